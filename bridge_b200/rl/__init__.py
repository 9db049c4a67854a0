"""RL objectives over the token tree, and distillation from a teacher policy."""

from .distill import distill_loss, teacher_alternatives
from .objective import SegmentPPOObjectiveAdapter
