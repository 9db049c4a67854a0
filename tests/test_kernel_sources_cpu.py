"""Rules that a kernel's source has to keep because no run can show that they hold: what the compiler may move, and what
orders a read of shared memory before the asynchronous copy that overwrites it."""

import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bridge_b200", "csrc")


def _sources():
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu*"))):
        with open(path) as f:
            yield os.path.basename(path), f.read()


def test_warp_collectives_in_assembly_are_volatile():
    """A statement that every lane of a warp has to reach may not be moved into a branch that only some lanes take."""
    seen = 0
    for name, text in _sources():
        for m in re.finditer(r"\basm(\s+volatile)?\s*\(((?:[^;\"]|\"(?:[^\"\\]|\\.)*\")*)\)\s*;", text):
            if re.search(r"\.sync\b", m.group(2)):
                seen += 1
                assert m.group(1), f"{name}: {' '.join(m.group(2).split())[:60]}"
    assert seen > 10


def test_slots_are_read_before_they_are_refilled():
    """Nothing but a barrier orders a lane's read of shared memory before the asynchronous copy into the same slot that
    it issues afterwards: reading a batch ends with one."""
    text = dict(_sources())["vocab_rows.cu"]
    body = re.search(r"void take\(Unit<T>\* u\) \{(.*?)\n  \}", text, re.S).group(1)
    assert body.rindex("__syncwarp()") > body.rindex("read<3>(")
    # and every read of a slot goes through it
    assert len(re.findall(r"\bread<\d>\(ring", text)) == len(re.findall(r"\bread<\d>\(ring", body)) == 4
