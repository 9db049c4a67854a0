"""Plans of adapters and the streams that read them."""

import pytest
import torch

from bridge_b200.models import AdapterSet, build_model, get_config
from bridge_b200.ops import adapter_linear, adapter_rows
from test_adapter_gpu import DEV, _inputs

pytestmark = pytest.mark.gpu


def _busy(stream):
    """Some 50 ms of waiting on a stream."""
    with torch.cuda.stream(stream):
        torch.cuda._sleep(100_000_000)


def _not_handed_out(table_ptr, like):
    return all(t.data_ptr() != table_ptr for t in [torch.empty(like, dtype=torch.int32, device=DEV) for _ in range(200)])


@pytest.mark.parametrize("t", [3, 40, 700])
@pytest.mark.parametrize("train", [False, True])
def test_a_plan_that_is_let_go_while_another_stream_reads_it(t, train):
    x, w, a, b, dy = _inputs(t, 512, 256, 3, 16, torch.bfloat16)
    cu, slots = [0, t // 3, t], [2, 0]
    with torch.no_grad():
        want = adapter_linear(x, w, a, b, adapter_rows(cu, slots, device=DEV))
    if train:
        a = a.clone().requires_grad_()
        # (the first backward of a process takes longer than the wait below)
        torch.autograd.grad(adapter_linear(x, w, a, b, adapter_rows(cu, slots, device=DEV)), (a,), dy)
    plan = adapter_rows(cu, slots, device=DEV)
    ptr, size = plan.table.data_ptr(), plan.table.numel()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    _busy(side)
    with torch.cuda.stream(side):
        y = adapter_linear(x, w, a, b, plan)
        if train:
            (da,) = torch.autograd.grad(y, (a,), dy)
        y = y.detach()
    del plan
    assert not side.query()
    assert _not_handed_out(ptr, size)
    torch.cuda.synchronize()
    assert torch.equal(y, want)


def test_plans_of_an_adapter_set():
    model = build_model(get_config("tiny"), seed=1, device=DEV)
    adapters = AdapterSet(model, slots=2, rank=8)
    p = adapters._modules_of[0]
    x = torch.randn(40, p.weight.shape[1], device=DEV, dtype=p.weight.dtype)
    side = torch.cuda.Stream()
    with torch.no_grad(), adapters.use(1):
        plan = adapters.rows_for(x)
        ptr, size = plan.table.data_ptr(), plan.table.numel()
        torch.cuda.synchronize()
        _busy(side)
        with torch.cuda.stream(side):
            p(x)
        del plan
        adapters._plans.clear()
        assert not side.query()
        assert _not_handed_out(ptr, size)
    torch.cuda.synchronize()
