"""What attention's kernels report to the host."""
import pytest
import torch

from attention_helpers import Problem, offsets
from sddmm_gpu_b200 import api

pytestmark = pytest.mark.gpu


def test_a_bad_index_and_a_wait_that_gave_up_are_both_reported(engine):
    p = Problem(torch.bfloat16, 64, 2, 2, [20, 30], window=(-1, 0))
    plan = p.plan(engine)
    p.q_offsets.copy_(offsets([20, 90]))
    plan.forward(p.Q, p.K, p.V, torch.empty_like(p.Q), flags=api.FLAG_ASYNC)
    got = [engine.selftest_wait_timeout()]
    for _ in range(2):
        try:
            engine.sync()
            got.append(api.OK)
        except api.SddmmError as e:
            got.append(e.status)
    assert got == [api.DEVICE_TIMEOUT, api.INDEX_OUT_OF_RANGE, api.OK]
    plan.close()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("max_q,max_k,backward", [(0, 8, False), (0, 0, False), (0, 8, True), (8, 0, True), (0, 0, True), (8, 0, False)])
def test_sequences_over_limits_of_zero_are_reported(engine, dtype, max_q, max_k, backward):
    p = Problem(dtype, 64, 2, 2, [5, 8], window=(-1, 0))
    plan = engine.attention_plan(dtype, 64, 2, 2, p.q_offsets, max_q, max_k, k_offsets=p.q_offsets, window=(-1, 0))
    O, l = torch.full_like(p.Q, 7.25), torch.full((2, 13), 7.25, device="cuda")
    grads = [torch.full_like(t, 7.25) for t in (p.Q, p.K, p.V)]
    with pytest.raises(api.SddmmError) as e:
        plan.backward(p.Q, p.K, p.V, O, l, p.dO, *grads) if backward else plan.forward(p.Q, p.K, p.V, O, l)
    assert e.value.status == api.INDEX_OUT_OF_RANGE
    assert all(bool((t == 7.25).all()) for t in (O, l, *grads))
    p.q_offsets.zero_()
    plan.forward(p.Q, p.K, p.V, O, l)
    plan.backward(p.Q, p.K, p.V, O, l, p.dO, *grads)
    assert all(bool((t == 7.25).all()) for t in (O, l, *grads))
    plan.close()
