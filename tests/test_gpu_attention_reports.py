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
