"""Attention on operands that hold infinities in places that are seen (a run that has diverged)."""
import math

import pytest
import torch

from attention_helpers import Problem, within

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
KINDS = [(F32, 64, [300, 40], None), (F16, 64, [300, 40], None), (BF16, 128, [600], None), (BF16, 128, [1, 1], [700, 33]), (F32, 64, [1], [3000]),
         (F16, 128, [300], [5000]), (F32, 64, [64], [2000])]


@pytest.mark.parametrize("value", [math.inf, -math.inf])
@pytest.mark.parametrize("kind", range(len(KINDS)))
def test_an_infinity_in_one_column_of_v(engine, kind, value):
    # that column is infinite where the key is seen, and a number elsewhere; the others keep their bits
    dtype, d, q, k = KINDS[kind]
    p = Problem(dtype, d, 2, 2, q, k, window=(-1, 0))
    plan = p.plan(engine)
    out = []
    for x in (0.0, value):
        p.V[5, :, 3] = x
        O, l = torch.empty_like(p.Q), torch.empty((2, p.q_rows), device="cuda")
        plan.forward(p.Q, p.K, p.V, O, l)
        out.append((O, l))
    (O, l), (O2, l2) = out
    assert torch.equal(l, l2)
    others = [c for c in range(d) if c != 3]
    assert torch.equal(O[..., others], O2[..., others])
    _, keys, seen, _ = next(iter(p.sequences()))
    sees = torch.zeros(p.q_rows, dtype=torch.bool, device="cuda")
    sees[:q[0]] = seen[:, 5]
    assert bool((O2[sees][..., 3] == value).all())
    o, _, tol, _ = p.forward(V=torch.where(p.V.isfinite(), p.V, 0.0))
    assert bool(((O2[~sees][..., 3].double() - o[~sees][..., 3]).abs() <= tol[~sees][..., 3]).all())
    plan.close()


@pytest.mark.parametrize("kind", [0, 1, 2])
def test_an_infinity_in_one_column_of_the_upstream_gradient(engine, kind):
    # dV: the column of the keys that the row sees; dK of the keys that it sees and its dQ are not finite
    dtype, d, q, k = KINDS[kind]
    p = Problem(dtype, d, 2, 2, q, k, window=(-1, 0))
    plan = p.plan(engine)
    O, l = torch.empty_like(p.Q), torch.empty((2, p.q_rows), device="cuda")
    plan.forward(p.Q, p.K, p.V, O, l)
    grads = [torch.empty_like(t) for t in (p.Q, p.K, p.V)]
    out = []
    for x in (0.0, math.inf):
        p.dO[200, :, 3] = x
        plan.backward(p.Q, p.K, p.V, O, l, p.dO, *grads)
        out.append([t.clone() for t in grads])
    (dq, dk, dv), (dq2, dk2, dv2) = out
    others = [c for c in range(d) if c != 3]
    assert bool((dv2[:201, :, 3] == math.inf).all()) and bool(dv2[:201][..., others].isfinite().all())
    # dP and delta of that row are infinite: their difference is infinite where the signs differ, else NaN
    assert not bool(dk2[:201].isfinite().any()) and not bool(dq2[200].isfinite().any())
    close = lambda a, b: bool(((a.double() - b.double()).abs() <= 2.0 ** -6 * b.double().abs().max()).all())  # noqa: E731  (computed anew: another order, unrounded weights)
    rest = [r for r in range(p.q_rows) if r != 200]
    assert close(dq2[rest], dq[rest]) and close(dk2[201:], dk[201:]) and close(dv2[201:], dv[201:])
    plan.close()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sums_that_run_over(engine, dtype):
    # values near the type's largest: the sum of weighted ones leaves fp32 before it is divided, the result does not
    p = Problem(dtype, 64, 2, 2, [200], window=(-1, 0))
    p.Q.zero_()
    p.V.fill_(3e38)
    plan = p.plan(engine)
    O = torch.empty_like(p.Q)
    plan.forward(p.Q, p.K, p.V, O)
    want = p.V[:200].double()
    # equal weights: n + 16 roundings, exp2's 2^-19, half a step of the type
    assert bool(((O.double() - want).abs() <= want * (2.0 ** -18 + 216 * 2.0 ** -24 + (2.0 ** -8 if dtype == BF16 else 0.0))).all())
    plan.close()


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d,q,k", [(64, [40], [30]), (128, [300, 140], [290, 100]), (64, [140], [100])])
def test_rows_that_see_nothing_have_no_gradient(engine, dtype, d, q, k, value):
    # their upstream gradient is not finite, and neither is a key that they do not see
    p = Problem(dtype, d, 2, 1, q, k, window=(-1, 0))
    plan = p.plan(engine)
    O, l = torch.empty_like(p.Q), torch.empty((2, p.q_rows), device="cuda")
    plan.forward(p.Q, p.K, p.V, O, l)
    nothing = torch.zeros(p.q_rows, dtype=torch.bool, device="cuda")
    for rows, _, seen, _ in p.sequences():
        nothing[rows] = ~seen.any(1)
    assert int(nothing.sum()) >= 10 and bool((l[:, nothing] == -math.inf).all())
    want, tol = p.backward()
    p.dO[nothing] = value
    p.K[k[0] - 1] = value              # seen by the last row of the first sequence alone
    dQ, dK, dV = (torch.full_like(t, 7.25) for t in (p.Q, p.K, p.V))
    plan.backward(p.Q, p.K, p.V, O, l, p.dO, dQ, dK, dV)
    assert bool((dQ[nothing] == 0).all())
    rest = torch.ones(p.q_rows, dtype=torch.bool, device="cuda")
    rest[q[0] - 1] = False
    keys = torch.ones(p.k_rows, dtype=torch.bool, device="cuda")
    keys[:k[0]] = False                # (the last row's score gradients are not numbers any more)
    within(dQ[rest], want[0][rest], tol[0][rest], "dQ")
    within(dK[keys], want[1][keys], tol[1][keys], "dK")
    within(dV[keys], want[2][keys], tol[2][keys], "dV")
    plan.close()
