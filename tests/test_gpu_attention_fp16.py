"""fp16 gradients of attention: as exact for small and large upstream gradients as for those of order one.

Gradients are linear in dO, and a power of two moves no bit of an fp16 value that stays normal: with dO times 2^e every gradient
has to be 2^e times as large, but for its own rounding where it is subnormal, 2^-25 (and, of the one at order one, half a step of its own).
"""
import pytest
import torch

from attention_helpers import Problem, within

pytestmark = pytest.mark.gpu

F16 = torch.float16


def _gradients(plan, p, O, l, dO):
    grads = [torch.full_like(t, 7.25) for t in (p.Q, p.K, p.V)]
    plan.backward(p.Q, p.K, p.V, O, l, dO, *grads)
    return grads


def _problem(engine, d, hq, hkv, q, k=None, **mask):
    p = Problem(F16, d, hq, hkv, q, k, **mask)
    # 2^-4 at least, so that 2^-10 of it is normal
    p.dO = torch.where(p.dO.abs() < 2.0 ** -4, torch.copysign(torch.full_like(p.dO, 2.0 ** -4), p.dO), p.dO)
    plan = p.plan(engine)
    O, l = torch.empty_like(p.Q), torch.empty((p.hq, p.q_rows), device="cuda")
    plan.forward(p.Q, p.K, p.V, O, l)
    return p, plan, O, l


def _scaled(first, second, by, what):
    # half a step of the first, rounded at its own size; of the second where it is subnormal
    tol = first.double().abs() * by * 2.0 ** -11 + 2.0 ** -25 * (1 + by)
    tol = torch.where(second.double().abs() >= 2.0 ** -13, torch.where(first.double().abs() >= 2.0 ** -13, 0.0, tol), tol)
    within(second, first.double() * by, tol, what)


SHAPES = [(64, 4, 2, [700, 130, 2048], None, dict(window=(-1, 0))), (128, 4, 4, [1500], None, dict(window=(-1, 0), cap=20.0)),
          (128, 2, 1, [300, 33], [900, 400], dict(window=(200, 0), prefix=40, bias=True)), (80, 6, 2, [129, 1, 64], None, dict()),
          (64, 1, 1, [2500], None, dict(window=(256, 256), prefix=20))]


@pytest.mark.parametrize("e", [-10, -9, -5, 3, 9])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_small_and_large_upstream_gradients(engine, shape, e):
    d, hq, hkv, q, k, mask = SHAPES[shape]
    p, plan, O, l = _problem(engine, d, hq, hkv, q, k, **mask)
    first = _gradients(plan, p, O, l, p.dO)
    dO = (p.dO.double() * 2.0 ** e).to(F16)
    assert bool((dO.double() == p.dO.double() * 2.0 ** e).all())
    for a, b, what in zip(first, _gradients(plan, p, O, l, dO), ("dQ", "dK", "dV")):
        _scaled(a, b, 2.0 ** e, what)
    for got, x, t, what in zip(first, *p.backward(), ("dQ", "dK", "dV")):
        within(got, x, t, what)
    plan.close()


def test_rows_of_different_sizes(engine):
    # every row of dQ by its own power of two, whatever the others are
    p, plan, O, l = _problem(engine, 64, 4, 2, [500, 70], window=(-1, 0))
    first = _gradients(plan, p, O, l, p.dO)
    by = torch.tensor([2.0 ** -(r % 11) for r in range(p.q_rows)], dtype=torch.float64, device="cuda")[:, None, None]   # exact
    second = _gradients(plan, p, O, l, (p.dO.double() * by).to(F16))
    tol = torch.where((second[0].double().abs() >= 2.0 ** -13) & (first[0].double().abs() >= 2.0 ** -13), 0.0, first[0].double().abs() * by * 2.0 ** -11 + 2.0 ** -25 * (1 + by))
    within(second[0], first[0].double() * by, tol, "dQ")
    p.dO = (p.dO.double() * by).to(F16)
    for got, x, t, what in zip(second, *p.backward(), ("dQ", "dK", "dV")):
        within(got, x, t, what)
    plan.close()


@pytest.mark.parametrize("value", [float("nan"), float("inf"), 65504.0])
def test_a_sequence_with_anything_next_to_a_small_one(engine, value):
    p, plan, O, l = _problem(engine, 64, 2, 2, [200, 60], window=(-1, 0))
    first = _gradients(plan, p, O, l, p.dO)
    dO = (p.dO.double() * 2.0 ** -10).to(F16)
    dO[200:] = value
    dO[100, 0, 5] = value if value != 65504.0 else dO[100, 0, 5]   # a row of the small one too: all gradients but its own and those of the keys that it sees
    second = _gradients(plan, p, O, l, dO)
    rows = [r for r in range(200) if r != 100]
    _scaled(first[0][rows], second[0][rows], 2.0 ** -10, "dQ")
    # keys whose tile meets what is not finite are computed anew, without rounded weights: as near to the definition as at order one
    want, tol = p.backward()
    for i, what in ((1, "dK"), (2, "dV")):
        within(second[i][101:200], want[i][101:200] * 2.0 ** -10, tol[i][101:200] * 2.0 ** -10 + 2.0 ** -25, what)
    plan.close()


def test_in_parts(engine):
    # few keys and many queries, and the other way round: blocks cut into parts, each with its own power of two
    for q, k in (([4000], [140]), ([140], [4000])):
        p, plan, O, l = _problem(engine, 64, 1, 1, q, k)
        first = _gradients(plan, p, O, l, p.dO)
        second = _gradients(plan, p, O, l, (p.dO.double() * 2.0 ** -10).to(F16))
        for a, b, what in zip(first, second, ("dQ", "dK", "dV")):
            _scaled(a, b, 2.0 ** -10, what)
        for got, x, t, what in zip(first, *p.backward(), ("dQ", "dK", "dV")):
            within(got, x, t, what)
        plan.close()


def test_no_gradient_at_all(engine):
    p, plan, O, l = _problem(engine, 64, 2, 2, [90, 200], window=(-1, 0))
    for g in _gradients(plan, p, O, l, torch.zeros_like(p.dO)):
        assert bool((g == 0).all())
    plan.close()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [60000, 200000])
def test_weights_of_many_keys(engine, d, n):
    # equal weights of 1 / n, below the least normal value of fp16
    nq = 70
    p = Problem(F16, d, 1, 1, [nq], [n])
    p.Q.zero_()
    p.dO.fill_(128.0)
    plan = p.plan(engine)
    O, l = torch.empty_like(p.Q), torch.empty((1, nq), device="cuda")
    plan.forward(p.Q, p.K, p.V, O, l)
    _, dK, dV = _gradients(plan, p, O, l, p.dO)
    assert plan.last_kernel_name() == "attention_backward_tc"
    # a weight: half a step, and exp (2^-19: its argument is of 2^5); dV: half a step, and where it is subnormal 2^-25
    within(dV, torch.full_like(dV, nq * 128.0 / n, dtype=torch.float64), nq * 128.0 / n * (2.0 ** -10 + 2.0 ** -18) + 2.0 ** -25, "dV")
    assert bool((dK == 0).all())
    plan.close()


def test_many_short_sequences(engine):
    # every tile of every sequence has a place of its own for its largest |dO|
    g = torch.Generator().manual_seed(5)
    q = [int(x) for x in torch.randint(0, 200, (150,), generator=g)]
    p, plan, O, l = _problem(engine, 64, 4, 2, q, window=(-1, 0))
    first = _gradients(plan, p, O, l, p.dO)
    # sequences of different sizes: each is exact by itself
    by = torch.cat([torch.full((n,), 2.0 ** -(b % 11), dtype=torch.float64) for b, n in enumerate(q)]).cuda()[:, None, None]
    second = _gradients(plan, p, O, l, (p.dO.double() * by).to(F16))
    for a, b, what in zip(first, second, ("dQ", "dK", "dV")):
        a = a.double() * by
        tol = torch.where((b.double().abs() >= 2.0 ** -13) & (a.abs() >= 2.0 ** -13 * by), 0.0, a.abs() * 2.0 ** -11 + 2.0 ** -25 * (1 + by))
        within(b, a, tol, what)
    plan.close()
