"""Capped scores of attention on the GPU against their definition in 64 bits, with a tolerance that goes by the score and not by the cap.

A capped score is off by at most 2^-21 of its size, and so of min(cap, |score before the cap|), beside what its product is off by:
  cap tanhf(x / cap)                 scale, division, tanhf (2 units), product: 7 roundings, 7 x 2^-24
  cap y (polynomial in y^2)          the polynomial 9e-8 = 1.5 x 2^-24, its factors (cap / scale, cap log2 e, their product) 4, last two steps, the
                                     product: 8.5 x 2^-24, of which the product's own term below holds 8
  cap - 2 cap / (1 + e^2y), y > 0.6  in units of cap: e^2y 2^-22.5 of itself and 2^-24 by its argument, the sum, the reciprocal 2^-23, together
                                     2^-21.4 of the quotient (0.46 at most), and the last rounding: 2^-22.4 <= 2^-21 x 0.6
"""
import math

import pytest
import torch

from attention_helpers import Problem, within
from sddmm_gpu_b200 import api

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


class Capped(Problem):
    def scores(self, Q, K, h, rows, keys, seen, far):
        q, k = Q[rows, h].double(), K[keys, h // (self.hq // self.hkv)].double()
        raw = q @ k.T * self.scale
        size = (q.abs() @ k.abs().T) * self.scale
        t = torch.tanh(raw / self.cap)
        x, slope = self.cap * t, 1 - t * t
        if self.slopes is not None:
            x = x - self.slopes[h].double() * far
            size = size + self.slopes[h].double() * far
        x = torch.where(seen, x, -math.inf)
        # fp32 products and sums (d terms, then 8 roundings), and the cap; a moved product moves its capped score by no more
        moved = size * (self.d + 8) * 2.0 ** -24 + raw.abs().clamp(max=self.cap) * 2.0 ** -21
        wobble = torch.where(seen, moved, 0.0)
        top = wobble.max(1).values if seen.shape[1] else torch.zeros(seen.shape[0], device="cuda", dtype=torch.float64)
        return x, slope, top


def _check(engine, p, backward=True):
    plan = p.plan(engine)
    O, l = torch.empty_like(p.Q), torch.empty((p.hq, p.q_rows), device="cuda")
    plan.forward(p.Q, p.K, p.V, O, l)
    o, lse, tol_o, tol_l = p.forward()
    within(O, o, tol_o, "O")
    within(l, lse, tol_l, "lse")
    name = plan.last_kernel_name()
    if backward:
        grads = [torch.empty_like(t) for t in (p.Q, p.K, p.V)]
        plan.backward(p.Q, p.K, p.V, O, l, p.dO, *grads)
        for got, x, t, what in zip(grads, *p.backward(), ("dQ", "dK", "dV")):
            within(got, x, t, what)
    plan.close()
    return name


SHAPES = [([40, 200], [90, 200]), ([1, 1], [700, 33])]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("cap", [0.05, 0.7, 30.0, 3000.0, 1e5, 1e9])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("q,k", SHAPES)
def test_caps_small_and_large(engine, dtype, cap, bias, q, k):
    _check(engine, Capped(dtype, 64, 4, 2, q, k, window=(-1, 0), cap=cap, bias=bias, gain=3.0))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("cap", [5e-5, 5e-6, 1.5e-6, 1e-6, 5e-7, 2e-7, 1.3e-7])
@pytest.mark.parametrize("zero", ["Q", "K", "both"])
@pytest.mark.parametrize("q,k", SHAPES)
def test_products_of_zero_under_tiny_caps(engine, dtype, cap, zero, q, k):
    # equal weights, whatever the cap; the cap's slope is one
    p = Capped(dtype, 64, 4, 2, q, k, window=(-1, 0), cap=cap)
    if zero != "K":
        p.Q.zero_()
    if zero != "Q":
        p.K.zero_()
    _check(engine, p)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("scale,cap", [(1e-2, 1e4), (1e-3, 1e3), (2e-2, 1e3)])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("q,k", SHAPES)
def test_large_products_far_below_their_cap(engine, dtype, scale, cap, bias, q, k):
    # products of up to 40,000; scores of up to 400, far below the cap: as exact as without one
    p = Capped(dtype, 8, 4, 2, q, k, window=(-1, 0), cap=cap, scale=scale, bias=bias, gain=3000.0)
    name = _check(engine, p)
    assert dtype == F32 or name in ("attention_tc", "attention_few_tc")


# Products of a warp that all lie within the range of tanh's polynomial go the short way; one that does not must change nothing for the others.
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("d,hq,hkv", [(64, 4, 2), (128, 4, 4)])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("q,k", [([40, 200], [90, 230]), ([1, 1], [700, 33])])
def test_bits_do_not_depend_on_hidden_places(engine, dtype, d, hq, hkv, bias, q, k):
    p = Capped(dtype, d, hq, hkv, q, k, slot=720, window=(30, 0), cap=30.0, bias=bias)
    plan = p.plan(engine)

    def run():
        O, l = torch.empty_like(p.Q), torch.empty((hq, p.q_rows), device="cuda")
        plan.forward(p.Q, p.K, p.V, O, l)
        grads = [torch.zeros_like(t) for t in (p.Q, p.K, p.V)]
        plan.backward(p.Q, p.K, p.V, O, l, p.dO, *grads)
        return O, l, *grads

    first = run()
    hidden = torch.ones(p.k_rows, dtype=torch.bool, device="cuda")
    for _, keys, seen, _ in p.sequences():
        hidden[keys] = ~seen.any(0)
    assert int(hidden[:k[0]].sum()) > 10
    p.K[hidden] *= 100
    p.V[hidden] *= 100
    second = run()
    for a, b, what in zip(first, second, ("O", "lse", "dQ", "dK", "dV")):
        assert torch.equal(a, b), f"keys that nobody sees: {what}"   # (their own gradients are zero or not written)
    # another sequence's rows lie in the same tile
    p.Q[q[0]:] *= 100
    third = run()
    for a, b, what in zip(second, third, ("O", "lse", "dQ", "dK", "dV")):
        part = (slice(None), slice(0, q[0])) if what == "lse" else slice(0, 720 if what in ("dK", "dV") else q[0])
        assert torch.equal(a[part], b[part]), f"another sequence: {what}"
    plan.close()
