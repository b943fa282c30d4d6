"""Rotary positions on the GPU against their definition in 64 bits, and the run of rotation, cache and attention as a program has it."""
import math

import numpy as np
import pytest
import torch

from attention_helpers import HALF_STEP, Problem, within
from sddmm_gpu_b200 import api

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _turned(x, positions, f, layout, inverse, m):
    """Result and tolerance: half a step of the type; cos and sin (angle off by 2^-25 of pi, and 2 units of fp32), two products and a sum in fp32."""
    n = f.shape[0]
    x = x.double().cpu()
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if layout == "interleaved" else (x[..., :n], x[..., n:2 * n])
    two_pi = np.longdouble("6.283185307179586476925286766559005768")
    angle = torch.from_numpy((np.multiply.outer(positions.cpu().numpy().astype(np.longdouble), f.astype(np.longdouble)) % two_pi).astype(np.float64))
    c, s = angle.cos()[:, None] * m, angle.sin()[:, None] * m * (-1 if inverse else 1)
    u, w = a * c - b * s, b * c + a * s
    size = (a.abs() + b.abs()) * abs(m)
    y, t = x.clone(), torch.zeros_like(x)
    for part, val in ((0, u), (1, w)):
        at = (slice(part, 2 * n, 2) if layout == "interleaved" else slice(part * n, part * n + n))
        y[..., at], t[..., at] = val, size
    return y, t


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("d,rot", [(128, 128), (64, 48), (80, 20), (6, 6), (5, 2), (64, 0), (256, 256)])
@pytest.mark.parametrize("rows,hq,hkv", [(1, 4, 1), (37, 6, 3), (300, 17, 5)])
def test_rotation(engine, dtype, layout, d, rot, rows, hq, hkv):
    g = torch.Generator("cuda").manual_seed(rows + d)
    q, k = (torch.randn((rows, h, d), device="cuda", generator=g).to(dtype) for h in (hq, hkv))
    f = api.rotary_frequencies(rot, factor=4.0, original_len=256) if rot else np.zeros(0)
    positions = torch.randint(0, 1 << 20, (rows,), device="cuda", generator=g)
    for inverse, m in ((False, 1.0), (True, 1.25)):
        out = [torch.full_like(t, 7.25) for t in (q, k)]
        engine.rotary([api.RotaryPart(q, out[0]), api.RotaryPart(k, out[1])], positions, f, layout, inverse, m)
        for x, y in zip((q, k), out):
            want, size = _turned(x, positions, f, layout, inverse, m)
            tol = size * (math.pi * 2.0 ** -25 + 5 * 2.0 ** -24) + HALF_STEP[dtype] * want.abs() * (size > 0) + (2.0 ** -24 if dtype == torch.float16 else 1e-30)
            within(y.cpu(), want, tol)
        both = [t.clone() for t in (q, k)]                       # in place: the same bits
        engine.rotary([api.RotaryPart(t) for t in both], positions, f, layout, inverse, m)
        assert all(torch.equal(a, b) for a, b in zip(both, out))


def test_there_and_back(engine):
    x = torch.randn((500, 3, 64), device="cuda")
    f = api.rotary_frequencies(64)
    y, z = torch.empty_like(x), torch.empty_like(x)
    engine.rotary([api.RotaryPart(x, y)], 12345, f)
    engine.rotary([api.RotaryPart(y, z)], 12345, f, inverse=True)
    pair = x[..., :32].abs() + x[..., 32:].abs()
    # forth and back: three roundings of pairs each way, and each angle's 2^-25 of pi and 2^-23 of its sine
    within(z, x.double(), torch.cat([pair, pair], -1).double() * 16 * 2.0 ** -24)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_far_positions(engine, layout):
    rows = torch.tensor([0, 1, -1, (1 << 31) + 5, -(1 << 40), (1 << 53) + 1, 10 ** 12], device="cuda")
    f = np.array([1.0, 0.7, 2.0 ** -20, 1e-9])
    x = torch.randn((7, 2, 8), device="cuda")
    y = torch.empty_like(x)
    engine.rotary([api.RotaryPart(x, y)], rows, f, layout)
    # the angle as whole numbers: position * (f / 2 pi), f / 2 pi to 64 bits as the definition of the frequency's rounding
    two_pi = np.longdouble("6.283185307179586476925286766559005768")
    turns = [int(np.floor(np.longdouble(v) / two_pi * np.longdouble(2) ** 64)) for v in f]
    angle = np.array([[(int(r) * t % (1 << 64)) / 2.0 ** 64 * 2 * math.pi for t in turns] for r in rows.cpu()])
    a, b = (x[..., 0::2], x[..., 1::2]) if layout == "interleaved" else (x[..., :4], x[..., 4:])
    u, w = (y[..., 0::2], y[..., 1::2]) if layout == "interleaved" else (y[..., :4], y[..., 4:])
    c, s = (torch.from_numpy(v(angle))[:, None].cuda() for v in (np.cos, np.sin))
    size = (a.abs() + b.abs()).double() * (math.pi * 2.0 ** -25 + 5 * 2.0 ** -24)
    within(u, a.double() * c - b.double() * s, size)
    within(w, b.double() * c + a.double() * s, size)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_a_cache(engine, dtype):
    n, h, d = 40, 3, 64
    k, v = (torch.randn((n, h, d), device="cuda").to(dtype) for _ in range(2))
    rows = torch.randperm(500, device="cuda")[:n]
    rows[5] = -1
    cache = torch.full((2, 500, h, d), 7.25, device="cuda", dtype=dtype)
    f = api.rotary_frequencies(d)
    want = torch.empty_like(k)
    pos = torch.arange(n, device="cuda")
    engine.rotary([api.RotaryPart(k, want)], pos, f)
    engine.rotary([api.RotaryPart(k, cache[0], rows), api.RotaryPart(v, cache[1], rows, rotate=False)], pos, f)
    kept = rows >= 0
    assert torch.equal(cache[0][rows[kept]], want[kept]) and torch.equal(cache[1][rows[kept]], v[kept])
    others = torch.ones(500, dtype=torch.bool, device="cuda")
    others[rows[kept]] = False
    assert bool((cache[:, others] == 7.25).all())
    # a row outside the cache: left out, reported
    rows[7] = 500
    with pytest.raises(api.SddmmError) as e:
        engine.rotary([api.RotaryPart(k, cache[0], rows)], pos, f)
    assert e.value.status == api.INDEX_OUT_OF_RANGE


@pytest.mark.parametrize("dtype", TYPES)
def test_odd_strides(engine, dtype):
    x = torch.randn((30, 4 * 65 + 1), device="cuda").to(dtype)[:, 1:].unflatten(1, (4, 65))[..., :64]
    y = torch.empty((4, 30, 64), device="cuda", dtype=dtype).transpose(0, 1)
    z = torch.empty((30, 4, 64), device="cuda", dtype=dtype)
    f = api.rotary_frequencies(64)
    engine.rotary([api.RotaryPart(x, y), api.RotaryPart(x.contiguous(), z)], 3, f)
    assert torch.equal(y, z)


def test_refusals(engine):
    x = torch.randn((10, 2, 64), device="cuda")
    f = api.rotary_frequencies(64)
    for args, kw in [(([api.RotaryPart(x)], 0, api.rotary_frequencies(66)), {}), (([api.RotaryPart(x)], 0, np.full(32, np.nan)), {}),
                     (([api.RotaryPart(x)], 0, f), dict(magnitude=math.nan)), (([api.RotaryPart(x)], 0, f), dict(flags=4)),
                     (([api.RotaryPart(x, x[:, :1].expand(-1, 2, -1))], 0, f), {})]:
        with pytest.raises(api.SddmmError) as e:
            engine.rotary(*args, **kw)
        assert e.value.status == api.INVALID_ARG
    for args in [([], 0, f), ([api.RotaryPart(x)] * 5, 0, f), ([api.RotaryPart(x, x.half())], 0, f), ([api.RotaryPart(x, x.cpu())], 0, f),
                 ([api.RotaryPart(x, torch.empty((9, 2, 64), device="cuda"))], 0, f), ([api.RotaryPart(x)], torch.arange(9, device="cuda"), f),
                 ([api.RotaryPart(x)], torch.arange(10), f), ([api.RotaryPart(x), api.RotaryPart(x[:5])], 0, f),
                 ([api.RotaryPart(x, x, torch.arange(10, device="cuda", dtype=torch.int32))], 0, f)]:
        with pytest.raises(ValueError):
            engine.rotary(*args)
    with pytest.raises(ValueError):
        engine.rotary([api.RotaryPart(x)], 0, f, layout="other")
    y = x[:0]
    engine.rotary([api.RotaryPart(y)], torch.empty(0, dtype=torch.int64, device="cuda"), f)   # nothing to do


def test_prompt_then_tokens(engine):
    """As a program has it: a prompt is rotated into a cache and attended to, then tokens one by one, in a captured step; the whole
    sequence at once gives the same."""
    dtype, d, hq, hkv, n, extra, slot = torch.bfloat16, 64, 8, 2, [37, 150], 5, 256
    g = torch.Generator("cuda").manual_seed(4)
    total = [x + extra for x in n]
    qkv = [[torch.randn((t, h, d), device="cuda", generator=g).to(dtype) for h in (hq, hkv, hkv)] for t in total]
    f = api.rotary_frequencies(d)
    cache = torch.full((2, 2 * slot, hkv, d), float("nan"), device="cuda", dtype=dtype)
    k_offsets = torch.tensor([0, slot, 2 * slot], dtype=torch.int32, device="cuda")
    k_len = torch.tensor(n, dtype=torch.int32, device="cuda")

    def step(q, k, v, positions, rows, plan, O, flags=0):
        r = torch.empty_like(q)
        engine.rotary([api.RotaryPart(q, r), api.RotaryPart(k, cache[0], rows), api.RotaryPart(v, cache[1], rows, rotate=False)], positions, f,
                      flags=flags)
        plan.forward(r, cache[0], cache[1], O, flags=flags)

    def plan_of(counts):
        off = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device="cuda")
        return engine.attention_plan(dtype, d, hq, hkv, off, max(counts), slot, k_offsets=k_offsets, k_len=k_len, window=(100, 0), softcap=20.0)

    cat = lambda i, a, b: torch.cat([s[i][a(t):b(t)] for s, t in zip(qkv, range(2))])  # noqa: E731
    pos = torch.cat([torch.arange(x, device="cuda") for x in n])
    rows = torch.cat([torch.arange(x, device="cuda") + b * slot for b, x in enumerate(n)])
    prompt = plan_of(n)
    O = torch.empty((sum(n), hq, d), device="cuda", dtype=dtype)
    step(*(cat(i, lambda t: 0, lambda t: n[t]) for i in range(3)), pos, rows, prompt, O)
    outs = [list(O[:n[0]]), list(O[n[0]:])]
    token = plan_of([1, 1])
    q, k, v = (torch.empty((2, h, d), device="cuda", dtype=dtype) for h in (hq, hkv, hkv))
    at, to = torch.zeros(2, dtype=torch.int64, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    O1 = torch.empty((2, hq, d), device="cuda", dtype=dtype)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        at.copy_(k_len)
        to.copy_(k_len + k_offsets[:2])
        k_len.add_(1)
        step(q, k, v, at, to, token, O1, api.FLAG_ASYNC)
    for t in range(extra):
        for i, x in enumerate((q, k, v)):
            x.copy_(torch.stack([s[i][m + t] for s, m in zip(qkv, n)]))
        graph.replay()
        for b in range(2):
            outs[b].append(O1[b].clone())
    torch.cuda.synchronize()
    engine.sync()
    # the whole sequences at once, from rotated operands in 64 bits as the cache rounds them
    p = Problem(dtype, d, hq, hkv, total, window=(100, 0), cap=20.0)
    for b in range(2):
        first = sum(total[:b])
        r = slice(first, first + total[b])
        where = torch.arange(total[b], device="cuda")
        y = [torch.empty_like(x) for x in qkv[b][:2]]
        engine.rotary([api.RotaryPart(x, o) for x, o in zip(qkv[b], y)], where, f)
        p.Q[r], p.K[r], p.V[r] = y[0], y[1], qkv[b][2]
    o, _, tol, _ = p.forward()
    within(torch.stack(outs[0] + outs[1]), o, tol)
