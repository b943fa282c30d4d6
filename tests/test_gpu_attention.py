"""Attention under described masks on the GPU against its definition in 64 bits (tests/attention_helpers.py)."""
import ctypes as C
import math
import struct

import pytest
import torch

from attention_helpers import Problem, offsets, within
from sddmm_gpu_b200 import api

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
NAN = float("nan")


def _forward(engine, p, lse=True, **more):
    plan = p.plan(engine, **more)
    O = torch.full((p.q_rows, p.hq, p.d), 7.25, dtype=p.dtype, device="cuda")
    l = torch.full((p.hq, p.q_rows), 7.25, device="cuda") if lse else None
    plan.forward(p.Q, p.K, p.V, O, l)
    return plan, O, l


def _check_forward(engine, p):
    plan, O, l = _forward(engine, p)
    o, lse, tol_o, tol_l = p.forward()
    used = ~o[:, 0, 0].isnan()
    within(O[used], o[used], tol_o[used], "O")
    within(l[:, used], lse[:, used], tol_l[:, used], "lse")
    assert bool((O[~used] == 7.25).all()) and bool((l[:, ~used] == 7.25).all())  # rows of no sequence
    O2 = torch.empty_like(O)
    plan.forward(p.Q, p.K, p.V, O2)                                             # without lse: the same bits
    assert torch.equal(O2[used], O[used])
    return plan, O, l


def _check_backward(engine, p):
    plan, O, l = _check_forward(engine, p)
    dQ, dK, dV = (torch.full_like(t, 7.25) for t in (p.Q, p.K, p.V))
    plan.backward(p.Q, p.K, p.V, O, l, p.dO, dQ, dK, dV)
    want, tol = p.backward()
    used_q = torch.zeros(p.q_rows, dtype=torch.bool, device="cuda")
    used_k = torch.zeros(p.k_rows, dtype=torch.bool, device="cuda")
    for rows, keys, _, _ in p.sequences():
        used_q[rows], used_k[keys] = True, True
    for got, x, t, used, name in zip((dQ, dK, dV), want, tol, (used_q, used_k, used_k), ("dQ", "dK", "dV")):
        within(got[used], x[used], t[used], name)
        assert bool((got[~used] == 7.25).all()), name
    again = [torch.empty_like(t) for t in (p.Q, p.K, p.V)]
    plan.backward(p.Q, p.K, p.V, O, l, p.dO, *again)
    assert all(torch.equal(a[u], b[u]) for a, b, u in zip(again, (dQ, dK, dV), (used_q, used_k, used_k)))
    return plan


def _array(address, row_stride, head_stride):
    return C.create_string_buffer(struct.pack("@Pqq", address, row_stride, head_stride))   # sddmm_head_array


MASKS = [dict(), dict(window=(-1, 0)), dict(window=(37, 0)), dict(window=(20, 50), prefix=9), dict(window=(-1, 0), prefix=70, cap=5.0),
         dict(window=(-1, 3), bias=True), dict(window=(130, 0), prefix=1, cap=3.0, bias=True), dict(window=(0, 0), prefix=0)]


@pytest.mark.parametrize("mask", range(len(MASKS)))
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d,hq,hkv", [(64, 4, 2), (128, 3, 3), (80, 4, 1), (8, 2, 2)])
def test_ragged_batch(engine, dtype, d, hq, hkv, mask):
    p = Problem(dtype, d, hq, hkv, [130, 1, 0, 64, 257, 3], seed=mask, extra_rows=5, gain=2.0, **MASKS[mask])
    _check_backward(engine, p).close()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("mask", range(len(MASKS)))
def test_queries_and_keys_of_other_lengths(engine, dtype, mask):
    # more keys than queries, more queries than keys (rows that see nothing under a causal mask), none of one or the other
    p = Problem(dtype, 64, 4, 2, [5, 140, 33, 0, 9, 200, 1], [300, 150, 7, 12, 0, 129, 1], seed=mask, **MASKS[mask])
    _check_backward(engine, p).close()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d,hq,hkv", [(64, 8, 2), (128, 4, 4), (128, 16, 1), (96, 32, 4)])
@pytest.mark.parametrize("mask", [0, 1, 3, 6])
def test_single_tokens_over_slots(engine, dtype, d, hq, hkv, mask):
    p = Problem(dtype, d, hq, hkv, [1] * 9, [1, 700, 64, 65, 2, 0, 1301, 128, 1000], slot=1310, seed=mask, **MASKS[mask])
    junk = torch.ones(p.k_rows, dtype=torch.bool, device="cuda")
    for _, keys, _, _ in p.sequences():
        junk[keys] = False
    p.K[junk], p.V[junk] = NAN, NAN   # what lies behind a slot's length does not matter
    _check_forward(engine, p)[0].close()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("d", [64, 128])
def test_gradients_of_slots(engine, dtype, d):
    # keys in slots that are not full: rows behind their length keep what they hold
    p = Problem(dtype, d, 4, 2, [30, 1, 200, 0], [50, 300, 260, 7], slot=301, window=(-1, 0), bias=True)
    _check_backward(engine, p).close()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("cap", [0.05, 0.7, 200.0, 3000.0, 1e5, 1e9])
@pytest.mark.parametrize("q,k", [([40, 200], [90, 200]), ([1, 1], [700, 33])])
def test_caps_small_and_large(engine, dtype, cap, q, k):
    p = Problem(dtype, 64, 4, 2, q, k, window=(-1, 0), cap=cap, gain=3.0)
    _check_backward(engine, p).close()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("cap", [1e-4, 1e-9, 1e-38])
@pytest.mark.parametrize("q,k", [([40, 200], [90, 200]), ([1, 1], [700, 33])])
def test_caps_next_to_nothing(engine, dtype, cap, q, k):
    # all scores are +-cap, and 0 where the product is: equal weights
    p = Problem(dtype, 64, 4, 2, q, k, window=(-1, 0), cap=cap)
    p.Q[0] = 0
    _check_forward(engine, p)[0].close()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_sequences(engine, dtype):
    g = torch.Generator().manual_seed(2)
    q = [int(x) for x in torch.randint(0, 30, (300,), generator=g)]
    p = Problem(dtype, 64, 2, 1, q, window=(-1, 0))
    _check_backward(engine, p).close()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("q,k,heads", [([700], [6000], 1), ([300, 20], [5000, 2100], 2), ([256], [4096], 2)])
def test_keys_in_parts(engine, dtype, q, k, heads):
    # too few blocks for the GPU: the keys of each are cut
    p = Problem(dtype, 128, heads, 1, q, k, window=(3000, 0), prefix=70, gain=2.0)
    plan, _, _ = _check_forward(engine, p)
    assert plan.last_kernel_name() in ("attention_tc", "attention_few_tc")
    plan.close()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("q", [1, 300])
def test_offsets_past_32_bits(engine, dtype, q):
    # rows 80,000 elements apart: the last ones lie beyond 2^31 elements and 2^32 bytes
    rows, stride = 27_000, 80_000
    p = Problem(dtype, 64, 2, 2, [q], [700], window=(-1, 0))
    K = torch.empty(rows * stride, dtype=dtype, device="cuda").view(rows, stride)[:, :128].unflatten(1, (2, 64))
    K[rows - 700:] = p.K
    plan = engine.attention_plan(dtype, 64, 2, 2, offsets([q]), q, 700, k_offsets=torch.tensor([rows - 700, rows], dtype=torch.int32, device="cuda"),
                                 window=(-1, 0), k_rows=rows)
    O = torch.empty_like(p.Q)
    plan.forward(p.Q, K, K, O)
    p.V = p.K
    o, _, tol, _ = p.forward()
    within(O, o, tol)
    plan.close()


def test_few_and_prompt_kernels_behind_other_work(engine):
    # what runs next on the stream finds all results, also of calls whose rows all have one part
    p = Problem(BF16, 128, 8, 8, [1] * 4, [5, 30, 17, 9], slot=8192, window=(-1, 0))
    plan = engine.attention_plan(BF16, 128, 8, 8, p.q_offsets, 1, 8192, k_offsets=p.k_offsets, k_len=p.k_len, window=(-1, 0), k_rows=p.k_rows)
    o, _, tol, _ = p.forward()
    for _ in range(50):
        O = torch.zeros_like(p.Q)
        plan.forward(p.Q, p.K, p.V, O, flags=api.FLAG_ASYNC)
        out = O + 0
        within(out, o, tol)
    plan.close()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("q,k", [([1], [9001]), ([3], [5000]), ([17, 2], [4100, 2500]), ([200], [3000])])
def test_few_queries_many_keys(engine, dtype, q, k):
    p = Problem(dtype, 128, 8, 2, q, k, window=(-1, 0), cap=30.0, gain=3.0)
    _check_forward(engine, p)[0].close()


@pytest.mark.parametrize("mask", range(len(MASKS)))
@pytest.mark.parametrize("d,hq,hkv,q,k", [(128, 8, 1, [1], [5000]), (8, 7, 7, [1, 2, 5], [900, 17, 2]), (72, 6, 2, [3, 0, 1], [4000, 90, 2100]),
                                          (64, 4, 4, [19], [3001])])
def test_few_queries_in_fp32(engine, d, hq, hkv, q, k, mask):
    p = Problem(F32, d, hq, hkv, q, k, seed=mask + 1, gain=2.0, **MASKS[mask])
    plan, _, _ = _check_forward(engine, p)
    if mask == 0 and k[0] > 3000:
        assert plan.last_kernel_name() == "attention_few_f32"
    plan.close()


@pytest.mark.parametrize("mask", range(len(MASKS)))
@pytest.mark.parametrize("d,hq,hkv,q,k", [(64, 4, 2, [200, 64, 0, 129], [1500, 900, 7, 129]), (104, 2, 1, [400], [1100]), (128, 2, 2, [65, 300], [600, 300])])
def test_keys_in_parts_in_fp32(engine, d, hq, hkv, q, k, mask):
    p = Problem(F32, d, hq, hkv, q, k, seed=mask + 1, gain=2.0, extra_rows=3, **MASKS[mask])
    plan, _, _ = _check_forward(engine, p)
    assert plan.last_kernel_name() == "attention_general" and plan._bytes[0] > 0
    plan.close()


@pytest.mark.parametrize("value", [NAN, math.inf, -math.inf])
def test_keys_in_parts_in_fp32_masked_places(engine, value):
    p = Problem(F32, 64, 4, 2, [200], [1500], window=(300, 0), prefix=5)
    o, lse, tol_o, tol_l = p.forward()
    for x in (p.K, p.V):
        x[5:1000] = value                  # hidden from all
        x[1499] = value                    # seen by the last row alone
    plan, O, l = _forward(engine, p)
    assert plan.last_kernel_name() == "attention_general" and plan._bytes[0] > 0
    within(O[:199], o[:199], tol_o[:199], "O")
    within(l[:, :199], lse[:, :199], tol_l[:, :199], "lse")
    assert not bool(O[199].isfinite().all())
    plan.close()


@pytest.mark.parametrize("value", [NAN, math.inf, -math.inf])
def test_few_queries_in_fp32_masked_places(engine, value):
    p = Problem(F32, 64, 4, 2, [1, 2], [3000, 2500], window=(700, 0), prefix=5)
    o, lse, tol_o, tol_l = p.forward()
    for x in (p.K, p.V):
        x[5:2298] = value                  # of the first sequence, hidden
        x[5499] = value                    # seen by the last row alone
    plan, O, l = _forward(engine, p)
    within(O[:2], o[:2], tol_o[:2], "O")
    within(l[:, :2], lse[:, :2], tol_l[:, :2], "lse")
    assert not bool(O[2].isfinite().all())
    plan.close()


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_long_band_with_global_tokens(engine, dtype):
    p = Problem(dtype, 64, 2, 2, [2300], window=(256, 256), prefix=80, gain=2.0)
    _check_backward(engine, p).close()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d,q,window,prefix,cap", [(64, [2300], (256, 256), 80, 0.0), (128, [900, 130, 1500], (-1, 0), 0, 0.0),
                                                   (128, [1, 700, 64], (90, 0), 7, 20.0), (64, [640] * 6, (-1, -1), 0, 0.0)])
def test_the_same_bits_every_time(engine, dtype, d, q, window, prefix, cap):
    # warps that run ahead of one another do so differently every time
    p = Problem(dtype, d, 4, 2, q, window=window, prefix=prefix, cap=cap)
    plan, O, l = _forward(engine, p)
    first = [torch.empty_like(t) for t in (p.Q, p.K, p.V)]
    plan.backward(p.Q, p.K, p.V, O, l, p.dO, *first)
    O2, l2, again = torch.empty_like(O), torch.empty_like(l), [torch.empty_like(t) for t in first]
    for _ in range(60):
        plan.forward(p.Q, p.K, p.V, O2, l2)
        plan.backward(p.Q, p.K, p.V, O, l, p.dO, *again)
        assert torch.equal(O, O2) and torch.equal(l, l2) and all(torch.equal(a, b) for a, b in zip(first, again))
    plan.close()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_scores_far_apart(engine, dtype):
    # weights that are nearly one-hot, maxima that move along the row
    p = Problem(dtype, 64, 2, 1, [300, 77], window=(-1, 0), gain=20.0)
    _check_backward(engine, p).close()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("layout", ["heads first", "fused", "odd"])
def test_strides(engine, dtype, layout):
    p = Problem(dtype, 64, 4, 4, [70, 129], window=(-1, 0), bias=True)
    want = _forward(engine, p)
    plan, O, l = want
    grads = [torch.empty_like(t) for t in (p.Q, p.K, p.V)]
    plan.backward(p.Q, p.K, p.V, O, l, p.dO, *grads)

    def place(t):
        if layout == "heads first":
            x = torch.empty((t.shape[1], t.shape[0], t.shape[2]), dtype=dtype, device="cuda").transpose(0, 1)
        elif layout == "fused":
            x = torch.empty((t.shape[0], 3 * t.shape[1], t.shape[2]), dtype=dtype, device="cuda")[:, t.shape[1]:2 * t.shape[1]]
        else:
            x = torch.empty((t.shape[0], t.shape[1] * (t.shape[2] + 1) + 1), dtype=dtype, device="cuda")[:, 1:].unflatten(1, (t.shape[1], -1))[..., :t.shape[2]]
        return x.copy_(t)

    Q, K, V, dO, O2 = place(p.Q), place(p.K), place(p.V), place(p.dO), place(torch.zeros_like(O))
    l2 = torch.empty_like(l)
    plan.forward(Q, K, V, O2, l2)
    o, lse, tol_o, tol_l = p.forward()
    within(O2, o, tol_o, "O")
    within(l2, lse, tol_l, "lse")
    out = [place(torch.zeros_like(t)) for t in (p.Q, p.K, p.V)]
    plan.backward(Q, K, V, O2, l2, dO, *out)
    for got, x, t in zip(out, *p.backward()):
        within(got, x, t)
    plan.close()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_repeated_heads(engine, dtype):
    # stride 0: one K and V for all heads, as an expanded tensor
    p = Problem(dtype, 64, 4, 4, [90], window=(-1, 0))
    p.K, p.V = p.K[:, :1].expand(-1, 4, -1), p.V[:, :1].expand(-1, 4, -1)
    plan, O, _ = _forward(engine, p)
    o, _, tol, _ = p.forward()
    within(O, o, tol)
    with pytest.raises(api.SddmmError):  # but not for what is written
        plan.forward(p.Q, p.K, p.V, torch.empty((90, 1, 64), dtype=dtype, device="cuda").expand(-1, 4, -1))
    plan.close()


@pytest.mark.parametrize("value", [NAN, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("q", [[200], [1], [2, 1]])
def test_masked_places_hold_anything(engine, dtype, value, q):
    # a key that a row does not see: nothing of it reaches that row, forward or backward
    k = [x + 60 for x in q]
    p = Problem(dtype, 64, 4, 2, q, k, window=(40, 0))
    clean_o, clean_l, tol_o, tol_l = p.forward()
    K, V = p.K.clone(), p.V.clone()
    last = sum(k) - 1
    first_hidden = 15                      # of the first sequence, no row sees it: 40 behind the first query's position is 20
    for x in (K, V):
        x[first_hidden] = value
        x[last] = value                    # seen by the last row alone
    plan = p.plan(engine)
    O, l = torch.empty_like(p.Q), torch.empty((p.hq, p.q_rows), device="cuda")
    plan.forward(p.Q, K, V, O, l)
    keep = slice(0, p.q_rows - 1)
    within(O[keep], clean_o[keep], tol_o[keep], "O")
    within(l[:, keep], clean_l[:, keep], tol_l[:, keep], "lse")
    # backward: the last row's gradient in masked places too
    dO = p.dO.clone()
    grads = [torch.empty_like(t) for t in (p.Q, p.K, p.V)]
    plan.forward(p.Q, p.K, p.V, O, l)
    V2 = p.V.clone()
    V2[first_hidden], K2 = value, p.K.clone()
    K2[first_hidden] = value
    plan.backward(p.Q, K2, V2, O, l, dO, *grads)
    for got, x, t in zip(grads, *p.backward()):
        within(got, x, t)
    if len(q) == 1 and q[0] > 1:
        # a query that holds anything reaches the keys that it sees alone: 40 behind the last key
        Q2 = p.Q.clone()
        Q2[-1] = value
        dO[-1] = value
        plan.backward(Q2, p.K, p.V, O, l, dO, *grads)
        (_, dK, dV), (_, tK, tV) = p.backward()
        seen = slice(0, k[0] - 41)
        within(grads[1][seen], dK[seen], tK[seen], "dK")
        within(grads[2][seen], dV[seen], tV[seen], "dV")
        within(grads[0][:-1], p.backward()[0][0][:-1], p.backward()[1][0][:-1], "dQ")
    plan.close()


def test_gradients_against_differences(engine):
    p = Problem(F32, 8, 2, 1, [9, 4], window=(-1, 1), prefix=2, cap=4.0, bias=True, gain=2.0)
    plan, O, l = _forward(engine, p)
    grads = [torch.empty_like(t) for t in (p.Q, p.K, p.V)]
    plan.backward(p.Q, p.K, p.V, O, l, p.dO, *grads)
    arrays = dict(Q=p.Q.double(), K=p.K.double(), V=p.V.double())

    def loss():
        return float((p.forward(**arrays)[0] * p.dO.double()).sum())

    g = torch.Generator().manual_seed(3)
    for name, grad in zip("QKV", grads):
        x = arrays[name]
        for _ in range(6):
            at = tuple(int(torch.randint(0, n, (1,), generator=g)) for n in x.shape)
            was, step = float(x[at]), 1e-4
            x[at] = was + step
            up = loss()
            x[at] = was - step
            slope = (up - loss()) / (2 * step)
            x[at] = was
            # differences: their own error is of step^2 times third derivatives (below 1e-6 here); gradients of fp32 as in the helper
            assert abs(float(grad[at]) - slope) <= 1e-5 * max(1.0, abs(slope)), (name, at)
    plan.close()


def test_streams_and_graphs(engine):
    p = Problem(BF16, 64, 8, 2, [1] * 3, [700, 30, 900], slot=1000, window=(-1, 0))
    plan = p.plan(engine)
    side = torch.cuda.Stream()
    O, l = torch.empty_like(p.Q), torch.empty((p.hq, p.q_rows), device="cuda")
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        q = p.Q.clone()
        plan.forward(q, p.K, p.V, O, l, flags=api.FLAG_ASYNC)
        out = O.clone()
    side.synchronize()
    o, _, tol, _ = p.forward()
    within(out, o, tol)
    # two captured calls of one plan, replayed in turn and at once; lengths change between replays
    graphs, outs = [], []
    for _ in range(2):
        outs.append(torch.zeros_like(p.Q))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            plan.forward(p.Q, p.K, p.V, outs[-1], flags=api.FLAG_ASYNC)
        graphs.append(g)
    p.k_counts = [1, 950, 333]
    p.k_len.copy_(torch.tensor(p.k_counts, dtype=torch.int32))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    # (the limits of the plan are those of its first lengths: 950 is over 900 and left out; 1 and 333 are followed)
    o, _, tol, _ = p.forward()
    for out in outs:
        within(out[[0, 2]], o[[0, 2]], tol[[0, 2]])
        assert torch.equal(out, outs[0])
    with pytest.raises(api.SddmmError) as e:
        engine.sync()
    assert e.value.status == api.INDEX_OUT_OF_RANGE
    plan.close()


def test_workspace_of_a_chosen_stream(engine):
    # a stream other than torch's current one: what the call gives back must not go to the current stream's next tensor
    p = Problem(BF16, 64, 8, 2, [1], [9000], window=(-1, 0))
    plan = p.plan(engine)
    assert plan._bytes[0] > 0
    side, seen, get = torch.cuda.Stream(), [], plan._workspace

    def watched(*a):
        w = get(*a)
        seen.append(w.data_ptr())
        return w

    plan._workspace = watched
    O = torch.empty_like(p.Q)
    torch.cuda.synchronize()
    try:
        engine.set_stream(side.cuda_stream)
        plan.forward(p.Q, p.K, p.V, O, flags=api.FLAG_ASYNC)
        assert torch.empty(plan._bytes[0], dtype=torch.uint8, device="cuda").data_ptr() != seen[0]
        engine.sync()
        o, _, tol, _ = p.forward()
        within(O, o, tol)
        engine.set_stream(0)
        with pytest.raises(ValueError):
            plan.forward(p.Q, p.K, p.V, O)
    finally:
        engine.set_stream(None)
    plan.close()


def test_backward_in_a_graph(engine):
    p = Problem(BF16, 64, 4, 2, [150, 40], window=(-1, 0))
    plan, O, l = _forward(engine, p)
    grads = [torch.empty_like(t) for t in (p.Q, p.K, p.V)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        plan.backward(p.Q, p.K, p.V, O, l, p.dO, *grads, flags=api.FLAG_ASYNC)
    p.Q.mul_(0.5)
    plan.forward(p.Q, p.K, p.V, O, l)
    g.replay()
    torch.cuda.synchronize()
    for got, x, t in zip(grads, *p.backward()):
        within(got, x, t)
    plan.close()


@pytest.mark.parametrize("which", ["q negative", "q behind", "q down", "q long", "k behind", "k long", "k over slot", "k negative"])
def test_bad_sequences_are_left_out_and_reported(engine, which):
    p = Problem(BF16, 64, 2, 2, [20, 30, 10], [25, 40, 12], slot=48, window=(-1, 0))
    plan = p.plan(engine)
    o, _, tol, _ = p.forward()
    offs, koffs, klen = [0, 20, 50, 60], [0, 48, 96, 144], [25, 40, 12]
    bad = 1
    if which == "q negative":
        offs[0], bad = -5, 0
    elif which == "q behind":
        offs[3], bad = 1 << 30, 2
    elif which == "q down":
        offs, bad = [0, 20, 15, 25], None
    elif which == "q long":
        offs = [0, 20, 60, 60]                  # 40 > max_q = 30
    elif which == "k behind":
        koffs[3], klen[2], bad = 1 << 30, 40, 2   # ends behind k_rows
        koffs[2] = 120
    elif which == "k long":
        klen[1] = 48                             # > max_k = 40
    elif which == "k over slot":
        koffs[2] = 80                            # 32 rows for 40 keys
    else:
        klen[1] = -1
    p.q_offsets.copy_(torch.tensor(offs, dtype=torch.int32))
    p.k_offsets.copy_(torch.tensor(koffs, dtype=torch.int32))
    p.k_len.copy_(torch.tensor(klen, dtype=torch.int32))
    O = torch.full_like(p.Q, 7.25)
    with pytest.raises(api.SddmmError) as e:
        plan.forward(p.Q, p.K, p.V, O)
    assert e.value.status == api.INDEX_OUT_OF_RANGE
    if bad is not None and which not in ("q long", "q negative", "k over slot", "k behind"):
        rows = [slice(0, 20), slice(20, 50), slice(50, 60)]
        for b in range(3):
            if b == bad:
                assert bool((O[rows[b]] == 7.25).all())
            else:
                within(O[rows[b]], o[rows[b]], tol[rows[b]])
    plan.close()


def test_refusals(engine):
    p = Problem(BF16, 64, 4, 2, [16], window=(-1, 0))
    for more, status in [(dict(head_dim=0), api.K_UNSUPPORTED), (dict(head_dim=60), api.K_UNSUPPORTED), (dict(head_dim=136), api.K_UNSUPPORTED),
                         (dict(q_heads=3), api.INVALID_ARG), (dict(q_heads=0), api.INVALID_ARG), (dict(scale=0.0), api.INVALID_ARG),
                         (dict(scale=NAN), api.INVALID_ARG), (dict(scale=-1.0), api.INVALID_ARG), (dict(softcap=-1.0), api.INVALID_ARG),
                         (dict(softcap=math.inf), api.INVALID_ARG), (dict(window=(-2, 0)), api.INVALID_ARG), (dict(max_q=-1), api.INVALID_ARG),
                         (dict(k_rows=7), api.INVALID_ARG), (dict(q_rows=1 << 30), api.INVALID_ARG),
                         (dict(k_len=offsets([])), api.INVALID_ARG)]:
        kw = dict(dtype=BF16, head_dim=64, q_heads=4, kv_heads=2, q_offsets=p.q_offsets, max_q=16, max_k=16)
        kw.update(more)
        with pytest.raises(api.SddmmError) as e:
            engine.attention_plan(**kw)
        assert e.value.status == status, more
    with pytest.raises(ValueError):
        engine.attention_plan(BF16, 64, 4, 2, p.q_offsets.long(), 16, 16)
    with pytest.raises(ValueError):
        engine.attention_plan(BF16, 64, 4, 2, p.q_offsets.cpu(), 16, 16)
    with pytest.raises(ValueError):
        engine.attention_plan(BF16, 64, 4, 2, p.q_offsets, 16, 16, slopes=torch.ones(3, device="cuda"))
    with pytest.raises(TypeError):
        engine.attention_plan(torch.float64, 64, 4, 2, p.q_offsets, 16, 16)
    plan = p.plan(engine)
    O = torch.empty_like(p.Q)
    for args in [(p.Q[:8], p.K, p.V, O), (p.Q, p.K.float(), p.V, O), (p.Q, p.K, p.V.cpu(), O), (p.Q, p.K, p.V, O[:, :2]),
                 (p.Q.transpose(1, 2).contiguous().transpose(1, 2), p.K, p.V, O)]:
        with pytest.raises(ValueError):
            plan.forward(*args)
    with pytest.raises(ValueError):
        plan.forward(p.Q, p.K, p.V, O, torch.empty((4, 8), device="cuda"))
    # at the C entry: host memory, no workspace, unknown flags
    q = _array(p.Q.data_ptr(), p.Q.stride(0), p.Q.stride(1))
    k = _array(p.K.data_ptr(), p.K.stride(0), p.K.stride(1))
    o = _array(O.data_ptr(), O.stride(0), O.stride(1))
    l = torch.empty((4, 16), device="cuda")
    L = api.lib()
    host = torch.empty_like(p.Q, device="cpu")
    bad = _array(host.data_ptr(), p.Q.stride(0), p.Q.stride(1))
    odd = _array(p.Q.data_ptr() + 1, p.Q.stride(0), p.Q.stride(1))
    back = _array(p.Q.data_ptr(), -p.Q.stride(0), p.Q.stride(1))
    tight = _array(O.data_ptr(), 64, 32)
    for args in [(bad, k, k, o), (odd, k, k, o), (back, k, k, o), (q, k, k, tight)]:
        assert L.sddmm_attention_forward(plan._a, *args, None, None, 0, 0) == api.INVALID_ARG
    assert L.sddmm_attention_forward(plan._a, q, k, k, o, None, None, 0, 2) == api.INVALID_ARG
    assert L.sddmm_attention_forward(plan._a, q, k, k, o, host.data_ptr(), None, 0, 0) == api.INVALID_ARG
    assert L.sddmm_attention_backward(plan._a, q, k, k, o, l.data_ptr(), o, q, k, k, None, 0, 0) == api.INVALID_ARG
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(api.SddmmError) as e:
            plan.forward(p.Q, p.K, p.V, O)   # a captured call that waits
    assert e.value.status == api.INVALID_ARG
    plan.close()


def test_refused_pointers(engine):
    p = Problem(F32, 64, 2, 2, [16], window=(-1, 0))
    plan = p.plan(engine)
    O, l = torch.empty_like(p.Q), torch.empty((2, 17), device="cuda")
    forward = api.lib().sddmm_attention_forward
    q, k, v, o = (_array(t.data_ptr(), t.stride(0), t.stride(1)) for t in (p.Q, p.K, p.V, O))
    w = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    assert forward(plan._a, q, k, v, o, l.data_ptr() + 2, w.data_ptr(), 1 << 20, 0) == api.INVALID_ARG  # not aligned
    for x in (q, k, v):
        assert forward(plan._a, q, k, v, x, None, w.data_ptr(), 1 << 20, 0) == api.INVALID_ARG          # written and read
    assert forward(plan._a, q, k, k, o, l.data_ptr(), w.data_ptr(), 1 << 20, 0) == api.OK               # K as V is fine
    grads = [torch.empty_like(p.Q) for _ in range(3)]
    dq, dk, dv = (_array(t.data_ptr(), t.stride(0), t.stride(1)) for t in grads)
    do = _array(p.dO.data_ptr(), p.dO.stride(0), p.dO.stride(1))
    for g in [(do, dk, dv), (dq, q, dv), (dq, dk, o), (dq, dq, dv), (dq, dk, dk), (dv, dk, dv)]:
        assert api.lib().sddmm_attention_backward(plan._a, q, k, v, o, l.data_ptr(), do, *g, w.data_ptr(), 1 << 20, 0) == api.INVALID_ARG
    assert api.lib().sddmm_attention_backward(plan._a, q, k, v, o, l.data_ptr(), do, dq, dk, dv, w.data_ptr(), 1 << 20, 0) == api.OK
    desc = api.AttentionDesc.from_buffer_copy(plan.desc)
    desc.q_offsets = p.q_offsets.data_ptr() + 1
    a = C.c_void_p()
    assert api.lib().sddmm_attention_plan(engine._h, C.byref(desc), C.byref(a)) == api.INVALID_ARG
    plan.close()


def test_nothing_to_do(engine):
    for q, k in [([], []), ([0], [5]), ([0, 0], [0, 0])]:
        p = Problem(BF16, 64, 2, 2, q, k)
        plan, O, l = _forward(engine, p)
        dQ, dK, dV = (torch.full_like(t, 7.25) for t in (p.Q, p.K, p.V))
        plan.backward(p.Q, p.K, p.V, O, l, p.dO, dQ, dK, dV)
        assert bool((dK == 0).all()) and bool((dV == 0).all())
        plan.close()
