"""Attention under a described mask, its gradient, and rotary positions: the calls whose speed matters, on one GPU.

A case is one call ("op"):

  attention  Attention.forward: prompts (packed documents), prompts behind a history, single tokens over a cache
  gradient   Attention.backward of packed documents, from the forward pass's output and log-sum-exp
  rotary     Handle.rotary: rotation of Q and K, to arrays of their own or (K, and V unrotated) to rows of a cache

Attention cases: "q" and "k" list the sequences' query and key counts; query i of a sequence stands at position
k - q + i.  A key j is seen if it is among the first "prefix" keys or at most "left" behind and "right" ahead of the
query (-1: no limit).  score = cap tanh(q.k / (sqrt(d) cap)) - slope distance; "cap" 0 and "bias" False leave
these out.  "slot" > 0: keys and values lie in cache slots of that many rows, filled up to their count; else packed.

`own` chooses between the framework's calls and the operators' plain form in elementary torch operations.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# no case has more entries in its padded score array or more multiplications than the largest listed ones
MOST_SCORES = 1 << 30
MOST_FLOPS = 7.0e11


def _attention(name, op, type, d, hq, hkv, q, k=None, slot=0, left=-1, right=0, prefix=0, cap=0.0, bias=False):
    case = dict(op=op, type=type, d=d, hq=hq, hkv=hkv, q=q, k=k or q, slot=slot, left=left, right=right, prefix=prefix, cap=cap,
                bias=bias)
    return dict(case, name=name) if name else case


def _rotary(name, type, d, rot, hq, hkv, tokens, layout, inverse=False, factor=1.0, far=0, cache=0):
    case = dict(op="rotary", type=type, d=d, rot=rot, hq=hq, hkv=hkv, tokens=tokens, layout=layout, inverse=inverse, factor=factor,
                far=far, cache=cache)
    return dict(case, name=name) if name else case


def listed():
    return [
        # a user's short question behind a conversation that the cache holds: the call's own cost counts
        _attention("question_48", "attention", "bf16", 64, 8, 2, "48", "311", slot=512),
        # a batch of prompts of different lengths, packed, scores capped
        _attention("prompts_ragged_cap", "attention", "bf16", 128, 16, 4, "1021 77 2048 1 640 1500 333 2111", cap=30.0),
        # one long prompt
        _attention("prompt_8k", "attention", "bf16", 128, 16, 16, "8192"),
        # the band with global tokens of the sparse-attention benchmark, on the first of its tokens
        _attention("band_16k", "attention", "f16", 64, 4, 4, "16384", left=256, right=256, prefix=80),
        # fp32, the framework's own type: text that sees its whole prefix, scores that fall with distance
        _attention("prefix_f32", "attention", "f32", 64, 8, 8, "1900 1333", prefix=500, bias=True),
        # single tokens: one long document
        _attention("token_33k", "attention", "bf16", 128, 32, 8, "1", "32801", slot=32896),
        # single tokens of a batch, lengths of all kinds, distance bias
        _attention("tokens_24", "attention", "f16", 64, 32, 4, " ".join(["1"] * 24),
                   "9000 17 4097 1 2222 812 16001 5120 64 3003 12345 700 129 7777 1024 6001 40 2500 15000 350 8191 1900 511 4400",
                   slot=16384, bias=True),
        # training on packed documents with capped scores, grouped heads
        _attention("gradient_ragged_cap", "gradient", "bf16", 128, 16, 4, "1500 900 33 2048 411 1204", cap=50.0),
        # training on one long document
        _attention("gradient_8k", "gradient", "bf16", 128, 8, 8, "8192"),
        # training in the framework's own type: a prefix that is seen whole, distance bias, a head of 80
        _attention("gradient_f32", "gradient", "f32", 80, 4, 2, "701 950", prefix=200, bias=True),
        # new tokens of a batch: rotated and stored in the cache, interleaved pairs, three quarters of the head
        _rotary("rotary_cache_48", "f16", 128, 96, 16, 4, 48, "interleaved", cache=8192),
        # gradient of the rotation of a training batch, frequencies scaled for a long context
        _rotary("rotary_inverse_32k", "bf16", 128, 128, 32, 8, 32768, "half", inverse=True, factor=8.0, far=100000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _fits(case):
    q, k = _lengths(case)
    return len(q) * case["hq"] * max(q) * max(k) <= MOST_SCORES and work(case)["flops"] <= MOST_FLOPS


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "history", "token", "token", "gradient", "gradient", "rotary"])
    if kind == "rotary":
        d = rng.choice([64, 80, 128])
        cache = rng.random() < 0.5
        return _rotary(None, rng.choice(list(TYPES)), d, rng.choice([d, d // 2, d * 3 // 4 // 2 * 2]), rng.choice([4, 8, 16, 32]),
                       rng.choice([1, 2, 4]), _log(rng, 1, 512 if cache else 32768), rng.choice(["half", "interleaved"]),
                       not cache and rng.random() < 0.5, rng.choice([1.0, 4.0, 8.0]), rng.choice([0, 1000, 100000]),
                       8192 if cache else 0)
    while True:
        type = "f32" if rng.random() < 0.15 else rng.choice(["f16", "bf16"])
        most = 2500 if type == "f32" else 8192
        group = rng.choice([1, 2, 4, 8])
        hkv = rng.choice([1, 2, 4, 8])
        mask = rng.choice([(-1, 0), (-1, 0), (-1, -1), (256, 256), (_log(rng, 16, 2000), 0)])
        more = dict(left=mask[0], right=mask[1], prefix=rng.choice([0, 0, _log(rng, 1, 600)]), cap=rng.choice([0.0, 0.0, 30.0, 50.0]),
                    bias=rng.random() < 0.3)
        d = rng.choice([64, 128, 64, 128, 80, 96])
        if kind == "token":
            n = _log(rng, 1, 32)
            k = [_log(rng, 1, 33000 if n <= 4 else 16000) for _ in range(n)]
            case = _attention(None, "attention", type, d, hkv * group, hkv, " ".join(["1"] * n), " ".join(map(str, k)),
                              slot=max(k) + rng.randrange(0, 100), **more)
        else:
            n = _log(rng, 1, 8)
            q = [_log(rng, 1, most / n ** 0.5) for _ in range(n)]
            if kind == "history":
                k = [x + _log(rng, 1, 4000) for x in q]
                case = _attention(None, "attention", type, d, hkv * group, hkv, " ".join(map(str, q)), " ".join(map(str, k)),
                                  slot=max(k) + rng.randrange(0, 100), **more)
            else:
                case = _attention(None, "gradient" if kind == "gradient" else "attention", type, d, hkv * group, hkv,
                                  " ".join(map(str, q)), **more)
        if _fits(case):
            return case


# ---- inputs ----------------------------------------------------------------------------------------------------------


def _lengths(case):
    return [int(x) for x in case["q"].split()], [int(x) for x in case["k"].split()]


def _frequencies(case):
    """Radians a position of every pair: base 10000; a factor > 1 slows the pairs that turn less than once in 4096 positions by it,
    leaves those of over 32 turns, and goes linearly between."""
    f = 10000.0 ** (-np.arange(0, case["rot"], 2, dtype=np.float64) / case["rot"])
    kept = np.clip((4096 * f / (2 * np.pi) - 1) / 31, 0, 1)
    return f * (kept + (1 - kept) / case["factor"])


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=g).to(t)

    d, hq, hkv = case["d"], case["hq"], case["hkv"]
    s = dict(case=case)
    if case["op"] == "rotary":
        n = case["tokens"]
        s["freq"] = _frequencies(case)
        s["magnitude"] = 0.1 * math.log(case["factor"]) + 1.0
        start = torch.randint(0, case["far"] + 1, (1,), device="cuda", generator=g)
        s["positions"] = start + torch.arange(n, device="cuda")
        s["q"], s["k"] = normal(n, hq, d), normal(n, hkv, d)
        s["q_out"] = torch.empty_like(s["q"])
        if case["cache"]:
            s["v"] = normal(n, hkv, d)
            s["rows"] = torch.randperm(case["cache"], device="cuda", generator=g)[:n]
            s["k_out"], s["v_out"] = normal(case["cache"], hkv, d), normal(case["cache"], hkv, d)
        else:
            s["k_out"] = torch.empty_like(s["k"])
        return s
    q, k = _lengths(case)

    def offsets(counts):
        return torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device="cuda")

    nq = sum(q)
    nk = len(k) * case["slot"] if case["slot"] else sum(k)
    s["q_offsets"] = offsets(q)
    s["k_offsets"] = offsets([case["slot"]] * len(k)) if case["slot"] else None
    s["k_len"] = torch.tensor(k, dtype=torch.int32, device="cuda") if case["slot"] else None
    s["prefix"] = torch.full((len(q),), case["prefix"], dtype=torch.int32, device="cuda") if case["prefix"] else None
    s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, hq + 1, device="cuda") / hq) if case["bias"] else None
    # heads differ in how sharply they look
    gain = torch.rand((hq, 1), device="cuda", generator=g) * 2 + 0.5
    s["q"] = (normal(nq, hq, d).float() * gain).to(t)
    s["k"], s["v"] = normal(nk, hkv, d), normal(nk, hkv, d)
    s["o"] = torch.empty_like(s["q"])
    s["lse"] = torch.empty((hq, nq), device="cuda")
    if case["op"] == "gradient":
        s["o"], s["lse"] = _forward(s)
        s["do"] = normal(nq, hq, d)
        s["dq"], s["dk"], s["dv"] = torch.empty_like(s["q"]), torch.empty_like(s["k"]), torch.empty_like(s["v"])
    return s


# ---- the framework's calls -------------------------------------------------------------------------------------------

_handle = None


def _engine():
    global _handle
    if _handle is None:
        from sddmm_gpu_b200 import api
        _handle = api.Handle(0)
    return _handle


def _own_plan(s):
    """A program keeps the plan with its masks; the plan reads lengths and offsets anew at every call."""
    if "plan" not in s:
        c = s["case"]
        q, k = _lengths(c)
        s["plan"] = _engine().attention_plan(s["q"].dtype, c["d"], c["hq"], c["hkv"], s["q_offsets"], max(q), max(k),
                                             k_offsets=s["k_offsets"], k_len=s["k_len"], prefix=s["prefix"], slopes=s["slopes"],
                                             softcap=c["cap"], window=(c["left"], c["right"]))
    return s["plan"]


def _own(s):
    from sddmm_gpu_b200 import api
    op = s["case"]["op"]
    if op == "attention":
        _own_plan(s).forward(s["q"], s["k"], s["v"], s["o"], s["lse"], flags=api.FLAG_ASYNC)
        return s["o"], s["lse"]
    if op == "gradient":
        _own_plan(s).backward(s["q"], s["k"], s["v"], s["o"], s["lse"], s["do"], s["dq"], s["dk"], s["dv"], flags=api.FLAG_ASYNC)
        return s["dq"], s["dk"], s["dv"]
    parts = [api.RotaryPart(s["q"], s["q_out"]), api.RotaryPart(s["k"], s["k_out"], rows=s.get("rows"))]
    if "v" in s:
        parts.append(api.RotaryPart(s["v"], s["v_out"], rows=s["rows"], rotate=False))
    c = s["case"]
    _engine().rotary(parts, s["positions"], s["freq"], layout=c["layout"], inverse=c["inverse"], magnitude=s["magnitude"],
                     flags=api.FLAG_ASYNC)
    return (s["q_out"], s["k_out"], s["v_out"]) if "v" in s else (s["q_out"], s["k_out"])


# ---- the plain form --------------------------------------------------------------------------------------------------


def _padded(x, start, count, most):
    """Rows start[b] .. start[b] + count[b] of x (rows, heads, d) as (b, heads, most, d) in 32 bits, zeros behind."""
    i = torch.arange(most, device=x.device)
    there = i < count[:, None]
    rows = torch.where(there, start[:, None] + i, 0)
    return torch.where(there[:, :, None, None], x[rows].float(), 0.0).transpose(1, 2)


def _unpadded(x, offsets, rows):
    """(b, heads, most, d) back to the packed rows (rows, heads, d)."""
    t = torch.arange(rows, device=x.device)
    b = torch.searchsorted(offsets[1:].long(), t, right=True)
    return x[b, :, t - offsets[b]]


def _scores(s):
    """Scores (b, kv heads, group, q, k) with -inf where nothing is seen, what they were before cap and bias came (over cap), and
    the padded operands."""
    c = s["case"]
    lq, lk = _lengths(c)
    hkv, group = c["hkv"], c["hq"] // c["hkv"]
    q0 = s["q_offsets"].long()
    k0 = q0 if s["k_offsets"] is None else s["k_offsets"].long()
    nq = q0[1:] - q0[:-1]
    nk = (k0[1:] - k0[:-1]) if s["k_len"] is None else s["k_len"].long()
    q = _padded(s["q"], q0[:-1], nq, max(lq)).unflatten(1, (hkv, group))
    k = _padded(s["k"], k0[:-1], nk, max(lk))[:, :, None]
    v = _padded(s["v"], k0[:-1], nk, max(lk))[:, :, None]
    x = torch.matmul(q.flatten(2, 3), k[:, :, 0].transpose(-1, -2)).unflatten(2, (group, max(lq))) * (1.0 / math.sqrt(c["d"]))
    th = None
    if c["cap"]:
        th = torch.tanh(x * (1.0 / c["cap"]))
        x = th * c["cap"]
    j = torch.arange(max(lk), device="cuda")
    pos = (nk - nq)[:, None] + torch.arange(max(lq), device="cuda")
    ahead = j - pos[:, :, None]
    if s["slopes"] is not None:
        x = x - s["slopes"].view(hkv, group, 1, 1) * ahead.abs()[:, None, None].float()
    seen = torch.ones_like(ahead, dtype=torch.bool)
    if c["left"] >= 0:
        seen &= ahead >= -c["left"]
    if c["right"] >= 0:
        seen &= ahead <= c["right"]
    if c["prefix"]:
        seen |= j < s["prefix"][:, None, None]
    seen &= (j < nk[:, None])[:, None, :] & (torch.arange(max(lq), device="cuda") < nq[:, None])[:, :, None]
    return x.masked_fill_(~seen[:, None, None], -math.inf), th, q, k, v


def _forward(s):
    c = s["case"]
    x, _, q, k, v = _scores(s)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), v[:, :, 0]).unflatten(2, p.shape[2:4]) / torch.where(total == 0, 1.0, total)
    lse = torch.where(total == 0, -math.inf, torch.log(total) + top)
    o = _unpadded(o.flatten(1, 2), s["q_offsets"], s["q"].shape[0])
    lse = _unpadded(lse.flatten(1, 2), s["q_offsets"], s["q"].shape[0])
    return o.to(s["q"].dtype), lse[..., 0].T.contiguous()


def _backward(s):
    c = s["case"]
    lq, _ = _lengths(c)
    hkv, group = c["hkv"], c["hq"] // c["hkv"]
    x, th, q, k, v = _scores(s)
    q0 = s["q_offsets"].long()
    nq = q0[1:] - q0[:-1]

    def of_queries(a):
        return _padded(a, q0[:-1], nq, max(lq)).unflatten(1, (hkv, group))

    lse = of_queries(s["lse"].T[:, :, None])
    p = torch.where(lse == -math.inf, 0.0, torch.exp(x - lse))
    del x
    do = of_queries(s["do"])
    delta = (do * of_queries(s["o"])).sum(-1, keepdim=True)
    dv = torch.matmul(p.flatten(2, 3).transpose(-1, -2), do.flatten(2, 3))
    dx = p * (torch.matmul(do.flatten(2, 3), v[:, :, 0].transpose(-1, -2)).unflatten(2, (group, max(lq))) - delta)
    if th is not None:
        dx = dx * (1.0 - th * th)
    dx = dx * (1.0 / math.sqrt(c["d"]))
    dq = torch.matmul(dx.flatten(2, 3), k[:, :, 0]).unflatten(2, (group, max(lq)))
    dk = torch.matmul(dx.flatten(2, 3).transpose(-1, -2), q.flatten(2, 3))
    rows = s["q"].shape[0]
    t = s["q"].dtype
    return (_unpadded(dq.flatten(1, 2), s["q_offsets"], rows).to(t), _unpadded(dk, s["q_offsets"], rows).to(t),
            _unpadded(dv, s["q_offsets"], rows).to(t))


def _rotated(x, positions, freq, layout, inverse, magnitude):
    rot = 2 * freq.shape[0]
    angle = positions.double()[:, None] * torch.from_numpy(freq).to(x.device)
    cos, sin = (angle.cos() * magnitude).float()[:, None], (angle.sin() * magnitude).float()[:, None]
    sin = -sin if inverse else sin
    y = x.float()
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if layout == "interleaved" else (y[..., :rot // 2], y[..., rot // 2:rot])
    u, w = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([u, w], -1).flatten(-2) if layout == "interleaved" else torch.cat([u, w], -1)
    return torch.cat([turned, y[..., rot:]], -1).to(x.dtype)


def _plain_rotary(s):
    c = s["case"]
    how = s["positions"], s["freq"], c["layout"], c["inverse"], s["magnitude"]
    s["q_out"].copy_(_rotated(s["q"], *how))
    if not c["cache"]:
        s["k_out"].copy_(_rotated(s["k"], *how))
        return s["q_out"], s["k_out"]
    s["k_out"][s["rows"]] = _rotated(s["k"], *how)
    s["v_out"][s["rows"]] = s["v"]
    return s["q_out"], s["k_out"], s["v_out"]


def run(state):
    if own:
        return _own(state)
    return {"attention": _forward, "gradient": _backward, "rotary": _plain_rotary}[state["case"]["op"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}[case["type"]]
    d, hq, hkv = case["d"], case["hq"], case["hkv"]
    if case["op"] == "rotary":
        n = case["tokens"]
        moved = 2 * n * d * (hq + (2 if case["cache"] else 1) * hkv) * size
        return {"bytes": moved + 8 * n * (2 if case["cache"] else 1), "flops": 3 * n * case["rot"] * (hq + hkv)}
    pairs = keys = queries = 0
    for q, k in zip(*_lengths(case)):
        pos = k - q + np.arange(q, dtype=np.int64)
        p = min(case["prefix"], k)
        lo = np.maximum(0, pos - case["left"]) if case["left"] >= 0 else np.zeros_like(pos)
        hi = np.minimum(k - 1, pos + case["right"]) if case["right"] >= 0 else np.full_like(pos, k - 1)
        band = np.maximum(0, hi - lo + 1)
        both = np.where(band > 0, np.maximum(0, np.minimum(hi, p - 1) - lo + 1), 0)
        pairs += int((band + p - both).sum())
        seen = lo[band > 0].min(initial=k)
        keys += int(max(0, hi.max() - seen + 1) + min(p, seen))
        queries += q
    rows = size * d * (hq * queries, hkv * keys)[0], size * d * hkv * keys
    if case["op"] == "attention":
        return {"bytes": 2 * rows[0] + 2 * rows[1] + 4 * hq * queries, "flops": 4 * d * hq * pairs}
    return {"bytes": 4 * rows[0] + 4 * rows[1] + 4 * hq * queries, "flops": 10 * d * hq * pairs}


# ---- the same from the definition, in 64 bits, one sequence and head at a time ---------------------------------------


def _exact_rotary(s, case):
    def turned(x):
        n = case["rot"] // 2
        x = x.double()
        z = x[..., :2 * n].unflatten(-1, (n, 2)) if case["layout"] == "interleaved" else x[..., :2 * n].unflatten(-1, (2, n)).transpose(-1, -2)
        z = torch.view_as_complex(z.contiguous())
        phase = torch.outer(s["positions"].double(), torch.as_tensor(s["freq"], device="cuda")) * (-1 if case["inverse"] else 1)
        z = torch.view_as_real(z * torch.polar(torch.full_like(phase, s["magnitude"]), phase)[:, None])
        z = z.flatten(-2) if case["layout"] == "interleaved" else z.transpose(-1, -2).flatten(-2)
        return torch.cat((z, x[..., 2 * n:]), -1)

    if not case["cache"]:
        return turned(s["q"]), turned(s["k"])
    k, v = s["k_out"].double(), s["v_out"].double()
    k.index_copy_(0, s["rows"], turned(s["k"]))
    v.index_copy_(0, s["rows"], s["v"].double())
    return turned(s["q"]), k, v


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(s, case)
    gradient = case["op"] == "gradient"
    hq, group = case["hq"], case["hq"] // case["hkv"]
    outs = [torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in (("dq", "dk", "dv") if gradient else ("o", "lse"))]
    q_row = k_row = 0
    for b, (n, m) in enumerate(zip(*_lengths(case))):
        if case["slot"]:
            k_row = b * case["slot"]
        at = torch.arange(n, device="cuda")[:, None] + (m - n)
        key = torch.arange(m, device="cuda")[None, :]
        hidden = torch.zeros(n, m, dtype=torch.bool, device="cuda")
        if case["left"] >= 0:
            hidden |= key < at - case["left"]
        if case["right"] >= 0:
            hidden |= key > at + case["right"]
        hidden &= key >= case["prefix"]
        far = (key - at).abs()
        for h in range(hq):
            rows, keys = slice(q_row, q_row + n), slice(k_row, k_row + m)
            q, k, v = s["q"][rows, h].double(), s["k"][keys, h // group].double(), s["v"][keys, h // group].double()
            raw = torch.einsum("nd,md->nm", q, k) / case["d"] ** 0.5
            x = case["cap"] * torch.tanh(raw / case["cap"]) if case["cap"] else raw
            if case["bias"]:
                x = x - float(s["slopes"][h]) * far
            x = x.masked_fill(hidden, -math.inf)
            lse = torch.logsumexp(x, 1)
            p = torch.nan_to_num(torch.exp(x - lse[:, None]), nan=0.0)
            o = p @ v
            if not gradient:
                outs[0][rows, h], outs[1][h, rows] = o, lse
                continue
            do = s["do"][rows, h].double()
            outs[2][keys, h // group] += p.T @ do
            dx = p * (do @ v.T - (p * (do @ v.T)).sum(1, keepdim=True)) / case["d"] ** 0.5
            if case["cap"]:
                dx = dx * (1 - torch.tanh(raw / case["cap"]) ** 2)
            outs[0][rows, h] = dx @ k
            outs[1][keys, h // group] += dx.T @ q
        q_row += n
        k_row += m
    return tuple(outs)
