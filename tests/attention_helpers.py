"""Attention and its gradient in 64 bits, from the definition, with the magnitudes that tolerances are made of."""
import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def offsets(counts, device="cuda"):
    out = [0]
    for c in counts:
        out.append(out[-1] + c)
    return torch.tensor(out, dtype=torch.int32, device=device)


class Problem:
    """A batch of sequences with its mask; random operands of it."""

    def __init__(self, dtype, d, hq, hkv, q, k=None, slot=0, window=(-1, -1), prefix=0, cap=0.0, bias=False, seed=1, scale=None, gain=1.0,
                 extra_rows=0):
        self.dtype, self.d, self.hq, self.hkv, self.q_counts, self.k_counts = dtype, d, hq, hkv, q, k or q
        self.window, self.cap, self.slot = window, cap, slot
        self.scale = d ** -0.5 if scale is None else scale
        g = torch.Generator("cuda").manual_seed(seed)
        n = len(q)
        self.q_offsets = offsets(q)
        separate = k is not None or slot
        self.k_offsets = offsets([slot] * n if slot else self.k_counts) if separate else None
        self.k_len = torch.tensor(self.k_counts, dtype=torch.int32, device="cuda") if slot else None
        self.prefix_of = [prefix if isinstance(prefix, int) else prefix[b] for b in range(n)]
        self.prefix = torch.tensor(self.prefix_of, dtype=torch.int32, device="cuda") if any(self.prefix_of) else None
        self.slopes = 2.0 ** (-4.0 * torch.arange(1, hq + 1, device="cuda") / hq) if bias else None
        self.q_rows = sum(q) + extra_rows
        self.k_rows = (n * slot if slot else sum(self.k_counts)) + extra_rows

        def normal(rows, heads, by=1.0):
            return (torch.randn((rows, heads, d), device="cuda", generator=g) * by).to(dtype)

        self.Q, self.K, self.V = normal(self.q_rows, hq, gain), normal(self.k_rows, hkv), normal(self.k_rows, hkv)
        self.dO = normal(self.q_rows, hq)

    def plan(self, engine, **more):
        kw = dict(k_offsets=self.k_offsets, k_len=self.k_len, prefix=self.prefix, slopes=self.slopes, scale=self.scale,
                  softcap=self.cap, window=self.window, q_rows=self.q_rows, k_rows=self.k_rows)
        kw.update(more)
        return engine.attention_plan(self.dtype, self.d, self.hq, self.hkv, self.q_offsets, max(self.q_counts, default=0),
                                     max(self.k_counts, default=0), **kw)

    def sequences(self):
        """(rows of Q, rows of K, seen) of each sequence; seen: queries x keys."""
        qr = kr = 0
        for b, (nq, nk) in enumerate(zip(self.q_counts, self.k_counts)):
            k0 = b * self.slot if self.slot else kr
            pos = torch.arange(nq, device="cuda")[:, None] + (nk - nq)
            j = torch.arange(nk, device="cuda")[None, :]
            seen = torch.ones((nq, nk), dtype=torch.bool, device="cuda")
            if self.window[0] >= 0:
                seen &= j >= pos - self.window[0]
            if self.window[1] >= 0:
                seen &= j <= pos + self.window[1]
            seen |= j < self.prefix_of[b]
            yield slice(qr, qr + nq), slice(k0, k0 + nk), seen, (pos - j).abs()
            qr += nq
            kr += nk

    def scores(self, Q, K, h, rows, keys, seen, far):
        """Scores of head h, slope of the cap, and the most that a product's rounding can move a score of the row."""
        q, k = Q[rows, h].double(), K[keys, h // (self.hq // self.hkv)].double()
        raw = q @ k.T * self.scale
        size = (q.abs() @ k.abs().T) * self.scale
        x, slope = raw, torch.ones_like(raw)
        if self.cap:
            t = torch.tanh(raw / self.cap)
            x, slope = self.cap * t, 1 - t * t
        if self.slopes is not None:
            x = x - self.slopes[h].double() * far
            size = size + self.slopes[h].double() * far
        x = torch.where(seen, x, -math.inf)
        # fp32 products and sums (d terms, then scale, cap, bias: 8 roundings), and a cap good to 2^-21 of itself
        wobble = torch.where(seen, size * (self.d + 8) * 2.0 ** -24 + self.cap * 2.0 ** -21, 0.0)
        top = wobble.max(1).values if seen.shape[1] else torch.zeros(seen.shape[0], device="cuda", dtype=torch.float64)
        return x, slope, top

    def forward(self, Q=None, K=None, V=None):
        """O, lse, their tolerances (rounded weights: half a step of the type each); rows of no sequence: NaN."""
        Q, K, V = (self.Q if Q is None else Q), (self.K if K is None else K), (self.V if V is None else V)
        u = HALF_STEP[self.dtype]
        O = torch.full((self.q_rows, self.hq, self.d), math.nan, dtype=torch.float64, device="cuda")
        lse = torch.full((self.hq, self.q_rows), math.nan, dtype=torch.float64, device="cuda")
        tol_o, tol_l = torch.zeros_like(O), torch.zeros_like(lse)
        for rows, keys, seen, far in self.sequences():
            n = seen.shape[1]
            for h in range(self.hq):
                x, _, wobble = self.scores(Q, K, h, rows, keys, seen, far)
                l = torch.logsumexp(x, 1) if n else torch.full((seen.shape[0],), -math.inf, device="cuda", dtype=torch.float64)
                p = torch.where(seen, torch.exp(x - torch.where(l == -math.inf, 0.0, l)[:, None]), 0.0)
                v = V[keys, h // (self.hq // self.hkv)].double()
                o = p @ v
                tiny = 2.0 ** -25 if self.dtype == torch.float16 else 0.0  # half a step of a subnormal weight
                # a weight: its score's error, exp (2^-22, and its argument of up to 2^5 rounded: 2^-19), its rounding; sums of n terms
                rel = 2 * wobble + 2.0 ** -19 + (n + 16) * 2.0 ** -24 + (u if u > 2.0 ** -24 else 0.0)
                O[rows, h], lse[h, rows] = o, l
                tol_o[rows, h] = rel[:, None] * (p @ v.abs()) * 2 + tiny * (seen.double() @ v.abs()) + u * o.abs() + 1e-30 + (2.0 ** -24 if self.dtype == torch.float16 else 0.0)
                tol_l[h, rows] = wobble + 2.0 ** -20 + (n + 16) * 2.0 ** -24 + 2.0 ** -22 * torch.where(l == -math.inf, 0.0, l).abs()
        return O, lse, tol_o, tol_l

    def backward(self):
        """dQ, dK, dV and their tolerances."""
        u = HALF_STEP[self.dtype]
        w = u if u > 2.0 ** -24 else 0.0  # weights and score gradients rounded before a product
        shape = lambda like: torch.zeros(like.shape, dtype=torch.float64, device="cuda")  # noqa: E731
        dQ, dK, dV, tQ, tK, tV = (shape(t) for t in (self.Q, self.K, self.V, self.Q, self.K, self.V))
        for rows, keys, seen, far in self.sequences():
            nq, nk = seen.shape
            if not nq or not nk:
                continue
            for h in range(self.hq):
                g = h // (self.hq // self.hkv)
                x, slope, wobble = self.scores(self.Q, self.K, h, rows, keys, seen, far)
                l = torch.logsumexp(x, 1)
                p = torch.where(seen, torch.exp(x - torch.where(l == -math.inf, 0.0, l)[:, None]), 0.0)
                q, k, v, do = self.Q[rows, h].double(), self.K[keys, g].double(), self.V[keys, g].double(), self.dO[rows, h].double()
                o = p @ v
                dp, size = do @ v.T, do.abs() @ v.abs().T
                delta, dsize = (do * o).sum(1, keepdim=True), (do.abs() * (p @ v.abs())).sum(1, keepdim=True)
                ds = p * (dp - delta) * slope * self.scale
                # error of ds: of p (its score, of lse, exp), of dp, of delta (O as rounded, and off by the forward's own tolerance), of the slope
                e_p = (3 * wobble + 2.0 ** -19 + (nk + 16) * 2.0 ** -24)[:, None]
                most = p * (dp - delta).abs() * self.scale
                e_ds = most * slope * e_p + p * self.scale * ((self.d + 8) * 2.0 ** -24 * (size + dsize) + (2 * w + u) * dsize)
                # weights and score gradients below 2^-14 are subnormal in fp16: half a step is 2^-25
                tiny = 2.0 ** -25 if self.dtype == torch.float16 else 0.0
                e_ds = e_ds + seen * tiny * self.scale + most * (2.0 ** -20 + (4 * wobble[:, None] / self.cap if self.cap else 0.0)) + w * ds.abs()
                dQ[rows, h] = ds @ k
                tQ[rows, h] = e_ds @ k.abs() + (nk + 16) * 2.0 ** -24 * (ds.abs() @ k.abs())
                dK[keys, g] += ds.T @ q
                tK[keys, g] += e_ds.T @ q.abs() + (nq * self.hq + 16) * 2.0 ** -24 * (ds.abs().T @ q.abs())
                dV[keys, g] += p.T @ do
                tV[keys, g] += (p * (e_p + w) + seen * tiny).T @ do.abs() + (nq * self.hq + 16) * 2.0 ** -24 * (p.T @ do.abs())
        floor = 1e-30 + (2.0 ** -24 if self.dtype == torch.float16 else 0.0)
        return (dQ, dK, dV), tuple(t + u * x.abs() + floor for t, x in ((tQ, dQ), (tK, dK), (tV, dV)))


def within(got, want, tol, what=""):
    got = got.double()
    same = (got == want) | ((got - want).abs() <= tol)
    assert bool(same.all()), f"{what}: {int((~same).sum())} of {same.numel()} out of tolerance, worst {float(((got - want).abs() / tol)[~same].max())} of it"
