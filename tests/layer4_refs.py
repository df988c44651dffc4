"""The operators of a layer whose cache has four bits an element, in float64, from their definitions: plain torch on
the CPU."""
import math

import torch

from layer_refs import F64, H, H0, U

NAN = float("nan")


def group_scale(x):
    """Scale of groups [..., 32] in float64: eight significant bits, then fp16; NaN where they do not reach."""
    x = x.to(F64)
    hi, lo = x.amax(-1), x.amin(-1)
    ext = torch.where(hi >= -lo, hi, lo) / -8
    m, e = torch.frexp(ext)
    d = torch.ldexp(torch.round(m * 256), e - 8)  # (half to even)
    d = torch.where(torch.isfinite(x).all(-1) & (d.abs() <= 8160), d, NAN)
    return d.half().to(F64) + 0.0  # (one zero)


def nibbles(x, d):
    """Elements 0 .. 15 of groups x [..., 32] at scales d."""
    d = d[..., None]
    q = torch.round(x.to(F64) / torch.where(d == 0, 1.0, d)).clamp(-8, 7) + 8
    return torch.where((d == 0) | torch.isnan(d), 8.0, q).to(torch.uint8)


def pack(q):
    """[..., D] elements 0 .. 15 as bytes [..., D / 2], element by element."""
    out = torch.zeros(q.shape[:-1] + (q.shape[-1] // 2,), dtype=torch.uint8)
    for e in range(q.shape[-1]):
        n = (e % 8) // 2 + 4 * (e % 2)
        out[..., e // 8 * 4 + n // 2] |= q[..., e] << (4 * (n % 2))
    return out


def unpack(b):
    D = 2 * b.shape[-1]
    out = torch.zeros(b.shape[:-1] + (D,), dtype=torch.uint8)
    for e in range(D):
        n = (e % 8) // 2 + 4 * (e % 2)
        out[..., e] = b[..., e // 8 * 4 + n // 2] >> (4 * (n % 2)) & 15
    return out


class Cache4:
    """A cache of the tests' own making with the sequences' tables, and the operators' definitions on it.  What no
    sequence has is random: bytes of any kind, scales of any bits, NaN and infinities among them."""

    def __init__(self, seqs, per_seq, heads, bt, D, extra=3, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.bt, self.D, self.heads = bt, D, heads
        n = seqs * per_seq + extra
        self.table = torch.randperm(n, generator=g)[:seqs * per_seq].reshape(seqs, per_seq).to(torch.int32)
        self.k, self.v = (torch.randint(0, 256, (n, heads, bt, D // 2), generator=g, dtype=torch.uint8) for _ in range(2))
        some = lambda *shape: torch.randint(-32768, 32768, shape, generator=g, dtype=torch.int16).view(torch.float16)  # noqa: E731
        self.ks, self.vs = some(n, heads, bt, D // 32), some(n, heads, D // 32, bt)
        self.n_kv = torch.zeros(seqs, dtype=torch.int32)

    def place(self, s, t):
        """(block, row) of token t of sequence s, or None."""
        i = int(self.table[s, t // self.bt])
        return (i, t % self.bt) if 0 <= i < self.k.shape[0] else None

    def length(self, s):
        return min(max(int(self.n_kv[s]), 0), self.table.shape[1] * self.bt)

    def set(self, s, t, k, v):
        """Writes tokens t, t + 1 .., k and v [tokens, heads, D]."""
        kg, vg = k.unflatten(-1, (-1, 32)), v.unflatten(-1, (-1, 32))
        dk, dv = group_scale(kg), group_scale(vg)
        bad = torch.isnan(dk).any(-1, keepdim=True) | torch.isnan(dv).any(-1, keepdim=True)
        dk, dv = torch.where(bad, NAN, dk), torch.where(bad, NAN, dv)
        kb, vb = pack(nibbles(kg, dk).flatten(-2)), pack(nibbles(vg, dv).flatten(-2))
        for j in range(k.shape[0]):
            at = self.place(s, t + j)
            if at is not None:
                i, r = at
                self.k[i, :, r], self.v[i, :, r], self.ks[i, :, r], self.vs[i, :, :, r] = kb[j], vb[j], dk[j].half(), dv[j].half()

    def fill(self, n_kv, std=1.0, seed=1):
        g = torch.Generator().manual_seed(seed)
        self.n_kv = torch.tensor(n_kv, dtype=torch.int32)
        for s in range(len(n_kv)):
            n = self.length(s)
            k, v = (torch.randn((n, self.heads, self.D), generator=g) * std * torch.exp(0.4 * torch.randn((n, self.heads, 1), generator=g)) for _ in range(2))
            self.set(s, 0, k, v)
        return self

    def write(self, k, v, n_new):
        """k, v [seqs, heads, tokens, D] float32 values; in place."""
        for s in range(self.table.shape[0]):
            end, m = self.length(s), min(max(int(n_new[s]), 0), k.shape[2])
            i = max(m - end, 0)  # none before token 0
            self.set(s, end - m + i, k[s, :, i:m].transpose(0, 1), v[s, :, i:m].transpose(0, 1))

    def on_gpu(self, mi):
        d = {n: getattr(self, n).cuda() for n in ("k", "v", "ks", "vs", "table", "n_kv")}
        d["cache"] = mi.kv_cache4(d["k"], d["v"], d["ks"], d["vs"])
        d["seqs"] = mi.kv_seqs(d["table"], d["n_kv"])
        return d

    def values(self, s, which, n=None):
        """Values of sequence s's tokens [heads, n_kv, D] in float64, and whether each is there."""
        n = self.length(s) if n is None else n
        out, ok = torch.zeros((self.heads, n, self.D), dtype=F64), torch.zeros(n, dtype=torch.bool)
        for b in range((n + self.bt - 1) // self.bt):
            i, lo, hi = int(self.table[s, b]), b * self.bt, min(n, (b + 1) * self.bt)
            if not 0 <= i < self.k.shape[0]:
                continue
            q = unpack((self.k if which == "k" else self.v)[i, :, :hi - lo]).to(F64) - 8
            d = self.ks[i, :, :hi - lo] if which == "k" else self.vs[i, :, :, :hi - lo].transpose(-1, -2)
            out[:, lo:hi] = (q.unflatten(-1, (-1, 32)) * d.to(F64)[..., None]).flatten(-2)
            ok[lo:hi] = True
        return out, ok

    def seen(self, s, m, causal, window, ok):
        """What the last m tokens' queries of sequence s see [m, n_kv]."""
        n = self.length(s)
        t, p = torch.arange(n), n - m + torch.arange(m)
        seen = ok[None].expand(m, n).clone()
        if causal:
            seen &= t <= p[:, None]
        if window:
            seen &= t > p[:, None] - window
        return seen

    def scores(self, s, h, q, scale, seen, group, q32):
        """Scores of q [m, D] of head h, -inf where hidden, and the bound on how far each is off: the products are exact
        and summed in fp32 ((D + 3) U of the magnitudes), an F32 q's two halves have 22 bits of the row's largest
        element or 2^-25 of it, and scale, reference and exponent round a score and the reference, 8 U of the largest."""
        key, ok = self.values(s, "k")
        k = torch.where(ok[:, None], key[h // group], 0.0)
        qq = q.to(F64)
        sc = scale * (qq @ k.T)
        mag = abs(scale) * (qq.abs() @ k.abs().T)
        E = mag * (self.D + 3) * U
        if q32:
            E = E + mag * 2.0 ** -22 + abs(scale) * 2.0 ** -25 * qq.abs().amax(-1, keepdim=True) * k.abs().sum(-1)
        big = torch.where(seen, sc.abs(), 0.0).amax(-1, keepdim=True) if sc.shape[1] else torch.zeros((sc.shape[0], 1), dtype=F64)
        E = torch.where(seen, E + 8 * U * big.clamp(min=1.0), 0.0)
        return sc.masked_fill(~seen, -math.inf), E

    def attn(self, q, n_q, scale, causal, window, q32, d32):
        """(out, its tolerance, lse, its tolerance) of q [seqs, n_q, heads, D]; rows past n_q are NaN.

        With E the bound on a score: a weight is off by the relative 2 E + 4 U (itself and the sum); it enters its
        product rounded by H relative (F32 dst: 2^-22), and for an F16 dst the sum is of the rounded ones, H again; a half
        has at least the step 2^-24, the reference being held at most 2^15 and at least 2^12 above the largest weight's
        place: 2^-37 of the largest weight a token; sums of n terms (n + 8) U.  The sum that lse takes is of unrounded
        weights."""
        S, NQ, NH, D = q.shape
        out, lse = torch.full((S, NQ, NH, D), math.nan, dtype=F64), torch.full((S, NQ, NH), math.nan, dtype=F64)
        tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
        group = NH // self.heads
        for s in range(S):
            val, ok = self.values(s, "v")
            m = min(max(int(n_q[s]), 0), NQ)
            seen = self.seen(s, m, causal, window, ok)
            n = seen.shape[1]
            for h in range(NH):
                sc, E = self.scores(s, h, q[s, :m, h], scale, seen, group, q32)
                vv = torch.where(ok[:, None], val[h // group], 0.0)
                w = torch.softmax(sc, -1)
                w = torch.where(seen.any(-1, keepdim=True), w, 0.0)
                vv = torch.where(seen.any(0)[:, None], vv, 0.0) if m else vv
                out[s, :m, h] = w @ vv
                lse[s, :m, h] = torch.logsumexp(sc, -1) if n else -math.inf
                if n == 0:
                    continue
                E = E.amax(-1, keepdim=True)
                W = w @ vv.abs()
                floor = n * 2.0 ** -37 * w.amax(-1, keepdim=True) * vv.abs().amax(0)
                tol[s, :m, h] = W * (2 * E + 4 * U + (2.0 ** -22 if d32 else 2 * H) + (n + 8) * U) + floor
                tol[s, :m, h] += U * out[s, :m, h].abs() if d32 else H * out[s, :m, h].abs() + H0
                ltol[s, :m, h] = (E + (n + 8) * U)[:, 0] + 4 * U * lse[s, :m, h].abs().nan_to_num(0, 0, 0)
        return out, tol, lse, ltol

    def weights(self, q, n_q, lse, scale, causal, window, q32):
        """(what is added [seqs, heads, room], its bound): a term is off by the relative E + 4 U and the difference's
        rounding, U of the larger of score and lse; sums of r terms in two levels of 64 tiles, at most (r + 8) U."""
        S, NQ, NH, D = q.shape
        room, group = self.table.shape[1] * self.bt, NH // self.heads
        out, tol = torch.zeros((S, self.heads, room), dtype=F64), torch.zeros((S, self.heads, room), dtype=F64)
        for s in range(S):
            _, ok = self.values(s, "k")
            m = min(max(int(n_q[s]), 0), NQ)
            seen = self.seen(s, m, causal, window, ok)
            n = seen.shape[1]
            for h in range(NH):
                sc, E = self.scores(s, h, q[s, :m, h], scale, seen, group, q32)
                l = lse[s, :m, h].to(F64)[:, None]
                p = torch.where(seen, torch.exp(sc - torch.where(seen.any(-1, keepdim=True), l, 0.0)), 0.0)
                out[s, h // group, :n] += p.sum(0)
                tol[s, h // group, :n] += (p * (E + 2 * U * l.abs().nan_to_num(0, 0, 0) + 4 * U)).sum(0) + p.sum(0) * (m * group + 8) * U
        return out, tol

    def evict(self, sums, n_keep, first, recent, sums_out, kept):
        """Lists of kept tokens by a sort; in place.  Returns the lengths."""
        k, v, ks, vs = self.k.clone(), self.v.clone(), self.ks.clone(), self.vs.clone()
        lengths = []
        for s in range(self.table.shape[0]):
            n = self.length(s)
            m = min(n, max(int(n_keep[s]), 0), kept.shape[2])
            rec = min(recent, m)
            fst = min(first, m - rec)
            for h in range(self.heads):
                def rank(t):
                    if t < fst or t >= n - rec:
                        return (0, 0.0, t)
                    if self.place(s, t) is None:
                        return (3, 0.0, t)
                    x = float(sums[s, h, t])
                    return (2, 0.0, t) if x != x else (1, -x, t)
                keep = list(range(n)) if m == n else sorted(sorted(range(n), key=rank)[:m])
                x = sums[s, h].clone()
                sums_out[s, h, :n] = 0
                for j, t in enumerate(keep):
                    kept[s, h, j] = t
                    sums_out[s, h, j] = x[t]
                    to, at = self.place(s, j), self.place(s, t)
                    if to is None or t == j:
                        continue
                    if at is None:
                        self.ks[to[0], h, to[1]] = NAN
                        self.vs[to[0], h, :, to[1]] = NAN
                        continue
                    self.k[to[0], h, to[1]], self.v[to[0], h, to[1]] = k[at[0], h, at[1]], v[at[0], h, at[1]]
                    self.ks[to[0], h, to[1]], self.vs[to[0], h, :, to[1]] = ks[at[0], h, at[1]], vs[at[0], h, :, at[1]]
            lengths.append(m)
        return lengths
