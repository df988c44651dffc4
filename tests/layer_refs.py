"""The operators around a layer's products in float64, from their definitions, and a cache of the tests' own
making: plain torch on the CPU or the GPU."""
import math

import torch

F64 = torch.float64
U = 2.0 ** -24   # half a step of float32, relative
H = 2.0 ** -11   # half a step of float16, relative
H0 = 2.0 ** -25  # half a step of float16 below its normal range


def step(dtype):
    return (H, H0) if dtype == torch.float16 else (U, 2.0 ** -150)


def tensor(mi, x, t=None):
    """mi355_tensor over a torch view, its last dimension first."""
    ne = list(reversed(x.shape))
    nb = [s * x.element_size() for s in reversed(x.stride())]
    nb += [nb[-1] * ne[-1]] * (4 - len(nb))
    return mi.from_torch(x, (mi.F16 if x.dtype == torch.float16 else mi.F32) if t is None else t, ne, nb)


def angles(pos, sections, n_dims, base, restart=False, interleaved=False, scale=1.0):
    """Angle of every pair: pos [axes, batch, tokens] -> [batch, tokens, n_dims / 2]."""
    n = n_dims // 2
    axes = []
    for i in range(n):
        if interleaved:
            a = i % 3
            axes.append(a if a and i < 3 * sections[a] else 0)
        else:
            axes.append(next(a for a in range(len(sections)) if i < sum(sections[:a + 1])))
    out, seen = [], [0] * 4
    for i, a in enumerate(axes):
        e = seen[a] / sections[a] if restart else i / n
        seen[a] += 1
        out.append(pos[a].to(F64) * (scale * base ** -e))
    return torch.stack(out, -1)


def rope(x, ang, halves):
    """x [batch, tokens, heads, ne0] turned by ang [batch, tokens, pairs]."""
    n = ang.shape[-1]
    y = x.to(F64).clone()
    i0 = torch.arange(n, device=x.device) * (1 if halves else 2)
    i1 = i0 + (n if halves else 1)
    c, s = torch.cos(ang)[:, :, None], torch.sin(ang)[:, :, None]
    a, b = x[..., i0].to(F64), x[..., i1].to(F64)
    y[..., i0], y[..., i1] = a * c - b * s, a * s + b * c
    return y


class Cache:
    """Bytes and scales [blocks, heads, tokens, D] / [blocks, heads] with the sequences' tables, and the
    operators' definitions on them, one block and head at a time."""

    def __init__(self, seqs, per_seq, heads, bt, D, extra=3, seed=0, device="cpu"):
        g = torch.Generator().manual_seed(seed)
        self.bt, self.D, self.heads = bt, D, heads
        n = seqs * per_seq + extra
        self.table = torch.randperm(n, generator=g)[:seqs * per_seq].reshape(seqs, per_seq).to(torch.int32)
        self.k, self.v = (torch.randint(0, 256, (n, heads, bt, D), generator=g, dtype=torch.uint8) for _ in range(2))
        self.ks, self.vs = (torch.full((n, heads), float("nan")) for _ in range(2))  # unwritten: anything
        self.n_kv = torch.zeros(seqs, dtype=torch.int32)

    def fill(self, n_kv, std=30.0, scale=0.03, seed=1):
        """Sequences of these lengths, as earlier writes left them."""
        g = torch.Generator().manual_seed(seed)
        self.n_kv = torch.tensor(n_kv, dtype=torch.int32)
        for s, n in enumerate(n_kv):
            for b in range((n + self.bt - 1) // self.bt):
                i = int(self.table[s, b])
                if not 0 <= i < self.k.shape[0]:
                    continue
                for x, sc in ((self.k, self.ks), (self.v, self.vs)):
                    q = torch.round(torch.randn((self.heads, self.bt, self.D), generator=g) * std).clamp(-127, 127)
                    x[i] = (q + 128).to(torch.uint8)
                    sc[i] = scale * torch.exp(0.5 * torch.randn(self.heads, generator=g))
        return self

    def on_gpu(self, mi):
        d = {n: getattr(self, n).cuda() for n in ("k", "v", "ks", "vs", "table", "n_kv")}
        d["cache"] = mi.kv_cache(d["k"], d["v"], d["ks"], d["vs"])
        d["seqs"] = mi.kv_seqs(d["table"], d["n_kv"])
        return d

    def write(self, k, v, n_new):
        """k, v [seqs, heads, tokens, D] float32 values; in place."""
        for s in range(self.table.shape[0]):
            end = min(max(int(self.n_kv[s]), 0), self.table.shape[1] * self.bt)
            m = min(max(int(n_new[s]), 0), k.shape[2])
            first = end - m
            for b in range(max(first, 0) // self.bt, (end + self.bt - 1) // self.bt):
                i, lo, hi = int(self.table[s, b]), max(first, 0, b * self.bt), min(end, (b + 1) * self.bt)
                if lo >= hi or not 0 <= i < self.k.shape[0]:
                    continue
                for x, q8, sc in ((k, self.k, self.ks), (v, self.v, self.vs)):
                    for h in range(self.heads):
                        keep = lo - b * self.bt
                        new = x[s, h, lo - first:hi - first].float()
                        d = new.abs().max() / torch.tensor(127.0)  # NaN wins
                        if keep:
                            d = torch.maximum(d, sc[i, h])
                            new = torch.cat([(q8[i, h, :keep].float() - 128) * sc[i, h], new])
                        q = torch.full(new.shape, 128, dtype=torch.uint8)
                        if torch.isfinite(d) and d > 0:
                            q = (torch.round(new.to(F64) / d.to(F64)).clamp(-127, 127) + 128).to(torch.uint8)
                        q8[i, h, :hi - b * self.bt] = q
                        sc[i, h] = d

    def values(self, s, which):
        """Values of sequence s's tokens [heads, n_kv, D] in float64, and whether each is there."""
        q8, sc = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        n = min(max(int(self.n_kv[s]), 0), self.table.shape[1] * self.bt)
        out, ok = torch.zeros((self.heads, n, self.D), dtype=F64), torch.zeros(n, dtype=torch.bool)
        for b in range((n + self.bt - 1) // self.bt):
            i, hi = int(self.table[s, b]), min(self.bt, n - b * self.bt)
            if 0 <= i < q8.shape[0]:
                out[:, b * self.bt:b * self.bt + hi] = (q8[i, :, :hi].to(F64) - 128) * sc[i].to(F64)[:, None, None]
                ok[b * self.bt:b * self.bt + hi] = True
        return out, ok

    def attn(self, q, n_q, scale, causal, window, q32, d32):
        """(out, tolerance) [seqs, n_q, heads, D] of q [seqs, n_q, heads, D]; rows past n_q are NaN.

        Tolerance, from the roundings of the products' operands and fp32 sums: a score is off by at most
          E = |scale| (sum |q k| ((D + 3) U + 2^-22 for an F32 q's two halves) + 2^-25 sum |k|, the halves' range)
        plus 4 U max(|score|, 1) for the scale, the running maximum and exp2's argument; its weight by
        the relative 2 E + 4 U (numerator and sum); a weight enters its product rounded by H (F32 dst: 2^-22) relative and
        2^-24 of the largest weighted step, over a sum of n terms by (n + 4) U."""
        S, NQ, NH, D = q.shape
        out = torch.full((S, NQ, NH, D), math.nan, dtype=F64)
        tol = torch.zeros_like(out)
        group = NH // self.heads
        for s in range(S):
            key, ok = self.values(s, "k")
            val, _ = self.values(s, "v")
            n, m = key.shape[1], min(max(int(n_q[s]), 0), NQ)
            t, p = torch.arange(n), n - m + torch.arange(m)
            seen = ok[None].expand(m, n).clone()
            if causal:
                seen &= t <= p[:, None]
            if window:
                seen &= t > p[:, None] - window
            for h in range(NH):
                kk, vv, qq = key[h // group], val[h // group], q[s, :m, h].to(F64)
                kk, vv = torch.where(ok[:, None], kk, 0.0), torch.where(ok[:, None], vv, 0.0)
                sc = scale * (qq @ kk.T)
                mag = (qq.abs() @ kk.abs().T) * abs(scale)
                w = torch.nan_to_num(torch.softmax(sc.masked_fill(~seen, -math.inf), -1))
                out[s, :m, h] = w @ vv
                if n == 0:
                    continue
                E = mag * ((D + 3) * U + (2.0 ** -22 if q32 else 0)) + (2.0 ** -25 * abs(scale) * kk.abs().sum(-1) if q32 else 0)
                E = torch.where(seen, E + 4 * U * torch.clamp(sc.abs(), min=1.0), 0.0).amax(-1, keepdim=True)
                W = w @ vv.abs()
                top = (w[:, :, None] * vv.abs()[None]).amax(1) if n * m < 400000 else W
                rel = 2 * E + 4 * U + (2.0 ** -22 if d32 else H) + (n + 4) * U
                tol[s, :m, h] = W * rel + n * 2.0 ** -24 * 127 * top.amax(-1, keepdim=True) * (2.0 ** -10 if d32 else 1.0)
                if not d32:
                    tol[s, :m, h] += H * out[s, :m, h].abs() + H0
        return out, tol
