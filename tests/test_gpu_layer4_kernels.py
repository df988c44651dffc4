"""Each kernel of the 4-bit cache's attention and of its weights' sums, named by the profile, over sizes that take it,
against float64 on the GPU; and the eviction of many sequences."""
import math

import pytest
import torch

import layer4_refs as R4
from layer_refs import F64, H, H0, U, tensor

pytestmark = pytest.mark.gpu
F16, F32, I32 = torch.float16, torch.float32, torch.int32
DEV = "cuda"


class Big:
    """A cache of random nibbles and scales on the GPU, and a sequence's values in float64."""

    def __init__(self, mi, n_kv, heads, bt, D, seed=0, miss=True, before=0):
        g = torch.Generator(DEV).manual_seed(seed)
        S, per = len(n_kv), max(n_kv) // bt + 1
        n = S * per + 2
        self.heads, self.bt, self.D = heads, bt, D
        self.table = before + torch.randperm(n, generator=g, device=DEV)[:S * per].reshape(S, per).to(I32)
        n += before  # (blocks that no sequence has)
        if miss and per > 3:
            self.table[0, 2] = -1
        self.n_kv = torch.tensor(n_kv, dtype=I32, device=DEV)
        self.k, self.v = (torch.randint(0, 256, (n, heads, bt, D // 2), generator=g, device=DEV, dtype=torch.uint8) for _ in range(2))
        scale = lambda *s: ((torch.rand(s, generator=g, device=DEV) - 0.5) * 0.6).bfloat16().to(F16)  # noqa: E731
        self.ks, self.vs = scale(n, heads, bt, D // 32), scale(n, heads, D // 32, bt)
        self.cache, self.seqs = mi.kv_cache4(self.k, self.v, self.ks, self.vs), mi.kv_seqs(self.table, self.n_kv)

    def rows(self, s, h, which):
        """Values [n, D] in float64, and which tokens are there."""
        ids, n = self.table[s].long(), int(self.n_kv[s])
        ok = (ids >= 0)[:, None].expand(-1, self.bt).flatten()[:n]
        ids = ids.clamp(min=0)
        b = (self.k if which == "k" else self.v)[ids, h]
        nib = torch.stack([b & 15, b >> 4], -1).flatten(-2).unflatten(-1, (-1, 2, 4)).transpose(-1, -2).flatten(-3)
        d = self.ks[ids, h] if which == "k" else self.vs[ids, h].transpose(-1, -2)
        x = ((nib.to(F64) - 8).unflatten(-1, (-1, 32)) * d.to(F64)[..., None]).flatten(-2)
        return x.flatten(0, 1)[:n], ok


def scores(c, s, h, q, group, causal, window, scale):
    """Scores of q [rows, D] in float64, -inf where hidden, and the bound on each (layer4_refs.py's, of the whole row)."""
    k, ok = c.rows(s, h // group, "k")
    n, m = k.shape[0], q.shape[0]
    t, p = torch.arange(n, device=DEV), n - m + torch.arange(m, device=DEV)
    seen = ok[None].expand(m, n)
    if causal:
        seen = seen & (t <= p[:, None])
    if window:
        seen = seen & (t > p[:, None] - window)
    q64 = q.to(F64)
    sc = scale * (q64 @ k.T.contiguous())
    E = abs(scale) * (q64.abs() @ k.abs().T.contiguous()) * ((c.D + 3) * U + (2.0 ** -22 if q.dtype == F32 else 0))
    if q.dtype == F32:
        E = E + abs(scale) * 2.0 ** -25 * q64.abs().amax(-1, keepdim=True) * k.abs().sum(-1)
    E = torch.where(seen, E, 0.0) + 8 * U * torch.where(seen, sc.abs(), 0.0).amax(-1, keepdim=True).clamp(min=1.0)
    return sc.masked_fill(~seen, -math.inf), E, seen


def check(mi, ctx, c, q, n_q, causal, window, d_type, want):
    """The attention (its kernel's name: want) and the sums of its weights."""
    S, NQ, NH, D = q.shape
    group, scale = NH // c.heads, D ** -0.5
    dst = torch.full((S, NQ, NH, D), math.nan, dtype=d_type, device=DEV)
    lse = torch.full((S, NQ, NH), math.nan, device=DEV)
    nq = torch.tensor(n_q, dtype=I32, device=DEV)
    room = c.table.shape[1] * c.bt
    sums = torch.zeros((S, c.heads, room), device=DEV)
    ctx.profile(True)
    qt = tensor(mi, q.transpose(1, 2))
    ctx.kv_cache4_attn(c.cache, c.seqs, qt, tensor(mi, dst), scale, n_q=nq.data_ptr(), causal=causal, window=window, lse=lse.data_ptr())
    ctx.kv_cache4_weights(c.cache, c.seqs, qt, lse.data_ptr(), sums.data_ptr(), scale, n_q=nq.data_ptr(), causal=causal, window=window)
    ctx.synchronize()
    names = set(ctx.profile_collect())
    ctx.profile(False)
    assert want in names and ("kv_cache4_weights_16" if NQ * group <= 16 else "kv_cache4_weights_32") in names, names
    d32 = d_type == F32
    for s in range(S):
        m = n_q[s]
        assert torch.isnan(dst[s, m:]).all() and torch.isnan(lse[s, m:]).all()
        add, atol = torch.zeros((c.heads, room), dtype=F64, device=DEV), torch.zeros((c.heads, room), dtype=F64, device=DEV)
        for h in range(NH):
            sc, E, seen = scores(c, s, h, q[s, :m, h], group, causal, window, scale)
            v, ok = c.rows(s, h // group, "v")
            n = v.shape[0]
            w = torch.where(seen.any(-1, keepdim=True), torch.softmax(sc, -1), 0.0)
            top = E.amax(-1, keepdim=True)
            y, W = w @ v, w @ v.abs()
            # (layer4_refs.py's Cache4.attn: the terms of the same roundings)
            tol = W * (2 * top + 4 * U + (2.0 ** -22 if d32 else 2 * H) + (n + 8) * U) + n * 2.0 ** -37 * w.amax(-1, keepdim=True) * v.abs().amax(0)
            tol = tol + (U * y.abs() if d32 else H * y.abs() + H0)
            got = dst[s, :m, h].to(F64)
            assert ((got - y).abs() <= tol).all(), (s, h, float(((got - y).abs() / tol).max()))
            want_l, l = torch.logsumexp(sc, -1), lse[s, :m, h].to(F64)
            some = seen.any(-1)
            assert (l[~some] == -math.inf).all()
            ltol = (top + (n + 8) * U)[:, 0] + 4 * U * want_l.abs().nan_to_num(0, 0, 0)
            assert ((l - want_l).abs()[some] <= ltol[some]).all()
            p = torch.where(seen, torch.exp(sc - torch.where(some, l, 0.0)[:, None]), 0.0)
            add[h // group, :n] += p.sum(0)
            atol[h // group, :n] += (p * (E + 2 * U * torch.where(some, l, 0.0).abs()[:, None] + 4 * U)).sum(0) + p.sum(0) * (m * group + 8) * U
        got = sums[s].to(F64)
        assert ((got - add).abs() <= atol + U * add).all(), float(((got - add).abs() - atol).max())


# sequences' lengths, queries, heads, key heads, tokens of a block, causal, window, the kernel
KERNELS = [([3000, 40, 1700], 1, 12, 3, 64, True, 0, "kv_cache4_attn_16"), ([700, 641], 40, 4, 2, 32, True, 0, "kv_cache4_attn_16"),
           ([900, 5, 830, 64, 1000, 77, 12, 801], 70, 32, 8, 16, True, 130, "kv_cache4_attn_128"),
           ([1800], 300, 16, 8, 128, True, 0, "kv_cache4_attn_128"), ([1290, 1201], 200, 12, 4, 64, False, 0, "kv_cache4_attn_128"),
           ([1800, 1555], 1501, 32, 4, 64, True, 0, "kv_cache4_attn_128_halves"), ([1500, 1999], 1501, 32, 4, 16, True, 333, "kv_cache4_attn_128_halves"),
           ([1700, 1], 1500, 40, 5, 128, False, 0, "kv_cache4_attn_128_halves"), ([4001], 4000, 4, 4, 64, True, 0, "kv_cache4_attn_128_halves")]


@pytest.mark.parametrize("q_type,d_type", [(F16, F16), (F32, F32), (F16, F32), (F32, F16)])
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("n_kv,nq,heads,kv,bt,causal,window,want", KERNELS)
def test_kernel(mi, ctx, n_kv, nq, heads, kv, bt, causal, window, want, D, q_type, d_type):
    c = Big(mi, n_kv, kv, bt, D, seed=nq)
    g = torch.Generator(DEV).manual_seed(D + nq)
    q = torch.randn((len(n_kv), nq, heads, D), generator=g, device=DEV).to(q_type)
    check(mi, ctx, c, q, [nq] + [max(nq - 3, 0)] * (len(n_kv) - 1), causal, window, d_type, want)


def test_write_ties_of_halves(mi, ctx):
    """F16 elements whose quotients are ties, and their neighbours, for scales of every significand and many magnitudes."""
    D = 64
    rows = []
    for m in range(128, 256, 3):
        for e in (-20, -12, -3, 2, 5):
            d = torch.tensor(float(m) * 2.0 ** (e - 7), dtype=F64)
            x = ((torch.arange(D, dtype=F64) % 16 - 7.5) * d).half()
            x[0] = x[32] = (-8 * d).half()
            if not torch.isfinite(x).all():
                continue
            up = torch.nextafter(x, torch.full_like(x, math.inf))
            down = torch.nextafter(x, torch.full_like(x, -math.inf))
            for y in (x, up, down):
                y = y.clone()
                y[0] = y[32] = x[0]
                rows.append(torch.where(y.abs() > x[0].abs(), x, y))
    n = len(rows) // 16 * 16
    x = torch.stack(rows[:n])[None, None]
    c = R4.Cache4(1, n // 16, 1, 16, D)
    c.n_kv[0] = n
    d = c.on_gpu(mi)
    c.write(x.float(), -x.float(), [n])
    kd, vd = x.cuda(), (-x).cuda()
    ctx.kv_cache4_write(d["cache"], d["seqs"], tensor(mi, kd), tensor(mi, vd))
    ctx.synchronize()
    assert torch.equal(d["k"].cpu(), c.k) and torch.equal(d["v"].cpu(), c.v)
    assert torch.equal(d["ks"].cpu()[c.table[0].long()], c.ks[c.table[0].long()])


@pytest.mark.parametrize("D", [64, 96, 128])
def test_evict_many(mi, ctx, D):
    """Lists, sums and rows of many sequences and heads against a sort of the whole: what is kept is read back unchanged."""
    n_kv = [5000, 4097, 17, 20000, 4096, 1, 16385]
    S, heads, bt, keep = len(n_kv), 3, 32, 9000
    c = Big(mi, n_kv, heads, bt, D, seed=D, miss=False)
    room = c.table.shape[1] * bt
    g = torch.Generator(DEV).manual_seed(1)
    sums = torch.where(torch.rand((S, heads, room), generator=g, device=DEV) < 0.4, 0.0, torch.randn((S, heads, room), generator=g, device=DEV).abs())
    n_keep = [4100, 1000, 9, 9000, 4096, 3, 8192]
    before = [[[c.rows(s, h, x)[0] for x in "kv"] for h in range(heads)] for s in range(S)]
    out, kept = torch.full_like(sums, 7.0), torch.full((S, heads, keep), -1, dtype=I32, device=DEV)
    n, nk = torch.zeros(S, dtype=I32, device=DEV), torch.tensor(n_keep, dtype=I32, device=DEV)
    ctx.kv_cache4_evict(c.cache, c.seqs, sums.data_ptr(), out.data_ptr(), keep, kept.data_ptr(), n.data_ptr(), n_keep=nk.data_ptr(), first=3, recent=500)
    ctx.synchronize()
    for s in range(S):
        end, m = n_kv[s], min(n_kv[s], n_keep[s])
        assert int(n[s]) == m
        rec = min(500, m)
        fst = min(3, m - rec)
        for h in range(heads):
            w = sums[s, h, :end].clone()
            w[:fst], w[end - rec:] = math.inf, math.inf
            order = torch.sort(w, descending=True, stable=True).indices[:m].sort().values
            assert torch.equal(kept[s, h, :m].long(), order) and (kept[s, h, m:] == -1).all()
            assert torch.equal(out[s, h, :m], sums[s, h, order]) and (out[s, h, m:end] == 0).all() and (out[s, h, end:] == 7).all()
            for x, was in zip("kv", before[s][h]):
                now = c.rows(s, h, x)[0]
                assert torch.equal(now[:m], was[order]) and torch.equal(now[m:], was[m:])


def test_weights_of_a_window_in_a_long_table(mi, ctx):
    """Ranges of the rows hold sums of the tokens that a window leaves, not of all places of the table."""
    c = Big(mi, [20000, 16411], 2, 64, 128, seed=5)
    g = torch.Generator(DEV).manual_seed(6)
    q = torch.randn((2, 1100, 8, 128), generator=g, device=DEV).to(F16)
    size = ctx.kv_cache4_weights_workspace_size(c.cache, c.seqs, tensor(mi, q.transpose(1, 2)), 100)
    assert 0 < size <= 32 * 2 * 2 * (100 + 1100 + 320) * 4  # at most 32 ranges; 64 tokens where the first one begins and 256 to a workgroup
    check(mi, ctx, c, q, [1100, 1097], True, 100, F16, "kv_cache4_attn_128_halves")


@pytest.mark.parametrize("nq,heads,want", [(1, 16, "kv_cache4_attn_16"), (300, 16, "kv_cache4_attn_128"), (1501, 64, "kv_cache4_attn_128_halves")])
def test_kernels_past_4_gib(mi, ctx, nq, heads, want):
    """Every kernel over blocks that begin more than 4 GiB into the keys and the values."""
    c = Big(mi, [1800], 8, 128, 128, seed=nq, before=70000)
    q = torch.randn((1, nq, heads, 128), generator=torch.Generator(DEV).manual_seed(nq), device=DEV).to(F16)
    assert int(c.table[0, 0]) * 8 * 128 * 64 > 1 << 32
    check(mi, ctx, c, q, [nq], True, 0, F16, want)
