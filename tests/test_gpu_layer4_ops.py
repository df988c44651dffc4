"""The operators of a layer with a 4-bit cache on the GPU against float64 (layer4_refs.py)."""
import math

import pytest
import torch

import layer_refs as R
import layer4_refs as R4
from layer_refs import F64, U, tensor

pytestmark = pytest.mark.gpu
F16, F32, I32 = torch.float16, torch.float32, torch.int32


def ints(x):
    return torch.tensor(x, dtype=I32, device="cuda")


# ---------------------------------------------------------------- norms and rotation
def qk_ref(x, w, eps, ang, halves):
    y = x.to(F64) / torch.sqrt(x.to(F64).square().mean(-1, keepdim=True) + eps)
    return R.rope(y * w.to(F64) if w is not None else y, ang, halves)


def qk_close(got, x, w, eps, ang, halves):
    """The squares' sum is off by (log2 of the lanes + 8) U, the root, quotient and products by 5 U, each counted of the
    pair's magnitude; a turn adds cos and sin to 2^-23 and three roundings: 24 U of |a| + |b| in all."""
    y = qk_ref(x, w, eps, ang, halves)
    n = ang.shape[-1]
    z = qk_ref(x, w, eps, torch.zeros_like(ang), halves).abs()
    i0 = torch.arange(n) * (1 if halves else 2)
    i1 = i0 + (n if halves else 1)
    pair = z.clone()
    pair[..., i0] = pair[..., i1] = z[..., i0] + z[..., i1]
    s, s0 = R.step(got.dtype)
    tol = 24 * U * pair + s * y.abs() * (got.dtype == F16) + s0
    assert ((got.cpu().to(F64) - y).abs() <= tol).all(), float(((got.cpu().to(F64) - y).abs() / tol).max())


QKS = [(64, 64, [32], {}), (128, 128, [64], {}), (96, 96, [48], {}), (128, 64, [16, 16], dict(restart=True)), (96, 96, [12, 18, 18], {}),
       (64, 64, [12, 10, 10], dict(order=1)), (256, 256, [128], {}), (80, 40, [20], {}), (33, 10, [5], {}), (7, 2, [1], {}), (250, 18, [9], {}),
       (256, 10, [5], {}), (64, 64, [32], dict(inverse=True)), (2, 2, [1], {})]


@pytest.mark.parametrize("ne0,n_dims,sections,kw", QKS)
@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("src,out", [(F32, F32), (F32, F16), (F16, F16), (F16, F32)])
def test_qk_norm_rope(mi, ctx, ne0, n_dims, sections, kw, halves, src, out):
    """Queries and keys as parts of one product's rows, every type; what lies beside them stays."""
    g = torch.Generator().manual_seed(ne0)
    for B, T, H, KV in ((2, 3, 5, 2), (1, 1, 1, 1)):
        x = (torch.randn((B, T, (H + 2 * KV) * ne0), generator=g) * 2).to(src)
        w = [1 + 0.2 * torch.randn(ne0, generator=g) for _ in range(2)]
        pos = torch.randint(-5, 100000, (len(sections), B, T), generator=g, dtype=I32)
        ang = R.angles(pos, sections, n_dims, 10000.0, kw.get("restart", False), kw.get("order", 0) == 1)
        ang = -ang if kw.get("inverse") else ang
        p = mi.rope_params(n_dims, sections, pairs=int(halves), **kw)
        xd, wd, pd = x.cuda(), [y.cuda() for y in w], pos.cuda()
        parts = xd.split([H * ne0, KV * ne0, KV * ne0], -1)
        qs, ks = (y.unflatten(-1, (-1, ne0)) for y in parts[:2])
        qd, kd = torch.full((B, T, H, ne0 + 3), 9.0, dtype=out, device="cuda"), torch.full((B, KV, T, ne0), 9.0, dtype=out, device="cuda").transpose(1, 2)
        ctx.qk_norm_rope(tensor(mi, qs), tensor(mi, ks), 1e-6, pd.data_ptr(), p, tensor(mi, qd[..., :ne0]), tensor(mi, kd), q_w=wd[0].data_ptr(),
                         k_w=wd[1].data_ptr())
        ctx.synchronize()
        xq, xk = x[..., :H * ne0].unflatten(-1, (-1, ne0)), x[..., H * ne0:(H + KV) * ne0].unflatten(-1, (-1, ne0))
        qk_close(qd[..., :ne0], xq, w[0], 1e-6, ang, halves)
        qk_close(kd, xk, w[1], 1e-6, ang, halves)
        assert (qd[..., ne0:] == 9).all() and torch.equal(xd.cpu(), x)
        # one side alone, without a weight; in place
        ctx.qk_norm_rope(None, tensor(mi, ks), 1e-6, pd.data_ptr(), p, None, tensor(mi, kd))
        ctx.synchronize()
        qk_close(kd, xk, None, 1e-6, ang, halves)
        if src == out:
            ctx.qk_norm_rope(tensor(mi, qs), tensor(mi, ks), 1e-6, pd.data_ptr(), p, tensor(mi, qs), tensor(mi, ks), q_w=wd[0].data_ptr())
            ctx.synchronize()
            qk_close(qs, xq, w[0], 1e-6, ang, halves)
            qk_close(ks, xk, None, 1e-6, ang, halves)
            assert torch.equal(parts[2].cpu(), x[..., (H + KV) * ne0:])


def test_qk_norm_rope_many_heads(mi, ctx):
    """Enough heads for several to a thread, a count that four do not divide, and no tokens or heads at all."""
    for H, KV, D in ((13, 3, 64), (32, 8, 128), (6, 0, 96)):
        B, T = 2, 1100
        x = torch.randn((B, T, H + KV, D), generator=torch.Generator().manual_seed(H))
        pos = torch.arange(T, dtype=I32).expand(1, B, T).contiguous()
        ang, p = R.angles(pos, [D // 2], D, 10000.0), mi.rope_params(D, [D // 2], pairs=1)
        xd, pd = x.cuda(), pos.cuda()
        q, k = torch.zeros((B, T, H, D), device="cuda"), torch.zeros((B, T, KV, D), device="cuda")
        ctx.qk_norm_rope(tensor(mi, xd[:, :, :H]), tensor(mi, xd[:, :, H:]), 1e-6, pd.data_ptr(), p, tensor(mi, q), tensor(mi, k))
        ctx.qk_norm_rope(tensor(mi, xd[:, :0, :H]), None, 1e-6, 0, p, tensor(mi, q[:, :0]), None)
        ctx.synchronize()
        qk_close(q, x[:, :, :H], None, 1e-6, ang, True)
        qk_close(k, x[:, :, H:], None, 1e-6, ang, True)


def test_qk_norm_rope_special_values(mi, ctx):
    """Zeros, one NaN or infinity spoil their own head only; squares beyond fp32 give zeros as their mean's root does."""
    x = torch.ones((1, 1, 6, 64))
    x[0, 0, 0] = 0
    x[0, 0, 1, 5] = math.nan
    x[0, 0, 2, 7] = math.inf
    x[0, 0, 3] = 1e20
    x[0, 0, 4] = 1e-25
    xd, y, pos = x.cuda(), torch.empty((1, 1, 6, 64), device="cuda"), torch.zeros((1, 1, 1), dtype=I32, device="cuda")
    ctx.qk_norm_rope(tensor(mi, xd), None, 1e-6, pos.data_ptr(), mi.rope_params(64, [32]), tensor(mi, y), None)
    ctx.synchronize()
    y = y.cpu()[0, 0]
    assert (y[0] == 0).all() and y[1].isnan().all() and y[2, 7].isnan() and (y[3] == 0).all()
    assert torch.allclose(y[4], torch.full((64,), 1e-22), rtol=1e-5) and torch.allclose(y[5], torch.ones(64), rtol=1e-5)


# ---------------------------------------------------------------- the cache
def same_bits(a, b):
    """Equal halves, NaN of any kind alike."""
    a, b = a.cpu(), b.cpu()
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a[~a.isnan()].view(torch.int16), b[~b.isnan()].view(torch.int16))


def same_cache(c, d):
    assert torch.equal(d["k"].cpu(), c.k) and torch.equal(d["v"].cpu(), c.v)
    assert same_bits(d["ks"], c.ks) and same_bits(d["vs"], c.vs)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("bt,D,heads", [(16, 64, 1), (32, 96, 3), (64, 128, 2), (128, 64, 2), (16, 128, 5), (128, 96, 1)])
def test_write(mi, ctx, bt, D, heads, dtype):
    """Bytes and scales equal those of the definition after every one of a run of writes, and nothing else changes."""
    S, per = 4, 5
    c = R4.Cache4(S, per, heads, bt, D, seed=bt + D)
    c.table[2, 1] = -1                     # blocks that are not there
    c.table[3, 0] = c.k.shape[0]
    d = c.on_gpu(mi)
    g = torch.Generator().manual_seed(5)
    n_kv = [0] * S
    for step, new in enumerate([[1, 3, bt, 0], [1, bt - 3, 2, 1], [2 * bt + 1, bt, 0, bt + 5], [bt - 1, 0, 3, 7]]):
        n_kv = [min(a + b, per * bt) for a, b in zip(n_kv, new)]
        c.n_kv = torch.tensor(n_kv, dtype=I32)
        d["n_kv"].copy_(c.n_kv)
        most = max(max(new), 1)
        k, v = ((torch.randn((S, heads, most, D), generator=g) * math.exp(0.7 * step * (-1) ** step)).to(dtype) for _ in range(2))
        c.write(k.float(), v.float(), new)
        kd = k.transpose(1, 2).contiguous().cuda().transpose(1, 2)  # a projection's order
        vd = torch.zeros((S, heads, most, D + 3), dtype=dtype, device="cuda")[..., 1:D + 1]
        vd.copy_(v)
        ctx.kv_cache4_write(d["cache"], d["seqs"], tensor(mi, kd), tensor(mi, vd), n_new=ints(new).data_ptr())
        ctx.synchronize()
        same_cache(c, d)
    # more new tokens than the sequence has, and counts and lengths out of range
    c.n_kv = torch.tensor([3, -4, per * bt + 9, 2], dtype=I32)
    d["n_kv"].copy_(c.n_kv)
    x = torch.randn((S, heads, 7, D), generator=g).to(dtype)
    c.write(x.float(), x.float(), [7, 2, 99, -3])
    xd = x.cuda()
    ctx.kv_cache4_write(d["cache"], d["seqs"], tensor(mi, xd), tensor(mi, xd), n_new=ints([7, 2, 99, -3]).data_ptr())
    ctx.synchronize()
    same_cache(c, d)


def test_write_roundings(mi, ctx):
    """Ties go to even, also beside fp32's own steps, for either sign; the ends of the scales' range; zeros."""
    D = 64
    for top in (8.0, 1.0, -3.3, 1e-3, -2.5e-5, 1e-6, 2.4e-7, 1e-7, 1e-30, 0.0, 255 * 256.0, 65407.9, -65408.0, 3e38):
        d = R4.group_scale(torch.full((1, 32), top))[0].float()
        x = torch.zeros((1, 1, 16, D))
        x[0, 0, 0] = (torch.arange(D) % 16 - 7.5) * (d if d == d else 1.0)     # halfway values
        for j, away in ((1, math.inf), (2, -math.inf)):                       # and one step of fp32 to either side
            x[0, 0, j] = torch.nextafter(x[0, 0, 0], torch.full((D,), away))
        x[0, 0, 3, 1], x[0, 0, 3, 40] = top, -top
        x[0, 0, 4, 2] = top
        x[0, 0, 4, 3] = -top                                                  # the positive one of two
        x[0, 0, 5:] = (torch.rand((11, D), generator=torch.Generator().manual_seed(3)) * 2 - 1) * top
        x = x.clamp(-abs(top), abs(top))
        x[0, 0, :3, 0] = x[0, 0, :3, 32] = top
        c = R4.Cache4(1, 1, 1, 16, D)
        c.n_kv[0] = 16
        dev = c.on_gpu(mi)
        c.write(x, x.flip(-1), [16])
        kd, vd = x.cuda(), x.flip(-1).contiguous().cuda()
        ctx.kv_cache4_write(dev["cache"], dev["seqs"], tensor(mi, kd), tensor(mi, vd))
        ctx.synchronize()
        same_cache(c, dev)


@pytest.mark.parametrize("D", [64, 96, 128])
def test_write_of_non_finite_values(mi, ctx, D):
    """They spoil their own token and head, keys and values, and nothing beside them."""
    c = R4.Cache4(2, 3, 2, 16, D)
    c.n_kv[:] = torch.tensor([40, 20])
    x = torch.randn((2, 2, 40, D), generator=torch.Generator().manual_seed(1))
    y = torch.randn((2, 2, 40, D), generator=torch.Generator().manual_seed(2))
    x[0, 1, 17, 3], x[1, 0, 2, D - 1], y[0, 0, 5, 33], y[1, 1, 7, 0] = math.nan, math.inf, -math.inf, math.nan
    x[0, 0, 9] = math.nan
    x[1, :, 20:] = math.nan  # behind the last token: not read
    d = c.on_gpu(mi)
    xd, yd = x.cuda(), y.cuda()
    c.write(x, y, [40, 20])
    ctx.kv_cache4_write(d["cache"], d["seqs"], tensor(mi, xd), tensor(mi, yd), n_new=ints([40, 20]).data_ptr())
    ctx.synchronize()
    same_cache(c, d)
    bad = torch.zeros((2, 2, 48), dtype=torch.bool)
    bad[0, 1, 17] = bad[1, 0, 2] = bad[0, 0, 5] = bad[1, 1, 7] = bad[0, 0, 9] = True
    for s in range(2):
        for n in "kv":
            val, _ = c.values(s, n)
            assert torch.equal(val.isnan().any(-1), bad[s, :, :c.length(s)]) and torch.equal(val.isnan().all(-1), bad[s, :, :c.length(s)])


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("bt,D,heads", [(16, 64, 2), (32, 96, 1), (64, 128, 3)])
def test_read(mi, ctx, bt, D, heads, dtype):
    """The values themselves, in order or by position; what is not there is left as it was."""
    c = R4.Cache4(3, 4, heads, bt, D).fill([3 * bt + 5, 1, 4 * bt])
    c.table[0, 1] = -7
    d = c.on_gpu(mi)
    T = 4 * bt + 3
    for pos in (None, torch.randint(-2, 4 * bt + 2, (3, T), generator=torch.Generator().manual_seed(3), dtype=I32)):
        k, v = (torch.full((3, T, heads, D + 5), 7.0, dtype=dtype, device="cuda") for _ in range(2))
        at = pos.cuda() if pos is not None else None
        kv = [tensor(mi, x[..., 2:D + 2].transpose(1, 2)) for x in (k, v)]
        ctx.kv_cache4_read(d["cache"], d["seqs"], kv[0], kv[1], pos=at.data_ptr() if at is not None else 0)
        ctx.synchronize()
        for x, n in ((k, "k"), (v, "v")):
            want = torch.full(x.shape, 7.0, dtype=F64)
            for s in range(3):
                val, ok = c.values(s, n)
                p = torch.arange(T) if pos is None else pos[s].long()
                there = (p >= 0) & (p < val.shape[1])
                there[there.clone()] &= ok[p[there]]
                want[s, there, :, 2:D + 2] = val[:, p[there]].transpose(0, 1)
            assert torch.equal(x.cpu().to(F64), want)
        ctx.kv_cache4_read(d["cache"], d["seqs"], None, kv[0], pos=at.data_ptr() if at is not None else 0)  # values alone
        ctx.synchronize()
        there = k[..., 2:D + 2] != 7.0
        assert torch.equal(k[..., 2:D + 2][there], v[..., 2:D + 2][there])


# ---------------------------------------------------------------- attention
def attend(mi, ctx, c, d, q, n_q, causal, window, dt, scale=None, lse=True):
    S, NQ, NH, D = q.shape
    qd = q.transpose(1, 2).contiguous().cuda() if NQ % 2 else q.cuda().transpose(1, 2)  # [S, NH, NQ, D] in either order
    dst = torch.full((S, NQ, NH, D), math.nan, dtype=dt, device="cuda")
    l = torch.full((S, NQ, NH), math.nan, device="cuda")
    ctx.kv_cache4_attn(d["cache"], d["seqs"], tensor(mi, qd), tensor(mi, dst), D ** -0.5 if scale is None else scale, n_q=ints(n_q).data_ptr(),
                       causal=causal, window=window, lse=l.data_ptr() if lse else 0)
    ctx.synchronize()
    return dst.cpu(), l.cpu()


def close(got, want, tol, what=""):
    a = got.to(F64)
    assert torch.equal(a.isnan(), want.isnan()), what
    inf = want.isinf()
    assert torch.equal(a[inf], want[inf]), what
    ok = ~want.isnan() & ~inf
    d = (a[ok] - want[ok]).abs()
    assert (d <= tol[ok]).all(), (what, float((d / tol[ok]).max()))


def check_attn(mi, ctx, c, d, q, n_q, causal, window, dt, scale=None):
    out, tol, lse, ltol = c.attn(q, n_q, q.shape[-1] ** -0.5 if scale is None else scale, causal, window, q.dtype == F32, dt == F32)
    got, l = attend(mi, ctx, c, d, q, n_q, causal, window, dt, scale)
    close(got, out, tol, "out")
    close(l, lse, ltol, "lse")
    again, _ = attend(mi, ctx, c, d, q, n_q, causal, window, dt, scale, lse=False)  # the same bits, with or without lse
    assert torch.equal(got.nan_to_num(0.0), again.nan_to_num(0.0))
    return got, l


# sequences' lengths, queries, heads, key heads, D, block, causal, window
ATTNS = [([1], 1, 1, 1, 64, 16, True, 0), ([777], 1, 16, 2, 64, 16, True, 0), ([0, 5], 1, 4, 4, 128, 32, True, 0),
         ([200, 33, 64], 1, 8, 1, 128, 64, True, 0), ([130, 257], 3, 5, 5, 96, 128, True, 0), ([95, 400], 7, 6, 2, 96, 16, True, 50),
         ([300], 40, 4, 2, 128, 32, True, 0), ([150, 20], 64, 2, 1, 64, 64, False, 0), ([513, 129], 130, 4, 2, 128, 64, True, 0),
         ([260], 300, 2, 2, 64, 16, True, 100), ([300, 1], 33, 7, 1, 96, 32, False, 0), ([1100], 2, 2, 1, 64, 128, True, 1),
         ([640, 600], 160, 2, 1, 96, 32, True, 0), ([257], 129, 8, 8, 64, 16, False, 64)]


@pytest.mark.parametrize("q_type,d_type", [(F16, F16), (F16, F32), (F32, F16), (F32, F32)])
@pytest.mark.parametrize("n_kv,nq,heads,kv,D,bt,causal,window", ATTNS)
def test_attn(mi, ctx, n_kv, nq, heads, kv, D, bt, causal, window, q_type, d_type):
    S = len(n_kv)
    per = max(n_kv) // bt + 2
    c = R4.Cache4(S, per, kv, bt, D, seed=nq).fill(n_kv)
    d = c.on_gpu(mi)
    q = (torch.randn((S, nq, heads, D), generator=torch.Generator().manual_seed(nq + D)) * 1.5).to(q_type)
    check_attn(mi, ctx, c, d, q, [nq] + [max(nq - 2, 0)] * (S - 1), causal, window, d_type)


@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("nq", [1, 20, 150])
def test_attn_over_missing_blocks_and_nan(mi, ctx, D, nq):
    """Blocks that are not there are not seen; a NaN token spoils the queries that see it and no others, also where its
    values alone were not finite; what lies behind a sequence's end never shows."""
    S, bt, kv = 3, 16, 2
    n_kv = [200, 161, 30]
    c = R4.Cache4(S, 14, kv, bt, D, seed=D).fill(n_kv)
    c.table[0, 2], c.table[0, 5], c.table[1, 0] = -1, c.k.shape[0] + 4, -9
    c.table[2, :2] = -1                     # nothing at all: zeros
    bad = torch.full((1, kv, D), 1.0)
    bad[0, 1, 3] = math.nan                 # key head 1 only
    c.set(1, 140, torch.ones((1, kv, D)), bad)
    d = c.on_gpu(mi)
    q = torch.randn((S, nq, 4, D), generator=torch.Generator().manual_seed(1))
    for dt in (F16, F32):
        for causal, window in ((True, 0), (True, 12), (False, 0)):
            got, lse = attend(mi, ctx, c, d, q, [nq] * S, causal, window, dt)
            w, tol, wl, ltol = c.attn(q, [nq] * S, D ** -0.5, causal, window, True, dt == F32)
            n = c.length(1)
            pos = n - nq + torch.arange(nq)
            sees = (pos >= 140) if causal else torch.ones(nq, dtype=torch.bool)
            if window:
                sees &= pos - window < 140
            w[1, :, 2:] = torch.where(sees[:, None, None], math.nan, w[1, :, 2:])
            wl[1, :, 2:] = torch.where(sees[:, None], math.nan, wl[1, :, 2:])
            if not sees.all():              # the others, without that token's NaN in the products
                e = R4.Cache4(S, 14, kv, bt, D, seed=D).fill(n_kv)
                e.table = c.table
                w2, tol2, wl2, ltol2 = e.attn(q, [nq] * S, D ** -0.5, causal, window, True, dt == F32)
                w[1], wl[1] = torch.where(w[1].isnan() & ~sees[:, None, None], w2[1], w[1]), torch.where(wl[1].isnan() & ~sees[:, None], wl2[1], wl[1])
                tol[1], ltol[1] = torch.where(sees[:, None, None], tol[1], tol2[1]), torch.where(sees[:, None], ltol[1], ltol2[1])
            close(got, w, tol, (causal, window))
            close(lse, wl, ltol, (causal, window))
            assert (got[2] == 0).all() and (lse[2] == -math.inf).all()


def test_attn_large_and_small(mi, ctx):
    """Scores far apart, scales of any size and sign, queries of any size: what the formula gives."""
    for D, std, qs, scale in ((64, 300.0, 1.0, 0.125), (128, 1e-3, 100.0, 0.7), (96, 1.0, 30.0, -0.3), (64, 1e3, 1e-6, 1.0), (128, 1.0, 1.0, 0.0)):
        c = R4.Cache4(1, 20, 1, 16, D, seed=3).fill([300], std=std)
        d = c.on_gpu(mi)
        for nq in (1, 140):
            q = torch.randn((1, nq, 2, D), generator=torch.Generator().manual_seed(2)) * qs
            for dt in (F16, F32):
                check_attn(mi, ctx, c, d, q, [nq], True, 0, dt, scale)


def test_attn_many_ranges(mi, ctx):
    """A long sequence beside short ones: several ranges, joined by the last workgroup; the same bits each time."""
    c = R4.Cache4(2, 160, 1, 128, 64, seed=8)
    c.n_kv[:] = torch.tensor([20000, 3], dtype=I32)
    g = torch.Generator().manual_seed(4)
    q8 = torch.randint(0, 256, c.k.shape, generator=g, dtype=torch.uint8)
    c.k, c.v = q8, q8.flip(-1)
    c.ks = (torch.rand(c.ks.shape, generator=g) * 0.2).bfloat16().half()
    c.vs = (torch.rand(c.vs.shape, generator=g) - 0.5).bfloat16().half()
    d = c.on_gpu(mi)
    for nq in (1, 5):
        q = torch.randn((2, nq, 3, 64), generator=g)
        got, _ = check_attn(mi, ctx, c, d, q, [nq] * 2, True, 0, F32)
        for _ in range(3):
            assert torch.equal(attend(mi, ctx, c, d, q, [nq] * 2, True, 0, F32)[0], got)


# ---------------------------------------------------------------- the weights' sums
@pytest.mark.parametrize("q_type", [F16, F32])
@pytest.mark.parametrize("n_kv,nq,heads,kv,D,bt,causal,window", ATTNS)
def test_weights(mi, ctx, n_kv, nq, heads, kv, D, bt, causal, window, q_type):
    S, per = len(n_kv), max(n_kv) // bt + 2
    c = R4.Cache4(S, per, kv, bt, D, seed=nq).fill(n_kv)
    c.table[0, min(1, per - 1)] = -1
    d = c.on_gpu(mi)
    q = (torch.randn((S, nq, heads, D), generator=torch.Generator().manual_seed(nq + D)) * 1.5).to(q_type)
    n_q = [nq] + [max(nq - 2, 0)] * (S - 1)
    _, lse = attend(mi, ctx, c, d, q, n_q, causal, window, F32)
    add, tol = c.weights(q, n_q, lse, D ** -0.5, causal, window, q_type == F32)
    before = torch.rand(add.shape, generator=torch.Generator().manual_seed(6)) * 3
    qd, ld = q.cuda().transpose(1, 2), lse.cuda()
    runs = []
    for _ in range(2):
        sums = before.cuda()
        ctx.kv_cache4_weights(d["cache"], d["seqs"], tensor(mi, qd), ld.data_ptr(), sums.data_ptr(), D ** -0.5, n_q=ints(n_q).data_ptr(), causal=causal,
                              window=window)
        ctx.synchronize()
        runs.append(sums.cpu())
    assert torch.equal(runs[0], runs[1])
    want = before.to(F64) + add
    assert torch.equal(runs[0][add == 0], before[add == 0])
    close(runs[0], want, tol + U * want)
    # the weights of a row are one in all
    total = (runs[0].to(F64) - before.to(F64)).sum()
    rows = int(torch.isfinite(lse).sum())
    assert abs(float(total) - rows) <= 1e-3 * max(rows, 1)


def test_weights_of_nan(mi, ctx):
    """A NaN token's queries give NaN to what they see; hidden tokens and other heads keep their numbers."""
    c = R4.Cache4(1, 8, 2, 16, 64).fill([100])
    bad = torch.ones((1, 2, 64))
    bad[0, 0, 1] = math.inf
    c.set(0, 60, bad, torch.ones((1, 2, 64)))
    d = c.on_gpu(mi)
    q = torch.randn((1, 50, 2, 64), generator=torch.Generator().manual_seed(1)).half()
    _, lse = attend(mi, ctx, c, d, q, [50], True, 0, F16)
    sums = torch.zeros((1, 2, 128), device="cuda")
    qd, ld = q.cuda().transpose(1, 2), lse.cuda()
    ctx.kv_cache4_weights(d["cache"], d["seqs"], tensor(mi, qd), ld.data_ptr(), sums.data_ptr(), 0.125)
    ctx.synchronize()
    s = sums.cpu()[0]
    assert s[0, :100].isnan().all() and (s[:, 100:] == 0).all() and torch.isfinite(s[1]).all()
    assert abs(float(s[1].sum()) - 50) < 1e-3


# ---------------------------------------------------------------- eviction
def evict(mi, ctx, c, d, sums, n_keep, max_keep, first, recent):
    S = c.table.shape[0]
    out, kept = torch.full(sums.shape, 7.0), torch.full((S, c.heads, max_keep), -1, dtype=I32)
    n = torch.full((S,), -5, dtype=I32, device="cuda")
    sd, od, kd = sums.cuda(), out.cuda(), kept.cuda()
    keep = ints(n_keep) if n_keep is not None else None
    ctx.kv_cache4_evict(d["cache"], d["seqs"], sd.data_ptr(), od.data_ptr(), max_keep, kd.data_ptr(), n.data_ptr(),
                        n_keep=keep.data_ptr() if keep is not None else 0, first=first, recent=recent)
    ctx.synchronize()
    want = c.evict(sums, n_keep if n_keep is not None else [max_keep] * S, first, recent, out, kept)
    assert n.tolist() == want
    assert torch.equal(kd.cpu(), kept)
    assert torch.equal(od.cpu().nan_to_num(-3.0), out.nan_to_num(-3.0)) and torch.equal(od.cpu().isnan(), out.isnan())
    same_cache(c, d)
    assert torch.equal(sd.cpu().nan_to_num(-3.0), sums.nan_to_num(-3.0))


def weights_like(shape, kind, seed=3):
    g = torch.Generator().manual_seed(seed)
    w = torch.exp(2.5 * torch.randn(shape, generator=g))
    if kind == "ties":
        w = torch.randint(0, 3, shape, generator=g).float()
    elif kind == "zeros":
        w = torch.where(torch.rand(shape, generator=g) < 0.9, 0.0, w)
    elif kind == "odd":  # signs, both zeros, infinities and NaN
        w = torch.randn(shape, generator=g)
        for i, x in enumerate((0.0, -0.0, math.inf, -math.inf, math.nan, 1e-42, -1e-42)):
            w = torch.where(torch.rand(shape, generator=g) < 0.06, x, w)
    return w


@pytest.mark.parametrize("kind", ["plain", "ties", "zeros", "odd"])
@pytest.mark.parametrize("bt,D,heads", [(16, 64, 1), (32, 96, 3), (64, 128, 2)])
def test_evict(mi, ctx, bt, D, heads, kind):
    n_kv = [5 * bt + 3, 2 * bt, 1, 0, 6 * bt]
    for n_keep, max_keep, first, recent in (([2 * bt, bt - 1, 1, 4, 3 * bt + 2], 3 * bt + 2, 2, bt), (None, bt + 5, 0, 0), ([0, 1, 0, 0, 6 * bt], 6 * bt, 4, 3),
                                            ([bt, 2 * bt + 1, -3, 9, 10], bt, 1000, 1000), (None, 0, 1, 1), ([7, 7, 7, 7, 7], 7, 5, 7)):
        c = R4.Cache4(5, 6, heads, bt, D, seed=D).fill(n_kv)
        d = c.on_gpu(mi)
        evict(mi, ctx, c, d, weights_like((5, heads, 6 * bt), kind), n_keep, max_keep, first, recent)


def test_evict_missing_blocks(mi, ctx):
    """Their tokens go first; one that is kept all the same leaves a NaN key, one that moves there is lost."""
    for n_keep in (60, 100, 110):
        c = R4.Cache4(1, 8, 2, 16, 64, seed=1).fill([120])
        c.table[0, 1], c.table[0, 4] = -1, 99
        d = c.on_gpu(mi)
        evict(mi, ctx, c, d, weights_like((1, 2, 128), "plain"), [n_keep], 128, 20, 70 if n_keep == 110 else 5)


@pytest.mark.parametrize("n", [1023, 1024, 1025, 5000, 40000])
def test_evict_long(mi, ctx, n):
    """More tokens than a workgroup has threads, with its steps' ends everywhere; random bytes stand for the tokens."""
    bt, per = 128, (n + 127) // 128
    c = R4.Cache4(1, per, 1, bt, 64, seed=n)
    c.n_kv[0] = n
    d = c.on_gpu(mi)
    for kind, keep in (("plain", n // 2), ("ties", n - 1), ("zeros", n // 3)):
        sums = weights_like((1, 1, per * bt), kind, seed=n)
        evict(mi, ctx, c, d, sums, [keep], n, 4, min(100, n // 4))


# ---------------------------------------------------------------- streams, graphs, far blocks
def test_on_another_stream_and_in_graphs(mi):
    """A context of its own stream; two graphs of one context, replayed in turn with eager work between."""
    st = torch.cuda.Stream()
    ctx = mi.Context(0, st.cuda_stream)
    c = R4.Cache4(2, 40, 2, 64, 128, seed=5).fill([1500, 700])
    d = c.on_gpu(mi)
    q = torch.randn((2, 1, 8, 128), generator=torch.Generator().manual_seed(2)).half()
    n_q = [1, 1]
    want, tol, wl, ltol = c.attn(q, n_q, 0.1, True, 0, False, False)
    add, wtol = c.weights(q, n_q, wl.float(), 0.1, True, 0, False)
    qd, dst, lse, nq = q.cuda().transpose(1, 2), torch.zeros((2, 1, 8, 128), dtype=F16, device="cuda"), torch.zeros((2, 1, 8), device="cuda"), ints(n_q)
    sums = torch.zeros((2, 2, 40 * 64), device="cuda")
    torch.cuda.synchronize()
    T = lambda x: tensor(mi, x)  # noqa: E731
    ctx.reserve_workspace(ctx.kv_cache4_attn_workspace_size(d["cache"], d["seqs"], T(qd)))

    def attn():
        ctx.kv_cache4_attn(d["cache"], d["seqs"], T(qd), T(dst), 0.1, n_q=nq.data_ptr(), lse=lse.data_ptr())

    def weigh():
        ctx.kv_cache4_weights(d["cache"], d["seqs"], T(qd), lse.data_ptr(), sums.data_ptr(), 0.1, n_q=nq.data_ptr())

    with torch.cuda.stream(st):
        attn()
        weigh()
        ctx.synchronize()
        graphs = []
        for f in (attn, weigh):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                f()
            graphs.append(g)
        close(dst.cpu(), want, tol)
        for _ in range(4):
            dst.zero_(), lse.zero_(), sums.zero_()
            graphs[0].replay()
            graphs[1].replay()
            torch.cuda.synchronize()
            close(dst.cpu(), want, tol)
            close(lse.cpu(), wl, ltol)
            got = sums.cpu().to(F64)
            assert ((got - add).abs() <= wtol + 2 * ltol.max() * add + 1e-30).all()
            attn()
            ctx.synchronize()
    ctx.close()


def test_blocks_past_4_gib(mi, ctx):
    """Offsets beyond 32 bits: tokens in the last blocks of a cache of 5 GiB a side."""
    n, heads, bt, D = 80000, 8, 128, 128
    k, v = (torch.empty((n, heads, bt, D // 2), dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = torch.zeros((n, heads, bt, 4), dtype=F16, device="cuda"), torch.zeros((n, heads, 4, bt), dtype=F16, device="cuda")
    table = ints([[n - 1, 3, n - 2]])
    n_kv = ints([300])
    cache, seqs = mi.kv_cache4(k, v, ks, vs), mi.kv_seqs(table, n_kv)
    x, y = (torch.randn((1, heads, 300, D), device="cuda", generator=torch.Generator("cuda").manual_seed(i)) for i in range(2))
    ctx.kv_cache4_write(cache, seqs, tensor(mi, x), tensor(mi, y))
    c = R4.Cache4(1, 3, heads, bt, D)
    c.table, c.n_kv = torch.tensor([[0, 1, 2]], dtype=I32), torch.tensor([300], dtype=I32)
    c.write(x.cpu(), y.cpu(), [300])
    back = torch.zeros((1, heads, 300, D), device="cuda")
    ctx.kv_cache4_read(cache, seqs, tensor(mi, back), None)
    q = torch.randn((1, 2, heads, D), generator=torch.Generator().manual_seed(9)).half()
    ctx.synchronize()
    assert torch.equal(back.cpu()[0].to(F64), c.values(0, "k")[0])
    d = {"cache": cache, "seqs": seqs}
    check_attn(mi, ctx, c, d, q, [2], True, 0, F16)
    sums, out = torch.rand((1, heads, 384), device="cuda"), torch.zeros((1, heads, 384), device="cuda")
    kept, m = torch.zeros((1, heads, 200), dtype=I32, device="cuda"), ints([0])
    ctx.kv_cache4_evict(cache, seqs, sums.data_ptr(), out.data_ptr(), 200, kept.data_ptr(), m.data_ptr())
    ctx.synchronize()
    old = c.values(0, "v")[0]
    ctx.kv_cache4_read(cache, mi.kv_seqs(table, m), None, tensor(mi, back))
    ctx.synchronize()
    for h in range(heads):
        assert torch.equal(back.cpu()[0, h, :200].to(F64), old[h, kept.cpu()[0, h].long()])


# ---------------------------------------------------------------- many heads to a key head, scales of any sign
def check_weights(mi, ctx, c, d, q, n_q, causal, window, scale):
    _, lse = attend(mi, ctx, c, d, q, n_q, causal, window, F32, scale)
    add, tol = c.weights(q, n_q, lse, scale, causal, window, q.dtype == F32)
    sums, qd, ld = torch.zeros(add.shape, device="cuda"), q.cuda().transpose(1, 2), lse.cuda()
    ctx.kv_cache4_weights(d["cache"], d["seqs"], tensor(mi, qd), ld.data_ptr(), sums.data_ptr(), scale, n_q=ints(n_q).data_ptr(), causal=causal, window=window)
    ctx.synchronize()
    close(sums.cpu(), add, tol + U * add)


@pytest.mark.parametrize("q_type", [F16, F32])
@pytest.mark.parametrize("nq,heads,kv,causal,window", [(1, 71, 1, True, 0), (5, 80, 2, True, 0), (30, 33, 1, True, 40), (3, 130, 1, False, 0), (64, 48, 1, True, 9)])
def test_many_heads_of_a_key_head(mi, ctx, nq, heads, kv, causal, window, q_type):
    """More heads to a key head than a step of the kernels has rows."""
    c = R4.Cache4(2, 12, kv, 32, 64, seed=heads).fill([300, 77])
    d = c.on_gpu(mi)
    q = torch.randn((2, nq, heads, 64), generator=torch.Generator().manual_seed(nq)).to(q_type)
    check_attn(mi, ctx, c, d, q, [nq, max(nq - 1, 1)], causal, window, q_type)
    check_weights(mi, ctx, c, d, q, [nq, max(nq - 1, 1)], causal, window, 0.125)


@pytest.mark.parametrize("q_type", [F16, F32])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-30, 0.7])
def test_weights_of_any_scale(mi, ctx, scale, q_type):
    c = R4.Cache4(1, 20, 2, 16, 128, seed=4).fill([290])
    d = c.on_gpu(mi)
    for nq in (1, 90):
        q = torch.randn((1, nq, 4, 128), generator=torch.Generator().manual_seed(nq)).to(q_type)
        check_weights(mi, ctx, c, d, q, [nq], True, 0, scale)
