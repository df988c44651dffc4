"""The operators around a layer's products on the GPU against float64 (layer_refs.py)."""
import math

import pytest
import torch

import layer_refs as R
from layer_refs import F64, H, H0, U, tensor

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


def rnd(seed, *shape, std=1.0, dtype=F32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


# ---------------------------------------------------------------- RMS norm
NORMS = [(1, 1), (3, 7), (5, 33), (2, 64), (7, 250), (4, 512), (3, 513), (9, 1024), (2, 2048), (3, 2056), (2, 4736), (1, 8192), (2, 8193), (1, 20000), (1, 32768)]


def norm_ref(x, add, w, eps):
    h = (x.float() + add.float()) if add is not None else x.float()
    y = h.to(F64) / torch.sqrt(h.to(F64).square().mean(-1, keepdim=True) + eps)
    return h, y * w.to(F64) if w is not None else y


@pytest.mark.parametrize("rows,n", NORMS)
@pytest.mark.parametrize("dtype", [F32, F16])
def test_rms_norm(mi, ctx, rows, n, dtype):
    """Eight roundings of half a fp32 step separate the passes from the exact norm of the fp32 sum: h's square,
    the mean and eps count half in the root; root, reciprocal, two products, and the mean's own rounding."""
    x, add, w = rnd(1, rows, n, std=2.0, dtype=dtype), rnd(2, rows, n, dtype=dtype), rnd(3, n) * 0.3 + 1
    for a, ww in ((add, w), (None, None)):
        h, y = norm_ref(x, a, ww, 1e-5)
        for out in (F32, F16):
            total, dst = torch.full_like(x, math.nan), torch.full((rows, n), math.nan, dtype=out, device="cuda")
            ctx.rms_norm(tensor(mi, x), tensor(mi, dst), 1e-5, add=tensor(mi, a) if a is not None else None,
                         w=ww.data_ptr() if ww is not None else 0, sum=tensor(mi, total))
            ctx.synchronize()
            assert torch.equal(total, h.to(dtype))
            tol = 8 * U * y.abs() + (H * y.abs() + H0 if out == F16 else 1e-44)
            assert ((dst.to(F64) - y).abs() <= tol).all(), float(((dst.to(F64) - y).abs() / tol).max())


@pytest.mark.parametrize("n", [32, 64, 96, 1024, 4736, 8192, 9216 + 32, 32768])
@pytest.mark.parametrize("dtype", [F32, F16])
def test_rms_norm_quantized(mi, ctx, n, dtype):
    """The 8-bit outputs are mi355_quantize_rows' bytes of the F32 output, and stand for it to half a step and
    the fp16 scale's rounding."""
    rows = 5
    x, add, w = rnd(4, rows, n, dtype=dtype), rnd(5, rows, n, dtype=dtype), rnd(6, n) * 0.3 + 1
    x[1] = 0
    add[1] = 0
    y = torch.empty((rows, n), device="cuda")
    args = dict(add=tensor(mi, add), w=w.data_ptr())
    ctx.rms_norm(tensor(mi, x), tensor(mi, y), 1e-6, **args)
    for t, size in ((mi.Q8_0, 34), (mi.Q8_1, 36)):
        got = torch.full((rows, n // 32 * size), 7, dtype=torch.uint8, device="cuda")
        want = torch.full_like(got, 9)
        ctx.rms_norm(tensor(mi, x), mi.from_torch(got, t, [n, rows]), 1e-6, **args)
        ctx.quantize_rows(t, mi.ACT_X86, tensor(mi, y), want.data_ptr())
        ctx.synchronize()
        assert torch.equal(got, want)
        for out in (F32, F16):
            back = torch.full((rows, n), math.nan, dtype=out, device="cuda")
            ctx.dequantize_rows(t, got.data_ptr(), tensor(mi, back))
            ctx.synchronize()
            top = y.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True).to(F64)
            tol = (top / 127 * (0.5 + 127 * (H + 4 * U)) + 128 * H0).expand(-1, -1, 32).flatten(-2)
            tol = tol + (H * y.abs() + H0 if out == F16 else 0)
            assert ((back.to(F64) - y.to(F64)).abs() <= tol).all()


def test_rms_norm_strides_and_places(mi, ctx):
    """Rows of a padded batch, four dimensions, in place; what lies between and behind the rows stays."""
    big = rnd(7, 2, 3, 4, 80)
    for dtype in (F32, F16):
        for n, off in ((64, 0), (64, 8), (64, 3), (37, 1)):
            x = big.to(dtype).clone()
            add = rnd(8, 2, 4, 3, n, dtype=dtype).transpose(1, 2)
            view = x[..., off:off + n]
            h, y = norm_ref(view, add, None, 1e-5)
            before = x.clone()
            dst = torch.full((2, 3, 4, 80), 5.0, device="cuda")
            ctx.rms_norm(tensor(mi, view), tensor(mi, dst[..., :n]), 1e-5, add=tensor(mi, add), sum=tensor(mi, view))
            ctx.synchronize()
            assert torch.equal(view, h.to(dtype))
            x[..., off:off + n] = before[..., off:off + n]
            assert torch.equal(x, before) and (dst[..., n:] == 5).all()
            assert ((dst[..., :n].to(F64) - y).abs() <= 8 * U * y.abs()).all()
            # the norm over its own input
            z = before.clone()
            ctx.rms_norm(tensor(mi, z[..., off:off + n]), tensor(mi, z[..., off:off + n]), 1e-5)
            _, y = norm_ref(before[..., off:off + n], None, None, 1e-5)
            ctx.synchronize()
            s, s0 = R.step(dtype)
            assert ((z[..., off:off + n].to(F64) - y).abs() <= (8 * U + s) * y.abs() + s0).all()
    q = torch.zeros((3, 40 * 34), dtype=torch.uint8, device="cuda")  # 8-bit rows at a wider pitch
    x = rnd(9, 3, 64)
    ctx.rms_norm(tensor(mi, x), mi.from_torch(q, mi.Q8_0, [64, 3], [34, 40 * 34, 120 * 34, 120 * 34]), 1e-5)
    y, want = torch.empty_like(x), torch.zeros((3, 68), dtype=torch.uint8, device="cuda")
    ctx.rms_norm(tensor(mi, x), tensor(mi, y), 1e-5)
    ctx.quantize_rows(mi.Q8_0, mi.ACT_X86, tensor(mi, y), want.data_ptr())
    ctx.synchronize()
    assert torch.equal(q[:, :68], want) and not q[:, 68:].any()


def test_rms_norm_special_values(mi, ctx):
    x = torch.zeros((6, 64), device="cuda")
    x[1, 3] = math.nan
    x[2, 5] = math.inf
    x[3] = 1e-30          # squares vanish in fp32
    x[4] = 1e19           # squares near the top of fp32
    x[5, 0] = -0.0
    y = torch.empty_like(x)
    ctx.rms_norm(tensor(mi, x), tensor(mi, y), 1e-5)
    ctx.rms_norm(tensor(mi, x[:0]), tensor(mi, y[:0]), 1e-5)  # no rows
    ctx.synchronize()
    assert torch.equal(y[0], x[0]) and y[1].isnan().all() and y[2, 5].isnan() and (y[2, :5] == 0).all()
    assert torch.allclose(y[3], torch.full((64,), 1e-30 / math.sqrt(1e-5), device="cuda"), rtol=1e-6, atol=0)
    assert torch.allclose(y[4], torch.ones(64, device="cuda"), rtol=1e-6) and not y[5].any()


@pytest.mark.parametrize("q8", ["Q8_0", "Q8_1"])
def test_rms_norm_special_values_in_eight_bits(mi, ctx, q8):
    """Rows with NaN and infinities become the blocks that the quantizer makes of the F32 norm: scales of NaN, not 0."""
    ty = getattr(mi, q8)
    x = rnd(11, 6, 96)
    x[1, 3] = math.nan
    x[2, 5] = math.inf
    x[3] = math.nan
    w = torch.ones(96, device="cuda")
    w[40], w[70] = math.nan, -math.inf
    bytes_ = 3 * (34 if q8 == "Q8_0" else 36)
    for weights in (None, w):
        y = torch.empty_like(x)
        got, want = (torch.full((6, bytes_), 0x55, dtype=torch.uint8, device="cuda") for _ in range(2))
        ctx.rms_norm(tensor(mi, x), tensor(mi, y), 1e-5, w=0 if weights is None else weights.data_ptr())
        ctx.rms_norm(tensor(mi, x), mi.from_torch(got, ty, [96, 6], [bytes_ // 3, bytes_, 6 * bytes_, 6 * bytes_]), 1e-5, w=0 if weights is None else weights.data_ptr())
        ctx.quantize_rows(ty, mi.ACT_X86, tensor(mi, y), want.data_ptr())
        ctx.synchronize()
        assert torch.equal(got, want)
        back = torch.zeros_like(x)
        ctx.dequantize_rows(ty, got.data_ptr(), tensor(mi, back))
        ctx.synchronize()
        assert back[1].isnan().all() and back[3].isnan().all()


@pytest.mark.parametrize("n", [32, 4736])
def test_dequantize_rows(mi, ctx, orc, n):
    import numpy as np
    x = rnd(10, 6, n)
    for t in (mi.Q8_0, mi.Q8_1, mi.Q4_0, mi.Q4_1):
        rows = torch.zeros((6, mi.row_size(t, n)), dtype=torch.uint8, device="cuda")
        if t == mi.Q8_1:
            ctx.quantize_rows(t, mi.ACT_X86, tensor(mi, x), rows.data_ptr())
        else:
            ctx.quantize_weights(t, tensor(mi, x), rows.data_ptr())
        ctx.synchronize()
        q, d, m = orc.decode_blocks(t, rows.cpu().numpy(), n)
        q, d = np.asarray(q, np.float32).reshape(6, -1, 32), np.asarray(d, np.float32).reshape(6, -1, 1)
        want = q * d  # each product and sum rounded to fp32
        if t == mi.Q4_1:
            want = want + np.asarray(m, np.float32).reshape(6, -1, 1)
        want = torch.from_numpy(want.reshape(3, 2, n)).cuda()
        for out in (F32, F16):
            dst = torch.full((2, 3, n + 4), 3.0, dtype=out, device="cuda").transpose(0, 1)
            ctx.dequantize_rows(t, rows.data_ptr(), tensor(mi, dst[..., :n]))
            ctx.synchronize()
            assert torch.equal(dst[..., :n], want.to(out)) and (dst[..., n:] == 3).all()


# ---------------------------------------------------------------- products of quantized rows
@pytest.mark.parametrize("M,N,K", [(1, 64, 32), (1, 4736, 1024), (5, 130, 96), (64, 1024, 512), (300, 257, 992), (1297, 771, 736), (5184, 288, 96)])
@pytest.mark.parametrize("wt", ["q8_0", "q4_0", "q4_1"])
def test_mul_mat_of_quantized_rows(mi, ctx, orc, M, N, K, wt):
    """The bits of the product of the F32 rows, on every route, with prepared weights and without allocation."""
    t = orc.NAME_TYPE[wt]
    at = mi.Q8_1 if wt == "q4_1" else mi.Q8_0
    w, x = rnd(11, N, K, std=0.05), rnd(12, M, K)
    rows = torch.zeros((N, mi.row_size(t, K)), dtype=torch.uint8, device="cuda")
    ctx.quantize_weights(t, tensor(mi, w), rows.data_ptr())
    x8 = torch.zeros((M, mi.row_size(at, K) + 4 * 36), dtype=torch.uint8, device="cuda")  # rows at a wider pitch
    flat = torch.zeros((M, mi.row_size(at, K)), dtype=torch.uint8, device="cuda")
    ctx.quantize_rows(at, mi.ACT_X86, tensor(mi, x), flat.data_ptr())
    ctx.synchronize()
    x8[:, :flat.shape[1]] = flat
    wide = x8.shape[1]
    src = mi.from_torch(x8, at, [K, M], [mi.TYPE_SIZE[at], wide, wide * M, wide * M])
    wt_ = mi.from_torch(rows, t, [K, N])
    want = torch.full((M, N), math.nan, device="cuda")
    ctx.mul_mat(wt_, tensor(mi, x), tensor(mi, want))
    buf = torch.empty(mi.weight_prepared_nbytes(wt_) + 256, dtype=torch.uint8, device="cuda")
    prep = ctx.weight_prepare(wt_, buf.data_ptr() + (-buf.data_ptr()) % 256, buf.numel() - 256)
    for kernel in (mi.MMQ_AUTO, mi.MMQ_F16, mi.MMQ_INT8):
        ctx.set_mmq_kernel(kernel)
        try:
            for ww, f in ((wt_, ctx.mul_mat), (prep, ctx.mul_mat), (wt_, ctx.mul_mat_noalloc)):
                got = torch.full((M, N), math.nan, device="cuda")
                f(ww, src, tensor(mi, got))
                ctx.synchronize()
                assert torch.equal(got, want)
        finally:
            ctx.set_mmq_kernel(mi.MMQ_AUTO)


def test_block_dots_of_quantized_rows(mi, ctx):
    M, N, K = 9, 40, 96
    w, x = rnd(13, N, K), rnd(14, M, K)
    rows, x8 = (torch.zeros((r, K // 32 * 34), dtype=torch.uint8, device="cuda") for r in (N, M))
    ctx.quantize_weights(mi.Q8_0, tensor(mi, w), rows.data_ptr())
    ctx.quantize_rows(mi.Q8_0, mi.ACT_X86, tensor(mi, x), x8.data_ptr())
    a, b = (torch.zeros((M, N, K // 32), dtype=torch.int32, device="cuda") for _ in range(2))
    wt = mi.from_torch(rows, mi.Q8_0, [K, N])
    ctx.mul_mat_block_dots(wt, tensor(mi, x), a.data_ptr())
    ctx.mul_mat_block_dots(wt, mi.from_torch(x8, mi.Q8_0, [K, M]), b.data_ptr())
    ctx.synchronize()
    assert a.any() and torch.equal(a, b)


# ---------------------------------------------------------------- rotary positions
ROPES = [dict(D=64, n_dims=64, sections=[32]), dict(D=128, n_dims=128, sections=[16, 24, 24], halves=True),
         dict(D=64, n_dims=64, sections=[16, 16], restart=True), dict(D=96, n_dims=96, sections=[16, 16, 16], interleaved=True, halves=True),
         dict(D=96, n_dims=64, sections=[8, 8, 8, 8], halves=True), dict(D=80, n_dims=20, sections=[3, 7]), dict(D=7, n_dims=6, sections=[0, 3], restart=True),
         dict(D=256, n_dims=256, sections=[128], halves=True), dict(D=2, n_dims=2, sections=[1])]


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("case", ROPES, ids=lambda c: "-".join(str(v) for v in c.values()))
def test_rope_multi(mi, ctx, case, dtype):
    """cos and sin are within 3 half steps of 1, each product and the sum within one of theirs: six of
    |a| + |b| in all; and the output's own rounding."""
    D, halves = case["D"], case.get("halves", False)
    kw = dict(restart=case.get("restart", False), order=1 if case.get("interleaved") else 0)
    p = mi.rope_params(case["n_dims"], case["sections"], 10000.0, pairs=1 if halves else 0, freq_scale=0.75, **kw)
    n, axes = case["n_dims"] // 2, len(case["sections"])
    for B, T, NH in ((1, 1, 1), (2, 5, 3), (1, 130, 17), (3, 1, 40)):
        g = torch.Generator(device="cuda").manual_seed(B * T)
        x = rnd(20, B, T, NH, D, dtype=dtype)
        pos = torch.randint(-200000, 200000, (axes, B, T), generator=g, device="cuda", dtype=torch.int32)
        pos[0, 0, 0] = 2 ** 31 - 1
        if T > 1:
            pos[-1, 0, 1] = -2 ** 31
        want = R.rope(x, R.angles(pos, case["sections"], case["n_dims"], 10000.0, kw["restart"], case.get("interleaved", False), 0.75), halves)
        mag = x.to(F64).abs()
        i = torch.arange(n, device="cuda") * (1 if halves else 2)
        j = i + (n if halves else 1)
        both = torch.zeros_like(mag)
        both[..., i] = both[..., j] = mag[..., i] + mag[..., j]
        s, s0 = R.step(dtype)
        tol = (6 * U + (s if dtype == F16 else 0)) * both + (s0 if dtype == F16 else 0)
        # odd strides (rows off 16 bytes), then a plain tensor, then in place
        wide = torch.full((B, T, NH, D + 1), 9.0, dtype=dtype, device="cuda")
        dst, same = torch.full_like(x, math.nan), x.clone()
        ctx.rope_multi(tensor(mi, x), pos.data_ptr(), p, tensor(mi, wide[..., :D]))
        ctx.rope_multi(tensor(mi, x), pos.data_ptr(), p, tensor(mi, dst))
        ctx.rope_multi(tensor(mi, same), pos.data_ptr(), p, tensor(mi, same))
        ctx.synchronize()
        assert ((dst.to(F64) - want).abs() <= tol).all(), float(((dst.to(F64) - want).abs() - tol).max())
        assert torch.equal(dst[..., 2 * n:], x[..., 2 * n:])
        assert torch.equal(dst, same) and torch.equal(dst, wide[..., :D]) and (wide[..., D:] == 9).all()


@pytest.mark.parametrize("base,scale", [(10000.0, 10.0), (10000.0, -0.5), (1.0, 0.3), (0.25, 1.0), (5e5, 0.0)])
def test_rope_multi_other_frequencies(mi, ctx, base, scale):
    """Turns of one and more a position, backwards, the same for every pair, growing with the pair, and none."""
    x = rnd(33, 1, 9, 2, 64)
    pos = torch.arange(-4, 5, dtype=torch.int32, device="cuda").reshape(1, 1, 9) * 1000003
    out = torch.empty_like(x)
    ctx.rope_multi(tensor(mi, x), pos.data_ptr(), mi.rope_params(64, [32], base, pairs=1, freq_scale=scale), tensor(mi, out))
    ctx.synchronize()
    # the float32 parameters as they are, and float64's own rounding of far angles
    f32 = lambda v: float(torch.tensor(v, dtype=F32))  # noqa: E731
    ang = R.angles(pos, [32], 64, f32(base), scale=f32(scale))
    both = x.abs().to(F64)
    both = both + both.roll(32, -1)
    far = torch.cat([ang, ang], -1).abs()[:, :, None] * 2.0 ** -51
    assert ((out.to(F64) - R.rope(x, ang, True)).abs() <= (6 * U + far) * both).all()


def test_rope_multi_is_the_image_encoders(mi, ctx):
    """Two axes with restart turn as the encoder's own table pass does (adjacent pairs, x first), to the table's rounding."""
    side, NH, hd = 6, 2, 64
    N = side * side
    f = 10000.0 ** (-4.0 * torch.arange(hd // 4, dtype=F64) / hd)
    t = torch.arange(N)
    ang = torch.cat([(t % side).to(F64)[:, None] * f, (t // side).to(F64)[:, None] * f], 1)
    table = torch.stack([torch.cos(ang), torch.sin(ang)], -1).float().cuda()
    qkv = rnd(30, N, 3 * NH * hd)
    q, k, v = (torch.empty((NH, N, hd), dtype=F16, device="cuda") for _ in range(3))
    bias = torch.zeros(3 * NH * hd, device="cuda")
    ctx.vit_qkv_rope(qkv.data_ptr(), bias.data_ptr(), table.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), N, N, NH, hd)
    x = qkv[:, :2 * NH * hd].reshape(1, N, 2 * NH, hd)  # queries and keys as heads of one view
    pos = torch.stack([t % side, t // side]).reshape(2, 1, N).to(torch.int32).cuda()
    out = torch.empty((1, N, 2 * NH, hd), device="cuda")
    ctx.rope_multi(tensor(mi, x), pos.data_ptr(), mi.rope_params(hd, [hd // 4, hd // 4], restart=True), tensor(mi, out))
    ctx.synchronize()
    want = torch.cat([q, k]).transpose(0, 1).to(F64)
    mag = x[0].abs().to(F64)
    both = mag + mag.unflatten(-1, (-1, 2)).flip(-1).flatten(-2)
    assert ((out[0].to(F64) - want).abs() <= (H + 12 * U) * both + H0).all()


def test_rope_multi_gradient(mi, ctx):
    """inverse is the transposed turn: against the formula's gradient, and against differences in float64 of the plain form."""
    B, T, NH, D = 2, 3, 4, 96
    x, g = rnd(31, B, T, NH, D), rnd(32, B, T, NH, D)
    pos = torch.arange(3 * B * T, dtype=torch.int32, device="cuda").reshape(3, B, T)
    kw = dict(n_dims=96, sections=[16, 16, 16], pairs=1)
    dx, back = torch.empty_like(x), x.clone()
    ctx.rope_multi(tensor(mi, g), pos.data_ptr(), mi.rope_params(inverse=True, **kw), tensor(mi, dx))
    for inverse in (False, True):
        ctx.rope_multi(tensor(mi, back), pos.data_ptr(), mi.rope_params(inverse=inverse, **kw), tensor(mi, back))
    ctx.synchronize()
    ang = R.angles(pos, [16, 16, 16], 96, 10000.0)
    mag = (g.to(F64).abs() + g.to(F64).abs().roll(48, -1))
    assert ((dx.to(F64) - R.rope(g, -ang, True)).abs() <= 6 * U * mag).all()
    mag = (x.to(F64).abs() + x.to(F64).abs().roll(48, -1))
    assert ((back - x).to(F64).abs() <= 2 * 12 * U * mag).all()
    for e in ((0, 0, 0, 0), (1, 2, 3, 47), (1, 0, 2, 95)):  # a difference quotient of a linear map is exact to rounding
        d = torch.zeros_like(x)
        d[e] = 1.0
        num = ((R.rope(x.to(F64) + d, ang, True) - R.rope(x.to(F64) - d, ang, True)) / 2 * g.to(F64)).sum()
        # two products of the gradient, six half steps of each, and float64's differences
        assert abs(float(num) - float(dx[e])) <= 6 * U * 2 * float(g.abs().max()) + 1e-9


# ---------------------------------------------------------------- the cache
def same_cache(c, d):
    assert torch.equal(d["ks"].cpu().view(torch.int32)[~c.ks.isnan()], c.ks.view(torch.int32)[~c.ks.isnan()])
    assert torch.equal(d["vs"].cpu().view(torch.int32)[~c.vs.isnan()], c.vs.view(torch.int32)[~c.vs.isnan()])
    assert torch.equal(d["ks"].cpu().isnan(), c.ks.isnan()) and torch.equal(d["vs"].cpu().isnan(), c.vs.isnan())
    assert torch.equal(d["k"].cpu(), c.k) and torch.equal(d["v"].cpu(), c.v)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("bt,D,heads", [(16, 64, 1), (32, 96, 3), (64, 128, 2), (128, 64, 2), (16, 128, 5), (128, 128, 1)])
def test_kv_cache_write(mi, ctx, bt, D, heads, dtype):
    """Bytes and scales equal those of the definition after every one of a run of writes of all lengths: into fresh
    blocks, behind kept tokens whose scale grows and does not, over several blocks, of nothing."""
    S, per = 4, 5
    c = R.Cache(S, per, heads, bt, D, seed=bt + D)
    c.table[2, 1] = -1                     # blocks that are not there
    c.table[3, 0] = c.k.shape[0]
    d = c.on_gpu(mi)
    g = torch.Generator().manual_seed(5)
    n_kv = [0] * S
    for step, new in enumerate([[1, 3, bt, 0], [1, bt - 3, 2, 1], [1, 1, 2 * bt, 2], [2 * bt + 1, bt, 0, bt + 5], [1, 1, 1, 1], [bt - 1, 0, 3, 7]]):
        n_kv = [min(a + b, per * bt) for a, b in zip(n_kv, new)]
        c.n_kv = torch.tensor(n_kv, dtype=torch.int32)
        d["n_kv"].copy_(c.n_kv)
        most = max(max(new), 1)
        k, v = ((torch.randn((S, heads, most, D), generator=g) * math.exp(0.7 * step * (-1) ** step)).to(dtype) for _ in range(2))
        c.write(k.float(), v.float(), new)
        kd = k.transpose(1, 2).contiguous().cuda().transpose(1, 2)  # a projection's order
        vd = torch.zeros((S, heads, most, D + 3), dtype=dtype, device="cuda")[..., 1:D + 1]
        vd.copy_(v)
        ctx.kv_cache_write(d["cache"], d["seqs"], tensor(mi, kd), tensor(mi, vd), n_new=torch.tensor(new, dtype=torch.int32, device="cuda").data_ptr())
        ctx.synchronize()
        same_cache(c, d)


def test_kv_cache_write_roundings(mi, ctx):
    """Ties go to even, also where the quotient's fp32 value is not the quotient; the smallest scales; zeros."""
    D, bt = 64, 16
    rows = torch.zeros((1, 1, 16, D))
    k = torch.arange(-63, 64, 2, dtype=F32)[:D] / 2
    cases = []
    for top in (127.0, 1.0, 3.3, 1e-3, 2.7e-37, 1e-42, 1.4e-45, 0.0, 3e38, 126.99999):
        d = torch.tensor(top) / torch.tensor(127.0)
        x = rows.clone()
        x[0, 0, 0] = k * d                               # halfway values, as near as fp32 has them
        for j, away in ((1, math.inf), (2, -math.inf)):  # and one step of fp32 to either side
            x[0, 0, j] = torch.nextafter(x[0, 0, 0], torch.full((D,), away))
        x[0, 0, 3, 0], x[0, 0, 3, 1] = top, -top
        x[0, 0, 4:] = (torch.rand((12, D), generator=torch.Generator().manual_seed(3)) * 2 - 1) * top
        x = x.clamp(-top, top)
        cases.append(x)
    for x in cases:
        c = R.Cache(1, 1, 1, bt, D)
        c.n_kv[0] = 16
        d = c.on_gpu(mi)
        c.write(x, x.flip(-1), [16])
        kd, vd = x.cuda(), x.flip(-1).contiguous().cuda()
        ctx.kv_cache_write(d["cache"], d["seqs"], tensor(mi, kd), tensor(mi, vd))
        ctx.synchronize()
        same_cache(c, d)


def test_kv_cache_write_of_non_finite_values(mi, ctx):
    """They spoil their own block and head, until it is written from its first row."""
    c = R.Cache(2, 3, 2, 16, 64)
    c.n_kv[:] = torch.tensor([40, 20])
    x = torch.randn((2, 2, 40, 64), generator=torch.Generator().manual_seed(1))
    x[0, 1, 17, 3], x[1, 0, 2, 9] = math.nan, math.inf
    x[1, :, 20:] = math.nan  # behind the last token: not read
    d = c.on_gpu(mi)
    xd, n_new = x.cuda(), torch.tensor([40, 20], dtype=torch.int32, device="cuda")
    ctx.kv_cache_write(d["cache"], d["seqs"], tensor(mi, xd), tensor(mi, xd), n_new=n_new.data_ptr())
    back = torch.full((2, 2, 40, 64), 5.0, device="cuda")
    ctx.kv_cache_read(d["cache"], d["seqs"], tensor(mi, back), None)
    ctx.synchronize()
    back = back.cpu()
    bad = torch.zeros((2, 2, 40), dtype=torch.bool)
    bad[0, 1, 16:32] = bad[1, 0, :16] = True
    there = torch.ones((2, 2, 40), dtype=torch.bool)
    there[1, :, 20:] = False
    assert (back[bad] != back[bad]).all() and (back[~there] == 5).all()
    ok = there & ~bad
    assert ((back - x)[ok].abs() <= 0.51 * 5 / 127).all()
    d["n_kv"].copy_(torch.tensor([32, 16]))  # the same blocks again, from their first rows
    y = torch.randn((2, 2, 16, 64), device="cuda")
    ctx.kv_cache_write(d["cache"], d["seqs"], tensor(mi, y), tensor(mi, y))
    ctx.kv_cache_read(d["cache"], d["seqs"], tensor(mi, back.cuda()), None)
    got = torch.zeros((2, 2, 16, 64), device="cuda")
    at = torch.stack([torch.arange(16, 32), torch.arange(16)]).to(torch.int32).cuda()
    ctx.kv_cache_read(d["cache"], d["seqs"], tensor(mi, got), None, pos=at.data_ptr())
    ctx.synchronize()
    assert ((got - y).abs() <= 0.51 * 5 / 127).all()


def test_kv_cache_write_takes_lengths_as_they_come(mi, ctx):
    """Counts beyond the rows, lengths below zero and beyond the table, more new tokens than the length."""
    c = R.Cache(5, 2, 1, 16, 64, seed=9)
    c.fill([20, 20, 20, 20, 20])
    d = c.on_gpu(mi)
    c.n_kv = torch.tensor([-3, 1000, 2, 25, 31], dtype=torch.int32)
    new = [4, 3, 5, 99, -2]
    x = torch.randn((5, 1, 5, 64), generator=torch.Generator().manual_seed(2))
    d["n_kv"].copy_(c.n_kv)
    c.write(x, -x, new)
    xd, yd = x.cuda(), (-x).cuda()
    ctx.kv_cache_write(d["cache"], d["seqs"], tensor(mi, xd), tensor(mi, yd), n_new=torch.tensor(new, dtype=torch.int32, device="cuda").data_ptr())
    ctx.synchronize()
    same_cache(c, d)


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("bt,D,heads", [(16, 64, 1), (32, 96, 3), (64, 128, 2), (128, 96, 2)])
def test_kv_cache_read(mi, ctx, bt, D, heads, dtype):
    S, per = 3, 4
    c = R.Cache(S, per, heads, bt, D)
    c.table[1, 1] = c.k.shape[0] + 5
    c.fill([3 * bt + 5, 2 * bt, 0])
    d = c.on_gpu(mi)
    n = 4 * bt
    ref = [c.values(s, w) for w in "kv" for s in range(S)]
    for pos in (None, torch.randint(-3, 4 * bt, (S, n), generator=torch.Generator().manual_seed(4)).to(torch.int32)):
        k = torch.full((S, n, heads, D), 9.0, dtype=dtype, device="cuda").transpose(1, 2)
        v = torch.full((S, heads, n, D + 1), 9.0, dtype=dtype, device="cuda")
        pd = pos.cuda() if pos is not None else None
        ctx.kv_cache_read(d["cache"], d["seqs"], tensor(mi, k), tensor(mi, v[..., :D]), pos=pd.data_ptr() if pos is not None else 0)
        ctx.synchronize()
        assert (v[..., D:] == 9).all()
        for i, got in enumerate((k, v[..., :D])):
            for s in range(S):
                val, ok = ref[i * S + s]
                p = pos[s].long() if pos is not None else torch.arange(n)
                there = (p >= 0) & (p < val.shape[1])
                there &= torch.cat([ok, torch.zeros(1, dtype=torch.bool)])[p.clamp(0, val.shape[1])]
                want = torch.full((heads, n, D), 9.0, dtype=dtype)
                want[:, there] = val[:, p[there]].float().to(dtype)
                assert torch.equal(got[s].cpu(), want)


# ---------------------------------------------------------------- attention over the cache
def check_attn(mi, ctx, c, q, n_q, scale, causal, window, dtype):
    S, NQ, NH, D = q.shape
    d = c.on_gpu(mi)
    qd = q.cuda()
    dst = torch.full((S, NQ, NH, D), 77.0, dtype=dtype, device="cuda")
    n = torch.tensor(n_q, dtype=torch.int32, device="cuda")
    ctx.kv_cache_attn(d["cache"], d["seqs"], tensor(mi, qd.transpose(1, 2)), tensor(mi, dst), scale, n_q=n.data_ptr(), causal=causal, window=window)
    ctx.synchronize()
    want, tol = c.attn(q, n_q, scale, causal, window, q.dtype == F32, dtype == F32)
    got = dst.cpu().to(F64)
    past = want.isnan()
    assert (got[past] == 77).all()
    off = (got - want).abs()[~past]
    assert got.isfinite().all() and (off <= tol[~past]).all(), float((off / tol[~past].clamp(min=1e-300)).max())
    return dst


TYPES = [(F16, F16), (F32, F32), (F32, F16), (F16, F32)]


@pytest.mark.parametrize("qt,ot", TYPES, ids=["hh", "ff", "fh", "hf"])
@pytest.mark.parametrize("D,bt", [(64, 16), (96, 32), (128, 64), (64, 128), (128, 16)])
@pytest.mark.parametrize("kv,group", [(1, 1), (2, 4), (1, 7), (2, 16), (1, 24)])
def test_attn_single_tokens(mi, ctx, D, bt, kv, group, qt, ot):
    """One query a sequence, lengths of none, one, around a block's and a step's end, and longer."""
    lens = [0, 1, bt - 1, bt, bt + 1, 63, 64, 65, 200, 333]
    c = R.Cache(len(lens), (333 + bt - 1) // bt, kv, bt, D, seed=D + bt).fill(lens)
    q = torch.randn((len(lens), 1, kv * group, D), generator=torch.Generator().manual_seed(6)).to(qt)
    check_attn(mi, ctx, c, q, [1] * len(lens), D ** -0.5, True, 0, ot)


@pytest.mark.parametrize("qt,ot", TYPES, ids=["hh", "ff", "fh", "hf"])
@pytest.mark.parametrize("D,bt,kv,group,nq,causal,window", [
    (64, 16, 2, 2, 3, True, 0), (128, 32, 1, 8, 5, True, 0), (96, 64, 2, 3, 17, True, 0), (64, 32, 1, 1, 70, True, 0),
    (128, 64, 2, 4, 67, True, 0), (128, 128, 1, 2, 150, True, 40), (64, 16, 1, 5, 33, False, 0), (96, 32, 2, 1, 130, False, 0),
    (64, 64, 1, 8, 40, True, 1), (96, 16, 1, 4, 9, False, 20), (128, 16, 1, 1, 300, True, 100)])
def test_attn_several_queries(mi, ctx, D, bt, kv, group, nq, causal, window, qt, ot):
    """Prompts, ragged and longer than what is cached (queries before the first token see nothing)."""
    lens, n_q = [190, 77, 30, 0, 333], [nq, max(nq // 2, 1), nq, nq, 0]
    c = R.Cache(5, (333 + bt - 1) // bt, kv, bt, D, seed=nq).fill(lens)
    q = torch.randn((5, nq, kv * group, D), generator=torch.Generator().manual_seed(7)).to(qt)
    check_attn(mi, ctx, c, q, n_q, D ** -0.5, causal, window, ot)


@pytest.mark.parametrize("nq", [1, 40, 200])
def test_attn_odd_caches(mi, ctx, nq):
    """Blocks that are not there are left out, also the first and all of them; scales of zero; values whose scales
    span thirty binades with the large ones out of sight; scores far apart."""
    D, bt = 64, 16
    c = R.Cache(4, 20, 2, bt, D, seed=3).fill([300, 290, 100, 160])
    c.table[0, 0], c.table[0, 7], c.table[1, 18] = -1, c.k.shape[0], -2 ** 31
    c.table[2] = -1
    ids = c.table[3].long()
    c.vs[ids[1]] = 0.0
    c.ks[ids[2]] = 0.0
    c.vs[ids[3:6]] = torch.tensor([1e-9, 1.0, 3e4])[:, None]
    c.k[ids[5]] = 128  # q . k = 0 there, and large elsewhere
    for qt, ot in ((F16, F32), (F32, F32)):
        q = (torch.randn((4, nq, 4, D), generator=torch.Generator().manual_seed(8)) * 3).to(qt)
        check_attn(mi, ctx, c, q, [nq] * 4, 0.5, nq > 1, 0, ot)


@pytest.mark.parametrize("nq", [16, 60, 300])
@pytest.mark.parametrize("qt,ot", TYPES[:2], ids=["hh", "ff"])
def test_attn_hides_what_is_not_finite(mi, ctx, nq, qt, ot):
    """A block spoilt by a NaN or an infinity reaches only the queries that see its tokens: none of those before it
    (causal), behind it (window) or of the other key head."""
    D, bt, n = 64, 16, 310
    for window, (ks, vs) in ((0, (math.nan, 1.0)), (40, (math.inf, math.nan)), (40, (1.0, math.inf))):
        c = R.Cache(1, 20, 2, bt, D, seed=11).fill([n])
        q = torch.randn((1, nq, 4, D), generator=torch.Generator().manual_seed(12)).to(qt)
        block = 18  # tokens 288 .. 303
        want, tol = c.attn(q, [nq], 0.125, True, window, qt == F32, ot == F32)
        i = int(c.table[0, block])
        c.ks[i, 1], c.vs[i, 1] = ks, vs
        d = c.on_gpu(mi)
        out = torch.full((1, nq, 4, D), 7.0, dtype=ot, device="cuda")
        qd = q.cuda()
        ctx.kv_cache_attn(d["cache"], d["seqs"], tensor(mi, qd.transpose(1, 2)), tensor(mi, out), 0.125, causal=True, window=window)
        ctx.synchronize()
        p = n - nq + torch.arange(nq)
        sees = p >= block * bt
        if window:
            sees &= p - window < block * bt + bt - 1
        got = out.cpu().to(F64)
        assert got[0, sees, 2:].isnan().any(-1).all() or not math.isnan(ks * vs)
        ok = torch.ones((nq, 4), dtype=torch.bool)
        ok[sees, 2:] = False
        assert ((got - want).abs() <= tol)[0, ok].all()


def test_far_blocks(mi, ctx):
    """A cache of more than 4 GiB: blocks at its end are written, read and attended to."""
    D, bt, heads = 128, 64, 8
    n = (1 << 32) // (bt * heads * D) + 700
    k, v = (torch.empty((n, heads, bt, D), dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.empty((n, heads), device="cuda") for _ in range(2))
    table = torch.tensor([[n - 1, 3, n - 2], [n - 600, n - 3, 0]], dtype=torch.int32, device="cuda")
    n_kv = torch.tensor([150, 190], dtype=torch.int32, device="cuda")
    cache, seqs = mi.kv_cache(k, v, ks, vs), mi.kv_seqs(table, n_kv)
    x = rnd(50, 2, heads, 190, D)
    new = n_kv.clone()
    ctx.kv_cache_write(cache, seqs, tensor(mi, x), tensor(mi, -x), n_new=new.data_ptr())
    kb, vb = torch.zeros_like(x), torch.zeros_like(x)
    ctx.kv_cache_read(cache, seqs, tensor(mi, kb), tensor(mi, vb))
    small = R.Cache(2, 3, heads, bt, D, extra=0)
    small.table = torch.arange(6, dtype=torch.int32).reshape(2, 3)
    small.n_kv = n_kv.cpu()
    small.write(x.cpu(), -x.cpu(), [150, 190])
    for nq in (1, 100):
        q = rnd(51, 2, nq, heads, D)
        out = torch.empty((2, nq, heads, D), device="cuda")
        ctx.kv_cache_attn(cache, seqs, tensor(mi, q.transpose(1, 2)), tensor(mi, out), 0.09)
        ctx.synchronize()
        want, tol = small.attn(q.cpu(), [nq, nq], 0.09, True, 0, True, True)
        assert ((out.cpu().to(F64) - want).abs() <= tol).all()
    for s, m in enumerate((150, 190)):
        assert torch.equal(kb[s, :, :m].cpu().to(F64), small.values(s, "k")[0].float().to(F64)) and torch.equal(vb[s, :, :m], -kb[s, :, :m])
        assert not kb[s, :, m:].any()


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_attn_scales(mi, ctx, scale):
    c = R.Cache(1, 10, 1, 32, 96).fill([300])
    for nq in (1, 90):
        q = torch.randn((1, nq, 2, 96), generator=torch.Generator().manual_seed(9))
        check_attn(mi, ctx, c, q, [nq], scale, True, 0, F32)


@pytest.mark.parametrize("nq,most,group", [(1, 9000, 4), (1, 40000, 1), (6, 5000, 2), (333, 3000, 1)])
def test_attn_long(mi, ctx, nq, most, group):
    """Lengths that are split over workgroups and joined again."""
    c = R.Cache(2, (most + 63) // 64, 1, 64, 64, seed=nq).fill([most, most // 3])
    q = torch.randn((2, nq, group, 64), generator=torch.Generator().manual_seed(10))
    check_attn(mi, ctx, c, q, [nq, nq], 0.125, True, 0, F32)
    check_attn(mi, ctx, c, q.half(), [nq, nq], 0.125, nq > 10, 0, F16)


def test_attn_strides(mi, ctx):
    """Queries and outputs in the orders that products leave and take, at odd offsets and pitches; n_q absent."""
    c = R.Cache(2, 8, 2, 16, 64).fill([100, 120])
    d = c.on_gpu(mi)
    for nq in (1, 33):
        base = rnd(40, 2, nq, 4, 64, dtype=F16)
        want = torch.empty((2, nq, 4, 64), dtype=F16, device="cuda")
        ctx.kv_cache_attn(d["cache"], d["seqs"], tensor(mi, base.transpose(1, 2)), tensor(mi, want), 0.125)
        for off in (0, 1, 4, 8):
            q = torch.zeros((2, 4, nq, 64 + 9), dtype=F16, device="cuda")[..., off:off + 64]
            q.copy_(base.transpose(1, 2))
            out = torch.full((nq, 2, 4, 80), 5.0, dtype=F16, device="cuda")
            ctx.kv_cache_attn(d["cache"], d["seqs"], tensor(mi, q), tensor(mi, out.transpose(0, 1)[..., off:off + 64]), 0.125)
            ctx.synchronize()
            assert torch.equal(out.transpose(0, 1)[..., off:off + 64], want)
            out[..., off:off + 64] = 5
            assert (out == 5).all()


def test_empty_calls(mi, ctx):
    """No sequences, no tokens, no blocks."""
    c = R.Cache(2, 1, 1, 16, 64).fill([3, 4])
    d = c.on_gpu(mi)
    before = d["k"].clone()
    none = torch.zeros((0, 1, 3, 64), device="cuda")
    one = torch.ones((2, 1, 3, 64), device="cuda")
    seqs0 = mi.kv_seqs(d["table"][:0].contiguous(), d["n_kv"][:0].contiguous())
    seqs0.table, seqs0.n_kv = d["table"].data_ptr(), d["n_kv"].data_ptr()
    empty = mi.make_tensor(one.data_ptr(), mi.F32, [64, 3, 1, 0])
    ctx.kv_cache_write(d["cache"], seqs0, empty, empty)
    ctx.kv_cache_read(d["cache"], seqs0, empty, empty)
    ctx.kv_cache_attn(d["cache"], seqs0, empty, mi.make_tensor(one.data_ptr(), mi.F32, [64, 1, 3, 0]), 1.0)
    nobody = mi.make_tensor(one.data_ptr(), mi.F32, [64, 0, 1, 2])
    ctx.kv_cache_write(d["cache"], d["seqs"], nobody, nobody)
    ctx.kv_cache_read(d["cache"], d["seqs"], nobody, None)
    ctx.kv_cache_attn(d["cache"], d["seqs"], nobody, mi.make_tensor(one.data_ptr(), mi.F32, [64, 1, 0, 2]), 1.0)
    bare = mi.kv_seqs(d["table"], d["n_kv"])
    bare.max_blocks = 0
    ctx.kv_cache_write(d["cache"], bare, tensor(mi, one), tensor(mi, one))
    out = torch.full((2, 3, 1, 64), 9.0, device="cuda")
    ctx.kv_cache_attn(d["cache"], bare, tensor(mi, one), tensor(mi, out), 1.0)
    p = mi.rope_params(64, [32])
    ctx.rope_multi(mi.make_tensor(one.data_ptr(), mi.F32, [64, 0, 5, 1]), d["n_kv"].data_ptr(), p, mi.make_tensor(one.data_ptr(), mi.F32, [64, 0, 5, 1]))
    ctx.rope_multi(mi.make_tensor(one.data_ptr(), mi.F32, [64, 2, 0, 1]), d["n_kv"].data_ptr(), p, mi.make_tensor(one.data_ptr(), mi.F32, [64, 2, 0, 1]))
    ctx.dequantize_rows(mi.Q8_0, one.data_ptr(), mi.make_tensor(one.data_ptr(), mi.F32, [64, 0]))
    ctx.synchronize()
    assert torch.equal(d["k"], before) and not none.numel() and (one == 1).all()
    assert not out.any()  # nothing to attend to
