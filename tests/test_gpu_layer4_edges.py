"""The operators of a layer with a 4-bit cache on the GPU at the ends of what they take: nothing at all, scales at the ends of
fp32, and sums over many rows."""
import math

import pytest
import torch

import layer4_refs as R4
from layer_refs import U, tensor
from test_gpu_layer4_ops import check_attn, close

pytestmark = pytest.mark.gpu
F16, F32, I32 = torch.float16, torch.float32, torch.int32


# ---------------------------------------------------------------- nothing to work on
def nothing_seen(mi, ctx, cache, seqs, S, nq, heads, D, dtype, causal, window):
    """An attention that sees no token gives zeros and an lse of -inf, and its weights' sums leave theirs."""
    q = torch.ones((S, heads, nq, D), dtype=dtype, device="cuda")
    out = torch.full((S, nq, heads, D), 9.0, dtype=dtype, device="cuda")
    lse = torch.full((S, nq, heads), 9.0, device="cuda")
    sums = torch.full((S, cache.n_head_kv, max(seqs.max_blocks, 1) * cache.block_tokens), 3.0, device="cuda")
    ctx.kv_cache4_attn(cache, seqs, tensor(mi, q), tensor(mi, out), 0.5, causal=causal, window=window, lse=lse.data_ptr())
    ctx.kv_cache4_weights(cache, seqs, tensor(mi, q), lse.data_ptr(), sums.data_ptr(), 0.5, causal=causal, window=window)
    ctx.synchronize()
    assert not out.any() and (lse == -math.inf).all() and (sums == 3).all()


# a single token, some, and as many as have the tokens' halves made before the attention in a longer table
@pytest.mark.parametrize("nq,heads,D", [(1, 4, 128), (40, 4, 96), (300, 4, 64), (4160, 32, 64)])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 70)])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_attn_without_blocks(mi, ctx, nq, heads, D, causal, window, dtype):
    """A table without blocks, a cache without, and sequences without tokens."""
    kv = heads // 4
    c = R4.Cache4(1, 2, kv, 64, D).fill([100])
    d = c.on_gpu(mi)
    bare = mi.kv_seqs(d["table"], d["n_kv"])
    bare.table, bare.max_blocks = None, 0
    nothing_seen(mi, ctx, d["cache"], bare, 1, nq, heads, D, dtype, causal, window)
    none = mi.KvCache4(None, None, None, None, 0, kv, 64, D)
    nothing_seen(mi, ctx, none, d["seqs"], 1, nq, heads, D, dtype, causal, window)
    d["n_kv"].zero_()
    nothing_seen(mi, ctx, d["cache"], d["seqs"], 1, nq, heads, D, dtype, causal, window)


def test_empty_calls(mi, ctx):
    """No sequences, no tokens or queries, no blocks: nothing is written but what says so."""
    c = R4.Cache4(2, 1, 1, 16, 64).fill([3, 4])
    d = c.on_gpu(mi)
    before = {n: d[n].clone() for n in ("k", "v", "ks", "vs")}
    one = torch.ones((2, 1, 3, 64), device="cuda")
    sums, out = torch.full((2, 1, 16), 2.0, device="cuda"), torch.full((2, 1, 16), 7.0, device="cuda")
    kept, n_out, lse = torch.full((2, 1, 3), -1, dtype=I32, device="cuda"), torch.full((2,), -5, dtype=I32, device="cuda"), torch.full((6,), 4.0, device="cuda")
    seqs0 = mi.KvSeqs(None, None, 0, 1)
    for ne_q, ne_d, s in (([64, 3, 1, 0], [64, 1, 3, 0], seqs0), ([64, 0, 1, 2], [64, 1, 0, 2], d["seqs"])):
        q, y = mi.make_tensor(None, mi.F32, ne_q), mi.make_tensor(None, mi.F32, ne_d)
        ctx.kv_cache4_write(d["cache"], s, q, q)
        ctx.kv_cache4_read(d["cache"], s, q, q)
        ctx.kv_cache4_read(d["cache"], s, None, q)
        ctx.kv_cache4_attn(d["cache"], s, q, y, 1.0, lse=lse.data_ptr())
        ctx.kv_cache4_weights(d["cache"], s, q, lse.data_ptr(), sums.data_ptr(), 1.0)
    ctx.kv_cache4_evict(d["cache"], seqs0, 0, 0, 3, 0, 0)
    bare = mi.KvSeqs(None, d["n_kv"].data_ptr(), 2, 0)
    none = mi.KvCache4(None, None, None, None, 0, 1, 16, 64)
    for cache, s in ((d["cache"], bare), (none, d["seqs"]), (none, bare)):
        ctx.kv_cache4_write(cache, s, tensor(mi, one), tensor(mi, one))
        ctx.kv_cache4_read(cache, s, tensor(mi, one), tensor(mi, one))
    ctx.kv_cache4_evict(d["cache"], bare, 0, 0, 3, 0, n_out.data_ptr())
    ctx.synchronize()
    assert n_out.tolist() == [0, 0]
    assert (sums == 2).all() and (out == 7).all() and (kept == -1).all() and (lse == 4).all() and (one == 1).all()
    assert all(torch.equal(d[n].view(torch.uint8), before[n].view(torch.uint8)) for n in before)
    # a cache without blocks under a table that has some: no token is there, so the lowest ones are kept
    sums[:] = torch.arange(16.0, device="cuda")
    ctx.kv_cache4_evict(none, d["seqs"], sums.data_ptr(), out.data_ptr(), 3, kept.data_ptr(), n_out.data_ptr(), recent=1)
    ctx.synchronize()
    assert n_out.tolist() == [3, 3] and kept.tolist() == [[[0, 1, 2]], [[0, 1, 3]]]
    assert out[0, 0].tolist() == [0, 1, 2] + [7] * 13 and out[1, 0].tolist() == [0, 1, 3, 0] + [7] * 12
    # none is kept
    kept.fill_(-1)
    ctx.kv_cache4_evict(d["cache"], d["seqs"], sums.data_ptr(), out.data_ptr(), 0, 0, n_out.data_ptr(), recent=1)
    ctx.synchronize()
    assert n_out.tolist() == [0, 0] and out[0, 0].tolist() == [0, 0, 0] + [7] * 13 and out[1, 0].tolist() == [0] * 4 + [7] * 12
    assert all(torch.equal(d[n].view(torch.uint8), before[n].view(torch.uint8)) for n in before)


# ---------------------------------------------------------------- scales at the ends of fp32
# (scale, size of the queries' elements or None: zeros, of the cache's): scores of a few units, or all zero
ENDS = [(1.4e-45, 1.0, 1.0), (1e-44, 1.0, 1.0), (-1e-42, 1.0, 1.0), (1e-43, 8e37, 2000.0), (-1e-41, 8e37, 40.0), (3e38, None, 1.0), (-3e38, 1e-38, 0.06)]


def at_the_end(scale, size, std, D, nq, dtype):
    scale = float(torch.tensor(scale, dtype=F32))
    c = R4.Cache4(1, 20, 1, 16, D, seed=5).fill([290], std=std)
    assert all(torch.isfinite(c.values(0, n)[0]).all() for n in "kv")
    q = torch.randn((1, nq, 2, D), generator=torch.Generator().manual_seed(nq))
    q = torch.zeros_like(q) if size is None else (q * size).clamp(-3e38, 3e38)
    if size is not None and size < 1:
        q[..., 0] = 2.0 ** -125  # the rows' largest elements are normal numbers
    return scale, c, q.to(dtype)


@pytest.mark.parametrize("scale,size,std", ENDS)
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("nq", [1, 140])
def test_attn_at_the_ends(mi, ctx, scale, size, std, D, nq):
    """Scales whose product with log2(e) is subnormal or infinite: the scores are what counts."""
    for dtype in (F32, F16):
        if dtype == F16 and size not in (None, 1.0):
            continue
        s, c, q = at_the_end(scale, size, std, D, nq, dtype)
        d = c.on_gpu(mi)
        for dt in (F16, F32):
            check_attn(mi, ctx, c, d, q, [nq], nq == 1, 0, dt, s)


@pytest.mark.parametrize("scale,size,std", ENDS)
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("nq", [1, 140])
def test_weights_at_the_ends(mi, ctx, scale, size, std, D, nq):
    """The same of the weights' sums, from the definition's logarithms."""
    for dtype in (F32, F16):
        if dtype == F16 and size not in (None, 1.0):
            continue
        s, c, q = at_the_end(scale, size, std, D, nq, dtype)
        d = c.on_gpu(mi)
        lse = c.attn(q, [nq], s, nq == 1, 0, dtype == F32, True)[2].float()
        add, tol = c.weights(q, [nq], lse, s, nq == 1, 0, dtype == F32)
        sums, qd, ld = torch.zeros(add.shape, device="cuda"), q.cuda().transpose(1, 2), lse.cuda()
        ctx.kv_cache4_weights(d["cache"], d["seqs"], tensor(mi, qd), ld.data_ptr(), sums.data_ptr(), s, causal=nq == 1)
        ctx.synchronize()
        close(sums.cpu(), add, tol + U * add)


# ---------------------------------------------------------------- sums over many rows
@pytest.mark.parametrize("seqs,blocks", [(16, 96), (4, 1)])
def test_weights_of_many_rows(mi, ctx, seqs, blocks):
    """32768 equal weights a token, in one range of the rows and in 32: 16 rows of a tile in a tree (4 additions deep), 32
    tiles one after another, then those (32 of one range; 2 of each of 32, which are 32 more), and two lanes' sums: no
    sum is more than 4 + 32 + 32 + 2 + 1 roundings deep, where one tile after another would be 1024.
    A weight is e^-lse, whose exponent is off by 4 U (log2(e), its product with the scale, their quotient, lse's product) and
    the exponential by 2 U: 7 U of it with lse up to 1.1.  (One tile after another is off by 7 to 214 U in these
    values, as fp32 on the CPU gives.)"""
    nq, heads, kv = 4096, 32, 4
    c = R4.Cache4(seqs, 1, kv, 128, 64).fill([64] * seqs)
    d = c.on_gpu(mi)
    table = torch.full((seqs, blocks), -1, dtype=I32, device="cuda")
    table[:, :1] = d["table"]
    q = torch.zeros((seqs, heads, nq, 64), dtype=F16, device="cuda")
    one = 0.1 + torch.arange(seqs * kv, device="cuda").reshape(seqs, 1, kv, 1) / (seqs * kv)
    lse = one.expand(seqs, nq, kv, heads // kv).reshape(seqs, nq, heads).contiguous()
    sums = torch.zeros((seqs, kv, blocks * 128), device="cuda")
    s = mi.kv_seqs(table, d["n_kv"])
    ctx.kv_cache4_weights(d["cache"], s, tensor(mi, q), lse.data_ptr(), sums.data_ptr(), 0.125, causal=False)
    ctx.synchronize()
    want = (nq * heads // kv * torch.exp(-one.reshape(seqs, kv, 1).double())).cpu()
    got = sums.cpu().double()
    assert (got[..., 64:] == 0).all()
    assert ((got[..., :64] - want).abs() <= (71 + 7) * U * want).all(), float(((got[..., :64] - want).abs() / want).max() / U)
