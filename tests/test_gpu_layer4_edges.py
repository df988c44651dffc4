"""The operators of a layer with a 4-bit cache on the GPU at the ends of what they take: nothing at all."""
import math

import pytest
import torch

import layer4_refs as R4
from layer_refs import tensor

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
