"""Every kernel of the cache's attention (16, 32 and 128 rows to a workgroup, one range of the tokens and several) against
float64, where the profile shows that the call took the kernel."""
import math

import pytest
import torch

import layer_refs as R
from layer_refs import F64, H, H0, U, tensor

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32
TYPES = [(F16, F16), (F32, F32), (F32, F16), (F16, F32)]
IDS = ["hh", "ff", "fh", "hf"]
# rows to a workgroup, whether the tokens' ranges are joined: sequences, key heads, group, queries, tokens that the table holds
CALLS = {(16, False): (3, 2, 4, 1, 320), (16, True): (2, 2, 1, 20, 960), (32, False): (1, 1, 7, 150, 512), (32, True): (2, 1, 7, 150, 960),
         (128, False): (2, 1, 8, 333, 320), (128, True): (1, 1, 7, 300, 640)}
KERNELS = sorted(CALLS)
NAMES = [f"{k}{'-joined' if j else ''}" for k, j in KERNELS]


def attend(mi, ctx, d, q, dst, scale, kernel, n_q=None, causal=True, window=0):
    """One call, and that it took this kernel and this many ranges: kernel = (rows, joined)."""
    ctx.profile(True)
    try:
        ctx.kv_cache_attn(d["cache"], d["seqs"], tensor(mi, q.transpose(1, 2)), tensor(mi, dst), scale,
                          n_q=0 if n_q is None else n_q.data_ptr(), causal=causal, window=window)
        took = ctx.profile_collect()
    finally:
        ctx.profile(False)
    assert list(took) == [f"kv_cache_attn_{kernel[0]}"]
    assert (ctx.kv_cache_attn_workspace_size(d["cache"], d["seqs"], tensor(mi, q.transpose(1, 2)), window) > 0) == kernel[1]


def exact(c, q, n_q, scale, causal, window, dtype):
    """(out, tolerance) [seqs, n_q, heads, D] in float64, rows past n_q NaN.

    Off by at most, with w the exact weights, W = sum w |v| and o the output:
      E = |scale| (sum |q k| (D + 3) U, for an F32 q with its two halves' 2^-22, + 2^-25 max |q| sum |k|, their range once the
        row's largest is between one and two) in a score;
      A = 2 U (|score| log2(e) + |log2 of the value scale| + 16) in exp2's argument, the reference and the lift in it: both
        move a weight's numerator and its part of the sum, 2 (E + A) W together;
      a weight enters its product as a half (F32 dst: as two): H relative, in the sum as well where that is of the halves,
        2 H W (2^-21 W); and 2^-25 where the largest is 2^8 at least: 2^-33 of the largest weighted step, 127 steps;
      thin blocks' weights of up to 2^-29 of the largest may leave the sum: n 2^-29 |o|;
      fp32 sums of n terms, 2 (n + 4) U W; and the output's own rounding."""
    S, NQ, NH, D = q.shape
    group = NH // c.heads
    out = torch.full((S, NQ, NH, D), math.nan, dtype=F64, device="cuda")
    tol = torch.zeros_like(out)
    q32, d32 = q.dtype == F32, dtype == F32
    for s in range(S):
        key, ok = c.values(s, "k")
        val, _ = c.values(s, "v")
        n, m = key.shape[1], min(max(int(n_q[s]), 0), NQ)
        if n == 0:
            out[s, :m] = 0.0
            continue
        vs = torch.zeros(c.heads, n, dtype=F64)  # value scale of every token
        for b in range((n + c.bt - 1) // c.bt):
            i = int(c.table[s, b])
            if 0 <= i < c.vs.shape[0]:
                vs[:, b * c.bt:(b + 1) * c.bt] = c.vs[i].to(F64)[:, None]
        key, val, ok, vs = key.cuda(), val.cuda(), ok.cuda(), vs.cuda()
        key, val = torch.where(ok[:, None], key, 0.0), torch.where(ok[:, None], val, 0.0)
        t, p = torch.arange(n, device="cuda"), n - m + torch.arange(m, device="cuda")
        seen = ok[None].expand(m, n).clone()
        if causal:
            seen &= t <= p[:, None]
        if window:
            seen &= t > p[:, None] - window
        for h in range(NH):
            kk, vv, sv, qq = key[h // group], val[h // group], vs[h // group], q[s, :m, h].cuda().to(F64)
            sc = scale * (qq @ kk.T)
            mag = (qq.abs() @ kk.abs().T) * abs(scale)
            w = torch.nan_to_num(torch.softmax(sc.masked_fill(~seen, -math.inf), -1))
            o = w @ vv
            W = w @ vv.abs()
            E = mag * ((D + 3) * U + (2.0 ** -22 if q32 else 0)) + (2.0 ** -25 * abs(scale) * qq.abs().amax(-1, keepdim=True) * kk.abs().sum(-1) if q32 else 0)
            A = 2 * U * (sc.abs() * 1.4427 + torch.where(sv > 0, torch.log2(sv.clamp(min=1e-300)).abs(), 0.0) + 16)
            EA = torch.where(seen, E + A, 0.0).amax(-1, keepdim=True)
            top = (w * sv).amax(-1, keepdim=True)
            tol[s, :m, h] = (W * (2 * EA + (2.0 ** -21 if d32 else 2 * H) + 2 * (n + 4) * U) + n * 2.0 ** -33 * 127 * top
                             + n * 2.0 ** -29 * o.abs() + (U * o.abs() if d32 else H * o.abs() + H0))
            out[s, :m, h] = o
    return out, tol


def check(mi, ctx, c, q, n_q, scale, kernel, dtype, causal=True, window=0):
    S, NQ, NH, D = q.shape
    d = c.on_gpu(mi)
    dst = torch.full((S, NQ, NH, D), 77.0, dtype=dtype, device="cuda")
    n = torch.tensor(n_q, dtype=torch.int32, device="cuda")
    attend(mi, ctx, d, q.cuda(), dst, scale, kernel, n, causal, window)
    want, tol = exact(c, q, n_q, scale, causal, window, dtype)
    got = dst.to(F64)
    past = want.isnan()
    assert (got[past] == 77).all()
    off = ((got - want).abs() / tol.clamp(min=1e-300))[~past]
    assert got.isfinite().all() and (off <= 1).all(), float(off.max())


def call(kernel, D, bt, qt, lens, seed, std=1.0):
    """Cache, queries and counts of a kernel's call; lens: lengths as parts of what the table holds."""
    S, kv, group, nq, most = CALLS[kernel]
    most = most // bt * bt
    c = R.Cache(S, most // bt, kv, bt, D, seed=seed).fill([int(most * x) for x in lens[:S]])
    q = (torch.randn((S, nq, kv * group, D), generator=torch.Generator().manual_seed(seed + 1)) * std).to(qt)
    return c, q, [nq] * S


@pytest.mark.parametrize("kernel", KERNELS, ids=NAMES)
@pytest.mark.parametrize("qt,ot", TYPES, ids=IDS)
def test_weights_do_not_depend_on_the_values_size(mi, ctx, kernel, qt, ot):
    """Blocks of small values beside others keep their tokens' part of the softmax's sum, however small: every second
    block's value scales are one ratio of the others', then ratios of all sizes mixed; the largest first and last."""
    for D, bt in ((64, 16), (96, 32), (128, 64)):
        for ratio in (2.0 ** -12, 2.0 ** -20, 2.0 ** -24, 1.5 * 2.0 ** -27, 2.0 ** -30, 1.5 * 2.0 ** -33, 2.0 ** -38, 2.0 ** -45, 2.0 ** -62, 2.0 ** -81, 0.0, None):
            c, q, n_q = call(kernel, D, bt, qt, (1.0, 0.77, 0.31), seed=D, std=0.3)
            for s in range(c.table.shape[0]):
                for b, i in enumerate(c.table[s].tolist()):
                    if ratio is None:
                        c.vs[i] *= 2.0 ** -((17 * b) % 64)
                    elif b % 2 == s % 2:
                        c.vs[i] *= ratio
            c.vs[:] = torch.where(c.vs < 1e-37, torch.where(c.vs.isnan(), c.vs, 0.0), c.vs)
            check(mi, ctx, c, q, n_q, D ** -0.5, kernel, ot)


@pytest.mark.parametrize("kernel", KERNELS, ids=NAMES)
@pytest.mark.parametrize("ot", [F32, F16], ids=["ff", "fh"])
def test_scales_at_the_ends_of_fp32(mi, ctx, kernel, ot):
    """Large queries at a scale of zero and over a cache of small keys, small ones over large keys: the scores are what
    their product says."""
    for D, bt in ((64, 16), (96, 32), (128, 64)):
        c, q, n_q = call(kernel, D, bt, F32, (0.97, 0.66, 0.83), seed=19)
        check(mi, ctx, c, q * 2.0 ** 119, n_q, 0.0, kernel, ot)
        keys = c.ks.clone()
        c.ks = keys * 2.0 ** -119
        check(mi, ctx, c, q * 2.0 ** 119, n_q, D ** -0.5, kernel, ot)
        c.ks = keys * 2.0 ** 119
        check(mi, ctx, c, q * 2.0 ** -132, n_q, 2.0 ** 10, kernel, ot)


WINDOWS = {(16, False): (1, 100), (16, True): (900,), (32, False): (1, 100), (32, True): (500, 700), (128, False): (1, 100), (128, True): (100, 300)}
SIZES = ((64, 16), (96, 32), (128, 64), (64, 128), (128, 16))
KERNEL = pytest.mark.parametrize("kernel", KERNELS, ids=NAMES)
TYPE = pytest.mark.parametrize("qt,ot", TYPES, ids=IDS)


@KERNEL
@TYPE
@pytest.mark.parametrize("D,bt", SIZES)
def test_causal_lengths(mi, ctx, kernel, D, bt, qt, ot):
    """Lengths at and off tiles' ends, of one token, of none, below the queries' number (the first see nothing); counts
    of all, a part and none of the queries."""
    for lens, part in (((1.0, 0.93, 0.5), (1, 1, 1)), ((0.999, 0.31, 0.7), (1, 0.5, 1)), ((0.07, 0.011, 0.002), (1, 1, 1)), ((0.004, 0, 0.4), (1, 1, 0)),
                       ((0.6, 0.21, 0.1), (0.17, 0.9, 1))):
        c, q, n_q = call(kernel, D, bt, qt, lens, seed=3)
        check(mi, ctx, c, q, [math.ceil(n * p) for n, p in zip(n_q, part)], D ** -0.5, kernel, ot)


@KERNEL
@TYPE
@pytest.mark.parametrize("D,bt", SIZES)
def test_masks_and_scales(mi, ctx, kernel, D, bt, qt, ot):
    """Every token seen, windows with and without the causal limit, negative scales and none, scores far apart."""
    c, q, n_q = call(kernel, D, bt, qt, (0.97, 0.66, 0.13), seed=5)
    check(mi, ctx, c, q, n_q, D ** -0.5, kernel, ot, causal=False)
    for window in WINDOWS[kernel]:
        check(mi, ctx, c, q, n_q, D ** -0.5, kernel, ot, causal=True, window=window)
        check(mi, ctx, c, q, n_q, D ** -0.5, kernel, ot, causal=False, window=window)
    for scale in (-0.2, 0.0, 2.0):
        check(mi, ctx, c, q, n_q, scale, kernel, ot)


@KERNEL
@TYPE
@pytest.mark.parametrize("D,bt", SIZES)
def test_blocks_that_are_not_there(mi, ctx, kernel, D, bt, qt, ot):
    """The first, some between, the last, all of a sequence's: left out.  Key scales of zero, value scales of zero, and
    scales that span twelve binades."""
    c, q, n_q = call(kernel, D, bt, qt, (0.97, 0.66, 0.83), seed=7)
    last = (int(c.n_kv[0]) - 1) // bt
    c.table[0, 0], c.table[0, min(3, last)], c.table[0, last] = -1, c.k.shape[0], -2 ** 31
    if c.table.shape[0] > 1:
        c.table[1, :] = -1
    ids = c.table[0].tolist()
    for b, i in enumerate(ids):
        if 0 <= i < c.k.shape[0]:
            c.vs[i] = c.vs[i] * 2.0 ** (b % 13 - 6) if b % 5 else torch.zeros(c.heads)
            if b % 7 == 1:
                c.ks[i] = 0.0
    c.vs[:] = torch.where(c.vs == 0, 0.0, c.vs)
    check(mi, ctx, c, q, n_q, D ** -0.5, kernel, ot)
    check(mi, ctx, c, q, n_q, D ** -0.5, kernel, ot, causal=False)


@KERNEL
@TYPE
@pytest.mark.parametrize("ks,vs", [(math.nan, 1.0), (1.0, math.nan), (math.inf, 1.0), (1.0, math.inf), (math.inf, math.inf)])
def test_scales_that_are_not_finite(mi, ctx, kernel, ks, vs, qt, ot):
    """Queries that see a token of such a block get NaN in every element, all others what they get without the block."""
    for D, bt in ((64, 16), (96, 32), (128, 64)):
        for window in (0, WINDOWS[kernel][-1]):
            c, q, n_q = call(kernel, D, bt, qt, (0.97, 0.8, 0.6), seed=11)
            S, NQ, NH, _ = q.shape
            want, tol = exact(c, q, n_q, D ** -0.5, True, window, ot)
            head, block = c.heads - 1, int(c.n_kv[0]) // bt - (1 if bt == 64 else 2)
            i = int(c.table[0, block])
            c.ks[i, head], c.vs[i, head] = ks, vs
            d = c.on_gpu(mi)
            dst = torch.full((S, NQ, NH, D), 77.0, dtype=ot, device="cuda")
            attend(mi, ctx, d, q.cuda(), dst, D ** -0.5, kernel, window=window)
            n = int(c.n_kv[0])
            p = n - NQ + torch.arange(NQ)
            sees = p >= block * bt
            if window:
                sees &= p - window < min(block * bt + bt, n) - 1
            hit = torch.zeros((S, NQ, NH), dtype=torch.bool)
            hit[0, :, head * (NH // c.heads):] = sees[:, None]
            got = dst.to(F64).cpu()
            assert hit.any() and got[hit].isnan().all()
            assert ((got - want.cpu()).abs() <= tol.cpu())[~hit].all()


@KERNEL
@TYPE
def test_orders_and_pitches(mi, ctx, kernel, qt, ot):
    """Queries in a product's rows and outputs at odd pitches and offsets: the bits of plain ones; what lies beside stays."""
    for D, bt in ((64, 16), (96, 32), (128, 64)):
        c, q, n_q = call(kernel, D, bt, qt, (0.97, 0.66, 0.83), seed=13)
        S, NQ, NH, _ = q.shape
        d = c.on_gpu(mi)
        want = torch.empty((S, NQ, NH, D), dtype=ot, device="cuda")
        attend(mi, ctx, d, q.cuda(), want, 0.11, kernel)
        for off in (0, 1, 2):
            wide = torch.zeros((NQ, S, NH, D + 5), dtype=qt, device="cuda")
            qd = wide.transpose(0, 1)[..., off:off + D]
            qd.copy_(q)
            out = torch.full((NH, S, NQ, D + 7), 5.0, dtype=ot, device="cuda")
            view = out.permute(1, 2, 0, 3)[..., off:off + D]
            attend(mi, ctx, d, qd, view, 0.11, kernel)
            assert torch.equal(view, want)
            view.fill_(5)
            assert (out == 5).all()


@KERNEL
def test_repeated_calls_have_the_same_bits(mi, ctx, kernel):
    c, q, n_q = call(kernel, 128, 16, F16, (1.0, 0.9, 0.8), seed=17)
    d, qd = c.on_gpu(mi), q.cuda()
    first = None
    for i in range(20):
        dst = torch.full(q.shape, float(i), dtype=F16, device="cuda")
        attend(mi, ctx, d, qd, dst, 0.1, kernel)
        first = dst if first is None else first
        assert torch.equal(dst, first)


def test_blocks_beyond_4_gib(mi, ctx):
    """Each kernel follows blocks that lie past 32 bits of offset in the cache as it follows near ones."""
    D, bt = 128, 64
    n = (1 << 32) // (bt * D) + 700
    k, v = (torch.empty(n * bt * D, dtype=torch.uint8, device="cuda") for _ in range(2))
    for kernel in KERNELS:
        c, q, n_q = call(kernel, D, bt, F16, (1.0, 0.77, 0.6), seed=23)
        near = c.on_gpu(mi)
        kv, blocks = c.heads, n // c.heads
        kf, vf = (x[:blocks * kv * bt * D].reshape(blocks, kv, bt, D) for x in (k, v))
        ks, vs = (torch.full((blocks, kv), math.nan, device="cuda") for _ in range(2))
        ids = near["table"].long().flatten()
        far = torch.arange(ids.numel(), device="cuda")
        far[1::2] = blocks - 1 - far[1::2]  # every second block at the far end
        kf[far], vf[far], ks[far], vs[far] = near["k"][ids], near["v"][ids], near["ks"][ids], near["vs"][ids]
        table = far.to(torch.int32).reshape(c.table.shape)
        there = dict(cache=mi.kv_cache(kf, vf, ks, vs), seqs=mi.kv_seqs(table, near["n_kv"]))
        want, got = (torch.full(q.shape, x, dtype=F16, device="cuda") for x in (1.0, 2.0))
        attend(mi, ctx, near, q.cuda(), want, 0.09, kernel)
        attend(mi, ctx, there, q.cuda(), got, 0.09, kernel)
        assert torch.equal(got, want)


@pytest.mark.parametrize("kernel", KERNELS, ids=NAMES)
def test_captured_and_replayed(mi, kernel):
    """Two graphs of one context over caches of their own, replayed in turn between its eager calls, also after a larger
    workspace has taken the place of theirs: the eager bits every time."""
    stream = torch.cuda.Stream()
    ctx = mi.Context(0, stream.cuda_stream)
    try:
        with torch.cuda.stream(stream):
            sets = []
            for seed in (29, 31):
                c, q, _ = call(kernel, 64, 16, F16, (1.0, 0.9, 0.7), seed=seed)
                d, qd = c.on_gpu(mi), q.cuda()
                want, out = (torch.zeros(q.shape, dtype=F16, device="cuda") for _ in range(2))
                sets.append((d, qd, want, out))
            args = lambda x, o: (x[0]["cache"], x[0]["seqs"], tensor(mi, x[1].transpose(1, 2)), tensor(mi, o), 0.125)  # noqa: E731
            ctx.reserve_workspace(max(ctx.kv_cache_attn_workspace_size(*args(x, x[3])[:3]) for x in sets))
            graphs = []
            for x in sets:
                stream.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    ctx.kv_cache_attn(*args(x, x[3]))
                graphs.append(graph)
                ctx.kv_cache_attn(*args(x, x[2]))
            for i in range(5):
                for x, graph in zip(sets, graphs):
                    x[3].fill_(i)
                    graph.replay()
                    ctx.kv_cache_attn(*args(sets[i & 1], sets[i & 1][2]))
                    stream.synchronize()
                    assert x[2].any() and torch.equal(x[3], x[2]), i
                ctx.reserve_workspace(1 << (20 + i))
    finally:
        ctx.close()
