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
