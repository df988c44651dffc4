"""The work of a transformer layer that keeps its tokens in a quantized cache.

Around the quantized products such a layer calls, per step: the residual's addition with a
root-mean-square norm whose output is the product's 8-bit operand; rotary positions over one to
three axes (text; time, height and width of video); the write of new keys and values into a cache of
one byte an element with a scale for each block of tokens and head, and its reading back; and the
attention over that cache, for single tokens and for prompts or frames.  Sizes are those of decoders
and of the image encoders here (5184 tokens a frame, head sizes 64, 96 and 128).

listed() names the cases, draw() gives others of the same ranges, prepare() makes what a program
holds before the call, run() is one pass, work() the bytes and operations that pass cannot do
without, exact() the same pass in float64.  Where `own` is false run() is the plain form.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

DEV = "cuda"
F16, F32, F64, I32 = torch.float16, torch.float32, torch.float64, torch.int32
TYPES = {"f16": F16, "f32": F32}
EPS = 1e-5
MOST_NORM = 8192 * 4736                  # elements of the largest listed norm
MOST_ROPE = 20736 * 16 * 64              # elements of the largest listed rotation
MOST_CACHE = 4 * 5200 * 8 * 128          # elements of the largest listed write or read, keys or values
MOST_TOKEN = 32 * 16384 * 8 * 128        # cached keys' elements of the largest single-token attention
MOST_PAIRS = 2 * 32 * 4096 * 5120        # query-key pairs of the largest listed prompt


def _package():
    """This repository's package, from the working folder."""
    name = "sam3_cpp_amd"
    if name not in sys.modules:
        path = os.path.join(os.getcwd(), "sam3.cpp_amd", "__init__.py")
        spec = importlib.util.spec_from_file_location(name, path)
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


def listed():
    return [
        # a decoder's single token before its first product: launch latency
        {"name": "norm_q8_token", "kind": "norm", "rows": 1, "n": 4096, "type": "f32", "out": "q8_0", "residual": True},
        # a frame's tokens at the image encoder's width, into a Q8_0 / Q4_0 product
        {"name": "norm_q8_frame", "kind": "norm", "rows": 5184, "n": 1024, "type": "f32", "out": "q8_0", "residual": True},
        # a long prompt at an odd width in half precision, into an F16 product
        {"name": "norm_f16_prompt", "kind": "norm", "rows": 8191, "n": 4736, "type": "f16", "out": "f16", "residual": True},
        # one token of each of many conversations, text and image positions, queries and keys in one tensor
        {"name": "rope_tokens", "kind": "rope", "batch": 32, "tokens": 1, "heads": 40, "D": 128, "type": "f16", "axes": 3, "halves": True},
        # four frames of 72 x 72 patches with axial positions
        {"name": "rope_frames", "kind": "rope", "batch": 4, "tokens": 5184, "heads": 16, "D": 64, "type": "f32", "axes": 2, "halves": False},
        # one token of each of 64 conversations into their last blocks
        {"name": "cache_token", "kind": "write", "seqs": 64, "most": 2000, "new": 1, "heads": 8, "D": 128, "block": 64, "type": "f16"},
        # four prompts written at once, one after a shared prefix that ends inside a block, and read back
        {"name": "cache_prompt", "kind": "write", "seqs": 4, "most": 5200, "new": 5101, "heads": 8, "D": 128, "block": 64, "type": "f16"},
        # a video's memory of three frames read back as the fp16 operands of a plain attention
        {"name": "cache_read", "kind": "read", "seqs": 1, "most": 15552, "heads": 8, "D": 64, "block": 32, "type": "f16"},
        # a short conversation's next token: latency
        {"name": "attn_token_short", "kind": "attn", "seqs": 1, "nq": 1, "most": 777, "heads": 16, "kv_heads": 2, "D": 64, "block": 16,
         "type": "f16", "causal": True, "window": 0},
        # the next token of 32 long conversations
        {"name": "attn_token_long", "kind": "attn", "seqs": 32, "nq": 1, "most": 16384, "heads": 32, "kv_heads": 8, "D": 128, "block": 64,
         "type": "f16", "causal": True, "window": 0},
        # two long prompts, ragged, after what is cached already
        {"name": "attn_prompt", "kind": "attn", "seqs": 2, "nq": 4096, "most": 5120, "heads": 32, "kv_heads": 8, "D": 128, "block": 64,
         "type": "f16", "causal": True, "window": 0},
        # a frame's tokens over a memory of three frames, fp32 in and out, every token seen
        {"name": "attn_memory_f32", "kind": "attn", "seqs": 1, "nq": 5184, "most": 15552, "heads": 8, "kv_heads": 8, "D": 64, "block": 32,
         "type": "f32", "causal": False, "window": 0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "rope", "rope", "write", "write", "read", "attn", "attn", "attn", "attn"])
    t = rng.choice(["f16", "f32"])
    if kind == "norm":
        out = rng.choice(["q8_0", "q8_0", "q8_1", t])
        n = 32 * _log_int(rng, 2, 256) if out.startswith("q8") else _log_int(rng, 33, 8192)
        rows = max(1, min(_log_int(rng, 1, 16384), MOST_NORM // n))
        return {"kind": kind, "rows": rows, "n": n, "type": t, "out": out, "residual": rng.random() < 0.7}
    if kind == "rope":
        D, heads, batch = rng.choice([64, 96, 128]), rng.choice([1, 2, 5, 8, 16, 32, 40]), rng.choice([1, 1, 2, 7, 32])
        tokens = max(1, min(_log_int(rng, 1, 20736), MOST_ROPE // (D * heads * batch)))
        return {"kind": kind, "batch": batch, "tokens": tokens, "heads": heads, "D": D, "type": t,
                "axes": rng.choice([1, 2, 3]), "halves": rng.random() < 0.5}
    D, block, kv = rng.choice([64, 96, 128, 128]), rng.choice([16, 32, 64, 128]), rng.choice([1, 2, 4, 8])
    seqs = rng.choice([1, 1, 2, 3, 8, 31])
    if kind in ("write", "read"):
        most = max(1, min(_log_int(rng, 1, 8192), MOST_CACHE // (seqs * kv * D)))
        case = {"kind": kind, "seqs": seqs, "most": most, "heads": kv, "D": D, "block": block, "type": t}
        if kind == "write":
            case["new"] = min(most, rng.choice([1, 1, _log_int(rng, 2, 8192)]))
        return case
    heads = kv * rng.choice([1, 1, 2, 4, 7, 8])
    most = _log_int(rng, 1, 32768)
    nq = rng.choice([1, 1, rng.randint(2, 16), _log_int(rng, 17, 5184)])
    most = max(1, min(most, MOST_TOKEN // (seqs * kv * D)))
    most = max(1, min(most, MOST_PAIRS // (seqs * heads * nq)))
    causal = rng.random() < 0.7
    return {"kind": kind, "seqs": seqs, "nq": nq, "most": most, "heads": heads, "kv_heads": kv, "D": D, "block": block,
            "type": t, "causal": causal, "window": rng.choice([0, 0, _log_int(rng, 16, 4096)]) if causal else 0}


# ---------------------------------------------------------------- what a program holds
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(0x5A3 + 7919 * int(seed))


def _normal(g, shape, std=1.0, mean=0.0):
    return torch.randn(shape, generator=g, device=DEV) * std + mean


def _int_between(g, lo, hi, n):
    return torch.randint(lo, hi + 1, (n,), generator=g, device=DEV, dtype=I32)


def _sections(case):
    """Pairs of each axis: time gets a quarter of three axes."""
    pairs = case["D"] // 2
    if case["axes"] == 1:
        return [pairs]
    if case["axes"] == 2:
        return [pairs // 2, pairs // 2]
    return [pairs // 4, (pairs - pairs // 4) // 2, (pairs - pairs // 4) // 2]


def _restart(case):
    """Whether every axis has all frequencies (frames) or the axes share them out (text and video)."""
    return case["axes"] == 2


def _cache(g, case, heads):
    """A cache with every block in use by somebody, and the tables of `seqs` sequences."""
    S, BT, D = case["seqs"], case["block"], case["D"]
    per = (case["most"] + BT - 1) // BT
    blocks = S * per + 3
    s = {"table": torch.randperm(blocks, generator=g, device=DEV)[:S * per].reshape(S, per).to(I32).contiguous()}
    for n in ("k", "v"):
        q = torch.clamp(torch.round(torch.randn((blocks, heads, BT, D), generator=g, device=DEV, dtype=F16) * 36), -127, 127)
        s[n + "8"] = (q + 128).to(torch.uint8)
        s[n + "_scale"] = torch.exp(_normal(g, (blocks, heads), 0.3)) / 36
    s["n_kv"] = torch.cat([torch.full((1,), case["most"], device=DEV, dtype=I32),
                           _int_between(g, (case["most"] + 1) // 2, case["most"], S - 1)])
    return s


def prepare(case, seed):
    g = _gen(seed)
    kind, ty = case["kind"], TYPES[case["type"]]
    if kind == "norm":
        rows, n = case["rows"], case["n"]
        s = {"x": _normal(g, (rows, n), 1.5).to(ty), "w": _normal(g, (n,), 0.2, 1.0)}
        if case["residual"]:
            s["add"] = _normal(g, (rows, n), 0.7).to(ty)
            s["sum"] = torch.zeros((rows, n), device=DEV, dtype=ty)
        if case["out"].startswith("q8"):
            s["rows8"] = torch.zeros((rows, n // 32 * (34 if case["out"] == "q8_0" else 36)), device=DEV, dtype=torch.uint8)
            s["dst"] = torch.zeros((rows, n), device=DEV, dtype=F16)
        else:
            s["dst"] = torch.zeros((rows, n), device=DEV, dtype=TYPES[case["out"]])
    elif kind == "rope":
        B, T, H, D = case["batch"], case["tokens"], case["heads"], case["D"]
        s = {"x": _normal(g, (B, T, H, D)).to(ty)}
        s["dst"] = torch.zeros_like(s["x"])
        t = torch.arange(T, device=DEV)[None] + torch.randint(0, 100000, (B, 1), generator=g, device=DEV)
        side = max(1, math.isqrt(T))
        hw = (torch.arange(T, device=DEV) + torch.randint(0, 5184, (B, 1), generator=g, device=DEV))
        pos = [t] if case["axes"] == 1 else [hw % side, hw // side] if case["axes"] == 2 else [t, hw // side, hw % side]
        s["pos"] = torch.stack([p.expand(B, T) for p in pos]).to(I32).contiguous()
    elif kind in ("write", "read"):
        S, H, D, BT = case["seqs"], case["heads"], case["D"], case["block"]
        s = _cache(g, case, H)
        if kind == "write":
            s["n_new"] = torch.minimum(_int_between(g, (case["new"] + 1) // 2, case["new"], S), s["n_kv"])
            # most new tokens are like the cached ones, some reach further
            for n in ("k", "v"):
                x = _normal(g, (S, H, case["new"], D))
                s[n] = (x * torch.exp(_normal(g, (S, H, case["new"], 1), 0.3))).to(ty)
            # from the first block that the call touches to the end
            first = (s["n_kv"] - s["n_new"]) // BT * BT
            s["pos"] = (first[:, None] + torch.arange(case["new"] + BT - 1, device=DEV, dtype=I32)).contiguous()
            n_read = case["new"] + BT - 1
        else:
            n_read = case["most"]
        s["k_dst"] = torch.zeros((S, H, n_read, D), device=DEV, dtype=ty)
        s["v_dst"] = torch.zeros((S, H, n_read, D), device=DEV, dtype=ty)
    else:
        S = case["seqs"]
        s = _cache(g, case, case["kv_heads"])
        s["n_q"] = torch.cat([torch.full((1,), case["nq"], device=DEV, dtype=I32),
                              _int_between(g, (case["nq"] + 1) // 2, case["nq"], S - 1)])
        # queries as a projection leaves them: the heads of a token together
        s["q"] = _normal(g, (S, case["nq"], case["heads"], case["D"])).to(ty)
        s["dst"] = torch.zeros((S, case["nq"], case["heads"], case["D"]), device=DEV, dtype=ty)
    s["case"] = dict(case)
    return s


# ---------------------------------------------------------------- the framework's calls
_ctx = None


def _own_call(s):
    """The calls of one pass over this state's buffers, whose descriptors a program makes once."""
    global _ctx
    mi = _package()
    if _ctx is None:
        _ctx = mi.Context(torch.cuda.current_device())
    c, ctx = s["case"], _ctx
    T = lambda x: mi.F16 if x.dtype == F16 else mi.F32  # noqa: E731

    def whole(x):  # a torch tensor, its last dimension first
        ne = list(reversed(x.shape))
        nb = [st * x.element_size() for st in reversed(x.stride())]
        return mi.from_torch(x, T(x), ne, nb + [nb[-1] * ne[-1]] * (4 - len(nb)))

    if c["kind"] == "norm":
        x, dst, w = whole(s["x"]), whole(s["dst"]), s["w"].data_ptr()
        add, total = (whole(s["add"]), whole(s["sum"])) if c["residual"] else (None, None)
        if "rows8" not in s:
            return lambda: ctx.rms_norm(x, dst, EPS, add=add, w=w, sum=total)
        t = mi.Q8_0 if c["out"] == "q8_0" else mi.Q8_1
        rows8, p8 = mi.from_torch(s["rows8"], t, [c["n"], c["rows"]]), s["rows8"].data_ptr()

        def norm_q8():
            ctx.rms_norm(x, rows8, EPS, add=add, w=w, sum=total)
            ctx.dequantize_rows(t, p8, dst)
        return norm_q8
    if c["kind"] == "rope":
        x, dst, pos = whole(s["x"]), whole(s["dst"]), s["pos"].data_ptr()
        p = mi.rope_params(c["D"], _sections(c), 10000.0, pairs=mi.ROPE_HALVES if c["halves"] else mi.ROPE_ADJACENT, restart=_restart(c))
        return lambda: ctx.rope_multi(x, pos, p, dst)
    cache, seqs = mi.kv_cache(s["k8"], s["v8"], s["k_scale"], s["v_scale"]), mi.kv_seqs(s["table"], s["n_kv"])
    if c["kind"] == "read":
        kd, vd = whole(s["k_dst"]), whole(s["v_dst"])
        return lambda: ctx.kv_cache_read(cache, seqs, kd, vd)
    if c["kind"] == "write":
        k, v, kd, vd, n, pos = whole(s["k"]), whole(s["v"]), whole(s["k_dst"]), whole(s["v_dst"]), s["n_new"].data_ptr(), s["pos"].data_ptr()

        def write_read():
            ctx.kv_cache_write(cache, seqs, k, v, n_new=n)
            ctx.kv_cache_read(cache, seqs, kd, vd, pos=pos)
        return write_read
    q, dst, n_q = whole(s["q"].transpose(1, 2)), whole(s["dst"]), s["n_q"].data_ptr()
    scale = c["D"] ** -0.5
    return lambda: ctx.kv_cache_attn(cache, seqs, q, dst, scale, n_q=n_q, causal=c["causal"], window=c["window"])


# ---------------------------------------------------------------- the plain forms
def _over(a, b):
    """a / b of float32 tensors (a number on either side would become a product with a reciprocal)."""
    a = a if torch.is_tensor(a) else torch.full_like(b, a)
    return a / (b if torch.is_tensor(b) else torch.full_like(a, b))


def _plain_norm(s):
    c = s["case"]
    h = s["x"].float()
    if c["residual"]:
        h = h + s["add"].float()
        s["sum"].copy_(h)
    mean = ((h * h).double().sum(-1, keepdim=True) / c["n"]).float()
    y = h * _over(1.0, torch.sqrt(mean + EPS)) * s["w"]
    if c["out"].startswith("q8"):
        b = y.reshape(c["rows"], -1, 32)
        top = b.abs().amax(-1, keepdim=True)
        q = torch.round(b * torch.where(top > 0, _over(127.0, top), torch.zeros_like(top)))
        y = (q * _over(top, 127.0).half().float()).reshape(c["rows"], -1)
    s["dst"].copy_(y)


def _frequencies(case):
    """Turns a position of each pair, and the pair's axis."""
    sec = _sections(case)
    axis = torch.repeat_interleave(torch.arange(len(sec), device=DEV), torch.tensor(sec, device=DEV), output_size=sum(sec))
    if _restart(case):
        size = torch.tensor(sec, device=DEV)
        e = torch.arange(sum(sec), device=DEV) - (torch.cumsum(size, 0) - size)[axis]
        return 10000.0 ** -(e.double() / size[axis]), axis
    return 10000.0 ** -(torch.arange(sum(sec), device=DEV).double() / sum(sec)), axis


def _plain_rope(s):
    c = s["case"]
    f, axis = _frequencies(c)
    angle = s["pos"].double()[axis].permute(1, 2, 0) * f  # batch, token, pair
    cos, sin = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]
    x = s["x"].float()
    if c["halves"]:
        a, b = x[..., :c["D"] // 2], x[..., c["D"] // 2:]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = x[..., 0::2], x[..., 1::2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    s["dst"].copy_(y)


def _nearest(x, d):
    """x / d rounded to the nearest whole number, ties to even, in -127 .. 127; 0 where d is 0."""
    return torch.clamp(torch.round(torch.where(d > 0, x.double() / d.double(), torch.zeros_like(x, dtype=F64))), -127, 127)


def _plain_write(s):
    c = s["case"]
    S, H, D, BT = c["seqs"], c["heads"], c["D"], c["block"]
    nb = (c["new"] + BT - 2) // BT + 1  # blocks that one sequence's new tokens may touch
    start = s["n_kv"] - s["n_new"]
    at = (start // BT * BT)[:, None] + torch.arange(nb * BT, device=DEV)  # positions of the touched blocks
    kept = (at < start[:, None]).reshape(S, nb, 1, BT, 1)
    new = ((at >= start[:, None]) & (at < s["n_kv"][:, None])).reshape(S, nb, 1, BT, 1)
    which = at.reshape(S, nb, BT)[:, :, 0] // BT
    seq, blk = torch.nonzero(which * BT < s["n_kv"][:, None], as_tuple=True)
    ids = s["table"][seq, which[seq, blk]].long()
    src = torch.clamp(at - start[:, None], 0, c["new"] - 1).reshape(S, nb, BT)[seq, blk]
    kept, new, zero = kept[seq, blk], new[seq, blk], torch.zeros((), device=DEV)
    has = kept.any(2, keepdim=True)
    for n in ("k", "v"):
        old_d = s[n + "_scale"][ids][..., None, None]
        old = (s[n + "8"][ids].float() - 128) * old_d
        x = s[n].float()[seq[:, None, None], torch.arange(H, device=DEV)[None, :, None], src[:, None, :]]  # pair, head, token
        d = _over(torch.where(new, x.abs(), zero).amax((2, 3), keepdim=True), 127.0)
        d = torch.where(has, torch.maximum(d, old_d), d)
        q = _nearest(torch.where(new, x, torch.where(kept, old, zero)), d) + 128
        s[n + "8"][ids] = torch.where(new | kept, q.to(torch.uint8), s[n + "8"][ids])
        s[n + "_scale"][ids] = d[..., 0, 0]


def _plain_read(s, pos):
    c = s["case"]
    BT = c["block"]
    ok = (pos >= 0) & (pos < s["n_kv"][:, None])
    p = torch.where(ok, pos, torch.zeros_like(pos)).long()
    ids = torch.gather(s["table"].long(), 1, p // BT)
    for n in ("k", "v"):
        val = (s[n + "8"][ids, :, p % BT].float() - 128) * s[n + "_scale"][ids][..., None]  # seq, row, head, element
        dst = s[n + "_dst"]
        dst.copy_(torch.where(ok[:, None, :, None], val.permute(0, 2, 1, 3).to(dst.dtype), dst))


def _plain_attn(s):
    c = s["case"]
    S, H, KV, D, nq = c["seqs"], c["heads"], c["kv_heads"], c["D"], c["nq"]
    ids = s["table"].long()
    key = (s["k8"][ids].float() - 128) * s["k_scale"][ids][..., None, None]  # seq, block, head, token, element
    val = (s["v8"][ids].float() - 128) * s["v_scale"][ids][..., None, None]
    key = key.permute(0, 2, 4, 1, 3).reshape(S * KV, D, -1)
    val = val.permute(0, 2, 1, 3, 4).reshape(S * KV, -1, D)
    n = key.shape[-1]
    q = s["q"].float().reshape(S, nq, KV, H // KV, D).permute(0, 2, 1, 3, 4).reshape(S * KV, nq * (H // KV), D)
    score = torch.bmm(q, key).reshape(S, KV, nq, H // KV, n) * D ** -0.5
    at = torch.arange(n, device=DEV)
    p = (s["n_kv"] - s["n_q"])[:, None] + torch.arange(nq, device=DEV)  # position of each query
    seen = (at < s["n_kv"][:, None, None]).expand(S, nq, n)
    if c["causal"]:
        seen = seen & (at <= p[..., None])
    if c["window"]:
        seen = seen & (at > p[..., None] - c["window"])
    seen = seen[:, None, :, None]
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = e.sum(-1, keepdim=True)
    out = torch.bmm(e.reshape(S * KV, -1, n), val).reshape(S, KV, nq, H // KV, D) / torch.where(total > 0, total, torch.ones_like(total))
    out = out.permute(0, 2, 1, 3, 4).reshape(S, nq, H, D)
    there = (torch.arange(nq, device=DEV) < s["n_q"][:, None])[..., None, None]
    s["dst"].copy_(torch.where(there, out.to(s["dst"].dtype), s["dst"]))


def _plain(s):
    kind = s["case"]["kind"]
    if kind == "norm":
        _plain_norm(s)
    elif kind == "rope":
        _plain_rope(s)
    elif kind == "write":
        _plain_write(s)
        _plain_read(s, s["pos"])
    elif kind == "read":
        _plain_read(s, torch.arange(s["case"]["most"], device=DEV)[None].expand(s["case"]["seqs"], -1))
    else:
        _plain_attn(s)


def run(state):
    if own:
        if "call" not in state:
            state["call"] = _own_call(state)
        state["call"]()
    else:
        _plain(state)
    return _outputs(state, state["case"]["kind"])


def _outputs(s, kind):
    if kind == "norm":
        return {"dst": s["dst"], "sum": s["sum"]} if "sum" in s else {"dst": s["dst"]}
    if kind == "write":
        return {"k": s["k_dst"], "v": s["v_dst"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if kind == "read":
        return {"k": s["k_dst"], "v": s["v_dst"]}
    return {"dst": s["dst"]}


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind, size = case["kind"], 2 if case["type"] == "f16" else 4
    if kind == "norm":
        n = case["rows"] * case["n"]
        if case["out"].startswith("q8"):  # the rows, and the values they stand for
            out = n * (34 if case["out"] == "q8_0" else 36) / 32 + 2 * n
        else:
            out = n * (2 if case["out"] == "f16" else 4)
        return {"bytes": n * size * (3 if case["residual"] else 1) + out + 4 * case["n"], "flops": 5 * n}
    if kind == "rope":
        n = case["batch"] * case["tokens"] * case["heads"] * case["D"]
        return {"bytes": 2 * n * size + 4 * case["axes"] * case["batch"] * case["tokens"], "flops": 3 * n}
    some = lambda most, seqs: most + (seqs - 1) * 0.75 * most  # tokens of ragged sequences  # noqa: E731
    if kind == "read":
        n = 2 * some(case["most"], case["seqs"]) * case["heads"] * case["D"]
        return {"bytes": n * (1 + size), "flops": n}
    if kind == "write":  # new elements in, one byte each out, and the touched blocks' values back
        n = 2 * 0.75 * case["new"] * case["seqs"] * case["heads"] * case["D"] if case["new"] > 1 else 2 * case["seqs"] * case["heads"] * case["D"]
        touched = n + 2 * case["seqs"] * case["heads"] * case["D"] * (case["block"] - 1) / 2
        return {"bytes": n * (size + 1) + touched * (1 + size), "flops": 2 * n}
    S, D = case["seqs"], case["D"]
    tokens, rows = some(case["most"], S), some(case["nq"], S) if case["nq"] > 1 else S
    per = tokens / S
    if case["causal"]:  # keys that a query sees on average
        nq = rows / S
        per = sum(max(0.0, min(per - nq + i + 1, case["window"] or 1 << 60)) for i in (0.125 * nq, 0.375 * nq, 0.625 * nq, 0.875 * nq)) / 4
    if case["window"]:
        tokens = min(tokens, S * (case["window"] + rows / S))
    return {"bytes": 2 * tokens * case["kv_heads"] * D + 2 * size * rows * case["heads"] * D,
            "flops": 4 * D * rows * case["heads"] * max(per, 1.0)}


# ---------------------------------------------------------------- the definitions in float64
def _exact_norm(s):
    c = s["case"]
    h = s["x"].double() + (s["add"].double() if c["residual"] else 0.0)
    y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + EPS) * s["w"].double()
    if c["out"].startswith("q8"):
        step = y.unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True) / 127
        y = (torch.round(y.unflatten(-1, (-1, 32)) / torch.where(step > 0, step, 1.0)) * step.half().double()).flatten(-2)
    return {"dst": y, "sum": h} if c["residual"] else {"dst": y}


def _exact_rope(s):
    c = s["case"]
    sec, D = _sections(c), c["D"]
    lead = s["x"].double()
    out = torch.empty_like(lead)
    pair = 0
    for axis, size in enumerate(sec):
        for e in range(size):
            f = 10000.0 ** (-e / size if _restart(c) else -pair / sum(sec))
            a = s["pos"][axis].double()[..., None] * f
            i, j = (pair, pair + D // 2) if c["halves"] else (2 * pair, 2 * pair + 1)
            out[..., i] = lead[..., i] * torch.cos(a) - lead[..., j] * torch.sin(a)
            out[..., j] = lead[..., i] * torch.sin(a) + lead[..., j] * torch.cos(a)
            pair += 1
    return {"dst": out}


def _exact_write(s):
    """Block by block, as the cache holds it: one float32 scale for each block and head."""
    c = s["case"]
    BT = c["block"]
    out = {"k": s["k_dst"].double(), "v": s["v_dst"].double()}
    for n in ("k", "v"):
        scale = s[n + "_scale"].double()
        for q in range(c["seqs"]):
            end = int(s["n_kv"][q])
            begin, row = end - int(s["n_new"][q]), 0
            for b in range(begin // BT, (end + BT - 1) // BT):
                at = int(s["table"][q, b])
                lo, hi = max(begin, b * BT), min(end, b * BT + BT)
                x = s[n][q, :, lo - begin:hi - begin].double()
                d = x.abs().amax((1, 2)) / 127
                if lo > b * BT:
                    was = (s[n + "8"][at, :, :lo - b * BT].double() - 128) * scale[at][:, None, None]
                    x, d = torch.cat([was.float().double(), x], 1), torch.maximum(d, scale[at])
                d = d.float().double()
                scale[at] = d
                whole = torch.round(x / torch.where(d > 0, d, 1.0)[:, None, None]).clamp(-127, 127)
                out[n][q, :, row:row + x.shape[1]] = whole * d[:, None, None]
                row += x.shape[1]
        out[n + "_scale"] = scale
    return out


def _exact_read(s):
    c = s["case"]
    out = {}
    for n in ("k", "v"):
        o = s[n + "_dst"].double()
        for q in range(c["seqs"]):
            ids, end = s["table"][q].long(), int(s["n_kv"][q])
            val = (s[n + "8"][ids].double() - 128) * s[n + "_scale"][ids].double()[..., None, None]
            o[q, :, :end] = val.transpose(0, 1).flatten(1, 2)[:, :end]
        out[n] = o
    return out


def _exact_attn(s):
    c = s["case"]
    group = c["heads"] // c["kv_heads"]
    out = s["dst"].double()
    for q in range(c["seqs"]):
        ids, end, rows = s["table"][q].long(), int(s["n_kv"][q]), int(s["n_q"][q])
        at, p = torch.arange(end, device=DEV), end - rows + torch.arange(rows, device=DEV)
        hidden = torch.zeros((rows, end), dtype=torch.bool, device=DEV)
        if c["causal"]:
            hidden |= at > p[:, None]
        if c["window"]:
            hidden |= at <= p[:, None] - c["window"]
        for h in range(c["kv_heads"]):
            key, val = (((s[n + "8"][ids, h].double() - 128) * s[n + "_scale"][ids, h].double()[:, None, None]).flatten(0, 1)[:end] for n in ("k", "v"))
            for m in range(h * group, h * group + group):
                w = s["q"][q, :rows, m].double() @ key.T / math.sqrt(c["D"])
                w = torch.softmax(w.masked_fill(hidden, -math.inf), -1)
                out[q, :rows, m] = torch.nan_to_num(w) @ val
    return {"dst": out}


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "rope": _exact_rope, "write": _exact_write, "read": _exact_read, "attn": _exact_attn}[case["kind"]](s)
