"""The work of a layer whose cache is held small: four bits an element, and its least used tokens dropped.

Per step such a layer calls, next to its quantized products: the norms of its queries and keys for each
head with the rotary positions in the same pass; the write of new keys and values into the cache, and its
reading back; the attention over it; the sums of the softmax weights that each cached token has got; and
the eviction of the tokens with the smallest sums.  Sizes are those of decoders and of the image encoders
here (5184 tokens a frame, head sizes 64, 96 and 128).

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
EPS = 1e-6
MOST_QK = 2 * 4096 * 40 * 128            # elements of the largest listed norm and rotation
MOST_CACHE = 4 * 5200 * 8 * 128          # elements of the largest listed write, keys or values
MOST_TOKEN = 32 * 16384 * 8 * 128        # cached keys' elements of the largest single-token attention
MOST_PAIRS = 2 * 32 * 4096 * 5120        # query-key pairs of the largest listed prompt
MOST_EVICT = 8 * 16384 * 8 * 128         # cached keys' elements of the largest listed eviction


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
        # one token of each of 32 conversations: a layer's products give floats, its attention takes halves
        {"name": "qk_tokens", "kind": "qk", "batch": 32, "tokens": 1, "heads": 32, "kv_heads": 8, "D": 128, "type": "f32", "out": "f16",
         "axes": 1, "halves": True},
        # two prompts out of one product of queries, keys and values
        {"name": "qk_prompt", "kind": "qk", "batch": 2, "tokens": 4096, "heads": 32, "kv_heads": 8, "D": 128, "type": "f32", "out": "f16",
         "axes": 1, "halves": True},
        # one token of each of 64 conversations, and the blocks' tokens read back
        {"name": "cache4_token", "kind": "write", "seqs": 64, "most": 2000, "new": 1, "heads": 8, "D": 128, "block": 64, "type": "f16"},
        # four prompts written at once, one after a shared prefix that ends inside a block, and read back
        {"name": "cache4_prompt", "kind": "write", "seqs": 4, "most": 5200, "new": 5101, "heads": 8, "D": 128, "block": 64, "type": "f16"},
        # a short conversation's next token: latency
        {"name": "attn4_token_short", "kind": "attn", "seqs": 1, "nq": 1, "most": 777, "heads": 16, "kv_heads": 2, "D": 64, "block": 16,
         "type": "f16", "causal": True, "window": 0},
        # the next token of 32 long conversations
        {"name": "attn4_token_long", "kind": "attn", "seqs": 32, "nq": 1, "most": 16384, "heads": 32, "kv_heads": 8, "D": 128, "block": 64,
         "type": "f16", "causal": True, "window": 0},
        # two long prompts, ragged, after what is cached already
        {"name": "attn4_prompt", "kind": "attn", "seqs": 2, "nq": 4096, "most": 5120, "heads": 32, "kv_heads": 8, "D": 128, "block": 64,
         "type": "f16", "causal": True, "window": 0},
        # a frame's tokens over a memory of three frames, fp32 in and out, every token seen
        {"name": "attn4_memory_f32", "kind": "attn", "seqs": 1, "nq": 5184, "most": 15552, "heads": 8, "kv_heads": 8, "D": 64, "block": 32,
         "type": "f32", "causal": False, "window": 0},
        # what the next token of 32 long conversations looked at
        {"name": "weights_token", "kind": "weights", "seqs": 32, "nq": 1, "most": 16384, "heads": 32, "kv_heads": 8, "D": 128, "block": 64,
         "type": "f16", "causal": True, "window": 0},
        # what two prompts looked at
        {"name": "weights_prompt", "kind": "weights", "seqs": 2, "nq": 2048, "most": 4099, "heads": 32, "kv_heads": 8, "D": 128, "block": 64,
         "type": "f16", "causal": True, "window": 0},
        # one conversation brought back to its budget, and the kept tokens read back
        {"name": "evict_one", "kind": "evict", "seqs": 1, "most": 1280, "keep": 1024, "first": 4, "recent": 64, "heads": 2, "D": 64, "block": 16, "type": "f16"},
        # eight long conversations halved
        {"name": "evict_long", "kind": "evict", "seqs": 8, "most": 16384, "keep": 8192, "first": 4, "recent": 1024, "heads": 8, "D": 128, "block": 64,
         "type": "f16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["qk", "qk", "write", "write", "attn", "attn", "attn", "attn", "weights", "weights", "evict", "evict"])
    t = rng.choice(["f16", "f32"])
    D, block, kv = rng.choice([64, 96, 128, 128]), rng.choice([16, 32, 64, 128]), rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 1, 2, 4, 7, 8])
    if kind == "qk":
        batch = rng.choice([1, 1, 2, 7, 32])
        tokens = max(1, min(_log_int(rng, 1, 20736), MOST_QK // (D * (heads + kv) * batch)))
        return {"kind": kind, "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv, "D": D, "type": t,
                "out": rng.choice(["f16", "f32"]), "axes": rng.choice([1, 2, 3]), "halves": rng.random() < 0.5}
    seqs = rng.choice([1, 1, 2, 3, 8, 31])
    if kind == "write":
        most = max(1, min(_log_int(rng, 1, 8192), MOST_CACHE // (seqs * kv * D)))
        return {"kind": kind, "seqs": seqs, "most": most, "new": min(most, rng.choice([1, 1, _log_int(rng, 2, 8192)])), "heads": kv, "D": D,
                "block": block, "type": t}
    if kind == "evict":
        most = max(1, min(_log_int(rng, 16, 32768), MOST_EVICT // (seqs * kv * D)))
        keep = max(1, int(most * rng.uniform(0.1, 1.0)))
        return {"kind": kind, "seqs": seqs, "most": most, "keep": keep, "first": rng.choice([0, 1, 4, 64]),
                "recent": rng.choice([0, 1, 32, keep // 4, keep]), "heads": kv, "D": D, "block": block, "type": t}
    most = _log_int(rng, 1, 32768)
    nq = rng.choice([1, 1, rng.randint(2, 16), _log_int(rng, 17, 5184)])
    most = max(1, min(most, MOST_TOKEN // (seqs * kv * D)))
    most = max(1, min(most, MOST_PAIRS // (seqs * heads * nq)))
    causal = rng.random() < 0.7
    return {"kind": kind, "seqs": seqs, "nq": nq, "most": most, "heads": heads, "kv_heads": kv, "D": D, "block": block,
            "type": t, "causal": causal, "window": rng.choice([0, 0, _log_int(rng, 16, 4096)]) if causal else 0}


# ---------------------------------------------------------------- what a program holds
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(0x45A3 + 7919 * int(seed))


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
    """A cache with every block in use by somebody, and the tables of `seqs` sequences.  Keys' scales are
    [block, head, token, group of 32], values' [block, head, group of 32, token]."""
    S, BT, D = case["seqs"], case["block"], case["D"]
    per = (case["most"] + BT - 1) // BT
    blocks = S * per + 3
    s = {"table": torch.randperm(blocks, generator=g, device=DEV)[:S * per].reshape(S, per).to(I32).contiguous()}
    # two elements of a group like normal ones to a byte, and scales of either sign with eight significant bits
    for n in ("k", "v"):
        q = [torch.clamp(torch.round(torch.randn((blocks, heads, BT, D // 2), generator=g, device=DEV, dtype=F16) * 3.1) + 8, 0, 15) for _ in range(2)]
        s[n + "4"] = (q[0] + 16 * q[1]).to(torch.uint8)
        d = torch.exp(_normal(g, (blocks, heads, BT, D // 32), 0.3)) / 3.1
        d = torch.where(torch.rand(d.shape, generator=g, device=DEV) < 0.5, d, -d)
        s[n + "_scale"] = d.bfloat16().to(F16)
    s["v_scale"] = s["v_scale"].transpose(2, 3).contiguous()
    s["n_kv"] = torch.cat([torch.full((1,), case["most"], device=DEV, dtype=I32),
                           _int_between(g, (case["most"] + 1) // 2, case["most"], S - 1)])
    return s


def prepare(case, seed):
    g = _gen(seed)
    kind, ty = case["kind"], TYPES[case["type"]]
    if kind == "qk":
        B, T, H, KV, D = case["batch"], case["tokens"], case["heads"], case["kv_heads"], case["D"]
        # one product's rows: queries, keys and values of a token behind one another
        s = {"qkv": _normal(g, (B, T, (H + 2 * KV) * D), 1.5).to(ty), "q_w": _normal(g, (D,), 0.2, 1.0), "k_w": _normal(g, (D,), 0.2, 1.0)}
        s["q"] = torch.zeros((B, T, H, D), device=DEV, dtype=TYPES[case["out"]])
        s["k"] = torch.zeros((B, T, KV, D), device=DEV, dtype=TYPES[case["out"]])
        t = torch.arange(T, device=DEV)[None] + torch.randint(0, 100000, (B, 1), generator=g, device=DEV)
        side = max(1, math.isqrt(T))
        hw = (torch.arange(T, device=DEV) + torch.randint(0, 5184, (B, 1), generator=g, device=DEV))
        pos = [t] if case["axes"] == 1 else [hw % side, hw // side] if case["axes"] == 2 else [t, hw // side, hw % side]
        s["pos"] = torch.stack([p.expand(B, T) for p in pos]).to(I32).contiguous()
    elif kind == "write":
        S, H, D, BT = case["seqs"], case["heads"], case["D"], case["block"]
        s = _cache(g, case, H)
        s["n_new"] = torch.minimum(_int_between(g, (case["new"] + 1) // 2, case["new"], S), s["n_kv"])
        # most new tokens are like the cached ones, some reach further
        for n in ("k", "v"):
            x = _normal(g, (S, H, case["new"], D))
            s[n] = (x * torch.exp(_normal(g, (S, H, case["new"], 1), 0.3))).to(ty)
        # from the first block that the call touches to the end
        first = (s["n_kv"] - s["n_new"]) // BT * BT
        s["pos"] = (first[:, None] + torch.arange(case["new"] + BT - 1, device=DEV, dtype=I32)).contiguous()
        s["k_dst"] = torch.zeros((S, H, case["new"] + BT - 1, D), device=DEV, dtype=ty)
        s["v_dst"] = torch.zeros((S, H, case["new"] + BT - 1, D), device=DEV, dtype=ty)
    elif kind == "evict":
        S, H, D = case["seqs"], case["heads"], case["D"]
        s = _cache(g, case, H)
        room = s["table"].shape[1] * case["block"]
        # a few tokens have most of the weight, and many of the others have got none
        w = torch.exp(_normal(g, (S, H, room), 2.5, -5.0))
        s["sums"] = torch.where(torch.rand(w.shape, generator=g, device=DEV) < 0.3, torch.zeros_like(w), w)
        s["n_keep"] = torch.cat([torch.full((1,), case["keep"], device=DEV, dtype=I32),
                                 _int_between(g, (case["keep"] + 1) // 2, case["keep"], S - 1)])
        s["sums_out"] = torch.zeros((S, H, room), device=DEV)
        s["kept"] = torch.full((S, H, case["keep"]), -1, device=DEV, dtype=I32)
        s["n_out"] = torch.zeros((S,), device=DEV, dtype=I32)
        s["k_dst"] = torch.zeros((S, H, case["keep"], D), device=DEV, dtype=ty)
        s["v_dst"] = torch.zeros((S, H, case["keep"], D), device=DEV, dtype=ty)
    else:
        S, H, D = case["seqs"], case["heads"], case["D"]
        s = _cache(g, case, case["kv_heads"])
        s["n_q"] = torch.cat([torch.full((1,), case["nq"], device=DEV, dtype=I32),
                              _int_between(g, (case["nq"] + 1) // 2, case["nq"], S - 1)])
        # queries as a projection leaves them: the heads of a token together
        s["q"] = _normal(g, (S, case["nq"], H, D)).to(ty)
        s["lse"] = torch.zeros((S, case["nq"], H), device=DEV)
        if kind == "attn":
            s["dst"] = torch.zeros((S, case["nq"], H, D), device=DEV, dtype=ty)
        else:  # what the attention before it left, and the sums of the steps before
            s["case"] = dict(case)
            s["lse"].copy_(_lse(_scores(s)))
            s["sums"] = torch.exp(_normal(g, (S, case["kv_heads"], s["table"].shape[1] * case["block"]), 1.5, -3.0))
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

    if c["kind"] == "qk":
        H, KV, D = c["heads"], c["kv_heads"], c["D"]
        q_src, k_src = (whole(x.unflatten(-1, (-1, D))) for x in s["qkv"].split([H * D, KV * D, KV * D], -1)[:2])
        q_dst, k_dst, q_w, k_w, pos = whole(s["q"]), whole(s["k"]), s["q_w"].data_ptr(), s["k_w"].data_ptr(), s["pos"].data_ptr()
        p = mi.rope_params(D, _sections(c), 10000.0, pairs=mi.ROPE_HALVES if c["halves"] else mi.ROPE_ADJACENT, restart=_restart(c))
        return lambda: ctx.qk_norm_rope(q_src, k_src, EPS, pos, p, q_dst, k_dst, q_w=q_w, k_w=k_w)
    cache, seqs = mi.kv_cache4(s["k4"], s["v4"], s["k_scale"], s["v_scale"]), mi.kv_seqs(s["table"], s["n_kv"])
    if c["kind"] == "write":
        k, v, kd, vd, n, pos = whole(s["k"]), whole(s["v"]), whole(s["k_dst"]), whole(s["v_dst"]), s["n_new"].data_ptr(), s["pos"].data_ptr()

        def write_read():
            ctx.kv_cache4_write(cache, seqs, k, v, n_new=n)
            ctx.kv_cache4_read(cache, seqs, kd, vd, pos=pos)
        return write_read
    if c["kind"] == "evict":
        kd, vd, after = whole(s["k_dst"]), whole(s["v_dst"]), mi.kv_seqs(s["table"], s["n_out"])
        sums, sums_out, n_keep, kept, n_out = (s[n].data_ptr() for n in ("sums", "sums_out", "n_keep", "kept", "n_out"))

        def evict_read():
            ctx.kv_cache4_evict(cache, seqs, sums, sums_out, c["keep"], kept, n_out, n_keep=n_keep, first=c["first"], recent=c["recent"])
            ctx.kv_cache4_read(cache, after, kd, vd)
        return evict_read
    q, n_q, lse, scale = whole(s["q"].transpose(1, 2)), s["n_q"].data_ptr(), s["lse"].data_ptr(), c["D"] ** -0.5
    if c["kind"] == "attn":
        dst = whole(s["dst"])
        return lambda: ctx.kv_cache4_attn(cache, seqs, q, dst, scale, n_q=n_q, causal=c["causal"], window=c["window"], lse=lse)
    sums = s["sums"].data_ptr()
    return lambda: ctx.kv_cache4_weights(cache, seqs, q, lse, sums, scale, n_q=n_q, causal=c["causal"], window=c["window"])


# ---------------------------------------------------------------- the plain forms
def _nibbles(b):
    """The elements 0 .. 15 of packed rows.  A 32-bit word holds eight, the even ones in its lower half."""
    n = torch.stack([b & 15, b >> 4], -1).flatten(-2)
    return n.unflatten(-1, (-1, 2, 4)).transpose(-1, -2).flatten(-3)


def _packed(q):
    """_nibbles' inverse."""
    n = q.unflatten(-1, (-1, 4, 2)).transpose(-1, -2).flatten(-3).unflatten(-1, (-1, 2))
    return (n[..., 0] + 16 * n[..., 1]).to(torch.uint8)


def _values(s, n, ids=slice(None)):
    """Keys or values of the blocks `ids` [..., head, token, element]."""
    d = s[n + "_scale"][ids].float()
    if n == "v":
        d = d.transpose(-1, -2)
    return ((_nibbles(s[n + "4"][ids]).float() - 8).unflatten(-1, (-1, 32)) * d[..., None]).flatten(-2)


def _frequencies(case):
    """Turns a position of each pair, and the pair's axis."""
    sec = _sections(case)
    axis = torch.repeat_interleave(torch.arange(len(sec), device=DEV), torch.tensor(sec, device=DEV), output_size=sum(sec))
    if _restart(case):
        size = torch.tensor(sec, device=DEV)
        e = torch.arange(sum(sec), device=DEV) - (torch.cumsum(size, 0) - size)[axis]
        return 10000.0 ** -(e.double() / size[axis]), axis
    return 10000.0 ** -(torch.arange(sum(sec), device=DEV).double() / sum(sec)), axis


def _plain_qk(s):
    c = s["case"]
    H, KV, D = c["heads"], c["kv_heads"], c["D"]
    f, axis = _frequencies(c)
    angle = s["pos"].double()[axis].permute(1, 2, 0) * f  # batch, token, pair
    cos, sin = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]
    x = s["qkv"][..., :(H + KV) * D].float().unflatten(-1, (H + KV, D))
    w = torch.cat([s["q_w"].expand(H, D), s["k_w"].expand(KV, D)])
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    if c["halves"]:
        a, b = x[..., :D // 2], x[..., D // 2:]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = x[..., 0::2], x[..., 1::2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    s["q"].copy_(y[:, :, :H])
    s["k"].copy_(y[:, :, H:])


def _plain_write(s):
    c = s["case"]
    S, H, BT = c["seqs"], c["heads"], c["block"]
    row = torch.arange(c["new"], device=DEV)
    at = (s["n_kv"] - s["n_new"])[:, None] + row  # place of each new token
    seq, r = torch.nonzero(row < s["n_new"][:, None], as_tuple=True)
    place = at[seq, r]
    ids, tok = s["table"][seq, place // BT].long(), place % BT
    for n in ("k", "v"):
        x = s[n].float()[seq, :, r].unflatten(-1, (-1, 32))  # token, head, group, element
        top, low = x.amax(-1, keepdim=True), x.amin(-1, keepdim=True)
        d = torch.where(top >= -low, top, low) * -0.125
        d = d.bfloat16().to(F16)
        d = torch.where(d.abs() <= 8160, d, torch.full_like(d, math.nan))
        w = d.double()
        q = torch.clamp(torch.round(torch.where(w.abs() > 0, x.double() / w, torch.zeros_like(w))), -8, 7) + 8
        s[n + "4"][ids, :, tok] = _packed(q.to(torch.uint8).flatten(-2))
        if n == "k":
            s["k_scale"][ids, :, tok] = d[..., 0]
        else:
            s["v_scale"][ids, :, :, tok] = d[..., 0]


def _plain_read(s, pos, n_kv):
    c = s["case"]
    BT = c["block"]
    ok = (pos >= 0) & (pos < n_kv[:, None])
    p = torch.where(ok, pos, torch.zeros_like(pos)).long()
    ids = torch.gather(s["table"].long(), 1, p // BT)
    seq, row = torch.nonzero(ok, as_tuple=True)
    ids, tok = ids[seq, row], (p % BT)[seq, row]
    for n in ("k", "v"):
        d = s["k_scale"][ids, :, tok] if n == "k" else s["v_scale"][ids, :, :, tok]
        val = ((_nibbles(s[n + "4"][ids, :, tok]).float() - 8).unflatten(-1, (-1, 32)) * d.float()[..., None]).flatten(-2)
        dst = s[n + "_dst"]
        dst[seq, :, row] = val.to(dst.dtype)


def _scores(s):
    """Scaled scores [seq, key head, query, head of the group, token], -inf where a query does not see the token."""
    c = s["case"]
    S, H, KV, D, nq = c["seqs"], c["heads"], c["kv_heads"], c["D"], c["nq"]
    key = _values(s, "k", s["table"].long()).permute(0, 2, 4, 1, 3).reshape(S * KV, D, -1)
    n = key.shape[-1]
    q = s["q"].float().reshape(S, nq, KV, H // KV, D).permute(0, 2, 1, 3, 4).reshape(S * KV, nq * (H // KV), D)
    score = torch.bmm(q, key).reshape(S, KV, nq, H // KV, n) * D ** -0.5
    at = torch.arange(n, device=DEV)
    p = (s["n_kv"] - s["n_q"])[:, None] + torch.arange(nq, device=DEV)  # position of each query
    seen = ((at < s["n_kv"][:, None, None]) & (torch.arange(nq, device=DEV) < s["n_q"][:, None])[..., None]).expand(S, nq, n)
    if c["causal"]:
        seen = seen & (at <= p[..., None])
    if c["window"]:
        seen = seen & (at > p[..., None] - c["window"])
    return score.masked_fill_(~seen[:, None, :, None], -math.inf)


def _lse(score):
    """log of the sum of exponentials [seq, query, head]."""
    return torch.logsumexp(score, -1).permute(0, 2, 1, 3).flatten(2)


def _there(s):
    return (torch.arange(s["case"]["nq"], device=DEV) < s["n_q"][:, None])[..., None]


def _plain_attn(s):
    c = s["case"]
    S, H, KV, D, nq = c["seqs"], c["heads"], c["kv_heads"], c["D"], c["nq"]
    score = _scores(s)
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    e = score.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    val = _values(s, "v", s["table"].long()).permute(0, 2, 1, 3, 4).reshape(S * KV, -1, D)
    out = torch.bmm(e.reshape(S * KV, -1, e.shape[-1]), val).reshape(S, KV, nq, H // KV, D) / torch.where(total > 0, total, torch.ones_like(total))
    out = out.permute(0, 2, 1, 3, 4).reshape(S, nq, H, D)
    lse = (torch.log(total) + top)[..., 0].permute(0, 2, 1, 3).flatten(2)
    there = _there(s)
    s["dst"].copy_(torch.where(there[..., None], out.to(s["dst"].dtype), s["dst"]))
    s["lse"].copy_(torch.where(there, lse, s["lse"]))


def _plain_weights(s):
    c = s["case"]
    S, H, KV, nq = c["seqs"], c["heads"], c["kv_heads"], c["nq"]
    lse = s["lse"].reshape(S, nq, KV, H // KV).permute(0, 2, 1, 3)[..., None]
    e = _scores(s).sub_(torch.where(torch.isfinite(lse), lse, torch.zeros_like(lse))).exp_()
    s["sums"].add_(e.flatten(2, 3).sum(2, dtype=F64).float())


def _plain_evict(s):
    c = s["case"]
    S, H, BT = c["seqs"], c["heads"], c["block"]
    at = torch.arange(s["sums"].shape[-1], device=DEV)
    n = torch.minimum(s["n_kv"], s["n_keep"])
    recent = torch.clamp(n, max=c["recent"])
    first = torch.clamp(n - recent, max=c["first"])
    always = (at < first[:, None]) | (at >= (s["n_kv"] - recent)[:, None])
    w = torch.where(always[:, None], torch.full_like(s["sums"], math.inf), s["sums"])
    w = torch.where((at < s["n_kv"][:, None])[:, None], w, torch.full_like(w, -math.inf))
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices  # the lower token first among equal ones
    rank = torch.empty_like(order).scatter_(-1, order, at.expand_as(order))
    order = torch.where(rank < n[:, None, None], at, torch.full_like(at, 1 << 40)).sort(-1).values[..., :c["keep"]]
    real = torch.arange(order.shape[-1], device=DEV) < n[:, None]  # sequence, kept token
    src = torch.where(real[:, None], order, torch.zeros_like(order))
    s["kept"][..., :order.shape[-1]].copy_(torch.where(real[:, None], order.to(I32), s["kept"][..., :order.shape[-1]]))
    s["n_out"].copy_(n)
    end = torch.where((at < s["n_kv"][:, None])[:, None], torch.zeros_like(w), s["sums_out"])
    end[..., :order.shape[-1]] = torch.where(real[:, None], torch.gather(s["sums"], -1, src), end[..., :order.shape[-1]])
    s["sums_out"].copy_(end)
    seq, head, j = torch.nonzero(real[:, None].expand_as(src), as_tuple=True)
    t = src[seq, head, j]
    f, ft, d, dt = s["table"][seq, t // BT].long(), t % BT, s["table"][seq, j // BT].long(), j % BT
    s["k4"][d, head, dt], s["v4"][d, head, dt] = s["k4"][f, head, ft], s["v4"][f, head, ft]
    s["k_scale"][d, head, dt], s["v_scale"][d, head, :, dt] = s["k_scale"][f, head, ft], s["v_scale"][f, head, :, ft]


def _plain(s):
    kind = s["case"]["kind"]
    if kind == "qk":
        _plain_qk(s)
    elif kind == "write":
        _plain_write(s)
        _plain_read(s, s["pos"], s["n_kv"])
    elif kind == "evict":
        _plain_evict(s)
        _plain_read(s, torch.arange(s["case"]["keep"], device=DEV)[None].expand(s["case"]["seqs"], -1), s["n_out"])
    elif kind == "attn":
        _plain_attn(s)
    else:
        _plain_weights(s)


def run(state):
    if own:
        if "call" not in state:
            state["call"] = _own_call(state)
        state["call"]()
    else:
        _plain(state)
    return _outputs(state, state["case"]["kind"])


def _outputs(s, kind):
    if kind == "qk":
        return {"q": s["q"], "k": s["k"]}
    if kind == "write":
        return {"k": s["k_dst"], "v": s["v_dst"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if kind == "evict":
        return {"k": s["k_dst"], "v": s["v_dst"], "sums": s["sums_out"], "kept": s["kept"], "n": s["n_out"]}
    return {"dst": s["dst"], "lse": s["lse"]} if kind == "attn" else {"sums": s["sums"]}


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind, size, D = case["kind"], 2 if case["type"] == "f16" else 4, case["D"]
    packed = D / 2 + D / 16  # bytes of a token and head, keys or values
    some = lambda most, seqs: most + (seqs - 1) * 0.75 * most  # tokens of ragged sequences  # noqa: E731
    if kind == "qk":
        n = case["batch"] * case["tokens"] * (case["heads"] + case["kv_heads"]) * D
        return {"bytes": n * (size + (2 if case["out"] == "f16" else 4)) + 4 * case["axes"] * case["batch"] * case["tokens"] + 8 * D, "flops": 8 * n}
    if kind == "write":  # new elements in, and packed, and the touched blocks' values back
        rows = 2 * case["seqs"] * case["heads"] * (0.75 * case["new"] if case["new"] > 1 else 1)
        touched = rows + 2 * case["seqs"] * case["heads"] * (case["block"] - 1) / 2
        return {"bytes": rows * (size * D + packed) + touched * (packed + size * D), "flops": 4 * rows * D}
    if kind == "evict":  # weights, and kept rows once out of the cache, into it, and as values
        tokens, kept = some(case["most"], case["seqs"]) * case["heads"], some(case["keep"], case["seqs"]) * case["heads"]
        return {"bytes": 8 * tokens + kept * (4 + 4 * packed + 2 * size * D), "flops": 2 * tokens}
    S, H, KV = case["seqs"], case["heads"], case["kv_heads"]
    tokens, rows = some(case["most"], S), some(case["nq"], S) if case["nq"] > 1 else S
    per = tokens / S
    if case["causal"]:  # keys that a query sees on average
        nq = rows / S
        per = sum(max(0.0, min(per - nq + i + 1, case["window"] or 1 << 60)) for i in (0.125 * nq, 0.375 * nq, 0.625 * nq, 0.875 * nq)) / 4
    if case["window"]:
        tokens = min(tokens, S * (case["window"] + rows / S))
    if kind == "attn":
        return {"bytes": 2 * tokens * KV * packed + rows * H * (2 * size * D + 4), "flops": 4 * D * rows * H * max(per, 1.0)}
    return {"bytes": tokens * KV * (packed + 8) + rows * H * (size * D + 4), "flops": 2 * D * rows * H * max(per, 1.0)}


# ---------------------------------------------------------------- the definitions in float64
def _element(b, i):
    """Element i of packed rows: nibble i / 2 of its word, of the upper half for odd ones."""
    place = i % 8 // 2 + 4 * (i % 2)
    return (b[..., i // 8 * 4 + place // 2] >> (4 * (place % 2))) & 15


def _rows(s, n, q, h, end):
    """Keys or values of the first `end` tokens of sequence q and head h, in float64."""
    ids = s["table"][q].long()
    b = s[n + "4"][ids, h].flatten(0, 1)[:end]
    d = s[n + "_scale"][ids, h].double()
    d = (d if n == "k" else d.transpose(1, 2)).flatten(0, 1)[:end]
    return torch.stack([(_element(b, i).double() - 8) * d[:, i // 32] for i in range(s["case"]["D"])], -1)


def _exact_qk(s):
    c = s["case"]
    H, KV, D, sec = c["heads"], c["kv_heads"], c["D"], _sections(c)
    out, begin = {}, 0
    for n, heads in (("q", H), ("k", KV)):
        x = s["qkv"][..., begin:begin + heads * D].double().unflatten(-1, (heads, D))
        begin += heads * D
        x = x * torch.rsqrt(x.square().sum(-1, keepdim=True) / D + EPS) * s[n + "_w"].double()
        y = torch.empty_like(x)
        pair = 0
        for axis, size in enumerate(sec):
            for e in range(size):
                a = s["pos"][axis].double()[..., None] * 10000.0 ** (-e / size if _restart(c) else -pair / sum(sec))
                i, j = (pair, pair + D // 2) if c["halves"] else (2 * pair, 2 * pair + 1)
                y[..., i] = x[..., i] * torch.cos(a) - x[..., j] * torch.sin(a)
                y[..., j] = x[..., i] * torch.sin(a) + x[..., j] * torch.cos(a)
                pair += 1
        out[n] = y
    return out


def _exact_write(s):
    """Sequence by sequence; what was in the cache before as it was."""
    c = s["case"]
    BT, out = c["block"], {"k": s["k_dst"].double(), "v": s["v_dst"].double()}
    for n in ("k", "v"):
        scale = s[n + "_scale"].double()
        for q in range(c["seqs"]):
            end, new = int(s["n_kv"][q]), int(s["n_new"][q])
            begin = end - new
            x = s[n][q, :, :new].double().unflatten(-1, (-1, 32))
            far = torch.gather(x, -1, x.abs().argmax(-1, keepdim=True))
            far = torch.where(x.amax(-1, keepdim=True) == -x.amin(-1, keepdim=True), far.abs(), far)
            # eight significant bits of far / -8, ties to even
            m, e = torch.frexp(far / -8)
            d = torch.ldexp(torch.round(m * 256), e - 8).half().double()
            d = torch.where(d.abs() > 8160, math.nan, d)
            val = torch.round(x / torch.where(d == 0, 1.0, d)).clamp(-8, 7) * d
            lo = begin // BT * BT
            for h in range(c["heads"]):
                if begin > lo:
                    out[n][q, h, :begin - lo] = _rows(s, n, q, h, end)[lo:begin]
            out[n][q, :, begin - lo:end - lo] = val.flatten(-2)
            at = torch.arange(begin, end, device=DEV)
            ids, tok = s["table"][q].long()[at // BT], at % BT
            if n == "k":
                scale[ids, :, tok] = d[..., 0].transpose(0, 1)
            else:
                scale[ids, :, :, tok] = d[..., 0].transpose(0, 1)
        out[n + "_scale"] = scale
    return out


def _exact_evict(s):
    c = s["case"]
    out = {"k": s["k_dst"].double(), "v": s["v_dst"].double(), "sums": s["sums_out"].double(), "kept": s["kept"].clone(), "n": s["n_out"].clone()}
    for q in range(c["seqs"]):
        end = int(s["n_kv"][q])
        n = min(end, int(s["n_keep"][q]))
        recent = min(c["recent"], n)
        first = min(c["first"], n - recent)
        middle = n - first - recent
        for h in range(c["heads"]):
            w = s["sums"][q, h, :end].double()
            best = torch.topk(w[first:end - recent], middle).values
            cut = float(best[-1]) if middle else math.inf
            body = torch.arange(first, end - recent, device=DEV)
            above = body[w[first:end - recent] > cut]
            equal = body[w[first:end - recent] == cut][:middle - len(above)]
            kept = torch.cat([torch.arange(first, device=DEV), torch.cat([above, equal]).sort().values, torch.arange(end - recent, end, device=DEV)])
            out["kept"][q, h, :n] = kept.to(I32)
            out["sums"][q, h, :end] = 0
            out["sums"][q, h, :n] = w[kept]
            for x in ("k", "v"):
                out[x][q, h, :n] = _rows(s, x, q, h, end)[kept]
        out["n"][q] = n
    return out


def _exact_scores(s, q, h):
    """What the queries of sequence q and head h score, with -inf for what they do not see."""
    c = s["case"]
    end, rows = int(s["n_kv"][q]), int(s["n_q"][q])
    at, p = torch.arange(end, device=DEV), end - rows + torch.arange(rows, device=DEV)
    hidden = torch.zeros((rows, end), dtype=torch.bool, device=DEV)
    if c["causal"]:
        hidden |= at > p[:, None]
    if c["window"]:
        hidden |= at <= p[:, None] - c["window"]
    key = _rows(s, "k", q, h * c["kv_heads"] // c["heads"], end)
    return (s["q"][q, :rows, h].double() @ key.T / math.sqrt(c["D"])).masked_fill(hidden, -math.inf)


def _exact_attn(s):
    c = s["case"]
    out = {"dst": s["dst"].double(), "lse": s["lse"].double()}
    for q in range(c["seqs"]):
        rows = int(s["n_q"][q])
        for h in range(c["heads"]):
            if h % (c["heads"] // c["kv_heads"]) == 0:
                val = _rows(s, "v", q, h * c["kv_heads"] // c["heads"], int(s["n_kv"][q]))
            w = _exact_scores(s, q, h)
            out["lse"][q, :rows, h] = torch.logsumexp(w, -1)
            out["dst"][q, :rows, h] = torch.nan_to_num(torch.softmax(w, -1)) @ val
    return out


def _exact_weights(s):
    c = s["case"]
    out = s["sums"].double()
    for q in range(c["seqs"]):
        end, rows = int(s["n_kv"][q]), int(s["n_q"][q])
        for h in range(c["heads"]):
            lse = s["lse"][q, :rows, h].double()[:, None]
            w = torch.exp(_exact_scores(s, q, h) - torch.where(torch.isfinite(lse), lse, 0.0))
            out[q, h * c["kv_heads"] // c["heads"], :end] += w.sum(0)
    return {"sums": out}


def exact(case, seed):
    s = prepare(case, seed)
    return {"qk": _exact_qk, "write": _exact_write, "evict": _exact_evict, "attn": _exact_attn, "weights": _exact_weights}[case["kind"]](s)
