"""The decode step's operators in 4 bits, over ragged batches: what a serving loop calls around the W8A8 linears.

  plan    block tables, slot maps and positions of a step from the requests' lengths, blocks taken from and given back to a free stack
  store   the new tokens' rows of the qkv projection: qk-norm, rotation, K and V into the paged cache in 4 bits, and read back
  attend  one query row per sequence over that cache
  linear  int8 activation codes times 4-bit weights with group scales, for a few rows

What a 4-bit group stands for: of its fp16 values, e is the one of largest magnitude (the positive one of two); the scale is
s = fp16(e / -8), a code is rint(x / s) held to [-8, 7] (0 where s is 0), a value is code * s.

Sizes are the repository's own: hidden 2560, 32 query / 8 kv heads of 128 (and their tensor-parallel shards), SwiGLU 9728, vocabulary
155776, 16-token blocks. K and V are normal values in which a few channels are larger than the rest, as in a trained network.
"""
import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

PACKAGE = "fish_audio_cpp_b200"
DIM, HEADS, KV_HEADS, HEAD_DIM, INTER, VOCAB = 2560, 32, 8, 128, 9728, 155776
QKV, BLOCK, EPS = (HEADS + 2 * KV_HEADS) * HEAD_DIM, 16, 1e-6
F16, F32, F64, I32, I64 = torch.float16, torch.float32, torch.float64, torch.int32, torch.int64


def _package():
    """The package directory carries a hyphen, so it is imported under an explicit module name."""
    if PACKAGE not in sys.modules:
        root = Path.cwd() / "fish-audio-cpp_b200"
        spec = importlib.util.spec_from_file_location(PACKAGE, root / "__init__.py", submodule_search_locations=[str(root)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[PACKAGE] = mod
        spec.loader.exec_module(mod)
    return sys.modules[PACKAGE]


_CTX = []


def _context():
    """The program's one library context (one per stream; everything here runs on the current stream)."""
    if not _CTX:
        torch.cuda.set_device(0)
        _CTX.append(_package().Context(0))
    return _CTX[0]


# ---- the cases -----------------------------------------------------------------------------------------------------


def listed():
    return [
        # One more token for each of eight sequences: what runs before every decode step.
        {"name": "plan_decode_b8", "kind": "plan", "batch": 8, "longest": 2048, "prompts": 0, "prompt": 0, "ended": 0, "room": 8},
        # A loaded server: 512 requests, most of them decoding, 48 prompts admitted, 40 requests over.
        {"name": "plan_mixed_b512", "kind": "plan", "batch": 512, "longest": 16384, "prompts": 48, "prompt": 4096, "ended": 40, "room": 200000},
        # The new rows of a decode step at the headline's batch.
        {"name": "store_b8_g32", "kind": "store", "tokens": 8, "n_q": 32, "n_kv": 8, "group": 32, "norm": True, "layers": 4},
        # A prompt of odd length in a stack without qk-norm.
        {"name": "store_prompt613_g64", "kind": "store", "tokens": 613, "n_q": 32, "n_kv": 8, "group": 64, "norm": False, "layers": 2},
        # The longest prompt there is.
        {"name": "store_prompt8192_g32", "kind": "store", "tokens": 8192, "n_q": 32, "n_kv": 8, "group": 32, "norm": True, "layers": 1},
        # One sequence at the start of its life: latency alone.
        {"name": "attend_b1_ctx37_g32", "kind": "attend", "batch": 1, "longest": 37, "spread": 0, "empty": 0, "n_q": 32, "n_kv": 8, "group": 32, "layers": 4},
        # The headline's batch and context.
        {"name": "attend_b8_ctx1024_g32", "kind": "attend", "batch": 8, "longest": 1024, "spread": 0, "empty": 0, "n_q": 32, "n_kv": 8, "group": 32, "layers": 4},
        # A server's ragged batch, two of its rows empty (a captured step with fewer requests than rows).
        {"name": "attend_b48_ragged_g64", "kind": "attend", "batch": 48, "longest": 8000, "spread": 1, "empty": 2, "n_q": 32, "n_kv": 8, "group": 64, "layers": 1},
        # Two long documents.
        {"name": "attend_b2_ctx131000_g32", "kind": "attend", "batch": 2, "longest": 131000, "spread": 0, "empty": 0, "n_q": 32, "n_kv": 8, "group": 32, "layers": 1},
        # One token through the qkv projection: the smallest linear of the step.
        {"name": "linear_qkv_m1_g128", "kind": "linear", "tokens": 1, "rows": QKV, "k": DIM, "group": 128, "epilogue": "none"},
        # Gate and up projection with SwiGLU at the headline's batch, the exporter's default groups.
        {"name": "linear_gate_up_m8_g64", "kind": "linear", "tokens": 8, "rows": 2 * INTER, "k": DIM, "group": 64, "epilogue": "swiglu"},
        # The whole vocabulary for sixteen sequences: the largest weight there is.
        {"name": "linear_head_m16_g256", "kind": "linear", "tokens": 16, "rows": VOCAB, "k": DIM, "group": 256, "epilogue": "none"},
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["plan", "store", "attend", "attend", "linear", "linear"])
    n_kv = rng.choice([1, 2, 4, 8])
    n_q = n_kv * rng.choice([1, 2, 4, 4, 4, 8] if n_kv < 8 else [1, 2, 4, 4])
    if kind == "plan":
        batch, longest = _spread(rng, 1, 512), _spread(rng, 40, 16384)
        prompts = rng.randint(0, max(0, batch // 8))
        ended = rng.randint(0, max(0, batch // 10))
        prompt = _spread(rng, 2, 4096)
        return {"kind": kind, "batch": batch, "longest": longest, "prompts": prompts, "prompt": prompt, "ended": ended,
                "room": batch + prompts * prompt + rng.randint(0, 100)}
    if kind == "store":
        return {"kind": kind, "tokens": _spread(rng, 1, 8191), "n_q": n_q, "n_kv": n_kv, "group": rng.choice([32, 64, 128]),
                "norm": rng.random() < 0.7, "layers": rng.randint(1, 4)}
    if kind == "attend":
        batch = _spread(rng, 1, 64)
        longest = _spread(rng, 1, min(131000, 262000 // batch))
        return {"kind": kind, "batch": batch, "longest": longest, "spread": rng.randint(0, 1), "empty": rng.randint(0, batch // 8),
                "n_q": n_q, "n_kv": n_kv, "group": rng.choice([32, 64, 128]), "layers": rng.randint(1, 2)}
    k = 32 * _spread(rng, 8, INTER // 32)
    rows = _spread(rng, 17, min(VOCAB, VOCAB * DIM // k))
    epilogue = rng.choice(["none", "none", "residual", "swiglu"])
    if epilogue == "swiglu":
        rows = max(16, rows // 16 * 16)
    return {"kind": kind, "tokens": rng.choice([1, 1, 2, 3, 4, 5, 7, 8, 11, 13, 16]), "rows": rows, "k": k, "group": rng.choice([32, 64, 128, 256]),
            "epilogue": epilogue}


# ---- inputs --------------------------------------------------------------------------------------------------------


def _gen(seed, tag):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + tag)
    return g


def _normal(gen, shape):
    return torch.randn(shape, dtype=F32, device="cuda", generator=gen)


def _channels(gen):
    """Gains of a head's channels: one in sixteen is four times the rest."""
    gain = torch.ones(HEAD_DIM, device="cuda")
    gain[torch.randperm(HEAD_DIM, device="cuda", generator=gen)[:HEAD_DIM // 16]] = 4.0
    return gain


def page_bytes(group):
    """K codes, V codes, then the scales of both, of 16 tokens of one kv head."""
    return 2 * BLOCK * HEAD_DIM // 2 + 2 * BLOCK * (HEAD_DIM // group) * 2


def _codes(x, group):
    """4-bit codes and scales of fp16 rows [..., 128]."""
    v = x.float().unflatten(-1, (HEAD_DIM // group, group))
    hi, lo = v.amax(-1), v.amin(-1)
    e = torch.where(hi >= -lo, hi, lo)
    s = (e / -8).half()
    s32 = s.float()[..., None]
    q = torch.where(s32 == 0, 0.0, torch.round(v / torch.where(s32 == 0, 1.0, s32))).clamp(-8, 7)
    bad = ~torch.isfinite(hi - lo)
    return torch.where(bad[..., None], 0.0, q).flatten(-2), torch.where(bad, float("nan"), s)


def _pages(k, v, group):
    """Pages [..., page_bytes] of fp16 K and V [..., 16, 128]: the cache's layout, in which a lane's 16 bytes are what it multiplies."""
    lead = k.shape[:-2]

    def nibbles(q):  # pairs (even, odd) -> bytes
        q = q.to(torch.uint8)
        return q[..., 0] | (q[..., 1] << 4)

    qk, sk = _codes(k, group)
    qv, sv = _codes(v, group)
    # K: token, quarter j of 8 channels, 32-channel run, nibble: channel 32 run + 8 j + nibble
    kb = nibbles((qk + 8).reshape(*lead, 16, 4, 4, 8).transpose(-3, -2).reshape(*lead, 16, 4, 4, 4, 2)).reshape(*lead, 1024)
    # V: pair of tokens, r, half, low / high, token of the pair, nibble: channel 64 high + 16 nibble + 8 half + r
    t = (qv + 8).reshape(*lead, 8, 2, 2, 4, 2, 8)  # pair, token, high, nibble, half, r
    n = len(lead)
    t = t.permute(*range(n), n, n + 5, n + 4, n + 2, n + 1, n + 3)
    vb = nibbles(t.reshape(*lead, 8, 8, 2, 2, 2, 2, 2)).reshape(*lead, 1024)

    def scales(s):  # pair of tokens, group, token of the pair
        s = s.reshape(*lead, 8, 2, HEAD_DIM // group).transpose(-1, -2).contiguous()
        return s.reshape(*lead, -1).view(torch.uint8)

    return torch.cat([kb, vb, scales(sk), scales(sv)], -1)


def _prepare_plan(c, seed):
    g = _gen(seed, 1)
    b, width = c["batch"], (c["longest"] + c["prompt"] + 1 + BLOCK - 1) // BLOCK
    cached = torch.exp(torch.rand(b, device="cuda", generator=g) * math.log(c["longest"])).int()
    new = torch.ones(b, dtype=I32, device="cuda")
    order = torch.randperm(b, device="cuda", generator=g)
    who = order[:c["prompts"]]
    cached[who] = 0
    if c["prompts"]:
        new[who] = 1 + (torch.rand(c["prompts"], device="cuda", generator=g) * (c["prompt"] - 1)).int()
    new[order[c["prompts"]:c["prompts"] + c["ended"]]] = -1
    capacity = b * width
    perm = torch.randperm(capacity, device="cuda", generator=g).to(I32)
    have = (cached + BLOCK - 1) // BLOCK
    first = torch.cumsum(have, 0) - have
    j = torch.arange(width, device="cuda")[None]
    used = j < have[:, None]
    table = torch.where(used, perm[(first[:, None] + j).clamp(max=capacity - 1)], -1).int()
    taken = int(have.sum())
    free = torch.zeros(capacity, dtype=I32, device="cuda")
    free[:capacity - taken] = perm[taken:]
    room = c["room"]
    return {"c": c, "cached": cached, "new": new, "table": table, "free": free, "count": torch.tensor([capacity - taken], dtype=I32, device="cuda"),
            "left": torch.zeros(1, dtype=I32, device="cuda"), "slots": torch.empty(room, dtype=I64, device="cuda"),
            "positions": torch.empty(room, dtype=I32, device="cuda"), "lens": torch.empty(b, dtype=I32, device="cuda"),
            "first": torch.empty(b + 1, dtype=I32, device="cuda"), "info": torch.empty(4, dtype=I32, device="cuda"),
            "width": width, "capacity": capacity}


def _prepare_store(c, seed):
    g = _gen(seed, 2)
    t, n_q, n_kv = c["tokens"], c["n_q"], c["n_kv"]
    blocks = (t + BLOCK - 1) // BLOCK + 3
    qkv = _normal(g, (t, n_q + 2 * n_kv, HEAD_DIM))
    qkv[:, n_q:n_q + n_kv] *= _channels(g)
    qkv = qkv.half().reshape(t, -1)
    norm = [1 + 0.1 * _normal(g, (HEAD_DIM,)) for _ in range(2)]
    freqs = (1.0 / torch.tensor(1e6, dtype=F64) ** (torch.arange(0, HEAD_DIM, 2, dtype=F64) / HEAD_DIM)).float().cuda()
    table = torch.randperm(blocks, device="cuda", generator=g)
    at = torch.arange(t, device="cuda")
    start = int(torch.randint(0, 2000, (1,), device="cuda", generator=g))
    if t <= 64:  # a decode step: every row is another sequence's
        slots = torch.randperm(blocks * BLOCK, device="cuda", generator=g)[:t]
        positions = torch.randint(0, 2048, (t,), device="cuda", generator=g).int()
    else:
        slots, positions = table[at // BLOCK] * BLOCK + at % BLOCK, (start + at).int()
    cache = torch.zeros((blocks, c["layers"], n_kv, page_bytes(c["group"])), dtype=torch.uint8, device="cuda")
    return {"c": c, "qkv": qkv, "q_norm": norm[0].half() if c["norm"] else None, "k_norm": norm[1].half() if c["norm"] else None, "freqs": freqs,
            "positions": positions, "slots": slots, "cache": cache, "blocks": blocks, "q": torch.empty((t, n_q, HEAD_DIM), dtype=F16, device="cuda"),
            "k": torch.empty((t, n_kv, HEAD_DIM), dtype=F16, device="cuda"), "v": torch.empty((t, n_kv, HEAD_DIM), dtype=F16, device="cuda")}


def _lengths(c, gen):
    b, longest = c["batch"], c["longest"]
    if c["spread"]:
        lens = torch.exp(torch.rand(b, device="cuda", generator=gen) * math.log(longest)).int().clamp(1, longest)
    else:
        lens = longest - (torch.rand(b, device="cuda", generator=gen) * (longest // 16)).int()
    if c["empty"]:
        lens[torch.randperm(b, device="cuda", generator=gen)[:c["empty"]]] = 0
    return lens.int()


def _prepare_attend(c, seed):
    g = _gen(seed, 3)
    b, n_q, n_kv = c["batch"], c["n_q"], c["n_kv"]
    width = (c["longest"] + BLOCK - 1) // BLOCK
    lens = _lengths(c, g)
    used = (lens.long() + BLOCK - 1) // BLOCK
    blocks = max(1, int(used.sum()))  # the pool holds what the batch uses; behind a sequence's end lie an earlier one's rows
    gain = _channels(g)
    cache = torch.empty((blocks, c["layers"], n_kv, page_bytes(c["group"])), dtype=torch.uint8, device="cuda")
    step = 1 << 14
    for at in range(0, blocks, step):
        n = min(step, blocks - at)
        for layer in range(c["layers"]):
            k = (_normal(g, (n, n_kv, BLOCK, HEAD_DIM)) * gain).half()
            v = _normal(g, (n, n_kv, BLOCK, HEAD_DIM)).half()
            cache[at:at + n, layer] = _pages(k, v, c["group"])
    perm = torch.randperm(blocks, device="cuda", generator=g).int()
    first = torch.cumsum(used, 0) - used
    j = torch.arange(width, device="cuda")[None]
    table = torch.where(j < used[:, None], perm[(first[:, None] + j).clamp(max=blocks - 1)], -1).int()
    q = _normal(g, (b, n_q, HEAD_DIM)).half()
    return {"c": c, "q": q, "cache": cache, "table": table, "lens": lens, "blocks": blocks, "width": width,
            "out": torch.empty((b, n_q, HEAD_DIM), dtype=F16, device="cuda")}


def _prepare_linear(c, seed):
    g = _gen(seed, 4)
    m, n, k, group = c["tokens"], c["rows"], c["k"], c["group"]
    groups = (k + group - 1) // group
    w = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=g)
    scale = torch.empty((n, groups), dtype=F32, device="cuda").uniform_(1e-3, 5e-3, generator=g).half()
    x = _normal(g, (m, k))
    x = torch.nn.functional.pad(x, (0, groups * group - k)).reshape(m, groups, group)
    xs = x.abs().amax(-1).clamp(min=1e-8) / 127
    xq = torch.round(x / xs[..., None]).clamp(-127, 127).to(torch.int8).reshape(m, -1)[:, :k].contiguous()
    columns = n // 2 if c["epilogue"] == "swiglu" else n
    return {"c": c, "w": w, "scale": scale, "xq": xq, "xs": xs, "residual": _normal(g, (m, n)).half() if c["epilogue"] == "residual" else None,
            "y": torch.empty((m, columns), dtype=F16, device="cuda")}


def prepare(case, seed):
    return {"plan": _prepare_plan, "store": _prepare_store, "attend": _prepare_attend, "linear": _prepare_linear}[case["kind"]](case, seed)


# ---- one pass ------------------------------------------------------------------------------------------------------


def run(state):
    kind = state["c"]["kind"]
    if own:
        return {"plan": _own_plan, "store": _own_store, "attend": _own_attend, "linear": _own_linear}[kind](state)
    return {"plan": _plain_plan, "store": _plain_store, "attend": _plain_attend, "linear": _plain_linear}[kind](state)


def _own_plan(s):
    c = s["c"]
    _context().plan_blocks(s["cached"], s["new"], c["batch"], s["table"], s["width"], s["free"], s["capacity"], s["count"], s["slots"], s["positions"],
                           s["lens"], s["first"], c["room"], s["info"], free_count_out=s["left"])
    return {n: s[n] for n in ("table", "free", "left", "slots", "positions", "lens", "first", "info")}


def _own_store(s):
    c, ctx = s["c"], _context()
    layer = c["layers"] - 1
    ctx.kv4_write(s["qkv"], s["slots"], s["cache"], s["blocks"], layer, c["layers"], c["tokens"], c["n_q"], c["n_kv"], HEAD_DIM, c["group"],
                  q_norm_w=s["q_norm"], k_norm_w=s["k_norm"], eps=EPS, freqs=s["freqs"], positions=s["positions"], q_out=s["q"])
    ctx.kv4_read(s["cache"], s["blocks"], s["slots"], layer, c["layers"], c["tokens"], c["n_kv"], HEAD_DIM, c["group"], s["k"], s["v"])
    return {"q": s["q"], "k": s["k"], "v": s["v"]}


def _own_attend(s):
    c = s["c"]
    _context().kv4_attention_decode(s["q"], s["cache"], s["blocks"], s["table"], s["lens"], s["out"], c["batch"], c["n_q"], HEAD_DIM, s["width"],
                                    1.0 / math.sqrt(HEAD_DIM), c["layers"] - 1, c["layers"], c["n_kv"], c["group"])
    return s["out"]


def _own_linear(s):
    c, pkg = s["c"], _package()
    epilogue = {"none": pkg.EPI_NONE, "residual": pkg.EPI_RESIDUAL, "swiglu": pkg.EPI_SWIGLU}[c["epilogue"]]
    _context().linear4_q(s["w"], s["scale"], c["group"], s["xq"], s["xs"], s["y"], c["tokens"], c["rows"], c["k"], epilogue=epilogue,
                         residual=s["residual"])
    return s["y"]


# ---- the plain forms -----------------------------------------------------------------------------------------------


def _plain_plan(s):
    cached, new, table, free, count = s["cached"].long(), s["new"].long(), s["table"], s["free"], s["count"].long()
    b, width, room = cached.numel(), s["width"], s["c"]["room"]
    dev = cached.device
    over = new < 0
    add = new.clamp(min=0)
    have = (cached + BLOCK - 1) // BLOCK
    give = torch.where(over, have, 0)
    take = torch.where(over, 0, (cached + add + BLOCK - 1) // BLOCK - have)
    j = torch.arange(width, device=dev)[None]
    # released blocks go on the stack, request by request; index `capacity` catches the rest
    free = torch.cat([free, free.new_zeros(1)])
    gone = j < give[:, None]
    at = torch.where(gone, count + (torch.cumsum(give, 0) - give)[:, None] + j, s["capacity"])
    free[at.reshape(-1)] = torch.where(gone, table, 0).reshape(-1)
    free = free[:s["capacity"]]
    top = count + give.sum()
    # blocks taken come from its top, in order
    fresh = (j >= have[:, None]) & (j < (have + take)[:, None])
    at = top - 1 - ((torch.cumsum(take, 0) - take)[:, None] + j - have[:, None])
    table = torch.where(fresh, free[at.clamp(0, s["capacity"] - 1)], table)
    left = top - take.sum()
    # tokens
    lens = torch.where(over, 0, cached + add)
    first = torch.cat([add.new_zeros(1), torch.cumsum(add, 0)])
    t = torch.arange(room, device=dev)
    who = torch.searchsorted(first, t, right=True) - 1
    real = t < first[-1]
    who = who.clamp(max=b - 1)
    pos = cached[who] + t - first[who]
    block = table[who, torch.where(real, pos // BLOCK, 0)].long()
    slots = torch.where(real, block * BLOCK + pos % BLOCK, -1)
    positions = torch.where(real, pos, 0).int()
    info = torch.stack([torch.zeros_like(top[0]), first[-1], take.sum(), left[0]]).int()
    return {"table": table, "free": free, "left": left.int(), "slots": slots, "positions": positions, "lens": lens.int(), "first": first.int(),
            "info": info}


def _normed(x, weight):
    v = x.float()
    return (v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS) * weight.float()).half()


def _rotated(x, freqs, positions):
    """Interleaved pairs; the angle is the fp32 product, as in the framework's other rotations."""
    angle = (positions.float()[:, None] * freqs[None]).double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[..., 0::2].float(), x[..., 1::2].float()
    return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2).half()


def _held(x, group):
    """What the 4-bit groups of fp16 rows stand for."""
    q, s = _codes(x, group)
    return (q.unflatten(-1, (-1, group)) * s.float()[..., None]).flatten(-2).half()


def _plain_store(s):
    c = s["c"]
    t, n_q, n_kv = c["tokens"], c["n_q"], c["n_kv"]
    q, k, v = s["qkv"].view(t, -1, HEAD_DIM).split([n_q, n_kv, n_kv], 1)
    if s["q_norm"] is not None:
        q, k = _normed(q, s["q_norm"]), _normed(k, s["k_norm"])
    q, k = _rotated(q, s["freqs"], s["positions"]), _rotated(k, s["freqs"], s["positions"])
    return {"q": q, "k": _held(k, c["group"]), "v": _held(v, c["group"])}


def _halves(b):
    """The two 4-bit numbers of a byte, the low one first, in a new last dimension; as signed codes."""
    return torch.stack([b & 15, b >> 4], -1).to(F32) - 8


def _opened(p, group):
    """K and V [..., 16, 128] in fp32 of pages [..., page_bytes]."""
    lead, n = p.shape[:-1], p.dim() - 1
    k = _halves(p[..., :1024]).view(*lead, 16, 4, 4, 8).transpose(-3, -2).reshape(*lead, 16, HEAD_DIM)
    v = _halves(p[..., 1024:2048]).view(*lead, 8, 8, 2, 2, 2, 4)  # pair, r, half, high, token, nibble
    v = v.permute(*range(n), n, n + 4, n + 3, n + 5, n + 2, n + 1).reshape(*lead, 16, HEAD_DIM)
    groups = HEAD_DIM // group
    s = p[..., 2048:].contiguous().view(F16).float().view(*lead, 2, 8, groups, 2).transpose(-1, -2).reshape(*lead, 2, 16, groups, 1)
    k = (k.unflatten(-1, (groups, group)) * s[..., 0, :, :, :]).flatten(-2)
    v = (v.unflatten(-1, (groups, group)) * s[..., 1, :, :, :]).flatten(-2)
    return k, v


def _plain_attend(s):
    c = s["c"]
    b, n_q, n_kv, width = c["batch"], c["n_q"], c["n_kv"], s["width"]
    p = s["cache"][:, c["layers"] - 1][s["table"].clamp(min=0).long()]  # [b, width, n_kv, page]
    k, v = _opened(p, c["group"])
    k = k.transpose(1, 2).reshape(b, n_kv, width * BLOCK, HEAD_DIM)
    v = v.transpose(1, 2).reshape(b, n_kv, width * BLOCK, HEAD_DIM)
    q = s["q"].float().view(b, n_kv, n_q // n_kv, HEAD_DIM)
    score = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(HEAD_DIM)
    there = torch.arange(width * BLOCK, device=q.device)[None] < s["lens"][:, None]
    score = torch.where(there[:, None, None], score, -1e30)
    w = torch.where(there[:, None, None], torch.exp(score - score.amax(-1, keepdim=True)), 0.0)
    out = torch.matmul(w, v) / w.sum(-1, keepdim=True).clamp(min=1e-30)
    return out.reshape(b, n_q, HEAD_DIM).half()


def _silu_product(y):
    """Rows of the weight come in blocks of 16: eight of the gate, then eight of the up projection."""
    gate, up = y.view(y.shape[0], -1, 2, 8).unbind(2)
    gate, up = gate.half().float(), up.half().float()
    return ((gate / (1 + torch.exp(-gate))).half().float() * up).half().flatten(1)


def _plain_linear(s):
    c = s["c"]
    m, n, k, group = c["tokens"], c["rows"], c["k"], c["group"]
    groups = s["scale"].shape[1]
    low, high = s["w"] & 15, s["w"] >> 4
    w = torch.stack([low, high], -1).view(n, k).to(F32)
    w = w - 16 * (w > 7)
    x = s["xq"].float()
    if groups * group > k:
        w, x = torch.nn.functional.pad(w, (0, groups * group - k)), torch.nn.functional.pad(x, (0, groups * group - k))
    sums = torch.bmm(x.view(m, groups, group).transpose(0, 1), w.view(n, groups, group).permute(1, 2, 0))  # whole numbers, exact in fp32
    y = (sums * s["scale"].float().t()[:, None] * s["xs"].t()[:, :, None]).sum(0)
    if c["epilogue"] == "swiglu":
        return _silu_product(y)
    y = y.half()
    return y if s["residual"] is None else (y.float() + s["residual"].float()).half()


# ---- what one pass cannot do without -------------------------------------------------------------------------------


def work(case):
    c, kind = case, case["kind"]
    if kind == "plan":
        tokens = c["batch"] + c["prompts"] * (c["prompt"] // 2)
        blocks = tokens // BLOCK + c["ended"] * (c["longest"] // (BLOCK * 8)) + 1
        return {"bytes": 12 * c["room"] + 16 * c["batch"] + 8 * blocks + 24, "flops": 4 * c["room"]}
    if kind == "store":
        per_head = HEAD_DIM // 2 + 2 * (HEAD_DIM // c["group"])
        row = 2 * HEAD_DIM
        bytes_ = c["tokens"] * (row * (c["n_q"] + 2 * c["n_kv"]) + row * c["n_q"] + 2 * c["n_kv"] * (2 * per_head + row) + 20)
        return {"bytes": bytes_, "flops": c["tokens"] * HEAD_DIM * (10 * (c["n_q"] + c["n_kv"]) + 12 * c["n_kv"])}
    if kind == "attend":
        mean = c["longest"] / max(1.0, math.log(max(2, c["longest"]))) if c["spread"] else c["longest"] * 31 / 32
        tokens = (c["batch"] - c["empty"]) * mean
        per_token = c["n_kv"] * (HEAD_DIM + 4 * (HEAD_DIM // c["group"])) + 4 / BLOCK
        return {"bytes": tokens * per_token + 4 * c["batch"] * c["n_q"] * HEAD_DIM, "flops": tokens * c["n_q"] * 4 * HEAD_DIM}
    m, n, k = c["tokens"], c["rows"], c["k"]
    groups = (k + c["group"] - 1) // c["group"]
    columns = n // 2 if c["epilogue"] == "swiglu" else n * (2 if c["epilogue"] == "residual" else 1)
    return {"bytes": n * k // 2 + 2 * n * groups + m * k + 4 * m * groups + 2 * m * columns, "flops": 2 * m * n * k}


# ---- the same from the definitions, in 64 bits ---------------------------------------------------------------------


def _exact_held(x, group):
    """x: fp64 rows that hold fp16 values."""
    v = x.reshape(*x.shape[:-1], HEAD_DIM // group, group)
    at = v.abs().argmax(-1, keepdim=True)
    e = v.gather(-1, at)
    both = (v == -e).any(-1, keepdim=True)
    e = torch.where(both, e.abs(), e)
    s = (e / -8).half().double()
    q = torch.round(v / torch.where(s == 0, 1.0, s)).clamp(-8, 7) * (s != 0)
    return (q * s).reshape(x.shape)


def _exact_store(s):
    c = s["c"]
    t, n_q, n_kv = c["tokens"], c["n_q"], c["n_kv"]
    x = s["qkv"].double().view(t, n_q + 2 * n_kv, HEAD_DIM)
    head, v = x[:, :n_q + n_kv], x[:, n_q + n_kv:]
    if s["q_norm"] is not None:
        weight = torch.cat([s["q_norm"].expand(n_q, -1), s["k_norm"].expand(n_kv, -1)]).double()
        head = (head / torch.sqrt((head ** 2).sum(-1, keepdim=True) / HEAD_DIM + EPS) * weight).half().double()
    turn = torch.polar(torch.ones((), dtype=F64, device=x.device), (s["positions"].float()[:, None] * s["freqs"][None]).double())
    head = torch.view_as_real(torch.view_as_complex(head.reshape(t, n_q + n_kv, HEAD_DIM // 2, 2).contiguous()) * turn[:, None]).flatten(-2)
    return {"q": head[:, :n_q], "k": _exact_held(head[:, n_q:].half().double(), c["group"]), "v": _exact_held(v, c["group"])}


def _exact_attend(s):
    c = s["c"]
    n_kv, ratio, group, dev = c["n_kv"], c["n_q"] // c["n_kv"], c["group"], s["q"].device
    token, channel = torch.arange(BLOCK)[:, None], torch.arange(HEAD_DIM)[None]
    # where the page keeps the code of (token, channel), as a count of 4-bit places, and its scale, as a count of fp16 values
    at_k = token * 128 + (channel % 32 // 8) * 32 + channel // 32 * 8 + channel % 8
    at_v = 2048 + token // 2 * 256 + channel % 8 * 32 + channel // 8 % 2 * 16 + channel // 64 * 8 + token % 2 * 4 + channel // 16 % 4
    groups = HEAD_DIM // group
    at_s = 1024 + token // 2 * groups * 2 + channel // group * 2 + token % 2
    at_k, at_v, at_s = (a.reshape(-1).to(dev) for a in (at_k, at_v, at_s))
    out = torch.zeros((c["batch"], c["n_q"], HEAD_DIM), dtype=F64, device=dev)
    for b, length in enumerate(s["lens"].tolist()):
        if not length:
            continue
        pages = s["cache"][s["table"][b, :(length + BLOCK - 1) // BLOCK].long(), c["layers"] - 1]
        halfs = pages.view(F16)
        for h in range(n_kv):
            def rows(at, scale):
                code = (pages[:, h][:, at // 2].int() >> (at % 2 * 4).int()) & 15
                return ((code - 8).double() * halfs[:, h][:, scale].double()).reshape(-1, HEAD_DIM)[:length]

            score = s["q"][b, h * ratio:(h + 1) * ratio].double() @ rows(at_k, at_s).T / math.sqrt(HEAD_DIM)
            out[b, h * ratio:(h + 1) * ratio] = torch.softmax(score, -1) @ rows(at_v, at_s + BLOCK * groups)
    return out


def _exact_linear(s):
    c = s["c"]
    n, k, group = c["rows"], c["k"], c["group"]
    out = []
    for at in range(0, n, 16384):
        part = s["w"][at:at + 16384]
        w = torch.empty((part.shape[0], k), dtype=F64, device=part.device)
        w[:, 0::2] = ((part << 4).view(torch.int8) // 16).double()
        w[:, 1::2] = (part.view(torch.int8) >> 4).double()
        w *= s["scale"][at:at + 16384].double().repeat_interleave(group, 1)[:, :k]
        out.append((s["xq"].double() * s["xs"].double().repeat_interleave(group, 1)[:, :k]) @ w.T)
    y = torch.cat(out, 1)
    if c["epilogue"] == "swiglu":
        y = y.view(y.shape[0], -1, 2, 8)
        return (y[:, :, 0] * torch.sigmoid(y[:, :, 0]) * y[:, :, 1]).flatten(1)
    return y if s["residual"] is None else y + s["residual"].double()


def exact(case, seed):
    if case["kind"] == "plan":
        return None
    s = prepare(case, seed)
    return {"store": _exact_store, "attend": _exact_attend, "linear": _exact_linear}[case["kind"]](s)
