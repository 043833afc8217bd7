"""The decode step in 4 bits on the GPU against its restatement in 64 bits: step plan, cache writes and reads, attention, linear."""
import math

import numpy as np
import pytest
import torch

from oracle import q4

pytestmark = pytest.mark.gpu

D, BS = 128, 16


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def i32(*shape, fill=-7):
    return torch.full(shape, fill, dtype=torch.int32, device="cuda")


# ---- the step plan -------------------------------------------------------------------------------------------------


def run_plan(ctx, cached, new, table, free, count, max_tokens, in_place=False, offset=0):
    B, width = len(cached), len(table[0]) if table else 1
    d = dict(cached=dev(np.array(cached, np.int32)), new=dev(np.array(new, np.int32)), table=dev(np.array(table, np.int32).reshape(B, width)),
             free=dev(np.array(free, np.int32)), count=dev(np.array([count], np.int32)))
    slots = torch.full((max_tokens + offset,), -7, dtype=torch.int64, device="cuda")[offset:]
    positions = i32(max_tokens + offset)[offset:]
    lens = d["cached"] if in_place else i32(B)
    first, info, left = i32(B + 1), i32(4), d["count"] if in_place else i32(1)
    ctx.plan_blocks(d["cached"], d["new"], B, d["table"], width, d["free"], len(free), d["count"], slots, positions, lens, first, max_tokens, info,
                    free_count_out=None if in_place else left)
    torch.cuda.synchronize()
    got = dict(table=d["table"].tolist(), free=d["free"].tolist(), left=left.item(), slots=slots.tolist(), positions=positions.tolist(),
               seq_lens=lens.tolist(), first=first.tolist(), info=info.tolist())
    if not in_place:
        assert d["cached"].tolist() == list(cached) and d["count"].item() == count
    return got


def plan_case(rng, B, longest, prompts, prompt, ended, spare=40):
    width = (longest + prompt + 1 + BS - 1) // BS
    cached = rng.integers(0, longest + 1, B)
    new = rng.integers(0, 3, B)
    who = rng.permutation(B)
    cached[who[:prompts]] = 0
    new[who[:prompts]] = rng.integers(1, prompt + 1, prompts)
    new[who[prompts:prompts + ended]] = -rng.integers(1, 5, len(who[prompts:prompts + ended]))
    have = (cached + BS - 1) // BS
    take = np.where(new < 0, 0, (cached + np.maximum(new, 0) + BS - 1) // BS - have)
    capacity = int(have.sum() + take.sum() + spare)
    perm = rng.permutation(capacity)
    table = np.full((B, width), -1)
    at = 0
    for b in range(B):
        table[b, :have[b]] = perm[at:at + have[b]]
        at += have[b]
    free = np.concatenate([perm[at:], np.full(at, -99)])
    return cached.tolist(), new.tolist(), table.tolist(), free.tolist(), capacity - at


@pytest.mark.parametrize("B,longest,prompts,prompt,ended", [(1, 40, 0, 1, 0), (1, 0, 1, 100, 0), (8, 300, 0, 1, 0), (7, 64, 2, 33, 3), (40, 500, 6, 700, 8),
                                                            (33, 16, 33, 64, 0), (300, 200, 20, 500, 100), (1500, 60, 40, 300, 200), (4096, 40, 0, 1, 4000)])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan_blocks(ctx, B, longest, prompts, prompt, ended, in_place):
    rng = np.random.default_rng(B + longest)
    case = plan_case(rng, B, longest, prompts, prompt, ended)
    tokens = sum(n for n in case[1] if n > 0) + int(rng.integers(0, 9))
    want = q4.plan(*case, max_tokens=tokens, capacity=len(case[3]))
    assert want["info"][0] == 0
    assert run_plan(ctx, *case, tokens, in_place=in_place) == want


@pytest.mark.parametrize("B,tokens", [(128, 512), (128, 513), (129, 512), (127, 300)])
def test_plan_blocks_around_one_round_of_few_threads(ctx, B, tokens):
    case = plan_case(np.random.default_rng(B + tokens), B, 50, 2, 60, 5)
    assert run_plan(ctx, *case, tokens) == q4.plan(*case, max_tokens=tokens, capacity=len(case[3]))


def test_plan_blocks_odd_addresses_and_no_requests(ctx):
    rng = np.random.default_rng(1)
    case = plan_case(rng, 9, 90, 3, 50, 1)
    tokens = sum(n for n in case[1] if n > 0) + 3
    assert run_plan(ctx, *case, tokens, offset=1) == q4.plan(*case, max_tokens=tokens, capacity=len(case[3]))
    nothing = run_plan(ctx, [], [], [], [5, 6], 2, 5)
    assert nothing["info"] == [0, 0, 0, 2] and nothing["slots"] == [-1] * 5 and nothing["first"] == [0] and nothing["left"] == 2
    full = run_plan(ctx, [16], [0], [[3, -1]], [5, 6], 2, 0)
    assert full["info"] == [0, 0, 0, 2] and full["seq_lens"] == [16] and full["table"] == [[3, -1]]


def test_plan_blocks_unmapped_rows_have_no_slots(ctx):
    """A cached block that the table does not name: its tokens get no slot."""
    got = run_plan(ctx, [3, 20], [2, 1], [[-1, -1], [4, -1]], [9], 1, 4)
    assert got["slots"] == [-1, -1, -1, -1] and got["info"] == [0, 3, 0, 1] and got["positions"] == [3, 4, 20, 0]


@pytest.mark.parametrize("status,change", [(1, dict(count=2)), (2, dict(cached0=16 * 6)), (3, dict(max_tokens=60)), (4, dict(cached0=-1)), (5, dict(count=-1)),
                                           (5, dict(count=-1, new=[0, 0, 0])), (5, dict(count=9)), (1, dict(new0=2**31 - 1)), (5, dict(cached0=2**31 - 1, new0=-1)),
                                           (1, dict(cached0=2**31 - 1, new0=2**31 - 1))])
def test_plan_blocks_all_or_nothing(ctx, status, change):
    cached, new = [16 * 3, 0, 20], [40, 30, -1]
    table = [[0, 1, 2, -1, -1, -1], [-1] * 6, [3, 4, -1, -1, -1, -1]]
    free = [7, 8, 9, 10, 11, 12, 13, -5, -5]
    new = change.get("new", new)
    cached[0], new[0] = change.get("cached0", cached[0]), change.get("new0", new[0])
    count, max_tokens = change.get("count", 7), change.get("max_tokens", 100)
    want = q4.plan(cached, new, table, free, count, max_tokens, len(free))
    assert want["info"][0] == status
    assert run_plan(ctx, cached, new, table, free, count, max_tokens) == want


def test_plan_blocks_steps_of_a_captured_graph(ctx):
    """The same captured call for every step of a batch: lengths and the stack are updated in place, tables grow, ended rows give back."""
    B, width, capacity = 6, 5, 24
    cached, table, free = [0] * B, [[-1] * width for _ in range(B)], list(range(100, 100 + capacity))
    count, rng = capacity, np.random.default_rng(3)
    d = dict(cached=dev(np.zeros(B, np.int32)), new=i32(B, fill=0), table=dev(np.array(table, np.int32)), free=dev(np.array(free, np.int32)),
             count=i32(1, fill=count))
    slots, positions, first, info = torch.empty(64, dtype=torch.int64, device="cuda"), i32(64), i32(B + 1), i32(4)
    side = torch.cuda.Stream()

    def call():
        ctx.plan_blocks(d["cached"], d["new"], B, d["table"], width, d["free"], capacity, d["count"], slots, positions, d["cached"], first, 64, info)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        call()  # nothing is new yet
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            call()
    for step in range(40):
        new = [int(x) for x in rng.integers(0, 9, B)]
        for b in range(B):
            if cached[b] + new[b] > 16 * width or (cached[b] and rng.random() < 0.15):
                new[b] = -1
        want = q4.plan(cached, new, table, free, count, 64, capacity)
        assert want["info"][0] == 0
        d["new"].copy_(dev(np.array(new, np.int32)))
        graph.replay()
        torch.cuda.synchronize()
        assert info.tolist() == want["info"] and slots.tolist() == want["slots"] and positions.tolist() == want["positions"]
        assert d["table"].tolist() == want["table"] and d["free"].tolist() == want["free"] and d["cached"].tolist() == want["seq_lens"]
        cached, table, free, count = want["seq_lens"], want["table"], want["free"], want["left"]
        live = [p for b in range(B) for p in table[b][:(cached[b] + 15) // 16]] + free[:count]
        assert sorted(live) == list(range(100, 100 + capacity))  # no block is lost or held twice


# ---- cache writes and reads ----------------------------------------------------------------------------------------


def wild_rows(rng, shape):
    """Normal values over many magnitudes, with zeros, subnormals, the largest fp16 and groups that are all the same."""
    x = rng.standard_normal(shape) * np.exp2(rng.integers(-24, 14, shape[:-1] + (1,)))
    x = np.clip(x, -65504, 65504).astype(np.float16)
    flat = x.reshape(-1, D)
    flat[::7, :40] = 0
    flat[1::11] = np.float16(6e-8) * rng.integers(-20, 21, flat[1::11].shape).astype(np.float16)
    flat[2::13, 5] = 65504
    flat[3::17] = flat[3::17, :1]
    return x


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("tokens,n_q,n_kv", [(1, 4, 1), (8, 32, 8), (37, 3, 3), (700, 8, 2)])
def test_kv4_write_is_the_rounding_of_the_groups(ctx, group, tokens, n_q, n_kv):
    """Without norm and rotation: codes and scales of k and v bit for bit, q untouched, and nothing else of the cache written."""
    rng = np.random.default_rng(tokens + group)
    blocks, layers, layer = tokens // 16 + 4, 3, 1
    qkv = wild_rows(rng, (tokens, n_q + 2 * n_kv, D))
    slots = rng.permutation(blocks * 16)[:tokens].astype(np.int64)
    page = q4.page_bytes(group)
    before = rng.integers(0, 256, (blocks, layers, n_kv, page), dtype=np.uint8)
    cache, q_out = dev(before), torch.zeros((tokens, n_q, D), dtype=torch.float16, device="cuda")
    ctx.kv4_write(dev(qkv), dev(slots), cache, blocks, layer, layers, tokens, n_q, n_kv, D, group, q_out=q_out)
    torch.cuda.synchronize()
    assert np.array_equal(q_out.cpu().numpy().view(np.uint16), qkv[:, :n_q].view(np.uint16))
    k_at, v_at, ks, vs = q4.page_places(group)
    nib = np.empty((blocks, layers, n_kv, 4096), np.uint8)
    nib[..., 0::2], nib[..., 1::2] = before[..., :2048] & 15, before[..., :2048] >> 4
    half = before.copy().view(np.uint16)
    for x, at, scale in ((qkv[:, n_q:n_q + n_kv], k_at, ks), (qkv[:, n_q + n_kv:], v_at, vs)):
        codes, s = q4.quantize(x, group)
        for t in range(tokens):
            b, r = slots[t] // 16, slots[t] % 16
            nib[b, layer][:, at[r]] = codes[t] + 8
            half[b, layer][:, scale[r, ::group]] = s[t].view(np.uint16)
    want = half.view(np.uint8)
    want[..., :2048] = nib[..., 0::2] | nib[..., 1::2] << 4
    got = cache.cpu().numpy()
    same = got == want
    # (-0 and 0 are the same scale: a group of zeros has either)
    zero = (got.view(np.uint16) & 0x7fff == 0) & (want.view(np.uint16) & 0x7fff == 0)
    assert (same[..., :2048]).all() and ((got.view(np.uint16) == want.view(np.uint16)) | zero)[..., 1024:].all()
    # and what is read back is what the groups stand for, rounded to fp16
    k, v = (torch.empty((tokens, n_kv, D), dtype=torch.float16, device="cuda") for _ in range(2))
    ctx.kv4_read(cache, blocks, dev(slots), layer, layers, tokens, n_kv, D, group, k, v)
    torch.cuda.synchronize()
    for got, x in ((k, qkv[:, n_q:n_q + n_kv]), (v, qkv[:, n_q + n_kv:])):
        assert np.array_equal(got.cpu().numpy(), q4.values(*q4.quantize(x, group), group).astype(np.float16))


def test_kv4_codes_at_every_border(ctx):
    """Values that lie on or next to the border between two codes, for scales of every kind: the codes are those of exact arithmetic."""
    rng = np.random.default_rng(0)
    rows = []
    for _ in range(3000):
        s = np.float16(np.uint16(rng.integers(1, 0x6c00)).view(np.float16))
        ext = np.float16(float(s) * 8)
        border = np.float16((rng.integers(-8, 8, 127) + 0.5) * float(s))
        bits = border.view(np.uint16).astype(np.int64) + rng.integers(-2, 3, 127)
        x = np.concatenate([[ext], np.clip(bits, 0, 0xffff).astype(np.uint16).view(np.float16)])
        x = np.where(np.abs(x) <= abs(ext), x, np.float16(0)).astype(np.float16)
        rows.append(x * np.float16(rng.choice([-1, 1])))
    x = np.stack(rows).reshape(-1, 1, D)
    x = np.where(np.isfinite(x), x, np.float16(0))
    T = x.shape[0]
    qkv = np.concatenate([x, x], 1)
    cache = torch.zeros((T // 16 + 1, 1, 1, q4.page_bytes(128)), dtype=torch.uint8, device="cuda")
    slots = torch.arange(T, dtype=torch.int64, device="cuda")
    k, v = (torch.empty((T, 1, D), dtype=torch.float16, device="cuda") for _ in range(2))
    ctx.kv4_write(dev(qkv), slots, cache, T // 16 + 1, 0, 1, T, 0, 1, D, 128)
    ctx.kv4_read(cache, T // 16 + 1, slots, 0, 1, T, 1, D, 128, k, v)
    torch.cuda.synchronize()
    want = q4.values(*q4.quantize(x, 128), 128).astype(np.float16)
    assert np.array_equal(k.cpu().numpy(), want) and np.array_equal(v.cpu().numpy(), want)


@pytest.mark.parametrize("B,with_norm,group", [(1, True, 32), (8, True, 64), (37, False, 128)])
def test_kv4_write_holds_what_the_fp16_cache_holds(ctx, oracle, B, with_norm, group):
    """q, and k and v before they are held in 4 bits, are those of w8a8_qknorm_rope_kvwrite, bit for bit."""
    rng = np.random.default_rng(B)
    n_q, n_kv, layers, layer, width = 32, 8, 2, 1, 300
    qkv = dev(rng.standard_normal((B, (n_q + 2 * n_kv) * D)).astype(np.float16))
    qw, kw = (dev(rng.uniform(0.5, 1.5, D).astype(np.float16)) if with_norm else None for _ in range(2))
    freqs, positions = dev(oracle.rope_freqs(D, 1e6)), rng.integers(0, width * BS, B).astype(np.int32)
    table = (np.arange(B)[:, None] + np.zeros((1, width))).astype(np.int32)  # a block a sequence
    kc, vc = (torch.zeros((B, layers, n_kv, BS, D), dtype=torch.float16, device="cuda") for _ in range(2))
    q16, q = (torch.empty((B, n_q, D), dtype=torch.float16, device="cuda") for _ in range(2))
    ctx.qknorm_rope_kvwrite(qkv, qw, kw, 1e-6, freqs, dev(positions), dev(table), width, kc, vc, layer, layers, B, n_q, n_kv, D, q16)
    slots = np.arange(B, dtype=np.int64) * BS + positions % BS
    cache = torch.zeros((B, layers, n_kv, q4.page_bytes(group)), dtype=torch.uint8, device="cuda")
    ctx.kv4_write(qkv, dev(slots), cache, B, layer, layers, B, n_q, n_kv, D, group, q_norm_w=qw, k_norm_w=kw, eps=1e-6, freqs=freqs,
                  positions=dev(positions), q_out=q)
    k, v = (torch.empty((B, n_kv, D), dtype=torch.float16, device="cuda") for _ in range(2))
    ctx.kv4_read(cache, B, dev(slots), layer, layers, B, n_kv, D, group, k, v)
    torch.cuda.synchronize()
    assert torch.equal(q, q16)
    at = np.arange(B)
    for got, c in ((k, kc), (v, vc)):
        x = c.cpu().numpy()[at, layer, :, positions % BS]
        assert np.array_equal(got.cpu().numpy(), q4.values(*q4.quantize(x, group), group).astype(np.float16))


def test_kv4_rows_without_a_slot_are_left_alone(ctx):
    rng = np.random.default_rng(2)
    T, n_q, n_kv, blocks, group = 9, 4, 1, 3, 32
    qkv = rng.standard_normal((T, n_q + 2 * n_kv, D)).astype(np.float16)
    slots = np.array([5, -1, 47, 48, 2**40, -2**40, 0, 1, -1], np.int64)  # 48 and 2^40 lie behind the last block
    before = rng.integers(0, 256, (blocks, 1, n_kv, q4.page_bytes(group)), dtype=np.uint8)
    cache, q = dev(before), torch.full((T, n_q, D), 7.0, dtype=torch.float16, device="cuda")
    ctx.kv4_write(dev(qkv), dev(slots), cache, blocks, 0, 1, T, n_q, n_kv, D, group, q_out=q)
    k, v = (torch.full((T, n_kv, D), 9.0, dtype=torch.float16, device="cuda") for _ in range(2))
    ctx.kv4_read(cache, blocks, dev(slots), 0, 1, T, n_kv, D, group, k, v)
    torch.cuda.synchronize()
    real = np.array([0, 2, 6, 7])
    rest = np.setdiff1d(np.arange(T), real)
    assert torch.equal(q[real].cpu(), torch.from_numpy(qkv[real, :n_q])) and (q[rest] == 7).all() and (k[rest] == 9).all() and (v[rest] == 9).all()
    assert np.array_equal(k[real].cpu().numpy(), q4.values(*q4.quantize(qkv[real, n_q:n_q + 1], group), group).astype(np.float16))
    after = cache.cpu().numpy()
    assert np.array_equal(after[1], before[1])  # no real slot lies there
    only_k = torch.full((T, n_kv, D), 9.0, dtype=torch.float16, device="cuda")
    ctx.kv4_read(cache, blocks, dev(slots), 0, 1, T, n_kv, D, group, only_k, None)
    assert torch.equal(only_k, k)


def test_kv4_rows_that_are_no_numbers(ctx):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((4, 3, D)).astype(np.float16)
    x[0, 1, 5], x[1, 2, 70], x[2, 1, 127], x[3, 2, 0] = np.nan, np.inf, -np.inf, np.nan
    cache = torch.zeros((1, 1, 1, q4.page_bytes(32)), dtype=torch.uint8, device="cuda")
    slots = torch.arange(4, dtype=torch.int64, device="cuda")
    k, v = (torch.empty((4, 1, D), dtype=torch.float16, device="cuda") for _ in range(2))
    ctx.kv4_write(dev(x), slots, cache, 1, 0, 1, 4, 1, 1, D, 32)
    ctx.kv4_read(cache, 1, slots, 0, 1, 4, 1, D, 32, k, v)
    torch.cuda.synchronize()
    for got, i in ((k, 1), (v, 2)):
        assert np.array_equal(got.cpu().numpy(), q4.values(*q4.quantize(x[:, i:i + 1], 32), 32).astype(np.float16), equal_nan=True)


# ---- attention -----------------------------------------------------------------------------------------------------


def attention_case(rng, lens, n_q, n_kv, group, layers, width, spare=2, junk=True):
    """q, pages (rows behind the lengths hold what is no number, where junk), table, lens."""
    B = len(lens)
    used = [(n + 15) // 16 for n in lens]
    blocks = sum(used) + spare
    perm = rng.permutation(blocks)
    gain = np.where(rng.random(D) < 0.06, 4.0, 1.0)
    K = (rng.standard_normal((blocks, layers, n_kv, BS, D)) * gain).astype(np.float16)
    V = rng.standard_normal((blocks, layers, n_kv, BS, D)).astype(np.float16)
    pages = q4.fill_pages(K, V, group)
    table = np.full((B, width), -1, np.int32)
    at = 0
    for b, n in enumerate(lens):
        table[b, :used[b]] = perm[at:at + used[b]]
        at += used[b]
        if junk and n % 16:
            _, _, ks, vs = q4.page_places(group)
            half = pages[table[b, used[b] - 1]].view(np.uint16)
            for scale in (ks, vs):
                half[..., np.unique(scale[n % 16:])] = rng.choice([0x7fff, 0x7c00, 0xfc00])
    if junk:
        pages[perm[at:]] = 255
    q = rng.standard_normal((B, n_q, D)).astype(np.float16)
    return q, pages, table, np.array(lens, np.int32)


def run_attention(ctx, q, pages, table, lens, n_kv, group, layer, sm, quant=0, out=True):
    B, n_q, _ = q.shape
    blocks, layers = pages.shape[:2]
    dout = torch.full((B, n_q, D), 9.0, dtype=torch.float16, device="cuda") if out else None
    xq = torch.full((B, n_q * D), 99, dtype=torch.int8, device="cuda") if quant else None
    xs = torch.full((B, n_q * D // quant), 99.0, dtype=torch.float32, device="cuda") if quant else None
    ctx.kv4_attention_decode(dev(q), dev(pages), blocks, dev(table), dev(lens), dout, B, n_q, D, table.shape[1], sm, layer, layers, n_kv, group,
                             quant_group_size=quant, Xq=xq, Xs=xs)
    torch.cuda.synchronize()
    ctx.check_device_status()
    return dout, xq, xs


def check_attention(ctx, case, n_kv, group, layer, sm):
    want, tol = q4.attention(*case, layer, sm, group)
    got = run_attention(ctx, *case, n_kv, group, layer, sm)[0].cpu().numpy().astype(np.float64)
    assert np.isfinite(got).all()
    worst = (np.abs(got - want).max(-1) / np.maximum(tol, 2.0**-24)).max()
    assert worst <= 1, worst
    for b, n in enumerate(case[3]):
        if n == 0:
            assert (got[b] == 0).all()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("lens", [[1], [15], [16], [17], [0], [33, 0, 1, 160], [5, 300, 0, 0, 1000, 16, 31], [2000] * 8, [0, 0, 7, 0], [1] * 70])
def test_kv4_attention(ctx, group, lens):
    rng = np.random.default_rng(len(lens) + group + lens[0])
    check_attention(ctx, attention_case(rng, lens, 8, 2, group, 2, 130), 2, group, 1, 1 / math.sqrt(D))


@pytest.mark.parametrize("n_q,n_kv", [(1, 1), (2, 1), (3, 1), (4, 1), (5, 1), (8, 1), (32, 8), (14, 2), (6, 6), (15, 3)])
def test_kv4_attention_heads(ctx, n_q, n_kv):
    rng = np.random.default_rng(n_q)
    lens = [40, 0, 3, 500, 129]
    check_attention(ctx, attention_case(rng, lens, n_q, n_kv, 32, 1, 32), n_kv, 32, 0, 0.11)


@pytest.mark.parametrize("n_q,n_kv,lens", [(4, 1, [40000]), (8, 1, [9000, 20000]), (16, 4, [12345, 1, 0, 30000]), (4, 4, [17000])])
def test_kv4_attention_long(ctx, n_q, n_kv, lens):
    """Pairs that lie in many CTAs: the pieces meet in the context's scratch; twice in a row, the tickets are as they were."""
    rng = np.random.default_rng(n_q)
    case = attention_case(rng, lens, n_q, n_kv, 64, 1, max(lens) // 16 + 5)
    for _ in range(2):
        check_attention(ctx, case, n_kv, 64, 0, 1 / math.sqrt(D))
    a = run_attention(ctx, *case, n_kv, 64, 0, 1 / math.sqrt(D))[0]
    for _ in range(5):
        assert torch.equal(a, run_attention(ctx, *case, n_kv, 64, 0, 1 / math.sqrt(D))[0])


def test_kv4_attention_large_batches(ctx):
    rng = np.random.default_rng(8)
    lens = [int(x) for x in rng.integers(0, 60, 1000)]
    check_attention(ctx, attention_case(rng, lens, 4, 1, 128, 1, 4), 1, 128, 0, 0.09)
    lens = [int(x) for x in rng.integers(0, 3, 4096)]
    check_attention(ctx, attention_case(rng, lens, 2, 1, 32, 1, 1), 1, 32, 0, 0.09)


def test_kv4_attention_sharp_and_flat_scores(ctx):
    """One token that takes all the weight, scores far apart, scores all alike, a scale of zero and a negative one."""
    rng = np.random.default_rng(9)
    q, pages, table, lens = attention_case(rng, [700, 64, 1], 4, 1, 32, 1, 44)
    for sm in (4.0, 0.5, 1e-6, 0.0, -0.3):
        check_attention(ctx, (q, pages, table, lens), 1, 32, 0, sm)


@pytest.mark.parametrize("n_q,n_kv,quants", [(32, 8, (64, 256, 512, 4, 32, 128)), (8, 1, (1024, 256)), (3, 1, (128, 64)), (6, 1, (256,))])
def test_kv4_attention_output_codes(ctx, oracle, n_q, n_kv, quants):
    rng = np.random.default_rng(n_q)
    case = attention_case(rng, [3, 0, 900, 77, 5000], n_q, n_kv, 32, 1, 320)
    plain = run_attention(ctx, *case, n_kv, 32, 0, 0.1)[0]
    for g in quants:
        out, xq, xs = run_attention(ctx, *case, n_kv, 32, 0, 0.1, quant=g)
        assert torch.equal(out, plain)
        wq, ws = oracle.quantize(out.cpu().numpy().reshape(5, -1), g)
        assert np.array_equal(xq.cpu().numpy(), wq) and np.array_equal(xs.cpu().numpy(), ws)
        _, only, scales = run_attention(ctx, *case, n_kv, 32, 0, 0.1, quant=g, out=False)
        assert torch.equal(only, xq) and torch.equal(scales, xs)


def test_kv4_attention_lengths_and_blocks_out_of_range(ctx):
    """Lengths are cut at the table's width, negative ones are none; block numbers outside the cache are read as block 0."""
    rng = np.random.default_rng(11)
    q, pages, table, lens = attention_case(rng, [64, 64, 40], 4, 1, 32, 1, 4, junk=False)
    base = run_attention(ctx, q, pages, table, lens, 1, 32, 0, 0.1)[0]
    long = run_attention(ctx, q, pages, table, np.array([2**31 - 1, 65, 40], np.int32), 1, 32, 0, 0.1)[0]
    assert torch.equal(base, long)
    none = run_attention(ctx, q, pages, table, np.array([-5, 64, 40], np.int32), 1, 32, 0, 0.1)[0]
    assert (none[0] == 0).all() and torch.equal(none[1:], base[1:])
    odd, zero = table.copy(), table.copy()
    odd[2, 1], odd[0, 2], zero[2, 1], zero[0, 2] = -9, 2**31 - 1, 0, 0
    assert torch.equal(run_attention(ctx, q, pages, odd, lens, 1, 32, 0, 0.1)[0], run_attention(ctx, q, pages, zero, lens, 1, 32, 0, 0.1)[0])


def test_kv4_attention_nan_stays_in_its_sequence_and_head(ctx):
    rng = np.random.default_rng(12)
    q, pages, table, lens = attention_case(rng, [200, 90, 33], 8, 2, 32, 1, 13)
    clean = run_attention(ctx, q, pages, table, lens, 2, 32, 0, 0.1)[0]
    _, _, ks, vs = q4.page_places(32)
    bad = pages.copy()
    bad[table[1, 2], 0, 1].view(np.float16)[ks[5, 0]] = np.nan   # a key of sequence 1, kv head 1
    bad[table[2, 0], 0, 0].view(np.float16)[vs[3, 64]] = np.nan  # a value's group of sequence 2, kv head 0
    got = run_attention(ctx, q, bad, table, lens, 2, 32, 0, 0.1)[0]
    nan = torch.isnan(got)
    assert nan[1, 4:].all() and nan[2, :4, 64:96].all()
    want = torch.zeros_like(nan)
    want[1, 4:] = True
    want[2, :4, 64:96] = True
    assert torch.equal(nan, want) and torch.equal(got[~nan], clean[~nan])


def test_kv4_cache_past_32_bits(ctx):
    """Offsets beyond 2^32 bytes: the last blocks of a cache of 5 GB."""
    rng = np.random.default_rng(13)
    group, n_kv, layers = 32, 8, 36
    page = q4.page_bytes(group)
    blocks = 5 * 2**30 // (layers * n_kv * page)
    if torch.cuda.mem_get_info()[0] < 8 * 2**30:
        pytest.skip("not enough free device memory")
    cache = torch.zeros(blocks * layers * n_kv * page, dtype=torch.uint8, device="cuda")
    T, n_q, layer = 40, 32, 35
    qkv = rng.standard_normal((T, n_q + 2 * n_kv, D)).astype(np.float16)
    table = np.array([[blocks - 1, blocks - 7, blocks - 2]], np.int32)
    slots = table[0].astype(np.int64)[np.arange(T) // 16] * 16 + np.arange(T) % 16
    q_out = torch.empty((T, n_q, D), dtype=torch.float16, device="cuda")
    ctx.kv4_write(dev(qkv), dev(slots), cache, blocks, layer, layers, T, n_q, n_kv, D, group, q_out=q_out)
    k, v = (torch.empty((T, n_kv, D), dtype=torch.float16, device="cuda") for _ in range(2))
    ctx.kv4_read(cache, blocks, dev(slots), layer, layers, T, n_kv, D, group, k, v)
    out = torch.empty((1, n_q, D), dtype=torch.float16, device="cuda")
    ctx.kv4_attention_decode(q_out[T - 1:], cache, blocks, dev(table), i32(1, fill=T), out, 1, n_q, D, 3, 0.1, layer, layers, n_kv, group)
    torch.cuda.synchronize()
    wk = q4.values(*q4.quantize(qkv[:, n_q:n_q + n_kv], group), group)
    assert np.array_equal(k.cpu().numpy(), wk.astype(np.float16))
    own = cache.view(blocks, layers, n_kv, page)[table[0].tolist()].cpu().numpy()
    want, tol = q4.attention(qkv[T - 1:, :n_q], own, np.array([[0, 1, 2]]), [T], layer, 0.1, group)
    assert (np.abs(out.cpu().numpy() - want).max(-1) <= tol).all()
    del cache


# ---- linear --------------------------------------------------------------------------------------------------------


def linear_case(rng, M, N, K, g):
    G = (K + g - 1) // g
    codes = rng.integers(-8, 8, (N, K))
    scale = rng.uniform(1e-3, 5e-3, (N, G)).astype(np.float16)
    Xq = rng.integers(-127, 128, (M, K)).astype(np.int8)
    Xs = rng.uniform(0.005, 0.05, (M, G)).astype(np.float32)
    return codes, scale, Xq, Xs


def check_linear(ctx, rng, M, N, K, g, epilogue, offset=0):
    """fp32 sums: G groups over at most 16 warps, three roundings a group: (G + 16 + 3) 2^-24 of the sum of magnitudes. Then fp16 (2^-11) for
    every rounding of the epilogue: gate g to g (1 + 2^-11), silu' is at most 1.1, silu and the product round again."""
    codes, scale, Xq, Xs = linear_case(rng, M, N, K, g)
    y, mag = q4.linear(codes, scale, g, Xq, Xs)
    err = (scale.shape[1] + 19) * 2.0**-24 * mag
    W = torch.empty(N * K // 2 + 32, dtype=torch.uint8, device="cuda")[offset:offset + N * K // 2]
    W.copy_(dev(q4.pack_codes(codes)).flatten())
    columns = N // 2 if epilogue == 2 else N
    out = torch.full((M + 1, columns), 7.0, dtype=torch.float16, device="cuda")
    residual = dev(rng.standard_normal((M, N)).astype(np.float16)) if epilogue == 1 else None
    ctx.linear4_q(W, dev(scale), g, dev(Xq), dev(Xs), out, M, N, K, epilogue=epilogue, residual=residual)
    torch.cuda.synchronize()
    got, half = out[:M].cpu().numpy().astype(np.float64), 2.0**-11
    assert (out[M] == 7).all()
    if epilogue == 2:
        gate, up = (a.reshape(M, -1) for a in (y.reshape(M, -1, 2, 8)[:, :, 0], y.reshape(M, -1, 2, 8)[:, :, 1]))
        eg, eu = (a.reshape(M, -1) for a in (err.reshape(M, -1, 2, 8)[:, :, 0], err.reshape(M, -1, 2, 8)[:, :, 1]))
        s = q4.silu(gate)
        ds = 1.1 * (eg + half * np.abs(gate)) + half * np.abs(s) + 2.0**-22
        du = eu + half * np.abs(up)
        want = s * up
        tol = (np.abs(s) + ds) * du + np.abs(up) * ds
        tol = tol + half * (np.abs(want) + tol)
    else:
        want, tol = y, err + half * (np.abs(y) + err)
        if residual is not None:
            want = y + residual.cpu().numpy()
            tol = tol + half * (np.abs(want) + tol)
    worst = (np.abs(got - want) / (tol + 2.0**-24)).max()
    assert worst <= 1, worst


@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 16, 17, 32, 33])
@pytest.mark.parametrize("N,K,g", [(16, 128, 128), (640, 2560, 64), (2560, 1024, 256), (33, 4096, 32), (1000, 320, 96), (48, 160, 128), (272, 9728, 128),
                                   (64, 96, 0), (8, 32, 32)])
def test_linear4(ctx, M, N, K, g):
    check_linear(ctx, np.random.default_rng(M + N + K + g), M, N, K, g if g else K, 0)


@pytest.mark.parametrize("epilogue", [1, 2])
@pytest.mark.parametrize("M,N,K,g", [(1, 640, 512, 64), (8, 1024, 2560, 32), (13, 160, 384, 128), (40, 64, 256, 256), (3, 16, 66, 22)])
def test_linear4_epilogues(ctx, epilogue, M, N, K, g):
    check_linear(ctx, np.random.default_rng(M + N), M, N, K, g, epilogue)


@pytest.mark.parametrize("M,N,K,g,offset", [(3, 17, 66, 22, 0), (2, 5, 2, 2, 0), (5, 40, 130, 64, 0), (2, 64, 128, 64, 1), (33, 31, 100, 10, 0), (2, 48, 96, 2000, 8)])
def test_linear4_shapes_of_the_generic_kernel(ctx, M, N, K, g, offset):
    check_linear(ctx, np.random.default_rng(M + N), M, N, K, min(g, K), 0, offset)


@pytest.mark.parametrize("M,N,K,g", [(16, 16, 65536, 32), (33, 16, 32768, 32), (9, 40, 65536, 64), (5, 16, 131072, 128), (32, 33, 16384, 256), (7, 4800, 32, 32)])
def test_linear4_long_rows(ctx, M, N, K, g):
    """Scales and codes that fill shared memory, so that fewer rows go into a launch."""
    check_linear(ctx, np.random.default_rng(K), M, N, K, g, 0)


def test_linear4_sums_are_exact(ctx):
    """Scales of one and the largest codes: whole numbers that fp16 holds come out as they are, and a long group's sum stays exact."""
    rng = np.random.default_rng(5)
    for M, N, K, g in ((4, 32, 2560, 64), (9, 64, 512, 256), (1, 16, 9728, 9728)):
        codes, Xq = rng.integers(-8, 8, (N, K)), np.zeros((M, K), np.int8)
        at = rng.choice(K, 8, replace=False)
        Xq[:, at] = rng.integers(-30, 31, (M, 8))
        ones = np.ones((N, K // g), np.float16)
        out = torch.empty((M, N), dtype=torch.float16, device="cuda")
        ctx.linear4_q(dev(q4.pack_codes(codes)), dev(ones), g, dev(Xq), dev(np.ones((M, K // g), np.float32)), out, M, N, K)
        torch.cuda.synchronize()
        assert np.array_equal(out.cpu().numpy().astype(np.int64), Xq.astype(np.int64) @ codes.T)
        full = np.full((M, K), -127, np.int8)
        tiny = np.full((N, K // g), 2.0**-10, np.float16)
        ctx.linear4_q(dev(q4.pack_codes(np.full((N, K), -8))), dev(tiny), g, dev(full), dev(np.full((M, K // g), 2.0**-8, np.float32)), out, M, N, K)
        torch.cuda.synchronize()
        assert (out.cpu().numpy() == np.float16(127 * 8 * K * 2.0**-18)).all()


def test_linear4_results_do_not_depend_on_the_run(ctx):
    rng = np.random.default_rng(6)
    codes, scale, Xq, Xs = linear_case(rng, 8, 2560, 9728, 64)
    W, s, x, xs = dev(q4.pack_codes(codes)), dev(scale), dev(Xq), dev(Xs)
    outs = [torch.empty((8, 2560), dtype=torch.float16, device="cuda") for _ in range(6)]
    for o in outs:
        ctx.linear4_q(W, s, 64, x, xs, o, 8, 2560, 9728)
    torch.cuda.synchronize()
    assert all(torch.equal(outs[0], o) for o in outs[1:])


@pytest.mark.parametrize("N,K,g", [(5, 64, 32), (64, 2560, 64), (17, 130, 64), (3, 34, 0), (8, 512, 256)])
def test_quantize_and_unpack_weight4(ctx, N, K, g):
    rng = np.random.default_rng(N)
    W = (rng.standard_normal((N, K)) * np.exp2(rng.integers(-20, 8, (N, 1)))).astype(np.float16)
    W[0, :3] = 0
    if N > 4:
        W[4, 1], W[3, K - 1] = np.nan, np.inf
    gg = g if g else K
    codes = torch.zeros((N, K // 2), dtype=torch.uint8, device="cuda")
    scale = torch.zeros((N, (K + gg - 1) // gg), dtype=torch.float16, device="cuda")
    ctx.quantize_weight4(dev(W), N, K, g, codes, scale)
    wide = torch.zeros((N, K), dtype=torch.int8, device="cuda")
    ctx.unpack_weight4(codes, N, K, wide)
    torch.cuda.synchronize()
    want, s = q4.quantize(W, gg)
    assert np.array_equal(wide.cpu().numpy(), want) and np.array_equal(codes.cpu().numpy(), q4.pack_codes(want))
    assert np.array_equal(scale.cpu().numpy(), s, equal_nan=True)


def test_linear4_agrees_with_the_8_bit_linear_over_unpacked_weights(ctx):
    """A prompt runs the W8A8 linear over the unpacked codes: same exact sums, fp32 sums in another order."""
    rng = np.random.default_rng(7)
    M, N, K, g = 24, 512, 1024, 64
    codes, scale, Xq, Xs = linear_case(rng, M, N, K, g)
    W4, s, x, xs = dev(q4.pack_codes(codes)), dev(scale), dev(Xq), dev(Xs)
    W8 = torch.empty((N, K), dtype=torch.int8, device="cuda")
    ctx.unpack_weight4(W4, N, K, W8)
    a, b = (torch.empty((M, N), dtype=torch.float16, device="cuda") for _ in range(2))
    ctx.linear4_q(W4, s, g, x, xs, a, M, N, K)
    ctx.linear_q(W8, s, g, x, xs, b, M, N, K)
    torch.cuda.synchronize()
    _, mag = q4.linear(codes, scale, g, Xq, Xs)
    tol = 2 * (K // g + 19) * 2.0**-24 * mag + 2 * 2.0**-11 * b.abs().cpu().numpy().astype(np.float64)
    assert (np.abs(a.cpu().numpy().astype(np.float64) - b.cpu().numpy()) <= tol + 2.0**-24).all()


# ---- a run of them together ----------------------------------------------------------------------------------------


def test_calls_refuse_another_current_device(ctx):
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    with torch.cuda.device(1), pytest.raises(Exception, match="current device"):
        ctx.unpack_weight4(1 << 20, 2, 2, 1 << 20, stream=0)


@pytest.mark.parametrize("captured", [False, True])
def test_requests_come_and_go(ctx, captured):
    """plan -> write -> attention over several steps of a changing batch (prompts, decoding, an ended request whose blocks another takes),
    with the output's codes going into a 4-bit linear; every step against 64 bits over the history of rows. The captured form replays one graph."""
    rng = np.random.default_rng(21)
    B, n_q, n_kv, group, g, width, capacity, room, N = 3, 8, 2, 32, 64, 6, 12, 48, 64
    K = n_q * D
    page, sm = q4.page_bytes(group), 1 / math.sqrt(D)
    cache = torch.full((capacity, 1, n_kv, page), 255, dtype=torch.uint8, device="cuda")
    cached, new, table = i32(B, fill=0), i32(B, fill=0), i32(B, width, fill=-1)
    free, count = torch.arange(capacity, dtype=torch.int32, device="cuda"), i32(1, fill=capacity)
    slots, positions, first, info = torch.empty(room, dtype=torch.int64, device="cuda"), i32(room), i32(B + 1), i32(4)
    qkv, q = (torch.zeros((room, h, D), dtype=torch.float16, device="cuda") for h in (n_q + 2 * n_kv, n_q))
    last, out = (torch.zeros((B, n_q, D), dtype=torch.float16, device="cuda") for _ in range(2))
    xq, xs = torch.empty((B, K), dtype=torch.int8, device="cuda"), torch.empty((B, K // g), dtype=torch.float32, device="cuda")
    codes, scale, _, _ = linear_case(rng, 1, N, K, g)
    W4, ws, y = dev(q4.pack_codes(codes)), dev(scale), torch.empty((B, N), dtype=torch.float16, device="cuda")

    def step():
        ctx.plan_blocks(cached, new, B, table, width, free, capacity, count, slots, positions, cached, first, room, info)
        ctx.kv4_write(qkv, slots, cache, capacity, 0, 1, room, n_q, n_kv, D, group, q_out=q)
        torch.index_select(q, 0, (first[1:] - 1).clamp(min=0), out=last)
        ctx.kv4_attention_decode(last, cache, capacity, table, cached, out, B, n_q, D, width, sm, 0, 1, n_kv, group, quant_group_size=g, Xq=xq, Xs=xs)
        ctx.linear4_q(W4, ws, g, xq, xs, y, B, N, K)

    run = step
    if captured:
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            step()
            side.synchronize()
            with torch.cuda.graph(graph, stream=side):
                step()
        torch.cuda.synchronize()
        run = graph.replay
    history = [[np.zeros((0, n_kv, D), np.float16)] * 2 for _ in range(B)]
    for news in ([20, 5, 3], [1, 1, 1], [1, 11, 1], [1, -1, 1], [1, 30, 0], [-1, 1, 1], [40, 1, 1], [1, 1, -1], [1, 1, 7]):
        rows = rng.standard_normal((room, n_q + 2 * n_kv, D)).astype(np.float16)
        qkv.copy_(dev(rows))
        new.copy_(dev(np.array(news, np.int32)))
        run()
        torch.cuda.synchronize()
        ctx.check_device_status()
        assert info[0].item() == 0
        at = 0
        for b, n in enumerate(news):
            if n < 0:
                history[b] = [np.zeros((0, n_kv, D), np.float16)] * 2
                continue
            new_rows = rows[at:at + n]
            history[b] = [np.concatenate([h, new_rows[:, n_q + i * n_kv:n_q + (i + 1) * n_kv]]) for i, h in enumerate(history[b])]
            at += n
        assert cached.tolist() == [len(h[0]) for h in history]
        own, tab, at = np.zeros((B * width, 1, n_kv, page), np.uint8), np.arange(B * width).reshape(B, width), 0
        for b in range(B):
            n = len(history[b][0])
            kv = [np.zeros((width * BS, n_kv, D), np.float16) for _ in range(2)]
            for x, h in zip(kv, history[b]):
                x[:n] = h
            own[tab[b], 0] = q4.fill_pages(*(x.reshape(width, BS, n_kv, D).transpose(0, 2, 1, 3) for x in kv), group)
        want, tol = q4.attention(last.cpu().numpy(), own, tab, cached.tolist(), 0, sm, group)
        got = out.cpu().numpy().astype(np.float64)
        assert (np.abs(got - want).max(-1) <= np.maximum(tol, 2.0**-24)).all()
        wy, mag = q4.linear(codes, scale, g, xq.cpu().numpy(), xs.cpu().numpy())
        assert (np.abs(y.cpu().numpy() - wy) <= (K // g + 20) * 2.0**-24 * mag + 2.0**-11 * (np.abs(wy) + 1e-3) + 2.0**-24).all()


# ---- calls that meet -----------------------------------------------------------------------------------------------


def test_two_contexts_on_two_streams(pkg):
    """A context of its own per stream: a run of calls on either, both on their way at once, gives what it gives alone."""
    rng = np.random.default_rng(30)
    n_q, n_kv, group, g = 8, 2, 32, 64
    contexts, streams = [pkg.Context(0, 0) for _ in range(2)], [torch.cuda.Stream() for _ in range(2)]
    jobs = []
    for lens in ([9000, 1, 700], [300] * 40):
        q, pages, table, n = attention_case(rng, lens, n_q, n_kv, group, 1, max(lens) // 16 + 1)
        B, K, N = len(lens), n_q * D, 320
        codes, scale, _, _ = linear_case(rng, 1, N, K, g)
        jobs.append(dict(q=dev(q), pages=dev(pages), blocks=len(pages), table=dev(table), lens=dev(n), B=B, K=K, N=N, W=dev(q4.pack_codes(codes)),
                         ws=dev(scale), xq=torch.empty((B, K), dtype=torch.int8, device="cuda"), xs=torch.empty((B, K // g), device="cuda"),
                         y=torch.empty((B, N), dtype=torch.float16, device="cuda"), zero=i32(B, fill=0), slots=torch.empty(9000, dtype=torch.int64, device="cuda"),
                         positions=i32(9000), plan_lens=i32(B), first=i32(B + 1), info=i32(4), count=i32(1, fill=0), free=i32(1)))

    def run(ctx, j, stream):
        ctx.kv4_attention_decode(j["q"], j["pages"], j["blocks"], j["table"], j["lens"], None, j["B"], n_q, D, j["table"].shape[1], 0.1, 0, 1, n_kv, group,
                                 quant_group_size=g, Xq=j["xq"], Xs=j["xs"], stream=stream)
        ctx.linear4_q(j["W"], j["ws"], g, j["xq"], j["xs"], j["y"], j["B"], j["N"], j["K"], stream=stream)
        ctx.plan_blocks(j["lens"], j["zero"], j["B"], j["table"], j["table"].shape[1], j["free"], 1, j["count"], j["slots"], j["positions"], j["plan_lens"],
                        j["first"], 9000, j["info"], stream=stream)

    alone = []
    for ctx, j in zip(contexts, jobs):
        run(ctx, j, None)
        torch.cuda.synchronize()
        alone.append(j["y"].clone())
        j["y"].fill_(7)
    torch.cuda.synchronize()
    for _ in range(20):
        for ctx, j, s in zip(contexts, jobs, streams):
            run(ctx, j, s.cuda_stream)
    torch.cuda.synchronize()
    for ctx, j, want in zip(contexts, jobs, alone):
        ctx.check_device_status()
        assert torch.equal(j["y"], want) and torch.equal(j["plan_lens"], j["lens"]) and j["info"].tolist() == [0, 0, 0, 0]
        ctx.close()


@pytest.mark.parametrize("lens", [[1], [17, 1, 33], [1000] * 8, [16, 48, 32, 0], [9000, 5]])
def test_kv4_attention_ahead_of_the_write(ctx, lens):
    """Layer after layer, the newest row written and attended over with nothing in between: the call that starts early gives what the
    other gives, also where the new row opens a block, and where a sequence has none."""
    rng = np.random.default_rng(len(lens) + lens[0])
    n_q, n_kv, group, layers, B = 8, 2, 32, 6, len(lens)
    width = max(lens) // 16 + 1
    q, pages, table, n = attention_case(rng, lens, n_q, n_kv, group, layers, width)
    slots = dev(np.array([table[b, (m - 1) // 16] * 16 + (m - 1) % 16 if m else -1 for b, m in enumerate(lens)], np.int64))
    qkv = [dev(rng.standard_normal((B, n_q + 2 * n_kv, D)).astype(np.float16)) for _ in range(layers)]
    dtable, dlens, blocks, side = dev(table), dev(n), len(pages), torch.cuda.Stream()

    def run(cache, rows, out, ahead):
        for l in range(layers):
            ctx.kv4_write(qkv[l], slots, cache, blocks, l, layers, B, n_q, n_kv, D, group, q_out=rows)
            ctx.kv4_attention_decode(rows, cache, blocks, dtable, dlens, out[l], B, n_q, D, width, 0.1, l, layers, n_kv, group, ahead=ahead)

    results = []
    for ahead in (False, True):
        for captured in (False, True):
            cache, rows, out = dev(pages), torch.zeros((B, n_q, D), dtype=torch.float16, device="cuda"), torch.zeros((layers, B, n_q, D), dtype=torch.float16, device="cuda")
            with torch.cuda.stream(side):
                side.wait_stream(torch.cuda.default_stream())
                if captured:
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph, stream=side):
                        run(cache, rows, out, ahead)
                    for _ in range(3):
                        graph.replay()
                else:
                    run(cache, rows, out, ahead)
            torch.cuda.synchronize()
            results.append((out, cache))
    ctx.check_device_status()
    for out, cache in results[1:]:
        assert torch.equal(out, results[0][0]) and torch.equal(cache, results[0][1])


def test_replays_and_eager_calls_in_turn(ctx):
    """Two graphs and eager calls of other sizes take turns on one stream: they share the context's scratch and tickets."""
    rng = np.random.default_rng(31)
    cases = [attention_case(rng, lens, 8, 2, 64, 1, max(lens) // 16 + 1) for lens in ([20000], [3000, 5, 8000], [40] * 30)]
    side, calls = torch.cuda.Stream(), []
    for q, pages, table, lens in cases:
        d = [dev(x) for x in (q, pages, table, lens)] + [torch.empty(q.shape, dtype=torch.float16, device="cuda")]

        def call(d=d, stream=None):
            ctx.kv4_attention_decode(d[0], d[1], d[1].shape[0], d[2], d[3], d[4], d[0].shape[0], 8, D, d[2].shape[1], 0.1, 0, 1, 2, 64, stream=stream)

        calls.append((call, d[4]))
    want = []
    with torch.cuda.stream(side):
        for call, out in calls:
            call()
            want.append(out.clone())
        side.synchronize()
        graphs = []
        for call, _ in calls[:2]:
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=side):
                call()
        for _ in range(5):
            for which in (0, 2, 1, 0, 1):
                calls[which][1].fill_(7)
                graphs[which].replay() if which < 2 else calls[2][0]()
            for (_, out), w in zip(calls, want):
                assert torch.equal(out, w)
    ctx.check_device_status()


def test_kv4_write_of_a_long_prompt_is_that_of_its_parts(ctx):
    """However many pairs of heads a warp takes: 20000 rows at once and in calls of 7 and up give the same cache and the same q."""
    rng = np.random.default_rng(32)
    T, n_q, n_kv, group = 20000, 5, 3, 64
    blocks = (T + 15) // 16
    qkv = torch.from_numpy(rng.standard_normal((T, n_q + 2 * n_kv, D)).astype(np.float16)).cuda()
    w = [dev(rng.uniform(0.5, 1.5, D).astype(np.float16)) for _ in range(2)]
    freqs = dev((10000.0 ** (-np.arange(64) / 64)).astype(np.float32))
    positions, slots = torch.arange(T, dtype=torch.int32, device="cuda"), torch.from_numpy(rng.permutation(blocks * 16)[:T]).cuda()
    got = []
    for cuts in ([0, T], [0, 7, 20, 1000, 1001, 9000, T]):
        cache = torch.zeros(blocks * n_kv * q4.page_bytes(group), dtype=torch.uint8, device="cuda")
        q = torch.zeros((T, n_q, D), dtype=torch.float16, device="cuda")
        for a, b in zip(cuts, cuts[1:]):
            ctx.kv4_write(qkv[a:b], slots[a:b], cache, blocks, 0, 1, b - a, n_q, n_kv, D, group, q_norm_w=w[0], k_norm_w=w[1], eps=1e-6, freqs=freqs,
                          positions=positions[a:b], q_out=q[a:b])
        torch.cuda.synchronize()
        got.append((cache, q))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


def test_plan_blocks_long_prompts(ctx):
    """More tokens than one CTA writes, into requests that take blocks which others give back in the same call."""
    cached, new = [160, 0, 48000, 7], [-1, 70001, -3, 9990]
    blocks = (70001 + 15) // 16 + 1
    table = np.full((4, blocks), -1, np.int64)
    perm = np.random.default_rng(33).permutation(6000)
    table[0, :10], table[2, :3000], table[3, 0] = perm[:10], perm[10:3010], perm[3010]
    free = np.concatenate([perm[3011:6000], np.full(3011, -5)])
    case = (cached, new, table.tolist(), free.tolist(), 2989)
    want = q4.plan(*case, max_tokens=80000, capacity=6000)
    assert want["info"][0] == 0
    for in_place in (False, True):
        assert run_plan(ctx, *case, 80000, in_place=in_place) == want


def test_linear4_many_rows_add_to_their_own_output(ctx):
    """More rows than a launch takes, the residual being the output itself; weight scales off the boundary that the wide reads want."""
    rng = np.random.default_rng(34)
    for M, N, K, g in ((70, 48, 512, 32), (45, 33, 1024, 64), (5, 64, 1024, 64)):
        codes, scale, Xq, Xs = linear_case(rng, M, N, K, g)
        y, mag = q4.linear(codes, scale, g, Xq, Xs)
        room = torch.empty(scale.size + 1, dtype=torch.float16, device="cuda")
        room[1:].copy_(dev(scale).flatten())
        start = rng.standard_normal((M, N)).astype(np.float16)
        out = dev(start)
        ctx.linear4_q(dev(q4.pack_codes(codes)), room[1:], g, dev(Xq), dev(Xs), out, M, N, K, epilogue=1, residual=out)
        torch.cuda.synchronize()
        err = (K // g + 19) * 2.0**-24 * mag  # as in check_linear
        tol = err + 2.0**-11 * (np.abs(y) + err)
        want = y + start
        tol = tol + 2.0**-11 * (np.abs(want) + tol)
        assert (np.abs(out.cpu().numpy() - want) <= tol + 2.0**-24).all()
