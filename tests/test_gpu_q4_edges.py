"""The decode step in 4 bits where a small mistake would be a large one: weights far below the largest, small and large queries, pages that must not be lost, several tiles a CTA, infinite scales, lengths near 2^31."""
import math

import numpy as np
import pytest
import torch

from oracle import q4

pytestmark = pytest.mark.gpu

D, BS = 128, 16


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


# ---- attention -----------------------------------------------------------------------------------------------------


def paged(rng, rows_k, rows_v, group):
    """fp16 rows [tokens, n_kv, 128] of every sequence -> (pages with one layer in a shuffled order, table, lengths)."""
    lens = [len(k) for k in rows_k]
    used = [(n + BS - 1) // BS for n in lens]
    n_kv = rows_k[0].shape[1]
    perm = rng.permutation(sum(used) + 3)
    pages = np.full((len(perm), 1, n_kv, q4.page_bytes(group)), 255, np.uint8)
    table = np.full((len(lens), max(max(used), 1)), -1, np.int32)
    at = 0
    for b, n in enumerate(lens):
        table[b, :used[b]] = perm[at:at + used[b]]
        at += used[b]
        padded = [np.zeros((used[b] * BS, n_kv, D), np.float16) for _ in range(2)]
        for x, rows in zip(padded, (rows_k[b], rows_v[b])):
            x[:n] = rows
        if n:
            pages[table[b, :used[b]], 0] = q4.fill_pages(*(x.reshape(-1, BS, n_kv, D).transpose(0, 2, 1, 3) for x in padded), group)
    return pages, table, np.array(lens, np.int32)


def run_attention(ctx, q, pages, table, lens, group, sm):
    B, n_q, _ = q.shape
    out = torch.full((B, n_q, D), 9.0, dtype=torch.float16, device="cuda")
    ctx.kv4_attention_decode(dev(q), dev(pages), len(pages), dev(table), dev(lens), out, B, n_q, D, table.shape[1], sm, 0, 1, pages.shape[2], group)
    torch.cuda.synchronize()
    ctx.check_device_status()
    return out.cpu().numpy().astype(np.float64)


def check_attention(ctx, q, pages, table, lens, group, sm):
    want, tol = q4.attention_bound(q, pages, table, lens, 0, sm, group)
    got = run_attention(ctx, q, pages, table, lens, group, sm)
    assert np.isfinite(got).all()
    worst = (np.abs(got - want) / (tol + 2.0**-40)).max()
    assert worst <= 1, worst


@pytest.mark.parametrize("below", [20.3, 23.5, 25.2, 27.0, 29.5])
@pytest.mark.parametrize("n,B", [(40000, 1), (3000, 1), (12000, 24)])
def test_kv4_attention_keeps_the_tail_behind_one_dominant_key(ctx, n, B, below):
    """One key takes the weight and has a value of zero; all others weigh 2^-below of it and have values of one: together they are the output.
    The warp that holds that key holds more of the pages the more sequences there are."""
    rng = np.random.default_rng(n)
    group, sm = 32, 1 / math.sqrt(D)
    for at in (0, 17, n - 1):
        K, V = np.zeros((n, 1, D), np.float16), np.ones((n, 1, D), np.float16)
        K[at, 0, 0] = 4.0
        V[at] = 0
        q = np.zeros((B, 4, D), np.float16)
        q[:, :, 0] = below * math.log(2) / (4 * sm)
        q[:, 2, 0] *= 0.75
        pages, table, lens = paged(rng, [K], [V], group)
        check_attention(ctx, q, pages, np.repeat(table, B, 0), np.repeat(lens, B), group, sm)  # (the sequences share their pages)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("size", [2.0**-24, 2.0**-17, 2.0**-13, 2.0**-9, 1.0, 2.0**9, 2.0**12])
def test_kv4_attention_queries_of_any_size(ctx, size, group):
    """The scale of the scores takes out what q is multiplied by, so that they are alike; heads of other sizes beside them."""
    rng = np.random.default_rng(group)
    lens = [900, 33, 1]
    rows = [[rng.standard_normal((n, 2, D)).astype(np.float16) for n in lens] for _ in range(2)]
    q = np.clip(rng.standard_normal((3, 8, D)) * size, -65504, 65504)
    q[:, 1] *= 2.0**-3
    q[:, 6] *= 2.0**2
    check_attention(ctx, np.clip(q, -65504, 65504).astype(np.float16), *paged(rng, *rows, group), group, 0.1 / size)


def pages_in_channels(n, n_kv):
    """Values that show which pages were added up: page i is one in channel 128 i / pages (times a sign per kv head), zero elsewhere."""
    V = np.zeros((n, n_kv, D), np.float16)
    pages = (n + BS - 1) // BS
    V[np.arange(n), :, np.arange(n) // BS * D // pages] = 1 - 2 * (np.arange(n_kv) % 2)
    return V


@pytest.mark.parametrize("n_q,n_kv,lens,group", [(4, 1, [40000], 64), (8, 1, [9000, 20000], 32), (16, 4, [12345, 1, 0, 30000], 128), (4, 4, [17000], 32),
                                                 (32, 8, [1024] * 8, 32), (32, 8, [1500, 40, 700], 64), (64, 8, [1024] * 8, 32)])
def test_kv4_attention_adds_up_every_page(ctx, n_q, n_kv, lens, group):
    rng = np.random.default_rng(n_q + lens[0])
    rows_k = [rng.standard_normal((n, n_kv, D)).astype(np.float16) for n in lens]
    q = rng.standard_normal((len(lens), n_q, D)).astype(np.float16)
    pages, table, n = paged(rng, rows_k, [pages_in_channels(m, n_kv) for m in lens], group)
    for _ in range(2):
        check_attention(ctx, q, pages, table, n, group, 1 / math.sqrt(D))


@pytest.mark.parametrize("n_q,n_kv,lens,group", [(4, 1, [40000], 64), (8, 2, [5, 300, 0, 1000, 16, 31], 32), (16, 4, [12345, 1, 30000], 128), (32, 8, [1024] * 4, 32)])
def test_kv4_attention_within_what_the_weights_allow(ctx, n_q, n_kv, lens, group):
    rng = np.random.default_rng(n_q + lens[0] + 1)
    gain = np.where(rng.random(D) < 0.06, 4.0, 1.0)
    rows_k = [(rng.standard_normal((n, n_kv, D)) * gain).astype(np.float16) for n in lens]
    rows_v = [rng.standard_normal((n, n_kv, D)).astype(np.float16) for n in lens]
    q = rng.standard_normal((len(lens), n_q, D)).astype(np.float16)
    check_attention(ctx, q, *paged(rng, rows_k, rows_v, group), group, 1 / math.sqrt(D))


# ---- linear --------------------------------------------------------------------------------------------------------


def part_of(g):
    """Channels that are promoted together: 256, 128, 64 or 32, the largest that divides the group's size."""
    return next(p for p in (256, 128, 64, 32) if g % p == 0)


@pytest.mark.parametrize("M", [1, 8, 16, 32])
@pytest.mark.parametrize("N,K,g", [(4752, 512, 64), (4760, 2560, 256), (9736, 2592, 32), (9728, 2560, 128), (9736, 1056, 96), (19456, 2560, 64), (19456, 512, 256),
                                   (40000, 2560, 256), (40000, 544, 544)])
def test_linear4_several_tiles_a_cta(ctx, M, N, K, g):
    """Two and many tiles a CTA, of several boxes each: runs that cross tiles, tiles that several warps share, with each epilogue. Sums of fp32 parts: (parts + 16
    warps + 3) 2^-24 of the magnitudes; every rounding to fp16 2^-11; silu' is at most 1.1."""
    gen = torch.Generator(device="cuda").manual_seed(M + N + K + g)
    G = (K + g - 1) // g
    codes = torch.randint(-8, 8, (N, K), generator=gen, device="cuda", dtype=torch.int8)
    scale = (torch.rand((N, G), generator=gen, device="cuda") * 4e-3 + 1e-3).half()
    x = torch.randint(-127, 128, (M, K), generator=gen, device="cuda", dtype=torch.int8)
    xs = torch.rand((M, G), generator=gen, device="cuda") * 0.045 + 0.005
    W = (codes[:, 0::2] & 15 | codes[:, 1::2] << 4).view(torch.uint8).contiguous()
    y, mag = (torch.zeros((M, N), dtype=torch.float64, device="cuda") for _ in range(2))
    starts = range(0, K, part_of(g))
    for k in starts:
        at, i = slice(k, min(K, k + part_of(g))), k // g
        term = x[:, at].double() @ codes[:, at].double().T * scale[:, i].double() * xs[:, i:i + 1].double()  # (whole numbers below 2^53: exact)
        y, mag = y + term, mag + term.abs()
    err, half = (len(starts) + 19) * 2.0**-24 * mag, 2.0**-11
    residual = torch.randn((M, N), generator=gen, device="cuda").half()
    for epilogue in (0, 1, 2):
        if epilogue == 2 and N % 16:
            continue
        out = torch.full((M + 1, N // 2 if epilogue == 2 else N), 7.0, dtype=torch.float16, device="cuda")
        ctx.linear4_q(W, scale, g, x, xs, out, M, N, K, epilogue=epilogue, residual=residual if epilogue == 1 else None)
        torch.cuda.synchronize()
        assert (out[M] == 7).all()
        if epilogue == 2:
            (gate, up), (eg, eu) = (a.view(M, -1, 2, 8).unbind(2) for a in (y, err))
            s = gate / (1 + torch.exp(-gate))
            ds = 1.1 * (eg + half * gate.abs()) + half * s.abs() + 2.0**-22
            want = s * up
            tol = (s.abs() + ds) * (eu + half * up.abs()) + up.abs() * ds
            want, tol = want.reshape(M, -1), (tol + half * (want.abs() + tol)).reshape(M, -1)
        else:
            want, tol = y, err + half * (y.abs() + err)
            if epilogue == 1:
                want = y + residual.double()
                tol = tol + half * (want.abs() + tol)
        worst = ((out[:M].double() - want).abs() / (tol + 2.0**-24)).max().item()
        assert worst <= 1, (epilogue, worst)


@pytest.mark.parametrize("M", [1, 7, 16, 20])
@pytest.mark.parametrize("N,K,g", [(32, 160, 32), (48, 288, 96), (16, 320, 64), (160, 2592, 32), (40, 66, 22), (32, 384, 128), (16, 544, 544)])
def test_linear4_infinite_scales(ctx, M, N, K, g):
    """Codes and activations of one: every group's sum is positive, so an infinite scale gives infinity in its row or token and nowhere else."""
    G = (K + g - 1) // g
    W = dev(q4.pack_codes(np.ones((N, K), np.int64)))
    x = torch.ones((M, K), dtype=torch.int8, device="cuda")
    for group in {0, G // 2, G - 1}:
        scale, xs = np.full((N, G), 2.0**-7, np.float16), np.full((M, G), 2.0**-3, np.float32)
        scale[3, group], scale[N - 1, group], xs[M // 2, group] = np.inf, -np.inf, np.inf
        want = np.full((M, N), K * 2.0**-10)
        want[M // 2] = np.inf
        want[:, 3], want[:, N - 1] = np.inf, -np.inf
        out = torch.empty((M, N), dtype=torch.float16, device="cuda")
        ctx.linear4_q(W, dev(scale), g, x, dev(xs), out, M, N, K)
        torch.cuda.synchronize()
        got = out.cpu().numpy().astype(np.float64)
        assert np.array_equal(np.isinf(got), np.isinf(want)) and not np.isnan(got).any(), (group, got[:, :8])
        assert np.array_equal(np.sign(got), np.sign(want))
        finite = np.isfinite(want)
        assert (np.abs(got[finite] - want[finite]) <= 2.0**-11 * want[finite]).all()


# ---- the step plan -------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("cached,new,status", [(2**31 - 5, 1, 2), (2**31 - 17, 2, 2), (2**31 - 1, 0, 2), (2**31 - 1, -1, 5), (0, 2**31 - 1, 1), (2**31 - 1, 2**31 - 1, 1),
                                               (2**31 - 17, 1, 0), (2**31 - 16, 0, 0)])
def test_plan_blocks_lengths_near_the_end_of_32_bits(ctx, cached, new, status):
    """A table row as wide as numbers go: tokens beyond 2^31 - 16 are refused like a row that is too short (after what comes ahead of that: blocks given
    back that the stack has no room for, blocks that it does not have)."""
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    width = 2**27
    table = torch.full((width,), 3, dtype=torch.int32, device="cuda")
    free, count, left = i32(8, 9), i32(2), i32(-7)
    slots, positions = torch.full((5,), -7, dtype=torch.int64, device="cuda"), i32(*[-7] * 5)
    lens, first, info = i32(-7), i32(-7, -7), i32(*[-7] * 4)
    ctx.plan_blocks(i32(cached), i32(new), 1, table, width, free, 2, count, slots, positions, lens, first, 5, info, free_count_out=left)
    torch.cuda.synchronize()
    assert (table == 3).all() and free.tolist() == [8, 9] and left.item() == 2
    if status:
        assert info.tolist() == [status, 0, 0, 2] and slots.tolist() == [-1] * 5 and positions.tolist() == [0] * 5 and lens.item() == cached
    else:
        assert info.tolist() == [0, new, 0, 2] and lens.item() == cached + new
        assert positions.tolist() == [cached] * new + [0] * (5 - new)
        assert slots.tolist() == [3 * 16 + cached % 16] * new + [-1] * (5 - new)
