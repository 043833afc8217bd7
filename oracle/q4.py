"""The decode step in 4 bits, restated in numpy from include/w8a8.h: 64-bit arithmetic, plain loops, no code of the library.
TEST INFRASTRUCTURE, NOT PRODUCT."""
from __future__ import annotations

import numpy as np

TOKENS, DIM = 16, 128


def quantize(x, g):
    """fp16 [..., K] in groups of g along the last axis -> (int codes [..., K], fp16 scales [..., ceil(K / g)])."""
    x = np.asarray(x, np.float16).astype(np.float64)
    K = x.shape[-1]
    G = (K + g - 1) // g
    codes, scales = np.zeros(x.shape, np.int64), np.zeros(x.shape[:-1] + (G,), np.float16)
    for i in range(G):
        v = x[..., i * g:(i + 1) * g]
        hi, lo = v.max(-1), v.min(-1)
        with np.errstate(all="ignore"):
            e = np.where(hi >= -lo, hi, lo)
            s = (e / -8).astype(np.float16)
            s = np.where(np.isfinite(v).all(-1), s, np.float16("nan"))
            d = s.astype(np.float64)[..., None]
            q = np.clip(np.rint(v / d), -8, 7)
            q = np.where((d == 0) | np.isnan(d), 0, q)
        codes[..., i * g:(i + 1) * g], scales[..., i] = q.astype(np.int64), s
    return codes, scales


def values(codes, scales, g):
    """fp64 values that codes and scales stand for."""
    return codes * np.repeat(scales.astype(np.float64), g, -1)[..., :codes.shape[-1]]


# ---- the page ----
def page_bytes(g):
    return 2048 + 64 * (DIM // g)


def page_places(g):
    """For (token, channel): the 4-bit place of its K code and of its V code in a page, and the fp16 places of its scales."""
    t, c = np.arange(TOKENS)[:, None], np.arange(DIM)[None]
    k = t * 128 + 8 * (4 * (c % 32 // 8) + c // 32) + c % 8
    v = 2048 + t // 2 * 256 + 8 * (4 * (c % 8) + 2 * (c // 8 % 2) + c // 64) + 4 * (t % 2) + c // 16 % 4
    ks = 1024 + (t // 2 * (DIM // g) + c // g) * 2 + t % 2
    return k, v, ks, ks + TOKENS * (DIM // g)


def open_pages(pages, g):
    """uint8 [..., page bytes] -> (K, V) fp64 [..., 16, 128]."""
    k, v, ks, vs = page_places(g)
    half = np.ascontiguousarray(pages).view(np.float16).astype(np.float64)

    def part(at, scale):
        code = (pages[..., at // 2] >> (at % 2 * 4).astype(np.uint8)) & 15
        with np.errstate(invalid="ignore"):  # (scales behind a sequence's end may be infinite)
            return (code.astype(np.int64) - 8) * half[..., scale]

    return part(k, ks), part(v, vs)


def fill_pages(K, V, g):
    """fp16 [..., 16, 128] twice -> uint8 pages."""
    k, v, ks, vs = page_places(g)
    lead = K.shape[:-2]
    nib = np.zeros(lead + (4096,), np.uint8)
    half = np.zeros(lead + (page_bytes(g) // 2,), np.float16)
    for x, at, scale in ((K, k, ks), (V, v, vs)):
        code, s = quantize(x, g)
        nib[..., at] = (code + 8).astype(np.uint8)
        half[..., scale] = np.repeat(s, g, -1)
    pages = half.view(np.uint8)
    pages[..., :2048] = nib[..., 0::2] | nib[..., 1::2] << 4
    return pages


def attention(q, pages, table, lens, layer, sm_scale, g):
    """q fp16 [B, H, 128], pages [blocks, layers, n_kv, page bytes] -> (fp64 out, a bound on what rounding may move it by).

    The bound, per (sequence, head), with m = max |v|, s the rounding of half a step of fp16 (2^-11): the softmax weights are rounded to
    fp16, relative s each (absolute 2^-25 for the smallest), and numerator and denominator use the same ones: they move the output by at most
    2 m (s + n 2^-25); the values code * scale are rounded: m s; the output is rounded: m s. A score is a sum of 128 products and four
    scaled group sums in fp32, then scaled and put through an exponential of 2^-22: it moves by at most d = 136 2^-24 sum |q k| sm
    + 2^-21 (1 + |score|), and the output by 2 m d. The fp32 sums of n weighted values move it by another n 2^-24 m at most, over
    numerator and denominator twice that."""
    B, H, _ = q.shape
    n_kv = pages.shape[2]
    ratio = H // n_kv
    out, tol = np.zeros(q.shape), np.zeros(q.shape[:2])
    q64 = q.astype(np.float64)
    for b in range(B):
        n = int(lens[b])
        if n <= 0:
            continue
        K, V = open_pages(pages[table[b, :(n + 15) // 16], layer], g)  # [blocks, n_kv, 16, 128]
        K = K.transpose(1, 0, 2, 3).reshape(n_kv, -1, DIM)[:, :n]
        V = V.transpose(1, 0, 2, 3).reshape(n_kv, -1, DIM)[:, :n]
        for h in range(H):
            k, v = K[h // ratio], V[h // ratio]
            s = k @ q64[b, h] * sm_scale
            p = np.exp(s - s.max())
            out[b, h] = p @ v / p.sum()
            m = np.abs(v).max()
            d = (136 * 2.0**-24 * (np.abs(k) @ np.abs(q64[b, h])).max() * abs(sm_scale)) + 2.0**-21 * (1 + np.abs(s).max())
            tol[b, h] = m * (4 * 2.0**-11 + 2 * d + n * (2.0**-24 + 2.0**-23)) + 2.0**-24
    return out, tol


# A weight of the softmax is held as two fp16 numbers relative to a reference that leaves the largest weight of a run of pages at 2^11 or more.
WEIGHTS_AT = 2.0**11


def attention_bound(q, pages, table, lens, layer, sm_scale, g, sms=148):
    """The same output with a bound for every element, from the row's own weights. With w_t = exp(s_t - max), D = sum w_t:

    * a score moves by at most d_t = 136 2^-24 sum |q k| sm + 2^-21 (1 + max |s|) (128 products and four scaled group sums in fp32, the scaling, the
      exponential), and with it its weight in numerator and denominator: sum w_t (e^d_t - 1) (|v_t| + |out|);
    * the denominator adds up the fp32 weights, the numerator takes them as two fp16 numbers: 2^-22 relative, or half a subnormal step where
      the largest weight is 2^11: sum max(2^-22 w_t, 2^-36) |v_t|;
    * code * scale of V is rounded to fp16: sum w_t (2^-11 |v_t| + 2^-25);
    * fp32 sums: two multiplies a page of a warp's run, each off by at most 2^-21 of what it adds up (seventeen terms, cut at the last place of the
      largest), and less than 64 sums where pieces meet, for the numerator; one sum a page and those, 2^-23 each, for the denominator. A run is at most a
      twelfth of a CTA's share of all pages, each pair counting three more, and of a pair of 96 pages kept whole;
    * the quotient and its rounding: (2^-22 + 2^-11) |out| + 2^-25.
    All of it over D but the last, and a hundredth more for products of these."""
    B, H, _ = q.shape
    n_kv = pages.shape[2]
    ratio = H // n_kv
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    q64 = q.astype(np.float64)
    in_use = [(max(int(n), 0) + 15) // 16 for n in lens]
    share = (sum(in_use) + 3 * B) * n_kv / sms
    for b in range(B):
        n = int(lens[b])
        if n <= 0:
            continue
        run = min(in_use[b], (share + 97) / 12 + 2)
        K, V = open_pages(pages[table[b, :in_use[b]], layer], g)  # [blocks, n_kv, 16, 128]
        K = K.transpose(1, 0, 2, 3).reshape(n_kv, -1, DIM)[:, :n]
        V = V.transpose(1, 0, 2, 3).reshape(n_kv, -1, DIM)[:, :n]
        for h in range(H):
            k, v = K[h // ratio], V[h // ratio]
            s = k @ q64[b, h] * sm_scale
            w = np.exp(s - s.max())
            total, size = w.sum(), np.abs(v)
            out[b, h] = w @ v / total
            d = 136 * 2.0**-24 * (np.abs(k) @ np.abs(q64[b, h])) * abs(sm_scale) + 2.0**-21 * (1 + np.abs(s).max())
            moved = w * np.expm1(d)
            weighted = w @ size
            e = moved @ size + moved.sum() * np.abs(out[b, h])
            e += np.maximum(2.0**-22 * w, 2.0**-25 / WEIGHTS_AT) @ size
            e += 2.0**-11 * weighted + 2.0**-25 * total
            e += (2 * run + 64) * 2.0**-21 * weighted + (run + 64) * 2.0**-23 * total * np.abs(out[b, h])
            tol[b, h] = 1.01 * (e / total + (2.0**-22 + 2.0**-11) * (np.abs(out[b, h]) + e / total)) + 2.0**-25
    return out, tol


# ---- the step plan ----
def plan(cached, new, table, free, count, max_tokens, capacity):
    """What w8a8_plan_blocks leaves, from Python lists: a dict of lists."""
    B, width = len(cached), min(len(table[0]) if table else 0, 2**27 - 1)
    table, free = [list(r) for r in table], list(free)
    blocks = lambda n: (n + 15) // 16
    give = sum(blocks(c) for c, n in zip(cached, new) if n < 0 and c >= 0)
    tokens = sum(n for n in new if n > 0)
    take = sum(blocks(max(c, 0) + n) - blocks(max(c, 0)) for c, n in zip(cached, new) if n >= 0)
    status = 0
    for code, bad in ((5, count < 0 or count + give > capacity), (1, take > count + give), (2, any(blocks(max(c, 0) + max(n, 0)) > width for c, n in zip(cached, new))),
                      (3, tokens > max_tokens), (4, any(c < 0 for c in cached))):
        if bad:
            status = code
            break
    if status:
        return dict(table=table, free=free, left=count, slots=[-1] * max_tokens, positions=[0] * max_tokens, seq_lens=[max(0, c) for c in cached],
                    first=[0] * (B + 1), info=[status, 0, 0, count])
    top = count
    for b in range(B):
        if new[b] < 0:
            for j in range(blocks(cached[b])):
                free[top] = table[b][j]
                top += 1
    slots, positions, lens, first = [], [], [], [0]
    for b in range(B):
        if new[b] < 0:
            lens.append(0)
        else:
            for j in range(blocks(cached[b]), blocks(cached[b] + new[b])):
                top -= 1
                table[b][j] = free[top]
            for pos in range(cached[b], cached[b] + new[b]):
                slots.append(table[b][pos // 16] * 16 + pos % 16 if table[b][pos // 16] >= 0 else -1)
                positions.append(pos)
            lens.append(cached[b] + new[b])
        first.append(len(slots))
    pad = max_tokens - len(slots)
    return dict(table=table, free=free, left=top, slots=slots + [-1] * pad, positions=positions + [0] * pad, seq_lens=lens, first=first,
                info=[0, tokens, take, top])


# ---- the linear ----
def pack_codes(codes):
    """int codes [N, K] in [-8, 7] -> uint8 [N, K / 2], the even k in the low four bits."""
    c = (np.asarray(codes, np.int64) & 15).astype(np.uint8)
    return c[:, 0::2] | c[:, 1::2] << 4


def linear(codes, scale, g, Xq, Xs):
    """fp64 [M, N] of 4-bit codes [N, K], fp16 scales [N, G], int8 activations [M, K] and their fp32 scales [M, G]; and the sum of
    the groups' absolute values, which bounds what fp32 sums may lose."""
    y = mag = 0.0
    for i in range(scale.shape[1]):
        P = Xq[:, i * g:(i + 1) * g].astype(np.int64) @ codes[:, i * g:(i + 1) * g].astype(np.int64).T
        term = P * scale[:, i].astype(np.float64)[None] * Xs[:, i].astype(np.float64)[:, None]
        y, mag = y + term, mag + np.abs(term)
    return y, mag


def silu(x):
    return x / (1 + np.exp(-x))
