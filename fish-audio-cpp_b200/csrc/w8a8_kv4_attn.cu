// Single-query attention over the paged cache in 4 bits (w8a8_q4.cuh), GQA, ragged lengths.
//
//   out[b, h] = sum_t p_t v_t / sum_t p_t,  p_t = exp(q_h . k_t sm_scale - max),  t < seq_lens[b];  zeros where seq_lens[b] is 0
//   k_t, v_t = code * scale of the row's group; one pass with the running maximum and sum of the softmax, both fp32
//
// Bound: HBM and the arithmetic, close to one another. A token costs 128 + 4 G bytes per kv head (K and V; G = 128 / group) instead of the fp16
// cache's 512; a warp executes some 325 instructions for the 2304 bytes of 16 tokens at groups of 32. 2 x 131000 tokens: 75 us, 60 % of
// the measured copy rate; the copies alone, without arithmetic, take 54, the arithmetic alone, without copies, 61 (the scores and the
// softmax 42 of them, a chain that three warps a scheduler cannot hide). Two pages at a time, one page's scores beside the sum over the page
// before it, scales folded into p, and 8 or 14 or 16 warps instead of 12 changed nothing or cost time.
//
// Split. The unit is a page: 16 tokens of one (sequence, kv head). All units of the batch, in the order sequence, head, page, are one
// range that is cut evenly over the warps of the grid (a CTA's warps take neighbouring runs), whatever the lengths are: nobody waits
// for the longest sequence. The cut is made on the device, where the lengths are. A warp that holds all pages of a (sequence, head)
// writes its output itself; pieces of a pair that lies in several warps meet in the CTA's shared memory, and where it lies in several
// CTAs in the context's scratch, where the CTA that comes last (a ticket per pair, reset by that CTA) adds them in the order of the pages.
//
// A warp streams its run through a ring of its own: one bulk copy per page, issued by a lane kStages ahead, across the borders of
// pairs; nothing in the steady state synchronises warps.
//
// Arithmetic. Scores: a masked nibble is, as the bits of an fp16 number, the subnormal code * 2^-24 (or, four bits up, code * 2^-20, which
// meets a q of a sixteenth), exact as a matrix operand: one instruction for two codes. Where a head's q stays below 512 the other channels take it sixteen times instead, so
// that nothing of a small q is lost; above, what a sixteenth rounds by is 2^-21 beside a q of 2^9. The 8 that stored codes carry leaves with the
// accumulator's start, -8 * sum of q over the group. Sums are fp32 per group, times the group's scale in fp32. P V: codes as fp16 numbers
// (1024 + code, less 1032), times the scale, rounded to fp16 (2^-11 relative; what w8a8_kv4_read returns); p as two fp16 numbers, the
// rounded one and what that left, which costs nothing here and takes the error from 3.3e-4 of the output to 2.6e-4,
// of which the output's own rounding is 2.1e-4; products are summed in fp32. The reference of the exponentials lies below the row's largest score and moves, and the
// sums with it, when a weight passes 2^kTop: a few times per row only.
#include "sm100_ptx.cuh"
#include "w8a8_internal.h"
#include "w8a8_q4.cuh"

#include <cmath>

namespace w8a8 {
namespace {

using q4::kDim;
using q4::kTokens;

constexpr int kMaxBatch = 4096;
constexpr float kNoScore = -1e30f;
// Pairs of at most kFewPages, and of at most twice a CTA's share (with eight heads, whose pieces are twice as long, four times) up to kWholePages, are not
// cut between CTAs: a join costs what a warp's two or three pages cost. us whole and cut, when the rule was made: 1 x 400 tokens 7.3 and 8.3, 8 x 400 8.0 and 9.5, 16 x 1024 11.5 and 13.1; 8 x 1024 11.3 and 11.0, 8 x 1500 13.8 and
// 12.0 (more than twice a share), with eight heads 8 x 1024 11.7 and 13.1; 64 x 4000 79 and 73 (whole up to 256 pages, and up to 96).
constexpr int kFewPages = 32, kWholePages = 96;
// Pages that a pair counts for beyond its own. us with 0, 2, 4 and 8, when it was chosen: 48 ragged sequences up to 8000 tokens 34, 23.5, 23.2, 23.4; 200 up to 2000
// tokens 50, 31.7, 32.1, 35.1; 64 x 512 20.5, 21.1, 21.3, 22.0.
constexpr int kPairCost = 3;
// The largest weight of a warp's pages so far stands between 2^kAt and 2^kTop, at the upper end of fp16: what a weight as two fp16 numbers loses is 2^-22 of itself
// or 2^-25, so a key that takes nearly all the weight leaves the others what they have down to 2^-36 of it. (With weights of up to one, others below
// 2^-25 were gone, which is all of the output where that key's value is small.) us for 2 x 131000 tokens and 64 heads over 8 x 1024 with kAt = 7, 10, 12, 13:
// 74.1, 74.1, 74.3, 74.5 and 11.3, 11.4, 11.5, 11.6.
constexpr float kTop = 15.0f, kAt = 11.0f;

struct Kv4Params {
    const __half* q;  // [batch, n_q, 128]
    const unsigned char* cache;
    const int* table;  // [batch, max_blocks]
    const int* lens;
    __half* out;  // [batch, n_q, 128] or null
    int8_t* Xq;   // [batch, n_q * 128] or null
    float* Xs;    // [batch, n_q * 128 / g]
    int g;
    int batch, n_q, n_kv, max_blocks, n_blocks, layer, n_layers;
    float scale_log2;  // sm_scale * log2(e) * 2^24: the scores' codes come as 2^-24 of themselves
    float* scratch;    // [CTAs][2] pieces
    int* tickets;      // [CTAs], zero between launches
    int* status;
    float over_grid;  // 1 / CTAs, rounded up
    bool ahead;  // lengths, table and all pages but each sequence's last were complete ahead of the launch ahead
};

// ---- helpers -------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t lop_and_or(uint32_t a, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(mask), "r"(bits));  // (a & mask) | bits
    return r;
}
__device__ __forceinline__ uint32_t as_u32(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }

// The eight stored codes (code + 8) of a word as fp16 pairs, nibbles (0, 4), (1, 5), (2, 6), (3, 7): times 2^-24, 2^-20, 2^-24, 2^-20.
__device__ __forceinline__ void unpack8_tiny(uint32_t w, uint32_t (&h)[4]) {
    const uint32_t up = w >> 8;
    h[0] = w & 0x000f000fu;
    h[1] = w & 0x00f000f0u;
    h[2] = up & 0x000f000fu;
    h[3] = up & 0x00f000f0u;
}
// The eight codes themselves: nibbles set into the mantissa of 1024 (Kim, Henry, Fahim and Awadalla, "Who says elephants can't run", 2022), the upper ones over 16.
__device__ __forceinline__ void unpack8(uint32_t w, uint32_t (&h)[4]) {
    const __half2 off = as_half2(0x64086408u);                                        // 1024 + 8
    const __half2 sixteenth = as_half2(0x2c002c00u), off16 = as_half2(0xd480d480u);  // 1 / 16; -(64 + 8)
    const uint32_t up = w >> 8;
    h[0] = as_u32(__hsub2(as_half2(lop_and_or(w, 0x000f000fu, 0x64006400u)), off));
    h[1] = as_u32(__hfma2(as_half2(lop_and_or(w, 0x00f000f0u, 0x64006400u)), sixteenth, off16));
    h[2] = as_u32(__hsub2(as_half2(lop_and_or(up, 0x000f000fu, 0x64006400u)), off));
    h[3] = as_u32(__hfma2(as_half2(lop_and_or(up, 0x00f000f0u, 0x64006400u)), sixteenth, off16));
}

// D(16x8) += A(16x16) B(16x8), fp16 in, fp32 out.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same into d from c, which stays.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
// Element (row, col) of an 8 x 8 matrix of 16-bit numbers goes to (col, row): lane 4 row + j holds columns 2 j, 2 j + 1.
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"(ptx::smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// x / d and what is left, for quotients below 2^20 (x below 2^31): the product with the reciprocal is off by less than a quarter there, the whole
// number below it by one at most.
struct Quotient {
    int q, rest;
};
__device__ __forceinline__ Quotient quotient(int x, int d) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(static_cast<float>(d)));
    int q = __float2int_rz(static_cast<float>(x) * r), rest = x - q * d;
    if (rest < 0) {
        --q;
        rest += d;
    } else if (rest >= d) {
        ++q;
        rest -= d;
    }
    return {q, rest};
}
template <int N>
__device__ __forceinline__ void lds_words(uint32_t (&w)[N], uint32_t addr) {
    if constexpr (N == 4)
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
    else if constexpr (N == 2)
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
    else
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
}

// A piece: the state of a softmax over part of a pair's pages. Numerators [heads][128], then maxima and denominators.
__host__ __device__ constexpr int piece_floats(int heads) { return heads * kDim + 2 * heads; }

// Adds the pieces base[i], i in `which`, in order; lane l holds channels 4 l .. of every head.
template <int R>
struct Merged {
    float4 acc[R];
    float m[R], l[R];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int h = 0; h < R; ++h) {
            acc[h] = {0.0f, 0.0f, 0.0f, 0.0f};
            m[h] = kNoScore;
            l[h] = 0.0f;
        }
    }
    __device__ __forceinline__ void add(int h, const float4& a, float ma, float la) {
        const float top = fmaxf(m[h], ma), x = exp2_fast(m[h] - top), y = exp2_fast(ma - top);
        acc[h].x = acc[h].x * x + a.x * y;
        acc[h].y = acc[h].y * x + a.y * y;
        acc[h].z = acc[h].z * x + a.z * y;
        acc[h].w = acc[h].w * x + a.w * y;
        l[h] = l[h] * x + la * y;
        m[h] = top;
    }
    __device__ __forceinline__ void store(float* piece, int lane) const {
#pragma unroll
        for (int h = 0; h < R; ++h) {
            reinterpret_cast<float4*>(piece + h * kDim)[lane] = acc[h];
            if (lane == 0) {
                piece[R * kDim + h] = m[h];
                piece[R * kDim + R + h] = l[h];
            }
        }
    }
};

// The pair's rows of the output, and their int8 codes (int8_gemm.cu:147-211) where asked for. heads <= R are real.
template <int R>
__device__ __forceinline__ void finish(const Kv4Params& p, const Merged<R>& s, int b, int kvh, int heads, int lane) {
    const int K = p.n_q * kDim;
    const size_t row = static_cast<size_t>(b) * K + static_cast<size_t>(kvh) * heads * kDim;
    float2 v[R][2];
#pragma unroll
    for (int h = 0; h < R; ++h) {
        const float inv = s.l[h] != 0.0f ? 1.0f / s.l[h] : 0.0f;
        const __half2 a = __floats2half2_rn(s.acc[h].x * inv, s.acc[h].y * inv), c = __floats2half2_rn(s.acc[h].z * inv, s.acc[h].w * inv);
        if (p.out && h < heads) *reinterpret_cast<uint2*>(p.out + row + h * kDim + 4 * lane) = {as_u32(a), as_u32(c)};
        v[h][0] = __half22float2(a);
        v[h][1] = __half22float2(c);
    }
    if (!p.Xq) return;
    float amax[R];
#pragma unroll
    for (int h = 0; h < R; ++h) {
        amax[h] = fmaxf(fmaxf(fabsf(v[h][0].x), fabsf(v[h][0].y)), fmaxf(fabsf(v[h][1].x), fabsf(v[h][1].y)));
#pragma unroll 1
        for (int d = 1; d < 32 && 4 * d < p.g; d <<= 1) amax[h] = fmaxf(amax[h], __shfl_xor_sync(0xffffffffu, amax[h], d));
    }
#pragma unroll
    for (int d = 1; d < R; d <<= 1)  // groups of several heads
        if (d * kDim < p.g) {
#pragma unroll
            for (int h = 0; h < R; ++h)
                if (!(h & d)) amax[h] = amax[h | d] = fmaxf(amax[h], amax[h | d]);
        }
#pragma unroll
    for (int h = 0; h < R; ++h) {
        float scale = amax[h] / 127.0f;
        if (scale < 1e-8f) scale = 1e-8f;
        const float inv = 1.0f / scale;
        const float x[4] = {v[h][0].x, v[h][0].y, v[h][1].x, v[h][1].y};
        uint32_t packed = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) packed |= static_cast<uint32_t>(max(-127, min(127, __float2int_rn(x[e] * inv))) & 255) << (8 * e);
        const size_t ch = row + h * kDim + 4 * lane;
        if (h < heads) {
            *reinterpret_cast<uint32_t*>(p.Xq + ch) = packed;
            if (ch % p.g == 0) p.Xs[ch / p.g] = scale;
        }
    }
}

// A pair that is one piece, or none (no tokens). One copy of this code: it runs cold.
template <int R>
__device__ __noinline__ void finish_whole(const Kv4Params& p, const float* piece, int b, int kvh) {
    const int lane = threadIdx.x & 31;
    Merged<R> s;
    s.clear();
    if (piece) {
#pragma unroll
        for (int h = 0; h < R; ++h) {
            s.acc[h] = reinterpret_cast<const float4*>(piece + h * kDim)[lane];
            s.l[h] = piece[R * kDim + R + h];
        }
    }
    finish<R>(p, s, b, kvh, p.n_q / p.n_kv, lane);
}

// Heads h0 .. h0 + E - 1 of pieces base[i], i in `which`, added and finished, or to the piece `to`. E is one, or the heads of a group of codes. Lane i
// sees to piece i's weights, so that the loop over the pieces has no chain but its sums. (Four heads by a warp each take half a microsecond less over
// 8 x 1024 tokens than all by one warp, piece by piece.)
template <int R, int E>
__device__ __noinline__ void merge_share(const Kv4Params& p, const float* base, uint32_t which, float* to, int b, int kvh, int h0) {
    constexpr int kPiece = piece_floats(R);
    const int lane = threadIdx.x & 31;
    const bool there = which >> lane & 1;
    const float* const mine = base + (there ? lane : __ffs(which) - 1) * kPiece + R * kDim + h0;
    Merged<E> s;
    s.clear();
    float w[E];
#pragma unroll
    for (int h = 0; h < E; ++h) {
        const float top_mine = there ? mine[h] : kNoScore, sum = there ? mine[R + h] : 0.0f;
        float top = top_mine;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        w[h] = exp2_fast(top_mine - top);
        float part = there ? sum * w[h] : 0.0f;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) part += __shfl_xor_sync(0xffffffffu, part, d);
        s.l[h] = part;
        s.m[h] = top;
    }
#pragma unroll 4
    for (; which; which &= which - 1) {
        const int i = __ffs(which) - 1;
        const float* const from = base + i * kPiece + h0 * kDim + 4 * lane;
#pragma unroll
        for (int h = 0; h < E; ++h) {
            const float4 a = *reinterpret_cast<const float4*>(from + h * kDim);
            const float x = __shfl_sync(0xffffffffu, w[h], i);
            s.acc[h] = {fmaf(a.x, x, s.acc[h].x), fmaf(a.y, x, s.acc[h].y), fmaf(a.z, x, s.acc[h].z), fmaf(a.w, x, s.acc[h].w)};
        }
    }
    const int heads = p.n_q / p.n_kv;
    if (!to) return finish<E>(p, s, b, (kvh * heads + h0) / E, E, lane);
#pragma unroll
    for (int h = 0; h < E; ++h) {
        reinterpret_cast<float4*>(to + (h0 + h) * kDim)[lane] = s.acc[h];
        if (lane == 0) {
            to[R * kDim + h0 + h] = s.m[h];
            to[R * kDim + R + h0 + h] = s.l[h];
        }
    }
}
template <int R>
__device__ __forceinline__ void merge_share(const Kv4Params& p, int each, const float* base, uint32_t which, float* to, int b, int kvh, int share) {
    if (each == 1) return merge_share<R, 1>(p, base, which, to, b, kvh, share);
    if (each == 2) return merge_share<R, 2>(p, base, which, to, b, kvh, 2 * share);
    if (each == 4) return merge_share<R, 4>(p, base, which, to, b, kvh, 4 * share);
    if constexpr (R == 8) merge_share<R, 8>(p, base, which, to, b, kvh, 8 * share);
}

// ---- the kernel ----------------------------------------------------------------------------------------------------
// G groups per head; R the most query heads per kv head (4 or 8); W warps.
// Twelve warps of 168 registers: with sixteen of 128 the long cases take the same (64 x 4000 tokens) and the short ones more (8 x 1024 tokens
// 0.5 us, 1 x 8192 0.8); with eight the long ones a fifth more. Four stages are 9 KB a warp on their way.
constexpr int kWarps = 12, kStages = 4;
template <int G, int R>
constexpr int kv4_smem(int batch) {
    return kWarps * (kStages * q4::page_bytes(G) + 2 * piece_floats(R) * 4) + (batch + 1) * 4;
}

template <int G, int R>
__global__ void __launch_bounds__(kWarps * 32, 1) kv4_attention_kernel(const __grid_constant__ Kv4Params p) {
    constexpr int W = kWarps, D = kStages, kPage = q4::page_bytes(G), kPiece = piece_floats(R);
    static_assert((D & (D - 1)) == 0 && D <= 32, "a stage is the low bits of a unit's number");
    extern __shared__ __align__(128) unsigned char kv4_smem_raw[];
    unsigned char* const ring_all = kv4_smem_raw;                                  // [W][D][kPage]
    float* const pieces = reinterpret_cast<float*>(kv4_smem_raw + W * D * kPage);  // [W][2][kPiece]
    int* const first_s = reinterpret_cast<int*>(pieces + W * 2 * kPiece);          // [batch + 1]: table entries in use ahead of a sequence
    __shared__ __align__(8) uint64_t full_bar[W][D];
    __shared__ int scan_s[W + 1];
    __shared__ int piece_pair[2 * W];  // the pair of a piece, or -1
    __shared__ int last_s[2];

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (lane < D) {
        ptx::mbar_init(&full_bar[warp][lane], 1);
        ptx::fence_barrier_init();
        ptx::fence_proxy_async();
    }
    if (tid < 2 * W) piece_pair[tid] = -1;
    if (!p.ahead) ptx::pdl_wait();

    // ---- table entries in use ahead of every sequence; each is n_kv units ----
    const int cap = p.max_blocks * kTokens;
    auto entries_of = [&](int b) { return (min(max(p.lens[b], 0), cap) + kTokens - 1) / kTokens; };
    if (p.batch <= 32) {
        if (warp == 0) {
            const int n = lane < p.batch ? entries_of(lane) : 0;
            int inc = n;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int o = __shfl_up_sync(0xffffffffu, inc, d);
                if (lane >= d) inc += o;
            }
            if (lane < p.batch) first_s[lane + 1] = inc;
            if (lane == 0) first_s[0] = 0;
        }
    } else {
        const int each = (p.batch + W * 32 - 1) / (W * 32), b0 = tid * each, b1 = min(p.batch, b0 + each);
        int sum = 0;
        for (int b = b0; b < b1; ++b) sum += entries_of(b);
        int inc = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, inc, d);
            if (lane >= d) inc += o;
        }
        if (lane == 31) scan_s[warp] = inc;
        __syncthreads();
        int at = inc - sum;
        for (int w = 0; w < warp; ++w) at += scan_s[w];
        if (tid == 0) first_s[0] = 0;
        for (int b = b0; b < b1; ++b) first_s[b + 1] = at += entries_of(b);
    }
    __syncthreads();
    const int units = first_s[p.batch] * p.n_kv;

    // ---- this warp's run (all numbers below 2^31: the host sees to it) ----
    // The range is cut by cost: a pair counts kPairCost pages more than it has (its q, its piece, its output; a run of many short pairs would
    // else last longest). Cost v of the range is cost v - of pairs ahead - kPairCost pages into its pair, none where that is negative.
    const int costs = units + kPairCost * p.batch * p.n_kv;
    const int grid = gridDim.x;
    int cta_cost = __float2int_ru(__fmul_ru(__int2float_ru(costs), p.over_grid));  // costs / grid or, of many, a few more
    if (static_cast<long long>(cta_cost - 1) * grid >= costs) --cta_cost;
    cta_cost = max(cta_cost, 1);
    auto cost_ahead = [&](int b) { return (first_s[b] + kPairCost * b) * p.n_kv; };
    auto last_at = [&](auto ahead, int v, int a) {  // the last sequence b >= a with ahead(b) <= v, where a is one: most often a
        int z = p.batch - 1;
        if (a >= z || ahead(a + 1) > v) return a;
#pragma unroll 1
        for (++a; a < z;) {
            const int mid = (a + z + 1) >> 1;
            if (ahead(mid) <= v) a = mid; else z = mid - 1;
        }
        return a;
    };
    struct Place {
        int b, h, in, of;  // cost `in` of `of` of the pair (b, h)
    };
    auto place_of = [&](int v, int a) {
        const int b = last_at(cost_ahead, v, a), of = first_s[b + 1] - first_s[b] + kPairCost, rest = v - cost_ahead(b);
        const Quotient x = quotient(rest, of);
        return Place{b, x.q, x.rest, of};
    };
    // Lanes 0, 1: where the CTA's run begins and ends; lanes 2, 3: the warp's. A CTA's borders are at multiples of cta_cost, but not inside a
    // pair of few pages, which goes to one side or the other as a whole.
    int at_border, b_border;  // in pages; the sequence (or one of no pages in front of it)
    {
        const int whole_pages = min(kWholePages, max(R / 2 * cta_cost, kFewPages));
        const long long nominal = static_cast<long long>(blockIdx.x + (lane & 1)) * cta_cost;
        int v = static_cast<int>(min(nominal, static_cast<long long>(costs))), a = 0;
#pragma unroll 1
        for (int step = 0; step < 2; ++step) {  // (two rounds through one copy of the code: the CTA's borders, then all four in pages)
            Place x = {0, 0, 0, kPairCost};
            if (v < costs) x = place_of(v, a);
            if (step == 0) {
                if (v < costs && x.of - kPairCost <= whole_pages) v += 2 * x.in < x.of ? -x.in : x.of - x.in;
                const int from = __shfl_sync(0xffffffffu, v, 0), to = __shfl_sync(0xffffffffu, v, 1);
                a = __shfl_sync(0xffffffffu, x.b, 0);  // (no border of the CTA's lies in front of its first one's sequence)
                if (lane & 2) v = min(to, from + (warp + (lane & 1)) * ((to - from + W - 1) / W));
            } else {
                b_border = x.b;
                v = v < costs ? first_s[x.b] * p.n_kv + x.h * (x.of - kPairCost) + max(0, x.in - kPairCost) : units;
            }
        }
        at_border = v;
    }
    const int cta_lo = __shfl_sync(0xffffffffu, at_border, 0), cta_hi = __shfl_sync(0xffffffffu, at_border, 1);
    const int lo = __shfl_sync(0xffffffffu, at_border, 2), n_mine = __shfl_sync(0xffffffffu, at_border, 3) - lo;
    auto units_ahead = [&](int b) { return first_s[b] * p.n_kv; };

    const uint32_t ring = ptx::smem_u32(ring_all) + warp * (D * kPage);
    const int first_b = __shfl_sync(0xffffffffu, b_border, 2);  // at or in front of the run's first sequence
    int page_of = 0;     // the page's number in the cache of unit (i & ~31) + lane of the run
    bool newest = false;  // it is its sequence's last
    auto look_up = [&](int i0) {
        const int i = i0 + lane;
        if (i < n_mine) {
            const int u = lo + i, b = last_at(units_ahead, u, first_b);  // (the last of those that start at or before u: empty ones in front of it start there too)
            const int blocks = first_s[b + 1] - first_s[b], rest = u - units_ahead(b);
            const Quotient x = quotient(rest, blocks);
            const int h = x.q, blk = x.rest;
            int phys = p.table[static_cast<size_t>(b) * p.max_blocks + blk];
            if (phys < 0 || phys >= p.n_blocks) phys = 0;  // (the caller's mistake; reads stay inside the cache)
            page_of = (phys * p.n_layers + p.layer) * p.n_kv + h;
            newest = blk == blocks - 1;
        }
    };
    auto issue = [&](int i) {  // the copy of unit i of the run, by the lane that knows where it is
        if (lane == (i & 31)) {
            uint64_t* bar = &full_bar[warp][i & (D - 1)];
            ptx::mbar_arrive_expect_tx(bar, kPage);
            bulk_load(ring + (i & (D - 1)) * kPage, p.cache + static_cast<size_t>(static_cast<uint32_t>(page_of)) * kPage, kPage, bar);
        }
    };
    // the pair at hand, and its q: asked for ahead of the pages, of a later pair ahead of the piece of the one before it
    const int g8 = lane >> 2, j4 = lane & 3, heads = p.n_q / p.n_kv;
    int b = first_b, blocks = 1, kvh = 0, blk0 = 0;
    uint4 q_raw[4];
    auto ask_q = [&](int u) {
        while (units_ahead(b + 1) <= u) ++b;
        blocks = first_s[b + 1] - first_s[b];
        const Quotient x = quotient(u - units_ahead(b), blocks);
        kvh = x.q;
        blk0 = x.rest;
#pragma unroll
        for (int run = 0; run < 4; ++run) {
            q_raw[run] = {0, 0, 0, 0};
            if (g8 < heads) q_raw[run] = ptx::ld_result_v4(p.q + (static_cast<size_t>(b) * p.n_q + kvh * heads + g8) * kDim + 32 * run + 8 * j4);
        }
    };
    if (n_mine > 0) {
        if (!p.ahead) ask_q(lo);
        look_up(0);
        if (p.ahead) {  // a sequence's last page may still be in the making
            const uint32_t later = __ballot_sync(0xffffffffu, newest && lane < min(n_mine, D));
#pragma unroll 1
            for (int i = 0; i < min(n_mine, D); ++i)
                if (!(later >> i & 1)) issue(i);
            ptx::pdl_wait();
#pragma unroll 1
            for (uint32_t rest = later; rest; rest &= rest - 1) issue(__ffs(rest) - 1);
            ask_q(lo);
        } else {
#pragma unroll 1  // (code size: it runs cold)
            for (int i = 0; i < min(n_mine, D); ++i) issue(i);
        }
    } else if (p.ahead) {
        ptx::pdl_wait();
    }
    ptx::pdl_launch_dependents();

    // rows of no tokens: zeros
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x)
        if (first_s[b] == first_s[b + 1])
            for (int h = warp; h < p.n_kv; h += W) finish_whole<R>(p, nullptr, b, h);

    bool failed = false;
    for (int i = 0; i < n_mine;) {
        // ---- the next pair of the run ----
        const int u0 = lo + i;
        const int i_end = min(n_mine, i + blocks - blk0);
        int tokens = min(max(p.lens[b], 0), cap) - blk0 * kTokens;  // from the page's first on

        // q of head g8 (nothing in columns without a head), the channels in the order of the K words; the start of the sums
        uint32_t qb[4][4];  // [run][channels 0, 4; 1, 5; 2, 6; 3, 7 of the lane's eight]; the odd ones a sixteenth of the even ones
        float start[G][4];  // of heads 2 j4, 2 j4 + 1, for the tokens of either half
        float to_log2[2];   // of these heads: what takes their raw scores to powers of two
        {
            uint32_t both = 0;  // bits 14 and 30: the two highest bits of a channel's exponent are set, it is 512 or more (or no number)
#pragma unroll
            for (int run = 0; run < 4; ++run)
                both |= (q_raw[run].x & q_raw[run].x << 1) | (q_raw[run].y & q_raw[run].y << 1) | (q_raw[run].z & q_raw[run].z << 1) | (q_raw[run].w & q_raw[run].w << 1);
            const uint32_t large = __ballot_sync(0xffffffffu, (both & 0x40004000u) != 0);
            const bool mine = (large >> (lane & 28) & 15) != 0;
            const __half2 even_by = as_half2(mine ? 0x3c003c00u : 0x4c004c00u), odd_by = as_half2(mine ? 0x2c002c00u : 0x3c003c00u);  // 1 or 16; 1 / 16 or 1
#pragma unroll
            for (int e = 0; e < 2; ++e) to_log2[e] = p.scale_log2 * ((large >> (8 * j4 + 4 * e) & 15) != 0 ? 1.0f : 0.0625f);
            float sum[G];
#pragma unroll
            for (int x = 0; x < G; ++x) sum[x] = 0.0f;
#pragma unroll
            for (int run = 0; run < 4; ++run) {
                const uint4 w = q_raw[run];
                qb[run][0] = as_u32(__hmul2(as_half2(__byte_perm(w.x, w.z, 0x5410)), even_by));
                qb[run][1] = as_u32(__hmul2(as_half2(__byte_perm(w.x, w.z, 0x7632)), odd_by));
                qb[run][2] = as_u32(__hmul2(as_half2(__byte_perm(w.y, w.w, 0x5410)), even_by));
                qb[run][3] = as_u32(__hmul2(as_half2(__byte_perm(w.y, w.w, 0x7632)), odd_by));
                float even = 0.0f, odd = 0.0f;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const float2 f = __half22float2(as_half2(qb[run][x]));
                    (x & 1 ? odd : even) += f.x + f.y;
                }
                sum[run * G / 4] += fmaf(16.0f, odd, even) * -0x1p-21f;  // -8 2^-24
            }
#pragma unroll
            for (int x = 0; x < G; ++x) {
                sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], 1);
                sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], 2);
                const float s0 = __shfl_sync(0xffffffffu, sum[x], 8 * j4), s1 = __shfl_sync(0xffffffffu, sum[x], 8 * j4 + 4);
                // (registers of their own, next to one another, as the multiply wants them: no copies per page)
                asm volatile("mov.b32 %0, %4;\n mov.b32 %1, %5;\n mov.b32 %2, %4;\n mov.b32 %3, %5;"
                             : "=f"(start[x][0]), "=f"(start[x][1]), "=f"(start[x][2]), "=f"(start[x][3]) : "f"(s0), "f"(s1));
            }
        }
        float m_run[2] = {kNoScore, kNoScore}, l_run[2] = {0.0f, 0.0f};  // of heads 2 j4, 2 j4 + 1
        float o[8][4];  // channels 16 n + g8 (+ 8) of heads 2 j4, 2 j4 + 1
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;

#pragma unroll 1
        for (; i < i_end; ++i, tokens -= kTokens) {
            if (!__all_sync(0xffffffffu, ptx::mbar_try_wait(&full_bar[warp][i & (D - 1)], (i / D) & 1)) && !failed &&
                !__all_sync(0xffffffffu, ptx::mbar_wait_bounded(&full_bar[warp][i & (D - 1)], (i / D) & 1))) {
                atomicExch(p.status, 900);
                failed = true;  // (the numbers are void from here on; counters and barriers still run their course)
            }
            const uint32_t page = ring + (i & (D - 1)) * kPage;

            // ---- scores: tokens g8, g8 + 8 of heads 2 j4, 2 j4 + 1 ----
            float sc[4];  // raw: times to_log2 they are in powers of two
            {
                uint32_t k0[4], k1[4], s0[G], s1[G];
                lds_words<4>(k0, page + g8 * 64 + j4 * 16);
                lds_words<4>(k1, page + (g8 + 8) * 64 + j4 * 16);
                lds_words<G>(s0, page + q4::kScaleOff + (g8 >> 1) * 4 * G);
                lds_words<G>(s1, page + q4::kScaleOff + (4 + (g8 >> 1)) * 4 * G);
                const uint32_t pick = g8 & 1 ? 0x7632 : 0x5410;  // the token's half of two groups' words
#pragma unroll
                for (int x = 0; x < G; ++x) {
                    float d[4];
#pragma unroll
                    for (int run = x * 4 / G; run < (x + 1) * 4 / G; ++run) {
                        uint32_t h0[4], h1[4];
                        unpack8_tiny(k0[run], h0);
                        unpack8_tiny(k1[run], h1);
                        if (run == x * 4 / G)
                            mma_f16(d, h0[0], h1[0], h0[1], h1[1], qb[run][0], qb[run][1], start[x]);
                        else
                            mma_f16(d, h0[0], h1[0], h0[1], h1[1], qb[run][0], qb[run][1]);
                        mma_f16(d, h0[2], h1[2], h0[3], h1[3], qb[run][2], qb[run][3]);
                    }
                    const int other = G > 1 ? x ^ 1 : x;
                    const float2 t0 = __half22float2(as_half2(__byte_perm(s0[x & ~1], s0[other | x], pick)));
                    const float2 t1 = __half22float2(as_half2(__byte_perm(s1[x & ~1], s1[other | x], pick)));
                    const float f0 = x & 1 ? t0.y : t0.x, f1 = x & 1 ? t1.y : t1.x;
                    sc[0] = x ? fmaf(d[0], f0, sc[0]) : d[0] * f0;
                    sc[1] = x ? fmaf(d[1], f0, sc[1]) : d[1] * f0;
                    sc[2] = x ? fmaf(d[2], f1, sc[2]) : d[2] * f1;
                    sc[3] = x ? fmaf(d[3], f1, sc[3]) : d[3] * f1;
                }
            }
            uint32_t v0[4], v1[4], vs0[G], vs1[G];  // V of token pairs j4 and 4 + j4
            lds_words<4>(v0, page + q4::kVOff + j4 * 128 + g8 * 16);
            lds_words<4>(v1, page + q4::kVOff + (4 + j4) * 128 + g8 * 16);
            lds_words<G>(vs0, page + q4::kScaleOff + 2 * kTokens * G + j4 * 4 * G);
            lds_words<G>(vs1, page + q4::kScaleOff + 2 * kTokens * G + (4 + j4) * 4 * G);
            if (tokens < kTokens) {  // what lies behind the sequence's end may not be a number: its scale becomes zero
                auto keep = [&](int left) { return left >= 2 ? 0xffffffffu : left == 1 ? 0x0000ffffu : 0u; };
                const uint32_t keep0 = keep(tokens - 2 * j4), keep1 = keep(tokens - 8 - 2 * j4);
#pragma unroll
                for (int x = 0; x < G; ++x) {
                    vs0[x] &= keep0;
                    vs1[x] &= keep1;
                }
            }
            // relative to the reference; what lies behind the sequence's end weighs nothing
            float y[4];
            auto relative = [&] {
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = g8 + 4 * (e & 2) < tokens ? fmaf(sc[e], to_log2[e & 1], -m_run[e & 1]) : -INFINITY;
            };
            relative();
            if (__any_sync(0xffffffffu, fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])) > kTop)) {
                const float before[2] = {m_run[0], m_run[1]};
                m_run[0] = m_run[1] = 0.0f;
                relative();
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float mx = fmaxf(y[e], y[2 + e]);
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
                    m_run[e] = fmaxf(before[e], mx - kAt);
                    const float corr = exp2_fast(before[e] - m_run[e]);
                    l_run[e] *= corr;
#pragma unroll
                    for (int n = 0; n < 8; ++n) {
                        o[n][e] *= corr;
                        o[n][2 + e] *= corr;
                    }
                }
                relative();
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = exp2_fast(y[e]);
            l_run[0] += y[0] + y[2];
            l_run[1] += y[1] + y[3];
            // as two fp16 numbers each: rounded, and what that left
            const __half2 p0 = __floats2half2_rn(y[0], y[1]), p1 = __floats2half2_rn(y[2], y[3]);
            const float2 f0 = __half22float2(p0), f1 = __half22float2(p1);
            const __half2 r0 = __floats2half2_rn(y[0] - f0.x, y[1] - f0.y), r1 = __floats2half2_rn(y[2] - f1.x, y[3] - f1.y);

            // ---- out^T += V^T P^T: rows are channels, columns heads, the contraction runs over tokens ----
            const uint32_t pb0 = transposed(as_u32(p0)), pb1 = transposed(as_u32(p1)), rb0 = transposed(as_u32(r0)), rb1 = transposed(as_u32(r1));
#pragma unroll
            for (int high = 0; high < 2; ++high) {
                uint32_t a0[4], a1[4], a2[4], a3[4];
                unpack8(v0[high], a0);
                unpack8(v0[2 + high], a1);
                unpack8(v1[high], a2);
                unpack8(v1[2 + high], a3);
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const __half2 s0 = as_half2(vs0[(4 * high + n) * G / 8]), s1 = as_half2(vs1[(4 * high + n) * G / 8]);
                    const uint32_t v[4] = {as_u32(__hmul2(as_half2(a0[n]), s0)), as_u32(__hmul2(as_half2(a1[n]), s0)), as_u32(__hmul2(as_half2(a2[n]), s1)),
                                           as_u32(__hmul2(as_half2(a3[n]), s1))};
                    mma_f16(o[4 * high + n], v[0], v[1], v[2], v[3], pb0, pb1);
                    mma_f16(o[4 * high + n], v[0], v[1], v[2], v[3], rb0, rb1);
                }
            }

            // ---- the stage is free: the copy of the unit kStages ahead ----
            const int next = i + D;
            if (next < n_mine) {
                ptx::fence_proxy_async();
                __syncwarp();
                if ((next & 31) == 0) look_up(next);
                if (!failed) issue(next);
            }
        }

        // ---- the pair's piece: of a pair that began in front of this run, or that begins in it ----
        const bool head = blk0 > 0, whole = !head && lo + i - u0 == blocks;
        const int this_b = b, this_kvh = kvh;
        if (i < n_mine) ask_q(lo + i);
        float* const piece = pieces + (2 * warp + (head ? 0 : 1)) * kPiece;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], d);
            const int h = 2 * j4 + e;
            if (h < R) {
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    piece[h * kDim + 16 * n + g8] = o[n][e];
                    piece[h * kDim + 16 * n + 8 + g8] = o[n][2 + e];
                }
                if (g8 == 0) {
                    piece[R * kDim + h] = m_run[e];
                    piece[R * kDim + R + h] = l_run[e];
                }
            }
        }
        __syncwarp();
        if (whole) {
            finish_whole<R>(p, piece, this_b, this_kvh);
            __syncwarp();
        } else if (lane == 0) {
            piece_pair[2 * warp + (head ? 0 : 1)] = this_b * p.n_kv + this_kvh;
        }
    }
    __syncthreads();

    // ---- pieces that meet in the CTA: chains of neighbours of one pair; a warp takes a head of a chain, or the heads of a group of codes ----
    const int each = p.Xq && p.g > kDim ? p.g / kDim : 1, shares = heads / each;
    auto pair_units = [&](int pair, int& from, int& to) {
        const Quotient x = quotient(pair, p.n_kv);
        const int pages = first_s[x.q + 1] - first_s[x.q];
        from = units_ahead(x.q) + x.rest * pages;
        to = from + pages;
        return x;
    };
    // (lane x of every warp looks at piece x; a chain starts where the piece in front of it is another pair's)
    const int pair_x = lane < 2 * W ? piece_pair[lane] : -1;
    const uint32_t there = __ballot_sync(0xffffffffu, pair_x >= 0);
    const uint32_t in_front = there & ((1u << lane) - 1);
    const int pair_before = __shfl_sync(0xffffffffu, pair_x, in_front ? 31 - __clz(in_front) : 0);
    const uint32_t starts = __ballot_sync(0xffffffffu, pair_x >= 0 && (!in_front || pair_before != pair_x));
    int open[2] = {-1, -1};  // pairs that go on in other CTAs: one that began ahead of this CTA's run, one that ends behind it
    int task = warp;  // of (chain, share), counted from the chain at hand: this warp's next
#pragma unroll 1
    for (uint32_t todo = starts; todo; todo &= todo - 1, task -= shares) {
        const int x = __ffs(todo) - 1;
        const uint32_t later = todo & (todo - 1);
        const uint32_t mine = there & (0xffffffffu << x) & (later ? (1u << (__ffs(later) - 1)) - 1 : 0xffffffffu);
        const int pair = __shfl_sync(0xffffffffu, pair_x, x);
        int from, to;
        const Quotient x_pair = pair_units(pair, from, to);
        const bool whole = from >= cta_lo && to <= cta_hi, before = from < cta_lo;
        if (!whole) open[before ? 0 : 1] = pair;
        for (; task < shares; task += W)
            merge_share<R>(p, each, pieces, mine, whole ? nullptr : p.scratch + (2ll * blockIdx.x + (before ? 0 : 1)) * kPiece, x_pair.q, x_pair.rest,
                                  task);
    }

    // ---- pairs that lie in several CTAs: the last of them to come here adds their pieces; half of the warps see to either open pair ----
    if (open[0] < 0 && open[1] < 0) goto done;  // (uniform over the CTA)
    __syncthreads();
    {
        constexpr int kHalf = W / 2;
        const int side = warp >= kHalf, w = warp - side * kHalf;
        const int pair = open[side];
        if (pair >= 0) {
            int from, to;
            const Quotient x_pair = pair_units(pair, from, to);
            const int first_cost = from + kPairCost * (pair + 1);  // of the pair's first page
            const int c0 = quotient(first_cost, cta_cost).q, c1 = quotient(first_cost + (to - from) - 1, cta_cost).q, n = c1 - c0 + 1;
            auto half_barrier = [&] { asm volatile("bar.sync %0, %1;" ::"r"(1 + side), "n"(kHalf * 32) : "memory"); };
            if (w == 0 && lane == 0) {  // (releases what the CTA's warps stored ahead of the barrier, acquires what the others' released)
                int before;
                asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(p.tickets + c0) : "memory");
                last_s[side] = before == n - 1;
                if (before == n - 1) p.tickets[c0] = 0;
            }
            half_barrier();
            if (last_s[side]) {
                // pieces in the order of the pages: warp w a run of them, the runs then in order
                const int run = (n + kHalf - 1) / kHalf, x0 = min(n, w * run), x1 = min(n, x0 + run);
                float* const sums = pieces + side * kHalf * kPiece;
                Merged<R> s;
                s.clear();
                for (int k = x0; k < x1; ++k) {
                    const float* piece = p.scratch + (2ll * (c0 + k) + (k == 0 ? 1 : 0)) * kPiece;
#pragma unroll
                    for (int h = 0; h < R; ++h)
                        s.add(h, __ldcg(reinterpret_cast<const float4*>(piece + h * kDim) + lane), __ldcg(piece + R * kDim + h), __ldcg(piece + R * kDim + R + h));
                }
                if (x0 < x1) s.store(sums + w * kPiece, lane);
                half_barrier();
                for (int x = w; x < shares; x += kHalf)
                    merge_share<R>(p, each, sums, (1u << ((n + run - 1) / run)) - 1, nullptr, x_pair.q, x_pair.rest, x);
            }
        }
    }
done:
    if (failed) {  // copies that may still be on their way land before the CTA goes
#pragma unroll 1
        for (int w = 0; w < 1000; ++w) __nanosleep(1000);
    }
}

template <int G, int R>
cudaError_t launch_kv4(const Kv4Params& p, int ctas, cudaStream_t stream) {
    static SmemAttribute attribute;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, 1, 1);
    cfg.blockDim = dim3(kWarps * 32, 1, 1);
    cfg.dynamicSmemBytes = kv4_smem<G, R>(p.batch);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled(kPdlAttn) ? 1 : 0;
    return launch_with_smem(attribute, kv4_smem<G, R>(kMaxBatch), cfg, kv4_attention_kernel<G, R>, p);
}

}  // namespace

int kv4_max_batch() { return kMaxBatch; }

size_t kv4_attention_scratch(int n_q, int n_kv) {
    return static_cast<size_t>(kKv4Tickets) * 2 * piece_floats(n_q / n_kv <= 4 ? 4 : 8) * sizeof(float);
}

int launch_kv4_attention(const __half* q, const void* cache, int n_blocks, const int* table, const int* lens, __half* out, int batch, int n_q,
                         int n_kv, int max_blocks, float sm_scale, int layer, int n_layers, int group, int g, int8_t* Xq, float* Xs,
                         float* scratch, int* tickets, int* status, bool ahead, cudaStream_t stream) {
    if (batch == 0) return W8A8_OK;
    const int ratio = n_q / n_kv;
    Kv4Params p = {q, static_cast<const unsigned char*>(cache), table, lens, out, Xq, Xs, g, batch, n_q, n_kv, max_blocks, n_blocks, layer, n_layers,
                   sm_scale * 1.4426950408889634f * 0x1p24f, scratch, tickets, status, 0.0f, ahead};
    const long long most = static_cast<long long>(batch) * n_kv * max_blocks;  // units, were all sequences as long as their rows
    const int sms = device_sms() < kKv4Tickets ? device_sms() : kKv4Tickets, ctas = most < sms ? static_cast<int>(most) : sms;
    p.over_grid = std::nextafter(1.0f / static_cast<float>(ctas > 0 ? ctas : 1), 1.0f);
    cudaError_t e;
    if (ratio <= 4)
        e = group == 32 ? launch_kv4<4, 4>(p, ctas, stream) : group == 64 ? launch_kv4<2, 4>(p, ctas, stream) : launch_kv4<1, 4>(p, ctas, stream);
    else
        e = group == 32 ? launch_kv4<4, 8>(p, ctas, stream) : group == 64 ? launch_kv4<2, 8>(p, ctas, stream) : launch_kv4<1, 8>(p, ctas, stream);
    if (e != cudaSuccess) return fail(W8A8_ERR_CUDA, "kv4_attention_decode launch: %s", cudaGetErrorString(e));
    return W8A8_OK;
}

}  // namespace w8a8
