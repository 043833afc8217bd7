// Single-query attention over the paged cache in 4 bits (w8a8_q4.cuh), GQA, ragged lengths.
//
//   out[b, h] = sum_t p_t v_t / sum_t p_t,  p_t = exp(q_h . k_t sm_scale - max),  t < seq_lens[b];  zeros where seq_lens[b] is 0
//   k_t, v_t = code * scale of the row's group; one pass with the running maximum and sum of the softmax, both fp32
//
// Bound: HBM. A token costs 128 + 8 G bytes per kv head (K and V; G = 128 / group) instead of the fp16 cache's 512, so the unpacking
// comes close behind: per 16 tokens of a kv head a warp executes some 300 instructions for 2304 bytes at groups of 32, where
// an SM is fed a page every ~100 clocks.
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
// Arithmetic. Codes become fp16 numbers by placing the four bits in the significand of 1024 (or, four bits further up, of 1024 in
// sixteenths) and taking that off: two values per instruction, exact. Scores: q (fp16) times codes, fp32 sums per group, times the
// group's scale in fp32. P V: p is rounded to fp16 (2^-11 relative; the denominator sums the rounded values), code * scale is rounded
// to fp16 (2^-11 relative, the values that w8a8_kv4_read returns), products are summed in fp32.
#include "sm100_ptx.cuh"
#include "w8a8_internal.h"
#include "w8a8_q4.cuh"

namespace w8a8 {
namespace {

using q4::kDim;
using q4::kTokens;

constexpr int kMaxBatch = 4096;
constexpr float kNoScore = -1e30f;

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
    float scale_log2;  // sm_scale * log2(e)
    int min_units;     // pages a warp takes at least
    float* scratch;    // [CTAs][2] pieces
    int* tickets;      // [CTAs], zero between launches
    int* status;
};

// ---- helpers -------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t lop_and_or(uint32_t a, uint32_t mask, uint32_t bits) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(mask), "r"(bits));  // (a & mask) | bits
    return r;
}
__device__ __forceinline__ uint32_t as_u32(__half2 v) { return *reinterpret_cast<uint32_t*>(&v); }
__device__ __forceinline__ __half2 as_half2(uint32_t v) { return *reinterpret_cast<__half2*>(&v); }

// The eight biased codes of a word as four fp16 pairs: nibbles (0, 4), (1, 5), (2, 6), (3, 7).
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

// Merges the pieces first, first + 1, ... of which at(i) is the address; lane l holds channels 4 l .. of every head.
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
    template <bool GLOBAL>
    __device__ __forceinline__ void add_piece(const float* piece, int lane) {
#pragma unroll
        for (int h = 0; h < R; ++h) {
            const float4* a = reinterpret_cast<const float4*>(piece + h * kDim) + lane;
            if constexpr (GLOBAL)
                add(h, __ldcg(a), __ldcg(piece + R * kDim + h), __ldcg(piece + R * kDim + R + h));
            else
                add(h, *a, piece[R * kDim + h], piece[R * kDim + R + h]);
        }
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
__device__ __noinline__ void finish(const Kv4Params& p, const Merged<R>& s, int b, int kvh, int heads, int lane) {
    const int K = p.n_q * kDim;
    const size_t row = static_cast<size_t>(b) * K + static_cast<size_t>(kvh) * heads * kDim;
    float2 v[R][2];
#pragma unroll
    for (int h = 0; h < R; ++h) {
        if (h >= heads) break;
        const float inv = s.l[h] != 0.0f ? 1.0f / s.l[h] : 0.0f;
        const __half2 a = __floats2half2_rn(s.acc[h].x * inv, s.acc[h].y * inv), c = __floats2half2_rn(s.acc[h].z * inv, s.acc[h].w * inv);
        if (p.out) *reinterpret_cast<uint2*>(p.out + row + h * kDim + 4 * lane) = {as_u32(a), as_u32(c)};
        v[h][0] = __half22float2(a);
        v[h][1] = __half22float2(c);
    }
    if (!p.Xq) return;
    float amax[R];
#pragma unroll
    for (int h = 0; h < R; ++h) {
        if (h >= heads) break;
        amax[h] = fmaxf(fmaxf(fabsf(v[h][0].x), fabsf(v[h][0].y)), fmaxf(fabsf(v[h][1].x), fabsf(v[h][1].y)));
        for (int d = 1; d < 32 && 4 * d < p.g; d <<= 1) amax[h] = fmaxf(amax[h], __shfl_xor_sync(0xffffffffu, amax[h], d));
    }
#pragma unroll
    for (int d = 1; d < R; d <<= 1)  // groups of several heads
        if (d * kDim < p.g) {
#pragma unroll
            for (int h = 0; h < R; ++h)
                if (!(h & d) && (h | d) < heads) amax[h] = amax[h | d] = fmaxf(amax[h], amax[h | d]);
        }
#pragma unroll
    for (int h = 0; h < R; ++h) {
        if (h >= heads) break;
        float scale = amax[h] / 127.0f;
        if (scale < 1e-8f) scale = 1e-8f;
        const float inv = 1.0f / scale;
        const float x[4] = {v[h][0].x, v[h][0].y, v[h][1].x, v[h][1].y};
        uint32_t packed = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) packed |= static_cast<uint32_t>(max(-127, min(127, __float2int_rn(x[e] * inv))) & 255) << (8 * e);
        const size_t ch = row + h * kDim + 4 * lane;
        *reinterpret_cast<uint32_t*>(p.Xq + ch) = packed;
        if (ch % p.g == 0) p.Xs[ch / p.g] = scale;
    }
}

// ---- the kernel ----------------------------------------------------------------------------------------------------
// G groups per head; R the most query heads per kv head (4 or 8); W warps.
template <int R>
struct Shape {
    static constexpr int kWarps = R == 4 ? 8 : 12;
    static constexpr int kStages = 4;
    static constexpr int kCtasPerSm = R == 4 ? 2 : 1;
};
template <int G, int R>
constexpr int kv4_smem(int batch) {
    return Shape<R>::kWarps * (Shape<R>::kStages * q4::page_bytes(G) + 2 * piece_floats(R) * 4) + (batch + 1) * 4;
}

template <int G, int R>
__global__ void __launch_bounds__(Shape<R>::kWarps * 32, Shape<R>::kCtasPerSm) kv4_attention_kernel(const Kv4Params p) {
    constexpr int W = Shape<R>::kWarps, D = Shape<R>::kStages, kPage = q4::page_bytes(G), kPiece = piece_floats(R);
    extern __shared__ __align__(128) unsigned char kv4_smem_raw[];
    unsigned char* const ring_all = kv4_smem_raw;                                          // [W][D][kPage]
    float* const pieces = reinterpret_cast<float*>(kv4_smem_raw + W * D * kPage);          // [W][2][kPiece]
    int* const first_s = reinterpret_cast<int*>(pieces + W * 2 * kPiece);                  // [batch + 1]: table entries in use ahead of a sequence
    __shared__ __align__(8) uint64_t full_bar[W][D];
    __shared__ int scan_s[W + 1];
    __shared__ long long piece_pair[2 * W];  // the pair of a piece, or -1
    __shared__ int last_s;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, j4 = lane & 3;
    const int heads = p.n_q / p.n_kv;
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < D; ++i) ptx::mbar_init(&full_bar[warp][i], 1);
        ptx::fence_barrier_init();
        ptx::fence_proxy_async();
    }
    if (tid < 2 * W) piece_pair[tid] = -1;
    ptx::pdl_wait();
    ptx::pdl_launch_dependents();

    // ---- table entries in use ahead of every sequence; each is n_kv units ----
    const int cap = p.max_blocks * kTokens;
    {
        const int each = (p.batch + W * 32 - 1) / (W * 32), b0 = tid * each, b1 = min(p.batch, b0 + each);
        int sum = 0;
        for (int b = b0; b < b1; ++b) sum += (min(max(p.lens[b], 0), cap) + kTokens - 1) / kTokens;
        int inc = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, inc, d);
            if (lane >= d) inc += o;
        }
        if (lane == 31) scan_s[warp + 1] = inc;
        if (tid == 0) scan_s[0] = 0;
        __syncthreads();
        int at = inc - sum;
        for (int w = 0; w <= warp; ++w) at += scan_s[w];
        for (int b = b0; b < b1; ++b) {
            first_s[b] = at;
            at += (min(max(p.lens[b], 0), cap) + kTokens - 1) / kTokens;
        }
        if (b1 == p.batch && (b0 < b1 || p.batch == 0)) first_s[p.batch] = at;
        __syncthreads();
    }
    const long long units = static_cast<long long>(first_s[p.batch]) * p.n_kv;
    // rows of no tokens: zeros
    for (int b = blockIdx.x; b < p.batch; b += gridDim.x)
        if (first_s[b] == first_s[b + 1])
            for (int h = warp; h < p.n_kv; h += W) {
                Merged<R> none;
                none.clear();
                finish<R>(p, none, b, h, heads, lane);
            }

    // ---- this warp's run ----
    const long long warps = static_cast<long long>(gridDim.x) * W;
    long long per = (units + warps - 1) / warps;
    if (per < p.min_units) per = p.min_units;
    const long long cta_units = per * W, cta_lo = min(units, blockIdx.x * cta_units), cta_hi = min(units, cta_lo + cta_units);
    const long long lo = min(cta_hi, cta_lo + warp * per), hi = min(cta_hi, lo + per);
    const int n_mine = static_cast<int>(hi - lo);

    // the sequence of a unit
    auto sequence_of = [&](long long u) {
        const int entry = static_cast<int>(u / p.n_kv);  // (a sequence's units are those of its entries, whatever their order in it)
        int a = 0, z = p.batch - 1;
        while (a < z) {
            const int mid = (a + z + 1) >> 1;
            if (first_s[mid] <= entry) a = mid; else z = mid - 1;
        }
        return a;  // (the last of those that start at or before u: empty ones in front of it start there too)
    };
    const uint32_t ring = ptx::smem_u32(ring_all) + warp * (D * kPage);
    long long page_of = 0;  // of unit lo + (i & ~31) + lane: its page's number in the cache
    auto look_up = [&](int i0) {
        const int i = i0 + lane;
        if (i < n_mine) {
            const long long u = lo + i;
            const int b = sequence_of(u);
            const int blocks = first_s[b + 1] - first_s[b];
            const int rest = static_cast<int>(u - static_cast<long long>(first_s[b]) * p.n_kv), h = rest / blocks, blk = rest - h * blocks;
            int phys = p.table[static_cast<size_t>(b) * p.max_blocks + blk];
            if (phys < 0 || phys >= p.n_blocks) phys = 0;  // (the caller's mistake; reads stay inside the cache)
            page_of = (static_cast<long long>(phys) * p.n_layers + p.layer) * p.n_kv + h;
        }
    };
    auto issue = [&](int i) {  // the copy of unit i of the run
        const int from = i & 31;
        const long long page = __shfl_sync(0xffffffffu, page_of, from);
        if (lane == 0) {
            uint64_t* bar = &full_bar[warp][i % D];
            ptx::mbar_arrive_expect_tx(bar, kPage);
            bulk_load(ring + (i % D) * kPage, p.cache + page * kPage, kPage, bar);
        }
    };
    int issued = 0;
    if (n_mine > 0) {
        look_up(0);
        for (; issued < min(n_mine, D); ++issued) issue(issued);
    }

    float* const my_head = pieces + (2 * warp) * kPiece;      // the piece of a pair that began in front of this run
    float* const my_tail = pieces + (2 * warp + 1) * kPiece;  // the piece of a pair that begins in it
    bool failed = false;
    int i = 0;
    int b = n_mine > 0 ? sequence_of(lo) : 0;
    while (i < n_mine) {
        // ---- the next pair of the run ----
        const long long u0 = lo + i;
        while (static_cast<long long>(first_s[b + 1]) * p.n_kv <= u0) ++b;
        const int blocks = first_s[b + 1] - first_s[b];
        const int rest = static_cast<int>(u0 - static_cast<long long>(first_s[b]) * p.n_kv), kvh = rest / blocks, blk0 = rest - kvh * blocks;
        const int n_here = min(n_mine - i, blocks - blk0);
        const int len = min(max(p.lens[b], 0), cap);

        // q: of head g8 (rows 8 .. 15 of the tile are zero), the channels in the order of the K words
        uint32_t qa[4][4];  // [run][a0, a2 of the first step; a0, a2 of the second]
#pragma unroll
        for (int run = 0; run < 4; ++run) {
            uint4 w = {0, 0, 0, 0};
            if (g8 < heads) w = ptx::ld_result_v4(p.q + (static_cast<size_t>(b) * p.n_q + kvh * heads + g8) * kDim + 32 * run + 8 * j4);
            qa[run][0] = __byte_perm(w.x, w.z, 0x5410);  // channels 0, 4
            qa[run][1] = __byte_perm(w.x, w.z, 0x7632);  // 1, 5
            qa[run][2] = __byte_perm(w.y, w.w, 0x5410);  // 2, 6
            qa[run][3] = __byte_perm(w.y, w.w, 0x7632);  // 3, 7
        }
        float m_run = kNoScore, l_run = 0.0f;
        float o[8][4];  // channels 16 n + g8 (+ 8) of heads 2 j4, 2 j4 + 1
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;

        for (int k = 0; k < n_here; ++k, ++i) {
            const int st = i % D;
            if (!failed && !__all_sync(0xffffffffu, ptx::mbar_wait_bounded(&full_bar[warp][st], (i / D) & 1))) {
                if (lane == 0) atomicExch(p.status, 900 + st);
                failed = true;  // (the numbers are void from here on; counters and barriers still run their course)
            }
            const uint32_t page = ring + st * kPage;
            const int tokens = min(kTokens, len - (blk0 + k) * kTokens);

            // ---- scores: tokens 2 j4, 2 j4 + 1 (and + 8) of head g8 ----
            float sc[2][2];
            uint32_t ks[2][G];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                uint32_t kw[4];
                lds_words<4>(kw, page + (g8 + 8 * t) * 64 + j4 * 16);
                lds_words<G>(ks[t], page + q4::kScaleOff + (j4 + 4 * t) * 4 * G);
                sc[t][0] = sc[t][1] = 0.0f;
                float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int run = 0; run < 4; ++run) {
                    uint32_t h[4];
                    unpack8(kw[run], h);
                    mma_f16(acc, qa[run][0], 0u, qa[run][1], 0u, h[0], h[1]);
                    mma_f16(acc, qa[run][2], 0u, qa[run][3], 0u, h[2], h[3]);
                    if ((run + 1) % (4 / G) == 0) {
                        const float2 s = __half22float2(as_half2(ks[t][run / (4 / G)]));
                        sc[t][0] = fmaf(acc[0], s.x, sc[t][0]);
                        sc[t][1] = fmaf(acc[1], s.y, sc[t][1]);
                        acc[0] = acc[1] = 0.0f;
                    }
                }
            }
            float mx = kNoScore;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    sc[t][e] = 8 * t + 2 * j4 + e < tokens ? sc[t][e] * p.scale_log2 : kNoScore;
                    mx = fmaxf(mx, sc[t][e]);
                }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            if (__any_sync(0xffffffffu, mx > m_run)) {
                const float top = fmaxf(m_run, mx), corr = exp2_fast(m_run - top);
                m_run = top;
                l_run *= corr;
                const float c0 = __shfl_sync(0xffffffffu, corr, 8 * j4), c1 = __shfl_sync(0xffffffffu, corr, 8 * j4 + 4);
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    o[n][0] *= c0;
                    o[n][1] *= c1;
                    o[n][2] *= c0;
                    o[n][3] *= c1;
                }
            }
            const __half2 p0 = __floats2half2_rn(exp2_fast(sc[0][0] - m_run), exp2_fast(sc[0][1] - m_run));
            const __half2 p1 = __floats2half2_rn(exp2_fast(sc[1][0] - m_run), exp2_fast(sc[1][1] - m_run));
            const float2 f0 = __half22float2(p0), f1 = __half22float2(p1);
            l_run += (f0.x + f0.y) + (f1.x + f1.y);

            // ---- out^T += V^T P^T: rows are channels, columns heads, the contraction runs over tokens ----
            uint32_t vw[2][4], vs[2][G];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                lds_words<4>(vw[t], page + q4::kVOff + (j4 + 4 * t) * 128 + g8 * 16);
                lds_words<G>(vs[t], page + q4::kScaleOff + 2 * kTokens * G + (j4 + 4 * t) * 4 * G);
            }
            if (tokens < kTokens)  // what lies behind the sequence's end may not be a number: its scale becomes zero
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const int left = tokens - (8 * t + 2 * j4);
                    const uint32_t keep = left >= 2 ? 0xffffffffu : left == 1 ? 0x0000ffffu : 0u;
#pragma unroll
                    for (int x = 0; x < G; ++x) vs[t][x] &= keep;
                }
#pragma unroll
            for (int high = 0; high < 2; ++high) {
                uint32_t a0[4], a1[4], a2[4], a3[4];
                unpack8(vw[0][high], a0);
                unpack8(vw[0][2 + high], a1);
                unpack8(vw[1][high], a2);
                unpack8(vw[1][2 + high], a3);
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const int x = (4 * high + n) * G / 8;
                    const __half2 s0 = as_half2(vs[0][x]), s1 = as_half2(vs[1][x]);
                    mma_f16(o[4 * high + n], as_u32(__hmul2(as_half2(a0[n]), s0)), as_u32(__hmul2(as_half2(a1[n]), s0)),
                            as_u32(__hmul2(as_half2(a2[n]), s1)), as_u32(__hmul2(as_half2(a3[n]), s1)), as_u32(p0), as_u32(p1));
                }
            }

            // ---- the stage is free: the copy of the unit kStages ahead ----
            if (issued < n_mine) {
                ptx::fence_proxy_async();
                __syncwarp();
                if ((issued & 31) == 0) look_up(issued);
                if (!failed) issue(issued);
                ++issued;
            }
        }

        // ---- the pair's piece ----
        l_run += __shfl_xor_sync(0xffffffffu, l_run, 1);
        l_run += __shfl_xor_sync(0xffffffffu, l_run, 2);
        float* const piece = blk0 > 0 ? my_head : my_tail;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int h = 2 * j4 + e;
            if (h < R) {
#pragma unroll
                for (int n = 0; n < 8; ++n) {
                    piece[h * kDim + 16 * n + g8] = o[n][e];
                    piece[h * kDim + 16 * n + 8 + g8] = o[n][2 + e];
                }
            }
        }
        if (j4 == 0 && g8 < R) {
            piece[R * kDim + g8] = m_run;
            piece[R * kDim + R + g8] = l_run;
        }
        __syncwarp();
        if (blk0 == 0 && n_here == blocks) {  // all of the pair
            Merged<R> s;
            s.clear();
            s.template add_piece<false>(piece, lane);
            finish<R>(p, s, b, kvh, heads, lane);
            __syncwarp();
        } else if (lane == 0) {
            piece_pair[2 * warp + (blk0 > 0 ? 0 : 1)] = static_cast<long long>(b) * p.n_kv + kvh;
        }
    }
    __syncthreads();

    // ---- pieces that meet in the CTA: chains of neighbours of one pair; a warp a chain ----
    auto pair_units = [&](long long pair, long long& from, long long& to) {
        const int pb = static_cast<int>(pair / p.n_kv), ph = static_cast<int>(pair % p.n_kv);
        const int blocks = first_s[pb + 1] - first_s[pb];
        from = static_cast<long long>(first_s[pb]) * p.n_kv + static_cast<long long>(ph) * blocks;
        to = from + blocks;
    };
    int chain = 0;
    long long open[2] = {-1, -1};  // pairs that go on in other CTAs: one that began ahead of this CTA's run, one that ends behind it
    for (int x = 0; x < 2 * W;) {
        const long long pair = piece_pair[x];
        if (pair < 0) { ++x; continue; }
        int y = x + 1, z = x;  // z: the last piece of the chain
        while (y < 2 * W && (piece_pair[y] < 0 || piece_pair[y] == pair)) {
            if (piece_pair[y] == pair) z = y;
            ++y;
        }
        long long from, to;
        pair_units(pair, from, to);
        const bool whole = from >= cta_lo && to <= cta_hi;
        if (!whole) open[from < cta_lo ? 0 : 1] = pair;
        if (chain % W == warp) {
            Merged<R> s;
            s.clear();
            for (int k = x; k <= z; ++k)
                if (piece_pair[k] == pair) s.template add_piece<false>(pieces + k * kPiece, lane);
            if (whole)
                finish<R>(p, s, static_cast<int>(pair / p.n_kv), static_cast<int>(pair % p.n_kv), heads, lane);
            else {
                s.store(p.scratch + (2ll * blockIdx.x + (from < cta_lo ? 0 : 1)) * kPiece, lane);
                __threadfence();
            }
        }
        ++chain;
        x = y;
    }

    // ---- pairs that lie in several CTAs: the last of them to come here adds their pieces ----
    for (int side = 0; side < 2; ++side) {
        if (open[side] < 0) continue;  // (uniform over the CTA)
        long long from, to;
        pair_units(open[side], from, to);
        const int c0 = static_cast<int>(from / cta_units), c1 = static_cast<int>((to - 1) / cta_units);
        __syncthreads();
        if (tid == 0) {
            __threadfence();
            const int before = atomicAdd(p.tickets + c0, 1);
            last_s = before == c1 - c0;
            if (last_s) p.tickets[c0] = 0;
            __threadfence();
        }
        __syncthreads();
        if (!last_s) continue;
        Merged<R> s;
        s.clear();
        // pieces in the order of the pages: warp w a run of them, the runs then in order
        const int n = c1 - c0 + 1, run = (n + W - 1) / W, a = min(n, warp * run), z = min(n, a + run);
#pragma unroll 2
        for (int k = a; k < z; ++k) s.template add_piece<true>(p.scratch + (2ll * (c0 + k) + (k == 0 ? 1 : 0)) * kPiece, lane);
        s.store(pieces + warp * kPiece, lane);
        __syncthreads();
        if (warp == 0) {
            s.clear();
            for (int w = 0; w < W; ++w) s.template add_piece<false>(pieces + w * kPiece, lane);
            finish<R>(p, s, static_cast<int>(open[side] / p.n_kv), static_cast<int>(open[side] % p.n_kv), heads, lane);
        }
        __syncthreads();
    }
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
    cfg.blockDim = dim3(Shape<R>::kWarps * 32, 1, 1);
    cfg.dynamicSmemBytes = kv4_smem<G, R>(p.batch);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled(kPdlAttn) ? 1 : 0;
    return launch_with_smem(attribute, kv4_smem<G, R>(kMaxBatch), cfg, kv4_attention_kernel<G, R>, p);
}

int kv4_ctas(int heads_per_kv, long long most_units, int sms) {
    const int W = heads_per_kv <= 4 ? Shape<4>::kWarps : Shape<8>::kWarps, per_sm = heads_per_kv <= 4 ? Shape<4>::kCtasPerSm : Shape<8>::kCtasPerSm;
    const long long want = (most_units + W - 1) / W, room = static_cast<long long>(sms) * per_sm;
    return static_cast<int>(want < 1 ? 1 : want < room ? want : room);
}

}  // namespace

int kv4_max_batch() { return kMaxBatch; }

size_t kv4_attention_scratch(int n_q, int n_kv) {
    return static_cast<size_t>(kKv4Tickets) * 2 * piece_floats(n_q / n_kv <= 4 ? 4 : 8) * sizeof(float);
}

int launch_kv4_attention(const __half* q, const void* cache, int n_blocks, const int* table, const int* lens, __half* out, int batch, int n_q,
                         int n_kv, int max_blocks, float sm_scale, int layer, int n_layers, int group, int g, int8_t* Xq, float* Xs,
                         float* scratch, int* tickets, int* status, cudaStream_t stream) {
    if (batch == 0) return W8A8_OK;
    const int ratio = n_q / n_kv;
    Kv4Params p = {q, static_cast<const unsigned char*>(cache), table, lens, out, Xq, Xs, g, batch, n_q, n_kv, max_blocks, n_blocks, layer, n_layers,
                   sm_scale * 1.4426950408889634f, 1, scratch, tickets, status};
    int ctas = kv4_ctas(ratio, static_cast<long long>(batch) * n_kv * max_blocks, device_sms());
    if (ctas > kKv4Tickets) ctas = kKv4Tickets;
    cudaError_t e;
    if (ratio <= 4)
        e = group == 32 ? launch_kv4<4, 4>(p, ctas, stream) : group == 64 ? launch_kv4<2, 4>(p, ctas, stream) : launch_kv4<1, 4>(p, ctas, stream);
    else
        e = group == 32 ? launch_kv4<4, 8>(p, ctas, stream) : group == 64 ? launch_kv4<2, 8>(p, ctas, stream) : launch_kv4<1, 8>(p, ctas, stream);
    if (e != cudaSuccess) return fail(W8A8_ERR_CUDA, "kv4_attention_decode launch: %s", cudaGetErrorString(e));
    return W8A8_OK;
}

}  // namespace w8a8
