// Rows of the qkv projection into the 4-bit paged cache (qk-norm, rotation, quantiser, write through a slot map), and back.
//
// Takes the place of the same reference code as qknorm_rope_kvwrite_kernel (src/engine/dual_ar_engine.cc:585-628; rope.cu:9-65;
// rms_norm.cu:10-58), with its rounding points and its summation order: q and k are the same fp16 numbers, and the cache holds what
// the fp16 cache would hold, in groups of 4 bits (w8a8_q4.cuh). Tokens are named by slots, so that a prompt's rows and a
// decode step's go the same way, and rows with a negative slot (a captured step's empty rows) are left alone, their q too.
//
// Bound: for prompts instructions and bytes alike (2 (n_q + 2 n_kv) 128 read and 2 n_q 128 written per token), latency for a decode step.
// 8192 tokens of 32 + 16 heads 43 us to write (27 for the bytes; 35 without the norm) and 10.9 to read back, a decode step's 8 tokens 3.6 for both.
// Half a warp holds a head, eight neighbouring channels a lane: 16-byte reads and writes, a K word a lane, and of the norm's tree three levels
// in the lane. A warp takes one token and one pair of heads after another, so that the angles are made once.
#include "sm100_ptx.cuh"
#include "w8a8_internal.h"
#include "w8a8_q4.cuh"

namespace w8a8 {
namespace {

constexpr int kStoreWarps = 4, kPairsAhead = 4;

struct StoreParams {
    const __half* qkv;       // [tokens, (n_q + 2 n_kv) * 128]
    const __half* q_norm_w;  // [128] or null
    const __half* k_norm_w;
    float eps;
    const float* freqs;      // [64] or null: no rotation
    const int* positions;    // [tokens], with freqs
    const long long* slots;  // [tokens]
    long long n_slots;
    unsigned char* cache;
    int tokens, n_q, n_kv, layer, n_layers;
    __half* q_out;           // [tokens, n_q, 128] or null
    int pairs_per_warp;
};

// Lane l of a half holds channels 8 l .. 8 l + 7 of a head, as four fp16 pairs.
struct Row {
    __half2 h[4];
};
__device__ __forceinline__ Row load_row(const __half* src, int l) {
    const uint4 v = ptx::ld_result_v4(src + 8 * l);
    Row r;
    r.h[0] = *reinterpret_cast<const __half2*>(&v.x);
    r.h[1] = *reinterpret_cast<const __half2*>(&v.y);
    r.h[2] = *reinterpret_cast<const __half2*>(&v.z);
    r.h[3] = *reinterpret_cast<const __half2*>(&v.w);
    return r;
}
__device__ __forceinline__ Row lds_row(uint32_t addr) {
    Row r;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(*reinterpret_cast<uint32_t*>(&r.h[0])), "=r"(*reinterpret_cast<uint32_t*>(&r.h[1])), "=r"(*reinterpret_cast<uint32_t*>(&r.h[2])),
                   "=r"(*reinterpret_cast<uint32_t*>(&r.h[3]))
                 : "r"(addr) : "memory");
    return r;
}
__device__ __forceinline__ void store_row(__half* dst, int l, const Row& r) {
    uint4 v;
    v.x = *reinterpret_cast<const uint32_t*>(&r.h[0]);
    v.y = *reinterpret_cast<const uint32_t*>(&r.h[1]);
    v.z = *reinterpret_cast<const uint32_t*>(&r.h[2]);
    v.w = *reinterpret_cast<const uint32_t*>(&r.h[3]);
    *reinterpret_cast<uint4*>(dst + 8 * l) = v;
}

using q4::F2;
using q4::f2;
// The lane's channels as x (even) and y (odd) of the rotation's pairs 0, 1 and 2, 3.
struct Wide {
    F2 x[2], y[2];
    Wide() = default;
    __device__ __forceinline__ explicit Wide(const Row& r) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float2 a = __half22float2(r.h[2 * i]), b = __half22float2(r.h[2 * i + 1]);
            x[i] = f2(a.x, b.x);
            y[i] = f2(a.y, b.y);
        }
    }
    __device__ __forceinline__ Row halves() const {
        Row r;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float2 a = parts(x[i]), b = parts(y[i]);
            r.h[2 * i] = __floats2half2_rn(a.x, b.x);
            r.h[2 * i + 1] = __floats2half2_rn(a.y, b.y);
        }
        return r;
    }
};

// Per-head RMSNorm, the sum of squares in the order of the reference's tree (rms_norm.cu:23-49 with 128 threads): over the five bits of
// an element's place in its run of 32, the highest first, then over the runs as (0 + 2) + (1 + 3). Place 8 (l & 3) + e of run
// l >> 2 is lane l's element e, so the first two levels are lanes, three are the lane's own, and the runs are lanes again.
__device__ __forceinline__ Row normed_row(const Row& r, const Wide& w, float eps) {
    const Wide v(r);
    F2 s[4] = {v.x[0] * v.x[0], v.x[1] * v.x[1], v.y[0] * v.y[0], v.y[1] * v.y[1]};
#pragma unroll
    for (int d = 2; d > 0; d >>= 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 a = parts(s[e]);
            s[e] = s[e] + f2(__shfl_xor_sync(0xffffffffu, a.x, d), __shfl_xor_sync(0xffffffffu, a.y, d));
        }
    const float2 even = parts(s[0] + s[1]), odd = parts(s[2] + s[3]);  // places e and e + 4
    float t = (even.x + even.y) + (odd.x + odd.y);
    t += __shfl_xor_sync(0xffffffffu, t, 8);
    t += __shfl_xor_sync(0xffffffffu, t, 4);
    const float rms = rsqrtf(t / q4::kDim + eps);
    const F2 rr = f2(rms, rms);
    Wide o;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        o.x[i] = v.x[i] * rr * w.x[i];
        o.y[i] = v.y[i] * rr * w.y[i];
    }
    return o.halves();
}

// Cosine and sine of one angle. (One copy of the code: it runs cold, and once per token.)
__device__ __noinline__ float2 cos_sin(float angle) { return make_float2(cosf(angle), sinf(angle)); }

// V's word of a lane holds eight r of one n; a 16-bit piece of the page holds the four n of one r. The four lanes that differ in n alone
// exchange their words (lanes are bits 1 and 2 of l): with `to_pieces` lane n gets the bytes of r = 2 n, 2 n + 1 (byte n' : n'), and back.
__device__ __forceinline__ uint32_t exchange_bytes(uint32_t w, int n) {
    const uint32_t x1 = __shfl_xor_sync(0xffffffffu, w, 2), x2 = __shfl_xor_sync(0xffffffffu, w, 4), x3 = __shfl_xor_sync(0xffffffffu, w, 6);
    const uint32_t pick = n | (n + 4) << 4;  // byte n of either
    const uint32_t own = __byte_perm(__byte_perm(w, x1, pick), __byte_perm(x2, x3, pick), 0x5410);  // of lanes n, n ^ 1, n ^ 2, n ^ 3
    return __byte_perm(own, 0, n | (n ^ 1) << 4 | (n ^ 2) << 8 | (n ^ 3) << 12);
}

// Pairs of heads of one kind: the query heads two by two, then k's, then v's (of an odd count the last pair's second half has nothing to do).
__host__ __device__ inline int store_pairs(int n_q, int n_kv) { return (n_q + 1) / 2 + 2 * ((n_kv + 1) / 2); }

template <int GROUPS>
__global__ void __launch_bounds__(kStoreWarps * 32, 10) kv4_write_kernel(const __grid_constant__ StoreParams p) {
    constexpr int kSpan = 16 / GROUPS;  // lanes of a group
    const int lane = threadIdx.x & 31, l = lane & 15, side = lane >> 4;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
    const int q_pairs = (p.n_q + 1) / 2, kv_pairs = (p.n_kv + 1) / 2, pairs = q_pairs + 2 * kv_pairs;
    const int per_token = (pairs + p.pairs_per_warp - 1) / p.pairs_per_warp;
    const long long item = static_cast<long long>(blockIdx.x) * kStoreWarps + warp;
    const int token = static_cast<int>(item / per_token), first = static_cast<int>(item % per_token) * p.pairs_per_warp;
    const int last = min(pairs, first + p.pairs_per_warp);
    const bool normed = p.q_norm_w != nullptr, turned = p.freqs != nullptr;
    Wide w;
    if (normed && first < q_pairs + kv_pairs) w = Wide(load_row(first < q_pairs ? p.q_norm_w : p.k_norm_w, l));  // parameters: asked for before the wait
    float f[2] = {0.0f, 0.0f};
    if (turned) { f[0] = p.freqs[4 * l + 2 * side]; f[1] = p.freqs[4 * l + 2 * side + 1]; }
    ptx::pdl_wait();
    ptx::pdl_launch_dependents();
    if (token >= p.tokens) return;
    const long long slot = p.slots[token];
    if (slot < 0 || slot >= p.n_slots) return;
    const __half* const row = p.qkv + static_cast<size_t>(token) * (p.n_q + 2 * p.n_kv) * q4::kDim;
    // Heads lie one behind the other, q, k, v; a pair's are two neighbours, but for the last of an odd kind, whose second half reads the next kind's
    // first (at the row's end its neighbour's) for nothing.
    const int heads = p.n_q + 2 * p.n_kv;
    int ahead = 2 * first - (first >= q_pairs ? p.n_q & 1 : 0) - (first >= q_pairs + kv_pairs ? p.n_kv & 1 : 0);  // the first head of the next pair to fetch
    // Through shared memory, kPairsAhead ahead; a lane copies what it reads itself, so that it waits for nobody else. (8192 tokens, one pair ahead in
    // registers 48 us, with the norm and without; ahead by 2, 3, 4, 8 42.6, 42.9, 43.0, 43.2 with it and 38.2, 36.1, 35.0, 34.2 without.)
    __shared__ __align__(16) uint4 ring_s[kStoreWarps][kPairsAhead][32];
    const uint32_t ring = ptx::smem_u32(&ring_s[warp][0][lane]);
    int asked = first;
    auto ask = [&] {
        if (asked < last) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ring + (asked - first) % kPairsAhead * 512),
                         "l"(row + min(ahead + side, heads - 1) * q4::kDim + 8 * l)
                         : "memory");
            ++asked;
            ahead += 2 - (asked == q_pairs ? p.n_q & 1 : asked == q_pairs + kv_pairs ? p.n_kv & 1 : 0);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll 1
    for (int i = 0; i < kPairsAhead; ++i) ask();
    auto take = [&](int pair) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kPairsAhead - 1) : "memory");
        const Row r = lds_row(ring + (pair - first) % kPairsAhead * 512);
        ask();
        return r;
    };
    // cosines and sines of the lane's four pairs; either half makes two
    F2 c[2], s[2], minus_s[2];
    if (turned && first < q_pairs + kv_pairs) {
        const float pos = static_cast<float>(p.positions[token]);
        const float2 a = cos_sin(f[0] * pos), b = cos_sin(f[1] * pos);
        const float2 ao = {__shfl_xor_sync(0xffffffffu, a.x, 16), __shfl_xor_sync(0xffffffffu, a.y, 16)};
        const float2 bo = {__shfl_xor_sync(0xffffffffu, b.x, 16), __shfl_xor_sync(0xffffffffu, b.y, 16)};
        const F2 mine_c = f2(a.x, b.x), mine_s = f2(a.y, b.y), other_c = f2(ao.x, bo.x), other_s = f2(ao.y, bo.y);
        c[0] = side ? other_c : mine_c;
        c[1] = side ? mine_c : other_c;
        s[0] = side ? other_s : mine_s;
        s[1] = side ? mine_s : other_s;
        minus_s[0] = -s[0];
        minus_s[1] = -s[1];
    }
    auto turn = [&](const Row& r) {  // norm and rotation of a q or k row
        const Row t = normed ? normed_row(r, w, p.eps) : r;
        if (!turned) return t;
        const Wide v(t);
        Wide o;
#pragma unroll
        for (int i = 0; i < 2; ++i) {  // interleaved pairs (rope.cu:36-45), rounded as qknorm_rope_kvwrite_kernel's are
            o.x[i] = fma2(v.x[i], c[i], v.y[i] * minus_s[i]);
            o.y[i] = fma2(v.y[i], c[i], v.x[i] * s[i]);
        }
        return o.halves();
    };

    // ---- query heads ----
    int pair = first;
    {
        __half* out = p.q_out + (static_cast<size_t>(token) * p.n_q + 2 * first + side) * q4::kDim;
#pragma unroll 1
        for (; pair < min(last, q_pairs); ++pair, out += 2 * q4::kDim) {
            const Row r = take(pair);
            if (!p.q_out) continue;
            const Row t = turn(r);
            if (2 * pair + side < p.n_q) store_row(out, l, t);
        }
    }
    if (pair < q_pairs + kv_pairs && pair < last && first < q_pairs && normed) w = Wide(load_row(p.k_norm_w, l));

    // ---- k, then v: in groups of 4 bits ----
    const int in_page = static_cast<int>(slot) & (q4::kTokens - 1);
    unsigned char* const block = p.cache + ((slot >> 4) * p.n_layers + p.layer) * p.n_kv * static_cast<long long>(q4::page_bytes(GROUPS));
#pragma unroll 1
    for (; pair < last; ++pair) {
        const bool is_v = pair >= q_pairs + kv_pairs;
        const int head = 2 * (pair - q_pairs - (is_v ? kv_pairs : 0)) + side;
        Row r = take(pair);
        if (!is_v) r = turn(r);
        __half2 hi = __hmax2_nan(__hmax2_nan(r.h[0], r.h[1]), __hmax2_nan(r.h[2], r.h[3]));
        __half2 lo = __hmin2_nan(__hmin2_nan(r.h[0], r.h[1]), __hmin2_nan(r.h[2], r.h[3]));
        __half2 mx = __halves2half2(__hmax_nan(__low2half(hi), __high2half(hi)), __hneg(__hmin_nan(__low2half(lo), __high2half(lo))));
#pragma unroll
        for (int d = kSpan / 2; d > 0; d >>= 1) mx = __hmax2_nan(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        const q4::Scale sc(mx);
        const uint32_t word = sc.codes_plus_8(r.h);
        const int n = (l >> 1) & 3;
        const uint32_t pieces = is_v ? exchange_bytes(word, n) : 0u;
        if (head >= p.n_kv) continue;
        unsigned char* const page = block + static_cast<long long>(head) * q4::page_bytes(GROUPS);
        if ((l & (kSpan - 1)) == 0) *reinterpret_cast<__half*>(page + q4::scale_off(GROUPS, is_v, in_page, l / kSpan)) = sc.s;
        if (!is_v) {  // the lane's word: run l >> 2, quarter l & 3
            *reinterpret_cast<uint32_t*>(page + in_page * 64 + (l & 3) * 16 + (l >> 2) * 4) = word;
        } else {  // channel 8 l + e is channel 64 high + 16 n + 8 half + r with high = l >> 3, n = (l >> 1) & 3, half = l & 1, r = e
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                uint32_t t = (pieces >> (4 * e)) & 0x0f0f0f0fu;  // a nibble of each of four bytes, to sixteen bits
                t = (t | t >> 4) & 0x00ff00ffu;
                *reinterpret_cast<uint16_t*>(page + q4::kVOff + (in_page >> 1) * 128 + (2 * n + e) * 16 + (l & 1) * 8 + (l >> 3) * 4 + (in_page & 1) * 2) =
                    static_cast<uint16_t>(t | t >> 8);
            }
        }
    }
}

// The values of listed slots, fp16: what a prompt that continues a cached prefix computes with. Half a warp per (token, kv head).
template <int GROUPS>
__global__ void __launch_bounds__(kStoreWarps * 32) kv4_read_kernel(const unsigned char* cache, const long long* slots, long long n_slots,
                                                                     int tokens, int n_kv, int layer, int n_layers, __half* k_out,
                                                                     __half* v_out) {
    constexpr int kSpan = 16 / GROUPS;
    const int lane = threadIdx.x & 31, l = lane & 15, n = (l >> 1) & 3;
    const long long item = (static_cast<long long>(blockIdx.x) * kStoreWarps + (threadIdx.x >> 5)) * 2 + (lane >> 4);
    const int token = static_cast<int>(item / n_kv), head = static_cast<int>(item % n_kv);
    ptx::pdl_wait();
    ptx::pdl_launch_dependents();
    const long long slot = token < tokens ? slots[token] : -1;
    const bool real = slot >= 0 && slot < n_slots;
    const int in_page = static_cast<int>(slot) & (q4::kTokens - 1);
    const unsigned char* page = cache + ((((real ? slot : 0) >> 4) * n_layers + layer) * n_kv + head) * static_cast<long long>(q4::page_bytes(GROUPS));
    uint32_t kw = 0, vw = 0;
    float ks = 0.0f, vs = 0.0f;
    if (real) {
        kw = *reinterpret_cast<const uint32_t*>(page + in_page * 64 + (l & 3) * 16 + (l >> 2) * 4);
        ks = __half2float(*reinterpret_cast<const __half*>(page + q4::scale_off(GROUPS, 0, in_page, l / kSpan)));
        vs = __half2float(*reinterpret_cast<const __half*>(page + q4::scale_off(GROUPS, 1, in_page, l / kSpan)));
#pragma unroll
        for (int e = 0; e < 2; ++e) {  // r = 2 n + e: sixteen bits to a nibble of each of four bytes
            uint32_t t = *reinterpret_cast<const uint16_t*>(page + q4::kVOff + (in_page >> 1) * 128 + (2 * n + e) * 16 + (l & 1) * 8 + (l >> 3) * 4 +
                                                            (in_page & 1) * 2);
            t = (t | t << 8) & 0x00ff00ffu;
            vw |= ((t | t << 4) & 0x0f0f0f0fu) << (4 * e);
        }
    }
    vw = exchange_bytes(vw, n);
    if (!real) return;
    const size_t at = (static_cast<size_t>(token) * n_kv + head) * q4::kDim;
    auto open = [&](uint32_t w, float s) {
        Row r;
#pragma unroll
        for (int x = 0; x < 4; ++x)
            r.h[x] = __floats2half2_rn(static_cast<float>(static_cast<int>((w >> (8 * x)) & 15) - 8) * s,
                                       static_cast<float>(static_cast<int>((w >> (8 * x + 4)) & 15) - 8) * s);
        return r;
    };
    if (k_out) store_row(k_out + at, l, open(kw, ks));
    if (v_out) store_row(v_out + at, l, open(vw, vs));
}

template <class... P, class... A>
cudaError_t launch_rows(long long warps, cudaStream_t stream, void (*kern)(P...), const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>((warps + kStoreWarps - 1) / kStoreWarps), 1, 1);
    cfg.blockDim = dim3(kStoreWarps * 32, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled(kPdlAttn) ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, args...);
}

}  // namespace

size_t kv4_page_bytes(int group) {
    return group == 32 || group == 64 || group == 128 ? q4::page_bytes(q4::kDim / group) : 0;
}

int launch_kv4_write(const __half* qkv, const __half* q_norm_w, const __half* k_norm_w, float eps, const float* freqs, const int* positions,
                     const long long* slots, void* cache, int n_blocks, int layer, int n_layers, int tokens, int n_q, int n_kv, int group,
                     __half* q_out, cudaStream_t stream) {
    if (tokens == 0) return W8A8_OK;
    StoreParams p = {qkv, q_norm_w, k_norm_w, eps, freqs, positions, slots, static_cast<long long>(n_blocks) * q4::kTokens,
                     static_cast<unsigned char*>(cache), tokens, n_q, n_kv, layer, n_layers, q_out, 1};
    // A warp takes one pair of heads while that does not fill the GPU (40 warps an SM run at once), else several, up to a token's: 48 warps an SM or
    // more. (With 32 and 96: 613 tokens 5.5 and 8.0 us instead of 6.0, 2048 tokens 16.7 and 17.3 instead of 14.9, 8192 tokens 42.6 and 44.3 instead of 42.6.)
    const int pairs = store_pairs(n_q, n_kv);
    const long long each = static_cast<long long>(tokens) * pairs / (48ll * device_sms());
    p.pairs_per_warp = each < 1 ? 1 : each < pairs ? static_cast<int>(each) : pairs;
    const long long warps = static_cast<long long>(tokens) * ((pairs + p.pairs_per_warp - 1) / p.pairs_per_warp);
    const cudaError_t e = group == 32   ? launch_rows(warps, stream, kv4_write_kernel<4>, p)
                          : group == 64 ? launch_rows(warps, stream, kv4_write_kernel<2>, p)
                                        : launch_rows(warps, stream, kv4_write_kernel<1>, p);
    if (e != cudaSuccess) return fail(W8A8_ERR_CUDA, "kv4_write launch: %s", cudaGetErrorString(e));
    return W8A8_OK;
}

int launch_kv4_read(const void* cache, int n_blocks, const long long* slots, int layer, int n_layers, int tokens, int n_kv, int group,
                    __half* k_out, __half* v_out, cudaStream_t stream) {
    if (tokens == 0) return W8A8_OK;
    const long long warps = (static_cast<long long>(tokens) * n_kv + 1) / 2, n_slots = static_cast<long long>(n_blocks) * q4::kTokens;
    const unsigned char* c = static_cast<const unsigned char*>(cache);
    const cudaError_t e =
        group == 32   ? launch_rows(warps, stream, kv4_read_kernel<4>, c, slots, n_slots, tokens, n_kv, layer, n_layers, k_out, v_out)
        : group == 64 ? launch_rows(warps, stream, kv4_read_kernel<2>, c, slots, n_slots, tokens, n_kv, layer, n_layers, k_out, v_out)
                      : launch_rows(warps, stream, kv4_read_kernel<1>, c, slots, n_slots, tokens, n_kv, layer, n_layers, k_out, v_out);
    if (e != cudaSuccess) return fail(W8A8_ERR_CUDA, "kv4_read launch: %s", cudaGetErrorString(e));
    return W8A8_OK;
}

}  // namespace w8a8
