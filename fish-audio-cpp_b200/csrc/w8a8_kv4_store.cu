// Rows of the qkv projection into the 4-bit paged cache (qk-norm, rotation, quantiser, write through a slot map), and back.
//
// Takes the place of the same reference code as qknorm_rope_kvwrite_kernel (src/engine/dual_ar_engine.cc:585-628; rope.cu:9-65;
// rms_norm.cu:10-58), with its rounding points and its summation order: q and k are the same fp16 numbers, and the cache holds what
// the fp16 cache would hold, in groups of 4 bits (w8a8_q4.cuh). Tokens are named by slots, so that a prompt's rows and a
// decode step's go the same way, and rows with a negative slot (a captured step's empty rows) are left alone, their q too.
//
// Bound: bytes for prompts (2 (n_q + 2 n_kv) 128 read and 2 n_q 128 written per token), latency for a decode step.
#include "sm100_ptx.cuh"
#include "w8a8_internal.h"
#include "w8a8_q4.cuh"

namespace w8a8 {
namespace {

constexpr int kStoreWarps = 4;

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
    int heads_per_warp;
};

// Lane l holds channels 4 l .. 4 l + 3 of a head.
struct Row {
    __half h[4];
};
__device__ __forceinline__ Row load_row(const __half* src, int lane) {
    const uint2 v = ptx::ld_result_v2(src + 4 * lane);
    const __half2 a = *reinterpret_cast<const __half2*>(&v.x), b = *reinterpret_cast<const __half2*>(&v.y);
    return {{__low2half(a), __high2half(a), __low2half(b), __high2half(b)}};
}

// Per-head RMSNorm, the sum of squares in the order of the reference's tree (rms_norm.cu:23-49 with 128 threads): over the five bits of
// an element's place in its run of 32, the highest first, then over the runs as (0 + 2) + (1 + 3). Place 4 (l & 7) + e of run
// l >> 3 is lane l's element e, so the first three levels are lanes, two are the lane's own, and the runs are lanes again.
__device__ __forceinline__ void norm_row(Row& r, const Row& w, float eps) {
    float s[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float v = __half2float(r.h[e]);
        s[e] = v * v;
    }
#pragma unroll
    for (int d = 4; d > 0; d >>= 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += __shfl_xor_sync(0xffffffffu, s[e], d);
    float t = (s[0] + s[2]) + (s[1] + s[3]);
    t += __shfl_xor_sync(0xffffffffu, t, 16);
    t += __shfl_xor_sync(0xffffffffu, t, 8);
    const float rms = rsqrtf(t / q4::kDim + eps);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float v = __half2float(r.h[e]) * rms;
        r.h[e] = __float2half(v * __half2float(w.h[e]));
    }
}

template <int GROUPS>
__global__ void __launch_bounds__(kStoreWarps * 32) kv4_write_kernel(const StoreParams p) {
    constexpr int kSpan = 32 / GROUPS;  // lanes of a group
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int heads = p.n_q + 2 * p.n_kv;
    const int per_token = (heads + p.heads_per_warp - 1) / p.heads_per_warp;
    const long long item = static_cast<long long>(blockIdx.x) * kStoreWarps + warp;
    const int token = static_cast<int>(item / per_token), h0 = static_cast<int>(item % per_token) * p.heads_per_warp;
    Row qw = {}, kw = {};
    const bool normed = p.q_norm_w != nullptr;
    if (normed) {  // parameters: asked for before the wait
        qw = load_row(p.q_norm_w, lane);
        kw = load_row(p.k_norm_w, lane);
    }
    float f[2] = {0.0f, 0.0f};
    if (p.freqs) { f[0] = p.freqs[2 * lane]; f[1] = p.freqs[2 * lane + 1]; }
    ptx::pdl_wait();
    ptx::pdl_launch_dependents();
    if (token >= p.tokens) return;
    const long long slot = p.slots[token];
    if (slot < 0 || slot >= p.n_slots) return;
    float c[2] = {1.0f, 1.0f}, s[2] = {0.0f, 0.0f};
    if (p.freqs) {
        const float pos = static_cast<float>(p.positions[token]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float angle = f[i] * pos;
            c[i] = cosf(angle);
            s[i] = sinf(angle);
        }
    }
    const int in_page = static_cast<int>(slot) & (q4::kTokens - 1);
    unsigned char* const block = p.cache + ((slot >> 4) * p.n_layers + p.layer) * p.n_kv * static_cast<long long>(q4::page_bytes(GROUPS));
    for (int head = h0; head < min(heads, h0 + p.heads_per_warp); ++head) {
        const bool is_q = head < p.n_q, is_v = head >= p.n_q + p.n_kv;
        if (is_q && !p.q_out) continue;
        Row r = load_row(p.qkv + (static_cast<size_t>(token) * heads + head) * q4::kDim, lane);
        if (!is_v) {
            if (normed) norm_row(r, is_q ? qw : kw, p.eps);
            if (p.freqs) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {  // interleaved pairs (rope.cu:36-45), rounded as qknorm_rope_kvwrite_kernel's are
                    const float a = __half2float(r.h[2 * i]), b = __half2float(r.h[2 * i + 1]);
                    r.h[2 * i] = __float2half(fmaf(a, c[i], -__fmul_rn(b, s[i])));
                    r.h[2 * i + 1] = __float2half(fmaf(b, c[i], __fmul_rn(a, s[i])));
                }
            }
        }
        if (is_q) {
            const __half2 a = __halves2half2(r.h[0], r.h[1]), b = __halves2half2(r.h[2], r.h[3]);
            uint2 v = {*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b)};
            *reinterpret_cast<uint2*>(p.q_out + (static_cast<size_t>(token) * p.n_q + head) * q4::kDim + 4 * lane) = v;
            continue;
        }
        __half2 mx = __hmax2_nan(q4::extremes(r.h[0], r.h[1]), q4::extremes(r.h[2], r.h[3]));
#pragma unroll
        for (int d = kSpan / 2; d > 0; d >>= 1) mx = __hmax2_nan(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        const q4::Scale sc(mx);
        unsigned char* const page = block + static_cast<long long>(head - p.n_q - (is_v ? p.n_kv : 0)) * q4::page_bytes(GROUPS);
        uint32_t code[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) code[e] = static_cast<uint32_t>(sc.code(r.h[e]) + 8);
        if ((lane & (kSpan - 1)) == 0)
            *reinterpret_cast<__half*>(page + q4::scale_off(GROUPS, is_v, in_page, lane / kSpan)) = sc.s;
        if (!is_v) {
            // channels 4 l .. 4 l + 3: run l >> 3, quarter (l & 7) >> 1, nibbles 4 (l & 1) ..; the even lane stores both halves
            uint32_t w = code[0] | code[1] << 4 | code[2] << 8 | code[3] << 12;
            w |= __shfl_down_sync(0xffffffffu, w, 1) << 16;
            if (!(lane & 1)) *reinterpret_cast<uint32_t*>(page + in_page * 64 + ((lane & 7) >> 1) * 16 + (lane >> 3) * 4) = w;
        } else {
            // channel 4 l + e is channel 64 high + 16 n + 8 half + r with high = l >> 4, n = (l >> 2) & 3, half = (l >> 1) & 1,
            // r = 4 (l & 1) + e: the four lanes that differ in n alone make four 16-bit pieces, one per e; each stores one
            const int n = (lane >> 2) & 3;
            uint32_t lo = (code[0] | code[1] << 16) << (4 * n), hi = (code[2] | code[3] << 16) << (4 * n);
#pragma unroll
            for (int d = 4; d <= 8; d <<= 1) {
                lo |= __shfl_xor_sync(0xffffffffu, lo, d);
                hi |= __shfl_xor_sync(0xffffffffu, hi, d);
            }
            const uint32_t both = n & 2 ? hi : lo;
            const uint16_t piece = static_cast<uint16_t>(n & 1 ? both >> 16 : both);
            const int r8 = 4 * (lane & 1) + n, half = (lane >> 1) & 1, high = lane >> 4;
            *reinterpret_cast<uint16_t*>(page + q4::kVOff + (in_page >> 1) * 128 + r8 * 16 + half * 8 + high * 4 + (in_page & 1) * 2) = piece;
        }
    }
}

// The values of listed slots, fp16: what a prompt that continues a cached prefix computes with. A warp per (token, kv head).
template <int GROUPS>
__global__ void __launch_bounds__(kStoreWarps * 32) kv4_read_kernel(const unsigned char* cache, const long long* slots, long long n_slots,
                                                                     int tokens, int n_kv, int layer, int n_layers, __half* k_out,
                                                                     __half* v_out) {
    constexpr int kSpan = 32 / GROUPS;
    const int lane = threadIdx.x & 31;
    const long long item = static_cast<long long>(blockIdx.x) * kStoreWarps + (threadIdx.x >> 5);
    const int token = static_cast<int>(item / n_kv), head = static_cast<int>(item % n_kv);
    ptx::pdl_wait();
    ptx::pdl_launch_dependents();
    if (token >= tokens) return;
    const long long slot = slots[token];
    if (slot < 0 || slot >= n_slots) return;
    const int in_page = static_cast<int>(slot) & (q4::kTokens - 1);
    const unsigned char* page = cache + (((slot >> 4) * n_layers + layer) * n_kv + head) * static_cast<long long>(q4::page_bytes(GROUPS));
    const float ks = __half2float(*reinterpret_cast<const __half*>(page + q4::scale_off(GROUPS, 0, in_page, lane / kSpan)));
    const float vs = __half2float(*reinterpret_cast<const __half*>(page + q4::scale_off(GROUPS, 1, in_page, lane / kSpan)));
    const uint32_t kc = *reinterpret_cast<const uint16_t*>(page + in_page * 64 + ((lane & 7) >> 1) * 16 + (lane >> 3) * 4 + (lane & 1) * 2);
    __half k[4], v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t piece = *reinterpret_cast<const uint16_t*>(page + q4::kVOff + (in_page >> 1) * 128 + (4 * (lane & 1) + e) * 16 +
                                                                  ((lane >> 1) & 1) * 8 + (lane >> 4) * 4 + (in_page & 1) * 2);
        k[e] = __float2half(static_cast<float>(static_cast<int>((kc >> (4 * e)) & 15) - 8) * ks);
        v[e] = __float2half(static_cast<float>(static_cast<int>((piece >> (4 * ((lane >> 2) & 3))) & 15) - 8) * vs);
    }
    const size_t at = (static_cast<size_t>(token) * n_kv + head) * q4::kDim + 4 * lane;
    if (k_out) {
        const __half2 a = __halves2half2(k[0], k[1]), b = __halves2half2(k[2], k[3]);
        *reinterpret_cast<uint2*>(k_out + at) = {*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b)};
    }
    if (v_out) {
        const __half2 a = __halves2half2(v[0], v[1]), b = __halves2half2(v[2], v[3]);
        *reinterpret_cast<uint2*>(v_out + at) = {*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b)};
    }
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
    const int heads = n_q + 2 * n_kv;
    // A warp a head while that does not fill the GPU.
    const long long all = static_cast<long long>(tokens) * heads, room = 32ll * device_sms();
    p.heads_per_warp = all > 4 * room ? 4 : all > 2 * room ? 2 : 1;
    const long long warps = static_cast<long long>(tokens) * ((heads + p.heads_per_warp - 1) / p.heads_per_warp);
    const cudaError_t e = group == 32   ? launch_rows(warps, stream, kv4_write_kernel<4>, p)
                          : group == 64 ? launch_rows(warps, stream, kv4_write_kernel<2>, p)
                                        : launch_rows(warps, stream, kv4_write_kernel<1>, p);
    if (e != cudaSuccess) return fail(W8A8_ERR_CUDA, "kv4_write launch: %s", cudaGetErrorString(e));
    return W8A8_OK;
}

int launch_kv4_read(const void* cache, int n_blocks, const long long* slots, int layer, int n_layers, int tokens, int n_kv, int group,
                    __half* k_out, __half* v_out, cudaStream_t stream) {
    if (tokens == 0) return W8A8_OK;
    const long long warps = static_cast<long long>(tokens) * n_kv, n_slots = static_cast<long long>(n_blocks) * q4::kTokens;
    const unsigned char* c = static_cast<const unsigned char*>(cache);
    const cudaError_t e =
        group == 32   ? launch_rows(warps, stream, kv4_read_kernel<4>, c, slots, n_slots, tokens, n_kv, layer, n_layers, k_out, v_out)
        : group == 64 ? launch_rows(warps, stream, kv4_read_kernel<2>, c, slots, n_slots, tokens, n_kv, layer, n_layers, k_out, v_out)
                      : launch_rows(warps, stream, kv4_read_kernel<1>, c, slots, n_slots, tokens, n_kv, layer, n_layers, k_out, v_out);
    if (e != cudaSuccess) return fail(W8A8_ERR_CUDA, "kv4_read launch: %s", cudaGetErrorString(e));
    return W8A8_OK;
}

}  // namespace w8a8
