// The linear over 4-bit weights for a few rows of int8 activation codes, and the loader's side of it.
//
//   Y[m, n] = sum over groups, ascending, of fma(float(P), ws[n, group], ...) * xs[m, group],   P = sum over the group of Xq[m, k] W4[n, k]
//
// the arithmetic of the W8A8 path (accumulate_group_kernel, int8_gemm.cu:213-234) with 4-bit codes in place of 8-bit ones: P is exact in
// int32, each group is promoted with both scales in fp32. W4 is row-major, two codes a byte (two's complement, the even k in the low
// four bits): a checkpoint's rows as they are, no packing step.
//
// Bound: the weights' bytes from HBM (N K / 2 + 2 N G); at decode sizes the fixed cost of a launch.
//
// A word of eight codes becomes two operand registers of mma.m16n8k32.s8 by a shift and two masks: w << 4 and w, both & 0xf0f0f0f0, are
// sixteen times the even and the odd codes as int8; the factor leaves with the weight scale (ws / 16, exact). The contraction index may
// be permuted freely as long as both operands agree, so lane (row, j) takes 4 V consecutive bytes of its row, and the activations of the
// same 8 V channels are split into even and odd bytes by two byte permutes per pair of words.
#include "sm100_ptx.cuh"
#include "w8a8_internal.h"
#include "w8a8_q4.cuh"

namespace w8a8 {
namespace {

constexpr int kL4Warps = 8;

struct L4Params {
    const uint8_t* W;       // [N, K / 2]
    const __half* w_scale;  // [N, G]
    const int8_t* Xq;       // [M, K]
    const float* Xs;        // [M, G]
    __half* Y;
    const __half* residual;
    int M, N, K, g, G;
    int epilogue;
    int tiles;  // of 16 rows
};

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <int V>
struct Words {
    uint32_t w[V];
};
template <int V>
__device__ __forceinline__ Words<V> load_weights(const uint8_t* p) {
    Words<V> r;
    if constexpr (V == 4)
        asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]) : "l"(p));
    else if constexpr (V == 2)
        asm volatile("ld.global.v2.u32 {%0,%1}, [%2];" : "=r"(r.w[0]), "=r"(r.w[1]) : "l"(p));
    else
        asm volatile("ld.global.u32 %0, [%1];" : "=r"(r.w[0]) : "l"(p));
    return r;
}

// What the epilogues make of a finished fp32 sum (roundings of the reference's separate kernels, ffn_activations.cu:12-17, :35-45).
__device__ __forceinline__ __half l4_swiglu(float gate, float up) {
    const float x = __half2float(__float2half_rn(gate));
    const float s = x / (1.0f + expf(-x));
    return __float2half_rn(__half2float(__float2half_rn(s)) * __half2float(__float2half_rn(up)));
}
__device__ __forceinline__ __half l4_plain(float v, const __half* residual, size_t at) {
    const __half h = __float2half_rn(v);
    return residual ? __float2half_rn(__half2float(h) + __half2float(residual[at])) : h;
}

// T token tiles of 8; V words a lane and row per step (a step is 32 V channels, all in one group).
template <int T, int V>
__global__ void __launch_bounds__(kL4Warps * 32) linear4_kernel(const L4Params p) {
    constexpr int U = 4;  // steps on their way
    __shared__ float part_s[2][kL4Warps][16][8 * T + 1];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g8 = lane >> 2, j4 = lane & 3;
    const int steps = (p.K + 32 * V - 1) / (32 * V);
    const int s0 = steps * warp / kL4Warps, s1 = steps * (warp + 1) / kL4Warps, mine = s1 - s0;
    const int n_tiles = blockIdx.x < p.tiles ? (p.tiles - 1 - blockIdx.x) / gridDim.x + 1 : 0;
    const int total = mine * n_tiles;
    const size_t pitch = static_cast<size_t>(p.K / 2);

    Words<V> wbuf[U][2];
    int l_tile = blockIdx.x, l_step = s0;  // the next step to load
    auto load = [&](Words<V> (&w)[2]) {
        const int k = 32 * V * l_step + 8 * V * j4;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int row = l_tile * 16 + 8 * half + g8;
#pragma unroll
            for (int v = 0; v < V; ++v) w[half].w[v] = 0u;
            if (k < p.K && row < p.N) w[half] = load_weights<V>(p.W + row * pitch + k / 2);
        }
        if (++l_step == s1) {
            l_step = s0;
            l_tile += gridDim.x;
        }
    };
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (u < total) load(wbuf[u]);
    ptx::pdl_wait();
    ptx::pdl_launch_dependents();

    int tile = blockIdx.x, step = s0, parity = 0;
    int sum[T][4];
    float acc[T][4];
#pragma unroll
    for (int t = 0; t < T; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            sum[t][e] = 0;
            acc[t][e] = 0.0f;
        }
    auto finish_tile = [&] {
#pragma unroll
        for (int t = 0; t < T; ++t) {
            part_s[parity][warp][g8][8 * t + 2 * j4] = acc[t][0];
            part_s[parity][warp][g8][8 * t + 2 * j4 + 1] = acc[t][1];
            part_s[parity][warp][g8 + 8][8 * t + 2 * j4] = acc[t][2];
            part_s[parity][warp][g8 + 8][8 * t + 2 * j4 + 1] = acc[t][3];
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[t][e] = 0.0f;
        }
        __syncthreads();
        auto added = [&](int r, int m) {
            float v = part_s[parity][0][r][m];
#pragma unroll
            for (int w = 1; w < kL4Warps; ++w) v += part_s[parity][w][r][m];
            return v;
        };
        if (p.epilogue == W8A8_EPI_SWIGLU) {
            for (int x = tid; x < 8 * p.M; x += kL4Warps * 32) {
                const int r = x & 7, m = x >> 3;
                p.Y[static_cast<size_t>(m) * (p.N / 2) + tile * 8 + r] = l4_swiglu(added(r, m), added(r + 8, m));
            }
        } else {
            for (int x = tid; x < 16 * p.M; x += kL4Warps * 32) {
                const int r = x & 15, m = x >> 4;
                const size_t at = static_cast<size_t>(m) * p.N + tile * 16 + r;
                if (tile * 16 + r < p.N) p.Y[at] = l4_plain(added(r, m), p.residual, at);
            }
        }
        parity ^= 1;  // (the next tile's sums go to the other buffer; its barrier comes before this one is written again)
    };
    if (mine == 0) {  // fewer steps than warps: nothing to add, but every barrier to meet
        for (int t = 0; t < n_tiles; ++t, tile += gridDim.x) finish_tile();
        return;
    }
    for (int i0 = 0; i0 < total; i0 += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i0 + u >= total) break;
            const int k = 32 * V * step + 8 * V * j4;
            uint32_t a[V][4];
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t w = wbuf[u][half].w[v];
                    a[v][half] = (w << 4) & 0xf0f0f0f0u;
                    a[v][2 + half] = w & 0xf0f0f0f0u;
                }
            if (i0 + u + U < total) load(wbuf[u]);
#pragma unroll
            for (int t = 0; t < T; ++t) {
                const int m = 8 * t + g8;
                uint32_t x[2 * V];
#pragma unroll
                for (int v = 0; v < 2 * V; ++v) x[v] = 0u;
                if (m < p.M && k < p.K) {
                    const uint32_t* src = reinterpret_cast<const uint32_t*>(p.Xq + static_cast<size_t>(m) * p.K + k);
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        const uint2 two = ptx::ld_result_v2(src + 2 * v);
                        x[2 * v] = two.x;
                        x[2 * v + 1] = two.y;
                    }
                }
#pragma unroll
                for (int v = 0; v < V; ++v)
                    mma_s8(sum[t], a[v][0], a[v][1], a[v][2], a[v][3], __byte_perm(x[2 * v], x[2 * v + 1], 0x6420),
                           __byte_perm(x[2 * v], x[2 * v + 1], 0x7531));
            }
            const int group = 32 * V * step / p.g;
            const bool tile_ends = step + 1 == s1;
            if (tile_ends || 32 * V * (step + 1) / p.g != group) {
                const int row = tile * 16 + g8;
                const float ws0 = row < p.N ? __half2float(p.w_scale[static_cast<size_t>(row) * p.G + group]) * 0.0625f : 0.0f;
                const float ws1 = row + 8 < p.N ? __half2float(p.w_scale[static_cast<size_t>(row + 8) * p.G + group]) * 0.0625f : 0.0f;
#pragma unroll
                for (int t = 0; t < T; ++t) {
                    const int m = 8 * t + 2 * j4;
                    const float x0 = m < p.M ? ptx::ld_result_f32(p.Xs + static_cast<size_t>(m) * p.G + group) : 0.0f;
                    const float x1 = m + 1 < p.M ? ptx::ld_result_f32(p.Xs + static_cast<size_t>(m + 1) * p.G + group) : 0.0f;
                    acc[t][0] = fmaf(static_cast<float>(sum[t][0]) * ws0, x0, acc[t][0]);
                    acc[t][1] = fmaf(static_cast<float>(sum[t][1]) * ws0, x1, acc[t][1]);
                    acc[t][2] = fmaf(static_cast<float>(sum[t][2]) * ws1, x0, acc[t][2]);
                    acc[t][3] = fmaf(static_cast<float>(sum[t][3]) * ws1, x1, acc[t][3]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[t][e] = 0;
                }
            }
            if (tile_ends) {
                finish_tile();
                tile += gridDim.x;
                step = s0;
            } else {
                ++step;
            }
        }
    }
}

// Any shape with an even K: a warp per row and token, groups in ascending order in every lane's share, shares added at the end. Coverage, not speed.
__global__ void __launch_bounds__(256) linear4_generic_kernel(const L4Params p) {
    const int lane = threadIdx.x & 31;
    const long long item = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const bool swiglu = p.epilogue == W8A8_EPI_SWIGLU;
    const int columns = swiglu ? p.N / 2 : p.N;
    const int m = static_cast<int>(item / columns), n = static_cast<int>(item % columns);
    ptx::pdl_wait();
    ptx::pdl_launch_dependents();
    if (m >= p.M) return;
    float y[2] = {0.0f, 0.0f};
    for (int part = 0; part < (swiglu ? 2 : 1); ++part) {
        const size_t row = swiglu ? static_cast<size_t>(n / 8) * 16 + 8 * part + n % 8 : n;
        for (int group = 0; group < p.G; ++group) {
            const int k0 = group * p.g, k1 = min(p.K, k0 + p.g);
            int sum = 0;
            for (int k = k0 + lane; k < k1; k += 32) {
                const int byte = p.W[row * (p.K / 2) + k / 2];
                const int code = static_cast<int8_t>((k & 1) ? byte & 0xf0 : byte << 4) >> 4;
                sum += code * p.Xq[static_cast<size_t>(m) * p.K + k];
            }
            sum = __reduce_add_sync(0xffffffffu, sum);
            y[part] = fmaf(static_cast<float>(sum) * __half2float(p.w_scale[row * p.G + group]), p.Xs[static_cast<size_t>(m) * p.G + group], y[part]);
        }
    }
    if (lane == 0) {
        const size_t at = static_cast<size_t>(m) * columns + n;
        p.Y[at] = swiglu ? l4_swiglu(y[0], y[1]) : l4_plain(y[0], p.residual, at);
    }
}

// fp16 weights to 4-bit codes and group scales (w8a8_q4.cuh); a warp a group, a lane two neighbours at a time. K and g are even.
__global__ void __launch_bounds__(256) quantize_weight4_kernel(const __half* W, int N, int K, int g, int G, uint8_t* codes, __half* scale) {
    const int lane = threadIdx.x & 31;
    const long long item = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    if (item >= static_cast<long long>(N) * G) return;
    const size_t row = static_cast<size_t>(item / G);
    const int group = static_cast<int>(item % G), k0 = group * g, k1 = min(K, k0 + g);
    const __half* src = W + row * K;
    __half2 mx = __halves2half2(__ushort_as_half(0xfc00u), __ushort_as_half(0xfc00u));
    for (int k = k0 + 2 * lane; k < k1; k += 64) mx = __hmax2_nan(mx, q4::extremes(src[k], src[k + 1]));
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) mx = __hmax2_nan(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    const q4::Scale sc(mx);
    for (int k = k0 + 2 * lane; k < k1; k += 64)
        codes[row * (K / 2) + k / 2] = static_cast<uint8_t>((sc.code(src[k]) & 15) | (sc.code(src[k + 1]) & 15) << 4);
    if (lane == 0) scale[row * G + group] = sc.s;
}

// Codes as int8 [N, K]: with the same scales a weight of the W8A8 path (prompts, more rows than the decode kernel takes).
__global__ void __launch_bounds__(256) unpack_weight4_kernel(const uint8_t* codes, long long bytes, char2* W) {
    for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < bytes; i += 256ll * gridDim.x) {
        const int b = codes[i];
        W[i] = make_char2(static_cast<int8_t>(b << 4) >> 4, static_cast<int8_t>(b) >> 4);
    }
}

template <class... P, class... A>
cudaError_t launch_l4(int ctas, cudaStream_t stream, void (*kern)(P...), const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, 1, 1);
    cfg.blockDim = dim3(256, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled(kPdlLinear) ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, args...);
}

template <int V>
cudaError_t launch_rows4(const L4Params& p, cudaStream_t stream) {
    const int room = 4 * device_sms(), ctas = p.tiles < room ? p.tiles : room;
    return p.M <= 8 ? launch_l4(ctas, stream, linear4_kernel<1, V>, p) : p.M <= 16 ? launch_l4(ctas, stream, linear4_kernel<2, V>, p)
                                                                                   : launch_l4(ctas, stream, linear4_kernel<4, V>, p);
}

}  // namespace

int launch_linear4(const void* W, const __half* w_scale, int group, const int8_t* Xq, const float* Xs, __half* Y, const __half* residual, int M, int N,
                   int K, int epilogue, cudaStream_t stream) {
    const int g = norm_group(K, group), G = num_groups(K, group);
    const bool swiglu = epilogue == W8A8_EPI_SWIGLU;
    const int columns = swiglu ? N / 2 : N;
    const bool fast = K % 32 == 0 && g % 32 == 0 && ((reinterpret_cast<uintptr_t>(W) | reinterpret_cast<uintptr_t>(Xq)) & 15u) == 0;
    for (int m0 = 0; m0 < M; m0 += 32) {  // (32 rows a launch; the weights are streamed once for each)
        const int m = fast ? (M - m0 < 32 ? M - m0 : 32) : M;
        L4Params p = {static_cast<const uint8_t*>(W), w_scale, Xq + static_cast<size_t>(m0) * K, Xs + static_cast<size_t>(m0) * G,
                      Y + static_cast<size_t>(m0) * columns, residual ? residual + static_cast<size_t>(m0) * N : nullptr, m, N, K, g, G, epilogue,
                      (N + 15) / 16};
        cudaError_t e;
        if (fast) {
            e = g % 128 == 0 ? launch_rows4<4>(p, stream) : g % 64 == 0 ? launch_rows4<2>(p, stream) : launch_rows4<1>(p, stream);
        } else {
            const long long warps = static_cast<long long>(M) * columns, ctas = (warps + 7) / 8;
            if (ctas > 0x7fffffffll) return fail(W8A8_ERR_UNSUPPORTED, "linear4_q: M=%d N=%d is too large for this shape's kernel", M, N);
            e = launch_l4(static_cast<int>(ctas), stream, linear4_generic_kernel, p);
        }
        if (e != cudaSuccess) return fail(W8A8_ERR_CUDA, "linear4_q launch: %s", cudaGetErrorString(e));
        if (!fast) break;
    }
    return W8A8_OK;
}

int launch_quantize_weight4(const __half* W, int N, int K, int group, void* codes, __half* scale, cudaStream_t stream) {
    const int g = norm_group(K, group), G = num_groups(K, group);
    const long long ctas = (static_cast<long long>(N) * G + 7) / 8;
    if (ctas > 0x7fffffffll) return fail(W8A8_ERR_UNSUPPORTED, "quantize_weight4: N=%d with %d groups is too large", N, G);
    quantize_weight4_kernel<<<static_cast<unsigned>(ctas), 256, 0, stream>>>(W, N, K, g, G, static_cast<uint8_t*>(codes), scale);
    return check_launch("quantize_weight4");
}

int launch_unpack_weight4(const void* codes, int N, int K, void* W, cudaStream_t stream) {
    const long long bytes = static_cast<long long>(N) * (K / 2), want = (bytes + 255) / 256, room = 16ll * device_sms();
    unpack_weight4_kernel<<<static_cast<unsigned>(want < room ? want : room), 256, 0, stream>>>(static_cast<const uint8_t*>(codes), bytes,
                                                                                               static_cast<char2*>(W));
    return check_launch("unpack_weight4");
}

}  // namespace w8a8
