// The linear over 4-bit weights for a few rows of int8 activation codes, and the loader's side of it.
//
//   Y[m, n] = sum over groups, ascending, of fma(float(P), ws[n, group], ...) * xs[m, group],   P = sum over the group of Xq[m, k] W4[n, k]
//
// the arithmetic of the W8A8 path (accumulate_group_kernel, int8_gemm.cu:213-234) with 4-bit codes in place of 8-bit ones: P is exact in
// int32, each group is promoted with both scales in fp32. W4 is row-major, two codes a byte (two's complement, the even k in the low
// four bits): a checkpoint's rows as they are, no packing step.
//
// Bound: the weights' bytes from HBM (N K / 2 + 2 N G): 155776 x 2560 at 16 rows in groups of 256 39.3 us in bursts, 81 % of the measured copy rate
// (41 to 44 in longer loops, at the card's power limit); at decode sizes latency: 19456 x 2560 with SwiGLU at 8 rows in groups of 64 8.2 us (3.9 for the bytes; 6.1 without activations and arithmetic), 6144 x 2560 at
// one row 3.6.
//
// A word of eight codes becomes two operand registers of mma.m16n8k32.s8 by a shift and two masks: w << 4 and w, both & 0xf0f0f0f0, are
// sixteen times the even and the odd codes as int8; the factor leaves with the weight scale (ws / 16, exact). The contraction index may
// be permuted freely as long as both operands agree and a multiply stays inside one group, so a lane reads its row's codes as they lie (16, 8
// or 4 bytes for groups of 128 and more, 64, 32), and the activations lie in shared memory in the same order, the eight channels of
// a word split into even and odd bytes.
//
// A warp streams boxes of 16 rows x 256 channels (2 KB) by TMA through a ring of its own, some stages ahead and ahead of the dependency wait, so
// no instructions are spent on addresses; rows and channels behind the matrix come as zeros. Row r of a box is row bitrev(r) of the tile: the
// rows that lanes read together then lie in different banks of the 128-byte swizzle.
//
// Split. A CTA has whole tiles of 16 rows; its warps take equal runs of their boxes, so that only tiles that a border cuts are added
// up over warps, in ascending channels, after one barrier at the end; all others leave from the registers.
#include "sm100_ptx.cuh"
#include "w8a8_internal.h"
#include "w8a8_q4.cuh"

namespace w8a8 {
namespace {

using q4::F2;
using q4::f2;

constexpr int kL4Warps = 8;
constexpr int kL4MaxSmem = 224 * 1024;
constexpr int kBoxRows = 16, kBoxBytes = 128, kBox = kBoxRows * kBoxBytes, kBoxK = 2 * kBoxBytes;

struct L4Params {
    const uint8_t* W;       // [N, K / 2]
    const __half* w_scale;  // [N, G]
    const int8_t* Xq;       // [M, K]
    const float* Xs;        // [M, G]
    __half* Y;
    const __half* residual;
    int M, N, K, g, G;
    int epilogue;
    int tiles;   // of 16 rows
    int boxes;   // per tile
    int stages;  // of a warp's ring
    int pitch;   // of a row of codes in shared memory
    int cta_tiles, longer;  // tiles of a CTA; the first `longer` CTAs have one more
    unsigned box_magic;     // 2^32 / boxes, rounded up (0: one box): x / boxes is the high word of x box_magic while x boxes < 2^32
    unsigned chunk_magic;   // the same for K / 16
    int pad;                // pitch - K
    int* status;
    int parts;            // of a row, what is promoted together: 256 / P channels
    unsigned part_magic;  // 2^31 over the parts of a group, rounded up
    int xs_rows;          // of the activation scales in shared memory: G where EXACT, else one more
};

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8_first(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(0));
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
}

__device__ __forceinline__ uint4 evens_first(uint4 v) {
    return {__byte_perm(v.x, v.y, 0x6420), __byte_perm(v.x, v.y, 0x7531), __byte_perm(v.z, v.w, 0x6420), __byte_perm(v.z, v.w, 0x7531)};
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

// The wait for a box that is not there yet. (One copy of this code.)
__device__ __noinline__ bool l4_wait_long(uint64_t* bar, uint32_t phase, int* status) {
    if (__all_sync(0xffffffffu, ptx::mbar_wait_bounded(bar, phase))) return false;
    atomicExch(status, 950);
    return true;  // (the numbers are void from here on; the barriers still run their course)
}

// T token tiles of 8; P promotes per box (256 / P channels each, all in one group); EXACT: groups of 256 / P channels, K in whole boxes and
// the scales of a box in one aligned read; DIRECT: the codes that meet a box come through the ring behind it (two boxes of 128 channels), by the
// warp that uses them.
// Shared memory: rings [warps][stages][box, codes]; pieces fp32 [warps][16][8 T + 1]; activation scales over 16, fp32 [xs_rows][8 T]; not DIRECT: codes
// [M][pitch], a pitch at which the rows that lanes read together lie in different banks. A run's last piece goes where its ring was.
// (reads run on to the end of the last box: what lies behind K meets weights of zero)
inline int l4_pitch(int K, int P) { return (K + 127) / 128 * 128 + (P <= 2 ? 16 : P == 4 ? 64 : 32); }
template <int T>
constexpr int l4_piece_floats() { return 16 * (8 * T + 1); }
template <int T>
__host__ __device__ constexpr int l4_stage_bytes(bool direct) { return kBox + (direct ? T * kBoxK * 8 : 0); }
template <int T>
constexpr int kDirectStages = T == 1 ? 3 : 2;
template <int T>
size_t l4_smem(int M, int K, int xs_rows, int stages, bool direct) {
    return 1024 + static_cast<size_t>(kL4Warps) * stages * l4_stage_bytes<T>(direct) + kL4Warps * l4_piece_floats<T>() * 4 + static_cast<size_t>(xs_rows) * 8 * T * 4 +
           (direct ? 0 : static_cast<size_t>(l4_pitch(K, 4)) * M + kBoxK);
}

template <int T, int P, bool EXACT, bool DIRECT>
__global__ void __launch_bounds__(kL4Warps * 32, 2) linear4_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ CUtensorMap x_map,
                                                                         const __grid_constant__ L4Params p) {
    constexpr int kPiece = l4_piece_floats<T>(), kCols = 8 * T + 1, kStage = l4_stage_bytes<T>(DIRECT);
    extern __shared__ unsigned char l4_smem_raw[];
    __shared__ __align__(8) uint64_t full_bar[kL4Warps][8];
    unsigned char* const base = l4_smem_raw + ((1024u - (ptx::smem_u32(l4_smem_raw) & 1023u)) & 1023u);  // (the swizzle repeats every 1024 bytes)
    float* const piece_s = reinterpret_cast<float*>(base + kL4Warps * p.stages * kStage);
    float* const xs_s = piece_s + kL4Warps * kPiece;
    auto end_piece = [&](int w) { return reinterpret_cast<float*>(base + w * p.stages * kStage); };  // of a finished run, in its ring
    const int xs_rows = EXACT ? p.G : p.G + 1;  // (one of zeros behind the last group)
    unsigned char* const codes_s = reinterpret_cast<unsigned char*>(xs_s + xs_rows * 8 * T);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, g8 = lane >> 2, j4 = lane & 3;
    const int row8 = (g8 & 1) << 2 | (g8 & 2) | g8 >> 2;  // the row of the tile that this lane's fragment row is (and + 8)
    // tiles [t0, t0 + nt) of this CTA, units [u0, u0 + n_mine) of this warp: the boxes of the CTA's tiles, one tile after the other
    const int cta = blockIdx.x, t0 = cta * p.cta_tiles + min(cta, p.longer), nt = p.cta_tiles + (cta < p.longer ? 1 : 0);
    const int all = nt * p.boxes;
    auto run_at = [&](int w) { return all * w / kL4Warps; };  // (below 2^31: the host sees to it; all is not negative)
    auto tile_of = [&](int unit) { return p.box_magic ? static_cast<int>(__umulhi(static_cast<unsigned>(unit), p.box_magic)) : unit; };
    const int u0 = run_at(warp), n_mine = run_at(warp + 1) - u0;
    const int first_tile = tile_of(u0);
    int tile = t0 + first_tile, box = u0 - first_tile * p.boxes;
    bool head = box > 0;  // the tile began in another warp's run

    const uint32_t ring = ptx::smem_u32(base) + warp * p.stages * kStage;
    int l_tile = tile, l_box = box;
    auto issue = [&](int stage) {  // (one lane)
        uint64_t* bar = &full_bar[warp][stage];
        ptx::mbar_arrive_expect_tx(bar, kStage);
        ptx::tma_load_2d_at(ring + stage * kStage, &map, bar, l_box * kBoxBytes, l_tile * kBoxRows);
        if (++l_box == p.boxes) {
            l_box = 0;
            ++l_tile;
        }
    };
    int c_box = box;
    auto issue_codes = [&](int stage) {  // (DIRECT; one lane) the codes that meet the box: two boxes of 8 T rows x 128 channels
#pragma unroll
        for (int h = 0; h < 2; ++h)
            ptx::tma_load_2d_at(ring + stage * kStage + kBox + h * 8 * T * 128, &x_map, &full_bar[warp][stage], c_box * kBoxK + h * 128, 0);
        if (++c_box == p.boxes) c_box = 0;
    };
    if (lane < p.stages) ptx::mbar_init(&full_bar[warp][lane], 1);
    ptx::fence_barrier_init();
    ptx::fence_proxy_async();
    __syncwarp();
    if (lane == 0)
        for (int i = 0; i < min(p.stages, n_mine); ++i) issue(i);
    // weight scales of the box that comes next, rows row8 and row8 + 8
    __half2 ws_next[P > 1 ? P : 1];  // EXACT, P > 1: [row half][P / 2 pairs of groups]; else one {row, row + 8} pair per promote
    // (a part behind K has no channels and takes two scales of zero: its sum of zero times an infinite one would be no number)
    auto missing = [&](int part) { return !EXACT && P > 1 && part >= p.parts; };
    auto group_of = [&](int part) { return EXACT ? part : missing(part) ? p.G : static_cast<int>(__umulhi(2u * part, p.part_magic)); };
    const __half *ws_row0 = nullptr, *ws_row1 = nullptr;  // of the tile that the next box belongs to
    auto scale_rows = [&](int tl) {
        ws_row0 = p.w_scale + static_cast<size_t>(min(tl * 16 + row8, p.N - 1)) * p.G;
        ws_row1 = p.w_scale + static_cast<size_t>(min(tl * 16 + row8 + 8, p.N - 1)) * p.G;
    };
    auto load_scales = [&](int bx) {
        if constexpr (EXACT && P > 1) {
            uint32_t* w = reinterpret_cast<uint32_t*>(ws_next);
            const __half *a = ws_row0 + bx * P, *b = ws_row1 + bx * P;
            if constexpr (P == 2) {
                w[0] = __ldg(reinterpret_cast<const uint32_t*>(a));
                w[1] = __ldg(reinterpret_cast<const uint32_t*>(b));
            } else if constexpr (P == 4) {
                const uint2 x = __ldg(reinterpret_cast<const uint2*>(a)), y = __ldg(reinterpret_cast<const uint2*>(b));
                w[0] = x.x; w[1] = x.y; w[2] = y.x; w[3] = y.y;
            } else {
                const uint4 x = __ldg(reinterpret_cast<const uint4*>(a)), y = __ldg(reinterpret_cast<const uint4*>(b));
                w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w; w[4] = y.x; w[5] = y.y; w[6] = y.z; w[7] = y.w;
            }
        } else {
#pragma unroll
            for (int pr = 0; pr < P; ++pr) {
                const int gr = min(p.G - 1, group_of(bx * P + pr));
                const __half2 w = __halves2half2(ws_row0[gr], ws_row1[gr]);
                ws_next[pr] = missing(bx * P + pr) ? __halves2half2(__ushort_as_half(0), __ushort_as_half(0)) : w;
            }
        }
    };
    if (n_mine > 0) {
        scale_rows(tile);
        load_scales(box);
    }
    ptx::pdl_wait();
    ptx::pdl_launch_dependents();  // (at the start it costs 1 % of a step: what is launched then takes room)

    // ---- the activations ----
    // DIRECT: each box's codes come with it. Else all rows to shared memory, the eight channels of a word even ones first.
    bool failed = false;
    constexpr int kAhead = 4;
    uint4 c_next[kAhead];
    const int chunks = p.M * (p.K / 16);  // of 16 codes; X is [M, K] without gaps
    auto ask = [&](int x0) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (x0 + i * kL4Warps * 32 < chunks) c_next[i] = ptx::ld_result_v4(p.Xq + 16ll * (x0 + i * kL4Warps * 32));
    };
    if constexpr (DIRECT) {
        if (lane == 0)
            for (int i = 0; i < min(p.stages, n_mine); ++i) issue_codes(i);
    } else {
        ask(tid);
    }
    for (int x = tid; x < xs_rows * 8 * T; x += kL4Warps * 32) {
        const int group = x / (8 * T), m = x % (8 * T);
        xs_s[x] = m < p.M && (EXACT || group < p.G) ? 0.0625f * ptx::ld_result_f32(p.Xs + static_cast<size_t>(m) * p.G + group) : 0.0f;
    }
    if constexpr (!DIRECT) {
#pragma unroll 1
        for (int x0 = tid; x0 < chunks; ask(x0 += kAhead * kL4Warps * 32)) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int x = x0 + i * kL4Warps * 32;
                if (x < chunks) *reinterpret_cast<uint4*>(codes_s + 16 * x + __umulhi(x, p.chunk_magic) * p.pad) = evens_first(c_next[i]);
            }
        }
    }
    __syncthreads();

    // ---- the run ----
    F2 sums[T][2];  // of rows row8, row8 + 8: tokens 8 t + 2 j4, + 1
#pragma unroll
    for (int t = 0; t < T; ++t) sums[t][0] = sums[t][1] = f2(0.0f, 0.0f);
    auto emit = [&](int at_tile, int r, int m, float v, float up) {  // rows r and (SwiGLU only) r + 8 of a tile, token m
        if (p.epilogue == W8A8_EPI_SWIGLU) {
            p.Y[static_cast<size_t>(m) * (p.N / 2) + at_tile * 8 + r] = l4_swiglu(v, up);
        } else if (at_tile * 16 + r < p.N) {
            const size_t at = static_cast<size_t>(m) * p.N + at_tile * 16 + r;
            p.Y[at] = l4_plain(v, p.residual, at);
        }
    };
    const uint32_t row_off = row8 * kBoxBytes;  // (the swizzle turns a row's 16-byte places by row8, the same for row8 + 8)
    uint32_t codes[T];  // (fragment rows behind the last row of X read that one: what becomes of them is not stored)
#pragma unroll
    for (int t = 0; t < T; ++t)
        codes[t] = ptx::smem_u32(codes_s) + min(8 * t + g8, p.M - 1) * p.pitch + j4 * (P <= 2 ? 32 : P == 4 ? 16 : 8);
    const uint32_t xs_at = ptx::smem_u32(xs_s) + 2 * j4 * 4;
    int stage = 0;
    uint32_t phase = 0;
    int left = n_mine;  // boxes of the run that are not done
#pragma unroll 1
    while (left > 0) {
        const int end = min(p.boxes, box + left);  // the run's boxes of this tile
        const bool tile_ends = end == p.boxes;
#pragma unroll 1
        for (; box < end; ++box, --left) {
            __half2 ws[P > 1 ? P : 1];
#pragma unroll
            for (int x = 0; x < (P > 1 ? P : 1); ++x) ws[x] = ws_next[x];
            if (box + 1 == end && left > 1) scale_rows(tile + 1);
            const int next_box = box + 1 < end ? box + 1 : left > 1 ? 0 : box;
            load_scales(next_box);
            if (!__all_sync(0xffffffffu, ptx::mbar_try_wait(&full_bar[warp][stage], phase)) && !failed) failed = l4_wait_long(&full_bar[warp][stage], phase, p.status);
            const uint32_t at = ring + stage * kStage + row_off;
            int sum[T][4];
            uint4 wide[2];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t w[2][2];  // [row half][word]
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t r = at + half * 8 * kBoxBytes;
                    if constexpr (P <= 2) {
                        if (!(q & 1)) wide[half] = lds128(r + (((2 * q + j4) ^ row8) << 4));
                        w[half][0] = q & 1 ? wide[half].z : wide[half].x;
                        w[half][1] = q & 1 ? wide[half].w : wide[half].y;
                    } else if constexpr (P == 4) {
                        const uint2 v = lds64(r + (((2 * q + (j4 >> 1)) ^ row8) << 4) + (j4 & 1) * 8);
                        w[half][0] = v.x;
                        w[half][1] = v.y;
                    } else {
                        w[half][0] = lds32(r + (((2 * q) ^ row8) << 4) + j4 * 4);
                        w[half][1] = lds32(r + (((2 * q + 1) ^ row8) << 4) + j4 * 4);
                    }
                }
                uint32_t a[2][4];
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    a[v][0] = (w[0][v] << 4) & 0xf0f0f0f0u;
                    a[v][1] = (w[1][v] << 4) & 0xf0f0f0f0u;
                    a[v][2] = w[0][v] & 0xf0f0f0f0u;
                    a[v][3] = w[1][v] & 0xf0f0f0f0u;
                }
                uint4 x[T];
#pragma unroll
                for (int t = 0; t < T; ++t) {
                    const uint32_t from = codes[t] + box * kBoxK + q * 64;
                    if constexpr (DIRECT) {  // chunks of 16 lie in the 128-byte swizzle
                        const uint32_t row = ring + stage * kStage + kBox + (8 * t + g8) * 128 + (q >> 1) * 8 * T * 128;
                        if constexpr (P <= 4) {
                            x[t] = evens_first(lds128(row + (((P <= 2 ? 2 * j4 + (q & 1) : (q & 1) * 4 + j4) ^ g8) << 4)));
                        } else {
                            const uint2 a = lds64(row + ((((q & 1) * 4 + (j4 >> 1)) ^ g8) << 4) + (j4 & 1) * 8);
                            const uint2 b = lds64(row + ((((q & 1) * 4 + 2 + (j4 >> 1)) ^ g8) << 4) + (j4 & 1) * 8);
                            x[t] = evens_first({a.x, a.y, b.x, b.y});
                        }
                    } else if constexpr (P <= 2) {
                        x[t] = lds128(from - (q & 1) * 48);  // quarters 0, 1: the first and second 16 of the lane's 32 channels
                    } else if constexpr (P == 4) {
                        x[t] = lds128(from);
                    } else {
                        const uint2 a = lds64(from), b = lds64(from + 32);
                        x[t] = {a.x, a.y, b.x, b.y};
                    }
                }
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    const bool first = P == 8 || (v == 0 && (P == 4 || (P == 2 && !(q & 1)) || (P == 1 && q == 0)));
#pragma unroll
                    for (int t = 0; t < T; ++t) {
                        const uint32_t b0 = v ? x[t].z : x[t].x, b1 = v ? x[t].w : x[t].y;
                        if (first)
                            mma_s8_first(sum[t], a[v][0], a[v][1], a[v][2], a[v][3], b0, b1);
                        else
                            mma_s8(sum[t], a[v][0], a[v][1], a[v][2], a[v][3], b0, b1);
                    }
                    if (P == 8 || (v == 1 && (P == 4 || (P == 2 && (q & 1)) || q == 3))) {  // promote
                        const int pr = P == 8 ? 2 * q + v : P == 4 ? q : P == 2 ? q >> 1 : 0;
                        float ws0, ws1;
                        if constexpr (EXACT && P > 1) {
                            ws0 = pr & 1 ? __high2float(ws[pr / 2]) : __low2float(ws[pr / 2]);
                            ws1 = pr & 1 ? __high2float(ws[P / 2 + pr / 2]) : __low2float(ws[P / 2 + pr / 2]);
                        } else {
                            ws0 = __low2float(ws[pr]);
                            ws1 = __high2float(ws[pr]);
                        }
                        const uint32_t xg = xs_at + group_of(box * P + pr) * (8 * T * 4);
#pragma unroll
                        for (int t = 0; t < T; ++t) {
                            const uint2 xx = lds64(xg + t * 32);
                            const F2 x01 = f2(__uint_as_float(xx.x), __uint_as_float(xx.y));
                            sums[t][0] = fma2(f2(static_cast<float>(sum[t][0]), static_cast<float>(sum[t][1])) * f2(ws0, ws0), x01, sums[t][0]);
                            sums[t][1] = fma2(f2(static_cast<float>(sum[t][2]), static_cast<float>(sum[t][3])) * f2(ws1, ws1), x01, sums[t][1]);
                        }
                    }
                }
            }
            // ---- the stage is free ----
            if (left > p.stages) {
                ptx::fence_proxy_async();
                __syncwarp();
                if (lane == 0 && !failed) {
                    issue(stage);
                    if constexpr (DIRECT) issue_codes(stage);
                }
            }
            if (++stage == p.stages) {
                stage = 0;
                phase ^= 1;
            }
        }
        float acc[T][4];
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const float2 a = parts(sums[t][0]), c = parts(sums[t][1]);
            acc[t][0] = a.x; acc[t][1] = a.y; acc[t][2] = c.x; acc[t][3] = c.y;
            sums[t][0] = sums[t][1] = f2(0.0f, 0.0f);
        }
        if (tile_ends && !head) {  // all of the tile
            const int columns = p.epilogue == W8A8_EPI_SWIGLU ? p.N / 2 : p.N, n = p.epilogue == W8A8_EPI_SWIGLU ? tile * 8 + row8 : tile * 16 + row8;
            const size_t first = static_cast<size_t>(2 * j4) * columns + n;
            __half* y = p.Y + first;
            auto each = [&](auto put) {  // put(y, t, e) for the lane's tokens
#pragma unroll
                for (int t = 0; t < T; ++t)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        if (8 * t + 2 * j4 + e < p.M) put(static_cast<size_t>(8 * t + e) * columns, t, e);
            };
            if (p.epilogue == W8A8_EPI_SWIGLU) {
                each([&](size_t at, int t, int e) { y[at] = l4_swiglu(acc[t][e], acc[t][2 + e]); });
            } else {
                const bool row0 = n < p.N, row1 = n + 8 < p.N;
                if (p.residual) {
                    const __half* const r = p.residual + first;
                    each([&](size_t at, int t, int e) {
                        if (row0) y[at] = l4_plain(acc[t][e], r, at);
                        if (row1) y[at + 8] = l4_plain(acc[t][2 + e], r, at + 8);
                    });
                } else {
                    each([&](size_t at, int t, int e) {
                        if (row0) y[at] = __float2half_rn(acc[t][e]);
                        if (row1) y[at + 8] = __float2half_rn(acc[t][2 + e]);
                    });
                }
            }
        } else {
            float* const piece = head ? piece_s + warp * kPiece : end_piece(warp);
#pragma unroll
            for (int t = 0; t < T; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) piece[(row8 + 4 * (e & 2)) * kCols + 8 * t + 2 * j4 + (e & 1)] = acc[t][e];
        }
        head = false;
        ++tile;
        box = 0;
    }
    __syncthreads();

    // ---- tiles that a border between warps cuts: lane w looks at the border in front of warp w; a tile counts at its first border ----
    const bool swiglu = p.epilogue == W8A8_EPI_SWIGLU;
    const int border = run_at(min(lane, kL4Warps)), cut_at = tile_of(border);
    const bool cuts = lane > 0 && lane < kL4Warps && border != cut_at * p.boxes;
    const bool cuts_before = __shfl_up_sync(0xffffffffu, cuts, 1);
    const int cut_before = __shfl_up_sync(0xffffffffu, cut_at, 1);
    const uint32_t cut_tiles = __ballot_sync(0xffffffffu, cuts && !(lane > 1 && cuts_before && cut_before == cut_at));
    const int n_cuts = __popc(cut_tiles);
    if (n_cuts > 0) {  // the warps take the cut tiles in turn; a lane has one row of the tile (SwiGLU: and the one 8 below) and every so many tokens
        int c = warp, share = 0, shares = 0;
        for (; c >= n_cuts; c -= n_cuts) ++share;
        for (int x = c; x < kL4Warps; x += n_cuts) ++shares;
        uint32_t later = cut_tiles;
        for (int x = 0; x < c; ++x) later &= later - 1;
        const int w = __ffs(later) - 1, to = (__shfl_sync(0xffffffffu, cut_at, w) + 1) * p.boxes;
        // its pieces: of warp w - 1, whose run it ends, and of those behind that border that begin inside it
        const int next_border = __shfl_down_sync(0xffffffffu, border, 1);
        const uint32_t has = __ballot_sync(0xffffffffu, lane >= w && lane < kL4Warps && border < to && next_border > border);
        const int cut = __shfl_sync(0xffffffffu, cut_at, w);
        const int rows_log = swiglu ? 3 : 4, r = lane & ((1 << rows_log) - 1);
#pragma unroll 1
        for (int m = (share << (5 - rows_log)) + (lane >> rows_log); m < p.M; m += shares << (5 - rows_log)) {
            const float* piece = end_piece(w - 1) + r * kCols + m;
            float v = piece[0], up = swiglu ? piece[8 * kCols] : 0.0f;
#pragma unroll 1
            for (uint32_t rest = has; rest; rest &= rest - 1) {
                piece = piece_s + (__ffs(rest) - 1) * kPiece + r * kCols + m;
                v += piece[0];
                if (swiglu) up += piece[8 * kCols];
            }
            emit(t0 + cut, r, m, v, up);
        }
    }
    if (failed) {  // copies that may still be on their way land before the CTA goes
#pragma unroll 1
        for (int w = 0; w < 1000; ++w) __nanosleep(1000);
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
cudaError_t launch_l4(SmemAttribute* attribute, int ctas, size_t smem, cudaStream_t stream, void (*kern)(P...), const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, 1, 1);
    cfg.blockDim = dim3(256, 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled(kPdlLinear) ? 1 : 0;
    return attribute ? launch_with_smem(*attribute, kL4MaxSmem, cfg, kern, args...) : cudaLaunchKernelEx(&cfg, kern, args...);
}

// Stages of a warp's ring: as many as leave room for two CTAs on an SM (more than four are not worth their space), else for one; 0: no room. (At
// least two: in the end the ring holds a piece of up to 2112 bytes.)
constexpr size_t kHalfSm = 112 * 1024, kThirdSm = 76 * 1024;
template <int T>
int l4_stages(int M, int K, int xs_rows, bool direct) {
    if (direct) return l4_smem<T>(M, K, xs_rows, kDirectStages<T>, true) <= kL4MaxSmem ? kDirectStages<T> : 0;
    for (int stages = 4; stages >= 2; --stages)
        if (l4_smem<T>(M, K, xs_rows, stages, direct) <= kHalfSm) return stages;
    for (int stages = 8; stages >= 2; --stages)
        if (l4_smem<T>(M, K, xs_rows, stages, direct) <= kL4MaxSmem) return stages;
    return 0;
}
int l4_stages(int M, int K, int xs_rows, bool direct) {
    return M > 16 ? l4_stages<4>(M, K, xs_rows, direct) : M > 8 ? l4_stages<2>(M, K, xs_rows, direct) : l4_stages<1>(M, K, xs_rows, direct);
}

// DIRECT where every CTA has one tile, so that a code is read once either way, and there are rows enough: eight rows of 4096 channels on 160 tiles
// in a run of launches 3.9 us, through shared memory 4.2; sixteen 4.7 and 5.7; one row 5.0 and 3.5 (between them the rule has not been measured); eight rows of 2560 on 1216 tiles 8.3 and 7.7.
// And where a CTA's codes leave no room for two CTAs on an SM (eight rows of 9728 channels: 10.7 us with one of them).
template <int T, int P, bool EXACT>
cudaError_t launch_boxes(L4Params p, const CUtensorMap& map, cudaStream_t stream) {
    static SmemAttribute attribute[2] = {SmemAttribute(true), SmemAttribute(true)};
    const bool direct = T <= 2 && ((p.M > 4 && p.tiles <= 2 * device_sms()) || l4_smem<T>(p.M, p.K, p.xs_rows, 2, false) > kHalfSm);
    p.stages = l4_stages<T>(p.M, p.K, p.xs_rows, direct);
    const int ctas = gemv_packed_ctas(p.tiles, device_sms(), l4_smem<T>(p.M, p.K, p.xs_rows, p.stages, direct) <= kHalfSm);
    p.cta_tiles = p.tiles / ctas;
    p.longer = p.tiles - p.cta_tiles * ctas;
    p.chunk_magic = static_cast<unsigned>(((1ull << 32) + p.K / 16 - 1) / (p.K / 16));
    p.pad = p.pitch - p.K;
    p.parts = (p.K + kBoxK / P - 1) / (kBoxK / P);
    const int group_parts = (p.g + kBoxK / P - 1) / (kBoxK / P);
    p.part_magic = static_cast<unsigned>(((1ull << 31) + group_parts - 1) / group_parts);
    p.box_magic = p.boxes == 1 ? 0u : static_cast<unsigned>(((1ull << 32) + p.boxes - 1) / p.boxes);
    // Never three CTAs on an SM: what the third takes from the others is more than its early start gives (four projections at one row 22.6 us with
    // three, 20.1 with two, 30.6 with one).
    size_t smem = l4_smem<T>(p.M, p.K, p.xs_rows, p.stages, direct);
    if (smem < kThirdSm) smem = kThirdSm;
    if constexpr (T <= 2)
        if (direct) {
            CUtensorMap x_map;
            if (make_tensor_map_2d_u8(&x_map, p.Xq, p.K, p.M, p.K, 128, 8 * T, 1)) return cudaErrorInvalidValue;
            return launch_l4(&attribute[1], ctas, smem, stream, linear4_kernel<T, P, EXACT, true>, map, x_map, p);
        }
    return launch_l4(&attribute[0], ctas, smem, stream, linear4_kernel<T, P, EXACT, false>, map, map, p);
}
template <int T, bool EXACT>
cudaError_t launch_rows4(const L4Params& p, const CUtensorMap& map, int P, cudaStream_t stream) {
    return P == 1   ? launch_boxes<T, 1, EXACT>(p, map, stream)
           : P == 2 ? launch_boxes<T, 2, EXACT>(p, map, stream)
           : P == 4 ? launch_boxes<T, 4, EXACT>(p, map, stream)
                    : launch_boxes<T, 8, EXACT>(p, map, stream);
}

}  // namespace

int launch_linear4(const void* W, const __half* w_scale, int group, const int8_t* Xq, const float* Xs, __half* Y, const __half* residual, int M, int N,
                   int K, int epilogue, int* status, cudaStream_t stream) {
    if (M == 0) return W8A8_OK;
    const int g = norm_group(K, group), G = num_groups(K, group);
    const bool swiglu = epilogue == W8A8_EPI_SWIGLU;
    const int columns = swiglu ? N / 2 : N;
    const int P = g % 256 == 0 ? 1 : g % 128 == 0 ? 2 : g % 64 == 0 ? 4 : 8;
    const bool exact = g == kBoxK / P && K % kBoxK == 0 && (reinterpret_cast<uintptr_t>(w_scale) & (2 * P - 1)) == 0;
    // rows of a launch: as many as fit shared memory; the weights are streamed once per launch
    const int xs_rows = G + (exact ? 0 : 1);
    int rows = 32;
    while (rows > 1 && l4_stages(rows, K, xs_rows, rows <= 16) == 0) rows /= 2;
    const bool fast = K % 32 == 0 && g % 32 == 0 && ((reinterpret_cast<uintptr_t>(W) | reinterpret_cast<uintptr_t>(Xq)) & 15u) == 0 &&
                      l4_stages(rows, K, xs_rows, rows <= 16) > 0 &&
                      // the kernel's 32-bit arithmetic
                      (static_cast<unsigned long long>((N + 15) / 16) / device_sms() + 2) * ((K + kBoxK - 1) / kBoxK) * ((K + kBoxK - 1) / kBoxK) < (1ull << 28);
    CUtensorMap map;
    if (fast)
        if (int rc = make_tensor_map_2d_u8(&map, W, K / 2, N, K / 2, kBoxBytes, kBoxRows, 1)) return rc;
    for (int m0 = 0; m0 < M; m0 += rows) {
        const int m = fast ? (M - m0 < rows ? M - m0 : rows) : M;
        L4Params p = {static_cast<const uint8_t*>(W), w_scale, Xq + static_cast<size_t>(m0) * K, Xs + static_cast<size_t>(m0) * G,
                      Y + static_cast<size_t>(m0) * columns, residual ? residual + static_cast<size_t>(m0) * N : nullptr, m, N, K, g, G, epilogue,
                      (N + 15) / 16, (K + kBoxK - 1) / kBoxK, 0, l4_pitch(K, P), 0, 0, 0, 0, 0, status, 0, 0, xs_rows};
        cudaError_t e;
        if (fast) {
            if (exact)
                e = m <= 8 ? launch_rows4<1, true>(p, map, P, stream) : m <= 16 ? launch_rows4<2, true>(p, map, P, stream) : launch_rows4<4, true>(p, map, P, stream);
            else
                e = m <= 8 ? launch_rows4<1, false>(p, map, P, stream) : m <= 16 ? launch_rows4<2, false>(p, map, P, stream) : launch_rows4<4, false>(p, map, P, stream);
        } else {
            const long long warps = static_cast<long long>(M) * columns, ctas = (warps + 7) / 8;
            if (ctas > 0x7fffffffll) return fail(W8A8_ERR_UNSUPPORTED, "linear4_q: M=%d N=%d is too large for this shape's kernel", M, N);
            e = launch_l4(nullptr, static_cast<int>(ctas), 0, stream, linear4_generic_kernel, p);
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
