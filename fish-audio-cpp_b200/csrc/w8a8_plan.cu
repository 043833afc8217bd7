// The step plan: block tables, slot maps and positions of a ragged batch, made on the GPU from the requests' lengths, with the
// paged cache's blocks taken from and given back to a stack of free block numbers. Takes the place of the reference's host free list and
// block-table upload (src/engine/block_manager.cc, src/engine/scheduler.cc), and of the host copy of the table in its decode step
// (src/engine/dual_ar_engine.cc:568-571).
//
// With have_b = ceil(cached_b / 16), over requests in order:
//   ended (new_b < 0): its have_b blocks go on the stack, give_b = have_b
//   others: take_b = ceil((cached_b + new_b) / 16) - have_b blocks come from the stack's top (after all that was given back)
//   token i of request b has the position cached_b + i and the slot 16 * table[b][position / 16] + position % 16
// Three exclusive prefix sums (tokens, blocks taken, blocks given) make every one of these independent of the others; a block that was given
// back and taken again in the same call is read from the row that gives it, so that nothing that is read is written by the call, but
// for the lengths and the stack's count where the caller has them updated in place.
//
// Bound: latency at decode sizes (one round trip for the lengths, one for block numbers; 8 requests 3.8 us), 12 bytes written per token for prompts (512
// requests, room for 200000 tokens 7.8 us). One
// launch: a CTA per 2048 tokens, each of which makes the sums again (200000 tokens: 20.1 us when a cluster of eight shared them) and then
// four tokens a thread. What is updated in place is written by the CTA that comes last (a ticket, reset by that CTA, which costs 0.9 us
// at 512 requests). All or nothing:
// where the blocks, the table's width, the token count or a length do not fit, no request gets anything, and `info` says why.
#include "sm100_ptx.cuh"
#include "w8a8_internal.h"

namespace w8a8 {
namespace {

// Threads of a CTA: 512, and 128 where that takes no more than one round. With 128, 512 and 1024 for 8 requests of a token 3.8, -, 4.5 us; with 256, 512 and
// 1024 for 64 requests with 4 prompts 6.2, 6.5, 7.1, 512 with room for 200000 tokens 8.0, 7.8, 9.2, 4000 of a token 21.5, 17.3, 16.7.
constexpr int kPlanThreads = 512, kPlanFew = 128;
static_assert(kPlanThreads <= 32 * 32, "a warp adds up the warps' sums");
constexpr int kPlanBlock = 16;
constexpr int kPlanMaxBatch = 4096;
constexpr int kPlanMaxBlocks = 0x7fffffff / kPlanBlock;  // of a request: its tokens, and their number rounded up to whole blocks, fit 32 bits

struct PlanParams {
    const int* cached;
    const int* fresh;
    int batch;
    int* table;
    int max_blocks;
    int* free_blocks;
    int capacity;
    const int* free_count;
    int* free_count_out;
    long long* slots;
    int* positions;
    int* seq_lens;
    int* first_token;
    int max_tokens;
    int* info;
    int vector_stores;  // slots and positions are 16-byte aligned
    int* ticket;        // zero between launches; null where nothing is updated in place, or by one CTA
};

struct Sums {
    long long tokens, take, give;
};
__device__ __forceinline__ Sums operator+(Sums a, Sums b) { return {a.tokens + b.tokens, a.take + b.take, a.give + b.give}; }
__device__ __forceinline__ Sums shfl_up(Sums v, int d) {
    return {__shfl_up_sync(0xffffffffu, v.tokens, d), __shfl_up_sync(0xffffffffu, v.take, d), __shfl_up_sync(0xffffffffu, v.give, d)};
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) plan_blocks_kernel(const PlanParams p) {
    constexpr int kWarps = THREADS / 32;
    extern __shared__ int plan_smem[];
    int* first_s = plan_smem;                      // [batch + 1] tokens ahead of request b
    int* take_s = first_s + p.batch + 1;           // [batch] blocks taken ahead of it
    int* give_s = take_s + p.batch;                // [batch] blocks given back ahead of it
    int* cached_s = give_s + p.batch;              // [batch]; minus one minus the length where the request ended
    __shared__ Sums warp_s[kWarps];
    __shared__ Sums run_s;
    __shared__ int bad_s, last_s;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int part = blockIdx.x, parts = gridDim.x;
    ptx::pdl_wait();
    ptx::pdl_launch_dependents();
    const long long count = *p.free_count;
    if (tid == 0) {
        run_s = {0, 0, 0};
        bad_s = 8;  // the lowest status found (5 comes before all); 8: none
    }
    __syncthreads();
    for (int b0 = 0; b0 < p.batch; b0 += THREADS) {
        const int b = b0 + tid;
        Sums mine = {0, 0, 0};
        int cached = 0;
        bool ended = false;
        if (b < p.batch) {
            cached = p.cached[b];
            const int fresh = p.fresh[b];
            ended = fresh < 0;
            if (cached < 0) {
                atomicMin(&bad_s, 4);
                cached = 0;
            }
            const long long have = (static_cast<long long>(cached) + kPlanBlock - 1) / kPlanBlock;
            const long long all = ended ? have : (static_cast<long long>(cached) + fresh + kPlanBlock - 1) / kPlanBlock;
            if (all > min(p.max_blocks, kPlanMaxBlocks)) atomicMin(&bad_s, 2);
            mine = {ended ? 0 : fresh, all - have, ended ? have : 0};
        }
        Sums inc = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const Sums o = shfl_up(inc, d);
            if (lane >= d) inc = inc + o;
        }
        if (lane == 31) warp_s[warp] = inc;
        __syncthreads();
        const Sums base = run_s;
        if (warp == 0) {
            Sums w = {0, 0, 0};
            if (lane < kWarps) w = warp_s[lane];
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const Sums o = shfl_up(w, d);
                if (lane >= d) w = w + o;
            }
            if (lane < kWarps) warp_s[lane] = w;
        }
        __syncthreads();
        Sums at = base + inc;
        if (warp > 0) at = at + warp_s[warp - 1];
        if (b < p.batch) {  // (numbers that do not fit 32 bits belong to a plan that is refused below)
            first_s[b + 1] = static_cast<int>(at.tokens);
            take_s[b] = static_cast<int>(at.take - mine.take);
            give_s[b] = static_cast<int>(at.give - mine.give);
            cached_s[b] = ended ? -1 - cached : cached;
        }
        if (tid == 0) run_s = base + warp_s[kWarps - 1];
        __syncthreads();
    }
    if (tid == 0) first_s[0] = 0;
    const Sums all = run_s;
    const long long top = count + all.give;
    int status = bad_s;
    if (all.tokens > p.max_tokens) status = min(status, 3);
    if (all.take > top) status = min(status, 1);
    if (count < 0 || top > p.capacity) status = 5;
    const bool ok = status == 8;

    __syncthreads();  // (first_s[0])
    const int threads = parts * THREADS, me = part * THREADS + tid;
    // the request that item x of a prefix sum belongs to: the last whose items start at or before it
    auto owner = [&](const int* ahead, int x) {
        int lo = 0, hi = p.batch - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (ahead[mid] <= x) lo = mid; else hi = mid - 1;
        }
        return lo;
    };
    auto given = [&](int x) {  // the x-th block given back
        const int b = owner(give_s, x);
        return p.table[static_cast<size_t>(b) * p.max_blocks + x - give_s[b]];
    };
    auto taken = [&](int x) {  // the x-th block taken: from the stack's top, what was given back first
        const long long at = top - 1 - x;
        return at < count ? p.free_blocks[at] : given(static_cast<int>(at - count));
    };
    if (ok) {  // a thread a block
        for (long long x = me; x < all.give; x += threads) p.free_blocks[count + x] = given(static_cast<int>(x));
        for (long long x = me; x < all.take; x += threads) {
            const int b = owner(take_s, static_cast<int>(x)), have = (cached_s[b] + kPlanBlock - 1) / kPlanBlock;
            p.table[static_cast<size_t>(b) * p.max_blocks + have + static_cast<int>(x) - take_s[b]] = taken(static_cast<int>(x));
        }
    }
    for (int b = me; b < p.batch; b += threads) p.first_token[b + 1] = ok ? first_s[b + 1] : 0;
    if (me == 0) {
        p.first_token[0] = 0;
        p.info[0] = ok ? 0 : status;
        p.info[1] = ok ? static_cast<int>(all.tokens) : 0;
        p.info[2] = ok ? static_cast<int>(all.take) : 0;
        p.info[3] = static_cast<int>(ok ? top - all.take : count);
    }
    // four tokens a thread: one search, then forward
    const int tokens = ok ? static_cast<int>(all.tokens) : 0;
    for (long long t0 = 4ll * me; t0 < p.max_tokens; t0 += 4ll * threads) {
        long long slot[4] = {-1, -1, -1, -1};
        int pos[4] = {0, 0, 0, 0};
        if (t0 < tokens) {
            int b = owner(first_s, static_cast<int>(t0)), seen_b = -1, seen_blk = -1, phys = -1;  // (four tokens lie in one block or two of a request, most of the time)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int t = static_cast<int>(t0) + e;
                if (t < tokens) {
                    while (first_s[b + 1] <= t) ++b;
                    const int cached = cached_s[b], have = (cached + kPlanBlock - 1) / kPlanBlock;
                    pos[e] = cached + t - first_s[b];
                    const int blk = pos[e] / kPlanBlock;
                    if (b != seen_b || blk != seen_blk) {
                        phys = blk >= have ? taken(take_s[b] + blk - have) : p.table[static_cast<size_t>(b) * p.max_blocks + blk];
                        seen_b = b;
                        seen_blk = blk;
                    }
                    slot[e] = phys < 0 ? -1 : static_cast<long long>(phys) * kPlanBlock + pos[e] % kPlanBlock;
                }
            }
        }
        if (p.vector_stores && t0 + 4 <= p.max_tokens) {
            reinterpret_cast<longlong2*>(p.slots + t0)[0] = make_longlong2(slot[0], slot[1]);
            reinterpret_cast<longlong2*>(p.slots + t0)[1] = make_longlong2(slot[2], slot[3]);
            *reinterpret_cast<int4*>(p.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
        } else {
            for (int e = 0; e < 4 && t0 + e < p.max_tokens; ++e) {
                p.slots[t0 + e] = slot[e];
                p.positions[t0 + e] = pos[e];
            }
        }
    }
    // what may be an input too: when every CTA has read it
    if (p.ticket) {
        __syncthreads();
        if (tid == 0) {
            int before;
            asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(before) : "l"(p.ticket) : "memory");
            last_s = before == parts - 1;
            if (last_s) *p.ticket = 0;
        }
        __syncthreads();
        if (!last_s) return;
    } else if (part > 0) {
        return;
    }
    for (int b = tid; b < p.batch; b += THREADS) {
        const int cached = cached_s[b], was = cached < 0 ? -1 - cached : cached;
        p.seq_lens[b] = !ok ? was : cached < 0 ? 0 : cached + first_s[b + 1] - first_s[b];
    }
    if (tid == 0) *p.free_count_out = static_cast<int>(ok ? top - all.take : count);
}

SmemAttribute plan_attribute[2];
constexpr int kPlanSmem = (4 * kPlanMaxBatch + 1) * 4;

}  // namespace

int plan_max_batch() { return kPlanMaxBatch; }

int launch_plan_blocks(const int* cached, const int* fresh, int batch, int* table, int max_blocks, int* free_blocks, int capacity,
                       const int* free_count, int* free_count_out, long long* slots, int* positions, int* seq_lens, int* first_token,
                       int max_tokens, int* info, int* ticket, cudaStream_t stream) {
    PlanParams p = {cached, fresh, batch, table, max_blocks, free_blocks, capacity, free_count, free_count_out, slots, positions,
                    seq_lens, first_token, max_tokens, info,
                    ((reinterpret_cast<uintptr_t>(slots) | reinterpret_cast<uintptr_t>(positions)) & 15u) == 0, ticket};
    const int want = (max_tokens + 4 * kPlanThreads - 1) / (4 * kPlanThreads), sms = device_sms(), parts = want < 1 ? 1 : want < sms ? want : sms;
    if (parts == 1 || (seq_lens != cached && free_count_out != free_count)) p.ticket = nullptr;
    const bool few = batch <= kPlanFew && max_tokens <= 4 * kPlanFew;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(parts, 1, 1);
    cfg.blockDim = dim3(few ? kPlanFew : kPlanThreads, 1, 1);
    cfg.dynamicSmemBytes = (4 * batch + 1) * 4;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled(kPdlRow) ? 1 : 0;
    const cudaError_t e = few ? launch_with_smem(plan_attribute[0], kPlanSmem, cfg, plan_blocks_kernel<kPlanFew>, p)
                              : launch_with_smem(plan_attribute[1], kPlanSmem, cfg, plan_blocks_kernel<kPlanThreads>, p);
    if (e != cudaSuccess) return fail(W8A8_ERR_CUDA, "plan_blocks launch: %s", cudaGetErrorString(e));
    return W8A8_OK;
}

}  // namespace w8a8
