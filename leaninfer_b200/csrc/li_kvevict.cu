// Eviction from a KV cache by accumulated attention weight.
//
// For each (sequence, kv head) with more than `budget` slots in use: keep the
// `budget` slots with the largest key, where the key is the weight's bit
// pattern (non-negative floats order as unsigned integers; negative and NaN
// count as 0) and 0xFFFFFFFF for the protected ones (n_sink first and n_recent
// newest positions), ties going to the lowest slot; then fill the freed slots
// below `budget`, ascending, with the kept ones behind it, ascending. Only
// those rows move: sources lie at or past `budget`, destinations below it, so
// all moves are independent and need no order.
//
//   kv_select   block per (sequence, kv head): the budget-th largest key by a
//               radix search over digits of 11, 11 and 10 bits, the two
//               ascending lists from a bit mask of the kept slots, and the first
//               kSelMoves moves themselves: 512 bytes (K and V row) each, plus
//               weight and position, eight a warp in flight. That is all there
//               is where a cache overshoots its budget by a little, as it does
//               in use;
//   kv_move     the moves beyond those, warps over all lists, and the lengths
//               (which every block of kv_select reads).
#include "li_kv.cuh"

LI_DEFINE_TU_STATUS(kvevict)

namespace li {
namespace {

constexpr int kSelCacheMax = 48 * 1024;     // keys held in shared memory up to this many slots
// From this many slots on, blocks of 1024 threads, below of 512, two an SM. Us with 512 and with 1024, caches cold: 1
// sequence x 8 heads 16 and 17 at 4352 slots, 24 and 17 at 8192; 2 x 8 at 18000 45 and 33; 64 x 8 at 4352 slots 29
// and 47 (3.5 blocks an SM), at 8192 48 and 48.
constexpr int kSelWide = 8192;
constexpr int kSelMoves = 256;              // moves that kv_select makes itself
constexpr int kBins = 2048;                 // of a digit
constexpr int kMovePer = 8;                 // moves of a warp in flight

struct EvictArgs {
    const float *weight;
    const int32_t *slot_pos, *pos;
    int32_t *len;
    int Hkv, max_ctx, budget, n_recent, max_moves;
    int64_t first_free;                // positions below are protected: the prefix's and the sinks'
    int32_t *count;                    // [n_seqs * Hkv] moves
    int2 *list;                        // [n_seqs * Hkv][max_moves] (from, to)
    uint32_t *masks;                   // [n_seqs * Hkv][mask_words]: kept slots, where shared memory is short
    int mask_words;                    // ceil(max_ctx / 32)
    __half *k, *v;
    float *weight_rw;
    int32_t *slot_pos_rw;
    int n_pairs;
};

__device__ __forceinline__ uint32_t evict_key(float w, int p, int64_t first_free, int64_t newest_free) {
    if (p < first_free || (int64_t)p > newest_free) return 0xffffffffu;
    return w > 0.f ? __float_as_uint(w) : 0u;
}

// Exclusive scan of v over the block's warps (one value per warp, given by
// every lane); returns this warp's offset and the total.
template <int W>
__device__ __forceinline__ int warp_offsets(int v, int *buf, int &total) {
    const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
    __syncthreads();
    if (lane == 0) buf[warp] = v;
    __syncthreads();
    int incl = lane < W ? buf[lane] : 0;
#pragma unroll
    for (int o = 1; o < W; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
    }
    total = __shfl_sync(0xffffffffu, incl, W - 1);
    const int before = __shfl_sync(0xffffffffu, incl, warp ? warp - 1 : 0);
    return warp ? before : 0;
}

// Rows m, m + stride, ... of a pair's moves: lanes 0-15 carry the K row, 16-31
// the V row, 16 bytes each; the loads of kMovePer rows go out together.
template <typename List>
__device__ __forceinline__ void move_rows(const EvictArgs &a, int pair, List move, int m, int n, int stride, int lane) {
    const int s = pair / a.Hkv, j = pair - s * a.Hkv;
    __half *base = (lane < 16 ? a.k : a.v) + ((size_t)s * a.max_ctx * a.Hkv + j) * kKvD + (lane & 15) * 8;
    const size_t row = (size_t)a.Hkv * kKvD;
    for (; m < n; m += kMovePer * stride) {
        uint4 d[kMovePer];
#pragma unroll
        for (int i = 0; i < kMovePer; ++i)
            if (m + i * stride < n) d[i] = *reinterpret_cast<const uint4 *>(base + (size_t)move(m + i * stride).x * row);
#pragma unroll
        for (int i = 0; i < kMovePer; ++i)
            if (m + i * stride < n) *reinterpret_cast<uint4 *>(base + (size_t)move(m + i * stride).y * row) = d[i];
    }
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) kv_select_kernel(EvictArgs a, bool cached) {
    constexpr int W = THREADS / kWarp, kPer = kBins / THREADS;
    extern __shared__ uint32_t keys[];             // cached: [max_ctx] keys, [mask_words] kept slots
    __shared__ int hist[kBins];
    __shared__ int buf[W];
    __shared__ int s_digit, s_want, s_all;
    __shared__ int2 mine[kSelMoves];
    grid_dep_wait();
    grid_dep_launch_dependents();
    const int pair = blockIdx.x, s = pair / a.Hkv;
    const int tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp;
    const int n = a.len[s], newest = a.pos[s];
    if (n < 0 || n > a.max_ctx) {
        if (tid == 0) {
            atomicExch(&g_device_error, LI_ERR_BAD_ARG);
            a.count[pair] = 0;
        }
        return;
    }
    if (n <= a.budget || a.budget == 0) {          // nothing to free, or nothing to keep: no rows move
        if (tid == 0) a.count[pair] = 0;
        return;
    }
    const float *w = a.weight + (size_t)pair * a.max_ctx;
    const int32_t *sp = a.slot_pos + (size_t)pair * a.max_ctx;
    const int64_t newest_free = (int64_t)newest - a.n_recent;
    auto key_of = [&](int i) -> uint32_t {
        return cached ? keys[i] : evict_key(w[i], sp[i], a.first_free, newest_free);
    };
    uint32_t *masks = cached ? keys + a.max_ctx : a.masks + (size_t)pair * a.mask_words;
    // the budget-th largest key, digit by digit from the top: `prefix` holds
    // the digits found, `want` the rank left among the keys that share them
    uint32_t prefix = 0, mask = 0;
    int want = a.budget;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const uint32_t digits = pass == 2 ? 1023u : 2047u;
        for (int i = tid; i < kBins; i += THREADS) hist[i] = 0;
        __syncthreads();
        if (pass == 0) {
#pragma unroll 8
            for (int i = tid; i < n; i += THREADS) {
                const uint32_t k = evict_key(w[i], sp[i], a.first_free, newest_free);
                if (cached) keys[i] = k;
                atomicAdd(&hist[k >> shift], 1);
            }
        } else {
            for (int i = tid; i < n; i += THREADS) {
                const uint32_t k = key_of(i);
                if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & digits], 1);
            }
        }
        __syncthreads();
        // thread t holds kPer bins, counted from the top; the digit is the bin where the running count reaches want
        int c[kPer], sum = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) sum += c[i] = hist[kBins - 1 - (tid * kPer + i)];
        int incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += x;
        }
        int total, before = warp_offsets<W>(__shfl_sync(0xffffffffu, incl, 31), buf, total) + incl - sum;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            if (before < want && before + c[i] >= want) {
                s_digit = kBins - 1 - (tid * kPer + i);
                s_want = want - before;
                s_all = c[i];
            }
            before += c[i];
        }
        __syncthreads();
        prefix |= ((uint32_t)s_digit & digits) << shift;
        mask |= digits << shift;
        want = s_want;
        const bool whole = s_all == want;          // all keys with these digits are kept: the others do not matter
        __syncthreads();
        if (whole) break;
    }
    // keys above `prefix` are kept, of those equal to it the first `want` (all
    // of them, unless weights are tied at the border): a bit per slot. A warp
    // owns whole groups of 32 slots, in order.
    const int groups = (n + 31) / 32, per = (groups + W - 1) / W;
    const int g0 = min(warp * per, groups), g1 = min(g0 + per, groups);
    const bool tied = s_all > want;
    int total, tie = 0;
    if (tied) {
        int ties = 0;
        for (int g = g0; g < g1; ++g) {
            const int i = g * 32 + lane;
            ties += __popc(__ballot_sync(0xffffffffu, i < n && key_of(i) == prefix));
        }
        tie = warp_offsets<W>(ties, buf, total);
    }
    for (int g = g0; g < g1; ++g) {
        const int i = g * 32 + lane;
        const uint32_t k = i < n ? key_of(i) : 0u;
        bool keep = i < n && (tied ? k > prefix : k >= prefix);
        if (tied) {
            const bool eq = i < n && k == prefix;
            const uint32_t eqs = __ballot_sync(0xffffffffu, eq);
            keep = keep || (eq && tie + __popc(eqs & ((1u << lane) - 1u)) < want);
            tie += __popc(eqs);
        }
        const uint32_t kept = __ballot_sync(0xffffffffu, keep);
        if (lane == 0) masks[g] = kept;
    }
    __syncthreads();
    // the lists, a run of groups per thread: freed slots below budget and kept ones behind it are few bits of a mask
    const int run = (groups + THREADS - 1) / THREADS, r0 = min(tid * run, groups), r1 = min(r0 + run, groups);
    auto bits = [&](int g, uint32_t &hole, uint32_t &from) {
        const uint32_t m = masks[g];
        const int left = a.budget - 32 * g;            // slots of the group below budget (budget < n)
        const uint32_t below = left <= 0 ? 0u : left >= 32 ? 0xffffffffu : (1u << left) - 1u;
        hole = ~m & below;
        from = m & ~below;
    };
    int holes = 0, froms = 0;
    for (int g = r0; g < r1; ++g) {
        uint32_t h, f;
        bits(g, h, f);
        holes += __popc(h);
        froms += __popc(f);
    }
    int hi = holes, fi = froms;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, hi, o), y = __shfl_up_sync(0xffffffffu, fi, o);
        if (lane >= o) { hi += x; fi += y; }
    }
    int moves;
    int at_h = warp_offsets<W>(__shfl_sync(0xffffffffu, hi, 31), buf, moves) + hi - holes;
    int at_f = warp_offsets<W>(__shfl_sync(0xffffffffu, fi, 31), buf, moves) + fi - froms;    // as many as freed slots
    int2 *list = a.list + (size_t)pair * a.max_moves;
    for (int g = r0; g < r1; ++g) {
        uint32_t h, f;
        bits(g, h, f);
        for (; h; h &= h - 1, ++at_h) (at_h < kSelMoves ? mine[at_h] : list[at_h]).y = 32 * g + __ffs(h) - 1;
        for (; f; f &= f - 1, ++at_f) (at_f < kSelMoves ? mine[at_f] : list[at_f]).x = 32 * g + __ffs(f) - 1;
    }
    if (tid == 0) a.count[pair] = moves;
    __syncthreads();
    const int here = min(moves, kSelMoves);
    static_assert(kSelMoves <= THREADS, "a move's weight and position a thread");
    float wv = 0.f;
    int32_t pv = 0;
    if (tid < here) {                              // on their way while the rows move
        wv = w[mine[tid].x];
        pv = sp[mine[tid].x];
    }
    move_rows(a, pair, [&](int m) { return mine[m]; }, warp, here, W, lane);
    if (tid < here) {
        const size_t at = (size_t)pair * a.max_ctx + mine[tid].y;
        a.weight_rw[at] = wv;
        a.slot_pos_rw[at] = pv;
    }
}

constexpr int kMoveWarps = 8;
constexpr int kMoveChunk = kMoveWarps * kMovePer;  // moves per block and step

__global__ void __launch_bounds__(kMoveWarps * kWarp) kv_move_kernel(EvictArgs a, int chunks) {
    grid_dep_wait();
    grid_dep_launch_dependents();
    const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
    for (int s = blockIdx.x * kMoveWarps * kWarp + threadIdx.x; s < a.n_pairs / a.Hkv; s += gridDim.x * kMoveWarps * kWarp)
        if (a.len[s] > a.budget && a.len[s] <= a.max_ctx) a.len[s] = a.budget;
    const int64_t items = (int64_t)a.n_pairs * chunks;
    for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
        const int pair = (int)(it / chunks), chunk = (int)(it % chunks);
        const int n = a.count[pair], m0 = kSelMoves + chunk * kMoveChunk;
        if (m0 >= n) continue;
        const int2 *list = a.list + (size_t)pair * a.max_moves;
        const int end = min(n, m0 + kMoveChunk);
        move_rows(a, pair, [&](int m) { return list[m]; }, m0 + warp, end, kMoveWarps, lane);
        const int m = m0 + threadIdx.x;
        if (m < end) {
            const size_t at = (size_t)pair * a.max_ctx;
            a.weight_rw[at + list[m].y] = a.weight_rw[at + list[m].x];
            a.slot_pos_rw[at + list[m].y] = a.slot_pos_rw[at + list[m].x];
        }
    }
}

size_t al256(size_t v) { return (v + 255) / 256 * 256; }

template <int THREADS>
int launch_select(const EvictArgs &a, bool cached, size_t smem, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    if (const int rc = allow_smem(kv_select_kernel<THREADS>, (kSelCacheMax + kSelCacheMax / 32) * 4, done)) return rc;
    return (int)launch_pdl(kv_select_kernel<THREADS>, dim3((unsigned)a.n_pairs), dim3(THREADS), smem, s, true, a, cached);
}

int moves_max(const li_kv_cache *C, int budget) {
    return budget < C->max_ctx - budget ? budget : C->max_ctx - budget;
}

}  // namespace
}  // namespace li

using namespace li;

extern "C" {

size_t li_kv_evict_workspace_size(const li_kv_cache *C, int budget) {
    if (check_kv_cache(C) || C->n_seqs == 0 || budget < 0 || budget > C->max_ctx) return 0;
    const size_t pairs = (size_t)C->n_seqs * C->n_kv_heads;
    return al256(pairs * sizeof(int32_t)) + al256(pairs * (size_t)moves_max(C, budget) * sizeof(int2)) +
           (C->max_ctx > kSelCacheMax ? al256(pairs * (((size_t)C->max_ctx + 31) / 32) * 4) : 0);
}

int li_launch_kv_evict(const li_kv_cache *C, const int32_t *pos, int budget, int n_sink, int n_recent,
                       void *workspace, size_t workspace_bytes, void *stream) {
    if (const int rc = check_kv_cache(C)) return rc;
    if (!pos || !C->weight || !C->slot_pos || budget < 0 || n_sink < 0 || n_recent < 0) return LI_ERR_BAD_ARG;
    if (budget > C->max_ctx || (int64_t)n_sink + n_recent > budget) return LI_ERR_BAD_SHAPE;
    if ((uintptr_t)pos & 3u) return LI_ERR_MISALIGNED;
    if (C->n_seqs == 0) return 0;
    if (!workspace || workspace_bytes < li_kv_evict_workspace_size(C, budget)) return LI_ERR_WORKSPACE;
    if (!aligned16(workspace)) return LI_ERR_MISALIGNED;
    EvictArgs a = {};
    const int pairs = C->n_seqs * C->n_kv_heads;
    a.weight = C->weight; a.slot_pos = C->slot_pos; a.pos = pos; a.len = C->len;
    a.Hkv = C->n_kv_heads; a.max_ctx = C->max_ctx; a.budget = budget; a.first_free = (int64_t)C->n_prefix + n_sink; a.n_recent = n_recent;
    a.max_moves = moves_max(C, budget);
    a.count = static_cast<int32_t *>(workspace);
    char *ws = static_cast<char *>(workspace) + al256((size_t)pairs * sizeof(int32_t));
    a.list = reinterpret_cast<int2 *>(ws);
    a.masks = reinterpret_cast<uint32_t *>(ws + al256((size_t)pairs * (size_t)a.max_moves * sizeof(int2)));
    a.mask_words = (C->max_ctx + 31) / 32;
    a.k = static_cast<__half *>(C->k); a.v = static_cast<__half *>(C->v);
    a.weight_rw = C->weight; a.slot_pos_rw = C->slot_pos;
    a.n_pairs = pairs;
    const cudaStream_t st = (cudaStream_t)stream;
    const bool cached = C->max_ctx <= kSelCacheMax;
    const size_t smem = cached ? ((size_t)C->max_ctx + a.mask_words) * 4 : 0;
    int rc = C->max_ctx < kSelWide ? launch_select<512>(a, cached, smem, st) : launch_select<1024>(a, cached, smem, st);
    if (rc) return rc;
    const int chunks = a.max_moves > kSelMoves ? (a.max_moves - kSelMoves + kMoveChunk - 1) / kMoveChunk : 0;
    const int64_t items = (int64_t)pairs * chunks, cap = (int64_t)num_sms() * 8;
    const int64_t lens = (C->n_seqs + kMoveWarps * kWarp - 1) / (kMoveWarps * kWarp);
    const int64_t grid = items > lens ? items : lens;
    return (int)launch_pdl(kv_move_kernel, dim3((unsigned)(grid < cap ? grid : cap)), dim3(kMoveWarps * kWarp), 0,
                           st, true, a, chunks);
}

}  // extern "C"
