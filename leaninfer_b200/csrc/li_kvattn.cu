// Attention of one token per sequence over a shared prefix and the
// sequence's own cache slots, with the accumulation of each own slot's
// attention weight.
//
//   o[s][h] = softmax_t(scale q[s][h] . K_t) V_t,  t over prefix and own slots
//   weight[s][j][t] = decay weight + sum_g p[s][jG+g][t]      (own slots)
//
// Both parts are cut along the tokens into pieces that fill the SMs evenly;
// a piece leaves (max, sum, o[128]) per q head, and the last kernel joins
// them. Every product takes q and p as two f16 parts (hi + lo: 22 bits), since
// K and V are f16 already: twice the tensor work of one part, for outputs that
// are as exact as fp32 sums (one part would leave 2^-12). Probabilities carry
// a factor 2^7, so that the lo part of a probability far below the largest is
// still a normal f16, and the running maximum is only raised when a score
// passes it by 2^8 (the factors cancel in o and sum alike; 2^15 fits f16).
// Rows of q are scaled by a power of two into [1, 2) first: any fp32 magnitude
// fits the f16 parts.
//
//   kv_prefix   tcgen05: the batch's q heads of one kv head are the rows of a
//               [seqs * G, 128] x [128, prefix] product. Two softmax
//               warpgroups work on two score tiles (128 rows x 128 tokens), so
//               that one's exponentials run under the other's products: two
//               row tiles that share each K / V tile, or, where one row tile
//               is all there is, alternate token tiles. P stays in tensor
//               memory (the A operand of P V, written over the scores).
//               Bound by the tensor cores from about 256 rows a kv head, by
//               HBM below.
//   kv_own      a warp per piece: 16 tokens at a time through a private ring of
//               cp.async stages, mma.sync m16n8k16 with the up to 8 q heads of
//               a kv head as rows 0-7 (hi) and 8-15 (lo). Bound by HBM: the
//               products of a step are 32 instructions for 8 KB, so what counts
//               is that warps run on their own (no block barrier per tile, any
//               length costs what it has), not the rate of the tensor pipe.
//   kv_join     joins the pieces of every (sequence, q head) and turns the
//               scores that kv_own kept into weights.
#include "li_kv.cuh"
#include "li_tc.cuh"

#include <cuda.h>   // CUtensorMap and its enums; the encoder is fetched at run time

#include <cstring>
#include <mutex>

LI_DEFINE_TU_STATUS(kvattn)

namespace li {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kPShift = 7.f;                 // probabilities carry 2^7
constexpr float kMaxLag = 8.f;                 // the running maximum may lag by 2^8

// ---- own part: pieces ------------------------------------------------------
constexpr int kOwnTok = 16;                    // tokens per step
constexpr int kOwnWarps = 8, kOwnThreads = kOwnWarps * kWarp;
constexpr int kOwnStages = 3;
constexpr int kOwnStageBytes = 2 * kOwnTok * kKvD * 2;      // K and V rows of a step: 8 KB
constexpr size_t kOwnSmem = (size_t)kOwnWarps * kOwnStages * kOwnStageBytes;   // 192 KB
constexpr int kOwnFlush = 16;                  // steps summed by mma before they join the record
constexpr int kOwnMinSteps = 2;                // steps a warp takes at least, where there are enough
constexpr int kScanMax = 2048;                 // entries of the length scan in shared memory

// ---- prefix part -----------------------------------------------------------
constexpr int kPreRows = 128, kPreTok = 128;
constexpr int kPreThreads = 512;               // warps 0-3, 4-7: softmax; 8: TMA; 9, 10: MMA; 12-15: records
constexpr uint32_t kPreSlotBytes = kPreTok * kKvD * 2;      // 128 tokens of K or V: 32 KB
constexpr uint32_t kPreQBytes = 2 * kPreRows * kKvD * 2;    // a row tile's hi and lo: 64 KB
constexpr int kPreSlots2 = 3, kPreSlots1 = 5;  // ring slots beside two / one row tiles of q
constexpr int kPreFlush = 4;                   // token tiles summed in tensor memory before they join the record
constexpr size_t kPreSmem = 1024 + 2 * kPreQBytes + kPreSlots2 * kPreSlotBytes + 256 + 3 * kPreRows * 4;
static_assert(kPreSmem <= 227 * 1024, "shared memory");
static_assert(2 * kPreQBytes + kPreSlots2 * kPreSlotBytes == kPreQBytes + kPreSlots1 * kPreSlotBytes, "ring");

struct KvAttnArgs {
    const float *q;
    int64_t q_stride;
    const __half *k, *v;
    const int32_t *len;
    int B, Hq, Hkv, G, max_ctx;
    float cscale;                      // |scale| log2(e)
    float qsign;                       // sign of scale, applied to q
    float decay;
    float *out, *weight;
    const float *gate;                 // sigmoid(gate) times the output, or nullptr
    int64_t gate_stride;
    // own part
    int own_warps;                     // warps of the kv_own grid
    int *base;                         // [B + 1] first step of every sequence (all kv heads), then the total
    float2 *own_ml;                    // [pairs + own_warps][G]
    float *own_o;                      // [pairs + own_warps][G][128]
    float *score;                      // [B][Hq][score_stride], log2 units (weight != nullptr)
    int score_stride;                  // max_ctx rounded up to 4
    bool after_prefix;
    int lead;                          // prefix tokens that kv_own takes as every sequence's first (else 0)
    const __half *kp, *vp;
    // prefix part
    int n_prefix, rows, n_rt, per_group, n_grp, n_tt;   // rows = B G; row tiles; row tiles per group; groups; tiles
    int pre_ctas, slots;
    float2 *pre_ml;                    // [Hkv n_grp + pre_ctas][2][128 rows]
    float *pre_o;                      // [Hkv n_grp + pre_ctas][2][32 groups of 4 dims][128 rows][4]
    // join
    int row_ctas, wpr, w_chunks;       // blocks that join rows, warps per row block, blocks per pair that write weights
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ int own_len(const KvAttnArgs &a, int s) {
    const int n = __ldcg(a.len + s);
    return n < 0 || n > a.max_ctx ? 0 : n;
}

// Tokens of sequence s that kv_own works on.
__device__ __forceinline__ int own_tokens(const KvAttnArgs &a, int s) { return own_len(a, s) + a.lead; }

__device__ __forceinline__ int own_steps(int n) { return (n + kOwnTok - 1) / kOwnTok; }

// Power of two 2^e with |x| / 2^e in [1, 2) (1 for infinities and NaN). The
// exponent stays within -126 .. 126, where 2^-e is a normal float too: below
// it |x| / 2^e is less than 1, above it in [2, 4), which fits f16 as well.
__device__ __forceinline__ float pow2_of(float x) {
    const uint32_t e = (__float_as_uint(x) >> 23) & 255u;
    return e == 255u ? 1.f : __uint_as_float(min(max(e, 1u), 253u) << 23);
}

__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// hi keeps the top 11 bits of x (exact in f16), lo the rest.
__device__ __forceinline__ float hi_part(float x) { return __uint_as_float(__float_as_uint(x) & 0xffffe000u); }

// 1 / 2^e of a power that pow2_of gave: exact.
__device__ __forceinline__ float inv_pow2(float p) { return __uint_as_float((254u << 23) - __float_as_uint(p)); }

// ---------------------------------------------------------------------------
// A line of T units dealt to W takers in runs whose lengths differ by at most
// one: the first T % W takers have T / W + 1.
// ---------------------------------------------------------------------------
struct Runs {
    int len, extra;
    __device__ __forceinline__ Runs(int T, int W) : len(T / W), extra(T % W) {}
    __device__ __forceinline__ int begin(int w) const { return w * len + min(w, extra); }
    __device__ __forceinline__ int taker(int unit) const {          // of a unit on the line
        const int cut = extra * (len + 1);
        return unit < cut ? unit / (len + 1) : extra + (unit - cut) / len;
    }
};

// Pieces of the own part: the steps of all (sequence, kv head) pairs in order,
// T of them, are dealt to W warps. The piece of pair p that warp w holds is
// record p + w: along the line of steps either p or w grows from piece to
// piece, so no two share a record.
__device__ __forceinline__ int own_active(int T, int warps) {
    const int w = T / kOwnMinSteps;
    return w < 1 ? 1 : w < warps ? w : warps;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// NG groups of 8 q heads. In a warp, lane l holds q head l / 4 of each group
// (scores of tokens 2 (l % 4), +1 of each 8; dims 2 (l % 4), +1 of each 8).
template <int NG, bool SCORE, bool LEAD>
__global__ void __launch_bounds__(kOwnThreads, 1) kv_own_kernel(const __grid_constant__ KvAttnArgs a) {
    extern __shared__ __align__(128) uint8_t own_smem[];
    __shared__ int cum[kScanMax], wsum[kOwnWarps];
    const int tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp;
    // behind a prefix kernel, this one starts when that one has passed its own
    // wait: everything either reads is in place; only the join needs both
    if (!a.after_prefix) {
        grid_dep_wait();
        grid_dep_launch_dependents();
    }
    // Lengths: `per` neighbouring sequences an entry, a running sum of their steps.
    const int per = (a.B + kScanMax - 1) / kScanMax, entries = (a.B + per - 1) / per;
    int T = 0;
    for (int e0 = 0; e0 < entries; e0 += kOwnThreads) {
        const int e = e0 + tid;
        int mine = 0;
        for (int i = 0; i < per; ++i) {
            const int s = e * per + i;
            if (e < entries && s < a.B) {
                const int n = __ldcg(a.len + s);
                const bool bad = n < 0 || n > a.max_ctx;
                if (bad && blockIdx.x == 0) atomicExch(&g_device_error, LI_ERR_BAD_ARG);
                mine += own_steps((bad ? 0 : n) + a.lead);
            }
        }
        mine *= a.Hkv;
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += x;
        }
        __syncthreads();
        if (lane == 31) wsum[warp] = incl;
        __syncthreads();
        int off = T, all = 0;
#pragma unroll
        for (int w = 0; w < kOwnWarps; ++w) {
            if (w < warp) off += wsum[w];
            all += wsum[w];
        }
        if (e < entries) {
            cum[e] = off + incl - mine;
            if (blockIdx.x == 0) {
                int at = off + incl - mine;
                for (int i = 0; i < per && e * per + i < a.B; ++i) {
                    a.base[e * per + i] = at;
                    at += own_steps(own_tokens(a, e * per + i)) * a.Hkv;
                }
            }
        }
        T += all;
    }
    if (blockIdx.x == 0 && tid == 0) a.base[a.B] = T;
    __syncthreads();

    const int W = own_active(T, a.own_warps);
    const int w = warp * gridDim.x + blockIdx.x;       // neighbouring pieces on different SMs
    const Runs runs(T, W);
    const int lo = w < W ? runs.begin(w) : 0, hi = w < W ? runs.begin(w + 1) : 0;
    const int n_steps = hi - lo;
    if (n_steps > 0) {
        // a cursor: sequence, kv head, step within the pair, and the sequence's length
        struct Cursor { int s, j, t, n; };
        Cursor ld;
        {
            int e = 0, end = entries;                  // the last entry that starts at or before lo
            while (end - e > 1) {
                const int mid = (e + end) / 2;
                if (cum[mid] <= lo) e = mid; else end = mid;
            }
            int at = cum[e], s = e * per, n = own_tokens(a, s);
            while (at + own_steps(n) * a.Hkv <= lo) {
                at += own_steps(n) * a.Hkv;
                n = own_tokens(a, ++s);
            }
            const int in = lo - at, st = own_steps(n);
            ld.s = s; ld.n = n; ld.j = in / st; ld.t = in - ld.j * st;
        }
        auto next = [&](Cursor &c) {
            if (++c.t < own_steps(c.n)) return;
            c.t = 0;
            if (++c.j < a.Hkv) return;
            c.j = 0;
            do {
                if (++c.s >= a.B) { c.n = 0; return; }
                c.n = own_tokens(a, c.s);
            } while (c.n == 0);
        };
        Cursor cu = ld;
        const uint32_t ring = smem_addr(own_smem) + (uint32_t)warp * kOwnStages * kOwnStageBytes;
        const size_t row = (size_t)a.Hkv * kKvD;
        const int lr = lane >> 4, lc = lane & 15;      // this lane's row (of two) and 16-byte piece in a copy
        auto issue = [&](const Cursor &c, int stage) {
            const int t0 = c.t * kOwnTok, left = c.n - t0;
            const size_t col = (size_t)c.j * kKvD + 8 * lc, seq = (size_t)c.s * a.max_ctx;
            const size_t at = (seq + t0) * row + col;
            const uint32_t dst = ring + (uint32_t)stage * kOwnStageBytes;
#pragma unroll
            for (int i = 0; i < kOwnTok / 2; ++i) {
                const int r = 2 * i + lr;
                const bool ok = r < left;              // past the length: zeros, whatever the slot holds
                const uint32_t d = dst + (uint32_t)(r * 256 + ((lc ^ (r & 7)) << 4));
                if (LEAD) {                            // the prefix, then the sequence's slots
                    const int t = t0 + (ok ? r : 0);
                    const bool pre = t < a.lead;
                    const size_t src = (pre ? (size_t)t : seq + (t - a.lead)) * row + col;
                    cp_async16(d, (pre ? a.kp : a.k) + src, ok);
                    cp_async16(d + kOwnTok * 256, (pre ? a.vp : a.v) + src, ok);
                } else {
                    const size_t src = at + (ok ? (size_t)r * row : 0);
                    cp_async16(d, a.k + src, ok);
                    cp_async16(d + kOwnTok * 256, a.v + src, ok);
                }
            }
        };
#pragma unroll
        for (int i = 0; i < kOwnStages - 1; ++i) {
            if (i < n_steps) {
                issue(ld, i);
                next(ld);
            }
            cp_async_commit();
        }
        uint32_t qf[NG][8][4];
        float o[NG][16][4], m[NG], l[NG], c2[NG], m_rec[NG];
        bool fresh = true;
        int since = 0;                                 // steps in o that are not in the record
        const int g = lane >> 2, tq = lane & 3;
        const int kc = lane >> 3, kr = lane & 7;       // ldmatrix: matrix and row this lane addresses
        int stage = 0, ld_stage = kOwnStages - 1;
        for (int i = 0; i < n_steps; ++i) {
            cp_async_wait<kOwnStages - 2>();
            __syncwarp();                              // this step has landed; the last one's stage is free
            if (i + kOwnStages - 1 < n_steps) {
                issue(ld, ld_stage);
                next(ld);
            }
            cp_async_commit();
            ld_stage = ld_stage + 1 == kOwnStages ? 0 : ld_stage + 1;
            if (fresh) {                               // a new pair: its q heads, scaled and split
#pragma unroll
                for (int e = 0; e < NG; ++e) {
                    const int h = 8 * e + g;
                    const float *qs = a.q + cu.s * a.q_stride + (size_t)(cu.j * a.G + h) * kKvD + 2 * tq;
                    float2 x[16];
                    float mx = 0.f;
#pragma unroll
                    for (int kk = 0; kk < 16; ++kk) {
                        x[kk] = h < a.G ? __ldcg(reinterpret_cast<const float2 *>(qs + 8 * kk)) : make_float2(0.f, 0.f);
                        mx = fmaxf(mx, fmaxf(fabsf(x[kk].x), fabsf(x[kk].y)));
                    }
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    const float p2 = pow2_of(mx), inv = inv_pow2(p2) * a.qsign;
                    c2[e] = a.cscale * p2;
#pragma unroll
                    for (int kk = 0; kk < 16; ++kk) {
                        const float y0 = x[kk].x * inv, y1 = x[kk].y * inv, h0 = hi_part(y0), h1 = hi_part(y1);
                        qf[e][kk >> 1][(kk & 1) * 2] = pack_h2(h0, h1);
                        qf[e][kk >> 1][(kk & 1) * 2 + 1] = pack_h2(y0 - h0, y1 - h1);
                    }
                    m[e] = m_rec[e] = -INFINITY;
                    l[e] = 0.f;
#pragma unroll
                    for (int nt = 0; nt < 16; ++nt)
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[e][nt][r] = 0.f;
                }
                fresh = false;
                since = 0;
            }
            const uint32_t kb = ring + (uint32_t)stage * kOwnStageBytes, vb = kb + kOwnTok * 256;
            stage = stage + 1 == kOwnStages ? 0 : stage + 1;
            // scores of 16 tokens: two 8-token tiles, 128 dims in eight k-steps
            float sc[NG][2][4];
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
#pragma unroll
                for (int e = 0; e < NG; ++e)
#pragma unroll
                    for (int r = 0; r < 4; ++r) sc[e][nt][r] = 0.f;
                const uint32_t tok = kb + (uint32_t)(8 * nt + kr) * 256;
#pragma unroll
                for (int kp = 0; kp < 4; ++kp) {
                    uint32_t b[4];
                    ldsm4(tok + (uint32_t)(((4 * kp + kc) ^ kr) << 4), b);
#pragma unroll
                    for (int e = 0; e < NG; ++e) {
                        mma_f16(sc[e][nt], qf[e][2 * kp], b[0], b[1]);
                        mma_f16(sc[e][nt], qf[e][2 * kp + 1], b[2], b[3]);
                    }
                }
            }
            const int t0 = cu.t * kOwnTok, left = cu.n - t0;
            uint32_t pf[NG][4];
#pragma unroll
            for (int e = 0; e < NG; ++e) {
                float s2[4];
                float mx = -INFINITY;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int nt = x >> 1, r = x & 1, tok = 8 * nt + 2 * tq + r;
                    s2[x] = (sc[e][nt][r] + sc[e][nt][2 + r]) * c2[e];
                    if (SCORE && 8 * e + g < a.G && tok < left && (!LEAD || t0 + tok >= a.lead))
                        a.score[((size_t)cu.s * a.Hq + (size_t)cu.j * a.G + 8 * e + g) * a.score_stride + t0 + tok -
                                (LEAD ? a.lead : 0)] = s2[x];
                    if (tok >= left) s2[x] = -INFINITY;
                    mx = fmaxf(mx, s2[x]);
                }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const bool grow = mx > m[e] + kMaxLag;     // also the first step: m = -inf
                if (__any_sync(0xffffffffu, grow)) {
                    const float f = !grow ? 1.f : m[e] == -INFINITY ? 0.f : ex2(m[e] - mx);
                    if (grow) m[e] = mx;
                    l[e] *= f;
#pragma unroll
                    for (int nt = 0; nt < 16; ++nt)
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[e][nt][r] *= f;
                }
                float p[4], ph[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    p[x] = ex2(s2[x] - m[e] + kPShift);
                    l[e] += p[x];
                    ph[x] = hi_part(p[x]);
                }
                pf[e][0] = pack_h2(ph[0], ph[1]);
                pf[e][1] = pack_h2(p[0] - ph[0], p[1] - ph[1]);
                pf[e][2] = pack_h2(ph[2], ph[3]);
                pf[e][3] = pack_h2(p[2] - ph[2], p[3] - ph[3]);
            }
            // o += P V: 16 tokens, 128 dims in 16 tiles
            const uint32_t vt = vb + (uint32_t)(((kc & 1) * 8 + kr) * 256);
#pragma unroll
            for (int dp = 0; dp < 8; ++dp) {
                uint32_t b[4];
                ldsm4_t(vt + (uint32_t)(((2 * dp + (kc >> 1)) ^ kr) << 4), b);
#pragma unroll
                for (int e = 0; e < NG; ++e) {
                    mma_f16(o[e][2 * dp], pf[e], b[0], b[1]);
                    mma_f16(o[e][2 * dp + 1], pf[e], b[2], b[3]);
                }
            }
            const int ps = cu.s, pj = cu.j;
            next(cu);
            fresh = cu.s != ps || cu.j != pj;
            const bool last = fresh || i + 1 == n_steps;
            if (last || ++since == kOwnFlush) {
                // o joins the record, whose values have the factor 2^(m_rec)
                const size_t rec = (size_t)ps * a.Hkv + pj + w;
                since = 0;
#pragma unroll
                for (int e = 0; e < NG; ++e) {
                    float sum = l[e] + __shfl_xor_sync(0xffffffffu, l[e], 1);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                    const int h = 8 * e + g;
                    if (h < a.G) {
                        if (last && tq == 0) a.own_ml[rec * a.G + h] = make_float2(m[e] - kPShift, sum);
                        float *d = a.own_o + (rec * a.G + h) * kKvD + 2 * tq;
                        const bool again = m_rec[e] != -INFINITY;
                        const float fr = again ? ex2(m_rec[e] - m[e]) : 0.f;
#pragma unroll
                        for (int nt = 0; nt < 16; ++nt) {
                            float2 x = make_float2(o[e][nt][0] + o[e][nt][2], o[e][nt][1] + o[e][nt][3]);
                            if (again) {
                                const float2 old = *reinterpret_cast<const float2 *>(d + 8 * nt);
                                x.x = fmaf(old.x, fr, x.x);
                                x.y = fmaf(old.y, fr, x.y);
                            }
                            *reinterpret_cast<float2 *>(d + 8 * nt) = x;
                        }
                    }
                    m_rec[e] = m[e];
#pragma unroll
                    for (int nt = 0; nt < 16; ++nt)
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[e][nt][r] = 0.f;
                }
            }
        }
        cp_async_wait<0>();
    }
    if (a.after_prefix) {
        grid_dep_launch_dependents();
        grid_dep_wait();       // the join follows both kernels
    }
}

// ---------------------------------------------------------------------------
// Pieces of the prefix part. Row tiles of one kv head go in groups of one or
// two (per_group); a group's token tile costs its number of row tiles. The
// line of all costs (kv heads, then groups) is dealt to the blocks in equal
// runs, a block's boundary rounded up to a whole token tile. The piece of
// group p that block c holds is record p + c, as above.
// ---------------------------------------------------------------------------
struct Group { int j, rt, nt, base; };         // kv head, first row tile, row tiles, place on the line

__device__ __forceinline__ Group group_at(const KvAttnArgs &a, int p) {
    Group g;
    g.j = p / a.n_grp;
    g.rt = (p - g.j * a.n_grp) * a.per_group;
    g.nt = a.n_rt - g.rt < a.per_group ? a.n_rt - g.rt : a.per_group;
    g.base = (g.j * a.n_rt + g.rt) * a.n_tt;
    return g;
}
// token tiles [t0, t1) in the run [lo, hi) of a group at `base` with nt (1 or 2) row tiles
__device__ __forceinline__ void tiles_of(const KvAttnArgs &a, int base, int nt, int lo, int hi, int &t0, int &t1) {
    t0 = lo <= base ? 0 : (lo - base + nt - 1) >> (nt - 1);
    t1 = hi <= base ? 0 : (hi - base + nt - 1) >> (nt - 1);
    if (t1 > a.n_tt) t1 = a.n_tt;
}

__device__ __forceinline__ void tma_load_3d(void *smem_dst, const CUtensorMap *map, int x, int y, int z,
                                            uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(smem_addr(smem_dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(bar))
        : "memory");
}

// A bounded wait that also gives up once another warp has.
__device__ __forceinline__ bool wait_or_abort(uint64_t *bar, uint32_t parity, volatile int *abort_flag) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*abort_flag) return false;
    if (!mbar_wait(bar, parity)) {
        *abort_flag = 1;
        return false;
    }
    return true;
}

// Named barrier 1 over the eight softmax warps, returning whether any passed v.
__device__ __forceinline__ bool softmax_bar_any(bool v) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred pi, po;\n\tsetp.ne.u32 pi, %1, 0;\n\t"
                 "bar.red.or.pred po, 1, 256, pi;\n\tselp.u32 %0, 1, 0, po;\n\t}"
                 : "=r"(r) : "r"((uint32_t)v) : "memory");
    return r != 0;
}

// Order in which the products of a piece of n token tiles are issued, and its
// K and V tiles go through the ring. The units u = 0 .. n nt - 1 are token tile
// u / 2 of row tile u % 2 (nt 2) or token tile u (nt 1), and unit u runs in
// score buffer u % 2: scores of units 0 and 1, then for each u P V of u and the
// scores of u + 2, which take the buffer that P of u leaves. So each buffer's
// softmax runs under the other's products. Tiles, by first use:
//   nt 2: K0 V0 K1 V1 ...;   nt 1: K0 K1 V0 K2 V1 K3 V2 ...
// o leaves tensor memory after unit i of a buffer's own count where this holds
// (and after its last): the two buffers at different times, since both at once
// would fill the SM's way to L2.
__device__ __forceinline__ bool sum_ends(int i, int b) { return (i + b * (kPreFlush / 2)) % kPreFlush == kPreFlush - 1; }

__device__ __forceinline__ int k_place(int t, int nt) { return nt == 2 ? 2 * t : t == 0 ? 0 : 2 * t - 1; }
__device__ __forceinline__ int v_place(int t, int nt, int n) { return nt == 2 ? 2 * t + 1 : t + (t + 2 < n ? t + 2 : n); }

__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float &a, float &b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__global__ void __launch_bounds__(kPreThreads, 1)
kv_prefix_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                 const __grid_constant__ KvAttnArgs a) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    uint8_t *qbuf = smem;                                          // [row tile][hi, lo][2 blocks of 64 dims][128 rows]
    uint8_t *ring = smem + (size_t)a.per_group * kPreQBytes;
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + 2 * kPreQBytes + kPreSlots2 * kPreSlotBytes);
    uint64_t *full = bars, *empty = full + kPreSlots1, *q_full = empty + kPreSlots1, *s_full = q_full + 1,
             *p_full = s_full + 2, *o_full = p_full + 4, *turn = o_full + 2, *fin = turn + 2, *m_full = fin + 2,
             *o_read = m_full + 2;
    uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(o_read + 2);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_holder + 1);
    float *m_of = reinterpret_cast<float *>(bars + 32);            // [buffer][row]: the maximum a sum of P V refers to
    float *c_of = m_of + 2 * kPreRows;                             // [row]: the scores' scale, where both buffers have it
    const int tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp;
    const int slots = a.slots;
    if (tid == 0) {
        for (int i = 0; i < slots; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], a.per_group); }
        mbar_init(q_full, 10);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&m_full[i], 4);
            mbar_init(&o_read[i], 4);
            mbar_init(&s_full[i], 1);
            mbar_init(&o_full[i], 1);
            mbar_init(&turn[i], 1);
            mbar_init(&fin[i], 1);
        }
        for (int i = 0; i < 4; ++i) mbar_init(&p_full[i], 4);      // [buffer][64 tokens]
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == 8) tmem_alloc(tmem_holder, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_holder;                            // scores / P of buffers 0, 1, then o of 0, 1
    grid_dep_wait();
    grid_dep_launch_dependents();

    const int cost = a.Hkv * a.n_rt * a.n_tt, c = blockIdx.x;
    const Runs runs(cost, a.pre_ctas);
    const int lo = runs.begin(c), hi = runs.begin(c + 1);
    int p0;                                                        // the group that lo falls into
    {
        const int per_j = a.n_rt * a.n_tt, j = lo / per_j;
        p0 = j * a.n_grp + (lo - j * per_j) / (a.per_group * a.n_tt);
    }
    const int p_end = a.Hkv * a.n_grp;

    if (warp >= 12) {
        // ---------------- records ----------------
        // The tensor cores' sums round towards zero, so o is taken out of
        // tensor memory every kPreFlush units and added, rounded to nearest, to
        // the record, by warps of its own: only the next sum's first product
        // waits for it, and that comes after its softmax. A row's words belong
        // to one thread. (red.global.add.v4.f32 in place of the load and store
        // was slower by far.)
        const int r = tid - 384;
        const uint32_t lane_base = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + 256u;
        uint32_t po = 0;                                           // phase of o_full and m_full, a bit per buffer
        bool ok = true;
        for (int p = p0; ok && p < p_end; ++p) {
            const Group g = group_at(a, p);
            if (g.base >= hi) break;
            int t0, t1;
            tiles_of(a, g.base, g.nt, lo, hi, t0, t1);
            const int n = t1 - t0, U = n * g.nt;
            float m_rec0 = -INFINITY, m_rec1 = -INFINITY;
            for (int u = 0; ok && u < U; ++u) {
                const int b = u & 1;
                if (u + 2 < U && !sum_ends(u >> 1, b)) continue;
                const bool live = (g.rt + (g.nt == 2 ? b : 0)) * kPreRows + r < a.rows;
                float4 *d = reinterpret_cast<float4 *>(a.pre_o + ((size_t)(p + c) * 2 + b) * kPreRows * kKvD) + r;
                const float m_old = b ? m_rec1 : m_rec0;
                const bool again = live && m_old != -INFINITY;
                float4 old[2][8];                                  // the record's values, a round ahead
                auto fetch = [&](float4 (&o)[8], int x) {
#pragma unroll
                    for (int y = 0; y < 8; ++y)
                        o[y] = again ? __ldcg(d + (8 * x + y) * kPreRows) : make_float4(0.f, 0.f, 0.f, 0.f);
                };
                fetch(old[0], 0);
                ok = __all_sync(0xffffffffu, wait_or_abort(&o_full[b], (po >> b) & 1u, abort_flag) &&
                                                 wait_or_abort(&m_full[b], (po >> b) & 1u, abort_flag));
                if (!ok) break;
                po ^= 1u << b;
                tc_fence_after();
                const float m = m_of[b * kPreRows + r], f = again ? ex2(m_old - m) : 0.f;
                (b ? m_rec1 : m_rec0) = m;
#pragma unroll 1
                for (int x0 = 0; x0 < 4; x0 += 2)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int x = x0 + e;
                        uint32_t v[32];
                        tmem_ld32_nowait(lane_base + 128u * b + 32u * x, v);
                        if (x < 3) fetch(old[e ^ 1], x + 1);
                        tmem_wait_ld();
                        if (x == 3) {                              // o may be overwritten
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(&o_read[b]);
                        }
                        if (live)
#pragma unroll
                            for (int y = 0; y < 8; ++y) {
                                const float4 w = old[e][y];
                                __stcg(d + (8 * x + y) * kPreRows,
                                       make_float4(fmaf(w.x, f, __uint_as_float(v[4 * y])),
                                                   fmaf(w.y, f, __uint_as_float(v[4 * y + 1])),
                                                   fmaf(w.z, f, __uint_as_float(v[4 * y + 2])),
                                                   fmaf(w.w, f, __uint_as_float(v[4 * y + 3]))));
                            }
                    }
            }
        }
    } else if (warp >= 8) {
        if (warp == 8 && lane == 0) {
            // ---------------- producer ----------------
            asm volatile("prefetch.tensormap [%0];" ::"l"(&tmK) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&tmV) : "memory");
            int slot = 0, used = 0;
            uint32_t par = 1;                                      // of the slot's previous release
            bool ok = true;
            for (int p = p0; ok && p < p_end; ++p) {
                const Group g = group_at(a, p);
                if (g.base >= hi) break;
                int t0, t1;
                tiles_of(a, g.base, g.nt, lo, hi, t0, t1);
                const int n = t1 - t0;
                auto load = [&](const CUtensorMap *map, int t) {
                    if (used >= slots && !(ok = ok && wait_or_abort(&empty[slot], par, abort_flag))) return;
                    mbar_arrive_expect_tx(&full[slot], kPreSlotBytes);
                    uint8_t *dst = ring + (size_t)slot * kPreSlotBytes;
                    const int z = (t0 + t) * kPreTok;
                    tma_load_3d(dst, map, 0, g.j, z, &full[slot]);
                    tma_load_3d(dst + kPreSlotBytes / 2, map, 64, g.j, z, &full[slot]);
                    ++used;
                    if (++slot == slots) { slot = 0; par ^= 1u; }
                };
                for (int t = 0; ok && t < n; ++t) {
                    if (g.nt == 2 || t == 0) load(&tmK, t);
                    if (g.nt == 1 && t + 1 < n) load(&tmK, t + 1);
                    load(&tmV, t);
                }
            }
            // every copy issued has landed before the block ends
            for (int k = used < slots ? 0 : used - slots; k < used; ++k)
                mbar_wait(&full[k % slots], (uint32_t)((k / slots) & 1));
        } else if ((warp == 9 || warp == 10) && lane == 0) {
            // ---------------- MMA issuer of buffer b ----------------
            // The thread stands still while an MMA is taken, so what it does
            // between them adds to the tensor pipe's time: descriptors advance
            // by constants, and the two issuers take turns, a batch (P V of a
            // unit, scores of the next) each, one's waits and commits running
            // under the other's products. Without turns the two batches would
            // mix, end together, and leave the tensor pipe idle while both
            // buffers' softmax runs.
            const int b = warp - 9;
            const uint32_t id_s = idesc_kf16(128, kPreTok, false);
            const uint32_t id_o = idesc_kf16(128, kKvD, false) | kIdescBMajorMN;
            const uint64_t k0 = sw128_desc(smem_addr(ring)), v0 = sw128_mn_desc(smem_addr(ring), kPreSlotBytes / 2);
            const uint32_t ts = tmem + 128u * b, to = tmem + 256u + 128u * b;
            struct Place { int slot; uint32_t par; };              // a ring place's slot and the phase of its copy
            auto advance = [&](Place &x, int by) {
                x.slot += by;
                while (x.slot >= slots) { x.slot -= slots; x.par ^= 1u; }
            };
            int place0 = 0;                                        // ring places before this piece
            uint32_t pq = 0, pp = 0, pt = 0, pr = 1;               // phases of q_full, p_full, turn, o_read (before)
            bool ok = true, have = b == 0;
            auto acquire = [&]() -> bool {
                if (!have && !wait_or_abort(&turn[b], pt, abort_flag)) return false;
                if (!have) pt ^= 1u;
                return have = true;
            };
            auto pass = [&]() {
                mbar_arrive(&turn[b ^ 1]);
                have = false;
            };
            for (int p = p0; ok && p < p_end; ++p) {
                const Group g = group_at(a, p);
                if (g.base >= hi) break;
                int t0, t1;
                tiles_of(a, g.base, g.nt, lo, hi, t0, t1);
                const int n = t1 - t0, U = n * g.nt;
                if (n <= 0) continue;
                mbar_arrive(q_full);                               // q_full counts the issuers too: none falls behind
                if (!(ok = wait_or_abort(q_full, pq, abort_flag))) break;
                pq ^= 1u;
                const uint64_t qd = sw128_desc(smem_addr(qbuf) + (g.nt == 2 ? (uint32_t)b * kPreQBytes : 0u));
                auto place = [&](int at) { return Place{at % slots, (uint32_t)((at / slots) & 1)}; };
                const int tb = g.nt == 2 ? 0 : b;                  // this buffer's first tile
                Place kp = place(place0 + k_place(tb, g.nt)), vp = place(place0 + v_place(tb, g.nt, n));
                place0 += 2 * n;
                if (b >= U) continue;                              // one unit: nothing for buffer 1
                auto release = [&](int slot) {
                    umma_commit(&empty[slot]);
                    if (g.nt < a.per_group) umma_commit(&empty[slot]);     // for the buffer that does not use it
                };
                // scores of unit u; lo first, so that only the hi products add to a sum of full size (the tensor
                // cores' sums round towards zero, once per instruction)
                auto scores = [&](uint64_t kd, bool turn_over) {
                    tc_fence_after();
#pragma unroll
                    for (int x = 0; x < 16; ++x) {
                        const uint32_t k = 1024u * ((x & 7) >> 2) + 2u * (x & 3);
                        umma_f16(ts, qd + (x < 8 ? 2048u : 0u) + k, kd + k, id_s, x ? 1u : 0u);
                        if (x == 12 && turn_over) pass();          // the other's first products queue behind the last
                    }
                };
                if (!(ok = wait_or_abort(&full[kp.slot], kp.par, abort_flag) && acquire())) break;
                scores(k0 + (uint64_t)(kp.slot * (kPreSlotBytes >> 4)), b == 1 || U > 1);
                umma_commit(&s_full[b]);
                release(kp.slot);
                for (int u = b; u < U; u += 2) {
                    const int t = g.nt == 2 ? u >> 1 : u;
                    const uint64_t vd = v0 + (uint64_t)(vp.slot * (kPreSlotBytes >> 4));
                    const uint32_t again = u >= 2 && !sum_ends((u >> 1) - 1, b) ? 1u : 0u;
                    const bool more = u + 2 < U;
                    if (!again) {                                  // a new sum: the last one has been read
                        if (!(ok = wait_or_abort(&o_read[b], pr, abort_flag))) break;
                        pr ^= 1u;
                    }
                    if (!(ok = wait_or_abort(&full[vp.slot], vp.par, abort_flag) &&
                               wait_or_abort(&p_full[2 * b], pp, abort_flag) && acquire()))
                        break;
                    tc_fence_after();
#pragma unroll
                    for (int x = 0; x < 8; ++x)
                        umma_f16_ta(to, ts + (x < 4 ? 16u : 0u) + 32u * ((x & 3) >> 1) + 8u * (x & 1), vd + 128u * (x & 3),
                                    id_o, x ? 1u : again);
                    // the first 64 tokens' products run while the softmax ends the other half
                    if (more) {
                        advance(kp, g.nt == 2 ? 2 : k_place(t + 2, 1) - k_place(t, 1));
                        ok = wait_or_abort(&full[kp.slot], kp.par, abort_flag);
                    }
                    if (!(ok = ok && wait_or_abort(&p_full[2 * b + 1], pp, abort_flag))) break;
                    pp ^= 1u;
                    tc_fence_after();
#pragma unroll
                    for (int x = 0; x < 8; ++x)
                        umma_f16_ta(to, ts + 64u + (x < 4 ? 16u : 0u) + 32u * ((x & 3) >> 1) + 8u * (x & 1),
                                    vd + 512u + 128u * (x & 3), id_o, 1u);
                    // at once, not behind the scores: the next K tile but one takes this slot, and the ring is short
                    release(vp.slot);
                    // o goes to the record: the buffer's last unit, or kPreFlush of them summed
                    if (!more || sum_ends(u >> 1, b)) umma_commit(&o_full[b]);
                    // an odd piece ends with buffer 0, which begins the next
                    if (more) scores(k0 + (uint64_t)(kp.slot * (kPreSlotBytes >> 4)), true);
                    else if (u + 1 < U || b == 1) pass();
                    if (more) {
                        umma_commit(&s_full[b]);
                        release(kp.slot);
                        advance(vp, g.nt == 2 ? 2 : v_place(t + 2, 1, n) - v_place(t, 1, n));
                    }
                }
            }
            umma_commit(&fin[b]);
            mbar_wait(&fin[b], 0u);
        }
    } else {
        // ---------------- softmax: a thread per row of its score buffer ----------------
        const int b = warp >> 2, r = tid & 127;
        const uint32_t lane_base = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        const uint32_t sb = lane_base + 128u * b, ob = lane_base + 256u + 128u * b;
        uint32_t ps = 0, pr = 1, pq = 0;                           // phases of s_full, o_read (before), q_full
        bool stop = false;
        for (int p = p0; !stop && p < p_end; ++p) {
            const Group g = group_at(a, p);
            if (g.base >= hi) break;
            int t0, t1;
            tiles_of(a, g.base, g.nt, lo, hi, t0, t1);
            const int n = t1 - t0;
            if (n <= 0) continue;
            // This warp's rows of q (32 of its buffer's tile, or 16 of the one tile), scaled and split into the
            // operand's rows. They are copied as they are first, all in flight at once: row r's 512 bytes are the
            // 128-byte rows r of the operand's four blocks (hi and lo, 64 dims each), so that each row is then
            // converted in its own place.
            const int tile0 = (g.rt + (g.nt == 2 ? b : 0)) * kPreRows, row = tile0 + r;
            const bool live = row < a.rows;
            float c2 = 0.f;
            {
                const int sub = lane >> 3, l8 = lane & 7;          // eight lanes a row, four rows a step
                const int steps = g.nt == 2 ? 8 : 4, first_row = g.nt == 2 ? 32 * (warp & 3) : 16 * warp;
                uint8_t *qd = qbuf + (g.nt == 2 ? (size_t)b * kPreQBytes : 0) + (first_row + sub) * 128;
                const int row0 = tile0 + first_row + sub, s0 = row0 / a.G;
                int h = row0 - s0 * a.G;
                const float *src = a.q + s0 * a.q_stride + (size_t)(g.j * a.G + h) * kKvD + 4 * l8;
                const int64_t wrap = a.q_stride - (int64_t)a.G * kKvD;         // to the next sequence's heads
                uint32_t dst = smem_addr(qd + l8 * 16);
#pragma unroll 1
                for (int i = 0; i < steps; ++i, dst += 512u) {
                    const bool in = row0 + 4 * i < a.rows;
                    const float *p = in ? src : a.q;
#pragma unroll
                    for (int k = 0; k < 4; ++k) cp_async16(dst + 16384u * k, p + 32 * k, in);
                    src += 4 * kKvD;
                    for (h += 4; h >= a.G; h -= a.G) src += wrap;
                }
                cp_async_commit();
                cp_async_wait<0>();
                __syncwarp();
#pragma unroll 2
                for (int i = 0; i < steps; ++i) {
                    float4 v[4];
                    float mx = 0.f;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        v[k] = *reinterpret_cast<const float4 *>(qd + i * 512 + l8 * 16 + 16384 * k);   // dims 32 k + 4 l8 ..
                        mx = fmaxf(mx, fmaxf(fmaxf(fabsf(v[k].x), fabsf(v[k].y)), fmaxf(fabsf(v[k].z), fabsf(v[k].w))));
                    }
#pragma unroll
                    for (int o = 4; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                    const float p2 = pow2_of(mx), inv = inv_pow2(p2) * a.qsign;
                    const float mine = __shfl_sync(0xffffffffu, p2, (lane & 3) * 8);    // also: the rows have been read
                    if (lane >> 2 == i) c2 = fmaxf(a.cscale * mine, 1.17549435e-38f);   // not 0: a masked score is -inf c2
                    if (g.nt == 1 && l8 == 0) c_of[first_row + 4 * i + sub] = fmaxf(a.cscale * p2, 1.17549435e-38f);
                    const uint32_t row7 = (uint32_t)(sub + 4 * i) & 7u;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float y[4] = {v[k].x * inv, v[k].y * inv, v[k].z * inv, v[k].w * inv};
                        const float h4[4] = {hi_part(y[0]), hi_part(y[1]), hi_part(y[2]), hi_part(y[3])};
                        // granule 4 (k % 2) + l8 / 2 of the row of block k / 2, swizzled as the operand wants it
                        uint8_t *to = qd + i * 512 + (k >> 1) * 16384 +
                                      (((4u * (k & 1) + (uint32_t)(l8 >> 1)) ^ row7) << 4) + (l8 & 1) * 8;
                        *reinterpret_cast<uint2 *>(to) = make_uint2(pack_h2(h4[0], h4[1]), pack_h2(h4[2], h4[3]));
                        *reinterpret_cast<uint2 *>(to + 32768) =
                            make_uint2(pack_h2(y[0] - h4[0], y[1] - h4[1]), pack_h2(y[2] - h4[2], y[3] - h4[3]));
                    }
                }
            }
            fence_proxy_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
            bool ok = true;
            if (g.nt == 1) {                                       // both buffers have all the rows
                ok = __all_sync(0xffffffffu, wait_or_abort(q_full, pq, abort_flag));
                c2 = c_of[r];
            }
            pq ^= 1u;
            float m = -INFINITY, l = 0.f;
            int unit = 0;
            // this buffer's token tiles: every one (nt 2), or every second one
            const int first = g.nt == 2 ? 0 : b, step = g.nt == 2 ? 1 : 2;
            for (int i = first; ok && i < n; i += step, ++unit) {
                ok = __all_sync(0xffffffffu, wait_or_abort(&s_full[b], ps, abort_flag));
                if (!ok) break;
                ps ^= 1u;
                tc_fence_after();
                // The scores are read twice, 32 tokens at a time, so that few are held in registers: for their
                // maximum, then for P, whose hi and lo parts (16 columns each) take the place of the 32 scores.
                const int left = a.n_prefix - (t0 + i) * kPreTok;
                float mx;
                {
                    float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
                    for (int x = 0; x < kPreTok && x < left; x += 32) {
                        uint32_t v[32];
                        tmem_ld32_nowait(sb + (uint32_t)x, v);
                        tmem_wait_ld();
                        if (left - x < 32) {
#pragma unroll
                            for (int y = 0; y < 32; ++y)
                                if (x + y >= left) v[y] = 0xff800000u;     // -inf
                        }
#pragma unroll
                        for (int y = 0; y < 32; y += 8)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                m4[e] = fmaxf(m4[e], fmaxf(__uint_as_float(v[y + e]), __uint_as_float(v[y + 4 + e])));
                    }
                    mx = c2 * fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                }
                const bool grow = mx > m + kMaxLag;
                const float f = !grow ? 1.f : m == -INFINITY ? 0.f : ex2(m - mx);
                if (grow) m = mx;
                l *= f;
                if (unit > 0 && !sum_ends(unit - 1, b) && __any_sync(0xffffffffu, grow)) {
                    // P V of this buffer's last tile is complete: these scores were issued after it
                    for (int x = 0; x < 4; ++x) {
                        uint32_t ov[32];
                        tmem_ld32_nowait(ob + 32u * x, ov);
                        tmem_wait_ld();
#pragma unroll
                        for (int y = 0; y < 32; ++y) ov[y] = __float_as_uint(__uint_as_float(ov[y]) * f);
                        tmem_st32(ob + 32u * x, ov);
                    }
                }
                const uint64_t cc = pack2(c2, c2), off = pack2(kPShift - m, kPShift - m), minus = pack2(-1.f, -1.f);
                uint64_t ls[2] = {0, 0};
#pragma unroll 1
                for (int x = 0; x < kPreTok; x += 32) {
                    uint32_t v[32], w[32];
                    tmem_ld32_nowait(sb + (uint32_t)x, v);
                    tmem_wait_ld();
                    if (left - x < 32) {
#pragma unroll
                        for (int y = 0; y < 32; ++y)
                            if (x + y >= left) v[y] = 0xff800000u;
                    }
#pragma unroll
                    for (int y = 0; y < 16; ++y) {
                        float p0, p1, d0, d1;
                        unpack2(fma2(pack2(__uint_as_float(v[2 * y]), __uint_as_float(v[2 * y + 1])), cc, off), p0, p1);
                        p0 = ex2(p0);
                        p1 = ex2(p1);
                        const uint64_t pp = pack2(p0, p1);
                        ls[y & 1] = add2(ls[y & 1], pp);
                        const float h0 = hi_part(p0), h1 = hi_part(p1);
                        w[y] = pack_h2(h0, h1);
                        unpack2(fma2(pack2(h0, h1), minus, pp), d0, d1);
                        w[16 + y] = pack_h2(d0, d1);
                    }
                    tmem_st32(sb + (uint32_t)x, w);
                    if (x & 32) {                                  // 64 tokens: their products may begin
                        tmem_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&p_full[2 * b + (x >> 6)]);
                    }
                }
                {
                    float l0, l1;
                    unpack2(add2(ls[0], ls[1]), l0, l1);
                    l += l0 + l1;
                }
                // P V of this unit ends a sum: the maximum it refers to, once the last sum's has been read
                if (i + step >= n || sum_ends(unit, b)) {
                    ok = __all_sync(0xffffffffu, wait_or_abort(&o_read[b], pr, abort_flag));
                    if (!ok) break;
                    pr ^= 1u;
                    m_of[b * kPreRows + r] = m;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&m_full[b]);
                }
            }
            if (ok && live && first < n) a.pre_ml[((size_t)(p + c) * 2 + b) * kPreRows + r] = make_float2(m - kPShift, l);
            // both buffers are done with q before the next piece's is written
            stop = softmax_bar_any(!ok);
        }
    }
    if (*abort_flag && tid == 0) atomicExch(&g_device_error, LI_ERR_TIMEOUT);
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ---------------------------------------------------------------------------
// The join of the pieces of row r = s G + g of kv head j. Pieces 0 .. n_pre-1
// are the prefix's (the same for all rows of a row tile), then the own part's.
// ---------------------------------------------------------------------------
struct RowPieces {
    int n_pre, n_own;
    int p, c0, streams, stream0, prow;     // prefix: group, first block, records per block
    int len, extra, base, nt;              //         the blocks' runs, the group's place and cost
    int rec0, gq;                          // own
};

// The prefix's share follows from the sizes alone; the sequences' own shares
// wait for kv_own's table.
__device__ __forceinline__ RowPieces prefix_pieces(const KvAttnArgs &a, int j, int row) {
    RowPieces x;
    x.gq = row % a.G;
    x.n_pre = x.n_own = 0;
    if (a.n_prefix > 0) {
        const int rt = row / kPreRows;
        x.prow = row - rt * kPreRows;
        x.p = j * a.n_grp + rt / a.per_group;
        const Group g = group_at(a, x.p);
        const Runs runs(a.Hkv * a.n_rt * a.n_tt, a.pre_ctas);
        x.len = runs.len; x.extra = runs.extra; x.base = g.base; x.nt = g.nt;
        x.c0 = runs.taker(g.base);
        const int c1 = runs.taker(g.base + g.nt * a.n_tt - 1);
        // one record per buffer; runs of one tile leave buffer 1 none
        x.streams = g.nt == 2 || runs.len + (runs.extra ? 1 : 0) <= 1 ? 1 : 2;
        x.stream0 = g.nt == 2 ? rt - g.rt : 0;
        x.n_pre = (c1 - x.c0 + 1) * x.streams;
    }
    return x;
}

__device__ __forceinline__ void own_pieces(const KvAttnArgs &a, RowPieces &x, int j, int s) {
    const int n = own_tokens(a, s), T = __ldcg(a.base + a.B), b0 = __ldcg(a.base + s);
    if (n > 0) {
        const Runs runs(T, own_active(T, a.own_warps));
        const int st = own_steps(n), at = b0 + j * st;
        const int w0 = runs.taker(at), w1 = runs.taker(at + st - 1);
        x.rec0 = s * a.Hkv + j + w0;
        x.n_own = w1 - w0 + 1;
    }
}

// Record of prefix piece i, or -1 where that piece holds no token.
__device__ __forceinline__ int pre_record(const KvAttnArgs &a, const RowPieces &x, int i) {
    const int c = x.c0 + (x.streams == 2 ? i >> 1 : i), w = x.streams == 2 ? i & 1 : x.stream0;
    const int lo = c * x.len + min(c, x.extra), hi = (c + 1) * x.len + min(c + 1, x.extra);
    int t0, t1;
    tiles_of(a, x.base, x.nt, lo, hi, t0, t1);
    return t1 - t0 > (x.streams == 2 ? w : 0) ? (x.p + c) * 2 + w : -1;
}

// (max, sum) of piece i; (-inf, 0) for an empty one.
__device__ __forceinline__ float2 piece_ml(const KvAttnArgs &a, const RowPieces &x, int i) {
    if (i < x.n_pre) {
        const int rec = pre_record(a, x, i);
        return rec < 0 ? make_float2(-INFINITY, 0.f) : __ldcg(a.pre_ml + (size_t)rec * kPreRows + x.prow);
    }
    return __ldcg(a.own_ml + (size_t)(x.rec0 + i - x.n_pre) * a.G + x.gq);
}

constexpr int kJoinWarps = 8;
constexpr int kJoinRun = kJoinWarps * kWarp * 4;     // slots of a weight block's step

// Rows: wpr neighbouring warps take ROWS rows of a kv head, each its share of
// the pieces; lane l holds row l % ROWS and the 4-dim groups l / ROWS,
// + 32 / ROWS, ... (the prefix's records lie dims first, so that with four rows
// a load reads whole sectors either way). With one row a warp has eight pieces
// in flight instead of two: few rows with many pieces each (one sequence's
// long cache is cut into hundreds).
template <int ROWS>
__global__ void __launch_bounds__(kJoinWarps * kWarp, 3) kv_join_kernel(const __grid_constant__ KvAttnArgs a) {
    constexpr int kPer = 8 / ROWS, kApart = kWarp / ROWS;
    __shared__ float red_m[kJoinWarps][ROWS], red_l[kJoinWarps][ROWS];
    __shared__ __align__(16) float4 red_o[kJoinWarps][ROWS][kWarp];
    __shared__ float gm[16], gi[16];
    const int tid = threadIdx.x, warp = tid / kWarp, lane = tid % kWarp;
    if ((int)blockIdx.x < a.row_ctas) {
        const int per = kJoinWarps / a.wpr, sub = warp % a.wpr;
        const int rows = a.B * a.G, blocks = (rows + ROWS - 1) / ROWS;      // row blocks of a kv head
        const int item = blockIdx.x * per + warp / a.wpr, j = item / blocks;
        const int rl = lane % ROWS, xq = lane / ROWS, row = (item - j * blocks) * ROWS + rl;
        const bool on = j < a.Hkv && row < rows;
        RowPieces x = prefix_pieces(a, on ? j : 0, on ? row : 0);
        grid_dep_wait();
        grid_dep_launch_dependents();
        float m = -INFINITY, l = 0.f;
        float4 o[ROWS];
#pragma unroll
        for (int i = 0; i < ROWS; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (on) {
            own_pieces(a, x, j, row / a.G);
            const int n = x.n_pre + x.n_own;
            // kPer pieces at a time, their loads in flight together (predicated, not branched over)
            for (int i0 = sub; i0 < n; i0 += kPer * a.wpr) {
                float4 v[kPer][ROWS];
                float2 ml[kPer];
#pragma unroll
                for (int e = 0; e < kPer; ++e) {
                    const int i = i0 + e * a.wpr;
                    const bool pre = i < x.n_pre;
                    const int rec = i >= n ? -1 : pre ? pre_record(a, x, i) : (x.rec0 + i - x.n_pre) * a.G + x.gq;
                    const float4 *src = pre ? reinterpret_cast<const float4 *>(a.pre_o) +
                                                  ((size_t)max(rec, 0) * 32 + xq) * kPreRows + x.prow
                                            : reinterpret_cast<const float4 *>(a.own_o) + (size_t)max(rec, 0) * 32 + xq;
                    const float2 *mp = pre ? a.pre_ml + (size_t)max(rec, 0) * kPreRows + x.prow : a.own_ml + max(rec, 0);
                    const int step = pre ? kApart * kPreRows : kApart;
                    ml[e] = rec >= 0 ? __ldcg(mp) : make_float2(-INFINITY, 0.f);
#pragma unroll
                    for (int k = 0; k < ROWS; ++k)
                        v[e][k] = rec >= 0 ? __ldcg(src + k * step) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
                float mx = m;
#pragma unroll
                for (int e = 0; e < kPer; ++e) mx = fmaxf(mx, ml[e].x);
                const float keep = m == -INFINITY ? 0.f : ex2(m - mx);
                m = mx;
                l *= keep;
#pragma unroll
                for (int k = 0; k < ROWS; ++k) { o[k].x *= keep; o[k].y *= keep; o[k].z *= keep; o[k].w *= keep; }
#pragma unroll
                for (int e = 0; e < kPer; ++e) {
                    const float f = ml[e].x == -INFINITY ? 0.f : ex2(ml[e].x - mx);
                    l = fmaf(f, ml[e].y, l);
#pragma unroll
                    for (int k = 0; k < ROWS; ++k) {
                        o[k].x = fmaf(f, v[e][k].x, o[k].x); o[k].y = fmaf(f, v[e][k].y, o[k].y);
                        o[k].z = fmaf(f, v[e][k].z, o[k].z); o[k].w = fmaf(f, v[e][k].w, o[k].w);
                    }
                }
            }
        }
        if (a.wpr > 1) {
            if (xq == 0) { red_m[warp][rl] = m; red_l[warp][rl] = l; }
#pragma unroll
            for (int k = 0; k < ROWS; ++k) red_o[warp][k][lane] = o[k];
            __syncthreads();
            if (sub == 0) {
                float M = m;
                for (int w = 1; w < a.wpr; ++w) M = fmaxf(M, red_m[warp + w][rl]);
                for (int w = 0; w < a.wpr; ++w) {
                    const float f = red_m[warp + w][rl] == -INFINITY ? 0.f : ex2(red_m[warp + w][rl] - M);
                    l = w ? fmaf(f, red_l[warp + w][rl], l) : f * l;
#pragma unroll
                    for (int k = 0; k < ROWS; ++k) {
                        const float4 v = red_o[warp + w][k][lane];
                        o[k].x = w ? fmaf(f, v.x, o[k].x) : f * v.x; o[k].y = w ? fmaf(f, v.y, o[k].y) : f * v.y;
                        o[k].z = w ? fmaf(f, v.z, o[k].z) : f * v.z; o[k].w = w ? fmaf(f, v.w, o[k].w) : f * v.w;
                    }
                }
                m = M;
            }
        }
        if (on && sub == 0) {
            const float inv = m == -INFINITY ? 0.f : 1.f / l;      // no token at all: zeros
            const int s = row / a.G;
            float4 *d = reinterpret_cast<float4 *>(a.out + ((size_t)s * a.Hq + (size_t)j * a.G + row - s * a.G) * kKvD) + xq;
#pragma unroll
            for (int k = 0; k < ROWS; ++k) {
                float4 v = make_float4(o[k].x * inv, o[k].y * inv, o[k].z * inv, o[k].w * inv);
                if (a.gate) {
                    const float4 gt = reinterpret_cast<const float4 *>(
                        a.gate + s * a.gate_stride + ((size_t)j * a.G + row - s * a.G) * kKvD)[xq + kApart * k];
                    v.x *= sigmoid(gt.x); v.y *= sigmoid(gt.y); v.z *= sigmoid(gt.z); v.w *= sigmoid(gt.w);
                }
                d[kApart * k] = v;
            }
        }
        return;
    }
    grid_dep_wait();
    grid_dep_launch_dependents();
    // weights of the pair (s, j), every w_chunks-th run of slots, four neighbouring ones a thread
    const int item = blockIdx.x - a.row_ctas, pair = item / a.w_chunks, chunk = item - pair * a.w_chunks;
    const int s = pair / a.Hkv, j = pair - s * a.Hkv, n = own_len(a, s);
    if (chunk * kJoinRun >= n) return;
    for (int gq = warp; gq < a.G; gq += kJoinWarps) {
        RowPieces x = prefix_pieces(a, j, s * a.G + gq);
        own_pieces(a, x, j, s);
        const int cnt = x.n_pre + x.n_own;
        float m = -INFINITY, l = 0.f;
        for (int i = lane; i < cnt; i += kWarp) {
            const float2 ml = piece_ml(a, x, i);
            if (ml.x != -INFINITY) {
                const float mx = fmaxf(m, ml.x);
                l = (m == -INFINITY ? 0.f : l * ex2(m - mx)) + ml.y * ex2(ml.x - mx);
                m = mx;
            }
        }
        float M = m;
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, k));
        const float L = warp_sum(m == -INFINITY ? 0.f : l * ex2(m - M));
        if (lane == 0) { gm[gq] = M; gi[gq] = 1.f / L; }
    }
    __syncthreads();
    float *wt = a.weight + (size_t)pair * a.max_ctx;
    const float *sc = a.score + ((size_t)s * a.Hq + (size_t)j * a.G) * a.score_stride;
    const bool vec = (a.max_ctx & 3) == 0 && ((uintptr_t)a.weight & 15u) == 0;
    for (int t = chunk * kJoinRun + 4 * tid; t < n; t += a.w_chunks * kJoinRun) {
        // the step's probabilities are summed first: one rounding against the accumulated weight
        float w[4] = {0.f, 0.f, 0.f, 0.f}, old[4] = {0.f, 0.f, 0.f, 0.f};
        const bool whole = vec && t + 4 <= n;
        if (a.decay != 0.f) {
            if (whole) {
                const float4 v = *reinterpret_cast<const float4 *>(wt + t);
                old[0] = v.x; old[1] = v.y; old[2] = v.z; old[3] = v.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (t + e < n) old[e] = wt[t + e];
            }
        }
        // a row of scores has score_stride floats, a multiple of 4: past n it holds nothing, and none of it is kept
#pragma unroll 4
        for (int gq = 0; gq < a.G; ++gq) {
            const float4 v = __ldcg(reinterpret_cast<const float4 *>(sc + (size_t)gq * a.score_stride + t));
            const float m = gm[gq], inv = gi[gq];
            w[0] = fmaf(ex2(v.x - m), inv, w[0]);
            w[1] = fmaf(ex2(v.y - m), inv, w[1]);
            w[2] = fmaf(ex2(v.z - m), inv, w[2]);
            w[3] = fmaf(ex2(v.w - m), inv, w[3]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = fmaf(a.decay, old[e], w[e]);
        if (whole) {
            *reinterpret_cast<float4 *>(wt + t) = make_float4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (t + e < n) wt[t + e] = w[e];
        }
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encoder() {
    static EncodeTiledFn fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
    });
    return fn;
}

// The prefix [n][Hkv][128] f16 as (dim, kv head, token) with a box of 128
// tokens by 64 dims, 128-byte swizzle; tokens past n come in as zeros.
int encode_prefix(CUtensorMap *m, const void *base, int Hkv, int n) {
    EncodeTiledFn fn = encoder();
    if (!fn) return LI_ERR_UNSUPPORTED;
    const cuuint64_t dims[3] = {(cuuint64_t)kKvD, (cuuint64_t)Hkv, (cuuint64_t)n};
    const cuuint64_t strides[2] = {(cuuint64_t)kKvD * 2, (cuuint64_t)Hkv * kKvD * 2};
    const cuuint32_t box[3] = {64, 1, (cuuint32_t)kPreTok};
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void *>(base), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : LI_ERR_BAD_SHAPE;
}

size_t al256(size_t v) { return (v + 255) / 256 * 256; }

// Grids and the workspace of a call; everything the size needs, nothing on
// the device. Returns the workspace's bytes, 0 when a count is beyond the
// kernels' integers.
size_t plan(const li_kv_cache *C, int n_q_heads, KvAttnArgs *a, size_t *off /* [6] */) {
    const int sms = num_sms();
    a->B = C->n_seqs; a->Hq = n_q_heads; a->Hkv = C->n_kv_heads; a->G = n_q_heads / C->n_kv_heads;
    a->max_ctx = C->max_ctx; a->n_prefix = C->n_prefix;
    const int64_t pairs = (int64_t)a->B * a->Hkv;
    // A prefix that is little to read even once per sequence (30 MB: about 5 us), or that has one reader, goes with
    // the own tokens: one kernel less, and no tile of 128 rows for a few. Us with the prefix kernel and without, 100
    // own tokens, caches cold: 4 sequences x 32 heads 20 and 16 at 256 tokens (4 MB), 26 and 20 at 1919 (30 MB), 28
    // and 24 at 4000 (62 MB), even at 8000; 16 sequences 22 and 20 at 480 (30 MB), 24 and 24 at 1000, 25 and 33 at
    // 2000 (125 MB); 64 sequences x 40 heads even at 30 tokens (7 MB), 23 and 24 at 119 (30 MB), 23 and 28 at 250. One
    // sequence: 20 and 15 at 512 tokens, 119 and 115 at 131072 with 8 kv heads, even with 4, but 41 and 57 with
    // one.
    if (a->n_prefix > 0 && (a->B == 1 || pairs * a->n_prefix <= (30ll << 20) / (4 * kKvD))) {
        a->lead = a->n_prefix;
        a->n_prefix = 0;
    }
    const int64_t most = pairs * ((a->max_ctx + (int64_t)a->lead + kOwnTok - 1) / kOwnTok);
    if (most >= (1ll << 30) || pairs * a->G >= (1ll << 30) || a->max_ctx + (int64_t)a->lead >= (1ll << 30)) return 0;
    int free_sms = sms;
    if (a->n_prefix > 0) {
        a->rows = a->B * a->G;
        a->n_rt = (a->rows + kPreRows - 1) / kPreRows;
        a->n_tt = (a->n_prefix + kPreTok - 1) / kPreTok;
        const int64_t cost = (int64_t)a->Hkv * a->n_rt * a->n_tt;
        if (cost >= (1ll << 30)) return 0;
        // Two row tiles share the K and V tiles they read, unless that leaves SMs idle. Us with one and with two: 33
        // and 35 at 1.3 units an SM (64 sequences x 1024 x 40 heads), 38 and 39 at 2.6, 53 and 53 at 10; where the
        // prefix is beyond L2 or the rows are many, 190 and 181 (64 x 65536), 369 and 346 (512 x 16384), though 661 and
        // 703 at 256 x 65536.
        a->per_group = a->n_rt > 1 && cost >= 2ll * sms ? 2 : 1;
        a->n_grp = (a->n_rt + a->per_group - 1) / a->per_group;
        a->slots = a->per_group == 2 ? kPreSlots2 : kPreSlots1;
        // With little to do, two token tiles a block: a tile for each score buffer, and SMs left for kv_own meanwhile
        // (16 x 2085 and weights: 29 us with a tile a block on 136 SMs, 24 with two on 68). A prefix of one tile has
        // no second one to add: a block a group (28 us from 34 at 201 x 123 x 16 heads).
        const int64_t blocks = a->per_group == 1 && a->n_tt > 1 ? (cost + 1) / 2 : cost;
        a->pre_ctas = (int)(blocks < sms ? blocks : sms);
        if (2 * a->pre_ctas <= sms) free_sms = sms - a->pre_ctas;
    }
    int64_t grid = most / kOwnMinSteps;
    grid = grid < 1 ? 1 : grid < free_sms ? grid : free_sms;
    a->own_warps = (int)grid * kOwnWarps;
    size_t at = 0;
    off[0] = at; at += al256(((size_t)a->B + 1) * 4);
    const size_t own_recs = (size_t)pairs + a->own_warps;
    off[1] = at; at += al256(own_recs * a->G * sizeof(float2));
    off[2] = at; at += al256(own_recs * a->G * kKvD * 4);
    a->score_stride = (a->max_ctx + 3) / 4 * 4;
    off[3] = at; at += C->weight ? al256((size_t)a->B * a->Hq * a->score_stride * 4) : 0;
    off[4] = off[5] = at;
    if (a->n_prefix > 0) {
        const size_t recs = ((size_t)a->Hkv * a->n_grp + a->pre_ctas) * 2 * kPreRows;
        off[4] = at; at += al256(recs * sizeof(float2));
        off[5] = at; at += al256(recs * kKvD * 4);
    }
    return at;
}

template <int NG, bool SCORE, bool LEAD>
int launch_own(const KvAttnArgs &a, cudaStream_t s) {
    static std::atomic<uint64_t> done{0};
    if (const int rc = allow_smem(kv_own_kernel<NG, SCORE, LEAD>, kOwnSmem, done)) return rc;
    return (int)launch_pdl(kv_own_kernel<NG, SCORE, LEAD>, dim3((unsigned)(a.own_warps / kOwnWarps)),
                           dim3(kOwnThreads), kOwnSmem, s, true, a);
}

template <int NG, bool SCORE>
int launch_own(const KvAttnArgs &a, cudaStream_t s) {
    return a.lead ? launch_own<NG, SCORE, true>(a, s) : launch_own<NG, SCORE, false>(a, s);
}

}  // namespace
}  // namespace li

using namespace li;

extern "C" {

size_t li_attn_kv_workspace_size(const li_kv_cache *C, int n_q_heads) {
    if (check_kv_cache(C) || C->n_seqs == 0 || n_q_heads <= 0 || n_q_heads % C->n_kv_heads ||
        n_q_heads / C->n_kv_heads > 16)
        return 0;
    KvAttnArgs a = {};
    size_t off[6];
    return plan(C, n_q_heads, &a, off);
}

int li_launch_attn_kv_decode(const li_kv_cache *C, const float *q, int64_t q_stride, int n_q_heads, float scale,
                             float *out, float decay, void *workspace, size_t workspace_bytes, void *stream) {
    return attn_kv_decode(C, q, q_stride, n_q_heads, scale, out, decay, nullptr, 0, workspace, workspace_bytes, stream);
}

}  // extern "C"

int li::attn_kv_decode(const li_kv_cache *C, const float *q, int64_t q_stride, int n_q_heads, float scale, float *out,
                       float decay, const float *gate, int64_t gate_stride, void *workspace, size_t workspace_bytes,
                       void *stream) {
    if (const int rc = check_kv_cache(C)) return rc;
    if (!q || !out || n_q_heads <= 0 || !(decay >= 0.0f) || isinf(decay) || !isfinite(scale)) return LI_ERR_BAD_ARG;
    if (n_q_heads % C->n_kv_heads) return LI_ERR_BAD_SHAPE;
    if (n_q_heads / C->n_kv_heads > 16) return LI_ERR_UNSUPPORTED;
    if (!aligned16(q) || !aligned16(out) || q_stride % 4) return LI_ERR_MISALIGNED;
    if (C->n_seqs == 0) return 0;
    KvAttnArgs a = {};
    size_t off[6];
    const size_t need = plan(C, n_q_heads, &a, off);
    if (need == 0) return LI_ERR_BAD_SHAPE;
    if (!workspace || workspace_bytes < need) return LI_ERR_WORKSPACE;
    if (!aligned16(workspace)) return LI_ERR_MISALIGNED;
    const cudaStream_t st = (cudaStream_t)stream;
    char *ws = static_cast<char *>(workspace);
    a.q = q; a.q_stride = q_stride;
    a.k = static_cast<const __half *>(C->k); a.v = static_cast<const __half *>(C->v);
    a.kp = static_cast<const __half *>(C->k_prefix); a.vp = static_cast<const __half *>(C->v_prefix);
    a.len = C->len;
    a.cscale = fabsf(scale) * kLog2e; a.qsign = scale < 0.f ? -1.f : 1.f;
    a.decay = decay; a.out = out; a.weight = C->weight;
    a.gate = gate; a.gate_stride = gate_stride;
    a.base = reinterpret_cast<int *>(ws + off[0]);
    a.own_ml = reinterpret_cast<float2 *>(ws + off[1]);
    a.own_o = reinterpret_cast<float *>(ws + off[2]);
    a.score = reinterpret_cast<float *>(ws + off[3]);
    a.pre_ml = reinterpret_cast<float2 *>(ws + off[4]);
    a.pre_o = reinterpret_cast<float *>(ws + off[5]);
    a.after_prefix = a.n_prefix > 0;
    int rc;
    if (a.n_prefix > 0) {
        CUtensorMap mk, mv;
        memset(&mk, 0, sizeof(mk));
        memset(&mv, 0, sizeof(mv));
        if ((rc = encode_prefix(&mk, C->k_prefix, a.Hkv, a.n_prefix)) ||
            (rc = encode_prefix(&mv, C->v_prefix, a.Hkv, a.n_prefix)))
            return rc;
        static std::atomic<uint64_t> done{0};
        if ((rc = allow_smem(kv_prefix_kernel, kPreSmem, done))) return rc;
        if ((rc = (int)launch_pdl(kv_prefix_kernel, dim3((unsigned)a.pre_ctas), dim3(kPreThreads), kPreSmem, st, true,
                                  mk, mv, a)))
            return rc;
    }
    if (a.G <= 8) rc = a.weight ? launch_own<1, true>(a, st) : launch_own<1, false>(a, st);
    else rc = a.weight ? launch_own<2, true>(a, st) : launch_own<2, false>(a, st);
    if (rc) return rc;
    // A row a warp where eight warps a row do not fill the SMs twice over, four rows where they do (a row a warp: 45 us
    // from 54 at 27 sequences x 40775 x 6 heads, 31 from 52 at 5 x 9910 x 16; 1 us behind at 180 rows with few
    // pieces, and 25 against 23 at 512 rows); and as many warps on them as it takes to fill the SMs, up to the pieces
    // that a row can have.
    const int pairs = a.B * a.Hkv;
    const int64_t pre = a.n_prefix ? 2ll * a.pre_ctas / (a.Hkv * a.n_grp) + 2 : 0;
    int64_t own = (a.max_ctx + (int64_t)a.lead + kOwnTok - 1) / kOwnTok / kOwnMinSteps + 1;
    if (own > a.own_warps / pairs + 2) own = a.own_warps / pairs + 2;
    const int rows_each = (int64_t)pairs * a.G <= 2ll * num_sms() ? 1 : 4;
    const int64_t row_blocks = (int64_t)a.Hkv * ((a.B * a.G + rows_each - 1) / rows_each);
    a.wpr = 1;
    while (a.wpr < kJoinWarps && a.wpr < pre + own && row_blocks * a.wpr < 16ll * num_sms()) a.wpr *= 2;
    const int per = kJoinWarps / a.wpr;
    a.row_ctas = (int)((row_blocks + per - 1) / per);
    int64_t blocks = a.row_ctas;
    if (a.weight) {
        // blocks per pair: enough for every SM to hold some, since each first joins its pair's sums
        const int64_t ch = ((int64_t)a.max_ctx + kJoinRun - 1) / kJoinRun, cap = (num_sms() * 4ll + pairs - 1) / pairs;
        a.w_chunks = (int)(ch < cap ? ch : cap);
        blocks += (int64_t)pairs * a.w_chunks;
    }
    if (blocks > 0x7fffffff) return LI_ERR_BAD_SHAPE;
    return rows_each == 1
               ? (int)launch_pdl(kv_join_kernel<1>, dim3((unsigned)blocks), dim3(kJoinWarps * kWarp), 0, st, true, a)
               : (int)launch_pdl(kv_join_kernel<4>, dim3((unsigned)blocks), dim3(kJoinWarps * kWarp), 0, st, true, a);
}
