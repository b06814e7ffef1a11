// Rotary positions, and the append of new tokens to a KV cache.
//
//   (y1, y2) = m (x1 cos a - x2 sin a, x2 cos a + x1 sin a) per pair, the
//   angle a of (position, pair) as described at li_rope.
//
// Bound by HBM: every value is read once and written once, a pair costs four
// products. The angles are the only costly arithmetic (double products, a
// sincospi), so a block takes whole tokens: it computes the cos and sin of
// its tokens' pairs once into shared memory and uses them for every head.
// A thread's unit of work is two vectors of E values (16 bytes each where
// alignment and sizes allow): the two halves of E pairs in the half layout,
// two vectors of E / 2 pairs half the rotated part apart in the interleaved
// one, and two as far apart in the part that passes through, so that the
// threads of a load or store have neighbouring vectors (neighbours in one
// thread put the halves of a 32-byte sector into two instructions, 1.8 times the
// L2 traffic: 47 us for the f16 prompts that take 39). A thread keeps its place in
// the head and walks over heads and tokens (no division per unit); the first
// units' loads are issued before the
// angles are computed, which hides the one behind the other.
#include "li_kv.cuh"

#include <math.h>

LI_DEFINE_TU_STATUS(rope)

namespace li {

int rope_args(const li_rope *R, RopeArgs *a) {
    if (R->layout != LI_ROPE_INTERLEAVED && R->layout != LI_ROPE_HALF) return LI_ERR_UNSUPPORTED;
    if (R->head_dim < 2 || R->head_dim > kRopeMaxDim || R->head_dim % 2) return LI_ERR_BAD_SHAPE;
    if (R->rope_dim < 0 || R->rope_dim % 2 || R->rope_dim > R->head_dim) return LI_ERR_BAD_SHAPE;
    if (!(R->theta > 1.0f) || isinf(R->theta) || !(R->freq_scale > 0.0f) || isinf(R->freq_scale) ||
        !isfinite(R->ext_factor) || !isfinite(R->attn_factor))
        return LI_ERR_BAD_ARG;
    if ((uintptr_t)R->freq_factors & 3u) return LI_ERR_MISALIGNED;
    const int d = R->rope_dim;
    const double two_pi = 6.283185307179586476925, lt = log((double)R->theta);
    double lo = 0.0, hi = 0.0, mag = R->attn_factor;
    if (R->ext_factor != 0.0f) {
        if (R->n_ctx_orig <= 0 || !(R->beta_fast > 0.0f) || !(R->beta_slow > 0.0f)) return LI_ERR_BAD_ARG;
        lo = fmax(0.0, floor(d * log(R->n_ctx_orig / (R->beta_fast * two_pi)) / (2.0 * lt)));
        hi = fmin(d - 1.0, ceil(d * log(R->n_ctx_orig / (R->beta_slow * two_pi)) / (2.0 * lt)));
        mag *= 1.0 + 0.1 * log(1.0 / R->freq_scale);
    }
    a->layout = R->layout;
    a->rope_dim = d;
    a->mag = (float)mag;
    a->factors = R->freq_factors;
    // theta^(-2i/d) by repeated products: off by 2^-46 of the value at worst (256 products), and by 2^-53 of a turn a
    // position, since the frequencies shrink meanwhile (bases of 100 and more)
    const double ratio = d > 0 ? exp(-2.0 / d * lt) : 1.0;
    double f = 1.0 / two_pi;
    for (int i = 0; i < d / 2; ++i, f *= ratio) {
        double c = R->freq_scale;
        if (R->ext_factor != 0.0f) {
            const double r = R->ext_factor * (1.0 - fmin(1.0, fmax(0.0, (i - lo) / fmax(0.001, hi - lo))));
            c = c * (1.0 - r) + r;
        }
        a->turns[i] = f * c;
    }
    return 0;
}

namespace {

constexpr int kRopeThreads = 256;      // at most
// Units of a thread in flight, and blocks per SM that the registers are held
// down to: more of the one costs the other. Two and four take 22.8 us for 4096
// tokens x 48 heads x 128 bf16 (of 15.6 at the copy rate), three units at four
// blocks 31 us, four at three 33 us, two at five blocks 29 us.
constexpr int kRopeBatch = 2, kRopeBlocks = 4;

// One launch over n_tokens tokens and `heads` head slots. Plain rotation: one
// source. Append: head slots are q heads, then k heads, then v heads.
struct RopeJob {
    RopeArgs r;
    const void *x;                     // plain: x; append: q
    void *dst;                         // plain: dst; append: q_out
    int64_t x_ts, x_hs, d_ts, d_hs;    // element strides (token, head)
    const int32_t *pos;
    int n_tokens, heads, D;
    int tb, hb, n_hblk;                // tokens and head slots per block, head blocks
    int hp, np;                        // heads a block takes at once, rounds of them per token
    int n_rot, units;                  // rotated units and all units per head
    float sin_sign;                    // -1: the transpose
    // append
    const void *k, *v;
    int64_t k_ts, v_ts;
    int Hq, Hkv, n_seqs, max_ctx;
    const int32_t *seq, *slot, *len;
    __half *k_cache, *v_cache;
    float *weight;
    int32_t *slot_pos;
};

template <int BYTES> struct VecOf;
template <> struct VecOf<16> { typedef uint4 type; };
template <> struct VecOf<8> { typedef uint2 type; };
template <> struct VecOf<4> { typedef uint32_t type; };
template <> struct VecOf<2> { typedef unsigned short type; };

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f(float &o, float v) { o = v; }
__device__ __forceinline__ void from_f(__half &o, float v) { o = __float2half_rn(v); }
__device__ __forceinline__ void from_f(__nv_bfloat16 &o, float v) { o = __float2bfloat16_rn(v); }

template <typename T, int E>
struct alignas(sizeof(T) * E) Pack {
    T v[E];
};

template <typename T, int E>
__device__ __forceinline__ Pack<T, E> load_pack(const T *p) {
    typedef typename VecOf<sizeof(T) * E>::type V;
    Pack<T, E> r;
    *reinterpret_cast<V *>(&r) = *reinterpret_cast<const V *>(p);   // x may be dst
    return r;
}

template <typename O, int E>
__device__ __forceinline__ void store_pack(O *p, const float (&f)[E]) {
    typedef typename VecOf<sizeof(O) * E>::type V;
    Pack<O, E> r;
#pragma unroll
    for (int e = 0; e < E; ++e) from_f(r.v[e], f[e]);
    *reinterpret_cast<V *>(p) = *reinterpret_cast<V *>(&r);
}

// A block's table of (cos, sin): two pairs are 16 bytes, and the 16-byte groups
// that a vector takes (kGroups of them) lie a stride apart, so that the threads
// of a read have neighbouring ones (in pair order they fell on a quarter of the
// banks). Place of pair i of `half`:
template <int E, bool HALF> struct Table {
    static constexpr int kPairs = HALF ? E : E > 1 ? E / 2 : 1;        // of a vector (E 1, interleaved: of two)
    static constexpr int kGroups = kPairs / 2;                         // 0: pair order
    static __device__ __forceinline__ int place(int i, int half) {
        constexpr int K = kGroups > 1 ? kGroups : 1;
        if (K == 1) return i;
        const int g = i >> 1;
        return 2 * ((g % K) * (half / kPairs) + g / K) + (i & 1);
    }
    // pairs of vector v
    static __device__ __forceinline__ void read(const float2 *t, int v, int half, float2 (&c)[kPairs]) {
        if (kGroups == 0) {
            c[0] = t[v];
        } else {
#pragma unroll
            for (int k = 0; k < kGroups; ++k) {
                const float4 x = reinterpret_cast<const float4 *>(t)[k * (half / kPairs) + v];
                c[2 * k] = make_float2(x.x, x.y);
                c[2 * k + 1] = make_float2(x.z, x.w);
            }
        }
    }
};

template <typename T, int E, bool HALF, bool APPEND>
__global__ void __launch_bounds__(kRopeThreads, kRopeBlocks) rope_kernel(const __grid_constant__ RopeJob j) {
    extern __shared__ __align__(16) uint8_t rope_smem[];
    const int half = j.r.rope_dim / 2;
    float2 *cs = reinterpret_cast<float2 *>(rope_smem);                               // [tb][half]
    int64_t *row = reinterpret_cast<int64_t *>(rope_smem + (size_t)8 * j.tb * half);  // [tb] cache row or -1
    grid_dep_wait();
    grid_dep_launch_dependents();
    const int tblk = blockIdx.x / j.n_hblk, hblk = blockIdx.x - tblk * j.n_hblk;
    const int t0 = tblk * j.tb, nt = min(j.tb, j.n_tokens - t0);
    const int h0 = hblk * j.hb, nh = min(j.hb, j.heads - h0);
    // this thread's place: unit u of head hd (of hp heads), the same in every round
    const int hd = threadIdx.x / j.units, u = threadIdx.x - hd * j.units;
    const bool rot = u < j.n_rot, worker = hd < j.hp;
    const int oa = !rot ? j.r.rope_dim + (u - j.n_rot) * E : !HALF && E == 1 ? 2 * u : u * E;
    const int ob = !rot ? oa + (j.units - j.n_rot) * E : !HALF && E == 1 ? oa + 1 : half + oa;
    const bool two = ob < j.D;
    // a walk over (token, round): the unit at (t, p) is head h0 + hd + p hp of token t0 + t
    struct Walk { int t, p; };
    auto step = [&](Walk &w) {
        if (++w.p == j.np) { w.p = 0; ++w.t; }
    };
    auto valid = [&](const Walk &w) { return worker && w.t < nt && hd + w.p * j.hp < nh; };

    Walk ld = {0, 0}, wk = {0, 0};
    for (bool first = true; wk.t < nt; first = false) {
        Pack<T, E> a[kRopeBatch], b[kRopeBatch];
#pragma unroll
        for (int i = 0; i < kRopeBatch; ++i, step(ld)) {
            if (!valid(ld)) continue;
            const int h = h0 + hd + ld.p * j.hp;
            const int64_t t = t0 + ld.t;
            const T *src;
            if (!APPEND || h < j.Hq) src = static_cast<const T *>(j.x) + t * j.x_ts + h * j.x_hs;
            else if (h < j.Hq + j.Hkv) src = static_cast<const T *>(j.k) + t * j.k_ts + (int64_t)(h - j.Hq) * j.D;
            else src = static_cast<const T *>(j.v) + t * j.v_ts + (int64_t)(h - j.Hq - j.Hkv) * j.D;
            a[i] = load_pack<T, E>(src + oa);
            if (two) b[i] = load_pack<T, E>(src + ob);
        }
        if (first) {                                // the block's angles, behind the first loads
            for (int i = threadIdx.x; i < nt * half; i += blockDim.x) {
                const int tok = i / half;
                float2 x = rope_cos_sin(j.r, j.pos[t0 + tok], i - tok * half);
                x.y *= j.sin_sign;
                cs[tok * half + Table<E, HALF>::place(i - tok * half, half)] = x;
            }
            if (APPEND && (int)threadIdx.x < nt) {
                const int t = t0 + threadIdx.x, s = j.seq ? j.seq[t] : t;
                int64_t r = -1;
                if (s >= 0 && s < j.n_seqs) {
                    const int sl = j.slot ? j.slot[t] : j.len[s] - 1;
                    if (sl >= 0 && sl < j.max_ctx) r = (int64_t)s * j.max_ctx + sl;
                }
                if (r < 0 && hblk == 0) atomicExch(&g_device_error, LI_ERR_BAD_ARG);
                row[threadIdx.x] = r;
            }
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < kRopeBatch; ++i, step(wk)) {
            if (!valid(wk)) continue;
            const int h = h0 + hd + wk.p * j.hp;
            const int64_t t = t0 + wk.t;
            float x[2][E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                x[0][e] = to_f(a[i].v[e]);
                x[1][e] = two ? to_f(b[i].v[e]) : 0.f;
            }
            if (rot && (!APPEND || h < j.Hq + j.Hkv)) {
                const float2 *cp = cs + wk.t * half;
                constexpr int P = Table<E, HALF>::kPairs;
                if constexpr (HALF || E == 1) {    // pair e: (a_e, b_e)
                    float2 c[P];
                    Table<E, HALF>::read(cp, u, half, c);
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const float p = x[0][e], q = x[1][e];
                        x[0][e] = p * c[e].x - q * c[e].y;
                        x[1][e] = q * c[e].x + p * c[e].y;
                    }
                } else {                           // pairs of neighbours in a (vector u) and in b (vector u + n_rot)
#pragma unroll
                    for (int v = 0; v < 2; ++v) {
                        float2 c[P];
                        Table<E, HALF>::read(cp, u + v * j.n_rot, half, c);
#pragma unroll
                        for (int e = 0; e < P; ++e) {
                            const float p = x[v][2 * e], q = x[v][2 * e + 1];
                            x[v][2 * e] = p * c[e].x - q * c[e].y;
                            x[v][2 * e + 1] = q * c[e].x + p * c[e].y;
                        }
                    }
                }
            }
            if (!APPEND || h < j.Hq) {
                T *o = static_cast<T *>(j.dst) + t * j.d_ts + h * j.d_hs;
                store_pack<T, E>(o + oa, x[0]);
                if (two) store_pack<T, E>(o + ob, x[1]);
            } else if (const int64_t r = row[wk.t]; r >= 0) {
                const bool is_k = h < j.Hq + j.Hkv;
                __half *o = (is_k ? j.k_cache : j.v_cache) + (r * j.Hkv + h - j.Hq - (is_k ? 0 : j.Hkv)) * j.D;
                store_pack<__half, E>(o + oa, x[0]);
                if (two) store_pack<__half, E>(o + ob, x[1]);
            }
        }
    }
    if (APPEND && hblk == 0 && (j.weight || j.slot_pos)) {
        for (int i = threadIdx.x; i < nt * j.Hkv; i += blockDim.x) {
            const int tok = i / j.Hkv, hd = i - tok * j.Hkv;
            const int64_t r = row[tok];
            if (r < 0) continue;
            const int64_t s = r / j.max_ctx, at = (s * j.Hkv + hd) * j.max_ctx + (r - s * j.max_ctx);
            if (j.weight) j.weight[at] = 0.f;
            if (j.slot_pos) j.slot_pos[at] = j.pos[t0 + tok];
        }
    }
}

template <typename T, int E, bool APPEND>
int rope_go(const RopeJob &j, unsigned grid, unsigned threads, size_t smem, cudaStream_t s) {
    if (j.r.layout == LI_ROPE_HALF)
        return (int)launch_pdl(rope_kernel<T, E, true, APPEND>, dim3(grid), dim3(threads), smem, s, true, j);
    return (int)launch_pdl(rope_kernel<T, E, false, APPEND>, dim3(grid), dim3(threads), smem, s, true, j);
}

// Launches with the widest vectors that sizes and addresses allow, in blocks
// of whole tokens with about 2 kRopeBatch units a thread; a call of few tokens
// is split over the heads too, so that it still spreads over the SMs.
template <typename T, bool APPEND>
int rope_launch(RopeJob &j, int e_max, cudaStream_t s) {
    int E = e_max;
    while (E > 1 && (j.r.rope_dim % (2 * E) || (j.D - j.r.rope_dim) % E)) E >>= 1;
    j.n_rot = j.r.rope_dim / (2 * E);
    j.units = j.n_rot + (j.D - j.r.rope_dim + 2 * E - 1) / (2 * E);      // at most 256: head_dim <= 512
    const int64_t per_tok = (int64_t)j.heads * j.units, all = per_tok * j.n_tokens;
    const int want = 2 * kRopeBatch * kRopeThreads;                     // two rounds a thread
    // units per block: all SMs busy first, then two rounds a thread
    int64_t share = (all + num_sms() - 1) / num_sms();
    share = share < kRopeThreads ? kRopeThreads : share < want ? share : want;
    j.tb = 1;
    j.hb = j.heads;
    if (per_tok > share) {
        const int64_t blocks = (per_tok + share - 1) / share;           // of about equally many heads
        j.hb = (int)((j.heads + blocks - 1) / blocks);
    } else {
        j.tb = (int)(share / per_tok);
        const int tb_max = 16384 / (8 + 4 * j.r.rope_dim);              // 16 KB of angles
        if (j.tb > tb_max) j.tb = tb_max;
        if (j.tb > kRopeThreads) j.tb = kRopeThreads;                   // small heads: a thread holds one token's row
        if (j.tb > j.n_tokens) j.tb = j.n_tokens;
    }
    j.n_hblk = (j.heads + j.hb - 1) / j.hb;
    // as many heads at once as 256 threads hold, in rounds of about equally many
    const int fit = kRopeThreads / j.units;
    j.np = (j.hb + fit - 1) / fit;
    j.hp = (j.hb + j.np - 1) / j.np;
    int threads = (j.hp * j.units + 31) / 32 * 32;
    if (threads < j.tb) threads = (j.tb + 31) / 32 * 32;                // a token each for the cache rows
    const int64_t grid = (int64_t)((j.n_tokens + j.tb - 1) / j.tb) * j.n_hblk;
    if (grid > 0x7fffffff) return LI_ERR_BAD_SHAPE;
    const size_t smem = (size_t)j.tb * (4 * j.r.rope_dim + (APPEND ? 8 : 0));
    if constexpr (sizeof(T) == 2)
        if (E == 8) return rope_go<T, 8, APPEND>(j, (unsigned)grid, (unsigned)threads, smem, s);
    switch (E) {
    case 4: return rope_go<T, 4, APPEND>(j, (unsigned)grid, (unsigned)threads, smem, s);
    case 2: return rope_go<T, 2, APPEND>(j, (unsigned)grid, (unsigned)threads, smem, s);
    default: return rope_go<T, 1, APPEND>(j, (unsigned)grid, (unsigned)threads, smem, s);
    }
}

template <bool APPEND>
int rope_dispatch(RopeJob &j, int dtype, int e_max, cudaStream_t s) {
    if (dtype == LI_DTYPE_F32) return rope_launch<float, APPEND>(j, e_max < 4 ? e_max : 4, s);
    if (dtype == LI_DTYPE_F16) return rope_launch<__half, APPEND>(j, e_max, s);
    return rope_launch<__nv_bfloat16, APPEND>(j, e_max, s);
}

// Elements per vector (a power of two up to e) that p and stride allow.
int vec_of(int e, const void *p, int64_t stride, int elem) {
    while (e > 1 && ((uintptr_t)p % (size_t)(e * elem) || stride % e)) e >>= 1;
    return e;
}

// Rows of `row` elements, `stride` apart: neighbours would overlap.
bool overlap(int n, int64_t stride, int64_t row) { return n > 1 && stride < row && stride > -row; }

int elem_size(int dtype) {
    return dtype == LI_DTYPE_F32 ? 4 : dtype == LI_DTYPE_F16 || dtype == LI_DTYPE_BF16 ? 2 : 0;
}

}  // namespace
}  // namespace li

using namespace li;

extern "C" int li_launch_rope(const li_rope *R, int dtype, const void *x, void *dst, const int32_t *pos, int n_tokens,
                              int n_heads, int64_t x_token_stride, int64_t x_head_stride, int64_t dst_token_stride,
                              int64_t dst_head_stride, int transpose, void *stream) {
    if (!R || !x || !dst || !pos || n_tokens < 0 || n_heads < 0) return LI_ERR_BAD_ARG;
    const int es = elem_size(dtype);
    if (!es) return LI_ERR_UNSUPPORTED;
    RopeJob j = {};
    if (const int rc = rope_args(R, &j.r)) return rc;
    if ((uintptr_t)x % es || (uintptr_t)dst % es || (uintptr_t)pos & 3u) return LI_ERR_MISALIGNED;
    if (n_tokens == 0 || n_heads == 0) return 0;
    if (overlap(n_tokens, dst_token_stride, R->head_dim) || overlap(n_heads, dst_head_stride, R->head_dim))
        return LI_ERR_BAD_SHAPE;
    j.x = x; j.dst = dst; j.pos = pos;
    j.x_ts = x_token_stride; j.x_hs = x_head_stride; j.d_ts = dst_token_stride; j.d_hs = dst_head_stride;
    j.n_tokens = n_tokens; j.heads = n_heads; j.D = R->head_dim;
    j.sin_sign = transpose ? -1.f : 1.f;
    int e = vec_of(16 / es, x, x_token_stride, es);
    e = vec_of(e, x, x_head_stride, es);
    e = vec_of(e, dst, dst_token_stride, es);
    e = vec_of(e, dst, dst_head_stride, es);
    return rope_dispatch<false>(j, dtype, e, (cudaStream_t)stream);
}

extern "C" int li_launch_kv_append(const li_kv_cache *C, const li_rope *R, int dtype, const void *q, int64_t q_stride,
                                   void *q_out, int64_t q_out_stride, int n_q_heads, const void *k, int64_t k_stride,
                                   const void *v, int64_t v_stride, const int32_t *pos, const int32_t *seq,
                                   const int32_t *slot, int n_tokens, void *stream) {
    if (const int rc = check_kv_cache(C)) return rc;
    if (!k || !v || !pos || n_tokens < 0 || (q && (!q_out || n_q_heads <= 0))) return LI_ERR_BAD_ARG;
    const int es = elem_size(dtype);
    if (!es) return LI_ERR_UNSUPPORTED;
    if (!seq && n_tokens > C->n_seqs) return LI_ERR_BAD_SHAPE;
    RopeJob j = {};
    j.r.layout = LI_ROPE_HALF;
    j.r.mag = 1.f;
    if (R) {
        if (const int rc = rope_args(R, &j.r)) return rc;
        if (R->head_dim != C->head_dim) return LI_ERR_BAD_SHAPE;
    }
    if ((uintptr_t)k % es || (uintptr_t)v % es || (uintptr_t)q % es || (uintptr_t)q_out % es ||
        ((uintptr_t)pos | (uintptr_t)seq | (uintptr_t)slot) & 3u)
        return LI_ERR_MISALIGNED;
    if (n_tokens == 0) return 0;
    j.x = q; j.dst = q_out; j.pos = pos;
    j.Hq = q ? n_q_heads : 0; j.Hkv = C->n_kv_heads; j.D = C->head_dim;
    if ((int64_t)j.Hq + 2ll * j.Hkv > (1 << 24)) return LI_ERR_BAD_SHAPE;
    if (q && overlap(n_tokens, q_out_stride, (int64_t)j.Hq * j.D)) return LI_ERR_BAD_SHAPE;
    j.x_ts = q_stride; j.x_hs = j.D; j.d_ts = q_out_stride; j.d_hs = j.D;
    j.n_tokens = n_tokens; j.heads = j.Hq + 2 * j.Hkv;
    j.sin_sign = 1.f;
    j.k = k; j.v = v; j.k_ts = k_stride; j.v_ts = v_stride;
    j.n_seqs = C->n_seqs; j.max_ctx = C->max_ctx;
    j.seq = seq; j.slot = slot; j.len = C->len;
    j.k_cache = static_cast<__half *>(C->k); j.v_cache = static_cast<__half *>(C->v);
    j.weight = C->weight; j.slot_pos = C->slot_pos;
    int e = vec_of(16 / es, k, k_stride, es);
    e = vec_of(e, v, v_stride, es);
    if (q) e = vec_of(vec_of(e, q, q_stride, es), q_out, q_out_stride, es);
    return rope_dispatch<true>(j, dtype, e, (cudaStream_t)stream);
}
