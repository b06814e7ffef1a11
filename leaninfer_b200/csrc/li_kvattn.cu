// Attention of one token per sequence over a shared prefix and the
// sequence's own cache slots, with the accumulation of each own slot's
// attention weight.
#include "li_kv.cuh"

LI_DEFINE_TU_STATUS(kvattn)

namespace li {
namespace {

struct KvAttnArgs {
    const float *q;
    int64_t q_stride;
    const __half *k, *v, *kp, *vp;
    const int32_t *len;
    int Hq, Hkv, G, max_ctx, n_prefix;
    float scale, decay;
    float *out, *weight;
};

// Block per (sequence, kv head), one q head after the other; a warp takes
// every fourth token (a lane holds four dims), the warps merge at the end.
__global__ void __launch_bounds__(128) kv_attn_kernel(KvAttnArgs a) {
    __shared__ float wm[4], wl[4], wo[4][kKvD], gm[16], gl[16];
    grid_dep_wait();
    grid_dep_launch_dependents();
    const int s = blockIdx.x / a.Hkv, j = blockIdx.x % a.Hkv;
    const int warp = threadIdx.x / kWarp, lane = threadIdx.x % kWarp;
    int n = a.len[s];
    if (n < 0 || n > a.max_ctx) {
        if (threadIdx.x == 0) atomicExch(&g_device_error, LI_ERR_BAD_ARG);
        n = 0;
    }
    const size_t row = (size_t)a.Hkv * kKvD, own0 = ((size_t)s * a.max_ctx * a.Hkv + j) * kKvD;
    auto at = [&](const __half *pre, const __half *own, int t) {
        const __half *p = t < a.n_prefix ? pre + (size_t)t * row + (size_t)j * kKvD
                                         : own + own0 + (size_t)(t - a.n_prefix) * row;
        const uint2 u = *reinterpret_cast<const uint2 *>(p + 4 * lane);
        const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&u.x));
        const float2 y = __half22float2(*reinterpret_cast<const __half2 *>(&u.y));
        return make_float4(x.x, x.y, y.x, y.y);
    };
    auto score = [&](const float4 q, int t) {
        const float4 k = at(a.kp, a.k, t);
        return warp_sum(q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w) * a.scale;
    };
    const int total = a.n_prefix + n;
    for (int g = 0; g < a.G; ++g) {
        const int h = j * a.G + g;
        const float4 q = *reinterpret_cast<const float4 *>(a.q + s * a.q_stride + (size_t)h * kKvD + 4 * lane);
        float m = -INFINITY, l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int t = warp; t < total; t += 4) {
            const float sc = score(q, t), mn = fmaxf(m, sc);
            const float al = m == -INFINITY ? 0.f : expf(m - mn), p = expf(sc - mn);
            const float4 v = at(a.vp, a.v, t);
            o.x = o.x * al + p * v.x; o.y = o.y * al + p * v.y; o.z = o.z * al + p * v.z; o.w = o.w * al + p * v.w;
            l = l * al + p;
            m = mn;
        }
        __syncthreads();
        *reinterpret_cast<float4 *>(&wo[warp][4 * lane]) = o;
        if (lane == 0) { wm[warp] = m; wl[warp] = l; }
        __syncthreads();
        float M = -INFINITY, L = 0.f, O = 0.f;
        for (int w = 0; w < 4; ++w) M = fmaxf(M, wm[w]);
        for (int w = 0; w < 4; ++w) {
            const float f = wm[w] == -INFINITY ? 0.f : expf(wm[w] - M);
            L += f * wl[w];
            O += f * wo[w][threadIdx.x];
        }
        a.out[((size_t)s * a.Hq + h) * kKvD + threadIdx.x] = total > 0 ? O / L : 0.f;
        if (threadIdx.x == 0) { gm[g] = M; gl[g] = L; }
    }
    if (!a.weight) return;
    __syncthreads();
    float *w = a.weight + ((size_t)s * a.Hkv + j) * a.max_ctx;
    for (int t = warp; t < n; t += 4) {
        float p = 0.f;
        for (int g = 0; g < a.G; ++g) {
            const float4 q = *reinterpret_cast<const float4 *>(a.q + s * a.q_stride + (size_t)(j * a.G + g) * kKvD +
                                                               4 * lane);
            p += expf(score(q, a.n_prefix + t) - gm[g]) / gl[g];
        }
        if (lane == 0) w[t] = a.decay == 0.f ? p : a.decay * w[t] + p;
    }
}

}  // namespace
}  // namespace li

using namespace li;

extern "C" {

size_t li_attn_kv_workspace_size(const li_kv_cache *C, int n_q_heads) {
    if (check_kv_cache(C) || C->n_seqs == 0 || n_q_heads <= 0) return 0;
    return 256;
}

int li_launch_attn_kv_decode(const li_kv_cache *C, const float *q, int64_t q_stride, int n_q_heads, float scale,
                             float *out, float decay, void *workspace, size_t workspace_bytes, void *stream) {
    if (const int rc = check_kv_cache(C)) return rc;
    if (!q || !out || n_q_heads <= 0 || !(decay >= 0.0f)) return LI_ERR_BAD_ARG;
    if (n_q_heads % C->n_kv_heads) return LI_ERR_BAD_SHAPE;
    if (n_q_heads / C->n_kv_heads > 16) return LI_ERR_UNSUPPORTED;
    if (!aligned16(q) || !aligned16(out) || q_stride % 4) return LI_ERR_MISALIGNED;
    if (C->n_seqs == 0) return 0;
    if (!workspace || workspace_bytes < li_attn_kv_workspace_size(C, n_q_heads)) return LI_ERR_WORKSPACE;
    if (!aligned16(workspace)) return LI_ERR_MISALIGNED;
    KvAttnArgs a = {};
    a.q = q; a.q_stride = q_stride;
    a.k = static_cast<const __half *>(C->k); a.v = static_cast<const __half *>(C->v);
    a.kp = static_cast<const __half *>(C->k_prefix); a.vp = static_cast<const __half *>(C->v_prefix);
    a.len = C->len; a.Hq = n_q_heads; a.Hkv = C->n_kv_heads; a.G = n_q_heads / C->n_kv_heads;
    a.max_ctx = C->max_ctx; a.n_prefix = C->n_prefix; a.scale = scale; a.decay = decay; a.out = out;
    a.weight = C->weight;
    return (int)launch_pdl(kv_attn_kernel, dim3((unsigned)(C->n_seqs * C->n_kv_heads)), dim3(128), 0,
                           (cudaStream_t)stream, true, a);
}

}  // extern "C"
