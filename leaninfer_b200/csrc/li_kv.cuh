// Shared pieces of the KV-cache operators (li_rope.cu, li_kvattn.cu,
// li_kvevict.cu): the host check of a cache descriptor and the rotary
// parameters in the form the kernels read.
#pragma once
#include "li_common.cuh"

#include <atomic>

namespace li {

constexpr int kKvD = 128;              // head_dim of the cache (the only built size)
constexpr int kRopeMaxDim = 512;

// 0, or the status a bad descriptor is refused with. Lengths live on the
// device and are checked by the kernels.
inline int check_kv_cache(const li_kv_cache *C) {
    if (!C || C->n_seqs < 0 || C->max_ctx <= 0 || C->n_kv_heads <= 0 || C->n_prefix < 0) return LI_ERR_BAD_ARG;
    if (!C->k || !C->v || !C->len) return LI_ERR_BAD_ARG;
    if (C->n_prefix > 0 && (!C->k_prefix || !C->v_prefix)) return LI_ERR_BAD_ARG;
    if (C->head_dim != kKvD) return LI_ERR_UNSUPPORTED;
    if (!aligned16(C->k) || !aligned16(C->v)) return LI_ERR_MISALIGNED;
    if (C->n_prefix > 0 && (!aligned16(C->k_prefix) || !aligned16(C->v_prefix))) return LI_ERR_MISALIGNED;
    if (((uintptr_t)C->len & 3u) || ((uintptr_t)C->weight & 3u) || ((uintptr_t)C->slot_pos & 3u))
        return LI_ERR_MISALIGNED;
    // (sequence, kv head) pairs stay below 2^31, (sequence, kv head, slot) counts below 2^40: more than any device
    // holds, and no size made of them overflows
    const int64_t pairs = (int64_t)C->n_seqs * C->n_kv_heads;
    if (pairs >= (1ll << 31) || pairs * C->max_ctx >= (1ll << 40)) return LI_ERR_BAD_SHAPE;
    return 0;
}

// Lets a kernel take `smem` bytes of dynamic shared memory on the current
// device, once per device (bit d of `done`: set on device d).
template <typename Kernel>
int allow_smem(Kernel kernel, size_t smem, std::atomic<uint64_t> &done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0ull;
    if (done.load(std::memory_order_relaxed) & bit) return 0;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return (int)e;
}

// li_rope as the kernels read it: the frequency of pair i in turns per
// position (angle / 2 pi), scaling included, divided by freq_factors[i] on
// the device.
struct RopeArgs {
    int layout, rope_dim;
    float mag;                         // magnitude m of the rotated values
    const float *factors;              // [rope_dim / 2] or nullptr
    double turns[kRopeMaxDim / 2];
};

// Fills *a from R; 0 or a status.
int rope_args(const li_rope *R, RopeArgs *a);

// cos and sin of pair i of the token at position pos, times the magnitude.
// The turn count is reduced to (-1/2, 1/2] in double, so the float argument
// of sincospif carries 24 bits of the angle: up to positions of about 2^24 the
// error is that of an angle known to 2^-25 of a half turn. Beyond, the
// frequency's own error shows (rope_args): for bases of 100 and more up to
// 2^-22 of a turn at the largest int32, 2^-17 for a base of 1.01.
__device__ __forceinline__ float2 rope_cos_sin(const RopeArgs &a, int pos, int i) {
    double t = (double)pos * a.turns[i];
    if (a.factors) t /= (double)a.factors[i];
    t -= rint(t);
    float sn, cs;
    sincospif((float)(2.0 * t), &sn, &cs);
    return make_float2(cs * a.mag, sn * a.mag);
}

// li_launch_attn_kv_decode, with an optional output gate: out = o *
// sigmoid(gate), gate [n_seqs][gate_stride] laid out as q (nullptr: none).
int attn_kv_decode(const li_kv_cache *C, const float *q, int64_t q_stride, int n_q_heads, float scale, float *out,
                   float decay, const float *gate, int64_t gate_stride, void *workspace, size_t workspace_bytes,
                   void *stream);

}  // namespace li
