// attn_packed.hip — causal grouped-query attention of a packed batch of prompts
// (AttentionPacked, 126).
#include <hip/hip_runtime.h>

#include <math.h>

#include "holo_kernels.h"
#include "packed_batch.h"

namespace holo {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// ---------------------------------------------------------- general form ----
// One wavefront a token and head, any head_dim, stride and alignment.
template <class E>
struct RowSrc {
    const typename E::T *kp, *vp;
    uint64_t ks, vs;
    __device__ float k(uint32_t j, uint32_t d) const { return E::widen(kp[j * ks + d]); }
    __device__ float v(uint32_t j, uint32_t d) const { return E::widen(vp[j * vs + d]); }
    __device__ float k_scale(uint32_t) const { return 1.0f; }
    __device__ float v_scale(uint32_t) const { return 1.0f; }
};

template <class E, int kDims>
__global__ __launch_bounds__(256) void packed_rows_kernel(AttnPackedArgs a, float mul) {
    __shared__ float qs[4][64 * kDims];
    if (blockIdx.x == 0) check_starts(a.pb);
    const uint32_t wave = pk_uni(threadIdx.x >> 6), lane = threadIdx.x & 63u;
    const uint64_t item = uint64_t(blockIdx.x) * 4 + wave;
    const uint32_t tok = uint32_t(item / a.H), h = uint32_t(item % a.H);
    if (tok >= a.pb.tokens) return;
    const uint32_t b = last_at_most(a.pb.batch, tok, [&](uint32_t s) { return start_of(a.pb, s); });
    const uint32_t r0 = start_of(a.pb, b);
    if (tok < r0 || tok >= start_of(a.pb, b + 1)) return;
    typedef typename E::T T;
    const T *q = static_cast<const T *>(a.q) + uint64_t(tok) * a.q_stride + uint64_t(h) * a.D;
    for (uint32_t d = lane; d < a.D; d += 64) qs[wave][d] = E::widen(q[d]) * mul;
    const uint32_t kh = h / (a.H / a.Hkv);
    const RowSrc<E> src{static_cast<const T *>(a.k) + uint64_t(r0) * a.k_stride + uint64_t(kh) * a.D,
                        static_cast<const T *>(a.v) + uint64_t(r0) * a.v_stride + uint64_t(kh) * a.D,
                        a.k_stride, a.v_stride};
    T *out = static_cast<T *>(a.out) + (uint64_t(tok) * a.H + h) * a.D;
    attend_row<kDims>(qs[wave], a.D, tok - r0 + 1, src, [&](uint32_t d, float v) { out[d] = E::narrow(v); });
}

template <class E>
void launch_rows(const AttnPackedArgs &a, float mul, hipStream_t stream) {
    const uint32_t grid = uint32_t((uint64_t(a.pb.tokens) * a.H + 3) / 4);
    if (a.D <= 128) packed_rows_kernel<E, 2><<<grid, 256, 0, stream>>>(a, mul);
    else packed_rows_kernel<E, kPackedMaxDim / 64><<<grid, 256, 0, stream>>>(a, mul);
}

}  // namespace

hipError_t launch_attn_packed(const AttnPackedArgs &a, hipStream_t stream) {
    const float mul = kLog2e / a.score_scale;
    if (a.dtype == 7) launch_rows<Bf16>(a, mul, stream);
    else if (a.dtype == 6) launch_rows<F16>(a, mul, stream);
    else launch_rows<F32>(a, mul, stream);
    return hipGetLastError();
}

}  // namespace holo
