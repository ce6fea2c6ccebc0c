// attn_selected.hip — attention of a packed batch's rows over the blocks of the int8
// cache that each row's list names (AttentionI8Selected, 133).
#include <hip/hip_runtime.h>

#include "holo_kernels.h"
#include "packed_batch.h"

namespace holo {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// General form: one wavefront a token and head, any head_dim, block and alignment.
struct BlockSrc {
    const int8_t *kp, *vp;
    const float *ks, *vs;
    uint32_t D, block;
    __device__ float k(uint32_t j, uint32_t d) const { return float(kp[uint64_t(j) * D + d]); }
    __device__ float v(uint32_t j, uint32_t d) const { return float(vp[uint64_t(j) * D + d]); }
    __device__ float k_scale(uint32_t j) const { return ks[j / block]; }
    __device__ float v_scale(uint32_t j) const { return vs[j / block]; }
};

template <class E, int kDims>
__global__ __launch_bounds__(256) void rows_kernel(AttnSelectedArgs s, float mul) {
    typedef typename E::T T;
    __shared__ float qs[4][64 * kDims];
    const AttnBlocksArgs &a = s.a;
    if (blockIdx.x == 0) check_starts(a.pb);
    const uint32_t wave = pk_uni(threadIdx.x >> 6), lane = threadIdx.x & 63u;
    const uint64_t item = uint64_t(blockIdx.x) * 4 + wave;
    const uint32_t tok = uint32_t(item / a.H), h = uint32_t(item % a.H);
    if (tok >= a.pb.tokens) return;
    const uint32_t b = last_at_most(a.pb.batch, tok, [&](uint32_t s) { return start_of(a.pb, s); });
    const uint32_t r0 = start_of(a.pb, b), r1 = start_of(a.pb, b + 1);
    if (tok < r0 || tok >= r1) return;
    const T *q = static_cast<const T *>(a.q) + uint64_t(tok) * a.q_stride + uint64_t(h) * a.D;
    for (uint32_t d = lane; d < a.D; d += 64) qs[wave][d] = E::widen(q[d]) * mul;
    const uint32_t kh = h / (a.H / a.Hkv), sees = visible_keys(a.lens[b], r1 - r0, tok - r0, a.bucket);
    const uint64_t plane = uint64_t(b) * a.Hkv + kh, nb = (uint64_t(a.bucket) + a.block - 1) / a.block;
    const BlockSrc src{a.kq + plane * a.bucket * a.D, a.vq + plane * a.bucket * a.D,
                       a.ks + plane * nb, a.vs + plane * nb, a.D, a.block};
    const int32_t *list = s.blocks + (uint64_t(tok) * a.Hkv + kh) * s.top;
    RowState<kDims> st;
    for (uint32_t e = 0; e < s.top; ++e) {
        const int64_t j = list[e];
        if (j < 0 || uint64_t(j) * a.block >= sees) continue;
        const uint64_t to = uint64_t(j + 1) * a.block;
        st.keys(qs[wave], a.D, uint32_t(j) * a.block, uint32_t(to < sees ? to : sees), src);
    }
    T *out = static_cast<T *>(a.out) + (uint64_t(tok) * a.H + h) * a.D;
    st.write(a.D, [&](uint32_t d, float v) { out[d] = E::narrow(v); });
}

template <class E>
void launch(const AttnSelectedArgs &s, float mul, hipStream_t stream) {
    const uint32_t grid = uint32_t(attn_selected_threads(s) / 256);
    if (s.a.D <= 128) rows_kernel<E, 2><<<grid, 256, 0, stream>>>(s, mul);
    else rows_kernel<E, kPackedMaxDim / 64><<<grid, 256, 0, stream>>>(s, mul);
}

}  // namespace

size_t attn_selected_scratch_bytes(const AttnSelectedArgs &) { return 0; }

uint64_t attn_selected_threads(const AttnSelectedArgs &s) {
    return (uint64_t(s.a.pb.tokens) * s.a.H + 3) / 4 * 256;
}

hipError_t launch_attn_selected(const AttnSelectedArgs &s, void *, hipStream_t stream) {
    const float mul = kLog2e / s.a.score_scale;
    if (s.a.dtype == 7) launch<Bf16>(s, mul, stream);
    else if (s.a.dtype == 6) launch<F16>(s, mul, stream);
    else launch<F32>(s, mul, stream);
    return hipGetLastError();
}

}  // namespace holo
