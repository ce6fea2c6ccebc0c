// attn_blocks.hip — attention of a packed batch's rows over the int8 cache with
// one scale a block of rows (AttentionI8Blocks, 128).
#include <hip/hip_runtime.h>

#include <math.h>

#include "holo_kernels.h"
#include "packed_batch.h"

namespace holo {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// Keys that row t of sequence b's n rows sees.
__device__ __forceinline__ uint32_t visible_keys(int64_t len, uint32_t n, uint32_t t, uint32_t bucket) {
    const int64_t v = len - int64_t(n - 1 - t);
    return v < 0 ? 0u : v > int64_t(bucket) ? bucket : uint32_t(v);
}

// ---------------------------------------------------------- general form ----
// One wavefront a token and head, any head_dim, block and alignment.
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
__global__ __launch_bounds__(256) void blocks_rows_kernel(AttnBlocksArgs a, float mul) {
    __shared__ float qs[4][64 * kDims];
    if (blockIdx.x == 0) check_starts(a.pb);
    const uint32_t wave = pk_uni(threadIdx.x >> 6), lane = threadIdx.x & 63u;
    const uint64_t item = uint64_t(blockIdx.x) * 4 + wave;
    const uint32_t tok = uint32_t(item / a.H), h = uint32_t(item % a.H);
    if (tok >= a.pb.tokens) return;
    const uint32_t b = last_at_most(a.pb.batch, tok, [&](uint32_t s) { return start_of(a.pb, s); });
    const uint32_t r0 = start_of(a.pb, b), r1 = start_of(a.pb, b + 1);
    if (tok < r0 || tok >= r1) return;
    typedef typename E::T T;
    const T *q = static_cast<const T *>(a.q) + uint64_t(tok) * a.q_stride + uint64_t(h) * a.D;
    for (uint32_t d = lane; d < a.D; d += 64) qs[wave][d] = E::widen(q[d]) * mul;
    const uint64_t plane = uint64_t(b) * a.Hkv + h / (a.H / a.Hkv);
    const uint64_t nb = (uint64_t(a.bucket) + a.block - 1) / a.block;
    const BlockSrc src{a.kq + plane * a.bucket * a.D, a.vq + plane * a.bucket * a.D,
                       a.ks + plane * nb, a.vs + plane * nb, a.D, a.block};
    T *out = static_cast<T *>(a.out) + (uint64_t(tok) * a.H + h) * a.D;
    attend_row<kDims>(qs[wave], a.D, visible_keys(a.lens[b], r1 - r0, tok - r0, a.bucket), src,
                      [&](uint32_t d, float v) { out[d] = E::narrow(v); });
}

template <class E>
void launch_rows(const AttnBlocksArgs &a, float mul, hipStream_t stream) {
    const uint32_t grid = uint32_t((uint64_t(a.pb.tokens) * a.H + 3) / 4);
    if (a.D <= 128) blocks_rows_kernel<E, 2><<<grid, 256, 0, stream>>>(a, mul);
    else blocks_rows_kernel<E, kPackedMaxDim / 64><<<grid, 256, 0, stream>>>(a, mul);
}

}  // namespace

size_t attn_blocks_scratch_bytes(const AttnBlocksArgs &) { return 0; }

hipError_t launch_attn_blocks(const AttnBlocksArgs &a, void *, hipStream_t stream) {
    const float mul = kLog2e / a.score_scale;
    if (a.dtype == 7) launch_rows<Bf16>(a, mul, stream);
    else if (a.dtype == 6) launch_rows<F16>(a, mul, stream);
    else launch_rows<F32>(a, mul, stream);
    return hipGetLastError();
}

}  // namespace holo
