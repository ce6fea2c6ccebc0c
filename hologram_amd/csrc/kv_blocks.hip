// kv_blocks.hip — int8 append with one power-of-two scale a block of rows
// (KvBlockAppend, 127), in place.
#include <hip/hip_runtime.h>

#include "holo_kernels.h"
#include "packed_batch.h"

namespace holo {
namespace {

constexpr uint32_t kThreads = 256;

// The least 2^e, e >= -126, with v <= 127 * 2^e, for a finite v > 0 given by its
// bits: 127 is 1.984375 * 2^6, so e is v's exponent less 6, one more where v's
// mantissa passes 1.984375. Exact, subnormal v included (the floor takes them).
__device__ __forceinline__ float block_scale(uint32_t bits) {
    const int e = int(bits >> 23) - 127 - 6 + ((bits & 0x7fffffu) > 0x7e0000u);
    return __uint_as_float(uint32_t((e < -126 ? -126 : e) + 127) << 23);
}

__device__ __forceinline__ int8_t to_i8(float r) {   // r finite
    return int8_t(rintf(fminf(fmaxf(r, -127.0f), 127.0f)));
}

// One workgroup a touched block and head. Sequence s owns the places [floor(
// starts[s] / block) + 2 s, floor(starts[s + 1] / block) + 2 (s + 1)) of the grid: n
// rows touch at most floor(n / block) + 2 blocks wherever they begin, so every
// touched block has a place and no prefix sum is needed.
template <class E>
__global__ __launch_bounds__(kThreads) void append_kernel(KvBlockArgs a) {
    __shared__ uint32_t top[kThreads / 64];
    const uint32_t kh = blockIdx.x % a.Hkv, place = blockIdx.x / a.Hkv, tid = threadIdx.x;
    if (blockIdx.x == 0) check_starts(a.pb);
    const uint32_t b = last_at_most(a.pb.batch, place, [&](uint32_t s) {
        return uint64_t(start_of(a.pb, s)) / a.block + 2ull * s;
    });
    const uint32_t r0 = start_of(a.pb, b), r1 = start_of(a.pb, b + 1);
    if (r1 <= r0) return;
    const uint64_t at = uint64_t(r0) / a.block + 2ull * b;
    if (place < at) return;
    const uint64_t pos = a.pos[b], end = pos + (r1 - r0);
    const uint64_t j = pos / a.block + (place - at), first = j * a.block;
    if (place == at && kh == 0 && tid == 0 && end > a.bucket) atomicOr(a.pb.err, 16);
    const uint64_t lo = first > pos ? first : pos;
    uint64_t hi = first + a.block < end ? first + a.block : end;
    hi = hi < a.bucket ? hi : a.bucket;
    if (lo >= hi) return;
    const uint64_t plane = uint64_t(b) * a.Hkv + kh;
    const uint32_t rows = uint32_t(hi - lo);
    const auto *nw = static_cast<const typename E::T *>(a.nw) + (r0 + (lo - pos)) * a.stride + uint64_t(kh) * a.D;
    uint32_t m = 0;   // of the magnitudes' bits: their order is the values', NaN and infinity on top
    for (uint32_t i = tid; i < rows * a.D; i += kThreads) {
        const uint32_t u = __float_as_uint(E::widen(nw[uint64_t(i / a.D) * a.stride + i % a.D])) & 0x7fffffffu;
        m = u > m ? u : m;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const uint32_t u = __shfl_xor(m, o, 64);
        m = u > m ? u : m;
    }
    if ((tid & 63u) == 0) top[tid >> 6] = m;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < kThreads / 64; ++w) m = top[w] > m ? top[w] : m;
    float s = m >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : m ? block_scale(m) : 0.0f;
    int8_t *rows0 = a.cache + (plane * a.bucket + first) * a.D;
    float *sp = a.scales + plane * ((uint64_t(a.bucket) + a.block - 1) / a.block) + j;
    const bool held = first < pos;
    const float old = held ? *sp : s;
    __syncthreads();   // every thread has read the block's scale
    if (held) {
        if (old != old || fabsf(old) > s) s = fabsf(old);
        if (s == s && old != s) {
            const float back = old / s;
            for (uint64_t i = tid; i < (lo - first) * a.D; i += kThreads) rows0[i] = to_i8(float(rows0[i]) * back);
        }
    }
    if (tid == 0) *sp = s;
    int8_t *dst = rows0 + (lo - first) * a.D;
    for (uint32_t i = tid; i < rows * a.D; i += kThreads) {
        const float x = E::widen(nw[uint64_t(i / a.D) * a.stride + i % a.D]);
        dst[i] = s > 0.0f ? to_i8(x / s) : int8_t(0);
    }
}

}  // namespace

hipError_t launch_kv_block_append(const KvBlockArgs &a, hipStream_t stream) {
    const uint32_t places = a.pb.tokens / a.block + 2 * a.pb.batch;
    const dim3 grid(places * a.Hkv);
    if (a.dtype == 7) append_kernel<Bf16><<<grid, kThreads, 0, stream>>>(a);
    else if (a.dtype == 6) append_kernel<F16><<<grid, kThreads, 0, stream>>>(a);
    else append_kernel<F32><<<grid, kThreads, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace holo
