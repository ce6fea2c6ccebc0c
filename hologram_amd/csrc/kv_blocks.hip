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

// Eight elements: their largest magnitude's bits, and them over a scale as int8.
template <class E>
struct Eight {
    uint4 raw[sizeof(typename E::T) / 2];
    __device__ __forceinline__ void load(const typename E::T *p) {
#pragma unroll
        for (uint32_t i = 0; i < sizeof raw / 16; ++i) raw[i] = reinterpret_cast<const uint4 *>(p)[i];
    }
    __device__ __forceinline__ float get(int i) const {
        const uint32_t *w = reinterpret_cast<const uint32_t *>(raw);
        if constexpr (sizeof(typename E::T) == 4) return __uint_as_float(w[i]);
        else return E::widen(uint16_t(w[i >> 1] >> (16 * (i & 1))));
    }
};

// One workgroup a touched block and head. Sequence s owns the places [floor(
// starts[s] / block) + 2 s, floor(starts[s + 1] / block) + 2 (s + 1)) of the grid: n
// rows touch at most floor(n / block) + 2 blocks wherever they begin, so every
// touched block has a place and no prefix sum is needed. The block's largest value
// is wanted before its first byte: in the wide form (16-byte rows) a thread keeps its
// eights of the rows in registers between the two, kHold of them, 64 rows of 128 dims;
// what is past those it reads again. A power-of-two scale divides by its reciprocal,
// exactly. Bound by the rows' bytes where they are many: 32 prompts of 1500 rows, 8 heads of
// 128 bf16, 98 MB in and 49 out, 29.5 us, 5.0 TB/s; by a launch and a workgroup's chain
// (search, offsets, rows, barrier, store) where each of 32 sequences has one row, 4.8 us (an
// empty launch, queued: 1.6). Between them both: 16 prompts of 100 to 1500 rows, 26 MB, 10 us,
// 2.6 TB/s (31 us in the narrow form, an element a thread).
constexpr uint32_t kHold = 4;
template <class E, bool kWide>
__global__ __launch_bounds__(kThreads) void append_kernel(KvBlockArgs a) {
    __shared__ uint32_t top[kThreads / 64];
    const uint32_t kh = blockIdx.x % a.Hkv, place = blockIdx.x / a.Hkv, tid = threadIdx.x;
    if (blockIdx.x == 0) check_starts(a.pb);
    const uint32_t b = last_at_most(a.pb.batch, place, [&](uint32_t s) {
        return uint64_t(start_of(a.pb, s) / a.block) + 2ull * s;
    });
    const uint32_t r0 = start_of(a.pb, b), r1 = start_of(a.pb, b + 1);
    if (r1 <= r0) return;
    const uint64_t at = uint64_t(r0 / a.block) + 2ull * b;
    if (place < at) return;
    const uint64_t pos = a.pos[b], end = pos + (r1 - r0);
    const uint64_t j = uint64_t(uint32_t(pos) / a.block) + (place - at), first = j * a.block;
    if (place == at && kh == 0 && tid == 0 && end > a.bucket) atomicOr(a.pb.err, 16);
    const uint64_t lo = first > pos ? first : pos;
    uint64_t hi = first + a.block < end ? first + a.block : end;
    hi = hi < a.bucket ? hi : a.bucket;
    if (lo >= hi) return;
    const uint64_t plane = uint64_t(b) * a.Hkv + kh;
    const uint32_t rows = uint32_t(hi - lo);
    const auto *nw = static_cast<const typename E::T *>(a.nw) + (r0 + (lo - pos)) * a.stride + uint64_t(kh) * a.D;
    int8_t *rows0 = a.cache + (plane * a.bucket + first) * a.D;
    float *sp = a.scales + plane * ((uint64_t(a.bucket) + a.block - 1) / a.block) + j;
    const bool held = first < pos;
    const float old = held ? *sp : 0.0f;
    uint32_t m = 0;   // of the magnitudes' bits: their order is the values', NaN and infinity on top
    auto see = [&](float x) {
        const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
        m = u > m ? u : m;
    };
    const uint32_t per = a.D / 8, eights = rows * per;      // (kWide)
    Eight<E> keep[kHold];
    auto eight_at = [&](uint32_t i) { return nw + uint64_t(i / per) * a.stride + 8 * (i % per); };
    if constexpr (kWide) {
#pragma unroll
        for (uint32_t q = 0; q < kHold; ++q)
            if (tid + q * kThreads < eights) keep[q].load(eight_at(tid + q * kThreads));
#pragma unroll
        for (uint32_t q = 0; q < kHold; ++q)
            if (tid + q * kThreads < eights)
#pragma unroll
                for (int e = 0; e < 8; ++e) see(keep[q].get(e));
        for (uint32_t i = tid + kHold * kThreads; i < eights; i += kThreads) {
            Eight<E> x;
            x.load(eight_at(i));
#pragma unroll
            for (int e = 0; e < 8; ++e) see(x.get(e));
        }
    } else {
        for (uint32_t i = tid; i < rows * a.D; i += kThreads) see(E::widen(nw[uint64_t(i / a.D) * a.stride + i % a.D]));
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const uint32_t u = __shfl_xor(m, o, 64);
        m = u > m ? u : m;
    }
    if ((tid & 63u) == 0) top[tid >> 6] = m;
    __syncthreads();       // (and every thread has read the block's scale)
#pragma unroll
    for (uint32_t w = 0; w < kThreads / 64; ++w) m = top[w] > m ? top[w] : m;
    float s = m >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : m ? block_scale(m) : 0.0f;
    if (held) {
        if (old != old || fabsf(old) > s) s = fabsf(old);
        if (s == s && old != s) {
            const float back = old / s;
            const uint32_t bytes = uint32_t(lo - first) * a.D;
            if constexpr (kWide) {
                for (uint32_t i = tid; i < bytes / 8; i += kThreads) {
                    uint2 v = reinterpret_cast<uint2 *>(rows0)[i];
                    uint32_t w[2] = {v.x, v.y};
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        uint32_t r = 0;
#pragma unroll
                        for (int e = 0; e < 4; ++e) r |= uint32_t(uint8_t(to_i8(float(int8_t(w[q] >> (8 * e))) * back))) << (8 * e);
                        w[q] = r;
                    }
                    reinterpret_cast<uint2 *>(rows0)[i] = make_uint2(w[0], w[1]);
                }
            } else {
                for (uint32_t i = tid; i < bytes; i += kThreads) rows0[i] = to_i8(float(rows0[i]) * back);
            }
        }
    }
    if (tid == 0) *sp = s;
    int8_t *dst = rows0 + (lo - first) * a.D;
    // (a scale that is no normal power of two can only be one that the block had)
    const uint32_t sb = __float_as_uint(s);
    const bool power = (sb & 0x7fffffu) == 0 && sb >= 0x00800000u && sb <= 0x7e000000u, some = s > 0.0f;
    const float inv = power ? 1.0f / s : 0.0f;
    auto quant = [&](float x) { return !some ? int8_t(0) : to_i8(power ? x * inv : x / s); };
    if constexpr (kWide) {
        auto store = [&](uint32_t i, const Eight<E> &x) {
            uint32_t w[2] = {0, 0};
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e >> 2] |= uint32_t(uint8_t(quant(x.get(e)))) << (8 * (e & 3));
            *reinterpret_cast<uint2 *>(dst + 8 * uint64_t(i)) = make_uint2(w[0], w[1]);
        };
#pragma unroll
        for (uint32_t q = 0; q < kHold; ++q)
            if (tid + q * kThreads < eights) store(tid + q * kThreads, keep[q]);
        for (uint32_t i = tid + kHold * kThreads; i < eights; i += kThreads) {
            Eight<E> x;
            x.load(eight_at(i));
            store(i, x);
        }
    } else {
        for (uint32_t i = tid; i < rows * a.D; i += kThreads)
            dst[i] = quant(E::widen(nw[uint64_t(i / a.D) * a.stride + i % a.D]));
    }
}

uint32_t blocks_of(const KvBlockArgs &a) { return (a.pb.tokens / a.block + 2 * a.pb.batch) * a.Hkv; }

template <class E>
void launch(const KvBlockArgs &a, hipStream_t stream) {
    const dim3 grid(blocks_of(a));
    const bool wide = a.D % 8 == 0 && a.stride * sizeof(typename E::T) % 16 == 0 &&
                      reinterpret_cast<uintptr_t>(a.nw) % 16 == 0 && reinterpret_cast<uintptr_t>(a.cache) % 8 == 0;
    if (wide) append_kernel<E, true><<<grid, kThreads, 0, stream>>>(a);
    else append_kernel<E, false><<<grid, kThreads, 0, stream>>>(a);
}

}  // namespace

uint64_t kv_block_append_threads(const KvBlockArgs &a) { return uint64_t(blocks_of(a)) * kThreads; }

hipError_t launch_kv_block_append(const KvBlockArgs &a, hipStream_t stream) {
    if (a.dtype == 7) launch<Bf16>(a, stream);
    else if (a.dtype == 6) launch<F16>(a, stream);
    else launch<F32>(a, stream);
    return hipGetLastError();
}

}  // namespace holo
