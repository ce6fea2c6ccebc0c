// packed_batch.h — what the packed-batch kernels (attn_packed.hip, attn_blocks.hip,
// kv_blocks.hip) share: finding a workgroup's sequence among the device-resident
// offsets, widening and narrowing, and the attention of one row at a time.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "holo_kernels.h"

namespace holo {

// A value every lane holds alike, moved to a scalar register.
__device__ __forceinline__ uint32_t pk_uni(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }

__device__ __forceinline__ uint32_t start_of(const PackedBatch &pb, uint32_t s) {
    const uint32_t v = pb.starts[s];
    return v < pb.tokens ? v : pb.tokens;
}

// The largest s in [0, n) with at(s) <= t, 0 if there is none, for `at` that does
// not decrease: the 64 lanes of a wavefront probe 64 places a step, so 4096
// sequences take two steps of loads. Every lane gets the answer; any `at` ends
// after the same steps with some s in [0, n).
template <class F>
__device__ __forceinline__ uint32_t last_at_most(uint32_t n, uint64_t t, F at) {
    uint32_t lo = 0, hi = n;
    const uint32_t lane = threadIdx.x & 63u;
    while (hi - lo > 1) {
        const uint32_t step = (hi - lo + 63) / 64;
        const uint64_t s = lo + uint64_t(lane) * step;
        const uint64_t hit = __ballot(s < hi && at(uint32_t(s)) <= t);
        const uint32_t at_lane = hit ? 63u - uint32_t(__builtin_clzll(hit)) : 0u;
        lo = pk_uni(lo + at_lane * step);
        hi = pk_uni(hi - lo > step ? lo + step : hi);
    }
    return lo;
}

// The sequence of place `t` where sequence s owns places [floor(starts[s] m / unit) +
// s, floor(starts[s + 1] m / unit) + s + 1): as many as its rows times m fill units of
// `unit`, or one more, so that neither a prefix sum nor the lengths are needed on the
// host. (tokens * m < 2^30.) Its first and one-past-last row and the place's number
// in it; false for a place that no unit of the sequence takes. As last_at_most, with
// the bounds taken from the probes of its last step.
struct Place {
    uint32_t b, lo, hi, unit;
};
__device__ __forceinline__ bool place_of(const PackedBatch &pb, uint32_t m, uint32_t unit, uint32_t t, Place *o) {
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t lo = 0, n = pb.batch, v;
    int at;
    for (;;) {
        const uint32_t step = (n + 63) / 64;
        const uint64_t s = lo + uint64_t(lane) * step;
        v = start_of(pb, s < pb.batch ? uint32_t(s) : pb.batch);
        const uint64_t hit = __ballot(lane * uint64_t(step) < n && v * m / unit + s <= t);
        at = hit ? 63 - __builtin_clzll(hit) : 0;
        lo = pk_uni(lo + at * step);
        if (step == 1) break;
        n = pk_uni(pb.batch - lo < step ? pb.batch - lo : step);
    }
    o->b = lo;
    o->lo = __builtin_amdgcn_readlane(v, at);
    o->hi = at < 63 ? __builtin_amdgcn_readlane(v, at + 1) : pk_uni(start_of(pb, lo + 1));
    const uint32_t first = o->lo * m / unit + lo;
    o->unit = t - first;
    return o->hi > o->lo && t >= first && o->unit * unit < (o->hi - o->lo) * m;
}

// Bit 8 of *err if the offsets decrease or pass `tokens`; the threads of one
// workgroup call it.
__device__ __forceinline__ void check_starts(const PackedBatch &pb) {
    bool bad = false;
    for (uint32_t s = threadIdx.x; s <= pb.batch; s += blockDim.x) {
        const uint32_t v = pb.starts[s];
        bad |= v > pb.tokens || (s && v < pb.starts[s - 1]);
    }
    if (bad) atomicOr(pb.err, 8);
}

struct Bf16 {
    static __device__ __forceinline__ float widen(uint16_t b) { return __uint_as_float(uint32_t(b) << 16); }
    // to nearest, ties to even; a NaN stays one
    static __device__ __forceinline__ uint16_t narrow(float v) {
        const uint32_t u = __float_as_uint(v);
        if ((u & 0x7fffffffu) > 0x7f800000u) return uint16_t((u >> 16) | 0x40u);
        return uint16_t((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
    }
    typedef uint16_t T;
};
struct F16 {
    static __device__ __forceinline__ float widen(uint16_t b) { return float(__builtin_bit_cast(_Float16, b)); }
    static __device__ __forceinline__ uint16_t narrow(float v) { return __builtin_bit_cast(uint16_t, _Float16(v)); }
    typedef uint16_t T;
};
struct F32 {
    static __device__ __forceinline__ float widen(float v) { return v; }
    static __device__ __forceinline__ float narrow(float v) { return v; }
    typedef float T;
};

// One wavefront's query row over `keys` keys: q (D floats in LDS, scaled by
// log2(e) / s), K row j's elements src.k(j, d) times src.k_scale(j), V's likewise.
// A lane takes one key of 64 for the scores and every 64th dim of the result, so
// any D and any layout go. Softmax in f32 with a running maximum and sum; keys at
// and past `keys` are not read. A row whose scores are all -inf is NaN (0 / 0), a
// row without keys zeros.
template <int kDims, class Src, class Put>
__device__ __forceinline__ void attend_row(const float *q, uint32_t D, uint32_t keys, const Src &src, Put put) {
    const uint32_t lane = threadIdx.x & 63u;
    float m = -INFINITY, l = 0.0f, acc[kDims];
#pragma unroll
    for (int i = 0; i < kDims; ++i) acc[i] = 0.0f;
    for (uint32_t j0 = 0; j0 < keys; j0 += 64) {
        const uint32_t n = keys - j0 < 64 ? keys - j0 : 64;
        float s = -INFINITY;
        if (lane < n) {
            float dot = 0.0f;
            for (uint32_t d = 0; d < D; ++d) dot = fmaf(q[d], src.k(j0 + lane, d), dot);
            s = dot * src.k_scale(j0 + lane);
        }
        float mn = s;
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) mn = fmaxf(mn, __shfl_xor(mn, o, 64));
        mn = fmaxf(mn, m);
        const float ref = mn == -INFINITY ? 0.0f : mn;
        const float al = m == -INFINITY ? 0.0f : exp2f(m - ref);
        const float p = lane < n ? (s == -INFINITY ? 0.0f : exp2f(s - ref)) : 0.0f;
        float sum = p;
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
        l = l * al + sum;
        m = mn;
#pragma unroll
        for (int i = 0; i < kDims; ++i) acc[i] *= al;
        for (uint32_t j = 0; j < n; ++j) {
            const float w = __shfl(p, int(j), 64) * src.v_scale(j0 + j);
#pragma unroll
            for (int i = 0; i < kDims; ++i)
                if (lane + 64u * i < D) acc[i] = fmaf(w, src.v(j0 + j, lane + 64u * i), acc[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < kDims; ++i)
        if (lane + 64u * i < D) put(lane + 64u * i, keys ? acc[i] / l : 0.0f);
}

}  // namespace holo
