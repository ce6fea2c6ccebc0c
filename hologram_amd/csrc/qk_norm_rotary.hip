// qk_norm_rotary.hip — q and k of a packed batch normed by the head and rotated by
// position (QkNormRotary, 130).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "holo_kernels.h"
#include "packed_tile.h"

namespace holo {
namespace {

// cos and sin of pos * freq. The product and its reduction to a quarter turn are f64:
// with n = rint(2 x / pi), x - n pi / 2 in two steps of one rounding each keeps 2^-50 of
// a radian for every |x| < 2^50, where f32 would lose the angle itself from some
// thousand positions on; what is left, at most pi / 4, is f32's.
__device__ __forceinline__ void turn(double pos, float freq, float *c, float *s) {
    const double x = pos * double(freq), low = fma(pos, double(freq), -x);
    const double n = rint(x * 0.63661977236758134308);
    double r = fma(-n, 1.57079632679489655800, x);
    r = fma(-n, 6.12323399573676603587e-17, r) + low;
    float sn, cs;
    sincosf(float(r), &sn, &cs);
    const int quarter = int(n - 4.0 * floor(n * 0.25));      // 0 to 3
    *c = quarter & 1 ? (quarter == 1 ? -sn : sn) : (quarter == 0 ? cs : -cs);
    *s = quarter & 1 ? (quarter == 1 ? cs : -cs) : (quarter == 0 ? sn : -sn);
}

// The position of token `tok` in its sequence (33 bits, pos[b] + t); false outside every
// sequence.
__device__ __forceinline__ bool position(const QkNormRotaryArgs &a, uint32_t tok, double *pos) {
    RowAt at;
    if (!row_of(a.pb, a.pos, tok, &at)) return false;
    *pos = double(at.of) + double(tok - at.lo);
    return true;
}

// General form: a wavefront a head's row, any head_dim, rotation and alignment.
template <class E>
__global__ __launch_bounds__(256) void rows_kernel(QkNormRotaryArgs a) {
    typedef typename E::T T;
    if (blockIdx.x == 0) check_starts(a.pb);
    const uint32_t lane = threadIdx.x & 63u, all = a.H + a.Hkv;
    const uint64_t item = uint64_t(blockIdx.x) * 4 + pk_uni(threadIdx.x >> 6);
    const uint32_t tok = uint32_t(item / all);
    uint32_t h = uint32_t(item - uint64_t(tok) * all);
    double pos;
    if (tok >= a.pb.tokens || !position(a, tok, &pos)) return;
    const int which = h >= a.H;
    h -= which ? a.H : 0;
    const T *x = static_cast<const T *>(a.x[which]) + uint64_t(tok) * a.stride[which] + uint64_t(h) * a.D;
    T *out = static_cast<T *>(a.out[which]) + (uint64_t(tok) * (which ? a.Hkv : a.H) + h) * a.D;
    const T *gamma = static_cast<const T *>(a.gamma[which]);
    float inv = 1.0f;
    const bool norm = a.norms >> which & 1;
    if (norm) {
        float sum = 0.0f;
        for (uint32_t d = lane; d < a.D; d += 64) {
            const float v = E::widen(x[d]);
            sum = fmaf(v, v, sum);
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
        inv = 1.0f / sqrtf(sum / float(a.D) + a.eps);
    }
    auto get = [&](uint32_t d) {
        const float v = E::widen(x[d]) * inv;
        return gamma ? v * E::widen(gamma[d]) : v;
    };
    const uint32_t half = a.rot / 2;
    for (uint32_t i = lane; i < half; i += 64) {
        const uint32_t d0 = a.interleaved ? 2 * i : i, d1 = a.interleaved ? 2 * i + 1 : i + half;
        float c, s;
        turn(pos, a.freqs[i], &c, &s);
        c *= a.magnitude, s *= a.magnitude;
        const float u = get(d0), v = get(d1);
        out[d0] = E::narrow(fmaf(u, c, -(v * s)));
        out[d1] = E::narrow(fmaf(v, c, u * s));
    }
    for (uint32_t d = a.rot + lane; d < a.D; d += 64) out[d] = E::narrow(get(d));
}

// ---------------------------------------------------------- wide form ----
// 16-byte accesses throughout. L lanes (a power of two) take a head's row, each two
// eights of it that hold whole pairs between them: eights l and l + rot / 16 of the
// rotated part, then two after another of the rest. A workgroup takes T tokens: their
// angles' cos and sin once, in LDS, for all heads; while those are taken the first rows
// are on their way, and each pass's under the one before. Bound by the bytes, each read
// and written once: 30,720 rows of 32 + 8 heads of 128 bf16, both normed, 629 MB in 110 us,
// 5.7 TB/s (a copy of as much: 117 us); 8576 rows of f16, half of each head turned, 176 MB
// in 33 us, 5.3 (34). The general form: 775 and 179 us. The stores go past the caches:
// 115 and 37 us where they did not. One token each of 32 sequences: 4.1 us, a workgroup's
// chain of search, angles and pass (an empty launch, queued: 1.6).
constexpr uint32_t kWideDim = 256;

// The sum over L lanes, in every one of them.
template <int L>
__device__ __forceinline__ float lane_sum(float v) {
    auto add = [&](auto ctrl) {
        v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    if constexpr (L >= 2) add(std::integral_constant<int, 0xb1>{});    // lane ^ 1
    if constexpr (L >= 4) add(std::integral_constant<int, 0x4e>{});    // lane ^ 2
    if constexpr (L >= 8) add(std::integral_constant<int, 0x141>{});   // 7 - lane of eight
    if constexpr (L >= 16) add(std::integral_constant<int, 0x140>{});  // 15 - lane of sixteen
    return v;
}

template <class E, int L>
__global__ __launch_bounds__(256) void wide_kernel(QkNormRotaryArgs a, uint32_t T) {
    typedef typename E::T V;
    constexpr uint32_t kRows = 256 / L;         // rows a pass
    __shared__ __align__(16) float cos_of[4][kWideDim / 2], sin_of[4][kWideDim / 2];
    __shared__ double pos_of[4];
    __shared__ bool in_of[4];
    const uint32_t tid = threadIdx.x, l = tid % L, tok0 = blockIdx.x * T, half = a.rot / 2, turned = a.rot / 8;
    const uint32_t toks = a.pb.tokens - tok0 < T ? a.pb.tokens - tok0 : T;
    if (blockIdx.x == 0 && blockIdx.y == 0) check_starts(a.pb);
    const bool pair = 2 * l < turned, live = 2 * l < a.D / 8;
    const uint32_t e0 = 8 * (pair ? l : 2 * l), e1 = 8 * (pair ? l + turned / 2 : 2 * l + 1);
    const uint32_t q_rows = toks * a.H, k_rows = toks * a.Hkv;
    const uint32_t q_passes = (q_rows + kRows - 1) / kRows, passes = q_passes + (k_rows + kRows - 1) / kRows;
    struct Row {
        Eight<E> x[2];
        uint32_t tok, h;
        bool in;
    };
    const float freq = tid < half ? a.freqs[tid] : 0.0f;      // (asked for ahead of the position)
    auto load = [&](uint32_t p, Row &r) __attribute__((always_inline)) {
        const int which = p >= q_passes;
        const uint32_t heads = which ? a.Hkv : a.H, i = (which ? p - q_passes : p) * kRows + tid / L;
        r.in = live && p < passes && i < (which ? k_rows : q_rows);
        r.tok = r.in ? i / heads : 0;
        r.h = i - r.tok * heads;
        if (!r.in) return;
        const V *x = static_cast<const V *>(a.x[which]) + uint64_t(tok0 + r.tok) * a.stride[which] + uint64_t(r.h) * a.D;
        r.x[0].load(x + e0);
        r.x[1].load(x + e1);
    };
    Row ring[2];
    const uint32_t p0 = blockIdx.y, dp = gridDim.y;
    load(p0, ring[0]);
    const uint32_t wave = pk_uni(tid >> 6);
    if (wave < toks) {
        double pos = 0.0;
        const bool in = position(a, tok0 + wave, &pos);
        if ((tid & 63u) == 0) pos_of[wave] = pos, in_of[wave] = in;
    }
    __syncthreads();
    for (uint32_t i = tid; i < toks * half; i += 256) {
        const uint32_t t = i / half, f = i - t * half;
        float c, s;
        turn(pos_of[t], i < half ? freq : a.freqs[f], &c, &s);
        cos_of[t][f] = c * a.magnitude, sin_of[t][f] = s * a.magnitude;
    }
    __syncthreads();
    float g[2][8];
    auto gamma = [&](int which) {
        const V *p = static_cast<const V *>(a.gamma[which]);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            Eight<E> x;
            if (p && live) x.load(p + (n ? e1 : e0));
#pragma unroll
            for (int e = 0; e < 8; ++e) g[n][e] = p && live ? x.get(e) : 1.0f;
        }
    };
    auto row = [&](uint32_t p, const Row &r) __attribute__((always_inline)) {
        const int which = p >= q_passes;
        float v[2][8];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[n][e] = r.in ? r.x[n].get(e) : 0.0f;
        if (a.norms >> which & 1) {
            float sum = 0.0f;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 8; ++e) sum = fmaf(v[n][e], v[n][e], sum);
            const float inv = 1.0f / sqrtf(lane_sum<L>(sum) / float(a.D) + a.eps);
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 8; ++e) v[n][e] = v[n][e] * inv * g[n][e];
        }
        if (!r.in || !in_of[r.tok]) return;
        const float *cs = cos_of[r.tok], *sn = sin_of[r.tok];
        if (pair && a.interleaved) {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float c = cs[(n ? e1 : e0) / 2 + e / 2], s = sn[(n ? e1 : e0) / 2 + e / 2];
                    const float x = v[n][e], y = v[n][e + 1];
                    v[n][e] = fmaf(x, c, -(y * s));
                    v[n][e + 1] = fmaf(y, c, x * s);
                }
        } else if (pair) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float c = cs[e0 + e], s = sn[e0 + e], x = v[0][e], y = v[1][e];
                v[0][e] = fmaf(x, c, -(y * s));
                v[1][e] = fmaf(y, c, x * s);
            }
        }
        V *out = static_cast<V *>(a.out[which]) + (uint64_t(tok0 + r.tok) * (which ? a.Hkv : a.H) + r.h) * a.D;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            u32x4 w[sizeof(V) / 2];
#pragma unroll
            for (uint32_t i = 0; i < 2 * sizeof(V); ++i) {
                if constexpr (sizeof(V) == 4) w[i / 4][i % 4] = __float_as_uint(v[n][i]);
                else w[0][i] = pack2<E>(v[n][2 * i], v[n][2 * i + 1]);
            }
#pragma unroll
            for (uint32_t i = 0; i < sizeof(V) / 2; ++i)
                __builtin_nontemporal_store(w[i], reinterpret_cast<u32x4 *>(out + (n ? e1 : e0)) + i);
        }
    };
    bool second = p0 >= q_passes;
    gamma(second);
    auto turn_to = [&](uint32_t p) {
        if (p >= q_passes && !second) gamma(second = true);
    };
    for (uint32_t p = p0; p < passes; p += 2 * dp) {
        load(p + dp, ring[1]);
        turn_to(p);
        row(p, ring[0]);
        if (p + dp >= passes) break;
        load(p + 2 * dp, ring[0]);
        turn_to(p + dp);
        row(p + dp, ring[1]);
    }
}

bool wide_applies(const QkNormRotaryArgs &a) {
    const uint32_t es = a.dtype == 8 ? 4 : 2;
    const auto at16 = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };   // (null too)
    return a.D <= kWideDim && a.D % 16 == 0 && a.rot % 16 == 0 && a.stride[0] * uint64_t(es) % 16 == 0 &&
           a.stride[1] * uint64_t(es) % 16 == 0 && at16(a.x[0]) && at16(a.x[1]) && at16(a.gamma[0]) &&
           at16(a.gamma[1]) && at16(a.out[0]) && at16(a.out[1]);
}

// Tokens a workgroup: more take the angles' part of its time once, fewer leave less of the
// GPU idle at the end, some 6000 workgroups are enough (8576 rows with 1, 2 and 4: 37, 38
// and 40 us; 30,720: 148, 121 and 115).
uint32_t tokens_of(const QkNormRotaryArgs &a) { return a.pb.tokens >= 24576 ? 4 : a.pb.tokens >= 12288 ? 2 : 1; }
// Workgroups that share a token's passes: one a pass while that leaves CUs free (32 rows:
// 4.1 us, 4.7 with one for all).
uint32_t shares_of(const QkNormRotaryArgs &a) {
    const uint32_t rows = a.D <= 64 ? 64 : a.D <= 128 ? 32 : 16;
    const uint32_t passes = (a.H + rows - 1) / rows + (a.Hkv + rows - 1) / rows;
    return a.pb.tokens > 1024 ? 1 : std::min(passes, 1024 / a.pb.tokens);
}

template <class E>
void launch(const QkNormRotaryArgs &a, hipStream_t stream) {
    if (!wide_applies(a)) {
        rows_kernel<E><<<uint32_t(qk_norm_rotary_threads(a) / 256), 256, 0, stream>>>(a);
        return;
    }
    const dim3 grid((a.pb.tokens + tokens_of(a) - 1) / tokens_of(a), shares_of(a));
    if (a.D <= 64) wide_kernel<E, 4><<<grid, 256, 0, stream>>>(a, tokens_of(a));
    else if (a.D <= 128) wide_kernel<E, 8><<<grid, 256, 0, stream>>>(a, tokens_of(a));
    else wide_kernel<E, 16><<<grid, 256, 0, stream>>>(a, tokens_of(a));
}

}  // namespace

uint64_t qk_norm_rotary_threads(const QkNormRotaryArgs &a) {
    if (wide_applies(a)) return (uint64_t(a.pb.tokens) + tokens_of(a) - 1) / tokens_of(a) * shares_of(a) * 256;
    return (uint64_t(a.pb.tokens) * (a.H + a.Hkv) + 3) / 4 * 256;
}

hipError_t launch_qk_norm_rotary(const QkNormRotaryArgs &a, hipStream_t stream) {
    if (a.dtype == 7) launch<Bf16>(a, stream);
    else if (a.dtype == 6) launch<F16>(a, stream);
    else launch<F32>(a, stream);
    return hipGetLastError();
}

}  // namespace holo
