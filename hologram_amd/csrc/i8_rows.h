// i8_rows.h — attention of up to sixteen rows at a time over int8 K and V whose 16-key
// steps have one scale each: what a wavefront does with 32 keys, and how wavefronts and
// workgroups join (attn_blocks.hip, attn_selected.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>

#include <type_traits>

#include "holo_kernels.h"
#include "packed_tile.h"

namespace holo {

// Sixteen rows are the columns of the matrix instructions, which read each byte of K and V
// once for all of them. Per 32 keys and wavefront:
//     S^T[32 keys x 16 rows] = K . Q^T    16x16x64 i8 on the cache's own bytes; a row
//                                         of Q as 23-bit integers in three int8
//                                         parts, its largest in [2^21, 2^22), so
//                                         the products are exact
//     scores, limits, online softmax      f32; a row is a lane column
//     O^T[DP x 16 rows] += V^T . P^T      16x16x32 f16; an int8 is an exact f16, built
//                                         by placing its byte under the exponent of
//                                         1024
// The scale of a 16-key step is one number (blocks are multiples of 16 keys): K's
// joins the scores, V's the weights, w = p vs 2^(7 - ve) with 2^ve above every finite
// |vs| of the keys the row sees so far. p is at most 2^8 (a row's maximum may lag that
// far behind before its sums are rescaled), so |w| <= 2^15, and weights down to 2^-31
// of the largest stay clear of f16's subnormals. 16-bit rows round w to f16 once, 11
// bits where the result has 8 or 11; f32 rows hold it in two parts, 22 bits.
// A row's sums, maximum and ve are its lanes' own, and a masked key's weight is 0 with
// the scales of steps it does not see left out, so nothing reaches another row.
constexpr float kLog2e = 1.4426950408889634f;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
constexpr uint32_t kUnit = 16, kStep = 32, kOob = 1u << 30;   // past every plane, twice it too
constexpr int kVeMin = -126;   // the floor of ve, where the result's own bits end

// A step's factor of its weights, v 2^(7 - ve). An infinite scale's is 2^100, whose weights
// are infinite in f16 where p is not 0 and 0 where it is: a key that the row does not see
// brings it no NaN.
__device__ __forceinline__ float weight_factor(float v, int ve) {
    const float f = ldexpf(v, 7 - ve);
    return fabsf(f) == INFINITY ? copysignf(0x1p100f, f) : f;
}
// A product as it is rounded to f32: the conversion to f16 behind it would else take the
// product unrounded, and its two parts, of which one does and the other not, be a step of
// f16 apart.
__device__ __forceinline__ float rounded(float w) {
    asm volatile("" : "+v"(w));
    return w;
}
// What a weight of at most 2^15 leaves over its f16, as f16; nothing of an infinite one's.
__device__ __forceinline__ float left_over(float w, float hi) { return fminf(fmaxf(w - hi, -16.0f), 16.0f); }

__device__ __forceinline__ __amdgpu_buffer_rsrc_t range(const void *base, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), 0, int(bytes), 0x00020000);
}

// The largest over a column's four lanes.
__device__ __forceinline__ float column_max(float v) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Dim t of four (bytes of words w[0..7], one a key, xor 0x80) for the eight keys, as
// f16: 1024 + byte by placement, less 1152.
__device__ __forceinline__ f16x8 key_column(const uint32_t (&w)[8], int t) {
    u32x4 m;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t two = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], t < 2 ? 0x05010400u : 0x07030602u);
        m[i] = __builtin_amdgcn_perm(0x64646464u, two, t & 1 ? 0x04030402u : 0x04010400u);
    }
    return __builtin_bit_cast(f16x8, m) - (f16x8)(_Float16)1152.0f;
}

// One wavefront's state of a unit's 16 rows: O^T (dim NDB * (4 g + i) + d of row r in
// o[d][i]), maximum, sum, ve.
template <int DP>
struct State {
    f32x4 o[DP / 16];
    float m, l;
    int ve;
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
        m = -INFINITY, l = 0.0f, ve = kVeMin;
    }
};

template <class E, int DP, int W>
struct FewLds {
    float o[W][kUnit][DP + 4];
    float m[W][kUnit], l[W][kUnit];
    int ve[W][kUnit];
};

// The bytes of two 16-key steps as a wavefront's lanes hold them, and where they are. K:
// keys 16 h + r, bytes 64 s + 16 g on. V: keys 16 (j / 4) + 4 g + j % 4, bytes NDB r on.
// (r = lane % 16, g = lane / 16.)
template <int DP>
struct KvStep {
    static constexpr int NKS = DP / 64, NDB = DP / 16, VW = NDB / 4;
    u32x4 k[2][NKS];
    uint32_t v[8][VW];
    float ks[2], vs[2];
};
template <int DP>
struct KvPlane {
    static constexpr int NKS = DP / 64, NDB = DP / 16, VW = NDB / 4;
    __amdgpu_buffer_rsrc_t rk, rv;
    uint32_t koff[NKS], voff, D;

    __device__ __forceinline__ KvPlane(const int8_t *k, const int8_t *v, uint32_t bucket, uint32_t dims)
        : rk(range(k, bucket * dims)), rv(range(v, bucket * dims)), D(dims) {
        const uint32_t lane = threadIdx.x & 63u, r = lane & 15u, g = lane >> 4;
#pragma unroll
        for (int s = 0; s < NKS; ++s) koff[s] = 64 * s + 16 * g < D ? r * D + 64 * s + 16 * g : kOob;
        voff = NDB * r < D ? 4 * g * D + NDB * r : kOob;
    }
    // The steps at bytes at[0] and at[1] of the plane (kOob: nothing is read, zeros).
    // kOnce: non-temporal, for a cache that is read once.
    template <bool kOnce>
    __device__ __forceinline__ void load(const uint32_t (&at)[2], KvStep<DP> &x) const {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int s = 0; s < NKS; ++s)
                x.k[h][s] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, koff[s] + at[h], 0, kOnce ? 2 : 0));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t o = voff + (at[j >> 2] + (j & 3) * D);
            if constexpr (VW == 1) {
                x.v[j][0] = __builtin_amdgcn_raw_buffer_load_b32(rv, o, 0, kOnce ? 2 : 0);
            } else if constexpr (VW == 2) {
                const auto w = __builtin_amdgcn_raw_buffer_load_b64(rv, o, 0, kOnce ? 2 : 0);
                x.v[j][0] = w[0], x.v[j][1] = w[1];
            } else {
                const auto w = __builtin_amdgcn_raw_buffer_load_b128(rv, o, 0, kOnce ? 2 : 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) x.v[j][i] = w[i];
            }
        }
    }
};

// A column's row of Q, dims 64 s + 16 g + e, in three int8 parts, and what its whole
// numbers' products are times.
template <class E, int DP>
struct RowQ {
    static constexpr int NKS = DP / 64;
    i32x4 part[3][NKS];
    float mul;

    // `q` the lane's row (any address where it is not live), `scale` log2(e) / divisor
    __device__ __forceinline__ void load(const typename E::T *q, bool live, uint32_t D, float scale) {
        typedef typename E::T T;
        constexpr bool kF32 = std::is_same_v<E, F32>;
        const uint32_t g = (threadIdx.x & 63u) >> 4;
        float qv[16 * NKS], top = 0.0f;
        {
#pragma unroll
            for (int s = 0; s < NKS; ++s) {
                const uint32_t d = 64 * s + 16 * g;
                const bool in = live && d < D;
#pragma unroll
                for (int w = 0; w < int(sizeof(T)); ++w) {
                    u32x4 x = {0, 0, 0, 0};
                    if (in) x = *reinterpret_cast<const u32x4 *>(q + d + w * (16 / sizeof(T)));
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float *to = qv + 16 * s + w * (16 / sizeof(T));
                        if constexpr (kF32) {
                            to[i] = __uint_as_float(x[i]);
                        } else {
                            to[2 * i] = E::widen(uint16_t(x[i]));
                            to[2 * i + 1] = E::widen(uint16_t(x[i] >> 16));
                        }
                    }
                }
            }
        }
        bool bad = false;      // a row with a NaN or infinity is NaN throughout
#pragma unroll
        for (int e = 0; e < 16 * NKS; ++e) {
            top = fmaxf(top, fabsf(qv[e]));
            bad |= !(fabsf(qv[e]) <= 3.4028235e38f);
        }
        top = column_max(top);
        bad = column_max(bad ? 1.0f : 0.0f) != 0.0f;
        int qe = 0;
        if (top > 0.0f && top <= 3.4028235e38f) {
            (void)frexpf(top, &qe);     // top < 2^qe
            qe = 22 - qe;
        }
#pragma unroll
        for (int s = 0; s < NKS; ++s)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                uint32_t bytes[3] = {0, 0, 0};
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    int v = bad ? 0 : int(rintf(ldexpf(qv[16 * s + 4 * w + t], qe)));
#pragma unroll
                    for (int p = 2; p >= 0; --p) {
                        const int up = (v + 128) >> 8;
                        bytes[p] |= uint32_t((p ? v - up * 256 : v) & 0xff) << (8 * t);
                        v = up;
                    }
                }
#pragma unroll
                for (int p = 0; p < 3; ++p) part[p][s][w] = int(bytes[p]);
            }
        mul = bad ? __uint_as_float(0x7fc00000u) : ldexpf(scale, -qe);
    }
};

// Two 16-key steps, keys key[h] on, joined to the rows' state; where `edge` is set, a key
// at or past `lim` (a column's own) or `end` does not count.
template <class E, int DP>
__device__ __forceinline__ void few_step(State<DP> &st, const KvStep<DP> &x, const RowQ<E, DP> &q, const uint32_t (&key)[2],
                                         bool edge, uint32_t lim, uint32_t end) {
    constexpr int NKS = DP / 64, NDB = DP / 16, VW = NDB / 4;
    constexpr bool kF32 = std::is_same_v<E, F32>;
    const uint32_t g = (threadIdx.x & 63u) >> 4;
    constexpr float kLag = 8.0f;
    float s[8], w[8];
    float vs_h[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        i32x4 a0 = {0, 0, 0, 0}, a1 = {0, 0, 0, 0}, a2 = {0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < NKS; ++c) {
            const i32x4 kf = __builtin_bit_cast(i32x4, x.k[h][c]);
            a0 = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf, q.part[0][c], a0, 0, 0, 0);
            a1 = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf, q.part[1][c], a1, 0, 0, 0);
            a2 = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf, q.part[2][c], a2, 0, 0, 0);
        }
        const float c = x.ks[h] * q.mul;
#pragma unroll
        for (int i = 0; i < 4; ++i) s[4 * h + i] = fmaf(float(a0[i]), 65536.0f, float(a1[i] * 256 + a2[i])) * c;
        vs_h[h] = x.vs[h];
    }
    if (edge) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t j = key[h] + 4 * g + i;
                s[4 * h + i] = j < lim && j < end ? s[4 * h + i] : -INFINITY;
            }
            vs_h[h] = key[h] < lim ? vs_h[h] : 0.0f;
        }
    }
    float mt = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
    mt = column_max(mt);
    int ve = st.ve;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float v = fabsf(vs_h[h]);
        int e = kVeMin;
        if (v > 0.0f && v <= 3.4028235e38f) (void)frexpf(v, &e);   // v < 2^e
        ve = e > ve ? e : ve;
    }
    if (__any(mt > st.m + kLag || ve > st.ve)) {
        const float mn = mt > st.m + kLag ? mt : st.m;
        const float al = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(st.m - mn);
        st.l *= al;
        const float sh = ldexpf(al, st.ve - ve);
#pragma unroll
        for (int d = 0; d < NDB; ++d) st.o[d] *= sh;
        st.m = mn, st.ve = ve;
    }
    const float ref = st.m == -INFINITY ? 0.0f : st.m;
    f16x8 hi, lo;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float f = weight_factor(vs_h[h], ve);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float p = __builtin_amdgcn_exp2f(s[4 * h + i] - ref);
            st.l += p;
            w[4 * h + i] = kF32 ? rounded(p * f) : p * f;
            hi[4 * h + i] = _Float16(w[4 * h + i]);
            if constexpr (kF32) lo[4 * h + i] = _Float16(left_over(w[4 * h + i], float(hi[4 * h + i])));
        }
    }
#pragma unroll
    for (int q = 0; q < VW; ++q) {
        uint32_t words[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) words[j] = x.v[j][q] ^ 0x80808080u;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const f16x8 v = key_column(words, t);
            st.o[4 * q + t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, hi, st.o[4 * q + t], 0, 0, 0);
            if constexpr (kF32) st.o[4 * q + t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, lo, st.o[4 * q + t], 0, 0, 0);
        }
    }
}

// few_step for at most eight rows: two column groups of eight, each over a 16-key step of its
// own, so that a lane's scores are four and not eight. Column r is row r % 8 over step r / 8: the
// products are made for all columns and those of a column's step kept, and its weights enter the
// products with V as zeros but for its step's keys. `key`, `ks` and `vs` are of the column's
// step.
template <class E, int DP>
__device__ __forceinline__ void group_step(State<DP> &st, const KvStep<DP> &x, const RowQ<E, DP> &q, uint32_t key,
                                           float ks, float vs, uint32_t lim) {
    constexpr int NKS = DP / 64, VW = DP / 64;
    constexpr bool kF32 = std::is_same_v<E, F32>;
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4;
    const bool second = (lane & 15u) >= 8;
    constexpr float kLag = 8.0f;
    i32x4 a[3];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        i32x4 b[3] = {{0, 0, 0, 0}, {0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int c = 0; c < NKS; ++c) {
            const i32x4 kf = __builtin_bit_cast(i32x4, x.k[h][c]);
#pragma unroll
            for (int p = 0; p < 3; ++p) b[p] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf, q.part[p][c], b[p], 0, 0, 0);
        }
#pragma unroll
        for (int p = 0; p < 3; ++p)
#pragma unroll
            for (int i = 0; i < 4; ++i) a[p][i] = h == 0 || second ? b[p][i] : a[p][i];
    }
    float s[4];
    const float c = ks * q.mul;
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = fmaf(float(a[0][i]), 65536.0f, float(a[1][i] * 256 + a[2][i])) * c;
    if (__any(key + 16 > lim)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = key + 4 * g + i < lim ? s[i] : -INFINITY;
        vs = key < lim ? vs : 0.0f;
    }
    const float mt = column_max(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])));
    const float av = fabsf(vs);
    int ve = kVeMin;
    if (av > 0.0f && av <= 3.4028235e38f) (void)frexpf(av, &ve);   // av < 2^ve
    ve = st.ve > ve ? st.ve : ve;
    if (__any(mt > st.m + kLag || ve > st.ve)) {
        const float mn = mt > st.m + kLag ? mt : st.m;
        const float al = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(st.m - mn);
        st.l *= al;
        const float sh = ldexpf(al, st.ve - ve);
#pragma unroll
        for (int d = 0; d < DP / 16; ++d) st.o[d] *= sh;
        st.m = mn, st.ve = ve;
    }
    const float ref = st.m == -INFINITY ? 0.0f : st.m, f = weight_factor(vs, ve);
    typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
    f16x4 hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float p = __builtin_amdgcn_exp2f(s[i] - ref);
        st.l += p;
        const float w = kF32 ? rounded(p * f) : p * f;
        hi[i] = _Float16(w);
        if constexpr (kF32) lo[i] = _Float16(left_over(w, float(hi[i])));
    }
    auto of_step = [&](f16x4 w) __attribute__((always_inline)) {
        const uint2 v = __builtin_bit_cast(uint2, w);
        return __builtin_bit_cast(f16x8, u32x4{second ? 0u : v.x, second ? 0u : v.y, second ? v.x : 0u, second ? v.y : 0u});
    };
    const f16x8 wh = of_step(hi);
    f16x8 wl;
    if constexpr (kF32) wl = of_step(lo);
#pragma unroll
    for (int n = 0; n < VW; ++n) {
        uint32_t words[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) words[j] = x.v[j][n] ^ 0x80808080u;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const f16x8 v = key_column(words, e);
            st.o[4 * n + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, wh, st.o[4 * n + e], 0, 0, 0);
            if constexpr (kF32) st.o[4 * n + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, wl, st.o[4 * n + e], 0, 0, 0);
        }
    }
}

// The wavefronts' states joined: 2^(m_w - M) of each, their units of 2^(ve - 7) made one; of C
// column groups too. put(row, dim, O, maximum, sum) of `rows` rows; the workgroup's LDS is
// free again after it.
template <class E, int DP, int W, int C = 1, class Put>
__device__ __forceinline__ void join_waves(State<DP> &st, uint32_t rows, uint32_t D, FewLds<E, DP, W> &lds, Put put) {
    constexpr int NDB = DP / 16;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, r = lane & 15u, g = lane >> 4, wave = pk_uni(tid >> 6);
    st.l += __shfl_xor(st.l, 16, 64);
    st.l += __shfl_xor(st.l, 32, 64);
#pragma unroll
    for (int d = 0; d < NDB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) lds.o[wave][r][NDB * (4 * g + i) + d] = st.o[d][i];
    if (g == 0) lds.m[wave][r] = st.m, lds.l[wave][r] = st.l, lds.ve[wave][r] = st.ve;
    __syncthreads();
    for (uint32_t i = tid; i < rows * D; i += 64 * W) {
        const uint32_t c = i / D, d = i - c * D;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
            for (int n = 0; n < C; ++n) M = fmaxf(M, lds.m[w][c + 16 / C * n]);
        const float ref = M == -INFINITY ? 0.0f : M;
        float o = 0.0f, l = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w)
#pragma unroll
            for (int n = 0; n < C; ++n) {
                const uint32_t r = c + 16 / C * n;
                const float e = __builtin_amdgcn_exp2f(lds.m[w][r] - ref);
                l += lds.l[w][r] * e;
                o += ldexpf(lds.o[w][r][d], lds.ve[w][r] - 7) * e;
            }
        put(c, d, o, M, l);
    }
    __syncthreads();
}

// One row of `np` partials, `stride` floats from one to the next, joined in order by a
// wavefront: its lanes take the partials' weights, 64 at a time, then the dims, eight
// partials in flight.
template <class E, int DP>
__device__ __forceinline__ void join_row(const float *p, uint32_t stride, uint32_t np, uint32_t D, bool none,
                                         typename E::T *out) {
    const uint32_t lane = threadIdx.x & 63u;
    float M = -INFINITY, l = 0.0f, o[DP / 64];
    for (uint32_t w = lane; w < np; w += 64) M = fmaxf(M, p[w * stride + DP]);
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) M = fmaxf(M, __shfl_xor(M, x, 64));
    const float ref = M == -INFINITY ? 0.0f : M;
#pragma unroll
    for (int i = 0; i < DP / 64; ++i) o[i] = 0.0f;
    for (uint32_t w0 = 0; w0 < np; w0 += 64) {
        const bool in = w0 + lane < np;
        const float e = in ? __builtin_amdgcn_exp2f(p[(w0 + lane) * stride + DP] - ref) : 0.0f;
        const float le = in ? p[(w0 + lane) * stride + DP + 1] * e : 0.0f;
        const uint32_t many = np - w0 < 64 ? np - w0 : 64;
        for (uint32_t w = 0; w < many; w += 8) {
            float x[8][DP / 64];
#pragma unroll
            for (uint32_t q = 0; q < 8; ++q)
#pragma unroll
                for (int i = 0; i < DP / 64; ++i) x[q][i] = w + q < many ? p[(w0 + w + q) * stride + lane + 64 * i] : 0.0f;
#pragma unroll
            for (uint32_t q = 0; q < 8; ++q) {
                if (w + q >= many) break;
                const float ew = __shfl(e, int(w + q), 64);
                l += __shfl(le, int(w + q), 64);
#pragma unroll
                for (int i = 0; i < DP / 64; ++i) o[i] = fmaf(x[q][i], ew, o[i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < DP / 64; ++i)
        if (lane + 64 * i < D) out[lane + 64 * i] = E::narrow(none ? 0.0f : o[i] / l);
}

}  // namespace holo
