// attn_blocks.hip — attention of a packed batch's rows over the int8 cache with
// one scale a block of rows (AttentionI8Blocks, 128).
#include <hip/hip_runtime.h>

#include <math.h>

#include <type_traits>

#include "holo_kernels.h"
#include "packed_tile.h"

namespace holo {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// Keys that row t of sequence b's n rows sees.
__device__ __forceinline__ uint32_t visible_keys(int64_t len, uint32_t n, uint32_t t, uint32_t bucket) {
    const int64_t v = len - int64_t(n - 1 - t);
    return v < 0 ? 0u : v > int64_t(bucket) ? bucket : uint32_t(v);
}

// ---------------------------------------------------------- few-row form ----
// Decode and drafts. Sixteen packed rows of a sequence and kv head (row r = token r /
// G, head r % G) are a unit: the columns of the matrix instructions, which read each
// byte of K and V once for all of them. The wavefronts of a workgroup take the 32-key
// blocks of its share in turn. Per block and wavefront:
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
//
// Two splits. Direct: a workgroup of eight wavefronts a unit, no second launch; for
// buckets up to kDirect rows and kDirectUnits units (one token of 8 kv heads of 128 dims
// for 8, 32 and 128 full sequences: 11, 13 and 47 us against the shares' 13, 18 and 34 at
// 512 rows, 15, 17 and 64 against 14, 22 and 52 at 1024, 23, 27 and 103 against 17, 31
// and 90 at 2048; ragged ones of up to 512 rows, 64 and 128 of them: 18 and 33 against 20
// and 29). Balanced: all units' 128-key quads laid end to end and cut into equal
// shares, one for each of the workgroups that the GPU holds at once, whatever the
// lengths; a unit that is cut leaves partials, which merge_kernel joins in order (a
// launch of its own: partials pass between XCDs' L2s at its boundary).
// Bound by the cache's bytes: 32 sequences of 512 to 32767 keys, 8 kv heads of 128 dims,
// 528 MB, 106 us or 5.0 TB/s, merge_kernel 5 us of them, 108 us of f32 rows; 128 of 8192
// keys, 2.2 GB, 6.6 TB/s. Short ones by their latency: 8 of 30 to 700 keys 9 us, up to three
// rounds of a workgroup's 256 keys.
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
constexpr uint32_t kUnit = 16, kStep = 32, kQuad = 128, kOob = 1u << 30;   // past every plane, twice it too
constexpr uint32_t kDirect = 1024, kDirectUnits = 640, kShares = 512, kMinQuads = 2;
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

struct Blocks {
    AttnBlocksArgs a;
    float mul;           // log2(e) / divisor
    uint32_t shift;      // block == 1 << shift
    uint32_t places;     // places of the grid (place_of)
    float *part;         // [places * Hkv + kShares][kUnit][DP + 2]: O, then the maximum and the sum
};

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
};

template <class E, int DP, int W>
struct FewLds {
    float o[W][kUnit][DP + 4];
    float m[W][kUnit], l[W][kUnit];
    int ve[W][kUnit];
};

// Keys [c0, c1) of unit `at.unit` of sequence at.b and kv head kh, by W wavefronts; the
// joined result goes to `out` (whole) or to a partial at dst.
template <class E, int DP, int W>
__device__ __forceinline__ void few_segment(const Blocks &k, const Place &at, uint32_t kh, uint32_t c0, uint32_t c1,
                                            bool whole, float *dst, FewLds<E, DP, W> &lds) {
    constexpr int NKS = DP / 64, NDB = DP / 16, VW = NDB / 4;
    constexpr bool kF32 = std::is_same_v<E, F32>;
    typedef typename E::T T;
    const AttnBlocksArgs &a = k.a;
    const uint32_t G = a.H / a.Hkv, n = at.hi - at.lo, R = n * G;
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const uint32_t wave = pk_uni(uint32_t(tid) >> 6);
    const uint32_t row = at.unit * kUnit + r, tok = row / G;
    const bool live = row < R;
    const int64_t len = a.lens[at.b];
    const uint32_t lim = live ? visible_keys(len, n, tok, a.bucket) : 0u;
    const uint32_t first = at.unit * kUnit / G, last = (at.unit * kUnit + kUnit - 1 < R ? at.unit * kUnit + kUnit - 1 : R - 1) / G;
    const uint32_t kmin = visible_keys(len, n, first, a.bucket), kmax = visible_keys(len, n, last, a.bucket);
    const uint32_t end = pk_uni(c1 < kmax ? c1 : kmax);
    const uint64_t plane = uint64_t(at.b) * a.Hkv + kh;
    const auto rk = range(a.kq + plane * a.bucket * a.D, a.bucket * a.D);
    const auto rv = range(a.vq + plane * a.bucket * a.D, a.bucket * a.D);
    const uint32_t nb = (a.bucket + a.block - 1) >> k.shift;
    const float *ks = a.ks + plane * nb, *vs = a.vs + plane * nb;

    // K: keys 16 h + r, bytes 64 s + 16 g on. V: keys 16 (j / 4) + 4 g + j % 4, bytes
    // NDB r on.
    uint32_t koff[NKS];
#pragma unroll
    for (int s = 0; s < NKS; ++s) koff[s] = uint32_t(64 * s + 16 * g) < a.D ? r * a.D + 64 * s + 16 * g : kOob;
    const uint32_t voff = uint32_t(NDB * r) < a.D ? 4 * g * a.D + NDB * r : kOob;
    struct Bytes {
        u32x4 k[2][NKS];
        uint32_t v[8][VW];
        float ks[2], vs[2];
    };
    // (non-temporal: the cache is read once)
    auto load = [&](uint32_t blk, Bytes &x) __attribute__((always_inline)) {
        const uint32_t so = blk < end ? blk * a.D : kOob;   // past the share: nothing is read
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int s = 0; s < NKS; ++s)
                x.k[h][s] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, koff[s] + (so + 16 * h * a.D), 0, 2));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t o = voff + (so + (16 * (j >> 2) + (j & 3)) * a.D);
            if constexpr (VW == 1) {
                x.v[j][0] = __builtin_amdgcn_raw_buffer_load_b32(rv, o, 0, 2);
            } else if constexpr (VW == 2) {
                const auto w = __builtin_amdgcn_raw_buffer_load_b64(rv, o, 0, 2);
                x.v[j][0] = w[0], x.v[j][1] = w[1];
            } else {
                const auto w = __builtin_amdgcn_raw_buffer_load_b128(rv, o, 0, 2);
#pragma unroll
                for (int i = 0; i < 4; ++i) x.v[j][i] = w[i];
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t i = (blk + 16 * h) >> k.shift, c = i < nb ? i : nb - 1;
            x.ks[h] = ks[c], x.vs[h] = vs[c];
        }
    };
    Bytes ring[2];
    const uint32_t mine = c0 + wave * kStep;
    load(mine, ring[0]);

    // Q: dims 64 s + 16 g + e of the lane's row
    float qv[16 * NKS], top = 0.0f;
    {
        const T *q = static_cast<const T *>(a.q) + uint64_t(at.lo + (live ? tok : 0u)) * a.q_stride +
                     (uint64_t(kh) * G + (live ? row - tok * G : 0u)) * a.D;
#pragma unroll
        for (int s = 0; s < NKS; ++s) {
            const uint32_t d = 64 * s + 16 * g;
            const bool in = live && d < a.D;
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
    i32x4 qp[3][NKS];
#pragma unroll
    for (int s = 0; s < NKS; ++s)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            uint32_t part[3] = {0, 0, 0};
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                int v = bad ? 0 : int(rintf(ldexpf(qv[16 * s + 4 * w + t], qe)));
#pragma unroll
                for (int p = 2; p >= 0; --p) {
                    const int up = (v + 128) >> 8;
                    part[p] |= uint32_t((p ? v - up * 256 : v) & 0xff) << (8 * t);
                    v = up;
                }
            }
#pragma unroll
            for (int p = 0; p < 3; ++p) qp[p][s][w] = int(part[p]);
        }
    const float mul = bad ? __uint_as_float(0x7fc00000u) : ldexpf(k.mul, -qe);

    State<DP> st;
#pragma unroll
    for (int d = 0; d < NDB; ++d) st.o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    st.m = -INFINITY, st.l = 0.0f, st.ve = kVeMin;
    constexpr float kLag = 8.0f;
    auto block = [&](uint32_t blk, const Bytes &x) __attribute__((always_inline)) {
        float s[8], w[8];
        float vs_h[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            i32x4 a0 = {0, 0, 0, 0}, a1 = {0, 0, 0, 0}, a2 = {0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < NKS; ++c) {
                const i32x4 kf = __builtin_bit_cast(i32x4, x.k[h][c]);
                a0 = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf, qp[0][c], a0, 0, 0, 0);
                a1 = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf, qp[1][c], a1, 0, 0, 0);
                a2 = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf, qp[2][c], a2, 0, 0, 0);
            }
            const float c = x.ks[h] * mul;
#pragma unroll
            for (int i = 0; i < 4; ++i) s[4 * h + i] = fmaf(float(a0[i]), 65536.0f, float(a1[i] * 256 + a2[i])) * c;
            vs_h[h] = x.vs[h];
        }
        if (blk + kStep > kmin || blk + kStep > end) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t key = blk + 16 * h + 4 * g + i;
                    s[4 * h + i] = key < lim && key < end ? s[4 * h + i] : -INFINITY;
                }
                vs_h[h] = blk + 16 * h < lim ? vs_h[h] : 0.0f;
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
    };
    for (uint32_t blk = mine; blk < end; blk += 2 * W * kStep) {
        load(blk + W * kStep, ring[1]);
        block(blk, ring[0]);
        if (blk + W * kStep >= end) break;
        load(blk + 2 * W * kStep, ring[0]);
        block(blk + W * kStep, ring[1]);
    }

    // The wavefronts' states joined: 2^(m_w - M) of each, their units of 2^(ve - 7) made
    // one
    st.l += __shfl_xor(st.l, 16, 64);
    st.l += __shfl_xor(st.l, 32, 64);
#pragma unroll
    for (int d = 0; d < NDB; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) lds.o[wave][r][NDB * (4 * g + i) + d] = st.o[d][i];
    if (g == 0) lds.m[wave][r] = st.m, lds.l[wave][r] = st.l, lds.ve[wave][r] = st.ve;
    __syncthreads();
    const uint32_t rows = R - at.unit * kUnit < kUnit ? R - at.unit * kUnit : kUnit;
    for (uint32_t i = tid; i < rows * a.D; i += 64 * W) {
        const uint32_t c = i / a.D, d = i - c * a.D;
        float M = lds.m[0][c];
#pragma unroll
        for (int w = 1; w < W; ++w) M = fmaxf(M, lds.m[w][c]);
        const float ref = M == -INFINITY ? 0.0f : M;
        float o = 0.0f, l = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float e = __builtin_amdgcn_exp2f(lds.m[w][c] - ref);
            l += lds.l[w][c] * e;
            o += ldexpf(lds.o[w][c][d], lds.ve[w][c] - 7) * e;
        }
        const uint32_t rr = at.unit * kUnit + c, t = rr / G;
        if (whole) {
            const bool none = visible_keys(len, n, t, a.bucket) == 0;
            static_cast<T *>(a.out)[(uint64_t(at.lo + t) * a.H + kh * G + (rr - t * G)) * a.D + d] =
                E::narrow(none ? 0.0f : o / l);
        } else {
            dst[c * (DP + 2) + d] = o;
            if (d == 0) dst[c * (DP + 2) + DP] = M, dst[c * (DP + 2) + DP + 1] = l;
        }
    }
    __syncthreads();
}

// Direct: grid places * Hkv. Eight wavefronts a unit, past 128 dims four, whose registers
// hold a block and its successor: with sixteen, 8 sequences of 30 to 700 keys of 64 dims
// took 9.8 us, not 8.8, and at 128 dims their registers spill.
template <class E, int DP, int W>
__global__ __launch_bounds__(64 * W) void few_direct_kernel(Blocks k) {
    __shared__ FewLds<E, DP, W> lds;
    if (blockIdx.x == 0) check_starts(k.a.pb);
    Place at;
    if (!place_of(k.a.pb, k.a.H / k.a.Hkv, kUnit, blockIdx.x / k.a.Hkv, &at)) return;
    few_segment<E, DP, W>(k, at, blockIdx.x % k.a.Hkv, 0, k.a.bucket, true, nullptr, lds);
}

// The quads of a sequence's units (one at least, so that rows without a key are
// written), and how many units it has.
__device__ __forceinline__ void sequence_quads(const AttnBlocksArgs &a, uint32_t b, uint32_t *units, uint32_t *quads) {
    const uint32_t lo = start_of(a.pb, b), hi = start_of(a.pb, b + 1);
    *units = hi > lo ? ((hi - lo) * (a.H / a.Hkv) + kUnit - 1) / kUnit : 0u;
    const uint32_t len = a.lens[b] < a.bucket ? a.lens[b] : a.bucket;
    *quads = len ? (len + kQuad - 1) / kQuad : 1u;
}

// The sequences' costs laid end to end.
struct Line {
    uint64_t total;
    uint64_t at;         // where sequence b's begin
    uint32_t b;
};
// Where the sequence that holds place `want(total)` of the line begins: 256 threads sum
// a run of sequences each, the run that holds it is walked.
template <class C, class F>
__device__ __forceinline__ Line find_line(uint32_t batch, C cost, F want, uint64_t *sums, Line *found) {
    const uint32_t tid = threadIdx.x, per = (batch + 255) / 256;
    const uint32_t b0 = tid * per, b1 = b0 + per < batch ? b0 + per : batch;
    uint64_t sum = 0;
    for (uint32_t b = b0; b < b1; ++b) sum += cost(b);
    // running sums: within a wavefront, then over the four
    uint64_t run = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t up = __shfl_up(run, o, 64);
        if ((tid & 63u) >= uint32_t(o)) run += up;
    }
    if ((tid & 63u) == 63u) sums[tid >> 6] = run;
    __syncthreads();
    uint64_t before = 0, total = 0;
#pragma unroll
    for (uint32_t w = 0; w < 4; ++w) {
        before += w < (tid >> 6) ? sums[w] : 0;
        total += sums[w];
    }
    const uint64_t at = want(total), base = before + run - sum;
    if (tid == 0) *found = Line{total, total, 0};
    __syncthreads();
    if (at >= base && at < base + sum) {
        uint64_t here = base;
        for (uint32_t b = b0; b < b1; ++b) {
            const uint64_t all = cost(b);
            if (at < here + all) {
                *found = Line{total, here, b};
                break;
            }
            here += all;
        }
    }
    __syncthreads();
    return *found;
}

__device__ __forceinline__ uint64_t share_of(uint64_t total) {
    const uint64_t s = (total + kShares - 1) / kShares;
    return s < kMinQuads ? kMinQuads : s;
}

template <class E, int DP>
__global__ __launch_bounds__(256, DP > 128 ? 1 : 2) void few_shares_kernel(Blocks k) {
    __shared__ FewLds<E, DP, 4> lds;
    __shared__ uint64_t sums[4];
    __shared__ Line found;
    const AttnBlocksArgs &a = k.a;
    if (blockIdx.x == 0) check_starts(a.pb);
    const uint32_t G = a.H / a.Hkv;
    // a sequence's quads come unit by unit, kv head by kv head
    const Line ln = find_line(a.pb.batch, [&](uint32_t b) {
        uint32_t units, quads;
        sequence_quads(a, b, &units, &quads);
        return uint64_t(units) * quads * a.Hkv;
    }, [&](uint64_t total) { return blockIdx.x * share_of(total); }, sums, &found);
    const uint64_t share = share_of(ln.total);
    uint64_t pos = blockIdx.x * share, end = pos + share < ln.total ? pos + share : ln.total;
    uint64_t base = ln.at;
    for (uint32_t b = ln.b; pos < end; ++b) {
        if (b >= a.pb.batch) return;
        uint32_t units, quads;
        sequence_quads(a, b, &units, &quads);
        const uint64_t all = uint64_t(units) * quads * a.Hkv;
        while (pos < end && pos < base + all) {
            const uint32_t u = uint32_t((pos - base) / quads), q0 = uint32_t((pos - base) - uint64_t(u) * quads);
            const uint32_t q1 = q0 + (end - pos) < quads ? uint32_t(q0 + (end - pos)) : quads;
            const uint32_t unit = pk_uni(u / a.Hkv), kh = pk_uni(u - unit * a.Hkv);   // (alike in all lanes)
            const Place at{pk_uni(b), pk_uni(start_of(a.pb, b)), pk_uni(start_of(a.pb, b + 1)), unit};
            const uint64_t id = uint64_t(at.lo * G / kUnit + at.b + unit) * a.Hkv + kh;
            few_segment<E, DP, 4>(k, at, kh, pk_uni(q0) * kQuad, pk_uni(q1) * kQuad, pk_uni(q0 == 0 && q1 == quads),
                                  k.part + (id + blockIdx.x) * (kUnit * (DP + 2)), lds);
            pos += q1 - q0;
        }
        base += all;
    }
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

// Joins the partials of a unit that shares cut: grid places * Hkv.
template <class E, int DP>
__global__ __launch_bounds__(256) void merge_kernel(Blocks k) {
    __shared__ uint64_t sums[4];
    const AttnBlocksArgs &a = k.a;
    const uint32_t G = a.H / a.Hkv, kh = blockIdx.x % a.Hkv;
    Place at;
    if (!place_of(a.pb, G, kUnit, blockIdx.x / a.Hkv, &at)) return;
    // quads before sequence at.b
    uint64_t sum = 0, all = 0;
    for (uint32_t b = threadIdx.x; b < a.pb.batch; b += 256) {
        uint32_t u, q;
        sequence_quads(a, b, &u, &q);
        all += uint64_t(u) * q * a.Hkv;
        if (b < at.b) sum += uint64_t(u) * q * a.Hkv;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        sum += __shfl_xor(sum, o, 64);
        all += __shfl_xor(all, o, 64);
    }
    __shared__ uint64_t alls[4];
    if ((threadIdx.x & 63u) == 0) sums[threadIdx.x >> 6] = sum, alls[threadIdx.x >> 6] = all;
    __syncthreads();
    sum = sums[0] + sums[1] + sums[2] + sums[3];
    all = alls[0] + alls[1] + alls[2] + alls[3];
    uint32_t units, quads;
    sequence_quads(a, at.b, &units, &quads);
    const uint64_t share = share_of(all);
    const uint64_t q0 = sum + (uint64_t(at.unit) * a.Hkv + kh) * quads;
    const uint64_t w0 = q0 / share, w1 = (q0 + quads - 1) / share;
    if (w0 == w1) return;      // one workgroup had all of it
    const uint64_t id = uint64_t(at.lo * G / kUnit + at.b + at.unit) * a.Hkv + kh;
    const float *src = k.part + (id + w0) * (kUnit * (DP + 2));
    const uint32_t np = uint32_t(w1 - w0 + 1), n = at.hi - at.lo, R = n * G;
    const uint32_t rows = R - at.unit * kUnit < kUnit ? R - at.unit * kUnit : kUnit;
    typedef typename E::T T;
    constexpr uint32_t kStride = kUnit * (DP + 2);
    const uint32_t wave = pk_uni(threadIdx.x >> 6);
    for (uint32_t c = wave; c < rows; c += 4) {
        const uint32_t rr = at.unit * kUnit + c, t = rr / G;
        const bool none = visible_keys(a.lens[at.b], n, t, a.bucket) == 0;
        T *out = static_cast<T *>(a.out) + (uint64_t(at.lo + t) * a.H + kh * G + (rr - t * G)) * a.D;
        join_row<E, DP>(src + c * (DP + 2), kStride, np, a.D, none, out);
    }
}

// -------------------------------------------------------------- tiled form ----
// Many rows a sequence. As AttentionPacked's tiles: 128 packed rows a workgroup, 32 a
// wavefront, over 64-key tiles, a tile's weights under the next one's scores; but the
// tiles are the cache's bytes, loaded into registers a tile ahead and widened to f16
// (exact) on their way into LDS. Q as f16, each row by a power of two so that its largest
// is in [2^14, 2^15): exact for 16-bit rows but for elements 2^-38 of the largest, and in
// two parts, 22 bits, for f32 rows; a row's power and log2(e) / divisor join K's scales.
// The scale of a 16-key step is one number: K's |ks| times the row's factor is the
// step's c, with s c - m one instruction; V's joins the weights as in the few-row form, w =
// p |vs| 2^(7 - ve), and the sum l takes p itself, in f32, whatever the scales are. (V's
// scale in the exponent and l's share of it taken back by 1 / |vs| was an instruction a
// weight less; scales far below the row's largest lost their keys' part of l that way.)
// 2^ve is above every finite |vs| of the steps the row sees so far. A scale's sign is put
// on the bytes on the way into LDS.
// In a tile that some row does not see to its end, s is scaled and limited first (c = 1),
// and a step that a row does not see brings it no scale.
// A row tile and kv head is a workgroup's, whole (chunk_tile_kernel), where that gives
// kManyRounds times what the GPU holds at once, or where the longest tile's keys are few
// beside the tiles there are (tiles_whole: known on the device, so all three kernels are
// launched and those not needed return; 7 us of the other split's 164). Else the tiles
// are dealt as equal shares of a line of keys, one share for each workgroup
// that the GPU holds: unit u (a row tile) of a sequence costs kStart + past' + S (u + 1)
// keys, past' what its rows see before their own to a multiple of 64, S = ceil(128 / G)
// the tokens that a unit spans at most, and kStart what starting and ending a unit
// takes in keys' time (14 to 17 us of head_dim 128 against 2.3 a 64-key tile with two
// workgroups a CU; 4 chunks of 301 to 1024 rows behind up to 6000 keys with 192, 384 and 768
// of them: 171, 165 and 179 us, 111, 117 and 129 of 64 dims, 434, 372 and 401 of 256, 287,
// 298 and 322 of f32 rows), so that a sequence's cost and the unit at a place of the line are
// closed forms. A unit's keys begin at its place kStart; cuts fall on tiles. A unit
// that is cut leaves partials for join_kernel.
// Bound by the vector units beside the matrix cores (450 vector instructions a wavefront
// and tile, a third of them the widening and the scales, against 32 matrix instructions:
// those are busy 29% of the cycles) and by the units' starts: 4 chunks of 301 to 1024 rows
// behind up to 6000 keys, 32 heads on 8 of 128 dims, 165 us, 0.53 PFLOP/s, join_kernel 15
// to 20 us of them; one of 1024 rows behind 4000 keys 0.57; f32 rows, whose every product is
// two, 298 us. A wavefront a row (below) took 793 us.
constexpr uint32_t kRows = 128, kKeys = 64, kManyRounds = 4, kMinKeys = 256, kStart = 384;

struct Chunk {
    AttnBlocksArgs a;
    float mul;
    uint32_t shift, places, shares;
    float *part;         // [places * Hkv + shares][kRows][DP + 2], as Blocks::part
};

// A partial: O as the lanes hold it, 4 dims (8 g + 4 (lane / 32) on) of row lane % 32 a
// 16-byte element, wavefront by wavefront and 8 dims by 8 dims (q), so that every access
// is 1 KB of whole lines; then the rows' maxima, then their sums.
template <int DP>
__device__ __forceinline__ uint32_t part_of(uint32_t wave, uint32_t q, uint32_t lane) {
    return ((wave * (DP / 8) + q) * 64 + lane) * 4;
}

// Four int8 (xor 0x80) as f16.
__device__ __forceinline__ uint2 widen4(uint32_t w) {
    typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
    const uint32_t b = w ^ 0x80808080u;
    const uint2 m = {__builtin_amdgcn_perm(0x64646464u, b, 0x04010400u), __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)};
    return __builtin_bit_cast(uint2, __builtin_bit_cast(f16x4, m) - (f16x4)(_Float16)1152.0f);
}

__device__ __forceinline__ f32x16 mfma_f16(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// The largest of a row's 64 scores, a step's times its factor (not below 0).
__device__ __forceinline__ float largest(const float (&mg)[4], const float (&c)[4]) {
    const float mt = fmaxf(fmaxf(mg[0] * c[0], mg[1] * c[1]), fmaxf(mg[2] * c[2], mg[3] * c[3]));
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(mt), __float_as_uint(mt), false, false);
    return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
}

template <int DP>
struct ChunkLds {
    uint8_t k0[128 * DP], k1[128 * DP], v0[128 * DP], v1[128 * DP];   // kKeys rows of 2 DP bytes each
};

// Keys [c0, c1) (whole tiles, but for the last) of row tile at.unit of sequence at.b and
// kv head kh, to the output (whole) or to a partial at dst.
template <class E, int DP>
__device__ __forceinline__ void chunk_segment(const Chunk &k, const Place &at, uint32_t kh, uint32_t c0, uint32_t c1,
                                              bool whole, float *dst, ChunkLds<DP> &lds) {
    constexpr int RB = 2 * DP, NK = DP / 16, DB = DP / 32, CT = DP / 64;   // CT: 16-byte chunks a thread widens
    constexpr bool kF32 = std::is_same_v<E, F32>;
    constexpr int P = kF32 ? 2 : 1;
    constexpr float kLag = 8.0f;
    typedef typename E::T T;
    uint8_t *const kb0 = lds.k0, *const kb1 = lds.k1, *const vb0 = lds.v0, *const vb1 = lds.v1;
    const AttnBlocksArgs &a = k.a;
    const uint32_t G = a.H / a.Hkv;
    const uint32_t t0 = at.lo, n = at.hi - at.lo, R = n * G, r0 = at.unit * kRows;
    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 31, lg = lane >> 5;
    const uint32_t wave = pk_uni(uint32_t(tid) >> 6);
    const int64_t len = a.lens[at.b];
    auto sees = [&](uint32_t r) { return visible_keys(len, n, (r < R ? r : R - 1) / G, a.bucket); };
    const uint32_t wr0 = r0 + 32 * wave, row = wr0 + lr < R ? wr0 + lr : R - 1, tok = row / G;
    const uint32_t lim = sees(row), wmin = pk_uni(sees(wr0));
    const uint32_t kall = pk_uni(sees(r0 + kRows - 1));
    const uint32_t j1 = c0 < kall ? c0 : kall, kmax = c1 < kall ? c1 : kall;
    const bool live = pk_uni(wr0 < R);

    // the tile's bytes: key tid / 4, chunks tid % 4 + 4 i of its row; its step's scales
    const uint64_t plane = uint64_t(at.b) * a.Hkv + kh;
    const auto rk = range(a.kq + plane * a.bucket * a.D, a.bucket * a.D);
    const auto rv = range(a.vq + plane * a.bucket * a.D, a.bucket * a.D);
    const uint32_t nb = (a.bucket + a.block - 1) >> k.shift;
    const float *ks = a.ks + plane * nb, *vs = a.vs + plane * nb;
    const uint32_t key = uint32_t(tid) >> 2, part = uint32_t(tid) & 3u;
    auto scale_at = [&](const float *x, uint32_t j) {
        const uint32_t i = j >> k.shift;
        return x[i < nb ? i : nb - 1];
    };
    auto uniform_at = [&](const float *x, uint32_t j) {   // alike in all lanes: a scalar load
        const uint32_t i = j >> k.shift;
        return reinterpret_cast<const __attribute__((address_space(4))) float *>(
            reinterpret_cast<uintptr_t>(x))[i < nb ? i : nb - 1];
    };
    u32x4 kr[CT], vr[CT];
    float ksk, vsk;
    auto fetch = [&](const __amdgpu_buffer_rsrc_t r, uint32_t j, u32x4 (&x)[CT]) {
#pragma unroll
        for (int i = 0; i < CT; ++i) {
            const uint32_t b = 16 * (part + 4 * i), off = j < kall && b < a.D ? (j + key) * a.D + b : kOob;
            x[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
        }
    };
    auto fetch_k = [&](uint32_t j) { fetch(rk, j, kr), ksk = scale_at(ks, j + key); };
    auto fetch_v = [&](uint32_t j) { fetch(rv, j, vr), vsk = scale_at(vs, j + key); };
    auto put = [&](uint8_t *buf, const u32x4 (&x)[CT], float scale, const uint32_t (&to)[2]) {
        const uint32_t flip = __float_as_uint(scale) >> 31 ? 0x80008000u : 0u;
        const bool plain = !__any(flip != 0);
#pragma unroll
        for (int i = 0; i < CT; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint2 lo = widen4(x[i][2 * h]), hi = widen4(x[i][2 * h + 1]);
                u32x4 v = {lo.x, lo.y, hi.x, hi.y};
                if (!plain) {
                    asm volatile("");      // a branch of its own
#pragma unroll
                    for (int w = 0; w < 4; ++w) v[w] ^= flip;
                }
                *reinterpret_cast<u32x4 *>(buf + (to[h] ^ (128u * i))) = v;
            }
    };
    // chunk 2 (part + 4 i) + h of the key's row, swizzled
    uint32_t kto[2], vto[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        kto[h] = key * RB + (((2u * part + h) ^ swz_k<DP>(key)) * 16u);
        vto[h] = key * RB + (((2u * part + h) ^ swz_v<DP>(key)) * 16u);
    }
    auto put_k = [&](uint8_t *buf) { put(buf, kr, ksk, kto); };
    auto put_v = [&](uint8_t *buf) { put(buf, vr, vsk, vto); };
    fetch_k(j1);
    fetch_v(j1);

    // Q's parts, by way of LDS: whole rows into 32 QB bytes of the wavefront's own, a row
    // past R a copy of the last
    constexpr uint32_t QB = sizeof(T) * DP, QC = QB / 16, QR = 1024 / QB;
    uint8_t *qbuf = kF32 ? (wave & 2 ? (wave & 1 ? vb1 : vb0) : (wave & 1 ? kb1 : kb0))
                         : (wave & 2 ? vb1 : kb1) + (wave & 1) * (32 * QB);
    auto chunk_at = [](uint32_t bytes, uint32_t r, uint32_t q) {   // 16-byte chunk q of row r
        return r * bytes + (q ^ (r & (bytes / 16 - 1u) & 15u)) * 16u;
    };
    {
        const uint32_t tok0 = r0 / G;
        const auto r = range(static_cast<const T *>(a.q) + uint64_t(t0 + tok0) * a.q_stride + kh * G * a.D, kOob);
#pragma unroll
        for (uint32_t i = 0; i < 32 / QR; ++i) {
            const uint32_t at_row = i * QR + lane / QC, rr = wr0 + at_row < R ? wr0 + at_row : R - 1, t = rr / G;
            const uint32_t q = (lane % QC) ^ (at_row & (QC - 1u) & 15u);
            const uint32_t off = ((t - tok0) * a.q_stride + (rr - t * G) * a.D) * uint32_t(sizeof(T)) + 16 * q;
            load_to_lds(r, qbuf + 1024 * i, 16 * q < a.D * sizeof(T) ? off : kOob);
        }
    }
    u32x4 qf[P][NK];
    float mul;
    {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt((15 << 8) | (7 << 4));   // vmcnt(0)
        asm volatile("" ::: "memory");
        float top = 0.0f;
        bool bad = false;
        auto chunk = [&](int i, float (&x)[8]) {   // dims 16 i + 8 lg on
#pragma unroll
            for (int w = 0; w < int(sizeof(T)) / 2; ++w) {
                const u32x4 v = *reinterpret_cast<const u32x4 *>(qbuf + chunk_at(QB, lr, (2 * i + lg) * (sizeof(T) / 2) + w));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (kF32) {
                        x[4 * w + e] = __uint_as_float(v[e]);
                    } else {
                        x[2 * e] = E::widen(uint16_t(v[e]));
                        x[2 * e + 1] = E::widen(uint16_t(v[e] >> 16));
                    }
                }
            }
        };
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            float x[8];
            chunk(i, x);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                top = fmaxf(top, fabsf(x[e]));
                bad |= !(fabsf(x[e]) <= 3.4028235e38f);
            }
        }
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        bad |= __shfl_xor(int(bad), 32, 64) != 0;
        int qe = 0;
        if (top > 0.0f && !bad) {
            (void)frexpf(top, &qe);     // top < 2^qe
            qe = 15 - qe;
        }
        mul = bad ? __uint_as_float(0x7fc00000u) : ldexpf(k.mul, -qe);
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            float x[8];
            chunk(i, x);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float y0 = bad ? 0.0f : ldexpf(x[2 * e], qe), y1 = bad ? 0.0f : ldexpf(x[2 * e + 1], qe);
                qf[0][i][e] = pack2<F16>(y0, y1);
                if constexpr (kF32) qf[P - 1][i][e] = pack2<F16>(y0 - float(_Float16(y0)), y1 - float(_Float16(y1)));
            }
        }
    }

    f32x16 o[DB], s[2];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    int ve = kVeMin;
    const uint32_t kat = k_place<DP>(lane), vat = v_place<DP>(lane);
    // of the steps of the tile in s: K's factor, and |vs| where the row sees a key of them, else 0
    float c[4], v[4];

    float nk[4], nv[4];      // the next tile's scales, loaded a tile's scores ahead of their use
    auto load_scales = [&](uint32_t j) __attribute__((always_inline)) {
#pragma unroll
        for (int g = 0; g < 4; ++g) nk[g] = uniform_at(ks, j + 16 * g), nv[g] = uniform_at(vs, j + 16 * g);
    };
    // the scales of tile j, and s limited; the largest exponent of the steps the row sees
    auto take = [&](int g) __attribute__((always_inline)) { c[g] = fabsf(nk[g]) * mul, v[g] = fabsf(nv[g]); };
    auto above = [&](float x) {        // the least 2^ve above x; kVeMin of a zero, an infinity or a NaN
        return x > 0.0f && x <= 3.4028235e38f ? __builtin_amdgcn_frexp_expf(x) : kVeMin;
    };
    auto limit = [&](uint32_t j, int *top) __attribute__((always_inline)) {
        take(0);
        const bool all = j + kKeys <= wmin;
        if (k.shift >= 6) {            // one block holds the tile
            asm volatile("");
            if (j >= lim) v[0] = 0.0f;
#pragma unroll
            for (int g = 1; g < 4; ++g) c[g] = c[0], v[g] = v[0];
            *top = above(v[0]);
        } else {
#pragma unroll
            for (int g = 1; g < 4; ++g) take(g);
            if (!all) {
                asm volatile("");
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    if (j + 16 * g >= lim) v[g] = 0.0f;
            }
            *top = kVeMin;
#pragma unroll
            for (int g = 0; g < 4; ++g) *top = above(v[g]) > *top ? above(v[g]) : *top;
        }
        if (all) return;
        int see = int(lim < kmax ? lim : kmax) - int(j) - 4 * lg;
        asm volatile("" : "+v"(see));
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                s[h][r] = 32 * h + 8 * (r >> 2) + (r & 3) < see ? s[h][r] * c[2 * h + (r >> 3)] : -INFINITY;
#pragma unroll
        for (int g = 0; g < 4; ++g) c[g] = 1.0f;
    };
    auto rescale = [&](float mt, int top) __attribute__((always_inline)) {
        if (__any(mt > m + kLag || top > ve)) {
            const float mn = mt > m + kLag ? mt : m;
            const int vn = top > ve ? top : ve;
            const float al = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            const float sh = ldexpf(al, ve - vn);
            l *= al;
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] *= sh;
            m = mn, ve = vn;
        }
    };
    u32x4 pf[P][4];
    float ref, f[4];              // per step: |vs| 2^(7 - ve)
    auto prepare = [&]() __attribute__((always_inline)) {
        ref = m == -INFINITY ? 0.0f : m;
        f[0] = weight_factor(v[0], ve);
        if (k.shift >= 6) {
            asm volatile("");
#pragma unroll
            for (int g = 1; g < 4; ++g) f[g] = f[0];
        } else {
#pragma unroll
            for (int g = 1; g < 4; ++g) f[g] = weight_factor(v[g], ve);
        }
    };
    auto weight_pair = [&](int i) __attribute__((always_inline)) {
        const int g = i >> 2;
        float w[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float p = __builtin_amdgcn_exp2f(fmaf(s[i >> 3][2 * (i & 7) + e], c[g], -ref));
            l += p;
            w[e] = kF32 ? rounded(p * f[g]) : p * f[g];
        }
        uint32_t hi = pack2<F16>(w[0], w[1]);
        if constexpr (kF32) {
            typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
            const f16x2 f = __builtin_bit_cast(f16x2, hi);
            uint32_t lo = pack2<F16>(left_over(w[0], float(f[0])), left_over(w[1], float(f[1])));
            asm volatile("" : "+v"(lo));
            pf[P - 1][i >> 2][i & 3] = lo;
        }
        asm volatile("" : "+v"(hi), "+v"(l));   // here, not where they are used
        pf[0][i >> 2][i & 3] = hi;
    };
    auto scores = [&](const uint8_t *buf, f32x16 (&to)[2], const bool weigh) __attribute__((always_inline)) {
        constexpr int kPairs = 16 / NK;
        uint32_t x = kat;
        asm volatile("" : "+v"(x));
        u32x4 kf[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) kf[i][h] = k_frag<DP>(buf, x, i, h);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 16; ++r) to[h][r] = 0.0f;
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int h = 0; h < 2; ++h) to[h] = mfma_f16(kf[i & 1][h], qf[p][i], to[h]);
            if (i + 2 < NK)
#pragma unroll
                for (int h = 0; h < 2; ++h) kf[i & 1][h] = k_frag<DP>(buf, x, i + 2, h);
            if (weigh)
#pragma unroll
                for (int q = kPairs * i; q < kPairs * (i + 1); ++q) weight_pair(q);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    // O^T += V^T . P^T of one tile, beside the largest of the next tile's scores
    auto products = [&](const uint8_t *buf) __attribute__((always_inline)) {
        constexpr int kSteps = 2 * DB, kMax = 32 / kSteps;
        uint32_t x = vat;
        asm volatile("" : "+v"(x));
        u32x4 vf[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) vf[i][h] = v_frag<DP>(buf, x, i / (DB / 2), 2 * (i % (DB / 2)) + h);
        float mg[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            const int st = i / (DB / 2), d = 2 * (i % (DB / 2));
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int h = 0; h < 2; ++h) o[d + h] = mfma_f16(vf[i & 1][h], pf[p][st], o[d + h]);
            if (i + 2 < kSteps)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    vf[i & 1][h] = v_frag<DP>(buf, x, (i + 2) / (DB / 2), 2 * ((i + 2) % (DB / 2)) + h);
#pragma unroll
            for (int r = kMax * i; r < kMax * (i + 1); ++r) mg[r >> 3] = fmaxf(mg[r >> 3], s[r >> 4][r & 15]);
        }
        __builtin_amdgcn_sched_barrier(0);
        return largest(mg, c);
    };
    auto step = [&](uint8_t *k_this, uint8_t *k_next, uint8_t *v_this, uint8_t *v_next, uint32_t j)
        __attribute__((always_inline)) {
        lds_barrier();     // k_next and v_this are filled, k_this and v_next are done with
        const bool more = j + kKeys < kmax;
        if (more) {
            load_scales(j + kKeys);
            put_k(k_this);
            put_v(v_next);
            fetch_k(j + 3 * kKeys);
            fetch_v(j + 2 * kKeys);
        }
        if (!live) return;
        prepare();
        int top = kVeMin;
        if (more) {
            f32x16 nx[2];
            scores(k_next, nx, true);
            s[0] = nx[0], s[1] = nx[1];
            limit(j + kKeys, &top);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) weight_pair(i);
        }
        const float mt = products(v_this);
        if (more) rescale(mt, top);
    };
    if (j1 < kmax) {
        load_scales(j1);
        if constexpr (kF32) lds_barrier();   // Q has been read where these go
        put_k(kb0);
        put_v(vb0);
        fetch_k(j1 + kKeys);
        fetch_v(j1 + kKeys);
        lds_barrier();     // and here
        put_k(kb1);
        fetch_k(j1 + 2 * kKeys);
        scores(kb0, s, false);
        int top;
        limit(j1, &top);
        float mg[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int r = 0; r < 32; ++r) mg[r >> 3] = fmaxf(mg[r >> 3], s[r >> 4][r & 15]);
        rescale(largest(mg, c), top);
        for (uint32_t j = j1; j < kmax; j += 2 * kKeys) {
            step(kb0, kb1, vb0, vb1, j);
            if (j + kKeys < kmax) step(kb1, kb0, vb1, vb0, j + kKeys);
        }
    }
    l += __shfl_xor(l, 32, 64);
    if (!whole) {
        if (!live) return;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                f32x4 x;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = ldexpf(o[d][4 * g + e], ve - 7);
                *reinterpret_cast<f32x4 *>(dst + part_of<DP>(wave, 4 * d + g, lane)) = x;
            }
        if (lg == 0) dst[kRows * DP + 32 * wave + lr] = m, dst[kRows * (DP + 1) + 32 * wave + lr] = l;
        return;
    }
    // rows stored whole through LDS (16-bit), or as they are (f32); 2^(ve - 7) last, for it
    // may be a subnormal
    const float inv = lim == 0 ? 0.0f : 1.0f / l;
    auto result = [&](float x) { return ldexpf(x * inv, ve - 7); };
    T *out = static_cast<T *>(a.out) + (uint64_t(t0) * a.H + kh * G) * a.D;
    if constexpr (kF32) {
        if (wr0 + lr >= R) return;
        T *to = out + (uint64_t(tok) * a.H + (row - tok * G)) * a.D;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const uint32_t dim = 32 * d + 8 * g + 4 * lg;
                if (dim < a.D)
#pragma unroll
                    for (int e = 0; e < 4; ++e) to[dim + e] = result(o[d][4 * g + e]);
            }
    } else {
        lds_barrier();
        uint8_t *turn = (wave & 2 ? kb1 : kb0) + (wave & 1) * (32 * RB);
        constexpr uint32_t CPR = RB / 16, RPL = 1024 / RB;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<uint2 *>(turn + chunk_at(RB, lr, 4 * d + g) + 8 * lg) =
                    make_uint2(pack2<E>(result(o[d][4 * g]), result(o[d][4 * g + 1])),
                               pack2<E>(result(o[d][4 * g + 2]), result(o[d][4 * g + 3])));
        __builtin_amdgcn_wave_barrier();
        const uint32_t q = lane % CPR;
#pragma unroll
        for (uint32_t i = 0; i < 32 / RPL; ++i) {
            const uint32_t r = i * RPL + lane / CPR, rr = wr0 + r, t = rr / G;
            if (rr < R && 8 * q < a.D)
                *reinterpret_cast<u32x4 *>(out + (uint64_t(t) * a.H + (rr - t * G)) * a.D + 8 * q) =
                    *reinterpret_cast<const u32x4 *>(turn + chunk_at(RB, r, q));
        }
    }
}

// The row tiles of sequence b and the line of their costs, one kv head's.
struct Units {
    uint32_t units, past, S;
    __device__ __forceinline__ uint64_t before(uint32_t u) const {   // cost of units 0 .. u - 1
        return uint64_t(u) * (kStart + past) + uint64_t(S) * (uint64_t(u) * (u + 1) / 2);
    }
    __device__ __forceinline__ uint32_t holding(uint64_t at) const {   // the unit at place `at`
        uint32_t lo = 0, hi = units;
        while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (before(mid) <= at) lo = mid;
            else hi = mid;
        }
        return lo;
    }
};
__device__ __forceinline__ Units sequence_units(const AttnBlocksArgs &a, uint32_t b) {
    const uint32_t lo = start_of(a.pb, b), hi = start_of(a.pb, b + 1), G = a.H / a.Hkv, n = hi > lo ? hi - lo : 0u;
    const uint32_t past = visible_keys(int64_t(a.lens[b]) - n, 1, 0, a.bucket);
    return Units{(n * G + kRows - 1) / kRows, (past + kKeys - 1) / kKeys * kKeys, (kRows + G - 1) / G};
}
__device__ __forceinline__ uint64_t keys_of(uint64_t total, uint32_t shares) {
    const uint64_t s = (total + shares - 1) / shares;
    return s < kMinKeys ? kMinKeys : s;
}

// Whether the row tiles go whole to workgroups. Whole, the GPU waits for the last long
// one, about half of its time; cut, each share starts one tile more and the partials are
// joined. In us whole and cut, of 128 dims, 64, 256 and 128 of f32 rows: 4 sequences of 301
// to 1024 rows, the longest tile's keys 1.7 for each tile: 45 and 76, 34 and 52, 100 and
// 146, 79 and 106; behind up to 6000 keys, 11 for each: 263 and 164, 195 and 117, 420 and
// 369, 333 and 298; 8 of 200 to 500 rows behind up to 3000, 4.7 for each: 120 and 94, 89 and
// 68, 225 and 200, 182 and 159; 16, 2.5 for each: 126 and 160, 95 and 117 (256 dims and f32
// are many times what the GPU holds). One of 1024 rows behind 4000, 20 for each: 159 and
// 131, 120 and 91, but 272 and 292, 215 and 237.
// The threads of a workgroup call it; all get the answer.
__device__ __forceinline__ bool tiles_whole(const AttnBlocksArgs &a, uint32_t (&most)[4], uint32_t (&many)[4]) {
    uint32_t keys = 0, units = 0;
    for (uint32_t b = threadIdx.x; b < a.pb.batch; b += 256) {
        const Units u = sequence_units(a, b);
        const uint32_t x = u.units ? u.past + u.S * u.units : 0u;
        keys = x > keys ? x : keys;
        units += u.units;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const uint32_t x = __shfl_xor(keys, o, 64);
        keys = x > keys ? x : keys;
        units += __shfl_xor(units, o, 64);
    }
    if ((threadIdx.x & 63u) == 0) most[threadIdx.x >> 6] = keys, many[threadIdx.x >> 6] = units;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) keys = most[w] > keys ? most[w] : keys;
    return keys <= 1000 + 2 * a.Hkv * (many[0] + many[1] + many[2] + many[3]);
}

// A row tile a workgroup: grid places * Hkv, those that see most keys first.
template <class E, int DP>
__global__ __launch_bounds__(256, (DP > 128 || sizeof(typename E::T) == 4 ? 1 : 2)) void chunk_tile_kernel(Chunk k) {
    __shared__ __attribute__((aligned(1024))) ChunkLds<DP> lds;
    if (blockIdx.x == 0) check_starts(k.a.pb);
    __shared__ uint32_t most[4], many[4];
    if (k.shares && !tiles_whole(k.a, most, many)) return;
    Place at;
    if (!place_of(k.a.pb, k.a.H / k.a.Hkv, kRows, k.places - 1 - blockIdx.x / k.a.Hkv, &at)) return;
    chunk_segment<E, DP>(k, at, blockIdx.x % k.a.Hkv, 0, k.a.bucket, true, nullptr, lds);
}

template <class E, int DP>
__global__ __launch_bounds__(256, (DP > 128 || sizeof(typename E::T) == 4 ? 1 : 2)) void chunk_shares_kernel(Chunk k) {
    __shared__ __attribute__((aligned(1024))) ChunkLds<DP> lds;
    __shared__ uint64_t sums[4];
    __shared__ uint32_t most[4], many[4];
    __shared__ Line found;
    const AttnBlocksArgs &a = k.a;
    if (tiles_whole(a, most, many)) return;
    const uint32_t G = a.H / a.Hkv;
    const Line ln = find_line(a.pb.batch, [&](uint32_t b) {
        const Units u = sequence_units(a, b);
        return u.before(u.units) * a.Hkv;
    }, [&](uint64_t total) { return blockIdx.x * keys_of(total, k.shares); }, sums, &found);
    const uint64_t share = keys_of(ln.total, k.shares);
    uint64_t pos = blockIdx.x * share, base = ln.at;
    const uint64_t end = pos + share < ln.total ? pos + share : ln.total;
    for (uint32_t b = ln.b; pos < end && b < a.pb.batch; ++b) {
        const Units u = sequence_units(a, b);
        const uint64_t one = u.before(u.units), all = one * a.Hkv;
        while (pos < end && pos < base + all) {
            const uint32_t kh = pk_uni(uint32_t((pos - base) / one));
            const uint64_t in = pos - base - kh * one;            // place in the head's line
            const uint32_t unit = pk_uni(u.holding(in));
            const uint64_t from = u.before(unit), cost = u.before(unit + 1) - from;
            const uint64_t left = in - from, right = left + (end - pos) < cost ? left + (end - pos) : cost;
            pos += right - left;
            // cuts at the next tile's end; the unit's own end takes what is left, and one
            // before its keys begin leaves them to the share behind it
            auto cut = [](uint64_t x) { return x <= kStart ? 0u : uint32_t((x - kStart + kKeys - 1) / kKeys * kKeys); };
            const uint32_t c0 = pk_uni(cut(left)), c1 = pk_uni(right == cost ? 0xffffffffu : cut(right));
            if (c1 == 0) continue;
            const Place at{pk_uni(b), pk_uni(start_of(a.pb, b)), pk_uni(start_of(a.pb, b + 1)), unit};
            const uint64_t id = uint64_t(at.lo * G / kRows + at.b) * a.Hkv + uint64_t(kh) * u.units + unit;
            lds_barrier();     // the segment before is done with the buffers
            chunk_segment<E, DP>(k, at, kh, c0, c1, pk_uni(c0 == 0 && right == cost),
                                 k.part + (id + blockIdx.x) * (kRows * (DP + 2)), lds);
        }
        base += all;
    }
}

// Joins the partials of a row tile that shares cut: grid places * Hkv * joins, a
// wavefront 32 rows and, in turn, 8 of their dims. `joins` fills 1024 workgroups with the
// places that there are, up to 8 dims a workgroup.
template <class E, int DP>
__global__ __launch_bounds__(256) void join_kernel(Chunk k, uint32_t joins) {
    __shared__ uint64_t sums[4], alls[4];
    __shared__ uint32_t most[4], many[4];
    const AttnBlocksArgs &a = k.a;
    const uint32_t G = a.H / a.Hkv, kh = blockIdx.x % a.Hkv, rest = blockIdx.x / a.Hkv, lane = threadIdx.x & 63u;
    Place at;
    if (!place_of(a.pb, G, kRows, rest / joins, &at) || tiles_whole(a, most, many)) return;
    uint64_t sum = 0, all = 0;       // costs before sequence at.b, and of all
    for (uint32_t b = threadIdx.x; b < a.pb.batch; b += 256) {
        const Units u = sequence_units(a, b);
        const uint64_t c = u.before(u.units) * a.Hkv;
        all += c;
        sum += b < at.b ? c : 0;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        sum += __shfl_xor(sum, o, 64);
        all += __shfl_xor(all, o, 64);
    }
    if (lane == 0) sums[threadIdx.x >> 6] = sum, alls[threadIdx.x >> 6] = all;
    __syncthreads();
    sum = sums[0] + sums[1] + sums[2] + sums[3];
    all = alls[0] + alls[1] + alls[2] + alls[3];
    const Units u = sequence_units(a, at.b);
    // the share that holds the unit's first keys, and its last
    const uint64_t share = keys_of(all, k.shares), q0 = sum + kh * u.before(u.units) + u.before(at.unit);
    const uint64_t w0 = (q0 + kStart) / share, w1 = (sum + kh * u.before(u.units) + u.before(at.unit + 1) - 1) / share;
    if (w0 == w1) return;            // one workgroup had all of it
    const uint32_t np = uint32_t(w1 - w0 + 1), n = at.hi - at.lo, R = n * G;
    const uint64_t id = uint64_t(at.lo * G / kRows + at.b) * a.Hkv + uint64_t(kh) * u.units + at.unit;
    constexpr uint32_t kStride = kRows * (DP + 2);
    const float *src = k.part + (id + w0) * kStride;
    const uint32_t wave = pk_uni(threadIdx.x >> 6), in = 32 * wave + (lane & 31u), rr = at.unit * kRows + in;
    if (at.unit * kRows + 32 * wave >= R) return;
    const float *ms = src + kRows * DP + in, *ls = ms + kRows;
    float M = -INFINITY, l = 0.0f;
    for (uint32_t w = 0; w < np; w += 8) {
        float x[8], y[8], mx = M;
#pragma unroll
        for (uint32_t q = 0; q < 8; ++q) {
            const bool is = w + q < np;
            x[q] = is ? ms[(w + q) * kStride] : -INFINITY, y[q] = is ? ls[(w + q) * kStride] : 0.0f;
        }
#pragma unroll
        for (uint32_t q = 0; q < 8; ++q) mx = fmaxf(mx, x[q]);
        const float ref = mx == -INFINITY ? 0.0f : mx;
        l *= __builtin_amdgcn_exp2f(M - ref);
#pragma unroll
        for (uint32_t q = 0; q < 8; ++q) l = fmaf(y[q], __builtin_amdgcn_exp2f(x[q] - ref), l);
        M = mx;
    }
    const float ref = M == -INFINITY ? 0.0f : M;
    const uint32_t t = (rr < R ? rr : R - 1) / G;
    const bool none = visible_keys(a.lens[at.b], n, t, a.bucket) == 0;
    auto *out = static_cast<typename E::T *>(a.out) + (uint64_t(at.lo + t) * a.H + kh * G + (rr - t * G)) * a.D;
    for (uint32_t c = rest % joins; 8 * c < a.D; c += joins) {
        f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
        const float *po = src + part_of<DP>(wave, c, lane);
        for (uint32_t w = 0; w < np; w += 8) {
            f32x4 x[8];
            float e[8];
#pragma unroll
            for (uint32_t q = 0; q < 8; ++q) {
                const uint32_t at_w = w + q < np ? w + q : np - 1;
                x[q] = *reinterpret_cast<const f32x4 *>(po + at_w * kStride);
                e[q] = ms[at_w * kStride];
            }
#pragma unroll
            for (uint32_t q = 0; q < 8; ++q) {
                const bool is = w + q < np;
                const float ew = is ? __builtin_amdgcn_exp2f(e[q] - ref) : 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = fmaf(is ? x[q][i] : 0.0f, ew, o[i]);
            }
        }
        if (rr >= R) continue;
        typename E::T v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = E::narrow(none ? 0.0f : o[i] / l);
        __builtin_memcpy(out + 8 * c + 4 * (lane >> 5), v, sizeof v);
    }
}

// What the matrix forms take: 16-byte rows of q, the caches and the output, offsets
// within a row tile's q below 2^30 bytes, whole 16-key steps in a block.
bool matrix_applies(const AttnBlocksArgs &a) {
    auto at16 = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    const uint32_t es = a.dtype == 8 ? 4 : 2;
    return a.D % 16 == 0 && a.D <= 256 && a.block >= 16 && (a.block & (a.block - 1)) == 0 && at16(a.kq) &&
           at16(a.vq) && at16(a.q) && at16(a.out) && uint64_t(a.q_stride) * es % 16 == 0 && a.q_stride < (1u << 21);
}
uint32_t few_places(const AttnBlocksArgs &a) {
    return uint32_t(uint64_t(a.pb.tokens) * (a.H / a.Hkv) / kUnit) + a.pb.batch;
}
uint32_t padded(uint32_t D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }
bool few_direct(const AttnBlocksArgs &a) {
    return a.bucket <= kDirect && uint64_t(few_places(a)) * a.Hkv <= kDirectUnits;
}
// At most 16 packed rows a sequence on average, 32 where no shares are cut: 32 sequences of
// 4000 keys, 58 us against the tiles' 94 with 16 rows, 80 and 95 with 32, 157 and 115 with
// 64, but 61 and 42 with 32 rows and 1 to 4000 keys; of 900 keys, 32 rows, 4 and 16
// sequences 17 and 32 us against 23 and 35. An average: the lengths are on the device. Empty
// sequences count (256 rows behind 4096 keys 54 us alone, 61 beside 63 of them), and rows of
// both kinds in one call take one form: 64 decode rows over 8192 keys 169 us, a chunk of 512
// rows 117, both in a call 443.
bool few_rows(const AttnBlocksArgs &a) {
    const uint32_t rows = few_direct(a) ? 2 * kUnit : kUnit;
    return uint64_t(a.pb.tokens) * (a.H / a.Hkv) <= uint64_t(rows) * a.pb.batch;
}

template <class E, int DP>
void launch_few(const Blocks &k, hipStream_t stream) {
    const uint32_t grid = k.places * k.a.Hkv;
    if (few_direct(k.a)) {
        constexpr int W = DP > 128 ? 4 : 8;
        few_direct_kernel<E, DP, W><<<grid, 64 * W, 0, stream>>>(k);
        return;
    }
    few_shares_kernel<E, DP><<<kShares, 256, 0, stream>>>(k);
    merge_kernel<E, DP><<<grid, 256, 0, stream>>>(k);
}
uint32_t chunk_places(const AttnBlocksArgs &a) {
    return uint32_t(uint64_t(a.pb.tokens) * (a.H / a.Hkv) / kRows) + a.pb.batch;
}
// Workgroups that the GPU holds at once (two a CU, one of f32 rows or 256 dims); 0 where
// the row tiles are many times as many and need no shares.
uint32_t chunk_shares(const AttnBlocksArgs &a) {
    const uint32_t held = a.dtype == 8 || a.D > 128 ? 256 : 512;
    return uint64_t(chunk_places(a)) * a.Hkv >= uint64_t(kManyRounds) * held ? 0 : held;
}

template <class E, int DP>
void launch_chunk(const Chunk &k, hipStream_t stream) {
    const uint32_t grid = k.places * k.a.Hkv;
    chunk_tile_kernel<E, DP><<<grid, 256, 0, stream>>>(k);
    if (k.shares == 0) return;
    chunk_shares_kernel<E, DP><<<k.shares, 256, 0, stream>>>(k);
    const uint32_t joins = grid * (DP / 8) <= 1024 ? DP / 8 : grid >= 256 ? 4 : 1024 / grid;
    join_kernel<E, DP><<<grid * joins, 256, 0, stream>>>(k, joins);
}
template <class E>
void launch_chunk(const Chunk &k, hipStream_t stream) {
    if (k.a.D <= 64) launch_chunk<E, 64>(k, stream);
    else if (k.a.D <= 128) launch_chunk<E, 128>(k, stream);
    else launch_chunk<E, 256>(k, stream);
}
template <class E>
void launch_few(const Blocks &k, hipStream_t stream) {
    if (k.a.D <= 64) launch_few<E, 64>(k, stream);
    else if (k.a.D <= 128) launch_few<E, 128>(k, stream);
    else launch_few<E, 256>(k, stream);
}

// ---------------------------------------------------------- general form ----
// One wavefront a token and head, any head_dim, block and alignment: for what the matrix
// forms do not take (32 sequences of up to 32768 keys, one token each: 18.7 ms, 0.11 on
// those).
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

size_t attn_blocks_scratch_bytes(const AttnBlocksArgs &a) {
    if (!matrix_applies(a)) return 0;
    if (!few_rows(a)) {
        const uint64_t s = chunk_shares(a);
        return s == 0 ? 0 : (uint64_t(chunk_places(a)) * a.Hkv + s) * kRows * (padded(a.D) + 2) * 4;
    }
    if (few_direct(a)) return 0;
    return (uint64_t(few_places(a)) * a.Hkv + kShares) * kUnit * (padded(a.D) + 2) * 4;
}

uint64_t attn_blocks_threads(const AttnBlocksArgs &a) {
    if (!matrix_applies(a)) return (uint64_t(a.pb.tokens) * a.H + 3) / 4 * 256;
    return uint64_t(few_rows(a) ? few_places(a) : chunk_places(a)) * a.Hkv * 256;
}

hipError_t launch_attn_blocks(const AttnBlocksArgs &a, void *scratch, hipStream_t stream) {
    const float mul = kLog2e / a.score_scale;
    if (matrix_applies(a) && !few_rows(a)) {
        Chunk k;
        k.a = a, k.mul = mul, k.places = chunk_places(a), k.shares = chunk_shares(a);
        k.part = static_cast<float *>(scratch), k.shift = uint32_t(__builtin_ctz(a.block));
        if (a.dtype == 7) launch_chunk<Bf16>(k, stream);
        else if (a.dtype == 6) launch_chunk<F16>(k, stream);
        else launch_chunk<F32>(k, stream);
        return hipGetLastError();
    }
    if (matrix_applies(a)) {
        Blocks k;
        k.a = a, k.mul = mul, k.places = few_places(a), k.part = static_cast<float *>(scratch);
        k.shift = uint32_t(__builtin_ctz(a.block));
        if (a.dtype == 7) launch_few<Bf16>(k, stream);
        else if (a.dtype == 6) launch_few<F16>(k, stream);
        else launch_few<F32>(k, stream);
        return hipGetLastError();
    }
    if (a.dtype == 7) launch_rows<Bf16>(a, mul, stream);
    else if (a.dtype == 6) launch_rows<F16>(a, mul, stream);
    else launch_rows<F32>(a, mul, stream);
    return hipGetLastError();
}

}  // namespace holo
