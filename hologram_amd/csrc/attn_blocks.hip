// attn_blocks.hip — attention of a packed batch's rows over the int8 cache with
// one scale a block of rows (AttentionI8Blocks, 128).
#include <hip/hip_runtime.h>

#include <math.h>

#include <type_traits>

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
// buckets up to kDirect rows, where a share of a unit would not fill a wavefront's
// pipeline. Balanced: all units' 128-key quads laid end to end and cut into equal
// shares, one for each of the workgroups that the GPU holds at once, whatever the
// lengths; a unit that is cut leaves partials, which merge_kernel joins in order (a
// launch of its own: partials pass between XCDs' L2s at its boundary).
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr uint32_t kUnit = 16, kStep = 32, kQuad = 128, kOob = 1u << 30;   // past every plane, twice it too
constexpr uint32_t kDirect = 2048, kShares = 512, kMinQuads = 2;
constexpr int kVeMin = -100;   // 2^ve's floor keeps 2^-ve finite

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
            const float f = ldexpf(vs_h[h], 7 - ve);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = __builtin_amdgcn_exp2f(s[4 * h + i] - ref);
                st.l += p;
                w[4 * h + i] = s[4 * h + i] == -INFINITY ? 0.0f : p * f;
                hi[4 * h + i] = _Float16(w[4 * h + i]);
                if constexpr (kF32) lo[4 * h + i] = _Float16(w[4 * h + i] - float(hi[4 * h + i]));
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

// Direct: grid places * Hkv. (Past 128 dims four wavefronts, whose registers hold a
// block and its successor.)
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

struct Line {
    uint64_t total;      // quads of all units of all kv heads
    uint64_t at;         // where sequence b's begin
    uint32_t b;
};
// Where the sequence that holds quad `want(total)` of the line begins: 256 threads sum
// a run of sequences each, the run that holds it is walked. A sequence's quads come
// unit by unit, kv head by kv head.
template <class F>
__device__ __forceinline__ Line find_line(const AttnBlocksArgs &a, F want, uint64_t *sums, Line *found) {
    const uint32_t tid = threadIdx.x, per = (a.pb.batch + 255) / 256;
    const uint32_t b0 = tid * per, b1 = b0 + per < a.pb.batch ? b0 + per : a.pb.batch;
    uint64_t sum = 0;
    uint32_t u, q;
    for (uint32_t b = b0; b < b1; ++b) {
        sequence_quads(a, b, &u, &q);
        sum += uint64_t(u) * q * a.Hkv;
    }
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
            sequence_quads(a, b, &u, &q);
            const uint64_t all = uint64_t(u) * q * a.Hkv;
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
    const Line ln = find_line(a, [&](uint64_t total) { return blockIdx.x * share_of(total); }, sums, &found);
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
    const int64_t len = a.lens[at.b];
    for (uint32_t i = threadIdx.x; i < rows * a.D; i += 256) {
        const uint32_t c = i / a.D, d = i - c * a.D;
        const float *p = src + c * (DP + 2);
        float M = -INFINITY;
        for (uint32_t w = 0; w < np; ++w) M = fmaxf(M, p[w * (kUnit * (DP + 2)) + DP]);
        const float ref = M == -INFINITY ? 0.0f : M;
        float o = 0.0f, l = 0.0f;
        for (uint32_t w = 0; w < np; ++w) {
            const float *x = p + w * (kUnit * (DP + 2));
            const float e = __builtin_amdgcn_exp2f(x[DP] - ref);
            o = fmaf(x[d], e, o);
            l = fmaf(x[DP + 1], e, l);
        }
        const uint32_t rr = at.unit * kUnit + c, t = rr / G;
        const bool none = visible_keys(len, n, t, a.bucket) == 0;
        static_cast<T *>(a.out)[(uint64_t(at.lo + t) * a.H + kh * G + (rr - t * G)) * a.D + d] =
            E::narrow(none ? 0.0f : o / l);
    }
}

// What the matrix forms take: 16-byte rows of q and the caches, whole 16-key steps in
// a block.
bool matrix_applies(const AttnBlocksArgs &a) {
    auto at16 = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    const uint32_t es = a.dtype == 8 ? 4 : 2;
    return a.D % 16 == 0 && a.D <= 256 && a.block >= 16 && (a.block & (a.block - 1)) == 0 && at16(a.kq) &&
           at16(a.vq) && at16(a.q) && uint64_t(a.q_stride) * es % 16 == 0;
}
uint32_t few_places(const AttnBlocksArgs &a) {
    return uint32_t(uint64_t(a.pb.tokens) * (a.H / a.Hkv) / kUnit) + a.pb.batch;
}
uint32_t padded(uint32_t D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }
// At most 16 packed rows a sequence on average.
bool few_rows(const AttnBlocksArgs &a) {
    return uint64_t(a.pb.tokens) * (a.H / a.Hkv) <= uint64_t(kUnit) * a.pb.batch;
}

template <class E, int DP>
void launch_few(const Blocks &k, hipStream_t stream) {
    const uint32_t grid = k.places * k.a.Hkv;
    if (k.a.bucket <= kDirect) {
        constexpr int W = DP > 128 ? 4 : 8;
        few_direct_kernel<E, DP, W><<<grid, 64 * W, 0, stream>>>(k);
        return;
    }
    few_shares_kernel<E, DP><<<kShares, 256, 0, stream>>>(k);
    merge_kernel<E, DP><<<grid, 256, 0, stream>>>(k);
}
template <class E>
void launch_few(const Blocks &k, hipStream_t stream) {
    if (k.a.D <= 64) launch_few<E, 64>(k, stream);
    else if (k.a.D <= 128) launch_few<E, 128>(k, stream);
    else launch_few<E, 256>(k, stream);
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

size_t attn_blocks_scratch_bytes(const AttnBlocksArgs &a) {
    if (!matrix_applies(a)) return 0;
    if (a.bucket <= kDirect) return 0;
    return (uint64_t(few_places(a)) * a.Hkv + kShares) * kUnit * (padded(a.D) + 2) * 4;
}

hipError_t launch_attn_blocks(const AttnBlocksArgs &a, void *scratch, hipStream_t stream) {
    const float mul = kLog2e / a.score_scale;
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
