// kv_select.hip — the bounds of a cache's blocks (KvBlockBounds, 131) and the blocks
// that each row attends to, chosen by them (KvBlockSelect, 132).
#include <hip/hip_runtime.h>

#include "i8_rows.h"

namespace holo {
namespace {

constexpr uint32_t kThreads = 256;

// ------------------------------------------------------------------ bounds ----
// One workgroup a touched block and head, found as KvBlockAppend finds them: sequence s
// owns the places [floor(starts[s] / block) + 2 s, floor(starts[s + 1] / block) + 2 (s +
// 1)).
__global__ __launch_bounds__(kThreads) void bounds_kernel(KvBoundsArgs a) {
    __shared__ int lo_of[kPackedMaxDim], hi_of[kPackedMaxDim];
    const uint32_t kh = blockIdx.x % a.Hkv, place = blockIdx.x / a.Hkv, tid = threadIdx.x;
    if (blockIdx.x == 0) check_starts(a.pb);
    const uint32_t b = last_at_most(a.pb.batch, place, [&](uint32_t s) {
        return uint64_t(start_of(a.pb, s) / a.block) + 2ull * s;
    });
    const uint32_t r0 = start_of(a.pb, b), r1 = start_of(a.pb, b + 1);
    if (r1 <= r0) return;
    const uint64_t at = uint64_t(r0 / a.block) + 2ull * b;
    if (place < at) return;
    const uint64_t pos = a.pos[b], end = pos + (r1 - r0) < a.bucket ? pos + (r1 - r0) : a.bucket;
    const uint64_t j = uint64_t(uint32_t(pos) / a.block) + (place - at), first = j * a.block;
    if (pos >= end || first >= end) return;
    const uint32_t rows = uint32_t(first + a.block < end ? a.block : end - first);
    const uint64_t plane = uint64_t(b) * a.Hkv + kh, nb = (uint64_t(a.bucket) + a.block - 1) / a.block;
    const int8_t *src = a.cache + (plane * a.bucket + first) * a.D;
    int8_t *dst = a.bounds + (plane * nb + j) * 2 * a.D;
    for (uint32_t d = tid; d < a.D; d += kThreads) lo_of[d] = 127, hi_of[d] = -128;
    __syncthreads();
    for (uint32_t i = tid; i < rows * a.D; i += kThreads) {
        const int v = src[i];
        atomicMin(&lo_of[i % a.D], v);
        atomicMax(&hi_of[i % a.D], v);
    }
    __syncthreads();
    for (uint32_t d = tid; d < a.D; d += kThreads) dst[d] = int8_t(lo_of[d]), dst[a.D + d] = int8_t(hi_of[d]);
}

uint32_t bounds_places(const KvBoundsArgs &a) { return (a.pb.tokens / a.block + 2 * a.pb.batch) * a.Hkv; }

// ------------------------------------------------------------------ select ----
// Two launches. The first leaves a row's sums over dims and heads of the larger of Q lo
// and Q hi, whole numbers: with P[d] the sum over the kv head's heads of Q's positive
// parts and N[d] of its negative ones, that is P . hi + N . lo (a negative scale: P . lo +
// N . hi), one product for all heads. The second takes a row's scores, sum times scale,
// exact in f64, and picks.
struct Select {
    KvSelectArgs a;
    int32_t *sums;       // [row1 - row0][Hkv][nb]
    uint32_t nb, row0, row1;
};

// The blocks that row t of a sequence's n rows sees.
__device__ __forceinline__ uint32_t blocks_seen(const KvSelectArgs &a, uint32_t len, uint32_t n, uint32_t t) {
    const uint32_t v = visible_keys(len, n, t, a.bucket);
    return v / a.block + (v % a.block != 0);
}

// Q of one element: its quotient by the group's power of two, the finite ones.
__device__ __forceinline__ int q8(float x, float inv) {
    return fabsf(x) <= 3.4028235e38f ? int(rintf(x * inv)) : 0;
}

// General form of the sums: a workgroup a row, kv head and 256 blocks, a block a thread.
template <class E>
__global__ __launch_bounds__(kThreads) void sums_kernel(Select k) {
    typedef typename E::T T;
    __shared__ int pos_of[kPackedMaxDim], neg_of[kPackedMaxDim];
    __shared__ uint32_t top[kThreads / 64];
    const KvSelectArgs &a = k.a;
    if (blockIdx.x == 0 && blockIdx.y == 0) check_starts(a.pb);
    const uint32_t tid = threadIdx.x, tok = k.row0 + blockIdx.x / a.Hkv, kh = blockIdx.x % a.Hkv, G = a.H / a.Hkv;
    RowAt at;
    if (!row_of(a.pb, a.lens, tok, &at)) return;
    const uint32_t seen = blocks_seen(a, at.of, at.hi - at.lo, tok - at.lo), j = blockIdx.y * kThreads + tid;
    if (seen <= a.top || blockIdx.y * kThreads >= seen - a.last) return;
    const T *q = static_cast<const T *>(a.q) + uint64_t(tok) * a.q_stride + uint64_t(kh) * G * a.D;
    uint32_t m = 0;
    for (uint32_t i = tid; i < G * a.D; i += kThreads) {
        const uint32_t u = __float_as_uint(E::widen(q[i])) & 0x7fffffffu;
        if (u < 0x7f800000u && u > m) m = u;
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
    const float inv = m ? 1.0f / block_scale(m) : 0.0f;
    for (uint32_t d = tid; d < a.D; d += kThreads) {
        int p = 0, n = 0;
        for (uint32_t h = 0; h < G; ++h) {
            const int v = q8(E::widen(q[h * a.D + d]), inv);
            p += v > 0 ? v : 0, n += v < 0 ? v : 0;
        }
        pos_of[d] = p, neg_of[d] = n;
    }
    __syncthreads();
    if (j >= seen - a.last) return;
    const uint64_t plane = uint64_t(at.b) * a.Hkv + kh;
    const int8_t *lo = a.bounds + (plane * k.nb + j) * 2 * a.D, *hi = lo + a.D;
    if (a.ks[plane * k.nb + j] < 0.0f) {
        const int8_t *t = lo;
        lo = hi, hi = t;
    }
    int sum = 0;
    for (uint32_t d = 0; d < a.D; ++d) sum += pos_of[d] * hi[d] + neg_of[d] * lo[d];
    k.sums[(uint64_t(tok - k.row0) * a.Hkv + kh) * k.nb + j] = sum;
}

// A score as a number in its order: NaN as infinity, -0 as 0. Never 0.
__device__ __forceinline__ uint64_t score_key(int32_t sum, float scale) {
    double v = double(sum) * double(scale);
    if (v != v) v = INFINITY;
    const uint64_t u = uint64_t(__double_as_longlong(v + 0.0));
    return u >> 63 ? ~u : u | (1ull << 63);
}

// The pick of any number of blocks: a workgroup a row and kv head. The `want` largest keys of n are those above
// a border that is found eight bits at a time from the top by counting, which ends as
// soon as what shares the border's bits is wanted whole; keys that are equal to the last
// bit go by their order.
__global__ __launch_bounds__(kThreads) void pick_any_kernel(Select k) {
    constexpr uint32_t kWaves = kThreads / 64;
    __shared__ uint32_t bins[256], waves[kWaves], picked[3], above_of[kWaves], ties_of[kWaves];
    const KvSelectArgs &a = k.a;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const uint32_t tok = k.row0 + blockIdx.x / a.Hkv, kh = blockIdx.x % a.Hkv;
    RowAt at;
    if (!row_of(a.pb, a.lens, tok, &at)) return;
    const uint32_t seen = blocks_seen(a, at.of, at.hi - at.lo, tok - at.lo);
    int32_t *out = a.out + (uint64_t(tok) * a.Hkv + kh) * a.top;
    if (seen <= a.top) {
        for (uint32_t i = tid; i < a.top; i += kThreads) out[i] = i < seen ? int32_t(i) : -1;
        return;
    }
    const uint32_t end = seen - a.last, n = end - a.first, want = a.top - a.first - a.last;
    for (uint32_t i = tid; i < a.first; i += kThreads) out[i] = int32_t(i);
    for (uint32_t i = tid; i < a.last; i += kThreads) out[a.top - a.last + i] = int32_t(end + i);
    if (want == 0) return;
    const int32_t *sums = k.sums + (uint64_t(tok - k.row0) * a.Hkv + kh) * k.nb + a.first;
    const float *ks = a.ks + (uint64_t(at.b) * a.Hkv + kh) * k.nb + a.first;
    auto each = [&](auto f) {
        for (uint32_t i0 = 0; i0 < n; i0 += kThreads) {
            const uint32_t i = i0 + tid;
            f(i < n, i < n ? score_key(sums[i], ks[i]) : 0);
        }
    };
    uint64_t border = 0, mask = 0;
    uint32_t left = want;
    for (int shift = 56; shift >= 0; shift -= 8) {
        bins[tid] = 0;
        __syncthreads();
        each([&](bool in, uint64_t key) {
            if (in && (key & mask) == border) atomicAdd(&bins[(key >> shift) & 255u], 1u);
        });
        __syncthreads();
        const uint32_t c = bins[255u - tid];
        uint32_t run = c;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t up = __shfl_up(run, o, 64);
            if (lane >= uint32_t(o)) run += up;
        }
        if (lane == 63u) waves[wave] = run;
        __syncthreads();
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) run += w < wave ? waves[w] : 0u;
        if (run >= left && run - c < left) picked[0] = 255u - tid, picked[1] = left - (run - c), picked[2] = c;
        __syncthreads();
        border |= uint64_t(picked[0]) << shift;
        mask |= 255ull << shift;
        left = picked[1];
        if (picked[2] == left) break;
    }
    // Those above the border, and of those at it the first `left` (all, but for equal keys)
    uint32_t above = 0, ties = 0, i = tid;
    each([&](bool in, uint64_t key) {
        const bool more = in && (key & mask) > border, tie = in && (key & mask) == border;
        const uint64_t m = __ballot(more), t = __ballot(tie), before = (1ull << lane) - 1;
        __syncthreads();
        if (lane == 0) above_of[wave] = __popcll(m), ties_of[wave] = __popcll(t);
        __syncthreads();
        uint32_t ab = above + __popcll(m & before), tb = ties + __popcll(t & before);
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) {
            ab += w < wave ? above_of[w] : 0u, tb += w < wave ? ties_of[w] : 0u;
            above += above_of[w], ties += ties_of[w];
        }
        if (more || (tie && tb < left)) out[a.first + ab + (tb < left ? tb : left)] = int32_t(a.first + i);
        i += kThreads;
    });
}

// The pick of at most 64 kWaves kHold blocks: kWaves wavefronts a row and kv head, a key
// kHold a lane in registers. The border is found by halving the range of the keys' upper
// words until `want` keys are at or above it (some twelve counts of ballots for scores that
// lie evenly; 64 at most, which leaves equal keys).
template <int kWaves, int kHold, class Sum>
__device__ __forceinline__ void pick_row(const KvSelectArgs &a, uint32_t seen, Sum sum, const float *ks, int32_t *out,
                                         uint32_t (*shared)[kWaves]) {
    const uint32_t lane = threadIdx.x & 63u, wave = kWaves == 1 ? 0u : pk_uni(threadIdx.x >> 6), tid = 64 * wave + lane;
    constexpr uint32_t kAll = 64 * kWaves;
    if (seen <= a.top) {
        for (uint32_t i = tid; i < a.top; i += kAll) out[i] = i < seen ? int32_t(i) : -1;
        return;
    }
    const uint32_t end = seen - a.last, n = end - a.first, want = a.top - a.first - a.last;
    for (uint32_t i = tid; i < a.first; i += kAll) out[i] = int32_t(i);
    for (uint32_t i = tid; i < a.last; i += kAll) out[a.top - a.last + i] = int32_t(end + i);
    if (want == 0) return;
    uint64_t key[kHold];
    uint32_t low = 0xffffffffu, high = 0;
#pragma unroll
    for (int q = 0; q < kHold; ++q) {
        const uint32_t i = tid + q * kAll;
        key[q] = 0;
        if (i < n) {
            key[q] = score_key(sum(a.first + i), ks[a.first + i]);
            const uint32_t u = uint32_t(key[q] >> 32);
            low = u < low ? u : low, high = u > high ? u : high;
        }
    }
    // what the wavefronts hold alike: a turn's numbers in one of two rows, so that one
    // barrier a turn is enough
    uint32_t turn = 0;
    auto others = [&](uint32_t mine, auto join) {
        if constexpr (kWaves == 1) return mine;
        uint32_t *row = shared[turn];
        turn ^= 1;
        if (lane == 0) row[wave] = mine;
        __syncthreads();
        uint32_t v = row[0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) v = join(v, row[w]);
        return pk_uni(v);
    };
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const uint32_t l = __shfl_xor(low, o, 64), h = __shfl_xor(high, o, 64);
        low = l < low ? l : low, high = h > high ? h : high;
    }
    low = others(pk_uni(low), [](uint32_t x, uint32_t y) { return x < y ? x : y; });
    high = others(pk_uni(high), [](uint32_t x, uint32_t y) { return x > y ? x : y; });
    auto count = [&](uint64_t border) {
        uint32_t c = 0;
#pragma unroll
        for (int q = 0; q < kHold; ++q) c += uint32_t(__popcll(__ballot(key[q] >= border)));
        return others(c, [](uint32_t x, uint32_t y) { return x + y; });
    };
    // at lo and above are `want` or more, at hi and above fewer
    uint64_t lo = uint64_t(low) << 32, hi = (uint64_t(high) + 1) << 32;
    uint32_t at_lo = n, at_hi = 0;
    while (at_lo != want && hi - lo > 1) {
        const uint64_t mid = lo + (hi - lo) / 2;
        const uint32_t c = count(mid);
        if (c >= want) lo = mid, at_lo = c;
        else hi = mid, at_hi = c;
    }
    // those above the border, and of those at it the first (all, but for equal keys)
    const bool exact = at_lo == want;
    const uint32_t left = exact ? 0u : want - at_hi;
    const uint64_t sure = exact ? lo : hi;
    uint32_t above = 0, ties = 0;
#pragma unroll
    for (int q = 0; q < kHold; ++q) {
        const bool more = key[q] >= sure, tie = !exact && key[q] == lo;
        const uint64_t m = __ballot(more), t = __ballot(tie), before = (1ull << lane) - 1;
        uint32_t ab = above, tb = ties;
        if constexpr (kWaves == 1) {
            above += uint32_t(__popcll(m)), ties += uint32_t(__popcll(t));
        } else {
            const uint32_t packed = uint32_t(__popcll(m)) | uint32_t(__popcll(t)) << 16;
            uint32_t *row = shared[turn];
            turn ^= 1;
            if (lane == 0) row[wave] = packed;
            __syncthreads();
#pragma unroll
            for (uint32_t w = 0; w < kWaves; ++w) {
                ab += w < wave ? row[w] & 0xffffu : 0u, tb += w < wave ? row[w] >> 16 : 0u;
                above += row[w] & 0xffffu, ties += row[w] >> 16;
            }
        }
        ab += uint32_t(__popcll(m & before)), tb += uint32_t(__popcll(t & before));
        if (more || (tie && tb < left)) out[a.first + ab + (tb < left ? tb : left)] = int32_t(a.first + tid + q * kAll);
    }
}

template <int kWaves, int kHold>
__global__ __launch_bounds__(256) void pick_kernel(Select k) {
    __shared__ uint32_t shared[2][kWaves];
    const KvSelectArgs &a = k.a;
    const uint32_t unit = kWaves == 1 ? blockIdx.x * 4 + pk_uni(threadIdx.x >> 6) : blockIdx.x;
    const uint32_t tok = k.row0 + unit / a.Hkv, kh = unit % a.Hkv;
    RowAt at;
    if (tok >= k.row1 || !row_of(a.pb, a.lens, tok, &at)) return;
    const int32_t *sums = k.sums + (uint64_t(tok - k.row0) * a.Hkv + kh) * k.nb;
    pick_row<kWaves, kHold>(a, blocks_seen(a, at.of, at.hi - at.lo, tok - at.lo), [&](uint32_t j) { return sums[j]; },
                            a.ks + (uint64_t(at.b) * a.Hkv + kh) * k.nb, a.out + (uint64_t(tok) * a.Hkv + kh) * a.top,
                            shared);
}

// ------------------------------------------------- the sums in matrix form ----
// Sixteen rows of a sequence are the columns of the matrix instructions, sixteen blocks
// the rows, whose operands are the bounds as they lie. P and N in two int8 parts each, 256 p1
// + p0 (up to 128 heads), so four products take all heads of the kv head at once:
//     S = 256 (p1 . hi + n1 . lo) + p0 . hi + n0 . lo       16x16x64 i8, exact
constexpr uint32_t kTile = 16;

template <int DP>
struct QParts {
    uint8_t b[4][kTile][DP + 16];     // p1, p0, n1, n0 of a row's dims (16 bytes on: other banks)
};

// P and N of rows [t0, t0 + m) of the sequence that begins at row `lo`: sixteen threads a
// row, DP / 16 dims each.
template <class E, int DP>
__device__ __forceinline__ void split_rows(const KvSelectArgs &a, uint32_t lo, uint32_t t0, uint32_t m, uint32_t kh,
                                           QParts<DP> &parts) {
    typedef typename E::T T;
    constexpr int VD = DP / 16;
    const uint32_t tid = threadIdx.x, row = tid >> 4, d0 = VD * (tid & 15u), G = a.H / a.Hkv;
    const bool live = row < m && d0 < a.D;
    const T *q = static_cast<const T *>(a.q) + uint64_t(lo + t0 + (live ? row : 0u)) * a.q_stride + uint64_t(kh) * G * a.D + d0;
    struct Dims {
        T x[VD];
    };
    uint32_t top = 0;
    if (live)
        for (uint32_t h = 0; h < G; ++h) {
            const Dims v = *reinterpret_cast<const Dims *>(__builtin_assume_aligned(q + h * a.D, sizeof(Dims) < 16 ? sizeof(Dims) : 16));
#pragma unroll
            for (int e = 0; e < VD; ++e) {
                const uint32_t u = __float_as_uint(E::widen(v.x[e])) & 0x7fffffffu;
                if (u < 0x7f800000u && u > top) top = u;
            }
        }
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) {
        const uint32_t u = __shfl_xor(top, o, 64);
        top = u > top ? u : top;
    }
    const float inv = top ? 1.0f / block_scale(top) : 0.0f;
    int p[VD] = {}, n[VD] = {};
    if (live)
        for (uint32_t h = 0; h < G; ++h) {
            const Dims v = *reinterpret_cast<const Dims *>(__builtin_assume_aligned(q + h * a.D, sizeof(Dims) < 16 ? sizeof(Dims) : 16));
#pragma unroll
            for (int e = 0; e < VD; ++e) {
                const int x = q8(E::widen(v.x[e]), inv);
                p[e] += x > 0 ? x : 0, n[e] += x < 0 ? x : 0;
            }
        }
#pragma unroll
    for (int w = 0; w < VD / 4; ++w) {
        uint32_t out[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int pv = p[4 * w + e], nv = n[4 * w + e], p1 = (pv + 128) >> 8, n1 = (nv + 128) >> 8;
            const int part[4] = {p1, pv - 256 * p1, n1, nv - 256 * n1};
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] |= uint32_t(part[i] & 0xff) << (8 * e);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<uint32_t *>(&parts.b[i][row][d0 + 4 * w]) = out[i];
    }
}

// The sums of blocks [j0, j1) for the rows in `parts`, by four wavefronts, sixteen blocks a
// step: put(row, block, four blocks' sums).
template <int DP, class Put>
__device__ __forceinline__ void tile_sums(const KvSelectArgs &a, uint64_t plane, uint32_t nb, uint32_t j0, uint32_t j1,
                                          const QParts<DP> &parts, Put put) {
    constexpr int NKS = DP / 64;
    const uint32_t lane = threadIdx.x & 63u, r = lane & 15u, g = lane >> 4, wave = pk_uni(threadIdx.x >> 6);
    const auto src = range(a.bounds + plane * nb * 2 * a.D, nb * 2 * a.D);
    const float *ks = a.ks + plane * nb;
    struct Bytes {
        i32x4 lo[NKS], hi[NKS];
        float scale;
    };
    auto load = [&](uint32_t jt, Bytes &x) __attribute__((always_inline)) {
        const uint32_t j = jt + r, at = j < j1 ? j * 2 * a.D + 16 * g : kOob;
#pragma unroll
        for (int s = 0; s < NKS; ++s) {
            const uint32_t o = 64 * s + 16 * g < a.D ? at + 64 * s : kOob;
            x.lo[s] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(src, o, 0, 0));
            x.hi[s] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(src, o + a.D, 0, 0));
        }
        x.scale = ks[j < j1 ? j : j0];
    };
    i32x4 part[4][NKS];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int s = 0; s < NKS; ++s) part[i][s] = *reinterpret_cast<const i32x4 *>(&parts.b[i][r][64 * s + 16 * g]);
    auto step = [&](uint32_t jt, Bytes &x) __attribute__((always_inline)) {
        if (__any(x.scale < 0.0f)) {
            const bool turn = x.scale < 0.0f;
#pragma unroll
            for (int s = 0; s < NKS; ++s) {
                const i32x4 lo = x.lo[s], hi = x.hi[s];
                x.lo[s] = turn ? hi : lo, x.hi[s] = turn ? lo : hi;
            }
        }
        i32x4 up = {0, 0, 0, 0}, down = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < NKS; ++s) {
            up = __builtin_amdgcn_mfma_i32_16x16x64_i8(x.hi[s], part[0][s], up, 0, 0, 0);
            down = __builtin_amdgcn_mfma_i32_16x16x64_i8(x.hi[s], part[1][s], down, 0, 0, 0);
            up = __builtin_amdgcn_mfma_i32_16x16x64_i8(x.lo[s], part[2][s], up, 0, 0, 0);
            down = __builtin_amdgcn_mfma_i32_16x16x64_i8(x.lo[s], part[3][s], down, 0, 0, 0);
        }
        put(r, jt + 4 * g, up * 256 + down);
    };
    Bytes ring[2];
    uint32_t jt = j0 + kTile * wave;
    if (jt < j1) load(jt, ring[0]);
    for (; jt < j1; jt += 8 * kTile) {
        load(jt + 4 * kTile, ring[1]);
        step(jt, ring[0]);
        if (jt + 4 * kTile >= j1) break;
        load(jt + 8 * kTile, ring[0]);
        step(jt + 4 * kTile, ring[1]);
    }
}

// The sums alone, kRange blocks a workgroup: grid places * Hkv, ranges.
constexpr uint32_t kRange = 256;
template <class E, int DP>
__global__ __launch_bounds__(256) void tile_sums_kernel(Select k) {
    __shared__ QParts<DP> parts;
    const KvSelectArgs &a = k.a;
    if (blockIdx.x == 0 && blockIdx.y == 0) check_starts(a.pb);
    Place at;
    if (!place_of(a.pb, 1, kTile, blockIdx.x / a.Hkv, &at)) return;
    const uint32_t kh = blockIdx.x % a.Hkv, n = at.hi - at.lo, t0 = at.unit * kTile, m = n - t0 < kTile ? n - t0 : kTile;
    const uint32_t first = at.lo + t0, seen = blocks_seen(a, a.lens[at.b], n, t0 + m - 1), j0 = blockIdx.y * kRange;
    if (first + m <= k.row0 || first >= k.row1 || seen <= a.top || j0 >= seen - a.last) return;
    const uint32_t end = seen - a.last, j1 = end - j0 < kRange ? end : j0 + kRange;
    split_rows<E, DP>(a, at.lo, t0, m, kh, parts);
    __syncthreads();
    tile_sums<DP>(a, uint64_t(at.b) * a.Hkv + kh, k.nb, j0, j1, parts, [&](uint32_t r, uint32_t j, i32x4 v) {
        if (r >= m || first + r < k.row0 || first + r >= k.row1) return;
        int32_t *to = k.sums + (uint64_t(first + r - k.row0) * a.Hkv + kh) * k.nb + j;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (j + i < j1) to[i] = v[i];
    });
}

// Sums and pick in one launch, the sums of sixteen rows in LDS: for up to kWhole blocks.
constexpr uint32_t kWhole = 640;
template <class E, int DP, int kHold>
__global__ __launch_bounds__(256) void whole_kernel(Select k) {
    __shared__ QParts<DP> parts;
    extern __shared__ __align__(16) int32_t sums[];       // [kTile][pitch]
    const KvSelectArgs &a = k.a;
    if (blockIdx.x == 0) check_starts(a.pb);
    Place at;
    if (!place_of(a.pb, 1, kTile, blockIdx.x / a.Hkv, &at)) return;
    const uint32_t kh = blockIdx.x % a.Hkv, n = at.hi - at.lo, t0 = at.unit * kTile, m = n - t0 < kTile ? n - t0 : kTile;
    const uint32_t len = a.lens[at.b], seen = blocks_seen(a, len, n, t0 + m - 1), pitch = k.nb + 4 + (4 - k.nb % 4) % 4;
    const uint64_t plane = uint64_t(at.b) * a.Hkv + kh;
    if (seen > a.top) {
        split_rows<E, DP>(a, at.lo, t0, m, kh, parts);
        __syncthreads();
        const uint32_t j1 = seen - a.last;
        tile_sums<DP>(a, plane, k.nb, 0, j1, parts, [&](uint32_t r, uint32_t j, i32x4 v) {
            if (j < j1) *reinterpret_cast<i32x4 *>(sums + r * pitch + j) = v;
        });
        __syncthreads();
    }
    for (uint32_t t = pk_uni(threadIdx.x >> 6); t < m; t += 4)
        pick_row<1, kHold>(a, blocks_seen(a, len, n, t0 + t), [&](uint32_t j) { return sums[t * pitch + j]; },
                           a.ks + plane * k.nb, a.out + (uint64_t(at.lo + t0 + t) * a.Hkv + kh) * a.top, nullptr);
}

uint32_t blocks_of(const KvSelectArgs &a) { return uint32_t((uint64_t(a.bucket) + a.block - 1) / a.block); }
// Rows a pass of the two launches, for sums of at most 256 MB (one row's, where those are
// more).
constexpr uint64_t kMaxSums = 1ull << 26;
uint32_t rows_a_pass(const KvSelectArgs &a) {
    const uint64_t one = uint64_t(a.Hkv) * blocks_of(a), rows = one >= kMaxSums ? 1 : kMaxSums / one;
    return uint32_t(rows < a.pb.tokens ? rows : a.pb.tokens);
}

bool matrix_applies(const KvSelectArgs &a) {
    const uint32_t es = a.dtype == 8 ? 4 : 2;
    return a.D <= 256 && a.D % 16 == 0 && a.H / a.Hkv <= 128 && reinterpret_cast<uintptr_t>(a.bounds) % 16 == 0 &&
           reinterpret_cast<uintptr_t>(a.q) % 16 == 0 && uint64_t(a.q_stride) * es % 16 == 0;
}
uint32_t places_of(const KvSelectArgs &a) { return a.pb.tokens / kTile + a.pb.batch; }
bool whole(const KvSelectArgs &a) { return matrix_applies(a) && blocks_of(a) <= kWhole; }

template <class E, int DP>
void launch_tiles(const Select &k, hipStream_t stream) {
    const uint32_t grid = places_of(k.a) * k.a.Hkv;
    if (!whole(k.a)) {
        if (k.nb > k.a.top) tile_sums_kernel<E, DP><<<dim3(grid, (k.nb + kRange - 1) / kRange), 256, 0, stream>>>(k);
        return;
    }
    const uint32_t pitch = k.nb + 4 + (4 - k.nb % 4) % 4, bytes = kTile * pitch * 4;
    if (k.nb <= 256) whole_kernel<E, DP, 4><<<grid, 256, bytes, stream>>>(k);
    else whole_kernel<E, DP, kWhole / 64><<<grid, 256, bytes, stream>>>(k);
}
template <class E>
void launch_sums(const Select &k, hipStream_t stream) {
    if (!matrix_applies(k.a)) {
        const dim3 grid((k.row1 - k.row0) * k.a.Hkv, (k.nb + kThreads - 1) / kThreads);
        if (k.nb > k.a.top) sums_kernel<E><<<grid, kThreads, 0, stream>>>(k);
    } else if (k.a.D <= 64) {
        launch_tiles<E, 64>(k, stream);
    } else if (k.a.D <= 128) {
        launch_tiles<E, 128>(k, stream);
    } else {
        launch_tiles<E, 256>(k, stream);
    }
}

void launch_pick(const Select &k, hipStream_t stream) {
    const uint32_t units = (k.row1 - k.row0) * k.a.Hkv;
    if (k.nb <= 2048 && units >= 2048) pick_kernel<1, 32><<<(units + 3) / 4, 256, 0, stream>>>(k);
    else if (k.nb <= 1024) pick_kernel<4, 4><<<units, 256, 0, stream>>>(k);
    else if (k.nb <= 2048) pick_kernel<4, 8><<<units, 256, 0, stream>>>(k);
    else if (k.nb <= 4096) pick_kernel<4, 16><<<units, 256, 0, stream>>>(k);
    else pick_any_kernel<<<units, kThreads, 0, stream>>>(k);
}

}  // namespace

uint64_t kv_bounds_threads(const KvBoundsArgs &a) { return uint64_t(bounds_places(a)) * kThreads; }

hipError_t launch_kv_bounds(const KvBoundsArgs &a, hipStream_t stream) {
    bounds_kernel<<<bounds_places(a), kThreads, 0, stream>>>(a);
    return hipGetLastError();
}

size_t kv_select_scratch_bytes(const KvSelectArgs &a) {
    return whole(a) ? 0 : size_t(rows_a_pass(a)) * a.Hkv * blocks_of(a) * 4;
}

uint64_t kv_select_threads(const KvSelectArgs &a) {
    const uint64_t units = uint64_t(rows_a_pass(a)) * a.Hkv, tiles = uint64_t(places_of(a)) * a.Hkv;
    if (whole(a)) return tiles * 256;
    const uint64_t sums = (matrix_applies(a) ? tiles : units) * ((blocks_of(a) + kRange - 1) / kRange);
    return (sums > units ? sums : units) * kThreads;
}

hipError_t launch_kv_select(const KvSelectArgs &a, void *scratch, hipStream_t stream) {
    Select k;
    k.a = a, k.sums = static_cast<int32_t *>(scratch), k.nb = blocks_of(a);
    const uint32_t step = whole(a) ? a.pb.tokens : rows_a_pass(a);
    for (uint32_t r = 0; r < a.pb.tokens; r += step) {
        k.row0 = r, k.row1 = a.pb.tokens - r < step ? a.pb.tokens : r + step;
        if (a.dtype == 7) launch_sums<Bf16>(k, stream);
        else if (a.dtype == 6) launch_sums<F16>(k, stream);
        else launch_sums<F32>(k, stream);
        if (!whole(a)) launch_pick(k, stream);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace holo
