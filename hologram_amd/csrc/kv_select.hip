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
struct Touched {
    const int8_t *src;       // its rows
    int8_t *dst;
    uint32_t rows;
};
__device__ __forceinline__ bool touched_block(const KvBoundsArgs &a, Touched *o) {
    const uint32_t kh = blockIdx.x % a.Hkv, place = blockIdx.x / a.Hkv;
    if (blockIdx.x == 0) check_starts(a.pb);
    const auto place_at = [&](uint32_t v, uint32_t s) { return uint64_t(v / a.block) + 2ull * s; };
    const RowAt at = sequence_at(a.pb, a.pos, place, place_at);
    const uint64_t begin = place_at(at.lo, at.b);
    if (at.hi <= at.lo || place < begin) return false;
    const uint64_t pos = at.of, past = pos + (at.hi - at.lo), end = past < a.bucket ? past : a.bucket;
    const uint64_t j = uint64_t(at.of / a.block) + (place - begin), first = j * a.block;
    if (pos >= end || first >= end) return false;
    const uint64_t plane = uint64_t(at.b) * a.Hkv + kh, nb = (uint64_t(a.bucket) + a.block - 1) / a.block;
    o->rows = uint32_t(first + a.block < end ? a.block : end - first);
    o->src = a.cache + (plane * a.bucket + first) * a.D;
    o->dst = a.bounds + (plane * nb + j) * 2 * a.D;
    return true;
}

// General form: an element a thread.
__global__ __launch_bounds__(kThreads) void bounds_any_kernel(KvBoundsArgs a) {
    __shared__ int lo_of[kPackedMaxDim], hi_of[kPackedMaxDim];
    const uint32_t tid = threadIdx.x;
    Touched t;
    if (!touched_block(a, &t)) return;
    for (uint32_t d = tid; d < a.D; d += kThreads) lo_of[d] = 127, hi_of[d] = -128;
    __syncthreads();
    for (uint32_t i = tid; i < t.rows * a.D; i += kThreads) {
        const int v = t.src[i];
        atomicMin(&lo_of[i % a.D], v);
        atomicMax(&hi_of[i % a.D], v);
    }
    __syncthreads();
    for (uint32_t d = tid; d < a.D; d += kThreads) t.dst[d] = int8_t(lo_of[d]), t.dst[a.D + d] = int8_t(hi_of[d]);
}

// Wide form: sixteen bytes a thread and row, so many rows at once as 256 threads hold. A
// byte's order is that of the 16-bit number whose upper half it is: two minima an
// instruction. The threads' bounds then meet in LDS, P threads a word of the result.
// Bound by a workgroup's chain (search, rows, LDS, store): behind one row of 32 sequences,
// 8 heads of 128 dims, 4.0 us; behind 16 prompts of 100 to 8000 rows in blocks of 64, 28 MB,
// 13.2 (the general form: 6.5 and 28; four rows a turn, two of them the first again in blocks
// of 64, 14.5).
constexpr uint32_t kBoundsDim = 256;
typedef short i16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t bytes_min(uint32_t x, uint32_t y) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(i16x2, x), __builtin_bit_cast(i16x2, y)));
}
__device__ __forceinline__ uint32_t bytes_max(uint32_t x, uint32_t y) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(i16x2, x), __builtin_bit_cast(i16x2, y)));
}
// Of four bytes the even and the odd ones as upper halves, and back.
__device__ __forceinline__ uint32_t even_of(uint32_t w) { return (w << 8) & 0xff00ff00u; }
__device__ __forceinline__ uint32_t odd_of(uint32_t w) { return w & 0xff00ff00u; }
__device__ __forceinline__ uint32_t joined(uint32_t even, uint32_t odd) { return (even >> 8 & 0x00ff00ffu) | (odd & 0xff00ff00u); }

template <int P>
__global__ __launch_bounds__(kThreads) void bounds_kernel(KvBoundsArgs a) {
    __shared__ __align__(16) uint32_t part[2][kThreads][4];      // smallest and largest, by thread
    const uint32_t tid = threadIdx.x, per = a.D / 16, groups = kThreads / per, c = tid % per, g = tid / per;
    Touched t;
    if (!touched_block(a, &t)) return;
    uint32_t lo[2][4], hi[2][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) lo[0][i] = lo[1][i] = 0x7f007f00u, hi[0][i] = hi[1][i] = 0x80008000u;
    if (g < groups) {
        const uint4 *row = reinterpret_cast<const uint4 *>(t.src) + c;
        for (uint32_t r = g; r < t.rows; r += 2 * groups) {
            uint4 v[2];
#pragma unroll
            for (uint32_t q = 0; q < 2; ++q)      // (a row past the block: the first one again)
                v[q] = row[uint64_t(r + q * groups < t.rows ? r + q * groups : r) * per];
#pragma unroll
            for (uint32_t q = 0; q < 2; ++q) {
                const uint32_t w[4] = {v[q].x, v[q].y, v[q].z, v[q].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t e = even_of(w[i]), o = odd_of(w[i]);
                    lo[0][i] = bytes_min(lo[0][i], e), lo[1][i] = bytes_min(lo[1][i], o);
                    hi[0][i] = bytes_max(hi[0][i], e), hi[1][i] = bytes_max(hi[1][i], o);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) part[0][tid][i] = joined(lo[0][i], lo[1][i]), part[1][tid][i] = joined(hi[0][i], hi[1][i]);
    }
    __syncthreads();
    const uint32_t o = tid / P, p = tid % P, words = a.D / 4;
    if (o >= 2 * words) return;
    const bool large = o >= words;
    const uint32_t word = large ? o - words : o, *from = &part[large][word / 4][word % 4];
    uint32_t e = large ? 0x80008000u : 0x7f007f00u, d = e;
    const uint32_t used = groups < t.rows ? groups : t.rows;
    for (uint32_t i = p; i < used; i += P) {
        const uint32_t w = from[i * per * 4];
        e = large ? bytes_max(e, even_of(w)) : bytes_min(e, even_of(w));
        d = large ? bytes_max(d, odd_of(w)) : bytes_min(d, odd_of(w));
    }
#pragma unroll
    for (int x = P / 2; x >= 1; x >>= 1) {
        const uint32_t e2 = __shfl_xor(e, x, 64), d2 = __shfl_xor(d, x, 64);
        e = large ? bytes_max(e, e2) : bytes_min(e, e2);
        d = large ? bytes_max(d, d2) : bytes_min(d, d2);
    }
    if (p == 0) reinterpret_cast<uint32_t *>(t.dst)[o] = joined(e, d);
}

uint32_t bounds_places(const KvBoundsArgs &a) { return (a.pb.tokens / a.block + 2 * a.pb.batch) * a.Hkv; }

// ------------------------------------------------------------------ select ----
// A row's sums over dims and heads of the larger of Q lo and Q hi are whole numbers: with
// P[d] the sum over the kv head's heads of Q's positive parts and N[d] of its negative
// ones, P . hi + N . lo (a negative scale: P . lo + N . hi), one product for all heads. The
// pick takes the scores, sum times scale, exactly. Up to 640 blocks both are one
// launch, the sums in LDS (whole_kernel); past that two, whose first reads the bounds with
// as many workgroups as there are blocks to read (tile_sums_kernel, pick_kernel).
// Bound by latency, the bytes are few: 32 rows over 2048 to 65536 keys in blocks of 32, 8 kv
// heads of 128 dims, 40 MB of bounds, 21 us, 14 of them the sums (a workgroup's chain of search,
// rows, bounds and store; 2.8 TB/s) and 7 the pick (a barrier a turn); 8 rows over up to 2000
// keys 5.4 us; 2459 rows of four chunks over up to 30000 keys in blocks of 64, 35 us, a third
// of the cycles in vector instructions of the pick, half of them waits. The general sums, and
// a pick by eight bits at a time in LDS: 55, 9.4 and 437 us.
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

// A score as a number in its order, exact: NaN as infinity, -0 as 0. Never 0. Sums of kBits bits:
// up to 29 of them times the scale's 24 are f64's 53; past that (a group of more than 2^15
// elements) the number is made of whole ones, 9 bits of exponent (1 to 308) and the 54 behind the
// leading one of the product's 55. That took 5% longer where f64 is enough (one row over 20000
// blocks: 127 and 120 us; 32 over 6000: 130 and 123).
template <int kBits>
__device__ __forceinline__ uint64_t score_key(int32_t sum, float scale) {
    if constexpr (kBits <= 29) {
        double v = double(sum) * double(scale);
        if (v != v) v = INFINITY;
        const uint64_t u = uint64_t(__double_as_longlong(v + 0.0));
        return u >> 63 ? ~u : u | (1ull << 63);
    }
    const uint32_t u = __float_as_uint(scale), e = u >> 23 & 255u, fraction = u & 0x7fffffu;
    bool down = (sum < 0) != (u >> 31 != 0);
    uint64_t size;
    if (e == 255u) {
        size = 511ull << 54;
        down = down && fraction == 0 && sum != 0;      // (0 times infinity is NaN too)
    } else {
        const uint64_t m = uint64_t(uint32_t(sum < 0 ? -sum : sum)) * (e ? fraction | 1u << 23 : fraction);
        const uint32_t lead = m ? uint32_t(__builtin_clzll(m)) : 63u;
        size = m ? uint64_t(63u - lead + (e ? e : 1u)) << 54 | (m << lead << 1) >> 10 : 0ull;
        down = down && m != 0;
    }
    return down ? (1ull << 63) - 1 - size : 1ull << 63 | size;
}

// The lists where the plane's blocks all fit: no sums, no pick. A workgroup a row and kv head.
__global__ __launch_bounds__(kThreads) void every_block_kernel(Select k) {
    const KvSelectArgs &a = k.a;
    if (blockIdx.x == 0) check_starts(a.pb);
    const uint32_t tok = k.row0 + blockIdx.x / a.Hkv, kh = blockIdx.x % a.Hkv;
    RowAt at;
    if (!row_of(a.pb, a.lens, tok, &at)) return;
    const uint32_t seen = blocks_seen(a, at.of, at.hi - at.lo, tok - at.lo);
    int32_t *out = a.out + (uint64_t(tok) * a.Hkv + kh) * a.top;
    for (uint32_t i = threadIdx.x; i < a.top; i += kThreads) out[i] = i < seen ? int32_t(i) : -1;
}

// The pick of any number of blocks: a workgroup a row and kv head. The `want` largest keys
// of n are those above a border that is found eight bits at a time from the top by counting,
// which ends as soon as what shares the border's bits is wanted whole; keys that are equal to
// the last bit go by their order.
template <int kBits>
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
            f(i < n, i < n ? score_key<kBits>(sums[i], ks[i]) : 0);
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

// The largest over a wavefront, in every lane.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    auto row = [&](auto ctrl) {
        const uint32_t o = uint32_t(__builtin_amdgcn_update_dpp(0, int(v), decltype(ctrl)::value, 0xf, 0xf, true));
        v = o > v ? o : v;
    };
    row(std::integral_constant<int, 0xb1>{});     // lane ^ 1
    row(std::integral_constant<int, 0x4e>{});     // lane ^ 2
    row(std::integral_constant<int, 0x141>{});    // 7 - lane of eight
    row(std::integral_constant<int, 0x140>{});    // 15 - lane of sixteen
    const auto x = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = x[0] > x[1] ? x[0] : x[1];
    const auto y = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return y[0] > y[1] ? y[0] : y[1];
}

// Lanes before this one whose bit is set.
__device__ __forceinline__ uint32_t before(uint64_t m) {
    return __builtin_amdgcn_mbcnt_hi(uint32_t(m >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(m), 0u));
}

// A number in the scores' order, equal for some that are not: for sums of 24 bits the product
// in f32, one rounding, which keeps the order; else score_key's upper word.
template <int kBits>
__device__ __forceinline__ uint32_t rough_key(int32_t sum, float scale) {
    if constexpr (kBits > 24) return uint32_t(score_key<kBits>(sum, scale) >> 32);
    float v = float(sum) * scale;
    if (v != v) v = INFINITY;
    const uint32_t u = __float_as_uint(v + 0.0f);
    return u ^ (uint32_t(int32_t(u) >> 31) | 0x80000000u);
}

// The pick of at most 64 kWaves kHold blocks: kWaves wavefronts a row and kv head, kHold
// rough keys a lane in registers. The border is found by halving their range until `want` of
// them are at or above it, some ten counts of ballots for scores that lie evenly. Where that
// leaves equal rough keys at the border, those are halved by their exact ones; what is
// equal then goes by its order.
// sum(j) and scale(j) may be asked for any j below 64 kWaves kHold.
template <int kWaves, int kHold, int kBits, class Sum, class Scale>
__device__ __forceinline__ void pick_row(const KvSelectArgs &a, uint32_t seen, Sum sum, Scale scale, int32_t *out,
                                         uint64_t *shared) {
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
    uint32_t key[kHold], high = 0, low = 0;      // (low: the complement of the smallest)
#pragma unroll
    for (int q = 0; q < kHold; ++q) {
        const uint32_t j = tid + q * kAll;
        const bool in = j - a.first < n;
        const uint32_t k = rough_key<kBits>(sum(j), scale(j));
        key[q] = in ? k : 0u;                                    // (below every key)
        high = key[q] > high ? key[q] : high;
        const uint32_t down = in ? ~k : 0u;
        low = down > low ? down : low;
    }
    // what the wavefronts hold, joined: a turn's numbers in one of two rows, so that one
    // barrier a turn is enough
    uint32_t turn = 0;
    auto others = [&](uint64_t mine, auto join) __attribute__((always_inline)) {
        if constexpr (kWaves == 1) return mine;
        uint64_t *row = shared + turn * kWaves;
        turn ^= 1;
        if (lane == 0) row[wave] = mine;
        __syncthreads();
        uint64_t v = row[0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) v = join(v, row[w]);
        return uint64_t(pk_uni(uint32_t(v))) | uint64_t(pk_uni(uint32_t(v >> 32))) << 32;
    };
    const uint64_t ends = others(uint64_t(pk_uni(wave_max(low))) << 32 | pk_uni(wave_max(high)), [](uint64_t x, uint64_t y) {
        const uint32_t xl = uint32_t(x), yl = uint32_t(y), xh = uint32_t(x >> 32), yh = uint32_t(y >> 32);
        return uint64_t(xh > yh ? xh : yh) << 32 | (xl > yl ? xl : yl);
    });
    // The border of the `want` largest of `all`: at lo and above are `want` or more, at hi and
    // above fewer. Several wavefronts take three borders a turn: half the turns, each a barrier.
    constexpr int kBorders = kWaves == 1 ? 1 : 3;
    struct Border {
        uint64_t at;
        uint32_t from, above;      // keys at it and above, keys above it
    };
    auto halve = [&](auto lo, auto hi, uint32_t all, uint32_t want, auto at_least) __attribute__((always_inline)) {
        uint32_t at_lo = all, at_hi = 0;
        while (at_lo != want && hi - lo > 1) {
            const auto half = (hi - lo) / 2;
            if constexpr (kBorders == 1) {
                const auto mid = lo + half;
                uint32_t c = 0;
#pragma unroll
                for (int q = 0; q < kHold; ++q) c += uint32_t(__popcll(__ballot(at_least(q, mid))));
                const bool up = c >= want;
                lo = up ? mid : lo, at_lo = up ? c : at_lo;
                hi = up ? hi : mid, at_hi = up ? at_hi : c;
            } else {
                const auto part = (hi - lo) / 4, m0 = lo + part, m1 = lo + half, m2 = m1 + part;
                uint32_t c[3] = {0, 0, 0};
#pragma unroll
                for (int q = 0; q < kHold; ++q) {
                    c[0] += uint32_t(__popcll(__ballot(at_least(q, m0))));
                    c[1] += uint32_t(__popcll(__ballot(at_least(q, m1))));
                    c[2] += uint32_t(__popcll(__ballot(at_least(q, m2))));
                }
                const uint64_t sum = others(c[0] | uint64_t(c[1]) << 20 | uint64_t(c[2]) << 40,
                                            [](uint64_t x, uint64_t y) { return x + y; });
                const uint32_t c0 = uint32_t(sum) & 0xfffffu, c1 = uint32_t(sum >> 20) & 0xfffffu, c2 = uint32_t(sum >> 40);
                // (a count of `want` is met by the highest border that has it)
                const bool u0 = c0 >= want, u1 = c1 >= want, u2 = c2 >= want;
                hi = u2 ? hi : u1 ? m2 : u0 ? m1 : m0, at_hi = u2 ? at_hi : u1 ? c2 : u0 ? c1 : c0;
                lo = u2 ? m2 : u1 ? m1 : u0 ? m0 : lo, at_lo = u2 ? c2 : u1 ? c1 : u0 ? c0 : at_lo;
            }
        }
        return Border{lo, at_lo, at_hi};
    };
    const uint32_t least = ~uint32_t(ends >> 32), past = uint32_t(ends) + 1;
    const Border rough = halve(least, past, n, want, [&](int q, uint32_t mid) { return key[q] >= mid; });
    const uint32_t lo = uint32_t(rough.at), at_lo = rough.from, at_hi = rough.above;
    // Lanes that hold a bit of `m`, in the blocks' order: how many before this one of key q
    uint32_t seen_before = 0;
    auto place = [&](uint64_t m) __attribute__((always_inline)) {
        uint32_t at = seen_before;
        if constexpr (kWaves == 1) {
            seen_before += uint32_t(__popcll(m));
        } else {
            uint64_t *row = shared + turn * kWaves;
            turn ^= 1;
            if (lane == 0) row[wave] = uint64_t(__popcll(m));
            __syncthreads();
#pragma unroll
            for (uint32_t w = 0; w < kWaves; ++w) {
                at += w < wave ? uint32_t(row[w]) : 0u;
                seen_before += uint32_t(row[w]);
            }
        }
        return at + before(m);
    };
    int32_t *to = out + a.first;
    if (at_lo == want) {
#pragma unroll
        for (int q = 0; q < kHold; ++q) {
            const bool chosen = key[q] >= lo;
            const uint32_t at = place(__ballot(chosen));
            if (chosen) to[at] = int32_t(tid + q * kAll);
        }
        return;
    }
    uint64_t exact[kHold];
    const uint32_t need = want - at_hi;
#pragma unroll
    for (int q = 0; q < kHold; ++q) {
        const uint32_t j = tid + q * kAll;
        exact[q] = key[q] == lo ? score_key<kBits>(sum(j), scale(j)) : 0;
    }
    const Border fine = halve(uint64_t(1), ~uint64_t(0), at_lo - at_hi, need, [&](int q, uint64_t mid) { return exact[q] >= mid; });
    // of the equal ones at the last border the first `left`
    const uint64_t sure = fine.from == need ? fine.at : fine.at + 1;
    const uint32_t left = fine.from == need ? 0u : need - fine.above;
    uint32_t chosen = 0;      // a bit a held key
#pragma unroll
    for (int q = 0; q < kHold; ++q) {
        const bool more = key[q] > lo || (key[q] == lo && exact[q] >= sure), tie = key[q] == lo && exact[q] == fine.at && !more;
        const uint32_t at = place(__ballot(tie));
        chosen |= uint32_t(more || (tie && at < left)) << q;
    }
    seen_before = 0;
#pragma unroll
    for (int q = 0; q < kHold; ++q) {
        const bool in = chosen >> q & 1;
        const uint32_t at = place(__ballot(in));
        if (in) to[at] = int32_t(tid + q * kAll);
    }
}

template <int kHold, int kBits>
__global__ __launch_bounds__(256) void pick_kernel(Select k) {
    __shared__ uint64_t shared[8];
    const KvSelectArgs &a = k.a;
    const uint32_t tok = k.row0 + blockIdx.x / a.Hkv, kh = blockIdx.x % a.Hkv;
    RowAt at;
    if (!row_of(a.pb, a.lens, tok, &at)) return;
    const int32_t *sums = k.sums + (uint64_t(tok - k.row0) * a.Hkv + kh) * k.nb;
    const float *ks = a.ks + (uint64_t(at.b) * a.Hkv + kh) * k.nb;
    const auto in = [&](uint32_t j) { return j < k.nb ? j : k.nb - 1; };
    pick_row<4, kHold, kBits>(a, blocks_seen(a, at.of, at.hi - at.lo, tok - at.lo), [&](uint32_t j) { return sums[in(j)]; },
                                    [&](uint32_t j) { return ks[in(j)]; }, a.out + (uint64_t(tok) * a.Hkv + kh) * a.top, shared);
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
    if (row >= kTile) return;
    const T *q = static_cast<const T *>(a.q) + uint64_t(lo + t0 + (live ? row : 0u)) * a.q_stride + uint64_t(kh) * G * a.D + d0;
    struct Dims {
        T x[VD];
    };
    constexpr uint32_t kHeld = 4;      // heads in registers between the two, asked for at once
    auto head = [&](uint32_t h) {
        return *reinterpret_cast<const Dims *>(__builtin_assume_aligned(q + h * a.D, sizeof(Dims) < 16 ? sizeof(Dims) : 16));
    };
    Dims held[kHeld] = {};
#pragma unroll
    for (uint32_t h = 0; h < kHeld; ++h)
        if (live && h < G) held[h] = head(h);
    uint32_t top = 0;
    auto see = [&](const Dims &v) {
#pragma unroll
        for (int e = 0; e < VD; ++e) {
            const uint32_t u = __float_as_uint(E::widen(v.x[e])) & 0x7fffffffu;
            if (u < 0x7f800000u && u > top) top = u;
        }
    };
#pragma unroll
    for (uint32_t h = 0; h < kHeld; ++h) see(held[h]);
    if (live)
        for (uint32_t h = kHeld; h < G; ++h) see(head(h));
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) {
        const uint32_t u = __shfl_xor(top, o, 64);
        top = u > top ? u : top;
    }
    const float inv = top ? 1.0f / block_scale(top) : 0.0f;
    int p[VD] = {}, n[VD] = {};
    auto add = [&](const Dims &v) {
#pragma unroll
        for (int e = 0; e < VD; ++e) {
            const int x = q8(E::widen(v.x[e]), inv);
            p[e] += x > 0 ? x : 0, n[e] += x < 0 ? x : 0;
        }
    };
#pragma unroll
    for (uint32_t h = 0; h < kHeld; ++h) add(held[h]);
    if (live)
        for (uint32_t h = kHeld; h < G; ++h) add(head(h));
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

// The sums of blocks [j0, j1) of a plane for the rows in `parts`, by W wavefronts, sixteen
// blocks a step. start() asks for a wavefront's first two steps, run() calls put(row, block,
// four blocks' sums).
template <int DP, int W>
struct TileSums {
    static constexpr int NKS = DP / 64, kDepth = 2;
    static constexpr uint32_t kNext = W * kTile;
    struct Bytes {
        i32x4 lo[NKS], hi[NKS];
        float scale;
    };
    __amdgpu_buffer_rsrc_t src;
    const float *ks;
    uint32_t D, j0, j1, jt;
    Bytes ring[kDepth];

    __device__ __forceinline__ void load(uint32_t from, Bytes &x) const {
        const uint32_t lane = threadIdx.x & 63u, r = lane & 15u, g = lane >> 4;
        const uint32_t j = from + r, at = j < j1 ? j * 2 * D + 16 * g : kOob;
#pragma unroll
        for (int s = 0; s < NKS; ++s) {
            const uint32_t o = 64 * s + 16 * g < D ? at + 64 * s : kOob;
            x.lo[s] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(src, o, 0, 0));
            x.hi[s] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(src, o + D, 0, 0));
        }
        x.scale = ks[j < j1 ? j : j0];
    }
    __device__ __forceinline__ void start(const KvSelectArgs &a, uint64_t plane, uint32_t nb, uint32_t first, uint32_t end) {
        src = range(a.bounds + plane * nb * 2 * a.D, nb * 2 * a.D);
        ks = a.ks + plane * nb, D = a.D, j0 = first, j1 = end, jt = j0 + kTile * pk_uni(threadIdx.x >> 6);
#pragma unroll
        for (int i = 0; i < kDepth; ++i)
            if (jt + i * kNext < j1) load(jt + i * kNext, ring[i]);
    }
    template <class Put>
    __device__ __forceinline__ void run(const QParts<DP> &parts, Put put) {
        const uint32_t lane = threadIdx.x & 63u, r = lane & 15u, g = lane >> 4;
        i32x4 part[4][NKS];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int s = 0; s < NKS; ++s) part[i][s] = *reinterpret_cast<const i32x4 *>(&parts.b[i][r][64 * s + 16 * g]);
        auto step = [&](uint32_t from, Bytes &x) __attribute__((always_inline)) {
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
            put(r, from + 4 * g, up * 256 + down);
        };
        while (jt < j1) {
#pragma unroll
            for (int i = 0; i < kDepth; ++i) {
                if (jt >= j1) break;
                step(jt, ring[i]);
                if (jt + kDepth * kNext < j1) load(jt + kDepth * kNext, ring[i]);
                jt += kNext;
            }
        }
    }
};

// The sums alone, kRange blocks a workgroup (32 rows of up to 2048 blocks with 64, 128, 256 and
// 512: 27, 17, 14 and 15 us of them): grid places * Hkv, ranges.
constexpr uint32_t kRange = 256;
template <class E, int DP>
__global__ __launch_bounds__(256) void tile_sums_kernel(Select k) {
    __shared__ QParts<DP> parts;
    const KvSelectArgs &a = k.a;
    if (blockIdx.x == 0 && blockIdx.y == 0) check_starts(a.pb);
    Place at;
    uint32_t len;
    if (!place_of(a.pb, 1, kTile, blockIdx.x / a.Hkv, &at, a.lens, &len)) return;
    const uint32_t kh = blockIdx.x % a.Hkv, n = at.hi - at.lo, t0 = at.unit * kTile, m = n - t0 < kTile ? n - t0 : kTile;
    const uint32_t first = at.lo + t0, seen = blocks_seen(a, len, n, t0 + m - 1), j0 = blockIdx.y * kRange;
    if (first + m <= k.row0 || first >= k.row1 || seen <= a.top || j0 >= seen - a.last) return;
    const uint32_t end = seen - a.last, j1 = end - j0 < kRange ? end : j0 + kRange;
    TileSums<DP, 4> tiles;
    tiles.start(a, uint64_t(at.b) * a.Hkv + kh, k.nb, j0, j1);
    split_rows<E, DP>(a, at.lo, t0, m, kh, parts);
    __syncthreads();
    tiles.run(parts, [&](uint32_t r, uint32_t j, i32x4 v) {
        if (r >= m || first + r < k.row0 || first + r >= k.row1) return;
        int32_t *to = k.sums + (uint64_t(first + r - k.row0) * a.Hkv + kh) * k.nb + j;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (j + i < j1) to[i] = v[i];
    });
}

// Sums and pick in one launch, the sums of kRows rows in LDS, for at most kMost blocks.
constexpr uint32_t kRows = 16;
constexpr int kWaves = 8;
template <class E, int DP, int kMost, int kBits>
__global__ __launch_bounds__(64 * kWaves) void whole_kernel(Select k) {
    __shared__ QParts<DP> parts;
    __shared__ __align__(16) int32_t sums[kRows][kMost + 4];
    __shared__ float scale_of[kMost];
    const KvSelectArgs &a = k.a;
    if (blockIdx.x == 0) check_starts(a.pb);
    Place at;
    uint32_t len;
    if (!place_of(a.pb, 1, kRows, blockIdx.x / a.Hkv, &at, a.lens, &len)) return;
    const uint32_t kh = blockIdx.x % a.Hkv, n = at.hi - at.lo, t0 = at.unit * kRows, m = n - t0 < kRows ? n - t0 : kRows;
    const uint32_t seen = blocks_seen(a, len, n, t0 + m - 1);
    const uint64_t plane = uint64_t(at.b) * a.Hkv + kh;
    if (seen > a.top) {
        const uint32_t j1 = seen - a.last;
        TileSums<DP, kWaves> tiles;
        tiles.start(a, plane, k.nb, 0, j1);
        for (uint32_t j = threadIdx.x; j < j1; j += 64 * kWaves) scale_of[j] = a.ks[plane * k.nb + j];
        split_rows<E, DP>(a, at.lo, t0, m, kh, parts);
        __syncthreads();
        tiles.run(parts, [&](uint32_t r, uint32_t j, i32x4 v) {
            if (r < m && j < j1) *reinterpret_cast<i32x4 *>(&sums[r][j]) = v;
        });
        __syncthreads();
    }
    for (uint32_t t = pk_uni(threadIdx.x >> 6); t < m; t += kWaves)
        pick_row<1, kMost / 64, kBits>(a, blocks_seen(a, len, n, t0 + t), [&](uint32_t j) { return sums[t][j]; },
                                        [&](uint32_t j) { return scale_of[j]; }, a.out + (uint64_t(at.lo + t0 + t) * a.Hkv + kh) * a.top, nullptr);
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
// One launch while sixteen rows' sums and their scales fit three workgroups into a CU's LDS (two
// past 128 dims): 32 rows of up to 512 blocks 11 us and two launches 15, 2459 rows of chunks 35
// and 95.
bool whole(const KvSelectArgs &a) { return matrix_applies(a) && blocks_of(a) <= 640; }
// A list of every block takes neither sums nor their scratch.
bool every_block(const KvSelectArgs &a) { return !whole(a) && blocks_of(a) <= a.top; }
uint32_t places_of(const KvSelectArgs &a) { return a.pb.tokens / (whole(a) ? kRows : kTile) + a.pb.batch; }
// Bits of the sums, of at most 127 * 128 an element: 24, 29 or 31 (the matrix form's groups of up
// to 128 heads of 256 dims: 24 or 29).
int sum_bits(const KvSelectArgs &a) {
    const uint64_t most = uint64_t(a.H / a.Hkv) * a.D * 127 * 128;
    return most < (1u << 24) ? 24 : most < (1u << 29) ? 29 : 31;
}

template <class E, int DP, int kBits>
void launch_whole(const Select &k, hipStream_t stream) {
    const uint32_t grid = places_of(k.a) * k.a.Hkv;
    if (k.nb <= 256) whole_kernel<E, DP, 256, kBits><<<grid, 64 * kWaves, 0, stream>>>(k);
    else if (k.nb <= 512) whole_kernel<E, DP, 512, kBits><<<grid, 64 * kWaves, 0, stream>>>(k);
    else whole_kernel<E, DP, 640, kBits><<<grid, 64 * kWaves, 0, stream>>>(k);
}
template <class E, int DP>
void launch_tiles(const Select &k, hipStream_t stream) {
    if (!whole(k.a)) {
        const dim3 grid(places_of(k.a) * k.a.Hkv, (k.nb + kRange - 1) / kRange);
        tile_sums_kernel<E, DP><<<grid, 256, 0, stream>>>(k);
    } else if (sum_bits(k.a) == 24) {
        launch_whole<E, DP, 24>(k, stream);
    } else {
        launch_whole<E, DP, 29>(k, stream);
    }
}
template <class E>
void launch_sums(const Select &k, hipStream_t stream) {
    if (!matrix_applies(k.a)) {
        const dim3 grid((k.row1 - k.row0) * k.a.Hkv, (k.nb + kThreads - 1) / kThreads);
        sums_kernel<E><<<grid, kThreads, 0, stream>>>(k);
    } else if (k.a.D <= 64) {
        launch_tiles<E, 64>(k, stream);
    } else if (k.a.D <= 128) {
        launch_tiles<E, 128>(k, stream);
    } else {
        launch_tiles<E, 256>(k, stream);
    }
}

template <int kBits>
void launch_pick(const Select &k, hipStream_t stream) {
    const uint32_t units = (k.row1 - k.row0) * k.a.Hkv;
    if (k.nb <= 1024) pick_kernel<4, kBits><<<units, 256, 0, stream>>>(k);
    else if (k.nb <= 2048) pick_kernel<8, kBits><<<units, 256, 0, stream>>>(k);
    else if (k.nb <= 4096) pick_kernel<16, kBits><<<units, 256, 0, stream>>>(k);
    else pick_any_kernel<kBits><<<units, kThreads, 0, stream>>>(k);
}

}  // namespace

uint64_t kv_bounds_threads(const KvBoundsArgs &a) { return uint64_t(bounds_places(a)) * kThreads; }

hipError_t launch_kv_bounds(const KvBoundsArgs &a, hipStream_t stream) {
    const uint32_t grid = bounds_places(a);
    if (a.D > kBoundsDim || a.D % 16 != 0 || reinterpret_cast<uintptr_t>(a.cache) % 16 != 0 ||
        reinterpret_cast<uintptr_t>(a.bounds) % 4 != 0)
        bounds_any_kernel<<<grid, kThreads, 0, stream>>>(a);
    else if (a.D <= 64) bounds_kernel<8><<<grid, kThreads, 0, stream>>>(a);
    else if (a.D <= 128) bounds_kernel<4><<<grid, kThreads, 0, stream>>>(a);
    else bounds_kernel<2><<<grid, kThreads, 0, stream>>>(a);
    return hipGetLastError();
}

size_t kv_select_scratch_bytes(const KvSelectArgs &a) {
    return whole(a) || every_block(a) ? 0 : size_t(rows_a_pass(a)) * a.Hkv * blocks_of(a) * 4;
}

uint64_t kv_select_threads(const KvSelectArgs &a) {
    const uint64_t units = uint64_t(rows_a_pass(a)) * a.Hkv, tiles = uint64_t(places_of(a)) * a.Hkv;
    if (whole(a)) return tiles * 64 * kWaves;
    const uint64_t sums = (matrix_applies(a) ? tiles : units) * ((blocks_of(a) + kRange - 1) / kRange);
    return (sums > units ? sums : units) * kThreads;
}

hipError_t launch_kv_select(const KvSelectArgs &a, void *scratch, hipStream_t stream) {
    Select k;
    k.a = a, k.sums = static_cast<int32_t *>(scratch), k.nb = blocks_of(a);
    const uint32_t step = whole(a) ? a.pb.tokens : rows_a_pass(a);
    for (uint32_t r = 0; r < a.pb.tokens; r += step) {
        k.row0 = r, k.row1 = a.pb.tokens - r < step ? a.pb.tokens : r + step;
        if (every_block(a)) {
            every_block_kernel<<<(k.row1 - k.row0) * a.Hkv, kThreads, 0, stream>>>(k);
        } else {
            if (a.dtype == 7) launch_sums<Bf16>(k, stream);
            else if (a.dtype == 6) launch_sums<F16>(k, stream);
            else launch_sums<F32>(k, stream);
            if (!whole(a)) {
                const int bits = sum_bits(a);
                if (bits == 24) launch_pick<24>(k, stream);
                else if (bits == 29) launch_pick<29>(k, stream);
                else launch_pick<31>(k, stream);
            }
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace holo
