// kv_select.hip — the bounds of a cache's blocks (KvBlockBounds, 131) and the blocks
// that each row attends to, chosen by them (KvBlockSelect, 132).
#include <hip/hip_runtime.h>

#include "holo_kernels.h"
#include "packed_batch.h"

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

// A row's place: its sequence and the blocks that it sees; false outside every sequence.
struct RowAt {
    uint32_t b, seen;
};
__device__ __forceinline__ bool row_at(const KvSelectArgs &a, uint32_t tok, RowAt *o) {
    const uint32_t b = last_at_most(a.pb.batch, tok, [&](uint32_t s) { return start_of(a.pb, s); });
    const uint32_t lo = start_of(a.pb, b), hi = start_of(a.pb, b + 1);
    if (tok < lo || tok >= hi) return false;
    const uint32_t v = visible_keys(a.lens[b], hi - lo, tok - lo, a.bucket);
    o->b = b;
    o->seen = v / a.block + (v % a.block != 0);
    return true;
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
    if (!row_at(a, tok, &at) || at.seen <= a.top) return;
    const uint32_t j = blockIdx.y * kThreads + tid;
    if (blockIdx.y * kThreads >= at.seen - a.last) return;
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
    if (j >= at.seen - a.last) return;
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

// The pick: a workgroup a row and kv head. The `want` largest keys of n are those above
// a border that is found eight bits at a time from the top by counting, which ends as
// soon as what shares the border's bits is wanted whole; keys that are equal to the last
// bit go by their order.
template <int kHold>
__global__ __launch_bounds__(kThreads) void pick_kernel(Select k) {
    constexpr uint32_t kWaves = kThreads / 64;
    __shared__ uint32_t bins[256], waves[kWaves], picked[3], above_of[kWaves], ties_of[kWaves];
    const KvSelectArgs &a = k.a;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const uint32_t tok = k.row0 + blockIdx.x / a.Hkv, kh = blockIdx.x % a.Hkv;
    RowAt at;
    if (!row_at(a, tok, &at)) return;
    int32_t *out = a.out + (uint64_t(tok) * a.Hkv + kh) * a.top;
    if (at.seen <= a.top) {
        for (uint32_t i = tid; i < a.top; i += kThreads) out[i] = i < at.seen ? int32_t(i) : -1;
        return;
    }
    const uint32_t end = at.seen - a.last, n = end - a.first, want = a.top - a.first - a.last;
    for (uint32_t i = tid; i < a.first; i += kThreads) out[i] = int32_t(i);
    for (uint32_t i = tid; i < a.last; i += kThreads) out[a.top - a.last + i] = int32_t(end + i);
    if (want == 0) return;
    const int32_t *sums = k.sums + (uint64_t(tok - k.row0) * a.Hkv + kh) * k.nb + a.first;
    const float *ks = a.ks + (uint64_t(at.b) * a.Hkv + kh) * k.nb + a.first;
    // in the order of the scores: NaN as infinity, -0 as 0
    auto key_at = [&](uint32_t i) {
        double v = double(sums[i]) * double(ks[i]);
        if (v != v) v = INFINITY;
        const uint64_t u = uint64_t(__double_as_longlong(v + 0.0));
        return u >> 63 ? ~u : u | (1ull << 63);
    };
    uint64_t held[kHold ? kHold : 1];
    if constexpr (kHold != 0) {
#pragma unroll
        for (int q = 0; q < kHold; ++q) held[q] = tid + q * kThreads < n ? key_at(tid + q * kThreads) : 0;
    }
    auto each = [&](auto f) {
        if constexpr (kHold != 0) {
#pragma unroll
            for (int q = 0; q < kHold; ++q) f(tid + q * kThreads < n, held[q]);
        } else {
            for (uint32_t i0 = 0; i0 < n; i0 += kThreads) f(i0 + tid < n, i0 + tid < n ? key_at(i0 + tid) : 0);
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

uint32_t blocks_of(const KvSelectArgs &a) { return uint32_t((uint64_t(a.bucket) + a.block - 1) / a.block); }
// Rows a pass of the two launches, for sums of at most 256 MB (one row's, where those are
// more).
constexpr uint64_t kMaxSums = 1ull << 26;
uint32_t rows_a_pass(const KvSelectArgs &a) {
    const uint64_t one = uint64_t(a.Hkv) * blocks_of(a), rows = one >= kMaxSums ? 1 : kMaxSums / one;
    return uint32_t(rows < a.pb.tokens ? rows : a.pb.tokens);
}

template <class E>
void launch_sums(const Select &k, hipStream_t stream) {
    const dim3 grid((k.row1 - k.row0) * k.a.Hkv, (k.nb + kThreads - 1) / kThreads);
    sums_kernel<E><<<grid, kThreads, 0, stream>>>(k);
}

void launch_pick(const Select &k, hipStream_t stream) {
    const uint32_t grid = (k.row1 - k.row0) * k.a.Hkv;
    if (k.nb <= 2 * kThreads) pick_kernel<2><<<grid, kThreads, 0, stream>>>(k);
    else if (k.nb <= 8 * kThreads) pick_kernel<8><<<grid, kThreads, 0, stream>>>(k);
    else pick_kernel<0><<<grid, kThreads, 0, stream>>>(k);
}

}  // namespace

uint64_t kv_bounds_threads(const KvBoundsArgs &a) { return uint64_t(bounds_places(a)) * kThreads; }

hipError_t launch_kv_bounds(const KvBoundsArgs &a, hipStream_t stream) {
    bounds_kernel<<<bounds_places(a), kThreads, 0, stream>>>(a);
    return hipGetLastError();
}

size_t kv_select_scratch_bytes(const KvSelectArgs &a) {
    return size_t(rows_a_pass(a)) * a.Hkv * blocks_of(a) * 4;
}

uint64_t kv_select_threads(const KvSelectArgs &a) {
    return uint64_t(rows_a_pass(a)) * a.Hkv * ((blocks_of(a) + kThreads - 1) / kThreads) * kThreads;
}

hipError_t launch_kv_select(const KvSelectArgs &a, void *scratch, hipStream_t stream) {
    Select k;
    k.a = a, k.sums = static_cast<int32_t *>(scratch), k.nb = blocks_of(a);
    const uint32_t step = rows_a_pass(a);
    for (uint32_t r = 0; r < a.pb.tokens; r += step) {
        k.row0 = r, k.row1 = a.pb.tokens - r < step ? a.pb.tokens : r + step;
        if (k.nb > a.top) {
            if (a.dtype == 7) launch_sums<Bf16>(k, stream);
            else if (a.dtype == 6) launch_sums<F16>(k, stream);
            else launch_sums<F32>(k, stream);
        }
        launch_pick(k, stream);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace holo
