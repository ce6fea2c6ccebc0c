// attn_selected.hip — attention of a packed batch's rows over the blocks of the int8
// cache that each row's list names (AttentionI8Selected, 133).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "i8_rows.h"

namespace holo {
namespace {

// -------------------------------------------------------------- matrix form ----
// A unit is a token, a kv head and sixteen of its heads: the columns of the matrix
// instructions (i8_rows.h). Its workgroup reads the list with the blocks' scales into LDS,
// drops the tail that names nothing, and its wavefronts take the 32-key steps of the
// blocks in turn. Where the units are many and have at most eight heads, the columns are two
// groups of eight, each over every other 16 keys (group_step): half the scores a lane.
// Bound by the bytes where each row has its own: 32 rows over 2048 keys of 8 kv heads of
// 128 dims, 134 MB, 28 us or 4.8 TB/s; 128 rows 89 us, 6.0 TB/s. By vector instructions where
// rows share them: 712 rows of two chunks over 2048 keys each, 270 us, 108 M of them, two thirds
// of the SIMDs' cycles (a third turn V's bytes into f16; the 3 GB out of the L2s are 11 TB/s, less
// than a third of what those hold; one group, whose registers leave two wavefronts a SIMD: 303).
// By latency where they are few: 8 rows over 256 keys 6.0 us, 26 f32 rows of drafts over 1280
// keys 15. A wavefront a row and head (below): 1560 us, 11.5 ms, 131 us, 754 us.
constexpr uint32_t kMaxList = 512;            // entries a workgroup takes at once
constexpr uint32_t kMostParts = 8192;         // shares' results in scratch: 135 MB at 256 dims, 68 at 128
constexpr uint32_t kNone = 0x80000000u;       // past every key

struct Selected {
    AttnSelectedArgs s;
    float mul;           // log2(e) / divisor
    uint32_t shift;      // block == 1 << shift
    uint32_t tiles;      // of sixteen heads a kv head
    uint32_t shares, per;   // of a list, and its entries each
    float *part;         // [units][shares][kUnit][DP + 2]: O, then the maximum and the sum (-1: no key)
};

struct Entry {
    uint32_t key;        // the block's first, kNone for none
    float ks, vs;
};

// C column groups (1 or 2). kRounds: a share's entries kMaxList at a time.
template <class E, int DP, int W, int C, bool kOnce, bool kRounds>
__global__ __launch_bounds__(64 * W, DP > 128 ? 1 : C == 2 ? 3 : 2) void few_kernel(Selected k) {
    constexpr uint32_t kHeads = kUnit / C;
    typedef typename E::T T;
    __shared__ FewLds<E, DP, W> lds;
    __shared__ Entry list[kMaxList];
    __shared__ uint32_t last;
    const AttnBlocksArgs &a = k.s.a;
    const uint32_t tid = threadIdx.x, wave = pk_uni(tid >> 6), share = blockIdx.y;
    if (blockIdx.x == 0 && share == 0) check_starts(a.pb);
    const uint32_t kh = blockIdx.x % a.Hkv, tile = blockIdx.x / a.Hkv % k.tiles, tok = blockIdx.x / a.Hkv / k.tiles;
    RowAt at;
    if (!row_of(a.pb, a.lens, tok, &at)) return;
    const uint32_t sees = visible_keys(at.of, at.hi - at.lo, tok - at.lo, a.bucket), G = a.H / a.Hkv;
    const uint64_t plane = uint64_t(at.b) * a.Hkv + kh, nb = (uint64_t(a.bucket) + a.block - 1) >> k.shift;
    const uint32_t e0 = share * k.per, mine = k.s.top - e0 < k.per ? k.s.top - e0 : k.per;
    const int32_t *ids = k.s.blocks + (uint64_t(tok) * a.Hkv + kh) * k.s.top + e0;
    auto read_list = [&](uint32_t from) __attribute__((always_inline)) {
        if (tid == 0) last = 0;
        __syncthreads();
        const uint32_t n = mine - from < kMaxList ? mine - from : kMaxList;
        for (uint32_t i = tid; i < n; i += 64 * W) {
            const int32_t id = ids[from + i];
            const bool ok = id >= 0 && uint64_t(id) << k.shift < sees;
            const uint64_t j = plane * nb + (ok ? uint32_t(id) : 0u);
            list[i] = Entry{ok ? uint32_t(id) << k.shift : kNone, a.ks[j], a.vs[j]};
            if (ok) atomicMax(&last, i + 1);
        }
    };
    read_list(0);
    const uint32_t r = tid & 15u, h0 = kh * G + tile * kUnit, rows = G - tile * kUnit < kUnit ? G - tile * kUnit : kUnit;
    const bool live = r % kHeads < rows;
    RowQ<E, DP> q;
    q.load(static_cast<const T *>(a.q) + uint64_t(tok) * a.q_stride + uint64_t(h0 + (live ? r % kHeads : 0u)) * a.D, live, a.D, k.mul);
    // 2^deep 16-key steps a block, of one longer than what the row sees those that hold it (so
    // the steps of a list are at most 2^31)
    const uint32_t reach = sees <= 16 ? 4u : 32u - uint32_t(__builtin_clz(sees - 1));
    const uint32_t deep = (k.shift < reach ? k.shift : reach) - 4;
    uint32_t halves;
    const KvPlane<DP> kv(a.kq + plane * a.bucket * a.D, a.vq + plane * a.bucket * a.D, a.bucket, a.D);
    struct Turn {
        KvStep<DP> x;         // two 16-key steps
        uint32_t key[2];      // their first keys (C == 1), or the column's step's
        float ks, vs;         // (C == 2) the column's step's
    };
    // A 16-key step of the list: its entry, and its first key (kNone past the list)
    auto half_at = [&](uint32_t half, Entry *e) __attribute__((always_inline)) {
        *e = list[half < halves ? half >> deep : 0u];
        return half < halves && e->key != kNone ? e->key + 16 * (half & ((1u << deep) - 1)) : kNone;
    };
    auto load = [&](uint32_t turn, Turn &o) __attribute__((always_inline)) {
        Entry e;
        uint32_t so[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t key = pk_uni(half_at(2 * turn + h, &e));
            so[h] = key == kNone ? kOob : key * a.D;
            if constexpr (C == 1) o.key[h] = key, o.x.ks[h] = e.ks, o.x.vs[h] = e.vs;
        }
        kv.template load<kOnce>(so, o.x);
        if constexpr (C == 2) {
            o.key[0] = half_at(2 * turn + r / kHeads, &e);
            o.ks = e.ks, o.vs = e.vs;
        }
    };
    State<DP> st;
    st.clear();
    auto take = [&](const Turn &o) __attribute__((always_inline)) {
        if constexpr (C == 1)
            few_step<E, DP>(st, o.x, q, o.key, o.key[0] + 16 > sees || o.key[1] + 16 > sees, sees, sees);
        else
            group_step<E, DP>(st, o.x, q, o.key[0], o.ks, o.vs, sees);
    };
    bool any = false;
    for (uint32_t from = 0;;) {
        __syncthreads();
        const uint32_t count = pk_uni(last);
        any |= count != 0;
        halves = count << deep;
        const uint32_t turns = (halves + 1) / 2;
        Turn ring[2];
        if (wave < turns) load(wave, ring[0]);
        for (uint32_t i = wave; i < turns; i += 2 * W) {
            if (i + W < turns) load(i + W, ring[1]);
            take(ring[0]);
            if (i + W >= turns) break;
            if (i + 2 * W < turns) load(i + 2 * W, ring[0]);
            take(ring[1]);
        }
        if (!kRounds || (from += kMaxList) >= mine) break;
        __syncthreads();      // (no wavefront reads the list that follows before all are done with this one)
        read_list(from);
    }
    float *dst = k.part + (uint64_t(blockIdx.x) * k.shares + share) * (kUnit * (DP + 2));
    join_waves<E, DP, W, C>(st, rows, a.D, lds, [&](uint32_t c, uint32_t d, float o, float M, float l) {
        if (k.shares == 1) {
            static_cast<T *>(a.out)[(uint64_t(tok) * a.H + h0 + c) * a.D + d] = E::narrow(any ? o / l : 0.0f);
        } else {
            dst[c * (DP + 2) + d] = o;
            if (d == 0) dst[c * (DP + 2) + DP] = M, dst[c * (DP + 2) + DP + 1] = any ? l : -1.0f;
        }
    });
}

// Joins the shares of a unit.
template <class E, int DP>
__global__ __launch_bounds__(256) void merge_kernel(Selected k) {
    typedef typename E::T T;
    const AttnBlocksArgs &a = k.s.a;
    const uint32_t kh = blockIdx.x % a.Hkv, tile = blockIdx.x / a.Hkv % k.tiles, tok = blockIdx.x / a.Hkv / k.tiles;
    RowAt at;
    if (!row_of(a.pb, nullptr, tok, &at)) return;
    const uint32_t G = a.H / a.Hkv, rows = G - tile * kUnit < kUnit ? G - tile * kUnit : kUnit;
    constexpr uint32_t kStride = kUnit * (DP + 2);
    const float *src = k.part + uint64_t(blockIdx.x) * k.shares * kStride;
    const uint32_t lane = threadIdx.x & 63u;
    bool any = false;
    for (uint32_t w = lane; w < k.shares; w += 64) any |= !(src[w * kStride + DP + 1] < 0.0f);
    const bool none = __ballot(any) == 0;
    for (uint32_t c = pk_uni(threadIdx.x >> 6); c < rows; c += 4)
        join_row<E, DP>(src + c * (DP + 2), kStride, k.shares, a.D, none,
                        static_cast<T *>(a.out) + (uint64_t(tok) * a.H + kh * G + tile * kUnit + c) * a.D);
}

bool matrix_applies(const AttnSelectedArgs &s) {
    const AttnBlocksArgs &a = s.a;
    const uint32_t es = a.dtype == 8 ? 4 : 2;
    const auto at16 = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    return a.D <= 256 && a.D % 16 == 0 && a.block >= 16 && (a.block & (a.block - 1)) == 0 && at16(a.q) &&
           uint64_t(a.q_stride) * es % 16 == 0 && at16(a.kq) && at16(a.vq);
}
uint32_t padded(uint32_t D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }
uint32_t tiles_of(const AttnBlocksArgs &a) { return (a.H / a.Hkv + kUnit - 1) / kUnit; }
uint64_t units_of(const AttnBlocksArgs &a) { return uint64_t(a.pb.tokens) * a.Hkv * tiles_of(a); }
// Entries a workgroup: at most kMaxList while that makes no more than kMostParts shares in all,
// else more, kMaxList at a time, and past kMostParts / 2 units all of them (4096 rows of 8 kv
// heads with 600 blocks of 16 keys: 6.37 ms, two shares each and 545 MB of scratch 6.50; 600
// with 1024: 3.03, 3.05). But where the units leave CUs idle and the list is four rounds of
// eight wavefronts, shares for as many workgroups as there are CUs, of four 32-key steps at
// least. One row of 8 kv heads over 2048 and 16384 keys whole and in shares: 19 and 117 us
// against 11 and 17; 4 rows over 8192, 67 against 20; 16 over 2048, 24 against 21; 8 rows over
// 256, 6.0 against 8.2. Every share has an entry.
uint32_t entries_of(const AttnSelectedArgs &s) {
    const uint64_t units = units_of(s.a), steps = uint64_t(s.top) * s.a.block / kStep;
    uint64_t shares = std::min<uint64_t>((s.top + kMaxList - 1) / kMaxList, std::max<uint64_t>(kMostParts / units, 1));
    if (steps >= 32 && units < 256) shares = std::max(shares, std::min(256 / units, steps / 4));
    shares = std::min<uint64_t>(shares, s.top);
    return uint32_t((s.top + shares - 1) / shares);
}
uint32_t shares_of(const AttnSelectedArgs &s) { return (s.top + entries_of(s) - 1) / entries_of(s); }
// Eight wavefronts a workgroup, four where there are two of them a CU and more (512 and 1024
// units over 2048 keys each: 54 and 105 us with eight, 49 and 93 with four) and past 128 dims,
// whose registers hold two steps.
bool four_waves(const AttnSelectedArgs &s) { return s.a.D > 128 || units_of(s.a) >= 512; }

// One row a sequence reads its blocks once; of several, the next may read them again from
// the caches (712 rows of two chunks: 359 us past the caches, 303 through them; 64 rows of as
// many sequences 48.6 and 51.6).
bool reads_once(const AttnSelectedArgs &s) { return s.a.pb.tokens <= s.a.pb.batch; }

template <class E, int DP, int W, int C, bool kRounds>
void launch_form(const Selected &k, dim3 grid, hipStream_t stream) {
    if (reads_once(k.s)) few_kernel<E, DP, W, C, true, kRounds><<<grid, 64 * W, 0, stream>>>(k);
    else few_kernel<E, DP, W, C, false, kRounds><<<grid, 64 * W, 0, stream>>>(k);
}
template <class E, int DP>
void launch_few(const Selected &k, hipStream_t stream) {
    const dim3 grid(uint32_t(units_of(k.s.a)), k.shares);
    const bool rounds = k.per > kMaxList;
    if constexpr (DP > 128) {
        if (rounds) launch_form<E, DP, 4, 1, true>(k, grid, stream);
        else launch_form<E, DP, 4, 1, false>(k, grid, stream);
    } else {
        const bool groups = k.s.a.H / k.s.a.Hkv <= kUnit / 2;
        if (rounds && groups) launch_form<E, DP, 4, 2, true>(k, grid, stream);
        else if (rounds) launch_form<E, DP, 4, 1, true>(k, grid, stream);
        else if (four_waves(k.s) && groups) launch_form<E, DP, 4, 2, false>(k, grid, stream);
        else if (four_waves(k.s)) launch_form<E, DP, 4, 1, false>(k, grid, stream);
        else launch_form<E, DP, 8, 1, false>(k, grid, stream);
    }
    if (k.shares > 1) merge_kernel<E, DP><<<grid.x, 256, 0, stream>>>(k);
}
template <class E>
void launch_few(const Selected &k, hipStream_t stream) {
    if (k.s.a.D <= 64) launch_few<E, 64>(k, stream);
    else if (k.s.a.D <= 128) launch_few<E, 128>(k, stream);
    else launch_few<E, 256>(k, stream);
}

// -------------------------------------------------------------- general form ----
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
__global__ __launch_bounds__(256) void rows_kernel(AttnSelectedArgs s, float mul) {
    typedef typename E::T T;
    __shared__ float qs[4][64 * kDims];
    const AttnBlocksArgs &a = s.a;
    if (blockIdx.x == 0) check_starts(a.pb);
    const uint32_t wave = pk_uni(threadIdx.x >> 6), lane = threadIdx.x & 63u;
    const uint64_t item = uint64_t(blockIdx.x) * 4 + wave;
    const uint32_t tok = uint32_t(item / a.H), h = uint32_t(item % a.H);
    if (tok >= a.pb.tokens) return;
    const uint32_t b = last_at_most(a.pb.batch, tok, [&](uint32_t s) { return start_of(a.pb, s); });
    const uint32_t r0 = start_of(a.pb, b), r1 = start_of(a.pb, b + 1);
    if (tok < r0 || tok >= r1) return;
    const T *q = static_cast<const T *>(a.q) + uint64_t(tok) * a.q_stride + uint64_t(h) * a.D;
    for (uint32_t d = lane; d < a.D; d += 64) qs[wave][d] = E::widen(q[d]) * mul;
    const uint32_t kh = h / (a.H / a.Hkv), sees = visible_keys(a.lens[b], r1 - r0, tok - r0, a.bucket);
    const uint64_t plane = uint64_t(b) * a.Hkv + kh, nb = (uint64_t(a.bucket) + a.block - 1) / a.block;
    const BlockSrc src{a.kq + plane * a.bucket * a.D, a.vq + plane * a.bucket * a.D,
                       a.ks + plane * nb, a.vs + plane * nb, a.D, a.block};
    const int32_t *list = s.blocks + (uint64_t(tok) * a.Hkv + kh) * s.top;
    RowState<kDims> st;
    for (uint32_t e = 0; e < s.top; ++e) {
        const int64_t j = list[e];
        if (j < 0 || uint64_t(j) * a.block >= sees) continue;
        const uint64_t to = uint64_t(j + 1) * a.block;
        st.keys(qs[wave], a.D, uint32_t(j) * a.block, uint32_t(to < sees ? to : sees), src);
    }
    T *out = static_cast<T *>(a.out) + (uint64_t(tok) * a.H + h) * a.D;
    st.write(a.D, [&](uint32_t d, float v) { out[d] = E::narrow(v); });
}

template <class E>
void launch(const AttnSelectedArgs &s, float mul, hipStream_t stream) {
    const uint32_t grid = uint32_t(attn_selected_threads(s) / 256);
    if (s.a.D <= 128) rows_kernel<E, 2><<<grid, 256, 0, stream>>>(s, mul);
    else rows_kernel<E, kPackedMaxDim / 64><<<grid, 256, 0, stream>>>(s, mul);
}

}  // namespace

size_t attn_selected_scratch_bytes(const AttnSelectedArgs &s) {
    if (!matrix_applies(s) || shares_of(s) == 1) return 0;
    return size_t(units_of(s.a)) * shares_of(s) * kUnit * (padded(s.a.D) + 2) * 4;
}

uint64_t attn_selected_threads(const AttnSelectedArgs &s) {
    if (matrix_applies(s)) return units_of(s.a) * shares_of(s) * (four_waves(s) ? 256 : 512);
    return (uint64_t(s.a.pb.tokens) * s.a.H + 3) / 4 * 256;
}

hipError_t launch_attn_selected(const AttnSelectedArgs &s, void *scratch, hipStream_t stream) {
    const float mul = kLog2e / s.a.score_scale;
    if (matrix_applies(s)) {
        Selected k;
        k.s = s, k.mul = mul, k.shift = uint32_t(__builtin_ctz(s.a.block)), k.tiles = tiles_of(s.a);
        k.shares = shares_of(s), k.per = entries_of(s), k.part = static_cast<float *>(scratch);
        if (s.a.dtype == 7) launch_few<Bf16>(k, stream);
        else if (s.a.dtype == 6) launch_few<F16>(k, stream);
        else launch_few<F32>(k, stream);
        return hipGetLastError();
    }
    if (s.a.dtype == 7) launch<Bf16>(s, mul, stream);
    else if (s.a.dtype == 6) launch<F16>(s, mul, stream);
    else launch<F32>(s, mul, stream);
    return hipGetLastError();
}

}  // namespace holo
