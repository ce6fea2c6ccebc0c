// attn_packed.hip — causal grouped-query attention of a packed batch of prompts
// (AttentionPacked, 126).
#include <hip/hip_runtime.h>

#include <math.h>

#include <algorithm>
#include <type_traits>

#include "holo_kernels.h"
#include "packed_tile.h"

namespace holo {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// ------------------------------------------------------------ tiled form ----
// bf16 and f16 rows. A sequence's n * G query rows of a kv head (G = H / Hkv; row
// r = token r / G, head r % G) go 128 to a workgroup, 32 to a wavefront, over
// 64-key tiles of the sequence, which come by LDS DMA, K's two tiles ahead and V's one,
// into one of two buffers while the other is multiplied. Per tile and wavefront:
//     S^T[64 keys x 32 rows] = K . Q^T    32x32x16, a row is a lane column
//     causal limit, online softmax in f32 (a row's keys are in its lane and in
//                                         the lane 32 apart)
//     O^T[DP x 32 rows] += V^T . P^T      32x32x16, P rounded to the rows' type:
//                                         the product the type can take, each
//                                         weight off by half a step at most, as the
//                                         result itself is; the sum l holds them
//                                         unrounded in f32
// f16 weights are held as 2^7 p (l too, so the quotient is the same): p reaches 2^8
// at most, and down to 2^-21 it stays clear of f16's subnormals.
// A workgroup a place (place_of) and kv head. Neighbouring workgroups take the kv
// heads of one place, so that with eight of them an XCD's L2 holds one head's K and
// V; late places, which see the most keys, go first. (All tiles of all sequences in
// the order of what they see gained nothing: 24 sequences of 17 to 2000 rows 161
// against 163 us, 60 of them 355 against 331.)
// Bound by the matrix cores where sequences are long (one of 8192 rows, 32 heads on 8 of
// 128 dims, 513 us, 1.07 PFLOP/s; of 96, 80 and 64 dims 485, 467 and 306: 80 and 96 are
// multiplied as 128). Where they are short by a workgroup's start and end, 6.8 us beside
// 2.0 us a 64-key step with two workgroups a CU (batches of equal sequences of 64 to 4096
// rows fit that within 1%; below 128 rows the bytes bound too): 24 of 17 to 2000 rows 140
// us, 37 of them starts and ends, 96 steps, 9% more of these than the visible pairs fill.
// A masked key's weight is 0, and 0 times a V that is not finite is NaN: in a tile
// that some row does not see to its end such elements are staged as 0, and then
// added by the rows that see their keys (add_odd); the other rows' bits are what
// they are without them.
constexpr uint32_t kRows = 128, kKeys = 64;
template <class E>
__device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (std::is_same_v<E, Bf16>)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <class E, int DP>
__device__ __forceinline__ void packed_tile(const AttnPackedArgs &a, const float mul, const uint32_t places) {
    constexpr int RB = 2 * DP, NK = DP / 16, DB = DP / 32, LPW = RB / 64;   // LPW: 1 KiB loads a wavefront
    constexpr uint32_t CPR = RB / 16, RPL = 1024 / RB, kOob = 0x80000000u;   // chunks a row, rows a load
    constexpr float kLag = 8.0f, kUp = std::is_same_v<E, F16> ? 7.0f : 0.0f;
    typedef uint8_t Buf[kKeys * RB];
    __shared__ __attribute__((aligned(1024))) Buf kb0, kb1, vb0, vb1;
    __shared__ uint32_t odd0[4], odd1[4];   // found in vb0, vb1, by wavefront
    if (blockIdx.x == 0) check_starts(a.pb);
    const uint32_t G = a.H / a.Hkv, kh = blockIdx.x % a.Hkv;
    Place at;
    if (!place_of(a.pb, G, kRows, places - 1 - blockIdx.x / a.Hkv, &at)) return;
    const uint32_t t0 = at.lo, n = at.hi - at.lo, R = n * G, r0 = at.unit * kRows;
    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 31, lg = lane >> 5;
    const uint32_t wave = pk_uni(uint32_t(tid) >> 6);
    // token of a row, the last one's past the end
    auto token = [&](uint32_t r) { return (r < R ? r : R - 1) / G; };
    const uint32_t wr0 = r0 + 32 * wave, row = wr0 + lr < R ? wr0 + lr : R - 1;
    const uint32_t lim = row / G + 1;
    const uint32_t kmin = pk_uni(token(r0) + 1), kmax = pk_uni(token(r0 + kRows - 1) + 1);
    const uint32_t wmin = pk_uni(token(wr0) + 1);
    const bool live = pk_uni(wr0 < R);   // the wavefront has rows

    // K and V straight into LDS: a load of a wavefront fills 1 KiB, RPL rows, and lane
    // i's 16 bytes land at 16 i, so the swizzle picks the chunk that the lane reads. A
    // resource a tile: rows past the sequence, like chunks past D, read as zeros.
    typedef typename E::T T;
    const T *kp = static_cast<const T *>(a.k) + uint64_t(t0) * a.k_stride + uint64_t(kh) * a.D;
    const T *vp = static_cast<const T *>(a.v) + uint64_t(t0) * a.v_stride + uint64_t(kh) * a.D;
    uint32_t koff[LPW], voff[LPW];
#pragma unroll
    for (int t = 0; t < LPW; ++t) {
        const uint32_t r = (wave * LPW + t) * RPL + lane / CPR, c = lane % CPR;
        const uint32_t ck = c ^ swz_k<DP>(r), cv = c ^ swz_v<DP>(r);
        koff[t] = 8 * ck < a.D ? (r * a.k_stride + 8 * ck) * 2u : kOob;
        voff[t] = 8 * cv < a.D ? (r * a.v_stride + 8 * cv) * 2u : kOob;
    }
    auto load_tile = [&](const T *base, uint32_t stride, uint32_t j0, const uint32_t (&off)[LPW], uint8_t *buf) {
        const uint32_t left = j0 < n ? (n - j0 < kKeys ? n - j0 : kKeys) : 0u;
        const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(base + uint64_t(left ? j0 : 0u) * stride), 0,
                                                         left ? int(((left - 1) * stride + a.D) * 2u) : 0, 0x00020000);
#pragma unroll
        for (int t = 0; t < LPW; ++t) load_to_lds(r, buf + (wave * LPW + t) * 1024u, off[t]);
    };
    auto load_k = [&](uint32_t j0, uint8_t *buf) { load_tile(kp, a.k_stride, j0, koff, buf); };
    auto load_v = [&](uint32_t j0, uint8_t *buf) { load_tile(vp, a.v_stride, j0, voff, buf); };
    // 16-byte chunk c of row r of a wavefront's 32 rows in LDS
    auto chunk_at = [&](uint32_t r, uint32_t c) { return r * RB + (c ^ (r & (CPR - 1u) & 15u)) * 16u; };
    // Q the same way, whole rows into the wavefront's part of the two buffers that are
    // needed last; a row past R is a copy of the last
    uint8_t *qbuf = (wave & 2 ? vb1 : kb1) + (wave & 1) * (32 * RB);
    {
        const uint32_t tok0 = r0 / G;
        const auto r = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<T *>(static_cast<const T *>(a.q) + uint64_t(t0 + tok0) * a.q_stride + kh * G * a.D), 0, int(kOob),
            0x00020000);
#pragma unroll
        for (int t = 0; t < 2 * LPW; ++t) {
            const uint32_t at = t * RPL + lane / CPR, rr = wr0 + at < R ? wr0 + at : R - 1, tq = rr / G;
            const uint32_t c = (lane % CPR) ^ (at & (CPR - 1u) & 15u);
            const uint32_t off = ((tq - tok0) * a.q_stride + (rr - tq * G) * a.D + 8 * c) * 2u;
            load_to_lds(r, qbuf + 1024 * t, 8 * c < a.D ? off : kOob);
        }
    }
    load_k(0, kb0);
    load_v(0, vb0);

    // (one of) a pair of f16 or bf16 with all exponent bits set
    constexpr uint32_t kExp = std::is_same_v<E, Bf16> ? 0x7f80u : 0x7c00u;
    auto odd = [](uint32_t w) { return (w & kExp) == kExp || ((w >> 16) & kExp) == kExp; };
    // V of a tile that some row does not see to its end: elements that are not finite
    // become zeros; whether there were any is *flag's.
    auto screen = [&](uint8_t *buf, uint32_t *flag) {
        constexpr int kMine = kKeys * RB / 4096;
        u32x4 x[kMine];
        bool any = false;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            x[i] = *reinterpret_cast<u32x4 *>(buf + tid * 16u + 4096u * i);
            any |= odd(x[i][0]) || odd(x[i][1]) || odd(x[i][2]) || odd(x[i][3]);
        }
        if (any)
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    x[i][w] = (x[i][w] & kExp) == kExp ? x[i][w] & 0xffff0000u : x[i][w];
                    x[i][w] = ((x[i][w] >> 16) & kExp) == kExp ? x[i][w] & 0xffffu : x[i][w];
                }
                *reinterpret_cast<u32x4 *>(buf + tid * 16u + 4096u * i) = x[i];
            }
        const bool found = __ballot(any) != 0;
        if (lane == 0) flag[wave] = found;
    };

    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    const uint32_t kat = k_place<DP>(lane), vat = v_place<DP>(lane);

    // The elements that `screen` left out, for the rows that see their keys: an infinity
    // or NaN with a weight above 0 is the sum it joins.
    auto add_odd = [&](uint32_t j0) __attribute__((always_inline)) {
#pragma unroll 1
        for (uint32_t j = j0; j < j0 + kKeys && j < n; ++j)
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const uint32_t dim = 32u * d + 8u * c + 4u * lg;
                    if (j >= lim || dim >= a.D) continue;
                    const uint2 v = *reinterpret_cast<const uint2 *>(vp + uint64_t(j) * a.v_stride + dim);
                    const uint16_t x[4] = {uint16_t(v.x), uint16_t(v.x >> 16), uint16_t(v.y), uint16_t(v.y >> 16)};
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (odd(x[e])) o[d][4 * c + e] += E::widen(x[e]);
                }
    };

    f32x16 s[2];
    u32x4 qf[NK];
    auto limit = [&](uint32_t j0) __attribute__((always_inline)) {   // keys the row does not see
        if (j0 + kKeys <= wmin) return;
        int sees = int(lim) - int(j0) - 4 * lg;
        asm volatile("" : "+v"(sees));   // a branch of its own: full tiles pass it by
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[h][r] = 32 * h + 8 * (r >> 2) + (r & 3) < sees ? s[h][r] : -INFINITY;
    };
    // m is a row's largest score up to kLag: a weight may reach 2^kLag, and the sums
    // are rescaled only where a row passes that
    auto rescale = [&](float mt) __attribute__((always_inline)) {
        if (__any(mt > m + kLag)) {
            const float mn = mt > m + kLag ? mt : m;   // (the other rows' bits stay as they are)
            const float al = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            l *= al;
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] *= al;
            m = mn;
        }
    };
    auto add_found = [&](const uint32_t *flag, uint32_t j0) __attribute__((always_inline)) {
        if (j0 + kKeys > kmin && __builtin_expect(flag[0] | flag[1] | flag[2] | flag[3], 0)) add_odd(j0);
    };
    // S = K . Q^T of a tile into `to`, beside the weights of the tile in s (kWeigh): a
    // product takes the matrix cores 32 cycles, the weights' vector instructions run
    // under it. The operands are read two steps ahead, and the barriers keep the
    // compiler from gathering the products behind the rest.
    u32x4 pf[4];
    auto weight_pair = [&](int i, float ref) __attribute__((always_inline)) {
        float p[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            p[e] = __builtin_amdgcn_exp2f(fmaf(s[i >> 3][2 * (i & 7) + e], mul, -ref));
            l += p[e];
        }
        uint32_t w = pack2<E>(p[0], p[1]);
        asm volatile("" : "+v"(w), "+v"(l));   // here, not where they are used
        pf[i >> 2][i & 3] = w;
    };
    auto reference = [&]() { return (m == -INFINITY ? 0.0f : m) - kUp; };
    auto scores = [&](const uint8_t *buf, f32x16 (&to)[2], const bool weigh) __attribute__((always_inline)) {
        constexpr int kPairs = 16 / NK;
        uint32_t at = kat;
        asm volatile("" : "+v"(at));   // one register, not one a step
        u32x4 kf[2][2];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int h = 0; h < 2; ++h) kf[k][h] = k_frag<DP>(buf, at, k, h);
        const float ref = reference();
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 16; ++r) to[h][r] = 0.0f;
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int h = 0; h < 2; ++h) to[h] = mfma<E>(kf[k & 1][h], qf[k], to[h]);
            if (k + 2 < NK)
#pragma unroll
                for (int h = 0; h < 2; ++h) kf[k & 1][h] = k_frag<DP>(buf, at, k + 2, h);
            if (weigh)
#pragma unroll
                for (int i = kPairs * k; i < kPairs * (k + 1); ++i) weight_pair(i, ref);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    // O^T += V^T . P^T, beside the largest of the scores in s
    auto products = [&](const uint8_t *buf) __attribute__((always_inline)) {
        constexpr int kSteps = 2 * DB, kMax = 32 / kSteps;
        uint32_t at = vat;
        asm volatile("" : "+v"(at));
        u32x4 vf[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) vf[i][h] = v_frag<DP>(buf, at, i / (DB / 2), 2 * (i % (DB / 2)) + h);
        float mt = -INFINITY;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            const int st = i / (DB / 2), d = 2 * (i % (DB / 2));
#pragma unroll
            for (int h = 0; h < 2; ++h) o[d + h] = mfma<E>(vf[i & 1][h], pf[st], o[d + h]);
            if (i + 2 < kSteps)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    vf[i & 1][h] = v_frag<DP>(buf, at, (i + 2) / (DB / 2), 2 * ((i + 2) % (DB / 2)) + h);
#pragma unroll
            for (int r = kMax * i; r < kMax * (i + 1); ++r) mt = fmaxf(mt, s[r >> 4][r & 15]);
        }
        __builtin_amdgcn_sched_barrier(0);
        const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(mt), __float_as_uint(mt), false, false);
        return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1])) * mul;
    };
    // Tile j0, whose scores are in s, limited and no more than kLag above m: its weights
    // beside the next tile's scores, then its products beside those scores' largest.
    auto step = [&](uint8_t *k_this, uint8_t *k_next, uint8_t *v_this, uint8_t *v_next, uint32_t *flag,
                    uint32_t j0) __attribute__((always_inline)) {
        all_barrier();     // k_next and v_this are filled, k_this and v_next are done with
        const bool more = j0 + kKeys < kmax;
        if (more) {
            load_k(j0 + 2 * kKeys, k_this);
            load_v(j0 + kKeys, v_next);
        }
        if (j0 + kKeys > kmin) {
            screen(v_this, flag);
            lds_barrier();
        }
        if (!live) return;
        if (more) {
            f32x16 nx[2];
            scores(k_next, nx, true);
            s[0] = nx[0], s[1] = nx[1];
            limit(j0 + kKeys);
        } else {
            const float ref = reference();
#pragma unroll
            for (int i = 0; i < 16; ++i) weight_pair(i, ref);
        }
        const float mt = products(v_this);
        add_found(flag, j0);
        if (more) rescale(mt);
    };
    all_barrier();
#pragma unroll
    for (int k = 0; k < NK; ++k) qf[k] = *reinterpret_cast<const u32x4 *>(qbuf + chunk_at(lr, 2 * k + lg));
    lds_barrier();   // the buffers that held Q are free
    load_k(kKeys, kb1);
    scores(kb0, s, false);
    limit(0);
    {
        float mt = -INFINITY;
#pragma unroll
        for (int r = 0; r < 32; ++r) mt = fmaxf(mt, s[r >> 4][r & 15]);
        rescale(fmaxf(mt, __shfl_xor(mt, 32, 64)) * mul);
    }
    for (uint32_t j0 = 0; j0 < kmax; j0 += 2 * kKeys) {
        step(kb0, kb1, vb0, vb1, odd0, j0);
        if (j0 + kKeys < kmax) step(kb1, kb0, vb1, vb0, odd1, j0 + kKeys);
    }
    l += __shfl_xor(l, 32, 64);
    // A lane holds dims 32 d + 8 c + 4 lg + i of row lr: through LDS (the wavefront's part
    // of a buffer that is done with), so that rows are stored whole
    lds_barrier();
    uint8_t *turn = (wave & 2 ? kb1 : kb0) + (wave & 1) * (32 * RB);
    const float inv = 1.0f / l;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int c = 0; c < 4; ++c)
            *reinterpret_cast<uint2 *>(turn + chunk_at(lr, 4 * d + c) + 8 * lg) =
                make_uint2(pack2<E>(o[d][4 * c] * inv, o[d][4 * c + 1] * inv),
                           pack2<E>(o[d][4 * c + 2] * inv, o[d][4 * c + 3] * inv));
    __builtin_amdgcn_wave_barrier();
    T *out = static_cast<T *>(a.out) + (uint64_t(t0) * a.H + kh * G) * a.D;
    const uint32_t c = lane % CPR;
#pragma unroll
    for (uint32_t i = 0; i < 32 / RPL; ++i) {
        const uint32_t r = i * RPL + lane / CPR, rr = wr0 + r, t = rr / G;
        if (rr < R && 8 * c < a.D)
            *reinterpret_cast<u32x4 *>(out + (uint64_t(t) * a.H + (rr - t * G)) * a.D + 8 * c) =
                *reinterpret_cast<const u32x4 *>(turn + chunk_at(r, c));
    }
}

template <class E, int DP>
__global__ __launch_bounds__(256, DP > 128 ? 1 : 2) void packed_tile_kernel(AttnPackedArgs a, float mul,
                                                                           uint32_t places) {
    packed_tile<E, DP>(a, mul, places);
}

// --------------------------------------------------------- tiled form, f32 ----
// f32 rows on the f32 matrix cores (32x32x2, 64 cycles): products and sums in f32
// throughout. They run at a sixteenth of the 16-bit rate, so a workgroup takes 32 rows
// and its wavefronts share the rows' keys, 32-key tiles in turn: four times the
// workgroups, a quarter of the chain. Each wavefront loads its own tiles into LDS, K's
// next while V is multiplied and V's next while K is, and meets the others once, at the
// end. A lane's scores are keys 8 (r / 4) + 4 (lane / 32) + r % 4 of row lane % 32, which
// is the order V's operands are read in; Q's dims go to the steps in the order in which
// 16-byte reads of K bring them. V that is not finite: as in the 16-bit form.
// 5 prompts of 33 to 1000 rows, 8 heads on 2 of 96 dims: 44 us, of which the longest
// prompt's last rows take most, 8 tiles a wavefront one after the other (1.9 GFLOP are 12
// us at the rate of an f32 product); a wavefront a row (below) took 583. 96 dims of rows of
// 128 are multiplied as 96: a quarter less of them.
constexpr uint32_t kRows32 = 32, kKeys32 = 32;

template <int DP, int W>
struct F32Lds {
    // K and V, [32 keys][DP], chunk c of row r at c ^ (r & 15); then O, [32 rows][DP] likewise
    float k[W][kKeys32 * DP], v[W][kKeys32 * DP];
    float m[W][kRows32], l[W][kRows32];
};

// DC: the dims that are multiplied, of rows of DP.
template <int DP, int DC, int W>
__device__ __forceinline__ void packed_f32(const AttnPackedArgs &a, const float mul, const uint32_t places) {
    constexpr int NC = DC / 8, DB = DC / 32;              // 16-byte chunks a lane reads of a key; 32-dim blocks
    constexpr uint32_t CPR = DP / 4, RPL = 256 / DP, kOob = 0x80000000u;
    __shared__ __attribute__((aligned(1024))) F32Lds<DP, W> lds;
    if (blockIdx.x == 0) check_starts(a.pb);
    const uint32_t G = a.H / a.Hkv, kh = blockIdx.x % a.Hkv;
    Place at;
    if (!place_of(a.pb, G, kRows32, places - 1 - blockIdx.x / a.Hkv, &at)) return;
    const uint32_t t0 = at.lo, n = at.hi - at.lo, R = n * G, r0 = at.unit * kRows32;
    const int tid = threadIdx.x, lane = tid & 63, lr = lane & 31, lg = lane >> 5;
    const uint32_t wave = pk_uni(uint32_t(tid) >> 6);
    const uint32_t row = r0 + lr < R ? r0 + lr : R - 1, tok = row / G, lim = tok + 1;
    const uint32_t kmin = pk_uni(r0 / G + 1), kmax = pk_uni((r0 + kRows32 - 1 < R ? r0 + kRows32 - 1 : R - 1) / G + 1);
    const float *kp = static_cast<const float *>(a.k) + uint64_t(t0) * a.k_stride + uint64_t(kh) * a.D;
    const float *vp = static_cast<const float *>(a.v) + uint64_t(t0) * a.v_stride + uint64_t(kh) * a.D;
    float *const kb = lds.k[wave], *const vb = lds.v[wave];
    auto place = [](uint32_t r, uint32_t c) { return r * DP + (c ^ (r & 15u)) * 4u; };   // of a 16-byte chunk

    auto load_tile = [&](const float *base, uint32_t stride, uint32_t j0, float *buf) {
        const uint32_t left = j0 < n ? (n - j0 < kKeys32 ? n - j0 : kKeys32) : 0u;
        const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(base + uint64_t(left ? j0 : 0u) * stride), 0,
                                                         left ? int(((left - 1) * stride + a.D) * 4u) : 0, 0x00020000);
#pragma unroll
        for (uint32_t t = 0; t < kKeys32 / RPL; ++t) {
            const uint32_t kr = t * RPL + lane / CPR, c = (lane % CPR) ^ (kr & 15u);
            load_to_lds(r, reinterpret_cast<uint8_t *>(buf) + 1024 * t, 4 * c < a.D ? (kr * stride + 4 * c) * 4u : kOob);
        }
    };
    load_tile(kp, a.k_stride, wave * kKeys32, kb);
    load_tile(vp, a.v_stride, wave * kKeys32, vb);

    // dims 8 i + 4 lg + e of the lane's row
    float4 q[NC];
    {
        const float *qp = static_cast<const float *>(a.q) + uint64_t(t0 + tok) * a.q_stride + (uint64_t(kh) * G + (row - tok * G)) * a.D;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const uint32_t d = 8 * i + 4 * lg;
            q[i] = d < a.D ? *reinterpret_cast<const float4 *>(qp + d) : float4{0, 0, 0, 0};
        }
    }
    auto odd = [](float x) { return !(fabsf(x) <= 3.4028235e38f); };

    f32x16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    for (uint32_t j0 = wave * kKeys32; j0 < kmax; j0 += W * kKeys32) {
        // K has landed (V's loads, the later ones, may not have)
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt((15 << 8) | (7 << 4) | ((kKeys32 / RPL) & 15) | (((kKeys32 / RPL) >> 4) << 14));
        asm volatile("" ::: "memory");
        f32x16 s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.0f;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const float4 x = *reinterpret_cast<const float4 *>(kb + place(lr, 2 * i + lg));
            s = __builtin_amdgcn_mfma_f32_32x32x2f32(x.x, q[i].x, s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x2f32(x.y, q[i].y, s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x2f32(x.z, q[i].z, s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x2f32(x.w, q[i].w, s, 0, 0, 0);
        }
        // V has landed; K's reads are done, its next tile may come
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(7 << 4);   // vmcnt(0) lgkmcnt(0)
        asm volatile("" ::: "memory");
        load_tile(kp, a.k_stride, j0 + W * kKeys32, kb);
        const bool full = j0 + kKeys32 <= kmin;
        bool found = false;
        if (!full) {
            const int see = int(lim) - int(j0) - 4 * lg;
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = 8 * (r >> 2) + (r & 3) < see ? s[r] : -INFINITY;
#pragma unroll 1
            for (uint32_t i = lane; i < kKeys32 * DP / 4; i += 64) {
                float4 x = *reinterpret_cast<float4 *>(vb + 4 * i);
                const bool here = odd(x.x) || odd(x.y) || odd(x.z) || odd(x.w);
                found |= here;
                if (!here) continue;
                x.x = odd(x.x) ? 0.0f : x.x, x.y = odd(x.y) ? 0.0f : x.y;
                x.z = odd(x.z) ? 0.0f : x.z, x.w = odd(x.w) ? 0.0f : x.w;
                *reinterpret_cast<float4 *>(vb + 4 * i) = x;
            }
            found = __ballot(found) != 0;
        }
        float mt = -INFINITY;
#pragma unroll
        for (int r = 0; r < 16; ++r) mt = fmaxf(mt, s[r]);
        mt = fmaxf(mt, __shfl_xor(mt, 32, 64)) * mul;
        if (__any(mt > m)) {
            const float mn = fmaxf(m, mt);
            const float al = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            l *= al;
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] *= al;
            m = mn;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], mul, -ref));
            l += s[r];
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const uint32_t kr = 8 * (r >> 2) + 4 * lg + (r & 3);
#pragma unroll
            for (int d = 0; d < DB; ++d)
                o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(vb[place(kr, 8 * d + (lr >> 2)) + (lr & 3)], s[r], o[d], 0, 0, 0);
        }
        if (__builtin_expect(found, 0)) {
#pragma unroll 1
            for (uint32_t j = j0; j < j0 + kKeys32 && j < n; ++j)
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const uint32_t dim = 32u * d + 8u * c + 4u * lg;
                        if (j >= lim || dim >= a.D) continue;
                        const float4 x = *reinterpret_cast<const float4 *>(vp + uint64_t(j) * a.v_stride + dim);
                        o[d][4 * c] += odd(x.x) ? x.x : 0.0f;
                        o[d][4 * c + 1] += odd(x.y) ? x.y : 0.0f;
                        o[d][4 * c + 2] += odd(x.z) ? x.z : 0.0f;
                        o[d][4 * c + 3] += odd(x.w) ? x.w : 0.0f;
                    }
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4));   // lgkmcnt(0): V's reads are done
        asm volatile("" ::: "memory");
        load_tile(vp, a.v_stride, j0 + W * kKeys32, vb);
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(7 << 4);   // (the loads past the last tile still write LDS)
    asm volatile("" ::: "memory");
    l += __shfl_xor(l, 32, 64);
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int c = 0; c < 4; ++c)
            *reinterpret_cast<float4 *>(kb + place(lr, 8 * d + 2 * c + lg)) =
                float4{o[d][4 * c], o[d][4 * c + 1], o[d][4 * c + 2], o[d][4 * c + 3]};
    if (lg == 0) lds.m[wave][lr] = m, lds.l[wave][lr] = l;
    __syncthreads();
    float *out = static_cast<float *>(a.out) + (uint64_t(t0) * a.H + kh * G) * a.D;
    for (uint32_t i = tid; i < kRows32 * CPR; i += 64 * W) {
        const uint32_t r = i / CPR, c = i % CPR, rr = r0 + r, t = rr / G;
        if (rr >= R || 4 * c >= a.D) continue;
        float M = lds.m[0][r];
#pragma unroll
        for (int w = 1; w < W; ++w) M = fmaxf(M, lds.m[w][r]);
        const float ref = M == -INFINITY ? 0.0f : M;
        float4 x = {0, 0, 0, 0};
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float e = __builtin_amdgcn_exp2f(lds.m[w][r] - ref);
            const float4 y = *reinterpret_cast<const float4 *>(lds.k[w] + place(r, c));
            sum = fmaf(lds.l[w][r], e, sum);
            x.x = fmaf(y.x, e, x.x), x.y = fmaf(y.y, e, x.y), x.z = fmaf(y.z, e, x.z), x.w = fmaf(y.w, e, x.w);
        }
        *reinterpret_cast<float4 *>(out + (uint64_t(t) * a.H + (rr - t * G)) * a.D + 4 * c) =
            float4{x.x / sum, x.y / sum, x.z / sum, x.w / sum};
    }
}

template <int DP, int DC, int W>
__global__ __launch_bounds__(64 * W, 1) void packed_f32_kernel(AttnPackedArgs a, float mul, uint32_t places) {
    packed_f32<DP, DC, W>(a, mul, places);
}

// What the tiles take: 16-byte rows of q, k, v and out, offsets within a tile's 64 keys
// and a workgroup's 128 rows below 2^31 bytes.
bool tiles_apply(const AttnPackedArgs &a) {
    auto at16 = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    const uint32_t far = std::max({a.q_stride, a.k_stride, a.v_stride});
    const uint32_t e = a.dtype == 8 ? 4 : 8;      // elements of 16 bytes
    return a.D % e == 0 && a.D <= 256 && a.q_stride % e == 0 && a.k_stride % e == 0 && a.v_stride % e == 0 &&
           at16(a.q) && at16(a.k) && at16(a.v) && at16(a.out) && far < (1u << 23);
}

uint32_t places_of(const AttnPackedArgs &a, uint32_t rows) {
    return uint32_t(uint64_t(a.pb.tokens) * (a.H / a.Hkv) / rows) + a.pb.batch;
}

template <class E>
void launch_tiles(const AttnPackedArgs &a, float mul, hipStream_t stream) {
    const uint32_t places = places_of(a, kRows), grid = places * a.Hkv;
    if (a.D <= 64) packed_tile_kernel<E, 64><<<grid, 256, 0, stream>>>(a, mul, places);
    else if (a.D <= 128) packed_tile_kernel<E, 128><<<grid, 256, 0, stream>>>(a, mul, places);
    else packed_tile_kernel<E, 256><<<grid, 256, 0, stream>>>(a, mul, places);
}

void launch_f32(const AttnPackedArgs &a, float mul, hipStream_t stream) {
    const uint32_t places = places_of(a, kRows32), grid = places * a.Hkv;
    if (a.D <= 64) packed_f32_kernel<64, 64, 4><<<grid, 256, 0, stream>>>(a, mul, places);
    else if (a.D <= 96) packed_f32_kernel<128, 96, 4><<<grid, 256, 0, stream>>>(a, mul, places);
    else if (a.D <= 128) packed_f32_kernel<128, 128, 4><<<grid, 256, 0, stream>>>(a, mul, places);
    else packed_f32_kernel<256, 256, 2><<<grid, 128, 0, stream>>>(a, mul, places);      // (LDS for two wavefronts)
}

// ---------------------------------------------------------- general form ----
// One wavefront a token and head, any head_dim, stride and alignment: for what the tiles
// do not take, 30 to 130 times as long where they do.
template <class E>
struct RowSrc {
    const typename E::T *kp, *vp;
    uint64_t ks, vs;
    __device__ float k(uint32_t j, uint32_t d) const { return E::widen(kp[j * ks + d]); }
    __device__ float v(uint32_t j, uint32_t d) const { return E::widen(vp[j * vs + d]); }
    __device__ float k_scale(uint32_t) const { return 1.0f; }
    __device__ float v_scale(uint32_t) const { return 1.0f; }
};

template <class E, int kDims>
__global__ __launch_bounds__(256) void packed_rows_kernel(AttnPackedArgs a, float mul) {
    __shared__ float qs[4][64 * kDims];
    if (blockIdx.x == 0) check_starts(a.pb);
    const uint32_t wave = pk_uni(threadIdx.x >> 6), lane = threadIdx.x & 63u;
    const uint64_t item = uint64_t(blockIdx.x) * 4 + wave;
    const uint32_t tok = uint32_t(item / a.H), h = uint32_t(item % a.H);
    if (tok >= a.pb.tokens) return;
    const uint32_t b = last_at_most(a.pb.batch, tok, [&](uint32_t s) { return start_of(a.pb, s); });
    const uint32_t r0 = start_of(a.pb, b);
    if (tok < r0 || tok >= start_of(a.pb, b + 1)) return;
    typedef typename E::T T;
    const T *q = static_cast<const T *>(a.q) + uint64_t(tok) * a.q_stride + uint64_t(h) * a.D;
    for (uint32_t d = lane; d < a.D; d += 64) qs[wave][d] = E::widen(q[d]) * mul;
    const uint32_t kh = h / (a.H / a.Hkv);
    const RowSrc<E> src{static_cast<const T *>(a.k) + uint64_t(r0) * a.k_stride + uint64_t(kh) * a.D,
                        static_cast<const T *>(a.v) + uint64_t(r0) * a.v_stride + uint64_t(kh) * a.D,
                        a.k_stride, a.v_stride};
    T *out = static_cast<T *>(a.out) + (uint64_t(tok) * a.H + h) * a.D;
    attend_row<kDims>(qs[wave], a.D, tok - r0 + 1, src, [&](uint32_t d, float v) { out[d] = E::narrow(v); });
}

template <class E>
void launch_rows(const AttnPackedArgs &a, float mul, hipStream_t stream) {
    const uint32_t grid = uint32_t((uint64_t(a.pb.tokens) * a.H + 3) / 4);
    if (a.D <= 128) packed_rows_kernel<E, 2><<<grid, 256, 0, stream>>>(a, mul);
    else packed_rows_kernel<E, kPackedMaxDim / 64><<<grid, 256, 0, stream>>>(a, mul);
}

}  // namespace

uint64_t attn_packed_threads(const AttnPackedArgs &a) {
    if (!tiles_apply(a)) return (uint64_t(a.pb.tokens) * a.H + 3) / 4 * 256;
    const bool f32 = a.dtype == 8;
    return uint64_t(places_of(a, f32 ? kRows32 : kRows)) * a.Hkv * (f32 && a.D > 128 ? 128 : 256);
}

hipError_t launch_attn_packed(const AttnPackedArgs &a, hipStream_t stream) {
    const float mul = kLog2e / a.score_scale;
    if (tiles_apply(a)) {
        if (a.dtype == 7) launch_tiles<Bf16>(a, mul, stream);
        else if (a.dtype == 6) launch_tiles<F16>(a, mul, stream);
        else launch_f32(a, mul, stream);
        return hipGetLastError();
    }
    if (a.dtype == 7) launch_rows<Bf16>(a, mul, stream);
    else if (a.dtype == 6) launch_rows<F16>(a, mul, stream);
    else launch_rows<F32>(a, mul, stream);
    return hipGetLastError();
}

}  // namespace holo
