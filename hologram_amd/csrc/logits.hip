// logits.hip — a request's sampling rules on its logits (LogitsProcess, 129).
#include <hip/hip_runtime.h>

#include "holo_kernels.h"
#include "packed_batch.h"

namespace holo {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// A workgroup takes kCols columns of a row. What the rules say of a column is one
// word in LDS: bits 0-18 how often it was generated, bits 19-30 one more than the
// place of its summed bias, bit 31 seen in the prompt. Every workgroup reads the
// row's whole history (it stays in L2) and keeps what falls into its columns, so
// counts are integers whose order does not matter, and no column's rule leaves
// the workgroup that writes it. The logits are copied, masked, while the rules are
// gathered; then the columns that a rule names, which their first finder listed, are
// written again, a thread each: few of a row's columns have one, and a division for every
// column that shares its 64 lanes with one took longer than that. Bound by the logits' own
// bytes, and by the gathering where many rows have long histories: 128 rows of 128000 bf16
// with masks, biases and 4096 tokens of history each, 70 MB, 21 us or 3.3 TB/s; without
// histories 14 us, 4.8 TB/s; one row 5 us, a workgroup's chain of history, barrier, copies
// and listed columns (an empty launch, queued: 1.6). 8192 columns read a row's
// history 16 times; 4096 and 256 threads, 32 times: 64 rows 13.3 us against 12.3, one row
// the same; 16384 and 512 threads 25 against 22.
constexpr uint32_t kCols = 8192, kThreads = kCols / 16, kList = 2048;

// 16 bytes of elements.
template <class E>
union Vec {
    u32x4 v;
    typename E::T e[16 / sizeof(typename E::T)];
};

template <class E>
__global__ __launch_bounds__(kThreads) void logits_kernel(LogitsArgs a, uint32_t chunks, bool wide) {
    constexpr uint32_t kV = 16 / sizeof(typename E::T);
    __shared__ __attribute__((aligned(16))) uint32_t word[kCols];
    __shared__ uint16_t list[kList];                    // places that a rule names
    __shared__ uint32_t listed, twice;                  // so many; some token of the workgroup's has two biases
    extern __shared__ int32_t ids[];                    // [biases], then their sums
    float *sums = reinterpret_cast<float *>(ids + a.biases);
    const uint32_t row = blockIdx.x / chunks, tid = threadIdx.x;
    const uint64_t at = uint64_t(row) * a.cols;
    const auto *in = static_cast<const typename E::T *>(a.logits) + at;
    auto *out = static_cast<typename E::T *>(a.out) + at;
    // columns [c0, c0 + kCols) of which those in [0, cols) are there; c0 falls on 16 bytes
    const uint32_t skew = wide ? uint32_t(reinterpret_cast<uintptr_t>(in) / sizeof(typename E::T)) % kV : 0u;
    const int64_t c0 = int64_t(blockIdx.x % chunks) * kCols - skew;
    auto place = [&](int32_t id) -> uint32_t {          // in word, kCols or more for none of them
        const uint32_t p = uint32_t(id) - uint32_t(int32_t(c0));
        return uint32_t(id) < a.cols ? p : uint32_t(kCols);
    };
    // the thread's logits and their mask bits, on their way while the rules are gathered
    constexpr int kMine = kCols / (kV * kThreads);
    const uint32_t *mask = a.mask ? a.mask + uint64_t(row) * ((a.cols + 31) / 32) : nullptr;
    Vec<E> x[kMine];
    uint32_t bits[kMine];
    auto whole = [&](int i) {
        const int64_t c = c0 + kV * (tid + uint32_t(i) * kThreads);
        return wide && c >= 0 && c + kV <= a.cols;
    };
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        const int64_t c = c0 + kV * (tid + uint32_t(i) * kThreads);
        bits[i] = 0xffffffffu;
        if (!whole(i)) continue;
        x[i].v = *reinterpret_cast<const u32x4 *>(in + c);
        if (mask) {
            const uint32_t sh = uint32_t(c) & 31u;
            bits[i] = mask[c >> 5] >> sh;
            if (sh + kV > 32) bits[i] |= mask[(c >> 5) + 1] << (32 - sh);
        }
    }
    // and its first tokens (as long as the row may be: what counts of it comes with them)
    const int32_t *h = a.history ? a.history + uint64_t(row) * a.history_len : nullptr;
    const bool by16 = reinterpret_cast<uintptr_t>(h) % 16 == 0;
    constexpr uint32_t kFirst = 2;
    int4 tokens[kFirst];
    uint32_t n = 0, prompt = 0;
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if (h) {
#pragma unroll
        for (uint32_t u = 0; u < kFirst; ++u)
            if (by16 && tid + u * kThreads < a.history_len / 4) tokens[u] = reinterpret_cast<const int4 *>(h)[tid + u * kThreads];
        prompt = a.spans[2 * uint64_t(row)];
        n = a.spans[2 * uint64_t(row) + 1];
        rep = a.params[3 * uint64_t(row)];
        freq = a.params[3 * uint64_t(row) + 1];
        pres = a.params[3 * uint64_t(row) + 2];
    }
    for (uint32_t c = 4 * tid; c < kCols; c += 4 * kThreads) *reinterpret_cast<u32x4 *>(word + c) = u32x4{0, 0, 0, 0};
    for (uint32_t j = tid; j < a.biases; j += kThreads) ids[j] = a.bias_ids[uint64_t(row) * a.biases + j];
    if (tid == 0) listed = 0, twice = 0;
    __syncthreads();
    // what no rule names is done: the mask's select
    const typename E::T none = E::narrow(-INFINITY);
    auto there = [&](uint32_t c) { return !mask || ((mask[c >> 5] >> (c & 31)) & 1u); };
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        const int64_t c = c0 + kV * (tid + uint32_t(i) * kThreads);
        if (whole(i)) {
#pragma unroll
            for (uint32_t e = 0; e < kV; ++e) x[i].e[e] = (bits[i] >> e) & 1u ? x[i].e[e] : none;
            *reinterpret_cast<u32x4 *>(out + c) = x[i].v;
        } else {
            for (uint32_t e = 0; e < kV; ++e)
                if (c + e >= 0 && c + e < a.cols) out[c + e] = there(uint32_t(c + e)) ? in[c + e] : none;
        }
    }
    // the one who finds a place without a rule lists it
    auto name = [&](uint32_t old, uint32_t p) {
        if (old) return;
        const uint32_t i = atomicAdd(&listed, 1u);
        if (i < kList) list[i] = uint16_t(p);
    };
    if (h) {
        n = n < a.history_len ? n : a.history_len;
        auto count = [&](int32_t id, uint32_t i) {
            const uint32_t p = place(id);
            if (p >= kCols) return;
            name(i < prompt ? atomicOr(&word[p], 0x80000000u) : atomicAdd(&word[p], 1u), p);
        };
        const uint32_t quads = by16 ? n / 4 : 0u;
        auto four = [&](const int4 &x, uint32_t q) {
            count(x.x, 4 * q), count(x.y, 4 * q + 1), count(x.z, 4 * q + 2), count(x.w, 4 * q + 3);
        };
#pragma unroll
        for (uint32_t u = 0; u < kFirst; ++u)
            if (tid + u * kThreads < quads) four(tokens[u], tid + u * kThreads);
        for (uint32_t q = tid + kFirst * kThreads; q < quads; q += kThreads) four(reinterpret_cast<const int4 *>(h)[q], q);
        for (uint32_t k = 4 * quads + tid; k < n; k += kThreads) count(h[k], k);
    }
    // A bias is its token's sum where the token has one; where a second is found, the
    // workgroup starts over with sums in the list's order.
    constexpr uint32_t kSlot = 0xfffu << 19;
    const float *bv = a.bias_values + uint64_t(row) * a.biases;
    for (uint32_t j = tid; j < a.biases; j += kThreads) {
        const uint32_t p = place(ids[j]);
        if (p >= kCols) continue;
        sums[j] = bv[j];
        const uint32_t old = atomicOr(&word[p], (j + 1) << 19);
        if (old & kSlot) twice = 1;
        name(old, p);
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((15 << 8) | (7 << 4));   // vmcnt(0): the copies are there, to be written over
    __syncthreads();
    if (twice) {
        for (uint32_t j = tid; j < a.biases; j += kThreads) {
            const uint32_t p = place(ids[j]);
            if (p < kCols) atomicAnd(&word[p], ~kSlot);
        }
        __syncthreads();
        for (uint32_t j = tid; j < a.biases; j += kThreads) {
            const int32_t id = ids[j];
            const uint32_t p = place(id);
            if (p >= kCols) continue;
            bool first = true;
            for (uint32_t k = 0; k < j; ++k) first &= ids[k] != id;
            if (!first) continue;
            float s = bv[j];
            for (uint32_t k = j + 1; k < a.biases; ++k)
                if (ids[k] == id) s += bv[k];
            sums[j] = s;
            atomicOr(&word[p], (j + 1) << 19);
        }
        __syncthreads();
    }
    auto rule = [&](uint32_t p) {
        const uint32_t c = uint32_t(c0 + p), w = word[p], n = w & 0x7ffffu, b = (w >> 19) & 0xfffu;
        if (!there(c)) return;
        float x = E::widen(in[c]);
        if (n || (w >> 31)) x = x > 0.0f ? x / rep : x * rep;
        if (n) x = x - (freq * float(n) + pres);
        if (b) x = x + sums[b - 1];
        out[c] = E::narrow(x);
    };
    if (listed <= kList) {
        for (uint32_t i = tid; i < listed; i += kThreads) rule(list[i]);
    } else {
        for (uint32_t p = tid; p < kCols; p += kThreads)
            if (word[p]) rule(p);
    }
}

// Workgroups a row; its columns begin up to 15 bytes into the first one's.
uint32_t chunks_of(const LogitsArgs &a) {
    const uint32_t kV = a.dtype == 8 ? 4 : 8;
    return uint32_t((uint64_t(a.cols) + kV - 1 + kCols - 1) / kCols);
}

template <class E>
void launch(const LogitsArgs &a, hipStream_t stream) {
    // the logits and the result as far past 16 bytes as each other
    const bool wide = (reinterpret_cast<uintptr_t>(a.logits) - reinterpret_cast<uintptr_t>(a.out)) % 16 == 0;
    const size_t lds = size_t(a.biases) * 8;
    const uint32_t chunks = chunks_of(a);
    logits_kernel<E><<<a.rows * chunks, kThreads, lds, stream>>>(a, chunks, wide);
}

}  // namespace

uint64_t logits_threads(const LogitsArgs &a) { return uint64_t(a.rows) * chunks_of(a) * kThreads; }

hipError_t launch_logits(const LogitsArgs &a, hipStream_t stream) {
    if (a.dtype == 7) launch<Bf16>(a, stream);
    else if (a.dtype == 6) launch<F16>(a, stream);
    else launch<F32>(a, stream);
    return hipGetLastError();
}

}  // namespace holo
