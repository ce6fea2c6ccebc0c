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
// the workgroup that writes it. Bound by the logits' own bytes where there are many
// rows: 128 rows of 128000 bf16 with masks, biases and 4096 tokens of
// history each, 70 MB, 22 us or 3.2 TB/s (every row's history is read 16 times, once a
// workgroup; 4096 columns and 256 threads, 32 times: 23 us; 64 rows 12.3 and 13.3, one row
// 6.1 and 6.1, the launch's own time).
constexpr uint32_t kCols = 8192, kThreads = kCols / 16;

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
    __shared__ uint32_t twice;                          // some token of the workgroup's has two biases
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
    int4 tokens = {-1, -1, -1, -1};
    uint32_t n = 0, prompt = 0;
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if (h) {
        if (by16 && tid < a.history_len / 4) tokens = reinterpret_cast<const int4 *>(h)[tid];
        prompt = a.spans[2 * uint64_t(row)];
        n = a.spans[2 * uint64_t(row) + 1];
        rep = a.params[3 * uint64_t(row)];
        freq = a.params[3 * uint64_t(row) + 1];
        pres = a.params[3 * uint64_t(row) + 2];
    }
    for (uint32_t c = 4 * tid; c < kCols; c += 4 * kThreads) *reinterpret_cast<u32x4 *>(word + c) = u32x4{0, 0, 0, 0};
    for (uint32_t j = tid; j < a.biases; j += kThreads) ids[j] = a.bias_ids[uint64_t(row) * a.biases + j];
    if (tid == 0) twice = 0;
    __syncthreads();
    if (h) {
        n = n < a.history_len ? n : a.history_len;
        auto count = [&](int32_t id, uint32_t i) {
            const uint32_t p = place(id);
            if (p >= kCols) return;
            if (i < prompt) atomicOr(&word[p], 0x80000000u);
            else atomicAdd(&word[p], 1u);
        };
        const uint32_t quads = by16 ? n / 4 : 0u;
        for (uint32_t q = tid; q < quads; q += kThreads) {
            if (q != tid) tokens = reinterpret_cast<const int4 *>(h)[q];
            count(tokens.x, 4 * q), count(tokens.y, 4 * q + 1), count(tokens.z, 4 * q + 2), count(tokens.w, 4 * q + 3);
        }
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
        if (atomicOr(&word[p], (j + 1) << 19) & kSlot) twice = 1;
    }
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
    const typename E::T none = E::narrow(-INFINITY);
    auto rule = [&](typename E::T bits, uint32_t w) {      // w != 0
        float x = E::widen(bits);
        const uint32_t n = w & 0x7ffffu, b = (w >> 19) & 0xfffu;
        if (n || (w >> 31)) x = x > 0.0f ? x / rep : x * rep;
        if (n) x = x - (freq * float(n) + pres);
        if (b) x = x + sums[b - 1];
        return E::narrow(x);
    };
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        const uint32_t p = kV * (tid + uint32_t(i) * kThreads);
        const int64_t c = c0 + p;
        if (whole(i)) {
            // what the mask leaves out is done at a select; few of the rest have a rule
            uint32_t w[kV], any = 0;
#pragma unroll
            for (uint32_t e = 0; e < kV; e += 4) {
                const u32x4 q = *reinterpret_cast<const u32x4 *>(word + p + e);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const bool in = (bits[i] >> (e + k)) & 1u;
                    any |= w[e + k] = in ? q[k] : 0u;
                    x[i].e[e + k] = in ? x[i].e[e + k] : none;
                }
            }
            if (any)
#pragma unroll
                for (uint32_t e = 0; e < kV; ++e)
                    if (w[e]) x[i].e[e] = rule(x[i].e[e], w[e]);
            *reinterpret_cast<u32x4 *>(out + c) = x[i].v;
        } else {
            for (uint32_t e = 0; e < kV; ++e) {
                const int64_t d = c + e;
                if (d < 0 || d >= a.cols) continue;
                const bool there = !mask || ((mask[d >> 5] >> (d & 31)) & 1u);
                out[d] = !there ? none : word[p + e] ? rule(in[d], word[p + e]) : in[d];
            }
        }
    }
}

template <class E>
void launch(const LogitsArgs &a, hipStream_t stream) {
    const uint32_t kV = 16 / sizeof(typename E::T);
    // the logits and the result as far past 16 bytes as each other
    const bool wide = (reinterpret_cast<uintptr_t>(a.logits) - reinterpret_cast<uintptr_t>(a.out)) % 16 == 0;
    const size_t lds = size_t(a.biases) * 8;
    const uint32_t chunks = uint32_t((uint64_t(a.cols) + kV - 1 + kCols - 1) / kCols);
    logits_kernel<E><<<a.rows * chunks, kThreads, lds, stream>>>(a, chunks, wide);
}

}  // namespace

hipError_t launch_logits(const LogitsArgs &a, hipStream_t stream) {
    if (a.dtype == 7) launch<Bf16>(a, stream);
    else if (a.dtype == 6) launch<F16>(a, stream);
    else launch<F32>(a, stream);
    return hipGetLastError();
}

}  // namespace holo
