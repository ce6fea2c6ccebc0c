// logits.hip — a request's sampling rules on its logits (LogitsProcess, 129).
#include <hip/hip_runtime.h>

#include "holo_kernels.h"
#include "packed_batch.h"

namespace holo {
namespace {

// A workgroup takes kCols columns of a row. What the rules say of a column is one
// word in LDS: bits 0-18 how often it was generated, bits 19-30 one more than the
// place of its summed bias, bit 31 seen in the prompt. Every workgroup reads the
// row's whole history (it stays in L2) and keeps what falls into its columns, so
// counts are integers whose order does not matter, and no column's rule leaves
// the workgroup that writes it.
constexpr uint32_t kCols = 4096, kThreads = 256;

template <class E>
__global__ __launch_bounds__(kThreads) void logits_kernel(LogitsArgs a, uint32_t chunks) {
    __shared__ uint32_t word[kCols];
    __shared__ int32_t ids[kLogitsMaxBiases];
    __shared__ float sums[kLogitsMaxBiases];
    const uint32_t row = blockIdx.x / chunks, c0 = (blockIdx.x % chunks) * kCols, tid = threadIdx.x;
    const uint32_t cols = a.cols - c0 < kCols ? a.cols - c0 : kCols;
    for (uint32_t c = tid; c < kCols; c += kThreads) word[c] = 0;
    const int32_t *bi = a.bias_ids + uint64_t(row) * a.biases;
    const float *bv = a.bias_values + uint64_t(row) * a.biases;
    if (a.bias_ids)
        for (uint32_t j = tid; j < a.biases; j += kThreads) ids[j] = bi[j];
    __syncthreads();
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if (a.history) {
        const int32_t *h = a.history + uint64_t(row) * a.history_len;
        const uint32_t n = a.spans[2 * row + 1] < a.history_len ? a.spans[2 * row + 1] : a.history_len;
        const uint32_t prompt = a.spans[2 * row];
        for (uint32_t i = tid; i < n; i += kThreads) {
            const uint32_t c = uint32_t(h[i]) - c0;
            if (h[i] < 0 || uint32_t(h[i]) < c0 || c >= cols) continue;
            if (i < prompt) atomicOr(&word[c], 0x80000000u);
            else atomicAdd(&word[c], 1u);
        }
        rep = a.params[3 * uint64_t(row)];
        freq = a.params[3 * uint64_t(row) + 1];
        pres = a.params[3 * uint64_t(row) + 2];
    }
    if (a.bias_ids)
        for (uint32_t j = tid; j < a.biases; j += kThreads) {
            const int32_t id = ids[j];
            if (id < 0 || uint32_t(id) < c0 || uint32_t(id) - c0 >= cols) continue;
            bool first = true;
            for (uint32_t k = 0; k < j; ++k) first &= ids[k] != id;
            if (!first) continue;
            float s = bv[j];
            for (uint32_t k = j + 1; k < a.biases; ++k)
                if (ids[k] == id) s += bv[k];
            sums[j] = s;
            atomicOr(&word[uint32_t(id) - c0], (j + 1) << 19);
        }
    __syncthreads();
    const auto *in = static_cast<const typename E::T *>(a.logits) + uint64_t(row) * a.cols + c0;
    auto *out = static_cast<typename E::T *>(a.out) + uint64_t(row) * a.cols + c0;
    const uint32_t *mask = a.mask ? a.mask + uint64_t(row) * ((a.cols + 31) / 32) : nullptr;
    for (uint32_t c = tid; c < cols; c += kThreads) {
        const uint32_t w = word[c];
        const bool allowed = !mask || ((mask[(c0 + c) >> 5] >> ((c0 + c) & 31u)) & 1u);
        typename E::T bits = in[c];
        if (w || !allowed) {
            float x = E::widen(bits);
            const uint32_t n = w & 0x7ffffu, at = (w >> 19) & 0xfffu;
            if (n || (w >> 31)) x = x > 0.0f ? x / rep : x * rep;
            if (n) x = x - (freq * float(n) + pres);
            if (at) x = x + sums[at - 1];
            bits = E::narrow(allowed ? x : -INFINITY);
        }
        out[c] = bits;
    }
}

}  // namespace

hipError_t launch_logits(const LogitsArgs &a, hipStream_t stream) {
    const uint32_t chunks = (a.cols + kCols - 1) / kCols;
    const dim3 grid(a.rows * chunks);
    if (a.dtype == 7) logits_kernel<Bf16><<<grid, kThreads, 0, stream>>>(a, chunks);
    else if (a.dtype == 6) logits_kernel<F16><<<grid, kThreads, 0, stream>>>(a, chunks);
    else logits_kernel<F32><<<grid, kThreads, 0, stream>>>(a, chunks);
    return hipGetLastError();
}

}  // namespace holo
