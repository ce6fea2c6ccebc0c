// qk_norm_rotary.hip — q and k of a packed batch normed by the head and rotated by
// position (QkNormRotary, 130).
#include <hip/hip_runtime.h>

#include "holo_kernels.h"
#include "packed_batch.h"

namespace holo {
namespace {

// cos and sin of pos * freq. The product and its reduction to a quarter turn are f64:
// with n = rint(2 x / pi), x - n pi / 2 in two steps of one rounding each keeps 2^-50 of
// a radian for every |x| < 2^50, where f32 would lose the angle itself from some
// thousand positions on; what is left, at most pi / 4, is f32's.
__device__ __forceinline__ void turn(uint32_t pos, float freq, float *c, float *s) {
    const double x = double(pos) * double(freq), low = fma(double(pos), double(freq), -x);
    const double n = rint(x * 0.63661977236758134308);
    double r = fma(-n, 1.57079632679489655800, x);
    r = fma(-n, 6.12323399573676603587e-17, r) + low;
    float sn, cs;
    sincosf(float(r), &sn, &cs);
    const int quarter = int(n - 4.0 * floor(n * 0.25));      // 0 to 3
    *c = quarter & 1 ? (quarter == 1 ? -sn : sn) : (quarter == 0 ? cs : -cs);
    *s = quarter & 1 ? (quarter == 1 ? cs : -cs) : (quarter == 0 ? sn : -sn);
}

// The position of token `tok` in its sequence; false outside every sequence.
__device__ __forceinline__ bool position(const QkNormRotaryArgs &a, uint32_t tok, uint32_t *pos) {
    const uint32_t b = last_at_most(a.pb.batch, tok, [&](uint32_t s) { return start_of(a.pb, s); });
    const uint32_t lo = start_of(a.pb, b), hi = start_of(a.pb, b + 1);
    if (tok < lo || tok >= hi) return false;
    *pos = a.rot ? a.pos[b] + (tok - lo) : 0u;
    return true;
}

// General form: a wavefront a head's row, any head_dim, rotation and alignment.
template <class E>
__global__ __launch_bounds__(256) void rows_kernel(QkNormRotaryArgs a) {
    typedef typename E::T T;
    if (blockIdx.x == 0) check_starts(a.pb);
    const uint32_t lane = threadIdx.x & 63u, all = a.H + a.Hkv;
    const uint64_t item = uint64_t(blockIdx.x) * 4 + pk_uni(threadIdx.x >> 6);
    const uint32_t tok = uint32_t(item / all);
    uint32_t h = uint32_t(item - uint64_t(tok) * all), pos;
    if (tok >= a.pb.tokens || !position(a, tok, &pos)) return;
    const int which = h >= a.H;
    h -= which ? a.H : 0;
    const T *x = static_cast<const T *>(a.x[which]) + uint64_t(tok) * a.stride[which] + uint64_t(h) * a.D;
    T *out = static_cast<T *>(a.out[which]) + (uint64_t(tok) * (which ? a.Hkv : a.H) + h) * a.D;
    const T *gamma = static_cast<const T *>(a.gamma[which]);
    float inv = 1.0f;
    const bool norm = a.norms >> which & 1;
    if (norm) {
        float sum = 0.0f;
        for (uint32_t d = lane; d < a.D; d += 64) {
            const float v = E::widen(x[d]);
            sum = fmaf(v, v, sum);
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
        inv = 1.0f / sqrtf(sum / float(a.D) + a.eps);
    }
    auto get = [&](uint32_t d) {
        const float v = E::widen(x[d]) * inv;
        return gamma ? v * E::widen(gamma[d]) : v;
    };
    const uint32_t half = a.rot / 2;
    for (uint32_t i = lane; i < half; i += 64) {
        const uint32_t d0 = a.interleaved ? 2 * i : i, d1 = a.interleaved ? 2 * i + 1 : i + half;
        float c, s;
        turn(pos, a.freqs[i], &c, &s);
        c *= a.magnitude, s *= a.magnitude;
        const float u = get(d0), v = get(d1);
        out[d0] = E::narrow(fmaf(u, c, -(v * s)));
        out[d1] = E::narrow(fmaf(v, c, u * s));
    }
    for (uint32_t d = a.rot + lane; d < a.D; d += 64) out[d] = E::narrow(get(d));
}

template <class E>
void launch(const QkNormRotaryArgs &a, hipStream_t stream) {
    rows_kernel<E><<<uint32_t(qk_norm_rotary_threads(a) / 256), 256, 0, stream>>>(a);
}

}  // namespace

uint64_t qk_norm_rotary_threads(const QkNormRotaryArgs &a) {
    return (uint64_t(a.pb.tokens) * (a.H + a.Hkv) + 3) / 4 * 256;
}

hipError_t launch_qk_norm_rotary(const QkNormRotaryArgs &a, hipStream_t stream) {
    if (a.dtype == 7) launch<Bf16>(a, stream);
    else if (a.dtype == 6) launch<F16>(a, stream);
    else launch<F32>(a, stream);
    return hipGetLastError();
}

}  // namespace holo
