// packed_tile.h — 64-key tiles of 16-bit K and V in LDS, as the tiled attention of a
// packed batch reads them (attn_packed.hip, attn_blocks.hip): rows of 2 DP bytes whose
// 16-byte chunks sit at chunk ^ swz(row), so that the K reads and the transposing V
// reads meet distinct banks.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "packed_batch.h"

namespace holo {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) uint8_t lds_u8;

// A workgroup barrier over LDS only: the loads in flight are not waited for.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_s_waitcnt(15 | (3 << 14) | (7 << 4));   // lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// The same, with the loads into LDS landed.
__device__ __forceinline__ void all_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(7 << 4);   // vmcnt(0) lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A wavefront's 1 KiB straight into LDS: each lane's 16 bytes at byte `off` of r, lane i's
// to dst + 16 i.
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t r, uint8_t *dst, uint32_t off) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_u8 *)dst, 16, off, 0, 0, 0);
}

// Two weights narrowed to nearest.
template <class E>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    if constexpr (std::is_same_v<E, Bf16>) {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, bf16x2{__bf16(lo), __bf16(hi)});
    } else {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, f16x2{_Float16(lo), _Float16(hi)});
    }
}

template <int DP>
__device__ __forceinline__ uint32_t swz_k(uint32_t row) {
    return DP >= 128 ? (row & 15u) : ((row >> 1) & 7u);
}
template <int DP>
__device__ __forceinline__ uint32_t swz_v(uint32_t row) {
    return DP >= 128 ? 4u * (row & 3u) : 4u * ((row >> 1) & 1u);
}

// Where a lane reads K: chunk lane / 32 of row lane % 32, swizzled; chunk 2 k + lane /
// 32 is that place with 2 k toggled. V's places likewise, for v_frag.
template <int DP>
__device__ __forceinline__ uint32_t k_place(uint32_t lane) {
    const uint32_t lr = lane & 31u, lg = lane >> 5;
    return lr * (2 * DP) + ((lg ^ swz_k<DP>(lr)) * 16u);
}
template <int DP>
__device__ __forceinline__ uint32_t v_place(uint32_t lane) {
    const uint32_t g16 = lane >> 4, r16 = lane & 15u;
    const uint32_t row = 4u * (g16 >> 1) + (r16 >> 2), chunk = 2u * (g16 & 1u) + ((r16 & 3u) >> 1);
    return row * (2 * DP) + ((chunk ^ swz_v<DP>(row)) * 16u) + (r16 & 1u) * 8u;
}
// Operand of dims 16 k .. 16 k + 15 of key rows 32 h .. 32 h + 31 of the K tile in
// `buf`; of 32-dim block d of key rows 16 st .. 16 st + 15 of V's, transposed: a lane's
// eight keys are 16 st + 8 c + 4 (lane / 32) + e, the order of its scores.
template <int DP>
__device__ __forceinline__ u32x4 k_frag(const uint8_t *buf, uint32_t at, int k, int h) {
    return *reinterpret_cast<const lds_u32x4 *>((const lds_u8 *)buf + (at ^ (32u * k)) + 64u * DP * h);
}
template <int DP>
__device__ __forceinline__ u32x4 v_frag(const uint8_t *buf, uint32_t at, int st, int d) {
    const lds_u8 *p = (const lds_u8 *)buf + (at ^ (64u * d)) + 32u * DP * st;
    const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_i16x4 *>(const_cast<lds_u8 *>(p)));
    const i16x4 hi =
        __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_i16x4 *>(const_cast<lds_u8 *>(p + 16u * DP)));
    return __builtin_bit_cast(u32x4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

}  // namespace holo
