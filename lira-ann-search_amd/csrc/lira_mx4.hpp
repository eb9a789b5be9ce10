// lira_mx4.hpp -- device helpers of the microscaled 4-bit format (lira_mx4.hip).
//
// A block is 32 consecutive elements of a row: 32 codes of 4 bits (sign, 2 exponent bits, 1
// mantissa bit: 0, .5, 1, 1.5, 2, 3, 4, 6) and one scale 2^(s - 127), s a byte (255: NaN).
// A plane is 128 elements = 4 blocks = 64 bytes of codes and 4 of scales; planes are the
// outer dimension, so the 16 x 128 fragment of v_mfma_scale_f32_16x16x128_f8f6f4 is 1 KiB
// of consecutive codes: lane l holds block l / 16 of row l % 16 (16 bytes) and its scale.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lira {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// 16 bytes to memory at any alignment, past the caches' write-back (nt): results are whole runs that this
// kernel does not read again.  8192 x 8192 fp32 out of a 512-deep product 103 us with plain stores, 75 so.
__device__ __forceinline__ void stream16(void *at, i32x4 v) {
    typedef int anywhere __attribute__((ext_vector_type(4), aligned(2)));
    __builtin_nontemporal_store((anywhere)v, (anywhere *)at);
}

// element types of lira_hip.h's LIRA_DTYPE_*
struct F32 {
    typedef float T;
    static constexpr uint32_t kNegInf = 0xff800000u;
    static __device__ __forceinline__ float up(float v) { return v; }
    static __device__ __forceinline__ float down(float v) { return v; }
};
struct BF16 {
    typedef __bf16 T;
    static constexpr uint32_t kNegInf = 0xff80u;
    static __device__ __forceinline__ float up(__bf16 v) { return (float)v; }
    static __device__ __forceinline__ __bf16 down(float v) { return (__bf16)v; }  // to nearest, ties to even
};
struct F16 {
    typedef _Float16 T;
    static constexpr uint32_t kNegInf = 0xfc00u;
    static __device__ __forceinline__ float up(_Float16 v) { return (float)v; }
    static __device__ __forceinline__ _Float16 down(float v) { return (_Float16)v; }
};

// |v| as an integer: orders like |v| and puts Inf and NaN above every number
__device__ __forceinline__ uint32_t mag(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// mag() of the largest of a block's 32 elements, 8 in each of 4 neighbouring lanes (DPP)
__device__ __forceinline__ uint32_t quad_max(const float (&v)[8]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, mag(v[i]));
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xf, 0xf, false));  // lane ^ 1
    return max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xf, 0xf, false));  // lane ^ 2
}

// the scale byte of a block whose largest magnitude has these bits: exponent - 2 (6 = 1.5 * 2^2
// is the largest element), not below 2^-127; 255 where the block holds Inf or NaN
__device__ __forceinline__ uint32_t scale_code(uint32_t m) {
    const uint32_t e = m >> 23;
    return e == 255 ? 255u : e < 2 ? 0u : e - 2;
}
// the operand form of v_cvt_scalef32_*: only the exponent field counts
__device__ __forceinline__ float scale_operand(uint32_t code) { return __uint_as_float(code << 23); }

// 8 floats -> 8 codes, element 0 in the low 4 bits; v / scale to nearest even, saturated at 6
__device__ __forceinline__ uint32_t to_codes(const float *v, float scale) {
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], scale, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], scale, 3);
    return r;
}

// N codes (the first in the low bits) -> the numbers they stand for; exact in fp32 but for 6 * 2^127
// and its like, which are past fp32's end
template <int N>
__device__ __forceinline__ void from_codes(uint32_t c, uint32_t s, float (&v)[N]) {
    const float scale = scale_operand(s);
    f32x2 t[4];
    t[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 0);
    t[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 1);
    if (N > 4) {
        t[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 2);
        t[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, scale, 3);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = s == 255 ? __uint_as_float(0x7fc00000u) : t[i / 2][i % 2];
}

// N = 8 or 32 consecutive elements of a row from element j (zeros past the row's end); VEC: the row's
// first element and the row stride are multiples of 16 bytes.  The ends of rows read their last
// element's place again: a branch round every load would wait for each.  ONCE: not kept in the L2.
template <class D, bool VEC, int N, bool ONCE = false>
__device__ __forceinline__ void load_run(const typename D::T *row, int64_t j, int64_t k, float (&v)[N]) {
    typedef typename D::T T;
    if (VEC && j + N <= k) {
        constexpr int E = 16 / sizeof(T);
        struct alignas(16) V {
            T e[E];
        } t[N / E];
#pragma unroll
        for (int i = 0; i < N / E; ++i) {
            const i32x4 *at = reinterpret_cast<const i32x4 *>(row + j + i * E);
            const i32x4 q = ONCE ? __builtin_nontemporal_load(at) : *at;
            __builtin_memcpy(&t[i], &q, 16);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = D::up(t[i / E].e[i % E]);
    } else {
        T t[N];
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = row[j + i < k ? j + i : k - 1];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = j + i < k ? D::up(t[i]) : 0.0f;
    }
}

}  // namespace lira
