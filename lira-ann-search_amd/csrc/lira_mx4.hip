// lira_mx4.hip -- microscaled 4-bit floats: packing, unpacking and the product on the matrix
// cores (layout and format: lira_mx4.hpp).
#include <string>

#include "lira_internal.hpp"
#include "lira_mx4.hpp"

namespace lira {

static constexpr int kPlane = 128;  // elements per plane

// ------------------------------------------------------------ pack / unpack
// 16 lanes per (row, plane), 8 elements each; the block's largest magnitude crosses its 4
// lanes by DPP.  A wave packs 4 consecutive rows: 256 bytes of codes and 16 of scales.
template <class D, bool VEC>
__global__ __launch_bounds__(256) void k_mx4_quantize(const typename D::T *__restrict__ x, int64_t n, int64_t k,
                                                      int64_t ld, uint8_t *__restrict__ codes,
                                                      uint8_t *__restrict__ scales, int64_t plane_rows) {
    const int lane = threadIdx.x & 15;
    const int64_t row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    const int64_t p = blockIdx.y;
    const bool live = row < n;
    float v[8];
    load8<D, VEC>(x + (live ? row : 0) * ld, p * kPlane + lane * 8, k, v);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, mag(v[i]));
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xf, 0xf, false));  // lane ^ 1
    m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xf, 0xf, false));  // lane ^ 2
    const uint32_t s = scale_code(m);
    const uint32_t c = s == 255 ? 0u : to_codes(v, scale_operand(s));
    if (!live) return;
    const int64_t at = p * plane_rows + row;
    *reinterpret_cast<uint32_t *>(codes + at * 64 + lane * 4) = c;
    if ((lane & 3) == 0) scales[at * 4 + (lane >> 2)] = (uint8_t)s;
}

template <class D>
__global__ __launch_bounds__(256) void k_mx4_dequantize(const uint8_t *__restrict__ codes,
                                                        const uint8_t *__restrict__ scales, int64_t plane_rows,
                                                        int64_t n, int64_t k, typename D::T *__restrict__ out,
                                                        int64_t ld) {
    const int lane = threadIdx.x & 15;
    const int64_t row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    const int64_t p = blockIdx.y;
    if (row >= n) return;
    const int64_t at = p * plane_rows + row;
    const uint32_t c = *reinterpret_cast<const uint32_t *>(codes + at * 64 + lane * 4);
    const uint32_t s = scales[at * 4 + (lane >> 2)];
    const int64_t j = p * kPlane + lane * 8;
    typename D::T *o = out + row * ld + j;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (j + i < k) o[i] = D::down(from_code((c >> (4 * i)) & 15u, s));
}

// ------------------------------------------------------------------ product
struct Epilogue {
    const float *bias;
    float alpha;
    int act;
};
__device__ __forceinline__ float finish(float acc, float bias, const Epilogue &e) {
    float y = fmaf(e.alpha, acc, bias);
    if (e.act == LIRA_ACT_RELU) y = y < 0.0f ? 0.0f : y;  // (NaN stays NaN)
    if (e.act == LIRA_ACT_SIGMOID) y = 1.0f / (1.0f + __expf(-y));
    return y;
}

// A wave computes 16 columns (rows of W) x 16 rows of the output; fragments straight from memory.
template <class D>
__global__ __launch_bounds__(256) void k_mx4_product(const uint8_t *__restrict__ ac, const uint8_t *__restrict__ as,
                                                     int64_t a_rows, int64_t m, const uint8_t *__restrict__ bc,
                                                     const uint8_t *__restrict__ bs, int64_t b_rows, int64_t n,
                                                     int planes, Epilogue ep, typename D::T *__restrict__ out,
                                                     int64_t ldo) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int64_t n0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 16, m0 = (int64_t)blockIdx.y * 16;
    if (n0 >= n) return;
    const int64_t ar = min(m0 + r, m - 1), br = min(n0 + r, n - 1);
    f32x4 acc = {0, 0, 0, 0};
    for (int p = 0; p < planes; ++p) {
        const i32x4 a = *reinterpret_cast<const i32x4 *>(ac + ((int64_t)p * a_rows + ar) * 64 + g * 16);
        const i32x4 b = *reinterpret_cast<const i32x4 *>(bc + ((int64_t)p * b_rows + br) * 64 + g * 16);
        const int sa = as[((int64_t)p * a_rows + ar) * 4 + g], sb = bs[((int64_t)p * b_rows + br) * 4 + g];
        const i32x8 A = {a.x, a.y, a.z, a.w, 0, 0, 0, 0}, B = {b.x, b.y, b.z, b.w, 0, 0, 0, 0};
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(B, A, acc, 4, 4, 0, sb, 0, sa);
    }
    // lane l: output row m0 + l % 16, columns n0 + 4 (l / 16) ..
    if (m0 + r >= m) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t c = n0 + g * 4 + i;
        if (c < n) out[(m0 + r) * ldo + c] = D::down(finish(acc[i], ep.bias ? ep.bias[c] : 0.0f, ep));
    }
}

// ---------------------------------------------------------------- launchers
static bool dtype_ok(int dtype) { return dtype >= LIRA_DTYPE_F32 && dtype <= LIRA_DTYPE_F16; }
static int64_t planes_of(int64_t k) { return (k + kPlane - 1) / kPlane; }
static int check_packed(const void *codes, const void *scales, int64_t rows, int64_t plane_rows, int64_t k) {
    if (rows < 0 || k <= 0) return fail(LIRA_EINVAL, "rows must be >= 0 and k >= 1");
    if (plane_rows < rows) return fail(LIRA_EINVAL, "plane_rows must be at least the number of rows");
    if (planes_of(k) > 65535) return fail(LIRA_EUNSUPPORTED, "k must be at most 8388480");
    if (rows > 0 && (!codes || !scales)) return fail(LIRA_EINVAL, "NULL buffer");
    if (((uintptr_t)codes & 15) != 0 || ((uintptr_t)scales & 3) != 0)
        return fail(LIRA_EINVAL, "codes must be 16-byte and scales 4-byte aligned");
    return LIRA_OK;
}
static int check_grid(int64_t blocks, const char *what) {
    return blocks > INT32_MAX ? fail(LIRA_EUNSUPPORTED, std::string(what) + ": too many rows for one launch") : LIRA_OK;
}

template <class D>
static int quantize(const void *x, int64_t n, int64_t k, int64_t ld, uint8_t *codes, uint8_t *scales,
                    int64_t plane_rows, hipStream_t st) {
    typedef typename D::T T;
    const bool vec = ((uintptr_t)x & 15) == 0 && (ld * sizeof(T)) % 16 == 0;
    const dim3 g((unsigned)((n + 15) / 16), (unsigned)planes_of(k));
    if (vec)
        hipLaunchKernelGGL((k_mx4_quantize<D, true>), g, dim3(256), 0, st, (const T *)x, n, k, ld, codes, scales,
                           plane_rows);
    else
        hipLaunchKernelGGL((k_mx4_quantize<D, false>), g, dim3(256), 0, st, (const T *)x, n, k, ld, codes, scales,
                           plane_rows);
    LIRA_HIP_TRY(hipGetLastError());
    return LIRA_OK;
}

template <class D>
static int product(const uint8_t *ac, const uint8_t *as, int64_t a_rows, int64_t m, const uint8_t *bc,
                   const uint8_t *bs, int64_t b_rows, int64_t n, int64_t k, const Epilogue &ep, void *out, int64_t ldo,
                   hipStream_t st) {
    const dim3 g((unsigned)((n + 63) / 64), (unsigned)((m + 15) / 16));
    hipLaunchKernelGGL((k_mx4_product<D>), g, dim3(256), 0, st, ac, as, a_rows, m, bc, bs, b_rows, n,
                       (int)planes_of(k), ep, (typename D::T *)out, ldo);
    LIRA_HIP_TRY(hipGetLastError());
    return LIRA_OK;
}

static int check_product(int64_t m, int64_t n, int act, const void *out, int out_dtype, int64_t ldo) {
    if (!dtype_ok(out_dtype)) return fail(LIRA_EINVAL, "unknown dtype");
    if (act < LIRA_ACT_NONE || act > LIRA_ACT_SIGMOID) return fail(LIRA_EINVAL, "unknown activation");
    if (ldo < n) return fail(LIRA_EINVAL, "ldo must be at least n");
    if (m > 0 && n > 0 && !out) return fail(LIRA_EINVAL, "NULL buffer");
    if ((m + 15) / 16 > 65535) return fail(LIRA_EUNSUPPORTED, "m must be at most 1048560");
    return check_grid((n + 63) / 64, "product");
}

}  // namespace lira

using namespace lira;

extern "C" {

int lira_mx4_quantize(const void *x, int dtype, int64_t n, int64_t k, int64_t ld, uint8_t *codes, uint8_t *scales,
                      int64_t plane_rows, void *stream) {
    if (!dtype_ok(dtype)) return fail(LIRA_EINVAL, "unknown dtype");
    if (int rc = check_packed(codes, scales, n, plane_rows, k)) return rc;
    if (ld < k) return fail(LIRA_EINVAL, "ld must be at least k");
    if (n == 0) return LIRA_OK;
    if (!x) return fail(LIRA_EINVAL, "NULL buffer");
    if (int rc = check_grid((n + 15) / 16, "mx4_quantize")) return rc;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == LIRA_DTYPE_F32) return quantize<F32>(x, n, k, ld, codes, scales, plane_rows, st);
    if (dtype == LIRA_DTYPE_BF16) return quantize<BF16>(x, n, k, ld, codes, scales, plane_rows, st);
    return quantize<F16>(x, n, k, ld, codes, scales, plane_rows, st);
}

int lira_mx4_dequantize(const uint8_t *codes, const uint8_t *scales, int64_t plane_rows, int64_t n, int64_t k,
                        void *out, int dtype, int64_t ld, void *stream) {
    if (!dtype_ok(dtype)) return fail(LIRA_EINVAL, "unknown dtype");
    if (int rc = check_packed(codes, scales, n, plane_rows, k)) return rc;
    if (ld < k) return fail(LIRA_EINVAL, "ld must be at least k");
    if (n == 0) return LIRA_OK;
    if (!out) return fail(LIRA_EINVAL, "NULL buffer");
    if (int rc = check_grid((n + 15) / 16, "mx4_dequantize")) return rc;
    hipStream_t st = (hipStream_t)stream;
    const dim3 g((unsigned)((n + 15) / 16), (unsigned)planes_of(k));
    if (dtype == LIRA_DTYPE_F32)
        hipLaunchKernelGGL((k_mx4_dequantize<F32>), g, dim3(256), 0, st, codes, scales, plane_rows, n, k, (float *)out,
                           ld);
    else if (dtype == LIRA_DTYPE_BF16)
        hipLaunchKernelGGL((k_mx4_dequantize<BF16>), g, dim3(256), 0, st, codes, scales, plane_rows, n, k,
                           (__bf16 *)out, ld);
    else
        hipLaunchKernelGGL((k_mx4_dequantize<F16>), g, dim3(256), 0, st, codes, scales, plane_rows, n, k,
                           (_Float16 *)out, ld);
    LIRA_HIP_TRY(hipGetLastError());
    return LIRA_OK;
}

int lira_mx4_matmul(const uint8_t *a_codes, const uint8_t *a_scales, int64_t a_plane_rows, int64_t m,
                    const uint8_t *b_codes, const uint8_t *b_scales, int64_t b_plane_rows, int64_t n, int64_t k,
                    float alpha, const float *bias, int act, void *out, int out_dtype, int64_t ldo, void *stream) {
    if (int rc = check_packed(a_codes, a_scales, m, a_plane_rows, k)) return rc;
    if (int rc = check_packed(b_codes, b_scales, n, b_plane_rows, k)) return rc;
    if (int rc = check_product(m, n, act, out, out_dtype, ldo)) return rc;
    if (m == 0 || n == 0) return LIRA_OK;
    hipStream_t st = (hipStream_t)stream;
    const Epilogue ep = {bias, alpha, act};
    if (out_dtype == LIRA_DTYPE_F32)
        return product<F32>(a_codes, a_scales, a_plane_rows, m, b_codes, b_scales, b_plane_rows, n, k, ep, out, ldo, st);
    if (out_dtype == LIRA_DTYPE_BF16)
        return product<BF16>(a_codes, a_scales, a_plane_rows, m, b_codes, b_scales, b_plane_rows, n, k, ep, out, ldo,
                             st);
    return product<F16>(a_codes, a_scales, a_plane_rows, m, b_codes, b_scales, b_plane_rows, n, k, ep, out, ldo, st);
}

int lira_mx4_linear_workspace_size(int64_t m, int64_t n, int64_t k, size_t *bytes) {
    if (!bytes) return fail(LIRA_EINVAL, "NULL buffer");
    if (m < 0 || n < 0 || k <= 0) return fail(LIRA_EINVAL, "bad shape");
    *bytes = m == 0 || n == 0 ? 0 : (size_t)(planes_of(k) * m * 68);
    return LIRA_OK;
}

int lira_mx4_linear(const void *x, int dtype, int64_t m, int64_t k, int64_t ldx, const uint8_t *b_codes,
                    const uint8_t *b_scales, int64_t b_plane_rows, int64_t n, float alpha, const float *bias, int act,
                    void *out, int out_dtype, int64_t ldo, void *workspace, size_t workspace_bytes, void *stream) {
    if (!dtype_ok(dtype)) return fail(LIRA_EINVAL, "unknown dtype");
    if (int rc = check_packed(b_codes, b_scales, n, b_plane_rows, k)) return rc;
    if (m < 0) return fail(LIRA_EINVAL, "bad shape");
    if (ldx < k) return fail(LIRA_EINVAL, "ldx must be at least k");
    if (int rc = check_product(m, n, act, out, out_dtype, ldo)) return rc;
    if (m == 0 || n == 0) return LIRA_OK;
    if (!x) return fail(LIRA_EINVAL, "NULL buffer");
    size_t need = 0;
    if (int rc = lira_mx4_linear_workspace_size(m, n, k, &need)) return rc;
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15) != 0))
        return fail(LIRA_EINVAL, "workspace too small (lira_mx4_linear_workspace_size) or not 16-byte aligned");
    uint8_t *ac = (uint8_t *)workspace, *as = ac + planes_of(k) * m * 64;
    if (int rc = lira_mx4_quantize(x, dtype, m, k, ldx, ac, as, m, stream)) return rc;
    return lira_mx4_matmul(ac, as, m, m, b_codes, b_scales, b_plane_rows, n, k, alpha, bias, act, out, out_dtype, ldo,
                           stream);
}

}  // extern "C"
