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
// alpha acc + bias and the activation, in place
template <int N>
__device__ __forceinline__ void finish(f32x4 (&acc)[N], f32x4 bias, const Epilogue &e) {
#pragma unroll
    for (int j = 0; j < N; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] = fmaf(e.alpha, acc[j][i], bias[i]);
    if (e.act == LIRA_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[j][i] = acc[j][i] < 0.0f ? 0.0f : acc[j][i];  // (NaN stays NaN)
    } else if (e.act == LIRA_ACT_SIGMOID) {
        // (hardware exp2 and reciprocal: 2 ulp of the exponent's rounding and 1 of the quotient's, under 2^-20)
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                acc[j][i] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(acc[j][i] * -1.44269504088896340736f));
    }
}
// 4 columns of the bias, 0 where there is none
__device__ __forceinline__ f32x4 bias4(const Epilogue &e, int64_t col, int64_t n) {
    f32x4 b = {0, 0, 0, 0};
    if (e.bias) {
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = col + i < n ? e.bias[col + i] : 0.0f;
    }
    return b;
}
template <class D>
struct alignas(4 * sizeof(typename D::T)) Four {
    typename D::T v[4];
};
// 4 columns of one output row, rounded: in one store (aligned), or those of them that there are
template <class D>
__device__ __forceinline__ void store4(typename D::T *at, f32x4 y) {
    Four<D> o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o.v[i] = D::down(y[i]);
    *reinterpret_cast<Four<D> *>(at) = o;
}
template <class D>
__device__ __forceinline__ void store_some(typename D::T *at, f32x4 y, int64_t left) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < left) at[i] = D::down(y[i]);
}

// LDS-DMA: lane l's `bytes` (16 or 4) at sbase + voff -> LDS byte lds + l * bytes.  Inline asm: hipcc
// would wait for every DMA in flight before each LDS read (it cannot tell their places apart);
// the pipeline below waits by count.  No register is written but M0, which is restored.
__device__ __forceinline__ void dma16(uint32_t lds, const uint8_t *sbase, uint32_t voff) {
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "s"(lds), "v"(voff), "s"(sbase)
                 : "memory");
}
__device__ __forceinline__ void dma4(uint32_t lds, const uint8_t *sbase, uint32_t voff) {
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %2, %3\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "s"(lds), "v"(voff), "s"(sbase)
                 : "memory");
}
template <int N>
__device__ __forceinline__ void wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// a row's 4 blocks of a plane sit in LDS at 16-byte slots (block ^ turn(row)): the 16 rows that a
// fragment read touches at one block then fall on different banks
__device__ __forceinline__ uint32_t turn(uint32_t row) { return ((row >> 2) & 1u) | ((((row >> 1) ^ (row >> 3)) & 1u) << 1); }

struct Product {
    const uint8_t *ac, *as;  // rows of the output (m)
    const uint8_t *bc, *bs;  // columns of the output (n)
    int64_t a_rows, b_rows, m, n, ldo;
    int planes;
    Epilogue ep;
    void *out;
};

// The tile kernel: TN columns x TM rows of the output, WN x WM waves of 64 lanes.  Planes of 128
// elements stream through kSlots LDS slots by LDS-DMA; a wave reads plane s + 1's fragments while
// the matrix instructions of plane s run, so both come from registers.
template <int TN, int TM, int WN, int WM, class D>
struct Tile {
    static constexpr int NW = WN * WM, FN = TN / WN / 16, FM = TM / WM / 16;
    static constexpr int kSlots = 4;
    static constexpr int kSlotBytes = (TN + TM) * 68;
    static constexpr int kCodeLoads = (TN + TM) / 16 / NW;                        // per wave and plane
    static constexpr int kScaleJobs = (TN + 63) / 64 + (TM + 63) / 64;            // of 64 rows
    static constexpr int kScaleLoads = (kScaleJobs + NW - 1) / NW;                // (some waves repeat one)
    static constexpr int kLoads = kCodeLoads + kScaleLoads;
    static constexpr int kBytes = kSlots * kSlotBytes;
    static_assert((TN + TM) / 16 % NW == 0, "whole loads per wave");

    struct Frags {
        i32x4 b[FN], a[FM];
        int sb[FN], sa[FM];
    };
};

template <int TN, int TM, int WN, int WM, class D>
__global__ __launch_bounds__(WN *WM * 64) void k_mx4_tile(Product P, int tiles_n, int tiles_m) {
    typedef Tile<TN, TM, WN, WM, D> C;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wn = w % WN, wm = w / WN;

    // Workgroups go to the 8 XCDs in turn: each XCD takes a run of tiles of its own, 8 tiles of rows
    // by as many of columns, so that the tiles in flight on it share their operands in its L2.
    const int64_t tiles = (int64_t)tiles_n * tiles_m;
    int64_t t = blockIdx.x;
    {
        const int64_t per = tiles / 8, rest = tiles % 8, x = t % 8;
        t = x * per + (x < rest ? x : rest) + t / 8;
    }
    const int64_t band = t / (8 * (int64_t)tiles_n), in = t % (8 * (int64_t)tiles_n);
    const int hb = (int)min((int64_t)8, tiles_m - band * 8);
    const int64_t m0 = (band * 8 + in % hb) * TM, n0 = in / hb * TN;

    const uint32_t lds = (uint32_t)(uintptr_t)smem;
    // this wave's loads of a plane: 16 rows each, codes first
    const uint8_t *cb = P.bc + n0 * 64, *ca = P.ac + m0 * 64, *sb = P.bs + n0 * 4, *sa = P.as + m0 * 4;
    const int64_t bstep = P.b_rows * 64, astep = P.a_rows * 64;
    const uint32_t nlast = (uint32_t)(min(P.n - n0, (int64_t)TN) - 1), mlast = (uint32_t)(min(P.m - m0, (int64_t)TM) - 1);
    uint32_t off[C::kCodeLoads], soff[C::kScaleLoads];
#pragma unroll
    for (int i = 0; i < C::kCodeLoads; ++i) {
        const uint32_t row = (uint32_t)((i * C::NW + w) * 16 + (lane >> 2));  // of the TN + TM rows
        const bool bside = (i * C::NW + w) * 16 < TN;
        const uint32_t rr = bside ? min(row, nlast) : min(row - TN, mlast);
        off[i] = rr * 64 + (((uint32_t)lane & 3u) ^ turn(row)) * 16;
    }
#pragma unroll
    for (int i = 0; i < C::kScaleLoads; ++i) {
        const int job = (i * C::NW + w) % C::kScaleJobs;
        constexpr int nb = (TN + 63) / 64;
        soff[i] = job < nb ? min((uint32_t)(job * 64 + lane), nlast) * 4 : min((uint32_t)((job - nb) * 64 + lane), mlast) * 4;
    }
    auto fetch = [&](int p, int slot) {
        const uint32_t base = lds + slot * C::kSlotBytes;
        const uint8_t *pb = cb + p * bstep, *pa = ca + p * astep;
#pragma unroll
        for (int i = 0; i < C::kCodeLoads; ++i) {
            const int rows = (i * C::NW + w) * 16;
            dma16(base + rows * 64, rows < TN ? pb : pa, off[i]);
        }
        const uint8_t *qb = sb + p * (bstep >> 4), *qa = sa + p * (astep >> 4);
#pragma unroll
        for (int i = 0; i < C::kScaleLoads; ++i) {
            const int job = (i * C::NW + w) % C::kScaleJobs;
            constexpr int nb = (TN + 63) / 64;
            dma4(base + (TN + TM) * 64 + (job < nb ? job * 256 : TN * 4 + (job - nb) * 256), job < nb ? qb : qa, soff[i]);
        }
    };
    const uint32_t frag_row = (uint32_t)r * 64 + (((uint32_t)g ^ turn((uint32_t)r)) * 16);
    auto read = [&](int slot, typename C::Frags &f) {
        const uint8_t *base = smem + slot * C::kSlotBytes;
        const uint8_t *fb = base + wn * (TN / WN) * 64 + frag_row, *fa = base + (TN + wm * (TM / WM)) * 64 + frag_row;
        const uint8_t *zb = base + (TN + TM) * 64 + wn * (TN / WN) * 4 + r * 4 + g;
        const uint8_t *za = base + (TN + TM) * 64 + TN * 4 + wm * (TM / WM) * 4 + r * 4 + g;
#pragma unroll
        for (int i = 0; i < C::FN; ++i) f.b[i] = *reinterpret_cast<const i32x4 *>(fb + i * 1024), f.sb[i] = zb[i * 64];
#pragma unroll
        for (int i = 0; i < C::FM; ++i) f.a[i] = *reinterpret_cast<const i32x4 *>(fa + i * 1024), f.sa[i] = za[i * 64];
    };
    f32x4 acc[C::FN][C::FM];
#pragma unroll
    for (int i = 0; i < C::FN; ++i)
#pragma unroll
        for (int j = 0; j < C::FM; ++j) acc[i][j] = (f32x4){0, 0, 0, 0};
    auto multiply = [&](const typename C::Frags &f) {
#pragma unroll
        for (int j = 0; j < C::FM; ++j)
#pragma unroll
            for (int i = 0; i < C::FN; ++i) {
                const i32x8 B = {f.b[i].x, f.b[i].y, f.b[i].z, f.b[i].w, 0, 0, 0, 0};
                const i32x8 A = {f.a[j].x, f.a[j].y, f.a[j].z, f.a[j].w, 0, 0, 0, 0};
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(B, A, acc[i][j], 4, 4, 0, f.sb[i], 0, f.sa[j]);
            }
    };
    const int planes = P.planes;
    // before plane s is read: its loads have landed (those of the two planes after it may be in
    // flight), and every wave has read plane s - 1, whose slot takes plane s + 3
    auto arrive = [&](int s) {
        if (s + 2 < planes)
            wait_vm<2 * C::kLoads>();
        else if (s + 1 < planes)
            wait_vm<C::kLoads>();
        else
            wait_vm<0>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (s + 3 < planes) fetch(s + 3, (s + 3) % C::kSlots);
    };
    for (int p = 0; p < 3 && p < planes; ++p) fetch(p, p);
    for (int s = 0; s < planes; ++s) {
        arrive(s);
        typename C::Frags f;
        read(s % C::kSlots, f);
        multiply(f);
    }

    // lane l of a fragment: output row l % 16, columns 4 (l / 16) ..
    typedef typename D::T T;
    const int64_t row0 = m0 + wm * (TM / WM) + r, col0 = n0 + wn * (TN / WN) + g * 4;
    T *out = (T *)P.out + row0 * P.ldo + col0;
    const bool whole = m0 + TM <= P.m && n0 + TN <= P.n && ((uintptr_t)P.out & (sizeof(Four<D>) - 1)) == 0 && P.ldo % 4 == 0;
#pragma unroll
    for (int i = 0; i < C::FN; ++i) {
        finish(acc[i], bias4(P.ep, col0 + i * 16, P.n), P.ep);
        if (whole) {
#pragma unroll
            for (int j = 0; j < C::FM; ++j) store4<D>(out + j * 16 * P.ldo + i * 16, acc[i][j]);
        } else {
#pragma unroll
            for (int j = 0; j < C::FM; ++j)
                if (row0 + j * 16 < P.m) store_some<D>(out + j * 16 * P.ldo + i * 16, acc[i][j], P.n - (col0 + i * 16));
        }
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

template <int TN, int TM, int WN, int WM, class D>
static int launch_tile(const Product &p, hipStream_t st) {
    typedef Tile<TN, TM, WN, WM, D> C;
    static std::atomic<uint64_t> latch{0};
    const void *fn = (const void *)&k_mx4_tile<TN, TM, WN, WM, D>;
    LIRA_HIP_TRY(set_smem_attr_once(latch, fn, C::kBytes));
    const int64_t tn = (p.n + TN - 1) / TN, tm = (p.m + TM - 1) / TM;
    if (tn * tm > INT32_MAX) return fail(LIRA_EUNSUPPORTED, "product: too many tiles for one launch");
    hipLaunchKernelGGL((k_mx4_tile<TN, TM, WN, WM, D>), dim3((unsigned)(tn * tm)), dim3(WN * WM * 64), C::kBytes, st, p,
                       (int)tn, (int)tm);
    LIRA_HIP_TRY(hipGetLastError());
    return LIRA_OK;
}

template <class D>
static int product(const Product &p, hipStream_t st) {
    const int64_t big = ((p.n + 255) / 256) * ((p.m + 255) / 256), mid = ((p.n + 127) / 128) * ((p.m + 127) / 128);
    if (big >= 256) return launch_tile<256, 256, 2, 4, D>(p, st);
    if (mid >= 256) return launch_tile<128, 128, 2, 2, D>(p, st);
    return launch_tile<64, 64, 2, 2, D>(p, st);
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
    const Product p = {a_codes, a_scales, b_codes, b_scales, a_plane_rows, b_plane_rows, m, n, ldo,
                       (int)planes_of(k), {bias, alpha, act}, out};
    if (out_dtype == LIRA_DTYPE_F32) return product<F32>(p, st);
    if (out_dtype == LIRA_DTYPE_BF16) return product<BF16>(p, st);
    return product<F16>(p, st);
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
