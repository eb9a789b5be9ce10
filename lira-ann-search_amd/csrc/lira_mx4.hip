// lira_mx4.hip -- microscaled 4-bit floats: packing, unpacking and the product on the matrix
// cores (layout and format: lira_mx4.hpp).
#include <algorithm>
#include <string>
#include <type_traits>

#include "lira_internal.hpp"
#include "lira_mx4.hpp"

namespace lira {

static constexpr int kPlane = 128;  // elements per plane

// ------------------------------------------------------------ pack / unpack
// 16 lanes per (row, plane), 8 elements each; the block's largest magnitude crosses its 4
// lanes by DPP.  A wave packs 4 consecutive rows: 256 bytes of codes and 16 of scales.
template <class D, bool VEC, bool ONCE>
__global__ __launch_bounds__(256) void k_mx4_quantize(const typename D::T *__restrict__ x, int64_t n, int64_t k,
                                                      int64_t ld, uint8_t *__restrict__ codes,
                                                      uint8_t *__restrict__ scales, int64_t plane_rows) {
    const int lane = threadIdx.x & 15;
    const int64_t row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    const int64_t p = blockIdx.y;
    const bool live = row < n;
    float v[8];
    load_run<D, VEC, 8, ONCE>(x + (live ? row : 0) * ld, p * kPlane + lane * 8, k, v);
    const uint32_t s = scale_code(quad_max(v));
    const uint32_t c = s == 255 ? 0u : to_codes(v, scale_operand(s));
    if (!live) return;
    const int64_t at = p * plane_rows + row;
    *reinterpret_cast<uint32_t *>(codes + at * 64 + lane * 4) = c;
    if ((lane & 3) == 0) scales[at * 4 + (lane >> 2)] = (uint8_t)s;
}

// A lane unpacks the E elements of one 16-byte store, so that a row's lanes write one run; a plane
// takes 128 / E lanes.
template <class D, bool VEC>
__global__ __launch_bounds__(256) void k_mx4_dequantize(const uint8_t *__restrict__ codes,
                                                        const uint8_t *__restrict__ scales, int64_t plane_rows,
                                                        int64_t n, int64_t k, typename D::T *__restrict__ out,
                                                        int64_t ld) {
    typedef typename D::T T;
    constexpr int E = 16 / sizeof(T), L = kPlane / E;
    const int lane = threadIdx.x % L;
    const int64_t row = (int64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
    const int64_t p = blockIdx.y;
    if (row >= n) return;
    const int64_t at = p * plane_rows + row;
    uint32_t c;
    if (E == 8)
        c = *reinterpret_cast<const uint32_t *>(codes + at * 64 + lane * 4);
    else
        c = *reinterpret_cast<const uint16_t *>(codes + at * 64 + lane * 2);
    const uint32_t s = scales[at * 4 + lane * E / 32];
    struct alignas(16) V {
        T e[E];
    } o;
    float v[E];
    from_codes<E>(c, s, v);
#pragma unroll
    for (int i = 0; i < E; ++i) o.e[i] = D::down(v[i]);
    const int64_t j = p * kPlane + lane * E;
    T *q = out + row * ld + j;
    if (VEC && j + E <= k) {
        stream16(q, *reinterpret_cast<const i32x4 *>(&o));
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (j + i < k) q[i] = o.e[i];
    }
}

// ------------------------------------------------------------------ product
struct Epilogue {
    const float *bias;
    float alpha;
    int act;
    bool bias16;  // whole runs of 4: aligned, and n a multiple of 4
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
        // (hardware exp2 and reciprocal, 1 ulp each, and the exponent's rounding, which grows with the argument x: off by
        // (1.5 |x| + 4) 2^-24 of the value, which is under 2^-21 absolutely, and 2^-17 of the value at x = -80)
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                acc[j][i] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(acc[j][i] * -1.44269504088896340736f));
    }
}
// 4 columns of the bias, 0 where there is none (past the end the last one's: not stored)
__device__ __forceinline__ f32x4 bias4(const Epilogue &e, int64_t col, int64_t n) {
    f32x4 b = {0, 0, 0, 0};
    if (e.bias16) {
        b = *reinterpret_cast<const f32x4 *>(e.bias + min(col, n - 4));
    } else if (e.bias) {
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = e.bias[min(col + i, n - 1)];
    }
    return b;
}
template <class D>
struct alignas(4 * sizeof(typename D::T)) Four {
    typename D::T v[4];
};
// 4 columns of one output row, rounded and stored (aligned)
template <class D>
__device__ __forceinline__ void store4(typename D::T *at, f32x4 y) {
    Four<D> o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o.v[i] = D::down(y[i]);
    *reinterpret_cast<Four<D> *>(at) = o;
}
// the same at any alignment, or the first `left` of them
template <class D>
__device__ __forceinline__ void store_run(typename D::T *at, f32x4 y, int64_t left) {
    Four<D> o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o.v[i] = D::down(y[i]);
    if (left >= 4) {
        __builtin_memcpy(at, &o, sizeof(o));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < left) at[i] = o.v[i];
    }
}

// LDS-DMA: lane l's `bytes` (16 or 4) at sbase + voff -> LDS byte lds + l * bytes.  Inline asm: hipcc
// would wait for every DMA in flight before each LDS read (it cannot tell their places apart);
// the pipeline below waits by count.  No register is written but M0, which is restored.
__device__ __forceinline__ const uint8_t *scalar(const uint8_t *p) {  // (the same in every lane)
    const uint64_t v = (uint64_t)p;
    return (const uint8_t *)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 |
                             (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}
__device__ __forceinline__ void dma16(uint32_t lds, const uint8_t *sbase, uint32_t voff) {
    uint32_t keep;
    sbase = scalar(sbase);
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "s"(lds), "v"(voff), "s"(sbase)
                 : "memory");
}
__device__ __forceinline__ void dma4(uint32_t lds, const uint8_t *sbase, uint32_t voff) {
    uint32_t keep;
    sbase = scalar(sbase);
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %2, %3\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "s"(lds), "v"(voff), "s"(sbase)
                 : "memory");
}
template <int N>
__device__ __forceinline__ void wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// A row's 4 blocks of a plane sit in LDS at 16-byte places (block ^ turn(row)).  An LDS read of 16 bytes a lane
// takes 16 lanes at a time over the 64 banks, lanes 0-3, 12-15, 20-27 first, then 4-11, 16-19,
// 28-31, and the upper half alike (measured): with this turn no two of them are on one bank.
__device__ __forceinline__ uint32_t turn(uint32_t row) { return (row >> 1) & 3u; }

struct Product {
    const uint8_t *ac, *as;  // rows of the output (m)
    const uint8_t *bc, *bs;  // columns of the output (n)
    int64_t a_rows, b_rows, m, n, ldo;
    int planes;
    Epilogue ep;
    void *out;
};

// W's fragment x the rows' fragment + acc: lane l holds block l / 16 of row l % 16.  (The 32 x 32 x 64 form
// has 1.4 times the rate by itself, 7.8 against 5.7 PFLOP/s, but the kernel around it is bound by its
// loads: 8192^3 0.30 ms with it, 0.29 so.)
__device__ __forceinline__ i32x8 wide(i32x4 v) { return (i32x8){v.x, v.y, v.z, v.w, 0, 0, 0, 0}; }
__device__ __forceinline__ f32x4 mfma(i32x4 b, int sb, i32x4 a, int sa, f32x4 acc) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wide(b), wide(a), acc, 4, 4, 0, sb, 0, sa);
}

// The tile kernel: TN columns x TM rows of the output by WN x WM x WK waves.  Planes of 128 elements
// stream through SLOTS LDS slots of PS planes by LDS-DMA, all slots but one in flight.  The WN x WM
// waves split the tile; where a tile is small, WK such sets of waves split a slot's planes (there
// is one barrier a slot, and a set's LDS reads and matrix instructions wait for each
// other: with more sets, less of that is left bare) and join their sums in LDS in a fixed order.
// PACK: the rows come as they are and are packed into their places by the workgroup itself, all planes (no more than
// there are slots) before the first product: a launch and the packed rows' way through memory less.
template <int TN, int TM, int WN, int WM, int WK, int SLOTS, int PS, bool PACK = false>
struct Tile {
    static constexpr int NW = WN * WM * WK, FN = TN / WN / 16, FM = TM / WM / 16;
    static constexpr int kNb = (TN + 63) / 64, kNa = (TM + 63) / 64;
    static constexpr int kCodeJobs = (TN + (PACK ? 0 : TM)) / 16;  // of 16 rows, a plane
    static constexpr int kScaleJobs = kNb + (PACK ? 0 : kNa);      // of up to 64 rows, a plane
    // per wave and slot (every wave makes the same number, so that it can wait by count: one without
    // a job of its own repeats another's)
    static constexpr int kCodeLoads = (kCodeJobs * PS + NW - 1) / NW, kScaleLoads = (kScaleJobs * PS + NW - 1) / NW;
    static constexpr int kLoads = kCodeLoads + kScaleLoads;
    // a plane of a slot: the codes of both sides, then their scales, 256 bytes a job (a side under 64 rows
    // fills its job's lanes by repeating its last row)
    static constexpr int kScaleAt = (TN + TM) * 64, kPlaneBytes = kScaleAt + (kNb + kNa) * 256;
    static constexpr int kBytes = SLOTS * PS * kPlaneBytes;
    // LDS that the sets' sums, or the rows on their way out (16 a wave, 16 bytes apart), take in the slots' place
    template <class D>
    static constexpr int epilogue_bytes() {
        return WK > 1 ? NW * FN * FM * 1024 : NW * 16 * (TN / WN * (int)sizeof(typename D::T) + 16);
    }
    static_assert(PS % WK == 0, "the sets split a slot's planes evenly");
    static_assert(!PACK || (PS == 1 && WK == 1), "packed rows: slot s is plane s");

    struct Frags {
        i32x4 b[FN], a[FM];
        int sb[FN], sa[FM];
    };
};

struct Rows {
    const void *x;  // (m, k), row stride ldx
    int64_t k, ldx;
    bool vec;  // first element and row stride are multiples of 16 bytes
};
// X: void, or the type of the rows that the tile packs
template <int TN, int TM, int WN, int WM, int WK, int SLOTS, int PS, class D, class X = void>
__global__ __launch_bounds__(WN *WM *WK * 64) void k_mx4_tile(Product P, Rows R, int tiles_n, int tiles_m) {
    constexpr bool PACK = !std::is_void<X>::value;
    typedef Tile<TN, TM, WN, WM, WK, SLOTS, PS, PACK> C;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wn = w % WN, wm = w / WN % WM, wk = w / (WN * WM);

    // Workgroups go to the 8 XCDs in turn: each XCD takes a run of tiles of its own, 4 tiles of rows
    // high, so that the tiles in flight on it share their operands in its L2 (8192^3, us: 328; 8 high 333;
    // in launch order 341).
    const int64_t tiles = (int64_t)tiles_n * tiles_m;
    int64_t t = blockIdx.x;
    {
        const int64_t per = tiles / 8, rest = tiles % 8, x = t % 8;
        t = x * per + (x < rest ? x : rest) + t / 8;
    }
    const int64_t band = t / (4 * (int64_t)tiles_n), in = t % (4 * (int64_t)tiles_n);
    const int hb = (int)min((int64_t)4, tiles_m - band * 4);
    const int64_t m0 = (band * 4 + in % hb) * TM, n0 = in / hb * TN;

    const uint32_t lds = (uint32_t)(uintptr_t)smem;
    const uint8_t *cb = P.bc + n0 * 64, *ca = P.ac + m0 * 64, *sb = P.bs + n0 * 4, *sa = P.as + m0 * 4;
    const int64_t bstep = P.b_rows * 64, astep = P.a_rows * 64;
    const uint32_t nlast = (uint32_t)(min(P.n - n0, (int64_t)TN) - 1), mlast = (uint32_t)(min(P.m - m0, (int64_t)TM) - 1);
    uint32_t off[C::kCodeLoads], soff[C::kScaleLoads];
#pragma unroll
    for (int i = 0; i < C::kCodeLoads; ++i) {
        const int first = (i * C::NW + w) % (C::kCodeJobs * PS) % C::kCodeJobs * 16;
        const uint32_t row = (uint32_t)(first + (lane >> 2));  // of the TN + TM rows
        const uint32_t rr = first < TN ? min(row, nlast) : min(row - TN, mlast);
        off[i] = rr * 64 + (((uint32_t)lane & 3u) ^ turn(row)) * 16;
    }
#pragma unroll
    for (int i = 0; i < C::kScaleLoads; ++i) {
        const int job = (i * C::NW + w) % (C::kScaleJobs * PS) % C::kScaleJobs;
        soff[i] = job < C::kNb ? min((uint32_t)(job * 64 + lane), nlast) * 4
                               : min((uint32_t)((job - C::kNb) * 64 + lane), mlast) * 4;
    }
    const int planes = P.planes, steps = (planes + PS - 1) / PS;
    auto fetch = [&](int s) {
        const uint32_t base = lds + s % SLOTS * (PS * C::kPlaneBytes);
#pragma unroll
        for (int i = 0; i < C::kCodeLoads; ++i) {
            const int job = (i * C::NW + w) % (C::kCodeJobs * PS), q = job / C::kCodeJobs, rows = job % C::kCodeJobs * 16;
            const int64_t p = PS == 1 ? s : min(s * PS + q, planes - 1);  // (past the end: any plane, not multiplied)
            dma16(base + q * C::kPlaneBytes + rows * 64, rows < TN ? cb + p * bstep : ca + p * astep, off[i]);
        }
#pragma unroll
        for (int i = 0; i < C::kScaleLoads; ++i) {
            const int all = (i * C::NW + w) % (C::kScaleJobs * PS), q = all / C::kScaleJobs, job = all % C::kScaleJobs;
            const int64_t p = PS == 1 ? s : min(s * PS + q, planes - 1);
            dma4(base + q * C::kPlaneBytes + C::kScaleAt + job * 256,
                 job < C::kNb ? sb + p * (bstep >> 4) : sa + p * (astep >> 4), soff[i]);
        }
    };
    const uint32_t turned = ((uint32_t)g ^ turn((uint32_t)r)) * 16;
    auto read = [&](int at, typename C::Frags &f) {
        const uint8_t *base = smem + at * C::kPlaneBytes;
        const uint8_t *fb = base + (wn * (TN / WN) + r) * 64 + turned, *fa = base + (TN + wm * (TM / WM) + r) * 64 + turned;
        const uint8_t *zb = base + C::kScaleAt + (wn * (TN / WN) + r) * 4 + g;
        const uint8_t *za = base + C::kScaleAt + C::kNb * 256 + (wm * (TM / WM) + r) * 4 + g;
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
            for (int i = 0; i < C::FN; ++i) acc[i][j] = mfma(f.b[i], f.sb[i], f.a[j], f.sa[j], acc[i][j]);
    };
    // before slot s is read: its loads have landed (those of the slots after it may be in flight),
    // and every wave has read slot s - 1, whose place takes the next one
    constexpr int kAhead = SLOTS - 1;
    static_assert((kAhead - 1) * C::kLoads <= 63, "vmcnt counts to 63");
    auto arrive = [&](int s) {
        const int after = steps - 1 - s;
        if (after >= kAhead - 1)
            wait_vm<(kAhead - 1) * C::kLoads>();
        else if (kAhead > 4 && after >= 3)
            wait_vm<3 * C::kLoads>();
        else if (kAhead > 3 && after == 2)
            wait_vm<2 * C::kLoads>();
        else if (kAhead > 2 && after == 1)
            wait_vm<C::kLoads>();
        else
            wait_vm<0>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (s + kAhead < steps) fetch(s + kAhead);
    };
    for (int s = 0; s < kAhead && s < steps; ++s) fetch(s);
    if constexpr (PACK) {
        // 8 elements a thread at a time, as in k_mx4_rows, a plane's all loaded before the first is packed;
        // the first wait's barrier is behind the last
        constexpr int U = TM * 16 / (C::NW * 64);
        const bool whole = R.vec && R.k % 8 == 0;  // (then a run is all in the row or all behind it, and k >= 8)
        for (int p = 0; p < planes; ++p) {
            const int run = threadIdx.x & 15, block = run >> 2;
            const int64_t at = p * kPlane + run * 8;
            uint8_t *slot = smem + p * C::kPlaneBytes;
            float v[U][8];
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const uint32_t row = i * (C::NW * 4) + (threadIdx.x >> 4);
                const typename X::T *x = (const typename X::T *)R.x + (m0 + min(row, mlast)) * R.ldx;
                if (whole)
                    load_run<X, true, 8>(x, min(at, R.k - 8), R.k, v[i]);
                else
                    load_run<X, false, 8>(x, at, R.k, v[i]);
            }
            if (whole && at >= R.k) {
#pragma unroll
                for (int i = 0; i < U; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[i][e] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const uint32_t row = i * (C::NW * 4) + (threadIdx.x >> 4), z = scale_code(quad_max(v[i]));
                *reinterpret_cast<uint32_t *>(slot + (TN + row) * 64 + ((uint32_t)block ^ turn(row)) * 16 + (run & 3) * 4) =
                    z == 255 ? 0u : to_codes(v[i], scale_operand(z));
                if ((run & 3) == 0) slot[C::kScaleAt + C::kNb * 256 + row * 4 + block] = (uint8_t)z;
            }
        }
    }
    for (int s = 0; s < steps; ++s) {
        arrive(s);
        typename C::Frags f[PS / WK];
#pragma unroll
        for (int q = 0; q < PS / WK; ++q) read(s % SLOTS * PS + q * WK + wk, f[q]);
#pragma unroll
        for (int q = 0; q < PS / WK; ++q)
            if (PS == 1 || s * PS + q * WK + wk < planes) multiply(f[q]);
    }
    if (WK > 1) {
        // set k's sums at [fragment][k]; the sets share the fragments out among themselves
        __syncthreads();  // (every slot has been read)
        f32x4 *red = reinterpret_cast<f32x4 *>(smem) + (w % (WN * WM)) * (C::FN * C::FM * WK * 64) + lane;
#pragma unroll
        for (int i = 0; i < C::FN; ++i)
#pragma unroll
            for (int j = 0; j < C::FM; ++j) red[((i * C::FM + j) * WK + wk) * 64] = acc[i][j];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < C::FN; ++i)
#pragma unroll
            for (int j = 0; j < C::FM; ++j) {
                if ((i * C::FM + j) % WK != wk) continue;
                f32x4 y = red[(i * C::FM + j) * WK * 64];
#pragma unroll
                for (int k = 1; k < WK; ++k) y += red[((i * C::FM + j) * WK + k) * 64];
                acc[i][j] = y;
            }
    }

    // lane l of a fragment: output row l % 16, columns 4 (l / 16) ..
    typedef typename D::T T;
    constexpr int TNw = TN / WN, TMw = TM / WM;
    const int64_t row0 = m0 + wm * TMw, col0 = n0 + wn * TNw;
    if (WK > 1) {
#pragma unroll
        for (int i = 0; i < C::FN; ++i) {
            const int64_t col = col0 + i * 16 + g * 4;
            finish(acc[i], bias4(P.ep, col, P.n), P.ep);
#pragma unroll
            for (int j = 0; j < C::FM; ++j) {
                const int64_t row = row0 + j * 16 + r;
                if ((i * C::FM + j) % WK != wk || row >= P.m) continue;
                store_run<D>((T *)P.out + row * P.ldo + col, acc[i][j], P.n - col);
            }
        }
        return;
    }
    // 16 rows at a time through LDS, a region a wave, so that a wave writes whole runs of a row: straight from
    // the fragments a bf16 store is runs of 32 bytes, 16 rows apart (8192^3 with them 0.35 ms, so 0.29)
    constexpr int E = 16 / sizeof(T), kRow = TNw + E, kUnits = 16 * TNw / E;
    static_assert(WK > 1 || C::NW * 16 * kRow * (int)sizeof(T) == C::template epilogue_bytes<D>(), "a region a wave");
    __syncthreads();  // (every slot has been read)
    T *stage = reinterpret_cast<T *>(smem) + w * (16 * kRow);
#pragma unroll
    for (int i = 0; i < C::FN; ++i) finish(acc[i], bias4(P.ep, col0 + i * 16 + g * 4, P.n), P.ep);
#pragma unroll
    for (int j = 0; j < C::FM; ++j) {
#pragma unroll
        for (int i = 0; i < C::FN; ++i) store4<D>(stage + r * kRow + i * 16 + g * 4, acc[i][j]);
        __builtin_amdgcn_wave_barrier();  // (a wave's LDS operations are in order)
#pragma unroll
        for (int u = 0; u < (kUnits + 63) / 64; ++u) {
            const int at = u * 64 + lane, rr = at / (TNw / E), c = at % (TNw / E) * E;
            const int64_t row = row0 + j * 16 + rr, col = col0 + c;
            if (at < kUnits && row < P.m && col < P.n) {
                const T *v = stage + rr * kRow + c;
                T *o = (T *)P.out + row * P.ldo + col;
                if (col + E <= P.n) {
                    stream16(o, *reinterpret_cast<const i32x4 *>(v));
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        if (col + e < P.n) o[e] = v[e];
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// The few-rows kernel: 16 NB columns of the output x up to 16 rows, a stream over W.  No operand is
// shared between waves, so W goes straight to registers: a wave's load of a fragment is 1 KiB in a row.
// KS waves of a workgroup split the planes and join their sums in LDS in a fixed order.  KS = 1, where there are
// few planes or many columns: four waves, each of its own columns, that go on to the next ones without a gap.  FUSED: the rows of x are
// packed here, 32 elements a thread, while the first planes of W are on their way; else they come
// packed and are read from the cache.
template <class X, class D, int NB, int KS, bool FUSED, bool VEC>
__global__ __launch_bounds__(KS == 1 ? 256 : KS * 64, 4) void k_mx4_rows(Product P, Rows R) {
    constexpr int U = KS == 1 ? 2 : FUSED ? 3 : 4;  // planes in flight
    constexpr int NT = KS == 1 ? 256 : KS * 64;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int planes = P.planes, first = KS == 1 ? 0 : w, m = (int)P.m;
    const int64_t groups = (P.n + 16 * NB - 1) / (16 * NB), step = KS == 1 ? (int64_t)gridDim.x * 4 : groups;
    int64_t group = KS == 1 ? (int64_t)blockIdx.x * 4 + w : blockIdx.x;
    const int64_t bplane = P.b_rows * 64, aplane = P.a_rows * 64;
    const int ao = min(r, m - 1);  // (rows past the end read the last one's place)
    struct Step {
        i32x4 b[NB], a;
        int sb[NB], sa;
        f32x4 bias[NB];  // (KS = 1, with a group's last plane: a load of its own would wait for those ahead of it)
    } f[U];
    const int stride = FUSED ? planes * 64 + 16 : 0;  // of a packed row in LDS (its banks turn by 4)
    uint8_t *xs = smem + (FUSED ? m * stride : 0);
    auto load = [&](Step &q, int64_t grp, int p) {
        const int64_t row = grp * (16 * NB);
        const uint8_t *c = P.bc + p * bplane + row * 64, *s = P.bs + p * (bplane >> 4) + row * 4;
        const int last = (int)min(P.n - row, (int64_t)16 * NB) - 1;  // (rows past the end read the last one's place)
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const uint32_t at = (uint32_t)min(i * 16 + r, last) * 4 + g;
            q.b[i] = __builtin_nontemporal_load(reinterpret_cast<const i32x4 *>(c + at * 16));
            q.sb[i] = s[at];
        }
        if (KS == 1 && p == planes - 1) {
#pragma unroll
            for (int i = 0; i < NB; ++i) q.bias[i] = bias4(P.ep, row + i * 16 + g * 4, P.n);
        }
        if (!FUSED) {
            q.a = *reinterpret_cast<const i32x4 *>(P.ac + p * aplane + ao * 64 + g * 16);
            q.sa = P.as[p * (aplane >> 4) + ao * 4 + g];
        }
    };
    // KS = 1: one run of planes, group after group; the loads are U planes ahead of the products
    int64_t ahead = group;
    int plane_ahead = 0;
    auto load_next = [&](Step &q) {
        if (ahead < groups) load(q, ahead, plane_ahead);
        if (++plane_ahead == planes) plane_ahead = 0, ahead += step;
    };
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (KS == 1)
            load_next(f[u]);
        else
            load(f[u], group, min(first + u * KS, planes - 1));
    }
    if (FUSED) {
        // 8 elements a thread, the blocks' largest by DPP as in k_mx4_quantize
        const int runs = planes * 16;
        for (int b = threadIdx.x; b < m * runs; b += NT) {
            const int row = m == 1 ? 0 : b / runs, run = b - row * runs;
            float v[8];
            load_run<X, VEC, 8>((const typename X::T *)R.x + row * R.ldx, run * 8, R.k, v);
            const uint32_t s = scale_code(quad_max(v));
            *reinterpret_cast<uint32_t *>(smem + row * stride + run * 4) = s == 255 ? 0u : to_codes(v, scale_operand(s));
            if ((run & 3) == 0) xs[row * planes * 4 + (run >> 2)] = (uint8_t)s;
        }
        __syncthreads();
    }
    auto store = [&](f32x4 y, f32x4 bias, int64_t col) {
        if (r >= m || col >= P.n) return;
        f32x4 t[1] = {y};
        finish(t, bias, P.ep);
        store_run<D>((typename D::T *)P.out + r * P.ldo + col, t[0], P.n - col);
    };
    auto packed = [&](Step &q, int p) {
        q.a = *reinterpret_cast<const i32x4 *>(smem + ao * stride + p * 64 + g * 16);
        q.sa = xs[ao * planes * 4 + p * 4 + g];
    };
    f32x4 acc[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) acc[i] = (f32x4){0, 0, 0, 0};
    auto multiply = [&](const Step &q) {
#pragma unroll
        for (int i = 0; i < NB; ++i) acc[i] = mfma(q.b[i], q.sb[i], q.a, q.sa, acc[i]);
    };
    if (KS == 1) {
        int p = 0;
        while (group < groups) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (group >= groups) break;  // (the whole wave)
                if (FUSED) packed(f[u], p);
                multiply(f[u]);
                if (++p == planes) {
#pragma unroll
                    for (int i = 0; i < NB; ++i) {
                        store(acc[i], f[u].bias[i], group * (16 * NB) + i * 16 + g * 4);
                        acc[i] = (f32x4){0, 0, 0, 0};
                    }
                    p = 0;
                    group += step;
                }
                load_next(f[u]);
            }
        }
        return;
    }
    for (int p = first; p < planes; p += U * KS) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (p + u * KS >= planes) break;  // (the whole wave)
            if (FUSED) packed(f[u], p + u * KS);
            multiply(f[u]);
            if (p + (U + u) * KS < planes) load(f[u], group, p + (U + u) * KS);
        }
    }
    __syncthreads();  // (the packed rows are no longer read)
    f32x4 *red = reinterpret_cast<f32x4 *>(smem);
#pragma unroll
    for (int i = 0; i < NB; ++i) red[(i * KS + w) * 64 + lane] = acc[i];
    __syncthreads();
    for (int t = w; t < NB; t += KS) {
        f32x4 y = red[t * KS * 64 + lane];
#pragma unroll
        for (int q = 1; q < KS; ++q) y += red[(t * KS + q) * 64 + lane];
        const int64_t col = group * (16 * NB) + t * 16 + g * 4;
        store(y, bias4(P.ep, col, P.n), col);
    }
}

// ---------------------------------------------------------------- launchers
static Epilogue epilogue(const float *bias, float alpha, int act, int64_t n) {
    return {bias, alpha, act, bias && ((uintptr_t)bias & 15) == 0 && n % 4 == 0};
}
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
    return blocks > INT32_MAX ? fail(LIRA_EUNSUPPORTED, std::string(what) + ": too many rows") : LIRA_OK;
}
// A launch has fewer than 2^32 threads along x: the rows that workgroups of 256 threads and `each` rows can take.
static constexpr int64_t launch_rows_most(int each) { return (int64_t)(UINT32_MAX / 256) * each; }

template <class D>
static int quantize(const void *x, int64_t n, int64_t k, int64_t ld, uint8_t *codes, uint8_t *scales,
                    int64_t plane_rows, hipStream_t st) {
    typedef typename D::T T;
    const bool vec = ((uintptr_t)x & 15) == 0 && (ld * sizeof(T)) % 16 == 0;
    // What the last kernel left of x may be in the caches; of x several times their size nothing is, and its
    // loads would push out the packed rows (1M x 128, packed and read back: 196 us, 184 with ONCE;
    // 10000 x 128 packed 2.9 us, 3.7 with it).
    const bool once = n * k * (int64_t)sizeof(T) >= (int64_t)128 << 20;
    constexpr int64_t most = launch_rows_most(16);
    for (int64_t r = 0; r < n; r += most) {
        const int64_t rows = std::min(n - r, most);
        const dim3 g((unsigned)((rows + 15) / 16), (unsigned)planes_of(k));
        const T *at = (const T *)x + r * ld;
        uint8_t *c = codes + r * 64, *s = scales + r * 4;
        if (!vec)
            hipLaunchKernelGGL((k_mx4_quantize<D, false, false>), g, dim3(256), 0, st, at, rows, k, ld, c, s, plane_rows);
        else if (once)
            hipLaunchKernelGGL((k_mx4_quantize<D, true, true>), g, dim3(256), 0, st, at, rows, k, ld, c, s, plane_rows);
        else
            hipLaunchKernelGGL((k_mx4_quantize<D, true, false>), g, dim3(256), 0, st, at, rows, k, ld, c, s, plane_rows);
        LIRA_HIP_TRY(hipGetLastError());
    }
    return LIRA_OK;
}

template <class D>
static int dequantize(const uint8_t *codes, const uint8_t *scales, int64_t plane_rows, int64_t n, int64_t k, void *out,
                      int64_t ld, hipStream_t st) {
    typedef typename D::T T;
    constexpr int R = 256 / (kPlane / (16 / (int)sizeof(T)));  // rows of a workgroup
    const bool vec = ((uintptr_t)out & 15) == 0 && (ld * sizeof(T)) % 16 == 0;
    constexpr int64_t most = launch_rows_most(R);
    for (int64_t r = 0; r < n; r += most) {
        const int64_t rows = std::min(n - r, most);
        const dim3 g((unsigned)((rows + R - 1) / R), (unsigned)planes_of(k));
        const uint8_t *c = codes + r * 64, *s = scales + r * 4;
        T *at = (T *)out + r * ld;
        if (vec)
            hipLaunchKernelGGL((k_mx4_dequantize<D, true>), g, dim3(256), 0, st, c, s, plane_rows, rows, k, at, ld);
        else
            hipLaunchKernelGGL((k_mx4_dequantize<D, false>), g, dim3(256), 0, st, c, s, plane_rows, rows, k, at, ld);
        LIRA_HIP_TRY(hipGetLastError());
    }
    return LIRA_OK;
}

template <int TN, int TM, int WN, int WM, int WK, int SLOTS, int PS, class D, class X = void>
static int launch_tile(const Product &p, hipStream_t st, const Rows &r = {nullptr, 0, 0, false}) {
    typedef Tile<TN, TM, WN, WM, WK, SLOTS, PS, !std::is_void<X>::value> C;
    static_assert(C::kBytes <= 163840 && C::template epilogue_bytes<D>() <= C::kBytes, "160 KB of LDS");
    static std::atomic<uint64_t> latch{0};
    const void *fn = (const void *)&k_mx4_tile<TN, TM, WN, WM, WK, SLOTS, PS, D, X>;
    LIRA_HIP_TRY(set_smem_attr_once(latch, fn, C::kBytes));
    // (few planes: only the slots that they fill, so that more workgroups share a compute unit:
    // 10000 x 1024 x 128 20 us -> 14)
    const int steps = (p.planes + PS - 1) / PS, slots = std::min(SLOTS, steps) * PS * C::kPlaneBytes;
    const int bytes = std::min<int>(C::kBytes, std::max<int>(slots, C::template epilogue_bytes<D>()));
    const int64_t tn = (p.n + TN - 1) / TN, tm = (p.m + TM - 1) / TM;
    hipLaunchKernelGGL((k_mx4_tile<TN, TM, WN, WM, WK, SLOTS, PS, D, X>), dim3((unsigned)(tn * tm)), dim3(C::NW * 64), bytes, st, p,
                       r, (int)tn, (int)tm);
    LIRA_HIP_TRY(hipGetLastError());
    return LIRA_OK;
}

template <class X, class D, int NB, int KS, bool FUSED, bool VEC>
static int launch_rows(const Product &p, const Rows &r, hipStream_t st) {
    static std::atomic<uint64_t> latch{0};
    const void *fn = (const void *)&k_mx4_rows<X, D, NB, KS, FUSED, VEC>;
    const int bytes = std::max(KS == 1 ? 0 : KS * NB * 1024, FUSED ? (int)p.m * (p.planes * 68 + 16) : 0);
    LIRA_HIP_TRY(set_smem_attr_once(latch, fn, 65536));
    const int64_t groups = (p.n + 16 * NB - 1) / (16 * NB);
    // (KS = 1: as many workgroups of 4 waves as the 256 compute units hold, 6 waves a SIMD)
    const int64_t blocks = KS == 1 ? std::min<int64_t>((groups + 3) / 4, 256 * 6) : groups;
    hipLaunchKernelGGL((k_mx4_rows<X, D, NB, KS, FUSED, VEC>), dim3((unsigned)blocks), dim3(KS == 1 ? 256 : KS * 64), bytes, st,
                       p, r);
    LIRA_HIP_TRY(hipGetLastError());
    return LIRA_OK;
}
// Rows that the product packs by itself: so few that every workgroup may do it again.  Up to 4 always (while they fit
// LDS); up to 16 of fewer planes, where that costs less than a launch of its own (kernels alone, us, packed here and
// by themselves: 16 x 8192 x 2048 6.9 and 7.1, 8 x 8192 x 4096 7.2 and 7.5, 16 x 8192 x 4096 10.3 and 7.4; 12 x 40000 x
// 2048 19.3 and 21.1, 8 x 40000 x 4096 27.3 and 24.5).
static bool rows_packed(int64_t m, int64_t n, int64_t k) {
    const int64_t planes = planes_of(k);
    return (m <= 4 && m * (planes * 68 + 16) <= 49152) || (m <= 16 && m * planes <= (n <= 8192 ? 256 : 192));
}

// 4096 tiles of 16 columns are enough loads in flight without the planes split (one row, us split and not: 32768 x
// 4096 18 and 26, 65536 x 4096 32 and 25, 200000 x 900 54 and 19).
static bool split_planes(const Product &p) { return p.planes >= 8 && (p.n + 15) / 16 < 4096; }

template <class X, class D>
static int linear_rows(const Product &p, const Rows &r, hipStream_t st) {
    // (32 columns a workgroup where that still leaves each compute unit one: the rows are packed half as often; 4 x 8192
    // x 8192 12.4 us, 14.4 with 16)
    if (split_planes(p) && p.n >= 256 * 32)
        return r.vec ? launch_rows<X, D, 2, 8, true, true>(p, r, st) : launch_rows<X, D, 2, 8, true, false>(p, r, st);
    if (split_planes(p))
        return r.vec ? launch_rows<X, D, 1, 8, true, true>(p, r, st) : launch_rows<X, D, 1, 8, true, false>(p, r, st);
    return r.vec ? launch_rows<X, D, 2, 1, true, true>(p, r, st) : launch_rows<X, D, 2, 1, true, false>(p, r, st);
}
// The tile of more than 16 rows: the one with the least estimated time.  A launch takes
// start + planes * plane + load * (tile + planes * step) us, where load is the tiles of a compute unit, between the
// average and the busiest's; the four numbers of each tile are least squares over 756 products (20 to 4096 rows, 256
// to 300000 columns, k 128 to 8192, 16-bit results).  On those, the choice is 1.7 % slower than the best tile, in
// the mean; the largest tile that leaves no compute unit idle was 16 %.  The first three tiles have four sets of
// waves and take four planes a barrier: less of a step is left bare, so they win while a compute unit has one tile
// of many planes (37 x 11111 x 5000: 11.8 us by the third, 13.3 by the fifth); the others are small enough in LDS for
// two or more a unit (37 x 300000 x 128: 11 us by the sixth, 28 by the third).
static const struct {
    int tn, tm, waves;
    float start, plane, tile, step;
} kTiles[] = {
    {32, 32, 8, 3.136f, 0.043f, 0.875f, 0.065f},
    {64, 32, 8, 3.796f, 0.017f, 1.108f, 0.138f},
    {64, 64, 8, 3.794f, 0.033f, 1.852f, 0.170f},
    {64, 32, 4, 2.975f, 0.133f, 0.417f, 0.073f},
    {64, 64, 4, 3.127f, 0.149f, 0.473f, 0.096f},
    {128, 64, 4, 3.607f, 0.179f, 0.699f, 0.160f},
    {128, 128, 4, 3.989f, 0.215f, 1.542f, 0.246f},
    {256, 256, 8, 3.441f, 0.340f, 6.660f, 0.784f},
};
static int tile_for(int64_t m, int64_t n, int64_t planes) {
    int best = 0;
    float least = INFINITY;
    for (int i = 0; i < (int)(sizeof(kTiles) / sizeof(kTiles[0])); ++i) {
        const auto &t = kTiles[i];
        const int64_t tiles = ((n + t.tn - 1) / t.tn) * ((m + t.tm - 1) / t.tm);
        const float load = 0.5f * ((float)((tiles + 255) / 256) + (float)tiles / 256.0f);
        const float us = t.start + planes * t.plane + load * (t.tile + planes * t.step);
        if (us < least) least = us, best = i;
    }
    return best;
}

template <class D>
static int product(const Product &p, hipStream_t st) {
    if (p.m <= 16) {
        const Rows r = {nullptr, 0, 0, false};
        if (split_planes(p)) return launch_rows<F32, D, 1, 8, false, false>(p, r, st);
        return launch_rows<F32, D, 2, 1, false, false>(p, r, st);
    }
    switch (tile_for(p.m, p.n, p.planes)) {
    case 0: return launch_tile<32, 32, 1, 2, 4, 4, 4, D>(p, st);
    case 1: return launch_tile<64, 32, 2, 1, 4, 4, 4, D>(p, st);
    case 2: return launch_tile<64, 64, 2, 1, 4, 4, 4, D>(p, st);
    case 3: return launch_tile<64, 32, 2, 2, 1, 4, 1, D>(p, st);
    case 4: return launch_tile<64, 64, 2, 2, 1, 4, 1, D>(p, st);
    case 5: return launch_tile<128, 64, 2, 2, 1, 4, 1, D>(p, st);
    case 6: return launch_tile<128, 128, 2, 2, 1, 4, 1, D>(p, st);
    default: return launch_tile<256, 256, 2, 4, 1, 4, 1, D>(p, st);
    }
}
// More rows, packed by their tiles: of whole runs of 8, for half a tile's columns or more, and of so few planes and
// tiles a compute unit that this takes no longer than a launch of its own does (kernels alone, fp32, us, packed here
// and by themselves: 1000 x 256 x 128 5.2 and 5.2, 4000 x 1024 x 128 6.8 and 8.0, 50000 x 256 x 128 14.8 and 19.2,
// 1000 x 1024 x 256 6.5 and 6.1; 1000 x 1024 x 384 9.3 and 6.4; a call from Python takes 4 less).  Rows that are not
// aligned, 4-byte loads, take the same way, since the workspace's size goes by shapes alone, but a launch of their own
// is faster: 1000 x 256 x 128 8.4 packed here and 5.8 by themselves, 4000 x 1024 x 128 12.6 and 8.4, 50000 x 256 x
// 128 31.1 and 26.2, 1000 x 1024 x 256 12.4 and 6.7.
static bool tile_packed(int64_t m, int64_t n, int64_t k) {
    const int64_t planes = planes_of(k), load = (((n + 127) / 128) * ((m + 63) / 64) + 255) / 256;
    return m > 16 && n >= 64 && k % 8 == 0 && planes <= 2 && load * planes <= 10;
}
static bool packed_inside(int64_t m, int64_t n, int64_t k) { return rows_packed(m, n, k) || tile_packed(m, n, k); }
template <class X, class D>
static int linear(const Product &p, const Rows &r, hipStream_t st) {
    if (p.m <= 16) return linear_rows<X, D>(p, r, st);
    return launch_tile<128, 64, 2, 2, 1, 4, 1, D, X>(p, st, r);
}
template <class X>
static int linear(const Product &p, const Rows &r, int out_dtype, hipStream_t st) {
    if (out_dtype == LIRA_DTYPE_F32) return linear<X, F32>(p, r, st);
    if (out_dtype == LIRA_DTYPE_BF16) return linear<X, BF16>(p, r, st);
    return linear<X, F16>(p, r, st);
}
static int product(const Product &p, int out_dtype, hipStream_t st) {
    if (out_dtype == LIRA_DTYPE_F32) return product<F32>(p, st);
    if (out_dtype == LIRA_DTYPE_BF16) return product<BF16>(p, st);
    return product<F16>(p, st);
}

static int check_product(int64_t m, int64_t n, int64_t k, int act, const void *out, int out_dtype, int64_t ldo) {
    if (!dtype_ok(out_dtype)) return fail(LIRA_EINVAL, "unknown dtype");
    if (act < LIRA_ACT_NONE || act > LIRA_ACT_SIGMOID) return fail(LIRA_EINVAL, "unknown activation");
    if (ldo < n) return fail(LIRA_EINVAL, "ldo must be at least n");
    if (m > 0 && n > 0 && !out) return fail(LIRA_EINVAL, "NULL buffer");
    if (m > INT32_MAX) return fail(LIRA_EUNSUPPORTED, "product: too many rows");
    if (int rc = check_grid((n + 15) / 16, "product")) return rc;
    if (m > 16) {  // (rows that their tiles pack have few)
        const auto &t = kTiles[tile_for(m, n, planes_of(k))];
        if (((n + t.tn - 1) / t.tn) * ((m + t.tm - 1) / t.tm) > (int64_t)(UINT32_MAX / (t.waves * 64)))
            return fail(LIRA_EUNSUPPORTED, "product: too many tiles for one launch, which has fewer than 2^32 threads");
    }
    return LIRA_OK;
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
    if (int rc = check_grid((n + 7) / 8, "mx4_dequantize")) return rc;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == LIRA_DTYPE_F32) return dequantize<F32>(codes, scales, plane_rows, n, k, out, ld, st);
    if (dtype == LIRA_DTYPE_BF16) return dequantize<BF16>(codes, scales, plane_rows, n, k, out, ld, st);
    return dequantize<F16>(codes, scales, plane_rows, n, k, out, ld, st);
}

int lira_mx4_matmul(const uint8_t *a_codes, const uint8_t *a_scales, int64_t a_plane_rows, int64_t m,
                    const uint8_t *b_codes, const uint8_t *b_scales, int64_t b_plane_rows, int64_t n, int64_t k,
                    float alpha, const float *bias, int act, void *out, int out_dtype, int64_t ldo, void *stream) {
    if (int rc = check_packed(a_codes, a_scales, m, a_plane_rows, k)) return rc;
    if (int rc = check_packed(b_codes, b_scales, n, b_plane_rows, k)) return rc;
    if (int rc = check_product(m, n, k, act, out, out_dtype, ldo)) return rc;
    if (m == 0 || n == 0) return LIRA_OK;
    hipStream_t st = (hipStream_t)stream;
    const Product p = {a_codes, a_scales, b_codes, b_scales, a_plane_rows, b_plane_rows, m, n, ldo,
                       (int)planes_of(k), epilogue(bias, alpha, act, n), out};
    return product(p, out_dtype, st);
}

int lira_mx4_linear_workspace_size(int64_t m, int64_t n, int64_t k, size_t *bytes) {
    if (!bytes) return fail(LIRA_EINVAL, "NULL buffer");
    if (m < 0 || n < 0 || k <= 0) return fail(LIRA_EINVAL, "bad shape");
    *bytes = m == 0 || n == 0 || packed_inside(m, n, k) ? 0 : (size_t)(planes_of(k) * m * 68);
    return LIRA_OK;
}

int lira_mx4_linear(const void *x, int dtype, int64_t m, int64_t k, int64_t ldx, const uint8_t *b_codes,
                    const uint8_t *b_scales, int64_t b_plane_rows, int64_t n, float alpha, const float *bias, int act,
                    void *out, int out_dtype, int64_t ldo, void *workspace, size_t workspace_bytes, void *stream) {
    if (!dtype_ok(dtype)) return fail(LIRA_EINVAL, "unknown dtype");
    if (int rc = check_packed(b_codes, b_scales, n, b_plane_rows, k)) return rc;
    if (m < 0) return fail(LIRA_EINVAL, "bad shape");
    if (ldx < k) return fail(LIRA_EINVAL, "ldx must be at least k");
    if (int rc = check_product(m, n, k, act, out, out_dtype, ldo)) return rc;
    if (m == 0 || n == 0) return LIRA_OK;
    if (!x) return fail(LIRA_EINVAL, "NULL buffer");
    size_t need = 0;
    if (int rc = lira_mx4_linear_workspace_size(m, n, k, &need)) return rc;
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15) != 0))
        return fail(LIRA_EINVAL, "workspace too small (lira_mx4_linear_workspace_size) or not 16-byte aligned");
    if (!need) {
        const Product p = {nullptr, nullptr, b_codes, b_scales, 0, b_plane_rows, m, n, ldo,
                           (int)planes_of(k), epilogue(bias, alpha, act, n), out};
        const Rows r = {x, k, ldx, ((uintptr_t)x & 15) == 0 && (ldx * (dtype == LIRA_DTYPE_F32 ? 4 : 2)) % 16 == 0};
        if (dtype == LIRA_DTYPE_F32) return linear<F32>(p, r, out_dtype, (hipStream_t)stream);
        if (dtype == LIRA_DTYPE_BF16) return linear<BF16>(p, r, out_dtype, (hipStream_t)stream);
        return linear<F16>(p, r, out_dtype, (hipStream_t)stream);
    }
    uint8_t *ac = (uint8_t *)workspace, *as = ac + planes_of(k) * m * 64;
    if (int rc = lira_mx4_quantize(x, dtype, m, k, ldx, ac, as, m, stream)) return rc;
    return lira_mx4_matmul(ac, as, m, m, b_codes, b_scales, b_plane_rows, n, k, alpha, bias, act, out, out_dtype, ldo,
                           stream);
}

}  // extern "C"
