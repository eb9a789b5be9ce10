// lira_distill.hip -- distillation from a teacher's top logits: loss and gradient.
//
// Row r: student logits z (vocab), teacher entries (i_j, t_j), j < top, i_j < 0 unused:
//   log p_j = t_j / T - L,  L = logsumexp_j(t_j / T) (or the teacher's own over all its outputs)
//   log q_v = z_v / T - logsumexp_v(z_v / T),  s = sum_j p_j
//   loss    = T^2 sum_{p_j > 0} p_j (log p_j - log q_{i_j})
//   d/dz_v  = T (s q_v - sum_{j: i_j = v} p_j)
// A row without a used entry has loss 0 and gradient 0.  z = -inf has q = 0.  NaN or +inf
// among the z, or an id >= vocab, makes the whole row NaN.  Sums in fp32; the gradient is
// rounded once, to the type of z.
#include <string>

#include "lira_internal.hpp"
#include "lira_mx4.hpp"

namespace lira {

static constexpr int kMaxTop = 1024;
static constexpr float kLog2e = 1.44269504088896340736f;

struct DistillArgs {
    const void *z;
    int64_t rows, vocab, ldz;
    const void *ids;
    const float *tv;
    int top, ids64;
    const float *teacher_lse;  // NULL: over the row's entries
    float t;                   // temperature
    const float *row_scale;    // factor of each row's gradient: row_scale[r * scale_stride]; NULL: 1
    int64_t scale_stride;
    float *loss;               // may be NULL
    float *stats;              // (rows, 2): student logsumexp of z / T, s (0: no entry counts, NaN: the row is NaN)
    void *dz;                  // NULL: loss alone
    int64_t ldd;
    int mode;                  // 0: loss (and dz) from scratch; 1: dz alone, from stats
};

// (max, sum of 2^((x - max) log2e)) pairs: joined as in a running softmax
struct MS {
    float m, s;
};
__device__ __forceinline__ float e2(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }
__device__ __forceinline__ MS join(MS a, MS b) {
    const float m = fmaxf(a.m, b.m);
    if (m == -INFINITY) return {m, a.s + b.s};  // (both sums are 0, or NaN)
    return {m, a.s * e2(a.m - m) + b.s * e2(b.m - m)};
}
__device__ __forceinline__ MS add(MS a, float x) { return join(a, {x, x == -INFINITY ? 0.0f : x != x ? x : 1.0f}); }

template <class D>
__global__ __launch_bounds__(256) void k_distill(DistillArgs a) {
    typedef typename D::T T;
    __shared__ float sm[4], ss[4], sp[kMaxTop], sx[kMaxTop];
    __shared__ int64_t sid[kMaxTop];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int64_t r = blockIdx.x;
    const T *z = (const T *)a.z + r * a.ldz;
    const float it = 1.0f / a.t;
    float lse;
    if (a.mode == 0) {
        MS v = {-INFINITY, 0.0f};
        for (int64_t j = tid; j < a.vocab; j += 256) {
            const float x = D::up(z[j]) * it;
            v = add(v, x == INFINITY ? NAN : x);
        }
#pragma unroll
        for (int s = 32; s >= 1; s >>= 1) v = join(v, {__shfl_xor(v.m, s), __shfl_xor(v.s, s)});
        if (lane == 0) sm[w] = v.m, ss[w] = v.s;
        __syncthreads();
        v = {sm[0], ss[0]};
        for (int i = 1; i < 4; ++i) v = join(v, {sm[i], ss[i]});
        lse = v.m == -INFINITY && v.s == 0.0f ? -INFINITY : v.m + logf(v.s);
        if (v.s != v.s) lse = NAN;
    } else {
        lse = a.stats[2 * r];
        if (a.stats[2 * r + 1] != a.stats[2 * r + 1]) lse = NAN;
    }
    // the teacher's entries
    float tm = -INFINITY;
    bool bad = false;
    for (int j = tid; j < a.top; j += 256) {
        const int64_t id = a.ids64 ? ((const int64_t *)a.ids)[r * a.top + j] : ((const int32_t *)a.ids)[r * a.top + j];
        bad |= id >= a.vocab;
        sid[j] = id;
        sp[j] = id < 0 ? -INFINITY : a.tv[r * a.top + j] * it;
    }
    if (__syncthreads_or(bad)) lse = NAN;
    MS tl = {-INFINITY, 0.0f};
    if (a.teacher_lse)
        tm = a.teacher_lse[r];
    else {
        for (int j = 0; j < a.top; ++j) tl = add(tl, sp[j]);
        tm = tl.m + logf(tl.s);
        if (tl.m == -INFINITY && tl.s == 0.0f) tm = -INFINITY;
    }
    __syncthreads();
    float l = 0.0f, sum = 0.0f;
    bool some = false;
    for (int j = tid; j < a.top; j += 256) {
        const int64_t id = sid[j];
        const float lp = sp[j] - tm;
        const float p = sp[j] == -INFINITY ? 0.0f : e2(lp);
        sp[j] = p;
        some |= id >= 0 && !(p == 0.0f);
        const float x = id >= 0 && id < a.vocab ? D::up(z[id]) * it : 0.0f;
        sx[j] = x;
        if (!(p == 0.0f)) {
            l += p * (lp - (x == -INFINITY ? x : x - lse));
        }
        sum += p;
    }
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) l += __shfl_xor(l, s), sum += __shfl_xor(sum, s);
    if (lane == 0) sm[w] = l, ss[w] = sum;
    some = __syncthreads_or(some);
    l = sm[0] + sm[1] + sm[2] + sm[3];
    sum = ss[0] + ss[1] + ss[2] + ss[3];
    if (lse != lse) l = sum = NAN, some = true;
    if (!some) l = sum = 0.0f;
    if (tid == 0) {
        if (a.loss) a.loss[r] = a.t * a.t * l;
        if (a.stats && a.mode == 0) a.stats[2 * r] = lse, a.stats[2 * r + 1] = sum;
    }
    if (!a.dz) return;
    T *dz = (T *)a.dz + r * a.ldd;
    const float g = a.t * (a.row_scale ? a.row_scale[r * a.scale_stride] : 1.0f);
    for (int64_t j = tid; j < a.vocab; j += 256) {
        const float x = D::up(z[j]) * it;
        const float q = x == -INFINITY && lse == lse ? 0.0f : e2(x - lse);
        dz[j] = D::down(some ? g * (sum * q) : 0.0f);
    }
    if (!some || lse != lse) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();  // (the entries' places are written again below, after every store above has ended)
    for (int j = tid; j < a.top; j += 256) {
        const int64_t id = sid[j];
        if (id < 0) continue;
        float p = 0.0f;
        bool first = true;
        for (int i = 0; i < a.top; ++i)
            if (sid[i] == id) p += sp[i], first &= i >= j;
        if (!first) continue;
        const float x = sx[j];  // (z's own place may hold dz by now)
        const float q = x == -INFINITY ? 0.0f : e2(x - lse);
        dz[id] = D::down(g * (sum * q - p));
    }
}

// out[0] = sum of the rows' losses, or their mean over the rows that count; out[1] = the factor
// of every row's gradient.  One workgroup, fixed order: the same bits every time.
__global__ __launch_bounds__(1024) void k_distill_reduce(const float *loss, const float *stats, int64_t rows, int mean,
                                                         float *out) {
    __shared__ float sl[16], sc[16];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    float l = 0.0f, c = 0.0f;
    for (int64_t r = tid; r < rows; r += 1024) {
        l += loss[r];
        c += stats[2 * r + 1] == 0.0f ? 0.0f : 1.0f;
    }
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) l += __shfl_xor(l, s), c += __shfl_xor(c, s);
    if (lane == 0) sl[w] = l, sc[w] = c;
    __syncthreads();
    if (tid != 0) return;
    l = c = 0.0f;
    for (int i = 0; i < 16; ++i) l += sl[i], c += sc[i];
    const float f = mean ? (c > 0.0f ? 1.0f / c : 0.0f) : 1.0f;
    out[0] = mean ? (c > 0.0f ? l / c : 0.0f) : l;
    out[1] = f;
}

static int run(const DistillArgs &a, int dtype, hipStream_t st) {
    const dim3 g((unsigned)a.rows);
    if (dtype == LIRA_DTYPE_F32)
        hipLaunchKernelGGL((k_distill<F32>), g, dim3(256), 0, st, a);
    else if (dtype == LIRA_DTYPE_BF16)
        hipLaunchKernelGGL((k_distill<BF16>), g, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((k_distill<F16>), g, dim3(256), 0, st, a);
    LIRA_HIP_TRY(hipGetLastError());
    return LIRA_OK;
}

}  // namespace lira

using namespace lira;

static int check_distill(const DistillArgs &a, int dtype, int ids_bits) {
    if (dtype < LIRA_DTYPE_F32 || dtype > LIRA_DTYPE_F16) return fail(LIRA_EINVAL, "unknown dtype");
    if (ids_bits != 32 && ids_bits != 64) return fail(LIRA_EINVAL, "ids_bits must be 32 or 64");
    if (a.rows < 0 || a.vocab <= 0) return fail(LIRA_EINVAL, "rows must be >= 0 and vocab >= 1");
    if (a.top < 1) return fail(LIRA_EINVAL, "top must be >= 1");
    if (a.top > kMaxTop) return fail(LIRA_EUNSUPPORTED, "top must be at most 1024");
    if (a.ldz < a.vocab || (a.dz && a.ldd < a.vocab)) return fail(LIRA_EINVAL, "row strides must be at least vocab");
    if (!(a.t > 0.0f) || !(a.t < INFINITY)) return fail(LIRA_EINVAL, "temperature must be positive and finite");
    if (a.row_scale && (a.scale_stride < 0 || a.scale_stride > 1))
        return fail(LIRA_EINVAL, "scale_stride must be 0 or 1");
    if (a.rows > INT32_MAX) return fail(LIRA_EUNSUPPORTED, "too many rows for one launch");
    if (a.rows > 0 && (!a.z || !a.ids || !a.tv)) return fail(LIRA_EINVAL, "NULL buffer");
    return LIRA_OK;
}

extern "C" {

int lira_distill_topk(const void *z, int dtype, int64_t rows, int64_t vocab, int64_t ldz, const void *ids, int ids_bits,
                      const float *teacher, int64_t top, float temperature, const float *teacher_lse, float *loss,
                      float *stats, const float *row_scale, int64_t scale_stride, void *dz, int64_t ldd,
                      void *stream) {
    const DistillArgs a = {z, rows, vocab, ldz, ids, teacher, (int)(top < 0 ? 0 : top > INT32_MAX ? INT32_MAX : top),
                           ids_bits == 64, teacher_lse, temperature, row_scale, scale_stride, loss, stats, dz, ldd, 0};
    if (int rc = check_distill(a, dtype, ids_bits)) return rc;
    if (rows == 0) return LIRA_OK;
    if (!loss) return fail(LIRA_EINVAL, "NULL buffer");
    return run(a, dtype, (hipStream_t)stream);
}

int lira_distill_topk_backward(const void *z, int dtype, int64_t rows, int64_t vocab, int64_t ldz, const void *ids,
                               int ids_bits, const float *teacher, int64_t top, float temperature,
                               const float *teacher_lse, const float *stats, const float *row_scale,
                               int64_t scale_stride, void *dz, int64_t ldd, void *stream) {
    const DistillArgs a = {z, rows, vocab, ldz, ids, teacher, (int)(top < 0 ? 0 : top > INT32_MAX ? INT32_MAX : top),
                           ids_bits == 64, teacher_lse, temperature, row_scale, scale_stride, nullptr,
                           const_cast<float *>(stats), dz, ldd, 1};
    if (int rc = check_distill(a, dtype, ids_bits)) return rc;
    if (rows == 0) return LIRA_OK;
    if (!stats || !dz) return fail(LIRA_EINVAL, "NULL buffer");
    return run(a, dtype, (hipStream_t)stream);
}

int lira_distill_reduce(const float *loss, const float *stats, int64_t rows, int mean, float *out, void *stream) {
    if (rows < 0) return fail(LIRA_EINVAL, "rows must be >= 0");
    if (!out || (rows > 0 && (!loss || !stats))) return fail(LIRA_EINVAL, "NULL buffer");
    hipLaunchKernelGGL(k_distill_reduce, dim3(1), dim3(1024), 0, (hipStream_t)stream, loss, stats, rows, mean ? 1 : 0,
                       out);
    LIRA_HIP_TRY(hipGetLastError());
    return LIRA_OK;
}

}  // extern "C"
