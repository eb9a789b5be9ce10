// lira_distill.hip -- distillation from a teacher's top logits: loss and gradient.
//
// Row r: student logits z (vocab), teacher entries (i_j, t_j), j < top, i_j < 0 unused:
//   log p_j = t_j / T - L,  L = logsumexp_j(t_j / T) (or the teacher's own over all its outputs)
//   log q_v = z_v / T - logsumexp_v(z_v / T),  s = sum_j p_j
//   loss    = T^2 sum_{p_j > 0} p_j (log p_j - log q_{i_j})
//   d/dz_v  = T (s q_v - sum_{j: i_j = v} p_j)
// A row in which no entry counts has loss 0 and gradient 0, whatever its logits.  z = -inf has
// q = 0.  NaN or +inf among the z, NaN among the entries, or an id >= vocab makes the row NaN.
//
// Memory-bound: the loss reads z once, the gradient writes as much.  Everything is in powers of 2
// of (z - max) c, c = log2(e) / T: one subtraction and one fma before the exp, no overflow where
// z holds its type's lowest value.  Sums in fp32 in a fixed order.
//
// A group of NT threads works on a row (or a slice of it).  Thread u holds the 16-byte vectors u,
// u + NT, ..: in registers (NV of them) where loss and gradient are wanted together, so that z is
// read from memory once.  Rows need not be aligned: the vectors begin where the gradient (the row
// itself, if only the loss is wanted) is, and up to two vectors' elements at the ends are single
// (2048 x 131071 bf16, loss and gradient: 251 us, 271 with vectors from the row's first element;
// the loss alone 99 and 117).  Which thread adds an element, so the last bits of a sum, follows from
// that alignment.
//
// The teacher's entries change single places of the gradient.  The first wave puts each entry
// into a list of the thread that stores its place (LDS); that thread stores the place once more
// after its vectors -- its own stores to one address stay in order, so no barrier waits for them.
#include <algorithm>
#include <cfloat>
#include <string>

#include "lira_device.hpp"
#include "lira_internal.hpp"
#include "lira_mx4.hpp"

namespace lira {

static constexpr int kMaxTop = 1024;
static constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

struct DistillArgs {
    const void *z;
    int64_t rows;
    int64_t vocab, ldz;
    const void *ids;
    const float *tv;
    int top, ids64;
    const float *teacher_lse;  // NULL: over the row's entries
    float t;                   // temperature
    const float *row_scale;    // factor of each row's gradient: row_scale[r * scale_stride]; NULL: 1
    int64_t scale_stride;
    float *loss;
    float *stats;  // (rows, 4): max z, log2 sum 2^((z - max) c), s (0: no entry counts, NaN: the row is NaN), 0
    void *dz;
    int64_t ldd;
    int slices;      // of a row, kSliceVecs vectors each (1: whole rows)
    float2 *part;    // [rows][slices] (max, sum) of the slices
    float *xs;       // [rows][top] the z that the entries name
};

enum Mode {
    kLoss,   // loss and stats
    kBoth,   // loss, stats and gradient
    kGrad,   // gradient from stats
    kPart,   // a slice's (max, sum) and, by slice 0, the entries' z
    kJoin,   // the slices' joined: loss by slice 0, and the slice's gradient if wanted
};

__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int m = 1; m <= 32; m <<= 1) v = fmaxf(v, __uint_as_float(xor_u32(__float_as_uint(v), m)));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int m = 1; m <= 32; m <<= 1) v += __uint_as_float(xor_u32(__float_as_uint(v), m));
    return v;
}

// 16 bytes of a row, at any alignment
template <class D>
struct Vec {
    typedef typename D::T T;
    static constexpr int E = 16 / sizeof(T);
    uint32_t w[4];
    __device__ __forceinline__ void load(const T *at) { __builtin_memcpy(w, at, 16); }
    __device__ __forceinline__ void store(T *at) const { stream16(at, (i32x4){(int)w[0], (int)w[1], (int)w[2], (int)w[3]}); }
    __device__ __forceinline__ float get(int i) const {
        if (sizeof(T) == 4) return __uint_as_float(w[i]);
        const uint16_t h = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        T t;
        __builtin_memcpy(&t, &h, sizeof(T) == 2 ? 2 : 0);
        return D::up(t);
    }
    // (the passes over a row unpack anew: unpacked values kept from one to the next would take
    // twice the registers that the row itself does)
    __device__ __forceinline__ void forget() { asm volatile("" : "+v"(w[0]), "+v"(w[1]), "+v"(w[2]), "+v"(w[3])); }
    __device__ __forceinline__ void mask(bool there) {
        constexpr uint32_t none = sizeof(T) == 4 ? 0xff800000u : D::kNegInf * 0x10001u;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = there ? w[i] : none;
    }
    __device__ __forceinline__ float max() const {
        float m = get(0);
#pragma unroll
        for (int i = 1; i < E; ++i) m = fmaxf(m, get(i));
        return m;
    }
    __device__ __forceinline__ float sum(float m, float c) const {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) s += ex2((get(i) - m) * c);
        return s;
    }
    __device__ __forceinline__ void grad(float m, float c, float l2, float f) {
        T o[E];
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] = D::down(f * ex2(fmaf(get(i) - m, c, -l2)));
        __builtin_memcpy(w, o, 16);
    }
};

static constexpr int kSliceVecs = 1024;  // 4 vectors a thread of 256

template <class D, int NT, int NV, int KM, Mode MODE>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void k_distill(DistillArgs a) {
    typedef typename D::T T;
    typedef Vec<D> V;
    constexpr int E = V::E, G = NT < 256 ? 256 / NT : 1, NW = NT / 64, J = KM / 64;
    constexpr bool kStats = MODE == kLoss || MODE == kBoth || MODE == kPart;
    constexpr bool kDz = MODE == kBoth || MODE == kGrad || MODE == kJoin;
    constexpr bool kEntries = MODE != kPart;
    static_assert(NT >= 64 && (G == 1 || NW == 1), "a group is a wave or a workgroup");
    __shared__ float sm[G][NW], ss[G][NW];
    __shared__ float s_p[G][kEntries ? KM : 1], s_x[G][kEntries ? KM : 1];
    __shared__ __attribute__((aligned(16))) int s_id[G][kEntries ? KM : 1];
    __shared__ int s_next[G][kEntries ? KM : 1], s_head[G][kDz ? NT : 1];
    constexpr int NC = NT < 256 ? NT : 256;
    __shared__ int s_count[G][kDz ? NC : 1];  // entries of the lists (of the threads u, u + 256, .. together)
    __shared__ float s_tot[G][2];
    __shared__ int s_many[G];
    const int gi = G == 1 ? 0 : threadIdx.x >> 6, u = G == 1 ? threadIdx.x : threadIdx.x & 63;
    const int lane = threadIdx.x & 63, w = G == 1 ? threadIdx.x >> 6 : 0;
    auto sync = [&]() {
        if (NW > 1)
            __syncthreads();
        else
            __builtin_amdgcn_wave_barrier();  // (one wave: LDS operations are in order)
    };
    int64_t r = (int64_t)blockIdx.x * G + gi;
    int slice = 0;
    if (MODE == kPart || MODE == kJoin || MODE == kGrad) {
        slice = (int)(r % a.slices);
        r /= a.slices;
    }
    if (r >= a.rows) return;  // (a whole wave, only where groups are waves)
    const T *z = (const T *)a.z + r * a.ldz;
    const float c = kLog2e / a.t;
    // the vectors begin h elements in; the slice's are [v0, v1); the elements before the first and behind the
    // last are single, one to each of the last slice's first threads
    const uintptr_t from = MODE != kLoss && kDz ? (uintptr_t)((const T *)a.dz + r * a.ldd) : (uintptr_t)z;
    const int h = min((int)a.vocab, (int)(-from & 15) / (int)sizeof(T));
    const int nvec = ((int)a.vocab - h) / E, shift = nvec * E;  // (element j + shift is single behind, j >= h)
    const int v0 = a.slices > 1 ? slice * kSliceVecs : 0;
    const int v1 = a.slices > 1 ? min(nvec, v0 + kSliceVecs) : nvec;
    const int singles = slice == a.slices - 1 ? (int)a.vocab - shift : 0;
    const bool single = u < singles;
    const int at1 = u < h ? u : u + shift;

    // ------------------------------------------- the entries' loads first
    int id[J];
    float tv[J];
    const bool first = kEntries && w == 0;
    if (first) {
#pragma unroll
        for (int i = 0; i < J; ++i) {
            const int j = i * 64 + lane;
            int64_t k = -1;
            tv[i] = -INFINITY;
            if (j < a.top) {
                k = a.ids64 ? ((const int64_t *)a.ids)[r * a.top + j] : ((const int32_t *)a.ids)[r * a.top + j];
                tv[i] = a.tv[r * a.top + j];
            }
            id[i] = k < 0 ? -1 : k >= a.vocab ? INT32_MAX : (int)k;  // (vocab < INT32_MAX)
        }
    }
    V x[NV ? NV : 1];
    float m = -INFINITY, s = 0.0f;
    if (kStats) {
        if (NV) {
            // (NV / 2 NT <= vectors <= NV NT: only the later half can be missing; a missing one is read
            // from the last one's place, which costs less than a branch round every load)
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int k = h + (i * NT + u) * E;
                x[i].load(z + (i < NV / 2 ? k : min(k, nvec ? h + shift - E : 0)));
            }
        }
    }
    const float x1 = single ? D::up(z[at1]) : -INFINITY;

    // Entries of a list that is walked, which takes the square of its length in steps that wait for each other; where
    // one is longer, the row's threads go over all entries for each id (256 x 4096, top 1024: ids apart 35 us and 42;
    // of one id 137 ms walked, 0.15 gone over; 4096 x 1024, top 64, padded with id 0: 700 us and 15).
    const int most = max(8, a.top / 16);

    // ------------------------------------------------------------ entries
    // of the first wave: p, log2 p and the z they name; in LDS p, z, the id and the owner's list
    float p[J], lp[J], xe[J];
    float tot = 0.0f;
    bool bad = false, any = false, many = false;
    if (first) {
        float L2;
        float tm = -INFINITY;
        if (a.teacher_lse) {
            tm = 0.0f;
            L2 = a.teacher_lse[r] * kLog2e;
        } else {
#pragma unroll
            for (int i = 0; i < J; ++i)
                if (id[i] >= 0) tm = fmaxf(tm, tv[i]);
            tm = wave_max(tm);
            if (tm == -INFINITY) tm = 0.0f;
            float ts = 0.0f;
#pragma unroll
            for (int i = 0; i < J; ++i)
                if (id[i] >= 0) ts += ex2((tv[i] - tm) * c);
            ts = wave_sum(ts);
            L2 = ts == 0.0f ? 0.0f : __builtin_amdgcn_logf(ts);
        }
        if (kDz) {
#pragma unroll
            for (int i = 0; i < NW; ++i) s_head[gi][i * 64 + lane] = -1;
#pragma unroll
            for (int i = 0; i < NC / 64; ++i) s_count[gi][i * 64 + lane] = 0;
            __builtin_amdgcn_wave_barrier();
        }
#pragma unroll
        for (int i = 0; i < J; ++i) {
            const int j = i * 64 + lane;
            bad |= id[i] == INT32_MAX;
            lp[i] = fmaf(tv[i] - tm, c, -L2);
            // (an entry of -inf is 0 whatever L: the logsumexp of a teacher row that is masked whole is -inf too)
            p[i] = id[i] < 0 || tv[i] == -INFINITY ? 0.0f : ex2(lp[i]);
            any |= !(p[i] == 0.0f);
            tot += p[i];
            xe[i] = 0.0f;
            const bool real = id[i] >= 0 && id[i] < a.vocab;
            if (MODE == kJoin)
                xe[i] = real ? a.xs[r * a.top + j] : 0.0f;
            else if (real)
                xe[i] = D::up(z[id[i]]);
            if (kDz) {
                s_p[gi][j] = p[i];
                s_x[gi][j] = xe[i];
                s_id[gi][j] = id[i];
                const int e = id[i] - h, v = e / E;
                const bool lone = e < 0 || e >= shift;
                // (an entry of p = 0 changes nothing: lists padded with id 0 would all be one thread's)
                if (real && !(p[i] == 0.0f) && (lone ? singles != 0 : v >= v0 && v < v1)) {
                    const int owner = !lone ? (v - v0) % NT : e < 0 ? id[i] : id[i] - shift;
                    s_next[gi][j] = atomicExch(&s_head[gi][owner], j);
                    many |= atomicAdd(&s_count[gi][owner % NC], 1) >= most;
                }
            }
        }
        tot = wave_sum(tot);
        if (__any(bad)) tot = NAN;
        any = __any(any) || tot != tot;
        many = __any(many);
    }
    if (MODE == kPart && slice == 0 && w == 0) {
        for (int j = lane; j < a.top; j += 64) {
            const int64_t k = a.ids64 ? ((const int64_t *)a.ids)[r * a.top + j] : ((const int32_t *)a.ids)[r * a.top + j];
            a.xs[r * a.top + j] = k >= 0 && k < a.vocab ? D::up(z[k]) : 0.0f;
        }
    }

    // -------------------------------------------------- softmax statistics
    if (kStats) {
        m = x1;
        if (NV) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (i >= NV / 2) x[i].mask(i * NT + u < nvec);
                x[i].forget();
                m = fmaxf(m, x[i].max());
            }
            m = wave_max(m);
            const float mu = m == -INFINITY ? 0.0f : m;
            s = single ? ex2((x1 - mu) * c) : 0.0f;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                x[i].forget();
                s += x[i].sum(mu, c);
            }
            s = wave_sum(s);
        } else {
            s = single ? ex2((x1 - (x1 == -INFINITY ? 0.0f : x1)) * c) : 0.0f;
            // 4 vectors at a time: their maximum joins the running one first
            for (int v = v0 + u; v < v1; v += 4 * NT) {
                V y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (v + i * NT < v1) y[i].load(z + h + (v + i * NT) * E);
                float n = m;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (v + i * NT < v1) n = fmaxf(n, y[i].max());
                const float nu = n == -INFINITY ? 0.0f : n;
                s *= m == -INFINITY ? (s != s ? s : 0.0f) : ex2((m - nu) * c);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (v + i * NT < v1) s += y[i].sum(nu, c);
                m = n;
            }
            const float wm = wave_max(m), wu = wm == -INFINITY ? 0.0f : wm;
            s = wave_sum(s * (m == -INFINITY ? (s != s ? s : 0.0f) : ex2((m - wu) * c)));
            m = wm;
        }
    }
    if (NW > 1 && kStats && lane == 0) sm[gi][w] = m, ss[gi][w] = s;
    if (NW > 1 && first && lane == 0) s_tot[gi][0] = tot, s_tot[gi][1] = any ? 1.0f : 0.0f, s_many[gi] = many;
    sync();
    if (NW > 1 && kEntries && !first) tot = s_tot[gi][0], any = s_tot[gi][1] != 0.0f;
    auto join = [&](float m1, float s1) {
        const float n = fmaxf(m, m1), nu = n == -INFINITY ? 0.0f : n;
        s = (m == -INFINITY ? (s != s ? s : 0.0f) : s * ex2((m - nu) * c)) +
            (m1 == -INFINITY ? (s1 != s1 ? s1 : 0.0f) : s1 * ex2((m1 - nu) * c));
        m = n;
    };
    if (kStats && NW > 1) {
        m = sm[gi][0], s = ss[gi][0];
#pragma unroll
        for (int i = 1; i < NW; ++i) join(sm[gi][i], ss[gi][i]);
    }
    if (MODE == kPart) {
        if (u == 0) a.part[r * a.slices + slice] = make_float2(m, s);
        return;
    }
    if (MODE == kJoin) {
        const float2 *q = a.part + r * a.slices;
        m = q[0].x, s = q[0].y;
        for (int i = 1; i < a.slices; ++i) join(q[i].x, q[i].y);
    }
    float l2;
    if (MODE == kGrad) {
        const float *st = a.stats + r * 4;
        m = st[0], l2 = st[1], tot = st[2];
        any = tot != 0.0f;
    } else {
        if (m == -INFINITY) m = 0.0f;
        l2 = s == 0.0f ? 0.0f : __builtin_amdgcn_logf(s);
        if (!any) tot = 0.0f;
        if (any && l2 != l2) tot = NAN;
    }

    // ---------------------------------------------------------------- loss
    if (MODE != kGrad && first && slice == 0) {
        float l = 0.0f;
#pragma unroll
        for (int i = 0; i < J; ++i)
            if (!(p[i] == 0.0f)) l += p[i] * (lp[i] - fmaf(xe[i] - m, c, -l2));
        l = wave_sum(l);
        if (tot != tot) l = NAN;
        if (lane == 0) {
            a.loss[r] = any ? a.t * a.t * kLn2 * l : 0.0f;
            if (a.stats) *reinterpret_cast<f32x4 *>(a.stats + r * 4) = (f32x4){m, l2, tot, 0.0f};
        }
    }

    // ------------------------------------------------------------ gradient
    if (kDz) {
        if (MODE == kJoin && !a.dz) return;
        T *dz = (T *)a.dz + r * a.ldd;
        const float g = a.t * (a.row_scale ? a.row_scale[r * a.scale_stride] : 1.0f), f = g * tot;
        // (without an entry that counts every gradient is 0, not 0 times what may be NaN)
        if (NV && MODE == kBoth) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                x[i].forget();
                if (any)
                    x[i].grad(m, c, l2, f);
                else
                    x[i] = V{};
                if (i < NV / 2 || i * NT + u < nvec) x[i].store(dz + h + (i * NT + u) * E);
            }
        } else {
            for (int v = v0 + u; v < v1; v += 4 * NT) {
                V y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (v + i * NT < v1) y[i].load(z + h + (v + i * NT) * E);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (v + i * NT < v1) {
                        if (any)
                            y[i].grad(m, c, l2, f);
                        else
                            y[i] = V{};
                        y[i].store(dz + h + (v + i * NT) * E);
                    }
            }
        }
        if (single) dz[at1] = D::down(any ? f * ex2(fmaf(x1 - m, c, -l2)) : 0.0f);
        if (!any || tot != tot) return;
        auto place = [&](int j, int k, float sum) {
            const float q = ex2(fmaf(s_x[gi][j] - m, c, -l2));
            dz[k] = D::down(g * (tot * q - sum));
        };
        // this thread's entries: of several with one id the first adds up all, in their order
        if (s_head[gi][u] < 0) return;
        if (NW > 1) many = s_many[gi];  // (read here: kept in a register from the barrier on, 131071 outputs take 1.5 % more)
        if (__builtin_expect(!many, 1)) {
            for (int j = s_head[gi][u]; j >= 0; j = s_next[gi][j]) {
                const int k = s_id[gi][j];
                bool lead = true;
                for (int i = s_head[gi][u]; i >= 0; i = s_next[gi][i]) lead &= !(s_id[gi][i] == k && i < j);
                if (!lead) continue;
                float sum = 0.0f;
                for (int at = j; at < KM;) {
                    sum += s_p[gi][at];
                    int next = KM;
                    for (int i = s_head[gi][u]; i >= 0; i = s_next[gi][i])
                        if (s_id[gi][i] == k && i > at && i < next) next = i;
                    at = next;
                }
                place(j, k, sum);
            }
            return;
        }
        // a long list: 16 entries at a time, and those found are struck out (an id has one owner: no other thread
        // looks for it)
        for (int j = s_head[gi][u]; j >= 0; j = s_next[gi][j]) {
            const int k = s_id[gi][j];
            if (k < 0) continue;
            float sum = 0.0f;
            for (int i = 0; i < a.top; i += 16) {
                i32x4 v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const i32x4 *>(&s_id[gi][i + e * 4]);
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (v[e / 4][e % 4] == k) {
                        sum += s_p[gi][i + e];
                        s_id[gi][i + e] = -1;
                    }
            }
            place(j, k, sum);
        }
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
        c += stats[4 * r + 2] == 0.0f ? 0.0f : 1.0f;
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

// A launch has fewer than 2^32 threads: more rows take another one.
template <class D, int NT, int NV, int KM, Mode MODE>
static int launch(DistillArgs a, hipStream_t st) {
    constexpr int G = NT < 256 ? 256 / NT : 1, threads = NT < 256 ? 256 : NT;
    const int64_t each = MODE == kPart || MODE == kJoin || MODE == kGrad ? a.slices : 1;  // groups a row
    const int64_t most = (int64_t)(UINT32_MAX / threads) * G / each;
    for (int64_t left = a.rows; left > 0;) {
        const int64_t n = a.rows = std::min(left, most);
        hipLaunchKernelGGL((k_distill<D, NT, NV, KM, MODE>), dim3((unsigned)((n * each + G - 1) / G)), dim3(threads), 0, st, a);
        LIRA_HIP_TRY(hipGetLastError());
        if ((left -= n) == 0) break;
        a.z = (const typename D::T *)a.z + n * a.ldz;
        a.ids = (const char *)a.ids + n * a.top * (a.ids64 ? 8 : 4);
        a.tv += n * a.top;
        if (a.teacher_lse) a.teacher_lse += n;
        if (a.row_scale) a.row_scale += n * a.scale_stride;
        if (a.loss) a.loss += n;
        if (a.stats) a.stats += n * 4;
        if (a.dz) a.dz = (typename D::T *)a.dz + n * a.ldd;
        if (a.part) a.part += n * a.slices;
        if (a.xs) a.xs += n * a.top;
    }
    return LIRA_OK;
}

// Slices of a row, where there are few long ones: 192 rows keep the 256 compute units busy by themselves
// (131072 outputs in bf16, us: 128 rows 28 in slices, 33 in whole rows; 256 rows 51 and 33).
static constexpr int kFewRows = 192;
static int64_t distill_slices(int64_t rows, int64_t vecs) {
    return rows < 1 || rows >= kFewRows ? 1 : std::max<int64_t>(1, (vecs + kSliceVecs - 1) / kSliceVecs);
}

template <class D>
static int run(DistillArgs a, bool grad_only, hipStream_t st) {
    const int64_t vecs = a.vocab / Vec<D>::E;
    const bool few = a.top <= 64;
    // A row to a wave where rows alone fill the chip or a wave reads it in two loads, else to a workgroup, which gets
    // it done sooner (loss and gradient, us by waves and by workgroups: 64 x 4096 bf16 8.4 and 5.7, 1024 x 8192
    // bf16 16.5 and 13.3, 16384 x 1024 fp32 31.7 and 41.8).
    const bool waves = vecs <= 64 * 2 || a.rows >= 4096;
    if (grad_only) {
        if (waves && vecs <= 64 * 16 && few) return launch<D, 64, 0, 64, kGrad>(a, st);
        a.slices = (int)std::max<int64_t>(1, (vecs + kSliceVecs - 1) / kSliceVecs);
        return few ? launch<D, 256, 0, 64, kGrad>(a, st) : launch<D, 256, 0, kMaxTop, kGrad>(a, st);
    }
    if (a.slices > 1) {
        if (int rc = launch<D, 256, 0, 64, kPart>(a, st)) return rc;
        return few ? launch<D, 256, 0, 64, kJoin>(a, st) : launch<D, 256, 0, kMaxTop, kJoin>(a, st);
    }
    if (!a.dz) {
        if (waves && vecs <= 64 * 16 && few) return launch<D, 64, 0, 64, kLoss>(a, st);
        return few ? launch<D, 256, 0, 64, kLoss>(a, st) : launch<D, 256, 0, kMaxTop, kLoss>(a, st);
    }
    if (!few) return launch<D, 256, 0, kMaxTop, kBoth>(a, st);
    // (the row in registers)
    if (vecs < 1) return launch<D, 64, 0, 64, kBoth>(a, st);
    if (vecs <= 64) return launch<D, 64, 1, 64, kBoth>(a, st);
    if (vecs <= 64 * 2) return launch<D, 64, 2, 64, kBoth>(a, st);
    if (waves) {
        if (vecs <= 64 * 4) return launch<D, 64, 4, 64, kBoth>(a, st);
        if (vecs <= 64 * 8) return launch<D, 64, 8, 64, kBoth>(a, st);
    } else {
        if (vecs <= 256) return launch<D, 256, 1, 64, kBoth>(a, st);
        if (vecs <= 256 * 2) return launch<D, 256, 2, 64, kBoth>(a, st);
    }
    if (vecs <= 256 * 4) return launch<D, 256, 4, 64, kBoth>(a, st);
    if (vecs <= 256 * 8) return launch<D, 256, 8, 64, kBoth>(a, st);
    if (vecs <= 256 * 16) return launch<D, 256, 16, 64, kBoth>(a, st);
    if (vecs <= 1024 * 8) return launch<D, 1024, 8, 64, kBoth>(a, st);
    if (vecs <= 1024 * 16) return launch<D, 1024, 16, 64, kBoth>(a, st);
    return launch<D, 256, 0, 64, kBoth>(a, st);
}
static int run(const DistillArgs &a, int dtype, bool grad_only, hipStream_t st) {
    if (dtype == LIRA_DTYPE_F32) return run<F32>(a, grad_only, st);
    if (dtype == LIRA_DTYPE_BF16) return run<BF16>(a, grad_only, st);
    return run<F16>(a, grad_only, st);
}

static int64_t vectors(int64_t vocab, int dtype) { return vocab / (dtype == LIRA_DTYPE_F32 ? 4 : 8); }

}  // namespace lira

using namespace lira;

static int check_distill(const DistillArgs &a, int dtype, int ids_bits) {
    if (dtype < LIRA_DTYPE_F32 || dtype > LIRA_DTYPE_F16) return fail(LIRA_EINVAL, "unknown dtype");
    if (ids_bits != 32 && ids_bits != 64) return fail(LIRA_EINVAL, "ids_bits must be 32 or 64");
    if (a.rows < 0 || a.vocab <= 0) return fail(LIRA_EINVAL, "rows must be >= 0 and vocab >= 1");
    if (a.top < 1) return fail(LIRA_EINVAL, "top must be >= 1");
    if (a.top > kMaxTop) return fail(LIRA_EUNSUPPORTED, "top must be at most 1024");
    if (a.ldz < a.vocab || (a.dz && a.ldd < a.vocab)) return fail(LIRA_EINVAL, "row strides must be at least vocab");
    if (!(a.t > 0.0f) || !(a.t < INFINITY) || !(kLog2e / a.t < INFINITY))
        return fail(LIRA_EINVAL, "temperature must be positive and finite");
    if (!(a.t * a.t < INFINITY) || a.t * a.t < FLT_MIN)  // (the loss's factor)
        return fail(LIRA_EINVAL, "temperature must have a square that fp32 holds, 1.1e-19 to 1.8e19");
    if (a.row_scale && (a.scale_stride < 0 || a.scale_stride > 1))
        return fail(LIRA_EINVAL, "scale_stride must be 0 or 1");
    if (a.vocab >= INT32_MAX) return fail(LIRA_EUNSUPPORTED, "vocab must be less than 2147483647");
    if (a.rows > INT32_MAX) return fail(LIRA_EUNSUPPORTED, "too many rows");
    if (a.rows > 0 && (!a.z || !a.ids || !a.tv)) return fail(LIRA_EINVAL, "NULL buffer");
    return LIRA_OK;
}

extern "C" {

int lira_distill_workspace_size(int64_t rows, int64_t vocab, int64_t top, int dtype, size_t *bytes) {
    if (!bytes) return fail(LIRA_EINVAL, "NULL buffer");
    if (dtype < LIRA_DTYPE_F32 || dtype > LIRA_DTYPE_F16) return fail(LIRA_EINVAL, "unknown dtype");
    if (rows < 0 || vocab <= 0 || top < 1) return fail(LIRA_EINVAL, "bad shape");
    const int64_t n = distill_slices(rows, vectors(vocab, dtype));
    *bytes = n > 1 ? (size_t)(rows * (n * sizeof(float2) + top * sizeof(float))) : 0;
    return LIRA_OK;
}

int lira_distill_topk(const void *z, int dtype, int64_t rows, int64_t vocab, int64_t ldz, const void *ids, int ids_bits,
                      const float *teacher, int64_t top, float temperature, const float *teacher_lse, float *loss,
                      float *stats, const float *row_scale, int64_t scale_stride, void *dz, int64_t ldd,
                      void *workspace, size_t workspace_bytes, void *stream) {
    DistillArgs a = {z, rows, vocab, ldz, ids, teacher, (int)(top < 0 ? 0 : top > INT32_MAX ? INT32_MAX : top),
                     ids_bits == 64, teacher_lse, temperature, row_scale, scale_stride, loss, stats, dz, ldd, 1,
                     nullptr, nullptr};
    if (int rc = check_distill(a, dtype, ids_bits)) return rc;
    if (rows == 0) return LIRA_OK;
    if (!loss) return fail(LIRA_EINVAL, "NULL buffer");
    if (((uintptr_t)stats & 15) != 0) return fail(LIRA_EINVAL, "stats must be 16-byte aligned");
    size_t need = 0;
    if (int rc = lira_distill_workspace_size(rows, vocab, top, dtype, &need)) return rc;
    if (need) {
        if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15) != 0)
            return fail(LIRA_EINVAL, "workspace too small (lira_distill_workspace_size) or not 16-byte aligned");
        a.slices = (int)distill_slices(rows, vectors(vocab, dtype));
        a.part = (float2 *)workspace;
        a.xs = (float *)(a.part + rows * a.slices);
    }
    return run(a, dtype, false, (hipStream_t)stream);
}

int lira_distill_topk_backward(const void *z, int dtype, int64_t rows, int64_t vocab, int64_t ldz, const void *ids,
                               int ids_bits, const float *teacher, int64_t top, float temperature,
                               const float *teacher_lse, const float *stats, const float *row_scale,
                               int64_t scale_stride, void *dz, int64_t ldd, void *stream) {
    const DistillArgs a = {z, rows, vocab, ldz, ids, teacher, (int)(top < 0 ? 0 : top > INT32_MAX ? INT32_MAX : top),
                           ids_bits == 64, teacher_lse, temperature, row_scale, scale_stride, nullptr,
                           const_cast<float *>(stats), dz, ldd, 1, nullptr, nullptr};
    if (int rc = check_distill(a, dtype, ids_bits)) return rc;
    if (rows == 0) return LIRA_OK;
    if (!stats || !dz) return fail(LIRA_EINVAL, "NULL buffer");
    if (((uintptr_t)stats & 15) != 0) return fail(LIRA_EINVAL, "stats must be 16-byte aligned");
    return run(a, dtype, true, (hipStream_t)stream);
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
