/*
 * lira_oracle.c -- CPU restatement of LIRA's query-time hot path.
 *
 * TEST INFRASTRUCTURE ONLY.  This file is the parity checker for the HIP
 * path in lira-ann-search_amd/csrc and the CPU baseline leg of bench.py.
 * Only tests/, __graft_entry__.smoke() and bench.py's cpu_baseline may load
 * it; the product path never does.
 *
 * Every function restates one piece of the reference (file:line into
 * qfshen23/LIRA-ANN-search @ 2025-11-28):
 *
 *   oracle_l2_sq              search.cpp:253-260  sequential fp32, no FMA
 *   oracle_ip                 search.cpp:263-269  sequential fp32, no FMA
 *   oracle_centroid_dist      search.cpp:220-235  sqrt(l2) to every centroid
 *   oracle_standardize        search.cpp:238-250  (d - mean) / scale, scale 0 -> 1
 *   oracle_build_csr          search.cpp:366-385  bucket -> sorted unique gids
 *   oracle_probe_threshold    search.cpp:447-466  score >= thr, argmax fallback
 *                             LIRA_smallscale.py:206 (score > thr, no fallback)
 *   oracle_probe_nearest      IVF nprobe ("nearest-nprobe" probe)
 *   oracle_scan_topk          search.cpp:471-514  scan + top-k, canonical order
 *   oracle_scan_per_partition LIRA_smallscale.py:145-174 (per (q, bucket) top-k)
 *
 * Numerics: must be compiled with -ffp-contract=off (see oracle/Makefile) so
 * that `acc += diff * diff` rounds the product before the add, exactly like
 * the reference binary (subps/mulps then sequential addss).
 *
 * Canonical top-k order: ascending (score, gid) where score = l2_sq for L2
 * and score = -ip for inner product (search.cpp:483-488).  The reference's
 * nth_element output is unordered and breaks boundary ties arbitrarily; this
 * restatement fixes the order so set equality with the reference holds
 * whenever the k-th boundary is not a tie.
 */
#include <math.h>
#include <stdint.h>
#include <stdlib.h>
#include <string.h>
#ifdef _OPENMP
#include <omp.h>
#endif

#define ORACLE_L2 0
#define ORACLE_IP 1

/* search.cpp:253-260 */
float oracle_l2_sq(const float *a, const float *b, int64_t dim) {
    float d = 0.0f;
    for (int64_t j = 0; j < dim; ++j) {
        float diff = a[j] - b[j];
        d += diff * diff;
    }
    return d;
}

/* search.cpp:263-269 */
float oracle_ip(const float *a, const float *b, int64_t dim) {
    float s = 0.0f;
    for (int64_t j = 0; j < dim; ++j) s += a[j] * b[j];
    return s;
}

/* search.cpp:220-235, batched over nq queries: out[q*B + c] */
void oracle_centroid_dist(const float *q, int64_t nq, const float *cent, int64_t nb,
                          int64_t dim, float *out) {
#pragma omp parallel for schedule(static)
    for (int64_t i = 0; i < nq; ++i) {
        for (int64_t c = 0; c < nb; ++c) {
            float dist = 0.0f;
            const float *x = q + i * dim, *y = cent + c * dim;
            for (int64_t j = 0; j < dim; ++j) {
                float diff = x[j] - y[j];
                dist += diff * diff;
            }
            out[i * nb + c] = sqrtf(dist);
        }
    }
}

/* search.cpp:238-250, in place over an (n, nb) matrix */
void oracle_standardize(float *dist, int64_t n, int64_t nb, const float *mean,
                        const float *scale) {
    for (int64_t i = 0; i < n; ++i)
        for (int64_t b = 0; b < nb; ++b) {
            float s = scale[b];
            if (s == 0.0f) s = 1.0f;
            dist[i * nb + b] = (dist[i * nb + b] - mean[b]) / s;
        }
}

static int cmp_i32(const void *a, const void *b) {
    int32_t x = *(const int32_t *)a, y = *(const int32_t *)b;
    return (x > y) - (x < y);
}

/*
 * search.cpp:366-385.  data_2_bkt is (n, n_mul) int32 with -1 = empty slot.
 * offsets (nb+1) and ids (capacity n*n_mul) are caller-allocated.  Returns the
 * total number of ids, or -1 when a bucket id is >= nb (search.cpp:375-377).
 */
int64_t oracle_build_csr(const int32_t *d2b, int64_t n, int64_t n_mul, int64_t nb,
                         int64_t *offsets, int32_t *ids) {
    int64_t *cnt = (int64_t *)calloc((size_t)nb + 1, sizeof(int64_t));
    for (int64_t i = 0; i < n * n_mul; ++i) {
        int32_t b = d2b[i];
        if (b < 0) continue;
        if (b >= nb) { free(cnt); return -1; }
        cnt[b + 1]++;
    }
    for (int64_t b = 0; b < nb; ++b) cnt[b + 1] += cnt[b];
    int64_t *cur = (int64_t *)malloc(sizeof(int64_t) * (size_t)nb);
    memcpy(cur, cnt, sizeof(int64_t) * (size_t)nb);
    for (int64_t i = 0; i < n; ++i)
        for (int64_t j = 0; j < n_mul; ++j) {
            int32_t b = d2b[i * n_mul + j];
            if (b < 0) continue;
            ids[cur[b]++] = (int32_t)i;
        }
    /* sort + unique per bucket, then compact */
    int64_t out = 0;
    offsets[0] = 0;
    for (int64_t b = 0; b < nb; ++b) {
        int64_t s = cnt[b], e = cnt[b + 1];
        qsort(ids + s, (size_t)(e - s), sizeof(int32_t), cmp_i32);
        for (int64_t i = s; i < e; ++i) {
            if (i > s && ids[i] == ids[i - 1]) continue;
            ids[out++] = ids[i];
        }
        offsets[b + 1] = out;
    }
    free(cur);
    free(cnt);
    return out;
}

/*
 * search.cpp:447-466 (strict=0: score >= thr, argmax fallback with first max)
 * LIRA_smallscale.py:206 (strict=1: score > thr, no fallback).
 * out is (n, nb) int32 padded with -1, buckets in ascending order; nprobe_out
 * receives the per-row count.
 */
void oracle_probe_threshold(const float *scores, int64_t n, int64_t nb, float thr,
                            int strict, int32_t *out, int32_t *nprobe_out) {
    for (int64_t i = 0; i < n; ++i) {
        const float *s = scores + i * nb;
        int32_t *o = out + i * nb;
        int32_t m = 0;
        for (int64_t b = 0; b < nb; ++b) {
            int take = strict ? (s[b] > thr) : (s[b] >= thr);
            if (take) o[m++] = (int32_t)b;
        }
        if (m == 0 && !strict) {
            int32_t best = 0;
            float bs = s[0];
            for (int64_t b = 1; b < nb; ++b)
                if (s[b] > bs) { bs = s[b]; best = (int32_t)b; }
            o[m++] = best;
        }
        for (int64_t b = m; b < nb; ++b) o[b] = -1;
        if (nprobe_out) nprobe_out[i] = m;
    }
}

/* (value, index) ascending; exact, deterministic */
typedef struct { float v; int64_t id; } pair_t;

static int pair_less(pair_t a, pair_t b) {
    return a.v < b.v || (a.v == b.v && a.id < b.id);
}

/*
 * IVF nearest-nprobe selection: the nprobe smallest dist (ties -> smaller b),
 * written in ascending (dist, b) order.
 */
void oracle_probe_nearest(const float *dist, int64_t n, int64_t nb, int64_t nprobe,
                          int32_t *out) {
    for (int64_t i = 0; i < n; ++i) {
        const float *d = dist + i * nb;
        int32_t *o = out + i * nprobe;
        pair_t best[4096];
        int64_t m = 0, cap = nprobe < nb ? nprobe : nb;
        if (cap > 4096) cap = 4096;
        for (int64_t b = 0; b < nb; ++b) {
            pair_t p = {d[b], b};
            if (m < cap) {
                int64_t j = m++;
                while (j > 0 && pair_less(p, best[j - 1])) { best[j] = best[j - 1]; --j; }
                best[j] = p;
            } else if (pair_less(p, best[cap - 1])) {
                int64_t j = cap - 1;
                while (j > 0 && pair_less(p, best[j - 1])) { best[j] = best[j - 1]; --j; }
                best[j] = p;
            }
        }
        for (int64_t j = 0; j < nprobe; ++j) o[j] = j < m ? (int32_t)best[j].id : -1;
    }
}

/* bounded sorted insertion list of the k smallest (score, gid) */
typedef struct {
    pair_t *a;
    int64_t n, cap;
} topk_t;

static void topk_push(topk_t *t, float v, int64_t id) {
    pair_t p = {v, id};
    if (t->n == t->cap && !pair_less(p, t->a[t->n - 1])) return;
    int64_t j = t->n < t->cap ? t->n++ : t->cap - 1;
    while (j > 0 && pair_less(p, t->a[j - 1])) { t->a[j] = t->a[j - 1]; --j; }
    t->a[j] = p;
}

static float score_of(const float *q, const float *v, int64_t dim, int metric) {
    return metric == ORACLE_IP ? -oracle_ip(q, v, dim) : oracle_l2_sq(q, v, dim);
}

/*
 * search.cpp:471-514 for a batch.  Buckets are stored as in search.cpp:387-403:
 * vecs holds bucket b's rows contiguously at rows offsets[b]..offsets[b+1],
 * ids the matching global ids.  probe is (nq, nprobe_max) int32, -1 padded.
 *
 * dedup=0 reproduces the reference multiset (a gid replicated in two probed
 * buckets may occupy two slots, search.cpp:496-514); dedup=r>0 keeps each gid
 * once, r being the largest number of buckets one gid sits in.  Outputs are faiss-ordered: D ascending for L2 (squared distance),
 * descending inner product for IP; pads are (+inf, -1) for L2 and (-inf, -1)
 * for IP.  ncand (nullable) receives search.cpp's cmp_for_query.
 */
void oracle_scan_topk(const float *q, int64_t nq, int64_t dim, const int64_t *offsets,
                      const int32_t *ids, const float *vecs, const int32_t *probe,
                      int64_t nprobe_max, int64_t k, int metric, int dedup, float *out_D,
                      int64_t *out_I, int64_t *ncand) {
    /* dedup: 0 = off (reference multiset); r > 0 = on, r = the most buckets
     * any one gid sits in (n_mul), which bounds the slots a winner can take */
#pragma omp parallel for schedule(dynamic, 1)
    for (int64_t i = 0; i < nq; ++i) {
        const float *qi = q + i * dim;
        int64_t cap = dedup > 0 ? k * dedup : k;
        pair_t *buf = (pair_t *)malloc(sizeof(pair_t) * (size_t)(cap > 0 ? cap : 1));
        topk_t t = {buf, 0, cap};
        int64_t cmp = 0;
        for (int64_t s = 0; s < nprobe_max; ++s) {
            int32_t b = probe[i * nprobe_max + s];
            if (b < 0) continue;
            for (int64_t r = offsets[b]; r < offsets[b + 1]; ++r)
                topk_push(&t, score_of(qi, vecs + r * dim, dim, metric), ids[r]);
            cmp += offsets[b + 1] - offsets[b];
        }
        int64_t m = 0;
        for (int64_t j = 0; j < t.n && m < k; ++j) {
            if (dedup && m > 0 && buf[j].id == out_I[i * k + m - 1]) continue;
            out_D[i * k + m] = metric == ORACLE_IP ? -buf[j].v : buf[j].v;
            out_I[i * k + m] = buf[j].id;
            ++m;
        }
        for (; m < k; ++m) {
            out_D[i * k + m] = metric == ORACLE_IP ? -INFINITY : INFINITY;
            out_I[i * k + m] = -1;
        }
        if (ncand) ncand[i] = cmp;
        free(buf);
    }
}

/*
 * LIRA_smallscale.py:145-174 (get_cmp_recall): the k best of every probed
 * bucket on its own.  out_D/out_I are (nq, nprobe_max, k); an unprobed slot
 * or a bucket with fewer than k rows is padded with (+-inf, -1) -- the
 * reference would wrap a -1 label to the bucket's last id (Appendix A), the
 * restatement does not.
 */
void oracle_scan_per_partition(const float *q, int64_t nq, int64_t dim,
                               const int64_t *offsets, const int32_t *ids,
                               const float *vecs, const int32_t *probe, int64_t nprobe_max,
                               int64_t k, int metric, float *out_D, int64_t *out_I) {
#pragma omp parallel for schedule(dynamic, 1)
    for (int64_t i = 0; i < nq; ++i) {
        pair_t *buf = (pair_t *)malloc(sizeof(pair_t) * (size_t)(k > 0 ? k : 1));
        for (int64_t s = 0; s < nprobe_max; ++s) {
            int32_t b = probe[i * nprobe_max + s];
            topk_t t = {buf, 0, k};
            if (b >= 0)
                for (int64_t r = offsets[b]; r < offsets[b + 1]; ++r)
                    topk_push(&t, score_of(q + i * dim, vecs + r * dim, dim, metric), ids[r]);
            float *D = out_D + (i * nprobe_max + s) * k;
            int64_t *I = out_I + (i * nprobe_max + s) * k;
            for (int64_t j = 0; j < k; ++j) {
                if (j < t.n) {
                    D[j] = metric == ORACLE_IP ? -buf[j].v : buf[j].v;
                    I[j] = buf[j].id;
                } else {
                    D[j] = metric == ORACLE_IP ? -INFINITY : INFINITY;
                    I[j] = -1;
                }
            }
        }
        free(buf);
    }
}

int oracle_num_threads(void) {
#ifdef _OPENMP
    return omp_get_max_threads();
#else
    return 1;
#endif
}

void oracle_set_num_threads(int n) {
#ifdef _OPENMP
    omp_set_num_threads(n);
#else
    (void)n;
#endif
}
