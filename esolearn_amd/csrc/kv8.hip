// An int8 KV cache of one layer and one sequence: rows are quantised as they
// are written, one f32 scale per row and head, and read back, or read by the
// attention (tree.hip) as they are.
//
// x [hd] -> s = f32(max|x| / 127), q = x / s rounded to the nearest integer,
// halves away from zero (the rounding of quantize_symmetric, quantize.rs:16-32,
// but of the exact quotient, where that rounds x * (1 / s) twice), |q| <= 127;
// the value that q stands for is f32(q) * s.  A row of zeros has s = 0.  A row
// with an infinity or a NaN has s = NaN: it reads back as NaN, whole.
//
// Layout, for the matrix-core attention: K [head][row][hdp] bytes, a lane's 16
// bytes of a row being an operand of the products q.k; V [head][row / 64][hdp]
// [64], the 64 rows of a block side by side per dimension, in the order in
// which a wave's scores of those rows lie in its lanes (kv8_perm), so that a
// lane's 16 bytes make an operand of the products p.v; V's bytes are q + 128.
// hdp = hd rounded up to 16.  Scales [head][row].
#include <cmath>
#include <new>

#include "kdev.h"
#include "kv8.h"

namespace scry {

int kv8_batch(const char *what, const scry_kv8 *caches, int n_seq, const DraftBatch &d, int rows, bool distinct,
              Kv8Batch *b) {
    if (!caches) return set_error(SCRY_ERR_INVALID, "%s: null caches", what);
    *b = Kv8Batch{};
    for (int s = 0; s < n_seq; s++) {
        const scry_kv8 c = caches[s];
        if (!c || !c->block) return set_error(SCRY_ERR_INVALID, "%s: null cache %d", what, s);
        if (c->n_kv != caches[0]->n_kv || c->hd != caches[0]->hd)
            return set_error(SCRY_ERR_INVALID, "%s: cache %d has %d heads of %d, cache 0 %d of %d", what, s, c->n_kv, c->hd,
                             caches[0]->n_kv, caches[0]->hd);
        if (d.len[s] > c->max_seq - rows)
            return set_error(SCRY_ERR_RANGE, "%s: rows [%d, %d) of cache %d, which holds %d", what, d.len[s],
                             d.len[s] + rows, s, c->max_seq);
        for (int t = 0; distinct && t < s; t++)
            if (caches[t] == c) return set_error(SCRY_ERR_INVALID, "%s: caches %d and %d are the same", what, t, s);
        b->k[s] = c->k;
        b->v[s] = c->v;
        b->ks[s] = c->ks;
        b->vs[s] = c->vs;
        b->rows_p[s] = c->rows_p;
    }
    b->n_kv = caches[0]->n_kv;
    b->hd = caches[0]->hd;
    b->hdp = caches[0]->hdp;
    return SCRY_OK;
}

namespace {

using namespace dev;

struct Kv8Rows {
    Kv8Batch c;
    int start[PF_MAX_SEQS];
    int rows;
};

// |x| / s, s > 0, to the nearest integer, halves up, at most 127.  f32 division
// may round a quotient up to an integer; the remainder x - k s is exact in f32
// (an fma of a multiple of ulp(s) below 2^24 ulp(s)) and decides.
__device__ __forceinline__ int steps_of(float x, float s) {
    const float ax = fabsf(x);
    const float k = floorf(ax / s);
    const float e = fmaf(-k, s, ax);
    const float r = e < 0.f ? k : 2.f * e >= s ? k + 1.f : k;
    const int q = (int)fminf(r, 127.f);
    return x < 0.f ? -q : q;
}

// blockIdx.y: K or V; blockIdx.z: the sequence.  G lanes hold a vector.
template <int G>
__global__ __launch_bounds__(256) void k_kv8_write(Kv8Rows a, const float *__restrict__ kx, const float *__restrict__ vx) {
    constexpr int NG = 256 / G;
    const int s = blockIdx.z, tid = threadIdx.x, gl = tid % G;
    const bool is_v = blockIdx.y;
    const int n_kv = a.c.n_kv, hd = a.c.hd, hdp = a.c.hdp, rows_p = a.c.rows_p[s];
    const size_t n = (size_t)a.rows * n_kv, at = (size_t)blockIdx.x * NG + tid / G;
    if (at >= n) return;  // whole groups of G lanes leave
    const int r = a.start[s] + (int)(at / n_kv), g = (int)(at % n_kv);
    const float *src = (is_v ? vx : kx) + ((size_t)s * n + at) * hd;
    const bool act = 4 * gl < hd;
    const float4 x = act ? *(const float4 *)(src + 4 * gl) : make_float4(0.f, 0.f, 0.f, 0.f);
    float m = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
    if (!(isfinite(x.x) && isfinite(x.y) && isfinite(x.z) && isfinite(x.w))) m = INFINITY;
#pragma unroll
    for (int off = G / 2; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
    const bool bad = m == INFINITY;
    const float sc = bad ? __builtin_nanf("") : m / 127.f;
    char4 q = make_char4(0, 0, 0, 0);
    if (!bad && sc > 0.f)
        q = make_char4((signed char)steps_of(x.x, sc), (signed char)steps_of(x.y, sc), (signed char)steps_of(x.z, sc),
                       (signed char)steps_of(x.w, sc));
    if (is_v) {
        if (act) {
            int8_t *d = a.c.v[s] + kv8_v_at(rows_p, hdp, g, r, 4 * gl) + kv8_perm(r & 63);
            d[0] = q.x ^ 0x80;
            d[64] = q.y ^ 0x80;
            d[128] = q.z ^ 0x80;
            d[192] = q.w ^ 0x80;
        }
    } else if (act) {
        *(char4 *)(a.c.k[s] + kv8_k_at(rows_p, hdp, g, r) + 4 * gl) = q;
    }
    if (gl == 0) (is_v ? a.c.vs[s] : a.c.ks[s])[(size_t)g * rows_p + r] = sc;
}

template <int G>
__global__ __launch_bounds__(256) void k_kv8_read(Kv8Rows a, float *__restrict__ kx, float *__restrict__ vx) {
    constexpr int NG = 256 / G;
    const int s = blockIdx.z, tid = threadIdx.x, gl = tid % G;
    const bool is_v = blockIdx.y;
    const int n_kv = a.c.n_kv, hd = a.c.hd, hdp = a.c.hdp, rows_p = a.c.rows_p[s];
    const size_t n = (size_t)a.rows * n_kv, at = (size_t)blockIdx.x * NG + tid / G;
    if (at >= n || 4 * gl >= hd) return;
    const int r = a.start[s] + (int)(at / n_kv), g = (int)(at % n_kv);
    const float sc = (is_v ? a.c.vs[s] : a.c.ks[s])[(size_t)g * rows_p + r];
    char4 q;
    if (is_v) {
        const int8_t *d = a.c.v[s] + kv8_v_at(rows_p, hdp, g, r, 4 * gl) + kv8_perm(r & 63);
        q = make_char4((signed char)(d[0] ^ 0x80), (signed char)(d[64] ^ 0x80), (signed char)(d[128] ^ 0x80),
                       (signed char)(d[192] ^ 0x80));
    } else {
        q = *(const char4 *)(a.c.k[s] + kv8_k_at(rows_p, hdp, g, r) + 4 * gl);
    }
    *(float4 *)((is_v ? vx : kx) + ((size_t)s * n + at) * hd + 4 * gl) =
        make_float4((float)q.x * sc, (float)q.y * sc, (float)q.z * sc, (float)q.w * sc);
}

struct Kv8Keep {
    Kv8Batch c;
    int start[PF_MAX_SEQS];
    int count[PF_MAX_SEQS];
    unsigned char path[PF_MAX_SEQS][DRAFT_MAX_TREE];
};

// Row start + path[i] moves to start + i, i ascending.  path[i] >= i ascends,
// so a row is read before a later move writes it if every byte's moves are
// done in order: one thread does them all for its bytes.  Eight rows are read
// ahead of their writes: rows i .. i + 7 are written, and the rows still to be
// read lie at path[i + 8] >= i + 8 or beyond.
__global__ __launch_bounds__(256) void k_kv8_keep(Kv8Keep a) {
    const int g = blockIdx.x, s = blockIdx.z, tid = threadIdx.x;
    const bool is_v = blockIdx.y;
    const int hdp = a.c.hdp, rows_p = a.c.rows_p[s], n = a.count[s], r0 = a.start[s];
    auto move = [&](auto *base, auto at) {
        for (int i = 0; i < n; i += 8) {
            std::remove_reference_t<decltype(*base)> x[8];
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (i + j < n) x[j] = base[at(r0 + a.path[s][i + j])];
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (i + j < n) base[at(r0 + i + j)] = x[j];
        }
    };
    if (is_v) {
        int8_t *v = a.c.v[s];
        for (int d = tid; d < hdp; d += 256)
            move(v, [&](int r) { return kv8_v_at(rows_p, hdp, g, r, d) + kv8_perm(r & 63); });
    } else {
        int *k = (int *)a.c.k[s];
        for (int d = tid; d < hdp / 4; d += 256) move(k, [&](int r) { return kv8_k_at(rows_p, hdp, g, r) / 4 + d; });
    }
    if (tid == 0) move(is_v ? a.c.vs[s] : a.c.ks[s], [&](int r) { return (size_t)g * rows_p + r; });
}

// vectors (row, head) of one sequence per workgroup, by the lanes of a head
template <class F>
int by_lanes(int hd, F f) {
    const int lanes = hd / 4;
    if (lanes <= 4) return f(std::integral_constant<int, 4>{});
    if (lanes <= 8) return f(std::integral_constant<int, 8>{});
    if (lanes <= 16) return f(std::integral_constant<int, 16>{});
    if (lanes <= 32) return f(std::integral_constant<int, 32>{});
    return f(std::integral_constant<int, 64>{});
}

int kv8_rows(const char *what, const scry_kv8 *caches, int n_seq, const int32_t *start, int rows, bool distinct,
             Kv8Rows *a, size_t *n) {
    DraftBatch d;
    SCRY_TRY(draft_batch(what, n_seq, rows, start, nullptr, &d));
    SCRY_TRY(kv8_batch(what, caches, n_seq, d, rows, distinct, &a->c));
    for (int s = 0; s < n_seq; s++) a->start[s] = d.len[s];
    a->rows = rows;
    *n = (size_t)rows * a->c.n_kv;  // vectors of a sequence
    return SCRY_OK;
}

}  // namespace
}  // namespace scry

using namespace scry;

#define API_LOCK std::lock_guard<std::recursive_mutex> _api_lock(scry::api_mutex())

extern "C" {

int scry_hip_kv8_new(int max_seq, int n_kv, int head_dim, scry_kv8 *out) {
    API_LOCK;
    SCRY_REQUIRE_INIT();
    if (!out) return set_error(SCRY_ERR_INVALID, "kv8_new: null output handle");
    *out = nullptr;
    SCRY_TRY(check_heads("kv8_new", 0, n_kv, head_dim));
    if (max_seq <= 0 || max_seq > 0x7fffffff - 64) return set_error(SCRY_ERR_INVALID, "kv8_new: max_seq %d", max_seq);
    DeviceScope dev;
    auto *c = new (std::nothrow) scry_kv8_s;
    if (!c) return set_error(SCRY_ERR_OOM, "host allocation failed");
    c->max_seq = max_seq;
    c->n_kv = n_kv;
    c->hd = head_dim;
    c->hdp = round_up(head_dim, 16);
    c->rows_p = round_up(max_seq, 64);
    const size_t rows = (size_t)n_kv * c->rows_p, plane = rows * c->hdp;
    int rc = dev_alloc((void **)&c->block, 2 * plane + 2 * rows * sizeof(float));
    // rows never written read as zero
    if (!rc) rc = launch_fill_u32((unsigned *)c->block, (2 * plane + 2 * rows * sizeof(float)) / 4, 0u, ctx().stream);
    if (rc) {
        dev_free(c->block);
        delete c;
        return rc;
    }
    c->k = (int8_t *)c->block;
    c->v = c->k + plane;
    c->ks = (float *)(c->v + plane);
    c->vs = c->ks + rows;
    *out = c;
    return SCRY_OK;
}

int scry_hip_kv8_free(scry_kv8 c) {
    API_LOCK;
    if (!c) return SCRY_OK;
    if (ctx().init) {
        DeviceScope dev;
        (void)hipStreamSynchronize(ctx().stream);
        dev_free(c->block);
    } else {
        dev_free(c->block);
    }
    delete c;
    return SCRY_OK;
}

int scry_hip_kv8_write(const scry_kv8 *caches, int n_seq, const int32_t *start, int rows, scry_buf k, scry_buf v) {
    API_LOCK;
    SCRY_REQUIRE_INIT();
    SCRY_TRY(check_f32(k, "kv8_write"));
    SCRY_TRY(check_f32(v, "kv8_write"));
    Kv8Rows a{};
    size_t n = 0;
    SCRY_TRY(kv8_rows("kv8_write", caches, n_seq, start, rows, true, &a, &n));
    if (k->n != n * n_seq * a.c.hd || v->n != k->n) return set_error(SCRY_ERR_INVALID, "kv8_write: shape mismatch");
    DeviceScope dev;
    return by_lanes(a.c.hd, [&](auto g) {
        constexpr int G = decltype(g)::value, NG = 256 / G;
        if ((n + NG - 1) / NG > 0x7fffffff) return set_error(SCRY_ERR_UNSUPPORTED, "kv8_write: %d rows", rows);
        hipLaunchKernelGGL(k_kv8_write<G>, dim3((unsigned)((n + NG - 1) / NG), 2, n_seq), dim3(256), 0, ctx().stream, a, k->d,
                           v->d);
        SCRY_HIP(hipGetLastError());
        return (int)SCRY_OK;
    });
}

int scry_hip_kv8_read(const scry_kv8 *caches, int n_seq, const int32_t *start, int rows, scry_buf *k, scry_buf *v) {
    API_LOCK;
    SCRY_REQUIRE_INIT();
    if (!k || !v) return set_error(SCRY_ERR_INVALID, "kv8_read: null output handle");
    Kv8Rows a{};
    size_t n = 0;
    SCRY_TRY(kv8_rows("kv8_read", caches, n_seq, start, rows, false, &a, &n));
    DeviceScope dev;
    scry_buf ok = nullptr, ov = nullptr;
    int rc = buf_new(n * n_seq * a.c.hd, &ok);
    if (!rc) rc = buf_new(n * n_seq * a.c.hd, &ov);
    if (!rc)
        rc = by_lanes(a.c.hd, [&](auto g) {
            constexpr int G = decltype(g)::value, NG = 256 / G;
            if ((n + NG - 1) / NG > 0x7fffffff) return set_error(SCRY_ERR_UNSUPPORTED, "kv8_read: %d rows", rows);
            hipLaunchKernelGGL(k_kv8_read<G>, dim3((unsigned)((n + NG - 1) / NG), 2, n_seq), dim3(256), 0, ctx().stream, a,
                               ok->d, ov->d);
            SCRY_HIP(hipGetLastError());
            return (int)SCRY_OK;
        });
    if (rc) {
        buf_del(ok);
        buf_del(ov);
        return rc;
    }
    *k = ok;
    *v = ov;
    return SCRY_OK;
}

int scry_hip_kv8_keep(const scry_kv8 *caches, int n_seq, const int32_t *start, const int32_t *paths, int n_path) {
    API_LOCK;
    SCRY_REQUIRE_INIT();
    const char *what = "kv8_keep";
    if (!paths || n_path < 1 || n_path > DRAFT_MAX_TREE)
        return set_error(SCRY_ERR_INVALID, "%s: paths of %d nodes (1..%d)", what, n_path, DRAFT_MAX_TREE);
    DraftBatch d;
    SCRY_TRY(draft_batch(what, n_seq, 1, start, nullptr, &d));
    Kv8Keep a{};
    bool moves = false;
    for (int s = 0; s < n_seq; s++) {
        const int32_t *p = paths + (size_t)s * n_path;
        int n = 0;
        while (n < n_path && p[n] != -1) {
            if (p[n] < 0 || p[n] >= DRAFT_MAX_TREE || (n && p[n] <= p[n - 1]))
                return set_error(SCRY_ERR_INVALID, "%s: node %d at place %d of sequence %d's path (ascending, below %d)", what,
                                 p[n], n, s, DRAFT_MAX_TREE);
            a.path[s][n] = (unsigned char)p[n];
            moves |= p[n] != n;
            n++;
        }
        a.count[s] = n;
        a.start[s] = d.len[s];
        if (n && caches && caches[s] && (long long)d.len[s] + p[n - 1] >= caches[s]->max_seq)
            return set_error(SCRY_ERR_RANGE, "%s: row %d + %d of cache %d, which holds %d", what, d.len[s], p[n - 1], s,
                             caches[s]->max_seq);
    }
    SCRY_TRY(kv8_batch(what, caches, n_seq, d, 0, true, &a.c));
    if (!moves) return SCRY_OK;
    DeviceScope dev;
    hipLaunchKernelGGL(k_kv8_keep, dim3(a.c.n_kv, 2, n_seq), dim3(256), 0, ctx().stream, a);
    SCRY_HIP(hipGetLastError());
    return SCRY_OK;
}

}  // extern "C"
