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

// Largest value of an aligned group of G lanes, in every lane: quad permutes and
// mirrors up to 16 lanes, then swaps of rows and halves, none through LDS.
template <int CTRL>
__device__ __forceinline__ float dpp_max(float v) {
    return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true)));
}
template <int G>
__device__ __forceinline__ float group_max(float v) {
    v = dpp_max<0xB1>(v);                       // quad_perm [1,0,3,2]
    v = dpp_max<0x4E>(v);                       // quad_perm [2,3,0,1]
    if constexpr (G >= 8) v = dpp_max<0x141>(v);   // row_half_mirror
    if constexpr (G >= 16) v = dpp_max<0x140>(v);  // row_mirror
    if constexpr (G >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    if constexpr (G >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    return v;
}

// |x| / s, s > 0, to the nearest integer r, halves up, at most 127.  r is off by
// one at most before the remainder x - r s, exact in f32 (an fma of a multiple of
// ulp(s) below 2^24 ulp(s)), decides.
__device__ __forceinline__ float to_nearest(float ax, float r, float s) {
    const float e = fmaf(-r, s, ax), e2 = e + e;
    return fminf(r + (e2 >= s ? 1.f : e2 < -s ? -1.f : 0.f), 127.f);
}

// A row's four values per lane of a group of G into steps; returns the scale.
// Rows of ordinary size take the product with 1 / s (to 1 ulp), and look at the
// remainders once for all four values: 2 |e| >= s is a quotient within rounding
// of a half, one in 10^5.
template <int G>
__device__ __forceinline__ float quantise(float4 x, int (&q)[4]) {
    const float v[4] = {x.x, x.y, x.z, x.w};
    float m = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
    if (__builtin_isunordered(x.x, x.y) || __builtin_isunordered(x.z, x.w)) m = INFINITY;
    m = group_max<G>(m);
    if (m >= 0x1p-100f && m < INFINITY) {
        // m / 127, correctly rounded: the product with f32(1 / 127), its
        // remainder exact, and one correction
        const float c = 1.f / 127.f, t = m * c, s = fmaf(fmaf(-127.f, t, m), c, t), inv = __builtin_amdgcn_rcpf(s);
        float r[4], worst = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            r[i] = rintf(fabsf(v[i]) * inv);
            worst = fmaxf(worst, fabsf(fmaf(-r[i], s, fabsf(v[i]))));
        }
        if (__any(worst + worst >= s)) {
#pragma unroll
            for (int i = 0; i < 4; i++) r[i] = to_nearest(fabsf(v[i]), r[i], s);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) q[i] = (int)copysignf(r[i], v[i]);
        return s;
    }
    const float s = m < INFINITY ? m / 127.f : __builtin_nanf("");
#pragma unroll
    for (int i = 0; i < 4; i++)
        q[i] = s > 0.f ? (int)copysignf(to_nearest(fabsf(v[i]), floorf(fabsf(v[i]) / s), s), v[i]) : 0;
    return s;
}
// the low bytes of four integers as a word
__device__ __forceinline__ unsigned bytes4(int a, int b, int c, int d) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm((unsigned)d, (unsigned)c, 0x0c0c0400u),
                                 __builtin_amdgcn_perm((unsigned)b, (unsigned)a, 0x0c0c0400u), 0x05040100u);
}

// A workgroup takes one 64-row block of one head, of K or of V (blockIdx.y), of
// a sequence (blockIdx.z): rows [lo, hi) of the block are the call's.  G lanes
// hold a row, four dimensions each.
struct Block {
    int g, r0, lo, hi;  // head, the block's first cache row, rows of it
    bool v;
    size_t src;  // row r of the block is vector src + r * n_kv of the call's rows (lo <= r < hi)
};
__device__ __forceinline__ bool block_of(const Kv8Rows &a, Block &b) {
    const int s = blockIdx.z, start = a.start[s];
    b.g = blockIdx.x % a.c.n_kv;
    b.r0 = (start & ~63) + 64 * (int)(blockIdx.x / a.c.n_kv);
    b.v = blockIdx.y;
    b.lo = max(start - b.r0, 0);
    b.hi = min(64, start + a.rows - b.r0);
    b.src = ((size_t)s * a.rows + (b.r0 - start)) * a.c.n_kv + b.g;  // (wraps below zero where lo > 0: lo takes it back)
    return b.lo < b.hi;
}
constexpr int V_LD = 17;  // words per dimension of a V block in LDS: 16, and one against bank conflicts

// Bound by HBM (4 bytes read, 1 written).  V's 64-byte groups hold one
// dimension of 64 rows: four rows of a dimension are a word, words are turned
// through LDS and written in 16-byte pieces (whole blocks) or one by one; the
// rows about a word that is not the call's alone, in bytes.
// 2047 rows of 32 heads of 128, 84 MB: 23 us (with V in bytes throughout 54 us).
template <int G>
__global__ __launch_bounds__(256) void k_kv8_write(Kv8Rows a, const float *__restrict__ kx, const float *__restrict__ vx) {
    constexpr int NG = 256 / G;
    __shared__ unsigned s_v[4 * G * V_LD];
    Block b;
    if (!block_of(a, b)) return;
    const int s = blockIdx.z, tid = threadIdx.x, gl = tid % G, grp = tid / G;
    const int n_kv = a.c.n_kv, hd = a.c.hd, hdp = a.c.hdp, rows_p = a.c.rows_p[s];
    const bool act = 4 * gl < hd;
    const float *src = (b.v ? vx : kx) + 4 * gl;
    float *scales = (b.v ? a.c.vs[s] : a.c.ks[s]) + (size_t)b.g * rows_p + b.r0;
    auto row = [&](int r) {
        return act ? *(const float4 *)(src + (b.src + (size_t)r * n_kv) * hd) : make_float4(0.f, 0.f, 0.f, 0.f);
    };
    auto put_row = [&](int r, const int (&q)[4]) {
        if (!act) return;
        if (b.v) {
            int8_t *d = a.c.v[s] + kv8_v_at(rows_p, hdp, b.g, b.r0, 4 * gl) + kv8_perm(r);
#pragma unroll
            for (int e = 0; e < 4; e++) d[64 * e] = (int8_t)(q[e] ^ 0x80);
        } else {
            *(unsigned *)(a.c.k[s] + kv8_k_at(rows_p, hdp, b.g, b.r0 + r) + 4 * gl) = bytes4(q[0], q[1], q[2], q[3]);
        }
    };
    constexpr int NQ = NG < 16 ? 16 / NG : 1;  // four rows at a time: rows 4 (grp + n NG) ..
    float4 x[NQ][4];
#pragma unroll
    for (int n = 0; n < NQ; n++)  // every load before the first use
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = 4 * (grp + n * NG) + i;
            x[n][i] = r >= b.lo && r < b.hi ? row(r) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
    for (int n = 0; n < NQ; n++) {
        const int r0 = 4 * (grp + n * NG);
        if (r0 + 4 <= b.lo || r0 >= b.hi) continue;
        int q[4][4];
        float sc[4];
#pragma unroll
        for (int i = 0; i < 4; i++) sc[i] = quantise<G>(x[n][i], q[i]);
        const bool whole = r0 >= b.lo && r0 + 4 <= b.hi;
        if (whole && gl == 0) *(float4 *)(scales + r0) = make_float4(sc[0], sc[1], sc[2], sc[3]);
        if (whole && b.v) {
            const int at = kv8_perm(r0) / 4;
#pragma unroll
            for (int e = 0; e < 4; e++) s_v[(4 * gl + e) * V_LD + at] = bytes4(q[0][e], q[1][e], q[2][e], q[3][e]) ^ 0x80808080u;
            continue;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (r0 + i < b.lo || r0 + i >= b.hi) continue;
            put_row(r0 + i, q[i]);
            if (!whole && gl == 0) scales[r0 + i] = sc[i];
        }
    }
    if (!b.v) return;
    __syncthreads();
    int8_t *d = a.c.v[s] + kv8_v_at(rows_p, hdp, b.g, b.r0, 0);
    if (b.lo == 0 && b.hi == 64) {
        for (int t = tid; t < hd * 4; t += 256) {  // dimension t / 4, words 4 (t % 4) ..
            const unsigned *w = s_v + (t >> 2) * V_LD + 4 * (t & 3);
            *(uint4 *)(d + 16 * t) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        return;
    }
    for (int t = tid; t < hd * 16; t += 256) {  // word t % 16: rows 16 (t % 4) + 4 (t / 4 % 4) ..
        const int r0 = 16 * (t & 3) + 4 * ((t >> 2) & 3);
        if (r0 >= b.lo && r0 + 4 <= b.hi) *(unsigned *)(d + 4 * t) = s_v[(t >> 4) * V_LD + (t & 15)];
    }
}

// The same blocks the other way (1 byte read, 4 written): 14.4 us for those rows.
template <int G>
__global__ __launch_bounds__(256) void k_kv8_read(Kv8Rows a, float *__restrict__ kx, float *__restrict__ vx) {
    constexpr int NG = 256 / G;
    __shared__ unsigned s_v[4 * G * V_LD];
    Block b;
    if (!block_of(a, b)) return;
    const int s = blockIdx.z, tid = threadIdx.x, gl = tid % G, grp = tid / G;
    const int n_kv = a.c.n_kv, hd = a.c.hd, hdp = a.c.hdp, rows_p = a.c.rows_p[s];
    const bool act = 4 * gl < hd;
    float *dst = (b.v ? vx : kx) + 4 * gl;
    const float *scales = (b.v ? a.c.vs[s] : a.c.ks[s]) + (size_t)b.g * rows_p + b.r0;
    auto put = [&](int r, unsigned w0, unsigned w1, unsigned w2, unsigned w3, int sh, float sc) {
        *(float4 *)(dst + (b.src + (size_t)r * n_kv) * hd) =
            make_float4((float)(int)(signed char)(w0 >> sh) * sc, (float)(int)(signed char)(w1 >> sh) * sc,
                        (float)(int)(signed char)(w2 >> sh) * sc, (float)(int)(signed char)(w3 >> sh) * sc);
    };
    if (b.v) {
        const int8_t *d = a.c.v[s] + kv8_v_at(rows_p, hdp, b.g, b.r0, 0);
        for (int t = tid; t < hd * 4; t += 256) {
            const uint4 x = *(const uint4 *)(d + 16 * t);
            unsigned *w = s_v + (t >> 2) * V_LD + 4 * (t & 3);
            w[0] = x.x ^ 0x80808080u;
            w[1] = x.y ^ 0x80808080u;
            w[2] = x.z ^ 0x80808080u;
            w[3] = x.w ^ 0x80808080u;
        }
        __syncthreads();
        if (!act) return;
        for (int w = grp; w < 16; w += NG) {
            if (4 * w + 4 <= b.lo || 4 * w >= b.hi) continue;
            const unsigned *x = s_v + 4 * gl * V_LD + kv8_perm(4 * w) / 4;
            const float4 sc = *(const float4 *)(scales + 4 * w);
            const float scs[4] = {sc.x, sc.y, sc.z, sc.w};
            const unsigned w0 = x[0], w1 = x[V_LD], w2 = x[2 * V_LD], w3 = x[3 * V_LD];
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (4 * w + i >= b.lo && 4 * w + i < b.hi) put(4 * w + i, w0, w1, w2, w3, 8 * i, scs[i]);
        }
        return;
    }
    if (!act) return;
#pragma unroll 4
    for (int r = b.lo + grp; r < b.hi; r += NG) {
        const float sc = scales[r];
        const unsigned w = *(const unsigned *)(a.c.k[s] + kv8_k_at(rows_p, hdp, b.g, b.r0 + r) + 4 * gl);
        put(r, w, w >> 8, w >> 16, w >> 24, 0, sc);
    }
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

// The lanes that hold a row, as a constant.
template <class F>
void by_lanes(int hd, F f) {
    const int lanes = hd / 4;
    if (lanes <= 4) return f(std::integral_constant<int, 4>{});
    if (lanes <= 8) return f(std::integral_constant<int, 8>{});
    if (lanes <= 16) return f(std::integral_constant<int, 16>{});
    if (lanes <= 32) return f(std::integral_constant<int, 32>{});
    return f(std::integral_constant<int, 64>{});
}

// Fills a and the grid of the block kernels (one more block than rows / 64 has
// where a sequence starts inside one).
int kv8_rows(const char *what, const scry_kv8 *caches, int n_seq, const int32_t *start, int rows, bool distinct,
             Kv8Rows *a, dim3 *grid) {
    DraftBatch d;
    SCRY_TRY(draft_batch(what, n_seq, rows, start, nullptr, &d));
    SCRY_TRY(kv8_batch(what, caches, n_seq, d, rows, distinct, &a->c));
    size_t blocks = 0;
    for (int s = 0; s < n_seq; s++) {
        a->start[s] = d.len[s];
        const size_t n = ((size_t)d.len[s] + rows + 63) / 64 - d.len[s] / 64;
        blocks = blocks > n ? blocks : n;
    }
    a->rows = rows;
    if (blocks * a->c.n_kv > DRAFT_MAX_GRID) return set_error(SCRY_ERR_UNSUPPORTED, "%s: %d rows of %d heads", what, rows, a->c.n_kv);
    *grid = dim3((unsigned)(blocks * a->c.n_kv), 2, n_seq);
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
    if (max_seq <= 0 || max_seq > DRAFT_MAX_ROW) return set_error(SCRY_ERR_INVALID, "kv8_new: max_seq %d (1 .. 2^30)", max_seq);
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
    dim3 grid;
    SCRY_TRY(kv8_rows("kv8_write", caches, n_seq, start, rows, true, &a, &grid));
    if (k->n != (size_t)n_seq * rows * a.c.n_kv * a.c.hd || v->n != k->n)
        return set_error(SCRY_ERR_INVALID, "kv8_write: shape mismatch");
    DeviceScope dev;
    by_lanes(a.c.hd, [&](auto g) {
        hipLaunchKernelGGL(k_kv8_write<decltype(g)::value>, grid, dim3(256), 0, ctx().stream, a, k->d, v->d);
    });
    SCRY_HIP(hipGetLastError());
    return SCRY_OK;
}

int scry_hip_kv8_read(const scry_kv8 *caches, int n_seq, const int32_t *start, int rows, scry_buf *k, scry_buf *v) {
    API_LOCK;
    SCRY_REQUIRE_INIT();
    if (!k || !v) return set_error(SCRY_ERR_INVALID, "kv8_read: null output handle");
    Kv8Rows a{};
    dim3 grid;
    SCRY_TRY(kv8_rows("kv8_read", caches, n_seq, start, rows, false, &a, &grid));
    const size_t n = (size_t)n_seq * rows * a.c.n_kv * a.c.hd;
    DeviceScope dev;
    scry_buf ok = nullptr, ov = nullptr;
    int rc = buf_new(n, &ok);
    if (!rc) rc = buf_new(n, &ov);
    if (!rc) {
        by_lanes(a.c.hd, [&](auto g) {
            hipLaunchKernelGGL(k_kv8_read<decltype(g)::value>, grid, dim3(256), 0, ctx().stream, a, ok->d, ov->d);
        });
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) rc = hip_fail(e, "kv8_read", __FILE__, __LINE__);
    }
    if (rc) {
        buf_del(ok);
        buf_del(ov);
        return rc;
    }
    *k = ok;
    *v = ov;
    return SCRY_OK;
}

int scry_hip_kv8_keep(const scry_kv8 *caches, int n_seq, const int32_t *start, const int64_t *paths, int n_path) {
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
        const int64_t *p = paths + (size_t)s * n_path;
        int n = 0;
        while (n < n_path && p[n] != -1) {
            if (p[n] < 0 || p[n] >= DRAFT_MAX_TREE || (n && p[n] <= p[n - 1]))
                return set_error(SCRY_ERR_INVALID, "%s: node %lld at place %d of sequence %d's path (ascending, below %d)", what,
                                 (long long)p[n], n, s, DRAFT_MAX_TREE);
            a.path[s][n] = (unsigned char)p[n];
            moves |= p[n] != n;
            n++;
        }
        a.count[s] = n;
        a.start[s] = d.len[s];
        if (n && caches && caches[s] && (long long)d.len[s] + p[n - 1] >= caches[s]->max_seq)
            return set_error(SCRY_ERR_RANGE, "%s: row %d + %d of cache %d, which holds %d", what, d.len[s], (int)p[n - 1], s,
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
