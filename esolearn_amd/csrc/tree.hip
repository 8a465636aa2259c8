// Attention of drafted tokens over a cache: row i of sequence s attends to its
// context's rows [0, len) and, among the drafted rows len + j, to its
// ancestors and itself.
//   o_i = sum_t p_t v_t / sum_t p_t,   p_t = exp(scale q_i.k_t - max)
// The cache is read in place: f32 rows [max_seq, n_kv * hd] or the int8 cache.
#include <cmath>

#include "kdev.h"
#include "kv8.h"

namespace scry {
namespace {

using namespace dev;

struct F32Batch {
    const float *k[PF_MAX_SEQS], *v[PF_MAX_SEQS];
};

struct TreeArgs {
    DraftBatch d;
    const float *q;  // [n_seq * rows, n_q * hd]
    float *out;
    int n_q, n_kv, hd;
    float scale;
};

// Whether drafted row j is an ancestor of row i or row i itself.
__device__ __forceinline__ bool tree_sees(const DraftBatch &d, int s, int i, int j) {
    if (!d.tree) return j <= i;
    while (i > j) i = d.parent[s][i];
    return i == j && d.parent[s][j] != -2;
}

// One workgroup per row and query head: each wave takes 64 keys at a time, a
// key per lane for the scores, a dimension per lane for the sums.
template <bool I8>
__global__ __launch_bounds__(256) void k_tree_simple(TreeArgs a, F32Batch f, Kv8Batch c) {
    __shared__ float s_q[DRAFT_MAX_HD], s_o[4][DRAFT_MAX_HD], s_m[4], s_l[4], s_p[4][64];
    const int row = blockIdx.x, h = blockIdx.y, s = row / a.d.rows, i = row % a.d.rows;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int hd = a.hd, g = h / (a.n_q / a.n_kv), len = a.d.len[s];
    const int end = len + a.d.rows;
    for (int d = tid; d < hd; d += 256) s_q[d] = a.q[((size_t)row * a.n_q + h) * hd + d];
    __syncthreads();
    float m = -INFINITY, l = 0.f, o[4] = {};
    const bool none = a.d.tree && a.d.parent[s][i] == -2;
    for (int t0 = wave * 64; t0 < end && !none; t0 += 256) {
        const int t = t0 + lane;
        const bool in = t < len || (t < end && tree_sees(a.d, s, i, t - len));
        float sc = -INFINITY;
        if (in) {
            sc = 0.f;
            if (I8) {
                const int8_t *k = c.k[s] + kv8_k_at(c.rows_p[s], c.hdp, g, t);
                for (int d = 0; d < hd; d++) sc = fmaf(s_q[d], (float)k[d], sc);
                sc *= c.ks[s][(size_t)g * c.rows_p[s] + t];
            } else {
                const float *k = f.k[s] + ((size_t)t * a.n_kv + g) * hd;
                for (int d = 0; d < hd; d++) sc = fmaf(s_q[d], k[d], sc);
            }
            sc *= a.scale;
        }
        float mx = sc;
        for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off));
        mx = fmaxf(m, mx);
        const float ref = mx == -INFINITY ? 0.f : mx;
        float p = in ? expf(sc - ref) : 0.f;
        const float alpha = expf(m - ref);
        l = l * alpha + wave_sum(p);
        m = mx;
        if (I8 && in) p *= c.vs[s][(size_t)g * c.rows_p[s] + t];
        s_p[wave][lane] = p;
        const unsigned long long mask = __ballot(in);
        for (int e = 0; e < 4; e++) {
            const int d = lane + 64 * e;
            if (d >= hd) break;
            float acc = o[e] * alpha;
            for (int j = 0; j < 64; j++) {
                if (!(mask >> j & 1)) continue;
                const float v = I8 ? (float)c.v[s][kv8_v_at(c.rows_p[s], c.hdp, g, t0 + j, d) + kv8_perm((t0 + j) & 63)]
                                   : f.v[s][((size_t)(t0 + j) * a.n_kv + g) * hd + d];
                acc = fmaf(s_p[wave][j], v, acc);
            }
            o[e] = acc;
        }
    }
    if (lane == 0) {
        s_m[wave] = m;
        s_l[wave] = l;
    }
    for (int e = 0; e < 4; e++)
        if (lane + 64 * e < hd) s_o[wave][lane + 64 * e] = o[e];
    __syncthreads();
    for (int d = tid; d < hd; d += 256) {
        float M = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
        if (M == -INFINITY) M = 0.f;
        float L = 0.f, O = 0.f;
        for (int w = 0; w < 4; w++) {
            const float e = expf(s_m[w] - M);
            L += s_l[w] * e;
            O += s_o[w][d] * e;
        }
        a.out[((size_t)row * a.n_q + h) * hd + d] = none ? 0.f : O / L;
    }
}

int tree_run(const char *what, scry_buf q, const TreeArgs &t, bool i8, const F32Batch &f, const Kv8Batch &c, scry_buf *out) {
    const size_t n = (size_t)t.d.n_seq * t.d.rows;
    if (n > 0x7fffffff) return set_error(SCRY_ERR_UNSUPPORTED, "%s: %zu rows", what, n);
    if (q->n != n * t.n_q * t.hd) return set_error(SCRY_ERR_INVALID, "%s: shape mismatch", what);
    DeviceScope dev;
    scry_buf o = nullptr;
    SCRY_TRY(buf_new(q->n, &o));
    TreeArgs a = t;
    a.q = q->d;
    a.out = o->d;
    if (i8)
        hipLaunchKernelGGL(k_tree_simple<true>, dim3((unsigned)n, a.n_q), dim3(256), 0, ctx().stream, a, f, c);
    else
        hipLaunchKernelGGL(k_tree_simple<false>, dim3((unsigned)n, a.n_q), dim3(256), 0, ctx().stream, a, f, c);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) {
        buf_del(o);
        return hip_fail(e, what, __FILE__, __LINE__);
    }
    *out = o;
    return SCRY_OK;
}

}  // namespace
}  // namespace scry

using namespace scry;

#define API_LOCK std::lock_guard<std::recursive_mutex> _api_lock(scry::api_mutex())

extern "C" {

int scry_hip_tree_attention(scry_buf q, const scry_buf *k_caches, const scry_buf *v_caches, int n_seq, const int32_t *len,
                            int rows, const int32_t *parents, int n_q, int n_kv, int head_dim, float scale, scry_buf *out) {
    API_LOCK;
    SCRY_REQUIRE_INIT();
    const char *what = "tree_attention";
    if (!out) return set_error(SCRY_ERR_INVALID, "%s: null output handle", what);
    SCRY_TRY(check_f32(q, what));
    TreeArgs t{};
    SCRY_TRY(draft_batch(what, n_seq, rows, len, parents, &t.d));
    if (n_q <= 0) return set_error(SCRY_ERR_INVALID, "%s: heads and head_dim must be > 0", what);
    SCRY_TRY(check_heads(what, n_q, n_kv, head_dim));
    if (!k_caches || !v_caches) return set_error(SCRY_ERR_INVALID, "%s: null caches", what);
    F32Batch f{};
    for (int s = 0; s < n_seq; s++) {
        SCRY_TRY(check_f32(k_caches[s], what));
        SCRY_TRY(check_f32(v_caches[s], what));
        const size_t need = ((size_t)t.d.len[s] + rows) * n_kv * head_dim;
        if (k_caches[s]->n < need || v_caches[s]->n < need)
            return set_error(SCRY_ERR_RANGE, "%s: rows [0, %d) of sequence %d's cache, which holds less", what,
                             t.d.len[s] + rows, s);
        f.k[s] = k_caches[s]->d;
        f.v[s] = v_caches[s]->d;
    }
    t.n_q = n_q;
    t.n_kv = n_kv;
    t.hd = head_dim;
    t.scale = scale;
    return tree_run(what, q, t, false, f, Kv8Batch{}, out);
}

int scry_hip_kv8_tree_attention(scry_buf q, const scry_kv8 *caches, int n_seq, const int32_t *len, int rows,
                                const int32_t *parents, int n_q, float scale, scry_buf *out) {
    API_LOCK;
    SCRY_REQUIRE_INIT();
    const char *what = "kv8_tree_attention";
    if (!out) return set_error(SCRY_ERR_INVALID, "%s: null output handle", what);
    SCRY_TRY(check_f32(q, what));
    TreeArgs t{};
    SCRY_TRY(draft_batch(what, n_seq, rows, len, parents, &t.d));
    Kv8Batch c;
    SCRY_TRY(kv8_batch(what, caches, n_seq, t.d, rows, false, &c));
    if (n_q <= 0) return set_error(SCRY_ERR_INVALID, "%s: heads and head_dim must be > 0", what);
    SCRY_TRY(check_heads(what, n_q, c.n_kv, c.hd));
    t.n_q = n_q;
    t.n_kv = c.n_kv;
    t.hd = c.hd;
    t.scale = scale;
    return tree_run(what, q, t, true, F32Batch{}, c, out);
}

}  // extern "C"
