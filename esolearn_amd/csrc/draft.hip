// Ops on drafted tokens: what they share (the batch of draft trees, its
// checks, pinned host memory), and the per-head norms of q and k with the
// rotation of every row at its own position.
//
// Row i of sequence s is a drafted token: a node of a tree whose parent is an
// earlier row (or the context), at position len[s] + its depth.  Without a
// tree row i follows row i - 1: one new token, a chain, a prompt.
#include <cmath>

#include "internal.h"
#include "kdev.h"

namespace scry {

int check_heads(const char *what, int n_q, int n_kv, int head_dim) {
    if (n_kv <= 0 || n_q < 0 || head_dim <= 0)
        return set_error(SCRY_ERR_INVALID, "%s: heads and head_dim must be > 0", what);
    if (n_q % n_kv) return set_error(SCRY_ERR_INVALID, "%s: n_q %% n_kv != 0", what);
    if (head_dim % 4 || head_dim > DRAFT_MAX_HD)
        return set_error(SCRY_ERR_UNSUPPORTED, "%s: head_dim %d (need %%4 == 0, <= %d)", what, head_dim, DRAFT_MAX_HD);
    // row offsets are 64-bit; one row of all heads is indexed in 32
    if ((size_t)(n_q + 2 * (size_t)n_kv) * head_dim > ((size_t)1 << 24))
        return set_error(SCRY_ERR_UNSUPPORTED, "%s: %d + 2 x %d heads in a row", what, n_q, n_kv);
    return SCRY_OK;
}

int draft_batch(const char *what, int n_seq, int rows, const int32_t *start, const int64_t *parents, DraftBatch *b) {
    if (n_seq < 1 || n_seq > PF_MAX_SEQS)
        return set_error(SCRY_ERR_INVALID, "%s: %d sequences (1..%d)", what, n_seq, PF_MAX_SEQS);
    if (rows < 1 || !start) return set_error(SCRY_ERR_INVALID, "%s: rows and start", what);
    if (parents && rows > DRAFT_MAX_TREE)
        return set_error(SCRY_ERR_UNSUPPORTED, "%s: a tree of %d nodes (at most %d)", what, rows, DRAFT_MAX_TREE);
    *b = DraftBatch{};
    b->n_seq = n_seq;
    b->rows = rows;
    b->tree = parents != nullptr;
    for (int s = 0; s < n_seq; s++) {
        if (start[s] < 0 || start[s] > DRAFT_MAX_ROW - rows)  // (the kernels count rows in 32 bits, past the last by a step)
            return set_error(SCRY_ERR_RANGE, "%s: rows %d .. of sequence %d (rows 0 .. 2^30)", what, start[s], s);
        b->len[s] = start[s];
        for (int i = 0; parents && i < rows; i++) {
            const int64_t p = parents[(size_t)s * rows + i];
            if (p < -2 || p >= i || (p >= 0 && b->parent[s][p] == -2))
                return set_error(SCRY_ERR_INVALID, "%s: node %d of sequence %d has parent %lld (an earlier node, -1: the context, -2: no node)",
                                 what, i, s, (long long)p);
            b->parent[s][i] = (signed char)p;
        }
    }
    return SCRY_OK;
}

namespace {
void *g_host = nullptr;
size_t g_host_bytes = 0;
unsigned *g_counters = nullptr;

void host_free() {
    if (g_host) (void)hipHostFree(g_host);
    g_host = nullptr;
    g_host_bytes = 0;
}
}  // namespace

int host_block(size_t bytes, void **p) {
    if (g_host_bytes < bytes) {
        SCRY_HIP(hipStreamSynchronize(ctx().stream));
        host_free();
        const size_t want = (bytes + 4095) & ~(size_t)4095;
        SCRY_HIP(hipHostMalloc(&g_host, want, hipHostMallocCoherent));
        g_host_bytes = want;
    }
    *p = g_host;
    return SCRY_OK;
}

int draft_counters(unsigned **ctr) {
    if (!g_counters) {
        void *p = nullptr;
        SCRY_TRY(dev_alloc(&p, DRAFT_COUNTERS * sizeof(unsigned)));
        const int rc = launch_fill_u32((unsigned *)p, DRAFT_COUNTERS, 0u, ctx().stream);
        if (rc) {
            dev_free(p);
            return rc;
        }
        g_counters = (unsigned *)p;
    }
    *ctr = g_counters;
    return SCRY_OK;
}

void draft_free() {
    host_free();
    dev_free(g_counters);
    g_counters = nullptr;
}

namespace {

using namespace dev;

struct QkArgs {
    const float *qkv, *freqs, *qw, *kw;
    float *q, *k, *v;
    int n_q, n_kv, hd;
    float eps, q_scale;
    // positions: start[s] + depth[s][i] (tree) or start[s] + i
    int rows, tree;
    int start[PF_MAX_SEQS];
    signed char depth[PF_MAX_SEQS][DRAFT_MAX_TREE];
};

// n = h / sqrt(mean(h^2) + eps) * w, then the pairs (2j, 2j + 1) of n turn by
// the angle f64(pos) f64(freq_j), its cos and sin rounded to f32 once (the
// values of the model cache's table); q is multiplied by q_scale.
// Bound by HBM: each value is read and written once.  One workgroup takes one
// row (few rows: a part of its heads), so its hd/2 angles, the expensive f64
// part, are computed once and lie in LDS; G lanes hold a head, a float4 each.
// The sum of squares of a head is an f32 tree over its lanes.
// 2047 rows of 96 heads of 128, 201 MB: 40 us, a large copy's rate; one row of
// 48: 3.6 us.
template <int G>
__global__ __launch_bounds__(256) void k_qk_norm_rope(QkArgs a) {
    constexpr int NG = 256 / G;
    __shared__ float2 s_cs[DRAFT_MAX_HD / 2];
    const int row = blockIdx.x, s = row / a.rows, i = row % a.rows;
    const int tid = threadIdx.x, gl = tid % G;
    const int heads = a.n_q + 2 * a.n_kv, hd = a.hd;
    const int pos = a.start[s] + (a.tree ? (int)a.depth[s][i] : i);
    const bool act = 4 * gl < hd;
    for (int j = tid; j < hd / 2; j += 256) {
        const double ang = (double)pos * (double)a.freqs[j];
        s_cs[j] = make_float2((float)cos(ang), (float)sin(ang));
    }
    __syncthreads();
    const float2 c0 = act ? s_cs[2 * gl] : make_float2(1.f, 0.f), c1 = act ? s_cs[2 * gl + 1] : make_float2(1.f, 0.f);
    const float4 one = make_float4(1.f, 1.f, 1.f, 1.f);
    const float4 qw = a.qw && act ? *(const float4 *)(a.qw + 4 * gl) : one;
    const float4 kw = a.kw && act ? *(const float4 *)(a.kw + 4 * gl) : one;
    const float *src = a.qkv + (size_t)row * heads * hd;
    for (int h = blockIdx.y * NG + tid / G; h < heads; h += gridDim.y * NG) {
        float4 x = act ? *(const float4 *)(src + h * hd + 4 * gl) : make_float4(0.f, 0.f, 0.f, 0.f);
        const bool is_q = h < a.n_q, is_v = h >= a.n_q + a.n_kv;
        float *o = is_q   ? a.q + ((size_t)row * a.n_q + h) * hd
                   : is_v ? a.v + ((size_t)row * a.n_kv + (h - a.n_q - a.n_kv)) * hd
                          : a.k + ((size_t)row * a.n_kv + (h - a.n_q)) * hd;
        if (!is_v) {
            if (is_q ? a.qw != nullptr : a.kw != nullptr) {
                float ss = x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w;
#pragma unroll
                for (int off = G / 2; off > 0; off >>= 1) ss += __shfl_xor(ss, off);
                const float r = 1.f / sqrtf(ss / (float)hd + a.eps);
                const float4 w = is_q ? qw : kw;
                x = make_float4(x.x * r * w.x, x.y * r * w.y, x.z * r * w.z, x.w * r * w.w);
            }
            x = make_float4(x.x * c0.x - x.y * c0.y, x.x * c0.y + x.y * c0.x, x.z * c1.x - x.w * c1.y, x.z * c1.y + x.w * c1.x);
            if (is_q) x = make_float4(x.x * a.q_scale, x.y * a.q_scale, x.z * a.q_scale, x.w * a.q_scale);
        }
        if (act) *(float4 *)(o + 4 * gl) = x;
    }
}

template <int G>
int launch_qk(const QkArgs &a, int n_rows, hipStream_t s) {
    constexpr int NG = 256 / G;
    // few rows: a row's heads over several workgroups, one group of heads each at most
    const int parts = (a.n_q + 2 * a.n_kv + NG - 1) / NG;
    int y = (1024 + n_rows - 1) / n_rows;
    if (y > parts) y = parts;
    hipLaunchKernelGGL(k_qk_norm_rope<G>, dim3(n_rows, y), dim3(256), 0, s, a);
    SCRY_HIP(hipGetLastError());
    return SCRY_OK;
}

}  // namespace
}  // namespace scry

using namespace scry;

extern "C" int scry_hip_qk_norm_rope(scry_buf qkv, int n_seq, int rows, const int32_t *start, const int64_t *parents,
                                     int n_q, int n_kv, int head_dim, scry_buf freqs, scry_buf q_weight,
                                     scry_buf k_weight, float eps, float q_scale, scry_buf *q, scry_buf *k, scry_buf *v) {
    std::lock_guard<std::recursive_mutex> lock(api_mutex());
    SCRY_REQUIRE_INIT();
    const char *what = "qk_norm_rope";
    if (!q || !k || !v) return set_error(SCRY_ERR_INVALID, "%s: null output handle", what);
    SCRY_TRY(check_f32(qkv, what));
    SCRY_TRY(check_f32(freqs, what));
    if (q_weight) SCRY_TRY(check_f32(q_weight, what));
    if (k_weight) SCRY_TRY(check_f32(k_weight, what));
    if (n_q <= 0) return set_error(SCRY_ERR_INVALID, "%s: heads and head_dim must be > 0", what);
    SCRY_TRY(check_heads(what, n_q, n_kv, head_dim));
    DraftBatch b;
    SCRY_TRY(draft_batch(what, n_seq, rows, start, parents, &b));
    const size_t n_rows = (size_t)n_seq * rows, hd = head_dim;
    if (n_rows > DRAFT_MAX_GRID) return set_error(SCRY_ERR_UNSUPPORTED, "%s: %zu rows", what, n_rows);
    if (qkv->n != n_rows * (n_q + 2 * (size_t)n_kv) * hd || freqs->n != hd / 2 || (q_weight && q_weight->n != hd) ||
        (k_weight && k_weight->n != hd))
        return set_error(SCRY_ERR_INVALID, "%s: shape mismatch", what);
    DeviceScope dev;
    QkArgs a{};
    a.qkv = qkv->d;
    a.freqs = freqs->d;
    a.qw = q_weight ? q_weight->d : nullptr;
    a.kw = k_weight ? k_weight->d : nullptr;
    a.n_q = n_q;
    a.n_kv = n_kv;
    a.hd = head_dim;
    a.eps = eps;
    a.q_scale = q_scale;
    a.rows = rows;
    a.tree = b.tree;
    for (int s = 0; s < n_seq; s++) {
        a.start[s] = b.len[s];
        for (int i = 0; b.tree && i < rows; i++) {
            const int p = b.parent[s][i];
            a.depth[s][i] = p >= 0 ? (signed char)(a.depth[s][p] + 1) : 0;
        }
    }
    scry_buf oq = nullptr, ok = nullptr, ov = nullptr;
    int rc = buf_new(n_rows * n_q * hd, &oq);
    if (!rc) rc = buf_new(n_rows * n_kv * hd, &ok);
    if (!rc) rc = buf_new(n_rows * n_kv * hd, &ov);
    if (!rc) {
        a.q = oq->d;
        a.k = ok->d;
        a.v = ov->d;
        hipStream_t s = ctx().stream;
        const int lanes = head_dim / 4;
        rc = lanes <= 4    ? launch_qk<4>(a, (int)n_rows, s)
             : lanes <= 8  ? launch_qk<8>(a, (int)n_rows, s)
             : lanes <= 16 ? launch_qk<16>(a, (int)n_rows, s)
             : lanes <= 32 ? launch_qk<32>(a, (int)n_rows, s)
                           : launch_qk<64>(a, (int)n_rows, s);
    }
    if (rc) {
        buf_del(oq);
        buf_del(ok);
        buf_del(ov);
        return rc;
    }
    *q = oq;
    *k = ok;
    *v = ov;
    return SCRY_OK;
}
