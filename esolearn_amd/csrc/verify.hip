// Verification of drafted tokens against the target's probabilities, from
// given random numbers (the reference decodes token by token, generate.rs:51-89,
// and has no counterpart).
//
// A drafted chain x_0 .. x_{n-1}, x_i drawn from q_i, against p_0 .. p_n:
//   x_i is accepted while u_i q_i(x_i) < p_i(x_i); at the first that is not,
//   the next token is drawn from max(p_i - q_i, 0), after the last from p_n.
// A drafted tree against p of the context (row 0) and of every node (row
// 1 + i): a token t_r is drawn from each row with u_r; the walk from row 0
// follows the child that holds the row's token, and ends with the token of the
// last row.  Either way the tokens are distributed as the target's.
//
// A draw from weights w is the lowest j whose running sum passes u sum(w), in
// f64.  Weights that are not positive and finite count as zero; where none is
// left, the residual falls back to p, and p to equal weights.
//
// The row is cut into chunks summed by a workgroup each; then one workgroup
// finds the chunk, and in it the token.  Bound by latency, and for trees by
// reading their rows once.
#include <cmath>
#include <cstring>

#include "internal.h"
#include "kdev.h"

namespace scry {
namespace {

using namespace dev;

constexpr int VF_MAX_ROWS = DRAFT_MAX_TREE;  // drafted tokens of a sequence
constexpr int VF_MAX_CHUNKS = 1024;
constexpr int VF_ARGS = 160;  // (token, number) pairs that travel in the kernel's arguments

struct VfIn {  // n_seq * (rows + 1) of each: a sequence's tokens (the last place unused) and its numbers
    double u[VF_ARGS];
    int tok[VF_ARGS];
};

struct VfArgs {
    const float *p, *q;  // [n_seq][rows + 1][V]; [n_seq][rows][V], null for a tree
    int V, rows, chunk, n_chunk, tree;
    signed char count[PF_MAX_SEQS];
    double *part;  // [n_seq][R][2][n_chunk]: sums of the weights and of p; R = rows + 1 (tree) or 1
    int *drawn;    // tree: [n_seq][rows + 1]
    int *out;      // pinned, [n_seq][2 + rows]: accepted, next token, path
    const double *u;  // null: in the arguments, with the tokens
    const int *tok;
};
__device__ __forceinline__ const double *vf_u(const VfArgs &a, const VfIn &in) { return a.u ? a.u : in.u; }
__device__ __forceinline__ const int *vf_tok(const VfArgs &a, const VfIn &in) { return a.u ? a.tok : in.tok; }

__device__ __forceinline__ double weight(float p, float q) {
    const double w = (double)p - (double)q;
    return w > 0.0 && w < (double)INFINITY ? w : 0.0;
}

// What sequence s draws from: row r of p, less row r of q where less is set.
struct VfRow {
    const float *p, *q;
    int r;
};
__device__ __forceinline__ VfRow vf_row(const VfArgs &a, const VfIn &in, int s, int r, int *n_ok) {
    const size_t V = a.V;
    const float *p = a.p + (size_t)s * (a.rows + 1) * V;
    if (a.tree) return {p + r * V, nullptr, r};
    const int n = a.count[s], lane = threadIdx.x & 63, at = s * (a.rows + 1) + lane;
    bool ok = true;
    if (lane < n) {
        const int x = vf_tok(a, in)[at];
        ok = vf_u(a, in)[at] * (double)a.q[((size_t)s * a.rows + lane) * V + x] < (double)p[lane * V + x];
    }
    const unsigned long long no = __ballot(!ok);
    const int k = no ? __ffsll((long long)no) - 1 : n;
    *n_ok = k;
    return {p + k * V, k < n ? a.q + ((size_t)s * a.rows + k) * V : nullptr, k};
}

__device__ __forceinline__ double block_sum(double v, double *red) {
    v = wave_sum_d(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

__global__ __launch_bounds__(256) void k_verify_sums(VfArgs a, VfIn args) {
    __shared__ double red[4];
    const int s = blockIdx.z, r = blockIdx.y, c = blockIdx.x;
    int n = 0;
    const VfRow w = vf_row(a, args, s, r, &n);
    const int lo = c * a.chunk, hi = min(a.V, lo + a.chunk);
    double sw = 0.0, sp = 0.0;
    for (int j = lo + (int)threadIdx.x; j < hi; j += 256) {
        sp += weight(w.p[j], 0.f);
        if (w.q) sw += weight(w.p[j], w.q[j]);
    }
    sp = block_sum(sp, red);
    if (w.q) sw = block_sum(sw, red);
    if (threadIdx.x == 0) {
        double *d = a.part + (((size_t)s * gridDim.y + r) * 2) * a.n_chunk + c;
        d[0] = w.q ? sw : sp;
        d[a.n_chunk] = sp;
    }
}

// Inclusive running sums over the workgroup's threads.
__device__ __forceinline__ double block_scan(double v, double *red) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const double o = __shfl_up(v, off);
        if (lane >= off) v += o;
    }
    __syncthreads();
    if (lane == 63) red[wave] = v;
    __syncthreads();
    for (int w = 0; w < wave; w++) v += red[w];
    return v;
}

// The lowest i in [0, n) with f(i) > 0 whose running sum of f, from `base` on,
// passes target; where rounding leaves none, the last i with f(i) > 0 (-1: no
// such i).  A thread takes ceil(n / 256) neighbours; the first thread whose end
// passes looks through its own.  *before: the running sum below i.
template <class F>
__device__ __forceinline__ int block_find(int n, double target, double base, F f, double *before, double *red) {
    __shared__ double s_end[256], s_before;
    __shared__ int s_first, s_last, s_i;
    const int tid = threadIdx.x, per = (n + 255) / 256, lo = min(n, tid * per), hi = min(n, lo + per);
    if (tid == 0) {
        s_first = 256;
        s_last = s_i = -1;
        s_before = base;
    }
    double own = 0.0;
    for (int i = lo; i < hi; i++) own += f(i);
    const double end = base + block_scan(own, red);  // (barriers: the shared values above are set)
    s_end[tid] = end;
    if (own > 0.0) {
        if (end > target) atomicMin(&s_first, tid);
        atomicMax(&s_last, tid);
    }
    __syncthreads();
    if (tid == (s_first < 256 ? s_first : s_last)) {
        double x = tid ? s_end[tid - 1] : base;
        for (int i = lo; i < hi; i++) {
            const double w = f(i);
            if (!(w > 0.0)) continue;
            s_i = i;
            s_before = x;
            x += w;
            if (x > target) break;
        }
    }
    __syncthreads();
    *before = s_before;
    const int r = s_i;
    __syncthreads();
    return r;
}

// The drawn index of sequence s, row r, in every thread.
__device__ __forceinline__ int vf_draw(const VfArgs &a, const VfRow &w, const double *part, double u, double *red) {
    double total = 0.0;
    const float *q = w.q;
    for (int c = threadIdx.x; c < a.n_chunk; c += 256) total += part[c];
    total = block_sum(total, red);
    if (!(total > 0.0)) {  // no residual: p itself
        q = nullptr;
        part += a.n_chunk;
        total = 0.0;
        for (int c = threadIdx.x; c < a.n_chunk; c += 256) total += part[c];
        total = block_sum(total, red);
        if (!(total > 0.0)) return min(a.V - 1, (int)(u * (double)a.V));
    }
    const double target = u * total;
    double before = 0.0;
    const int c = block_find(a.n_chunk, target, 0.0, [&](int i) { return part[i]; }, &before, red);
    const int lo = c * a.chunk, n = min(a.chunk, a.V - lo);
    __syncthreads();
    double unused;
    const int j = block_find(n, target, before, [&](int i) { return weight(w.p[lo + i], q ? q[lo + i] : 0.f); }, &unused, red);
    return lo + max(j, 0);
}

__global__ __launch_bounds__(256) void k_verify_draw(VfArgs a, VfIn args) {
    __shared__ double red[4];
    const int s = blockIdx.z, r = blockIdx.y;
    int n = 0;
    const VfRow w = vf_row(a, args, s, r, &n);
    const double *part = a.part + (((size_t)s * gridDim.y + r) * 2) * a.n_chunk;
    const int j = vf_draw(a, w, part, vf_u(a, args)[s * (a.rows + 1) + (a.tree ? r : a.rows)], red);
    if (threadIdx.x) return;
    if (a.tree) {
        a.drawn[s * (a.rows + 1) + r] = j;
    } else {
        a.out[s * (2 + a.rows)] = n;
        a.out[s * (2 + a.rows) + 1] = j;
    }
}

// One wave per sequence, a node per lane.
__global__ __launch_bounds__(64) void k_verify_walk(VfArgs a, VfIn args, DraftBatch d) {
    const int s = blockIdx.x, i = threadIdx.x;
    const int parent = i < a.rows ? (int)d.parent[s][i] : -2;
    const int tok = i < a.rows ? vf_tok(a, args)[s * (a.rows + 1) + i] : 0;
    int *out = a.out + s * (2 + a.rows);
    int cur = -1, n = 0, t;
    for (;;) {
        t = a.drawn[s * (a.rows + 1) + cur + 1];
        const unsigned long long hit = __ballot(parent == cur && tok == t);
        if (!hit) break;
        cur = __ffsll((long long)hit) - 1;  // above the last one: at most `rows` turns
        if (i == 0) out[2 + n] = cur;
        n++;
    }
    if (i >= n && i < a.rows) out[2 + i] = -1;
    if (i == 0) {
        out[0] = n;
        out[1] = t;
    }
}

// Checks, uploads, runs and waits: *res is the pinned result [n_seq][2 + rows].
int vf_run(const char *what, scry_buf p, scry_buf q, const int64_t *tokens, const int32_t *counts, const int32_t *parents,
           const double *u, int n_seq, int rows, int vocab, const int **res) {
    const bool tree = !q;
    if (vocab <= 0 || rows < 1) return set_error(SCRY_ERR_INVALID, "%s: vocabulary and rows must be > 0", what);
    if (rows > VF_MAX_ROWS)
        return set_error(SCRY_ERR_UNSUPPORTED, "%s: %d drafted tokens a sequence (at most %d)", what, rows, VF_MAX_ROWS);
    const int32_t zero[PF_MAX_SEQS] = {};
    DraftBatch d;
    SCRY_TRY(draft_batch(what, n_seq, rows, zero, parents, &d));
    if (!tokens || !u) return set_error(SCRY_ERR_INVALID, "%s: null tokens or random numbers", what);
    const size_t V = vocab, m = rows, n = n_seq * (m + 1);
    if (p->n != n * V || (q && q->n != n_seq * m * V)) return set_error(SCRY_ERR_INVALID, "%s: shape mismatch", what);
    // workgroups of 256 threads: at least 8 values a thread, at most VF_MAX_CHUNKS chunks
    VfArgs a{};
    a.p = p->d;
    a.q = q ? q->d : nullptr;
    a.V = vocab;
    a.rows = rows;
    a.tree = tree;
    a.chunk = 2048;
    while ((V + a.chunk - 1) / a.chunk > VF_MAX_CHUNKS) a.chunk *= 2;
    a.n_chunk = (int)((V + a.chunk - 1) / a.chunk);
    const int R = tree ? rows + 1 : 1;

    VfIn in{};
    double hu[PF_MAX_SEQS * (VF_MAX_ROWS + 1)];
    int ht[PF_MAX_SEQS * (VF_MAX_ROWS + 1)];
    for (int s = 0; s < n_seq; s++) {
        const int c = counts ? counts[s] : rows;
        if (c < 0 || c > rows)
            return set_error(SCRY_ERR_INVALID, "%s: %d drafted tokens in sequence %d (0..%d)", what, c, s, rows);
        a.count[s] = (signed char)c;
        for (size_t i = 0; i <= m; i++) {
            const size_t at = s * (m + 1) + i;
            hu[at] = u[at];
            if (!(u[at] >= 0.0 && u[at] < 1.0))
                return set_error(SCRY_ERR_INVALID, "%s: random number %zu of sequence %d is %g, outside [0, 1)", what, i, s,
                                 u[at]);
            ht[at] = 0;
            if (i == m || (tree ? d.parent[s][i] == -2 : (int)i >= c)) continue;  // no drafted token
            const int64_t t = tokens[s * m + i];
            if (t < 0 || t >= vocab)
                return set_error(SCRY_ERR_RANGE, "%s: token %lld at place %zu of sequence %d, vocabulary %d", what, (long long)t,
                                 i, s, vocab);
            ht[at] = (int)t;
        }
    }
    const bool big = n > VF_ARGS;
    const size_t out_bytes = (n_seq * (m + 2) * sizeof(int) + 255) & ~(size_t)255;
    DeviceScope dev;
    char *host = nullptr;
    SCRY_TRY(host_block(out_bytes + n * (sizeof(double) + sizeof(int)), (void **)&host));
    a.out = (int *)host;
    std::memcpy(big ? (double *)(host + out_bytes) : in.u, hu, n * sizeof(double));
    std::memcpy(big ? (int *)(host + out_bytes + n * sizeof(double)) : in.tok, ht, n * sizeof(int));

    // workspace: chunk sums, drawn tokens, inputs too many for the arguments
    const size_t part = (size_t)n_seq * R * 2 * a.n_chunk * sizeof(double), drawn = (n * sizeof(int) + 7) & ~(size_t)7;
    char *ws = nullptr;
    SCRY_TRY(ctx_workspace(part + drawn + n * (sizeof(double) + sizeof(int)), (void **)&ws));
    a.part = (double *)ws;
    a.drawn = (int *)(ws + part);
    hipStream_t st = ctx().stream;
    if (big) {
        a.u = (double *)(ws + part + drawn);
        a.tok = (int *)(a.u + n);
        SCRY_HIP(hipMemcpyAsync((void *)a.u, host + out_bytes, n * (sizeof(double) + sizeof(int)), hipMemcpyHostToDevice, st));
    }
    hipLaunchKernelGGL(k_verify_sums, dim3(a.n_chunk, R, n_seq), dim3(256), 0, st, a, in);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess) {
        hipLaunchKernelGGL(k_verify_draw, dim3(1, R, n_seq), dim3(256), 0, st, a, in);
        e = hipGetLastError();
    }
    if (e == hipSuccess && tree) {
        hipLaunchKernelGGL(k_verify_walk, dim3(n_seq), dim3(64), 0, st, a, in, d);
        e = hipGetLastError();
    }
    // the pinned block is read and written until here, whatever happened
    const hipError_t w = hipStreamSynchronize(st);
    if (e == hipSuccess) e = w;
    if (e != hipSuccess) return hip_fail(e, what, __FILE__, __LINE__);
    *res = a.out;
    return SCRY_OK;
}

}  // namespace
}  // namespace scry

using namespace scry;

extern "C" {

int scry_hip_verify_draft(scry_buf p, scry_buf q, const int64_t *tokens, const int32_t *counts, const double *u, int n_seq,
                          int rows, int vocab, int64_t *accepted, int64_t *token) {
    std::lock_guard<std::recursive_mutex> lock(api_mutex());
    SCRY_REQUIRE_INIT();
    const char *what = "verify_draft";
    SCRY_TRY(check_f32(p, what));
    SCRY_TRY(check_f32(q, what));
    if (!accepted || !token) return set_error(SCRY_ERR_INVALID, "%s: null output", what);
    const int *r = nullptr;
    SCRY_TRY(vf_run(what, p, q, tokens, counts, nullptr, u, n_seq, rows, vocab, &r));
    for (int s = 0; s < n_seq; s++) {
        accepted[s] = r[(size_t)s * (rows + 2)];
        token[s] = r[(size_t)s * (rows + 2) + 1];
    }
    return SCRY_OK;
}

int scry_hip_verify_tree(scry_buf p, const int64_t *tokens, const int32_t *parents, const double *u, int n_seq, int rows,
                         int vocab, int64_t *paths, int64_t *accepted, int64_t *token) {
    std::lock_guard<std::recursive_mutex> lock(api_mutex());
    SCRY_REQUIRE_INIT();
    const char *what = "verify_tree";
    SCRY_TRY(check_f32(p, what));
    if (!parents) return set_error(SCRY_ERR_INVALID, "%s: null parents", what);
    if (!paths || !accepted || !token) return set_error(SCRY_ERR_INVALID, "%s: null output", what);
    const int *r = nullptr;
    SCRY_TRY(vf_run(what, p, nullptr, tokens, nullptr, parents, u, n_seq, rows, vocab, &r));
    for (int s = 0; s < n_seq; s++) {
        const int *x = r + (size_t)s * (rows + 2);
        accepted[s] = x[0];
        token[s] = x[1];
        for (int i = 0; i < rows; i++) paths[(size_t)s * rows + i] = x[2 + i];
    }
    return SCRY_OK;
}

}  // extern "C"
