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
// One launch.  A row is cut into chunks, a workgroup each, whose four waves
// leave the sums of their parts; the last workgroup of a row to arrive finds
// the part, and in it the token; for a tree, the last row of a sequence walks.
// A chain reads one row of p (and of q) of a sequence and is bound by the
// latency of that sequence of steps (V = 32000: 9 us, 16 chains at 128256: 13);
// a tree reads its rows once, at the rate of the memory, before the draws (four
// trees of 31 nodes at V = 128256, 66 MB: 27 us).
#include <atomic>
#include <chrono>
#include <cmath>
#include <cstring>

#include "arrive.h"
#include "internal.h"
#include "kdev.h"

namespace scry {
namespace {

using namespace dev;

constexpr int VF_MAX_ROWS = DRAFT_MAX_TREE;  // drafted tokens of a sequence
constexpr int VF_ARGS = 160;  // (token, number) pairs that travel in the kernel's arguments

struct VfIn {  // n_seq * (rows + 1) of each: a sequence's tokens (the last place unused) and its numbers
    double u[VF_ARGS];
    int tok[VF_ARGS];
};

struct VfArgs {
    const float *p, *q;  // [n_seq][rows + 1][V]; [n_seq][rows][V], null for a tree
    int V, rows, sub, n_sub, tree, wide;  // sub: values of a wave's part; wide: rows are 16-byte aligned
    signed char count[PF_MAX_SEQS];
    double *part;       // [n_seq][R][2][n_sub]: sums of the weights and of p; R = rows + 1 (tree) or 1
    int *drawn;         // tree: [n_seq][rows + 1]
    unsigned *arrived;  // [n_seq][VF_MAX_ROWS + 2]: workgroups per row, rows per sequence; zero between launches
    int *out;           // pinned, [n_seq][3 + rows]: done, accepted, next token, path
    const double *u;    // null: in the arguments, with the tokens
    const int *tok;
};
__device__ __forceinline__ const double *vf_u(const VfArgs &a, const VfIn &in) { return a.u ? a.u : in.u; }
__device__ __forceinline__ const int *vf_tok(const VfArgs &a, const VfIn &in) { return a.u ? a.tok : in.tok; }

__device__ __forceinline__ double weight(float p) { return p > 0.f && p < INFINITY ? (double)p : 0.0; }
__device__ __forceinline__ double weight(float p, float q) {
    const double w = (double)p - (double)q;
    return w > 0.0 && w < (double)INFINITY ? w : 0.0;
}

// What sequence s draws from: row p, less row q where it is set.  For a chain
// every wave looks at all of the sequence's tokens, one a lane.
struct VfRow {
    const float *p, *q;
    int n;  // chain: accepted
};
__device__ __forceinline__ VfRow vf_row(const VfArgs &a, const VfIn &in, int s, int r) {
    const size_t V = a.V;
    const float *p = a.p + (size_t)s * (a.rows + 1) * V;
    if (a.tree) return {p + r * V, nullptr, 0};
    const int n = a.count[s], lane = threadIdx.x & 63, at = s * (a.rows + 1) + lane;
    bool ok = true;
    if (lane < n) {
        const int x = vf_tok(a, in)[at];
        ok = vf_u(a, in)[at] * (double)a.q[((size_t)s * a.rows + lane) * V + x] < (double)p[lane * V + x];
    }
    const unsigned long long no = __ballot(!ok);
    const int k = no ? __ffsll((long long)no) - 1 : n;
    return {p + k * V, k < n ? a.q + ((size_t)s * a.rows + k) * V : nullptr, k};
}

// Inclusive running sums over the wave's lanes.
__device__ __forceinline__ double wave_scan(double v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const double o = __shfl_up(v, off);
        if (lane >= off) v += o;
    }
    return v;
}

// One wave: the lowest i in [lo, hi) with f(i) > 0 whose running sum of f, from
// `base` on, passes target; where rounding leaves none, the last with f(i) > 0
// (-1: no such i).  *base: the running sum below that i.  A lane takes PER
// neighbours of 64 PER at a time.
template <int PER, class F>
__device__ __forceinline__ int wave_find(int lo, int hi, double target, double *base, F f) {
    const int lane = threadIdx.x & 63;
    int last = -1;
    double below = *base, run = *base;  // below: the sum below `last`
    for (int i0 = lo; i0 < hi; i0 += 64 * PER) {
        double w[PER], own = 0.0;
#pragma unroll
        for (int k = 0; k < PER; k++) {
            const int i = i0 + lane * PER + k;
            w[k] = i < hi ? f(i) : 0.0;
            own += w[k];
        }
        const double end = run + wave_scan(own);
        const double prev = __shfl_up(end, 1);
        const unsigned long long some = __ballot(own > 0.0), pass = __ballot(own > 0.0 && end > target);
        if (some) {
            const int who = pass ? __ffsll((long long)pass) - 1 : 63 - __clzll((long long)some);
            // that lane looks through its own
            double x = lane ? prev : run, at = x;
            int mine = -1;
#pragma unroll
            for (int k = 0; k < PER; k++) {
                if (!(w[k] > 0.0) || (mine >= 0 && x > target)) continue;
                mine = i0 + lane * PER + k;
                at = x;
                x += w[k];
            }
            last = __shfl(mine, who);
            below = __shfl(at, who);
            if (pass) break;
        }
        run = __shfl(end, 63);
    }
    *base = below;
    return last;
}

// The index drawn from a row by the first wave of the workgroup, from the sums
// of its parts.
__device__ __forceinline__ int vf_draw(const VfArgs &a, const VfRow &w, const double *part, double u) {
    const int lane = threadIdx.x & 63;
    const float *q = w.q;
    double total = 0.0;
    for (int turn = 0; turn < 2; turn++) {
        for (int c = lane; c < a.n_sub; c += 64) total += get(part + c);
        total = wave_sum_d(total);
        if (total > 0.0) break;
        if (turn || !q) return min(a.V - 1, (int)(u * (double)a.V));  // no mass at all
        q = nullptr;  // no residual: p itself
        part += a.n_sub;
        total = 0.0;
    }
    const double target = u * total;
    double base = 0.0;
    const int c = wave_find<4>(0, a.n_sub, target, &base, [&](int i) { return get(part + i); });
    const int lo = max(c, 0) * a.sub, hi = min(a.V, lo + a.sub);
    const int j = wave_find<8>(lo, hi, target, &base, [&](int i) { return q ? weight(w.p[i], q[i]) : weight(w.p[i]); });
    return max(j, 0);
}

// A result's value to host memory, past every cache of the device; and, by the
// wave that wrote them, once those stores are complete, that the result is there.
__device__ __forceinline__ void to_host(int *p, int v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM); }
__device__ __forceinline__ void vf_done(const VfArgs &a, int s) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if ((threadIdx.x & 63) == 0) to_host(a.out + s * (3 + a.rows), 1);
}

// From row 0 to the child that holds the row's token, a node per lane.
__device__ __forceinline__ void vf_walk(const VfArgs &a, const VfIn &in, const DraftBatch &d, int s) {
    const int i = threadIdx.x & 63;
    const int parent = i < a.rows ? (int)d.parent[s][i] : -2;
    const int tok = i < a.rows ? vf_tok(a, in)[s * (a.rows + 1) + i] : 0;
    const int t_row = i < a.rows ? get(a.drawn + s * (a.rows + 1) + 1 + i) : 0;  // drawn after node i
    int *out = a.out + s * (3 + a.rows) + 1;
    int cur = -1, n = 0, t = get(a.drawn + s * (a.rows + 1));
    for (;;) {
        const unsigned long long hit = __ballot(parent == cur && tok == t);
        if (!hit) break;
        cur = __ffsll((long long)hit) - 1;  // above the last one: at most `rows` turns
        if (i == 0) to_host(out + 2 + n, cur);
        t = __shfl(t_row, cur);
        n++;
    }
    if (i >= n && i < a.rows) to_host(out + 2 + i, -1);
    if (i == 0) {
        to_host(out, n);
        to_host(out + 1, t);
    }
}

__global__ __launch_bounds__(256) void k_verify(VfArgs a, VfIn in, DraftBatch d) {
    const int s = blockIdx.z, r = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const VfRow w = vf_row(a, in, s, r);
    const int c = blockIdx.x * 4 + wave;
    double *part = a.part + (((size_t)s * gridDim.y + r) * 2) * a.n_sub;
    if (c < a.n_sub) {
        const int lo = c * a.sub, hi = min(a.V, lo + a.sub);
        double sw = 0.0, sp = 0.0;
        auto add = [&](float p, float q) {
            sp += weight(p);
            if (w.q) sw += weight(p, q);
        };
        if (a.wide) {
#pragma unroll 4
            for (int j = lo + 4 * lane; j < hi; j += 256) {
                const float4 p = *(const float4 *)(w.p + j);
                const float4 q = w.q ? *(const float4 *)(w.q + j) : make_float4(0.f, 0.f, 0.f, 0.f);
                add(p.x, q.x);
                add(p.y, q.y);
                add(p.z, q.z);
                add(p.w, q.w);
            }
        } else {
#pragma unroll 8
            for (int j = lo + lane; j < hi; j += 64) add(w.p[j], w.q ? w.q[j] : 0.f);
        }
        sp = wave_sum_d_dpp(sp);
        sw = w.q ? wave_sum_d_dpp(sw) : sp;
        if (lane == 0) {
            put(part + c, sw);
            put(part + a.n_sub + c, sp);
        }
    }
    unsigned *arrived = a.arrived + s * (VF_MAX_ROWS + 2);
    if (!last_to_arrive(arrived + 1 + r, gridDim.x)) return;
    if (wave == 0) {
        const int j = vf_draw(a, w, part, vf_u(a, in)[s * (a.rows + 1) + (a.tree ? r : a.rows)]);
        if (lane == 0) {
            if (a.tree) {
                put(a.drawn + s * (a.rows + 1) + r, j);
            } else {
                to_host(a.out + s * (3 + a.rows) + 1, w.n);
                to_host(a.out + s * (3 + a.rows) + 2, j);
            }
        }
        if (!a.tree) vf_done(a, s);
    }
    if (!a.tree || !last_to_arrive(arrived, gridDim.y)) return;
    if (wave != 0) return;
    vf_walk(a, in, d, s);
    vf_done(a, s);
}

// Checks, uploads, runs and waits: *res is the pinned result [n_seq][3 + rows].
int vf_run(const char *what, scry_buf p, scry_buf q, const int64_t *tokens, const int32_t *counts, const int64_t *parents,
           const double *u, int n_seq, int rows, int vocab, const int **res) {
    const bool tree = !q;
    if (vocab <= 0 || rows < 1) return set_error(SCRY_ERR_INVALID, "%s: vocabulary and rows must be > 0", what);
    if (vocab > 1 << 30) return set_error(SCRY_ERR_UNSUPPORTED, "%s: vocabulary %d (at most 2^30)", what, vocab);
    if (rows > VF_MAX_ROWS)
        return set_error(SCRY_ERR_UNSUPPORTED, "%s: %d drafted tokens a sequence (at most %d)", what, rows, VF_MAX_ROWS);
    const int32_t zero[PF_MAX_SEQS] = {};
    DraftBatch d;
    SCRY_TRY(draft_batch(what, n_seq, rows, zero, parents, &d));
    if (!tokens || !u) return set_error(SCRY_ERR_INVALID, "%s: null tokens or random numbers", what);
    const size_t V = vocab, m = rows, n = n_seq * (m + 1);
    if (p->n != n * V || (q && q->n != n_seq * m * V)) return set_error(SCRY_ERR_INVALID, "%s: shape mismatch", what);
    VfArgs a{};
    a.p = p->d;
    a.q = q ? q->d : nullptr;
    a.V = vocab;
    a.rows = rows;
    a.tree = tree;
    a.wide = V % 4 == 0;
    const int R = tree ? rows + 1 : 1;
    // a wave's part: 512 values (8 a lane; 16 chains at V = 128256 22 us a call, 25
    // at 256 values, 24 at 1024), more where that gives more workgroups than the
    // chip runs at once (four trees of 31 nodes 38 us; 42 at half as many workgroups
    // or twice as many)
    size_t sub = 512;
    while (sub < 4096 && (V + 4 * sub - 1) / (4 * sub) * R * n_seq > 2048) sub *= 2;
    a.sub = (int)sub;
    a.n_sub = (int)((V + sub - 1) / sub);

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
    const size_t out_bytes = (n_seq * (m + 3) * sizeof(int) + 255) & ~(size_t)255;
    DeviceScope dev;
    char *host = nullptr;
    SCRY_TRY(host_block(out_bytes + n * (sizeof(double) + sizeof(int)), (void **)&host));
    a.out = (int *)host;
    for (int s = 0; s < n_seq; s++) a.out[s * (m + 3)] = 0;  // (no launch writes them any more)
    std::memcpy(big ? (double *)(host + out_bytes) : in.u, hu, n * sizeof(double));
    std::memcpy(big ? (int *)(host + out_bytes + n * sizeof(double)) : in.tok, ht, n * sizeof(int));

    // workspace: sums of the parts, drawn tokens, inputs too many for the arguments
    const size_t part = (size_t)n_seq * R * 2 * a.n_sub * sizeof(double), drawn = (n * sizeof(int) + 7) & ~(size_t)7;
    char *ws = nullptr;
    SCRY_TRY(ctx_workspace(part + drawn + n * (sizeof(double) + sizeof(int)), (void **)&ws));
    a.part = (double *)ws;
    a.drawn = (int *)(ws + part);
    hipStream_t st = ctx().stream;
    static_assert((size_t)PF_MAX_SEQS * (VF_MAX_ROWS + 2) <= DRAFT_COUNTERS, "counters");
    SCRY_TRY(draft_counters(&a.arrived));
    if (big) {
        a.u = (double *)(ws + part + drawn);
        a.tok = (int *)(a.u + n);
        SCRY_HIP(hipMemcpyAsync((void *)a.u, host + out_bytes, n * (sizeof(double) + sizeof(int)), hipMemcpyHostToDevice, st));
    }
    hipLaunchKernelGGL(k_verify, dim3((a.n_sub + 3) / 4, R, n_seq), dim3(256), 0, st, a, in, d);
    hipError_t e = hipGetLastError();
    // The results are there when every sequence is done: the host looks for that
    // for a while, which is 4 us sooner than the stream's own end is known (one chain
    // at V = 32000 22.5 -> 18.3 us), and behind longer work, or where a result does
    // not come, waits for the stream, which says why.
    const volatile int *flag = a.out;
    auto done = [&] {
        for (int s = 0; s < n_seq; s++)
            if (!flag[s * (m + 3)]) return false;
        return true;
    };
    const auto until = std::chrono::steady_clock::now() + std::chrono::milliseconds(20);
    bool seen = false;
    while (e == hipSuccess && !(seen = done()) && std::chrono::steady_clock::now() < until) {
    }
    std::atomic_thread_fence(std::memory_order_acquire);
    if (!seen) {
        const hipError_t w = hipStreamSynchronize(st);
        if (e == hipSuccess) e = w;
        if (e != hipSuccess) return hip_fail(e, what, __FILE__, __LINE__);
    }
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
        accepted[s] = r[(size_t)s * (rows + 3) + 1];
        token[s] = r[(size_t)s * (rows + 3) + 2];
    }
    return SCRY_OK;
}

int scry_hip_verify_tree(scry_buf p, const int64_t *tokens, const int64_t *parents, const double *u, int n_seq, int rows,
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
        const int *x = r + (size_t)s * (rows + 3) + 1;
        accepted[s] = x[0];
        token[s] = x[1];
        for (int i = 0; i < rows; i++) paths[(size_t)s * rows + i] = x[2 + i];
    }
    return SCRY_OK;
}

}  // extern "C"
