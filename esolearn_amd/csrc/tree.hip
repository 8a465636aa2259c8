// Attention of drafted tokens over a cache: row i of sequence s attends to its
// context's rows [0, len) and, among the drafted rows len + j, to its
// ancestors and itself.
//   o_i = sum_t p_t v_t / sum_t p_t,   p_t = 2^(s_t - c),  s_t = scale log2(e) q_i.k_t
// for any c, the running reference of one pass over the keys.  The cache is
// read in place: f32 rows [max_seq, n_kv * hd] or the int8 cache.
//
// A column is one (row, query head) of a KV head, rows * nrep of them, in tiles
// of 16.  Both kernels compute the scores transposed, keys x columns, so that a
// lane holds the scores of one column for 4 keys of each 16: the running
// maximum and sum are lane values joined over 4 lanes, and the weights are
// already the operand that the products p.v take, without a pass through LDS.
// Few columns (narrow kernels): a workgroup has one tile, each of its four waves
// every fourth step of keys, and they are joined through LDS.  Many (wide): a
// wave has a tile, and the workgroup's tiles share each step's keys through LDS.
// Where the keys are split over workgroups too, the last of them or k_tree_merge*
// joins the splits.
//
// Workgroups go to the XCDs round-robin: those of one (sequence, KV head,
// split) share their keys and sit on one XCD, so the keys come from its L2
// after the first.
#include <cmath>

#include "arrive.h"
#include "kdev.h"
#include "kv8.h"

namespace scry {
namespace {

using namespace dev;

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

struct F32Batch {
    const float *k[PF_MAX_SEQS], *v[PF_MAX_SEQS];
};

struct TreeArgs {
    DraftBatch d;
    const float *q;  // [n_seq * rows, n_q * hd]
    float *out;
    float *part_o, *part_ml;  // n_split > 1: [column][split][hd], [column][split][2] (c, sum)
    int n_q, n_kv, hd, nrep, cols;  // cols = rows * nrep
    // Key splits of each sequence, alike in size across them; a split's unit is
    // (sequence, KV head, split), numbered from pair0[s] on.  n_split: the most.
    int n_split, n_qg, near;  // n_qg: groups of the workgroup's columns; near: of a chain's pairs, those in one order
    int splits[PF_MAX_SEQS], pair0[PF_MAX_SEQS + 1];
    float scale2;                   // scale * log2(e)
    unsigned *arrived;  // splits per (sequence, KV head, column group), zero between launches; null: k_tree_merge* join
};

constexpr int WAVES = 4;

// What a wave's lane knows of its column (lane % 16 of a tile): keys below lim
// and the drafted rows of mask are seen.
struct Column {
    int lim;
    unsigned long long mask;
    bool none;  // no such column, or no node
};

struct Unit {  // a workgroup's part of the work
    int s, g, split, qg;
};
// A chain's later column groups see more keys: `near` pairs at a time, the groups
// go from the longest to the shortest, and to and fro over an XCD's 32 CUs
// (neighbours in the order sit on neighbours), so that each gets long and short
// ones (a 2000-row prompt, 32 heads of 128: f32 332 us, in plain order 591, int8
// 104 and 138; half as many pairs near 357 and 109, twice as many the same).
__device__ __forceinline__ bool unit_of(const TreeArgs &a, Unit &u) {
    const int i = blockIdx.x;
    int t = i >> 3, local = t / a.n_qg;
    u.qg = t % a.n_qg;
    if (!a.d.tree && a.n_qg > 1) {
        const int all = (a.pair0[a.d.n_seq] + 7) >> 3, at = local / a.near * a.near, n = min(a.near, all - at);
        const int r = t - at * a.n_qg, row = r & ~31, end = min(row + 32, n * a.n_qg);
        t = r & 32 ? row + end - 1 - r : r;
        local = at + t % n;
        u.qg = a.n_qg - 1 - t / n;
    }
    const int pair = (i & 7) + 8 * local;
    if (pair >= a.pair0[a.d.n_seq]) return false;  // padding of the last eight
    u.s = 0;
    while (pair >= a.pair0[u.s + 1]) u.s++;
    const int own = pair - a.pair0[u.s];
    u.split = own % a.splits[u.s];
    u.g = own / a.splits[u.s];
    return true;
}

// Node `lane`'s ancestors and itself, by pointer jumping: after k steps a mask
// holds the nearest 2^k of them.
__device__ __forceinline__ unsigned long long ancestor_mask(const DraftBatch &d, int s) {
    const int lane = threadIdx.x & 63;
    int up = lane < d.rows ? (int)d.parent[s][lane] : -1;
    unsigned long long m = up == -2 ? 0 : 1ull << lane;
#pragma unroll
    for (int k = 0; k < 6; k++) {
        const unsigned long long pm = __shfl(m, up & 63);
        const int pu = __shfl(up, up & 63);
        if (up >= 0) {
            m |= pm;
            up = pu;
        }
    }
    return m;
}

__device__ __forceinline__ Column column_of(const TreeArgs &a, int s, int c, unsigned long long anc) {
    const int node = c < a.cols ? c / a.nrep : -1, len = a.d.len[s];
    Column r{0, 0, true};
    if (!a.d.tree) {
        if (node >= 0) r = {len + node + 1, 0, false};
    } else {
        const unsigned long long m = __shfl(anc, node & 63);
        if (node >= 0 && m) r = {len, m, false};
    }
    return r;
}
__device__ __forceinline__ bool sees(const Column &c, int t, int len) {
    const int j = t - len;
    return t < c.lim || ((unsigned)j < 64u && (c.mask >> j & 1));
}

// Largest value over the four lanes of a column; their sum.  The swaps give
// every lane its own value and that of the lane 16 (32) away, without LDS.
__device__ __forceinline__ float2 swap16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float2 swap32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float col_max(float v) {
    float2 p = swap16(v);
    p = swap32(fmaxf(p.x, p.y));
    return fmaxf(p.x, p.y);
}
__device__ __forceinline__ float col_sum(float v) {
    float2 p = swap16(v);
    p = swap32(p.x + p.y);
    return p.x + p.y;
}
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Four dimensions of column c's output: o times 1 / l, or zero where there is no node.
__device__ __forceinline__ void store_out(const TreeArgs &a, int s, int g, int c, int d, float4 o, float inv) {
    const int node = c / a.nrep, h = g * a.nrep + c % a.nrep;
    float4 r = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    if (a.d.tree && a.d.parent[s][node] == -2) r = make_float4(0.f, 0.f, 0.f, 0.f);
    *(float4 *)(a.out + (((size_t)s * a.d.rows + node) * a.n_q + h) * a.hd + d) = r;
}
__device__ __forceinline__ size_t part_of(const TreeArgs &a, const Unit &u, int c) {
    return (((size_t)u.s * a.n_kv + u.g) * a.cols + c) * a.n_split + u.split;
}
// A split's partial: read in this launch by the last split to arrive (put /
// get), or by the next launch.
__device__ __forceinline__ void store_part(const TreeArgs &a, size_t at, int d, float4 v) {
    float *p = a.part_o + at * a.hd + d;
    if (a.arrived) {
        put((unsigned long long *)p, __builtin_bit_cast(unsigned long long, make_float2(v.x, v.y)));
        put((unsigned long long *)p + 1, __builtin_bit_cast(unsigned long long, make_float2(v.z, v.w)));
    } else {
        *(float4 *)p = v;
    }
}
__device__ __forceinline__ void store_ml(const TreeArgs &a, size_t at, float c, float l) {
    float *p = a.part_ml + at * 2;
    if (a.arrived)
        put((unsigned long long *)p, __builtin_bit_cast(unsigned long long, make_float2(c, l)));
    else
        *(float2 *)p = make_float2(c, l);
}
__device__ __forceinline__ float2 get2(const float *p) {
    return __builtin_bit_cast(float2, get((const unsigned long long *)p));
}
__device__ __forceinline__ bool last_split(const TreeArgs &a, const Unit &u) {
    return last_to_arrive(a.arrived + ((size_t)u.s * a.n_kv + u.g) * a.n_qg + u.qg, a.splits[u.s]);
}

// The tile of a wide kernel's wave: a wave stays on its SIMD, so tiles that are
// not there (seven in two groups of four) go round.
template <int W>
__device__ __forceinline__ int tile_of(const Unit &u, int wave) {
    return (wave + u.g + u.split) % W;
}

// A wide kernel's wave ends: the output of its columns, or a split's partial.
template <int N, class DIM>
__device__ __forceinline__ void finish_wide(const TreeArgs &a, const Unit &u, int c, float own_c, float own_l, float4 (&o)[N], DIM dim) {
    if (c >= a.cols) return;
    const size_t at = part_of(a, u, c);
    const float inv = 1.f / own_l;
#pragma unroll
    for (int x = 0; x < N; x++) {
        if (dim(x) >= a.hd) continue;
        if (a.n_split == 1)
            store_out(a, u.s, u.g, c, dim(x), o[x], inv);
        else
            *(float4 *)(a.part_o + at * a.hd + dim(x)) = o[x];
    }
    if (a.n_split > 1 && (threadIdx.x & 63) < 16) *(float2 *)(a.part_ml + at * 2) = make_float2(own_c, own_l);
}

// The four waves' (c, sum, out) of each column joined in wave order, from
// s_o [wave][column][ld], s_c and s_l [wave][column]: the output, or one split's
// partial.  Factors are 2^(c - max c); a wave without keys has c = -inf.
template <int COLS>
__device__ __forceinline__ void join_waves(const TreeArgs &a, const Unit &u, const float *s_o, const float *s_c,
                                           const float *s_l, int ld) {
    __syncthreads();
    const int hd = a.hd, n4 = hd / 4;
    for (int x = threadIdx.x; x < COLS * n4; x += 64 * WAVES) {
        const int col = x / n4, d = 4 * (x % n4), c = u.qg * COLS + col;
        if (c >= a.cols) break;  // columns ascend
        float C = -INFINITY;
#pragma unroll
        for (int w = 0; w < WAVES; w++) C = fmaxf(C, s_c[w * COLS + col]);
        const float ref = C == -INFINITY ? 0.f : C;
        float L = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            const float f = exp2_fast(s_c[w * COLS + col] - ref);
            const float4 v = *(const float4 *)(s_o + (w * COLS + col) * ld + d);
            L += s_l[w * COLS + col] * f;
            o.x += v.x * f;
            o.y += v.y * f;
            o.z += v.z * f;
            o.w += v.w * f;
        }
        if (a.n_split == 1) {
            store_out(a, u.s, u.g, c, d, o, 1.f / L);
        } else {
            const size_t at = part_of(a, u, c);
            store_part(a, at, d, o);
            if (d == 0) store_ml(a, at, C, L);
        }
    }
    if (a.n_split == 1 || !a.arrived || !last_split(a, u)) return;
    // the last split of these columns: a thread per four dimensions
    const int ns = a.splits[u.s];
    for (int x = threadIdx.x; x < COLS * n4; x += 64 * WAVES) {
        const int d = 4 * (x % n4), c = u.qg * COLS + x / n4;
        if (c >= a.cols) break;
        const size_t at = part_of(a, u, c) - u.split;
        float C = -INFINITY, L = 0.f;
        float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int p0 = 0; p0 < ns; p0 += 8) {  // eight splits' loads before their first use
            float2 ml[8], lo[8], hi[8];
#pragma unroll
            for (int p = 0; p < 8; p++) {
                const size_t q = at + min(p0 + p, ns - 1);
                ml[p] = get2(a.part_ml + q * 2);
                lo[p] = get2(a.part_o + q * hd + d);
                hi[p] = get2(a.part_o + q * hd + d + 2);
            }
            float top = C;
#pragma unroll
            for (int p = 0; p < 8; p++) top = fmaxf(top, ml[p].x);
            const float ref = top == -INFINITY ? 0.f : top, f0 = exp2_fast(C - ref);
            C = top;
            L *= f0;
            r = make_float4(r.x * f0, r.y * f0, r.z * f0, r.w * f0);
#pragma unroll
            for (int p = 0; p < 8; p++) {
                if (p0 + p >= ns) break;
                const float f = exp2_fast(ml[p].x - ref);
                L += ml[p].y * f;
                r.x += lo[p].x * f;
                r.y += lo[p].y * f;
                r.z += hi[p].x * f;
                r.w += hi[p].y * f;
            }
        }
        store_out(a, u.s, u.g, c, d, r, 1.f / L);
    }
}

// The splits of a column joined in a fixed order.  A workgroup takes `per`
// columns: a wave finds a column's factors, a lane per split; then 256 / per
// threads sum its splits, lanes of four dimensions times groups of splits, and
// the groups are joined through LDS.
constexpr int MAX_SPLIT = 64;
__global__ __launch_bounds__(256) void k_tree_merge(TreeArgs a, int per, int lanes) {
    __shared__ float s_f[16 * MAX_SPLIT], s_l[16];
    __shared__ float4 s_p[256];
    const int tid = threadIdx.x, lane = tid & 63, hd = a.hd, g = blockIdx.y, s = blockIdx.z, ns = a.splits[s];
    const int c0 = blockIdx.x * per;
    const size_t col0 = ((size_t)s * a.n_kv + g) * a.cols + c0;
    for (int i = tid >> 6; i < per && c0 + i < a.cols; i += 4) {
        float2 ml = make_float2(-INFINITY, 0.f);
        if (lane < ns) ml = *(const float2 *)(a.part_ml + ((col0 + i) * a.n_split + lane) * 2);
        float C = ml.x;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) C = fmaxf(C, __shfl_xor(C, off));
        const float f = exp2_fast(ml.x - (C == -INFINITY ? 0.f : C));
        const float L = wave_sum(ml.y * f);
        s_f[i * MAX_SPLIT + lane] = f;
        if (lane == 0) s_l[i] = L;
    }
    __syncthreads();
    const int n_grp = 256 / (per * lanes), x = tid % lanes, grp = tid / lanes % n_grp, i = tid / (lanes * n_grp);
    const bool act = c0 + i < a.cols && 4 * x < hd;
    float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
    if (act) {
        const float *o = a.part_o + (col0 + i) * a.n_split * hd + 4 * x;
#pragma unroll 8
        for (int p = grp; p < ns; p += n_grp) {
            const float f = s_f[i * MAX_SPLIT + p];
            const float4 v = *(const float4 *)(o + (size_t)p * hd);
            r.x += v.x * f;
            r.y += v.y * f;
            r.z += v.z * f;
            r.w += v.w * f;
        }
    }
    s_p[tid] = r;
    __syncthreads();
    if (grp || !act) return;
    for (int k = 1; k < n_grp; k++) {
        const float4 v = s_p[tid + k * lanes];
        r.x += v.x;
        r.y += v.y;
        r.z += v.z;
        r.w += v.w;
    }
    store_out(a, s, g, c0 + i, 4 * x, r, 1.f / s_l[i]);
}

// Many columns: a thread takes four dimensions of one, its splits eight at a
// time (loads before their first use: a round trip to memory each time).
// blockIdx.y: the KV head, blockIdx.z: the sequence (64-bit divisions of one
// linear index took more time than the loads).
__global__ __launch_bounds__(256) void k_tree_merge_flat(TreeArgs a) {
    const unsigned t = blockIdx.x * 256 + threadIdx.x, n4 = (unsigned)a.hd / 4;
    const int x = (int)(t % n4), c = (int)(t / n4), g = blockIdx.y, s = blockIdx.z;
    if (c >= a.cols) return;
    const size_t col = ((size_t)s * a.n_kv + g) * a.cols + c;
    const int ns = a.splits[s];
    const float2 *ml = (const float2 *)(a.part_ml + col * a.n_split * 2);
    const float *o = a.part_o + col * a.n_split * a.hd + 4 * x;
    float C = -INFINITY, L = 0.f;
    float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p0 = 0; p0 < ns; p0 += 8) {
        float2 m[8];
        float4 v[8];
#pragma unroll
        for (int p = 0; p < 8; p++) {
            const int q = min(p0 + p, ns - 1);
            m[p] = ml[q];
            v[p] = *(const float4 *)(o + (size_t)q * a.hd);
        }
        float top = C;
#pragma unroll
        for (int p = 0; p < 8; p++) top = fmaxf(top, m[p].x);
        const float ref = top == -INFINITY ? 0.f : top, f0 = exp2_fast(C - ref);
        C = top;
        L *= f0;
        r = make_float4(r.x * f0, r.y * f0, r.z * f0, r.w * f0);
#pragma unroll
        for (int p = 0; p < 8; p++) {
            if (p0 + p >= ns) break;
            const float f = exp2_fast(m[p].x - ref);
            L += m[p].y * f;
            r.x += v[p].x * f;
            r.y += v[p].y * f;
            r.z += v[p].z * f;
            r.w += v[p].w * f;
        }
    }
    store_out(a, s, g, c, 4 * x, r, 1.f / L);
}

// The steps of SK keys that a workgroup takes of the keys that its columns see.
template <int SK>
__device__ __forceinline__ void step_range(const TreeArgs &a, const Unit &u, int cols, int *lo, int *hi) {
    int rows = a.d.rows;
    if (!a.d.tree) rows = min(rows, (min(a.cols, (u.qg + 1) * cols) - 1) / a.nrep + 1);
    const unsigned steps = (unsigned)(a.d.len[u.s] + rows + SK - 1) / SK, ns = a.splits[u.s], each = steps / ns, more = steps % ns;
    *lo = (int)(u.split * each + min((unsigned)u.split, more));
    *hi = *lo + (int)(each + ((unsigned)u.split < more));
}

// ------------------------------------------------------------ int8 cache
// q.k: K's bytes are an operand as they lie; q is held as 24-bit integers of
// its row's largest value in three balanced int8 digits, so the products and
// their sums over hd are exact integers.
// p.v: V's bytes become f16 (exact), and w = p * (the row's scale) is split
// into two f16 terms, each rounded to the nearest: 2^-24 of w, or where w is
// small f16's smallest steps.  c starts as max s + log2(the largest scale) - 12
// and moves where a w passes 2^15, so those steps lie 2^-36 below the largest w
// or further.  Scales below 2^-80 count as 2^-80 there, which keeps 2^-c in f32's
// range.
// KS: steps of 64 dimensions (hdp <= 64 KS).

// Column c's query as digits: lane (cl, j) holds dimensions 64 k + 16 j ..;
// returns what a score's integer is multiplied by (but the key's scale).
template <int KS>
__device__ __forceinline__ float query_digits(const TreeArgs &a, const Unit &u, int c, int j, i32x4 (&qd)[3][KS]) {
    const int cc = min(c, a.cols - 1), node = cc / a.nrep, rep = cc % a.nrep, hd = a.hd;
    const float *q = a.q + (((size_t)u.s * a.d.rows + node) * a.n_q + u.g * a.nrep + rep) * hd;
    float4 x[KS][4];
    float m = 0.f;
    bool nan = false;
#pragma unroll
    for (int k = 0; k < KS; k++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int d = 64 * k + 16 * j + 4 * e;
            x[k][e] = d < hd ? *(const float4 *)(q + d) : make_float4(0.f, 0.f, 0.f, 0.f);
            const float4 v = x[k][e];
            m = fmaxf(m, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
            nan |= __builtin_isunordered(v.x, v.y) || __builtin_isunordered(v.z, v.w);
        }
    // a query with an infinity or NaN has no finite softmax over any key
    m = col_max(nan ? INFINITY : fmaxf(m, 0x1p-96f));
    const float up = m < INFINITY ? 8290000.f / m : 0.f;  // 126.5 * 2^16: the top digit stays below 128
#pragma unroll
    for (int k = 0; k < KS; k++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float v[4] = {x[k][e].x, x[k][e].y, x[k][e].z, x[k][e].w};
            int X[4];
#pragma unroll
            for (int i = 0; i < 4; i++) X[i] = __float2int_rn(v[i] * up);
#pragma unroll
            for (int g = 0; g < 3; g++) {  // a digit is the low byte; with it taken off, (X + 128) >> 8 is left
                const unsigned w01 = __builtin_amdgcn_perm((unsigned)X[1], (unsigned)X[0], 0x0c0c0400u);
                const unsigned w23 = __builtin_amdgcn_perm((unsigned)X[3], (unsigned)X[2], 0x0c0c0400u);
                qd[g][k][e] = (int)__builtin_amdgcn_perm(w23, w01, 0x05040100u);
#pragma unroll
                for (int i = 0; i < 4; i++) X[i] = (X[i] + 128) >> 8;
            }
        }
    return m < INFINITY ? m / 8290000.f * a.scale2 : __builtin_nanf("");
}

// The integer scores of N blocks of 16 keys, digits joined: h 256 + b, the sums
// h and b exact.  b starts at the bits of 1.5 * 2^23, so that b + 1.5 * 2^23 is
// an f32 as it stands (|b| < 2^22: hd products of two digits), and h at -192,
// which its two bytes take back.  The blocks' products are interleaved: a
// chain of one block's would wait for itself.
template <int KS, int N>
__device__ __forceinline__ void digit_scores(const i32x4 (&kk)[N][KS], const i32x4 (&qd)[3][KS], f32x4 *sc) {
    i32x4 h[N], b[N];
#pragma unroll
    for (int x = 0; x < N; x++) {
        h[x] = i32x4{-192, -192, -192, -192};
        b[x] = i32x4{0x4b400000, 0x4b400000, 0x4b400000, 0x4b400000};
    }
#pragma unroll
    for (int k = 0; k < KS; k++)
#pragma unroll
        for (int x = 0; x < N; x++) {
            h[x] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kk[x][k], qd[2][k], h[x], 0, 0, 0);
            b[x] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kk[x][k], qd[0][k], b[x], 0, 0, 0);
        }
#pragma unroll
    for (int x = 0; x < N; x++) h[x] = h[x] << 8;
#pragma unroll
    for (int k = 0; k < KS; k++)
#pragma unroll
        for (int x = 0; x < N; x++) h[x] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kk[x][k], qd[1][k], h[x], 0, 0, 0);
#pragma unroll
    for (int x = 0; x < N; x++)
#pragma unroll
        for (int i = 0; i < 4; i++) sc[x][i] = fmaf((float)h[x][i], 256.f, __int_as_float(b[x][i]));
}

// A column's running state: the reference c, the largest score and the
// exponent of the largest scale - 12 when it last moved, the sum of the weights.
struct RunI8 {
    float c = -INFINITY, m = -INFINITY, ve = -92.f, l = 0.f;
};

// Weights as two f16 terms, in the order of the operands of w.v.
__device__ __forceinline__ void split_weights(const float (&w)[4], int x, f16x8 (&wh)[2], f16x8 (&wl)[2]) {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const f16x2 h = __builtin_convertvector((f32x2{w[i], w[i + 1]}), f16x2);
        const f16x2 lo = __builtin_convertvector((f32x2{fmaf(-(float)h[0], 1.f, w[i]), fmaf(-(float)h[1], 1.f, w[i + 1])}), f16x2);
        wh[x / 2][4 * (x % 2) + i] = h[0];
        wh[x / 2][4 * (x % 2) + i + 1] = h[1];
        wl[x / 2][4 * (x % 2) + i] = lo[0];
        wl[x / 2][4 * (x % 2) + i + 1] = lo[1];
    }
}

// One step's 64 scores of a column (16 a lane; key 16 x + 4 j + i at [x][i];
// sc is multiplied by kq for the score) and the rows' scales into the operands
// of w.v.  Where the reference moves, l is rescaled and o's factor is returned
// (1: o stays).  The reference need not be the largest score: it is kept while
// the weights fit f16 and the sum f32, so most steps neither look for a
// maximum nor rescale (a 512-row chunk over 1500 rows of 32 heads: 63 -> 58 us).
template <class KQ, class VS>
__device__ __forceinline__ float softmax_step(RunI8 &r, const f32x4 (&sc)[4], KQ &&kq, VS &&vs, bool full, const Column &co, int t,
                                              int len, f16x8 (&wh)[2], f16x8 (&wl)[2]) {
    if (full) {
        float sum = 0.f, top = 0.f;
#pragma unroll
        for (int x = 0; x < 4; x++) {
            const f32x4 k = kq(x), v = vs(x);
            float w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float p = exp2_fast(fmaf(sc[x][i], k[i], -r.c));
                sum += p;
                w[i] = p * v[i];
            }
            top = fmaxf(fmaxf(fmaxf(fmaxf(top, w[0]), w[1]), w[2]), w[3]);
            split_weights(w, x, wh, wl);
        }
        // (a NaN weight makes the sum a NaN)
        if (!__any(!(top <= 0x1p15f && sum <= 0x1p96f))) {
            r.l += sum;
            return 1.f;
        }
    }
    float vm = 0.f, mx = -INFINITY, s[4][4];
    unsigned seen = 0;
#pragma unroll
    for (int x = 0; x < 4; x++) {
        const f32x4 k = kq(x), v = vs(x);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const bool in = full || sees(co, t + 16 * x + i, len);
            seen |= (unsigned)in << (4 * x + i);
            s[x][i] = in ? sc[x][i] * k[i] : -INFINITY;
            vm = fmaxf(vm, in ? v[i] : 0.f);
            mx = fmaxf(mx, s[x][i]);
        }
    }
    vm = col_max(vm);
    r.m = fmaxf(r.m, col_max(mx));
    // 2^e >= the largest scale * 2^-12, e >= -92
    r.ve = fmaxf(r.ve, (float)((int)((__float_as_uint(fmaxf(vm, 0x1p-80f)) + 0x7fffffu) >> 23) - 127 - 12));
    // no score yet: a reference that the first one exceeds
    const float c = r.m == -INFINITY ? -INFINITY : r.m + r.ve, ref = c == -INFINITY ? 0.f : c;
    const float al = r.c == -INFINITY ? 0.f : exp2_fast(r.c - ref);
    r.c = c;
    float sum = 0.f;
#pragma unroll
    for (int x = 0; x < 4; x++) {
        const f32x4 v = vs(x);
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float p = exp2_fast(s[x][i] - ref);
            sum += p;
            w[i] = seen >> (4 * x + i) & 1 ? p * v[i] : 0.f;  // an unseen scale may be NaN
        }
        split_weights(w, x, wh, wl);
    }
    r.l = r.l * al + sum;
    return al;
}

// Eight of a dimension's V bytes (two words of four rows) as f16: byte v + 128
// behind 0x64 is 1024 + v + 128.
__device__ __forceinline__ f16x8 v_operand(int w0, int w1) {
    i32x4 r;
#pragma unroll
    for (int i = 0; i < 4; i++)
        r[i] = __builtin_bit_cast(int, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, (unsigned)(i < 2 ? w0 : w1),
                                                                                        i % 2 ? 0x04030402u : 0x04010400u)) -
                                           f16x2{(_Float16)1152.f, (_Float16)1152.f});
    return __builtin_bit_cast(f16x8, r);
}

// Few columns (one tile a workgroup): bound by reading the cache.  Keys go
// from memory to the operands, every wave with steps of its own.  One token of
// 32 heads (8 of K and V, 128 dimensions) over 65001 rows: 137 MB in 28.7 us.
template <int KS>
__global__ __launch_bounds__(64 * WAVES, KS <= 2 ? 2 : 1) void k_tree_i8(TreeArgs a, Kv8Batch cb) {
    constexpr int DT = 4 * KS, COLS = 16;
    extern __shared__ __align__(16) float sm[];
    Unit u;
    if (!unit_of(a, u)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cl = lane & 15, j = lane >> 4;
    const int hd = a.hd, hdp = cb.hdp, len = a.d.len[u.s];
    const int c = u.qg * COLS + cl;
    const Column co = column_of(a, u.s, c, a.d.tree ? ancestor_mask(a.d, u.s) : 0);
    i32x4 qd[3][KS];
    const float qs = query_digits<KS>(a, u, c, j, qd);
    RunI8 r;
    f32x4 o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int rows_p = cb.rows_p[u.s];
    const int8_t *kb = cb.k[u.s] + (size_t)u.g * rows_p * hdp, *vb = cb.v[u.s] + (size_t)u.g * rows_p * hdp;
    const float *ksb = cb.ks[u.s] + (size_t)u.g * rows_p, *vsb = cb.vs[u.s] + (size_t)u.g * rows_p;
    int lo, hi;
    step_range<64>(a, u, COLS, &lo, &hi);

    i32x4 kk[4][KS];
    f32x4 ks[4];
    auto load_k = [&](int st) {
        const int8_t *kt = kb + (size_t)st * 64 * hdp;
#pragma unroll
        for (int x = 0; x < 4; x++) {
#pragma unroll
            for (int k = 0; k < KS; k++)
                kk[x][k] = 64 * k + 16 * j < hdp ? *(const i32x4 *)(kt + (16 * x + cl) * hdp + 64 * k + 16 * j) : i32x4{0, 0, 0, 0};
            ks[x] = *(const f32x4 *)(ksb + st * 64 + 16 * x + 4 * j);
        }
    };
    if (lo + wave < hi) load_k(lo + wave);
    for (int st = lo + wave; st < hi; st += WAVES) {
        const int t0 = st * 64;
        const int8_t *vt = vb + (size_t)t0 * hdp;
        f32x4 vs[4], sc[4], kq[4];
#pragma unroll
        for (int x = 0; x < 4; x++) vs[x] = *(const f32x4 *)(vsb + t0 + 16 * x + 4 * j);
        digit_scores<KS, 4>(kk, qd, sc);
#pragma unroll
        for (int x = 0; x < 4; x++) kq[x] = ks[x] * qs;
        i32x4 vv[DT];  // K is used up: its registers take V
#pragma unroll
        for (int d = 0; d < DT; d++)
            vv[d] = 16 * d < hdp ? *(const i32x4 *)(vt + (16 * d + cl) * 64 + 16 * j) : i32x4{0, 0, 0, 0};
        f16x8 wh[2], wl[2];
        const float al = softmax_step(r, sc, [&](int x) { return kq[x]; }, [&](int x) { return vs[x]; }, t0 + 64 <= len, co, t0 + 4 * j, len, wh, wl);
        if (__any(al != 1.f)) {
#pragma unroll
            for (int d = 0; d < DT; d++) o[d] *= al;
        }
        load_k(min(st + WAVES, hi - 1));  // under the products below
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
            for (int d = 0; d < DT; d += 4) {  // four dimensions' products between two of one
                f16x8 va[4];
#pragma unroll
                for (int e = 0; e < 4; e++) va[e] = v_operand(vv[d + e][2 * x], vv[d + e][2 * x + 1]);
#pragma unroll
                for (int e = 0; e < 4; e++) o[d + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[e], wh[x], o[d + e], 0, 0, 0);
#pragma unroll
                for (int e = 0; e < 4; e++) o[d + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[e], wl[x], o[d + e], 0, 0, 0);
            }
    }

    const int ld = hd + 4, col = wave * COLS + cl;
    float *s_o = sm, *s_c = sm + WAVES * COLS * ld, *s_l = s_c + WAVES * COLS;
    const float sum = col_sum(r.l);
    if (j == 0) {
        s_c[col] = r.c;
        s_l[col] = sum;
    }
#pragma unroll
    for (int d = 0; d < DT; d++)
        if (16 * d + 4 * j < hd) *(f32x4 *)(s_o + col * ld + 16 * d + 4 * j) = o[d];
    join_waves<COLS>(a, u, s_o, s_c, s_l, ld);
}

// Many columns: bound by the arithmetic of the softmax and the conversions, so
// W waves with a tile each share the keys through LDS: each stages a part of
// a step, V as f16 (converted once for the W tiles), in the order in which the
// lanes take their operands, and holds the next step's part in registers.
// 64-node trees of eight 4000-row contexts, 32 heads over 8 of 128: 26 GFLOP (65
// in digits and terms) in 74 us.
template <int KS, int W>
__global__ __launch_bounds__(64 * W, (KS == 1 ? 4 : KS == 2 ? 3 : 2) - (W < 4 ? 1 : 0)) void k_tree_i8_wide(TreeArgs a, Kv8Batch cb) {
    constexpr int DT = 4 * KS, XB = (4 + W - 1) / W, DB = (DT + W - 1) / W;
    __shared__ i32x4 s_k[4][KS][64];
    __shared__ f16x8 s_v[DT][2][64];
    __shared__ f32x4 s_sc[2][16];  // scales of K and V
    Unit u;
    if (!unit_of(a, u)) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int cl = lane & 15, j = lane >> 4;
    const int hd = a.hd, hdp = cb.hdp, len = a.d.len[u.s];
    const int c0 = (u.qg * W + tile_of<W>(u, wave)) * 16, c = c0 + cl;
    const Column co = column_of(a, u.s, c, a.d.tree ? ancestor_mask(a.d, u.s) : 0);
    i32x4 qd[3][KS];
    const float qs = query_digits<KS>(a, u, c, j, qd);
    // keys that any column of this wave sees
    const int end = c0 >= a.cols ? 0 : a.d.tree ? len + a.d.rows : len + min(c0 + 15, a.cols - 1) / a.nrep + 1;
    RunI8 r;
    f32x4 o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int rows_p = cb.rows_p[u.s];
    const int8_t *kb = cb.k[u.s] + (size_t)u.g * rows_p * hdp, *vb = cb.v[u.s] + (size_t)u.g * rows_p * hdp;
    const float *scb = (tid < 64 ? cb.ks[u.s] : cb.vs[u.s]) + (size_t)u.g * rows_p + lane;
    int lo, hi;
    step_range<64>(a, u, 16 * W, &lo, &hi);

    // A lane's offsets in a step's K and V.  Dimensions past hdp are taken from
    // the last ones: they meet zero digits of q, or make outputs nobody stores.
    i32x4 kr[XB][KS], vr[DB];
    int ko[XB][KS], vo[DB];
    float sr = 0.f;
#pragma unroll
    for (int b = 0; b < XB; b++)
#pragma unroll
        for (int k = 0; k < KS; k++) ko[b][k] = (16 * min(W * b + wave, 3) + cl) * hdp + min(64 * k + 16 * j, hdp - 16);
#pragma unroll
    for (int b = 0; b < DB; b++) vo[b] = min(16 * (W * b + wave) + cl, hdp - 1) * 64 + 16 * j;
    auto fetch = [&](int st) {
        const int8_t *kt = kb + (size_t)st * 64 * hdp, *vt = vb + (size_t)st * 64 * hdp;
#pragma unroll
        for (int b = 0; b < XB; b++)
#pragma unroll
            for (int k = 0; k < KS; k++) kr[b][k] = *(const i32x4 *)(kt + ko[b][k]);
#pragma unroll
        for (int b = 0; b < DB; b++) vr[b] = *(const i32x4 *)(vt + vo[b]);
        if (tid < 128) sr = scb[(size_t)st * 64];
    };
    if (lo < hi) fetch(lo);
    for (int st = lo; st < hi; st++) {
        const int t0 = st * 64;
        __syncthreads();  // the step before has been read
#pragma unroll
        for (int b = 0; b < XB; b++)
            if (W * b + W <= 4 || W * b + wave < 4)
#pragma unroll
                for (int k = 0; k < KS; k++) s_k[W * b + wave][k][lane] = kr[b][k];
#pragma unroll
        for (int b = 0; b < DB; b++)
            if (W * b + W <= DT || W * b + wave < DT) {
                s_v[W * b + wave][0][lane] = v_operand(vr[b][0], vr[b][1]);
                s_v[W * b + wave][1][lane] = v_operand(vr[b][2], vr[b][3]);
            }
        if (tid < 128) ((float *)s_sc)[tid] = sr;
        __syncthreads();
        fetch(min(st + 1, hi - 1));
        if (t0 >= end) continue;  // (uniform in the wave)
        f32x4 sc[4];
#pragma unroll
        for (int x = 0; x < 4; x += 2) {
            i32x4 kk[2][KS];
#pragma unroll
            for (int k = 0; k < KS; k++) {
                kk[0][k] = s_k[x][k][lane];
                kk[1][k] = s_k[x + 1][k][lane];
            }
            digit_scores<KS, 2>(kk, qd, sc + x);
        }
        f16x8 wh[2], wl[2];
        const float al = softmax_step(r, sc, [&](int x) { return s_sc[0][4 * x + j] * qs; }, [&](int x) { return s_sc[1][4 * x + j]; }, t0 + 64 <= len, co, t0 + 4 * j, len, wh, wl);
        if (__any(al != 1.f)) {
#pragma unroll
            for (int d = 0; d < DT; d++) o[d] *= al;
        }
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
            for (int d = 0; d < DT; d += 4) {  // four dimensions' products between two of one
                f16x8 va[4];
#pragma unroll
                for (int e = 0; e < 4; e++) va[e] = s_v[d + e][x][lane];
#pragma unroll
                for (int e = 0; e < 4; e++) o[d + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[e], wh[x], o[d + e], 0, 0, 0);
#pragma unroll
                for (int e = 0; e < 4; e++) o[d + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va[e], wl[x], o[d + e], 0, 0, 0);
            }
    }

    float4 v[DT];
#pragma unroll
    for (int d = 0; d < DT; d++) v[d] = make_float4(o[d][0], o[d][1], o[d][2], o[d][3]);
    finish_wide(a, u, c, r.c, col_sum(r.l), v, [&](int d) { return 16 * d + 4 * j; });
}

// ------------------------------------------------------------- f32 cache
// Products on the f32 matrix instructions (16 x 16 x 4): f32 sums of f32
// products.  Which four dimensions, or keys, an instruction takes is free as
// long as both operands agree: lane (cl, j) loads K rows as float4 of
// dimensions 16 c + 4 j .. (element e is instruction (c, e)'s operand), and V
// rows 4 j + i as float4 of dimensions 64 e + 4 cl .., so every load is 16
// bytes wide and a row's lanes are neighbours.
// ET: blocks of 64 dimensions.

// One step's 16 KB scores of a column (4 KB a lane; key 16 y + 4 j + i at [y][i])
// into weights; l is rescaled where the reference moves and o's factor returned
// (1: o stays).
template <int KB>
__device__ __forceinline__ float softmax_f32(float &m, float &l, f32x4 (&s)[KB], float scale2, bool full, const Column &co, int t,
                                             int len, float (&p)[KB][4]) {
    float mx = -INFINITY;
#pragma unroll
    for (int y = 0; y < KB; y++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            s[y][i] *= scale2;
            if (!full) s[y][i] = sees(co, t + 16 * y + i, len) ? s[y][i] : -INFINITY;
            mx = fmaxf(mx, s[y][i]);
        }
    mx = fmaxf(m, col_max(mx));
    const float ref = mx == -INFINITY ? 0.f : mx;
    float al = 1.f;
    if (__any(mx != m)) {
        al = m == -INFINITY ? 0.f : exp2_fast(m - ref);
        l *= al;
        m = mx;
    }
#pragma unroll
    for (int y = 0; y < KB; y++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            p[y][i] = exp2_fast(s[y][i] - ref);
            l += p[y][i];
        }
    return al;
}

// Adds the values of V that are not finite, of the keys that the column sees:
// o[e][f][r] is dimension 64 e + 16 j + 4 r + f.
template <int ET>
__device__ __forceinline__ void add_odd(f32x4 (&o)[ET][4], const float (&p)[4], const Column &co, const float *vt, int ldk, int hd, int t0,
                                        int left, int len) {
    const int lane = threadIdx.x & 63, cl = lane & 15, j = lane >> 4;
#pragma unroll 1
    for (int k = 0; k < 16; k += 4) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float pk = __shfl(p[i], 4 * k + cl);
            if (k + i >= left || !sees(co, t0 + k + i, len)) continue;
#pragma unroll
            for (int e = 0; e < ET; e++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int d = 64 * e + 16 * j + 4 * r;
                    if (d >= hd) continue;
                    const f32x4 v = *(const f32x4 *)(vt + (size_t)(k + i) * ldk + d);
#pragma unroll
                    for (int f = 0; f < 4; f++)
                        if (!isfinite(v[f])) o[e][f][r] += pk * v[f];
                }
        }
    }
}

// Few columns (one tile a workgroup): bound by reading the cache.
template <int ET>
__global__ __launch_bounds__(64 * WAVES, ET <= 3 ? 2 : 1) void k_tree_f32(TreeArgs a, F32Batch fb) {
    constexpr int CT = 4 * ET, COLS = 16;
    extern __shared__ __align__(16) float sm[];
    Unit u;
    if (!unit_of(a, u)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cl = lane & 15, j = lane >> 4;
    const int hd = a.hd, len = a.d.len[u.s], ldk = a.n_kv * hd, end = len + a.d.rows;
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    const int c = u.qg * COLS + cl;
    const Column co = column_of(a, u.s, c, a.d.tree ? ancestor_mask(a.d, u.s) : 0);
    f32x4 q[CT], o[ET][4];
    {
        const int cc = min(c, a.cols - 1);
        const float *qr = a.q + (((size_t)u.s * a.d.rows + cc / a.nrep) * a.n_q + u.g * a.nrep + cc % a.nrep) * hd;
#pragma unroll
        for (int x = 0; x < CT; x++) q[x] = 16 * x + 4 * j < hd ? *(const f32x4 *)(qr + 16 * x + 4 * j) : zero;
    }
#pragma unroll
    for (int e = 0; e < ET; e++)
#pragma unroll
        for (int f = 0; f < 4; f++) o[e][f] = zero;
    float m = -INFINITY, l = 0.f;
    const float *kb = fb.k[u.s] + (size_t)u.g * hd, *vb = fb.v[u.s] + (size_t)u.g * hd;
    int lo, hi;
    step_range<16>(a, u, COLS, &lo, &hi);

    f32x4 kk[CT];
    auto load_k = [&](int st) {
        const float *kt = kb + (size_t)st * 16 * ldk + (size_t)cl * ldk + 4 * j;
        const bool in = cl < end - st * 16;
#pragma unroll
        for (int x = 0; x < CT; x++) kk[x] = in && 16 * x + 4 * j < hd ? *(const f32x4 *)(kt + 16 * x) : zero;
    };
    if (lo + wave < hi) load_k(lo + wave);
    for (int st = lo + wave; st < hi; st += WAVES) {
        const int t0 = st * 16;
        const float *vt = vb + (size_t)t0 * ldk;
        const int left = end - t0;  // rows that there are, from t0 on
        f32x4 vv[4][ET];
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int e = 0; e < ET; e++)
                vv[i][e] = 4 * j + i < left && 64 * e + 4 * cl < hd ? *(const f32x4 *)(vt + (size_t)(4 * j + i) * ldk + 64 * e + 4 * cl) : zero;
        f32x4 s0 = zero, s1 = zero;
#pragma unroll
        for (int x = 0; x < CT; x++)
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                s0 = __builtin_amdgcn_mfma_f32_16x16x4f32(kk[x][e], q[x][e], s0, 0, 0, 0);
                s1 = __builtin_amdgcn_mfma_f32_16x16x4f32(kk[x][e + 1], q[x][e + 1], s1, 0, 0, 0);
            }
        load_k(min(st + WAVES, hi - 1));  // K is used up: under the products p.v
        const bool full = t0 + 16 <= len;
        // In drafted rows a value that is not finite may be seen by one column
        // and not by another: 0 * inf must not reach the latter.  Such values
        // leave the products here and are added one by one below.
        bool odd = false;
        if (!full) {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int e = 0; e < ET; e++)
#pragma unroll
                    for (int f = 0; f < 4; f++)
                        if (!isfinite(vv[i][e][f])) {
                            odd = true;
                            vv[i][e][f] = 0.f;
                        }
            odd = __any(odd);
        }
        float p[1][4];
        f32x4 sc[1] = {s0 + s1};
        const float al = softmax_f32<1>(m, l, sc, a.scale2, full, co, t0 + 4 * j, len, p);
        if (__any(al != 1.f)) {
#pragma unroll
            for (int e = 0; e < ET; e++)
#pragma unroll
                for (int f = 0; f < 4; f++) o[e][f] *= al;
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int e = 0; e < ET; e++)
#pragma unroll
                for (int f = 0; f < 4; f++) o[e][f] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv[i][e][f], p[0][i], o[e][f], 0, 0, 0);
        if (odd) add_odd<ET>(o, p[0], co, vt, ldk, hd, t0, left, len);
    }

    const int ld = hd + 4, col = wave * COLS + cl;
    float *s_o = sm, *s_c = sm + WAVES * COLS * ld, *s_l = s_c + WAVES * COLS;
    const float sum = col_sum(l);
    if (j == 0) {
        s_c[col] = m;
        s_l[col] = sum;
    }
#pragma unroll
    for (int e = 0; e < ET; e++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int d = 64 * e + 16 * j + 4 * r;
            if (d < hd) *(f32x4 *)(s_o + col * ld + d) = f32x4{o[e][0][r], o[e][1][r], o[e][2][r], o[e][3][r]};
        }
    join_waves<COLS>(a, u, s_o, s_c, s_l, ld);
}

// Many columns: bound by the f32 matrix rate.  W waves with a tile each share
// a step's keys through LDS, in operand order; the next step's part waits in
// registers.  A step is 16 keys, 32 where heads are short (at 128 dimensions 32
// keys a step left fewer waves: 26-node trees of four contexts 62 against 56 us).
// Those trees over 2047 rows, 32 heads over 8 of 128: 2.8 GFLOP in 47 us.
constexpr int tree_f32_blocks(int et) { return et == 1 ? 2 : 1; }
template <int ET, int W>
__global__ __launch_bounds__(64 * W, ET <= 2 ? 3 : ET == 4 && W == 2 ? 1 : 2) void k_tree_f32_wide(TreeArgs a, F32Batch fb) {
    constexpr int CT = 4 * ET, KB = tree_f32_blocks(ET), NB = (KB * CT + W - 1) / W;
    __shared__ f32x4 s_k[KB * CT][64], s_v[KB * CT][64];  // block y, x: [y CT + x]; V's x = i ET + e
    __shared__ int s_odd[W];
    Unit u;
    if (!unit_of(a, u)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cl = lane & 15, j = lane >> 4;
    const int hd = a.hd, len = a.d.len[u.s], ldk = a.n_kv * hd, rows_end = len + a.d.rows;
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    const int c0 = (u.qg * W + tile_of<W>(u, wave)) * 16, c = c0 + cl;
    const Column co = column_of(a, u.s, c, a.d.tree ? ancestor_mask(a.d, u.s) : 0);
    const int end = c0 >= a.cols ? 0 : a.d.tree ? rows_end : len + min(c0 + 15, a.cols - 1) / a.nrep + 1;
    f32x4 q[CT], o[ET][4];
    {
        const int cc = min(c, a.cols - 1);
        const float *qr = a.q + (((size_t)u.s * a.d.rows + cc / a.nrep) * a.n_q + u.g * a.nrep + cc % a.nrep) * hd;
#pragma unroll
        for (int x = 0; x < CT; x++) q[x] = 16 * x + 4 * j < hd ? *(const f32x4 *)(qr + 16 * x + 4 * j) : zero;
    }
#pragma unroll
    for (int e = 0; e < ET; e++)
#pragma unroll
        for (int f = 0; f < 4; f++) o[e][f] = zero;
    float m = -INFINITY, l = 0.f;
    const float *kb = fb.k[u.s] + (size_t)u.g * hd, *vb = fb.v[u.s] + (size_t)u.g * hd;
    int lo, hi;
    step_range<16 * KB>(a, u, 16 * W, &lo, &hi);

    // Steps whose rows are all there, of heads that fill their 64-dimension
    // blocks, take a lane's fixed offsets: the checks took 2% of the time.
    f32x4 kr[NB], vr[NB];
    int ko[NB], vo[NB];
#pragma unroll
    for (int b = 0; b < NB; b++) {
        const int at = min(W * b + wave, KB * CT - 1), y = at / CT, x = at % CT, i = x / ET, e = x % ET;
        ko[b] = (16 * y + cl) * ldk + 16 * x + 4 * j;
        vo[b] = (16 * y + 4 * j + i) * ldk + 64 * e + 4 * cl;
    }
    auto fetch = [&](int st) {
        const float *kt = kb + (size_t)st * 16 * KB * ldk, *vt = vb + (size_t)st * 16 * KB * ldk;
        const int left = rows_end - st * 16 * KB;
        if (left >= 16 * KB && hd == 64 * ET) {
#pragma unroll
            for (int b = 0; b < NB; b++) {
                kr[b] = *(const f32x4 *)(kt + ko[b]);
                vr[b] = *(const f32x4 *)(vt + vo[b]);
            }
            return;
        }
#pragma unroll
        for (int b = 0; b < NB; b++) {
            const int at = min(W * b + wave, KB * CT - 1), y = at / CT, x = at % CT, i = x / ET, e = x % ET;
            kr[b] = 16 * y + cl < left && 16 * x + 4 * j < hd ? *(const f32x4 *)(kt + ko[b]) : zero;
            vr[b] = 16 * y + 4 * j + i < left && 64 * e + 4 * cl < hd ? *(const f32x4 *)(vt + vo[b]) : zero;
        }
    };
    if (lo < hi) fetch(lo);
    for (int st = lo; st < hi; st++) {
        const int t0 = st * 16 * KB;
        const bool full = t0 + 16 * KB <= len;
        bool odd = false;
        if (!full) {  // values that are not finite leave the products, as in k_tree_f32
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int f = 0; f < 4; f++)
                    if (!isfinite(vr[b][f])) {
                        odd = true;
                        vr[b][f] = 0.f;
                    }
            odd = __any(odd);
        }
        __syncthreads();  // the step before has been read
#pragma unroll
        for (int b = 0; b < NB; b++)
            if (W * b + W <= KB * CT || W * b + wave < KB * CT) {
                s_k[W * b + wave][lane] = kr[b];
                s_v[W * b + wave][lane] = vr[b];
            }
        if (lane == 0) s_odd[wave] = odd;
        __syncthreads();
        fetch(min(st + 1, hi - 1));
        if (t0 >= end) continue;  // (uniform in the wave)
        f32x4 s0[KB], s1[KB];
#pragma unroll
        for (int y = 0; y < KB; y++) s0[y] = s1[y] = zero;
#pragma unroll
        for (int x = 0; x < CT; x++)
#pragma unroll
            for (int y = 0; y < KB; y++) {
                const f32x4 kk = s_k[y * CT + x][lane];
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    s0[y] = __builtin_amdgcn_mfma_f32_16x16x4f32(kk[e], q[x][e], s0[y], 0, 0, 0);
                    s1[y] = __builtin_amdgcn_mfma_f32_16x16x4f32(kk[e + 1], q[x][e + 1], s1[y], 0, 0, 0);
                }
            }
        float p[KB][4];
        f32x4 sc[KB];
#pragma unroll
        for (int y = 0; y < KB; y++) sc[y] = s0[y] + s1[y];
        const float al = softmax_f32<KB>(m, l, sc, a.scale2, full, co, t0 + 4 * j, len, p);
        if (__any(al != 1.f)) {
#pragma unroll
            for (int e = 0; e < ET; e++)
#pragma unroll
                for (int f = 0; f < 4; f++) o[e][f] *= al;
        }
#pragma unroll
        for (int y = 0; y < KB; y++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int e = 0; e < ET; e++) {
                    const f32x4 vv = s_v[y * CT + i * ET + e][lane];
#pragma unroll
                    for (int f = 0; f < 4; f++) o[e][f] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv[f], p[y][i], o[e][f], 0, 0, 0);
                }
        if (!full) {
            int any = 0;
#pragma unroll
            for (int w = 0; w < W; w++) any |= s_odd[w];
            if (any)
#pragma unroll
                for (int y = 0; y < KB; y++)
                    add_odd<ET>(o, p[y], co, vb + ((size_t)t0 + 16 * y) * ldk, ldk, hd, t0 + 16 * y, rows_end - t0 - 16 * y, len);
        }
    }

    float4 v[4 * ET];
#pragma unroll
    for (int e = 0; e < ET; e++)
#pragma unroll
        for (int r = 0; r < 4; r++) v[4 * e + r] = make_float4(o[e][0][r], o[e][1][r], o[e][2][r], o[e][3][r]);
    finish_wide(a, u, c, m, col_sum(l), v, [&](int x) { return 64 * (x / 4) + 16 * j + 4 * (x % 4); });
}

// Key splits: about `want` workgroups in all, each of `least` steps or more,
// the sequences' splits of like sizes.
void pick_splits(TreeArgs &a, int step_keys, int want, int least) {
    long long steps[PF_MAX_SEQS], all = 0;
    for (int s = 0; s < a.d.n_seq; s++) all += steps[s] = ((long long)a.d.len[s] + a.d.rows + step_keys - 1) / step_keys;
    long long size = (all * a.n_kv * a.n_qg + want - 1) / want;
    if (size < least) size = least;
    if (a.cols > 1 << 20) size = all;  // (many columns fill the chip: their splits' sums would be large)
    a.n_split = 1;
    for (int s = 0; s < a.d.n_seq; s++) {
        long long n = (steps[s] + size / 2) / size;
        n = n < 1 ? 1 : n > MAX_SPLIT ? MAX_SPLIT : n;
        a.splits[s] = (int)n;
        if (a.n_split < n) a.n_split = (int)n;
    }
}

// waves: of a workgroup; cols: its columns
template <class K, class B>
int launch_tree(K kernel, TreeArgs a, const B &b, int waves, int cols, size_t lds, int step_keys, int want, int least, int fused, hipStream_t s) {
    a.n_qg = (a.cols + cols - 1) / cols;
    a.near = (127 + a.n_qg) / a.n_qg;  // (an XCD runs about 128 workgroups at once)
    pick_splits(a, step_keys, want, least);
    const size_t n_col = (size_t)a.d.n_seq * a.n_kv * a.cols;
    void *ws = nullptr;
    SCRY_TRY(split_workspace(n_col * (a.hd + 2) * sizeof(float), &a.n_split, &ws));
    a.part_o = (float *)ws;
    a.part_ml = a.part_o + n_col * a.n_split * a.hd;
    for (int i = 0; i < a.d.n_seq; i++) {
        if (a.n_split == 1) a.splits[i] = 1;  // one is enough, or no memory for more
        a.pair0[i + 1] = a.pair0[i] + a.n_kv * a.splits[i];
    }
    const size_t grid = (size_t)((a.pair0[a.d.n_seq] + 7) / 8) * 8 * a.n_qg;
    if (grid > DRAFT_MAX_GRID) return set_error(SCRY_ERR_UNSUPPORTED, "attention: %zu workgroups", grid);
    // Few splits of few columns: the last to arrive joins them, without a second
    // launch (one token of 4 query heads a KV head over 2000 int8 rows: 14.8 ->
    // 12.7 us).  From 2 MB of partial sums on, a launch of its own has more
    // workgroups for them (16 rows of 32 heads of 128: over 4000 int8 rows, 2 MB,
    // 18.5 us joined by the last and 19.0 by a launch, over 6000, 3 MB, 24.7 and
    // 22.0), and so for the wide kernels' columns.
    a.arrived = nullptr;
    if (a.n_split > 1 && a.n_split <= fused && n_col * a.n_split * a.hd <= (size_t)1 << 19 &&
        (size_t)a.d.n_seq * a.n_kv * a.n_qg <= DRAFT_COUNTERS)
        SCRY_TRY(draft_counters(&a.arrived));
    if (lds > 65536)
        SCRY_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(64 * waves), lds, s, a, b);
    SCRY_HIP(hipGetLastError());
    // a thread per four dimensions where they fill the chip, else the groups of
    // k_tree_merge (16384 columns of 128 by 3 splits: 8 against 13 us; 32 columns
    // by 64 splits: 19 against 4 us)
    const size_t n = n_col * (a.hd / 4);
    if (a.n_split == 1 || a.arrived) return SCRY_OK;
    if (n >= (size_t)1 << 15) {
        hipLaunchKernelGGL(k_tree_merge_flat, dim3((a.cols * (a.hd / 4) + 255) / 256, a.n_kv, a.d.n_seq), dim3(256), 0, s, a);
        SCRY_HIP(hipGetLastError());
    } else {
        int lanes = 1;
        while (4 * lanes < a.hd) lanes *= 2;
        // threads of a column: its lanes, times up to as many groups as it has splits
        int per = 256 / lanes;
        while (per > 1 && 256 / (per * lanes) * 2 <= a.n_split) per /= 2;
        if (per > 16) per = 16;
        hipLaunchKernelGGL(k_tree_merge, dim3((a.cols + per - 1) / per, a.n_kv, a.d.n_seq), dim3(256), 0, s, a, per, lanes);
        SCRY_HIP(hipGetLastError());
    }
    return SCRY_OK;
}

// Workgroups that a launch aims at: three of four waves a CU (what the wide
// int8 kernel's registers allow at 128 dimensions: 64-node trees of eight
// 4000-row contexts 84 us at two, 75 at three, 76 at four, of which some wait;
// a 512-row chunk over 1500 rows of 32 heads 50, 50 and 56).  The f32 kernels:
// 26-node trees of four 2047-row contexts 51 us at two, 50 at three, 52 at four.
constexpr int WANT = 768;
constexpr int FUSED = 16;  // key splits that the last of a narrow kernel's workgroups joins

// Columns in tiles of 16: three or four tiles share the keys (W waves).  One tile,
// over int8 caches two, have the narrow kernel (8-node trees of 32 columns over
// 2000 rows of four sequences: int8 19.4 us wide, 17.3 narrow, f32 32.6 and 40.0).
template <int KS>
int launch_i8(const TreeArgs &a, const Kv8Batch &b, hipStream_t s) {
    const int tiles = (a.cols + 15) / 16, groups = (tiles + 3) / 4, w = (tiles + groups - 1) / groups;
    const size_t lds = (size_t)WAVES * 16 * (a.hd + 4 + 2) * sizeof(float);
    if (tiles <= 2) return launch_tree(k_tree_i8<KS>, a, b, WAVES, 16, lds, 64, WANT, 8, FUSED, s);
    if (w == 3) return launch_tree(k_tree_i8_wide<KS, 3>, a, b, 3, 48, 0, 64, 4 * WANT / 3, 4, 0, s);
    return launch_tree(k_tree_i8_wide<KS, 4>, a, b, 4, 64, 0, 64, WANT, 4, 0, s);
}
template <int ET>
int launch_f32(const TreeArgs &a, const F32Batch &b, hipStream_t s) {
    const int tiles = (a.cols + 15) / 16, groups = (tiles + 3) / 4, w = (tiles + groups - 1) / groups;
    const size_t lds = (size_t)WAVES * 16 * (a.hd + 4 + 2) * sizeof(float);
    if (w == 1) return launch_tree(k_tree_f32<ET>, a, b, WAVES, 16, lds, 16, WANT, 8, FUSED, s);
    if (w == 2) return launch_tree(k_tree_f32_wide<ET, 2>, a, b, 2, 32, 0, 16 * tree_f32_blocks(ET), 2 * WANT, 4, 0, s);
    if (w == 3) return launch_tree(k_tree_f32_wide<ET, 3>, a, b, 3, 48, 0, 16 * tree_f32_blocks(ET), 4 * WANT / 3, 4, 0, s);
    return launch_tree(k_tree_f32_wide<ET, 4>, a, b, 4, 64, 0, 16 * tree_f32_blocks(ET), WANT, 4, 0, s);
}

int tree_run(const char *what, scry_buf q, const TreeArgs &t, bool i8, const F32Batch &f, const Kv8Batch &c, scry_buf *out) {
    const size_t n = (size_t)t.d.n_seq * t.d.rows;
    if (q->n != n * t.n_q * t.hd) return set_error(SCRY_ERR_INVALID, "%s: shape mismatch", what);
    TreeArgs a = t;
    a.nrep = a.n_q / a.n_kv;
    if ((size_t)a.d.rows * a.nrep > (size_t)1 << 30) return set_error(SCRY_ERR_UNSUPPORTED, "%s: %d rows", what, a.d.rows);
    a.cols = a.d.rows * a.nrep;
    DeviceScope dev;
    scry_buf o = nullptr;
    SCRY_TRY(buf_new(q->n, &o));
    a.q = q->d;
    a.out = o->d;
    hipStream_t s = ctx().stream;
    const int blocks = (a.hd + 63) / 64;
    const int rc = i8 ? blocks == 1   ? launch_i8<1>(a, c, s)
                        : blocks == 2 ? launch_i8<2>(a, c, s)
                        : blocks == 3 ? launch_i8<3>(a, c, s)
                                      : launch_i8<4>(a, c, s)
                   : blocks == 1 ? launch_f32<1>(a, f, s)
                   : blocks == 2 ? launch_f32<2>(a, f, s)
                   : blocks == 3 ? launch_f32<3>(a, f, s)
                                 : launch_f32<4>(a, f, s);
    if (rc) {
        buf_del(o);
        return rc;
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
                            int rows, const int64_t *parents, int n_q, int n_kv, int head_dim, float scale, scry_buf *out) {
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
    t.scale2 = scale * 1.4426950408889634f;
    return tree_run(what, q, t, false, f, Kv8Batch{}, out);
}

int scry_hip_kv8_tree_attention(scry_buf q, const scry_kv8 *caches, int n_seq, const int32_t *len, int rows,
                                const int64_t *parents, int n_q, float scale, scry_buf *out) {
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
    t.scale2 = scale * 1.4426950408889634f;
    return tree_run(what, q, t, true, F32Batch{}, c, out);
}

}  // extern "C"
