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
// A wave takes QT tiles and every fourth step of keys; the four waves of a
// workgroup are joined through LDS, and where the keys are split over
// workgroups too, by k_tree_merge.
//
// Workgroups go to the XCDs round-robin: those of one (sequence, KV head,
// split) share their keys and sit on one XCD, so the keys come from its L2
// after the first.
#include <cmath>

#include "kdev.h"
#include "kv8.h"

namespace scry {
namespace {

using namespace dev;

typedef int i32x4 __attribute__((ext_vector_type(4)));
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
    int n_split, n_qg, n_pair;      // key splits, groups of QT tiles, (sequence, KV head, split)s
    float scale2;                   // scale * log2(e)
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
__device__ __forceinline__ bool unit_of(const TreeArgs &a, Unit &u) {
    const int i = blockIdx.x, pair = (i & 7) + 8 * ((i >> 3) / a.n_qg);
    u.qg = (i >> 3) % a.n_qg;
    if (pair >= a.n_pair) return false;  // padding of the last eight
    u.split = pair % a.n_split;
    const int sg = pair / a.n_split;
    u.g = sg % a.n_kv;
    u.s = sg / a.n_kv;
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

// Largest value over the four lanes of a column; their sum.
__device__ __forceinline__ float col_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float col_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

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
        const int node = c / a.nrep, h = u.g * a.nrep + c % a.nrep;
        if (a.n_split == 1) {
            float4 r = make_float4(o.x / L, o.y / L, o.z / L, o.w / L);
            if (a.d.tree && a.d.parent[u.s][node] == -2) r = make_float4(0.f, 0.f, 0.f, 0.f);
            *(float4 *)(a.out + (((size_t)u.s * a.d.rows + node) * a.n_q + h) * hd + d) = r;
        } else {
            const size_t at = (((size_t)u.s * a.n_kv + u.g) * a.cols + c) * a.n_split + u.split;
            *(float4 *)(a.part_o + at * hd + d) = o;
            if (d == 0) *(float2 *)(a.part_ml + at * 2) = make_float2(C, L);
        }
    }
}

// The splits of a column joined in split order: a wave per column, a lane per
// four dimensions (and per split, for the factors).
__global__ __launch_bounds__(256) void k_tree_merge(TreeArgs a, size_t n_col) {
    const size_t col = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (col >= n_col) return;
    const int c = (int)(col % a.cols), g = (int)(col / a.cols % a.n_kv), s = (int)(col / a.cols / a.n_kv);
    const int node = c / a.nrep, h = g * a.nrep + c % a.nrep, hd = a.hd;
    const float *ml = a.part_ml + col * a.n_split * 2;
    float cc = -INFINITY, l = 0.f;
    if (lane < a.n_split) {
        cc = ml[2 * lane];
        l = ml[2 * lane + 1];
    }
    float C = cc;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) C = fmaxf(C, __shfl_xor(C, off));
    const float f = exp2_fast(cc - (C == -INFINITY ? 0.f : C));
    const float L = wave_sum(l * f);
    const bool act = 4 * lane < hd;
    const float *o = a.part_o + col * a.n_split * hd + 4 * lane;
    float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int p = 0; p < a.n_split; p++) {
        const float fp = __shfl(f, p);
        const float4 v = act ? *(const float4 *)(o + (size_t)p * hd) : r;
        r.x += v.x * fp;
        r.y += v.y * fp;
        r.z += v.z * fp;
        r.w += v.w * fp;
    }
    if (!act) return;
    r = make_float4(r.x / L, r.y / L, r.z / L, r.w / L);
    if (a.d.tree && a.d.parent[s][node] == -2) r = make_float4(0.f, 0.f, 0.f, 0.f);
    *(float4 *)(a.out + (((size_t)s * a.d.rows + node) * a.n_q + h) * hd + 4 * lane) = r;
}

// The steps of SK keys that a workgroup takes of the keys that its columns see.
template <int SK, int COLS>
__device__ __forceinline__ void step_range(const TreeArgs &a, const Unit &u, int *lo, int *hi) {
    int rows = a.d.rows;
    if (!a.d.tree) rows = min(rows, (min(a.cols, (u.qg + 1) * COLS) - 1) / a.nrep + 1);
    const long long steps = ((long long)a.d.len[u.s] + rows + SK - 1) / SK;
    *lo = (int)(steps * u.split / a.n_split);
    *hi = (int)(steps * (u.split + 1) / a.n_split);
}

// ------------------------------------------------------------ int8 cache
// q.k: K's bytes are an operand as they lie; q is held as 24-bit integers of
// its row's largest value in three balanced int8 digits, so the products and
// their sums over hd are exact integers.
// p.v: V's bytes become f16 (exact), and w = p * (the row's scale) is split
// into two f16 terms, 22 bits.  c = max s + log2(the largest scale seen) - 14:
// the largest w is 2^14, and f16's smallest steps lie 2^-38 below.  Scales
// below 2^-80 count as 2^-80 there, which keeps 2^-c in f32's range.
// KS: steps of 64 dimensions (hdp <= 64 KS).
template <int KS, int QT>
__global__ __launch_bounds__(64 * WAVES, KS <= 3 ? 2 : 1) void k_tree_i8(TreeArgs a, Kv8Batch cb) {
    constexpr int DT = 4 * KS, COLS = 16 * QT;
    extern __shared__ __align__(16) float sm[];
    Unit u;
    if (!unit_of(a, u)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cl = lane & 15, j = lane >> 4;
    const int hd = a.hd, hdp = cb.hdp, len = a.d.len[u.s];

    // the columns' queries as digits: lane (cl, j) holds dimensions 64 x + 16 j ..
    const unsigned long long anc = a.d.tree ? ancestor_mask(a.d, u.s) : 0;
    Column co[QT];
    i32x4 qd[QT][3][KS];
    float qs[QT];
#pragma unroll
    for (int t = 0; t < QT; t++) {
        const int c = u.qg * COLS + 16 * t + cl;
        co[t] = column_of(a, u.s, c, anc);
        const int node = min(c, a.cols - 1) / a.nrep, rep = min(c, a.cols - 1) % a.nrep;
        const float *q = a.q + (((size_t)u.s * a.d.rows + node) * a.n_q + u.g * a.nrep + rep) * hd;
        float4 x[KS][4];
        float m = 0.f;
        bool fin = true;
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int d = 64 * k + 16 * j + 4 * e;
                x[k][e] = d < hd ? *(const float4 *)(q + d) : make_float4(0.f, 0.f, 0.f, 0.f);
                const float4 v = x[k][e];
                m = fmaxf(m, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
                fin &= isfinite(v.x) && isfinite(v.y) && isfinite(v.z) && isfinite(v.w);
            }
        // a query with an infinity or NaN has no finite softmax over any key
        m = col_max(fin ? fmaxf(m, 0x1p-96f) : INFINITY);
        const float up = m < INFINITY ? 8290000.f / m : 0.f;  // 126.5 * 2^16: the top digit stays below 128
        qs[t] = m < INFINITY ? m / 8290000.f * a.scale2 : __builtin_nanf("");
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float v[4] = {x[k][e].x, x[k][e].y, x[k][e].z, x[k][e].w};
                unsigned w[3] = {0, 0, 0};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int X = up > 0.f ? (int)rintf(v[i] * up) : 0;
                    const int d0 = (int)(signed char)X, X1 = (X - d0) >> 8, d1 = (int)(signed char)X1, d2 = (X1 - d1) >> 8;
                    w[0] |= (unsigned)(d0 & 255) << (8 * i);
                    w[1] |= (unsigned)(d1 & 255) << (8 * i);
                    w[2] |= (unsigned)(d2 & 255) << (8 * i);
                }
#pragma unroll
                for (int g = 0; g < 3; g++) qd[t][g][k][e] = (int)w[g];
            }
    }

    float m[QT], ve[QT], l[QT];  // largest score, exponent of the largest scale - 14, sum
    f32x4 o[QT][DT];
#pragma unroll
    for (int t = 0; t < QT; t++) {
        m[t] = -INFINITY;
        ve[t] = -94.f;
        l[t] = 0.f;
#pragma unroll
        for (int d = 0; d < DT; d++) o[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const int rows_p = cb.rows_p[u.s];
    const int8_t *kb = cb.k[u.s] + (size_t)u.g * rows_p * hdp, *vb = cb.v[u.s] + (size_t)u.g * rows_p * hdp;
    const float *ksb = cb.ks[u.s] + (size_t)u.g * rows_p, *vsb = cb.vs[u.s] + (size_t)u.g * rows_p;
    int lo, hi;
    step_range<64, COLS>(a, u, &lo, &hi);

    i32x4 kk[4][KS];
    float4 ks[4];
    auto load_k = [&](int st) {
        const int8_t *kt = kb + (size_t)st * 64 * hdp;
#pragma unroll
        for (int x = 0; x < 4; x++) {
#pragma unroll
            for (int k = 0; k < KS; k++)
                kk[x][k] = 64 * k + 16 * j < hdp ? *(const i32x4 *)(kt + (16 * x + cl) * hdp + 64 * k + 16 * j) : i32x4{0, 0, 0, 0};
            ks[x] = *(const float4 *)(ksb + st * 64 + 16 * x + 4 * j);
        }
    };
    if (lo + wave < hi) load_k(lo + wave);
    for (int st = lo + wave; st < hi; st += WAVES) {
        const int t0 = st * 64;
        const int8_t *vt = vb + (size_t)t0 * hdp;
        float4 vs[4];
#pragma unroll
        for (int x = 0; x < 4; x++) vs[x] = *(const float4 *)(vsb + t0 + 16 * x + 4 * j);
        i32x4 vv[DT];

        const bool full = t0 + 64 <= len;  // every column sees every key
        float vmax = 0.f;
        if (full) {
#pragma unroll
            for (int x = 0; x < 4; x++) vmax = fmaxf(vmax, fmaxf(fmaxf(vs[x].x, vs[x].y), fmaxf(vs[x].z, vs[x].w)));
            vmax = col_max(vmax);
        }
        f16x8 wh[QT][2], wl[QT][2];
#pragma unroll
        for (int t = 0; t < QT; t++) {
            float sc[4][4];
            float mx = -INFINITY;
#pragma unroll
            for (int x = 0; x < 4; x++) {
                i32x4 h = {0, 0, 0, 0}, b = {0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < KS; k++) h = __builtin_amdgcn_mfma_i32_16x16x64_i8(kk[x][k], qd[t][2][k], h, 0, 0, 0);
                // (|h| <= 2^22: hd products of two digits)
                h = h << 8;
#pragma unroll
                for (int k = 0; k < KS; k++) h = __builtin_amdgcn_mfma_i32_16x16x64_i8(kk[x][k], qd[t][1][k], h, 0, 0, 0);
#pragma unroll
                for (int k = 0; k < KS; k++) b = __builtin_amdgcn_mfma_i32_16x16x64_i8(kk[x][k], qd[t][0][k], b, 0, 0, 0);
                const float kx[4] = {ks[x].x, ks[x].y, ks[x].z, ks[x].w};
#pragma unroll
                for (int i = 0; i < 4; i++) sc[x][i] = fmaf((float)h[i], 256.f, (float)b[i]) * (qs[t] * kx[i]);
            }
            if (t == QT - 1) {  // K is used up: its registers take V
#pragma unroll
                for (int d = 0; d < DT; d++)
                    vv[d] = 16 * d < hdp ? *(const i32x4 *)(vt + (16 * d + cl) * 64 + 16 * j) : i32x4{0, 0, 0, 0};
            }
            float vm = vmax;
            unsigned seen = 0xffffu;
            if (!full) {
                seen = 0;
                vm = 0.f;
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const float vx[4] = {vs[x].x, vs[x].y, vs[x].z, vs[x].w};
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const bool in = sees(co[t], t0 + 16 * x + 4 * j + i, len);
                        seen |= (unsigned)in << (4 * x + i);
                        sc[x][i] = in ? sc[x][i] : -INFINITY;
                        vm = fmaxf(vm, in ? vx[i] : 0.f);
                    }
                }
                vm = col_max(vm);
            }
#pragma unroll
            for (int x = 0; x < 4; x++) mx = fmaxf(mx, fmaxf(fmaxf(sc[x][0], sc[x][1]), fmaxf(sc[x][2], sc[x][3])));
            mx = fmaxf(m[t], col_max(mx));
            // 2^e >= the largest scale, e >= -80
            const float e = fmaxf(ve[t], (float)((int)((__float_as_uint(fmaxf(vm, 0x1p-80f)) + 0x7fffffu) >> 23) - 127 - 14));
            const float ref = mx == -INFINITY ? 0.f : mx + e;
            if (__any(mx != m[t] || e != ve[t])) {
                const float al = m[t] == -INFINITY ? 0.f : exp2_fast(m[t] + ve[t] - ref);
                l[t] *= al;
#pragma unroll
                for (int d = 0; d < DT; d++) o[t][d] *= al;
                m[t] = mx;
                ve[t] = e;
            }
            float sum = 0.f;
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const float vx[4] = {vs[x].x, vs[x].y, vs[x].z, vs[x].w};
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float p = exp2_fast(sc[x][i] - ref);
                    sum += p;
                    w[i] = p * vx[i];
                    if (!full && !(seen >> (4 * x + i) & 1)) w[i] = 0.f;  // the scale may be NaN
                }
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const f16x2 h = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(w[i], w[i + 1]));
                    const f16x2 r = __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_pkrtz(w[i] - (float)h[0], w[i + 1] - (float)h[1]));
                    wh[t][x / 2][4 * (x % 2) + i] = h[0];
                    wh[t][x / 2][4 * (x % 2) + i + 1] = h[1];
                    wl[t][x / 2][4 * (x % 2) + i] = r[0];
                    wl[t][x / 2][4 * (x % 2) + i + 1] = r[1];
                }
            }
            l[t] += sum;
        }
        load_k(min(st + WAVES, hi - 1));  // under the products below
#pragma unroll
        for (int d = 0; d < DT; d++) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
                // byte b = v + 128 behind 0x64 is f16 1024 + b
                i32x4 hv;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const unsigned by = (unsigned)vv[d][2 * x + i / 2];
                    const f16x2 r = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, by, i % 2 ? 0x04030402u : 0x04010400u)) -
                                    f16x2{(_Float16)1152.f, (_Float16)1152.f};
                    hv[i] = __builtin_bit_cast(int, r);
                }
                const f16x8 va = __builtin_bit_cast(f16x8, hv);
#pragma unroll
                for (int t = 0; t < QT; t++) {
                    o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, wh[t][x], o[t][d], 0, 0, 0);
                    o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, wl[t][x], o[t][d], 0, 0, 0);
                }
            }
        }
    }

    const int ld = hd + 4;
    float *s_o = sm, *s_c = sm + WAVES * COLS * ld, *s_l = s_c + WAVES * COLS;
#pragma unroll
    for (int t = 0; t < QT; t++) {
        const int col = wave * COLS + 16 * t + cl;
        const float sum = col_sum(l[t]);
        if (j == 0) {
            s_c[col] = m[t] == -INFINITY ? m[t] : m[t] + ve[t];
            s_l[col] = sum;
        }
#pragma unroll
        for (int d = 0; d < DT; d++)
            if (16 * d + 4 * j < hd) *(f32x4 *)(s_o + col * ld + 16 * d + 4 * j) = o[t][d];
    }
    join_waves<COLS>(a, u, s_o, s_c, s_l, ld);
}

// ------------------------------------------------------------- f32 cache
// Products on the f32 matrix instructions (16 x 16 x 4): f32 sums of f32
// products.  Which four dimensions, or keys, an instruction takes is free as
// long as both operands agree: lane (cl, j) loads K rows as float4 of
// dimensions 16 c + 4 j .. (element e is instruction (c, e)'s operand), and V
// rows 4 j + i as float4 of dimensions 64 e + 4 cl .., so every load is 16
// bytes wide and a row's lanes are neighbours.
// ET: blocks of 64 dimensions.
template <int ET, int QT>
__global__ __launch_bounds__(64 * WAVES, ET <= 3 ? 2 : 1) void k_tree_f32(TreeArgs a, F32Batch fb) {
    constexpr int CT = 4 * ET, COLS = 16 * QT;
    extern __shared__ __align__(16) float sm[];
    Unit u;
    if (!unit_of(a, u)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cl = lane & 15, j = lane >> 4;
    const int hd = a.hd, len = a.d.len[u.s], ldk = a.n_kv * hd, end = len + a.d.rows;

    const unsigned long long anc = a.d.tree ? ancestor_mask(a.d, u.s) : 0;
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    Column co[QT];
    f32x4 q[QT][CT], o[QT][ET][4];
    float m[QT], l[QT];
#pragma unroll
    for (int t = 0; t < QT; t++) {
        const int c = u.qg * COLS + 16 * t + cl;
        co[t] = column_of(a, u.s, c, anc);
        const int node = min(c, a.cols - 1) / a.nrep, rep = min(c, a.cols - 1) % a.nrep;
        const float *qr = a.q + (((size_t)u.s * a.d.rows + node) * a.n_q + u.g * a.nrep + rep) * hd;
#pragma unroll
        for (int x = 0; x < CT; x++) q[t][x] = 16 * x + 4 * j < hd ? *(const f32x4 *)(qr + 16 * x + 4 * j) : zero;
#pragma unroll
        for (int e = 0; e < ET; e++)
#pragma unroll
            for (int f = 0; f < 4; f++) o[t][e][f] = zero;
        m[t] = -INFINITY;
        l[t] = 0.f;
    }
    const float *kb = fb.k[u.s] + (size_t)u.g * hd, *vb = fb.v[u.s] + (size_t)u.g * hd;
    int lo, hi;
    step_range<16, COLS>(a, u, &lo, &hi);

    for (int st = lo + wave; st < hi; st += WAVES) {
        const int t0 = st * 16;
        const float *kt = kb + (size_t)t0 * ldk, *vt = vb + (size_t)t0 * ldk;
        const int left = end - t0;  // rows that there are, from t0 on
        f32x4 kk[CT], vv[4][ET];
#pragma unroll
        for (int x = 0; x < CT; x++) kk[x] = cl < left && 16 * x + 4 * j < hd ? *(const f32x4 *)(kt + (size_t)cl * ldk + 16 * x + 4 * j) : zero;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int e = 0; e < ET; e++)
                vv[i][e] = 4 * j + i < left && 64 * e + 4 * cl < hd ? *(const f32x4 *)(vt + (size_t)(4 * j + i) * ldk + 64 * e + 4 * cl) : zero;

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
#pragma unroll
        for (int t = 0; t < QT; t++) {
            f32x4 s0 = zero, s1 = zero;
#pragma unroll
            for (int x = 0; x < CT; x++) {
                if (16 * x < hd)
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    s0 = __builtin_amdgcn_mfma_f32_16x16x4f32(kk[x][e], q[t][x][e], s0, 0, 0, 0);
                    s1 = __builtin_amdgcn_mfma_f32_16x16x4f32(kk[x][e + 1], q[t][x][e + 1], s1, 0, 0, 0);
                }
            }
            float sc[4];
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                sc[i] = (s0[i] + s1[i]) * a.scale2;
                if (!full) sc[i] = sees(co[t], t0 + 4 * j + i, len) ? sc[i] : -INFINITY;
                mx = fmaxf(mx, sc[i]);
            }
            mx = fmaxf(m[t], col_max(mx));
            const float ref = mx == -INFINITY ? 0.f : mx;
            if (__any(mx != m[t])) {
                const float al = m[t] == -INFINITY ? 0.f : exp2_fast(m[t] - ref);
                l[t] *= al;
#pragma unroll
                for (int e = 0; e < ET; e++)
#pragma unroll
                    for (int f = 0; f < 4; f++) o[t][e][f] *= al;
                m[t] = mx;
            }
            float p[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                p[i] = exp2_fast(sc[i] - ref);
                l[t] += p[i];
            }
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int e = 0; e < ET; e++)
#pragma unroll
                    for (int f = 0; f < 4; f++)
                        o[t][e][f] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv[i][e][f], p[i], o[t][e][f], 0, 0, 0);
            if (odd) {
                // o[e][f][r] is dimension 64 e + 16 j + 4 r + f of column cl
#pragma unroll 1
                for (int k = 0; k < 16; k += 4) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float pk = __shfl(p[i], 4 * k + cl);
                        if (k + i >= left || !sees(co[t], t0 + k + i, len)) continue;
#pragma unroll
                        for (int e = 0; e < ET; e++)
#pragma unroll
                            for (int r = 0; r < 4; r++) {
                                const int d = 64 * e + 16 * j + 4 * r;
                                const f32x4 v = d < hd ? *(const f32x4 *)(vt + (size_t)(k + i) * ldk + d) : zero;
#pragma unroll
                                for (int f = 0; f < 4; f++)
                                    if (!isfinite(v[f])) o[t][e][f][r] += pk * v[f];
                            }
                    }
                }
            }
        }
    }

    const int ld = hd + 4;
    float *s_o = sm, *s_c = sm + WAVES * COLS * ld, *s_l = s_c + WAVES * COLS;
#pragma unroll
    for (int t = 0; t < QT; t++) {
        const int col = wave * COLS + 16 * t + cl;
        const float sum = col_sum(l[t]);
        if (j == 0) {
            s_c[col] = m[t];
            s_l[col] = sum;
        }
#pragma unroll
        for (int e = 0; e < ET; e++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int d = 64 * e + 16 * j + 4 * r;
                if (d < hd) *(f32x4 *)(s_o + col * ld + d) = f32x4{o[t][e][0][r], o[t][e][1][r], o[t][e][2][r], o[t][e][3][r]};
            }
    }
    join_waves<COLS>(a, u, s_o, s_c, s_l, ld);
}

constexpr int MAX_SPLIT = 64;  // k_tree_merge has a lane per split

// Key splits: enough workgroups to fill the chip, each wave with a few steps.
int pick_splits(const TreeArgs &a, int step_keys) {
    int len = 0;
    for (int s = 0; s < a.d.n_seq; s++) len = len > a.d.len[s] ? len : a.d.len[s];
    const long long steps = ((long long)len + a.d.rows + step_keys - 1) / step_keys;
    const long long units = (long long)a.d.n_seq * a.n_kv * a.n_qg;
    long long n = (768 + units - 1) / units;
    const long long most = steps / (2 * WAVES);
    if (n > most) n = most;
    if (n > MAX_SPLIT) n = MAX_SPLIT;
    return n < 1 ? 1 : (int)n;
}

template <class K, class B>
int launch_tree(K kernel, TreeArgs a, const B &b, int qt, int step_keys, hipStream_t s) {
    const int cols = 16 * qt;
    a.n_qg = (a.cols + cols - 1) / cols;
    a.n_split = pick_splits(a, step_keys);
    const size_t n_col = (size_t)a.d.n_seq * a.n_kv * a.cols;
    void *ws = nullptr;
    SCRY_TRY(split_workspace(n_col * (a.hd + 2) * sizeof(float), &a.n_split, &ws));
    a.part_o = (float *)ws;
    a.part_ml = a.part_o + n_col * a.n_split * a.hd;
    a.n_pair = a.d.n_seq * a.n_kv * a.n_split;
    const size_t grid = (size_t)((a.n_pair + 7) / 8) * 8 * a.n_qg;
    if (grid > 0x7fffffff) return set_error(SCRY_ERR_UNSUPPORTED, "attention: %zu workgroups", grid);
    const size_t lds = (size_t)WAVES * cols * (a.hd + 4 + 2) * sizeof(float);
    SCRY_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(64 * WAVES), lds, s, a, b);
    SCRY_HIP(hipGetLastError());
    if (a.n_split > 1) {
        hipLaunchKernelGGL(k_tree_merge, dim3((unsigned)((n_col + 3) / 4)), dim3(256), 0, s, a, n_col);
        SCRY_HIP(hipGetLastError());
    }
    return SCRY_OK;
}

int tree_run(const char *what, scry_buf q, const TreeArgs &t, bool i8, const F32Batch &f, const Kv8Batch &c, scry_buf *out) {
    const size_t n = (size_t)t.d.n_seq * t.d.rows;
    if (q->n != n * t.n_q * t.hd) return set_error(SCRY_ERR_INVALID, "%s: shape mismatch", what);
    TreeArgs a = t;
    a.nrep = a.n_q / a.n_kv;
    if ((size_t)a.d.rows * a.nrep > 0x7fffff00) return set_error(SCRY_ERR_UNSUPPORTED, "%s: %d rows", what, a.d.rows);
    a.cols = a.d.rows * a.nrep;
    DeviceScope dev;
    scry_buf o = nullptr;
    SCRY_TRY(buf_new(q->n, &o));
    a.q = q->d;
    a.out = o->d;
    hipStream_t s = ctx().stream;
    const int blocks = (a.hd + 63) / 64;
    const bool two = a.cols > 16;  // two tiles a wave where there are two
    int rc;
    if (i8)
        rc = blocks == 1   ? two ? launch_tree(k_tree_i8<1, 2>, a, c, 2, 64, s) : launch_tree(k_tree_i8<1, 1>, a, c, 1, 64, s)
             : blocks == 2 ? two ? launch_tree(k_tree_i8<2, 2>, a, c, 2, 64, s) : launch_tree(k_tree_i8<2, 1>, a, c, 1, 64, s)
             : blocks == 3 ? launch_tree(k_tree_i8<3, 1>, a, c, 1, 64, s)
                           : launch_tree(k_tree_i8<4, 1>, a, c, 1, 64, s);
    else
        rc = blocks == 1   ? two ? launch_tree(k_tree_f32<1, 2>, a, f, 2, 16, s) : launch_tree(k_tree_f32<1, 1>, a, f, 1, 16, s)
             : blocks == 2 ? two ? launch_tree(k_tree_f32<2, 2>, a, f, 2, 16, s) : launch_tree(k_tree_f32<2, 1>, a, f, 1, 16, s)
             : blocks == 3 ? launch_tree(k_tree_f32<3, 1>, a, f, 1, 16, s)
                           : launch_tree(k_tree_f32<4, 1>, a, f, 1, 16, s);
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
    t.scale2 = scale * 1.4426950408889634f;
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
    t.scale2 = scale * 1.4426950408889634f;
    return tree_run(what, q, t, true, F32Batch{}, c, out);
}

}  // extern "C"
