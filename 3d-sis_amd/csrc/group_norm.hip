// Group norm with an activation on channels-last rows, forward and backward.
//
// Sample s has n_s rows (voxels) of C channels in G groups of c = C / G; m = n_s c.  Per (sample, group)
//     mu = 1/m sum x,  var = 1/m sum (x - mu)^2,  r = (var + eps)^-1/2,  h = (x - mu) r,  z = h w + b,  y = act(z)
// and backward, with d = dy act'(z):
//     db = sum d,  dw = sum d h  (over samples and rows),  dx = r (w d - (sum_group w d + h sum_group w d h) / m).
//
// Both directions are bound by memory: forward has to read x and write y, backward to read x and dy and write dx, and every group
// needs all of its rows before the first result can be written.  Two launches each: the first reduces TILES of rows to partial sums
// (a deterministic tree, no atomics), the second adds the partials of its own sample and applies.  Samples of which a workgroup can
// hold a column block's rows in cache take one launch for both.  A tile is processed by the same
// workgroup number in both, i.e. on the same XCD, so that what fits its L2 is not fetched twice.
//
// Ragged batches: sample s owns rows [off[s], off[s + 1]) of one buffer, off on the device.  Tiles never cross samples: sample s uses the
// workgroup numbers from  floor(off[s] / T) + s  on, which leaves it at least ceil(n_s / T) of them whatever the lengths are, so the grid
// and the workspace depend on the row count and the number of samples alone and the call captures into a graph.
//
// Statistics: a thread keeps the mean a of its rows so far, in 32 bits and relative to its first row K, and the sum M2 of squared deviations
// from it.  Four rows at a time: with s = sum d and q = sum d^2 of d = x - K - a, and n rows now, a += s / n, M2 += q - s^2 / n.  No row, the
// first one included, stands so far out that the others are lost beside it (sums about K alone: 5e-4 of the variance of a flat map of 118
// rows a thread with one peak).  Threads, then tiles, are joined in 64 bits as such pairs, relative to the first one's mean c:
//     mean = c + sum n_i (mean_i - c) / n,  M2 = sum M2_i + sum n_i (mean_i - c)^2 - (sum n_i (mean_i - c))^2 / n.  c is the mean of n_1
// of the n values, so the two sides of the last difference are at most n / n_1 times their result: no level of the map, however large,
// cancels in it, and a constant map has variance 0.
//
// Measured (kernel alone; rate of the bytes that it moves itself, the rows' second reading included):
//   96 x 48 x 96 x 32 fp32, ReLU   gn_stats 13.2 us (4.3 TB/s), gn_apply 17.3 (6.5), gn_back_sums 22.6 (5.0), gn_back_apply 24.9 (6.8):  78 us
//                                  for 226 MB that have to move once
//   24 x 12 x 24 x 128 fp32, ReLU  5.0, 5.6, 6.8, 7.0 us: the loads' way and back, twice a launch; the calls take the host 34 us
//   16 crops, 43995 x 64 in all    7.2, 8.0, 9.1, 9.0 us
//   12 x 6 x 12 x 128 fp32         gn_one 7.0 us
#include "elem.h"

namespace {

constexpr int NT = 512, U = 4;    // threads of a workgroup; rows a thread has in flight

struct GnArgs {
    const void *x, *dy;
    void *y;                      // forward: y; backward: dx
    const float *w, *b;
    float *mean, *rstd;           // (S, G)
    const int64_t *off;           // S + 1 row offsets, or NULL: S samples of `rows` rows each
    int64_t rows;                 // per sample, or of the whole buffer (ragged)
    int64_t x_n, x_v, d_n, d_v, y_n, y_v;     // element strides between samples and rows of x, dy, y / dx
    int S, C, G, cpg, gpb, T, t_log, tiles, zero_tail;     // T rows a tile; ragged: T = 1 << t_log
    float eps;
    double2 *part;                // forward: [G][workgroups] (mean, sum of squared deviations from it)
    float2 *part_g, *part_c;      // backward: [G][workgroups] and [workgroups][C]
    float *dw, *db;
};

struct Tile {
    int s;                        // sample; S = the rows behind the last one; -1 = nothing to do
    int t;                        // tile of that sample
    int n;                        // rows in the tile
    int first;                    // workgroup number of the sample's tile 0
    int ntiles;
    int64_t row0, len;            // first row of the tile (of the sample when dense, of the buffer when ragged), rows of the sample
};

__device__ inline int64_t clamp_off(const GnArgs &a, int s)
{
    if (s == 0) return 0;                           // the first sample starts at row 0
    const int64_t o = a.off[s];
    return o < 0 ? 0 : (o > a.rows ? a.rows : o);
}

// the tile of workgroup number `b`; uniform over the workgroup, which calls it together
__device__ inline Tile find_tile(const GnArgs &a, int b)
{
    Tile r;
    int64_t begin;
    if (!a.off) {
        const int tps = a.tiles / a.S;
        r.s = b / tps;
        r.t = b - r.s * tps;
        r.first = r.s * tps;
        r.len = a.rows;
        begin = 0;
    } else {
        // the last s with floor(off[s] / T) + s <= b, which is one of b - floor(rows / T) .. b: a thread looks at one of every `step` of
        // these (one of each, mostly), then at those in between
        int lo = max(0, b - (int)(a.rows >> a.t_log)), n = min(a.S, b) + 1 - lo;
        while (n > 1) {
            const int step = (n + NT - 1) / NT, s = lo + threadIdx.x * step;
            const bool before = (int)threadIdx.x * step < n && (clamp_off(a, s) >> a.t_log) + s <= b;
            const int up = (max(__syncthreads_count(before), 1) - 1) * step;
            lo += up;
            n = min(step, n - up);
        }
        r.s = lo;
        begin = clamp_off(a, lo);
        const int64_t end = lo < a.S ? clamp_off(a, lo + 1) : a.rows;
        r.first = (int)(begin >> a.t_log) + lo;
        r.t = b - r.first;
        r.len = end > begin ? end - begin : 0;      // offsets that decrease give empty samples, never rows outside the buffer
    }
    r.ntiles = a.off ? (int)((r.len + a.T - 1) >> a.t_log) : a.tiles / a.S;
    const int64_t left = r.len - (int64_t)r.t * a.T;
    r.n = r.t < 0 || left < 0 ? 0 : (left < a.T ? (int)left : a.T);
    r.row0 = begin + (int64_t)r.t * a.T;
    if (r.t < 0 || r.n == 0) {
        if (!(r.s < a.S && r.t == 0)) r.s = -1;     // an empty sample keeps its tile 0: it still has statistics to write
    }
    return r;
}

// thread -> (row lane, vector column) of a column block of `nv` vectors
struct Cols {
    int g0, gl, nv, rpb, ri, cv, c;                  // first group, groups, vector columns, rows in parallel, this thread's row lane / column / first channel
    bool live;
};
template <int VEC> __device__ inline Cols columns(const GnArgs &a)
{
    Cols k;
    k.g0 = blockIdx.y * a.gpb;
    k.gl = min(a.gpb, a.G - k.g0);
    k.nv = k.gl * a.cpg / VEC;
    k.rpb = NT / k.nv;
    k.ri = threadIdx.x / k.nv;
    k.cv = threadIdx.x - k.ri * k.nv;
    k.live = k.ri < k.rpb;
    k.c = k.g0 * a.cpg + k.cv * VEC;
    return k;
}

// lanes (a power of two, at most a wave) that share the sums of one of `gl` groups
__device__ inline int lanes_per_group(int gl)
{
    int lp = 64;
    while (lp > 1 && lp * gl > NT) lp >>= 1;
    return lp;
}
template <typename F> __device__ inline void finish_group(double s0, double s1, int lp, int l, int g, F out)
{
    for (int o = lp >> 1; o > 0; o >>= 1) {
        s0 += __shfl_xor(s0, o);
        s1 += __shfl_xor(s1, o);
    }
    if (l == 0) out(g, s0, s1);
}

// Adds the weighted channel sums (backward) of a column block's groups, `cpg` pairs a group in LDS
template <typename F> __device__ inline void reduce_channels(const float2 *lds, int gl, int cpg, F out)
{
    const int lp = lanes_per_group(gl), l = threadIdx.x & (lp - 1);
    for (int g = threadIdx.x / lp; g < gl; g += NT / lp) {
        double s0 = 0, s1 = 0;
        for (int i = l; i < cpg; i += lp) {
            const float2 v = lds[g * cpg + i];
            s0 += v.x;
            s1 += v.y;
        }
        finish_group(s0, s1, lp, l, g, out);
    }
}

// f(there, p[i * stride]) for i = from, from + step, ...: in that order, N of them on their way at a time, the last ones perhaps not there
template <int N, typename P, typename F> __device__ inline void each_pair(const P *p, int64_t stride, int from, int n, int step, F f)
{
    int i = from;
    for (; i + step < n; i += N * step) {
        P v[N];
#pragma unroll
        for (int u = 0; u < N; ++u) v[u] = p[min(i + u * step, n - 1) * stride];
#pragma unroll
        for (int u = 0; u < N; ++u) f(i + u * step < n, v[u]);
    }
    if (i < n) f(true, p[i * stride]);               // all there is, mostly, where samples are small
}

// The sums of a sample's tiles: part[g * tiles + first + p], so that a wave reads neighbouring tiles
template <typename F> __device__ inline void reduce_tiles(const float2 *part, int tiles, int first, int ntiles, int g0, int gl, F out)
{
    const int lp = lanes_per_group(gl), l = threadIdx.x & (lp - 1);
    for (int g = threadIdx.x / lp; g < gl; g += NT / lp) {
        double s0 = 0, s1 = 0;
        each_pair<8>(part + (size_t)(g0 + g) * tiles + first, 1, l, ntiles, lp, [&](bool there, float2 v) {
            s0 += there ? v.x : 0.f;
            s1 += there ? v.y : 0.f;
        });
        finish_group(s0, s1, lp, l, g, out);
    }
}

// 1 / n of a count of values: Newton's iteration from an estimate of 23 bits or more, two steps
__device__ inline double inverse(double n)
{
    double r = __builtin_amdgcn_rcp(n);
    r = __builtin_fma(r, __builtin_fma(-n, r, 1.0), r);
    return __builtin_fma(r, __builtin_fma(-n, r, 1.0), r);
}

__device__ inline float inverse(float n)
{
    const float r = __builtin_amdgcn_rcpf(n);
    return fmaf(r, fmaf(-n, r, 1.f), r);
}

// (mean, M2) of several such pairs with their numbers of values, joined relative to c, the mean of the first one
struct Joined {
    double c, s0, s1;
    __device__ Joined(double c_) : c(c_), s0(0), s1(0) {}
    __device__ void add(double n, double2 v)
    {
        const double d = v.x - c, nd = n * d;
        s0 += nd;
        s1 += v.y + nd * d;
    }
};
__device__ inline double2 joined(double c, double s0, double s1, double inv_n) { return make_double2(c + s0 * inv_n, s1 - s0 * (s0 * inv_n)); }

// Joins, per group of the column block, what the threads left in LDS for `n` rows: `epg` entries a group and row lane, each of `chans` channels
template <typename F> __device__ inline void join_groups(const double2 *lds, int rpb, int n, int gl, int epg, int chans, F out)
{
    const int lp = lanes_per_group(gl), l = threadIdx.x & (lp - 1), all = n / rpb, more = n - all * rpb;      // a lane's rows: all, or one more
    const int per = min(rpb, n) * epg;               // lanes without a row have left nothing
    for (int g = threadIdx.x / lp; g < gl; g += NT / lp) {
        Joined j(n ? lds[g * epg].x : 0);
        for (int i = l; i < per; i += lp) {
            const int r = i / epg;
            j.add((double)((all + (r < more)) * chans), lds[(r * gl + g) * epg + (i - r * epg)]);
        }
        const double c = j.c, inv = inverse((double)n * epg * chans);
        finish_group(j.s0, j.s1, lp, l, g, [&](int g_, double s0, double s1) { out(g_, joined(c, s0, s1, inv)); });
    }
}

// The same over the tiles of one sample of `len` rows: all have T rows but the last one, which its lane adds by itself (an empty sample's one
// place is read and not used).  N pairs on their way: four with one channel a thread, so that three workgroups fit a CU (5000 samples, C 18,
// fp32: 75 us, 85 with eight), else eight, where two fit either way (40 MB fp32, one group: 22.2 us, 23.0 with four).
template <int N, typename F> __device__ inline void join_tiles(const GnArgs &a, int first, int ntiles, int64_t len, int g0, int gl, F out)
{
    const int lp = lanes_per_group(gl), l = threadIdx.x & (lp - 1), before = max(ntiles - 1, 0);
    for (int g = threadIdx.x / lp; g < gl; g += NT / lp) {
        const double2 *p = a.part + (size_t)(g0 + g) * a.tiles + first;
        Joined j(p[0].x);
        const double2 end = p[before];
        double d0 = 0, d1 = 0;
        each_pair<N>(p, 1, l, before, lp, [&](bool there, double2 v) {
            const double d = there ? v.x - j.c : 0;
            d0 += d;
            d1 = __builtin_fma(d, d, d1);
            j.s1 += there ? v.y : 0;
        });
        const double whole = (double)a.T * a.cpg;
        j.s0 = whole * d0;
        j.s1 = __builtin_fma(whole, d1, j.s1);
        if (l == (before & (lp - 1))) j.add((double)(len - (int64_t)before * a.T) * a.cpg, end);
        const double c = j.c, inv = inverse((double)len * a.cpg);
        finish_group(j.s0, j.s1, lp, l, g, [&](int g_, double s0, double s1) { out(g_, joined(c, s0, s1, inv)); });
    }
}

constexpr int ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2;

// h w + b.  ReLU's slope is 0 or 1 by its sign, so it is taken there as written, the product rounded, and forward and backward take the same
// steps: a row's gradient then passes exactly where its output does, and where it does when the formula is written out one operation a time.
template <int ACT> __device__ inline float affine(float h, float w, float b)
{
#pragma clang fp contract(off)
    if constexpr (ACT == ACT_RELU) return h * w + b;
    else return __builtin_fmaf(h, w, b);
}

__device__ inline float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }      // two units in the last place
template <int ACT> __device__ inline float act(float z)
{
    if constexpr (ACT == ACT_RELU) return z < 0.f ? 0.f : z;                 // NaN stays NaN
    else if constexpr (ACT == ACT_SILU) return z * sigmoid(z);
    else return z;
}
template <int ACT> __device__ inline float act_slope(float z)
{
    if constexpr (ACT == ACT_RELU) return z > 0.f ? 1.f : 0.f;
    else if constexpr (ACT == ACT_SILU) {
        const float s = sigmoid(z);
        return s * (1.f + z * (1.f - s));
    } else return 1.f;
}

// This thread's rows of a tile, U of them at a time and the next U on their way while these are worked on; the first are asked for when the
// object is made, so that they travel with whatever else is waited for.  f(row, there, vector); in the last batch rows that are not there
// repeat the tile's last one (there = false), so that no condition stands between the loads.  ONCE: read for the last time.
template <typename T, int VEC, bool ONCE> struct Rows {
    const T *x;
    int64_t stride;
    int r, rpb, n;
    SisVec<T, VEC> cur[U];
    __device__ Rows(const T *x_, int64_t stride_, const Cols &k, int n_) : x(x_), stride(stride_), r(k.ri), rpb(k.rpb), n(n_) { load(cur, r); }
    __device__ void load(SisVec<T, VEC> (&v)[U], int at) const
    {
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = sis3d_raw<T, VEC, ONCE>(x + min(at + u * rpb, n - 1) * stride);
    }
    __device__ const SisVec<T, VEC> &first() const { return cur[0]; }
};
template <typename T, int VEC, bool ONCE, typename F> __device__ inline void each_batch(Rows<T, VEC, ONCE> &x, F f)        // f(U vectors from row x.r on)
{
    SisVec<T, VEC> next[U];
    const int step = U * x.rpb;
    for (; x.r < x.n; x.r += step) {
        if (x.r + step < x.n) x.load(next, x.r + step);
        f(x.cur);
#pragma unroll
        for (int u = 0; u < U; ++u) x.cur[u] = next[u];
    }
}
template <typename T, int VEC, bool ONCE, typename F> __device__ inline void each_row(Rows<T, VEC, ONCE> &x, F f)
{
    each_batch(x, [&](const SisVec<T, VEC> (&v)[U]) {
#pragma unroll
        for (int u = 0; u < U; ++u) f(x.r + u * x.rpb, x.r + u * x.rpb < x.n, v[u]);
    });
}
template <typename T, int VEC, bool ONCE, typename F> __device__ inline void each_row2(Rows<T, VEC, ONCE> &x, Rows<T, VEC, ONCE> &d, F f)
{
    SisVec<T, VEC> nx[U], nd[U];
    const int step = U * x.rpb;
    for (; x.r < x.n; x.r += step) {
        if (x.r + step < x.n) {
            x.load(nx, x.r + step);
            d.load(nd, x.r + step);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) f(x.r + u * x.rpb, x.r + u * x.rpb < x.n, x.cur[u], d.cur[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            x.cur[u] = nx[u];
            d.cur[u] = nd[u];
        }
    }
}

// group, inside the column block, of element i of this thread's vectors
template <int VEC> struct GroupOf {
    int g[VEC];
    __device__ GroupOf(const GnArgs &a, const Cols &k)
    {
        g[0] = k.cv * VEC / a.cpg;
        if (a.cpg % VEC == 0) {
#pragma unroll
            for (int i = 1; i < VEC; ++i) g[i] = g[0];
        } else {
#pragma unroll
            for (int i = 1; i < VEC; ++i) g[i] = (k.cv * VEC + i) / a.cpg;
        }
    }
};

// One tile's rows: mean and sum of squared deviations of every group, to out(group, pair); n = 0: not a number
template <typename T, int VEC, typename F> __device__ inline void tile_sums(const GnArgs &a, const Cols &k, const T *px, int n, double2 *lds, F out)
{
    const bool fold = a.cpg % VEC == 0;              // a vector's channels are of one group: one entry a thread
    if (k.live && n > 0) {
        Rows<T, VEC, false> x(px, a.x_v, k, n);
        float K[VEC], mean[VEC], M2[VEC];            // of each channel's m rows so far, the mean relative to K
        int m = 0;
        sis3d_unpack<T, VEC>(x.first(), K);
#pragma unroll
        for (int i = 0; i < VEC; ++i) mean[i] = M2[i] = 0.f;
        each_batch(x, [&](const SisVec<T, VEC> (&v)[U]) {
            float s[VEC], q[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) s[i] = q[i] = 0.f;
            auto add = [&](const SisVec<T, VEC> &row) {
                float f[VEC];
                sis3d_unpack<T, VEC>(row, f);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float d = f[i] - K[i] - mean[i];
                    s[i] += d;
                    q[i] = fmaf(d, d, q[i]);
                }
            };
            if (x.r + (U - 1) * x.rpb < x.n) {
#pragma unroll
                for (int u = 0; u < U; ++u) add(v[u]);
                m += U;
            } else {
#pragma unroll
                for (int u = 0; u + 1 < U; ++u)
                    if (x.r + u * x.rpb < x.n) add(v[u]), ++m;
            }
            const float im = inverse((float)m);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float t = s[i] * im;
                mean[i] += t;
                M2[i] += fmaf(-s[i], t, q[i]);
            }
        });
        if (m > 0) {
            if (!fold)
#pragma unroll
                for (int i = 0; i < VEC; ++i) lds[(k.ri * k.nv + k.cv) * VEC + i] = make_double2((double)K[i] + mean[i], M2[i]);
            if (fold) {
                // the mean is made of the channels' K in 64 bits, so that it is rounded no more than they are; deviations from it need no more
                // than 32, but their squares may leave them
                double k_all = 0, sq = 0;
                float a_all = 0.f;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    k_all += K[i];
                    a_all += mean[i];
                }
                const double all = (k_all + a_all) * (1.0 / VEC);
                const float near = (float)(all - K[0]);          // relative to the first channel's K, as the channels' means below
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const double d = K[i] - K[0] + mean[i] - near;
                    sq = __builtin_fma(d * m, d, sq) + M2[i];
                }
                lds[k.ri * k.nv + k.cv] = make_double2(all, sq);
            }
        }
    }
    __syncthreads();
    join_groups(lds, k.rpb, n, k.gl, fold ? a.cpg / VEC : a.cpg, fold ? VEC : 1, out);
}

// mean and r of a group from its mean and sum of squared deviations; 0 for an empty sample
__device__ inline void group_stats(const GnArgs &a, const Cols &k, const Tile &t, float *st, int g, double2 v)
{
    double mu = 0, r = 0;
    if (t.len > 0) {
        mu = v.x;
        const double var = v.y * inverse((double)t.len * a.cpg);
        r = 1.0 / sqrt((var < 0 ? 0 : var) + (double)a.eps);      // NaN passes
    }
    st[g] = (float)mu;
    st[k.gl + g] = (float)r;
    if (t.t == 0 && a.mean) {
        a.mean[(size_t)t.s * a.G + k.g0 + g] = (float)mu;
        a.rstd[(size_t)t.s * a.G + k.g0 + g] = (float)r;
    }
}

// What a thread needs for its channels and its first rows, asked for before the statistics are known
template <typename T, int VEC, int ACT, bool ONCE> struct Apply {
    float w[VEC], b[VEC];
    GroupOf<VEC> g;
    Rows<T, VEC, ONCE> x;
    __device__ Apply(const GnArgs &a, const Cols &k, const T *px, int n) : g(a, k), x(px, a.x_v, k, n)
    {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            w[i] = a.w ? a.w[k.c + i] : 1.f;
            b[i] = a.b ? a.b[k.c + i] : 0.f;
        }
    }
    __device__ void run(const GnArgs &a, const Cols &k, const float *st, T *y)
    {
        float mu[VEC], rs[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            mu[i] = st[g.g[i]];
            rs[i] = st[k.gl + g.g[i]];
            if constexpr (ACT != ACT_RELU) w[i] *= rs[i];
        }
        each_row(x, [&](int r, bool there, const SisVec<T, VEC> &v) {
            float o[VEC];
            sis3d_unpack<T, VEC>(v, o);
#pragma unroll
            for (int i = 0; i < VEC; ++i) o[i] = act<ACT>(affine<ACT>(ACT == ACT_RELU ? (o[i] - mu[i]) * rs[i] : o[i] - mu[i], w[i], b[i]));
            if (there) sis3d_store<T, VEC, ONCE>(y + r * a.y_v, o);
        });
    }
};

// rows behind the last sample
template <typename T, int VEC> __device__ inline void zero_rows(const GnArgs &a, const Cols &k, T *y, int n)
{
    if (!a.zero_tail || !k.live) return;
    const float z[VEC] = {};
    for (int r = k.ri; r < n; r += k.rpb) sis3d_store<T, VEC>(y + r * a.y_v, z);
}

template <typename T> __device__ inline const T *rows_at(const void *p, const GnArgs &a, const Cols &k, const Tile &t, int64_t sn, int64_t sv)
{
    return (const T *)p + (a.off ? 0 : t.s * sn) + t.row0 * sv + k.c;
}

template <typename T, int VEC> __global__ __launch_bounds__(NT) void gn_stats(GnArgs a)
{
    extern __shared__ double2 lds[];
    const Tile t = find_tile(a, blockIdx.x);
    if (t.s < 0 || t.s >= a.S || t.n == 0) return;
    const Cols k = columns<VEC>(a);
    tile_sums<T, VEC>(a, k, rows_at<T>(a.x, a, k, t, a.x_n, a.x_v), t.n, lds,
                      [&](int g, double2 v) { a.part[(size_t)(k.g0 + g) * a.tiles + blockIdx.x] = v; });
}

// ONCE: x and y are more than the L2 holds, they are read and written past it
template <typename T, int VEC, int ACT, bool ONCE> __global__ __launch_bounds__(NT) void gn_apply(GnArgs a)
{
    extern __shared__ double2 ldsd[];
    float *st = (float *)ldsd;                       // [gl] mean, [gl] r
    const Tile t = find_tile(a, blockIdx.x);
    if (t.s < 0) return;
    const Cols k = columns<VEC>(a);
    T *y = (T *)rows_at<T>(a.y, a, k, t, a.y_n, a.y_v);
    if (t.s >= a.S) { zero_rows<T, VEC>(a, k, y, t.n); return; }
    if (t.n == 0) {                                  // an empty sample has statistics only
        join_tiles<VEC == 1 ? 4 : 8>(a, t.first, 0, 0, k.g0, k.gl, [&](int g, double2 v) { group_stats(a, k, t, st, g, v); });
        return;
    }
    Cols safe = k;                                   // threads beyond the block's vectors read its first and write nothing
    if (!k.live) safe.ri = safe.cv = 0, safe.c = k.g0 * a.cpg;
    Apply<T, VEC, ACT, ONCE> ap(a, safe, rows_at<T>(a.x, a, safe, t, a.x_n, a.x_v), t.n);
    join_tiles<VEC == 1 ? 4 : 8>(a, t.first, t.ntiles, t.len, k.g0, k.gl, [&](int g, double2 v) { group_stats(a, k, t, st, g, v); });
    __syncthreads();
    if (k.live) ap.run(a, k, st, y);
}

// both in one launch where a sample is one tile (T >= every sample): the second reading of the rows comes from cache
template <typename T, int VEC, int ACT> __global__ __launch_bounds__(NT) void gn_one(GnArgs a)
{
    extern __shared__ double2 lds[];
    __shared__ float st[2 * NT];
    const Tile t = find_tile(a, blockIdx.x);
    if (t.s < 0) return;
    const Cols k = columns<VEC>(a);
    T *y = (T *)rows_at<T>(a.y, a, k, t, a.y_n, a.y_v);
    if (t.s >= a.S) { zero_rows<T, VEC>(a, k, y, t.n); return; }
    const T *x = rows_at<T>(a.x, a, k, t, a.x_n, a.x_v);
    tile_sums<T, VEC>(a, k, x, t.n, lds, [&](int g, double2 v) { group_stats(a, k, t, st, g, v); });
    __syncthreads();
    if (k.live && t.n > 0) Apply<T, VEC, ACT, false>(a, k, x, t.n).run(a, k, st, y);
}

// what a thread needs of its channels in the backward direction
template <int VEC> struct Chan {
    float mu[VEC], rs[VEC], w[VEC], b[VEC];
    __device__ Chan(const GnArgs &a, const Cols &k, int s)
    {
        const GroupOf<VEC> of(a, k);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const size_t g = (size_t)s * a.G + k.g0 + of.g[i];
            mu[i] = a.mean[g];
            rs[i] = a.rstd[g];
            w[i] = a.w ? a.w[k.c + i] : 1.f;
            b[i] = a.b ? a.b[k.c + i] : 0.f;
        }
    }
};

// Channel sums (d, d h) of a tile: to chan(channel, s0, s1), and their weighted sums per group to group(group, S1, S2)
template <typename T, int VEC, int ACT, typename FC, typename FG>
__device__ inline void tile_grad_sums(const GnArgs &a, const Cols &k, const Tile &t, const T *x, const T *dy, float2 *lds, FC chan, FG group)
{
    const int cl = k.gl * a.cpg;
    if (k.live) {
        Rows<T, VEC, false> rx(x, a.x_v, k, t.n), rd(dy, a.d_v, k, t.n);
        const Chan<VEC> c(a, k, t.s);
        float s0[VEC], s1[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) s0[i] = s1[i] = 0.f;
        each_row2(rx, rd, [&](int, bool there, const SisVec<T, VEC> &v, const SisVec<T, VEC> &d) {
            float xf[VEC], df[VEC];
            sis3d_unpack<T, VEC>(v, xf);
            sis3d_unpack<T, VEC>(d, df);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float h = (xf[i] - c.mu[i]) * c.rs[i];
                const float e = df[i] * act_slope<ACT>(affine<ACT>(h, c.w[i], c.b[i]));
                s0[i] += there ? e : 0.f;
                s1[i] += there ? e * h : 0.f;
            }
        });
#pragma unroll
        for (int i = 0; i < VEC; ++i) lds[k.ri * cl + k.cv * VEC + i] = make_float2(s0[i], s1[i]);
    }
    __syncthreads();
    // over the row lanes: q threads a channel, thread (channel, part) adds the rows part, part + q, ... into row `part`, which it alone reads
    const int q = cl < NT ? min(NT / cl, k.rpb) : 1;
    for (int i = threadIdx.x; i < q * cl; i += NT) {
        double s0 = 0, s1 = 0;
        for (int j = i; j < k.rpb * cl; j += q * cl) {
            const float2 v = lds[j];
            s0 += v.x;
            s1 += v.y;
        }
        lds[i] = make_float2((float)s0, (float)s1);
    }
    __syncthreads();
    for (int c = threadIdx.x; c < cl; c += NT) {
        double s0 = 0, s1 = 0;
        for (int j = c; j < q * cl; j += cl) {
            const float2 v = lds[j];
            s0 += v.x;
            s1 += v.y;
        }
        const int cg = k.g0 * a.cpg + c;
        chan(cg, s0, s1);
        const float w = a.w ? a.w[cg] : 1.f;
        lds[c] = make_float2((float)(w * s0), (float)(w * s1));
    }
    __syncthreads();
    reduce_channels(lds, k.gl, a.cpg, group);
}

template <typename T, int VEC, int ACT, bool ONCE> struct ApplyGrad {
    Rows<T, VEC, ONCE> x, d;
    Chan<VEC> c;
    GroupOf<VEC> g;
    __device__ ApplyGrad(const GnArgs &a, const Cols &k, const Tile &t, const T *px, const T *pd)
        : x(px, a.x_v, k, t.n), d(pd, a.d_v, k, t.n), c(a, k, t.s), g(a, k) {}
    __device__ void run(const GnArgs &a, const Cols &k, const float *st, T *dx)
    {
        float m1[VEC], m2[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            m1[i] = st[g.g[i]];
            m2[i] = st[k.gl + g.g[i]];
        }
        each_row2(x, d, [&](int r, bool there, const SisVec<T, VEC> &v, const SisVec<T, VEC> &dv) {
            float o[VEC], df[VEC];
            sis3d_unpack<T, VEC>(v, o);
            sis3d_unpack<T, VEC>(dv, df);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float h = (o[i] - c.mu[i]) * c.rs[i];
                const float e = df[i] * act_slope<ACT>(affine<ACT>(h, c.w[i], c.b[i])) * c.w[i];
                o[i] = c.rs[i] * (e - fmaf(h, m2[i], m1[i]));
            }
            if (there) sis3d_store<T, VEC, ONCE>(dx + r * a.y_v, o);
        });
    }
};

template <typename T, int VEC, int ACT> __global__ __launch_bounds__(NT) void gn_back_sums(GnArgs a)
{
    extern __shared__ double2 ldsd[];
    const Tile t = find_tile(a, blockIdx.x);
    const Cols k = columns<VEC>(a);
    if (t.s < 0 || t.s >= a.S || t.n == 0) {         // no rows: its channel sums are read all the same
        for (int c = threadIdx.x; c < k.gl * a.cpg; c += NT) a.part_c[(size_t)blockIdx.x * a.C + k.g0 * a.cpg + c] = make_float2(0.f, 0.f);
        return;
    }
    tile_grad_sums<T, VEC, ACT>(
        a, k, t, rows_at<T>(a.x, a, k, t, a.x_n, a.x_v), rows_at<T>(a.dy, a, k, t, a.d_n, a.d_v), (float2 *)ldsd,
        [&](int c, double s0, double s1) { a.part_c[(size_t)blockIdx.x * a.C + c] = make_float2((float)s0, (float)s1); },
        [&](int g, double s0, double s1) { a.part_g[(size_t)(k.g0 + g) * a.tiles + blockIdx.x] = make_float2((float)s0, (float)s1); });
}

template <typename T, int VEC, int ACT, bool ONCE> __global__ __launch_bounds__(NT) void gn_back_apply(GnArgs a)
{
    extern __shared__ double2 ldsd[];
    float *st = (float *)ldsd;                       // [gl] S1 / m, [gl] S2 / m
    if ((int)blockIdx.x >= a.tiles) {                // the last workgroups add the channel sums of all tiles: dw, db
        if (blockIdx.y) return;
        __shared__ double acc[NT][2];
        const int c = ((int)blockIdx.x - a.tiles) * 32 + (threadIdx.x & 31), l = threadIdx.x >> 5;
        double s0 = 0, s1 = 0;
        if (c < a.C)
            each_pair<8>(a.part_c + c, a.C, l, a.tiles, NT / 32, [&](bool there, float2 v) {
                s0 += there ? v.x : 0.f;
                s1 += there ? v.y : 0.f;
            });
        acc[threadIdx.x][0] = s0;
        acc[threadIdx.x][1] = s1;
        __syncthreads();
        if (threadIdx.x < 32 && c < a.C) {
            for (int i = 1; i < NT / 32; ++i) {
                s0 += acc[i * 32 + threadIdx.x][0];
                s1 += acc[i * 32 + threadIdx.x][1];
            }
            if (a.db) a.db[c] = (float)s0;
            if (a.dw) a.dw[c] = (float)s1;
        }
        return;
    }
    const Tile t = find_tile(a, blockIdx.x);
    if (t.s < 0 || t.n == 0) return;
    const Cols k = columns<VEC>(a);
    T *dx = (T *)rows_at<T>(a.y, a, k, t, a.y_n, a.y_v);
    if (t.s >= a.S) { zero_rows<T, VEC>(a, k, dx, t.n); return; }
    Cols safe = k;
    if (!k.live) safe.ri = safe.cv = 0, safe.c = k.g0 * a.cpg;
    ApplyGrad<T, VEC, ACT, ONCE> ap(a, safe, t, rows_at<T>(a.x, a, safe, t, a.x_n, a.x_v), rows_at<T>(a.dy, a, safe, t, a.d_n, a.d_v));
    const double m = (double)t.len * a.cpg;
    reduce_tiles(a.part_g, a.tiles, t.first, t.ntiles, k.g0, k.gl, [&](int g, double s0, double s1) {
        st[g] = (float)(s0 / m);
        st[k.gl + g] = (float)(s1 / m);
    });
    __syncthreads();
    if (k.live) ap.run(a, k, st, dx);
}

// both in one launch for one dense sample that is one tile: dw and db are its own channel sums
template <typename T, int VEC, int ACT> __global__ __launch_bounds__(NT) void gn_back_one(GnArgs a)
{
    extern __shared__ double2 ldsd[];
    __shared__ float st[2 * NT];
    const Tile t = find_tile(a, blockIdx.x);
    const Cols k = columns<VEC>(a);
    const double m = (double)t.len * a.cpg;
    const T *x = rows_at<T>(a.x, a, k, t, a.x_n, a.x_v), *dy = rows_at<T>(a.dy, a, k, t, a.d_n, a.d_v);
    tile_grad_sums<T, VEC, ACT>(
        a, k, t, x, dy, (float2 *)ldsd,
        [&](int c, double s0, double s1) {
            if (a.db) a.db[c] = (float)s0;
            if (a.dw) a.dw[c] = (float)s1;
        },
        [&](int g, double s0, double s1) {
            st[g] = (float)(s0 / m);
            st[k.gl + g] = (float)(s1 / m);
        });
    __syncthreads();
    if (k.live) ApplyGrad<T, VEC, ACT, false>(a, k, t, x, dy).run(a, k, st, (T *)rows_at<T>(a.y, a, k, t, a.y_n, a.y_v));
}

struct Plan {
    int vec, gpb, ncol, T, t_log, one, once, rc;
    int64_t tiles;
};

int gcd_(int a, int b) { return b ? gcd_(b, a % b) : a; }

// Tiles of rows and column blocks of whole groups.  `wide`: 16-byte accesses are possible (alignment of every pointer and stride).
Plan make_plan(int dtype, int S, int64_t rows, int ragged, int C, int G, bool wide, bool backward)
{
    Plan p{};
    const int es = sis3d_elem_bytes(dtype), cpg = C / G;
    p.vec = wide && C % (16 / es) == 0 ? 16 / es : 1;
    const int gu = p.vec / gcd_(cpg, p.vec);               // groups whose channels are whole vectors
    const int fit = (int)((int64_t)NT * p.vec / cpg), most = (fit < NT ? fit : NT) / gu * gu;        // a block has at most NT groups
    if (most < 1) { p.rc = SIS3D_EUNSUPPORTED; return p; }
    // a column block is one 128-byte line of a row, or one group if that is wider: the narrower it is, the fewer groups a workgroup of
    // the second launch has to add the tiles' sums of
    p.gpb = gu;
    const int64_t total = ragged ? rows : rows * S;
    // one workgroup takes a whole sample where that is little: up to 128 KB of a line it is sooner done than a second launch.  Its column
    // blocks are narrower than a line while there are fewer than 512 of them: the rows come from cache, and more CUs take part
    p.one = rows * (cpg * gu * es > 128 ? cpg * gu * es : 128) <= 128 * 1024 && !(backward && (S != 1 || ragged));
    // Samples of few rows: wider, so that a workgroup has 64 KB to work on (5000 samples of 31 rows of
    // 256 fp32 channels: forward 385 us by lines, 76 by whole rows; 1000 of 156: 90 us by lines, 53 by 16 KB, 38 by 64)
    const int64_t mean_rows = S ? total / S : total;
    while (p.gpb < G && (p.gpb * cpg * es < 128 || mean_rows * p.gpb * cpg * es < 64 << 10) && p.gpb + gu <= most &&
           !(p.one && (int64_t)S * G / p.gpb <= 512))
        p.gpb += gu;
    // whole rows where groups do not fill lines: neighbouring blocks would fetch the line they share twice (40 MB fp32, forward / backward,
    // 48 channels in 16 groups 42 / 65 us by blocks, 30 / 45 by rows; 96 in 32 48 / 71, 29 / 44)
    if (p.gpb > G || (!p.one && p.gpb * cpg * es % 128 && G <= most)) p.gpb = G;
    p.ncol = (G + p.gpb - 1) / p.gpb;
    int64_t T;
    if (p.one) T = rows;
    else {
        // a workgroup per CU, two where the second launch's sums over the tiles are little against the rows (48 x 24 x 48 x 64 bf16: 512
        // tiles 6.6 + 13.0 us, 256 tiles 5.6 + 10.2 us)
        const int blocks = total * C * es < 16 << 20 ? 256 : 512;
        T = (total * p.ncol + blocks - 1) / blocks;
        const int rpb = (int)(NT / (p.gpb * cpg / p.vec));
        if (T < rpb) T = rpb;
        if (T > 1024 * rpb) T = 1024 * rpb;                // rows of a thread, which adds them in 32 bits
    }
    if (T < 1) T = 1;                                      // no rows
    p.once = total * C * es > 16 << 20;                    // half of what the eight L2s hold
    p.t_log = 0;
    while (((int64_t)1 << p.t_log) < T) ++p.t_log;
    if (ragged) T = (int64_t)1 << p.t_log;                 // a shift in place of divisions by T
    p.T = (int)T;
    p.tiles = ragged ? (rows >> p.t_log) + S + 1 : S * ((rows + T - 1) / T);
    // a launch has at most 2^32 - 1 threads in one dimension and 65535 workgroups in the other
    if (p.tiles + (C + 31) / 32 > 0xffffffffll / NT || p.ncol > 65535) p.rc = SIS3D_EUNSUPPORTED;
    return p;
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

size_t ws_bytes_of(const Plan &p, int C, int G, bool backward)
{
    const size_t t = (size_t)p.tiles;
    return p.one ? 0 : backward ? t * ((size_t)C + G) * sizeof(float2) : t * G * sizeof(double2);
}

#define GN_ACT(KERN, ...)                                                                                       \
    switch (act) {                                                                                                 \
    case ACT_RELU: hipLaunchKernelGGL((KERN<T, VEC, ACT_RELU __VA_ARGS__>), grid, dim3(NT), lds, st, a); break;                \
    case ACT_SILU: hipLaunchKernelGGL((KERN<T, VEC, ACT_SILU __VA_ARGS__>), grid, dim3(NT), lds, st, a); break;                \
    default: hipLaunchKernelGGL((KERN<T, VEC, ACT_NONE __VA_ARGS__>), grid, dim3(NT), lds, st, a); break;                      \
    }

template <typename T, int VEC> int launch(const GnArgs &a, const Plan &p, int act, bool backward, hipStream_t st)
{
    dim3 grid((unsigned)p.tiles, p.ncol);
    // forward: a pair of doubles a thread, or a channel where groups are not whole vectors; backward: a pair of floats a channel.  The last
    // column block may have fewer groups, and then more rows in parallel, than the others
    size_t lds = 0;
    for (int groups : {p.gpb, a.G - (p.ncol - 1) * p.gpb}) {
        const int cl = groups * a.cpg, rpb = NT / (cl / VEC);
        const size_t need = backward ? (size_t)rpb * cl * sizeof(float2) : (size_t)rpb * (a.cpg % VEC ? cl : cl / VEC) * sizeof(double2);
        if (need > lds) lds = need;
    }
    if (p.one) {
        if (backward) { GN_ACT(gn_back_one) }
        else { GN_ACT(gn_one) }
        return sis3d_check_launch();
    }
    if (backward) { GN_ACT(gn_back_sums) }
    else hipLaunchKernelGGL((gn_stats<T, VEC>), grid, dim3(NT), lds, st, a);
    const int rc = sis3d_check_launch();
    if (rc) return rc;
    if (backward) grid.x += (a.C + 31) / 32;
    lds = 2 * p.gpb * sizeof(float);
    if (backward) {
        if (p.once) { GN_ACT(gn_back_apply, , true) }
        else { GN_ACT(gn_back_apply, , false) }
    } else {
        if (p.once) { GN_ACT(gn_apply, , true) }
        else { GN_ACT(gn_apply, , false) }
    }
    return sis3d_check_launch();
}

int dispatch(const GnArgs &a, const Plan &p, int dtype, int act, bool backward, hipStream_t st)
{
    switch (dtype) {
    case SIS3D_F32: return p.vec > 1 ? launch<float, 4>(a, p, act, backward, st) : launch<float, 1>(a, p, act, backward, st);
    case SIS3D_BF16: return p.vec > 1 ? launch<__bf16, 8>(a, p, act, backward, st) : launch<__bf16, 1>(a, p, act, backward, st);
    default: return p.vec > 1 ? launch<_Float16, 8>(a, p, act, backward, st) : launch<_Float16, 1>(a, p, act, backward, st);
    }
}

int check_args(int dtype, int S, int64_t rows, int C, int G, int act)
{
    if (!sis3d_elem_bytes(dtype) || S < 0 || rows < 0 || C <= 0 || G <= 0 || C % G || act < ACT_NONE || act > ACT_SILU) return SIS3D_EINVAL;
    return SIS3D_OK;
}

} // namespace

extern "C" size_t sis3d_group_norm_workspace_bytes(int dtype, int S, int64_t rows, int ragged, int C, int G, int backward)
{
    if (check_args(dtype, S, rows, C, G, 0)) return 0;
    size_t most = 0;
    for (int wide = 0; wide < 2; ++wide) {                 // whichever access width the pointers will allow
        const Plan p = make_plan(dtype, S, rows, ragged, C, G, wide, backward);
        const size_t b = p.rc ? 0 : ws_bytes_of(p, C, G, backward);
        if (b > most) most = b;
    }
    return most;
}

extern "C" int sis3d_group_norm_forward(const void *x, int dtype, int S, int64_t rows, const int64_t *offsets, int64_t x_sample, int64_t x_row,
                                        int C, int G, const float *weight, const float *bias, float eps, int act, void *y, int64_t y_sample,
                                        int64_t y_row, int zero_tail, float *mean, float *rstd, void *workspace, size_t workspace_bytes,
                                        sis3d_stream_t stream)
{
    const int rc = check_args(dtype, S, rows, C, G, act);
    if (rc) return rc;
    if ((mean == nullptr) != (rstd == nullptr) || !(eps >= 0.f)) return SIS3D_EINVAL;
    hipStream_t st = as_stream(stream);
    if ((S == 0 && !offsets) || rows == 0) {               // no rows: statistics of nothing
        if (!mean || !S) return SIS3D_OK;
        const int rz = sis3d_fill32(mean, 0, (size_t)S * G * 4, st);
        return rz ? rz : sis3d_fill32(rstd, 0, (size_t)S * G * 4, st);
    }
    if (!x || !y) return SIS3D_EINVAL;
    const int es = sis3d_elem_bytes(dtype);
    const int64_t strides = (offsets ? 0 : (x_sample | y_sample)) | x_row | y_row;
    const Plan p = make_plan(dtype, S, rows, offsets != nullptr, C, G, aligned16(x) && aligned16(y) && strides * es % 16 == 0, false);
    if (p.rc) return p.rc;
    if (workspace_bytes < ws_bytes_of(p, C, G, false)) return SIS3D_EWORKSPACE;
    if (!p.one && (!workspace || !aligned16(workspace))) return SIS3D_EINVAL;
    GnArgs a{};
    a.x = x; a.y = y; a.w = weight; a.b = bias; a.mean = mean; a.rstd = rstd; a.off = offsets; a.rows = rows;
    a.x_n = x_sample; a.x_v = x_row; a.y_n = y_sample; a.y_v = y_row;
    a.S = S; a.C = C; a.G = G; a.cpg = C / G; a.gpb = p.gpb; a.T = p.T; a.t_log = p.t_log; a.tiles = (int)p.tiles; a.zero_tail = zero_tail; a.eps = eps;
    a.part = (double2 *)workspace;
    return dispatch(a, p, dtype, act, false, st);
}

extern "C" int sis3d_group_norm_backward(const void *dy, int64_t dy_sample, int64_t dy_row, const void *x, int dtype, int S, int64_t rows,
                                         const int64_t *offsets, int64_t x_sample, int64_t x_row, int C, int G, const float *mean,
                                         const float *rstd, const float *weight, const float *bias, int act, void *dx, int64_t dx_sample,
                                         int64_t dx_row, float *dweight, float *dbias, void *workspace, size_t workspace_bytes,
                                         sis3d_stream_t stream)
{
    const int rc = check_args(dtype, S, rows, C, G, act);
    if (rc) return rc;
    hipStream_t st = as_stream(stream);
    if (S == 0 || rows == 0) {
        int rz = dweight ? sis3d_fill32(dweight, 0, (size_t)C * 4, st) : SIS3D_OK;
        if (!rz && dbias) rz = sis3d_fill32(dbias, 0, (size_t)C * 4, st);
        if (rz || rows == 0 || !offsets) return rz;
    }
    if (!x || !dy || !dx || ((!mean || !rstd) && S)) return SIS3D_EINVAL;
    const int es = sis3d_elem_bytes(dtype);
    const int64_t strides = (offsets ? 0 : (x_sample | dy_sample | dx_sample)) | x_row | dy_row | dx_row;
    const Plan p = make_plan(dtype, S, rows, offsets != nullptr, C, G, aligned16(x) && aligned16(dy) && aligned16(dx) && strides * es % 16 == 0, true);
    if (p.rc) return p.rc;
    if (workspace_bytes < ws_bytes_of(p, C, G, true)) return SIS3D_EWORKSPACE;
    if (!p.one && (!workspace || !aligned16(workspace))) return SIS3D_EINVAL;
    GnArgs a{};
    a.x = x; a.dy = dy; a.y = dx; a.w = weight; a.b = bias; a.mean = (float *)mean; a.rstd = (float *)rstd; a.off = offsets; a.rows = rows;
    a.x_n = x_sample; a.x_v = x_row; a.d_n = dy_sample; a.d_v = dy_row; a.y_n = dx_sample; a.y_v = dx_row;
    a.S = S; a.C = C; a.G = G; a.cpg = C / G; a.gpb = p.gpb; a.T = p.T; a.t_log = p.t_log; a.tiles = (int)p.tiles; a.zero_tail = 1;
    a.part_c = (float2 *)workspace;
    a.part_g = a.part_c + (size_t)p.tiles * C;
    a.dw = dweight; a.db = dbias;
    return dispatch(a, p, dtype, act, true, st);
}
