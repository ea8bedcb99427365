// Group norm with an activation on channels-last rows, forward and backward.
//
// Sample s has n_s rows (voxels) of C channels in G groups of c = C / G; m = n_s c.  Per (sample, group)
//     mu = 1/m sum x,  var = 1/m sum (x - mu)^2,  r = (var + eps)^-1/2,  h = (x - mu) r,  z = h w + b,  y = act(z)
// and backward, with d = dy act'(z):
//     db = sum d,  dw = sum d h  (over samples and rows),  dx = r (w d - (sum_group w d + h sum_group w d h) / m).
//
// Both directions are bound by memory: forward has to read x and write y, backward to read x and dy and write dx, and every group
// needs all of its rows before the first result can be written.  Two launches each: the first reduces TILES of rows to partial sums
// (a deterministic tree, no atomics), the second adds the partials of its own sample and applies.  A tile is processed by the same
// workgroup number in both, i.e. on the same XCD, so that what fits its L2 is not fetched twice.
//
// Ragged batches: sample s owns rows [off[s], off[s + 1]) of one buffer, off on the device.  Tiles never cross samples: sample s uses the
// workgroup numbers from  floor(off[s] / T) + s  on, which leaves it at least ceil(n_s / T) of them whatever the lengths are, so the grid
// and the workspace depend on the row count and the number of samples alone and the call captures into a graph.
//
// Sums: a thread adds d = x - K and d^2 in 32 bits over its (at most a few hundred) rows, K its own first row, so a mean that is large
// against the deviation does not cancel; everything across threads is added in 64 bits.
#include "elem.h"

namespace {

constexpr int NT = 512;

struct GnArgs {
    const void *x, *dy;
    void *y;                      // forward: y; backward: dx
    const float *w, *b;
    float *mean, *rstd;           // (S, G)
    const int64_t *off;           // S + 1 row offsets, or NULL: S samples of `rows` rows each
    int64_t rows;                 // per sample, or of the whole buffer (ragged)
    int64_t x_n, x_v, d_n, d_v, y_n, y_v;     // element strides between samples and rows of x, dy, y / dx
    int S, C, G, cpg, gpb, T, tiles, act, zero_tail;
    float eps;
    double2 *part;                // forward: [workgroups][G] (sum, sum of squares)
    float2 *part_g, *part_c;      // backward: [workgroups][G] and [workgroups][C]
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

// the tile of workgroup number `b`; uniform over the workgroup
__device__ inline Tile find_tile(const GnArgs &a, int b)
{
    Tile r;
    int64_t begin;
    if (!a.off) {
        const int tps = (int)((a.rows + a.T - 1) / a.T);
        r.s = b / tps;
        r.t = b - r.s * tps;
        r.first = r.s * tps;
        r.len = a.rows;
        begin = 0;
    } else {
        // the last s with floor(off[s] / T) + s <= b
        int lo = 0, hi = a.S + 1;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (clamp_off(a, mid) / a.T + mid <= b) lo = mid;
            else hi = mid;
        }
        r.s = lo;
        begin = clamp_off(a, lo);
        const int64_t end = lo < a.S ? clamp_off(a, lo + 1) : a.rows;
        r.first = (int)(begin / a.T) + lo;
        r.t = b - r.first;
        r.len = end > begin ? end - begin : 0;      // offsets that decrease give empty samples, never rows outside the buffer
    }
    r.ntiles = (int)((r.len + a.T - 1) / a.T);
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

// Adds, per group of the column block, pairs that the threads left in LDS: lds[row lane][channel of the block] -> out(group, pair).
template <typename P, typename F> __device__ inline void reduce_groups(const P *lds, int rpb, int gl, int cpg, F out)
{
    int lp = 1;
    while (lp < 64 && lp * 2 * gl <= NT) lp *= 2;
    const int per = rpb * cpg;
    for (int g = threadIdx.x / lp; g < gl; g += NT / lp) {
        const int l = threadIdx.x % lp;
        double s0 = 0, s1 = 0;
        for (int i = l; i < per; i += lp) {
            const int r = i / cpg;
            const P v = lds[(size_t)r * gl * cpg + g * cpg + (i - r * cpg)];
            s0 += v.x;
            s1 += v.y;
        }
        for (int o = lp >> 1; o > 0; o >>= 1) {
            s0 += __shfl_xor(s0, o);
            s1 += __shfl_xor(s1, o);
        }
        if (l == 0) out(g, s0, s1);
    }
}

// The same over the tiles of one sample: part[(first + p) * G + g]
template <typename P, typename F> __device__ inline void reduce_tiles(const P *part, int first, int ntiles, int G, int g0, int gl, F out)
{
    int lp = 1;
    while (lp < 64 && lp * 2 * gl <= NT) lp *= 2;
    for (int g = threadIdx.x / lp; g < gl; g += NT / lp) {
        const int l = threadIdx.x % lp;
        double s0 = 0, s1 = 0;
        for (int p = l; p < ntiles; p += lp) {
            const P v = part[(size_t)(first + p) * G + g0 + g];
            s0 += v.x;
            s1 += v.y;
        }
        for (int o = lp >> 1; o > 0; o >>= 1) {
            s0 += __shfl_xor(s0, o);
            s1 += __shfl_xor(s1, o);
        }
        if (l == 0) out(g, s0, s1);
    }
}

constexpr int ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2;

template <int ACT> __device__ inline float act(float z)
{
    if constexpr (ACT == ACT_RELU) return z < 0.f ? 0.f : z;                 // NaN stays NaN
    else if constexpr (ACT == ACT_SILU) return z / (1.f + __expf(-z));
    else return z;
}
template <int ACT> __device__ inline float act_slope(float z)
{
    if constexpr (ACT == ACT_RELU) return z > 0.f ? 1.f : 0.f;
    else if constexpr (ACT == ACT_SILU) {
        const float s = 1.f / (1.f + __expf(-z));
        return s * (1.f + z * (1.f - s));
    } else return 1.f;
}

template <typename T, int VEC> __global__ __launch_bounds__(NT) void gn_stats(GnArgs a)
{
    extern __shared__ double2 lds[];
    const Tile t = find_tile(a, blockIdx.x);
    if (t.s < 0 || t.s >= a.S || t.n == 0) return;
    const Cols k = columns<VEC>(a);
    const T *x = (const T *)a.x + (a.off ? 0 : t.s * a.x_n) + t.row0 * a.x_v + k.c;
    if (k.live) {
        float K[VEC], s1[VEC], s2[VEC], v[VEC];
        int n = 0;
#pragma unroll
        for (int i = 0; i < VEC; ++i) K[i] = s1[i] = s2[i] = 0.f;
        if (k.ri < t.n) sis3d_load<T, VEC>(x + k.ri * a.x_v, K);
        for (int r = k.ri; r < t.n; r += k.rpb, ++n) {
            sis3d_load<T, VEC>(x + r * a.x_v, v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float d = v[i] - K[i];
                s1[i] += d;
                s2[i] = fmaf(d, d, s2[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const double kk = K[i];
            lds[(size_t)k.ri * k.nv * VEC + k.cv * VEC + i] = make_double2(n * kk + s1[i], s2[i] + kk * (2.0 * s1[i] + n * kk));
        }
    }
    __syncthreads();
    reduce_groups(lds, k.rpb, k.gl, a.cpg, [&](int g, double s0, double s1) { a.part[(size_t)blockIdx.x * a.G + k.g0 + g] = make_double2(s0, s1); });
}

template <typename T, int VEC, int ACT> __global__ __launch_bounds__(NT) void gn_apply(GnArgs a)
{
    extern __shared__ float st[];                    // [gl] mean, [gl] r
    const Tile t = find_tile(a, blockIdx.x);
    if (t.s < 0) return;
    const Cols k = columns<VEC>(a);
    T *y = (T *)a.y + (a.off ? 0 : t.s * a.y_n) + t.row0 * a.y_v + k.c;
    if (t.s >= a.S) {                                // rows behind the last sample
        if (a.zero_tail && k.live) {
            const float z[VEC] = {};
            for (int r = k.ri; r < t.n; r += k.rpb) sis3d_store<T, VEC>(y + r * a.y_v, z);
        }
        return;
    }
    const double m = (double)t.len * a.cpg;
    reduce_tiles(a.part, t.first, t.ntiles, a.G, k.g0, k.gl, [&](int g, double s0, double s1) {
        double mu = 0, r = 0;
        if (m > 0) {
            mu = s0 / m;
            const double var = s1 / m - mu * mu;
            r = 1.0 / sqrt((var < 0 ? 0 : var) + (double)a.eps);      // NaN passes
        }
        st[g] = (float)mu;
        st[k.gl + g] = (float)r;
        if (t.t == 0 && a.mean) {
            a.mean[(size_t)t.s * a.G + k.g0 + g] = (float)mu;
            a.rstd[(size_t)t.s * a.G + k.g0 + g] = (float)r;
        }
    });
    __syncthreads();
    if (!k.live) return;
    const T *x = (const T *)a.x + (a.off ? 0 : t.s * a.x_n) + t.row0 * a.x_v + k.c;
    float mu[VEC], sc[VEC], sh[VEC], v[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        const int g = (k.cv * VEC + i) / a.cpg;
        mu[i] = st[g];
        sc[i] = st[k.gl + g] * (a.w ? a.w[k.c + i] : 1.f);
        sh[i] = a.b ? a.b[k.c + i] : 0.f;
    }
    for (int r = k.ri; r < t.n; r += k.rpb) {
        sis3d_load<T, VEC>(x + r * a.x_v, v);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = act<ACT>(fmaf(v[i] - mu[i], sc[i], sh[i]));
        sis3d_store<T, VEC>(y + r * a.y_v, v);
    }
}

template <typename T, int VEC, int ACT> __global__ __launch_bounds__(NT) void gn_back_sums(GnArgs a)
{
    extern __shared__ double2 ldsd[];
    float2 *lds = (float2 *)ldsd;
    const Tile t = find_tile(a, blockIdx.x);
    const Cols k = columns<VEC>(a);
    const int cl = k.gl * a.cpg;
    if (t.s < 0 || t.s >= a.S || t.n == 0) {         // no rows: its channel sums are read all the same
        for (int c = threadIdx.x; c < cl; c += NT) a.part_c[(size_t)blockIdx.x * a.C + k.g0 * a.cpg + c] = make_float2(0.f, 0.f);
        return;
    }
    if (k.live) {
        const T *x = (const T *)a.x + (a.off ? 0 : t.s * a.x_n) + t.row0 * a.x_v + k.c;
        const T *dy = (const T *)a.dy + (a.off ? 0 : t.s * a.d_n) + t.row0 * a.d_v + k.c;
        float mu[VEC], rs[VEC], w[VEC], b[VEC], v[VEC], d[VEC], s0[VEC], s1[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const size_t g = (size_t)t.s * a.G + (k.c + i) / a.cpg;
            mu[i] = a.mean[g];
            rs[i] = a.rstd[g];
            w[i] = a.w ? a.w[k.c + i] : 1.f;
            b[i] = a.b ? a.b[k.c + i] : 0.f;
            s0[i] = s1[i] = 0.f;
        }
        for (int r = k.ri; r < t.n; r += k.rpb) {
            sis3d_load<T, VEC>(x + r * a.x_v, v);
            sis3d_load<T, VEC>(dy + r * a.d_v, d);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float h = (v[i] - mu[i]) * rs[i];
                const float e = d[i] * act_slope<ACT>(fmaf(h, w[i], b[i]));
                s0[i] += e;
                s1[i] = fmaf(e, h, s1[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) lds[(size_t)k.ri * cl + k.cv * VEC + i] = make_float2(s0[i], s1[i]);
    }
    __syncthreads();
    // per channel over the row lanes, then per group with the weights
    for (int c = threadIdx.x; c < cl; c += NT) {
        double s0 = 0, s1 = 0;
        for (int r = 0; r < k.rpb; ++r) {
            const float2 v = lds[(size_t)r * cl + c];
            s0 += v.x;
            s1 += v.y;
        }
        const int cg = k.g0 * a.cpg + c;
        a.part_c[(size_t)blockIdx.x * a.C + cg] = make_float2((float)s0, (float)s1);
        const float w = a.w ? a.w[cg] : 1.f;
        lds[c] = make_float2((float)(w * s0), (float)(w * s1));      // row lane 0's place of the same channel: read by this thread alone before
    }
    __syncthreads();
    reduce_groups(lds, 1, k.gl, a.cpg, [&](int g, double s0, double s1) { a.part_g[(size_t)blockIdx.x * a.G + k.g0 + g] = make_float2((float)s0, (float)s1); });
}

template <typename T, int VEC, int ACT> __global__ __launch_bounds__(NT) void gn_back_apply(GnArgs a)
{
    extern __shared__ float st[];                    // [gl] S1 / m, [gl] S2 / m
    if ((int)blockIdx.x >= a.tiles) {                // the last workgroups add the channel sums of all tiles: dw, db
        if (blockIdx.y) return;
        __shared__ double acc[NT][2];
        const int c = ((int)blockIdx.x - a.tiles) * 32 + (threadIdx.x & 31), l = threadIdx.x >> 5;
        double s0 = 0, s1 = 0;
        if (c < a.C)
            for (int p = l; p < a.tiles; p += NT / 32) {
                const float2 v = a.part_c[(size_t)p * a.C + c];
                s0 += v.x;
                s1 += v.y;
            }
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
    T *dx = (T *)a.y + (a.off ? 0 : t.s * a.y_n) + t.row0 * a.y_v + k.c;
    if (t.s >= a.S) {
        if (a.zero_tail && k.live) {
            const float z[VEC] = {};
            for (int r = k.ri; r < t.n; r += k.rpb) sis3d_store<T, VEC>(dx + r * a.y_v, z);
        }
        return;
    }
    const double m = (double)t.len * a.cpg;
    reduce_tiles(a.part_g, t.first, t.ntiles, a.G, k.g0, k.gl, [&](int g, double s0, double s1) {
        st[g] = (float)(s0 / m);
        st[k.gl + g] = (float)(s1 / m);
    });
    __syncthreads();
    if (!k.live) return;
    const T *x = (const T *)a.x + (a.off ? 0 : t.s * a.x_n) + t.row0 * a.x_v + k.c;
    const T *dy = (const T *)a.dy + (a.off ? 0 : t.s * a.d_n) + t.row0 * a.d_v + k.c;
    float mu[VEC], rs[VEC], w[VEC], b[VEC], m1[VEC], m2[VEC], v[VEC], d[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        const int gl = (k.cv * VEC + i) / a.cpg;
        const size_t g = (size_t)t.s * a.G + k.g0 + gl;
        mu[i] = a.mean[g];
        rs[i] = a.rstd[g];
        w[i] = a.w ? a.w[k.c + i] : 1.f;
        b[i] = a.b ? a.b[k.c + i] : 0.f;
        m1[i] = st[gl];
        m2[i] = st[k.gl + gl];
    }
    for (int r = k.ri; r < t.n; r += k.rpb) {
        sis3d_load<T, VEC>(x + r * a.x_v, v);
        sis3d_load<T, VEC>(dy + r * a.d_v, d);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const float h = (v[i] - mu[i]) * rs[i];
            const float e = d[i] * act_slope<ACT>(fmaf(h, w[i], b[i])) * w[i];
            v[i] = rs[i] * (e - fmaf(h, m2[i], m1[i]));
        }
        sis3d_store<T, VEC>(dx + r * a.y_v, v);
    }
}

struct Plan {
    int vec, gpb, ncol, T;
    int64_t tiles;
    int rc;
};

int gcd_(int a, int b) { return b ? gcd_(b, a % b) : a; }

// Tiles of rows and column blocks of whole groups.  `wide`: 16-byte accesses are possible (alignment of every pointer and stride).
Plan make_plan(int dtype, int S, int64_t rows, int ragged, int C, int G, bool wide)
{
    Plan p{};
    const int es = sis3d_elem_bytes(dtype), cpg = C / G;
    p.vec = wide && C % (16 / es) == 0 ? 16 / es : 1;
    const int gu = p.vec / gcd_(cpg, p.vec);               // groups whose channels are whole vectors
    int most = (int)((int64_t)NT * p.vec / cpg) / gu * gu;
    if (most > G) most = G;
    if (most < gu || most < 1) { p.rc = SIS3D_EUNSUPPORTED; return p; }
    if (most > 32) most = 32 / gu * gu > 0 ? 32 / gu * gu : gu;    // bounds what a workgroup of the second launch has to add up
    p.gpb = most;
    p.ncol = (G + p.gpb - 1) / p.gpb;
    const int64_t total = ragged ? rows : rows * S;
    int64_t T = (total * p.ncol + 511) / 512;              // about two workgroups per CU
    const int rpb = NT * p.vec / (p.gpb * cpg);
    if (T < rpb) T = rpb;
    if (T < 1) T = 1;
    if (T > (1 << 24)) T = 1 << 24;
    p.T = (int)T;
    p.tiles = ragged ? rows / T + S + 1 : S * ((rows + T - 1) / T);
    if (p.tiles > 0x7fffff00) p.rc = SIS3D_EUNSUPPORTED;
    return p;
}

bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

size_t ws_bytes_of(const Plan &p, int C, int G, bool backward)
{
    const size_t t = (size_t)p.tiles;
    return backward ? t * ((size_t)C + G) * sizeof(float2) : t * G * sizeof(double2);
}

#define GN_ACT(T, VEC, KERN)                                                                                       \
    switch (a.act) {                                                                                               \
    case ACT_RELU: hipLaunchKernelGGL((KERN<T, VEC, ACT_RELU>), grid, dim3(NT), lds, st, a); break;                \
    case ACT_SILU: hipLaunchKernelGGL((KERN<T, VEC, ACT_SILU>), grid, dim3(NT), lds, st, a); break;                \
    default: hipLaunchKernelGGL((KERN<T, VEC, ACT_NONE>), grid, dim3(NT), lds, st, a); break;                      \
    }

template <typename T, int VEC> int launch(const GnArgs &a, const Plan &p, bool backward, hipStream_t st)
{
    const int cl = p.gpb * a.cpg;
    const int rpb = NT / (cl / VEC);
    {
        const dim3 grid((unsigned)p.tiles, p.ncol);
        const size_t lds = (size_t)rpb * cl * (backward ? sizeof(float2) : sizeof(double2));
        if (backward) { GN_ACT(T, VEC, gn_back_sums) }
        else hipLaunchKernelGGL((gn_stats<T, VEC>), grid, dim3(NT), lds, st, a);
        const int rc = sis3d_check_launch();
        if (rc) return rc;
    }
    const dim3 grid((unsigned)p.tiles + (backward ? (a.C + 31) / 32 : 0), p.ncol);
    const size_t lds = 2 * p.gpb * sizeof(float);
    if (backward) { GN_ACT(T, VEC, gn_back_apply) }
    else { GN_ACT(T, VEC, gn_apply) }
    return sis3d_check_launch();
}

int dispatch(const GnArgs &a, const Plan &p, int dtype, bool backward, hipStream_t st)
{
    switch (dtype) {
    case SIS3D_F32: return p.vec > 1 ? launch<float, 4>(a, p, backward, st) : launch<float, 1>(a, p, backward, st);
    case SIS3D_BF16: return p.vec > 1 ? launch<__bf16, 8>(a, p, backward, st) : launch<__bf16, 1>(a, p, backward, st);
    default: return p.vec > 1 ? launch<_Float16, 8>(a, p, backward, st) : launch<_Float16, 1>(a, p, backward, st);
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
        const Plan p = make_plan(dtype, S, rows, ragged, C, G, wide);
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
    const Plan p = make_plan(dtype, S, rows, offsets != nullptr, C, G, aligned16(x) && aligned16(y) && strides * es % 16 == 0);
    if (p.rc) return p.rc;
    if (workspace_bytes < ws_bytes_of(p, C, G, false)) return SIS3D_EWORKSPACE;
    if (!workspace || !aligned16(workspace)) return SIS3D_EINVAL;
    GnArgs a{};
    a.x = x; a.y = y; a.w = weight; a.b = bias; a.mean = mean; a.rstd = rstd; a.off = offsets; a.rows = rows;
    a.x_n = x_sample; a.x_v = x_row; a.y_n = y_sample; a.y_v = y_row;
    a.S = S; a.C = C; a.G = G; a.cpg = C / G; a.gpb = p.gpb; a.T = p.T; a.tiles = (int)p.tiles; a.act = act; a.zero_tail = zero_tail; a.eps = eps;
    a.part = (double2 *)workspace;
    return dispatch(a, p, dtype, false, st);
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
    const Plan p = make_plan(dtype, S, rows, offsets != nullptr, C, G, aligned16(x) && aligned16(dy) && aligned16(dx) && strides * es % 16 == 0);
    if (p.rc) return p.rc;
    if (workspace_bytes < ws_bytes_of(p, C, G, true)) return SIS3D_EWORKSPACE;
    if (!workspace || !aligned16(workspace)) return SIS3D_EINVAL;
    GnArgs a{};
    a.x = x; a.dy = dy; a.y = dx; a.w = weight; a.b = bias; a.mean = (float *)mean; a.rstd = (float *)rstd; a.off = offsets; a.rows = rows;
    a.x_n = x_sample; a.x_v = x_row; a.d_n = dy_sample; a.d_v = dy_row; a.y_n = dx_sample; a.y_v = dx_row;
    a.S = S; a.C = C; a.G = G; a.cpg = C / G; a.gpb = p.gpb; a.T = p.T; a.tiles = (int)p.tiles; a.act = act; a.zero_tail = 1;
    a.part_c = (float2 *)workspace;
    a.part_g = a.part_c + (size_t)p.tiles * C;
    a.dw = dweight; a.db = dbias;
    return dispatch(a, p, dtype, true, st);
}
