// Rows of class scores: log probabilities of given labels with entropy and top alternatives, distillation from a teacher's kept
// logits, and the gradients of both with respect to the scores.
//
// Row l of K scores, temperature T (1 for the log probabilities):  L = log sum_j exp(l_j / T),  p_j = exp(l_j / T - L)
//     log probabilities:  logp = l_y - L,  H = L - sum_j p_j l_j,  the k largest l_j - L (equal scores: the lowest class first)
//     their gradient:     dl_j = a (1[j = y] - p_j) - e p_j (l_j - L + H)
//     distillation:       q = softmax of the kept teacher logits / T,  loss = T^2 sum_i q_i (log q_i - l_ci / T + L)
//     its gradient:       dl_j = g T (p_j - sum over i with c_i = j of q_i)
//
// All of it is bound by reading the scores once (and writing the gradient once).  Forward keeps a running maximum m and the sums
// s = sum e^((l - m) / T) and t = sum (l - m) e^((l - m) / T) per lane, rescaled when m grows, so a row is read once whatever its length;
// H = log s - t / s needs no second pass.  Everything is held in 32 bits.
// A row's L is kept as the pair (m, s): p = exp((l - m) / T) / s then has no rounding of a large L in it, and rows of the type's lowest
// value come out as what they are (all classes alike).
//
// Three forms, by the number of classes:
//   short rows       (contiguous: as long as 64 lanes would not have a vector each; class-strided: K <= 1024)  a lane, or up to 32 of them,
//                    takes a row; contiguous rows come through LDS in vectors, class-strided (planar) scores are read in place, with
//                    neighbouring rows on neighbouring lanes
//   longer rows      a wave or a workgroup streams a row with 16-byte loads from its first aligned element on; distillation of up to 4 KB
//                    by 16 lanes, so that four rows share what is done once a row
//   few long rows    the class axis is split over workgroups and a second launch joins their sums and alternatives
//
// Alternatives of a long row without sorting it or reading it twice: every lane knows the largest score it has seen.  The lanes of a wave
// are put into >= k groups; the smallest of the group maxima is a bound that at least k elements reach, and so is any number that k lanes'
// maxima reach.  It is taken after 1, 2, 4, ... batches of loads, and vectors with an element that reaches it are noted while they pass.
// Those that still reach the last bound, a few more than k, are read again and their elements at or above it ranked by counting, by
// (score, class).
//
// Measured (kernel alone):
//   tile_forward / tile_backward   55296 x 41 fp32 planar, one alternative: 6.8 / 7.9 us.  200 x 19 fp32: 5 / 5 us, the loads' way and back
//   four_distill                   40000 x 1203 fp16, 8 entries: 21.6 us (4.6 TB/s)
//   long_backward by waves         the same: 44.9 us (4.4 TB/s)
//   long_forward by workgroups     4096 x 32768 bf16, 32 entries: 57 us (4.7 TB/s), backward 86 (6.3: what the L2s and the memory-side cache
//                                  keep of the scores).  2000 x 20011 bf16: 21 us without alternatives, 31 with eight
//   split_forward, split_join      3 x 65536 fp32, five alternatives: 8.4 + 4.0 us
// What bounds the 16-bit forms next to memory is arithmetic: an exponential is four instructions' time, and with conversion, maximum and
// the sums an element takes about ten.
#include "elem.h"

namespace {

constexpr int TOP_MAX = 32, KEPT_MAX = 128, K_STRIDED = 1024, K_WAVE = 4096;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f, LOWEST = -3.402823466e38f;
constexpr int LP = 0, KD = 1;

struct RowArgs {
    const void *score;
    void *dscore;
    int64_t s_n, s_v, s_c, d_n, d_v, d_c;      // element strides: outer index, row inside it, class
    int64_t V, R;                              // row r = n * V + v
    int K, N;
    const int32_t *num;                        // live rows, or NULL
    const int64_t *labels;
    int top;
    float *logp, *entropy, *top_logp;
    float2 *norm;                              // (m, s) of each row
    int64_t *top_class;
    const float *kept;                         // (R, nk)
    const int64_t *cls;
    int nk;
    float tau, inv, inv_lo, c2;                // T, 1 / T in two parts, log2(e) / T
    float *loss;
    const float *g1, *g2;                      // gradients: of logp and entropy, or of the loss
    const float2 *norm_in;
    const float *entropy_in;
    int planar, parts;
    int g_log, sk, chunk;                      // tiles: lanes per row, floats of a row in LDS, classes of a lane
    uint32_t per4;                             // 2^32 / (K / 4), rounded up
    float *part;                               // [R * parts][4]
    uint64_t *part_keys;                       // [R * parts][top]
};

__device__ inline int64_t live_rows(const RowArgs &a)
{
    if (!a.num) return a.R;
    const int64_t n = a.num[0];
    return n < 0 ? 0 : (n < a.R ? n : a.R);
}
__device__ inline int64_t row_at(const RowArgs &a, int64_t r, int64_t sn, int64_t sv)
{
    if (a.N == 1) return r * sv;
    const int64_t n = r / a.V;
    return n * sn + (r - n * a.V) * sv;
}

__device__ inline float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ inline float log_(float x) { return LN2 * __builtin_amdgcn_logf(x); }        // of sums: normal numbers
// a product that is rounded by itself and not fused with what is done with it
__device__ inline float mul_rounded(float a, float b)
{
#pragma clang fp contract(off)
    return a * b;
}
__device__ inline float rcp_(float x) { return __builtin_amdgcn_rcpf(x); }

// a score as a whole number of the same order; -0 counts as 0, NaN as -inf
__device__ inline uint32_t ordered(float v)
{
    const uint32_t b = __float_as_uint(fmaxf(v, -INFINITY) + 0.f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ inline float score_of(uint32_t o) { return __uint_as_float(o ^ ((o & 0x80000000u) ? 0x80000000u : 0xffffffffu)); }
// (score, class) as one number: larger score first, then the lower class
__device__ inline uint64_t key_of(float v, int c) { return ((uint64_t)ordered(v) << 32) | (uint32_t)~c; }
__device__ inline int key_class(uint64_t k) { return (int)~(uint32_t)k; }
__device__ inline float key_score(uint64_t k) { return score_of((uint32_t)(k >> 32)); }
__device__ inline uint64_t shfl_xor64(uint64_t v, int o) { return (uint64_t)__shfl_xor((unsigned long long)v, o); }
__device__ inline uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ inline uint64_t min64(uint64_t a, uint64_t b) { return a < b ? a : b; }

// maximum of three in one instruction.  Written out because the compiler puts a canonicalising instruction in front of every operand that
// it has only seen as bits; what that guards against (a signalling NaN) would at worst cost a NaN row the order of its alternatives.
__device__ inline float max3_(float a, float b, float c)
{
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
template <int N> __device__ inline float max_of(const float (&x)[N])
{
    float m = x[0];
#pragma unroll
    for (int i = 1; i + 1 < N; i += 2) m = max3_(m, x[i], x[i + 1]);
    return N % 2 ? m : fmaxf(m, x[N - 1]);
}

// sum over a wave in the vector pipe (row shifts by 1, 2, 4, 8, then the rows' last lanes broadcast): every lane gets it
template <int CTRL, int ROWS> __device__ inline float dpp(float old, float v)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(old), __float_as_int(v), CTRL, ROWS, 0xf, false));
}
__device__ inline float last_lane(float v) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63)); }
__device__ inline float wave_sum(float v)
{
    v += dpp<0x111, 0xf>(0.f, v);
    v += dpp<0x112, 0xf>(0.f, v);
    v += dpp<0x114, 0xf>(0.f, v);
    v += dpp<0x118, 0xf>(0.f, v);
    v += dpp<0x142, 0xa>(0.f, v);
    v += dpp<0x143, 0xc>(0.f, v);
    return last_lane(v);
}
// one step of a maximum over the 16 lanes of a row, rotated by N: every lane takes part, so one instruction does it (written out for the
// reason given at max3_; the waits are those between a vector result and its use across lanes)
template <int N> __device__ inline float max_ror(float v)
{
    float r;
    asm("s_nop 1\n\tv_max_f32_dpp %0, %1, %1 row_ror:%2 row_mask:0xf bank_mask:0xf\n\ts_nop 1" : "=v"(r) : "v"(v), "n"(N));
    return r;
}
__device__ inline float lane_at(float v, int i) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), i)); }
__device__ inline float wave_max(float v)
{
    v = max_ror<8>(max_ror<4>(max_ror<2>(max_ror<1>(v))));
    return max3_(lane_at(v, 0), lane_at(v, 16), fmaxf(lane_at(v, 32), lane_at(v, 48)));
}
__device__ inline float wave_min(float v) { return -wave_max(-v); }
// the same over 16 lanes: rotated and added, every lane gets the same bits
__device__ inline float row_sum(float v)
{
    v += dpp<0x128, 0xf>(0.f, v);
    v += dpp<0x124, 0xf>(0.f, v);
    v += dpp<0x122, 0xf>(0.f, v);
    return v + dpp<0x121, 0xf>(0.f, v);
}
__device__ inline float row_max(float v) { return max_ror<1>(max_ror<2>(max_ror<4>(max_ror<8>(v)))); }
// of the L lanes that a row has
template <int L> __device__ inline float lanes_sum(float v) { return L == 16 ? row_sum(v) : wave_sum(v); }
template <int L> __device__ inline float lanes_max(float v) { return L == 16 ? row_max(v) : wave_max(v); }
template <int L> __device__ inline bool lanes_any(bool v)
{
    const uint64_t mask = __ballot(v);
    return L == 16 ? (mask >> (threadIdx.x & 48) & 0xffff) != 0 : mask != 0;
}
// the largest of the 2, 4, 8 or 16 neighbouring lanes that v's lane is one of: quads by permutation, then mirrored halves and rows
__device__ inline float neighbours_max(float v, int lanes)
{
    v = fmaxf(v, dpp<0xb1, 0xf>(v, v));
    if (lanes >= 4) v = fmaxf(v, dpp<0x4e, 0xf>(v, v));
    if (lanes >= 8) v = fmaxf(v, dpp<0x141, 0xf>(v, v));
    if (lanes >= 16) v = fmaxf(v, dpp<0x140, 0xf>(v, v));
    return v;
}

// running sums of a softmax: m in score units (never below LOWEST), s = sum 2^x and, where an entropy is wanted, t = sum x 2^x,
// x = (l - m) c2
template <bool ENT> struct Soft {
    float m, s, t;
    __device__ void init() { m = LOWEST; s = t = 0.f; }
    __device__ void raise(float to, float c2)
    {
        const float x = (m - to) * c2, f = exp2_(x);
        if constexpr (ENT) t = f * fmaf(fmaxf(x, -200.f), s, t);          // -200: 2^x is 0 from there on, and 0 * inf is not wanted
        s *= f;
        m = to;
    }
    __device__ void add(float l, float c2)             // l <= m
    {
        const float x = (l - m) * c2, e = exp2_(x);
        s += e;
        if constexpr (ENT) t = fmaf(fmaxf(x, -200.f), e, t);
    }
    __device__ void join(float m2, float s2, float t2, float c2)
    {
        Soft o{m2, s2, t2};
        const float to = fmaxf(m, m2);
        raise(to, c2);
        o.raise(to, c2);
        s += o.s;
        t += o.t;
    }
    __device__ void join_wave(float c2)
    {
        raise(wave_max(m), c2);
        s = wave_sum(s);
        if constexpr (ENT) t = wave_sum(t);
    }
    __device__ float log_s() const { return s == 0.f ? -INFINITY : log_(s); }      // s = 0: a row of nothing but -inf
    __device__ float entropy() const { return s == 0.f ? 0.f : log_(s) - LN2 * (t / s); }
};

// The same sums for one lane of a long row, x = l c2 - M in one fused operation (its rounding is that of x; one of M would be common to all
// classes and cancels).  M, in units of x, need only be near the largest: it follows it when it is exceeded by more than 2.  It starts at
// -NEAR: scores that far below 0 (masks) add 0.  Where the largest lies above NEAR the rounding of M itself is no longer small in x; where it
// lies below -NEAR, which M does not follow, the largest term may be a number and smaller ones that count beside it may not.  Such rows,
// masked ones and those that are not finite end in a sum of 0, inf or NaN and are taken again class by class.
constexpr float NEAR = 4194304.f;          // 2^22: M is rounded by at most 1/4
__device__ inline bool sums_hold(float m, float c2) { return fabsf(mul_rounded(m, c2)) < NEAR; }        // m: a row's largest score
template <bool ENT> struct Lane {
    float M, s, t;
    __device__ void init() { M = -NEAR; s = t = 0.f; }
    __device__ void raise(float to)
    {
        const float x = M - to, f = exp2_(x);
        if constexpr (ENT) t = f * fmaf(fmaxf(x, -200.f), s, t);
        s *= f;
        M = to;
    }
    __device__ void follow(float top, float c2)
    {
        const float to = mul_rounded(top, c2);
        if (to > M + 2.f) raise(to);
    }
    __device__ void add(float l, float c2)
    {
        const float x = fmaf(l, c2, -M), e = exp2_(x);
        s += e;
        if constexpr (ENT) t = fmaf(fmaxf(x, -200.f), e, t);
    }
    // L lanes, relative to their largest score m: divided by m's own term, so that a row of one class has s = 1 exactly
    template <int L> __device__ Soft<ENT> join(float largest, float c2)
    {
        const float m = fmaxf(lanes_max<L>(largest), LOWEST);
        raise(fmaxf(mul_rounded(m, c2), -NEAR));
        s = lanes_sum<L>(s);
        if constexpr (ENT) t = lanes_sum<L>(t);
        if (s == 0.f) return Soft<ENT>{LOWEST, 0.f, 0.f};              // nothing but masks here
        const float x = fmaf(m, c2, -M), e = exp2_(x);
        return Soft<ENT>{m, sums_hold(m, c2) ? s / e : NAN, ENT ? fmaf(-x, s, t) / e : 0.f};
    }
};

// (m, log s) of a row, for the few log probabilities that it reports
struct Norm { float m, ls; };

// l / T - L, -inf where L is
__device__ inline float log_p(float l, Norm n, float inv, float inv_lo)
{
    const float d = l - n.m;
    return n.ls == -INFINITY ? -INFINITY : fmaf(d, inv, fmaf(fmaxf(d, LOWEST), inv_lo, -n.ls));
}

__device__ inline float label_logp(const RowArgs &a, int64_t y, float ly, Norm n)
{
    return y < 0 ? 0.f : (y >= a.K ? NAN : log_p(ly, n, 1.f, 0.f));
}

// A row in the backward direction, prepared so that a class costs one exponential and a few operations:
//     log probabilities   -p (ga + ge (log p + H)) = 2^x (k1 max(x, -288) + k0),  x = (l - m) log2(e)
//     distillation        ga p = 2^x k0,  x = (l - m) log2(e) / T
// (p is 0 from x = -288 on, and 0 * inf is not wanted; a row of nothing but -inf has 1 / s = 0).  `near` takes x from one fused operation
// with M = m c2 rounded, whose rounding is taken out of k0 and k1 beforehand; `exact` serves rows where that is not small.
template <int MODE> struct Back {
    float m, ga, k0, k1, c2, M, n0, n1;
    bool in_range;
    __device__ void finish()
    {
        M = mul_rounded(m, c2);
        in_range = fabsf(M) < NEAR;
        const float off = fmaf(m, c2, -M), f = exp2_(-off);        // l c2 - M = x + off
        n1 = MODE == LP ? k1 * f : 0.f;
        n0 = MODE == LP ? f * fmaf(-k1, off, k0) : f * k0;
    }
    __device__ void scores(float2 norm, float h, float ga_, float ge)
    {
        const float is = norm.y == 0.f ? 0.f : 1.f / norm.y;
        m = norm.x;
        ga = ga_;
        k1 = -is * ge * LN2;
        k0 = -is * (ga + ge * (h - (norm.y == 0.f ? 0.f : log_(norm.y))));
        c2 = LOG2E;
        finish();
    }
    __device__ void loss(float2 norm, float ga_, float c2_)
    {
        m = norm.x;
        ga = ga_;
        k0 = norm.y == 0.f ? 0.f : ga / norm.y;
        c2 = c2_;
        finish();
    }
    // without the label's or the teacher's share
    __device__ float exact(float l) const
    {
        const float x = (l - m) * c2, e = exp2_(x);
        if constexpr (MODE == LP) return e * fmaf(k1, fmaxf(x, -288.f), k0);
        else return e * k0;
    }
    __device__ float near(float l) const
    {
        const float x = fmaf(l, c2, -M), e = exp2_(x);
        if constexpr (MODE == LP) return e * fmaf(n1, fmaxf(x, -288.f), n0);
        else return e * n0;
    }
};

// a teacher's entry: 0 = absent, 1 = present, 2 = no such class
__device__ inline int entry(const RowArgs &a, int64_t c) { return c < 0 ? 0 : (c >= a.K ? 2 : 1); }

// --------------------------------------------------------------------------- the lanes that share a short row --
struct Group {
    int64_t r, at;                             // row; the row that may be read (0 where r is none: such lanes take part in the shuffles only)
    int sub, lpr, step;                        // lane of the row, lanes per row, distance of neighbouring row lanes
    bool in, live;                             // a row of the call; a live one
};
__device__ inline float group_sum(float v, const Group &g)
{
    for (int o = g.lpr >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o * g.step);
    return v;
}
__device__ inline float group_max(float v, const Group &g)
{
    for (int o = g.lpr >> 1; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o * g.step));
    return v;
}

// A row's kept entries, shared by the lanes of a group: entry i is lane i % lpr's
struct Teacher { float m, s; bool any, bad; };     // largest kept logit, sum of exponentials; an entry that counts, one that cannot
__device__ inline Teacher group_teacher(const RowArgs &a, const Group &g)
{
    Teacher t{-INFINITY, 0.f, false, false};
    const float *kept = a.kept + g.at * a.nk;
    const int64_t *cls = a.cls + g.at * a.nk;
    float bad = 0.f;
    for (int i = g.sub; i < a.nk; i += g.lpr) {
        const int e = entry(a, cls[i]);
        if (e) t.m = fmaxf(t.m, kept[i]);
        if (e == 2 || (e && kept[i] != kept[i])) bad = 1.f;
    }
    t.m = group_max(t.m, g);
    t.bad = group_max(bad, g) > 0.f;
    t.any = t.m > -INFINITY;
    if (t.any)
        for (int i = g.sub; i < a.nk; i += g.lpr)
            if (entry(a, cls[i])) t.s += exp2_((kept[i] - t.m) * a.c2);
    t.s = group_sum(t.s, g);
    return t;
}
// Every entry of a row, in their order, to all lanes of the group: f(number, class or -1, q).  Each is read and its q made by one lane.
template <typename F> __device__ inline void each_entry(const RowArgs &a, const Group &g, const Teacher &t, F f)
{
    const int first = g.step == 1 ? (threadIdx.x & 63) - g.sub : (threadIdx.x & (g.step - 1));      // the wave's lane with sub = 0
    const float is = t.any ? rcp_(t.s) : 0.f;
    for (int i0 = 0; i0 < a.nk; i0 += g.lpr) {
        int c = -1;
        float q = 0.f;
        if (i0 + g.sub < a.nk) {
            const int64_t k = a.cls[g.at * a.nk + i0 + g.sub];
            if (entry(a, k) == 1) {
                c = (int)k;
                q = exp2_((a.kept[g.at * a.nk + i0 + g.sub] - t.m) * a.c2) * is;
            }
        }
        for (int s = 0; s < g.lpr && i0 + s < a.nk; ++s) f(i0 + s, __shfl(c, first + s * g.step), __shfl(q, first + s * g.step));
    }
}
// an entry's share of the loss; q log q is 0 at q = 0
__device__ inline float entry_loss(const RowArgs &a, const Teacher &t, float ls, float kept, float l, Norm norm)
{
    const float x = (kept - t.m) * a.c2, q = exp2_(x) * rcp_(t.s);
    return q != 0.f ? q * (x * LN2 - ls - log_p(l, norm, a.inv, a.inv_lo)) : 0.f;
}

template <int W> __device__ inline int team_of() { return W == 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0; }
template <int W> __device__ inline void team_sync()
{
    if constexpr (W == 1) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        __builtin_amdgcn_wave_barrier();
    } else __syncthreads();
}

// ------------------------------------------------------------------------- short rows: a lane, or a few, to a row --
// A workgroup has 256 / G rows.  Dense rows are one run of memory: it is read by vectors into LDS, as floats, and G neighbouring lanes take
// a row from there, a stretch of classes each -- no shuffle within a stretch, and with G = 1 none at all.  Scores in any other layout are
// read in place, neighbouring lanes having neighbouring rows.  The gradient of a dense tile is made in LDS and leaves as it came.
// LDS rows are K floats apart where K is no multiple of 4 (banks differ from row to row by themselves), else an odd number of fours.
struct TileRow {
    Group g;
    int row, lo, n;                            // row of the tile; this lane's classes are lo .. lo + n - 1
};
constexpr int IN_PLACE = 0, BY_ONE = 1, BY_FOUR = 2;

// (score, class) of a short row as one number, a larger one for a larger score and then for a lower class; 0 is none.  Scores of 16 bits,
// as floats, are 0 in their last 13 bits and more, where the class (below 1024) goes; 32-bit scores take the mantissa of a double, whose maximum
// and minimum are one instruction each.
static_assert(K_STRIDED <= 1024, "10 bits of a key are the class");
template <typename T> struct Rank {
    using Key = uint32_t;
    static __device__ Key key(float v, int c) { return (ordered(v) & ~1023u) | (uint32_t)(1023 - c); }
    static __device__ int cls(Key k) { return 1023 - (int)(k & 1023u); }
    static __device__ float score(Key k) { return __uint_as_float(__float_as_uint(score_of(k)) & ~1023u); }
    static __device__ Key larger(Key a, Key b) { return a > b ? a : b; }
    template <int N> static __device__ void insert(Key (&t)[N], Key k)       // t descending: the middle of a place, the one above it and k
    {
#pragma unroll
        for (int i = N - 1; i > 0; --i) t[i] = larger(t[i], k < t[i - 1] ? k : t[i - 1]);
        t[0] = larger(t[0], k);
    }
    static __device__ Key other(Key k, int o) { return __shfl_xor(k, o); }
};
template <> struct Rank<float> {
    using Key = double;
    static __device__ Key key(float v, int c)
    {
        const uint32_t o = ordered(v);
        return __hiloint2double((int)(0x3ff00000u | o >> 22), (int)(o << 10 | (uint32_t)(1023 - c)));
    }
    static __device__ int cls(Key k) { return 1023 - (__double2loint(k) & 1023); }
    static __device__ float score(Key k) { return score_of((uint32_t)__double2hiint(k) << 22 | (uint32_t)__double2loint(k) >> 10); }
    static __device__ Key larger(Key a, Key b) { return fmax(a, b); }
    template <int N> static __device__ void insert(Key (&t)[N], Key k)
    {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const Key a = fmax(t[i], k);
            k = fmin(t[i], k);
            t[i] = a;
        }
    }
    static __device__ Key other(Key k, int o) { return __hiloint2double(__shfl_xor(__double2hiint(k), o), __shfl_xor(__double2loint(k), o)); }
};

template <int HOW> __device__ inline TileRow tile_row(const RowArgs &a)
{
    TileRow t;
    const int G = 1 << a.g_log, rpw_log = 6 - a.g_log, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    t.g.lpr = G;
    if (HOW == IN_PLACE && a.planar) {
        t.row = (w << rpw_log) + (lane & ((1 << rpw_log) - 1));
        t.g.sub = lane >> rpw_log;
        t.g.step = 1 << rpw_log;
    } else {
        t.row = threadIdx.x >> a.g_log;
        t.g.sub = lane & (G - 1);
        t.g.step = 1;
    }
    t.g.r = (int64_t)blockIdx.x * (256 >> a.g_log) + t.row;
    t.g.in = t.g.r < a.R;
    t.g.live = t.g.in && t.g.r < live_rows(a);
    t.g.at = t.g.live ? t.g.r : 0;
    t.lo = t.g.sub * a.chunk;
    t.n = t.g.live ? max(0, min(a.chunk, a.K - t.lo)) : 0;
    return t;
}

// rows of the tile that are live, times K, between memory and LDS
template <typename T, int HOW, bool IN> __device__ inline void move_tile(const RowArgs &a, T *mem, float *lds)
{
    constexpr int VEC = 16 / sizeof(T);
    const int rb = 256 >> a.g_log;
    const int64_t r0 = (int64_t)blockIdx.x * rb, left = (IN ? live_rows(a) : a.R) - r0;
    const int total = left <= 0 ? 0 : (int)(left < rb ? left : rb) * a.K;
    mem += r0 * a.K;
    auto place = [&](int i) {                      // of the float with number i, a multiple of 4
        if constexpr (HOW == BY_ONE) return i;
        const int row = __umulhi((uint32_t)i >> 2, a.per4);
        return i + row * (a.sk - a.K);
    };
    for (int i = threadIdx.x * VEC; i < total; i += 256 * VEC) {
        float x[VEC];
        if (i + VEC <= total) {
            if constexpr (IN) {
                sis3d_unpack<T, VEC>(sis3d_load_once<T, VEC>(mem + i), x);
#pragma unroll
                for (int j = 0; j < VEC; j += 4) *(float4 *)(lds + place(i + j)) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; j += 4) *(float4 *)(x + j) = *(const float4 *)(lds + place(i + j));
                sis3d_store<T, VEC>(mem + i, x);
            }
        } else
            for (int j = 0; i + j < total; ++j) {
                const int at = place((i + j) & ~3) + ((i + j) & 3);
                if constexpr (IN) lds[at] = sis3d_f32(mem[i + j]);
                else mem[i + j] = sis3d_from_f32<T>(lds[at]);
            }
    }
    __syncthreads();
}

// A lane's classes, eight at a time: f(first class, x[8], how many of them there are)
template <typename T, int HOW, typename F> __device__ inline void each_eight(const RowArgs &a, const TileRow &t, const T *p, const float *row, F f)
{
    const int all = a.K - (((1 << a.g_log) - 1) * a.chunk);        // classes that every lane of a row has
    for (int i = 0; i < a.chunk; i += 8) {
        float x[8];
        const bool whole = i + 8 <= all;
        if constexpr (HOW == IN_PLACE) {
            if (t.n > i) {
                const T *q = p + (t.lo + i) * a.s_c;
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = sis3d_f32(q[min(j, t.n - 1 - i) * a.s_c]);
            }
        } else if constexpr (HOW == BY_FOUR) {
#pragma unroll
            for (int j = 0; j < 8; j += 4) *(float4 *)(x + j) = *(const float4 *)(row + t.lo + i + j);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = row[t.lo + i + j];
        }
        if (!whole || !t.g.live)
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = i + j < t.n ? x[j] : -INFINITY;
        f(i, x);
    }
}

template <typename T, int MODE, int HOW, int TK> __global__ __launch_bounds__(256) void tile_forward(RowArgs a)
{
    extern __shared__ float4 lds4[];
    float *lds = (float *)lds4;
    const TileRow t = tile_row<HOW>(a);
    const Group &g = t.g;
    const T *p = (const T *)a.score + (HOW == IN_PLACE ? row_at(a, g.at, a.s_n, a.s_v) : 0);
    const float *row = lds + t.row * a.sk;
    if constexpr (HOW != IN_PLACE) move_tile<T, HOW, true>(a, (T *)a.score, lds);
    auto score = [&](int64_t c) { return HOW == IN_PLACE ? sis3d_f32(p[c * a.s_c]) : row[c]; };
    Lane<MODE == LP> ln;
    ln.init();
    float best = -INFINITY;
    using Key = typename Rank<T>::Key;
    Key first[TK ? TK : 1];                            // this lane's best ones
#pragma unroll
    for (int k = 0; k < TK; ++k) first[k] = 0;
    each_eight<T, HOW>(a, t, p, row, [&](int i, const float (&x)[8]) {
        const float top = max_of(x);
        if constexpr (TK == 1)
            if (top > best) {
                int at = 0;
#pragma unroll
                for (int j = 7; j > 0; --j) at = x[j] == top ? j : at;
                at = x[0] == top ? 0 : at;
                first[0] = Rank<T>::key(top, t.lo + i + at);
            }
        best = fmaxf(best, top);
        ln.follow(top, a.c2);
#pragma unroll
        for (int j = 0; j < 8; ++j) ln.add(x[j], a.c2);
        if constexpr (TK > 1)
#pragma unroll
            for (int j = 0; j < 8; ++j) Rank<T>::insert(first, i + j < t.n ? Rank<T>::key(x[j], t.lo + i + j) : (Key)0);
    });
    if (TK == 1 && t.n > 0 && best == -INFINITY) first[0] = Rank<T>::key(best, t.lo);         // nothing was more than -inf
    // the lanes of a row, relative to its largest score, which has s = 1 if it is the only one
    Soft<MODE == LP> so;
    so.m = fmaxf(group_max(best, g), LOWEST);
    ln.raise(fmaxf(mul_rounded(so.m, a.c2), -NEAR));
    const float x0 = fmaf(so.m, a.c2, -ln.M), e0 = exp2_(x0);
    so.s = group_sum(ln.s, g);
    so.t = MODE == LP ? group_sum(ln.t, g) : 0.f;
    so.t = fmaf(-x0, so.s, so.t) / e0;
    so.s = so.s / e0;
    if (!(so.s > 0.f && so.s < INFINITY && sums_hold(so.m, a.c2))) {
        so.init();
        for (int i = 0; i < t.n; ++i) so.m = fmaxf(so.m, score(t.lo + i));
        so.m = group_max(so.m, g);
        for (int i = 0; i < t.n; ++i) so.add(score(t.lo + i), a.c2);
        so.s = group_sum(so.s, g);
        so.t = group_sum(so.t, g);
    }
    const Norm norm{so.m, so.log_s()};
    if constexpr (MODE == KD) {
        const Teacher te = group_teacher(a, g);
        float loss = 0.f;
        if (te.any && g.live) {
            const float ls = log_(te.s);
            for (int i = g.sub; i < a.nk; i += g.lpr) {
                const int64_t c = a.cls[g.at * a.nk + i];
                if (entry(a, c) == 1) loss += entry_loss(a, te, ls, a.kept[g.at * a.nk + i], score(c), norm);
            }
        }
        loss = a.tau * a.tau * group_sum(loss, g);
        if (g.sub == 0 && g.in) {
            a.loss[g.r] = !g.live ? 0.f : (te.bad ? NAN : loss);
            a.norm[g.r] = g.live ? make_float2(so.m, so.s) : make_float2(0.f, 0.f);
        }
        return;
    }
    if (g.sub == 0 && g.in) {
        const int64_t y = g.live ? a.labels[g.at] : -1;
        a.logp[g.r] = label_logp(a, y, y >= 0 && y < a.K ? score(y) : 0.f, norm);
        a.entropy[g.r] = g.live ? so.entropy() : 0.f;
        a.norm[g.r] = g.live ? make_float2(so.m, so.s) : make_float2(0.f, 0.f);
    }
    if constexpr (TK > 0)
        for (int i = 0; i < a.top; ++i) {
            // the best of the lanes' first ones; its lane goes on to the next
            Key k = first[0];
            for (int o = g.lpr >> 1; o > 0; o >>= 1) k = Rank<T>::larger(k, Rank<T>::other(k, o * g.step));
            const bool mine = k == first[0];
#pragma unroll
            for (int j = 0; j + 1 < TK; ++j) first[j] = mine ? first[j + 1] : first[j];
            first[TK - 1] = mine ? (Key)0 : first[TK - 1];
            if (g.sub == 0 && g.in) {
                a.top_class[g.r * a.top + i] = g.live ? Rank<T>::cls(k) : 0;
                a.top_logp[g.r * a.top + i] = g.live ? log_p(Rank<T>::score(k), norm, 1.f, 0.f) : 0.f;
            }
        }
}

template <typename T, int MODE, int HOW> __global__ __launch_bounds__(256) void tile_backward(RowArgs a)
{
    extern __shared__ float4 lds4[];
    float *lds = (float *)lds4;
    const TileRow t = tile_row<HOW>(a);
    const Group &g = t.g;
    const T *p = (const T *)a.score + (HOW == IN_PLACE ? row_at(a, g.at, a.s_n, a.s_v) : 0);
    T *d = (T *)a.dscore + (HOW == IN_PLACE ? row_at(a, g.in ? g.r : 0, a.d_n, a.d_v) : 0);
    float *row = lds + t.row * a.sk;
    if constexpr (HOW != IN_PLACE) move_tile<T, HOW, true>(a, (T *)a.score, lds);
    Back<MODE> k;
    Teacher te;
    int y = -1;
    if constexpr (MODE == LP) {
        const int64_t label = a.labels[g.at];
        k.scores(a.norm_in[g.at], a.entropy_in[g.at], label < 0 ? 0.f : (label >= a.K ? NAN : a.g1[g.at]), a.g2 ? a.g2[g.at] : 0.f);
        if (g.live && label >= 0 && label < a.K) y = (int)label;
    } else {
        te = group_teacher(a, g);
        k.loss(a.norm_in[g.at], te.bad ? NAN : (te.any ? a.g1[g.at] * a.tau : 0.f), a.c2);
    }
    if constexpr (HOW == IN_PLACE) {
        auto grad = [&](int c) {
            const float l = sis3d_f32(p[c * a.s_c]);
            return k.in_range ? k.near(l) : k.exact(l);
        };
        if (g.live)
            each_eight<T, HOW>(a, t, p, row, [&](int i, const float (&x)[8]) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (i + j < t.n) d[(t.lo + i + j) * a.d_c] = sis3d_from_f32<T>(k.in_range ? k.near(x[j]) : k.exact(x[j]));
            });
        else if (g.in)
            for (int i = 0; i < max(0, min(a.chunk, a.K - t.lo)); ++i) d[(t.lo + i) * a.d_c] = sis3d_from_f32<T>(0.f);
        // the label's class, or the kept ones, again by the lane that has written it
        if constexpr (MODE == LP) {
            if (y >= t.lo && y < t.lo + t.n) d[y * a.d_c] = sis3d_from_f32<T>(grad(y) + k.ga);
        } else {
            // a class that may have been kept before is written once more, with the sum so far; `seen` is of classes modulo 64
            uint64_t seen = 0;
            each_entry(a, g, te, [&](int i, int c, float q) {
                if (!te.any || c < t.lo || c >= t.lo + t.n) return;
                const uint64_t bit = 1ull << (c & 63);
                if (seen & bit)
                    for (int j = i - 1; j >= 0; --j)
                        if (a.cls[g.at * a.nk + j] == c) q += exp2_((a.kept[g.at * a.nk + j] - te.m) * a.c2) * rcp_(te.s);
                seen |= bit;
                d[c * a.d_c] = sis3d_from_f32<T>(grad(c) - k.ga * q);
            });
        }
    } else {
        if (g.live) {
            // the lane's stretch in place, then the label's or the teacher's share by the lane that has that class
            float *mine = row + t.lo;
            if (k.in_range) {
#pragma unroll 4
                for (int i = 0; i < t.n; ++i) mine[i] = k.near(mine[i]);
            } else
                for (int i = 0; i < t.n; ++i) mine[i] = k.exact(mine[i]);
        } else if (g.in)
            for (int i = 0; i < max(0, min(a.chunk, a.K - t.lo)); ++i) row[t.lo + i] = 0.f;
        if constexpr (MODE == LP) {
            if (y >= t.lo && y < t.lo + t.n) row[y] += k.ga;
        } else
            each_entry(a, g, te, [&](int, int c, float q) {
                if (te.any && c >= t.lo && c < t.lo + t.n) row[c] -= k.ga * q;
            });
        __syncthreads();
        move_tile<T, HOW, false>(a, (T *)a.dscore, lds);
    }
}

// ---------------------------------------------------------------------------- long rows, classes contiguous --
// A team of W waves (1: four teams to a workgroup; 4: the workgroup) has a row or a part of one.
// [k0, k1) of a row: elements in front of the first 16-byte boundary and behind the last whole vector are taken one by one
template <typename T> struct Span {
    static constexpr int VEC = 16 / sizeof(T);
    const T *row, *body;
    int k0, head, nvec, tail;
    __device__ Span(const T *row_, int k0_, int k1) : row(row_), k0(k0_)
    {
        const int n = k1 - k0;
        head = (int)((16 - ((uintptr_t)(row + k0) & 15)) & 15) / (int)sizeof(T);
        if (head > n) head = n;
        nvec = (n - head) / VEC;
        tail = n - head - nvec * VEC;
        body = row + k0 + head;
    }
    __device__ int first_class(int v) const { return k0 + head + v * VEC; }
    // the i-th of the single elements, i < head + tail
    __device__ int edge_class(int i) const { return i < head ? k0 + i : k0 + head + nvec * VEC + (i - head); }
    __device__ int edges() const { return head + tail; }
};

// A lane's vectors lane, lane + NL, ... of a span, UL at a time and the next UL on their way while these are worked on; the first are
// asked for when the object is made, so that a row's other loads travel with them.  f(count, v, vectors): `count` of them from v on, all
// there but perhaps the last one of the last batch.
// UL: 4 where a workgroup has a row, 2 where fewer lanes have one (40000 x 1203 fp16, distillation forward, a wave to a row: 39.4 us with 4,
// 36.5 with 2; 16 lanes to a row: 27.6 with 4, 24.1 with 2)
constexpr int loads_of(int NL) { return NL > 64 ? 4 : 2; }
template <int N> struct Count { static constexpr int value = N; };
template <typename T, int NL, bool ONCE> struct Stream {
    static constexpr int VEC = 16 / sizeof(T), UL = loads_of(NL);
    const Span<T> &sp;
    const int lane, steps;                                     // steps of NL vectors, the same for all lanes of a wave
    SisVec<T, VEC> raw[UL];
    __device__ Stream(const Span<T> &s, int l) : Stream(s, l, s.nvec) {}
    __device__ Stream(const Span<T> &s, int l, int vectors) : sp(s), lane(l), steps((vectors + NL - 1) / NL) { load(raw, l); }
    __device__ void load(SisVec<T, VEC> (&r)[UL], int v) const
    {
#pragma unroll
        for (int u = 0; u < UL; ++u) r[u] = sis3d_raw<T, VEC, ONCE>(sp.body + (int64_t)min(v + u * NL, sp.nvec - 1) * VEC);
    }
    template <typename F> __device__ void each(F f)
    {
        int v = lane, left = steps;
        SisVec<T, VEC> next[UL];
        while (left > UL) {
            load(next, v + UL * NL);
            f(Count<UL>(), v, raw);
            left -= UL, v += UL * NL;
            if (left <= UL) { last(left, v, next, f); return; }
            load(raw, v + UL * NL);
            f(Count<UL>(), v, next);
            left -= UL, v += UL * NL;
        }
        last(left, v, raw, f);
    }
    // the same with less code (one batch and one vector of it), for work that takes more instructions than a cache of them holds ten times
    template <typename F> __device__ void each_compact(F f)
    {
        int v = lane, left = steps;
        for (; left > UL; left -= UL, v += UL * NL) {
            SisVec<T, VEC> next[UL];
            load(next, v + UL * NL);
            f(Count<UL>(), v, raw);
#pragma unroll
            for (int u = 0; u < UL; ++u) raw[u] = next[u];
        }
#pragma unroll 1
        for (; left > 0; --left, v += NL) {
            f(Count<1>(), v, raw);
#pragma unroll
            for (int u = 0; u + 1 < UL; ++u) raw[u] = raw[u + 1];
        }
    }
    template <typename F> __device__ void last(int left, int v, const SisVec<T, VEC> (&r)[UL], F f)
    {
        if (left == 1) f(Count<1>(), v, r);
        else if (left == 2) f(Count<2>(), v, r);
        if constexpr (UL > 2) {
            if (left == 3) f(Count<3>(), v, r);
            else if (left == 4) f(Count<4>(), v, r);
        }
    }
};

template <typename T, int W, int MODE, bool TOP> struct Long {
    static constexpr int NL = 64 * W, ROOM = 256, VEC = 16 / sizeof(T), UL = loads_of(NL);
    struct Vec { float m; int v; };            // a vector and its largest score
    struct Shared {
        uint64_t cand[TOP ? W : 1][TOP ? ROOM : 1], bound[W];       // a wave's elements
        Vec vecs[TOP ? W : 1][TOP ? ROOM : 1]; // and the vectors they are in
        float red[W][5];
        int lanes[W][64], count[W], total;
    };
    static __device__ int lane() { return W == 1 ? threadIdx.x & 63 : threadIdx.x; }
    static __device__ int wave() { return W == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

    // What a wave notes while it reads; all but `best` is the same in all lanes
    struct Noted {
        float best, b;                         // this lane's largest score; the bound
        int want, lanes, count, batch, next;
        bool over;                             // there was no room
        __device__ void init(int want_)
        {
            want = want_;
            best = b = -INFINITY;
            lanes = want > 16 ? 2 : want > 8 ? 4 : want > 4 ? 8 : 16;
            count = batch = 0;
            next = 1;
            over = false;
        }
        // The smallest maximum of as many groups of lanes as are wanted.  For more alternatives then closer, by halves, to the largest number
        // that as many lanes' maxima reach: every step's bound is one (10000 x 2500 fp32: ten alternatives 37 us without, 25 with, 32 of
        // them 93 and 28; by workgroups, 2500 x 20000 bf16, eight of them 35 and 36)
        __device__ void tighten()
        {
            b = fmaxf(b, wave_min(neighbours_max(best, lanes)));
            if (want <= (W == 1 ? 4 : 8)) return;
            float above = wave_max(best);
            for (int i = 0; i < 6; ++i) {
                const float mid = 0.5f * b + 0.5f * above;
                const bool reached = __popcll(__ballot(best >= mid)) >= want;
                b = reached ? mid : b;
                above = reached ? above : mid;
            }
        }
        // keeps the vectors that reach the bound
        __device__ void compact(Vec *list)
        {
            const int ln = threadIdx.x & 63;
            int kept = 0;
            for (int i = 0; i < count; i += 64) {
                const Vec e = list[min(i + ln, count - 1)];
                const uint64_t mask = __ballot(i + ln < count && e.m >= b);
                if (mask >> ln & 1) list[kept + __popcll(mask & ((1ull << ln) - 1))] = e;         // not behind its own place
                kept += __popcll(mask);
                team_sync<1>();
            }
            count = kept;
        }
        // puts entries of the lanes that have one behind the list's others
        template <typename E> __device__ void note(E *list, bool there, E entry)
        {
            const uint64_t mask = __ballot(there);
            if (!mask) return;
            const int n = __popcll(mask);
            if (count + n > ROOM) { over = true; return; }
            if (there) list[count + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0))] = entry;
            count += n;
        }
    };

    static __device__ float team_max(float v, Shared &sh)
    {
        v = wave_max(v);
        if constexpr (W > 1) {
            __syncthreads();
            if ((threadIdx.x & 63) == 0) sh.red[threadIdx.x >> 6][0] = v;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < W; ++w) v = fmaxf(v, sh.red[w][0]);
        }
        return v;
    }
    static __device__ float team_sum(float v, Shared &sh)
    {
        v = wave_sum(v);
        if constexpr (W > 1) {
            __syncthreads();
            if ((threadIdx.x & 63) == 0) sh.red[threadIdx.x >> 6][0] = v;
            __syncthreads();
            v = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) v += sh.red[w][0];
        }
        return v;
    }
    // The sums of a row that is masked throughout, holds the lowest or nearly the largest numbers, or is not finite: class by class, the
    // largest score first
    static __device__ Soft<MODE == LP> exact_row(const RowArgs &a, const Span<T> &sp, Shared &sh)
    {
        const int k1 = sp.k0 + sp.nvec * VEC + sp.edges();
        Soft<MODE == LP> so;
        so.init();
        float m = LOWEST;
        for (int c = sp.k0 + lane(); c < k1; c += NL) m = fmaxf(m, sis3d_f32(sp.row[c]));
        so.m = team_max(m, sh);
        for (int c = sp.k0 + lane(); c < k1; c += NL) so.add(sis3d_f32(sp.row[c]), a.c2);
        so.s = team_sum(so.s, sh);
        if constexpr (MODE == LP) so.t = team_sum(so.t, sh);
        return so;
    }

    // one pass over the span: the team's sums in every lane, and this lane's largest (score, class) among its vectors
    static __device__ Soft<MODE == LP> pass(const RowArgs &a, const Span<T> &sp, Stream<T, NL, !TOP> &st, Shared &sh, Noted &nt)
    {
        Lane<MODE == LP> ln;
        ln.init();
        nt.init(a.top);
        const float edge = lane() < sp.edges() ? sis3d_f32(sp.row[sp.edge_class(lane())]) : -INFINITY;
        auto batch = [&](auto count, int v, const SisVec<T, VEC> (&raw)[UL]) {
            constexpr int N = decltype(count)::value;
            const bool last = v + (N - 1) * NL < sp.nvec;       // no vector: -inf adds nothing
            float x[N][VEC], mx[N];
#pragma unroll
            for (int u = 0; u < N; ++u) {
                sis3d_unpack<T, VEC>(raw[u], x[u]);
                if (u == N - 1)
#pragma unroll
                    for (int i = 0; i < VEC; ++i) x[u][i] = last ? x[u][i] : -INFINITY;
                mx[u] = max_of(x[u]);
            }
            const float top = max_of(mx);
            nt.best = fmaxf(nt.best, top);
            ln.follow(top, a.c2);
            if constexpr (TOP) {
                if (++nt.batch == nt.next || nt.b == -INFINITY) {
                    nt.tighten();
                    nt.next = 2 * nt.batch;
                }
                // many alternatives: the list may fill before the bound is next due (10000 x 2500 fp32, 32 of them: 93 us, 160 without this)
                if (nt.count > ROOM - 64 * N) {
                    nt.tighten();
                    nt.compact(sh.vecs[wave()]);
                }
#pragma unroll
                for (int u = 0; u < N; ++u) nt.note(sh.vecs[wave()], mx[u] >= nt.b && mx[u] > -INFINITY, Vec{mx[u], v + u * NL});
            }
#pragma unroll
            for (int u = 0; u < N; ++u)
#pragma unroll
                for (int i = 0; i < VEC; ++i) ln.add(x[u][i], a.c2);
        };
        // by the same rule with and without alternatives: the same sums, bit for bit (50000 x 1000 bf16, five alternatives: 61 us compact,
        // 56 not; by workgroups 5000 x 10000: 43, 50)
        if constexpr (MODE == LP && W > 1) st.each_compact(batch);
        else st.each(batch);
        ln.follow(edge, a.c2);
        if (lane() < sp.edges()) ln.add(edge, a.c2);
        float block = INFINITY;                 // a bound from all waves' groups together, a quarter as many of each
        if constexpr (TOP) {
            nt.tighten();
            if (W > 1) block = wave_min(neighbours_max(nt.best, a.top > 16 ? 8 : 16));
        }
        auto so = ln.template join<64>(fmaxf(nt.best, edge), a.c2);
        if constexpr (W > 1) {
            if ((threadIdx.x & 63) == 0) {
                sh.red[threadIdx.x >> 6][0] = so.m;
                sh.red[threadIdx.x >> 6][1] = so.s;
                sh.red[threadIdx.x >> 6][2] = so.t;
                sh.red[threadIdx.x >> 6][3] = nt.b;
                sh.red[threadIdx.x >> 6][4] = block;
            }
            __syncthreads();
            if constexpr (TOP) {
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    nt.b = fmaxf(nt.b, sh.red[w][3]);
                    block = fminf(block, sh.red[w][4]);
                }
                nt.b = fmaxf(nt.b, block);
            }
            so = Soft<MODE == LP>{sh.red[0][0], sh.red[0][1], sh.red[0][2]};
#pragma unroll
            for (int w = 1; w < W; ++w) so.join(sh.red[w][0], sh.red[w][1], sh.red[w][2], a.c2);
        }
        if (!(so.s > 0.f && so.s < INFINITY)) so = exact_row(a, sp, sh);        // the same for all lanes of the team
        return so;
    }

    // Elements of the span that pass `keep(score, class)`, from the lanes whose `again` says that they have one and from the edges: read
    // again into sh.cand as one list, and their number as the answer, which may be more than there is room for
    template <typename F> static __device__ int collect(const Span<T> &sp, Shared &sh, bool again, F keep)
    {
        const int w = wave(), ln = threadIdx.x & 63;
        uint64_t *cand = sh.cand[0];
        team_sync<W>();
        if (lane() == 0) sh.total = 0;
        const uint64_t mask = __ballot(again);
        if (again) sh.lanes[w][__popcll(mask & ((1ull << ln) - 1))] = ln;
        team_sync<W>();
        auto offer = [&](float v, int c) {
            if (keep(v, c)) {
                const int i = atomicAdd(&sh.total, 1);
                if (i < W * ROOM) cand[i] = key_of(v, c);
            }
        };
        const int per = (sp.nvec + NL - 1) / NL, items = __popcll(mask) * per;
        for (int i = ln; i < items; i += 64) {
            const int j = i / per, v = sh.lanes[w][j] + w * 64 + (i - j * per) * NL;
            if (v >= sp.nvec) continue;
            float x[VEC];
            sis3d_load<T, VEC>(sp.body + (int64_t)v * VEC, x);
#pragma unroll
            for (int e = 0; e < VEC; ++e) offer(x[e], sp.first_class(v) + e);
        }
        if (lane() < sp.edges()) {
            const int c = sp.edge_class(lane());
            offer(sis3d_f32(sp.row[c]), c);
        }
        team_sync<W>();
        return sh.total;
    }

    // The `top` largest keys of the span, out(rank, key) once for each rank, from what the waves have noted
    template <typename F> static __device__ void alternatives(const RowArgs &a, const Span<T> &sp, Shared &sh, Noted &nt, F out)
    {
        const int want = a.top, w = wave(), ln = threadIdx.x & 63;       // a span has far more classes
        // of the vectors noted, those that reach the last bound are read again and their elements that do are noted
        if (nt.over) nt.count = 0;
        nt.compact(sh.vecs[w]);
        const int kept = nt.count;
        nt.count = 0;
        for (int i = 0; i < kept; i += 64) {
            const int v = sh.vecs[w][min(i + ln, kept - 1)].v, c = sp.first_class(v);
            float x[VEC];
            sis3d_load<T, VEC>(sp.body + (int64_t)v * VEC, x);
#pragma unroll
            for (int e = 0; e < VEC; ++e) nt.note(sh.cand[w], i + ln < kept && x[e] >= nt.b && x[e] > -INFINITY, key_of(x[e], c + e));
        }
        const float edge = lane() < sp.edges() ? sis3d_f32(sp.row[sp.edge_class(lane())]) : -INFINITY;
        nt.note(sh.cand[w], edge >= nt.b && edge > -INFINITY, key_of(edge, sp.edge_class(lane())));
        bool over = nt.over;
        int m = nt.count;
        if constexpr (W > 1) {
            if (ln == 0) sh.count[w] = over ? -1 : m;
            __syncthreads();
            m = 0;
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const int n = sh.count[i];
                over = over || n < 0;
                m += n;
            }
        } else team_sync<1>();
        if (!over && m >= want) {
            for (int i = ln; i < nt.count; i += 64) {
                const uint64_t k = sh.cand[w][i];
                int rank = 0;
#pragma unroll
                for (int q = 0; q < W; ++q) {
                    const int n = W == 1 ? nt.count : sh.count[q];
#pragma unroll 4
                    for (int j = 0; j < n; ++j) rank += sh.cand[q][j] > k;
                }
                if (rank < want) out(rank, k);
            }
            return;
        }
        const int room = W * ROOM;
        uint64_t *cand = sh.cand[0];
        if (!over) {
            // fewer numbers than that: -inf (and NaN, which counts as that) from the lowest class on; the first 64 classes hold enough
            m = collect(sp, sh, nt.best > -INFINITY, [](float v, int) { return v > -INFINITY; });
            const int c = sp.k0 + ln;
            const float v = sis3d_f32(sp.row[c]);
            const bool none = !(v > -INFINITY);
            const uint64_t mask = __ballot(none);
            const int i = m + __popcll(mask & ((1ull << ln) - 1));
            if (none && i < want && w == 0) cand[i] = key_of(v, c);
            team_sync<W>();
            m = want;
        } else {
            // Many equal scores at the bound: a bound on (score, class).  A vector's last class stands for the place of its maximum,
            // vectors being disjoint ranges of classes.
            int groups = 1;
            while (groups < want) groups *= 2;
            int at = lane();
            for (int v = lane(); v < sp.nvec; v += NL) {
                float x[VEC];
                sis3d_load<T, VEC>(sp.body + (int64_t)v * VEC, x);
                if (max_of(x) == nt.best) { at = v; break; }
            }
            const uint64_t mine = lane() < sp.nvec ? key_of(nt.best, sp.first_class(at) + VEC - 1) : 0;
            uint64_t k = mine;
            for (int o = 32; o >= groups; o >>= 1) k = max64(k, shfl_xor64(k, o));
            for (int o = groups >> 1; o > 0; o >>= 1) k = min64(k, shfl_xor64(k, o));
            if constexpr (W > 1) {
                if (ln == 0) sh.bound[w] = k;
                __syncthreads();
#pragma unroll
                for (int i = 0; i < W; ++i) k = max64(k, sh.bound[i]);
            }
            m = collect(sp, sh, mine != 0 && mine >= k, [&](float v, int c) { return key_of(v, c) >= k; });
        }
        if (m <= room) {
            for (int i = lane(); i < m; i += NL) {
                const uint64_t k = cand[i];
                int rank = 0;
                for (int j = 0; j < m; ++j) rank += cand[j] > k;
                if (rank < want) out(rank, k);
            }
            return;
        }
        // rows made to have more elements at the bound than there is room for: the largest below the last one, `want` times
        const int n = sp.nvec * VEC + sp.edges();
        uint64_t last = ~0ull;
        for (int r = 0; r < want; ++r) {
            uint64_t k = 0;
            for (int c = sp.k0 + lane(); c < sp.k0 + n; c += NL) {
                const uint64_t q = key_of(sis3d_f32(sp.row[c]), c);
                if (q < last) k = max64(k, q);
            }
            for (int o = 32; o > 0; o >>= 1) k = max64(k, shfl_xor64(k, o));
            if constexpr (W > 1) {
                __syncthreads();
                if (ln == 0) sh.bound[w] = k;
                __syncthreads();
                for (int i = 0; i < W; ++i) k = max64(k, sh.bound[i]);
            }
            if (lane() == 0) out(r, k);
            last = k;
        }
    }
};

// A row's kept entries in the L lanes that it has, at most two a lane.  Loads return in the order in which they were asked for: first the
// entries, then the row's vectors, then the scores of the entries' classes, which need wait for the entries alone.
template <int L> struct Kept {
    float x[2], l[2];                          // teacher's logit, student's score; -inf: no such entry
    int c[2];                                  // class, -1: none
    int64_t k[2];
    bool bad;
    __device__ Kept(const RowArgs &a, int64_t r, bool on = true) : bad(false)
    {
        const int lane = threadIdx.x & (L - 1), nk = on ? a.nk : 0;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            x[j] = -INFINITY;
            k[j] = -1;
            if (lane + L * j < nk) {
                k[j] = a.cls[r * a.nk + lane + L * j];
                x[j] = a.kept[r * a.nk + lane + L * j];
            }
        }
    }
    template <typename T> __device__ void scores(const RowArgs &a, const T *row)
    {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            c[j] = -1;
            l[j] = 0.f;
            if (k[j] < 0) x[j] = -INFINITY;
            else if (k[j] >= a.K || x[j] != x[j]) bad = true;
            else {
                c[j] = (int)k[j];
                l[j] = sis3d_f32(row[k[j]]);
            }
        }
    }
    __device__ Teacher teacher(const RowArgs &a) const
    {
        Teacher t;
        t.m = lanes_max<L>(fmaxf(x[0], x[1]));
        t.bad = lanes_any<L>(bad);
        t.any = t.m > -INFINITY;
        t.s = t.any ? lanes_sum<L>(exp2_((x[0] - t.m) * a.c2) + exp2_((x[1] - t.m) * a.c2)) : 0.f;
        return t;
    }
};

template <int L> __device__ inline void row_loss(const RowArgs &a, int64_t r, const Kept<L> &kept, const Soft<false> &so)
{
    const Norm norm{so.m, so.log_s()};
    const Teacher t = kept.teacher(a);
    float loss = 0.f;
    if (t.any) {
        const float ls = log_(t.s);
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (kept.c[j] >= 0) loss += entry_loss(a, t, ls, kept.x[j], kept.l[j], norm);
    }
    loss = a.tau * a.tau * lanes_sum<L>(loss);
    if ((threadIdx.x & (L - 1)) == 0) {
        a.loss[r] = t.bad ? NAN : loss;
        a.norm[r] = make_float2(so.m, so.s);
    }
}

// A row's label and, behind the row's vectors, its score
struct Label {
    int64_t y;
    float l;
    __device__ Label() : y(-1), l(0.f) {}
    __device__ Label(const RowArgs &a, int64_t r) : y(a.labels[r]), l(0.f) {}
    template <typename T> __device__ void score(const RowArgs &a, const T *row) { l = y >= 0 && y < a.K ? sis3d_f32(row[y]) : 0.f; }
};

__device__ inline void row_outputs(const RowArgs &a, int64_t r, const Label &label, const Soft<true> &so, Norm norm)
{
    a.logp[r] = label_logp(a, label.y, label.l, norm);
    a.entropy[r] = so.entropy();
    a.norm[r] = make_float2(so.m, so.s);
}

// outputs of a row past the live count, by a team of `n` lanes
template <int MODE> __device__ inline void zero_row(const RowArgs &a, int64_t r, int lane, int n)
{
    if (lane == 0) {
        a.norm[r] = make_float2(0.f, 0.f);
        if constexpr (MODE == KD) a.loss[r] = 0.f;
        else a.logp[r] = a.entropy[r] = 0.f;
    }
    if constexpr (MODE == LP)
        for (int i = lane; i < a.top; i += n) {
            a.top_logp[r * a.top + i] = 0.f;
            a.top_class[r * a.top + i] = 0;
        }
}

template <typename T, int W, int MODE, bool TOP> __global__ __launch_bounds__(256) void long_forward(RowArgs a)
{
    using L = Long<T, W, MODE, TOP>;
    __shared__ typename L::Shared shared[4 / W];
    auto &sh = shared[team_of<W>()];
    const int64_t r = (int64_t)blockIdx.x * (4 / W) + team_of<W>();
    if (r >= a.R) return;                                  // the whole team
    if (r >= live_rows(a)) { zero_row<MODE>(a, r, L::lane(), L::NL); return; }
    const T *row = (const T *)a.score + row_at(a, r, a.s_n, a.s_v);
    const Span<T> sp(row, 0, a.K);
    typename L::Noted nt;
    if constexpr (MODE == KD) {
        const bool first = W == 1 || threadIdx.x < 64;
        Kept<64> kept(a, r, first);
        Stream<T, L::NL, !TOP> st(sp, L::lane());
        kept.scores(a, row);
        const auto so = L::pass(a, sp, st, sh, nt);
        if (first) row_loss(a, r, kept, so);
    } else {
        Label label(a, r);
        Stream<T, L::NL, !TOP> st(sp, L::lane());
        label.score(a, row);
        const auto so = L::pass(a, sp, st, sh, nt);
        const Norm norm{so.m, so.log_s()};
        if (L::lane() == 0) row_outputs(a, r, label, so, norm);
        if constexpr (TOP)
            L::alternatives(a, sp, sh, nt, [&](int rank, uint64_t k) {
                a.top_class[r * a.top + rank] = key_class(k);
                a.top_logp[r * a.top + rank] = log_p(key_score(k), norm, 1.f, 0.f);
            });
    }
}

// Distillation of rows that are not so long: 16 lanes to a row, four rows to a wave, which share all that is done once a row
template <typename T> __global__ __launch_bounds__(256) void four_distill(RowArgs a)
{
    constexpr int L = 16, VEC = 16 / sizeof(T), UL = loads_of(L);
    const int64_t r0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 4, r = r0 + ((threadIdx.x & 63) >> 4), live = live_rows(a);
    const int lane = threadIdx.x & (L - 1);
    if (r >= live && r < a.R) zero_row<KD>(a, r, lane, L);
    if (r0 >= live) return;                                    // the whole wave
    const int64_t at = r < live ? r : live - 1;                // lanes of a row that is not there go over the last one and write nothing
    const T *row = (const T *)a.score + row_at(a, at, a.s_n, a.s_v);
    const Span<T> sp(row, 0, a.K);
    Kept<L> kept(a, at);
    Stream<T, L, true> st(sp, lane, a.K / VEC);
    kept.scores(a, row);
    const float edge = lane < sp.edges() ? sis3d_f32(row[sp.edge_class(lane)]) : -INFINITY;
    Lane<false> ln;
    ln.init();
    float best = edge;
    st.each([&](auto count, int v, const SisVec<T, VEC> (&raw)[UL]) {
        constexpr int N = decltype(count)::value;
        const bool last = v + (N - 1) * L < sp.nvec;
        float x[N][VEC], mx[N];
#pragma unroll
        for (int u = 0; u < N; ++u) {
            sis3d_unpack<T, VEC>(raw[u], x[u]);
            if (u == N - 1)
#pragma unroll
                for (int i = 0; i < VEC; ++i) x[u][i] = last ? x[u][i] : -INFINITY;
            mx[u] = max_of(x[u]);
        }
        const float top = max_of(mx);
        best = fmaxf(best, top);
        ln.follow(top, a.c2);
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
            for (int i = 0; i < VEC; ++i) ln.add(x[u][i], a.c2);
    });
    ln.follow(edge, a.c2);
    if (lane < sp.edges()) ln.add(edge, a.c2);
    Soft<false> so = ln.join<L>(best, a.c2);
    if (!(so.s > 0.f && so.s < INFINITY)) {                    // class by class, as exact_row; the same for the row's lanes
        so.init();
        for (int c = lane; c < a.K; c += L) so.m = fmaxf(so.m, sis3d_f32(row[c]));
        so.m = row_max(so.m);
        for (int c = lane; c < a.K; c += L) so.add(sis3d_f32(row[c]), a.c2);
        so.s = row_sum(so.s);
    }
    const int64_t out = r < live ? r : a.R;
    if (out < a.R) row_loss(a, out, kept, so);
}

// one part of a row to a workgroup
template <typename T, int MODE, bool TOP> __global__ __launch_bounds__(256) void split_forward(RowArgs a)
{
    using L = Long<T, 4, MODE, TOP>;
    __shared__ typename L::Shared sh;
    const int64_t r = blockIdx.x / a.parts;
    const int part = blockIdx.x - (int)(r * a.parts);
    if (r >= live_rows(a)) return;
    const T *row = (const T *)a.score + row_at(a, r, a.s_n, a.s_v);
    const int k0 = (int)((int64_t)a.K * part / a.parts), k1 = (int)((int64_t)a.K * (part + 1) / a.parts);
    const Span<T> sp(row, k0, k1);
    Stream<T, L::NL, !TOP> st(sp, L::lane());
    typename L::Noted nt;
    const auto so = L::pass(a, sp, st, sh, nt);
    if (threadIdx.x == 0) *(float4 *)(a.part + (size_t)blockIdx.x * 4) = make_float4(so.m, so.s, so.t, 0.f);
    if constexpr (TOP) L::alternatives(a, sp, sh, nt, [&](int rank, uint64_t k) { a.part_keys[(size_t)blockIdx.x * a.top + rank] = k; });
}

// joins the parts of a row: one wave
template <typename T, int MODE> __global__ __launch_bounds__(64) void split_join(RowArgs a)
{
    __shared__ uint64_t cand[64 * TOP_MAX];
    __shared__ int count;
    const int64_t r = blockIdx.x;
    const int lane = threadIdx.x;
    if (r >= live_rows(a)) { zero_row<MODE>(a, r, lane, 64); return; }
    const T *row = (const T *)a.score + row_at(a, r, a.s_n, a.s_v);
    Soft<MODE == LP> so;
    so.init();
    if (lane < a.parts) {
        const float4 v = *(const float4 *)(a.part + ((size_t)r * a.parts + lane) * 4);
        so = Soft<MODE == LP>{v.x, v.y, v.z};
    }
    so.join_wave(a.c2);
    const Norm norm{so.m, so.log_s()};
    if constexpr (MODE == KD) {
        Kept<64> kept(a, r);
        kept.scores(a, row);
        row_loss(a, r, kept, so);
    } else {
        Label label(a, r);
        label.score(a, row);
        if (lane == 0) row_outputs(a, r, label, so, norm);
        if (!a.top) return;
        // a part's last alternative bounds the row's from below: only keys that reach the largest of these bounds are ranked
        const uint64_t *keys = a.part_keys + (size_t)r * a.parts * a.top;
        uint64_t b = lane < a.parts ? keys[lane * a.top + a.top - 1] : 0;
        for (int o = 32; o > 0; o >>= 1) b = max64(b, shfl_xor64(b, o));
        if (lane == 0) count = 0;
        __syncthreads();
        for (int i = lane; i < a.parts * a.top; i += 64)
            if (keys[i] >= b) cand[atomicAdd(&count, 1)] = keys[i];
        __syncthreads();
        for (int i = lane; i < count; i += 64) {
            const uint64_t k = cand[i];
            int rank = 0;
            for (int j = 0; j < count; ++j) rank += cand[j] > k;
            if (rank < a.top) {
                a.top_class[r * a.top + rank] = key_class(k);
                a.top_logp[r * a.top + rank] = log_p(key_score(k), norm, 1.f, 0.f);
            }
        }
    }
}

// gradient of a row's part; `parts` workgroups or one team to a row
template <typename T, int W, int MODE> __global__ __launch_bounds__(256) void long_backward(RowArgs a)
{
    constexpr int NL = 64 * W, VEC = 16 / sizeof(T), UL = loads_of(NL);
    __shared__ float q_s[4 / W][MODE == KD ? KEPT_MAX : 1], l_s[4 / W][MODE == KD ? KEPT_MAX : 1];
    __shared__ int c_s[4 / W][MODE == KD ? KEPT_MAX : 1];
    const int team = team_of<W>(), lane = W == 1 ? threadIdx.x & 63 : threadIdx.x;
    const int64_t item = (int64_t)blockIdx.x * (4 / W) + team, r = a.parts == 1 ? item : item / a.parts;
    if (r >= a.R) return;
    int k0 = 0, k1 = a.K;
    if (a.parts > 1) {
        const int part = (int)(item - r * a.parts);
        k0 = (int)((int64_t)a.K * part / a.parts);
        k1 = (int)((int64_t)a.K * (part + 1) / a.parts);
    }
    const T *row = (const T *)a.score + row_at(a, r, a.s_n, a.s_v);
    T *out = (T *)a.dscore + row_at(a, r, a.d_n, a.d_v);
    if (r >= live_rows(a)) {
        for (int c = k0 + lane; c < k1; c += NL) out[c] = sis3d_from_f32<T>(0.f);
        return;
    }
    const Span<T> sp(row, k0, k1);
    Back<MODE> k;
    int y = -1;
    float ly = 0.f;
    const float2 norm = a.norm_in[r];
    const float g1 = a.g1[r];
    const Label label = MODE == LP ? Label(a, r) : Label();
    Kept<64> kept(a, r, MODE == KD);
    Stream<T, NL, true> st(sp, lane);
    const float edge = lane < sp.edges() ? sis3d_f32(row[sp.edge_class(lane)]) : 0.f;
    if constexpr (MODE == LP) {
        y = label.y >= k0 && label.y < k1 ? (int)label.y : -1;
        if (y >= 0) ly = sis3d_f32(row[y]);
        k.scores(norm, a.entropy_in[r], label.y < 0 ? 0.f : (label.y >= a.K ? NAN : g1), a.g2 ? a.g2[r] : 0.f);
    } else {
        kept.scores(a, row);
        const Teacher t = kept.teacher(a);
        k.loss(norm, t.bad ? NAN : (t.any ? g1 * a.tau : 0.f), a.c2);
        if (W == 1 || threadIdx.x < 64)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                c_s[team][lane + 64 * j] = kept.c[j];
                q_s[team][lane + 64 * j] = t.any ? exp2_((kept.x[j] - t.m) * a.c2) * rcp_(t.s) : 0.f;
                l_s[team][lane + 64 * j] = kept.l[j];
            }
    }
    const bool wide = ((uintptr_t)(out + k0 + sp.head) & 15) == 0;
    if (!k.in_range) {
        for (int c = k0 + lane; c < k1; c += NL) out[c] = sis3d_from_f32<T>(k.exact(sis3d_f32(row[c])));
    } else st.each([&](auto count, int v, const SisVec<T, VEC> (&raw)[UL]) {
        constexpr int N = decltype(count)::value;
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int c = sp.first_class(v + u * NL);
            float x[VEC];
            sis3d_unpack<T, VEC>(raw[u], x);
#pragma unroll
            for (int i = 0; i < VEC; ++i) x[i] = k.near(x[i]);
            if (u == N - 1 && v + u * NL >= sp.nvec) continue;
            if (wide) sis3d_store<T, VEC>(out + c, x);
            else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) out[c + i] = sis3d_from_f32<T>(x[i]);
            }
        }
    });
    if (lane < sp.edges() && k.in_range) out[sp.edge_class(lane)] = sis3d_from_f32<T>(k.exact(edge));
    // The label's class, or the kept classes of this part, again with their share: written behind the team's own stores.  A class that
    // is kept twice is written by its first entry with the sum of both.
    team_sync<W>();
    if constexpr (MODE == LP) {
        if (lane == 0 && y >= 0) out[y] = sis3d_from_f32<T>(k.exact(ly) + k.ga);
    } else {
        for (int i = lane; i < a.nk; i += NL) {
            const int c = c_s[team][i];
            if (c < k0 || c >= k1) continue;
            float q = 0.f;
            bool first = true;
            for (int j = 0; j < a.nk; ++j)
                if (c_s[team][j] == c) {
                    q += q_s[team][j];
                    first = first && j >= i;
                }
            if (first) out[c] = sis3d_from_f32<T>(k.exact(l_s[team][i]) - k.ga * q);
        }
    }
}

// The same with 16 lanes to a row, four rows to a wave, as four_distill
template <typename T, int MODE> __global__ __launch_bounds__(256) void four_backward(RowArgs a)
{
    constexpr int L = 16, VEC = 16 / sizeof(T), UL = loads_of(L);
    __shared__ float q_s[16][MODE == KD ? 2 * L : 1];
    __shared__ int c_s[16][MODE == KD ? 2 * L : 1];
    const int64_t r0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 4, r = r0 + ((threadIdx.x & 63) >> 4), n = live_rows(a);
    const int lane = threadIdx.x & (L - 1), team = threadIdx.x >> 4;
    if (r0 >= a.R) return;                                     // the whole wave
    T *out = (T *)a.dscore + row_at(a, r < a.R ? r : 0, a.d_n, a.d_v);
    if (r >= n) {
        if (r < a.R)
            for (int c = lane; c < a.K; c += L) out[c] = sis3d_from_f32<T>(0.f);
        return;                                                // all lanes of the row
    }
    const T *row = (const T *)a.score + row_at(a, r, a.s_n, a.s_v);
    const Span<T> sp(row, 0, a.K);
    Back<MODE> k;
    const float2 norm = a.norm_in[r];
    const float g1 = a.g1[r];
    const Label label = MODE == LP ? Label(a, r) : Label();
    Kept<L> kept(a, r, MODE == KD);
    Stream<T, L, true> st(sp, lane, a.K / VEC);
    const float edge = lane < sp.edges() ? sis3d_f32(row[sp.edge_class(lane)]) : 0.f;
    float ly = 0.f;
    if constexpr (MODE == LP) {
        if (label.y >= 0 && label.y < a.K) ly = sis3d_f32(row[label.y]);
        k.scores(norm, a.entropy_in[r], label.y < 0 ? 0.f : (label.y >= a.K ? NAN : g1), a.g2 ? a.g2[r] : 0.f);
    } else {
        kept.scores(a, row);
        const Teacher t = kept.teacher(a);
        k.loss(norm, t.bad ? NAN : (t.any ? g1 * a.tau : 0.f), a.c2);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            c_s[team][lane + L * j] = kept.c[j];
            q_s[team][lane + L * j] = t.any ? exp2_((kept.x[j] - t.m) * a.c2) * rcp_(t.s) : 0.f;
        }
    }
    const bool wide = ((uintptr_t)(out + sp.head) & 15) == 0;
    if (!k.in_range) {
        for (int c = lane; c < a.K; c += L) out[c] = sis3d_from_f32<T>(k.exact(sis3d_f32(row[c])));
    } else {
        st.each([&](auto count, int v, const SisVec<T, VEC> (&raw)[UL]) {
            constexpr int N = decltype(count)::value;
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const int c = sp.first_class(v + u * L);
                float x[VEC];
                sis3d_unpack<T, VEC>(raw[u], x);
#pragma unroll
                for (int i = 0; i < VEC; ++i) x[i] = k.near(x[i]);
                if (u == N - 1 && v + u * L >= sp.nvec) continue;
                if (wide) sis3d_store<T, VEC>(out + c, x);
                else {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) out[c + i] = sis3d_from_f32<T>(x[i]);
                }
            }
        });
        if (lane < sp.edges()) out[sp.edge_class(lane)] = sis3d_from_f32<T>(k.exact(edge));
    }
    team_sync<1>();                                            // the label's class or the kept ones again, behind the row's other stores
    if constexpr (MODE == LP) {
        if (lane == 0 && label.y >= 0 && label.y < a.K) out[label.y] = sis3d_from_f32<T>(k.exact(ly) + k.ga);
    } else {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = lane + L * j, c = kept.c[j];
            if (i >= a.nk || c < 0) continue;
            float q = 0.f;
            bool first = true;
            for (int m = 0; m < a.nk; ++m)
                if (c_s[team][m] == c) {
                    q += q_s[team][m];
                    first = first && m >= i;
                }
            if (first) out[c] = sis3d_from_f32<T>(k.exact(kept.l[j]) - k.ga * q);
        }
    }
}

// ------------------------------------------------------------------------------------------------------ host --
// a launch has at most 2^32 - 1 threads
bool too_many(int64_t workgroups) { return workgroups > 0xffffffffll / 256; }

// fp16, log probabilities, forward / backward: 50000 x 1000 48 / 59 us as short rows, 35 / 37 as longer ones; 83000 x 600 44 / 42 and 52 / 41
bool is_short(int K, int64_t s_c, int es) { return s_c != 1 ? K <= K_STRIDED : K <= 64 * (16 / es) + 16; }

// few long rows: parts of at least 4096 classes, enough for two workgroups per CU, at most one per lane of the joining wave
int parts_of(int64_t R, int K, int64_t s_c)
{
    if (K <= K_WAVE || s_c != 1 || R >= 256 || R <= 0) return 1;
    int64_t p = (512 + R - 1) / R;
    if (p > K / 4096) p = K / 4096;
    return (int)(p > 64 ? 64 : (p < 1 ? 1 : p));
}

// a wave to a row rather than a workgroup: up to 4096 classes, or 1536 vectors where there are rows enough (5000 x 10000 bf16, five
// alternatives: 46 us by workgroups, 27 by waves; 5000 x 5000 fp32 38 and 22)
bool wave_rows(const RowArgs &a, int es) { return a.parts == 1 && (a.K <= K_WAVE || (a.K <= 24576 / es && a.R >= 4096)); }

// distillation with 16 lanes to a row: rows of up to 4 KB, of 96 classes at least (tiles and waves against it, 8 entries, 100 MB:  fp32
// x 64 31 / 41 us, x 100 41 / 32, x 300 38 / 23, x 1000 21 / 22;  fp16 x 100 61 / 56, x 300 52 / 31, x 600 46 / 23, x 1203 36 / 24, x 2000
// 26 / 24, x 4000 23 / 25)
bool four_rows(const RowArgs &a, int es) { return a.s_c == 1 && a.nk <= 32 && a.K >= 96 && a.K * es <= 4096 && a.R >= 16 * 256; }

// how a tile's rows are had, its lanes per row and its LDS; LDS for dense, aligned rows of at most 56 floats a lane
template <typename T> int plan_tile(RowArgs &a, bool backward)
{
    const bool dense = a.s_c == 1 && a.s_v == a.K && (a.N == 1 || a.s_n == a.V * a.K) && ((uintptr_t)a.score & 15) == 0 &&
                       (!backward || (a.d_c == 1 && a.d_v == a.K && (a.N == 1 || a.d_n == a.V * a.K) && ((uintptr_t)a.dscore & 15) == 0));
    const int how = !dense ? IN_PLACE : a.K % 4 ? BY_ONE : BY_FOUR;
    a.sk = how == BY_FOUR ? ((a.K / 4) | 1) * 4 : a.K;
    a.per4 = how == BY_FOUR ? (uint32_t)((((uint64_t)1 << 32) + a.K / 4 - 1) / (a.K / 4)) : 0;
    // a teacher's entries are shared by up to eight lanes, two or, where the row's gradient is made in LDS, four of them a lane.  Half a
    // million x 41 fp32, planar, 16 entries: forward 361 us by two lanes, 147 by four, 100 by eight, backward 467, 262, 178; 32 entries:
    // 183 / 196 us forward by eight / sixteen, 356 / 455 backward.  Rows, 16 entries, backward: 276 us by two, 81 by four, 93 by eight.
    a.g_log = 0;
    while (a.g_log < 3 && (backward && dense ? 4 : 2) << a.g_log < a.nk && 4 << a.g_log < a.K) ++a.g_log;
    // 32 classes a lane (400000 x 41 fp32: 20 us by two lanes, 28 by one); 56 where the lanes' lists of alternatives have to be joined (400000 x 100 bf16, ten alternatives: 120 us by 24, 99 by
    // 48, 90 by 96, which is 64 KB of LDS and more)
    const int stretch = a.top > 4 && a.K > 48 ? 56 : 32;
    if (dense || !a.planar)
        while (a.g_log < 5 && stretch << a.g_log < a.K) ++a.g_log;
    // more lanes to a row while there are CUs without a workgroup
    while (a.g_log < 4 && 8 << a.g_log < a.K && (a.R << a.g_log) < 256 * 256) ++a.g_log;
    a.chunk = (a.K + (1 << a.g_log) - 1) >> a.g_log;
    // the lanes of a row meet different banks (125000 x 400 bf16 with stretches of 16: backward 105 us, of 28: 54)
    if (how == BY_FOUR) a.chunk = ((a.chunk + 3) / 4 | 1) * 4;
    if (how == BY_ONE) a.chunk |= 1;
    return how;
}
size_t tile_lds(const RowArgs &a, int how) { return how == IN_PLACE ? 0 : ((size_t)(256 >> a.g_log) * a.sk + ((size_t)a.chunk << a.g_log) + 16) * sizeof(float); }

template <typename T, int MODE, int TK> void tile_launch(RowArgs &a, int how, hipStream_t st)
{
    const int rb = 256 >> a.g_log;
    const dim3 grid((unsigned)((a.R + rb - 1) / rb)), block(256);
    const size_t lds = tile_lds(a, how);
    if (how == IN_PLACE) hipLaunchKernelGGL((tile_forward<T, MODE, IN_PLACE, TK>), grid, block, lds, st, a);
    else if (how == BY_ONE) hipLaunchKernelGGL((tile_forward<T, MODE, BY_ONE, TK>), grid, block, lds, st, a);
    else hipLaunchKernelGGL((tile_forward<T, MODE, BY_FOUR, TK>), grid, block, lds, st, a);
}

template <typename T, int MODE> int run_forward(RowArgs &a, hipStream_t st)
{
    if constexpr (MODE == KD)
        if (four_rows(a, sizeof(T))) {
            if (too_many((a.R + 15) / 16)) return SIS3D_EUNSUPPORTED;
            hipLaunchKernelGGL((four_distill<T>), dim3((unsigned)((a.R + 15) / 16)), dim3(256), 0, st, a);
            return sis3d_check_launch();
        }
    if (is_short(a.K, a.s_c, sizeof(T))) {
        const int how = plan_tile<T>(a, false);
        if (too_many((a.R + (256 >> a.g_log) - 1) / (256 >> a.g_log))) return SIS3D_EUNSUPPORTED;
        if (MODE == KD || a.top == 0) tile_launch<T, MODE, 0>(a, how, st);
        else if (a.top == 1) tile_launch<T, LP, 1>(a, how, st);
        else if (a.top <= 4) tile_launch<T, LP, 4>(a, how, st);
        else if (a.top <= 8) tile_launch<T, LP, 8>(a, how, st);
        else if (a.top <= 16) tile_launch<T, LP, 16>(a, how, st);
        else tile_launch<T, LP, 32>(a, how, st);
        return sis3d_check_launch();
    }
    const bool by_wave = wave_rows(a, sizeof(T));
    const int64_t workgroups = by_wave ? (a.R + 3) / 4 : a.R * a.parts;
    if (too_many(workgroups)) return SIS3D_EUNSUPPORTED;
    const dim3 block(256), each((unsigned)workgroups);
    auto launch = [&](auto top) {
        constexpr bool TOP = decltype(top)::value && MODE == LP;
        if (a.parts > 1) hipLaunchKernelGGL((split_forward<T, MODE, TOP>), each, block, 0, st, a);
        else if (by_wave) hipLaunchKernelGGL((long_forward<T, 1, MODE, TOP>), each, block, 0, st, a);
        else hipLaunchKernelGGL((long_forward<T, 4, MODE, TOP>), each, block, 0, st, a);
    };
    if (a.top) launch(Count<1>());
    else launch(Count<0>());
    const int rc = sis3d_check_launch();
    if (rc || a.parts == 1) return rc;
    hipLaunchKernelGGL((split_join<T, MODE>), dim3((unsigned)a.R), dim3(64), 0, st, a);
    return sis3d_check_launch();
}

template <typename T, int MODE> int run_backward(RowArgs &a, hipStream_t st)
{
    // 16 lanes to a row where a wave has too little of it and a tile too few rows (100 MB bf16, log probabilities: x 100 50 us by tiles, 60 by
    // 16 lanes; x 200 54 / 42, x 400 54 / 40, x 600 44 / 42, x 1000 37 by waves, 40; fp32 x 200 47 / 40, x 300 40 / 40)
    if (a.d_c == 1 && a.K >= 200 && a.K * (int)sizeof(T) <= 1200 && four_rows(a, sizeof(T))) {
        if (too_many((a.R + 15) / 16)) return SIS3D_EUNSUPPORTED;
        hipLaunchKernelGGL((four_backward<T, MODE>), dim3((unsigned)((a.R + 15) / 16)), dim3(256), 0, st, a);
        return sis3d_check_launch();
    }
    if (is_short(a.K, a.s_c, sizeof(T)) || a.d_c != 1) {
        const int how = plan_tile<T>(a, true), rb = 256 >> a.g_log;
        if (too_many((a.R + rb - 1) / rb)) return SIS3D_EUNSUPPORTED;
        const dim3 grid((unsigned)((a.R + rb - 1) / rb)), block(256);
        const size_t lds = tile_lds(a, how);
        if (how == IN_PLACE) hipLaunchKernelGGL((tile_backward<T, MODE, IN_PLACE>), grid, block, lds, st, a);
        else if (how == BY_ONE) hipLaunchKernelGGL((tile_backward<T, MODE, BY_ONE>), grid, block, lds, st, a);
        else hipLaunchKernelGGL((tile_backward<T, MODE, BY_FOUR>), grid, block, lds, st, a);
        return sis3d_check_launch();
    }
    const bool by_wave = wave_rows(a, sizeof(T));
    const int64_t workgroups = by_wave ? (a.R + 3) / 4 : a.R * a.parts;
    if (too_many(workgroups)) return SIS3D_EUNSUPPORTED;
    const dim3 each((unsigned)workgroups);
    if (by_wave) hipLaunchKernelGGL((long_backward<T, 1, MODE>), each, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((long_backward<T, 4, MODE>), each, dim3(256), 0, st, a);
    return sis3d_check_launch();
}

template <int MODE> int run(RowArgs &a, int dtype, bool backward, hipStream_t st)
{
    switch (dtype) {
    case SIS3D_F32: return backward ? run_backward<float, MODE>(a, st) : run_forward<float, MODE>(a, st);
    case SIS3D_BF16: return backward ? run_backward<__bf16, MODE>(a, st) : run_forward<__bf16, MODE>(a, st);
    default: return backward ? run_backward<_Float16, MODE>(a, st) : run_forward<_Float16, MODE>(a, st);
    }
}

// the arguments that all four entry points share; EUNSUPPORTED for scores that are neither short nor contiguous along the classes
int fill(RowArgs &a, const void *score, int dtype, int N, int64_t V, int K, int64_t s_n, int64_t s_v, int64_t s_c, const int32_t *num)
{
    if (!sis3d_elem_bytes(dtype) || N < 0 || V < 0 || K <= 0) return SIS3D_EINVAL;
    if (V && N > ((int64_t)1 << 40) / V) return SIS3D_EUNSUPPORTED;
    a.score = score; a.N = N; a.V = V; a.R = N * V; a.K = K; a.s_n = s_n; a.s_v = s_v; a.s_c = s_c; a.num = num;
    if (K > K_STRIDED && s_c != 1) return SIS3D_EUNSUPPORTED;
    if (((uintptr_t)score) % sis3d_elem_bytes(dtype)) return SIS3D_EINVAL;
    a.planar = s_c != 1 && s_v < s_c;
    a.parts = parts_of(a.R, K, s_c);
    if (a.R * a.parts > 0x7fffffff) return SIS3D_EUNSUPPORTED;
    return SIS3D_OK;
}

void temperature(RowArgs &a, float t)
{
    const double inv = 1.0 / t;
    a.tau = t;
    a.inv = (float)inv;
    a.inv_lo = (float)(inv - a.inv);
    a.c2 = (float)(1.4426950408889634 * inv);
}

size_t ws_of(int64_t R, int parts, int top) { return parts > 1 ? (size_t)R * parts * (16 + 8 * (size_t)top) : 0; }

} // namespace

extern "C" size_t sis3d_class_rows_workspace_bytes(int64_t rows, int K, int64_t s_c, int top)
{
    return rows > 0 && K > 0 ? ws_of(rows, parts_of(rows, K, s_c), top > 0 ? top : 0) : 0;
}

extern "C" int sis3d_class_logprobs_forward(const void *score, int dtype, int N, int64_t V, int K, int64_t s_n, int64_t s_v, int64_t s_c,
                                            const int64_t *labels, const int32_t *num_rows, int top, float *logp, float *entropy,
                                            float *norm, float *top_logp, int64_t *top_class, void *workspace, size_t workspace_bytes,
                                            sis3d_stream_t stream)
{
    RowArgs a{};
    const int rc = fill(a, score, dtype, N, V, K, s_n, s_v, s_c, num_rows);
    if (rc) return rc;
    if (top < 0 || top > TOP_MAX || top > K) return SIS3D_EINVAL;
    if (a.R == 0) return SIS3D_OK;
    if (!score || !labels || !logp || !entropy || !norm || (top && (!top_logp || !top_class))) return SIS3D_EINVAL;
    if (workspace_bytes < ws_of(a.R, a.parts, top)) return SIS3D_EWORKSPACE;
    if (a.parts > 1 && (!workspace || ((uintptr_t)workspace & 15))) return SIS3D_EINVAL;
    a.labels = labels; a.top = top; a.logp = logp; a.entropy = entropy; a.norm = (float2 *)norm; a.top_logp = top_logp; a.top_class = top_class;
    a.part = (float *)workspace;
    a.part_keys = (uint64_t *)((char *)workspace + (size_t)a.R * a.parts * 16);
    temperature(a, 1.f);
    return run<LP>(a, dtype, false, as_stream(stream));
}

extern "C" int sis3d_class_logprobs_backward(const void *score, int dtype, int N, int64_t V, int K, int64_t s_n, int64_t s_v, int64_t s_c,
                                             const int64_t *labels, const int32_t *num_rows, const float *norm, const float *entropy,
                                             const float *grad_logp, const float *grad_entropy, void *dscore, int64_t d_n, int64_t d_v,
                                             int64_t d_c, sis3d_stream_t stream)
{
    RowArgs a{};
    const int rc = fill(a, score, dtype, N, V, K, s_n, s_v, s_c, num_rows);
    if (rc) return rc;
    if (K > K_STRIDED && d_c != 1) return SIS3D_EUNSUPPORTED;
    if (a.R == 0) return SIS3D_OK;
    if (!score || !labels || !norm || !entropy || !grad_logp || !dscore) return SIS3D_EINVAL;
    a.labels = labels; a.norm_in = (const float2 *)norm; a.entropy_in = entropy; a.g1 = grad_logp; a.g2 = grad_entropy;
    a.dscore = dscore; a.d_n = d_n; a.d_v = d_v; a.d_c = d_c;
    temperature(a, 1.f);
    return run<LP>(a, dtype, true, as_stream(stream));
}

extern "C" int sis3d_distill_forward(const void *score, int dtype, int N, int64_t V, int K, int64_t s_n, int64_t s_v, int64_t s_c,
                                     const float *kept, const int64_t *classes, int nkept, const int32_t *num_rows, float temp, float *loss,
                                     float *norm, void *workspace, size_t workspace_bytes, sis3d_stream_t stream)
{
    RowArgs a{};
    const int rc = fill(a, score, dtype, N, V, K, s_n, s_v, s_c, num_rows);
    if (rc) return rc;
    if (nkept < 1 || nkept > KEPT_MAX || !(temp >= 1e-3f && temp <= 1e3f)) return SIS3D_EINVAL;
    if (a.R == 0) return SIS3D_OK;
    if (!score || !kept || !classes || !loss || !norm) return SIS3D_EINVAL;
    if (workspace_bytes < ws_of(a.R, a.parts, 0)) return SIS3D_EWORKSPACE;
    if (a.parts > 1 && (!workspace || ((uintptr_t)workspace & 15))) return SIS3D_EINVAL;
    a.kept = kept; a.cls = classes; a.nk = nkept; a.loss = loss; a.norm = (float2 *)norm;
    a.part = (float *)workspace;
    temperature(a, temp);
    return run<KD>(a, dtype, false, as_stream(stream));
}

extern "C" int sis3d_distill_backward(const void *score, int dtype, int N, int64_t V, int K, int64_t s_n, int64_t s_v, int64_t s_c,
                                      const float *kept, const int64_t *classes, int nkept, const int32_t *num_rows, float temp,
                                      const float *norm, const float *grad_loss, void *dscore, int64_t d_n, int64_t d_v, int64_t d_c,
                                      sis3d_stream_t stream)
{
    RowArgs a{};
    const int rc = fill(a, score, dtype, N, V, K, s_n, s_v, s_c, num_rows);
    if (rc) return rc;
    if (nkept < 1 || nkept > KEPT_MAX || !(temp >= 1e-3f && temp <= 1e3f)) return SIS3D_EINVAL;
    if (K > K_STRIDED && d_c != 1) return SIS3D_EUNSUPPORTED;
    if (a.R == 0) return SIS3D_OK;
    if (!score || !kept || !classes || !norm || !grad_loss || !dscore) return SIS3D_EINVAL;
    a.kept = kept; a.cls = classes; a.nk = nkept; a.norm_in = (const float2 *)norm; a.g1 = grad_loss;
    a.dscore = dscore; a.d_n = d_n; a.d_v = d_v; a.d_c = d_c;
    temperature(a, temp);
    return run<KD>(a, dtype, true, as_stream(stream));
}
