// Sampling from rows of scores with given random numbers: temperature, top-k, top-p and min-p, with replacement (inverse of the cumulative
// mass) and without (the n largest keys of an exponential race).
//
//   score x: NaN and -inf (a weight: anything not positive) are excluded, +inf counts as the type's largest value
//   l = x / T or log(x) / T,   mass w = exp(l - max l), or x itself for weights at T = 1
//   top-k keeps the k best, ties to the lowest index; top-p the shortest prefix of those, best first, that carries p of their mass;
//   min-p what has at least min_p of the best mass
//   with replacement:    smallest i with (w_0 + ... + w_i) > u * total
//   without:             the n largest l_i - log(-log(1 - u_i)), in index order
//
// All masses, sums and keys are in 64 bits: an index has to be the same as the definition's however many categories there are.  A mass below
// 2^-1074 of the row's best is 0 and never drawn.  Masses that
// are added by atomics (top-p's histograms) are added as integers, so that neither their order nor the launch changes a result: of 63 fraction
// bits of the largest mass.  Floating sums have one fixed order.
//
// What bounds it: not the bytes (3 M scores are 3 us of memory, 10 M with their numbers 18).  A short row is the work of one compute unit
// (100 ns for each instruction that 15 k elements cost); a long one a chain of passes, each of which pays 4 to 5 us to be launched behind the
// one before, some 2 us for a round trip between the chip's eight L2 caches, and its vector instructions.
#include "lg_common.h"
#include "lg_types.h"
#include "litegs_hip.h"


#define SM_BINS 2048                   // bins of one level of a radix selection
#define SM_MAX_WAVES 16
#define SM_SHORT 12288                 // longest row of one workgroup: 768 threads of 16 elements (a CU has 168 registers for each of 12 waves; with 16 waves 128 are too few)

enum { SM_LOGITS = 0, SM_LINEAR = 1, SM_POWER = 2 };

struct SmRule { int mode; double inv_t /*1 / temperature*/, top_p, min_p; long long top_k; };

// ---- scores ------------------------------------------------------------------------------------------------------------------------------
// A row's passes are bound by their instructions (a vector instruction takes a wave four cycles: 69 of them per element were 27 us for 10 M),
// so that scores are compared as the floats that they are, and taken apart as ordered integers only where a bin is wanted.
template <typename T> struct SmMax;
template <> struct SmMax<float> { static constexpr float v = 3.402823466e38f; };
template <> struct SmMax<LgHalf> { static constexpr float v = 65504.0f; };
template <> struct SmMax<LgBf16> { static constexpr float v = 3.3895313892515355e38f; };

__device__ __forceinline__ float sm_floor(const SmRule& r) { return r.mode == SM_LOGITS ? -INFINITY : 0.0f; }
// the score itself (-0 + 0 = +0: equal scores have equal bits); -inf = excluded
template <typename T> __device__ __forceinline__ float sm_score(T raw, float floor)
{
    const float x = lg_to_float(raw);
    return x > floor ? fminf(x, SmMax<T>::v) + 0.0f : -INFINITY;
}
// larger float <=> larger integer, and back
__device__ __forceinline__ uint32_t sm_order(float k)
{
    const uint32_t b = __float_as_uint(k);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float sm_unorder(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o); }

// exp(x) for x <= 0 and log(x) for x > 0 in 64 bits, without the general functions' special cases (which cost as much again, and registers):
// x = n ln 2 + r with |r| <= ln 2 / 2 and the Taylor polynomial of degree 13 (first term left out < 5e-18);  x = 2^e m with m in
// [sqrt(1/2), sqrt(2)), log m = 2 atanh(s), s = (m - 1) / (m + 1), |s| < 0.172, eleven terms behind the first (next: 4e-19).  ln 2 in two
// parts, the first of 32 bits so that its products with n are exact.  Good to about one step.
__device__ __forceinline__ double sm_exp(double x)
{
    x = fmax(x, -800.0);                                               // (below 2^-1074 all is 0)
    const double n = rint(x * 1.4426950408889634);
    const double r = fma(n, -1.90821492927058770e-10, fma(n, -6.93147180369123816e-01, x));
    double p = fma(r, 1.6059043836821613e-10, 2.08767569878681e-09);
    p = fma(r, p, 2.505210838544172e-08);
    p = fma(r, p, 2.755731922398589e-07);
    p = fma(r, p, 2.7557319223985893e-06);
    p = fma(r, p, 2.48015873015873e-05);
    p = fma(r, p, 0.0001984126984126984);
    p = fma(r, p, 0.001388888888888889);
    p = fma(r, p, 0.008333333333333333);
    p = fma(r, p, 0.041666666666666664);
    p = fma(r, p, 0.16666666666666666);
    p = fma(r, p, 0.5);
    return ldexp(fma(r * r, p, r) + 1.0, (int)n);
}
__device__ __forceinline__ double sm_ln(double x)
{
    int e = __builtin_amdgcn_frexp_exp(x);
    double m = __builtin_amdgcn_frexp_mant(x);                          // [1/2, 1)
    if (m < 0.70710678118654752) { m *= 2.0; e -= 1; }
    const double f = m - 1.0, s = f / (m + 1.0), z = s * s;
    double p = fma(z, 1.0 / 23, 1.0 / 21);
    p = fma(z, p, 1.0 / 19);
    p = fma(z, p, 1.0 / 17);
    p = fma(z, p, 1.0 / 15);
    p = fma(z, p, 1.0 / 13);
    p = fma(z, p, 1.0 / 11);
    p = fma(z, p, 1.0 / 9);
    p = fma(z, p, 1.0 / 7);
    p = fma(z, p, 1.0 / 5);
    p = fma(z, p, 1.0 / 3);
    const double n = (double)e;
    return fma(n, 6.93147180369123816e-01, fma(n, 1.90821492927058770e-10, 2.0 * fma(s * z, p, s)));
}

struct SmScale { int mode; double inv_t, top /*l of the best score, or its weight*/, shift /*power of two that brings a linear weight below one*/; };

// The best one's l has to come from the function that gives the others' (`ln`): at a temperature of 1e-20 the last bit of a logarithm is
// as much as e^1000.
template <typename Ln> __device__ __forceinline__ SmScale sm_scale(const SmRule& r, float best, const Ln& ln)
{
    SmScale s = { r.mode, r.inv_t, 0.0, 1.0 };
    if (best == -INFINITY) return s;
    const double x = (double)best;
    if (r.mode == SM_LOGITS) s.top = x * s.inv_t;
    else if (r.mode == SM_POWER) s.top = ln(x) * s.inv_t;
    else { s.top = x; s.shift = ldexp(1.0, -ilogb(x) - 1); }
    return s;
}
__device__ __forceinline__ SmScale sm_scale(const SmRule& r, float best)                      // for sm_mass
{
    return sm_scale(r, best, [](double x) { return sm_ln(x); });
}
__device__ __forceinline__ double sm_log(const SmScale& s, float score)
{
    const double x = (double)score;
    return s.mode == SM_LOGITS ? x * s.inv_t : s.mode == SM_POWER ? sm_ln(x) * s.inv_t : sm_ln(x);
}
__device__ __forceinline__ double sm_mass(const SmScale& s, float score)                      // (NaN of a NaN)
{
    return s.mode == SM_LINEAR ? (double)score : sm_exp(sm_log(s, score) - s.top);
}
// The same masses in about a third of the instructions, for passes over whole rows, with two tables in LDS that each workgroup works out for
// itself: 1 / c and log c for the middles c of 128 parts of [1, 2) -- a score has 24 bits, m / c - 1 is one product, below 1 / 256, and six
// terms of its logarithm remain -- and 2^(j / 64): five terms of the exponential.  Good to two steps of the logarithm, as the above.
struct SmTables { double inv[128], log[128], exp[64]; };

__device__ __forceinline__ void sm_tables(SmTables& t, int mode)      // a barrier has to follow
{
    const int k = threadIdx.x;
    if (mode == SM_POWER && k < 128) {
        const double inv = 1.0 / (1.0 + (k + 0.5) * 0x1p-7);
        t.inv[k] = inv;
        t.log[k] = -sm_ln(inv);
    }
    if (mode != SM_LINEAR && k >= 128 && k < 192) t.exp[k - 128] = 2.0 * sm_exp((k - 192) * (0.69314718055994531 / 64));
}
__device__ __forceinline__ double sm_exp(const SmTables& t, double x)
{
    x = fmax(x, -800.0);
    const double k = rint(x * 92.332482616893657);                     // 64 / ln 2
    const double r = fma(k, -1.90821492927058770e-10 / 64, fma(k, -6.93147180369123816e-01 / 64, x));
    double p = fma(r, 1.0 / 120, 1.0 / 24);
    p = fma(r, p, 1.0 / 6);
    p = fma(r, p, 0.5);
    const int i = (int)k;
    const double e = t.exp[i & 63];
    return ldexp(fma(e, fma(r * r, p, r), e), i >> 6);
}
__device__ __forceinline__ double sm_ln(const SmTables& t, float x)
{
    const bool small = x < 0x1p-126f;
    const uint32_t b = __float_as_uint(small ? x * 0x1p32f : x);
    const int i = (int)(b >> 16) & 127;
    const double r = fma((double)__uint_as_float((b & 0x7fffffu) | 0x3f800000u), t.inv[i], -1.0), n = (double)((int)(b >> 23) - (small ? 159 : 127));
    double p = fma(r, -1.0 / 6, 1.0 / 5);
    p = fma(r, p, -1.0 / 4);
    p = fma(r, p, 1.0 / 3);
    p = fma(r, p, -0.5);
    return fma(n, 6.93147180369123816e-01, fma(n, 1.90821492927058770e-10, t.log[i] + fma(r * r, p, r)));
}
__device__ __forceinline__ SmScale sm_scale(const SmTables& t, const SmRule& r, float best)        // for sm_masses
{
    return sm_scale(r, best, [&](double x) { return sm_ln(t, (float)x); });
}
// N masses at once (x: scores, -inf where excluded), without a branch between them: one after the other each waits for its own chain of some
// twenty dependent instructions
template <int N> __device__ __forceinline__ void sm_masses(const SmTables& t, const SmScale& s, const float (&x)[N], double (&m)[N])
{
    bool any = false;
#pragma unroll
    for (int k = 0; k < N; k++) any = any || x[k] > -INFINITY;
    if (__ballot(any) == 0) {                                          // (the same for the wave)
#pragma unroll
        for (int k = 0; k < N; k++) m[k] = 0.0;
        return;
    }
    if (s.mode == SM_LINEAR) {
#pragma unroll
        for (int k = 0; k < N; k++) m[k] = (double)fmaxf(x[k], 0.0f);
        return;
    }
    if (s.mode == SM_POWER) {
#pragma unroll
        for (int k = 0; k < N; k++) m[k] = sm_ln(t, x[k] > -INFINITY ? x[k] : 1.0f);
    } else {
#pragma unroll
        for (int k = 0; k < N; k++) m[k] = (double)(x[k] > -INFINITY ? x[k] : 0.0f);
    }
#pragma unroll
    for (int k = 0; k < N; k++) m[k] = sm_exp(t, m[k] * s.inv_t - s.top);
#pragma unroll
    for (int k = 0; k < N; k++) m[k] = x[k] > -INFINITY ? m[k] : 0.0;
}

// key of the exponential race, ordered as an unsigned integer; 0 = excluded
__device__ __forceinline__ unsigned long long sm_race(const SmScale& s, float score, float u)
{
    if (score == -INFINITY) return 0ull;
    u = u == u ? fminf(fmaxf(u, 0x1p-33f), 1.0f - 0x1p-24f) : 1.0f - 0x1p-24f;
    const double k = sm_log(s, score) - log(-log1p(-(double)u)) + 0.0;
    const unsigned long long b = (unsigned long long)__double_as_longlong(k);
    return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}

// ---- sums of masses that do not depend on their order --------------------------------------------------------------------------------
struct SmSum { unsigned long long hi, lo; };                           // (hi + lo / 2^32) / 2^31, both limbs carry-free up to 2^31 terms
struct SmLimbs { uint32_t hi, lo; };
__device__ __forceinline__ SmLimbs sm_limbs(double m)                  // 0 <= m <= 1
{
    const double a = m * 0x1p31;
    const uint32_t hi = (uint32_t)a;
    return SmLimbs{ hi, (uint32_t)((a - (double)hi) * 0x1p32) };
}
__device__ __forceinline__ double sm_sum_value(SmSum s)
{
    const unsigned long long hi = s.hi + (s.lo >> 32), lo = s.lo & 0xffffffffull;
    return (double)hi * 0x1p-31 + (double)lo * 0x1p-63;
}

// ---- scans of a wave and of a workgroup, in one fixed order ----------------------------------------------------------------------------
// Lane exchange by DPP (row shifts of 16 lanes, then two broadcasts): a shuffle through the LDS crossbar costs a hundred cycles a step, and a
// selection is little else than scans.
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t sm_dpp(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false); }
template <int CTRL, int ROWS> __device__ __forceinline__ unsigned long long sm_dpp(unsigned long long v)
{
    return (unsigned long long)sm_dpp<CTRL, ROWS>((uint32_t)v) | (unsigned long long)sm_dpp<CTRL, ROWS>((uint32_t)(v >> 32)) << 32;
}
template <int CTRL, int ROWS> __device__ __forceinline__ double sm_dpp(double v)
{
    return __longlong_as_double((long long)sm_dpp<CTRL, ROWS>((unsigned long long)__double_as_longlong(v)));
}
__device__ __forceinline__ uint32_t sm_lane(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }
__device__ __forceinline__ unsigned long long sm_lane(unsigned long long v, int lane)
{
    return (unsigned long long)sm_lane((uint32_t)v, lane) | (unsigned long long)sm_lane((uint32_t)(v >> 32), lane) << 32;
}
__device__ __forceinline__ float sm_lane(float v, int lane) { return __uint_as_float(sm_lane(__float_as_uint(v), lane)); }
__device__ __forceinline__ double sm_lane(double v, int lane) { return __longlong_as_double((long long)sm_lane((unsigned long long)__double_as_longlong(v), lane)); }

struct SmAdd { template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return a + b; } };
struct SmMaxOf { template <typename V> __device__ __forceinline__ V operator()(V a, V b) const { return a > b ? a : b; } };

// inclusive scan over the wave (ROWS16: over each row of 16 lanes); lanes without a neighbour see 0, the identity of both operations here
template <bool ROWS16, typename Op, typename V> __device__ __forceinline__ V sm_wave_scan(V v, Op op)
{
    v = op(v, sm_dpp<0x111, 0xf>(v));
    v = op(v, sm_dpp<0x112, 0xf>(v));
    v = op(v, sm_dpp<0x114, 0xf>(v));
    v = op(v, sm_dpp<0x118, 0xf>(v));
    if (!ROWS16) {
        v = op(v, sm_dpp<0x142, 0xa>(v));
        v = op(v, sm_dpp<0x143, 0xc>(v));
    }
    return v;
}

struct SmScratch { unsigned long long a[SM_MAX_WAVES], b[SM_MAX_WAVES], word[6]; };

// inclusive scan over the workgroup; `before` and `total` are the operation over the waves before this one and over all.  lds: 8 bytes a wave
template <typename Op, typename V> __device__ __forceinline__ V sm_block_op(V v, Op op, void* lds, V& before, V& total)
{
    V* part = (V*)lds;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const V inc = sm_wave_scan<false>(v, op);
    __syncthreads();
    if (lane == 63) part[wave] = inc;
    __syncthreads();
    const V p = sm_wave_scan<true>((lane & 15) < waves ? part[lane & 15] : (V)0, op);
    total = sm_lane(p, 15);
    before = wave ? sm_lane(p, wave - 1) : (V)0;
    return op(before, inc);
}
// exclusive prefix sum over the workgroup, and the total
template <typename V> __device__ __forceinline__ V sm_block_scan(V v, void* lds, V& total)
{
    V before;
    return sm_block_op(v, SmAdd(), lds, before, total) - v;
}
// The same for floating sums: handed up one lane (and one wave), not the inclusive sum less the thread's own, which would lose what lies before
// a thread whose own is 2^53 times as large.
__device__ __forceinline__ double sm_block_sum_before(double v, void* lds, double& total)
{
    double before;
    const double prev = sm_dpp<0x138, 0xf>(sm_block_op(v, SmAdd(), lds, before, total));        // one lane up; lane 0: 0
    return (threadIdx.x & 63) ? prev : before;
}
// inclusive maximum over the threads up to this one: sums that rounding made fall, or rise without a mass, are flat again
__device__ __forceinline__ double sm_block_rise(double v, void* lds, double& total)
{
    double before;
    return sm_block_op(v, SmMaxOf(), lds, before, total);
}
__device__ __forceinline__ double sm_block_rise_before(double v, void* lds, double& total)       // ... up to the thread before this one
{
    double before;
    const double inc = sm_block_op(v, SmMaxOf(), lds, before, total);
    const double prev = sm_dpp<0x138, 0xf>(inc);                       // one lane up; lane 0: 0
    return fmax(before, prev);
}
template <typename V> __device__ __forceinline__ V sm_block_max(V v, void* lds)
{
    V before, total;
    sm_block_op(v, SmMaxOf(), lds, before, total);
    return total;
}

// ---- radix selection: histograms of one level, and the bin in which the selection ends -------------------------------------------------
// Bin b of 64 * 2^p lies at sm_slot(b, p) in LDS: the 2^p bins of one lane of the wave that walks them lie 65 apart, so that neither that walk
// nor one in the bins' order meets a bank twice.  In memory, where workgroups merge them, bins lie in the order of the slots; counts of a level
// in their own, so that the bins that hold anything lie close together and a wave's additions to one line are one access (top-k of 3 M 54 ->
// 51 us; top-p's sums of 8 bytes and the race's counts are merged as fast or faster spread out).
// A row of one workgroup keeps the counts above bit 48 of the low limb's sums (at most SM_SHORT terms: 46 bits), one atomic less an element.
#define SM_SLOTS 2080                  // sm_slots(5)
struct SmHist { uint32_t n[SM_SLOTS]; unsigned long long hi[SM_SLOTS], lo[SM_SLOTS]; };
struct SmMerged { uint32_t n[SM_BINS]; unsigned long long hi[SM_BINS], lo[SM_BINS]; };
union SmShortHist { uint32_t n[SM_SLOTS]; struct { unsigned long long hi[SM_SLOTS], lo[SM_SLOTS]; }; };
#define SM_PACK 48
__host__ __device__ constexpr int sm_slots(int p) { return 65 << p; }
__device__ __forceinline__ int sm_slot(int b, int p) { return (b & ((1 << p) - 1)) * 65 + (b >> p); }
__device__ __forceinline__ int sm_nth_slot(int k) { return (k >> 6) * 65 + (k & 63); }

// An element is taken while what lies before it (best first) is less than the target, counted in elements or in mass.
struct SmTake { double target; uint32_t before_n; SmSum before_m; };
struct SmBin { int bin; uint32_t count, total; };

template <bool MASS> __device__ __forceinline__ bool sm_room(const SmTake& t, uint32_t n, unsigned long long hi, unsigned long long lo)
{
    return MASS ? sm_sum_value(SmSum{ t.before_m.hi + hi, t.before_m.lo + lo }) < t.target : (double)(t.before_n + n) < t.target;
}

// The lowest bin with anything in it (a mass, where mass is what counts) whose predecessors (the bins above it) leave room: a wave sums 2^p bins a lane, best first, scans, and does the
// same once more inside the lane it ends in.  Updates take.before_* to the amount above that bin; bin -1: there is none.  All threads call it
// behind a barrier; a barrier has to follow before the histogram or sc is written again.
template <bool MASS, bool PACKED = false>
__device__ SmBin sm_boundary(const uint32_t* hn, const unsigned long long* hhi, const unsigned long long* hlo, int p, SmTake& take, SmScratch& sc)
{
    const unsigned long long low = PACKED ? (1ull << SM_PACK) - 1 : ~0ull;
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x, per = 1 << p;
        uint32_t n = 0;
        unsigned long long hi = 0, lo = 0;
#pragma unroll 8
        for (int k = 0; k < per; k++) {
            const int at = k * 65 + 63 - lane;
            if (!PACKED) n += hn[at];
            if (MASS) { const unsigned long long v = hlo[at]; hi += hhi[at]; lo += v & low; if (PACKED) n += (uint32_t)(v >> SM_PACK); }
        }
        const uint32_t in = sm_wave_scan<false>(n, SmAdd());
        unsigned long long ihi = 0, ilo = 0;
        if (MASS) { ihi = sm_wave_scan<false>(hi, SmAdd()); ilo = sm_wave_scan<false>(lo, SmAdd()); }
        const unsigned long long enter = __ballot((MASS ? (hi | lo) != 0 : n != 0) && sm_room<MASS>(take, in - n, ihi - hi, ilo - lo));
        const uint32_t total = sm_lane(in, 63);
        int bin = -1;
        uint32_t bn = take.before_n, count = 0;
        SmSum bm = take.before_m;
        if (enter) {
            const int l = 63 - __clzll((long long)enter);
            bn += sm_lane(in - n, l);
            if (MASS) { bm.hi += sm_lane(ihi - hi, l); bm.lo += sm_lane(ilo - lo, l); }
            const int at = (per - 1 - lane) * 65 + 63 - l;
            uint32_t n2 = 0;
            unsigned long long hi2 = 0, lo2 = 0, ihi2 = 0, ilo2 = 0;
            if (lane < per) {
                if (!PACKED) n2 = hn[at];
                if (MASS) { hi2 = hhi[at]; lo2 = hlo[at] & low; if (PACKED) n2 = (uint32_t)(hlo[at] >> SM_PACK); }
            }
            const uint32_t in2 = sm_wave_scan<false>(n2, SmAdd());
            if (MASS) { ihi2 = sm_wave_scan<false>(hi2, SmAdd()); ilo2 = sm_wave_scan<false>(lo2, SmAdd()); }
            const SmTake inner = { take.target, bn, bm };
            const int l2 = 63 - __clzll((long long)__ballot((MASS ? (hi2 | lo2) != 0 : n2 != 0) && sm_room<MASS>(inner, in2 - n2, ihi2 - hi2, ilo2 - lo2)));
            bin = ((63 - l) << p) | (per - 1 - l2);
            bn += sm_lane(in2 - n2, l2);
            count = sm_lane(n2, l2);
            if (MASS) { bm.hi += sm_lane(ihi2 - hi2, l2); bm.lo += sm_lane(ilo2 - lo2, l2); }
        }
        if (lane == 0) {
            sc.word[0] = (unsigned long long)(long long)bin;
            sc.word[1] = bn;
            sc.word[2] = (unsigned long long)count | (unsigned long long)total << 32;
            sc.word[3] = bm.hi;
            sc.word[4] = bm.lo;
        }
    }
    __syncthreads();
    const SmBin b = { (int)(long long)sc.word[0], (uint32_t)sc.word[2], (uint32_t)(sc.word[2] >> 32) };
    take.before_n = (uint32_t)sc.word[1];
    take.before_m = SmSum{ sc.word[3], sc.word[4] };
    return b;
}

// of `count` elements of equal key behind what is before them: how many are taken (at least one, by the choice of the bin)
template <bool MASS> __device__ __forceinline__ uint32_t sm_ties(const SmTake& take, uint32_t count, double mass)
{
    if (!MASS) {
        const double left = take.target - (double)take.before_n;
        return left >= (double)count ? count : (uint32_t)ceil(left);
    }
    const SmLimbs l = sm_limbs(mass);
    const SmSum one = { l.hi, l.lo };
    uint32_t lo = 1, hi = count;                                       // the first j (from 0) that finds no room
    while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (sm_room<true>(take, 0, mid * one.hi, mid * one.lo)) lo = mid + 1; else hi = mid;
    }
    return lo;
}
// every element of the boundary bin is taken: the selection needs no further level
template <bool MASS> __device__ __forceinline__ bool sm_whole_bin(const SmTake& take, uint32_t count)
{
    return count == 1 || (!MASS && take.target - (double)take.before_n >= (double)count);
}

// What passes the filters: scores above thr, and those equal to it up to index `end` (thr = -inf, end = 0: all but the excluded)
struct SmKept { float thr; uint32_t end; };
#define SM_ALL 0xffffffffu
__device__ __forceinline__ bool sm_in(const SmKept& k, float x, uint32_t i) { return x > k.thr || (x == k.thr && i < k.end); }

// min-p as a cut of the scores: the smallest one whose mass is at least min_p of the best one's (the mass grows with the score), looked for
// among the ordered integers from `lo` to `hi`, the best one's, that `of` makes scores.  Every wave for itself, 64 probes a round.
template <typename Of> __device__ __forceinline__ float sm_min_p(const SmRule& rule, uint32_t lo, uint32_t hi, const Of& of)
{
    const SmScale s = sm_scale(rule, of(hi));
    const double least = rule.min_p * sm_mass(s, of(hi));
    const uint32_t lane = threadIdx.x & 63;
    while (lo < hi) {
        const uint32_t gap = (hi - lo) / 64 + 1;
        const unsigned long long p = (unsigned long long)lo + (unsigned long long)lane * gap;
        const unsigned long long ok = __ballot(p >= hi || sm_mass(s, of((uint32_t)p)) >= least);
        const uint32_t f = ok ? (uint32_t)__ffsll((long long)ok) - 1 : 64;
        const unsigned long long nhi = (unsigned long long)lo + (unsigned long long)f * gap;
        if (f) lo += (f - 1) * gap + 1;
        hi = nhi < hi ? (uint32_t)nhi : hi;
    }
    return of(lo);
}
__device__ __forceinline__ void sm_min_p(const SmRule& rule, float best, SmKept& kept)
{
    const float thr = sm_min_p(rule, rule.mode == SM_LOGITS ? 1u : 0x80000001u /*the least weight*/, sm_order(best), [](uint32_t k) { return sm_unorder(k); });
    if (thr > kept.thr) kept = SmKept{ thr, SM_ALL };
}

// ---- approximate race keys ---------------------------------------------------------------------------------------------------------------
// The n-th largest race key is found from approximate keys in 32 bits: k ~ log2(mass) - log2(-ln(1 - u)).  Levels of histograms of the ordered
// float bound it to a bin; what lies above the bin by more than twice the approximation's error wins, what lies below by as much loses, and
// the few in the zone between are ranked by their exact 64-bit keys.
//
// Error of k, with the logarithm instruction good to a step of its result or, for arguments next to one, to 2^-22:
//   -ln(1 - u): below u = 2^-6 a series, good to 2^-21 relative.  From there on log2(1 - u) is at least 2^-5.5 and off by the instruction's
//   2^-22 and by the rounding of 1 - u (2^-25, i.e. 2^-23.5 in the logarithm): 2^-16 relative, so that its own logarithm is off by 2^-15.4;
//   that logarithm (at most 33), log2(mass) (at most |k| + 33), slope and products round by 2^-21 of them at most: 2^-15.9 + |k| 2^-21;
//   the logarithm of a weight next to one: 2^-22 of the slope.
// Together less than 2^-14.6 + |k| 2^-21 + slope 2^-22.  sm_margin allows twice each of the three and more.
__device__ __forceinline__ float sm_log2(float x)                      // x > 0, subnormals too
{
    const bool small = x < 0x1p-100f;
    return __builtin_amdgcn_logf(small ? x * 0x1p64f : x) - (small ? 64.0f : 0.0f);
}
__device__ __forceinline__ float sm_margin(float k, float slope) { return 0x1p-13f + fabsf(k) * 0x1p-18f + slope * 0x1p-21f; }
__device__ __forceinline__ float sm_slope(const SmRule& r) { return (float)((r.mode == SM_LOGITS ? 1.4426950408889634 : 1.0) * r.inv_t); }

// approximate key of a candidate.  `slope`: log2(e) / T or 1 / T in 32 bits
__device__ __forceinline__ float sm_race32(bool logits, float slope, float x, float u)
{
    u = u == u ? fminf(fmaxf(u, 0x1p-33f), 1.0f - 0x1p-24f) : 1.0f - 0x1p-24f;
    const float a = (logits ? x : sm_log2(x)) * slope;
    const float e = u < 0x1p-6f ? u * (1.0f + u * (0.5f + u * (0.33333333f + u * 0.25f))) : -0.69314718f * __builtin_amdgcn_logf(1.0f - u);
    const float k = fminf(fmaxf(a, -3e38f), 3e38f) - __builtin_amdgcn_logf(e);
    return k + 0.0f;
}

// zone of the n-th key given that its approximation lies in [lo, hi]: ordered keys below zone.lo lose, above zone.hi win
struct SmZone { uint32_t lo, hi; };
__device__ __forceinline__ SmZone sm_zone(uint32_t lo, uint32_t hi, float slope)
{
    const float klo = sm_unorder(lo), khi = sm_unorder(hi);
    const uint32_t a = sm_order(klo - 2.0f * sm_margin(klo, slope)), b = sm_order(khi + 2.0f * sm_margin(khi, slope));
    return SmZone{ a ? a : 1u, b };
}

// (out of line: sixteen of them inlined, with their constants, spill two thousand registers)
__device__ __attribute__((noinline)) unsigned long long sm_race_call(SmScale s, float x, float u) { return sm_race(s, x, u); }

// ---- short rows: one workgroup per row, EPT consecutive elements of a thread in registers ----------------------------------------------
// One CU works on a row, so that every instruction an element costs is 0.1 us for 15 k of them: scores are kept as floats (-inf: excluded)
// and compared as they are, and a level of a selection spreads the range that is left evenly over its bins (floats of either sign linearly,
// weights by their bits, i.e. by their logarithm).  A level leaves some tens of elements then, which a wave ranks.

// Radix selection.  at(k, w): whether element threadIdx.x * EPT + k is a candidate, and its word.  Ends with one element in the bin or one
// word: lo is then the bin's lowest word, take.before_* what lies above it, and the result its count.
template <int TPB, int EPT, typename At>
__device__ __forceinline__ SmBin sm_select_short(const At& at_, SmTake& take, SmShortHist& h, SmScratch& sc, unsigned long long& lo)
{
    unsigned long long prefix = 0;
    int shift = 64;
    SmBin b = { -1, 0, 0 };
    while (shift > 0) {
        const int width = shift >= 11 ? 11 : shift < 6 ? 6 : shift, at = shift > width ? shift - width : 0, p = width - 6;
        __syncthreads();
        for (int i = threadIdx.x; i < sm_slots(p); i += TPB) h.n[i] = 0;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < EPT; k++) {
            unsigned long long w;
            if (!at_(k, w) || (shift < 64 && (w >> shift) != prefix)) continue;
            atomicAdd(&h.n[sm_slot((int)((w >> at) & ((1ull << (shift - at)) - 1)), p)], 1u);
        }
        __syncthreads();
        b = sm_boundary<false>(h.n, nullptr, nullptr, p, take, sc);
        if (b.bin < 0) { lo = 0; return b; }                           // no candidate at all
        prefix = (prefix << (shift - at)) | (unsigned)b.bin;
        shift = at;
        if (b.count == 1) break;
    }
    lo = prefix << shift;
    return b;
}

// index of the n-th (from 1) flagged element
template <int EPT> __device__ __forceinline__ uint32_t sm_nth_short(const bool (&flag)[EPT], uint32_t n, SmScratch& sc)
{
    uint32_t c = 0, total;
#pragma unroll
    for (int k = 0; k < EPT; k++) c += flag[k];
    uint32_t at = sm_block_scan<uint32_t>(c, sc.a, total);
#pragma unroll
    for (int k = 0; k < EPT; k++) if (flag[k] && ++at == n) sc.word[0] = threadIdx.x * EPT + k;
    __syncthreads();
    return (uint32_t)sc.word[0];
}

// four consecutive scores from i on; what lies behind V is NaN, which is never drawn
template <typename T> __device__ __forceinline__ LgVec4<T> sm_load4(const T* x, long long i, long long V, bool vec)
{
    if (vec && i + 4 <= V) return *(const LgVec4<T>*)(x + i);
    LgVec4<T> v;
#pragma unroll
    for (int k = 0; k < 4; k++) v.v[k] = i + k < V ? x[i + k] : lg_from_float<T>(__uint_as_float(0x7fc00000u));
    return v;
}
template <typename T> __device__ __forceinline__ bool sm_aligned(const T* x) { return (uintptr_t)x % (4 * sizeof(T)) == 0; }

// a boundary bin of at most 64 elements, ranked by a wave; or those and up to 63 above them
struct SmFew { unsigned long long hi[64], lo[64]; double sum[128]; float x[128], u[128]; uint32_t index[128], order[64], ahead[128]; };
union SmShortLds { SmShortHist hist; SmFew few; struct { unsigned long long rank[SM_BINS]; uint32_t index[SM_BINS]; } zone; };

// Bins of the numbers from lo to hi, and the one that is wanted (-1: all of them).  Grows with x; lo and hi are never in one bin.
struct SmBins {
    float lo, hi, f, s;
    uint32_t low;
    int down, want;
    bool linear;
    __device__ __forceinline__ int of(float x) const
    {
        if (!linear) return (int)((__float_as_uint(x) - low) >> down);
        return (int)fminf(fmaxf((x * f - lo * f) * s, 0.0f), (float)(SM_BINS - 1));
    }
    __device__ __forceinline__ bool in(float x) const { return x >= lo && x <= hi && (want < 0 || of(x) == want); }
};
__device__ __forceinline__ SmBins sm_bins(bool linear, float lo, float hi)
{
    SmBins b = { lo, hi, 1.0f, 0.0f, __float_as_uint(lo), 0, -1, linear };
    if (linear) {
        if (hi - lo == INFINITY) b.f = 0.25f;
        b.s = (float)SM_BINS / (hi * b.f - lo * b.f);                  // (infinite for a range below 1e-35: lo is then in bin 0, the others in the last)
    } else {
        const uint32_t range = __float_as_uint(hi) - b.low;
        b.down = range >> 11 ? 21 - __clz(range) : 0;
    }
    return b;
}

// the smallest and the largest of the numbers that are in (inf and -inf: none is)
template <int EPT, typename In> __device__ __forceinline__ void sm_range_short(const float (&x)[EPT], const In& in, SmScratch& sc, float& lo, float& hi)
{
    float a = INFINITY, b = -INFINITY;
#pragma unroll
    for (int k = 0; k < EPT; k++) if (in(k)) { a = fminf(a, x[k]); b = fmaxf(b, x[k]); }
    const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
    uint32_t low = sm_wave_scan<false>(~sm_order(a), SmMaxOf()), high = sm_wave_scan<false>(sm_order(b), SmMaxOf());
    __syncthreads();
    if (lane == 63) sc.a[threadIdx.x >> 6] = (unsigned long long)high << 32 | low;
    __syncthreads();
    const unsigned long long part = (lane & 15) < waves ? sc.a[lane & 15] : 0ull;
    low = sm_lane(sm_wave_scan<true>((uint32_t)part, SmMaxOf()), 15);
    high = sm_lane(sm_wave_scan<true>((uint32_t)(part >> 32), SmMaxOf()), 15);
    lo = sm_unorder(~low);
    hi = sm_unorder(high);
}

// Where a selection of the candidates x (> -inf; from lo to hi) ends: the bins that are left hold at most `small` elements, or only equal ones (lo == hi).
// take.before_* is what lies above them, the result their count and the number of candidates (0: there are none).
template <bool MASS, int TPB, int EPT>
__device__ __forceinline__ SmBin sm_find_short(const float (&x)[EPT], const double* mass /*LDS, [EPT][TPB], at most one each*/, bool linear, float lo, float hi, SmTake& take, uint32_t small,
                               SmShortHist& h, SmScratch& sc, SmBins& bins)
{
    uint32_t candidates = 0;
    if (!(lo <= hi)) return SmBin{ -1, 0, 0 };
    for (int level = 0; ; level++) {
        if (level) sm_range_short<EPT>(x, [&](int k) { return x[k] > -INFINITY && bins.in(x[k]); }, sc, lo, hi);
        bins = sm_bins(linear, lo, hi);
        for (int i = threadIdx.x; i < SM_SLOTS; i += TPB) { if (MASS) { h.hi[i] = 0; h.lo[i] = 0; } else h.n[i] = 0; }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < EPT; k++) {
            if (!(x[k] >= lo && x[k] <= hi)) continue;
            const int i = sm_slot(bins.of(x[k]), 5);
            if (MASS) {
                const SmLimbs m = sm_limbs(mass[k * TPB + threadIdx.x]);
                if (m.hi) atomicAdd(&h.hi[i], (unsigned long long)m.hi);
                atomicAdd(&h.lo[i], (unsigned long long)m.lo | 1ull << SM_PACK);
            } else atomicAdd(&h.n[i], 1u);
        }
        __syncthreads();
        SmBin b = sm_boundary<MASS, MASS>(h.n, h.hi, h.lo, 5, take, sc);
        if (level == 0) candidates = b.total;
        b.total = candidates;
        if (b.bin < 0) return b;
        bins.want = b.bin;
        if (b.count <= small || lo == hi) return b;
        __syncthreads();                                               // (lo and hi are never in one bin: every round has fewer)
    }
}

// what a top-k (MASS false) or top-p with that target leaves of the candidates
template <bool MASS, int TPB, int EPT>
__device__ __forceinline__ SmKept sm_filter_short(const float (&x)[EPT], const double* mass, bool linear, float lo, float hi, SmTake take, SmShortLds& h, SmScratch& sc)
{
    SmBins bins;
    const SmBin bin = sm_find_short<MASS, TPB, EPT>(x, mass, linear, lo, hi, take, 64, h.hist, sc, bins);
    if (bin.count > 64) {                                              // equal ones: the first of them
        bool tie[EPT];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < EPT; k++) {
            tie[k] = x[k] == bins.lo;
            if (MASS && tie[k]) sc.word[5] = (unsigned long long)__double_as_longlong(mass[k * TPB + threadIdx.x]);        // (all the same)
        }
        __syncthreads();
        const uint32_t ties = sm_ties<MASS>(take, bin.count, MASS ? __longlong_as_double((long long)sc.word[5]) : 0.0);
        return SmKept{ bins.lo, ties < bin.count ? sm_nth_short<EPT>(tie, ties, sc) + 1 : SM_ALL };
    }
    __syncthreads();
    if (threadIdx.x == 0) sc.word[5] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < EPT; k++)
        if (bins.in(x[k])) {
            const uint32_t a = (uint32_t)atomicAdd(&sc.word[5], 1ull);
            h.few.x[a] = x[k];
            h.few.index[a] = threadIdx.x * EPT + k;
            if (MASS) { const SmLimbs m = sm_limbs(mass[k * TPB + threadIdx.x]); h.few.hi[a] = m.hi; h.few.lo[a] = m.lo; }
        }
    __syncthreads();
    if (threadIdx.x < 64) {
        const uint32_t n = bin.count, l = threadIdx.x, i = l < n ? h.few.index[l] : 0u;
        const float mine = l < n ? h.few.x[l] : 0.0f;
        uint32_t ahead = 0;
        for (uint32_t c = 0; c < n; c++) { const float other = sm_lane(mine, (int)c); ahead += other > mine || (other == mine && sm_lane(i, (int)c) < i); }
        if (l < n) h.few.order[ahead] = l;
        __threadfence_block();                                         // (one wave: in order, and the compiler is told)
        const uint32_t a = l < n ? h.few.order[l] : 0u;                // the l-th best
        bool room;
        if (MASS) {
            const SmSum m = { l < n ? h.few.hi[a] : 0ull, l < n ? h.few.lo[a] : 0ull };
            room = sm_room<true>(take, 0, sm_wave_scan<false>(m.hi, SmAdd()) - m.hi, sm_wave_scan<false>(m.lo, SmAdd()) - m.lo);
        } else room = sm_room<false>(take, l, 0, 0);
        const unsigned long long taken = __ballot(l < n && room);
        const int e = taken ? 63 - __clzll((long long)taken) : 0;      // (the first one always is)
        if ((int)l == e) { sc.word[0] = __float_as_uint(h.few.x[a]); sc.word[1] = h.few.index[a]; }
    }
    __syncthreads();
    return SmKept{ __uint_as_float((uint32_t)sc.word[0]), (uint32_t)sc.word[1] + 1 };
}

// A row from beginning to end in one launch: scores in registers, masses in LDS (worked out once), and one histogram level a filter as a rule.
// 10 k scores: a plain draw 10.4 us, behind top-k 50 and top-p 10, behind top-p 21, 500 distinct 18; a launch alone is 5.  64 rows take what one takes (a compute
// unit each).
template <typename T, int TPB, int EPT, bool DISTINCT>
__global__ void __launch_bounds__(TPB) sample_short_kernel(const T* __restrict__ scores, long long sstride, const float* __restrict__ u, long long ustride,
                                                            int V, long long n, SmRule rule, const uint32_t* __restrict__ names /*nullable [R, V]*/,
                                                            long long* __restrict__ out)
{
    __shared__ double mass[TPB * EPT];                                 // element k of thread t at k * TPB + t; at the end the cumulative ones
    __shared__ SmShortLds h;
    __shared__ SmTables tables;
    __shared__ uint32_t won[DISTINCT ? TPB * EPT / 32 : 1];
    __shared__ SmScratch sc;
    const long long r = blockIdx.x;
    const T* row = scores + r * sstride;
    const bool logits = rule.mode == SM_LOGITS;
    const float floor = sm_floor(rule);
    u += r * ustride;
    out += r * n;
    if (names) names += r * V;
    auto name = [&](uint32_t i) { return names ? (long long)names[i] : (long long)i; };          // of element i, where the row is what a filter left
    const int i0 = threadIdx.x * EPT;
    const bool filtered = (rule.top_k > 0 && rule.top_k < V) || rule.top_p < 1.0;
    float x[EPT], most = -INFINITY, lowest = -INFINITY;
    {
        LgVec4<T> v[EPT / 4];
#pragma unroll
        for (int k = 0; k < EPT / 4; k++) v[k] = sm_load4(row, i0 + 4 * k, V, sm_aligned(row));
        sm_tables(tables, rule.mode);                                  // (the first scan is the barrier)
#pragma unroll
        for (int k = 0; k < EPT; k++) { x[k] = sm_score(v[k / 4].v[k % 4], floor); most = fmaxf(most, x[k]); }
    }
    if (filtered) sm_range_short<EPT>(x, [&](int k) { return x[k] > -INFINITY; }, sc, lowest, most);
    else most = sm_unorder(sm_block_max(sm_order(most), sc.a));
    if (most == -INFINITY) {                                           // nothing to draw from
        for (long long j = (long long)blockIdx.y * TPB + threadIdx.x; j < n; j += (long long)gridDim.y * TPB) out[j] = -1;
        return;
    }
    const SmScale scale = sm_scale(tables, rule, most);
    // masses, once: linear ones by a power of two below one
    const double unit = rule.mode == SM_LINEAR ? scale.shift : 1.0;
    auto masses = [&]() {
#pragma unroll
        for (int k = 0; k < EPT; k += 4) {
            const float four[4] = { x[k], x[k + 1], x[k + 2], x[k + 3] };
            double m[4];
            sm_masses(tables, scale, four, m);
#pragma unroll
            for (int j = 0; j < 4; j++) mass[(k + j) * TPB + threadIdx.x] = m[j] * unit;
        }
    };
    if (rule.top_k > 0 && rule.top_k <= 64 && rule.top_k < V) {
        // What such a top-k leaves is the work of one wave: the bin in which it ends and what lies above are listed in index order and ranked by
        // all threads; the first wave applies the other filters, best first, and sums or ranks (10 k scores: 1 behind top-k 50 and
        // top-p 24 -> 10 us, 10 distinct 31 -> 15, behind top-k alone 20 -> 15; 300 scores 11.5 -> 7.2, 15.5 -> 11, 10.3 -> 10.7)
        SmTake take = { (double)rule.top_k, 0, { 0, 0 } };
        SmBins bins;
        const SmBin bin = sm_find_short<false, TPB, EPT>(x, mass, logits, lowest, most, take, 64, h.hist, sc, bins);
        if (bin.count <= 64) {                                         // (else equal numbers)
            uint32_t in = 0, found;
#pragma unroll
            for (int k = 0; k < EPT; k++) if (x[k] >= bins.lo && bins.of(x[k]) >= bins.want) in |= 1u << k;
            uint32_t at = sm_block_scan<uint32_t>(__popc(in), sc.a, found);          // at most 63 + 64
#pragma unroll
            for (int k = 0; k < EPT; k++) if ((in >> k) & 1) {
                    h.few.x[at] = x[k];
                    if (DISTINCT) h.few.u[at] = u[i0 + k];
                    h.few.index[at++] = i0 + k;
                }
            if (threadIdx.x < 128) { h.few.ahead[threadIdx.x] = 0; h.few.sum[threadIdx.x] = 0.0; }
            __syncthreads();
            {
                constexpr uint32_t PARTS = TPB / 128;                  // threads that share an element's comparisons
                const uint32_t a = threadIdx.x % 128, each = (found + PARTS - 1) / PARTS, from = threadIdx.x / 128 * each;
                if (a < found) {
                    const float mine = h.few.x[a];
                    uint32_t ahead = 0;
#pragma unroll 4
                    for (uint32_t c = from; c < found && c < from + each; c++) ahead += h.few.x[c] > mine || (h.few.x[c] == mine && c < a);
                    if (ahead) atomicAdd(&h.few.ahead[a], ahead);
                }
            }
            __syncthreads();
            if (threadIdx.x < 64) {
                const uint32_t l = threadIdx.x, K = found < (uint32_t)rule.top_k ? found : (uint32_t)rule.top_k;
                for (uint32_t a = l; a < found; a += 64) if (h.few.ahead[a] < K) h.few.order[h.few.ahead[a]] = a;
                __threadfence_block();                                 // (one wave: in order, and the compiler is told)
                const uint32_t a = l < K ? h.few.order[l] : 0u;        // the l-th best
                const float z[1] = { l < K ? h.few.x[a] : -INFINITY };
                double m[1];
                sm_masses(tables, scale, z, m);
                bool keep = l < K;
                if (rule.top_p < 1.0) {
                    const SmLimbs one = sm_limbs(m[0] * unit);
                    const unsigned long long hi = sm_wave_scan<false>((unsigned long long)one.hi, SmAdd()), lo = sm_wave_scan<false>((unsigned long long)one.lo, SmAdd());
                    const SmTake part = { rule.top_p * sm_sum_value(SmSum{ sm_lane(hi, 63), sm_lane(lo, 63) }), 0, { 0, 0 } };
                    keep = keep && sm_room<true>(part, 0, hi - one.hi, lo - one.lo);
                }
                if (rule.min_p > 0.0) keep = keep && m[0] >= rule.min_p * sm_lane(m[0], 0);
                h.few.ahead[l] = 0;
                h.few.ahead[l + 64] = 0;
                __threadfence_block();
                if (DISTINCT) {
                    uint32_t ahead = 0;
                    if (__popcll(__ballot(keep)) > n) {                // (else all of them win)
                        const unsigned long long key = keep ? sm_race_call(scale, z[0], h.few.u[a]) : 0ull;
                        for (uint32_t c = 0; c < K; c++) { const unsigned long long other = sm_lane(key, (int)c); ahead += other > key || (other == key && sm_lane(a, (int)c) < a); }
                    }
                    if (keep && ahead < n) h.few.ahead[a] = 1;
                    __threadfence_block();
                    // in index order, two a lane
                    const uint32_t w0 = h.few.ahead[2 * l], w1 = h.few.ahead[2 * l + 1], upto = sm_wave_scan<false>(w0 + w1, SmAdd());
                    if (w0) out[upto - w0 - w1] = name(h.few.index[2 * l]);
                    if (w1) out[upto - w1] = name(h.few.index[2 * l + 1]);
                    if (l == 63) sc.word[0] = upto;
                } else {
                    if (keep) h.few.sum[a] = m[0];
                    __threadfence_block();
                    const double m0 = h.few.sum[2 * l], m1 = h.few.sum[2 * l + 1], upto = sm_wave_scan<false>(m0 + m1, SmAdd()), before = sm_dpp<0x138, 0xf>(upto);
                    const double c0 = m0 > 0.0 ? before + m0 : 0.0, c1 = m1 > 0.0 ? fmax(c0, before + (m0 + m1)) : c0;        // rise with a mass only
                    const double risen = sm_dpp<0x138, 0xf>(sm_wave_scan<false>(c1, SmMaxOf()));
                    h.few.sum[2 * l] = fmax(risen, c0);
                    h.few.sum[2 * l + 1] = fmax(risen, c1);
                    const unsigned long long b0 = __ballot(m0 > 0.0), b1 = __ballot(m1 > 0.0);
                    const int l0 = 2 * (63 - (b0 ? __clzll((long long)b0) : 64)), l1 = 2 * (63 - (b1 ? __clzll((long long)b1) : 64)) + 1;
                    if (l == 63) { sc.word[0] = (unsigned long long)__double_as_longlong(upto); sc.word[1] = (unsigned long long)(l0 > l1 ? l0 : l1); }
                }
            }
            __syncthreads();
            if (DISTINCT) {
                for (long long j = (long long)sc.word[0] + threadIdx.x; j < n; j += TPB) out[j] = -1;
            } else {
                const double total = __longlong_as_double((long long)sc.word[0]);
                const uint32_t last = (uint32_t)sc.word[1];
                for (long long j = (long long)blockIdx.y * TPB + threadIdx.x; j < n; j += (long long)gridDim.y * TPB) {
                    const float uj = u[j];
                    const double t = (uj > 0.0f ? (double)uj : 0.0) * total;
                    uint32_t lo = uj >= 1.0f ? last : 0, hi = last;    // the first sum that passes t, or the last one
                    while (lo < hi) { const uint32_t mid = (lo + hi) >> 1; if (h.few.sum[mid] > t) hi = mid; else lo = mid + 1; }
                    out[j] = name(h.few.index[lo]);
                }
            }
            return;
        }
    }
    // filters: an element that one of them drops becomes -inf
    for (int pass = 0; pass < 2; pass++) {
        SmTake take = { 0.0, 0, { 0, 0 } };
        SmKept left;
        if (pass == 0) {
            if (rule.top_k <= 0 || rule.top_k >= V) continue;
            take.target = (double)rule.top_k;
            left = sm_filter_short<false, TPB, EPT>(x, mass, logits, lowest, most, take, h, sc);
            lowest = left.thr;
        } else {
            if (rule.top_p >= 1.0) continue;
            SmSum mine = { 0, 0 }, total;
            masses();
#pragma unroll
            for (int k = 0; k < EPT; k++) { const SmLimbs m = sm_limbs(mass[k * TPB + threadIdx.x]); mine.hi += m.hi; mine.lo += m.lo; }
            sm_block_scan<unsigned long long>(mine.hi, sc.a, total.hi);
            sm_block_scan<unsigned long long>(mine.lo, sc.b, total.lo);
            take.target = rule.top_p * sm_sum_value(total);
            left = sm_filter_short<true, TPB, EPT>(x, mass, logits, lowest, most, take, h, sc);
        }
#pragma unroll
        for (int k = 0; k < EPT; k++) if (!sm_in(left, x[k], (uint32_t)(i0 + k))) x[k] = -INFINITY;
    }
    if (rule.min_p > 0.0) {
        SmKept kept = { -INFINITY, 0u };
        sm_min_p(rule, most, kept);
#pragma unroll
        for (int k = 0; k < EPT; k++) if (!(x[k] >= kept.thr)) x[k] = -INFINITY;
    }
    if (DISTINCT) {
        float race[EPT];                                               // approximate keys; -inf: not a candidate
        uint32_t wins = 0;
        const float slope = sm_slope(rule);
#pragma unroll
        for (int k = 0; k < EPT / 4; k++) {                            // (loads first)
            const LgVec4<float> four = sm_load4(u, i0 + 4 * k, V, sm_aligned(u));
#pragma unroll
            for (int j = 0; j < 4; j++) race[4 * k + j] = four.v[j];
        }
#pragma unroll
        for (int k = 0; k < EPT; k++) race[k] = x[k] > -INFINITY ? sm_race32(logits, slope, x[k], race[k]) : -INFINITY;
        float rlo, rhi;
        sm_range_short<EPT>(race, [&](int k) { return race[k] > -INFINITY; }, sc, rlo, rhi);
        SmTake take = { (double)n, 0, { 0, 0 } };
        SmBins bins;
        const SmBin bin = sm_find_short<false, TPB, EPT>(race, nullptr, true, rlo, rhi, take, 64, h.hist, sc, bins);
        float zlo = -INFINITY, zhi = -INFINITY;                        // nothing to rank where everything wins
        const bool ranked = bin.total > (uint32_t)n;
        if (ranked) {
            sm_range_short<EPT>(race, [&](int k) { return bins.in(race[k]); }, sc, zlo, zhi);
            zlo -= 2.0f * sm_margin(zlo, slope);
            zhi += 2.0f * sm_margin(zhi, slope);
        }
        __syncthreads();
        if (threadIdx.x == 0) sc.word[5] = 0;
        for (int i = threadIdx.x; i < TPB * EPT / 32; i += TPB) won[i] = 0;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < EPT; k++) {
            if (race[k] > zhi) wins |= 1u << k;
            else if (ranked && race[k] >= zlo) {
                const uint32_t at = (uint32_t)atomicAdd(&sc.word[5], 1ull);
                if (at < SM_BINS) h.zone.index[at] = i0 + k;
            }
        }
        uint32_t sure;
        sm_block_scan<uint32_t>(__popc(wins), sc.a, sure);
        const uint32_t found = (uint32_t)sc.word[5], room = (uint32_t)n > sure ? (uint32_t)n - sure : 0;
        if (found <= SM_BINS) {
            for (uint32_t a = threadIdx.x; a < found; a += TPB) {
                const uint32_t i = h.zone.index[a];
                h.zone.rank[a] = sm_race_call(scale, sm_score(row[i], floor), u[i]);
            }
            __syncthreads();
            for (uint32_t a = threadIdx.x; a < found; a += TPB) {
                const unsigned long long mine = h.zone.rank[a];
                const uint32_t i = h.zone.index[a];
                uint32_t ahead = 0;
                for (uint32_t c = 0; c < found; c++) ahead += h.zone.rank[c] > mine || (h.zone.rank[c] == mine && h.zone.index[c] < i);
                if (ahead < room) atomicOr(&won[i >> 5], 1u << (i & 31));
            }
            __syncthreads();
            wins |= (won[i0 >> 5] >> (i0 & 31)) & ((1u << EPT) - 1);
        } else {
            // many elements next to the border (equal numbers, or a slope that spreads nothing): radix selection of their exact keys
            unsigned long long *mine = (unsigned long long*)mass + threadIdx.x, elo;        // (the masses are done)
#pragma unroll
            for (int k = 0; k < EPT; k++) mine[k * TPB] = race[k] > -INFINITY && race[k] >= zlo && race[k] <= zhi ? sm_race_call(scale, x[k], u[i0 + k]) : 0ull;
            SmTake left = { (double)room, 0, { 0, 0 } };
            const SmBin e = sm_select_short<TPB, EPT>([&](int k, unsigned long long& w) { w = mine[k * TPB]; return w != 0ull; }, left, h.hist, sc, elo);
            const uint32_t ties = e.bin < 0 ? 0 : e.count == 1 ? 1 : sm_ties<false>(left, e.count, 0.0);
            uint32_t last = SM_ALL;
            if (ties < e.count) {
                bool tie[EPT];
                __syncthreads();
#pragma unroll
                for (int k = 0; k < EPT; k++) tie[k] = mine[k * TPB] == elo;
                last = sm_nth_short<EPT>(tie, ties, sc);
            }
            if (e.bin >= 0)
#pragma unroll
                for (int k = 0; k < EPT; k++) {
                    const unsigned long long w = mine[k * TPB];
                    if (w != 0 && (w > elo || (w == elo && (uint32_t)(i0 + k) <= last))) wins |= 1u << k;
                }
        }
        uint32_t total;
        long long at = sm_block_scan<uint32_t>(__popc(wins), sc.a, total);
#pragma unroll
        for (int k = 0; k < EPT; k++) if ((wins >> k) & 1) out[at++] = name(i0 + k);
        for (long long j = (long long)total + threadIdx.x; j < n; j += TPB) out[j] = -1;
    } else {
        double m[EPT], sum = 0.0, total, most_sum;
        uint32_t last = 0;
        if (rule.top_p >= 1.0) masses();
#pragma unroll
        for (int k = 0; k < EPT; k++) m[k] = x[k] > -INFINITY ? mass[k * TPB + threadIdx.x] : 0.0;
#pragma unroll
        for (int k = 0; k < EPT; k++) {
            sum += m[k];
            if (m[k] > 0.0) last = (uint32_t)(i0 + k) + 1;
        }
        // cumulative masses that rise at elements with a mass only, and never fall (a sum along the lanes and one along a thread's elements
        // round differently): the search then ends at an element that can be drawn
        const double before = sm_block_sum_before(sum, sc.a, total);
        last = sm_block_max(last, sc.b);
        double at = before, high = 0.0;
#pragma unroll
        for (int k = 0; k < EPT; k++) { at += m[k]; if (m[k] > 0.0) high = fmax(high, at); }
        high = sm_block_rise_before(high, sc.a, most_sum);
        at = before;
#pragma unroll
        for (int k = 0; k < EPT; k++) { at += m[k]; if (m[k] > 0.0) high = fmax(high, at); mass[k * TPB + threadIdx.x] = high; }
        __syncthreads();
        for (long long j = (long long)blockIdx.y * TPB + threadIdx.x; j < n; j += (long long)gridDim.y * TPB) {         // (blockIdx.y: its share of the draws)
            const float uj = u[j];
            const double t = (uj > 0.0f ? (double)uj : 0.0) * total;
            uint32_t lo = uj >= 1.0f ? last - 1 : 0, hi = last - 1;    // first element whose sum passes t; from one on the last one with a mass
            while (lo < hi) { const uint32_t mid = (lo + hi) >> 1; if (mass[mid % EPT * TPB + mid / EPT] > t) hi = mid; else lo = mid + 1; }
            out[j] = name(lo);
        }
    }
}

// ---- long rows: B workgroups per row ---------------------------------------------------------------------------------------------------
// Every step is one launch over (row, workgroup); the last workgroup of a row to finish a step (SmRowState::ticket) draws its conclusion and
// leaves it in the row's state for the next launch.
#define SM_LTPB 1024
#define SM_RBITS1 12                   // levels of the race's approximate keys: 12 bits, then 10 (a finer second level costs more to merge than it saves to rank)
#define SM_RBITS2 10
#define SM_RBINS (1 << SM_RBITS1)
#define SM_TILE 8192                   // elements per workgroup step of the race's last pass: 128 words of winners
#define SM_STILE 4096                  // elements per tile of prefix sums
#define SM_GROUP 16                    // elements per stored prefix
#define SM_STEPS 12

struct SmRowState {                    // (sm_begin_kernel knows where kept and before are)
    SmKept kept, before;               // what passes the filters; ... before the selection under way
    SmTake take;
    double total, top;                 // with replacement: total mass of the kept; the largest l
    unsigned long long sure;           // race: winners
    float best, least;                 // largest score; least score that passes min-p
    uint32_t prefix, ties, ended, cut, zone_lo, zone_hi, candidates, end_tile /*with replacement: the last tile with a mass*/;
    uint32_t ticket[SM_STEPS], sub[16][32];       // (sub: one of 32 words, 128 bytes apart)
};

struct SmWork {                        // workspace of a call
    char* clear;                       // per row, `clear_bytes` each: state, then what is there of: race bins, histogram or 16-bit counts
    long long clear_bytes, rbins_at, hist_at;
    uint32_t *best, *tile_n, *tile_eq, *keys, *list, *names;
    unsigned long long* words;
    double *group, *tile_sum, *tile_top;
    char *few, *few_u;                 // what top-k left: scores and numbers, rule.top_k a row
    long long B, tiles, stiles, capacity, vpad;
    __device__ __forceinline__ SmRowState& state(long long r) const { return *(SmRowState*)(clear + r * clear_bytes); }
    __device__ __forceinline__ uint32_t* rbins(long long r) const { return (uint32_t*)(clear + r * clear_bytes + rbins_at); }
    __device__ __forceinline__ SmMerged& hist(long long r) const { return *(SmMerged*)(clear + r * clear_bytes + hist_at); }
    __device__ __forceinline__ uint32_t* counts(long long r) const { return (uint32_t*)(clear + r * clear_bytes + hist_at); }
};

template <typename V> __device__ __forceinline__ V sm_peek(const V* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename V> __device__ __forceinline__ void sm_poke(V* p, V v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// The last workgroup of a row to get here.  What it reads of the others' work was written by device-wide atomics (adds, or sm_poke's stores, which
// go through the XCD's own L2) and is read by sm_peek: each wave waits for its own to be done before the ticket is drawn, and no L2 has to be
// written back (a release fence in every wave of every workgroup took longer than the pass over the data).
__device__ __forceinline__ uint32_t sm_draw_ticket(uint32_t* t) { return __hip_atomic_fetch_add(t, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
// Adds to one line of memory take 5 ns each, so of more than 128 workgroups sixteen groups draw among themselves first, on lines of their own (3 M
// scores: a plain draw, 733 workgroups, 26.5 -> 23.5 us, top-k of 1.5 M, four steps of 256, 51.8 -> 48.1).  The last of a group leaves its word
// clear for the next step.
__device__ __forceinline__ bool sm_last_block(SmRowState& st, int step, uint32_t block, uint32_t blocks, uint32_t* lds)
{
    if (blocks == 1) { __syncthreads(); return true; }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        bool last;
        if (blocks <= 128) last = sm_draw_ticket(&st.ticket[step]) == blocks - 1;
        else {
            const uint32_t g = block & 15;
            last = sm_draw_ticket(st.sub[g]) == (blocks - g + 15) / 16 - 1;
            if (last) {
                sm_poke(st.sub[g], 0u);
                last = sm_draw_ticket(&st.ticket[step]) == 15;
            }
        }
        *lds = last;
    }
    __syncthreads();
    return *lds != 0;
}

// Clears the row's part of the workspace and, where a mass needs the row's best score, leaves the best of each workgroup's share.  (10 M scores
// 8.4 us, 4.8 TB/s; without the best 2 us.)
template <typename T>
__global__ void __launch_bounds__(SM_LTPB) sm_begin_kernel(const T* __restrict__ scores, long long sstride, long long V, SmRule rule, SmWork wk, int want_best)
{
    __shared__ SmScratch sc;
    const long long r = blockIdx.x / wk.B, b = blockIdx.x % wk.B;
    uint4* clear = (uint4*)(wk.clear + r * wk.clear_bytes);
    for (long long i = b * SM_LTPB + threadIdx.x; i < wk.clear_bytes / 16; i += wk.B * SM_LTPB) clear[i] = i == 0 ? uint4{ 0xff800000u, 0, 0xff800000u, 0 } : uint4{ 0, 0, 0, 0 };        // (kept, before)
    if (!want_best) return;
    const T* x = scores + r * sstride;
    const bool vec = sm_aligned(x);
    const float floor = sm_floor(rule);
    const long long stride = wk.B * SM_LTPB * 4;
    float best = -INFINITY;
    for (long long i = (b * SM_LTPB + threadIdx.x) * 4; i < V; i += 4 * stride) {
        LgVec4<T> v[4];
#pragma unroll
        for (int g = 0; g < 4; g++) v[g] = sm_load4(x, i + g * stride, V, vec);
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int j = 0; j < 4; j++) best = fmaxf(best, sm_score(v[g].v[j], floor));
    }
    const uint32_t order = sm_block_max(sm_order(best), sc.a);
    if (threadIdx.x == 0) wk.best[r * wk.B + b] = order;
}
// the row's best (every wave on its own)
__device__ __forceinline__ float sm_best(const SmWork& wk, long long r)
{
    uint32_t best = 0;
    for (long long i = threadIdx.x & 63; i < wk.B; i += 64) { const uint32_t k = wk.best[r * wk.B + i]; best = k > best ? k : best; }
    return sm_unorder(sm_lane(sm_wave_scan<false>(best, SmMaxOf()), 63));
}

// what a selection leaves in the row's state (one thread): `ties` of `count` elements of score thr are taken, and all above it
__device__ __forceinline__ void sm_conclude(SmRowState& st, const SmKept& kept, float thr, uint32_t ties, uint32_t count)
{
    if (thr < kept.thr) return;                                        // a whole bin around the earlier filter's cut: that one stands
    st.kept = SmKept{ thr, thr == kept.thr ? kept.end : SM_ALL };
    if (ties < count) { st.cut = 1; st.ties = ties; }
}

// A mass as two integers that LDS adds up: so many of 2^bits parts that a workgroup's share of the row cannot overflow 63 bits (50 for short
// rows, 47 for 10 M scores), and what that leaves, of either sign, in 2^-bits of a part.  The addition of 2^(52 - bits) rounds, and leaves the
// integer in the low bits of the sum.  (One integer alone is 4 us faster for 10 M scores, but then ten million equal scores behind a larger one
// are cut some elements off.)
struct SmParts { int bits; double one, rest; };
__device__ __forceinline__ SmParts sm_parts(const SmWork& wk, long long V)
{
    const long long share = (V + wk.B * SM_LTPB * 4 - 1) / (wk.B * SM_LTPB * 4) * (SM_LTPB * 4);
    const int b = __clzll(share - 1) - 1, bits = b < 51 ? b : 51;      // 63 - ceil(log2(share))
    return SmParts{ bits, ldexp(1.0, 52 - bits), ldexp(1.5, 52 - 2 * bits) };
}
__device__ __forceinline__ unsigned long long sm_bits_above(double sum, double one) { return (unsigned long long)__double_as_longlong(sum) - (unsigned long long)__double_as_longlong(one); }
__device__ __forceinline__ void sm_add_parts(const SmParts& p, double mass, unsigned long long& whole, unsigned long long& rest)
{
    const double sum = mass + p.one;
    atomicAdd(&whole, sm_bits_above(sum, p.one));
    atomicAdd(&rest, sm_bits_above(mass - (sum - p.one) + p.rest, p.rest));
}
__device__ __forceinline__ SmSum sm_sum_of_parts(const SmParts& p, unsigned long long whole, unsigned long long rest)
{
    const long long lo = (long long)((whole << (63 - p.bits)) & 0xffffffffull) + ((long long)rest >> (2 * p.bits - 63));
    return SmSum{ (whole >> (p.bits - 31)) + (unsigned long long)(lo >> 32), (unsigned long long)lo & 0xffffffffull };
}

// One level of top-k (MASS false) or top-p: bits [shift - width, shift) of the ordered scores that pass the filters and match the prefix found
// so far.  Three levels of 11, 10 and 11 bits name the last key that is taken, whatever the scores are like; a level of 2^13 bins instead
// would merge four times as many words.  10 M weights under a temperature: 42 us for the first level (a logarithm and an exponential in 64
// bits each: the vector pipe), 18 and 17 for the others (2.2 TB/s); 3 M counted: 13, 13 and 8 us, of which the data are 3 each.
template <typename T, bool MASS>
__global__ void __launch_bounds__(SM_LTPB) sm_level_kernel(const T* __restrict__ scores, long long sstride, long long V, SmRule rule, SmWork wk, int step,
                                                           int shift, int width)
{
    __shared__ SmHist h;
    __shared__ SmTables tables;
    __shared__ SmScratch sc;
    __shared__ uint32_t ticket;
    constexpr int G = MASS ? 2 : 4;                                    // groups of four loaded ahead
    const long long r = blockIdx.x / wk.B, b = blockIdx.x % wk.B;
    SmRowState& st = wk.state(r);
    const bool first = shift == 32;
    const T* x = scores + r * sstride;
    const bool vec = sm_aligned(x);
    const float floor = sm_floor(rule);
    const int at = shift - width, nbins = 1 << width, p = width - 6;
    const long long stride = wk.B * SM_LTPB * 4;
    long long i = (b * SM_LTPB + threadIdx.x) * 4;
    LgVec4<T> v[G];
#pragma unroll
    for (int g = 0; g < G; g++) v[g] = sm_load4(x, i + g * stride, V, vec);
    if (!first && st.ended) return;
    const SmKept kept = first ? st.kept : st.before;
    const bool filtered = kept.thr > -INFINITY;
    const uint32_t prefix = st.prefix;
    // the prefix as a range of scores (its last one is not -0, which equals the first one of the next range)
    float least = -SmMax<float>::v, most = SmMax<float>::v;
    if (!first) {
        const uint32_t last = (prefix << shift) | ((1u << shift) - 1);
        least = sm_unorder(prefix << shift);
        most = sm_unorder(last == 0x7fffffffu ? last - 1 : last);
    }
    const float best = MASS ? (first ? sm_best(wk, r) : st.best) : 0.0f;
    const SmParts parts = sm_parts(wk, V);
    const bool counted = !MASS || at == 0;                             // masses need no counts before the last level
    if (MASS) sm_tables(tables, rule.mode);
    for (int k = threadIdx.x; k < sm_slots(p); k += SM_LTPB) { h.n[k] = 0; if (MASS) { h.hi[k] = 0; h.lo[k] = 0; } }
    __syncthreads();
    const SmScale scale = sm_scale(tables, rule, best);
    const double unit = rule.mode == SM_LINEAR ? scale.shift : 1.0;
    while (i < V) {
        float z[4 * G];
        int found = 0;
#pragma unroll
        for (int g = 0; g < G; g++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float y = sm_score(v[g].v[j], floor);
                y = y >= least && y <= most ? y : -INFINITY;
                if (filtered) y = sm_in(kept, y, (uint32_t)(i + g * stride + j)) ? y : -INFINITY;
                z[4 * g + j] = y;
                if (MASS) found += __popcll(__ballot(y > -INFINITY));
            }
        double mass[4 * G];
        const bool many = MASS && found >= 64;                         // (the same for the wave: all masses at once, or one at a time)
        if (many) sm_masses(tables, scale, z, mass);
#pragma unroll
        for (int j = 0; j < 4 * G; j++) {
            if (!(z[j] > -INFINITY)) continue;
            const int bin = sm_slot((int)(sm_order(z[j]) >> at) & (nbins - 1), p);
            if (counted) atomicAdd(&h.n[bin], 1u);
            if (MASS) {
                if (!many) { const float one[1] = { z[j] }; double m[1]; sm_masses(tables, scale, one, m); mass[j] = m[0]; }
                sm_add_parts(parts, mass[j] * unit, h.hi[bin], h.lo[bin]);
            }
        }
        i += G * stride;
        if (i >= V) break;
#pragma unroll
        for (int g = 0; g < G; g++) v[g] = sm_load4(x, i + g * stride, V, vec);
    }
    __syncthreads();
    if (MASS)
        for (int k = threadIdx.x; k < sm_slots(p); k += SM_LTPB) { const SmSum m = sm_sum_of_parts(parts, h.hi[k], h.lo[k]); h.hi[k] = m.hi; h.lo[k] = m.lo; }
    __syncthreads();
    if (wk.B > 1) {
        SmMerged& g = wk.hist(r);
        for (int k = threadIdx.x; k < nbins; k += SM_LTPB) {
            const int slot = MASS ? sm_nth_slot(k) : sm_slot(k, p);
            if (counted && h.n[slot]) atomicAdd(&g.n[k], h.n[slot]);
            if (MASS) { if (h.hi[slot]) atomicAdd(&g.hi[k], h.hi[slot]); if (h.lo[slot]) atomicAdd(&g.lo[k], h.lo[slot]); }
        }
        if (!sm_last_block(st, step, (uint32_t)b, (uint32_t)wk.B, &ticket)) return;
        // taken over (all loads before the first store: each is a round trip to memory), and left clear for the next level
        constexpr int K = SM_BINS / SM_LTPB;
        uint32_t n[K];
        unsigned long long hi[K], lo[K];
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int bin = k * SM_LTPB + threadIdx.x;
            n[k] = counted ? sm_peek(&g.n[bin]) : 0u;
            if (MASS) { hi[k] = sm_peek(&g.hi[bin]); lo[k] = sm_peek(&g.lo[bin]); }
        }
#pragma unroll
        for (int k = 0; k < K; k++) {
            const int bin = k * SM_LTPB + threadIdx.x, slot = MASS ? sm_nth_slot(bin) : sm_slot(bin, p);
            if (bin >= nbins) continue;
            h.n[slot] = n[k]; g.n[bin] = 0;
            if (MASS) { h.hi[slot] = hi[k]; h.lo[slot] = lo[k]; g.hi[bin] = 0; g.lo[bin] = 0; }
        }
        __syncthreads();
    }
    SmTake take = st.take;
    if (first) {
        take = SmTake{ (double)rule.top_k, 0, { 0, 0 } };
        if (MASS) {
            SmSum mine = { 0, 0 }, total;
            for (int k = threadIdx.x; k < sm_slots(p); k += SM_LTPB) { mine.hi += h.hi[k]; mine.lo += h.lo[k]; }
            sm_block_scan<unsigned long long>(mine.hi, sc.a, total.hi);
            sm_block_scan<unsigned long long>(mine.lo, sc.b, total.lo);
            take.target = rule.top_p * sm_sum_value(total);
        }
    }
    const SmBin bin = sm_boundary<MASS>(h.n, h.hi, h.lo, p, take, sc);
    if (threadIdx.x != 0) return;
    st.before = kept;
    st.take = take;
    st.best = best;
    st.ended = 0;
    st.cut = 0;
    if (bin.bin < 0) { st.ended = 1; return; }                         // no candidate: the filter in force (or an empty row) stands
    const uint32_t found = (first ? 0u : prefix << width) | (uint32_t)bin.bin;
    st.prefix = found;
    const bool whole = counted && sm_whole_bin<MASS>(take, bin.count);
    if (!whole && at > 0) return;
    // the key is found, or the lowest key of a bin that is taken whole; a cut among the equal ones is left to sm_cut_kernel
    const float thr = sm_unorder(found << at), one[1] = { thr };
    double mass[1] = { 0.0 };
    if (MASS) sm_masses(tables, scale, one, mass);
    st.ended = 1;
    sm_conclude(st, kept, thr, whole ? bin.count : sm_ties<MASS>(take, bin.count, mass[0] * unit), bin.count);
}

// ---- scores of 16 bits: both filters from one histogram of all keys ----------------------------------------------------------------------
// The 65536 ordered keys of a 16-bit type are counted in LDS (two counters a word: a workgroup takes at most SM_SHARE16 elements), added up in
// memory, and the last workgroup works top-k and top-p out of the counts: one pass over the row and one exponential per distinct score, in
// the place of one pass for the best and three for each filter.  16 rows of 100 k: 24 us, about half of it the last workgroup's conclusion.
// Rows of 50 k behind top-p: 1 row 45 us a call (by levels 63), 64 rows 58 (83), 256 rows 131 (160), 512 rows 231 (287); behind top-k alone 64
// rows 51 (57), 128 rows 72 (82), 256 rows 118 (110).  So up to 256 rows, where the counts are 64 MB, and without top-p up to 128.
#define SM_SHARE16 32768
__device__ __forceinline__ uint32_t sm_bits(LgHalf v) { return (uint32_t)__builtin_bit_cast(uint16_t, v); }
__device__ __forceinline__ uint32_t sm_bits(LgBf16 v) { return v.bits; }
__device__ __forceinline__ uint32_t sm_bits(float) { return 0u; }                            // (no such path)
template <typename T> __device__ __forceinline__ T sm_from_bits(uint32_t b);
template <> __device__ __forceinline__ LgHalf sm_from_bits<LgHalf>(uint32_t b) { return __builtin_bit_cast(LgHalf, (uint16_t)b); }
template <> __device__ __forceinline__ LgBf16 sm_from_bits<LgBf16>(uint32_t b) { return LgBf16{ (uint16_t)b }; }

// a score as an ordered key of 16 bits, 0 = excluded, and back
template <typename T> __device__ __forceinline__ uint32_t sm_key16(T raw, float floor)
{
    const float x = sm_score(raw, floor);
    if (x == -INFINITY) return 0u;
    const uint32_t b = sm_bits(lg_from_float<T>(x));
    return (b & 0x8000u) ? (~b & 0xffffu) : (b | 0x8000u);
}
template <typename T> __device__ __forceinline__ float sm_unkey16(uint32_t k) { return lg_to_float(sm_from_bits<T>((k & 0x8000u) ? (k & 0x7fffu) : (~k & 0xffffu))); }

// per chunk of 64 keys: count, and mass in limbs, of what a filter left
struct SmChunks { uint32_t n[1024]; unsigned long long hi[1024], lo[1024]; };

template <typename T>
__global__ void __launch_bounds__(1024) sm_count16_kernel(const T* __restrict__ scores, long long sstride, long long V, SmRule rule, SmWork wk, int step, int top_k, int top_p)
{
    __shared__ union { uint32_t pair[32768]; SmChunks chunk; } h;
    __shared__ SmScratch sc;
    __shared__ uint32_t ticket;
    const long long r = blockIdx.x / wk.B, b = blockIdx.x % wk.B;
    SmRowState& st = wk.state(r);
    const T* x = scores + r * sstride;
    const bool vec = sm_aligned(x);
    const float floor = sm_floor(rule);
    const long long stride = wk.B * 4096;
    long long i = (b * 1024 + threadIdx.x) * 4;
    LgVec4<T> v[4];
#pragma unroll
    for (int g = 0; g < 4; g++) v[g] = sm_load4(x, i + g * stride, V, vec);
    for (int k = threadIdx.x; k < 8192; k += 1024) ((uint4*)h.pair)[k] = uint4{ 0, 0, 0, 0 };
    __syncthreads();
    while (i < V) {
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t k = sm_key16(v[g].v[j], floor);
                if (k) atomicAdd(&h.pair[k >> 1], 1u << (16 * (k & 1)));
            }
        i += 4 * stride;
        if (i >= V) break;
#pragma unroll
        for (int g = 0; g < 4; g++) v[g] = sm_load4(x, i + g * stride, V, vec);
    }
    __syncthreads();
    uint32_t* counts = wk.counts(r);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // chunk c: keys 64 c ... 64 c + 63.  A wave merges, and walks at the end, the chunks (b / 2) * 32 + wave * 2 + b % 2, b = 0 ... 63: the scores
    // that occur lie close together
    auto chunk_of = [](int b, int w) { return (b >> 1) * 32 + w * 2 + (b & 1); };
    unsigned long long live = 0;
    for (int it = 0; it < 32; it++) {
        const int k = it * 1024 + threadIdx.x;
        const uint32_t w = h.pair[k];
        if (w & 0xffffu) atomicAdd(&counts[2 * k], w & 0xffffu);
        if (w >> 16) atomicAdd(&counts[2 * k + 1], w >> 16);
        const unsigned long long any = __ballot(w != 0);
        live |= ((unsigned long long)((uint32_t)any != 0) | (unsigned long long)((any >> 32) != 0) << 1) << (2 * it);
    }
    unsigned long long* all_live = (unsigned long long*)(counts + 65536);        // a word of each wave, 128 bytes apart (adds to one line wait for each other)
    if (lane == 0 && live) atomicOr(&all_live[wave * 16], live);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (!sm_last_block(st, step, (uint32_t)b, (uint32_t)wk.B, &ticket)) return;
    const unsigned long long lives = sm_peek(&all_live[(lane & 15) * 16]);
    live = sm_lane(lives, wave);
    const int top = (int)sm_lane(sm_wave_scan<true>(lives ? (uint32_t)chunk_of(63 - __clzll((long long)lives), lane & 15) + 1 : 0u, SmMaxOf()), 15) - 1;
    uint32_t best = 0;                                                 // every wave on its own
    if (top >= 0) best = (uint32_t)top * 64 + 63 - __clzll((long long)__ballot(sm_peek(&counts[top * 64 + lane]) != 0));
    const float most = best ? sm_unkey16<T>(best) : -INFINITY;
    const SmScale scale = sm_scale(rule, most);
    const double unit = rule.mode == SM_LINEAR ? scale.shift : 1.0;
    SmKept kept = { -INFINITY, 0u };
    uint32_t cut_key = 0, cut_n = 0;                                   // top-k: keys above cut_key whole, cut_n of it
    uint32_t thr = 0, ties = 0, equal = 0;
    for (int pass = 0; pass < 2 && best != 0; pass++) {
        if (!(pass == 0 ? top_k : top_p)) continue;
        const bool mass = pass == 1;
        SmTake take = { (double)rule.top_k, 0, { 0, 0 } };
        // what is left of key k's count
        auto left = [&](uint32_t k) {
            const uint32_t n = sm_peek(&counts[k]);
            return k > cut_key ? n : k == cut_key ? cut_n : 0u;
        };
        auto limbs = [&](uint32_t k, uint32_t n) {
            SmSum m = { 0, 0 };
            if (n) { const SmLimbs one = sm_limbs(sm_mass(scale, sm_unkey16<T>(k)) * unit); m = SmSum{ (unsigned long long)one.hi * n, (unsigned long long)one.lo * n }; }
            return m;
        };
        if (mass) { h.chunk.hi[threadIdx.x] = 0; h.chunk.lo[threadIdx.x] = 0; } else h.chunk.n[threadIdx.x] = 0;
        __syncthreads();
        // eight chunks a round: their counts are eight round trips to memory otherwise
        for (unsigned long long todo = live; todo; ) {
            uint32_t n[8];
            int chunk[8];
#pragma unroll
            for (int q = 0; q < 8; q++) {
                chunk[q] = todo ? chunk_of(__ffsll((long long)todo) - 1, wave) : -1;
                todo &= todo - 1;
                n[q] = chunk[q] < 0 ? 0u : left((uint32_t)chunk[q] * 64 + lane);
            }
#pragma unroll
            for (int q = 0; q < 8; q++) {
                if (chunk[q] < 0) continue;
                if (mass) {
                    SmSum m = limbs((uint32_t)chunk[q] * 64 + lane, n[q]);
                    m.hi = sm_lane(sm_wave_scan<false>(m.hi, SmAdd()), 63);
                    m.lo = sm_lane(sm_wave_scan<false>(m.lo, SmAdd()), 63);
                    if (lane == 0) { h.chunk.hi[chunk[q]] = m.hi; h.chunk.lo[chunk[q]] = m.lo; }
                } else {
                    const uint32_t sum = sm_lane(sm_wave_scan<false>(n[q], SmAdd()), 63);
                    if (lane == 0) h.chunk.n[chunk[q]] = sum;
                }
            }
        }
        __syncthreads();
        // the chunk in which the selection ends: thread t stands for chunk 1023 - t
        const int chunk = 1023 - (int)threadIdx.x;
        uint32_t n = 0, before = 0, all;
        SmSum m = { 0, 0 }, total = { 0, 0 }, upto = { 0, 0 };
        if (!mass) {
            n = h.chunk.n[chunk];
            before = sm_block_scan<uint32_t>(n, sc.a, all);
        } else {
            m = SmSum{ h.chunk.hi[chunk], h.chunk.lo[chunk] };
            upto.hi = sm_block_scan<unsigned long long>(m.hi, sc.a, total.hi);
            upto.lo = sm_block_scan<unsigned long long>(m.lo, sc.b, total.lo);
            take.target = rule.top_p * sm_sum_value(total);
        }
        const bool room = mass ? (m.hi | m.lo) != 0 && sm_room<true>(take, 0, upto.hi, upto.lo) : n != 0 && sm_room<false>(take, before, 0, 0);
        const uint32_t end = sm_block_max<uint32_t>(room ? threadIdx.x + 1 : 0u, sc.a);
        if (room && threadIdx.x + 1 == end) { sc.word[0] = before; sc.word[1] = upto.hi; sc.word[2] = upto.lo; }
        __syncthreads();
        take.before_n = (uint32_t)sc.word[0];
        take.before_m = SmSum{ sc.word[1], sc.word[2] };
        // inside it: lane l stands for its key 63 - l (every wave the same)
        const uint32_t k = (1024 - end) * 64 + 63 - (uint32_t)lane;
        const uint32_t n2 = left(k);
        SmSum m2 = { 0, 0 }, in2 = { 0, 0 };
        const uint32_t in = sm_wave_scan<false>(n2, SmAdd());
        if (mass) {
            m2 = limbs(k, n2);
            in2.hi = sm_wave_scan<false>(m2.hi, SmAdd());
            in2.lo = sm_wave_scan<false>(m2.lo, SmAdd());
        }
        const unsigned long long enter = __ballot(mass ? (m2.hi | m2.lo) != 0 && sm_room<true>(take, 0, in2.hi - m2.hi, in2.lo - m2.lo) : n2 != 0 && sm_room<false>(take, in - n2, 0, 0));
        const int l = enter ? 63 - __clzll((long long)enter) : 0;
        equal = sm_lane(n2, l);
        thr = sm_lane(k, l);
        take.before_n += sm_lane(in - n2, l);
        if (mass) { take.before_m.hi += sm_lane(in2.hi - m2.hi, l); take.before_m.lo += sm_lane(in2.lo - m2.lo, l); }
        const double unit_mass = mass ? sm_mass(scale, sm_unkey16<T>(thr)) * unit : 0.0;
        ties = mass ? sm_ties<true>(take, equal, unit_mass) : sm_ties<false>(take, equal, 0.0);
        // equal ones that top-k had left out count as cut too
        equal = sm_peek(&counts[thr]);
        cut_key = thr;
        cut_n = ties;
        __syncthreads();
    }
    float least = -INFINITY;
    if (best != 0 && rule.min_p > 0.0) least = sm_min_p(rule, rule.mode == SM_LOGITS ? 1u : 0x8001u, best, [](uint32_t k) { return sm_unkey16<T>(k); });
    if (threadIdx.x != 0) return;
    st.before = kept;
    st.best = most;
    st.least = least;
    st.ended = 1;
    st.cut = 0;
    if (best != 0) sm_conclude(st, kept, sm_unkey16<T>(thr), ties, equal);
}

// ---- cuts among equal keys, and what top-k left ------------------------------------------------------------------------------------------
// Index of the last equal element that is kept, where a selection ends inside equal keys.  GATHER: also every tile's first place among the
// elements that are left.  (4.5 us where there is nothing to cut, 8.8 for 16 rows of 100 k in half width, where there always is.)
template <typename T, bool GATHER>
__global__ void __launch_bounds__(SM_LTPB) sm_cut_kernel(const T* __restrict__ scores, long long sstride, long long V, SmRule rule, SmWork wk, int step)
{
    __shared__ SmScratch sc;
    __shared__ uint32_t ticket;
    const long long r = blockIdx.x / wk.B, b = blockIdx.x % wk.B;
    SmRowState& st = wk.state(r);
    const bool cut = st.cut;
    if (!GATHER && !cut) return;
    const T* x = scores + r * sstride;
    const bool vec = sm_aligned(x);
    const float floor = sm_floor(rule);
    const SmKept kept = st.kept;
    uint32_t *tile_n = wk.tile_n + r * wk.tiles, *tile_eq = wk.tile_eq + r * wk.tiles;
    for (long long t = b; t < wk.tiles; t += wk.B) {
        // (counts do not care for the order: groups of four as they load best)
        LgVec4<T> v[SM_TILE / SM_LTPB / 4];
#pragma unroll
        for (int g = 0; g < SM_TILE / SM_LTPB / 4; g++) v[g] = sm_load4(x, t * SM_TILE + (g * SM_LTPB + threadIdx.x) * 4, V, vec);
        uint32_t eq = 0, more = 0, total;
#pragma unroll
        for (int g = 0; g < SM_TILE / SM_LTPB / 4; g++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float y = sm_score(v[g].v[j], floor);
                const uint32_t i = (uint32_t)(t * SM_TILE + (g * SM_LTPB + threadIdx.x) * 4 + j);
                eq += y == kept.thr && i < kept.end;
                more += y > kept.thr;
            }
        sm_block_scan<uint32_t>(eq, sc.a, total);
        if (threadIdx.x == 0) sm_poke(&tile_eq[t], total);
        if (GATHER) {
            sm_block_scan<uint32_t>(more, sc.b, total);
            if (threadIdx.x == 0) sm_poke(&tile_n[t], total);
        }
    }
    if (!sm_last_block(st, step, (uint32_t)b, (uint32_t)wk.B, &ticket)) return;
    const uint32_t want = cut ? st.ties : SM_ALL;                      // equal elements that are kept
    unsigned long long equal = 0, run = 0;
    long long tile = -1;
    uint32_t rest = 0;
    for (long long base = 0; base < wk.tiles; base += SM_LTPB) {
        const long long t = base + threadIdx.x;
        const uint32_t c = t < wk.tiles ? sm_peek(&tile_eq[t]) : 0u;
        uint32_t total;
        const uint32_t before = sm_block_scan<uint32_t>(c, sc.a, total);
        const unsigned long long from = equal + before;                // equal ones before this tile
        const uint32_t mine = from >= want ? 0u : want - from < c ? (uint32_t)(want - from) : c;
        if (cut && mine != 0 && from + mine == want) { sc.word[0] = (unsigned long long)t; sc.word[1] = want - from; }
        if (GATHER) {
            uint32_t kept_here = mine + (t < wk.tiles ? sm_peek(&tile_n[t]) : 0u), all;
            const uint32_t at = sm_block_scan<uint32_t>(kept_here, sc.b, all);
            if (t < wk.tiles) tile_n[t] = (uint32_t)(run + at);
            run += all;
        }
        __syncthreads();
        if (cut && tile < 0 && equal + total >= want) { tile = (long long)sc.word[0]; rest = (uint32_t)sc.word[1]; }        // uniform
        equal += total;
        __syncthreads();
    }
    if (GATHER && threadIdx.x == 0) st.sure = run;
    if (tile < 0) return;
    // inside the tile: eight consecutive elements a thread
    constexpr int E = SM_TILE / SM_LTPB;
    const long long i0 = tile * SM_TILE + (long long)threadIdx.x * E;
    LgVec4<T> v[E / 4];
#pragma unroll
    for (int g = 0; g < E / 4; g++) v[g] = sm_load4(x, i0 + 4 * g, V, vec);
    uint32_t is = 0, total;
#pragma unroll
    for (int k = 0; k < E; k++) {
        if (sm_score(v[k / 4].v[k % 4], floor) == kept.thr && (uint32_t)(i0 + k) < kept.end) is |= 1u << k;
    }
    uint32_t before = sm_block_scan<uint32_t>(__popc(is), sc.a, total);
#pragma unroll
    for (int k = 0; k < E; k++) if (((is >> k) & 1) && ++before == rest) { st.kept.end = (uint32_t)(i0 + k) + 1; st.cut = 0; }
}

// A top-k of at most SM_SHORT elements leaves a short row, which one more launch finishes: 3 M scores behind top-k 50 and top-p 46 us, by the
// long way 83; behind k = 5000 alone, where the long way is shortest, a draw 55 and 54, 500 distinct 65 and 70 (of 50 k scores 43 and 36, 53 and
// 44: the case that loses).
// What top-k left, in index order: scores, their names and (without replacement) their numbers; rule.top_k places a row, the last ones empty
template <typename T>
__global__ void __launch_bounds__(SM_LTPB) sm_gather_kernel(const T* __restrict__ scores, long long sstride, const float* __restrict__ u /*nullable*/, long long ustride,
                                                            long long V, SmRule rule, SmWork wk)
{
    __shared__ SmScratch sc;
    const long long r = blockIdx.x / wk.tiles, t = blockIdx.x % wk.tiles, K = rule.top_k;
    const SmRowState& st = wk.state(r);
    const T* x = scores + r * sstride;
    const bool vec = sm_aligned(x);
    const float floor = sm_floor(rule);
    const SmKept kept = st.kept;
    constexpr int E = SM_TILE / SM_LTPB;                               // consecutive elements a thread
    const long long i0 = t * SM_TILE + (long long)threadIdx.x * E;
    LgVec4<T> v[E / 4];
#pragma unroll
    for (int g = 0; g < E / 4; g++) v[g] = sm_load4(x, i0 + 4 * g, V, vec);
    uint32_t in = 0, total;
#pragma unroll
    for (int k = 0; k < E; k++) if (sm_in(kept, sm_score(v[k / 4].v[k % 4], floor), (uint32_t)(i0 + k))) in |= 1u << k;
    long long at = (long long)wk.tile_n[r * wk.tiles + t] + sm_block_scan<uint32_t>(__popc(in), sc.a, total);
    T* few = (T*)wk.few + r * K;
    uint32_t* names = wk.names + r * K;
    float* few_u = (float*)wk.few_u + r * K;
#pragma unroll
    for (int k = 0; k < E; k++)
        if ((in >> k) & 1) {
            if (at < K) {
                few[at] = v[k / 4].v[k % 4];
                names[at] = (uint32_t)(i0 + k);
                if (u) few_u[at] = u[r * ustride + i0 + k];
            }
            at++;
        }
    for (long long j = (long long)st.sure + t * SM_LTPB + threadIdx.x; j < K; j += wk.tiles * SM_LTPB) few[j] = lg_from_float<T>(__uint_as_float(0x7fc00000u));
}

// filter in force with min-p (every wave works the cut out for itself where the histogram of all keys has not)
__device__ __forceinline__ SmKept sm_final(const SmWork& wk, long long r, const SmRowState& st, const SmRule& rule)
{
    SmKept kept = st.kept;
    if (rule.min_p <= 0.0) return kept;
    if (!wk.best) return st.least > kept.thr ? SmKept{ st.least, SM_ALL } : kept;
    const float best = sm_best(wk, r);
    if (best > -INFINITY) sm_min_p(rule, best, kept);
    return kept;
}

// ---- long rows, with replacement -------------------------------------------------------------------------------------------------------
// Prefix sums of the kept masses inside tiles, one stored per SM_GROUP elements, relative to the tile's best element (so that no pass for the
// row's best is needed); the last workgroup puts the tiles on a common scale.  Fixed order everywhere.  Workgroups of 256, five a compute unit,
// hide each other's scans: 3 M weights 12.6 us, scores 14 (the exponentials; a plain draw of 10 M scores 40.7 us, of weights 34).
template <typename T>
__global__ void __launch_bounds__(256) sm_sums_kernel(const T* __restrict__ scores, long long sstride, long long V, SmRule rule, SmWork wk, SmWork whole, int step)
{
    __shared__ SmTables tables;
    __shared__ SmScratch sc;
    __shared__ uint32_t ticket;
    const long long r = blockIdx.x / wk.B, b = blockIdx.x % wk.B;
    SmRowState& st = wk.state(r);
    const T* x = scores + r * sstride;
    const bool vec = sm_aligned(x);
    const float floor = sm_floor(rule);
    sm_tables(tables, rule.mode);                                      // (the scans below are the barrier)
    const SmKept kept = sm_final(whole, r, st, rule);
    double *sums = wk.tile_sum + r * wk.stiles, *tops = wk.tile_top + r * wk.stiles, *groups = wk.group + r * wk.stiles * (SM_STILE / SM_GROUP);
    for (long long t = b; t < wk.stiles; t += wk.B) {
        const long long i0 = t * SM_STILE + threadIdx.x * SM_GROUP;
        LgVec4<T> v[SM_GROUP / 4];
#pragma unroll
        for (int k = 0; k < SM_GROUP / 4; k++) v[k] = sm_load4(x, i0 + 4 * k, V, vec);
        float z[SM_GROUP], best = -INFINITY;
#pragma unroll
        for (int k = 0; k < SM_GROUP; k++) {
            const float y = sm_score(v[k / 4].v[k % 4], floor);
            z[k] = sm_in(kept, y, (uint32_t)(i0 + k)) ? y : -INFINITY;
            best = fmaxf(best, z[k]);
        }
        best = sm_unorder(sm_block_max(sm_order(best), sc.b));
        const SmScale scale = sm_scale(tables, rule, best);
        double mass[SM_GROUP], sum = 0.0, total, most;
        sm_masses(tables, scale, z, mass);
#pragma unroll
        for (int k = 0; k < SM_GROUP; k++) sum += mass[k];
        const double before = sm_block_scan<double>(sum, sc.a, total);
        groups[t * (SM_STILE / SM_GROUP) + threadIdx.x] = sm_block_rise(sum > 0.0 ? before + sum : 0.0, sc.b, most);
        if (threadIdx.x == 0) {
            sm_poke(&sums[t], total);
            sm_poke(&tops[t], best > -INFINITY ? scale.top : -INFINITY);
        }
    }
    if (!sm_last_block(st, step, (uint32_t)b, (uint32_t)wk.B, &ticket)) return;
    double top = -INFINITY;
    for (long long t = threadIdx.x; t < wk.stiles; t += 256) top = fmax(top, sm_peek(&tops[t]));
    const unsigned long long ordered = (unsigned long long)__double_as_longlong(top + 0.0);
    const unsigned long long m = sm_block_max<unsigned long long>((ordered >> 63) ? ~ordered : (ordered | 0x8000000000000000ull), sc.b);
    top = __longlong_as_double((long long)((m >> 63) ? (m & 0x7fffffffffffffffull) : ~m));
    double run = 0.0, risen = 0.0;
    uint32_t end = 0;
    constexpr int K = 4;                                               // tiles a thread
    for (long long base = 0; base < wk.stiles; base += 256 * K) {
        const long long t0 = base + threadIdx.x * K;
        double mass[K], tt[K], sum = 0.0, total, most;
#pragma unroll
        for (int k = 0; k < K; k++) {
            mass[k] = t0 + k < wk.stiles ? sm_peek(&sums[t0 + k]) : 0.0;
            tt[k] = t0 + k < wk.stiles ? sm_peek(&tops[t0 + k]) : -INFINITY;
        }
#pragma unroll
        for (int k = 0; k < K; k++) {
            if (rule.mode != SM_LINEAR) mass[k] = tt[k] == -INFINITY ? 0.0 : mass[k] * sm_exp(tables, tt[k] - top);
            sum += mass[k];
        }
        double at = run + sm_block_sum_before(sum, sc.a, total);
        double rise[K], high = 0.0;
#pragma unroll
        for (int k = 0; k < K; k++) {
            at += mass[k];
            if (mass[k] > 0.0) { end = (uint32_t)(t0 + k); if (at > high) high = at; }
            rise[k] = high;
        }
        const double below = fmax(sm_block_rise_before(high, sc.b, most), risen);
#pragma unroll
        for (int k = 0; k < K; k++) if (t0 + k < wk.stiles) sums[t0 + k] = fmax(rise[k], below);
        risen = fmax(risen, most);
        run += total;
    }
    end = sm_wave_scan<false>(end, SmMaxOf());
    if ((threadIdx.x & 63) == 63) atomicMax(&st.end_tile, end);
    if (threadIdx.x == 0) { st.total = run; st.top = top; st.kept = kept; }
}

// how many of the n ascending values are not past (`past(a[i])` is false up to there and true behind)
template <typename Past> __device__ __forceinline__ int sm_rank(const double* a, int n, const Past& past)
{
    int lo = 0;
    while (n > 0) {
        const int half = n >> 1;
        if (past(a[lo + half])) n = half; else { lo += half + 1; n -= half + 1; }
    }
    return lo;
}
// the same, three values a round loaded together (half the round trips to memory for half as many loads again)
template <typename Past> __device__ __forceinline__ int sm_rank4(const double* a, int n, const Past& past)
{
    int lo = 0;
    while (n >= 4) {
        const int part = n >> 2;
        const bool x = past(a[lo + part - 1]), y = past(a[lo + 2 * part - 1]), z = past(a[lo + 3 * part - 1]);
        const int c = x ? 0 : y ? 1 : z ? 2 : 3;
        lo += c * part;
        n = c < 3 ? part - 1 : n - 3 * part;
    }
    return lo + sm_rank(a + lo, n, past);
}

// One draw a thread: its tile by binary search in LDS, its group of 16 by search in memory, its element by the masses worked out once more.
// Bound by those dependent loads: 8 us for a few draws, 13 for 100 k of 3 M.  (Sixteen-way search: 30 us in the place of 17.)
#define SM_DRAW_ENDS 2048              // tiles whose ends a workgroup of draws keeps in LDS (or ends of groups of tiles, where there are more)

template <typename T>
__global__ void __launch_bounds__(256) sm_draw_kernel(const T* __restrict__ scores, long long sstride, const float* __restrict__ u, long long ustride,
                                                      long long V, long long n, SmRule rule, SmWork wk, long long* __restrict__ out)
{
    __shared__ double ends[SM_DRAW_ENDS];
    __shared__ SmTables tables;
    const long long blocks = (n + 255) / 256, r = blockIdx.x / blocks, j = blockIdx.x % blocks * 256 + threadIdx.x, at = r * n + j;
    const SmRowState& st = wk.state(r);
    const double* sums = wk.tile_sum + r * wk.stiles;
    const int tiles = (int)wk.stiles, group = (tiles + SM_DRAW_ENDS - 1) / SM_DRAW_ENDS, ngroups = (tiles + group - 1) / group;
    sm_tables(tables, rule.mode);
    for (int k = threadIdx.x; k < ngroups; k += 256) ends[k] = sums[((k + 1) * group < tiles ? (k + 1) * group : tiles) - 1];
    __syncthreads();
    if (j >= n) return;
    const double* tops = wk.tile_top + r * wk.stiles;
    const double total = ends[ngroups - 1];
    if (!(total > 0.0)) { out[at] = -1; return; }
    const float uj = u[r * ustride + j];
    const double target = (uj > 0.0f ? (double)uj : 0.0) * st.total;
    auto tile_of = [&](auto&& past) {
        const int k = sm_rank(ends, ngroups, past), t = k * group;
        return k < ngroups && group > 1 ? t + sm_rank(sums + t, t + group < tiles ? group : tiles - t, past) : t;
    };
    int t = uj >= 1.0f ? tiles : tile_of([&](double s) { return s > target; });
    const bool last = t >= tiles;                                      // (or rounding: the last one with a mass)
    if (last) t = (int)st.end_tile;
    const double* g = wk.group + (r * wk.stiles + t) * (long long)(SM_STILE / SM_GROUP);
    const int ng = SM_STILE / SM_GROUP;
    const double scale_up = rule.mode == SM_LINEAR ? 1.0 : sm_exp(tables, tops[t] - st.top);
    const double local = fmax((target - (t ? sums[t - 1] : 0.0)) / scale_up, 0.0), here = g[ng - 1];
    int k = last ? ng - 1 : sm_rank4(g, ng, [&](double s) { return s > local; });
    if (k >= ng) k = sm_rank4(g, ng, [&](double s) { return s >= here; });
    // Inside the group: the masses once more, in the same order.  A mass that is nothing next to the row's best (below 2^-1074 of it) may be
    // something next to the tile's: it is not drawn, and where a group holds no other, the next that does is taken (the one before, on the way to
    // the last).  There is one: the tile's sum is something, and so is its best.
    const T* x = scores + r * sstride;
    const SmScale scale = { rule.mode, rule.inv_t, tops[t], 1.0 };
    const SmKept kept = st.kept;
    const bool vec = sm_aligned(x);
    long long drawn = -1;
    for (int q = 0; q < ng && drawn < 0; q++, k = last ? k - 1 : k + 1 < ng ? k + 1 : 0) {
        const long long i0 = (long long)t * SM_STILE + k * SM_GROUP;
        double acc = k ? g[k - 1] : 0.0;
        LgVec4<T> v[SM_GROUP / 4];
#pragma unroll
        for (int e = 0; e < SM_GROUP / 4; e++) v[e] = sm_load4(x, i0 + 4 * e, V, vec);
        float z[SM_GROUP];
        double mass[SM_GROUP];
#pragma unroll
        for (int e = 0; e < SM_GROUP; e++) {
            const float y = sm_score(v[e / 4].v[e % 4], sm_floor(rule));
            z[e] = sm_in(kept, y, (uint32_t)(i0 + e)) ? y : -INFINITY;
        }
        sm_masses(tables, scale, z, mass);
        int found = -1, any = -1;
#pragma unroll
        for (int e = 0; e < SM_GROUP; e++) {
            acc += mass[e];
            if (mass[e] * scale_up > 0.0) { any = e; if (found < 0 && !last && acc > local) found = e; }
        }
        if (any >= 0) drawn = i0 + (found >= 0 ? found : any);
    }
    out[at] = drawn;
}

// ---- long rows, without replacement ----------------------------------------------------------------------------------------------------
// Approximate keys and their first level: one pass over scores and numbers, keys written for the passes to come (4 bytes an element in the
// place of 8, and two logarithms less).  3 M: 17 us (36 MB moved), 10 M 23 us behind top-p.
template <typename T>
__global__ void __launch_bounds__(SM_LTPB) sm_race_kernel(const T* __restrict__ scores, long long sstride, const float* __restrict__ u, long long ustride,
                                                          long long V, long long n, SmRule rule, SmWork wk, int step)
{
    constexpr int P = SM_RBITS1 - 6;
    __shared__ uint32_t h[sm_slots(P)];
    __shared__ SmScratch sc;
    __shared__ uint32_t ticket;
    const long long r = blockIdx.x / wk.B, b = blockIdx.x % wk.B;
    SmRowState& st = wk.state(r);
    const T* x = scores + r * sstride;
    u += r * ustride;
    uint32_t* keys = wk.keys + r * wk.vpad;
    const bool logits = rule.mode == SM_LOGITS, vec = sm_aligned(x), uvec = sm_aligned(u);
    const float floor = sm_floor(rule);
    const float slope = sm_slope(rule);
    const SmKept kept = sm_final(wk, r, st, rule);
    const long long stride = wk.B * SM_LTPB * 4;
    constexpr int G = 2;
    long long i = (b * SM_LTPB + threadIdx.x) * 4;
    LgVec4<T> v[G];
    LgVec4<float> uk[G];
#pragma unroll
    for (int g = 0; g < G; g++) { v[g] = sm_load4(x, i + g * stride, V, vec); uk[g] = sm_load4(u, i + g * stride, V, uvec); }
    for (int k = threadIdx.x; k < sm_slots(P); k += SM_LTPB) h[k] = 0;
    __syncthreads();
    while (i < V) {
#pragma unroll
        for (int g = 0; g < G; g++) {
            const long long at = i + g * stride;
            LgVec4<uint32_t> o;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float y = sm_score(v[g].v[j], floor);
                o.v[j] = sm_in(kept, y, (uint32_t)(at + j)) ? sm_order(sm_race32(logits, slope, y, uk[g].v[j])) : 0u;
                if (o.v[j]) atomicAdd(&h[sm_slot((int)(o.v[j] >> (32 - SM_RBITS1)), P)], 1u);
            }
            if (at < V) *(LgVec4<uint32_t>*)(keys + at) = o;           // (padded to a multiple of four: what lies behind V is key 0)
        }
        i += G * stride;
        if (i >= V) break;
#pragma unroll
        for (int g = 0; g < G; g++) { v[g] = sm_load4(x, i + g * stride, V, vec); uk[g] = sm_load4(u, i + g * stride, V, uvec); }
    }
    __syncthreads();
    uint32_t* g = wk.rbins(r);
    for (int i = threadIdx.x; i < SM_RBINS; i += SM_LTPB) if (const uint32_t c = h[sm_nth_slot(i)]) atomicAdd(&g[i], c);
    if (!sm_last_block(st, step, (uint32_t)b, (uint32_t)wk.B, &ticket)) return;
    uint32_t n4[SM_RBINS / SM_LTPB];
#pragma unroll
    for (int k = 0; k < SM_RBINS / SM_LTPB; k++) n4[k] = sm_peek(&g[k * SM_LTPB + threadIdx.x]);
#pragma unroll
    for (int k = 0; k < SM_RBINS / SM_LTPB; k++) { h[sm_nth_slot(k * SM_LTPB + threadIdx.x)] = n4[k]; g[k * SM_LTPB + threadIdx.x] = 0; }
    __syncthreads();
    SmTake take = { (double)n, 0, { 0, 0 } };
    const SmBin bin = sm_boundary<false>(h, nullptr, nullptr, P, take, sc);
    if (threadIdx.x != 0) return;
    st.kept = kept;
    st.candidates = 0;
    st.take = take;
    st.prefix = (uint32_t)(bin.bin < 0 ? 0 : bin.bin);
    st.ended = 0;
    if (bin.total <= (unsigned long long)n) { st.ended = 1; st.zone_lo = 1u; st.zone_hi = 0u; }        // whatever is left wins: nothing to rank
}

// Second level, and the zone (3 M: 9 us, one read of the keys)
__global__ void __launch_bounds__(SM_LTPB) sm_race_level_kernel(long long V, SmRule rule, SmWork wk, int step)
{
    constexpr int P = SM_RBITS2 - 6;
    __shared__ uint32_t h[sm_slots(P)];
    __shared__ SmScratch sc;
    __shared__ uint32_t ticket;
    const long long r = blockIdx.x / wk.B, b = blockIdx.x % wk.B;
    SmRowState& st = wk.state(r);
    if (st.ended) return;
    const uint32_t* keys = wk.keys + r * wk.vpad;
    const uint32_t prefix = st.prefix;
    const int nbins = 1 << SM_RBITS2, at = 32 - SM_RBITS1 - SM_RBITS2;
    for (int i = threadIdx.x; i < sm_slots(P); i += SM_LTPB) h[i] = 0;
    __syncthreads();
    const long long stride = wk.B * SM_LTPB * 4;
    for (long long i = (b * SM_LTPB + threadIdx.x) * 4; i < V; i += 4 * stride) {
        LgVec4<uint32_t> o[4];
#pragma unroll
        for (int g = 0; g < 4; g++) o[g] = i + g * stride < V ? *(const LgVec4<uint32_t>*)(keys + i + g * stride) : LgVec4<uint32_t>{ { 0, 0, 0, 0 } };
#pragma unroll
        for (int g = 0; g < 4; g++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (o[g].v[j] && (o[g].v[j] >> (32 - SM_RBITS1)) == prefix) atomicAdd(&h[sm_slot((int)(o[g].v[j] >> at) & (nbins - 1), P)], 1u);
    }
    __syncthreads();
    uint32_t* g = wk.rbins(r);
    for (int i = threadIdx.x; i < nbins; i += SM_LTPB) if (const uint32_t c = h[sm_nth_slot(i)]) atomicAdd(&g[i], c);
    if (!sm_last_block(st, step, (uint32_t)b, (uint32_t)wk.B, &ticket)) return;
    for (int i = threadIdx.x; i < nbins; i += SM_LTPB) h[sm_nth_slot(i)] = sm_peek(&g[i]);
    __syncthreads();
    SmTake take = st.take;
    const SmBin bin = sm_boundary<false>(h, nullptr, nullptr, P, take, sc);
    if (threadIdx.x != 0) return;
    const uint32_t lo = (prefix << (32 - SM_RBITS1)) | ((uint32_t)(bin.bin < 0 ? 0 : bin.bin) << at);
    const SmZone zone = sm_zone(lo, lo | ((1u << at) - 1), sm_slope(rule));
    st.zone_lo = zone.lo;
    st.zone_hi = zone.hi;
}

#define SM_ZTILES 4096                 // tiles whose winners are counted in LDS
// Winners as a bit per element, the zone's elements as a list, winners counted per tile; the last workgroup ranks the list (3 M: 13 us, 10 M
// 18).  That holds while the zone is small.  Where a good part of the row has one key next to the border -- equal scores at a temperature of a
// thousandth of them or less, which outweigh the numbers, or equal scores with equal numbers -- every one of them is added to the list by an
// atomic on one word, and one workgroup works out their exact keys again and again: a call for 5 % of 100 k, 1 M and 10 M such scores takes 1.6, 18
// and 190 ms (2.4, 25 and 250 with one number for all).
template <typename T>
__global__ void __launch_bounds__(SM_LTPB) sm_zone_kernel(const T* __restrict__ scores, long long sstride, const float* __restrict__ u, long long ustride,
                                                          long long V, long long n, SmRule rule, SmWork wk, int step)
{
    __shared__ union { SmHist hist; struct { unsigned long long rank[SM_BINS]; uint32_t index[SM_BINS]; }; } h;
    __shared__ uint32_t wins[SM_ZTILES], ahead[SM_BINS];
    __shared__ SmScratch sc;
    __shared__ uint32_t ticket;
    const long long r = blockIdx.x / wk.B, b = blockIdx.x % wk.B;
    SmRowState& st = wk.state(r);
    const uint32_t zlo = st.zone_lo, zhi = st.zone_hi;
    const uint32_t* keys = wk.keys + r * wk.vpad;
    unsigned long long* words = wk.words + r * wk.tiles * (SM_TILE / 64);
    uint32_t* tile_n = wk.tile_n + r * wk.tiles;
    uint32_t* list = wk.list + r * wk.capacity;
    const int lane = threadIdx.x & 63;
    for (long long t = b; t < wk.tiles; t += wk.B) {
        uint32_t c = 0, total;
        uint32_t key[SM_TILE / SM_LTPB];
#pragma unroll
        for (int k = 0; k < SM_TILE / SM_LTPB; k++) {
            const long long i = t * SM_TILE + k * SM_LTPB + threadIdx.x;
            key[k] = i < V ? keys[i] : 0u;
        }
#pragma unroll
        for (int k = 0; k < SM_TILE / SM_LTPB; k++) {
            const long long i = t * SM_TILE + k * SM_LTPB + threadIdx.x;
            const unsigned long long w = __ballot(key[k] > zhi);
            if (lane == 0) { sm_poke(&words[i >> 6], w); c += (uint32_t)__popcll(w); }
            if (key[k] >= zlo && key[k] <= zhi) {
                const uint32_t at = atomicAdd(&st.candidates, 1u);
                if (at < (uint32_t)wk.capacity) sm_poke(&list[at], (uint32_t)i);
            }
        }
        sm_block_scan<uint32_t>(c, sc.a, total);
        if (threadIdx.x == 0) { sm_poke(&tile_n[t], total); }
    }
    if (!sm_last_block(st, step, (uint32_t)b, (uint32_t)wk.B, &ticket)) return;
    unsigned long long mine = 0, sure;
    const bool in_lds = wk.tiles <= SM_ZTILES;
    const uint32_t found = sm_peek(&st.candidates);
    for (uint32_t a = threadIdx.x; a < found && a < SM_BINS; a += SM_LTPB) h.index[a] = sm_peek(&list[a]);
    for (long long t = threadIdx.x; t < wk.tiles; t += SM_LTPB) {
        const uint32_t c = sm_peek(&tile_n[t]);
        mine += c;
        if (in_lds) wins[t] = c;
    }
    sm_block_scan<unsigned long long>(mine, sc.a, sure);
    const T* x = scores + r * sstride;
    u += r * ustride;
    const float floor = sm_floor(rule);
    const SmKept kept = st.kept;
    const SmScale scale = sm_scale(rule, -INFINITY);                          // (race keys need no common scale)
    auto race = [&](long long i) {
        const float y = sm_score(x[i], floor);
        return sm_race(scale, sm_in(kept, y, (uint32_t)i) ? y : -INFINITY, u[i]);
    };
    auto win = [&](uint32_t i) {
        atomicOr(&words[i >> 6], 1ull << (i & 63));
        if (in_lds) atomicAdd(&wins[i / SM_TILE], 1u); else atomicAdd(&tile_n[i / SM_TILE], 1u);
    };
    const unsigned long long room = (unsigned long long)n - sure;      // winners still to be named
    if (found <= (uint32_t)wk.capacity && found <= SM_BINS) {
        for (uint32_t a = threadIdx.x; a < found; a += SM_LTPB) h.rank[a] = race((long long)h.index[a]);
        __syncthreads();
        // `parts` threads share a candidate's comparisons
        const uint32_t parts = found <= SM_LTPB / 8 ? 8 : found <= SM_LTPB / 2 ? 2 : 1, each = (found + parts - 1) / parts;
        for (uint32_t a = threadIdx.x; a < found; a += SM_LTPB) ahead[a] = 0;
        __syncthreads();
        for (uint32_t q = threadIdx.x; q < found * parts; q += SM_LTPB) {
            const uint32_t a = q / parts, part = q % parts, i = h.index[a];
            const unsigned long long k = h.rank[a];
            uint32_t n = 0;
            for (uint32_t c = part * each; c < found && c < (part + 1) * each; c++) n += h.rank[c] > k || (h.rank[c] == k && h.index[c] < i);
            if (n) atomicAdd(&ahead[a], n);
        }
        __syncthreads();
        for (uint32_t a = threadIdx.x; a < found; a += SM_LTPB) if (ahead[a] < room) win(h.index[a]);
    } else {
        // many elements next to the border: all but equal keys in numbers.  Radix selection of the exact keys by this workgroup, over the list
        // or, where that was too short, over the row.
        const bool all = found > (uint32_t)wk.capacity;
        const long long m = all ? V : (long long)found;
        auto index = [&](long long a) { return all ? a : (long long)sm_peek(&list[a]); };
        auto key_of = [&](long long a) {
            const long long i = index(a);
            const uint32_t o = keys[i];
            return o >= zlo && o <= zhi ? race(i) : 0ull;
        };
        // one selection of `bits` bits among of(a) != 0: lowest key of the bin it ends in, and that bin
        auto select = [&](int bits, double target, auto&& of, unsigned long long& thr, SmTake& take) {
            take = SmTake{ target, 0, { 0, 0 } };
            SmBin bin = { -1, 0, 0 };
            unsigned long long prefix = 0;
            int shift = bits;
            while (shift > 0) {
                const int width = shift >= 11 ? 11 : shift < 6 ? 6 : shift, low = shift > width ? shift - width : 0;
                __syncthreads();
                for (int k = threadIdx.x; k < sm_slots(width - 6); k += SM_LTPB) h.hist.n[k] = 0;
                __syncthreads();
                for (long long a = threadIdx.x; a < m; a += SM_LTPB) {
                    const unsigned long long k = of(a);
                    if (k != 0ull && (shift == 64 || (k >> shift) == prefix)) atomicAdd(&h.hist.n[sm_slot((int)((k >> low) & ((1ull << (shift - low)) - 1)), width - 6)], 1u);
                }
                __syncthreads();
                bin = sm_boundary<false>(h.hist.n, nullptr, nullptr, width - 6, take, sc);
                if (bin.bin < 0) break;
                prefix = (prefix << (shift - low)) | (unsigned)bin.bin;
                shift = low;
                if (bin.count == 1) break;
            }
            thr = prefix << shift;
            return bin;
        };
        unsigned long long thr = ~0ull;
        uint32_t last = SM_ALL;
        SmTake take;
        const SmBin e = room ? select(64, (double)room, key_of, thr, take) : SmBin{ -1, 0, 0 };
        if (e.bin < 0) thr = ~0ull;
        else if (e.count > 1) {
            const uint32_t ties = sm_ties<false>(take, e.count, 0.0);
            if (ties < e.count) {                                      // the lowest indices among equal keys: selected by the indices' complement
                unsigned long long cut;
                const unsigned long long equal = thr;
                select(32, (double)ties, [&](long long a) { return key_of(a) == equal ? (unsigned long long)~(uint32_t)index(a) : 0ull; }, cut, take);
                last = ~(uint32_t)cut;
            }
        }
        __syncthreads();
        for (long long a = threadIdx.x; a < m; a += SM_LTPB) {
            const unsigned long long k = key_of(a);
            const uint32_t i = (uint32_t)index(a);
            if (k != 0ull && (k > thr || (k == thr && i <= last))) win(i);
        }
    }
    if (!in_lds) __threadfence();
    __syncthreads();
    // tiles' first positions in the output
    unsigned long long run = 0;
    for (long long base = 0; base < wk.tiles; base += SM_LTPB) {
        const long long t = base + threadIdx.x;
        const uint32_t c = t < wk.tiles ? (in_lds ? wins[t] : sm_peek(&tile_n[t])) : 0u;
        unsigned long long total;
        const unsigned long long before = sm_block_scan<unsigned long long>(c, sc.a, total);
        if (t < wk.tiles) tile_n[t] = (uint32_t)(run + before);
        run += total;
    }
    if (threadIdx.x == 0) st.sure = run;
}

// winners' indices, ascending; one workgroup of two waves per tile, one word of winners per thread (150 k of 3 M: 4 us)
__global__ void __launch_bounds__(SM_TILE / 64) sm_emit_kernel(long long n, SmWork wk, long long* __restrict__ out)
{
    __shared__ SmScratch sc;
    const long long r = blockIdx.x / wk.tiles, t = blockIdx.x % wk.tiles;
    out += r * n;
    unsigned long long w = wk.words[(r * wk.tiles + t) * (SM_TILE / 64) + threadIdx.x];
    uint32_t total;
    long long at = (long long)wk.tile_n[r * wk.tiles + t] + sm_block_scan<uint32_t>((uint32_t)__popcll(w), sc.a, total);
    const long long i0 = t * SM_TILE + (long long)threadIdx.x * 64;
    while (w) {
        const int k = __ffsll((long long)w) - 1;
        w &= w - 1;
        if (at < n) out[at] = i0 + k;
        at++;
    }
    // the row's end where fewer than n were left
    const long long m = (long long)wk.state(r).sure;
    for (long long j = m + t * (SM_TILE / 64) + threadIdx.x; j < n; j += wk.tiles * (SM_TILE / 64)) out[j] = -1;
}

// ---- entry points ----------------------------------------------------------------------------------------------------------------------
static bool sm_rule(int logits, double temperature, long long top_k, double top_p, double min_p, SmRule& r)
{
    if (!(temperature >= 1e-30 && temperature <= 1e30) || top_k < 0 || !(top_p > 0.0 && top_p <= 1.0) || !(min_p >= 0.0 && min_p <= 1.0)) return false;
    r = SmRule{ logits ? SM_LOGITS : temperature == 1.0 ? SM_LINEAR : SM_POWER, 1.0 / temperature, top_p, min_p, top_k };
    return true;
}

// How a call runs.  Short rows: one workgroup each, as far as its LDS and registers reach (12288 scores, short and long: plain 10 and 17 us, behind
// top-p 22 and 53, 614 distinct 18 and 25; 64 rows 11 / 18, 22 / 59, 19 / 28).  Long ones: the filters by levels of a histogram, or, for 16-bit
// scores, from one histogram of all keys; what a small top-k leaves goes on as a short row.  Both sides of these two stand at their kernels.
struct SmPlan { bool is_short, top_k, top_p, counts, few; };
#define SM_COUNTS_ROWS 256

static SmPlan sm_plan(long long R, long long V, int bytes, long long top_k, double top_p)
{
    SmPlan p;
    p.is_short = V <= SM_SHORT;
    p.top_k = top_k > 0 && top_k < V;
    p.top_p = top_p < 1.0;
    p.counts = bytes == 2 && (p.top_k || p.top_p) && R <= (p.top_p ? SM_COUNTS_ROWS : SM_COUNTS_ROWS / 2);
    p.few = p.top_k && top_k <= SM_SHORT;
    return p;
}

// lays the workspace out; returns its size in bytes
static long long sm_layout(const SmPlan& plan, long long R, long long V, int bytes, bool distinct, long long top_k, char* base, SmWork& w)
{
    char* p = base;
    auto align = [](long long b) { return (b + 255) & ~255ll; };
    auto take = [&](bool want, long long b) { char* at = p; if (want) p += align(b); return at; };
    const bool race = distinct && !plan.few;
    w.rbins_at = align(sizeof(SmRowState));
    w.hist_at = w.rbins_at + (race ? align(SM_RBINS * 4) : 0);
    w.clear_bytes = w.hist_at + (plan.counts ? 65536 * 4 + 16 * 128 : plan.top_k || plan.top_p ? align(sizeof(SmMerged)) : 0);
    w.tiles = (V + SM_TILE - 1) / SM_TILE;
    w.stiles = (V + SM_STILE - 1) / SM_STILE;
    w.vpad = (V + 3) & ~3ll;
    w.capacity = V / 256 > 4096 ? V / 256 : 4096;
    // 256 workgroups fill the chip, and every further one adds its histogram to the same words of memory (3 M scores behind top-p: 79 us with 256,
    // 95 with 512, 83 with 128)
    const long long want = (V + SM_LTPB * 8 - 1) / (SM_LTPB * 8), most = R >= 256 ? 1 : 256 / R;
    w.B = want < most ? want : most;
    w.clear = take(true, R * w.clear_bytes);
    w.best = plan.counts ? nullptr : (uint32_t*)take(true, R * w.B * 4);        // (else the histogram of all keys tells)
    w.tile_n = (uint32_t*)take(true, R * w.tiles * 4);
    w.tile_eq = (uint32_t*)take(true, R * w.tiles * 4);
    w.names = (uint32_t*)take(plan.few, R * top_k * 4);
    w.few = take(plan.few, R * top_k * bytes);
    w.few_u = take(plan.few && distinct, R * top_k * 4);
    w.keys = (uint32_t*)take(race, R * w.vpad * 4);
    w.words = (unsigned long long*)take(race, R * w.tiles * (SM_TILE / 64) * 8);
    w.list = (uint32_t*)take(race, R * w.capacity * 4);
    const bool sums = !distinct && !plan.few;
    w.group = (double*)take(sums, R * w.stiles * (SM_STILE / SM_GROUP) * 8);
    w.tile_sum = (double*)take(sums, R * w.stiles * 8);
    w.tile_top = (double*)take(sums, R * w.stiles * 8);
    return p - base;
}

template <typename T>
static void sample_short(const T* scores, long long ss, const float* u, long long us, long long R, long long V, long long n, const SmRule& rule,
                         const uint32_t* names, long long* out, bool distinct, hipStream_t s)
{
    // Many draws of few rows: workgroups that would idle filter the row once more and share its draws.  By one workgroup 5000 draws of 1000
    // scores take 22 us and 100000 of 10000 171 us; with 4096 draws a workgroup 13 and 17 us, with 1024 7 and 12 us (7 and 12 us are 1000 draws).
    const long long share = (n + 1023) / 1024, most = R < 256 ? 256 / R : 1;
    const long long rows = 1ll << 21;                                  // of a launch: its threads are counted in 32 bits
    for (long long r = 0; r < R; r += rows) {
        const dim3 grid((unsigned)(R - r < rows ? R - r : rows), distinct ? 1u : (unsigned)(share < most ? share : most));
        const T* x = scores + r * ss;
        const float* v = u + r * us;
        const uint32_t* nm = names ? names + r * V : nullptr;
        long long* o = out + r * n;
#define SM_LAUNCH_SHORT(TPB_, EPT_)                                                                                                                 \
    do {                                                                                                                                            \
        if (distinct) hipLaunchKernelGGL((sample_short_kernel<T, TPB_, EPT_, true>), grid, dim3(TPB_), 0, s, x, ss, v, us, (int)V, n, rule, nm, o); \
        else hipLaunchKernelGGL((sample_short_kernel<T, TPB_, EPT_, false>), grid, dim3(TPB_), 0, s, x, ss, v, us, (int)V, n, rule, nm, o);         \
    } while (0)
        // 300 scores in 256 x 4, 1024 x 4 and 768 x 16 threads x elements: a plain draw 4.4, 5.8 and 8.4 us, 512 rows of them 5.4, 11.3 and 16.6; 3000
        // scores in the last two 5.9 and 8.6, 512 rows 12.3 and 17.2
        if (V <= 1024) SM_LAUNCH_SHORT(256, 4);
        else if (V <= 4096) SM_LAUNCH_SHORT(1024, 4);
        else SM_LAUNCH_SHORT(768, 16);
#undef SM_LAUNCH_SHORT
    }
}

template <typename T>
static int sample_launch(const T* scores, long long ss, const float* u, long long us, long long R, long long V, long long n,
                         const SmRule& rule, long long* out, bool distinct, void* temp, long long temp_bytes, hipStream_t s)
{
    const SmPlan plan = sm_plan(R, V, (int)sizeof(T), rule.top_k, rule.top_p);
    if (plan.is_short) {
        sample_short(scores, ss, u, us, R, V, n, rule, nullptr, out, distinct, s);
        LG_RETURN_LAST();
    }
    SmWork wk;
    const long long need = sm_layout(plan, R, V, (int)sizeof(T), distinct, rule.top_k, (char*)temp, wk);
    const long long draws = R * ((n + 255) / 256);
    if (temp == nullptr || temp_bytes < need || (uintptr_t)temp % 16 != 0 || R * wk.tiles > 0x3fffffll || draws > 0xffffffll) return (int)hipErrorInvalidValue;        // (threads of a launch: 32 bits)
    const dim3 grid((unsigned)(R * wk.B)), block(SM_LTPB);
    int step = 0;
    const int want_best = !plan.counts && (plan.top_p || rule.min_p > 0.0);
    hipLaunchKernelGGL((sm_begin_kernel<T>), grid, block, 0, s, scores, ss, V, rule, wk, want_best);
    if (plan.counts) {
        if constexpr (sizeof(T) == 2) {
            SmWork cw = wk;                                            // counters of 16 bits: a bounded share of the row each
            const long long shares = (V + SM_SHARE16 - 1) / SM_SHARE16;
            cw.B = shares > wk.B ? shares : wk.B;
            hipLaunchKernelGGL((sm_count16_kernel<T>), dim3((unsigned)(R * cw.B)), dim3(1024), 0, s, scores, ss, V, rule, cw, step++, (int)plan.top_k, (int)plan.top_p);
        }
    }
    for (int pass = 0; pass < 2; pass++) {
        if (plan.counts ? pass == 0 : !(pass == 0 ? plan.top_k : plan.top_p && !plan.few)) continue;
        if (!plan.counts)
            for (int shift = 32; shift > 0; ) {
                const int width = shift == 21 ? 10 : 11;               // 11, 10, 11: the second level is the one that may fill all its bins, and all workgroups merge theirs
                if (pass == 0) hipLaunchKernelGGL((sm_level_kernel<T, false>), grid, block, 0, s, scores, ss, V, rule, wk, step++, shift, width);
                else hipLaunchKernelGGL((sm_level_kernel<T, true>), grid, block, 0, s, scores, ss, V, rule, wk, step++, shift, width);
                shift -= width;
            }
        SmWork tw = wk;
        tw.B = wk.tiles < 256 ? wk.tiles : 256;
        const dim3 tgrid((unsigned)(R * tw.B));
        if (plan.few) hipLaunchKernelGGL((sm_cut_kernel<T, true>), tgrid, block, 0, s, scores, ss, V, rule, tw, step++);
        else hipLaunchKernelGGL((sm_cut_kernel<T, false>), tgrid, block, 0, s, scores, ss, V, rule, tw, step++);
    }
    if (plan.few) {
        const long long K = rule.top_k;
        hipLaunchKernelGGL((sm_gather_kernel<T>), dim3((unsigned)(R * wk.tiles)), block, 0, s, scores, ss, distinct ? u : nullptr, us, V, rule, wk);
        SmRule rest = rule;
        rest.top_k = 0;
        if (plan.counts) rest.top_p = 1.0;
        if (distinct) sample_short((const T*)wk.few, K, (const float*)wk.few_u, K, R, K, n, rest, wk.names, out, true, s);
        else sample_short((const T*)wk.few, K, u, us, R, K, n, rest, wk.names, out, false, s);
        LG_RETURN_LAST();
    }
    if (!distinct) {
        SmWork sw = wk;
        sw.B = wk.stiles < 5 * wk.B ? wk.stiles : 5 * wk.B;            // (five workgroups of four waves fit a CU)
        hipLaunchKernelGGL((sm_sums_kernel<T>), dim3((unsigned)(R * sw.B)), dim3(256), 0, s, scores, ss, V, rule, sw, wk, step++);
        hipLaunchKernelGGL((sm_draw_kernel<T>), dim3((unsigned)draws), dim3(256), 0, s, scores, ss, u, us, V, n, rule, wk, out);
        LG_RETURN_LAST();
    }
    hipLaunchKernelGGL((sm_race_kernel<T>), grid, block, 0, s, scores, ss, u, us, V, n, rule, wk, step++);
    hipLaunchKernelGGL(sm_race_level_kernel, grid, block, 0, s, V, rule, wk, step++);
    SmWork zw = wk;
    zw.B = wk.tiles < wk.B ? wk.tiles : wk.B;
    hipLaunchKernelGGL((sm_zone_kernel<T>), dim3((unsigned)(R * zw.B)), block, 0, s, scores, ss, u, us, V, n, rule, zw, step++);
    hipLaunchKernelGGL(sm_emit_kernel, dim3((unsigned)(R * wk.tiles)), dim3(SM_TILE / 64), 0, s, n, wk, out);
    LG_RETURN_LAST();
}

LG_API long long lg_sample_temp_bytes(long long R, long long V, long long n, int dtype, int distinct, long long top_k, double top_p)
{
    if (R <= 0 || n <= 0 || V <= SM_SHORT || V >= (1ll << 31)) return 0;
    const int bytes = dtype == LG_F32 ? 4 : 2;
    SmWork w;
    return sm_layout(sm_plan(R, V, bytes, top_k, top_p), R, V, bytes, distinct != 0, top_k, nullptr, w);
}

LG_API int lg_sample(const void* scores, int dtype, long long score_stride, const float* u, long long u_stride, long long R, long long V,
                     long long n, int distinct, int logits, double temperature, long long top_k, double top_p, double min_p,
                     int64_t* out, void* temp, long long temp_bytes, void* stream)
{
    SmRule rule;
    if (R < 0 || V < 0 || n < 0 || R > 0x7fffffffll || V >= (1ll << 31) || !sm_rule(logits, temperature, top_k, top_p, min_p, rule)) return (int)hipErrorInvalidValue;
    if (R == 0 || n == 0) return 0;
    LG_REQUIRE(out);
    if (V > 0) LG_REQUIRE(scores, u);
    if (distinct && n > V) return (int)hipErrorInvalidValue;
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
    case LG_F32: return sample_launch((const float*)scores, score_stride, u, u_stride, R, V, n, rule, (long long*)out, distinct != 0, temp, temp_bytes, s);
    case LG_F16: return sample_launch((const LgHalf*)scores, score_stride, u, u_stride, R, V, n, rule, (long long*)out, distinct != 0, temp, temp_bytes, s);
    case LG_BF16: return sample_launch((const LgBf16*)scores, score_stride, u, u_stride, R, V, n, rule, (long long*)out, distinct != 0, temp, temp_bytes, s);
    }
    return (int)hipErrorInvalidValue;
}
