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
// All masses, sums and keys are in 64 bits: an index has to be the same as the definition's however many categories there are.  Masses that
// are added by atomics (top-p's histograms) are added as integers (two 64-bit limbs of 32 fraction bits each, relative to the largest mass),
// so that neither their order nor the launch changes a result; floating sums have one fixed order.
#include "lg_common.h"
#include "lg_types.h"
#include "litegs_hip.h"

#define SM_TPB 1024
#define SM_BINS 2048
#define SM_EPT 4                       // consecutive elements per thread of a prefix-sum step
#define SM_STEP (SM_TPB * SM_EPT)

enum { SM_LOGITS = 0, SM_LINEAR = 1, SM_POWER = 2 };

struct SmRule { int mode; double temperature, top_p, min_p; long long top_k; };

// ---- scores as ordered keys ----------------------------------------------------------------------------------------------------------
template <typename T> struct SmMax;
template <> struct SmMax<float> { static constexpr float v = 3.402823466e38f; };
template <> struct SmMax<LgHalf> { static constexpr float v = 65504.0f; };
template <> struct SmMax<LgBf16> { static constexpr float v = 3.3895313892515355e38f; };

// larger score <=> larger key; 0 = excluded
template <typename T> __device__ __forceinline__ uint32_t sm_key(T raw, bool logits)
{
    float x = lg_to_float(raw);
    if (!(x == x) || (logits ? x == -INFINITY : x <= 0.0f)) return 0u;
    x = fminf(x, SmMax<T>::v) + 0.0f;                                  // (-0 + 0 = +0: equal scores have equal keys)
    const uint32_t b = __float_as_uint(x);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ double sm_value(uint32_t key)
{
    return (double)__uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}

struct SmScale { int mode; double temperature, top /*l of the best score, or its weight*/, shift /*power of two that brings a linear weight below one*/; };

__device__ __forceinline__ SmScale sm_scale(const SmRule& r, uint32_t best)
{
    SmScale s = { r.mode, r.temperature, 0.0, 1.0 };
    if (best == 0u) return s;
    const double x = sm_value(best);
    if (r.mode == SM_LOGITS) s.top = x / r.temperature;
    else if (r.mode == SM_POWER) s.top = log(x) / r.temperature;
    else { s.top = x; s.shift = ldexp(1.0, -ilogb(x) - 1); }
    return s;
}
__device__ __forceinline__ double sm_log(const SmScale& s, uint32_t key)
{
    const double x = sm_value(key);
    return s.mode == SM_LOGITS ? x / s.temperature : s.mode == SM_POWER ? log(x) / s.temperature : log(x);
}
__device__ __forceinline__ double sm_mass(const SmScale& s, uint32_t key)
{
    if (key == 0u) return 0.0;
    return s.mode == SM_LINEAR ? sm_value(key) : exp(sm_log(s, key) - s.top);
}
// key of the exponential race, ordered as an unsigned integer; 0 = excluded
__device__ __forceinline__ unsigned long long sm_race(const SmScale& s, uint32_t key, float u)
{
    if (key == 0u) return 0ull;
    u = u == u ? fminf(fmaxf(u, 0x1p-33f), 1.0f - 0x1p-24f) : 1.0f - 0x1p-24f;
    const double k = sm_log(s, key) - log(-log1p(-(double)u)) + 0.0;
    const unsigned long long b = (unsigned long long)__double_as_longlong(k);
    return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}

// ---- sums of masses that do not depend on their order --------------------------------------------------------------------------------
struct SmSum { unsigned long long hi, lo; };                           // (hi + lo / 2^32) / 2^32, both limbs carry-free up to 2^31 terms
__device__ __forceinline__ SmSum sm_limbs(double m)                    // 0 <= m <= 1
{
    const double a = m * 4294967296.0;
    const unsigned long long hi = (unsigned long long)a;
    return SmSum{ hi, (unsigned long long)((a - (double)hi) * 4294967296.0) };
}
__device__ __forceinline__ double sm_sum_value(SmSum s)
{
    const unsigned long long hi = s.hi + (s.lo >> 32), lo = s.lo & 0xffffffffull;
    return (double)hi * 0x1p-32 + (double)lo * 0x1p-64;
}

// ---- workgroup-wide scans (fixed order) ----------------------------------------------------------------------------------------------
template <typename V> __device__ __forceinline__ V sm_shfl_up(V v, int d) { return __shfl_up(v, d); }

// exclusive prefix of v over the workgroup and the total; `part` is LDS for one value per wave (+ 1)
template <typename V> __device__ __forceinline__ V sm_block_scan(V v, V* part, V& total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    V inc = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const V o = sm_shfl_up(inc, d);
        if (lane >= d) inc += o;
    }
    __syncthreads();
    if (lane == 63) part[wave] = inc;
    __syncthreads();
    if (wave == 0) {
        V w = lane < waves ? part[lane] : (V)0;
        V winc = w;
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) {
            const V o = sm_shfl_up(winc, d);
            if (lane >= d) winc += o;
        }
        if (lane < waves) part[lane] = winc - w;
        if (lane == waves - 1) part[waves] = winc;
    }
    __syncthreads();
    total = part[waves];
    return part[wave] + (inc - v);
}

__device__ __forceinline__ unsigned long long sm_block_max(unsigned long long v, unsigned long long* part)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) { const unsigned long long o = __shfl_xor(v, d); v = o > v ? o : v; }
    __syncthreads();
    if (lane == 0) part[wave] = v;
    __syncthreads();
    v = part[0];
    for (int w = 1; w < waves; w++) v = part[w] > v ? part[w] : v;
    return v;
}

// ---- histogram of one level of a radix selection, and the bin in which the selection ends ---------------------------------------------
struct SmHist { uint32_t n[SM_BINS]; unsigned long long hi[SM_BINS], lo[SM_BINS]; };

// An element is taken while what lies before it (best first) is less than the target.  `by_mass` false: counted in elements; true: in mass.
struct SmTake { bool by_mass; double target; unsigned long long before_n; SmSum before_m; };

struct SmScratch { unsigned long long u64[20], u64b[20], u64c[20]; double f64[20]; uint32_t u32[20]; unsigned long long word[4]; };

// The lowest non-empty bin whose predecessors (the bins above it) leave room.  Updates take.before_* to the amount above that bin and
// returns the bin and its count; bin = -1: nothing there.
__device__ int sm_boundary(const SmHist& h, int nbins, SmTake& take, SmScratch& sc, unsigned long long& count)
{
    const int per = (nbins + SM_TPB - 1) / SM_TPB;                     // 1 or 2; thread t owns the bins nbins-1 - per*t - k
    unsigned long long n[2] = { 0, 0 }, hi[2] = { 0, 0 }, lo[2] = { 0, 0 };
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const int b = nbins - 1 - ((int)threadIdx.x * per + k);
        if (k < per && b >= 0) {
            n[k] = h.n[b];
            if (take.by_mass) { hi[k] = h.hi[b]; lo[k] = h.lo[b]; }
        }
    }
    unsigned long long tn, thi = 0, tlo = 0, bhi = 0, blo = 0;
    unsigned long long bn = sm_block_scan<unsigned long long>(n[0] + n[1], sc.u64, tn);
    if (take.by_mass) {
        bhi = sm_block_scan<unsigned long long>(hi[0] + hi[1], sc.u64b, thi);
        blo = sm_block_scan<unsigned long long>(lo[0] + lo[1], sc.u64c, tlo);
    }
    unsigned long long mine = 0;                                       // 1 + position in descending order of the last bin that is entered
    unsigned long long an = 0, ahi = 0, alo = 0, ac = 0;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const unsigned long long before_n = take.before_n + bn;
        const SmSum before_m = { take.before_m.hi + bhi, take.before_m.lo + blo };
        const bool room = take.by_mass ? sm_sum_value(before_m) < take.target : (double)before_n < take.target;
        if (k < per && n[k] != 0 && room) {
            mine = (unsigned long long)threadIdx.x * per + k + 1;
            an = before_n; ahi = before_m.hi; alo = before_m.lo; ac = n[k];
        }
        bn += n[k]; bhi += hi[k]; blo += lo[k];
    }
    const unsigned long long best = sm_block_max(mine, sc.u64);
    if (best == 0) { count = 0; return -1; }
    __syncthreads();
    if (mine == best) { sc.word[0] = an; sc.word[1] = ahi; sc.word[2] = alo; sc.word[3] = ac; }
    __syncthreads();
    take.before_n = sc.word[0];
    take.before_m = SmSum{ sc.word[1], sc.word[2] };
    count = sc.word[3];
    __syncthreads();
    return nbins - (int)best;
}

// of `count` elements of equal key behind what is before them: how many are taken (at least one, by the choice of the bin)
__device__ __forceinline__ unsigned long long sm_ties(const SmTake& take, unsigned long long count, double mass)
{
    if (!take.by_mass) {
        const double left = take.target - (double)take.before_n;
        return left >= (double)count ? count : (unsigned long long)ceil(left);
    }
    const SmSum one = sm_limbs(mass);
    auto room = [&](unsigned long long j) {                            // is the j-th equal (from 0) taken?
        return sm_sum_value(SmSum{ take.before_m.hi + j * one.hi, take.before_m.lo + j * one.lo }) < take.target;
    };
    unsigned long long lo = 1, hi = count;                             // room(0) holds; the answer is the first j without room
    while (lo < hi) {
        const unsigned long long mid = lo + (hi - lo) / 2;
        if (room(mid)) lo = mid + 1; else hi = mid;
    }
    return lo;
}

// ---- one workgroup per row -----------------------------------------------------------------------------------------------------------
// what passes the filters: key > thr, or key == thr and index <= last; and mass >= least
struct SmKept { uint32_t thr; long long last; double least; };

template <typename T> struct SmRow {
    const T* x; long long V; bool logits; SmScale scale;
    __device__ __forceinline__ uint32_t key(long long i) const { return sm_key(x[i], logits); }
    __device__ __forceinline__ bool in(const SmKept& k, uint32_t key, long long i) const
    {
        return key != 0u && (key > k.thr || (key == k.thr && i <= k.last)) && (k.least <= 0.0 || sm_mass(scale, key) >= k.least);
    }
};

// shrinks `kept` to the elements that `take` leaves; keys(i) is an unsigned key of `bits` bits (0: not a candidate)
template <int BITS, typename Key, typename Mass>
__device__ void sm_select(long long V, const Key& keys, const Mass& mass_of, SmTake take, SmHist& h, SmScratch& sc,
                          unsigned long long& thr, unsigned long long& ties, unsigned long long& equal)
{
    unsigned long long prefix = 0, count = 0;
    int shift = BITS;
    while (shift > 0) {
        const int width = shift >= 11 ? 11 : shift;
        const int at = shift - width, nbins = 1 << width;
        __syncthreads();
        for (int b = threadIdx.x; b < nbins; b += SM_TPB) { h.n[b] = 0; if (take.by_mass) { h.hi[b] = 0; h.lo[b] = 0; } }
        __syncthreads();
        for (long long i = threadIdx.x; i < V; i += SM_TPB) {
            const unsigned long long k = keys(i);
            if (k == 0ull || (shift < 64 && (k >> shift) != prefix)) continue;
            const int b = (int)((k >> at) & (unsigned long long)(nbins - 1));
            atomicAdd(&h.n[b], 1u);
            if (take.by_mass) {
                const SmSum m = sm_limbs(mass_of(k));
                if (m.hi) atomicAdd(&h.hi[b], m.hi);
                if (m.lo) atomicAdd(&h.lo[b], m.lo);
            }
        }
        __syncthreads();
        const int b = sm_boundary(h, nbins, take, sc, count);
        if (b < 0) { thr = ~0ull; ties = 0; equal = 0; return; }       // no candidate at all
        prefix = (prefix << width) | (unsigned)b;
        shift = at;
    }
    thr = prefix;
    equal = count;
    ties = sm_ties(take, count, take.by_mass ? mass_of(thr) : 0.0);
}

// index of the n-th (from 1) element with is(i), in index order
template <typename Is> __device__ long long sm_nth(long long V, unsigned long long n, const Is& is, SmScratch& sc)
{
    unsigned long long done = 0;
    __syncthreads();
    if (threadIdx.x == 0) sc.word[0] = ~0ull;
    __syncthreads();
    for (long long base = 0; base < V; base += SM_TPB) {
        const long long i = base + threadIdx.x;
        const bool f = i < V && is(i);
        uint32_t total;
        const uint32_t before = sm_block_scan<uint32_t>(f ? 1u : 0u, sc.u32, total);
        if (f && done + before + 1 == n) sc.word[0] = (unsigned long long)i;
        done += total;
        if (done >= n) break;
    }
    __syncthreads();
    const long long at = (long long)sc.word[0];
    __syncthreads();
    return at;
}

template <typename T>
__device__ SmKept sm_filter_row(SmRow<T>& row, const SmRule& rule, SmHist& h, SmScratch& sc)
{
    unsigned long long best = 0;
    for (long long i = threadIdx.x; i < row.V; i += SM_TPB) { const unsigned long long k = row.key(i); best = k > best ? k : best; }
    best = sm_block_max(best, sc.u64);
    row.scale = sm_scale(rule, (uint32_t)best);
    SmKept kept = { 0u, 0x7fffffffffffffffll, 0.0 };
    if (best == 0) return kept;
    const double unit = row.scale.mode == SM_LINEAR ? row.scale.shift : 1.0;
    auto mass_of = [&](unsigned long long k) { return sm_mass(row.scale, (uint32_t)k) * unit; };
    for (int pass = 0; pass < 2; pass++) {
        SmTake take = { pass == 1, 0.0, 0, { 0, 0 } };
        if (pass == 0) {
            if (rule.top_k <= 0 || rule.top_k >= row.V) continue;
            take.target = (double)rule.top_k;
        } else {
            if (rule.top_p >= 1.0) continue;
            unsigned long long hi = 0, lo = 0;
            for (long long i = threadIdx.x; i < row.V; i += SM_TPB) {
                const uint32_t k = row.key(i);
                if (!row.in(kept, k, i)) continue;
                const SmSum m = sm_limbs(mass_of(k));
                hi += m.hi; lo += m.lo;
            }
            SmSum total;
            sm_block_scan<unsigned long long>(hi, sc.u64, total.hi);
            sm_block_scan<unsigned long long>(lo, sc.u64b, total.lo);
            take.target = rule.top_p * sm_sum_value(total);
        }
        unsigned long long thr, ties, equal;
        const SmKept before = kept;
        auto keys = [&](long long i) { const uint32_t k = row.key(i); return row.in(before, k, i) ? (unsigned long long)k : 0ull; };
        sm_select<32>(row.V, keys, mass_of, take, h, sc, thr, ties, equal);
        kept.thr = (uint32_t)thr;
        if (kept.thr != before.thr) kept.last = 0x7fffffffffffffffll;      // an earlier filter's cut was among other equals
        if (ties < equal) kept.last = sm_nth(row.V, ties, [&](long long i) { return keys(i) == thr; }, sc);
    }
    if (rule.min_p > 0.0) kept.least = rule.min_p * sm_mass(row.scale, (uint32_t)best);
    return kept;
}

template <typename T>
__global__ void __launch_bounds__(SM_TPB) sample_row_kernel(const T* __restrict__ scores, long long sstride, const float* __restrict__ u, long long ustride,
                                                            long long V, long long n, SmRule rule, long long* __restrict__ out)
{
    __shared__ SmHist h;
    __shared__ SmScratch sc;
    double* cdf = (double*)&h;                                         // the histograms are done when the prefix sums begin
    static_assert(sizeof(SmHist) >= SM_STEP * sizeof(double), "");
    const long long r = blockIdx.x;
    SmRow<T> row = { scores + r * sstride, V, rule.mode == SM_LOGITS, {} };
    const SmKept kept = sm_filter_row(row, rule, h, sc);
    out += r * n;
    u += r * ustride;
    // two passes over the prefix sums of the kept masses, in the same order: the first for the total, the second finds the draws of each step
    auto weight = [&](long long i) {
        if (i >= V) return 0.0;
        const uint32_t k = row.key(i);
        return row.in(kept, k, i) ? sm_mass(row.scale, k) : 0.0;
    };
    double total = 0.0;
    unsigned long long last = 0;
    for (int pass = 0; pass < 2; pass++) {
        double run = 0.0;
        for (long long base = 0; base < V; base += SM_STEP) {
            double w[SM_EPT], sum = 0.0, step;
#pragma unroll
            for (int k = 0; k < SM_EPT; k++) {
                const long long i = base + (long long)threadIdx.x * SM_EPT + k;
                w[k] = weight(i);
                sum += w[k];
                if (pass == 0 && w[k] > 0.0) last = (unsigned long long)i + 1;
            }
            double at = run + sm_block_scan<double>(sum, sc.f64, step);
            if (pass == 1) {
#pragma unroll
                for (int k = 0; k < SM_EPT; k++) { at += w[k]; cdf[threadIdx.x * SM_EPT + k] = at; }
                __syncthreads();
                const double end = run + step;
                for (long long j = threadIdx.x; j < n; j += SM_TPB) {
                    const float uj = u[j];
                    const double t = (uj > 0.0f ? (double)uj : 0.0) * total;
                    if (!(t >= run && (t < end || base + SM_STEP >= V))) continue;
                    int lo = 0, hi = SM_STEP;                          // first position with cdf > t
                    while (lo < hi) { const int mid = (lo + hi) >> 1; if (cdf[mid] > t) hi = mid; else lo = mid + 1; }
                    long long i = base + lo;
                    while (i < (long long)last && !(weight(i) > 0.0)) i++;      // rounding at a border never lands on an excluded element
                    out[j] = i < (long long)last ? i : (long long)last - 1;
                }
            }
            run += step;
        }
        if (pass == 0) {
            total = run;
            last = sm_block_max(last, sc.u64);
            if (last == 0) {                                           // nothing to draw from
                for (long long j = threadIdx.x; j < n; j += SM_TPB) out[j] = -1;
                return;
            }
        }
        __syncthreads();
    }
}

template <typename T>
__global__ void __launch_bounds__(SM_TPB) sample_distinct_row_kernel(const T* __restrict__ scores, long long sstride, const float* __restrict__ u,
                                                                     long long ustride, long long V, long long n, SmRule rule, long long* __restrict__ out)
{
    __shared__ SmHist h;
    __shared__ SmScratch sc;
    const long long r = blockIdx.x;
    SmRow<T> row = { scores + r * sstride, V, rule.mode == SM_LOGITS, {} };
    const SmKept kept = sm_filter_row(row, rule, h, sc);
    out += r * n;
    u += r * ustride;
    auto race = [&](long long i) {
        const uint32_t k = row.key(i);
        return row.in(kept, k, i) ? sm_race(row.scale, k, u[i]) : 0ull;
    };
    unsigned long long thr, ties, equal;
    const SmTake take = { false, (double)n, 0, { 0, 0 } };
    sm_select<64>(V, race, [](unsigned long long) { return 0.0; }, take, h, sc, thr, ties, equal);
    // winners in index order; of the last key's ties the first ones
    unsigned long long done = 0, tied = 0;
    for (long long base = 0; base < V && done < (unsigned long long)n; base += SM_TPB) {
        const long long i = base + threadIdx.x;
        const unsigned long long k = i < V ? race(i) : 0ull;
        bool win = k > thr;
        uint32_t total;
        if (ties < equal) {
            const uint32_t before = sm_block_scan<uint32_t>(k != 0 && k == thr ? 1u : 0u, sc.u32, total);
            win = win || (k != 0 && k == thr && tied + before < ties);
            tied += total;
        } else win = win || (k != 0 && k == thr);
        const uint32_t before = sm_block_scan<uint32_t>(win ? 1u : 0u, sc.u32, total);
        if (win) out[done + before] = i;
        done += total;
    }
    for (long long j = (long long)done + threadIdx.x; j < n; j += SM_TPB) out[j] = -1;
}

// ---- entry points --------------------------------------------------------------------------------------------------------------------
static bool sm_rule(int logits, double temperature, long long top_k, double top_p, double min_p, SmRule& r)
{
    if (!(temperature > 0.0) || !(temperature <= 1e30) || top_k < 0 || !(top_p > 0.0 && top_p <= 1.0) || !(min_p >= 0.0 && min_p <= 1.0)) return false;
    r = SmRule{ logits ? SM_LOGITS : temperature == 1.0 ? SM_LINEAR : SM_POWER, temperature, top_p, min_p, top_k };
    return true;
}

template <typename T>
static int sample_launch(const T* scores, long long sstride, const float* u, long long ustride, long long R, long long V, long long n,
                         const SmRule& rule, long long* out, bool distinct, hipStream_t s)
{
    if (distinct)
        hipLaunchKernelGGL((sample_distinct_row_kernel<T>), dim3((unsigned)R), dim3(SM_TPB), 0, s, scores, sstride, u, ustride, V, n, rule, out);
    else
        hipLaunchKernelGGL((sample_row_kernel<T>), dim3((unsigned)R), dim3(SM_TPB), 0, s, scores, sstride, u, ustride, V, n, rule, out);
    LG_RETURN_LAST();
}

LG_API long long lg_sample_temp_bytes(long long R, long long V, long long n, int distinct, int filtered) { return 0; }

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
    case LG_F32: return sample_launch((const float*)scores, score_stride, u, u_stride, R, V, n, rule, (long long*)out, distinct != 0, s);
    case LG_F16: return sample_launch((const LgHalf*)scores, score_stride, u, u_stride, R, V, n, rule, (long long*)out, distinct != 0, s);
    case LG_BF16: return sample_launch((const LgBf16*)scores, score_stride, u, u_stride, R, V, n, rule, (long long*)out, distinct != 0, s);
    }
    return (int)hipErrorInvalidValue;
}
