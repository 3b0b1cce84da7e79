// Counter-based dropout (forward = backward), uniform and normal draws.  No operator here stores a mask or a state: the words come from
// lg_philox.h.
//
// What bounds them: HBM.  A word costs ~120 issue cycles per wave of 64 lanes and 64 words (20 32x32->64 products per four words), i.e. 3 M
// words take 2.6 us of the chip's vector issue while the 24 MB that dropout moves for them take 5 us; so one thread draws the four words of a
// block once and applies them to as many rows as share them.
#include "lg_common.h"
#include "lg_philox.h"
#include "lg_types.h"
#include "litegs_hip.h"

#define DR_TPB 256

struct DrKey { unsigned long long seed, offset; const long long* offset_dev; };

__device__ __forceinline__ unsigned long long dr_offset(const DrKey& k)
{
    return k.offset_dev ? k.offset + (unsigned long long)*k.offset_dev : k.offset;
}

// y[r, i] = keep(i) ? x[r, i] * scale : 0, keep(i) = word(index(i)) >= threshold, for a group of four consecutive i and `rows` rows.
// index(i) = i, or chunk_ids[i / S] * S + i % S when the columns are chunks compacted out of a larger cloud.
// The product is rounded to 32 bits and then to T, for every T: dr_product keeps the compiler from folding multiply and conversion into one
// mixed-width instruction, which rounds float16 results once and would make them differ from what the same formula gives anywhere else.
// A dropped element is zero whatever it held (NaN and infinity too): selected, not multiplied.
__device__ __forceinline__ float dr_product(float a, float b)
{
    float c = a * b;
    asm volatile("" : "+v"(c));
    return c;
}
// Measured, launch behind launch: 3 M float32 4.9 us a direction (24 MB: 4.9 TB/s), by chunk id 5.6, 45 rows of 500 k 27.5 us (180 MB: 6.5 TB/s, part
// of it from the last-level cache), 8 M bfloat16 8.7 (their words' issue alone 7).  What a forward and a backward pass take of a user's program
// for less than 10 M elements is the autograd engine's host time (40 us).
// Work items are (block of DR_ROWS rows, group), groups innermost, so that short rows fill a workgroup too.
#define DR_ROWS 8
template <typename T, bool VEC>
__global__ void __launch_bounds__(DR_TPB) dropout_kernel(const T* __restrict__ x, T* __restrict__ y, long long lead, long long M,
                                                         unsigned long long threshold, float scale, DrKey key,
                                                         const long long* __restrict__ chunk_ids, int S)
{
    const long long item = (long long)blockIdx.x * DR_TPB + threadIdx.x, groups = (M + 3) >> 2;
    long long rb = 0, g = item;
    if (lead > DR_ROWS) {
        rb = (item | groups) >> 32 ? item / groups : (long long)((uint32_t)item / (uint32_t)groups);
        g = item - rb * groups;
    }
    const long long i0 = 4 * g, r0 = rb * DR_ROWS;
    if (i0 >= M || r0 >= lead) return;
    const unsigned long long offset = dr_offset(key);
    bool keep[4];
    if (chunk_ids == nullptr) {
        const LgWords w = lg_philox((unsigned long long)g, offset, key.seed);
#pragma unroll
        for (int k = 0; k < 4; k++) keep[k] = w.w[k] >= threshold;
    } else if (S % 4 == 0) {                                           // four consecutive columns are one block of words
        const long long a = (i0 | S) >> 32 ? i0 / S : (long long)((uint32_t)i0 / (uint32_t)S);
        const LgWords w = lg_philox(((unsigned long long)chunk_ids[a] * (unsigned)S + (unsigned long long)(i0 - a * S)) >> 2, offset, key.seed);
#pragma unroll
        for (int k = 0; k < 4; k++) keep[k] = w.w[k] >= threshold;
    } else {                                                           // the block may change at each of them
        unsigned long long block = ~0ull;
        LgWords w = {};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const long long i = i0 + k < M ? i0 + k : M - 1;
            const unsigned long long at = (unsigned long long)chunk_ids[i / S] * (unsigned)S + (unsigned long long)(i % S);
            if ((at >> 2) != block) { block = at >> 2; w = lg_philox(block, offset, key.seed); }
            const int m = (int)(at & 3);
            keep[k] = (m == 0 ? w.w[0] : m == 1 ? w.w[1] : m == 2 ? w.w[2] : w.w[3]) >= threshold;
        }
    }
    const int nr = (int)(lead - r0 < DR_ROWS ? lead - r0 : DR_ROWS);
    for (int r = 0; r < nr; r++) {
        const size_t at = (size_t)(r0 + r) * M + i0;
        if (VEC) {
            LgVec4<T> v = *(const LgVec4<T>*)(x + at);
#pragma unroll
            for (int k = 0; k < 4; k++) v.v[k] = keep[k] ? lg_from_float<T>(dr_product(lg_to_float(v.v[k]), scale)) : lg_from_float<T>(0.0f);
            *(LgVec4<T>*)(y + at) = v;
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (i0 + k < M) y[at + k] = keep[k] ? lg_from_float<T>(dr_product(lg_to_float(x[at + k]), scale)) : lg_from_float<T>(0.0f);
        }
    }
}

template <typename T>
static int dropout_launch(const T* x, T* y, long long lead, long long M, unsigned long long threshold, float scale, const DrKey& key,
                          const long long* ids, int S, hipStream_t s)
{
    const long long items = (M + 3) / 4 * ((lead + DR_ROWS - 1) / DR_ROWS), blocks = (items + DR_TPB - 1) / DR_TPB;
    if (blocks > 0xffffffll) return (int)hipErrorInvalidValue;         // (threads of a launch: 32 bits; four elements each)
    const bool vec = M % 4 == 0 && ((uintptr_t)x | (uintptr_t)y) % (4 * sizeof(T)) == 0;
    const dim3 grid((unsigned)blocks);
    if (vec) hipLaunchKernelGGL((dropout_kernel<T, true>), grid, dim3(DR_TPB), 0, s, x, y, lead, M, threshold, scale, key, ids, S);
    else hipLaunchKernelGGL((dropout_kernel<T, false>), grid, dim3(DR_TPB), 0, s, x, y, lead, M, threshold, scale, key, ids, S);
    LG_RETURN_LAST();
}

LG_API int lg_dropout(const void* x, void* y, int dtype, long long lead, long long M, double p, long long seed, long long offset,
                      const int64_t* offset_dev, const int64_t* chunk_ids, int S, void* stream)
{
    if (lead <= 0 || M <= 0) return 0;
    LG_REQUIRE(x, y);
    if (!(p >= 0.0 && p <= 1.0) || (chunk_ids && (S <= 0 || M % S != 0))) return (int)hipErrorInvalidValue;
    const unsigned long long threshold = (unsigned long long)__builtin_rint(p * 4294967296.0);      // 2^32: no word is kept
    const float scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.0f;
    const DrKey key = { (unsigned long long)seed, (unsigned long long)offset, (const long long*)offset_dev };
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
    case LG_F32: return dropout_launch((const float*)x, (float*)y, lead, M, threshold, scale, key, (const long long*)chunk_ids, S, s);
    case LG_F16: return dropout_launch((const LgHalf*)x, (LgHalf*)y, lead, M, threshold, scale, key, (const long long*)chunk_ids, S, s);
    case LG_BF16: return dropout_launch((const LgBf16*)x, (LgBf16*)y, lead, M, threshold, scale, key, (const long long*)chunk_ids, S, s);
    }
    return (int)hipErrorInvalidValue;
}

// -ln(a) for a = (k + 1/2) / 2^32.  In the upper half a is written as 1 - b, so that nothing is lost next to one: ln(1 - b) =
// b * ln(y) / (y - 1) with y = fl(1 - b) (the rounding of y cancels to first order).
__device__ __forceinline__ float dr_neg_log(uint32_t k)
{
    if (k < 0x80000000u) return -logf(((float)k + 0.5f) * 0x1p-32f);
    const float b = ((float)(0xffffffffu - k) + 0.5f) * 0x1p-32f;
    const float y = 1.0f - b;
    return y == 1.0f ? b : logf(y) * b / (y - 1.0f);
}

// (cos, sin) of the angle 2 pi k / 2^32: the quadrant is taken off in integers, what is left lies in [-pi/4, pi/4] and goes through the
// Taylor polynomials (first term left out: x^11 / 11! < 2e-9 and x^12 / 12! < 2e-10).
__device__ __forceinline__ void dr_cos_sin(uint32_t k, float& c, float& s)
{
    const uint32_t q = (k + 0x20000000u) >> 30;
    const float x = (float)(int32_t)(k - (q << 30)) * 1.46291807926715968e-9f;          // 2 pi / 2^32
    const float z = x * x;
    const float sn = fmaf(x * z, fmaf(z, fmaf(z, fmaf(z, 2.7557319224e-6f, -1.9841269841e-4f), 8.3333333333e-3f), -1.6666666667e-1f), x);
    const float cs = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -2.7557319224e-7f, 2.4801587302e-5f), -1.3888888889e-3f), 4.1666666667e-2f), -0.5f), 1.0f);
    const float a = (q & 1) ? sn : cs, b = (q & 1) ? cs : sn;
    c = (q == 1 || q == 2) ? -a : a;
    s = (q >= 2 && q < 4) ? -b : b;
}

// One thread, one block of four words.  10 M uniform float32 9.1 us (40 MB: 4.4 TB/s); normal ones 15.5 us (80 MB: 5.2 TB/s), 3 M 6.8, 150 k 2.6
// (a launch).  Radius, angle and product are worked out in 32 bits: float32 results are then off by some 6e-8 of the largest where 64 bits would
// leave 3e-8, which is no use to a random number and costs several times the instructions.
template <typename T, bool NORMAL, bool VEC>
__global__ void __launch_bounds__(DR_TPB) draw_kernel(const T* __restrict__ std_, T* __restrict__ out, long long n, DrKey key, float top)
{
    const long long g = (long long)blockIdx.x * DR_TPB + threadIdx.x;
    const long long i0 = 4 * g;
    if (i0 >= n) return;
    const LgWords w = lg_philox((unsigned long long)g, dr_offset(key), key.seed);
    float v[4];
    if (NORMAL) {
#pragma unroll
        for (int h = 0; h < 4; h += 2) {
            const float r = sqrtf(2.0f * dr_neg_log(w.w[h]));
            float c, s;
            dr_cos_sin(w.w[h + 1], c, s);
            v[h] = r * c;
            v[h + 1] = r * s;
        }
    } else {
        // (k + 1/2) / 2^32 in (0, 1): rounded to 32 bits, then to T, and kept below one
#pragma unroll
        for (int h = 0; h < 4; h++) v[h] = fminf(lg_to_float(lg_from_float<T>((float)(((double)w.w[h] + 0.5) * 0x1p-32))), top);
    }
    if (VEC && i0 + 4 <= n) {
        LgVec4<T> o;
        if (NORMAL) {
            const LgVec4<T> d = *(const LgVec4<T>*)(std_ + i0);
#pragma unroll
            for (int h = 0; h < 4; h++) v[h] *= lg_to_float(d.v[h]);
        }
#pragma unroll
        for (int h = 0; h < 4; h++) o.v[h] = lg_from_float<T>(v[h]);
        *(LgVec4<T>*)(out + i0) = o;
    } else {
#pragma unroll
        for (int h = 0; h < 4; h++)
            if (i0 + h < n) out[i0 + h] = lg_from_float<T>(NORMAL ? v[h] * lg_to_float(std_[i0 + h]) : v[h]);
    }
}

template <typename T>
static int draw_launch(const T* std_, T* out, long long n, const DrKey& key, float top, hipStream_t s)
{
    const long long blocks = ((n + 3) / 4 + DR_TPB - 1) / DR_TPB;
    if (blocks > 0xffffffll) return (int)hipErrorInvalidValue;         // (threads of a launch: 32 bits; four elements each)
    const bool vec = ((uintptr_t)std_ | (uintptr_t)out) % (4 * sizeof(T)) == 0;
    const dim3 grid((unsigned)blocks);
    if (std_ && vec) hipLaunchKernelGGL((draw_kernel<T, true, true>), grid, dim3(DR_TPB), 0, s, std_, out, n, key, top);
    else if (std_) hipLaunchKernelGGL((draw_kernel<T, true, false>), grid, dim3(DR_TPB), 0, s, std_, out, n, key, top);
    else if (vec) hipLaunchKernelGGL((draw_kernel<T, false, true>), grid, dim3(DR_TPB), 0, s, std_, out, n, key, top);
    else hipLaunchKernelGGL((draw_kernel<T, false, false>), grid, dim3(DR_TPB), 0, s, std_, out, n, key, top);
    LG_RETURN_LAST();
}

LG_API int lg_random_draw(const void* std_ /*nullable*/, void* out, int dtype, long long n, long long seed, long long offset,
                          const int64_t* offset_dev, void* stream)
{
    if (n <= 0) return 0;
    LG_REQUIRE(out);
    const DrKey key = { (unsigned long long)seed, (unsigned long long)offset, (const long long*)offset_dev };
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
    case LG_F32: return draw_launch((const float*)std_, (float*)out, n, key, 1.0f - 0x1p-24f, s);
    case LG_F16: return draw_launch((const LgHalf*)std_, (LgHalf*)out, n, key, 1.0f - 0x1p-11f, s);
    case LG_BF16: return draw_launch((const LgBf16*)std_, (LgBf16*)out, n, key, 1.0f - 0x1p-8f, s);
    }
    return (int)hipErrorInvalidValue;
}
