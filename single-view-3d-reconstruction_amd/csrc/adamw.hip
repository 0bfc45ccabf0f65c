// The optimizer step over many tensors at once: the gradients' common norm, unscaling, clipping and AdamW with
// 32-bit or 8-bit moments (formulas and code formats in sv3d_hip.h).
//
// Tensors reach a kernel as a table in its arguments (captured with the launch, nothing on the device has to
// be kept up to date), at most kTable of them per launch, cut into chunks; a workgroup looks up its chunk's tensor.
#include "element.h"

#include <cfloat>
#include <cmath>
#include <type_traits>

// fused products and sums are written out: the same bits wherever a function is inlined
#pragma clang fp contract(off)

namespace {

using namespace sv3d;

constexpr int kThreads = 256;
// tensors of one launch: the tables have to fit 4 KB of kernel arguments
constexpr int kTable = 76;
constexpr int kSumTable = 250;
constexpr int64_t kPiece = (int64_t)1 << 31;    // elements of one table entry at most
constexpr int kChunk = 2048;        // elements of one workgroup of the update, 32-bit moments
constexpr int kChunk8 = 2048;       // 8-bit moments
constexpr int kBlock = SV3D_STATE_BLOCK;
constexpr int kSumChunk = 4096;
constexpr int kSumGroups = 1024;

// the sum over a workgroup's threads, known to thread 0; `part`: one number per wave
__device__ inline double group_sum(double v, double *part, int waves)
{
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x / 64] = v;
    __syncthreads();
    if (threadIdx.x == 0)
        for (int w = 1; w < waves; ++w) v += part[w];
    return v;
}

// ---- the norm: sums of squares --------------------------------------------------------------------
// Squares and sums in double: a square of an fp32 number neither overflows nor is rounded there, and the order of
// the sum stops to matter for the fp32 norm that is made of it.
struct SumTable {
    const void *grad[kSumTable];
    uint32_t numel[kSumTable];
    int32_t first[kSumTable + 1];   // of each tensor's chunks
    int32_t count;
};
static_assert(sizeof(SumTable) + 8 <= 4096, "kernel arguments");

template <class T>
__global__ __launch_bounds__(kThreads) void grad_square_sums_kernel(SumTable t, double *__restrict__ sums)
{
    __shared__ double part[kThreads / 64];
    double acc[4] = {0.0, 0.0, 0.0, 0.0};
    int k = 0;
    for (int chunk = blockIdx.x; chunk < t.first[t.count]; chunk += gridDim.x) {
        while (chunk >= t.first[k + 1]) ++k;
        const T *g = (const T *)t.grad[k];
        const int64_t at = (int64_t)(chunk - t.first[k]) * kSumChunk;
        const int64_t left = (int64_t)t.numel[k] - at;
        constexpr int V = 16 / (int)sizeof(T), U = kSumChunk / (kThreads * V);
        Words<T, V> w[U];
        // a whole chunk's loads go out together; with the ends checked they would wait for each other
        if (left >= kSumChunk) {
#pragma unroll
            for (int u = 0; u < U; ++u) w[u] = load_words<T, V>(g + at + (u * kThreads + threadIdx.x) * V);
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int o = (u * kThreads + threadIdx.x) * V;
                w[u] = load_words<T, V>(g + at + o, (int)left - o);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j & 3] += (double)w[u][j] * (double)w[u][j];
    }
    const double sum = group_sum((acc[0] + acc[1]) + (acc[2] + acc[3]), part, kThreads / 64);
    if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

// ---- what each tensor's update multiplies by -------------------------------------------------------
struct Factors {
    float grad;         // unscaling, clipping and sign
    float rate;         // lr / (1 - beta1^t)
    float root;         // 1 / sqrt(1 - beta2^t)
    float small_root;   // 2^-16 of that
    float decay;        // lr weight_decay
    float keep;         // 1 - lr weight_decay
    uint32_t key;       // of the dither
    int32_t skip;
};

// What the kernels need of the call's parameters.
struct Scalars {
    double lr, log_b1, log_b2, weight_decay, max_norm;
    const float *lr_device, *grad_scale, *found_inf;
    float *total_norm;
    uint32_t seed;
    int32_t maximize;
};

// What gradients are multiplied by, from the sum of their squares (or none of it); one thread of a call.
__device__ inline double grad_factor(const Scalars &p, double square_sum)
{
    const double inv = p.grad_scale ? 1.0 / (double)*p.grad_scale : 1.0;
    double c = 1.0;
    if (p.max_norm > 0.0) {
        const double norm = sqrt(square_sum) * inv;
        if (p.total_norm) *p.total_norm = (float)norm;
        c = p.max_norm / (norm + 1e-6);
        if (c > 1.0) c = 1.0;                   // a norm that is no number goes through, into every weight
    }
    return (p.maximize ? -inv : inv) * c;
}

// Takes a tensor's step count forward.  In double: beta^t close to 1 is subtracted from 1.
// `grad` is left to the caller.
__device__ inline Factors factors_of(const Scalars &p, float *step)
{
    const int32_t skip = p.found_inf && *p.found_inf != 0.f;
    const double lr = p.lr_device ? (double)*p.lr_device : p.lr;
    const float n = *step + 1.f;
    if (!skip) *step = n;
    Factors f;
    f.grad = 0.f;
    f.rate = (float)(lr / -expm1((double)n * p.log_b1));
    f.root = (float)(1.0 / sqrt(-expm1((double)n * p.log_b2)));
    f.small_root = f.root * 0x1p-16f;
    f.decay = (float)(lr * p.weight_decay);
    f.keep = (float)(1.0 - lr * p.weight_decay);
    f.key = (uint32_t)n * 0x9E3779B1u + p.seed * 0x6A09E667u;
    f.skip = skip;
    return f;
}

constexpr int kSteps = 384;
struct StepTable {
    float *step[kSteps];
    int32_t base, count;
};
static_assert(sizeof(StepTable) + sizeof(Scalars) + 32 <= 4096, "kernel arguments");

// One workgroup: the factors of up to kSteps tensors.  All that does not depend on the norm goes before the wait for its
// partial sums, whose loads go out together (14 M weights, clipped: 75.9 -> 74.8 us).
__global__ __launch_bounds__(kThreads) void adamw_factors_kernel(StepTable t, Scalars p, const double *__restrict__ sums,
                                                                 int num_sums, Factors *__restrict__ out)
{
    __shared__ double part[kThreads / 64];
    __shared__ double grad;
    constexpr int U = kSumGroups / kThreads;
    double sum[U];
#pragma unroll
    for (int u = 0; u < U; ++u) sum[u] = u * kThreads + (int)threadIdx.x < num_sums ? sums[u * kThreads + threadIdx.x] : 0.0;
    Factors mine;
    if ((int)threadIdx.x < t.count) mine = factors_of(p, t.step[threadIdx.x]);
    double acc = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    static_assert(U == 4, "what one launch of sums leaves");
    for (int i = kSumGroups + threadIdx.x; i < num_sums; i += kThreads) acc += sums[i];
    acc = group_sum(acc, part, kThreads / 64);
    if (threadIdx.x == 0) grad = grad_factor(p, acc);
    __syncthreads();
    mine.grad = (float)grad;
    if ((int)threadIdx.x < t.count) out[t.base + threadIdx.x] = mine;
    for (int i = kThreads + threadIdx.x; i < t.count; i += kThreads) {
        Factors f = factors_of(p, t.step[i]);
        f.grad = (float)grad;
        out[t.base + i] = f;
    }
}

// ---- 8-bit moments -----------------------------------------------------------------------------------
// Two rounds of multiplying and folding the high bits down (multipliers: the fractions of sqrt 2 and sqrt 3).
__device__ inline uint32_t dither(uint32_t element, uint32_t key)
{
    uint32_t x = element + key;
    x = (x ^ (x >> 16)) * 0x6A09E667u;
    x = (x ^ (x >> 15)) * 0xBB67AE85u;
    return x ^ (x >> 16);
}

// First moments are the e4m3 numbers that the hardware converts, rounding included: it adds 20 bits below the last kept one
// and cuts (here the 16 bits of the dither and half a one).  They are scaled so that a block's largest value lands in
// [2^7, 2^8).
//
// A code of a second moment is the upper bits of a float32 whose exponent field is as narrow as the code's: with the
// block's values scaled so that the code's smallest exponent meets float32's, bits 20 and up of a value ARE its code, its
// subnormal codes included (float32's own subnormal numbers), and the same 20 bits go in below before they are cut off.
// The block's largest value has code 0xf0 to 0xf8.
constexpr int kFirstBias = 134, kSecondBias = 30;
constexpr int kFirstFloor = 20, kSecondFloor = 34;      // so that every value is a normal number, also as bf16

__device__ inline float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// a byte below the lowest that is ever written (fresh state: 0) counts as that one
__device__ inline float first_unit(uint32_t e) { return power_of_two(max((int)e, kFirstFloor) - kFirstBias); }
__device__ inline int second_power(uint32_t e) { return max((int)e, kSecondFloor) - kSecondBias; }

constexpr uint32_t kInfinity = 0x7f800000u;
__device__ inline uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// what a moment contributes to its block's exponent: an infinity or NaN does not
__device__ inline uint32_t finite_bits(float v) { return magnitude_bits(v) < kInfinity ? magnitude_bits(v) : 0u; }

// four codes of one word
__device__ inline void decode_first(uint32_t codes, float unit, float *out)
{
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
    out[0] = lo[0] * unit;
    out[1] = lo[1] * unit;
    out[2] = hi[0] * unit;
    out[3] = hi[1] * unit;
}

__device__ inline void decode_second(uint32_t codes, int power, float *out)
{
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = ldexpf(__uint_as_float((codes >> (8 * j) & 0xffu) << 20), power);
    // 0xff is no number: the only byte whose low seven bits and one carry into its top bit, and whose top bit is set
    const uint32_t nan = ((codes & 0x7f7f7f7fu) + 0x01010101u) & codes & 0x80808080u;
    if (nan) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (nan >> (8 * j) & 0xffu) out[j] = NAN;
    }
}

// four values, all of them finite, to one word; `h` their dithers
__device__ inline uint32_t encode_first(const float *m, float scale, const uint32_t *h)
{
    int w = 0;
    w = __builtin_amdgcn_cvt_sr_fp8_f32(m[0] * scale, (int)((h[0] & 0xffff0000u) | 0x8000u), w, 0);
    w = __builtin_amdgcn_cvt_sr_fp8_f32(m[1] * scale, (int)((h[1] & 0xffff0000u) | 0x8000u), w, 1);
    w = __builtin_amdgcn_cvt_sr_fp8_f32(m[2] * scale, (int)((h[2] & 0xffff0000u) | 0x8000u), w, 2);
    w = __builtin_amdgcn_cvt_sr_fp8_f32(m[3] * scale, (int)((h[3] & 0xffff0000u) | 0x8000u), w, 3);
    return (uint32_t)w;
}

__device__ inline uint32_t encode_second(const float *v, int power, const uint32_t *h)
{
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t q = (__float_as_uint(ldexpf(v[j], -power)) + ((h[j] & 0xffffu) << 4) + 8u) >> 20 & 0xffu;
        w |= max(q, min(__float_as_uint(v[j]), 1u)) << (8 * j);         // nothing above zero becomes zero
    }
    return w;
}

// in place of the codes that the above made of infinities and NaN
__device__ inline void mark_not_finite(const float *v, uint32_t code, uint32_t *w)
{
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (magnitude_bits(v[j]) >= kInfinity) *w = (*w & ~(0xffu << (8 * j))) | (code | (code == 0x7fu ? __float_as_uint(v[j]) >> 31 << 7 : 0u)) << (8 * j);
}

// ---- the update --------------------------------------------------------------------------------------
struct Entry {
    void *param;
    const void *grad;
    void *exp_avg, *exp_avg_sq;
    uint8_t *scales;
};

struct Table {
    Entry t[kTable];
    uint32_t numel[kTable];
    int32_t first[kTable + 1];
    int32_t order[kTable];              // whose factors
    uint8_t odd[kTable];                // whether the piece starts at an odd multiple of 2^31 elements
    int32_t count;
};

struct Betas {
    float b1, c1, b2, c2, eps;          // c = 1 - b, taken in double
    float eps_of_zero;                  // where the second moment is zero
    int32_t tiny_eps;                   // whether roots below 2^-63 count next to eps
};
static_assert(sizeof(Table) + sizeof(Betas) + 16 <= 4096, "kernel arguments");

// New moments and weight.  For fp32 weights the root and the quotient are rounded to nearest.  For 16-bit weights they are
// the hardware's, off by one unit in fp32's last place where the exact ones are off by half: the weight that the step
// goes into is rounded to 8 or 11 of its 24 bits.  (134 M bf16 weights with 8-bit moments 354 us, 399 with the exact ones; 62 M
// fp32 weights wait for memory: 305 with either, with 8-bit moments 269 with the exact ones and 268 with the hardware's.)
// The hardware's root takes numbers below the normal ones (2^-126) for zero, and squares of first gradients get there.  What
// it leaves out of the denominator is then at most 2^-63 times the bias correction.  With an eps of 2^24 times that or more
// (5.8e-11 for beta2 = 0.999) it is below fp32's last place; TINY, the form for a smaller eps, scales small ones by 2^32
// (357 us in the case above: six more of some sixty instructions for each element).
// The decay of an fp32 weight is added to the step and both are taken off with one rounding: a factor 1 - decay would be
// 2^-24 off, more than a decay of 1e-8 and a fifth of one of 1e-7, the same way in every step.  A weight that is an infinity
// stays one.  The rounding of a 16-bit weight is far above that.
// A second moment of zero, that of an element without a gradient or of squares that fp32 does not hold, has at least
// 2^-63 (the root of the smallest normal number) in place of eps: there the quotient is 0/0 or nearly so.
template <class T, bool TINY>
__device__ inline float step_of(float p, float &m, float &v, float g, const Betas &b, const Factors &f)
{
    g *= f.grad;
    m = fmaf(b.c1, g, b.b1 * m);
    v = fmaf(b.c2 * g, g, b.b2 * v);
    const float eps = !TINY || v > 0.f ? b.eps : b.eps_of_zero;
    if constexpr (sizeof(T) == 4) {
        const float u = m / fmaf(sqrtf(v), f.root, eps);
        return p - fmaf(f.rate, u, f.decay * __builtin_amdgcn_fmed3f(p, -FLT_MAX, FLT_MAX));
    } else {
        const bool small = TINY && v < 0x1p-96f;
        const float root = __builtin_amdgcn_sqrtf(small ? v * 0x1p32f : v);
        const float u = m * __builtin_amdgcn_rcpf(fmaf(root, small ? f.small_root : f.root, eps));
        return fmaf(-f.rate, u, p * f.keep);
    }
}

// f(a constant TINY)
template <bool V>
struct Bool {
    static constexpr bool value = V;
};

template <class T, class F>
__device__ inline void with_eps(const Betas &b, F f)
{
    if (sizeof(T) == 2 && !b.tiny_eps)
        f(Bool<false>());
    else
        f(Bool<true>());
}

// The tensor of chunk `chunk`: the lanes look at the table's entries at once, two each.
template <int TABLE>
__device__ inline int tensor_of(const int32_t *first, int count, int chunk)
{
    static_assert(TABLE <= 128, "two entries per lane");
    const int lane = threadIdx.x & 63;
    int k = __popcll(__ballot(lane < count && chunk >= first[lane + 1]));
    if (TABLE > 64) k += __popcll(__ballot(lane + 64 < count && chunk >= first[min(lane + 65, TABLE)]));
    return k;
}

// A whole chunk's loads go out together; with the ends checked they would wait for each other, which only a tensor's last
// chunk does.  Weights and moments are read and written past the caches: nothing of this step reads them again, and what
// the step before left to be written back does not come in between (62 M weights, 32-bit moments, clipped: 383 us through
// the caches, 303 us past them; only the loads or only the stores gain nothing).  Gradients are read past the caches if no
// norm was taken of them just before (134 M bf16 gradients: 367 and 353 us), out of the caches if one was, by this call or by
// the caller for several of them (62 M with 8-bit moments: 303 and 291 us; in two groups 221 and 206).
template <bool WHOLE, class T, int V, bool STREAM = true>
__device__ inline Words<T, V> load_some(const T *p, int n)
{
    if constexpr (WHOLE && STREAM) return stream_words<T, V>(p);
    if constexpr (WHOLE) return load_words<T, V>(p);
    return load_words<T, V>(p, n);
}

template <bool WHOLE, class T, int V, bool STREAM = true>
__device__ inline void store_some(T *p, const Words<T, V> &w, int n)
{
    if constexpr (WHOLE && STREAM)
        stream_words<T, V>(p, w);
    else if constexpr (WHOLE)
        store_words<T, V>(p, w);
    else
        store_words<T, V>(p, w, n);
}

template <bool WHOLE, bool STREAM_G, class T>
__device__ inline void update_chunk(const Entry &e, int64_t at, int left, const Betas &b, const Factors &f)
{
    constexpr int V = 4, U = kChunk / (kThreads * V);
    T *p = (T *)e.param + at;
    const T *g = (const T *)e.grad + at;
    float *em = (float *)e.exp_avg + at, *ev = (float *)e.exp_avg_sq + at;
    Words<T, V> wp[U], wg[U];
    Words<float, V> wm[U], wv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int o = u * kThreads * V, n = left - o;
        wg[u] = load_some<WHOLE, T, V, STREAM_G>(g + o, n);
        wm[u] = load_some<WHOLE, float, V>(em + o, n);
        wv[u] = load_some<WHOLE, float, V>(ev + o, n);
        wp[u] = load_some<WHOLE, T, V>(p + o, n);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int o = u * kThreads * V, n = left - o;
        float np[V], nm[V], nv[V];
        with_eps<T>(b, [&](auto tiny) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                nm[j] = wm[u][j];
                nv[j] = wv[u][j];
                np[j] = step_of<T, decltype(tiny)::value>(wp[u][j], nm[j], nv[j], wg[u][j], b, f);
            }
        });
        store_some<WHOLE, float, V>(em + o, to_words<float, V>(nm), n);
        store_some<WHOLE, float, V>(ev + o, to_words<float, V>(nv), n);
        store_some<WHOLE, T, V>(p + o, to_words<T, V>(np), n);
    }
}

template <class T, bool STREAM_G>
__global__ __launch_bounds__(kThreads) void adamw_kernel(Table t, Betas b, const Factors *__restrict__ factors)
{
    const int chunk = blockIdx.x, k = __builtin_amdgcn_readfirstlane(tensor_of<kTable>(t.first, t.count, chunk));
    const Factors f = factors[t.order[k]];
    if (f.skip) return;
    const int64_t from = (int64_t)(chunk - t.first[k]) * kChunk, left = (int64_t)t.numel[k] - from;
    const int mine = threadIdx.x * 4;
    if (left >= kChunk)
        update_chunk<true, STREAM_G, T>(t.t[k], from + mine, 0, b, f);
    else
        update_chunk<false, STREAM_G, T>(t.t[k], from + mine, (int)left - mine, b, f);
}

// the largest of 16 neighbouring lanes, in each of them
__device__ inline uint32_t largest16(uint32_t v)
{
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true));
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, true));
}

// 16 lanes share a block of 128 elements, eight each.  Elements behind the end are zero: they add nothing to the
// block's exponents and are not stored.
template <bool WHOLE, bool STREAM_G, class T>
__device__ inline void update_chunk8(const Entry &e, int64_t at, int n, uint32_t element, const Betas &b, const Factors &f)
{
    constexpr int V = 8;
    T *p = (T *)e.param + at;
    const T *g = (const T *)e.grad + at;
    uint8_t *cm = (uint8_t *)e.exp_avg + at, *cv = (uint8_t *)e.exp_avg_sq + at;
    uint8_t *scales = e.scales + at / kBlock * 2;
    const auto bm = load_some<WHOLE, uint8_t, V>(cm, n), bv = load_some<WHOLE, uint8_t, V>(cv, n);
    const uint32_t em = scales[0], ev = scales[1];
    const auto wg = load_some<WHOLE, T, V, STREAM_G>(g, n), wp = load_some<WHOLE, T, V>(p, n);
    float m[V], v[V], np[V];
    const float unit = first_unit(em);
    const int power = second_power(ev);
#pragma unroll
    for (int q = 0; q < V; q += 4) {
        decode_first(bm.w[q / 4], unit, m + q);
        decode_second(bv.w[q / 4], power, v + q);
    }
    uint32_t top_m = 0, top_v = 0;
    with_eps<T>(b, [&](auto tiny) {
#pragma unroll
        for (int j = 0; j < V; ++j) np[j] = step_of<T, decltype(tiny)::value>(wp[j], m[j], v[j], wg[j], b, f);
    });
#pragma unroll
    for (int j = 0; j < V; ++j) {
        top_m = max(top_m, magnitude_bits(m[j]));
        top_v = max(top_v, magnitude_bits(v[j]));
    }
    store_some<WHOLE, T, V>(p, to_words<T, V>(np), n);
    top_m = largest16(top_m);
    top_v = largest16(top_v);
    const bool wild = max(top_m, top_v) >= kInfinity;       // the same in the block's 16 lanes
    if (wild) {
        top_m = top_v = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            top_m = max(top_m, finite_bits(m[j]));
            top_v = max(top_v, finite_bits(v[j]));
        }
        top_m = largest16(top_m);
        top_v = largest16(top_v);
    }
    const int xm = max((int)(top_m >> 23), kFirstFloor), xv = max((int)(top_v >> 23), kSecondFloor);
    uint32_t h[V];
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = dither(element + j, f.key);
    Words<uint8_t, V> om, ov;
#pragma unroll
    for (int q = 0; q < V; q += 4) {
        om.w[q / 4] = encode_first(m + q, power_of_two(kFirstBias - xm), h + q);
        ov.w[q / 4] = encode_second(v + q, second_power(xv), h + q);
    }
    if (wild) {
#pragma unroll
        for (int q = 0; q < V; q += 4) {
            mark_not_finite(m + q, 0x7fu, &om.w[q / 4]);
            mark_not_finite(v + q, 0xffu, &ov.w[q / 4]);
        }
    }
    store_some<WHOLE, uint8_t, V>(cm, om, n);
    store_some<WHOLE, uint8_t, V>(cv, ov, n);
    if ((threadIdx.x & 15) == 0) {
        scales[0] = (uint8_t)xm;
        scales[1] = (uint8_t)xv;
    }
}

template <class T, bool STREAM_G>
__global__ __launch_bounds__(kThreads) void adamw8_kernel(Table t, Betas b, const Factors *__restrict__ factors)
{
    const int chunk = blockIdx.x, k = __builtin_amdgcn_readfirstlane(tensor_of<kTable>(t.first, t.count, chunk));
    const Factors f = factors[t.order[k]];
    if (f.skip) return;
    const int64_t from = (int64_t)(chunk - t.first[k]) * kChunk8, left = (int64_t)t.numel[k] - from;
    const int mine = threadIdx.x * 8;
    const uint32_t element = (uint32_t)from + mine + ((uint32_t)t.odd[k] << 31);
    if (left >= kChunk8) {
        update_chunk8<true, STREAM_G, T>(t.t[k], from + mine, 0, element, b, f);
    } else {
        // the 16 lanes of a block stay or go together: each of them passes on what others found
        if (mine / kBlock * kBlock >= left) return;
        update_chunk8<false, STREAM_G, T>(t.t[k], from + mine, (int)left - mine, element, b, f);
    }
}

// ---- small calls: everything in one workgroup, one launch ----------------------------------------------
// The norm, the factors and the update of at most kSmallChunks chunks: four teams of 256 threads take a chunk each.
constexpr int kSmallThreads = 1024, kSmallTable = 64;
constexpr int kSmallChunks = 8;
static_assert(kChunk == kChunk8, "one count of chunks for both");

struct SmallTable {
    Entry t[kSmallTable];
    float *step[kSmallTable];
    uint32_t numel[kSmallTable];
    int32_t first[kSmallTable + 1];
    int32_t count;
};
static_assert(sizeof(SmallTable) + sizeof(Scalars) + sizeof(Betas) + 32 <= 4096, "kernel arguments");

template <class T, int BITS>
__global__ __launch_bounds__(kSmallThreads) void adamw_small_kernel(SmallTable t, Scalars p, Betas b)
{
    __shared__ double part[kSmallThreads / 64];
    __shared__ double grad;
    __shared__ Factors factors[kSmallTable];
    const int chunks = t.first[t.count];
    const int team = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kThreads), mine = threadIdx.x % kThreads;
    double acc = 0.0;
    if (p.max_norm > 0.0)
        for (int chunk = team; chunk < chunks; chunk += kSmallThreads / kThreads) {
            const int k = __builtin_amdgcn_readfirstlane(tensor_of<kSmallTable>(t.first, t.count, chunk));
            const int at = (chunk - t.first[k]) * kChunk + mine * 8;
            const auto w = load_words<T, 8>((const T *)t.t[k].grad + at, (int)t.numel[k] - at);
#pragma unroll
            for (int j = 0; j < 8; ++j) acc += (double)w[j] * (double)w[j];
        }
    if ((int)threadIdx.x < t.count) factors[threadIdx.x] = factors_of(p, t.step[threadIdx.x]);
    acc = group_sum(acc, part, kSmallThreads / 64);
    if (threadIdx.x == 0) grad = grad_factor(p, acc);
    __syncthreads();
    for (int chunk = team; chunk < chunks; chunk += kSmallThreads / kThreads) {
        const int k = __builtin_amdgcn_readfirstlane(tensor_of<kSmallTable>(t.first, t.count, chunk));
        Factors f = factors[k];
        if (f.skip) return;
        f.grad = (float)grad;
        const int at = (chunk - t.first[k]) * kChunk, left = (int)t.numel[k] - at;
        if constexpr (BITS == 32) {
            if (left >= kChunk)
                update_chunk<true, false, T>(t.t[k], at + mine * 4, 0, b, f);
            else
                update_chunk<false, false, T>(t.t[k], at + mine * 4, left - mine * 4, b, f);
        } else {
            if (left >= kChunk8)
                update_chunk8<true, false, T>(t.t[k], at + mine * 8, 0, at + mine * 8, b, f);
            else if (mine * 8 / kBlock * kBlock < left)
                update_chunk8<false, false, T>(t.t[k], at + mine * 8, left - mine * 8, at + mine * 8, b, f);
        }
    }
}

template <bool WHOLE>
__device__ inline void values_of(const uint8_t *cm, const uint8_t *cv, const uint8_t *scales, int n, bf16 *m, bf16 *v)
{
    constexpr int V = 8;
    const auto bm = load_some<WHOLE, uint8_t, V, false>(cm, n), bv = load_some<WHOLE, uint8_t, V, false>(cv, n);
    const float unit = first_unit(scales[0]);
    const int power = second_power(scales[1]);
    float om[V], ov[V];
#pragma unroll
    for (int q = 0; q < V; q += 4) {
        decode_first(bm.w[q / 4], unit, om + q);
        decode_second(bv.w[q / 4], power, ov + q);
    }
    store_some<WHOLE, bf16, V>(m, to_words<bf16, V>(om), n);
    store_some<WHOLE, bf16, V>(v, to_words<bf16, V>(ov), n);
}

// eight elements per thread, so that a thread's all belong to one block
__global__ __launch_bounds__(kThreads) void moment_values_kernel(const uint8_t *__restrict__ cm, const uint8_t *__restrict__ cv,
                                                                 const uint8_t *__restrict__ scales, int64_t numel,
                                                                 bf16 *__restrict__ m, bf16 *__restrict__ v)
{
    constexpr int V = 8;
    const int64_t step = (int64_t)gridDim.x * kThreads * V;
    for (int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * V; i < numel; i += step) {
        const uint8_t *e = scales + i / kBlock * 2;
        if (numel - i >= V)
            values_of<true>(cm + i, cv + i, e, V, m + i, v + i);
        else
            values_of<false>(cm + i, cv + i, e, (int)(numel - i), m + i, v + i);
    }
}

// ---- host ----------------------------------------------------------------------------------------------
int check(const sv3d_adamw_tensor *tensors, int32_t n, bool grads_only)
{
    if (n < 0 || (n > 0 && !tensors)) return SV3D_ERR_INVALID_ARG;
    for (int32_t i = 0; i < n; ++i) {
        const sv3d_adamw_tensor &t = tensors[i];
        if (t.numel < 0 || !known_type(t.type)) return SV3D_ERR_INVALID_ARG;
        if (t.numel > 0 && (!t.grad || !aligned(t.grad, type_bytes(t.type)))) return SV3D_ERR_INVALID_ARG;
        if (t.numel > ((int64_t)1 << 40)) return SV3D_ERR_UNSUPPORTED;
        if (grads_only) continue;
        if ((t.state_bits != 8 && t.state_bits != 32) || !t.step || !aligned(t.step, 4)) return SV3D_ERR_INVALID_ARG;
        if (t.numel == 0) continue;
        if (!t.param || !t.exp_avg || !t.exp_avg_sq || !aligned(t.param, type_bytes(t.type))) return SV3D_ERR_INVALID_ARG;
        if (t.state_bits == 8 ? !t.scales : !aligned(t.exp_avg, 4) || !aligned(t.exp_avg_sq, 4)) return SV3D_ERR_INVALID_ARG;
    }
    return SV3D_OK;
}

// Collects tensors into launches of at most TABLE pieces and kMaxChunks chunks (a launch holds fewer than 2^32
// threads) and calls launch(pieces, first chunk of each, number of pieces).  A tensor of more than kPiece elements is
// several pieces.
constexpr int64_t kMaxChunks = 1 << 23;
static_assert(kPiece / kChunk <= kMaxChunks && kPiece % kChunk == 0 && kPiece % kChunk8 == 0 && kPiece % kSumChunk == 0, "a piece fits a launch");

struct Piece {
    int32_t index;
    int64_t from, numel;
};

template <int TABLE, class Take, class Launch>
int in_launches(const sv3d_adamw_tensor *tensors, int32_t n, int64_t chunk, Take take, Launch launch)
{
    Piece piece[TABLE];
    int32_t first[TABLE + 1] = {0};
    int count = 0;
    for (int32_t i = 0; i < n; ++i) {
        if (!take(tensors[i])) continue;
        for (int64_t from = 0; from < tensors[i].numel; from += kPiece) {
            const int64_t left = tensors[i].numel - from, now = left < kPiece ? left : kPiece;
            const int64_t chunks = (now + chunk - 1) / chunk;
            if (count == TABLE || first[count] + chunks > kMaxChunks) {
                if (const int st = launch(piece, first, count)) return st;
                count = 0;
            }
            piece[count] = {i, from, now};
            first[count + 1] = first[count] + (int32_t)chunks;
            ++count;
        }
    }
    return count ? launch(piece, first, count) : (int)SV3D_OK;
}

template <class F>
int for_each_type(F f)
{
    if (const int st = f((float *)nullptr, (int32_t)SV3D_F32)) return st;
    if (const int st = f((f16 *)nullptr, (int32_t)SV3D_F16)) return st;
    return f((bf16 *)nullptr, (int32_t)SV3D_BF16);
}

int sum_groups(int32_t chunks) { return chunks < kSumGroups ? chunks : kSumGroups; }

}  // namespace

extern "C" int sv3d_grad_square_sums_count(const sv3d_adamw_tensor *tensors, int32_t num_tensors, int32_t *count)
{
    if (!count) return SV3D_ERR_INVALID_ARG;
    if (const int st = check(tensors, num_tensors, true)) return st;
    int32_t total = 0;
    for_each_type([&](auto *, int32_t type) {
        return in_launches<kSumTable>(tensors, num_tensors, kSumChunk, [&](const sv3d_adamw_tensor &t) { return t.type == type; },
                           [&](const Piece *, const int32_t *first, int n) {
                               total += sum_groups(first[n]);
                               return (int)SV3D_OK;
                           });
    });
    *count = total;
    return SV3D_OK;
}

extern "C" int sv3d_grad_square_sums(const sv3d_adamw_tensor *tensors, int32_t num_tensors, double *sums, int32_t count,
                                     void *stream)
{
    int32_t need = 0, at = 0;
    if (const int st = sv3d_grad_square_sums_count(tensors, num_tensors, &need)) return st;
    if (count != need || (need > 0 && (!sums || !aligned(sums, 8)))) return SV3D_ERR_INVALID_ARG;
    return for_each_type([&](auto *T, int32_t type) {
        using E = std::remove_pointer_t<decltype(T)>;
        return in_launches<kSumTable>(tensors, num_tensors, kSumChunk, [&](const sv3d_adamw_tensor &t) { return t.type == type; },
                           [&](const Piece *piece, const int32_t *first, int n) {
                               SumTable t;
                               t.count = n;
                               for (int k = 0; k < n; ++k) {
                                   t.grad[k] = (const E *)tensors[piece[k].index].grad + piece[k].from;
                                   t.numel[k] = (uint32_t)piece[k].numel;
                               }
                               for (int k = 0; k <= n; ++k) t.first[k] = first[k];
                               const int groups = sum_groups(first[n]);
                               hipLaunchKernelGGL(grad_square_sums_kernel<E>, dim3(groups), dim3(kThreads), 0,
                                                  (hipStream_t)stream, t, sums + at);
                               at += groups;
                               return launch_status();
                           });
    });
}

extern "C" int sv3d_adamw_workspace(const sv3d_adamw_params *p, const sv3d_adamw_tensor *tensors, int32_t num_tensors,
                                    size_t *bytes)
{
    if (!p || num_tensors < 0 || !bytes) return SV3D_ERR_INVALID_ARG;
    int32_t sums = 0;
    if (p->max_norm > 0.0 && !p->square_sums)
        if (const int st = sv3d_grad_square_sums_count(tensors, num_tensors, &sums)) return st;
    *bytes = (size_t)num_tensors * sizeof(Factors) + (size_t)sums * sizeof(double);
    return SV3D_OK;
}

namespace {

// Whether the call is the small kernel's: one type and kind of moments, few elements, and no norm from elsewhere.  Where that
// kernel has work for its four teams once or twice, it takes the time of one launch in place of three (5136 elements,
// clipped, 15.3 -> 7.8 us with the call's host time; at 16 chunks 15.4 and 13.4 us, not clipped 11.3 and 11.6).
bool small_call(const sv3d_adamw_params *p, const sv3d_adamw_tensor *tensors, int32_t n)
{
    if (n > kSmallTable || p->square_sums) return false;
    int64_t chunks = 0;
    for (int32_t i = 0; i < n; ++i) {
        if (tensors[i].type != tensors[0].type || tensors[i].state_bits != tensors[0].state_bits) return false;
        if (tensors[i].numel > kSmallChunks * kChunk) return false;
        chunks += (tensors[i].numel + kChunk - 1) / kChunk;
    }
    return chunks <= kSmallChunks;
}

int small_step(const Scalars &scalars, const Betas &b, const sv3d_adamw_tensor *tensors, int32_t n, hipStream_t stream)
{
    SmallTable t;
    t.count = n;
    t.first[0] = 0;
    for (int i = 0; i < n; ++i) {
        const sv3d_adamw_tensor &s = tensors[i];
        t.t[i] = {s.param, s.grad, s.exp_avg, s.exp_avg_sq, s.scales};
        t.step[i] = s.step;
        t.numel[i] = (uint32_t)s.numel;
        t.first[i + 1] = t.first[i] + (int32_t)((s.numel + kChunk - 1) / kChunk);
    }
    return for_each_type([&](auto *T, int32_t type) {
        using E = std::remove_pointer_t<decltype(T)>;
        if (type != tensors[0].type) return (int)SV3D_OK;
        const auto kernel = tensors[0].state_bits == 32 ? adamw_small_kernel<E, 32> : adamw_small_kernel<E, 8>;
        hipLaunchKernelGGL(kernel, dim3(1), dim3(kSmallThreads), 0, stream, t, scalars, b);
        return launch_status();
    });
}

}  // namespace

extern "C" int sv3d_adamw_step(const sv3d_adamw_params *p, const sv3d_adamw_tensor *tensors, int32_t num_tensors,
                               void *workspace, size_t workspace_bytes, void *stream)
{
    if (!p) return SV3D_ERR_INVALID_ARG;
    if (const int st = check(tensors, num_tensors, false)) return st;
    if (!(p->beta1 >= 0.0 && p->beta1 < 1.0 && p->beta2 >= 0.0 && p->beta2 < 1.0 && p->eps >= 0.0)) return SV3D_ERR_INVALID_ARG;
    if (!(p->max_norm >= 0.0) || p->num_square_sums < 0) return SV3D_ERR_INVALID_ARG;
    if (!aligned(p->lr_device, 4) || !aligned(p->grad_scale, 4) || !aligned(p->found_inf, 4) || !aligned(p->total_norm, 4) ||
        !aligned(p->square_sums, 8))
        return SV3D_ERR_INVALID_ARG;
    if (num_tensors == 0) return SV3D_OK;
    size_t need = 0;
    if (const int st = sv3d_adamw_workspace(p, tensors, num_tensors, &need)) return st;
    if (!workspace || !aligned(workspace, 16)) return SV3D_ERR_INVALID_ARG;
    if (workspace_bytes < need) return SV3D_ERR_WORKSPACE;
    const Scalars scalars = {p->lr,         log(p->beta1), log(p->beta2), p->weight_decay, p->max_norm, p->lr_device,
                             p->grad_scale, p->found_inf,  p->total_norm, p->seed,         p->maximize};
    const Betas b = {(float)p->beta1, (float)(1.0 - p->beta1), (float)p->beta2, (float)(1.0 - p->beta2),
                     (float)p->eps, (float)(p->eps > 0x1p-63 ? p->eps : 0x1p-63), p->eps < 0x1p-39 / sqrt(1.0 - p->beta2)};
    if (small_call(p, tensors, num_tensors)) return small_step(scalars, b, tensors, num_tensors, (hipStream_t)stream);
    Factors *factors = (Factors *)workspace;
    const bool clip = p->max_norm > 0.0;
    const double *sums = p->square_sums;
    int32_t num_sums = clip ? p->num_square_sums : 0;
    if (clip && !p->square_sums) {
        num_sums = (int32_t)((need - num_tensors * sizeof(Factors)) / sizeof(double));
        double *own = (double *)(factors + num_tensors);
        if (const int st = sv3d_grad_square_sums(tensors, num_tensors, own, num_sums, stream)) return st;
        sums = own;
    }
    for (int32_t base = 0; base < num_tensors; base += kSteps) {
        StepTable s;
        s.base = base;
        s.count = num_tensors - base < kSteps ? num_tensors - base : kSteps;
        for (int i = 0; i < s.count; ++i) s.step[i] = tensors[base + i].step;
        hipLaunchKernelGGL(adamw_factors_kernel, dim3(1), dim3(kThreads), 0, (hipStream_t)stream, s, scalars, sums, num_sums, factors);
        if (const int st = launch_status()) return st;
    }
    return for_each_type([&](auto *T, int32_t type) {
        using E = std::remove_pointer_t<decltype(T)>;
        for (int32_t bits : {32, 8}) {
            const int64_t state = bits == 32 ? 4 : 1;
            const int st = in_launches<kTable>(
                tensors, num_tensors, bits == 32 ? kChunk : kChunk8,
                [&](const sv3d_adamw_tensor &t) { return t.type == type && t.state_bits == bits; },
                [&](const Piece *piece, const int32_t *first, int n) {
                    Table t;
                    t.count = n;
                    for (int k = 0; k < n; ++k) {
                        const sv3d_adamw_tensor &s = tensors[piece[k].index];
                        const int64_t from = piece[k].from;
                        t.t[k] = {(E *)s.param + from, (const E *)s.grad + from, (char *)s.exp_avg + from * state,
                                  (char *)s.exp_avg_sq + from * state, s.scales ? s.scales + from / kBlock * 2 : nullptr};
                        t.numel[k] = (uint32_t)piece[k].numel;
                        t.order[k] = piece[k].index;
                        t.odd[k] = (uint8_t)(from >> 31 & 1);
                    }
                    for (int k = 0; k <= n; ++k) t.first[k] = first[k];
                    const auto kernel = bits == 32 ? (clip ? adamw_kernel<E, false> : adamw_kernel<E, true>)
                                                   : (clip ? adamw8_kernel<E, false> : adamw8_kernel<E, true>);
                    hipLaunchKernelGGL(kernel, dim3(first[n]), dim3(kThreads), 0, (hipStream_t)stream, t, b, factors);
                    return launch_status();
                });
            if (st) return st;
        }
        return (int)SV3D_OK;
    });
}

extern "C" int sv3d_moment_values(const uint8_t *exp_avg, const uint8_t *exp_avg_sq, const uint8_t *scales, int64_t numel,
                                  void *exp_avg_out, void *exp_avg_sq_out, void *stream)
{
    if (numel < 0) return SV3D_ERR_INVALID_ARG;
    if (numel == 0) return SV3D_OK;
    if (!exp_avg || !exp_avg_sq || !scales || !exp_avg_out || !exp_avg_sq_out || !aligned(exp_avg_out, 2) || !aligned(exp_avg_sq_out, 2))
        return SV3D_ERR_INVALID_ARG;
    const int64_t groups = (numel + kThreads * 8 - 1) / (kThreads * 8);
    hipLaunchKernelGGL(moment_values_kernel, dim3((uint32_t)(groups < (1 << 20) ? groups : (1 << 20))), dim3(kThreads), 0,
                       (hipStream_t)stream, exp_avg, exp_avg_sq, scales, numel, (bf16 *)exp_avg_out, (bf16 *)exp_avg_sq_out);
    return launch_status();
}
