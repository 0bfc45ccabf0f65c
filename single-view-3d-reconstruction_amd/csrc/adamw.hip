// The optimizer step over many tensors at once: the gradients' common norm, unscaling, clipping and AdamW with
// 32-bit or 8-bit moments (formulas and code formats in sv3d_hip.h).
//
// Tensors reach a kernel as a table in its arguments (captured with the launch, nothing on the device has to
// be kept up to date), at most kTable of them per launch, cut into chunks; a workgroup looks up its chunk's tensor.
#include "element.h"

#include <type_traits>

namespace {

using namespace sv3d;

constexpr int kThreads = 256;
constexpr int kTable = 64;          // tensors of one launch: the table has to fit 4 KB of kernel arguments
constexpr int kChunk = 2048;        // elements of one workgroup of the update
constexpr int kBlock = SV3D_STATE_BLOCK;
constexpr int kSumChunk = 4096;
constexpr int kSumGroups = 1024;
constexpr float kSmallest = 0x1p-126f;

// ---- the norm: sums of squares --------------------------------------------------------------------
// Squares and sums in double: a square of an fp32 number neither overflows nor is rounded there, and the order of
// the sum stops to matter for the fp32 norm that is made of it.
struct SumTable {
    const void *grad[kTable];
    int64_t numel[kTable];
    int32_t first[kTable + 1];      // of each tensor's chunks
    int32_t count;
};

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
        const int left = (int)min(t.numel[k] - at, (int64_t)kSumChunk);
        constexpr int V = 16 / (int)sizeof(T);
#pragma unroll
        for (int u = 0; u < kSumChunk / (kThreads * V); ++u) {
            const int o = (u * kThreads + threadIdx.x) * V;
            const auto w = load_words<T, V>(g + at + o, left - o);
#pragma unroll
            for (int j = 0; j < V; ++j) acc[j & 3] += (double)w[j] * (double)w[j];
        }
    }
    double sum = (acc[0] + acc[1]) + (acc[2] + acc[3]);
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x / 64] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kThreads / 64; ++w) sum += part[w];
        sums[blockIdx.x] = sum;
    }
}

// ---- what each tensor's update multiplies by -------------------------------------------------------
struct Factors {
    float grad;         // unscaling, clipping and sign
    float decay;        // 1 - lr weight_decay
    float rate;         // lr / (1 - beta1^t)
    float root;         // 1 / sqrt(1 - beta2^t)
    uint32_t key;       // of the dither
    int32_t skip;
    int32_t pad[2];
};

constexpr int kSteps = 384;
struct StepTable {
    float *step[kSteps];
    int32_t base, count;
};

// One workgroup.  Takes the step counts forward, in double: beta^t close to 1 is subtracted from 1.
__global__ __launch_bounds__(kThreads) void adamw_factors_kernel(StepTable t, sv3d_adamw_params p, Factors *__restrict__ out)
{
    __shared__ double part[kThreads / 64];
    __shared__ double scale;
    const double inv = p.grad_scale ? 1.0 / (double)*p.grad_scale : 1.0;
    if (p.square_sums) {
        double acc = 0.0;
        for (int i = threadIdx.x; i < p.num_square_sums; i += kThreads) acc += p.square_sums[i];
        for (int d = 32; d > 0; d >>= 1) acc += __shfl_xor(acc, d);
        if ((threadIdx.x & 63) == 0) part[threadIdx.x / 64] = acc;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < kThreads / 64; ++w) acc += part[w];
            const double norm = sqrt(acc) * inv;
            if (p.total_norm) *p.total_norm = (float)norm;
            const double c = p.max_norm / (norm + 1e-6);
            scale = inv * (c > 1.0 ? 1.0 : c);      // a norm that is no number goes through, into every weight
        }
        __syncthreads();
    } else {
        if (threadIdx.x == 0) scale = inv;
        __syncthreads();
    }
    const int32_t skip = p.found_inf && *p.found_inf != 0.f;
    const double lr = p.lr_device ? (double)*p.lr_device : p.lr;
    for (int i = threadIdx.x; i < t.count; i += kThreads) {
        const float n = *t.step[i] + 1.f;
        if (!skip) *t.step[i] = n;
        Factors f;
        f.grad = (float)(p.maximize ? -scale : scale);
        f.decay = (float)(1.0 - lr * p.weight_decay);
        f.rate = (float)(lr / (1.0 - pow(p.beta1, (double)n)));
        f.root = (float)(1.0 / sqrt(1.0 - pow(p.beta2, (double)n)));
        f.key = (uint32_t)n * 0x9E3779B1u + p.seed * 0x6A09E667u;
        f.skip = skip;
        f.pad[0] = f.pad[1] = 0;
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

__device__ inline float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// A code is the upper bits of a float32 whose exponent field is as narrow as the code's: with a block's values scaled so
// that the code's smallest exponent meets float32's, bits 20 and up of a value ARE its code, its subnormal codes included
// (float32's own subnormal numbers), and the dither (16 bits and half a one) goes in below before they are cut off.
//   first:  field = exponent + 7,  sign in bit 31;     second: field = exponent + 15
constexpr int kFirstBias = 134, kSecondBias = 142;      // a block's largest value lands in [2^7, 2^8) and [2^15, 2^16)
constexpr int kFirstFloor = 20, kSecondFloor = 34;      // so that every value is a normal number, also as bf16
constexpr int kFirstField = 127 - 7, kSecondField = 127 - 15;

// what to multiply by two to the power of, from a value to its code's place; a byte below the lowest that is ever
// written (fresh state: 0) counts as that one
__device__ inline int first_power(uint32_t e) { return kFirstBias - kFirstField - max((int)e, kFirstFloor); }
__device__ inline int second_power(uint32_t e) { return kSecondBias - kSecondField - max((int)e, kSecondFloor); }

__device__ inline uint32_t block_exponent(uint32_t largest_bits, int floor) { return (uint32_t)max((int)(largest_bits >> 23), floor); }

constexpr uint32_t kInfinity = 0x7f800000u;
__device__ inline uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// what a moment contributes to its block's exponent: an infinity or NaN does not
__device__ inline uint32_t finite_bits(float v) { return magnitude_bits(v) < kInfinity ? magnitude_bits(v) : 0u; }

// `low`: the dither bits in place, (bits << 4) + 8
__device__ inline uint32_t encode_first(float m, int power, uint32_t low)
{
    const uint32_t q = (__float_as_uint(ldexpf(m, power)) + low) >> 20;
    return (magnitude_bits(m) < kInfinity ? q & 0x7fu : 0x7fu) | (q >> 4 & 0x80u);
}

__device__ inline uint32_t encode_second(float v, int power, uint32_t low)
{
    const uint32_t q = (__float_as_uint(ldexpf(v, power)) + low) >> 20;
    return !(v < INFINITY) ? 0xffu : v > 0.f ? max(q, 1u) : q;
}

__device__ inline float decode_first(uint32_t code, int power)
{
    const float v = ldexpf(__uint_as_float((code & 0x7fu) << 20 | (code & 0x80u) << 24), -power);
    return (code & 0x7fu) == 0x7fu ? NAN : v;
}

__device__ inline float decode_second(uint32_t code, int power) { return code == 0xffu ? NAN : ldexpf(__uint_as_float(code << 20), -power); }

// ---- the update --------------------------------------------------------------------------------------
struct Entry {
    void *param;
    const void *grad;
    void *exp_avg, *exp_avg_sq;
    uint8_t *scales;
    int64_t numel;
};

struct Table {
    Entry t[kTable];
    int32_t first[kTable + 1];
    int32_t order[kTable];              // whose factors
    int32_t count;
};

struct Betas {
    float b1, c1, b2, c2, eps;          // c = 1 - b, taken in double
};

// Products and sums of the moments as they stand, each rounded: the same bits on every path.  The root and the
// quotient are the hardware's (off by one unit in the last place where the exact ones are off by half); it takes numbers
// below the normal ones for zero, hence the lower end.
__device__ inline float step_of(float &m, float &v, float g, const Betas &b, const Factors &f)
{
    m = __fadd_rn(__fmul_rn(b.b1, m), __fmul_rn(b.c1, g));
    v = __fadd_rn(__fmul_rn(b.b2, v), __fmul_rn(b.c2, __fmul_rn(g, g)));
    const float root = __builtin_amdgcn_sqrtf(v < kSmallest ? kSmallest : v);       // NaN stays
    return f.rate * (m * __builtin_amdgcn_rcpf(root * f.root + b.eps));
}

// The tensor of chunk `chunk`: the lanes look at the 64 table entries at once.
__device__ inline int tensor_of(const int32_t *first, int count, int chunk)
{
    const int lane = threadIdx.x & 63;
    return __popcll(__ballot(lane < count && chunk >= first[lane + 1]));
}

template <class T>
__global__ __launch_bounds__(kThreads) void adamw_kernel(Table t, Betas b, const Factors *__restrict__ factors)
{
    const int k = __builtin_amdgcn_readfirstlane(tensor_of(t.first, t.count, blockIdx.x));
    const Entry e = t.t[k];
    const Factors f = factors[t.order[k]];
    if (f.skip) return;
    constexpr int V = 4, U = kChunk / (kThreads * V);
    const int64_t at = (int64_t)((int)blockIdx.x - t.first[k]) * kChunk + threadIdx.x * V;
    T *p = (T *)e.param + at;
    const T *g = (const T *)e.grad + at;
    float *em = (float *)e.exp_avg + at, *ev = (float *)e.exp_avg_sq + at;
    const int left = (int)min(e.numel - at, (int64_t)kChunk);
    Words<T, V> wp[U], wg[U];
    Words<float, V> wm[U], wv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int o = u * kThreads * V, n = left - o;
        wg[u] = load_words<T, V>(g + o, n);
        wm[u] = load_words<float, V>(em + o, n);
        wv[u] = load_words<float, V>(ev + o, n);
        wp[u] = load_words<T, V>(p + o, n);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int o = u * kThreads * V, n = left - o;
        float np[V], nm[V], nv[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            nm[j] = wm[u][j];
            nv[j] = wv[u][j];
            const float s = step_of(nm[j], nv[j], wg[u][j] * f.grad, b, f);
            np[j] = wp[u][j] * f.decay - s;
        }
        store_pack<float, V>(em + o, nm, n);
        store_pack<float, V>(ev + o, nv, n);
        store_pack<T, V>(p + o, np, n);
    }
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
template <class T>
__global__ __launch_bounds__(kThreads) void adamw8_kernel(Table t, Betas b, const Factors *__restrict__ factors)
{
    const int k = __builtin_amdgcn_readfirstlane(tensor_of(t.first, t.count, blockIdx.x));
    const Entry e = t.t[k];
    const Factors f = factors[t.order[k]];
    if (f.skip) return;
    constexpr int V = 8;
    const int64_t at = (int64_t)((int)blockIdx.x - t.first[k]) * kChunk + threadIdx.x * V;
    // the 16 lanes of a block stay or go together: each of them passes on what others found
    if (at - (int)(threadIdx.x & 15) * V >= e.numel) return;
    const int n = (int)max(min(e.numel - at, (int64_t)V), (int64_t)0);
    T *p = (T *)e.param + at;
    const T *g = (const T *)e.grad + at;
    uint8_t *cm = (uint8_t *)e.exp_avg + at, *cv = (uint8_t *)e.exp_avg_sq + at;
    uint8_t *scales = e.scales + at / kBlock * 2;
    const auto wg = load_words<T, V>(g, n);
    const auto bm = load_words<uint8_t, V>(cm, n), bv = load_words<uint8_t, V>(cv, n);
    const auto wp = load_words<T, V>(p, n);
    const int pm = first_power(scales[0]), pv = second_power(scales[1]);
    float m[V], v[V], np[V];
    uint32_t top_m = 0, top_v = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        m[j] = decode_first(bm.byte(j), pm);
        v[j] = decode_second(bv.byte(j), pv);
        const float s = step_of(m[j], v[j], wg[j] * f.grad, b, f);
        np[j] = wp[j] * f.decay - s;
        top_m = max(top_m, finite_bits(m[j]));
        top_v = max(top_v, finite_bits(v[j]));
    }
    store_pack<T, V>(p, np, n);
    const uint32_t xm = block_exponent(largest16(top_m), kFirstFloor), xv = block_exponent(largest16(top_v), kSecondFloor);
    const int qm = first_power(xm), qv = second_power(xv);
    Words<uint8_t, V> om = {}, ov = {};
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const uint32_t h = dither((uint32_t)at + j, f.key);
        om.w[j / 4] |= encode_first(m[j], qm, (h >> 12 & 0xffff0u) + 8u) << (j % 4 * 8);
        ov.w[j / 4] |= encode_second(v[j], qv, (h << 4 & 0xffff0u) + 8u) << (j % 4 * 8);
    }
    store_words<uint8_t, V>(cm, om, n);
    store_words<uint8_t, V>(cv, ov, n);
    if ((threadIdx.x & 15) == 0) {
        scales[0] = (uint8_t)xm;
        scales[1] = (uint8_t)xv;
    }
}

// eight elements per thread, so that a thread's all belong to one block
__global__ __launch_bounds__(kThreads) void moment_values_kernel(const uint8_t *__restrict__ cm, const uint8_t *__restrict__ cv,
                                                                 const uint8_t *__restrict__ scales, int64_t numel,
                                                                 bf16 *__restrict__ m, bf16 *__restrict__ v)
{
    constexpr int V = 8;
    const int64_t step = (int64_t)gridDim.x * kThreads * V;
    for (int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * V; i < numel; i += step) {
        const int n = (int)min(numel - i, (int64_t)V);
        const auto bm = load_words<uint8_t, V>(cm + i, n), bv = load_words<uint8_t, V>(cv + i, n);
        const int64_t block = i / kBlock;
        const int pm = first_power(scales[2 * block]), pv = second_power(scales[2 * block + 1]);
        float om[V], ov[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            om[j] = decode_first(bm.byte(j), pm);
            ov[j] = decode_second(bv.byte(j), pv);
        }
        store_pack<bf16, V>(m + i, om, n);
        store_pack<bf16, V>(v + i, ov, n);
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
        if ((t.state_bits != 8 && t.state_bits != 32) || !t.step) return SV3D_ERR_INVALID_ARG;
        if (t.numel == 0) continue;
        if (!t.param || !t.exp_avg || !t.exp_avg_sq || !aligned(t.param, type_bytes(t.type))) return SV3D_ERR_INVALID_ARG;
        if (t.state_bits == 8 ? !t.scales : !aligned(t.exp_avg, 4) || !aligned(t.exp_avg_sq, 4)) return SV3D_ERR_INVALID_ARG;
    }
    return SV3D_OK;
}

// Collects tensors into launches of at most kTable of them and kMaxChunks chunks (a launch holds fewer than 2^32
// threads) and calls launch(pieces, first chunk of each, number of pieces).  Only a tensor that is larger than a
// launch is cut, at multiples of kMaxChunks chunks.
constexpr int64_t kMaxChunks = 1 << 23;
static_assert(kMaxChunks * kChunk % ((int64_t)1 << 32) == 0, "the dither takes an element's index modulo 2^32");

struct Piece {
    int32_t index;
    int64_t from, numel;
};

template <class Take, class Launch>
int in_launches(const sv3d_adamw_tensor *tensors, int32_t n, int64_t chunk, Take take, Launch launch)
{
    Piece piece[kTable];
    int32_t first[kTable + 1] = {0};
    int count = 0;
    for (int32_t i = 0; i < n; ++i) {
        if (!take(tensors[i])) continue;
        for (int64_t from = 0; from < tensors[i].numel; from += kMaxChunks * chunk) {
            const int64_t left = tensors[i].numel - from, most = kMaxChunks * chunk;
            const int64_t now = left < most ? left : most, chunks = (now + chunk - 1) / chunk;
            if (count == kTable || first[count] + chunks > kMaxChunks) {
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
        return in_launches(tensors, num_tensors, kSumChunk, [&](const sv3d_adamw_tensor &t) { return t.type == type; },
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
        return in_launches(tensors, num_tensors, kSumChunk, [&](const sv3d_adamw_tensor &t) { return t.type == type; },
                           [&](const Piece *piece, const int32_t *first, int n) {
                               SumTable t;
                               t.count = n;
                               for (int k = 0; k < n; ++k) {
                                   t.grad[k] = (const E *)tensors[piece[k].index].grad + piece[k].from;
                                   t.numel[k] = piece[k].numel;
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

extern "C" int sv3d_adamw_workspace(int32_t num_tensors, size_t *bytes)
{
    if (num_tensors < 0 || !bytes) return SV3D_ERR_INVALID_ARG;
    *bytes = (size_t)num_tensors * sizeof(Factors);
    return SV3D_OK;
}

extern "C" int sv3d_adamw_step(const sv3d_adamw_params *p, const sv3d_adamw_tensor *tensors, int32_t num_tensors,
                               void *workspace, size_t workspace_bytes, void *stream)
{
    if (!p) return SV3D_ERR_INVALID_ARG;
    if (const int st = check(tensors, num_tensors, false)) return st;
    if (!(p->beta1 >= 0.0 && p->beta1 < 1.0 && p->beta2 >= 0.0 && p->beta2 < 1.0 && p->eps >= 0.0)) return SV3D_ERR_INVALID_ARG;
    if (p->square_sums && (p->num_square_sums < 0 || !(p->max_norm >= 0.0))) return SV3D_ERR_INVALID_ARG;
    if (num_tensors == 0) return SV3D_OK;
    if (!workspace || !aligned(workspace, 16)) return SV3D_ERR_INVALID_ARG;
    if (workspace_bytes < (size_t)num_tensors * sizeof(Factors)) return SV3D_ERR_WORKSPACE;
    Factors *factors = (Factors *)workspace;
    for (int32_t base = 0; base < num_tensors; base += kSteps) {
        StepTable s;
        s.base = base;
        s.count = num_tensors - base < kSteps ? num_tensors - base : kSteps;
        for (int i = 0; i < s.count; ++i) s.step[i] = tensors[base + i].step;
        hipLaunchKernelGGL(adamw_factors_kernel, dim3(1), dim3(kThreads), 0, (hipStream_t)stream, s, *p, factors);
        if (const int st = launch_status()) return st;
    }
    const Betas b = {(float)p->beta1, (float)(1.0 - p->beta1), (float)p->beta2, (float)(1.0 - p->beta2), (float)p->eps};
    return for_each_type([&](auto *T, int32_t type) {
        using E = std::remove_pointer_t<decltype(T)>;
        for (int32_t bits : {32, 8}) {
            const int64_t state = bits == 32 ? 4 : 1;
            const int st = in_launches(
                tensors, num_tensors, kChunk,
                [&](const sv3d_adamw_tensor &t) { return t.type == type && t.state_bits == bits; },
                [&](const Piece *piece, const int32_t *first, int n) {
                    Table t;
                    t.count = n;
                    for (int k = 0; k < n; ++k) {
                        const sv3d_adamw_tensor &s = tensors[piece[k].index];
                        const int64_t from = piece[k].from;
                        t.t[k] = {(E *)s.param + from, (const E *)s.grad + from, (char *)s.exp_avg + from * state,
                                  (char *)s.exp_avg_sq + from * state, s.scales ? s.scales + from / kBlock * 2 : nullptr,
                                  piece[k].numel};
                        t.order[k] = piece[k].index;
                    }
                    for (int k = 0; k <= n; ++k) t.first[k] = first[k];
                    const auto kernel = bits == 32 ? adamw_kernel<E> : adamw8_kernel<E>;
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
