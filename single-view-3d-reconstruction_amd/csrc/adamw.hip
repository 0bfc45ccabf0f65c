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
    double acc = 0.0;
    int k = 0;
    for (int chunk = blockIdx.x; chunk < t.first[t.count]; chunk += gridDim.x) {
        while (chunk >= t.first[k + 1]) ++k;
        const T *g = (const T *)t.grad[k];
        const int64_t at = (int64_t)(chunk - t.first[k]) * kSumChunk, end = min(at + kSumChunk, t.numel[k]);
        for (int64_t i = at + threadIdx.x; i < end; i += kThreads) {
            const double v = (double)to_float(g[i]);
            acc += v * v;
        }
    }
    for (int d = 32; d > 0; d >>= 1) acc += __shfl_xor(acc, d);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x / 64] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kThreads / 64; ++w) acc += part[w];
        sums[blockIdx.x] = acc;
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

// A magnitude t < 2^(17 or 8) to a code with three mantissa bits whose smallest normal value is 2^LOWEST: 20 bits
// of the fp32 mantissa fall off, after `bits` (16 of them, and half a one) has been added to them.  Below 2^LOWEST
// the codes are evenly spaced, as they are in the octave above it, so t is moved there.
template <int LOWEST>
__device__ inline uint32_t cut(float t, uint32_t bits)
{
    const bool small = t < power_of_two(LOWEST);
    t += small ? power_of_two(LOWEST) : 0.f;
    return ((__float_as_uint(t) + (bits << 4) + 8u) >> 20) - ((126u + LOWEST) << 3) - (small ? 8u : 0u);
}

// what a moment contributes to its block's exponent: an infinity or NaN does not
__device__ inline float finite_magnitude(float v) { return fabsf(v) < INFINITY ? fabsf(v) : 0.f; }

constexpr int kFirstBias = 134, kSecondBias = 142;      // a block's largest value lands in [2^7, 2^8) and [2^15, 2^16)
constexpr int kFirstFloor = 20, kSecondFloor = 34;      // so that every value is a normal number, also as bf16

__device__ inline uint32_t block_exponent(float largest, int floor) { return (uint32_t)max((int)(__float_as_uint(largest) >> 23), floor); }

__device__ inline uint32_t encode_first(float m, float scale, uint32_t bits)
{
    const float a = fabsf(m);
    const uint32_t code = a < INFINITY ? cut<-6>(a * scale, bits) : 0x7fu;
    return code | (__float_as_uint(m) >> 31 << 7);
}

__device__ inline uint32_t encode_second(float v, float scale, uint32_t bits)
{
    if (!(v < INFINITY)) return 0xffu;
    const uint32_t code = cut<-14>(v * scale, bits);
    return v > 0.f ? max(code, 1u) : code;
}

template <int LOWEST>
__device__ inline float magnitude(uint32_t code)
{
    const bool small = code < 8u;
    const float t = __uint_as_float((code + ((126u + LOWEST) << 3) + (small ? 8u : 0u)) << 20);
    return t - (small ? power_of_two(LOWEST) : 0.f);
}

__device__ inline float decode_first(uint32_t code, float unit)
{
    const uint32_t c = code & 0x7fu;
    const float a = c == 0x7fu ? NAN : magnitude<-6>(c) * unit;
    return code & 0x80u ? -a : a;
}

__device__ inline float decode_second(uint32_t code, float unit) { return code == 0xffu ? NAN : magnitude<-14>(code) * unit; }

// the power of two of a block's codes; a byte below the lowest that is ever written (fresh state: 0) counts as that one
__device__ inline float first_unit(uint32_t e) { return power_of_two(max((int)e, kFirstFloor) - kFirstBias); }
__device__ inline float second_unit(uint32_t e) { return power_of_two(max((int)e, kSecondFloor) - kSecondBias); }

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

// products and sums as they stand, each rounded: the same moments on every path
__device__ inline float step_of(float &m, float &v, float g, const Betas &b, const Factors &f)
{
    m = __fadd_rn(__fmul_rn(b.b1, m), __fmul_rn(b.c1, g));
    v = __fadd_rn(__fmul_rn(b.b2, v), __fmul_rn(b.c2, __fmul_rn(g, g)));
    return f.rate * (m / (sqrtf(v) * f.root + b.eps));
}

template <class T>
__global__ __launch_bounds__(kThreads) void adamw_kernel(Table t, Betas b, const Factors *__restrict__ factors)
{
    int k = 0;
    while ((int)blockIdx.x >= t.first[k + 1]) ++k;
    const Entry e = t.t[k];
    const Factors f = factors[t.order[k]];
    if (f.skip) return;
    const int64_t at = (int64_t)((int)blockIdx.x - t.first[k]) * kChunk, end = min(at + kChunk, e.numel);
    T *p = (T *)e.param;
    const T *g = (const T *)e.grad;
    float *em = (float *)e.exp_avg, *ev = (float *)e.exp_avg_sq;
    for (int64_t i = at + threadIdx.x; i < end; i += kThreads) {
        float m = em[i], v = ev[i];
        const float s = step_of(m, v, to_float(g[i]) * f.grad, b, f);
        em[i] = m;
        ev[i] = v;
        p[i] = from_float<T>(to_float(p[i]) * f.decay - s);
    }
}

// 16 lanes share a block of 128 elements, eight each
template <class T>
__global__ __launch_bounds__(kThreads) void adamw8_kernel(Table t, Betas b, const Factors *__restrict__ factors)
{
    int k = 0;
    while ((int)blockIdx.x >= t.first[k + 1]) ++k;
    const Entry e = t.t[k];
    const Factors f = factors[t.order[k]];
    if (f.skip) return;
    const int64_t i0 = (int64_t)((int)blockIdx.x - t.first[k]) * kChunk + threadIdx.x * 8, block = i0 / kBlock;
    const bool live = i0 < e.numel;
    T *p = (T *)e.param;
    const T *g = (const T *)e.grad;
    uint8_t *cm = (uint8_t *)e.exp_avg, *cv = (uint8_t *)e.exp_avg_sq;
    const float um = live ? first_unit(e.scales[2 * block]) : 0.f;
    const float uv = live ? second_unit(e.scales[2 * block + 1]) : 0.f;
    float m[8], v[8], top_m = 0.f, top_v = 0.f;
    for (int j = 0; j < 8; ++j) {
        const int64_t i = i0 + j;
        m[j] = v[j] = 0.f;
        if (i >= e.numel) continue;
        m[j] = decode_first(cm[i], um);
        v[j] = decode_second(cv[i], uv);
        const float s = step_of(m[j], v[j], to_float(g[i]) * f.grad, b, f);
        p[i] = from_float<T>(to_float(p[i]) * f.decay - s);
        top_m = fmaxf(top_m, finite_magnitude(m[j]));
        top_v = fmaxf(top_v, finite_magnitude(v[j]));
    }
    for (int d = 8; d > 0; d >>= 1) {
        top_m = fmaxf(top_m, __shfl_xor(top_m, d));
        top_v = fmaxf(top_v, __shfl_xor(top_v, d));
    }
    if (!live) return;
    const uint32_t xm = block_exponent(top_m, kFirstFloor), xv = block_exponent(top_v, kSecondFloor);
    const float sm = power_of_two(kFirstBias - (int)xm), sv = power_of_two(kSecondBias - (int)xv);
    for (int j = 0; j < 8; ++j) {
        const int64_t i = i0 + j;
        if (i >= e.numel) break;
        const uint32_t h = dither((uint32_t)i, f.key);
        cm[i] = (uint8_t)encode_first(m[j], sm, h >> 16);
        cv[i] = (uint8_t)encode_second(v[j], sv, h & 0xffffu);
    }
    if ((threadIdx.x & 15) == 0) {
        e.scales[2 * block] = (uint8_t)xm;
        e.scales[2 * block + 1] = (uint8_t)xv;
    }
}

__global__ __launch_bounds__(kThreads) void moment_values_kernel(const uint8_t *__restrict__ cm, const uint8_t *__restrict__ cv,
                                                                 const uint8_t *__restrict__ scales, int64_t numel,
                                                                 bf16 *__restrict__ m, bf16 *__restrict__ v)
{
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < numel; i += (int64_t)gridDim.x * kThreads) {
        const int64_t block = i / kBlock;
        m[i] = from_float<bf16>(decode_first(cm[i], first_unit(scales[2 * block])));
        v[i] = from_float<bf16>(decode_second(cv[i], second_unit(scales[2 * block + 1])));
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
    const int64_t groups = (numel + kThreads - 1) / kThreads;
    hipLaunchKernelGGL(moment_values_kernel, dim3((uint32_t)(groups < (1 << 20) ? groups : (1 << 20))), dim3(kThreads), 0,
                       (hipStream_t)stream, exp_avg, exp_avg_sq, scales, numel, (bf16 *)exp_avg_out, (bf16 *)exp_avg_sq_out);
    return launch_status();
}
