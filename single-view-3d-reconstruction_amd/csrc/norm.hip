// Layer norm over rows of `cols` elements, forward and backward.
//   forward:  mu = mean x, r = 1/sqrt(mean (x-mu)^2 + eps), y = (x-mu) r w + b
//   backward: h = (x-mu) r, u = dy w, dx = r (u - mean u - h mean(u h)), dw = sum_rows dy h, db = sum_rows dy
// Statistics, gradients and their sums are fp32; only what is stored is rounded to its type.
#include "element.h"

#include <type_traits>

namespace {

using namespace sv3d;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

__device__ inline float wave_sum(float v)
{
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// A wave per row, the row read three times.
template <class X, class Y, class P>
__global__ __launch_bounds__(kThreads) void layer_norm_forward_kernel(
    const X *__restrict__ x, const P *__restrict__ weight, const P *__restrict__ bias, int64_t rows, int64_t cols,
    int64_t x_stride, float eps, Y *__restrict__ y, float *__restrict__ mean, float *__restrict__ rstd)
{
    const int lane = threadIdx.x & 63;
    for (int64_t row = (int64_t)blockIdx.x * kWaves + threadIdx.x / 64; row < rows; row += (int64_t)gridDim.x * kWaves) {
        const X *xr = x + row * x_stride;
        float s = 0.f;
        for (int64_t c = lane; c < cols; c += 64) s += to_float(xr[c]);
        const float mu = wave_sum(s) / (float)cols;
        float q = 0.f;
        for (int64_t c = lane; c < cols; c += 64) {
            const float d = to_float(xr[c]) - mu;
            q += d * d;
        }
        const float r = 1.f / sqrtf(wave_sum(q) / (float)cols + eps);
        Y *yr = y + row * cols;
        for (int64_t c = lane; c < cols; c += 64) {
            const float h = (to_float(xr[c]) - mu) * r;
            yr[c] = from_float<Y>(h * (weight ? to_float(weight[c]) : 1.f) + (bias ? to_float(bias[c]) : 0.f));
        }
        if (lane == 0) {
            if (mean) mean[row] = mu;
            if (rstd) rstd[row] = r;
        }
    }
}

template <class X, class Y, class P>
__global__ __launch_bounds__(kThreads) void layer_norm_dx_kernel(
    const X *__restrict__ x, const Y *__restrict__ dy, const P *__restrict__ weight, const float *__restrict__ mean,
    const float *__restrict__ rstd, int64_t rows, int64_t cols, int64_t x_stride, int64_t dy_stride, X *__restrict__ dx)
{
    const int lane = threadIdx.x & 63;
    for (int64_t row = (int64_t)blockIdx.x * kWaves + threadIdx.x / 64; row < rows; row += (int64_t)gridDim.x * kWaves) {
        const X *xr = x + row * x_stride;
        const Y *dr = dy + row * dy_stride;
        const float mu = mean[row], r = rstd[row];
        float su = 0.f, sh = 0.f;
        for (int64_t c = lane; c < cols; c += 64) {
            const float u = to_float(dr[c]) * (weight ? to_float(weight[c]) : 1.f);
            su += u;
            sh += u * ((to_float(xr[c]) - mu) * r);
        }
        su = wave_sum(su) / (float)cols;
        sh = wave_sum(sh) / (float)cols;
        X *o = dx + row * cols;
        for (int64_t c = lane; c < cols; c += 64) {
            const float u = to_float(dr[c]) * (weight ? to_float(weight[c]) : 1.f);
            o[c] = from_float<X>((u - su - (to_float(xr[c]) - mu) * r * sh) * r);
        }
    }
}

// dweight and dbias: a thread per column adds up a slice of the rows ...
constexpr int kSlices = 64;

template <class X, class Y>
__global__ __launch_bounds__(kThreads) void layer_norm_slices_kernel(
    const X *__restrict__ x, const Y *__restrict__ dy, const float *__restrict__ mean, const float *__restrict__ rstd,
    int64_t rows, int64_t cols, int64_t x_stride, int64_t dy_stride, float *__restrict__ part)
{
    const int64_t c = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (c >= cols) return;
    float w = 0.f, b = 0.f;
    for (int64_t row = blockIdx.y; row < rows; row += kSlices) {
        const float d = to_float(dy[row * dy_stride + c]);
        w += d * ((to_float(x[row * x_stride + c]) - mean[row]) * rstd[row]);
        b += d;
    }
    part[(2 * (int64_t)blockIdx.y) * cols + c] = w;
    part[(2 * (int64_t)blockIdx.y + 1) * cols + c] = b;
}

// ... and then the slices
template <class P>
__global__ __launch_bounds__(kThreads) void layer_norm_join_kernel(const float *__restrict__ part, int64_t cols,
                                                                   P *__restrict__ dweight, P *__restrict__ dbias)
{
    const int64_t c = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (c >= cols) return;
    float w = 0.f, b = 0.f;
    for (int s = 0; s < kSlices; ++s) {
        w += part[(2 * (int64_t)s) * cols + c];
        b += part[(2 * (int64_t)s + 1) * cols + c];
    }
    if (dweight) dweight[c] = from_float<P>(w);
    if (dbias) dbias[c] = from_float<P>(b);
}

// workgroups for a wave per row; beyond the cap (a launch holds fewer than 2^32 threads) a wave takes several rows
uint32_t row_blocks(int64_t rows)
{
    const int64_t n = (rows + kWaves - 1) / kWaves;
    return (uint32_t)(n < (1 << 20) ? n : (1 << 20));
}

int check(const sv3d_layer_norm_params *p)
{
    if (!p || p->rows < 0 || p->cols <= 0 || p->x_stride < 0) return SV3D_ERR_INVALID_ARG;
    if (!known_type(p->x_type) || !(p->eps >= 0.f)) return SV3D_ERR_INVALID_ARG;
    if ((p->y_type != p->x_type && p->y_type != SV3D_F32) || (p->param_type != p->x_type && p->param_type != SV3D_F32))
        return SV3D_ERR_INVALID_ARG;
    if (p->rows > ((int64_t)1 << 40) || p->cols > ((int64_t)1 << 24)) return SV3D_ERR_UNSUPPORTED;
    return SV3D_OK;
}

// calls f(x, y, param) with null pointers of the element types
template <class X, class F>
int with_types_of(const sv3d_layer_norm_params *p, F f)
{
    const bool y32 = p->y_type == SV3D_F32, p32 = p->param_type == SV3D_F32;
    if (y32 && p32) return f((X *)nullptr, (float *)nullptr, (float *)nullptr);
    if (y32) return f((X *)nullptr, (float *)nullptr, (X *)nullptr);
    if (p32) return f((X *)nullptr, (X *)nullptr, (float *)nullptr);
    return f((X *)nullptr, (X *)nullptr, (X *)nullptr);
}

template <class F>
int with_types(const sv3d_layer_norm_params *p, F f)
{
    if (p->x_type == SV3D_F32) return f((float *)nullptr, (float *)nullptr, (float *)nullptr);
    return p->x_type == SV3D_F16 ? with_types_of<f16>(p, f) : with_types_of<bf16>(p, f);
}

}  // namespace

extern "C" int sv3d_layer_norm_forward(const sv3d_layer_norm_params *p, const void *x, const void *weight,
                                       const void *bias, void *y, float *mean, float *rstd, void *stream)
{
    if (const int st = check(p)) return st;
    if (p->rows == 0) return SV3D_OK;
    if (!x || !y) return SV3D_ERR_INVALID_ARG;
    return with_types(p, [&](auto *X, auto *Y, auto *P) {
        using XT = std::remove_pointer_t<decltype(X)>;
        using YT = std::remove_pointer_t<decltype(Y)>;
        using PT = std::remove_pointer_t<decltype(P)>;
        hipLaunchKernelGGL((layer_norm_forward_kernel<XT, YT, PT>), dim3(row_blocks(p->rows)),
                           dim3(kThreads), 0, (hipStream_t)stream, (const XT *)x, (const PT *)weight, (const PT *)bias,
                           p->rows, p->cols, p->x_stride, p->eps, (YT *)y, mean, rstd);
        return launch_status();
    });
}

extern "C" int sv3d_layer_norm_workspace(const sv3d_layer_norm_params *p, size_t *bytes)
{
    if (!bytes) return SV3D_ERR_INVALID_ARG;
    if (const int st = check(p)) return st;
    *bytes = (size_t)2 * kSlices * p->cols * sizeof(float);
    return SV3D_OK;
}

extern "C" int sv3d_layer_norm_backward(const sv3d_layer_norm_params *p, const void *x, const void *dy,
                                        const void *weight, const float *mean, const float *rstd, void *dx,
                                        void *dweight, void *dbias, void *workspace, size_t workspace_bytes,
                                        void *stream)
{
    if (const int st = check(p)) return st;
    if (p->dy_stride < 0) return SV3D_ERR_INVALID_ARG;
    if (p->rows > 0 && (!x || !dy || !mean || !rstd)) return SV3D_ERR_INVALID_ARG;
    const bool params = dweight || dbias;
    if (params) {
        size_t need = 0;
        sv3d_layer_norm_workspace(p, &need);
        if (!workspace || !aligned(workspace, 16)) return SV3D_ERR_INVALID_ARG;
        if (workspace_bytes < need) return SV3D_ERR_WORKSPACE;
    }
    return with_types(p, [&](auto *X, auto *Y, auto *P) {
        using XT = std::remove_pointer_t<decltype(X)>;
        using YT = std::remove_pointer_t<decltype(Y)>;
        using PT = std::remove_pointer_t<decltype(P)>;
        if (dx && p->rows > 0) {
            hipLaunchKernelGGL((layer_norm_dx_kernel<XT, YT, PT>), dim3(row_blocks(p->rows)),
                               dim3(kThreads), 0, (hipStream_t)stream, (const XT *)x, (const YT *)dy, (const PT *)weight,
                               mean, rstd, p->rows, p->cols, p->x_stride, p->dy_stride, (XT *)dx);
            if (const int st = launch_status()) return st;
        }
        if (params) {
            const uint32_t blocks = (uint32_t)((p->cols + kThreads - 1) / kThreads);
            hipLaunchKernelGGL((layer_norm_slices_kernel<XT, YT>), dim3(blocks, kSlices), dim3(kThreads), 0,
                               (hipStream_t)stream, (const XT *)x, (const YT *)dy, mean, rstd, p->rows, p->cols,
                               p->x_stride, p->dy_stride, (float *)workspace);
            if (const int st = launch_status()) return st;
            hipLaunchKernelGGL((layer_norm_join_kernel<PT>), dim3(blocks), dim3(kThreads), 0, (hipStream_t)stream,
                               (const float *)workspace, p->cols, (PT *)dweight, (PT *)dbias);
            return launch_status();
        }
        return (int)SV3D_OK;
    });
}
