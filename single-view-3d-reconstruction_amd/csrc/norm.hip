// Layer norm over rows of `cols` elements, forward and backward.
//   forward:  mu = mean x, r = 1/sqrt(mean (x-mu)^2 + eps), y = (x-mu) r w + b
//   backward: h = (x-mu) r, u = dy w, dx = r (u - mean u - h mean(u h)), dw = sum_rows dy h, db = sum_rows dy
// Statistics, gradients and a workgroup's sums are fp32, the join of those over the rows is double; only what is stored
// is rounded to its type.
#include "element.h"

#include <type_traits>

namespace {

using namespace sv3d;

constexpr int kThreads = 256;

// ---- rows in registers ------------------------------------------------------------------------------
// G threads share a row, each holds K packs of 16 bytes of it, G packs apart.  Rows shorter than a wave's packs
// share the wave; rows longer than 64 threads hold take a workgroup, whose waves add up through LDS.
template <class X>
constexpr int kPack = 16 / (int)sizeof(X);

template <int G>
constexpr int kGroup = G > 64 ? G : 256;        // threads of the workgroup

// Which of a workgroup's rows a thread works on: known to the whole wave (and kept in scalar registers, the row's
// addresses with it) where a wave has no more than one.
template <int G>
__device__ inline int row_of_group()
{
    const int r = threadIdx.x / G;
    return G >= 64 ? __builtin_amdgcn_readfirstlane(r) : r;
}

// The sum over the row's threads.  `part` is not written again before every thread has passed another row_sum on
// another buffer, so one barrier is enough.
template <int G>
__device__ inline float row_sum(float v, float *part)
{
    if (G <= 64) return lane_sum<(G < 64 ? G : 64)>(v);
    v = lane_sum<64>(v);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x / 64] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int w = 1; w < G / 64; ++w) v += part[w];
    return v;
}

template <int V>
__device__ inline float sum_of(const float *v)
{
    float s = v[0];
#pragma unroll
    for (int j = 1; j < V; ++j) s += v[j];
    return s;
}

// A row's packs.  Where the row's end cuts one, the pack that ends with the row is loaded in its place and what it
// repeats is dropped when the values are used (drop_end): put together from single elements, a pack would have to
// be waited for where it is loaded, and no load of the next row would be on its way during the work on this one.  Rows of
// eight packs at most, which may be shorter than one, are put together.
template <class X, int G, bool ENDS>
__device__ inline int cut_by(int n)
{
    return ENDS && G > 8 && n > 0 && n < kPack<X> ? kPack<X> - n : 0;
}

template <class T, int V, int G, bool ENDS>
__device__ inline Words<T, V> load_row(const T *p, int n, int cut)
{
    return load_words<T, V, (ENDS && G <= 8)>(p - cut, n);
}

template <int G, bool ENDS, class T, int V>
__device__ inline void drop_end(Words<T, V> &w, int cut)
{
    if (ENDS && G > 8 && cut) drop_words(w, cut);
}

// weights of either type, kept in registers over all the rows of a thread
template <class X, int V, bool ENDS>
__device__ inline void load_params(const void *p, bool f32, float missing, int c, int n, float *out)
{
    if (!p) {
#pragma unroll
        for (int j = 0; j < V; ++j) out[j] = missing;
    } else if (f32 || __is_same(X, float)) {
        const auto r = load_words<float, V, ENDS>((const float *)p + c, n);
#pragma unroll
        for (int j = 0; j < V; ++j) out[j] = r[j];
    } else {
        const auto r = load_words<X, V, ENDS>((const X *)p + c, n);
#pragma unroll
        for (int j = 0; j < V; ++j) out[j] = r[j];
    }
}

template <class X, class Y, int G, int K, bool ENDS, bool STREAM>
__global__ __launch_bounds__(kGroup<G>) void layer_norm_forward_kernel(
    const X *__restrict__ x, const void *__restrict__ weight, const void *__restrict__ bias, int params_f32, int cols,
    int64_t rows, int64_t x_stride, float eps, Y *__restrict__ y, float *__restrict__ mean, float *__restrict__ rstd)
{
    constexpr int V = kPack<X>, R = kGroup<G> / G;
    __shared__ float part[2][G > 64 ? G / 64 : 1];
    const int lane = threadIdx.x % G;
    const int64_t step = (int64_t)gridDim.x * R;
    int64_t row = (int64_t)blockIdx.x * R + row_of_group<G>();
    const float inv = 1.f / (float)cols;
    int cut[K];
    Words<X, V> next[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = (k * G + lane) * V;
        cut[k] = cut_by<X, G, ENDS>(cols - c);
        if (row < rows) next[k] = load_row<X, V, G, ENDS>(x + row * x_stride + c, cols - c, cut[k]);
    }
    float w[K][V], b[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = (k * G + lane) * V;
        load_params<X, V, ENDS>(weight, params_f32, 1.f, c, cols - c, w[k]);
        load_params<X, V, ENDS>(bias, params_f32, 0.f, c, cols - c, b[k]);
    }
    for (; row < rows; row += step) {
        float v[K][V], s = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            drop_end<G, ENDS>(next[k], cut[k]);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[k][j] = next[k][j];
                s += v[k][j];                       // zero behind the row's end
            }
        }
        if (row + step < rows) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int c = (k * G + lane) * V;
                next[k] = load_row<X, V, G, ENDS>(x + (row + step) * x_stride + c, cols - c, cut[k]);
            }
        }
        const float mu = row_sum<G>(s, part[0]) * inv;
        float q = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[k][j] -= mu;
                q += (k * G + lane) * V + (ENDS ? j : 0) < cols ? v[k][j] * v[k][j] : 0.f;
            }
        const float r = 1.f / sqrtf(row_sum<G>(q, part[1]) * inv + eps);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * G + lane) * V;
#pragma unroll
            for (int j = 0; j < V; ++j) v[k][j] = v[k][j] * r * w[k][j] + b[k][j];
            store_pack<Y, V, ENDS, STREAM>(y + row * cols + c, v[k], cols - c);
        }
        if (lane == 0) {
            if (mean) mean[row] = mu;
            if (rstd) rstd[row] = r;
        }
    }
}

// ---- rows beyond registers: a workgroup per row, which it reads three times ----------------------------
constexpr int kLong = 1024;

template <class X, class Y>
__global__ __launch_bounds__(kLong) void layer_norm_forward_long_kernel(
    const X *__restrict__ x, const void *__restrict__ weight, const void *__restrict__ bias, int params_f32, int cols,
    int64_t rows, int64_t x_stride, float eps, Y *__restrict__ y, float *__restrict__ mean, float *__restrict__ rstd)
{
    constexpr int V = kPack<X>;
    __shared__ float part[2][kLong / 64];
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const X *xr = x + row * x_stride;
        float s[V] = {};
        for (int c = threadIdx.x * V; c < cols; c += kLong * V) {
            const auto w = load_words<X, V>(xr + c, cols - c);
#pragma unroll
            for (int j = 0; j < V; ++j) s[j] += w[j];           // zero behind the row's end
        }
        const float mu = row_sum<kLong>(sum_of<V>(s), part[0]) / (float)cols;
        float q[V] = {};
        for (int c = threadIdx.x * V; c < cols; c += kLong * V) {
            const auto w = load_words<X, V>(xr + c, cols - c);
#pragma unroll
            for (int j = 0; j < V; ++j) q[j] += c + j < cols ? (w[j] - mu) * (w[j] - mu) : 0.f;
        }
        const float r = 1.f / sqrtf(row_sum<kLong>(sum_of<V>(q), part[1]) / (float)cols + eps);
        for (int c = threadIdx.x * V; c < cols; c += kLong * V) {
            const auto v = load_words<X, V>(xr + c, cols - c);
            float w[V], b[V];
            load_params<X, V, true>(weight, params_f32, 1.f, c, cols - c, w);
            load_params<X, V, true>(bias, params_f32, 0.f, c, cols - c, b);
#pragma unroll
            for (int j = 0; j < V; ++j) w[j] = (v[j] - mu) * r * w[j] + b[j];
            store_pack<Y, V>(y + row * cols + c, w, cols - c);
        }
        if (threadIdx.x == 0) {
            if (mean) mean[row] = mu;
            if (rstd) rstd[row] = r;
        }
    }
}

// The compiler takes the values for new ones.
template <class T, int N>
__device__ inline void forget(Words<T, N> &w)
{
#pragma unroll
    for (int i = 0; i < w.kCount; ++i) asm("" : "+v"(w.w[i]));
}

// ---- backward, rows in registers --------------------------------------------------------------------
// One pass over x and dy: dx, and the weights' gradients of the workgroup's rows, which stay in registers until its last
// row, are added up over the rows that the workgroup has at a time and go to `part` [workgroup][2][cols].  x and dy
// are held as they were loaded and converted where they are used: with the weight and the two gradients in registers
// there is no room for the values in fp32 as well, and arithmetic is not what this waits for.
template <int G>
constexpr int kBack = G > 512 ? G : 512;

template <class X, class Y, int G, int K, bool ENDS, bool STREAM>
__global__ __launch_bounds__(kBack<G>, 4) void layer_norm_backward_kernel(
    const X *__restrict__ x, const Y *__restrict__ dy, const void *__restrict__ weight, int params_f32, int cols, int64_t rows,
    const float *__restrict__ mean, const float *__restrict__ rstd, int64_t x_stride, int64_t dy_stride, X *__restrict__ dx,
    float *__restrict__ part)
{
    constexpr int V = kPack<X>, R = kBack<G> / G, E = K * V;
    __shared__ float both[2][2][kBack<G> / 64];
    const int lane = threadIdx.x % G, wave = threadIdx.x / 64;
    const int64_t step = (int64_t)gridDim.x * R;
    int64_t row = (int64_t)blockIdx.x * R + row_of_group<G>();
    const float inv = 1.f / (float)cols;
    int cut[K];
#pragma unroll
    for (int k = 0; k < K; ++k) cut[k] = cut_by<X, G, ENDS>(cols - (k * G + lane) * V);
    Words<X, V> nx[K];
    Words<Y, V> nd[K];
    float nmu, nr;
    // a row behind the last one has dy = 0 and adds nothing anywhere
    const auto fetch = [&](int64_t at) {
        const bool there = at < rows;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * G + lane) * V, n = there ? cols - c : 0;
            nx[k] = load_row<X, V, G, ENDS>(x + at * x_stride + c, n, cut[k]);
            nd[k] = load_row<Y, V, G, ENDS>(dy + at * dy_stride + c, n, cut[k]);
        }
        nmu = there ? mean[at] : 0.f;
        nr = there ? rstd[at] : 0.f;
    };
    fetch(row);
    float w[E], dw[E], db[E];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = (k * G + lane) * V;
        load_params<X, V, ENDS>(weight, params_f32, 1.f, c, cols - c, w + k * V);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) dw[e] = db[e] = 0.f;
    int turn = 0;
    for (int64_t base = (int64_t)blockIdx.x * R; base < rows; base += step, row += step, turn ^= 1) {
        Words<X, V> cx[K];
        Words<Y, V> cd[K];
#pragma unroll
        for (int k = 0; k < K; ++k) {
            cx[k] = nx[k];
            cd[k] = nd[k];
            drop_end<G, ENDS>(cx[k], cut[k]);
            drop_end<G, ENDS>(cd[k], cut[k]);
        }
        const float mu = nmu, r = nr;
        if (base + step < rows) fetch(row + step);
        float su = 0.f, sh = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float d = cd[e / V][e % V];       // zero behind the row's end, and so is all that it enters
            const float h = (cx[e / V][e % V] - mu) * r, u = d * w[e];
            dw[e] += d * h;
            db[e] += d;
            su += u;
            sh += u * h;
        }
        if (!dx) continue;
        su = lane_sum<(G < 64 ? G : 64)>(su);
        sh = lane_sum<(G < 64 ? G : 64)>(sh);
        if constexpr (G > 64) {
            // both sums with one barrier; the buffers of two turns alternate
            if ((threadIdx.x & 63) == 0) {
                both[turn][0][wave] = su;
                both[turn][1][wave] = sh;
            }
            __syncthreads();
            const int first = threadIdx.x / G * (G / 64);
            su = both[turn][0][first];
            sh = both[turn][1][first];
#pragma unroll
            for (int i = 1; i < G / 64; ++i) {
                su += both[turn][0][first + i];
                sh += both[turn][1][first + i];
            }
        }
        su *= inv;
        sh *= inv;
        // what follows is worked out from x and dy again: kept from above, it would take 16 registers more
#pragma unroll
        for (int k = 0; k < K; ++k) {
            forget(cx[k]);
            forget(cd[k]);
        }
        if (row >= rows) continue;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * G + lane) * V;
            float o[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float h = (cx[k][j] - mu) * r, u = cd[k][j] * w[k * V + j];
                o[j] = (u - su - h * sh) * r;
            }
            store_pack<X, V, ENDS, STREAM>(dx + row * cols + c, o, cols - c);
        }
    }
    if (!part) return;
    // the rows that share a wave, then the others by halves
#pragma unroll
    for (int e = 0; e < E; ++e) {
#pragma unroll
        for (int d = G; d < 64; d *= 2) {
            dw[e] += __shfl_xor(dw[e], d);
            db[e] += __shfl_xor(db[e], d);
        }
    }
    constexpr int kTeam = G < 64 ? 64 : G, kHalf = kBack<G> / kTeam / 2;
    const int team = threadIdx.x / kTeam;
    const bool first = threadIdx.x % kTeam < G;
    if constexpr (kHalf > 0) {
        __shared__ float fold[kHalf][E][G];
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            float(&acc)[E] = which ? db : dw;
            for (int half = kHalf; half > 0; half /= 2) {
                __syncthreads();
                if (first && team >= half && team < 2 * half)
#pragma unroll
                    for (int e = 0; e < E; ++e) fold[team - half][e][lane] = acc[e];
                __syncthreads();
                if (first && team < half)
#pragma unroll
                    for (int e = 0; e < E; ++e) acc[e] += fold[team][e][lane];
            }
        }
    }
    if (team != 0 || !first) return;
    float *out = part + (int64_t)blockIdx.x * 2 * cols;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = (k * G + lane) * V;
        store_pack<float, V, ENDS>(out + c, dw + k * V, cols - c);
        store_pack<float, V, ENDS>(out + cols + c, db + k * V, cols - c);
    }
}

// Rows beyond registers: a workgroup per row, which it reads twice.
template <class X, class Y>
__global__ __launch_bounds__(kLong) void layer_norm_dx_long_kernel(
    const X *__restrict__ x, const Y *__restrict__ dy, const void *__restrict__ weight, int params_f32, int cols, int64_t rows,
    const float *__restrict__ mean, const float *__restrict__ rstd, int64_t x_stride, int64_t dy_stride, X *__restrict__ dx)
{
    constexpr int V = kPack<X>;
    __shared__ float part[2][kLong / 64];
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const X *xr = x + row * x_stride;
        const Y *dr = dy + row * dy_stride;
        const float mu = mean[row], r = rstd[row];
        float su[V] = {}, sh[V] = {};
        for (int c = threadIdx.x * V; c < cols; c += kLong * V) {
            const auto v = load_words<X, V>(xr + c, cols - c);
            const auto d = load_words<Y, V>(dr + c, cols - c);
            float w[V];
            load_params<X, V, true>(weight, params_f32, 1.f, c, cols - c, w);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float u = d[j] * w[j];                    // zero behind the row's end
                su[j] += u;
                sh[j] += u * ((v[j] - mu) * r);
            }
        }
        const float mu_u = row_sum<kLong>(sum_of<V>(su), part[0]) / (float)cols;
        const float mu_uh = row_sum<kLong>(sum_of<V>(sh), part[1]) / (float)cols;
        for (int c = threadIdx.x * V; c < cols; c += kLong * V) {
            const auto v = load_words<X, V>(xr + c, cols - c);
            const auto d = load_words<Y, V>(dr + c, cols - c);
            float w[V];
            load_params<X, V, true>(weight, params_f32, 1.f, c, cols - c, w);
#pragma unroll
            for (int j = 0; j < V; ++j) w[j] = (d[j] * w[j] - mu_u - (v[j] - mu) * r * mu_uh) * r;
            store_pack<X, V>(dx + row * cols + c, w, cols - c);
        }
    }
}

// dweight and dbias of such rows: a thread for a few columns adds up a slice of the rows
constexpr int kSlices = 64, kSliceColumns = 4;

template <class X, class Y>
__global__ __launch_bounds__(kThreads) void layer_norm_slices_kernel(
    const X *__restrict__ x, const Y *__restrict__ dy, const float *__restrict__ mean, const float *__restrict__ rstd,
    int64_t rows, int cols, int64_t x_stride, int64_t dy_stride, float *__restrict__ part)
{
    constexpr int V = kSliceColumns;
    const int c = (blockIdx.x * kThreads + threadIdx.x) * V, n = cols - c;
    if (n <= 0) return;
    float w[V] = {}, b[V] = {};
#pragma unroll 4
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const auto v = load_words<X, V>(x + row * x_stride + c, n);
        const auto d = load_words<Y, V>(dy + row * dy_stride + c, n);
        const float mu = mean[row], r = rstd[row];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            w[j] += d[j] * ((v[j] - mu) * r);
            b[j] += d[j];
        }
    }
    float *out = part + 2 * (int64_t)blockIdx.y * cols + c;
    store_pack<float, V>(out, w, n);
    store_pack<float, V>(out + cols, b, n);
}

// The sum over the `count` partial sums: 16 columns of one of the two gradients per workgroup, 64 threads each.  In
// double: there are up to 512 of either sign, and this waits for its loads.
template <class P>
__global__ __launch_bounds__(1024) void layer_norm_join_kernel(const float *__restrict__ part, int count, int cols,
                                                               P *__restrict__ dweight, P *__restrict__ dbias)
{
    __shared__ double fold[64][17];
    P *out = blockIdx.y ? dbias : dweight;
    if (!out) return;
    const int c = blockIdx.x * 16 + threadIdx.x % 16, slice = threadIdx.x / 16;
    double s = 0.0;
    if (c < cols)
        for (int i = slice; i < count; i += 64) s += (double)part[(2 * (int64_t)i + blockIdx.y) * cols + c];
    fold[slice][threadIdx.x % 16] = s;
    __syncthreads();
    if (threadIdx.x >= 256) return;
    // 16 lanes for each of the 16 columns
    const int column = threadIdx.x / 16, l = threadIdx.x % 16;
    s = (fold[l][column] + fold[l + 16][column]) + (fold[l + 32][column] + fold[l + 48][column]);
#pragma unroll
    for (int d = 1; d < 16; d *= 2) s += __shfl_xor(s, d);
    if (l == 0 && blockIdx.x * 16 + column < cols) out[blockIdx.x * 16 + column] = from_float<P>((float)s);
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

// Threads per row and packs per thread that hold `cols` columns, as a call f(G, K): the fewest threads that do with one
// pack each, but two before a row needs more than a wave (with a wave to itself it is added up without a barrier: 32768 x
// 1024 bf16 24.1 us, 25.9 with one pack in 128 threads), and more than one beyond 1024 threads; f(0, 0) beyond those.
// With one pack a thread needs no more than 64 registers and a CU holds 2048 of them: 16384 x 4096 bf16 53.3 us with two
// packs in 256 threads, 49.8 with one in 512.  These widths fill their threads; one that does not leaves threads idle (5003 x
// 1336 fp16, 167 packs in 256 threads: 8.8 us, where the bytes take 4.4), and was not measured with other shapes.
template <int G_, int K_>
struct Shape {
    static constexpr int G = G_, K = K_;
};

template <class X, class F>
int with_shape(int64_t cols, F f)
{
    const int64_t packs = (cols + kPack<X> - 1) / kPack<X>;
    if (packs <= 8) return f(Shape<8, 1>());
    if (packs <= 16) return f(Shape<16, 1>());
    if (packs <= 32) return f(Shape<32, 1>());
    if (packs <= 64) return f(Shape<64, 1>());
    if (packs <= 128) return f(Shape<64, 2>());
    if (packs <= 256) return f(Shape<256, 1>());
    if (packs <= 512) return f(Shape<512, 1>());
    if (packs <= 1024) return f(Shape<1024, 1>());
    if (packs <= 2048) return f(Shape<1024, 2>());
    if constexpr (kPack<X> == 4)
        if (packs <= 4096) return f(Shape<1024, 4>());
    return f(Shape<0, 0>());
}

// The same for the backward, which holds five values for each element: eight elements per thread, up to 8192 columns
// (sixteen do not fit the 128 registers of a thread in a workgroup of 1024).
template <class X, class F>
int with_back_shape(int64_t cols, F f)
{
    const int64_t packs = (cols + kPack<X> - 1) / kPack<X>;
    constexpr int K = 8 / kPack<X>;
    if (packs <= 8) return f(Shape<8, 1>());
    if (packs <= 16) return f(Shape<16, 1>());
    if (packs <= 32) return f(Shape<32, 1>());
    if (packs <= 64) return f(Shape<64, 1>());
    if constexpr (K == 2)
        if (packs <= 128) return f(Shape<64, 2>());
    if (packs <= 128 * K) return f(Shape<128, K>());
    if (packs <= 256 * K) return f(Shape<256, K>());
    if (packs <= 512 * K) return f(Shape<512, K>());
    if (packs <= 1024 * K) return f(Shape<1024, K>());
    return f(Shape<0, 0>());
}

// What a kernel is compiled for: whether a row's end cuts a pack (or only leaves packs out), and whether its output goes
// past the caches, f(ENDS, STREAM).  The output of a layer is what the next one reads; but where the call reads and
// writes more than the 256 MB of the last cache, the start of it is gone when that one comes, and what is left to be
// written back meets the next reads (16384 x 4096 bf16 forward and backward 133 us through the caches, 120 past them; 32768 x 512
// forward 11.3 and 11.2).
template <bool V>
struct Bool {
    static constexpr bool value = V;
};
constexpr int64_t kLastCache = (int64_t)256 << 20;

template <class F>
int with_ends(bool ends, bool stream, F f)
{
    if (ends) return stream ? f(Bool<true>(), Bool<true>()) : f(Bool<true>(), Bool<false>());
    return stream ? f(Bool<false>(), Bool<true>()) : f(Bool<false>(), Bool<false>());
}

// A workgroup for each set of rows, but no more than the device holds at once: more rows are taken in turn, with the
// weights in registers and the next row's load on its way.
uint32_t persistent_groups(int64_t rows, int rows_per_group, int threads, int per_cu = 2048)
{
    const int64_t want = (rows + rows_per_group - 1) / rows_per_group, fit = 256 * (per_cu / threads);
    return (uint32_t)(want < fit ? want : fit);
}

template <class X, class F>
int with_output(const sv3d_layer_norm_params *p, F f)
{
    return p->y_type == SV3D_F32 ? f((X *)nullptr, (float *)nullptr) : f((X *)nullptr, (X *)nullptr);
}

// calls f(x, y) with null pointers of the element types
template <class F>
int with_xy(const sv3d_layer_norm_params *p, F f)
{
    if (p->x_type == SV3D_F32) return f((float *)nullptr, (float *)nullptr);
    return p->x_type == SV3D_F16 ? with_output<f16>(p, f) : with_output<bf16>(p, f);
}

// Workgroups of the backward, each of which leaves one partial sum of dweight and dbias: two for each CU, enough to fill
// the device.  The partial sums, written and read once more, are little where a workgroup has many rows (16384 x 4096 bf16: 34 of
// 437 MB), not where it has few (4224 x 512 fp32: 4 of 30 MB; 512 x 8192 bf16: 67 of 92 MB, backward 14.8 us, join 12.7).
constexpr int kBackGroups = 512;

template <class X>
int partial_sums(const sv3d_layer_norm_params *p)
{
    return with_back_shape<X>(p->cols, [&](auto shape) {
        constexpr int G = decltype(shape)::G;
        if constexpr (G == 0) {
            return (int)(p->rows < kSlices ? p->rows : kSlices);
        } else {
            constexpr int R = kBack<G> / G;
            const int64_t want = (p->rows + R - 1) / R;
            return (int)(want < kBackGroups ? want : kBackGroups);
        }
    });
}

int partial_sums(const sv3d_layer_norm_params *p)
{
    return p->x_type == SV3D_F32 ? partial_sums<float>(p) : partial_sums<f16>(p);
}

}  // namespace

extern "C" int sv3d_layer_norm_forward(const sv3d_layer_norm_params *p, const void *x, const void *weight,
                                       const void *bias, void *y, float *mean, float *rstd, void *stream)
{
    if (const int st = check(p)) return st;
    if (p->rows == 0) return SV3D_OK;
    if (!x || !y) return SV3D_ERR_INVALID_ARG;
    if (!aligned(x, type_bytes(p->x_type)) || !aligned(y, type_bytes(p->y_type)) || !aligned(weight, type_bytes(p->param_type)) ||
        !aligned(bias, type_bytes(p->param_type)) || !aligned(mean, 4) || !aligned(rstd, 4))
        return SV3D_ERR_INVALID_ARG;
    return with_xy(p, [&](auto *xt, auto *yt) {
        using X = std::remove_pointer_t<decltype(xt)>;
        using Y = std::remove_pointer_t<decltype(yt)>;
        return with_shape<X>(p->cols, [&](auto shape) {
            constexpr int G = decltype(shape)::G, K = decltype(shape)::K;
            const int f32 = p->param_type == SV3D_F32, cols = (int)p->cols;
            if constexpr (G == 0)
                hipLaunchKernelGGL((layer_norm_forward_long_kernel<X, Y>), dim3(persistent_groups(p->rows, 1, kLong)),
                                   dim3(kLong), 0, (hipStream_t)stream, (const X *)x, weight, bias, f32, cols, p->rows,
                                   p->x_stride, p->eps, (Y *)y, mean, rstd);
            else
                with_ends(cols % kPack<X> != 0, p->rows * cols * (int64_t)(sizeof(X) + sizeof(Y)) >= kLastCache, [&](auto ends, auto past) {
                    hipLaunchKernelGGL((layer_norm_forward_kernel<X, Y, G, K, decltype(ends)::value, decltype(past)::value>),
                                       dim3(persistent_groups(p->rows, kGroup<G> / G, kGroup<G>, G == 1024 && K > 1 ? 1024 : 2048)),
                                       dim3(kGroup<G>), 0,
                                       (hipStream_t)stream, (const X *)x, weight, bias, f32, cols, p->rows, p->x_stride, p->eps,
                                       (Y *)y, mean, rstd);
                    return 0;
                });
            return launch_status();
        });
    });
}

extern "C" int sv3d_layer_norm_workspace(const sv3d_layer_norm_params *p, size_t *bytes)
{
    if (!bytes) return SV3D_ERR_INVALID_ARG;
    if (const int st = check(p)) return st;
    *bytes = (size_t)2 * partial_sums(p) * p->cols * sizeof(float);
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
    if (!aligned(x, type_bytes(p->x_type)) || !aligned(dy, type_bytes(p->y_type)) || !aligned(dx, type_bytes(p->x_type)) ||
        !aligned(weight, type_bytes(p->param_type)) || !aligned(dweight, type_bytes(p->param_type)) ||
        !aligned(dbias, type_bytes(p->param_type)) || !aligned(mean, 4) || !aligned(rstd, 4))
        return SV3D_ERR_INVALID_ARG;
    const bool params = dweight || dbias;
    if (params && p->rows > 0) {
        size_t need = 0;
        sv3d_layer_norm_workspace(p, &need);
        if (!workspace || !aligned(workspace, 16)) return SV3D_ERR_INVALID_ARG;
        if (workspace_bytes < need) return SV3D_ERR_WORKSPACE;
    }
    const int cols = (int)p->cols, count = partial_sums(p), f32 = p->param_type == SV3D_F32;
    float *part = params ? (float *)workspace : nullptr;
    hipStream_t s = (hipStream_t)stream;
    if (p->rows > 0 && (dx || params)) {
        const int st = with_xy(p, [&](auto *xt, auto *yt) {
            using X = std::remove_pointer_t<decltype(xt)>;
            using Y = std::remove_pointer_t<decltype(yt)>;
            return with_back_shape<X>(p->cols, [&](auto shape) {
                constexpr int G = decltype(shape)::G, K = decltype(shape)::K;
                if constexpr (G > 0) {
                    const int64_t bytes = p->rows * cols * (int64_t)(2 * sizeof(X) + sizeof(Y));
                    with_ends(cols % kPack<X> != 0, bytes >= kLastCache, [&](auto ends, auto past) {
                        hipLaunchKernelGGL((layer_norm_backward_kernel<X, Y, G, K, decltype(ends)::value, decltype(past)::value>),
                                           dim3(count), dim3(kBack<G>), 0, s, (const X *)x, (const Y *)dy, weight, f32, cols,
                                           p->rows, mean, rstd, p->x_stride, p->dy_stride, (X *)dx, part);
                        return 0;
                    });
                } else {
                    if (dx)
                        hipLaunchKernelGGL((layer_norm_dx_long_kernel<X, Y>), dim3(persistent_groups(p->rows, 1, kLong)),
                                           dim3(kLong), 0, s, (const X *)x, (const Y *)dy, weight, f32, cols, p->rows, mean,
                                           rstd, p->x_stride, p->dy_stride, (X *)dx);
                    if (part)
                        hipLaunchKernelGGL((layer_norm_slices_kernel<X, Y>), dim3((cols + kThreads * kSliceColumns - 1) / (kThreads * kSliceColumns), count),
                                           dim3(kThreads), 0, s, (const X *)x, (const Y *)dy, mean, rstd, p->rows, cols,
                                           p->x_stride, p->dy_stride, part);
                }
                return launch_status();
            });
        });
        if (st) return st;
    }
    if (!params) return SV3D_OK;
    const dim3 grid((cols + 15) / 16, 2);
    if (p->param_type == SV3D_F32)
        hipLaunchKernelGGL(layer_norm_join_kernel<float>, grid, dim3(1024), 0, s, part, count, cols, (float *)dweight, (float *)dbias);
    else if (p->param_type == SV3D_F16)
        hipLaunchKernelGGL(layer_norm_join_kernel<f16>, grid, dim3(1024), 0, s, part, count, cols, (f16 *)dweight, (f16 *)dbias);
    else
        hipLaunchKernelGGL(layer_norm_join_kernel<bf16>, grid, dim3(1024), 0, s, part, count, cols, (bf16 *)dweight, (bf16 *)dbias);
    return launch_status();
}
