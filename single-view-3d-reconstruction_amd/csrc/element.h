// Element types of the layer norm and optimizer kernels: fp32 in registers, fp32 / fp16 / bf16 in memory.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "sv3d_hip.h"

namespace sv3d {

using f16 = _Float16;
using bf16 = __bf16;

// to_float is exact; from_float rounds to nearest even (at most half a step: 2^-11 of the value for fp16,
// 2^-8 for bf16)
template <class T>
__device__ inline float to_float(T v) { return (float)v; }
template <class T>
__device__ inline T from_float(float v) { return (T)v; }

// N consecutive elements, loaded and stored at once from any address that is a multiple of the element's size (global
// memory takes wide accesses at any alignment; rows of odd length start anywhere)
template <class T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
    T v[N];
};

// The same elements as the 32-bit words that they fill, for values that wait in registers: two of 16 bits in each, where a
// Pack that is put together from single elements would take a register for every one of them.
template <class T, int N>
struct Words {
    static constexpr int kCount = N * (int)sizeof(T) / 4;
    uint32_t w[kCount];
    __device__ inline uint32_t byte(int i) const { return w[i / 4] >> (i % 4 * 8) & 0xffu; }
    __device__ inline float operator[](int i) const
    {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        const uint32_t h = w[i / 2];
        if constexpr (__is_same(T, bf16)) return __uint_as_float(i & 1 ? h & 0xffff0000u : h << 16);
        return (float)__builtin_bit_cast(f16, (uint16_t)(i & 1 ? h >> 16 : h & 0xffffu));
    }
};

template <int BYTES> struct Bits;
template <> struct Bits<1> { using type = uint8_t; };
template <> struct Bits<2> { using type = uint16_t; };
template <> struct Bits<4> { using type = uint32_t; };

// all of them
template <class T, int N>
__device__ inline Words<T, N> load_words(const T *p)
{
    Words<T, N> r;
    const auto q = *reinterpret_cast<const Pack<T, N> *>(p);
    __builtin_memcpy(r.w, q.v, sizeof(r.w));
    return r;
}

template <class T, int N>
__device__ inline void store_words(T *p, const Words<T, N> &r)
{
    Pack<T, N> q;
    __builtin_memcpy(q.v, r.w, sizeof(r.w));
    *reinterpret_cast<Pack<T, N> *>(p) = q;
}

// the same past the caches, for what nobody reads again soon
template <class T, int N>
__device__ inline Words<T, N> stream_words(const T *p)
{
    using V = uint32_t __attribute__((ext_vector_type(Words<T, N>::kCount), aligned(sizeof(T))));
    const V q = __builtin_nontemporal_load(reinterpret_cast<const V *>(p));
    Words<T, N> r;
    __builtin_memcpy(r.w, &q, sizeof(r.w));
    return r;
}

template <class T, int N>
__device__ inline void stream_words(T *p, const Words<T, N> &r)
{
    using V = uint32_t __attribute__((ext_vector_type(Words<T, N>::kCount), aligned(sizeof(T))));
    V q;
    __builtin_memcpy(&q, r.w, sizeof(r.w));
    __builtin_nontemporal_store(q, reinterpret_cast<V *>(p));
}

// `n` of the elements exist (n <= 0: none), the others are zero.  Without ENDS it is all or none of them.
template <class T, int N, bool ENDS = true, bool STREAM = false>
__device__ inline Words<T, N> load_words(const T *p, int n)
{
    if constexpr (!ENDS) {
        Words<T, N> r = {};
        if (n > 0) r = STREAM ? stream_words<T, N>(p) : load_words<T, N>(p);
        return r;
    }
    if (n >= N) return STREAM ? stream_words<T, N>(p) : load_words<T, N>(p);
    Words<T, N> r = {};
    if (n <= 0) return r;
    constexpr int kBytes = (int)sizeof(T);
#pragma unroll
    for (int j = 0; j < N; ++j)
        if (j < n)
            r.w[j * kBytes / 4] |= (uint32_t) reinterpret_cast<const typename Bits<kBytes>::type *>(p)[j] << (j * kBytes % 4 * 8);
    return r;
}

// Drops the lowest `off` elements, zeros come in at the top.
template <class T, int N>
__device__ inline void drop_words(Words<T, N> &r, int off)
{
    constexpr int C = Words<T, N>::kCount;
    const int bytes = off * (int)sizeof(T);
#pragma unroll
    for (int step = C / 2; step > 0; step /= 2)
        if (bytes & (4 * step)) {
#pragma unroll
            for (int i = 0; i < C; ++i) r.w[i] = i + step < C ? r.w[i + step] : 0u;
        }
    if (sizeof(T) == 2 && (bytes & 2)) {
#pragma unroll
        for (int i = 0; i < C; ++i) r.w[i] = r.w[i] >> 16 | (i + 1 < C ? r.w[i + 1] << 16 : 0u);
    }
}

// the first n of the elements, all of them at once where they are there
template <class T, int N, bool ENDS = true, bool STREAM = false>
__device__ inline void store_words(T *p, const Words<T, N> &r, int n)
{
    if (!ENDS && n <= 0) return;
    if (!ENDS || n >= N) return STREAM ? stream_words<T, N>(p, r) : store_words<T, N>(p, r);
    using B = typename Bits<(int)sizeof(T)>::type;
    constexpr int kBytes = (int)sizeof(T);
#pragma unroll
    for (int j = 0; j < N; ++j)
        if (j < n) reinterpret_cast<B *>(p)[j] = (B)(r.w[j * kBytes / 4] >> (j * kBytes % 4 * 8));
}

template <class T, int V>
__device__ inline Words<T, V> to_words(const float *v)
{
    Pack<T, V> r;
#pragma unroll
    for (int j = 0; j < V; ++j) r.v[j] = from_float<T>(v[j]);
    Words<T, V> w;
    __builtin_memcpy(w.w, r.v, sizeof(w.w));
    return w;
}

template <class T, int V, bool ENDS = true, bool STREAM = false>
__device__ inline void store_pack(T *p, const float *v, int n) { store_words<T, V, ENDS, STREAM>(p, to_words<T, V>(v), n); }

// ---- sums over the lanes of a wave ----------------------------------------------------------------
// Every one of G neighbouring lanes gets the sum of their values, added in an order that G fixes.
template <int CTRL>
__device__ inline float dpp(float v)
{
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xf, 0xf, true));
}

__device__ inline float swap16_sum(float v)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ inline float swap32_sum(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <int G>
__device__ inline float lane_sum(float v)
{
    static_assert(G == 8 || G == 16 || G == 32 || G == 64, "lanes of one group");
    v += dpp<0xB1>(v);                      // lane ^ 1
    v += dpp<0x4E>(v);                      // lane ^ 2
    v += dpp<0x141>(v);                     // 7 - lane in each eight: the other four
    if (G >= 16) v += dpp<0x140>(v);        // 15 - lane in each sixteen: the other eight
    if (G >= 32) v = swap16_sum(v);
    if (G >= 64) v = swap32_sum(v);
    return v;
}

inline bool known_type(int32_t t) { return t == SV3D_F32 || t == SV3D_F16 || t == SV3D_BF16; }
inline int type_bytes(int32_t t) { return t == SV3D_F32 ? 4 : 2; }
inline bool aligned(const void *p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

inline int launch_status() { return hipGetLastError() == hipSuccess ? SV3D_OK : SV3D_ERR_LAUNCH; }

}  // namespace sv3d
