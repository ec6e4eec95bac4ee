// Element types of the kernels that take more than fp32, and the vector accesses they share.
#pragma once

#include "tfc_common.h"

typedef __bf16 tfc_bf16;
typedef _Float16 tfc_f16;

template <class T>
struct TfcType;
template <>
struct TfcType<float> {
    static constexpr int V = 4;  // elements of a 16-byte access
};
template <>
struct TfcType<tfc_bf16> {
    static constexpr int V = 8;
};
template <>
struct TfcType<tfc_f16> {
    static constexpr int V = 8;
};

inline size_t tfc_dtype_size(int dtype) { return dtype == TFC_F32 ? 4 : 2; }
inline bool tfc_dtype_ok(int dtype) { return dtype == TFC_F32 || dtype == TFC_BF16 || dtype == TFC_F16; }

// Calls F<T>(args) with the type a TFC_* dtype code names (checked before).
#define TFC_BY_DTYPE(dtype, F, ...)                                                          \
    ((dtype) == TFC_F32 ? F<float>(__VA_ARGS__) : (dtype) == TFC_BF16 ? F<tfc_bf16>(__VA_ARGS__) : F<tfc_f16>(__VA_ARGS__))

// N elements at a pointer that is aligned to ONE element only: rows of odd width and views into flat buffers start anywhere,
// and global memory takes 8- and 16-byte accesses at any address.  They are held as whole words until they are used: an access
// whose elements are named apart is taken apart by the compiler too, into narrower ones with a wait in every branch.
typedef unsigned tfc_u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned tfc_u32x2 __attribute__((ext_vector_type(2)));
template <int BYTES>
struct TfcWords;
template <>
struct TfcWords<32> {
    typedef unsigned type __attribute__((ext_vector_type(8)));
};
template <>
struct TfcWords<16> {
    typedef tfc_u32x4 type;
};
template <>
struct TfcWords<8> {
    typedef tfc_u32x2 type;
};
template <>
struct TfcWords<4> {
    typedef uint32_t type;
};
template <>
struct TfcWords<2> {
    typedef uint16_t type;
};
template <class T, int N>
using TfcRaw = typename TfcWords<N * (int)sizeof(T)>::type;

template <class T, int N>
__device__ __forceinline__ TfcRaw<T, N> tfc_load(const T* p) {
    TfcRaw<T, N> r;
    __builtin_memcpy(&r, p, sizeof(r));
    return r;
}
template <class T, int N>
__device__ __forceinline__ void tfc_store(T* p, TfcRaw<T, N> v) {
    __builtin_memcpy(p, &v, sizeof(v));
}
template <class T, int N>
__device__ __forceinline__ void tfc_unpack(TfcRaw<T, N> r, float (&v)[N]) {
    T e[N];
    __builtin_memcpy(e, &r, sizeof(r));
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float)e[i];
}
template <class T, int N>
__device__ __forceinline__ TfcRaw<T, N> tfc_pack(const float (&v)[N]) {
    T e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = (T)v[i];
    TfcRaw<T, N> r;
    __builtin_memcpy(&r, e, sizeof(r));
    return r;
}

// The same with `left` elements up to the end of the row: those at or behind it are zeros / not written.
template <class T, int N>
__device__ __forceinline__ TfcRaw<T, N> tfc_load_left(const T* p, long left) {
    TfcRaw<T, N> r = {};
    if (left >= N) {
        r = tfc_load<T, N>(p);
    } else if (left > 0) {
        T e[N];
#pragma unroll
        for (int i = 0; i < N; ++i) e[i] = i < left ? p[i] : (T)0.f;
        __builtin_memcpy(&r, e, sizeof(r));
    }
    return r;
}
template <class T, int N>
__device__ __forceinline__ void tfc_load_f(const T* p, long left, float (&v)[N]) {
    tfc_unpack<T, N>(tfc_load_left<T, N>(p, left), v);
}
template <class T, int N>
__device__ __forceinline__ void tfc_store_f(T* p, long left, const float (&v)[N]) {
    if (left >= N) {
        tfc_store<T, N>(p, tfc_pack<T, N>(v));
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < left) p[i] = (T)v[i];
    }
}

// a[c] = sum over p of part[p][c] for c < na, b[c - na] for the nb columns behind them, in a fixed order (tfc_norm.hip): the join of
// per-workgroup column sums.  a, b may be null.
int tfc_join_columns(const float* part, int64_t n_part, int64_t na, void* a, int64_t nb, void* b, int dtype, hipStream_t stream);
