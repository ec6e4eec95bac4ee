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
// and global memory takes 8- and 16-byte accesses at any address.
template <class T, int N>
struct TfcPack {
    T e[N];
};
template <class T, int N>
__device__ __forceinline__ TfcPack<T, N> tfc_load(const T* p) {
    TfcPack<T, N> r;
    __builtin_memcpy(&r, p, sizeof(r));
    return r;
}
template <class T, int N>
__device__ __forceinline__ void tfc_store(T* p, const TfcPack<T, N>& v) {
    __builtin_memcpy(p, &v, sizeof(v));
}

// N elements as floats, those at or behind `left` as zeros / not written (left >= N: one access).
template <class T, int N>
__device__ __forceinline__ void tfc_load_f(const T* p, long left, float (&v)[N]) {
    if (left >= N) {
        const TfcPack<T, N> r = tfc_load<T, N>(p);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (float)r.e[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < left ? (float)p[i] : 0.f;
    }
}
template <class T, int N>
__device__ __forceinline__ void tfc_store_f(T* p, long left, const float (&v)[N]) {
    if (left >= N) {
        TfcPack<T, N> r;
#pragma unroll
        for (int i = 0; i < N; ++i) r.e[i] = (T)v[i];
        tfc_store<T, N>(p, r);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < left) p[i] = (T)v[i];
    }
}

// a[c] = sum over p of part[p][c] for c < na, b[c - na] for the nb columns behind them, in a fixed order (tfc_norm.hip): the join of
// per-workgroup column sums.  a, b may be null.
int tfc_join_columns(const float* part, int64_t n_part, int64_t na, void* a, int64_t nb, void* b, int dtype, hipStream_t stream);
