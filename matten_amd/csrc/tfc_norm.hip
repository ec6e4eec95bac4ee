// Layer norm over the last axis: y = (x - mean) rstd w + b with mean = sum x / d, rstd = (sum (x - mean)^2 / d + eps)^-1/2, and
// its backward pass with the reduction of the weights' gradients.  No counterpart in the reference's two target models; it is
// the normalisation of the scalar head (nn/mlp.py).
//
// Both passes are bound by HBM: a row is read once into registers, its statistics are formed there (two sums over centred
// values, so no cancellation), and the result is written from there.  A row belongs to G lanes - 8 to 64 of a wave for short
// rows, so that no lane idles at d = 32, or a whole workgroup - each holding NV vectors of 16 bytes.  Lanes keep their
// columns of w and b in registers over all rows they visit.  The backward pass also keeps the column sums of dw and db there:
// a fixed number of workgroups walks the rows and writes one partial row each; tfc_join_columns adds them in a fixed order.
// Measured: 65536 x 1024 in bf16 46 us forward (5.8 TB/s, some of it from the last-level cache), 79 + 4 backward (5.1 TB/s); 6911 x
// 1001 in fp32 (rows that start anywhere) 11.4 and 17.4 + 4.8 (4.8 TB/s); 2048 x 64 3.7 and 5.0 + 2.2, launches.
#include "tfc_types.h"

#include <algorithm>

namespace {

constexpr int NORM_MAX_PARTIALS = 1024;

// Sums of two values over the G lanes of a row (G a power of two <= 64, or the whole workgroup of G threads).
template <int G>
__device__ __forceinline__ void row_sums(float& a, float& b, float* lds) {
    if constexpr (G < 64) {
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) {
            a += __shfl_xor(a, o);
            b += __shfl_xor(b, o);
        }
    } else {
        a = tfc_wave_sum(a);
        b = tfc_wave_sum(b);
        if constexpr (G > 64) {
            constexpr int W = G / 64;
            const int wave = threadIdx.x >> 6;
            __syncthreads();  // the sums before these have been read
            if ((threadIdx.x & 63) == 0) {
                lds[wave] = a;
                lds[W + wave] = b;
            }
            __syncthreads();
            a = b = 0.f;
#pragma unroll
            for (int i = 0; i < W; ++i) {
                a += lds[i];
                b += lds[W + i];
            }
        }
    }
}

constexpr int norm_threads(int g) { return g > 256 ? g : 256; }

template <class T, int G, int NV>
struct NormShape {
    static constexpr int V = TfcType<T>::V;
    static constexpr int THREADS = norm_threads(G);
    static constexpr int ROWS = THREADS / G;  // rows a workgroup has in hand
};

template <class T, int G, int NV>
__global__ __launch_bounds__(norm_threads(G)) void tfc_layer_norm_fwd_kernel(
    const T* __restrict__ x, const T* __restrict__ w, const T* __restrict__ b, long rows, int d, float eps,
    T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
    using S = NormShape<T, G, NV>;
    constexpr int V = S::V;
    __shared__ float lds[2 * (S::THREADS / 64)];
    const int lane = threadIdx.x % G, slot = threadIdx.x / G;
    float wv[NV][V], bv[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * G + lane) * V;
#pragma unroll
        for (int j = 0; j < V; ++j) wv[i][j] = 1.f, bv[i][j] = 0.f;
        if (w && c < d) tfc_load_f<T, V>(w + c, d - c, wv[i]);
        if (b && c < d) tfc_load_f<T, V>(b + c, d - c, bv[i]);
    }
    const float fd = (float)d;  // (divided by, not multiplied with its rounded inverse: a row without spread centres to zeros)
    for (long r0 = (long)blockIdx.x * S::ROWS; r0 < rows; r0 += (long)gridDim.x * S::ROWS) {
        const long r = r0 + slot;
        const bool live = r < rows;  // (a row's lanes agree; the others keep step for the barriers)
        const T* xr = x + (live ? r : 0) * (long)d;
        float v[NV][V];
        float s = 0.f, q = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + lane) * V;
            tfc_load_f<T, V>(xr + c, live ? (long)d - c : 0, v[i]);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) s += v[i][j];
        row_sums<G>(s, q, lds);
        const float mu = s / fd;
        s = q = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + lane) * V;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[i][j] = c + j < d ? v[i][j] - mu : 0.f;
                s += v[i][j] * v[i][j];
            }
        }
        row_sums<G>(s, q, lds);
        const float rs = 1.f / sqrtf(s / fd + eps);
        if (live) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * G + lane) * V;
#pragma unroll
                for (int j = 0; j < V; ++j) v[i][j] = v[i][j] * rs * wv[i][j] + bv[i][j];
                if (c < d) tfc_store_f<T, V>(y + r * (long)d + c, (long)d - c, v[i]);
            }
            if (lane == 0 && mean) {
                mean[r] = mu;
                rstd[r] = rs;
            }
        }
    }
}

// With h = (x - mean) rstd and u = dy w:  dx = rstd (u - sum(u)/d - h sum(u h)/d),  dw = sum_rows dy h,  db = sum_rows dy.
template <class T, int G, int NV, bool PART>
__global__ __launch_bounds__(norm_threads(G)) void tfc_layer_norm_bwd_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, const T* __restrict__ w, const float* __restrict__ mean,
    const float* __restrict__ rstd, long rows, int d, T* __restrict__ dx, float* __restrict__ part) {
    using S = NormShape<T, G, NV>;
    constexpr int V = S::V;
    __shared__ float lds[G <= 64 ? 2 * 64 * NV * V : 2 * (S::THREADS / 64)];
    const int lane = threadIdx.x % G, slot = threadIdx.x / G;
    float wv[NV][V], gw[NV][V], gb[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * G + lane) * V;
#pragma unroll
        for (int j = 0; j < V; ++j) wv[i][j] = 1.f, gw[i][j] = 0.f, gb[i][j] = 0.f;
        if (w && c < d) tfc_load_f<T, V>(w + c, d - c, wv[i]);
    }
    const float fd = (float)d;
    for (long r0 = (long)blockIdx.x * S::ROWS; r0 < rows; r0 += (long)gridDim.x * S::ROWS) {
        const long r = r0 + slot;
        const bool live = r < rows;
        const long at = (live ? r : 0) * (long)d;
        const float mu = live ? mean[r] : 0.f, rs = live ? rstd[r] : 0.f;
        float h[NV][V], g[NV][V];
        float s = 0.f, q = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + lane) * V;
            tfc_load_f<T, V>(x + at + c, live ? (long)d - c : 0, h[i]);
            tfc_load_f<T, V>(dy + at + c, live ? (long)d - c : 0, g[i]);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * G + lane) * V;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                h[i][j] = live && c + j < d ? (h[i][j] - mu) * rs : 0.f;
                if (PART) {
                    gw[i][j] += g[i][j] * h[i][j];
                    gb[i][j] += g[i][j];
                }
                g[i][j] *= wv[i][j];
                s += g[i][j];
                q += g[i][j] * h[i][j];
            }
        }
        if (!dx) continue;
        row_sums<G>(s, q, lds);
        s /= fd;
        q /= fd;
        if (live) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * G + lane) * V;
#pragma unroll
                for (int j = 0; j < V; ++j) g[i][j] = rs * (g[i][j] - s - h[i][j] * q);
                if (c < d) tfc_store_f<T, V>(dx + r * (long)d + c, (long)d - c, g[i]);
            }
        }
    }
    if constexpr (PART) {
        float* pw = part + (long)blockIdx.x * 2 * d;
        if constexpr (G <= 64) {
            // rows side by side in a wave first, then the workgroup's waves one after the other through LDS
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j)
#pragma unroll
                    for (int o = G; o < 64; o <<= 1) {
                        gw[i][j] += __shfl_xor(gw[i][j], o);
                        gb[i][j] += __shfl_xor(gb[i][j], o);
                    }
            for (int k = 0; k < S::THREADS / 64; ++k) {
                if ((int)(threadIdx.x >> 6) == k && (threadIdx.x & 63) < G) {
#pragma unroll
                    for (int i = 0; i < NV; ++i)
#pragma unroll
                        for (int j = 0; j < V; ++j) {
                            const int c = (i * V + j) * G + lane;  // (transposed: neighbouring lanes, neighbouring banks)
                            lds[c] = k ? lds[c] + gw[i][j] : gw[i][j];
                            lds[G * NV * V + c] = k ? lds[G * NV * V + c] + gb[i][j] : gb[i][j];
                        }
                }
                __syncthreads();
            }
            for (int c = threadIdx.x; c < d; c += S::THREADS) {
                const int vec = c / V, i = vec / G, l = vec - i * G, j = c - vec * V;
                pw[c] = lds[(i * V + j) * G + l];
                pw[d + c] = lds[G * NV * V + (i * V + j) * G + l];
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const int c = (i * G + lane) * V + j;
                    if (c < d) {
                        pw[c] = gw[i][j];
                        pw[d + c] = gb[i][j];
                    }
                }
        }
    }
}

// Rows too long for the registers of a workgroup: the row is walked again for every sum (it is in the caches by then).
template <class T>
__global__ __launch_bounds__(1024) void tfc_layer_norm_long_fwd_kernel(
    const T* __restrict__ x, const T* __restrict__ w, const T* __restrict__ b, long rows, long d, float eps,
    T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd) {
    __shared__ float lds[32];
    for (long r = blockIdx.x; r < rows; r += gridDim.x) {
        const T* xr = x + r * d;
        float s = 0.f, q = 0.f;
        for (long c = threadIdx.x; c < d; c += 1024) s += (float)xr[c];
        row_sums<1024>(s, q, lds);
        const float mu = s / (float)d;
        s = q = 0.f;
        for (long c = threadIdx.x; c < d; c += 1024) {
            const float v = (float)xr[c] - mu;
            s += v * v;
        }
        row_sums<1024>(s, q, lds);
        const float rs = 1.f / sqrtf(s / (float)d + eps);
        for (long c = threadIdx.x; c < d; c += 1024)
            y[r * d + c] = (T)(((float)xr[c] - mu) * rs * (w ? (float)w[c] : 1.f) + (b ? (float)b[c] : 0.f));
        if (threadIdx.x == 0 && mean) {
            mean[r] = mu;
            rstd[r] = rs;
        }
    }
}

template <class T>
__global__ __launch_bounds__(1024) void tfc_layer_norm_long_bwd_kernel(
    const T* __restrict__ dy, const T* __restrict__ x, const T* __restrict__ w, const float* __restrict__ mean,
    const float* __restrict__ rstd, long rows, long d, T* __restrict__ dx) {
    __shared__ float lds[32];
    for (long r = blockIdx.x; r < rows; r += gridDim.x) {
        const float mu = mean[r], rs = rstd[r];
        float s = 0.f, q = 0.f;
        for (long c = threadIdx.x; c < d; c += 1024) {
            const float u = (float)dy[r * d + c] * (w ? (float)w[c] : 1.f);
            s += u;
            q += u * ((float)x[r * d + c] - mu) * rs;
        }
        row_sums<1024>(s, q, lds);
        s /= (float)d;
        q /= (float)d;
        for (long c = threadIdx.x; c < d; c += 1024) {
            const float u = (float)dy[r * d + c] * (w ? (float)w[c] : 1.f);
            dx[r * d + c] = (T)(rs * (u - s - ((float)x[r * d + c] - mu) * rs * q));
        }
    }
}

// Column sums for the long rows: a thread owns a column of one slab of rows.
template <class T>
__global__ __launch_bounds__(256) void tfc_layer_norm_long_cols_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                                       const float* __restrict__ mean,
                                                                       const float* __restrict__ rstd, long rows, long d,
                                                                       long slab, float* __restrict__ part) {
    const long c = (long)blockIdx.x * 256 + threadIdx.x;
    if (c >= d) return;
    const long r0 = (long)blockIdx.y * slab, r1 = r0 + slab < rows ? r0 + slab : rows;
    float gw = 0.f, gb = 0.f;
    for (long r = r0; r < r1; ++r) {
        const float g = (float)dy[r * d + c];
        gw += g * ((float)x[r * d + c] - mean[r]) * rstd[r];
        gb += g;
    }
    part[(long)blockIdx.y * 2 * d + c] = gw;
    part[(long)blockIdx.y * 2 * d + d + c] = gb;
}

// 32 columns x 32 walkers; walker k adds the partial rows k, k + 32, ..., the walkers are joined in order.
// Columns [0, na) go to `a`, the others to `b` (either null: not written).
template <class T>
__global__ __launch_bounds__(1024) void tfc_join_columns_kernel(const float* __restrict__ part, long n_part, long stride, long n,
                                                                long na, T* __restrict__ out_a, T* __restrict__ out_b) {
    __shared__ float lds[32][33];
    const int cl = threadIdx.x & 31, k = threadIdx.x >> 5;
    const long c = (long)blockIdx.x * 32 + cl;
    float s = 0.f;
    if (c < n) {
        long p = k;
        for (; p + 96 < n_part; p += 128) {
            const float a = part[p * stride + c], b = part[(p + 32) * stride + c];
            const float e = part[(p + 64) * stride + c], f = part[(p + 96) * stride + c];
            s += (a + b) + (e + f);
        }
        for (; p < n_part; p += 32) s += part[p * stride + c];
    }
    lds[k][cl] = s;
    __syncthreads();
    if (k == 0 && c < n) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) t += lds[i][cl];
        if (c < na) {
            if (out_a) out_a[c] = (T)t;
        } else if (out_b) {
            out_b[c - na] = (T)t;
        }
    }
}

template <class T>
int join_columns(const float* part, int64_t n_part, int64_t na, void* out_a, int64_t nb, void* out_b, hipStream_t stream) {
    TfcProfScope prof("tfc_join_columns", stream);
    const int64_t n = na + nb;
    hipLaunchKernelGGL(tfc_join_columns_kernel<T>, dim3((unsigned)((n + 31) / 32)), dim3(1024), 0, stream, part, (long)n_part,
                       (long)n, (long)n, (long)na, (T*)out_a, (T*)out_b);
    TFC_LAUNCH_CHECK("tfc_join_columns");
    return TFC_OK;
}

struct NormArgs {
    const void *x, *w, *b, *dy;
    int64_t rows, d;
    float eps;
    void *y, *dx;
    float *mean, *rstd, *part;
    int64_t n_part;
    hipStream_t stream;
};

// Workgroups of the backward pass: each leaves one partial row, so no more than are needed to fill the chip, and each is
// given a few rows.
int64_t norm_partials(int64_t rows, int64_t rows_per_group) {
    const int64_t groups = (rows + rows_per_group - 1) / rows_per_group;
    return std::max<int64_t>(1, std::min<int64_t>((groups + 1) / 2, NORM_MAX_PARTIALS));
}

template <class T, int G, int NV>
int norm_fwd(const NormArgs& a) {
    using S = NormShape<T, G, NV>;
    const int64_t groups = (a.rows + S::ROWS - 1) / S::ROWS;
    hipLaunchKernelGGL((tfc_layer_norm_fwd_kernel<T, G, NV>), dim3((unsigned)std::min<int64_t>(groups, 4096)), dim3(S::THREADS), 0,
                       a.stream, (const T*)a.x, (const T*)a.w, (const T*)a.b, (long)a.rows, (int)a.d, a.eps, (T*)a.y, a.mean,
                       a.rstd);
    TFC_LAUNCH_CHECK("tfc_layer_norm_fwd");
    return TFC_OK;
}

template <class T, int G, int NV>
int norm_bwd(const NormArgs& a) {
    using S = NormShape<T, G, NV>;
    const int64_t groups = (a.rows + S::ROWS - 1) / S::ROWS;
    if (a.part)
        hipLaunchKernelGGL((tfc_layer_norm_bwd_kernel<T, G, NV, true>), dim3((unsigned)a.n_part), dim3(S::THREADS), 0, a.stream,
                           (const T*)a.dy, (const T*)a.x, (const T*)a.w, a.mean, a.rstd, (long)a.rows, (int)a.d, (T*)a.dx, a.part);
    else
        hipLaunchKernelGGL((tfc_layer_norm_bwd_kernel<T, G, NV, false>), dim3((unsigned)std::min<int64_t>(groups, 4096)),
                           dim3(S::THREADS), 0, a.stream, (const T*)a.dy, (const T*)a.x, (const T*)a.w, a.mean, a.rstd,
                           (long)a.rows, (int)a.d, (T*)a.dx, (float*)nullptr);
    TFC_LAUNCH_CHECK("tfc_layer_norm_bwd");
    return TFC_OK;
}

// Lanes and vectors by the row's length in vectors: the fewest lanes that hold the row in 16 registers each (NV <= 4 vectors of
// fp32, 2 of 16 bits: the backward pass keeps five such sets), a workgroup's only where a wave's do not.
template <class T, template <class, int, int> class F>
int norm_by_width(const NormArgs& a) {
    const int64_t nv = (a.d + TfcType<T>::V - 1) / TfcType<T>::V;
    if (nv <= 8) return F<T, 8, 1>::run(a);
    if (nv <= 16) return F<T, 16, 1>::run(a);
    if (nv <= 32) return F<T, 32, 1>::run(a);
    if (nv <= 64) return F<T, 64, 1>::run(a);
    if (nv <= 128) return F<T, 64, 2>::run(a);
    if constexpr (TfcType<T>::V == 4) {
        if (nv <= 256) return F<T, 64, 4>::run(a);
        if (nv <= 512) return F<T, 256, 2>::run(a);
        if (nv <= 1024) return F<T, 256, 4>::run(a);
        if (nv <= 2048) return F<T, 1024, 2>::run(a);
        return F<T, 1024, 4>::run(a);
    } else {
        if (nv <= 512) return F<T, 256, 2>::run(a);
        return F<T, 1024, 2>::run(a);
    }
}
constexpr int64_t NORM_MAX_D = 16384;

template <class T, int G, int NV>
struct Fwd {
    static int run(const NormArgs& a) { return norm_fwd<T, G, NV>(a); }
};
template <class T, int G, int NV>
struct Bwd {
    static int run(const NormArgs& a) { return norm_bwd<T, G, NV>(a); }
};

// Rows a workgroup of the backward pass has in hand (NormShape::ROWS of the shape norm_by_width takes).
int rows_per_group(int64_t d, int dtype) {
    const int64_t v = dtype == TFC_F32 ? 4 : 8, nv = (d + v - 1) / v;
    return nv <= 8 ? 32 : nv <= 16 ? 16 : nv <= 32 ? 8 : nv * v <= 1024 ? 4 : 1;
}

bool norm_long(int64_t d) { return d > NORM_MAX_D; }

int64_t long_slab(int64_t rows) { return std::max<int64_t>(1, (rows + 63) / 64); }

template <class T>
int layer_norm_fwd(const NormArgs& a) {
    if (!norm_long(a.d)) return norm_by_width<T, Fwd>(a);
    hipLaunchKernelGGL(tfc_layer_norm_long_fwd_kernel<T>, dim3((unsigned)std::min<int64_t>(a.rows, 2048)), dim3(1024), 0, a.stream,
                       (const T*)a.x, (const T*)a.w, (const T*)a.b, (long)a.rows, (long)a.d, a.eps, (T*)a.y, a.mean, a.rstd);
    TFC_LAUNCH_CHECK("tfc_layer_norm_long_fwd");
    return TFC_OK;
}

template <class T>
int layer_norm_bwd(const NormArgs& a) {
    if (!norm_long(a.d)) return norm_by_width<T, Bwd>(a);
    if (a.dx) {
        hipLaunchKernelGGL(tfc_layer_norm_long_bwd_kernel<T>, dim3((unsigned)std::min<int64_t>(a.rows, 2048)), dim3(1024), 0,
                           a.stream, (const T*)a.dy, (const T*)a.x, (const T*)a.w, a.mean, a.rstd, (long)a.rows, (long)a.d,
                           (T*)a.dx);
        TFC_LAUNCH_CHECK("tfc_layer_norm_long_bwd");
    }
    if (a.part) {
        hipLaunchKernelGGL(tfc_layer_norm_long_cols_kernel<T>, dim3((unsigned)((a.d + 255) / 256), (unsigned)a.n_part), dim3(256), 0,
                           a.stream, (const T*)a.dy, (const T*)a.x, a.mean, a.rstd, (long)a.rows, (long)a.d, (long)long_slab(a.rows),
                           a.part);
        TFC_LAUNCH_CHECK("tfc_layer_norm_long_cols");
    }
    return TFC_OK;
}

int64_t partial_rows(int64_t rows, int64_t d, int dtype) {
    if (norm_long(d)) return (rows + long_slab(rows) - 1) / long_slab(rows);
    return norm_partials(rows, rows_per_group(d, dtype));
}

}  // namespace

int tfc_join_columns(const float* part, int64_t n_part, int64_t na, void* out_a, int64_t nb, void* out_b, int dtype,
                     hipStream_t stream) {
    return TFC_BY_DTYPE(dtype, join_columns, part, n_part, na, out_a, nb, out_b, stream);
}

extern "C" int tfc_layer_norm_fwd(const void* x, const void* w, const void* b, int64_t rows, int64_t d, float eps, int32_t dtype,
                                  void* y, float* mean, float* rstd, tfc_stream_t stream) {
    TFC_REQUIRE(tfc_dtype_ok(dtype), TFC_EINVAL, "tfc_layer_norm_fwd: unknown dtype %d", (int)dtype);
    TFC_REQUIRE(rows >= 0 && d > 0, TFC_EINVAL, "tfc_layer_norm_fwd: bad sizes %lld x %lld", (long long)rows, (long long)d);
    TFC_REQUIRE(eps >= 0.f, TFC_EINVAL, "tfc_layer_norm_fwd: eps must not be negative");
    if (rows == 0) return TFC_OK;
    TFC_REQUIRE(x && y && (!mean == !rstd), TFC_EINVAL, "tfc_layer_norm_fwd: null pointer");
    hipStream_t s = (hipStream_t)stream;
    TfcProfScope prof("tfc_layer_norm_fwd", s);
    NormArgs a{};
    a.x = x, a.w = w, a.b = b, a.rows = rows, a.d = d, a.eps = eps, a.y = y, a.mean = mean, a.rstd = rstd, a.stream = s;
    return TFC_BY_DTYPE(dtype, layer_norm_fwd, a);
}

extern "C" int64_t tfc_layer_norm_bwd_workspace_floats(int64_t rows, int64_t d, int32_t dtype) {
    if (rows <= 0 || d <= 0 || !tfc_dtype_ok(dtype)) return 0;
    return partial_rows(rows, d, dtype) * 2 * d;
}

extern "C" int tfc_layer_norm_bwd(const void* dy, const void* x, const void* w, const float* mean, const float* rstd, int64_t rows,
                                  int64_t d, int32_t dtype, void* dx, void* dw, void* db, float* workspace, int64_t workspace_floats,
                                  tfc_stream_t stream) {
    TFC_REQUIRE(tfc_dtype_ok(dtype), TFC_EINVAL, "tfc_layer_norm_bwd: unknown dtype %d", (int)dtype);
    TFC_REQUIRE(rows >= 0 && d > 0, TFC_EINVAL, "tfc_layer_norm_bwd: bad sizes %lld x %lld", (long long)rows, (long long)d);
    hipStream_t s = (hipStream_t)stream;
    if (rows == 0) return dw || db ? tfc_join_columns(nullptr, 0, d, dw, d, db, dtype, s) : TFC_OK;  // sums over no rows
    TFC_REQUIRE(dy && x && mean && rstd, TFC_EINVAL, "tfc_layer_norm_bwd: null pointer");
    if (!dx && !dw && !db) return TFC_OK;
    NormArgs a{};
    a.dy = dy, a.x = x, a.w = w, a.mean = const_cast<float*>(mean), a.rstd = const_cast<float*>(rstd);
    a.rows = rows, a.d = d, a.dx = dx, a.stream = s;
    if (dw || db) {
        a.n_part = partial_rows(rows, d, dtype);
        TFC_REQUIRE(workspace && workspace_floats >= a.n_part * 2 * d, TFC_EINVAL, "tfc_layer_norm_bwd: workspace too small");
        a.part = workspace;
    }
    {
        TfcProfScope prof("tfc_layer_norm_bwd", s);
        const int rc = TFC_BY_DTYPE(dtype, layer_norm_bwd, a);
        if (rc) return rc;
    }
    return a.part ? tfc_join_columns(workspace, a.n_part, d, dw, d, db, dtype, s) : TFC_OK;
}
