// The backward pass of a dense layer of at most 64 x 64 (the hidden layers of the radial network and of small heads) in one kernel.
//
//   z = alpha x W + bias,  dz = act'(z) dy,  dx = alpha cst dz W^T,  dW = alpha cst x^T dz,  db = cst (column sums of dz)
//
// Such a layer has so few products for each row that three kernels, with z and dz in memory between them, are bound by HBM several
// times over (200000 rows of fp32: dz 28, dx 34, dW 24 + 7 us on top of 13 us for writing z).  Here a workgroup walks tiles of 64
// rows: x and dy are read once, z is formed again from x and the weights that stay in LDS, dz goes from the accumulators to
// LDS, dx = dz W^T goes out, and x^T dz stays in the accumulators over all tiles; one partial result a workgroup, joined in a
// fixed order (tfc_join_columns).  The next tile's x and dy are in flight meanwhile.  200000 rows of fp32: 59 + 4 us for 154 MB, which
// a copy moves in 32; what is left is the six piece products of three products, 26 us of the matrix units, and the cuts into pieces
// between them.
//
// LDS holds x, dz and W as [64][64] images of 16-bit elements (fp32: three of them, the bf16 pieces; dz of 16-bit types: two pieces, which
// costs nothing here and makes the gradients as good as their own rounding), 16-byte units swizzled by
// the row, so that both ways of reading are served by one image: eight neighbours of a row in one access, or four rows of a
// column by the transposing read.  fp32: 72 KB, two workgroups on a CU.
#include "tfc_dense_act.h"

#include <algorithm>

namespace {

constexpr int S = TFC_NARROW;
constexpr int IMAGE = S * S;

struct Narrow {
    long m;
    int n, k;
    const void *x, *w, *bias, *dy;
    long ldx;
    int wk, wn;  // strides of the weight along k and n
    void* dx;
    float* part;  // [workgroups][k n + n], the weight's gradient in the weight's own order
    int pk, pn;   // its strides
    float alpha, cst, factor;  // factor = alpha cst, for 16 bits / TFC_DZ_SCALE: what dz lacks in the images
    int act;
    int want_dw;
};

// Element index of (row, col) in an image; col a multiple of 4 is the start of half a unit.  The swizzle is row / 2 % 8 with its bits
// reversed: eight rows of one parity (which share 128 of the banks' 256 bytes) differ, so that 16 rows of one unit meet all banks, and two
// such neighbours differ in the upper bit, so that four rows of four units do.
__device__ __forceinline__ int at(int row, int col) {
    const int swizzle = (row << 1 & 4) | (row >> 1 & 2) | (row >> 3 & 1);
    return row * S + (((col >> 3) ^ swizzle) << 3) + (col & 7);
}

// Fragment whose lane l holds row r0 + l % 32, eight columns from c0 + 8 (l / 32) on.
__device__ __forceinline__ uintx4 frag_row(const uint16_t* im, int r0, int c0) {
    const int lane = threadIdx.x & 63;
    return *(const uintx4*)(im + at(r0 + (lane & 31), c0 + (lane >> 5) * 8));
}
// Fragment whose lane l holds COLUMN c0 + l % 32, eight rows from r0 + 8 (l / 32) on.
__device__ __forceinline__ uintx4 frag_col(const uint16_t* im, int c0, int r0) {
    const int lane = threadIdx.x & 63;
    const int row = r0 + (lane >> 5) * 8 + ((lane & 15) >> 2), col = c0 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
    typedef __attribute__((address_space(3))) shortx4* Lds;
    struct {
        shortx4 a, b;
    } both = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(im + at(row, col))),
              __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(im + at(row + 4, col)))};
    return __builtin_bit_cast(uintx4, both);
}

// Eight neighbours of a row into the image(s) of x or W; c a multiple of 8.
template <class T>
__device__ __forceinline__ void put8(uint16_t* im, int row, int c, const float (&v)[8]) {
    if constexpr (std::is_same<T, float>::value) {
        const Unit3 u = split8(v);
        *(uintx4*)(im + at(row, c)) = u.h;
        *(uintx4*)(im + IMAGE + at(row, c)) = u.m;
        *(uintx4*)(im + 2 * IMAGE + at(row, c)) = u.l;
    } else {
        *(uintx4*)(im + at(row, c)) = tfc_pack<T, 8>(v);
    }
}
// Four neighbours of a row into the images of dz; c a multiple of 4.
template <class T>
__device__ __forceinline__ void put4(uint16_t* im, int row, int c, const float (&v)[4]) {
    if constexpr (std::is_same<T, float>::value) {
        const float w[8] = {v[0], v[1], v[2], v[3], 0.f, 0.f, 0.f, 0.f};
        const Unit3 u = split8(w);
        *(tfc_u32x2*)(im + at(row, c)) = tfc_u32x2{u.h[0], u.h[1]};
        *(tfc_u32x2*)(im + IMAGE + at(row, c)) = tfc_u32x2{u.m[0], u.m[1]};
        *(tfc_u32x2*)(im + 2 * IMAGE + at(row, c)) = tfc_u32x2{u.l[0], u.l[1]};
    } else {
        *(tfc_u32x2*)(im + at(row, c)) = tfc_pack<T, 4>(v);
        float lo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) lo[j] = second_piece(T(), v[j]);
        *(tfc_u32x2*)(im + IMAGE + at(row, c)) = tfc_pack<T, 4>(lo);
    }
}

// acc += A^T-side fragments a[] times b[] (all piece products)
template <class T, int P>
__device__ __forceinline__ void terms(const uintx4 (&a)[P], const uintx4 (&b)[P], floatx16& acc) {
#pragma unroll
    for (int q = 0; q < (P == 3 ? 6 : 1); ++q) acc = mma(Mma<T>(), a[P == 3 ? TFC_TERM_B[q] : 0], b[P == 3 ? TFC_TERM_A[q] : 0], acc);
}

template <class T>
__global__ __launch_bounds__(256, 2) void tfc_dense_narrow_bwd_kernel(const Narrow g) {
    constexpr int P = Pieces<T>::N, D = P == 3 ? 3 : 2;  // pieces of x and W; of dz
    __shared__ __attribute__((aligned(16))) uint16_t lds[(2 * P + D) * IMAGE];
    uint16_t *wi = lds, *xi = lds + P * IMAGE, *di = lds + 2 * P * IMAGE;
    static_assert((P + D) * IMAGE * 2 >= S * S * 4, "dx passes through the images of x and dz");
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, half = lane >> 5;
    constexpr float LO = std::is_same<T, tfc_f16>::value ? 1.f / TFC_LO_SCALE : 1.f;
    const int r32 = (wave >> 1) * 32, c32 = (wave & 1) * 32;  // the wave's quarter of every 64 x 64 product
    // ---- weights, once: image [k][n]
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int row = t / 8 + 32 * i, c = (t % 8) * 8;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = row < g.k && c + j < g.n ? (float)((const T*)g.w)[(long)row * g.wk + (long)(c + j) * g.wn] : 0.f;
        put8<T>(wi, row, c, v);
    }
    float bias[16];
#pragma unroll
    for (int q = 0; q < 16; ++q) {
        const int n = c32 + (q >> 2) * 8 + half * 4 + (q & 3);
        bias[q] = g.bias && n < g.n ? (float)((const T*)g.bias)[n] : 0.f;
    }
    // ---- operands of a tile, in flight: x as two units of 8 a thread, dy as the accumulators of z lie
    TfcRaw<T, 8> rx[2];
    TfcRaw<T, 4> rd[4];
    auto ask = [&](long m0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const long row = m0 + t / 8 + 32 * i;
            const int c = (t % 8) * 8;
            rx[i] = tfc_load_left<T, 8>((const T*)g.x + row * g.ldx + c, row < g.m ? g.k - c : 0);
        }
        const long row = m0 + r32 + (lane & 31);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int c = c32 + 8 * q + half * 4;
            rd[q] = tfc_load_left<T, 4>((const T*)g.dy + row * g.n + c, row < g.m ? g.n - c : 0);
        }
    };
    floatx16 dw = floatx16(0.f), dw_lo = floatx16(0.f);  // (16 bits: products with the second pieces of dz apart)
    float db[16];
#pragma unroll
    for (int q = 0; q < 16; ++q) db[q] = 0.f;
    const long tiles = (g.m + S - 1) / S;
    ask((long)blockIdx.x * S);
    for (long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const long m0 = tile * S;
        __syncthreads();  // the images of the tile before have been read
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float v[8];
            tfc_unpack<T, 8>(rx[i], v);
            put8<T>(xi, t / 8 + 32 * i, (t % 8) * 8, v);
        }
        float dz[16];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float v[4];
            tfc_unpack<T, 4>(rd[q], v);
#pragma unroll
            for (int e = 0; e < 4; ++e) dz[4 * q + e] = v[e];
        }
        if (tile + gridDim.x < tiles) ask(m0 + (long)gridDim.x * S);
        __syncthreads();
        // z of rows r32.., columns c32..: lane l has row l % 32 and, in register 4 q + e, column 8 q + 4 (l / 32) + e
        if (g.act != TFC_ACT_IDENTITY) {
            floatx16 z = floatx16(0.f);
#pragma unroll
            for (int kk = 0; kk < S; kk += 16) {
                uintx4 a[P], b[P];
#pragma unroll
                for (int p = 0; p < P; ++p) a[p] = frag_col(wi + p * IMAGE, c32, kk), b[p] = frag_row(xi + p * IMAGE, r32, kk);
                terms<T, P>(a, b, z);
            }
            float f[16];
#pragma unroll
            for (int q = 0; q < 16; ++q) f[q] = z[q] * g.alpha + bias[q];
            act_grad_apply<sizeof(T) == 2>(g.act, f);
#pragma unroll
            for (int q = 0; q < 16; ++q) dz[q] *= f[q];
        }
        const bool live = m0 + r32 + (lane & 31) < g.m;
#pragma unroll
        for (int q = 0; q < 16; ++q) {  // (behind the last row and column dy is zero: 0 x a derivative that is not finite must not come in)
            const int n = c32 + (q >> 2) * 8 + half * 4 + (q & 3);
            dz[q] = live && n < g.n ? dz[q] : 0.f;
            db[q] += dz[q];
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float v[4] = {dz[4 * q], dz[4 * q + 1], dz[4 * q + 2], dz[4 * q + 3]};
            if constexpr (P == 1) v[0] *= TFC_DZ_SCALE, v[1] *= TFC_DZ_SCALE, v[2] *= TFC_DZ_SCALE, v[3] *= TFC_DZ_SCALE;
            put4<T>(di, r32 + (lane & 31), c32 + 8 * q + half * 4, v);
        }
        __syncthreads();
        floatx16 dx = floatx16(0.f), dx_lo = floatx16(0.f);
#pragma unroll
        for (int kk = 0; kk < S; kk += 16) {
            uintx4 w[P], d[D];
            if (g.dx) {  // rows r32.., columns (of k) c32..
#pragma unroll
                for (int p = 0; p < P; ++p) w[p] = frag_row(wi + p * IMAGE, c32, kk);
#pragma unroll
                for (int p = 0; p < D; ++p) d[p] = frag_row(di + p * IMAGE, r32, kk);
                if constexpr (P == 3)
                    terms<T, P>(w, d, dx);
                else
                    dx_lo = mma(T(), w[0], d[1], dx_lo), dx = mma(T(), w[0], d[0], dx);
            }
            if (g.want_dw) {  // rows (of k) r32.., columns c32..
#pragma unroll
                for (int p = 0; p < P; ++p) w[p] = frag_col(xi + p * IMAGE, r32, kk);
#pragma unroll
                for (int p = 0; p < D; ++p) d[p] = frag_col(di + p * IMAGE, c32, kk);
                if constexpr (P == 3)
                    terms<T, P>(d, w, dw);
                else
                    dw_lo = mma(T(), d[1], w[0], dw_lo), dw = mma(T(), d[0], w[0], dw);
            }
        }
        if constexpr (P == 1) dx += dx_lo * LO;
        if (!g.dx) continue;
        // dx through LDS ([64][64] floats where x and dz lay, units swizzled), out in whole rows
        __syncthreads();
        float* out = (float*)xi;
        const int rr = r32 + (lane & 31);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int u = (c32 + 8 * q + half * 4) >> 2;
            *(floatx4*)(out + rr * S + ((u ^ (rr & 15)) << 2)) = floatx4{dx[4 * q], dx[4 * q + 1], dx[4 * q + 2], dx[4 * q + 3]} * g.factor;
        }
        __syncthreads();
        constexpr int V = TfcType<T>::V, LPR = S / V, RPP = 256 / LPR;
#pragma unroll
        for (int p = 0; p < S / RPP; ++p) {
            const int row = p * RPP + t / LPR, c = (t % LPR) * V;
            float v[V];
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                const floatx4 w = *(const floatx4*)(out + row * S + ((((c + e) >> 2) ^ (row & 15)) << 2));
#pragma unroll
                for (int f = 0; f < 4; ++f) v[e + f] = w[f];
            }
            if (m0 + row < g.m && c < g.k) tfc_store_f<T, V>((T*)g.dx + (m0 + row) * g.k + c, g.k - c, v);
        }
    }
    // ---- partial sums
    if constexpr (P == 1) dw += dw_lo * LO;
    float* part = g.part + (long)blockIdx.x * ((long)g.k * g.n + g.n);
    if (g.want_dw) {
        const int k = r32 + (lane & 31);
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            const int n = c32 + (q >> 2) * 8 + half * 4 + (q & 3);
            if (k < g.k && n < g.n) part[k * g.pk + n * g.pn] = dw[q] * g.factor;
        }
    }
    __syncthreads();
    float* sums = (float*)lds;  // [2 row halves][64]
#pragma unroll
    for (int q = 0; q < 16; ++q) {
        float s = db[q];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) s += __shfl_xor(s, o);
        if ((lane & 31) == 0) sums[(wave >> 1) * S + c32 + (q >> 2) * 8 + half * 4 + (q & 3)] = s;
    }
    __syncthreads();
    if (t < g.n) part[(long)g.k * g.n + t] = (sums[t] + sums[S + t]) * g.cst;
}

template <class T>
int launch(const Narrow& g, int64_t blocks, hipStream_t s) {
    hipLaunchKernelGGL(tfc_dense_narrow_bwd_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, s, g);
    TFC_LAUNCH_CHECK("tfc_dense_narrow_bwd");
    return TFC_OK;
}

}  // namespace

// Workgroups, each of which leaves one partial result: two for every CU, as many as its LDS holds.
int64_t tfc_dense_narrow_partials(int64_t m) { return std::max<int64_t>(1, std::min<int64_t>((m + S - 1) / S, 512)); }

int tfc_dense_narrow_bwd(const tfc_dense_bwd_desc* d, float* part, hipStream_t stream) {
    Narrow g{};
    g.m = d->m, g.n = (int)d->n, g.k = (int)d->k;
    g.x = d->x, g.w = d->w, g.bias = d->bias, g.dy = d->dy, g.ldx = d->ldx;
    TFC_REQUIRE(d->ldw < INT32_MAX, TFC_EUNSUPPORTED, "tfc_dense_bwd: weight rows of 2^31 elements or more");
    g.wk = d->w_along_k ? 1 : (int)d->ldw, g.wn = d->w_along_k ? (int)d->ldw : 1;
    g.dx = d->dx, g.part = part;
    g.pk = d->w_along_k ? 1 : g.n, g.pn = d->w_along_k ? g.k : 1;
    g.alpha = d->alpha, g.cst = d->act_cst, g.act = d->act, g.want_dw = d->dw != nullptr;
    g.factor = d->alpha * d->act_cst * (d->dtype == TFC_F32 ? 1.f : 1.f / TFC_DZ_SCALE);
    const int64_t blocks = tfc_dense_narrow_partials(d->m);
    {
        TfcProfScope prof("tfc_dense_narrow_bwd", stream);
        const int rc = TFC_BY_DTYPE(d->dtype, launch, g, blocks, stream);
        if (rc) return rc;
    }
    if (!d->dw && !d->db) return TFC_OK;
    return tfc_join_columns(part, blocks, d->k * d->n, d->dw, d->n, d->db, d->dtype, stream);
}
