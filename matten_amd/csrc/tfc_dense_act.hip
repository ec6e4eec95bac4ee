// Matrix product with its epilogue: C = c act(alpha A B + bias) + residual, for fp32, bf16 and fp16, and the elementwise half of
// its backward pass (dz = c act'(z) dy with the column sums that are the bias's gradient).  The products of the backward
// pass are the same kernel without the epilogue: dA = dz B^T, dB = A^T dz.
//
// A tile of C belongs to a workgroup of four waves.  Operand tiles go through registers into LDS as rows of 16-bit elements with
// the contraction index contiguous (row stride padded by 16 bytes: consecutive rows start 16-byte units of different banks), so a
// lane reads its eight k of a matrix instruction in one access; an operand whose memory runs along the rows instead is
// transposed on the way, in registers.  The loads of the next step are in flight while this one is multiplied.
// bf16 and fp16 feed v_mfma_f32_32x32x16 directly.  fp32 is cut into three bf16 pieces, x = h + m + l exactly (8 + 8 + 8
// significant bits), and the product is the six largest of the nine piece products, the dropped ones below 2^-24 |a b|: 2.67
// times the rate of the fp32 matrix instruction and no less exact (an infinity has no pieces: it gives NaN).
// The instruction's rows are the columns of C, so that a lane ends up with four neighbouring columns of a row.
//
// What the backward pass needs of the forward one is z = alpha A B + bias.  Rounded to a 16-bit type it would be wrong by as much as the
// results are, and the gradients by 1.5 times what their own rounding is worth: store_z() keeps more of it.  dz is rounded for the
// products, as the matrix instruction takes it, or kept in two pieces (dz_pieces()).
//
// Measured, with the library's product of the same sizes without an epilogue: fp32 6912 x 511 x 2048 118 us (library 157), with bias, ssp
// and z 132, its gradients' products 106 and 98 (169, 125); bf16 16384 x 1024 x 4096 173 us (139), with gelu, z and residual 221,
// its gradients' 117 and 124 (98, 197); bf16 1 x 4096 x 4096 7.3 us for 7.1 us of weights.
//
// Few tiles and a long contraction (a weight's gradient over many rows): the contraction is split, partial tiles go to the
// workspace and a second kernel adds them in order and applies the epilogue.
#include "tfc_dense_act.h"

#include <algorithm>

namespace {

// ------------------------------------------------------------------------------------------------ operands
struct Operand {
    const void* p;
    long ld;  // elements between rows (k contiguous) / between k (rows contiguous)
};

// The comparisons of a step at an edge are made when it comes: kept from step to step they would cost the registers that a second
// workgroup on the CU needs.
__device__ __forceinline__ void hide(int& t) { asm volatile("" : "+v"(t)); }

// What a thread has in flight of an operand tile of R rows and a step of K, and its way to LDS.
//  along k: units of eight k of a row; LDS [row][K + 8].
//  along the rows, 16 bits: units of eight rows of a k; LDS [k][R + 32], turned by the transposing LDS read (fragment()).  The padding
//    puts the four k that such a read takes side by side into different quarters of the banks.
//  along the rows, fp32: the pieces are formed on the way to LDS, so the turning is done there too: a thread takes RV neighbouring
//    rows x eight k and writes units of eight k; LDS [row][K + 8].
// A step is loaded without a comparison, from an address that is the workgroup's plus a 32-bit offset that is the thread's for
// good (nothing touches the values before store(): all accesses are in flight together), wherever its accesses stay inside
// the operand's memory: rows behind the last one are the last one again (their products are not stored), and an access that
// begins in the last rows may run into the next k's.  The others (the tail of the contraction; along the rows, the edge
// tile's last step) go element by element.
template <class T, int R, bool ALONG_K>
struct Stage {
    static constexpr bool F32 = std::is_same<T, float>::value, TURN = !ALONG_K && F32, TR_READ = !ALONG_K && !F32;
    static constexpr int P = Pieces<T>::N, K = Pieces<T>::K, UNITS = R * K / 8 / 256;
    static constexpr int LD = TR_READ ? R + 32 : K + 8;                  // 16-bit elements of an LDS row
    static constexpr int IMAGE = TR_READ ? K * LD : P * R * LD;          // and of the operand's whole image
    static constexpr int RV = TURN ? UNITS : 8;                          // rows of an access along the rows
    static constexpr int NR = TURN ? 8 : UNITS, NE = TURN ? RV : 8;      // accesses, elements of one
    static constexpr int SIDE = ALONG_K ? K / 8 : R / RV, HOP = 256 / SIDE;  // threads side by side; rows (or k) between accesses
    TfcRaw<T, NE> raw[NR];
    uint32_t off[NR];  // bytes from the tile's first element of this step
    const char* base;
    long adv;  // bytes to the next step

    // Row and k, in the tile and step, of access i of thread t.
    static __device__ __forceinline__ int row_of(int t, int i) { return ALONG_K ? t / SIDE + i * HOP : (t % SIDE) * RV; }
    static __device__ __forceinline__ int k_of(int t, int i) {
        return ALONG_K ? (t % SIDE) * 8 : TURN ? (t / SIDE) * 8 + i : t / SIDE + i * HOP;
    }

    __device__ __forceinline__ void start(const Operand& o, long r0, long rows, long k0) {
        const int t = threadIdx.x, last = (int)(rows < R ? rows : R) - 1;
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const uint32_t r = (uint32_t)min(row_of(t, i), last), k = (uint32_t)k_of(t, i), ld = (uint32_t)o.ld;
            off[i] = (uint32_t)sizeof(T) * (ALONG_K ? r * ld + k : k * ld + r);
        }
        base = (const char*)o.p + sizeof(T) * (ALONG_K ? r0 * o.ld + k0 : k0 * o.ld + r0);
        adv = sizeof(T) * (ALONG_K ? K : K * o.ld);
    }

    // rows, k: how many of each there are from the tile's first on (PLAIN: accesses that need no comparison).
    template <bool PLAIN>
    __device__ __forceinline__ void load(long rows, long k) {
        int t = threadIdx.x;
        if (!PLAIN) hide(t);
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const T* q = (const T*)(base + off[i]);
            if constexpr (PLAIN) {
                raw[i] = tfc_load<T, NE>(q);
            } else {
                const int r = row_of(t, i), kk = k_of(t, i);
                T e[NE];
#pragma unroll
                for (int j = 0; j < NE; ++j) e[j] = (ALONG_K ? r < rows && kk + j < k : r + j < rows && kk < k) ? q[j] : (T)0.f;
                __builtin_memcpy(&raw[i], e, sizeof(e));
            }
        }
        base += adv;
    }

    __device__ __forceinline__ void store(uint16_t* lds) const {
        const int t = threadIdx.x;
        if constexpr (!F32) {
#pragma unroll
            for (int i = 0; i < NR; ++i)
                *(uintx4*)(lds + (ALONG_K ? row_of(t, i) * LD + k_of(t, i) : k_of(t, i) * LD + row_of(t, i))) = raw[i];
        } else {
            float f[NR][NE];
#pragma unroll
            for (int i = 0; i < NR; ++i) tfc_unpack<T, NE>(raw[i], f[i]);
#pragma unroll
            for (int i = 0; i < UNITS; ++i) {
                const int row = TURN ? row_of(t, 0) + i : row_of(t, i), k = k_of(t, 0);
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = TURN ? f[j % NR][i % NE] : f[i % NR][j % NE];
                const Unit3 u = split8(v);
                uint16_t* q = lds + row * LD + k;
                *(uintx4*)q = u.h;
                *(uintx4*)(q + R * LD) = u.m;
                *(uintx4*)(q + 2 * R * LD) = u.l;
            }
        }
    }

    // Piece p of 32 rows from r0 on and 16 k from kk on, as the matrix instruction takes it: lane l has row l % 32, eight k from
    // 8 (l / 32) on.  The transposing read gives, in each group of 16 lanes, lane i the column i of four rows of LDS of 16
    // elements each, whose quarters the lanes 4 j .. 4 j + 3 address.
    static __device__ __forceinline__ uintx4 fragment(const uint16_t* lds, int p, int r0, int kk) {
        const int lane = threadIdx.x & 63;
        if constexpr (!TR_READ) return *(const uintx4*)(lds + (p * R + r0 + (lane & 31)) * LD + kk + (lane >> 5) * 8);
        const uint16_t* q = lds + (kk + (lane >> 5) * 8 + ((lane & 15) >> 2)) * LD + r0 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
        typedef __attribute__((address_space(3))) shortx4* Lds;
        struct {
            shortx4 a, b;
        } both = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(q)), __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(q + 4 * LD))};
        return __builtin_bit_cast(uintx4, both);
    }
};

// ------------------------------------------------------------------------------------------------ the product
// How much of a contraction of k elements from k0 to k1 goes in whole steps without comparisons.  An operand along the rows whose tile
// is not full must have eight elements between k and must not be at its last k: its accesses then end inside its memory.
__device__ __forceinline__ long plain_part(long k0, long k1, long k, long step, bool full_a, long lda, bool full_b, long ldb) {
    long n = (k1 - k0) / step * step;
    if ((!full_a && lda < 8) || (!full_b && ldb < 8)) return 0;
    if ((!full_a || !full_b) && k0 + n == k) n -= step;
    return n < 0 ? 0 : n;
}

struct Args {
    Operand a, b;
    long m, n, k;
    void* c;
    long ldc;
    const void *bias, *res;
    long ldr;
    void* z;  // alpha A B + bias, for the backward pass (store_z)
    float alpha, cst;
    int act;
    float* part;  // split contraction: [split][m][n]
    long k_split;
    int tiles_m, tiles_n;
    int passes;        // 2 (16 bits only): one operand is the sum of two pieces, the second lo_a or lo_b bytes behind the first
    long lo_a, lo_b;
};

// z [m, n], packed.  fp32: as it is.  bf16: as fp16, three bits better in the same two bytes: what lies beyond that range is cut to its
// end, where every act' has reached its limit, and what is not zero does not become zero (abs).  fp16: the upper three bytes of the
// fp32 number, a plane of two and behind it a plane of one.
__device__ __forceinline__ tfc_f16 z_half(float v) {
    const float a = fminf(fmaxf(fabsf(v), 0x1p-24f), 65504.f);
    return v != 0.f && v == v ? (tfc_f16)__builtin_copysignf(a, v) : (tfc_f16)v;
}
template <class T, int N>
__device__ __forceinline__ void store_z(void* z, long count, long at, const float (&v)[N]) {
    if constexpr (std::is_same<T, float>::value) {
        tfc_store<float, N>((float*)z + at, tfc_pack<float, N>(v));
    } else if constexpr (std::is_same<T, tfc_bf16>::value) {
        tfc_f16 h[N];
#pragma unroll
        for (int j = 0; j < N; ++j) h[j] = z_half(v[j]);
        __builtin_memcpy((tfc_f16*)z + at, h, sizeof(h));
    } else {
        uint16_t hi[N];
        uint8_t lo[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t u = __float_as_uint(v[j]);
            hi[j] = (uint16_t)(u >> 16), lo[j] = (uint8_t)(u >> 8);
        }
        __builtin_memcpy((uint16_t*)z + at, hi, sizeof(hi));
        __builtin_memcpy((uint8_t*)z + 2 * count + at, lo, sizeof(lo));
    }
}
template <class T, int N>
__device__ __forceinline__ void load_z(const void* z, long count, long at, long left, float (&v)[N]) {
    if constexpr (std::is_same<T, float>::value) {
        tfc_load_f<float, N>((const float*)z + at, left, v);
    } else if constexpr (std::is_same<T, tfc_bf16>::value) {
        tfc_load_f<tfc_f16, N>((const tfc_f16*)z + at, left, v);
    } else if (left >= N) {
        TfcRaw<T, N> hi;
        typename TfcWords<N>::type lo;
        __builtin_memcpy(&hi, (const uint16_t*)z + at, sizeof(hi));
        __builtin_memcpy(&lo, (const uint8_t*)z + 2 * count + at, sizeof(lo));
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = __uint_as_float((hi[j / 2] >> (j % 2 * 16)) << 16 | (lo[j / 4] >> (j % 4 * 8) & 255) << 8);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            v[j] = j < left ? __uint_as_float((uint32_t)((const uint16_t*)z)[at + j] << 16 | (uint32_t)((const uint8_t*)z)[2 * count + at + j] << 8)
                            : 0.f;
    }
}

// N neighbouring columns of one row of C, all inside; `res`: their residual where there is one.
template <class T, int N>
__device__ __forceinline__ void epilogue(const Args& g, long row, long col, float (&v)[N], TfcRaw<T, N> res) {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] *= g.alpha;
    if (g.bias) {
        float b[N];
        tfc_unpack<T, N>(tfc_load<T, N>((const T*)g.bias + col), b);
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] += b[j];
    }
    if (g.z) store_z<T, N>(g.z, g.m * g.n, row * g.n + col, v);
    act_apply<sizeof(T) == 2>(g.act, v);
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] *= g.cst;
    if (g.res) {
        float r[N];
        tfc_unpack<T, N>(res, r);
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] += r[j];
    }
    tfc_store<T, N>((T*)g.c + row * g.ldc + col, tfc_pack<T, N>(v));
}

template <class T, int N>
__device__ __forceinline__ TfcRaw<T, N> residual(const Args& g, long row, long col) {
    TfcRaw<T, N> r = {};
    if (g.res) r = tfc_load<T, N>((const T*)g.res + row * g.ldr + col);
    return r;
}

// Columns [col, col + N) of a row as far as there are any: whole, or one by one.
template <class T, int N>
__device__ __forceinline__ void epilogue_left(const Args& g, long row, long col, const float (&v)[N]) {
    if (g.n - col >= N) {
        float w[N];
#pragma unroll
        for (int j = 0; j < N; ++j) w[j] = v[j];
        epilogue<T, N>(g, row, col, w, residual<T, N>(g, row, col));
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            float w[1] = {v[j]};
            if (col + j < g.n) epilogue<T, 1>(g, row, col + j, w, residual<T, 1>(g, row, col + j));
        }
    }
}

constexpr int corner_floats(int ni) { return 32 * (32 * ni + 4); }

// A wave's 32 MI x 32 NI part of C, first element (m0, n0).  A lane holds 4 columns of 32 rows apart: 32 rows x 32 NI columns at a time
// go through the wave's own corner of LDS and come back as whole 16-byte accesses of neighbouring lanes (128 bytes of a row at
// least: storing the accumulators where they lie, 16 bytes of 32 different rows an instruction, took 255 us longer in the
// product of 16384 x 1024 x 4096).  The residual of the next 32 rows is asked for before this one's results are stored: a wait
// for a load is a wait for every access before it, stores too.
template <class T, int MI, int NI, bool SPLIT>
__device__ __forceinline__ void write_out(const Args& g, const floatx16 (&acc)[MI][NI], float* corner, long m0, long n0) {
    constexpr int V = SPLIT ? 4 : TfcType<T>::V, WC = 32 * NI, LW = WC + 4;
    constexpr int LPR = WC / V, RPP = 64 / LPR, PASSES = 32 / RPP;  // lanes of a row, rows of a pass
    constexpr int TOGETHER = PASSES < 4 ? PASSES : 4;               // passes whose residuals are in flight together
    const int lane = threadIdx.x & 63, fr = lane & 31, cl = (lane % LPR) * V;
    const long col = n0 + cl;
    const bool whole = g.n - n0 >= WC && g.m - m0 >= 32 * MI;  // (the same in all lanes)
    TfcRaw<T, V> next[TOGETHER];
    auto ask = [&](int i, int p0) {
        if constexpr (!SPLIT) {
            if (whole) {
#pragma unroll
                for (int p = 0; p < TOGETHER; ++p) next[p] = residual<T, V>(g, m0 + 32 * i + (p0 + p) * RPP + lane / LPR, col);
            }
        }
    };
    ask(0, 0);
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        wave_step();
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                floatx4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * q + e];
                *(floatx4*)(corner + fr * LW + 32 * j + 8 * q + (lane >> 5) * 4) = v;
            }
        wave_step();
        if (!whole) {  // an edge: element by element, straight from LDS
#pragma unroll 1
            for (int at = lane; at < 32 * WC; at += 64) {
                const long row = m0 + 32 * i + at / WC, c = n0 + at % WC;
                float v[1] = {corner[at / WC * LW + at % WC]};
                if (row >= g.m || c >= g.n) continue;
                if constexpr (SPLIT)
                    g.part[((long)blockIdx.y * g.m + row) * g.n + c] = v[0];
                else
                    epilogue<T, 1>(g, row, c, v, residual<T, 1>(g, row, c));
            }
            continue;
        }
#pragma unroll
        for (int p0 = 0; p0 < PASSES; p0 += TOGETHER) {
            TfcRaw<T, V> res[TOGETHER];
#pragma unroll
            for (int p = 0; p < TOGETHER; ++p) res[p] = next[p];
            if (p0 + TOGETHER < PASSES)
                ask(i, p0 + TOGETHER);
            else if (i + 1 < MI)
                ask(i + 1, 0);
#pragma unroll
            for (int p = 0; p < TOGETHER; ++p) {
                const int rl = (p0 + p) * RPP + lane / LPR;
                const long row = m0 + 32 * i + rl;
                float v[V];
#pragma unroll
                for (int e = 0; e < V; e += 4) {
                    const floatx4 w = *(const floatx4*)(corner + rl * LW + cl + e);
#pragma unroll
                    for (int f = 0; f < 4; ++f) v[e + f] = w[f];
                }
                if constexpr (SPLIT)
                    tfc_store<float, V>(g.part + ((long)blockIdx.y * g.m + row) * g.n + col, tfc_pack<float, V>(v));
                else
                    epilogue<T, V>(g, row, col, v, res[p]);
            }
        }
    }
}

// (row of tiles << 32) + column of this workgroup's tile.  Neighbouring workgroups of an XCD share its L2: they take tiles in columns of
// GROUP, so that those in flight read few panels of both operands and write long stretches of rows.  16384 x 1024 x 4096 in bf16,
// GROUP 1, 4, 8, 32: 180, 175, 175, 186 us; with residual and z, bound by writing, 232, 221, 241, 232.
__device__ __forceinline__ long tile_of(const Args& g) {
    constexpr unsigned GROUP = 4;
    const unsigned tile = tfc_xcd_remap(blockIdx.x, gridDim.x), strip = GROUP * (unsigned)g.tiles_n;
    const unsigned top = tile / strip * GROUP, in = tile % strip, high = min(GROUP, (unsigned)g.tiles_m - top);
    return ((long)(top + in % high) << 32) + in / high;
}

// BM x BN tile, waves 2 x 2.  SPLIT: this workgroup's part of the contraction to g.part.
template <class T, bool AK, bool BK, int BM, int BN, bool SPLIT>
__global__ __launch_bounds__(256, 2) void tfc_dense_kernel(const Args g) {
    using A = Stage<T, BM, AK>;
    using B = Stage<T, BN, BK>;
    constexpr int P = Pieces<T>::N, K = Pieces<T>::K;
    constexpr int MI = BM / 64, NI = BN / 64;  // 32 x 32 tiles of a wave
    constexpr int LDS = A::IMAGE + B::IMAGE > 8 * corner_floats(NI) ? A::IMAGE + B::IMAGE : 8 * corner_floats(NI);
    __shared__ __attribute__((aligned(16))) uint16_t lds[LDS];
    uint16_t* la = lds;
    uint16_t* lb = lds + A::IMAGE;
    const long tile = tile_of(g);
    const long m0 = (tile >> 32) * BM, n0 = (tile & 0xFFFFFFFF) * BN;
    const long k0 = SPLIT ? (long)blockIdx.y * g.k_split : 0;
    const long k1 = SPLIT ? (k0 + g.k_split < g.k ? k0 + g.k_split : g.k) : g.k;
    const int wave = threadIdx.x >> 6;
    const int wm = (wave >> 1) * 32 * MI, wn = (wave & 1) * 32 * NI;
    floatx16 acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = floatx16(0.f);
    A sa;
    B sb;
    const long ra = g.m - m0, rb = g.n - n0;
    // One step: its operands to LDS, then (MORE) the loads of the next one and the products.
    auto step = [&](auto more, long left) {
        __syncthreads();  // the step before has been read
        sa.store(la);
        sb.store(lb);
        __syncthreads();
        if constexpr (more == 1) sa.template load<true>(ra, left), sb.template load<true>(rb, left);
        if constexpr (more == 2) sa.template load<false>(ra, left), sb.template load<false>(rb, left);
#pragma unroll
        for (int kk = 0; kk < K; kk += 16) {
            uintx4 fa[MI][P], fb[NI][P];
#pragma unroll
            for (int p = 0; p < P; ++p) {
#pragma unroll
                for (int i = 0; i < MI; ++i) fa[i][p] = A::fragment(la, p, wm + 32 * i, kk);
#pragma unroll
                for (int j = 0; j < NI; ++j) fb[j][p] = B::fragment(lb, p, wn + 32 * j, kk);
            }
            // (fp32: smallest terms first; the tiles take turns, so that no instruction waits for the one before it)
            constexpr int TERMS = P == 3 ? 6 : 1;
#pragma unroll
            for (int q = 0; q < TERMS; ++q)
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int j = 0; j < NI; ++j)
                        acc[i][j] = mma(Mma<T>(), fb[j][P == 3 ? TFC_TERM_B[q] : 0], fa[i][P == 3 ? TFC_TERM_A[q] : 0], acc[i][j]);
        }
    };
    const int passes = P == 1 ? g.passes : 1;
#pragma unroll 1
    for (int lo = passes - 1; lo >= 0; --lo) {  // (the second pieces first: the smaller terms)
        sa.start({(const char*)g.a.p + lo * g.lo_a, g.a.ld}, m0, ra, k0);
        sb.start({(const char*)g.b.p + lo * g.lo_b, g.b.ld}, n0, rb, k0);
        long left = k1 - k0;  // of the contraction, from the step in hand on
        long plain = plain_part(k0, k1, g.k, K, AK || ra >= BM, g.a.ld, BK || rb >= BN, g.b.ld);
        if (plain > 0)
            sa.template load<true>(ra, left), sb.template load<true>(rb, left);
        else
            sa.template load<false>(ra, left), sb.template load<false>(rb, left);
        for (; plain > K; plain -= K, left -= K) step(std::integral_constant<int, 1>(), left - K);
#pragma unroll 1
        for (; left > K; left -= K) step(std::integral_constant<int, 2>(), left - K);
        step(std::integral_constant<int, 0>(), 0);
        if (std::is_same<T, tfc_f16>::value && lo) {
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j) acc[i][j] *= 1.f / TFC_LO_SCALE;
        }
    }
    __syncthreads();
    write_out<T, MI, NI, SPLIT>(g, acc, (float*)lds + wave * corner_floats(NI), m0 + wm, n0 + wn);
}

// ------------------------------------------------------------------------------------------------ large 16-bit products
// 256 x 256 tile of eight waves (2 x 4, 128 x 64 of C each: eight 32 x 32 products for six operand reads).  The operands of a step of
// 64 go straight from memory to LDS while the step before is multiplied (two images of 64 KB, one barrier a step): what bounds
// the kernel above on large products is the wait for operands on their way through registers.  A step of 64 and not 32: a
// row's part of it is a whole line of 128 bytes (16384 x 4096 x 1024 along k: 128 us with steps of 32, three of them in flight,
// 121 with steps of 64).  A wave reads the operands of the next 16 k between the products of this one (121 -> 115).
// Rows of an image have no padding (a wave's 64 x 16 bytes land side by side); their 16-byte units are swizzled by which unit a lane
// asks memory for, so that 16 lanes of a read meet all banks: along k, unit ^ (row / 2 % 8); along the rows, 64-byte part ^ (k % 4).
// Operands start at multiples of 16 bytes, have strides and, along the rows, sizes of multiples of 8; the contraction is a
// multiple of 64.  Rows behind the last one are the last one again.
constexpr int DEEP = 256, DEEP_K = 64, DEEP_IMAGE = DEEP * DEEP_K;

// 16 bytes a lane from base + off to `to` + 16 lane.  Written out, because for the transposing LDS reads the compiler cannot tell the
// image being filled from the one being read and waits for every access of the wave; nothing is loaded into registers, and
// the kernel's own waits (TFC_DEEP_STEP) are the ones there are.  M0 is read one state after it was set.
__device__ __forceinline__ void memory_to_lds(const char* base, uint32_t off, uint16_t* to) {
    const uint32_t lds = (uint32_t)tfc_uniform((int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)to);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory");
}

template <class T, bool ALONG_K>
struct DeepStage {
    uint32_t off[4];  // bytes, of this lane's four accesses a step
    const char* base;
    long adv;

    __device__ __forceinline__ void start(const Operand& o, long r0, long rows, long k0) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, last = (int)(rows < DEEP ? rows : DEEP) - 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t r, k;
            if constexpr (ALONG_K) {
                const int row = (i * 8 + wave) * 8 + lane / 8;
                r = min(row, last), k = ((lane & 7) ^ ((row >> 1) & 7)) * 8;
                off[i] = 2u * (r * (uint32_t)o.ld + k);
            } else {
                k = (i * 8 + wave) * 2 + lane / 32;
                r = min((int)((((lane & 31) >> 2) ^ (k & 3)) * 32 + (lane & 3) * 8), last & ~7);
                off[i] = 2u * (k * (uint32_t)o.ld + r);
            }
        }
        base = (const char*)o.p + 2 * (ALONG_K ? r0 * o.ld + k0 : k0 * o.ld + r0);
        adv = 2 * (ALONG_K ? DEEP_K : DEEP_K * o.ld);
    }
    __device__ __forceinline__ void load(uint16_t* image) {
        const int wave = tfc_uniform(threadIdx.x >> 6);
#pragma unroll
        for (int i = 0; i < 4; ++i) memory_to_lds(base, off[i], image + (i * 8 + wave) * 512);
        base += adv;
    }
    static __device__ __forceinline__ uintx4 fragment(const uint16_t* im, int r0, int kk) {
        const int lane = threadIdx.x & 63;
        if constexpr (ALONG_K) {
            const int r = r0 + (lane & 31), u = kk / 8 + (lane >> 5);
            return *(const uintx4*)(im + r * DEEP_K + ((u ^ ((r >> 1) & 7)) << 3));
        }
        const int k = kk + (lane >> 5) * 8 + ((lane & 15) >> 2), r = r0 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
        const uint16_t* q = im + k * DEEP + (((r >> 5) ^ (k & 3)) << 5) + (r & 31);  // (k + 4: the same swizzle)
        typedef __attribute__((address_space(3))) shortx4* Lds;
        struct {
            shortx4 a, b;
        } both = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(q)), __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(q + 4 * DEEP))};
        return __builtin_bit_cast(uintx4, both);
    }
};

template <class T, bool AK, bool BK, bool SPLIT>
__global__ __launch_bounds__(512, 2) void tfc_dense_deep_kernel(const Args g) {
    __shared__ __attribute__((aligned(16))) uint16_t s0[2 * DEEP_IMAGE], s1[2 * DEEP_IMAGE];
    const long tile = tile_of(g);
    const long m0 = (tile >> 32) * DEEP, n0 = (tile & 0xFFFFFFFF) * DEEP;
    const long k0 = SPLIT ? (long)blockIdx.y * g.k_split : 0;
    const long k1 = SPLIT ? (k0 + g.k_split < g.k ? k0 + g.k_split : g.k) : g.k;
    const int wave = threadIdx.x >> 6, wm = (wave >> 2) * 128, wn = (wave & 3) * 64;
    floatx16 acc[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = floatx16(0.f);
    DeepStage<T, AK> sa;
    DeepStage<T, BK> sb;
    sa.start(g.a, m0, g.m - m0, k0);
    sb.start(g.b, n0, g.n - n0, k0);
    int ahead = (int)((k1 - k0) / DEEP_K), todo = ahead;  // steps to ask for, steps to multiply
    auto ask = [&](uint16_t* s) {
        if (ahead > 0) {
            sa.load(s);
            sb.load(s + DEEP_IMAGE);
            --ahead;
        }
    };
    auto multiply = [&](const uint16_t* s) {
        uintx4 fa[2][4], fb[2][2];
        auto read = [&](int q) {
#pragma unroll
            for (int j = 0; j < 2; ++j) fb[q & 1][j] = DeepStage<T, BK>::fragment(s + DEEP_IMAGE, wn + 32 * j, 16 * q);
#pragma unroll
            for (int i = 0; i < 4; ++i) fa[q & 1][i] = DeepStage<T, AK>::fragment(s, wm + 32 * i, 16 * q);
        };
        read(0);
#pragma unroll
        for (int q = 0; q < DEEP_K / 16; ++q) {
            if (q + 1 < DEEP_K / 16) read(q + 1);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = mma(T(), fb[q & 1][j], fa[q & 1][i], acc[i][j]);
        }
        constexpr int READS = (AK ? 4 : 8) + (BK ? 2 : 4);  // of a part of 16
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
#pragma unroll
        for (int q = 0; q < DEEP_K / 16; ++q) {
            int left = q + 1 < DEEP_K / 16 ? READS : 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                if (left > 0) __builtin_amdgcn_sched_group_barrier(0x100, READS > 8 ? 2 : 1, 0);
                left -= READS > 8 ? 2 : 1;
            }
        }
        --todo;
    };
    // Every wave waits for its own accesses of the step in hand and for its reads of the image before, and then for the other waves; behind
    // the barrier that image is free.
#define TFC_DEEP_STEP(HERE, FREE)                                            \
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); \
    ask(FREE);                                                               \
    multiply(HERE);                                                          \
    if (todo == 0) break;
    ask(s0);
    while (true) {
        TFC_DEEP_STEP(s0, s1)
        TFC_DEEP_STEP(s1, s0)
    }
#undef TFC_DEEP_STEP
    __syncthreads();
    static_assert(4 * corner_floats(2) * 4 <= 4 * DEEP_IMAGE, "four waves' corners in an image pair");
    write_out<T, 4, 2, SPLIT>(g, acc, (float*)(wave & 1 ? s1 : s0) + (wave >> 1) * corner_floats(2), m0 + wm, n0 + wn);
}

// ------------------------------------------------------------------------------------------------ a few rows
// At most ROWS rows (a single token): bound by reading B once.  One launch without partial results, where the tiles above, mostly empty,
// split the contraction and join it in a second one (1 x 4096 x 4096 with B along k: bf16 12.9 -> 7.3 us, which is reading B at the speed of
// a copy, fp32 28 -> 13; 4 rows 13.5 -> 9.3, 29 -> 14).  The products
// are fp32 multiply-adds on the vector units, which up to four rows keep pace with memory.
// B along k: a workgroup has COLS columns, its four waves take turns along the contraction; sums over the lanes, then the waves.
// B along the rows: a workgroup has 128 bytes of every row (fp32; 16 bits: 64, so that there are workgroups enough) and 16 waves side by
// side along the contraction.
constexpr int ROWS = 4, COLS = 4, STRIP = 32;

// Row r of A from k on: N elements as far as `left` goes, with their second pieces where there are any.
template <class T, int N, bool WHOLE>
__device__ __forceinline__ void row_part(const Args& g, int r, long k, long left, float (&x)[N]) {
    const T* p = (const T*)g.a.p + min((long)r, g.m - 1) * g.a.ld + k;
    tfc_unpack<T, N>(WHOLE ? tfc_load<T, N>(p) : tfc_load_left<T, N>(p, left), x);
    if (sizeof(T) == 2 && g.lo_a) {
        const T* q = (const T*)((const char*)p + g.lo_a);
        float lo[N];
        tfc_unpack<T, N>(WHOLE ? tfc_load<T, N>(q) : tfc_load_left<T, N>(q, left), lo);
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] += lo[j] * (std::is_same<T, tfc_f16>::value ? 1.f / TFC_LO_SCALE : 1.f);
    }
}

template <class T, int M>
__global__ __launch_bounds__(256) void tfc_dense_rows_k_kernel(const Args g) {
    constexpr int V = TfcType<T>::V, STEP = 4 * 64 * V;
    __shared__ float lds[4][M * COLS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long n0 = (long)blockIdx.x * COLS;
    const T* w[COLS];
#pragma unroll
    for (int c = 0; c < COLS; ++c) w[c] = (const T*)g.b.p + min(n0 + c, g.n - 1) * g.b.ld;
    float acc[M][COLS];
#pragma unroll
    for (int r = 0; r < M; ++r)
#pragma unroll
        for (int c = 0; c < COLS; ++c) acc[r][c] = 0.f;
    auto part = [&](auto whole, long k) {
        TfcRaw<T, V> raw[COLS];
#pragma unroll
        for (int c = 0; c < COLS; ++c) raw[c] = whole ? tfc_load<T, V>(w[c] + k) : tfc_load_left<T, V>(w[c] + k, g.k - k);
        float x[M][V];
#pragma unroll
        for (int r = 0; r < M; ++r) row_part<T, V, whole>(g, r, k, g.k - k, x[r]);
#pragma unroll
        for (int c = 0; c < COLS; ++c) {
            float v[V];
            tfc_unpack<T, V>(raw[c], v);
#pragma unroll
            for (int r = 0; r < M; ++r)
#pragma unroll
                for (int j = 0; j < V; ++j) acc[r][c] += x[r][j] * v[j];
        }
    };
    const long mine = (long)(wave * 64 + lane) * V;
    long k0 = 0;
    for (; k0 + STEP <= g.k; k0 += STEP) part(std::true_type(), k0 + mine);
    if (k0 + mine < g.k) part(std::false_type(), k0 + mine);
    if constexpr (M * COLS == 16) {
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = acc[i / COLS][i % COLS];
        const float s = tfc_wave_reduce16(v);
        if ((lane & 3) == 0) lds[wave][tfc_reduce16_index(lane)] = s;
    } else {
#pragma unroll
        for (int r = 0; r < M; ++r) {
            float v[4] = {acc[r][0], acc[r][1], acc[r][2], acc[r][3]};
            const float s = tfc_wave_reduce4(v);
            if ((lane & 15) == 0) lds[wave][r * COLS + tfc_reduce4_index(lane)] = s;
        }
    }
    __syncthreads();
    const int t = threadIdx.x;
    if (t < M * COLS && t / COLS < g.m && n0 + t % COLS < g.n) {
        float v[1] = {(lds[0][t] + lds[1][t]) + (lds[2][t] + lds[3][t])};
        epilogue<T, 1>(g, t / COLS, n0 + t % COLS, v, residual<T, 1>(g, t / COLS, n0 + t % COLS));
    }
}

template <class T, int M>
__global__ __launch_bounds__(1024) void tfc_dense_rows_n_kernel(const Args g) {
    constexpr int V = TfcType<T>::V, LC = STRIP / V, STEP = 1024 / LC * V;  // lanes side by side; a lane has V neighbouring k
    __shared__ float lds[16][M * STRIP];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, cl = (threadIdx.x % LC) * V;
    const long n0 = (long)blockIdx.x * STRIP, left = g.n - n0 - cl;
    const T* w = (const T*)g.b.p + n0 + cl;
    float acc[M][V];
#pragma unroll
    for (int r = 0; r < M; ++r)
#pragma unroll
        for (int j = 0; j < V; ++j) acc[r][j] = 0.f;
    auto multiply = [&](TfcRaw<T, V> raw, const float (&x)[M][V], int u) {
        float v[V];
        tfc_unpack<T, V>(raw, v);
#pragma unroll
        for (int r = 0; r < M; ++r)
#pragma unroll
            for (int j = 0; j < V; ++j) acc[r][j] += x[r][u] * v[j];
    };
    long k = (long)(threadIdx.x / LC) * V;
    if (g.n - n0 >= STRIP) {
        for (; k + V <= g.k; k += STEP) {
            TfcRaw<T, V> raw[V];
#pragma unroll
            for (int u = 0; u < V; ++u) raw[u] = tfc_load<T, V>(w + (k + u) * g.b.ld);
            float x[M][V];
#pragma unroll
            for (int r = 0; r < M; ++r) row_part<T, V, true>(g, r, k, V, x[r]);
#pragma unroll
            for (int u = 0; u < V; ++u) multiply(raw[u], x, u);
        }
    }
    for (; k < g.k; k += STEP) {
        float x[M][V];
#pragma unroll
        for (int r = 0; r < M; ++r) row_part<T, V, false>(g, r, k, g.k - k, x[r]);
#pragma unroll
        for (int u = 0; u < V; ++u)
            if (k + u < g.k) multiply(tfc_load_left<T, V>(w + (k + u) * g.b.ld, left), x, u);
    }
    // Sums over the lanes of a column: rows of 16 lanes pair by pair, each keeping half of the V columns, then inside the rows.
    const int half = lane >> 5, odd = lane >> 4 & 1, p = lane & 15;
#pragma unroll
    for (int r = 0; r < M; ++r) {
        float h[V / 2], q[V / 4];
#pragma unroll
        for (int j = 0; j < V / 2; ++j) h[j] = tfc_swap_add32(acc[r][j], acc[r][j + V / 2]);
#pragma unroll
        for (int j = 0; j < V / 4; ++j) {
            q[j] = tfc_swap_add16(h[j], h[j + V / 4]);
            q[j] += tfc_dpp<0x128>(q[j]);                        // row_ror:8
            if constexpr (LC == 4) q[j] += tfc_dpp<0x124>(q[j]);  // row_ror:4
            if (p < LC) lds[wave][r * STRIP + p * V + half * (V / 2) + odd * (V / 4) + j] = q[j];
        }
    }
    __syncthreads();
    const int t = threadIdx.x;
    if (t < M * STRIP && t / STRIP < g.m && n0 + t % STRIP < g.n) {
        float v[1] = {0.f};
#pragma unroll
        for (int i = 0; i < 16; ++i) v[0] += lds[i][t];
        epilogue<T, 1>(g, t / STRIP, n0 + t % STRIP, v, residual<T, 1>(g, t / STRIP, n0 + t % STRIP));
    }
}

// 256 / W quads of columns x W walkers: walker w adds the parts w, w + W, ..., the walkers are joined in order.
template <class T, int W>
__global__ __launch_bounds__(256) void tfc_dense_join_kernel(const Args g, int splits) {
    constexpr int Q = 256 / W;
    __shared__ float lds[W > 1 ? W : 1][Q][4];
    const long nv = (g.n + 3) / 4, total = g.m * nv, slab = g.m * g.n;
    const int ql = threadIdx.x % Q, w = threadIdx.x / Q;
    const long i = (long)blockIdx.x * Q + ql;
    const long row = i / nv, col = (i - row * nv) * 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (i < total) {
        const float* p = g.part + row * g.n + col;
#pragma unroll 4
        for (int s = w; s < splits; s += W) {
            float x[4];
            tfc_load_f<float, 4>(p + s * slab, g.n - col, x);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += x[j];
        }
    }
    if constexpr (W > 1) {
#pragma unroll
        for (int j = 0; j < 4; ++j) lds[w][ql][j] = v[j];
        __syncthreads();
        if (w > 0) return;
#pragma unroll
        for (int k = 1; k < W; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += lds[k][ql][j];
    }
    if (i < total) epilogue_left<T, 4>(g, row, col, v);
}

// An empty contraction: the epilogue of zeros.
template <class T>
__global__ __launch_bounds__(256) void tfc_dense_empty_kernel(const Args g) {
    const long nv = (g.n + 3) / 4, total = g.m * nv;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
        const long row = i / nv, col = (i - row * nv) * 4;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        epilogue_left<T, 4>(g, row, col, v);
    }
}

// ------------------------------------------------------------------------------------------------ backward, elementwise
// dz / cst = act'(z) dy, for 16 bits times TFC_DZ_SCALE (both are undone in the products' factor), its second pieces `lo` elements behind
// the first (0: none), and the column sums of dz: a workgroup walks a slab of rows, cw threads side by side on a chunk of
// columns, 256 / cw rows at a time; its sums go to one partial row.  z null: act is the identity.
template <class T>
__global__ __launch_bounds__(256) void tfc_dense_dz_kernel(const T* __restrict__ dy, const void* __restrict__ z, long rows, long n,
                                                           int act, float cst, int cw, long slab, T* __restrict__ dz, long lo,
                                                           float* __restrict__ part) {
    constexpr int V = TfcType<T>::V;
    const int cl = threadIdx.x % cw, rl = threadIdx.x / cw, step = 256 / cw;
    const long c = ((long)blockIdx.x * cw + cl) * V, left = n - c;
    const long r0 = (long)blockIdx.y * slab, r1 = r0 + slab < rows ? r0 + slab : rows;
    float sum[V];
#pragma unroll
    for (int j = 0; j < V; ++j) sum[j] = 0.f;
    if (left > 0) {
        for (long r = r0 + rl; r < r1; r += step) {
            float g[V], x[V];
            tfc_load_f<T, V>(dy + r * n + c, left, g);
            if (z) {
                load_z<T, V>(z, rows * n, r * n + c, left, x);
                act_grad_apply<sizeof(T) == 2>(act, x);
#pragma unroll
                for (int j = 0; j < V; ++j) g[j] *= x[j];
            }
#pragma unroll
            for (int j = 0; j < V; ++j) {
                sum[j] += j < left ? g[j] : 0.f;
                if (sizeof(T) == 2) g[j] *= TFC_DZ_SCALE;
            }
            if (dz) tfc_store_f<T, V>(dz + r * n + c, left, g);
            if (sizeof(T) == 2 && lo) {
#pragma unroll
                for (int j = 0; j < V; ++j) g[j] = second_piece(T(), g[j]);
                tfc_store_f<T, V>(dz + lo + r * n + c, left, g);
            }
        }
    }
    if (!part) return;
    __shared__ float lds[256 * V];
#pragma unroll
    for (int j = 0; j < V; ++j) lds[(rl * V + j) * cw + cl] = sum[j];
    __syncthreads();
    if (rl == 0 && left > 0) {
        for (int k = 1; k < step; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) sum[j] += lds[(k * V + j) * cw + cl];
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] *= cst;
        tfc_store_f<float, V>(part + (long)blockIdx.y * n + c, left, sum);
    }
}

// ------------------------------------------------------------------------------------------------ host
struct Plan {
    int bm, bn;
    int64_t tiles_m, tiles_n, splits, k_split;
};

// What the kernel for large products asks of sizes and of operands.
bool deep_shape(int64_t m, int64_t n, int64_t k, int dtype) {
    return dtype != TFC_F32 && m >= DEEP && n >= DEEP && k % DEEP_K == 0;
}
bool deep_operands(const tfc_dense_desc& d) {
    return deep_shape(d.m, d.n, d.k, d.dtype) && (((uintptr_t)d.a | (uintptr_t)d.b) & 15) == 0 && d.lda % 8 == 0 && d.ldb % 8 == 0 &&
           (d.a_along_k || d.m % 8 == 0) && (d.b_along_k || d.n % 8 == 0);
}

// Tiles: 128 x 128, or narrower ones for a narrow C (64 x 64 moves twice as many operand bytes through LDS for each product).  Where
// the tiles alone do not put three workgroups (fp32: two, by LDS) on every CU the contraction is split, in parts of at least eight
// steps; and where the partial tiles would not stay in the caches (over 16 MB) in parts long enough that writing and adding them
// up takes less than half the time of the products: 1024 of k for 16 bits, 192 for fp32, whose products cost six times as much.
// deep: whether the kernel for large products may be taken.
Plan plan(int64_t m, int64_t n, int64_t k, int dtype, bool deep) {
    Plan p{};
    const bool wide = dtype == TFC_F32;
    const int64_t step = wide ? 32 : 64, steps = (k + step - 1) / step, want = wide ? 512 : 768;
    auto take = [&](int bm, int bn, int64_t want) {
        p.bm = bm, p.bn = bn;
        p.tiles_m = (m + bm - 1) / bm;
        p.tiles_n = (n + bn - 1) / bn;
        const int64_t have = p.tiles_m * p.tiles_n;
        p.splits = 1;
        if (have < want) {
            p.splits = std::max<int64_t>(1, std::min<int64_t>((want + have / 2) / have, steps / 8));
            if (p.splits * m * n * 4 > (16 << 20)) p.splits = std::max<int64_t>(1, std::min<int64_t>(p.splits, k / (wide ? 192 : 1024)));
        }
        const int64_t each = (steps + p.splits - 1) / p.splits;
        p.k_split = each * step;
        p.splits = steps ? (steps + each - 1) / each : 1;
        return have * p.splits >= 256;
    };
    if (deep && take(256, 256, 256)) return p;
    if (m > 64 && n > 64 && take(128, 128, want)) return p;
    if (m > 64 && take(128, 64, want)) return p;
    take(64, 64, want);
    return p;
}

// Whether the kernels for a few rows are taken.  A workgroup's share of B grows with k: along k (16 bits, 16 columns of 16384: 4.4 us,
// 9 with four rows; tiles 8) up to 32 KB a column.  Along the rows (16 bits, 4096 x 128: 6.1 us, 9 with four
// rows, tiles 8; 4096 x 4096: 14.2, 17, tiles 12.9, 14.5; fp32 4096 x 4096: 19, 21, tiles 28; 8192 x 64: 12.5, 13, the same) up to 2048 of 16
// bits, 4096 of fp32.
bool few_rows(const tfc_dense_desc& d) {
    const int64_t size = (int64_t)tfc_dtype_size(d.dtype);
    return d.a_along_k && d.m <= ROWS && d.k > 0 && d.k <= (d.b_along_k ? (1 << 15) / size : 1024 * size);
}

template <class T, int M>
int launch_rows(const Args& g, bool b_k, hipStream_t s) {
    if (b_k)
        hipLaunchKernelGGL((tfc_dense_rows_k_kernel<T, M>), dim3((unsigned)((g.n + COLS - 1) / COLS)), dim3(256), 0, s, g);
    else
        hipLaunchKernelGGL((tfc_dense_rows_n_kernel<T, M>), dim3((unsigned)((g.n + STRIP - 1) / STRIP)), dim3(1024), 0, s, g);
    TFC_LAUNCH_CHECK("tfc_dense_rows");
    return TFC_OK;
}
template <class T>
int dense_rows(const Args& g, bool b_k, hipStream_t s) {
    return g.m == 1 ? launch_rows<T, 1>(g, b_k, s) : g.m == 2 ? launch_rows<T, 2>(g, b_k, s) : launch_rows<T, ROWS>(g, b_k, s);
}

template <class T, bool AK, bool BK, int BM, int BN>
int launch_tile(const Args& g, const Plan& p, hipStream_t s) {
    const dim3 grid((unsigned)(p.tiles_m * p.tiles_n), (unsigned)p.splits);
    if (p.splits > 1)
        hipLaunchKernelGGL((tfc_dense_kernel<T, AK, BK, BM, BN, true>), grid, dim3(256), 0, s, g);
    else
        hipLaunchKernelGGL((tfc_dense_kernel<T, AK, BK, BM, BN, false>), grid, dim3(256), 0, s, g);
    TFC_LAUNCH_CHECK("tfc_dense");
    return TFC_OK;
}

template <class T, bool AK, bool BK>
int launch_layout(const Args& g, const Plan& p, hipStream_t s) {
    if constexpr (sizeof(T) == 2) {
        if (p.bn == 256) {
            const dim3 grid((unsigned)(p.tiles_m * p.tiles_n), (unsigned)p.splits);
            if (p.splits > 1)
                hipLaunchKernelGGL((tfc_dense_deep_kernel<T, AK, BK, true>), grid, dim3(512), 0, s, g);
            else
                hipLaunchKernelGGL((tfc_dense_deep_kernel<T, AK, BK, false>), grid, dim3(512), 0, s, g);
            TFC_LAUNCH_CHECK("tfc_dense_deep");
            return TFC_OK;
        }
    }
    if (p.bn == 128) return launch_tile<T, AK, BK, 128, 128>(g, p, s);
    if (p.bm == 128) return launch_tile<T, AK, BK, 128, 64>(g, p, s);
    return launch_tile<T, AK, BK, 64, 64>(g, p, s);
}

template <class T>
int dense(Args g, const Plan& p, bool a_k, bool b_k, hipStream_t s) {
    const long quads = g.m * ((g.n + 3) / 4);
    const unsigned flat = (unsigned)std::min<long>((quads + 255) / 256, 8192);
    if (g.k == 0) {
        hipLaunchKernelGGL(tfc_dense_empty_kernel<T>, dim3(flat), dim3(256), 0, s, g);
        TFC_LAUNCH_CHECK("tfc_dense_empty");
        return TFC_OK;
    }
    g.tiles_m = (int)p.tiles_m, g.tiles_n = (int)p.tiles_n, g.k_split = p.k_split;
    const int rc = !a_k ? launch_layout<T, false, false>(g, p, s)
                   : b_k ? launch_layout<T, true, true>(g, p, s)
                         : launch_layout<T, true, false>(g, p, s);
    if (rc || p.splits == 1) return rc;
    if (p.splits >= 32)  // (many parts: few columns, or they would fill the chip; walkers side by side keep the accesses in flight)
        hipLaunchKernelGGL((tfc_dense_join_kernel<T, 16>), dim3((unsigned)((quads + 15) / 16)), dim3(256), 0, s, g, (int)p.splits);
    else
        hipLaunchKernelGGL((tfc_dense_join_kernel<T, 1>), dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, s, g, (int)p.splits);
    TFC_LAUNCH_CHECK("tfc_dense_join");
    return TFC_OK;
}

struct DzPlan {
    int cw;
    int64_t chunks, slab, slabs;
};
DzPlan dz_plan(int64_t rows, int64_t n, int dtype) {
    DzPlan p{};
    const int64_t v = dtype == TFC_F32 ? 4 : 8, nv = (n + v - 1) / v;
    p.cw = 1;
    while (p.cw < nv && p.cw < 256) p.cw *= 2;
    p.chunks = (nv + p.cw - 1) / p.cw;
    const int64_t step = 256 / p.cw;
    const int64_t want = std::max<int64_t>(1, 2048 / p.chunks);  // slabs that fill the chip
    p.slab = std::max<int64_t>(4 * step, (rows + want - 1) / want);
    p.slabs = (rows + p.slab - 1) / p.slab;
    return p;
}

template <class T>
int dense_dz(const DzPlan& p, const void* dy, const void* z, int64_t rows, int64_t n, int act, float cst, void* dz, int64_t lo,
             float* part, hipStream_t s) {
    hipLaunchKernelGGL(tfc_dense_dz_kernel<T>, dim3((unsigned)p.chunks, (unsigned)p.slabs), dim3(256), 0, s, (const T*)dy, z, (long)rows,
                       (long)n, act, cst, p.cw, (long)p.slab, (T*)dz, (long)lo, part);
    TFC_LAUNCH_CHECK("tfc_dense_dz");
    return TFC_OK;
}

bool act_ok(int act) {
    return act == TFC_ACT_IDENTITY || act == TFC_ACT_SSP || act == TFC_ACT_SILU || act == TFC_ACT_TANH || act == TFC_ACT_ABS ||
           act == TFC_ACT_SIGMOID || act == TFC_ACT_GELU;
}

}  // namespace

// For operands of any layout, aligned or not.
static int64_t product_floats(int64_t m, int64_t n, int64_t k, int dtype) {
    if (m <= 0 || n <= 0 || k <= 0) return 0;
    int64_t splits = plan(m, n, k, dtype, false).splits;
    if (deep_shape(m, n, k, dtype)) splits = std::max(splits, plan(m, n, k, dtype, true).splits);
    return splits > 1 ? splits * m * n : 0;
}

extern "C" int64_t tfc_dense_workspace_floats(const tfc_dense_desc* d) {
    if (!d || d->m <= 0 || d->n <= 0 || d->k <= 0 || !tfc_dtype_ok(d->dtype) || few_rows(*d)) return 0;
    const int64_t splits = plan(d->m, d->n, d->k, d->dtype, deep_operands(*d)).splits;
    return splits > 1 ? splits * d->m * d->n : 0;
}

// A thread's offset in a tile has 32 bits: 256 rows, or a step of 64, of the longest row.
constexpr int64_t TFC_LD_MAX = 1 << 22;

// lo_a, lo_b: bytes from an operand's first pieces to its second ones (0: there are none).
static int dense_product(const tfc_dense_desc* d, int64_t lo_a, int64_t lo_b, float* workspace, int64_t workspace_floats,
                         tfc_stream_t stream) {
    TFC_REQUIRE(d, TFC_EINVAL, "tfc_dense: null descriptor");
    TFC_REQUIRE(tfc_dtype_ok(d->dtype), TFC_EINVAL, "tfc_dense: unknown dtype %d", (int)d->dtype);
    TFC_REQUIRE(act_ok(d->act), TFC_EINVAL, "tfc_dense: unknown activation %d", (int)d->act);
    TFC_REQUIRE(d->m >= 0 && d->n >= 0 && d->k >= 0, TFC_EINVAL, "tfc_dense: negative size");
    if (d->m == 0 || d->n == 0) return TFC_OK;
    TFC_REQUIRE(d->c && (d->k == 0 || (d->a && d->b)), TFC_EINVAL, "tfc_dense: null pointer");
    TFC_REQUIRE(d->a_along_k || !d->b_along_k, TFC_EUNSUPPORTED,
                "tfc_dense: an A that runs along its rows needs a B that runs along its columns");
    TFC_REQUIRE(d->lda >= 0 && d->ldb >= 0 && d->ldc >= d->n && (!d->residual || d->ldr >= 0), TFC_EINVAL, "tfc_dense: bad stride");
    const bool few = few_rows(*d) && !lo_b;
    const Plan p = d->k && !few ? plan(d->m, d->n, d->k, d->dtype, !lo_a && !lo_b && deep_operands(*d)) : Plan{64, 64, 1, 1, 1, 0};
    TFC_REQUIRE(d->lda < TFC_LD_MAX && d->ldb < TFC_LD_MAX, TFC_EUNSUPPORTED, "tfc_dense: operand rows of 2^22 elements or more");
    TFC_REQUIRE(p.tiles_m * p.tiles_n < (int64_t)1 << 31, TFC_EUNSUPPORTED, "tfc_dense: %lld x %lld has too many tiles",
                (long long)d->m, (long long)d->n);
    TFC_REQUIRE(p.splits == 1 || (workspace && workspace_floats >= p.splits * d->m * d->n), TFC_EINVAL,
                "tfc_dense: workspace too small");
    hipStream_t s = (hipStream_t)stream;
    TfcProfScope prof("tfc_dense", s);
    Args g{};
    g.a = {d->a, (long)d->lda}, g.b = {d->b, (long)d->ldb};
    g.m = d->m, g.n = d->n, g.k = d->k;
    g.c = d->c, g.ldc = d->ldc, g.bias = d->bias, g.res = d->residual, g.ldr = d->ldr, g.z = d->z;
    g.alpha = d->alpha, g.cst = d->act_cst, g.act = d->act, g.part = workspace;
    g.passes = lo_a || lo_b ? 2 : 1, g.lo_a = lo_a, g.lo_b = lo_b;
    if (few) return TFC_BY_DTYPE(d->dtype, dense_rows, g, d->b_along_k != 0, s);
    return TFC_BY_DTYPE(d->dtype, dense, g, p, d->a_along_k != 0, d->b_along_k != 0, s);
}

extern "C" int tfc_dense(const tfc_dense_desc* d, float* workspace, int64_t workspace_floats, tfc_stream_t stream) {
    return dense_product(d, 0, 0, workspace, workspace_floats, stream);
}

static int dense_dz_pass(const void* dy, const void* z, int64_t rows, int64_t n, int dtype, int act, float cst, void* dz, int64_t lo,
                         void* db, float* part, hipStream_t s) {
    if (rows == 0) return db ? tfc_join_columns(nullptr, 0, n, db, 0, nullptr, dtype, s) : TFC_OK;
    const DzPlan p = dz_plan(rows, n, dtype);
    {
        TfcProfScope prof("tfc_dense_dz", s);
        const int rc = TFC_BY_DTYPE(dtype, dense_dz, p, dy, act == TFC_ACT_IDENTITY ? nullptr : z, rows, n, act, cst, dz,
                                    lo, db ? part : nullptr, s);
        if (rc) return rc;
    }
    return db ? tfc_join_columns(part, p.slabs, n, db, 0, nullptr, dtype, s) : TFC_OK;
}

extern "C" int tfc_dense_keeps_z(int64_t n, int64_t k, int32_t act) { return act != TFC_ACT_IDENTITY && !tfc_dense_is_narrow(n, k); }

extern "C" int64_t tfc_dense_z_bytes(int64_t m, int64_t n, int32_t dtype) {
    return m > 0 && n > 0 && tfc_dtype_ok(dtype) ? m * n * (dtype == TFC_F32 ? 4 : dtype == TFC_BF16 ? 2 : 3) : 0;
}

// Pieces of the element type that dz is kept in.  One is what the matrix instruction takes; the gradients' error then is sqrt 2 of what
// their own rounding is worth.  Two take that away and double the products (backward pass in bf16 with one and two, in us:
// 16384 x 1024 x 4096: 389, 830; 200000 x 128 x 128: 103, 144; 414 x 1281 x 21: 29, 35).  bf16: one where there are elements enough on
// all sides for the errors to come out at that; a gradient of few elements, or from few of dz, may have several times its share.
// fp16: always two.  One piece of what lies below 2^-14 (a small dy, a saturated act') has 2^-25 as its error whatever its size, and
// a sum over n or m carries that into results that are not small; the second piece takes it to 2^-36 (training step with gelu in us,
// one and two: 16384 x 1024 x 4096: 622, 1033; 6912 x 512 x 2048: 144, 176; 200000 x 128 x 128: 181, 220).
// exact: the caller's choice of two.
static int dz_pieces(int64_t m, int64_t n, int64_t k, int dtype, int act, bool exact) {
    if (dtype == TFC_F32 || act == TFC_ACT_IDENTITY) return 1;
    return exact || dtype == TFC_F16 || std::min(m * n, std::min(m * k, n * k)) < 1 << 14 ? 2 : 1;
}

// The general backward pass's workspace: [dz | what one of its parts needs at a time], in floats.
struct BwdSpace {
    int64_t dz, rest;
};
static BwdSpace bwd_space(int64_t m, int64_t n, int64_t k, int dtype, int act, bool exact) {
    BwdSpace w{};
    if (act != TFC_ACT_IDENTITY) w.dz = (m * n * dz_pieces(m, n, k, dtype, act, exact) * (int64_t)tfc_dtype_size(dtype) + 15) / 16 * 4;
    w.rest = std::max(m > 0 && n > 0 ? dz_plan(m, n, dtype).slabs * n : 0,
                      std::max(product_floats(m, k, n, dtype),
                               std::max(product_floats(k, n, m, dtype), product_floats(n, k, m, dtype))));
    return w;
}

static int64_t bwd_floats(int64_t m, int64_t n, int64_t k, int dtype, int act, bool exact) {
    if (m < 0 || n < 0 || k < 0 || !tfc_dtype_ok(dtype)) return 0;
    if (m > 0 && tfc_dense_is_narrow(n, k)) return tfc_dense_narrow_partials(m) * (k * n + n);
    const BwdSpace w = bwd_space(m, n, k, dtype, act, exact);
    return w.dz + w.rest;
}

extern "C" int64_t tfc_dense_bwd_workspace_floats(int64_t m, int64_t n, int64_t k, int32_t dtype, int32_t act) {
    return bwd_floats(m, n, k, dtype, act, false);
}

extern "C" int64_t tfc_dense_bwd_desc_workspace_floats(const tfc_dense_bwd_desc* d) {
    return d ? bwd_floats(d->m, d->n, d->k, d->dtype, d->act, d->exact_dz != 0) : 0;
}

extern "C" int tfc_dense_bwd(const tfc_dense_bwd_desc* d, float* workspace, int64_t workspace_floats, tfc_stream_t stream) {
    TFC_REQUIRE(d, TFC_EINVAL, "tfc_dense_bwd: null descriptor");
    TFC_REQUIRE(tfc_dtype_ok(d->dtype), TFC_EINVAL, "tfc_dense_bwd: unknown dtype %d", (int)d->dtype);
    TFC_REQUIRE(act_ok(d->act), TFC_EINVAL, "tfc_dense_bwd: unknown activation %d", (int)d->act);
    TFC_REQUIRE(d->m >= 0 && d->n >= 0 && d->k >= 0, TFC_EINVAL, "tfc_dense_bwd: negative size");
    TFC_REQUIRE(d->ldx >= 0 && d->ldw >= 0, TFC_EINVAL, "tfc_dense_bwd: bad stride");
    if (!d->dx && !d->dw && !d->db) return TFC_OK;
    const int64_t m = d->m, n = d->n, k = d->k;
    TFC_REQUIRE(m == 0 || n == 0 || (d->dy && (k == 0 || (d->x && d->w))), TFC_EINVAL, "tfc_dense_bwd: null pointer");
    TFC_REQUIRE(m == 0 || n == 0 || d->z || !tfc_dense_keeps_z(n, k, d->act), TFC_EINVAL, "tfc_dense_bwd: activation %d needs z",
                (int)d->act);
    TFC_REQUIRE(workspace_floats >= tfc_dense_bwd_desc_workspace_floats(d) && (workspace || workspace_floats == 0), TFC_EINVAL,
                "tfc_dense_bwd: workspace too small");
    hipStream_t s = (hipStream_t)stream;
    if (m > 0 && tfc_dense_is_narrow(n, k)) return tfc_dense_narrow_bwd(d, workspace, s);
    const int64_t ldz = m > 1 ? n : 0;  // (one row: nothing strides)
    TFC_REQUIRE((!d->dx && !d->dw) || (ldz < TFC_LD_MAX && (!d->dx || d->ldw < TFC_LD_MAX) && (!d->dw || d->ldx < TFC_LD_MAX)), TFC_EUNSUPPORTED,
                "tfc_dense_bwd: operand rows of 2^22 elements or more");  // (before anything is launched)
    const bool exact = d->exact_dz != 0;
    const BwdSpace space = bwd_space(m, n, k, d->dtype, d->act, exact);
    const bool plain = d->act == TFC_ACT_IDENTITY;  // dz is dy
    const void* dz = plain ? d->dy : (const void*)workspace;
    float* rest = workspace + space.dz;
    const int64_t lo = dz_pieces(m, n, k, d->dtype, d->act, exact) == 2 ? m * n : 0;
    if (n > 0 && ((!plain && (d->dx || d->dw)) || d->db)) {
        const int rc = dense_dz_pass(d->dy, d->z, m, n, d->dtype, d->act, d->act_cst, plain || !(d->dx || d->dw) ? nullptr : workspace,
                                     d->dx || d->dw ? lo : 0, d->db, rest, s);
        if (rc) return rc;
    }
    tfc_dense_desc g{};
    g.alpha = d->alpha * d->act_cst * (plain || d->dtype == TFC_F32 ? 1.f : 1.f / TFC_DZ_SCALE);
    g.act_cst = 1.f, g.act = TFC_ACT_IDENTITY, g.dtype = d->dtype;
    if (d->dx) {  // dz W^T
        g.m = m, g.n = k, g.k = n;
        g.a = dz, g.lda = ldz, g.a_along_k = 1;
        g.b = d->w, g.ldb = d->ldw, g.b_along_k = !d->w_along_k;
        g.c = d->dx, g.ldc = k;
        const int rc = dense_product(&g, 2 * lo, 0, rest, space.rest, stream);
        if (rc) return rc;
    }
    if (d->dw) {  // x^T dz, or its transpose, in the weight's own order
        g.k = m, g.a_along_k = g.b_along_k = 0;
        if (d->w_along_k) {
            g.m = n, g.n = k;
            g.a = dz, g.lda = ldz, g.b = d->x, g.ldb = d->ldx;
        } else {
            g.m = k, g.n = n;
            g.a = d->x, g.lda = d->ldx, g.b = dz, g.ldb = ldz;
        }
        g.c = d->dw, g.ldc = g.n;
        return dense_product(&g, d->w_along_k ? 2 * lo : 0, d->w_along_k ? 0 : 2 * lo, rest, space.rest, stream);
    }
    return TFC_OK;
}
