// One AdamW step over many parameter tensors.  With g the gradient (times min(1, max_norm / (|all g| + 1e-6)) when a largest
// norm is given), t the tensor's own step count:
//
//   m = b1 m + (1 - b1) g        p = (1 - lr wd) p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//   v = b2 v + (1 - b2) g g
//
// all in fp32 whatever the parameters' type, every operation rounded once (no contraction), so that a program that writes the
// line above out in torch operations gets the same bits with 32-bit moments.
//
// Moments in 8 bits: m and sqrt(v) are kept as e4m3 codes (sign, 4 exponent, 3 mantissa bits) with one power-of-two scale for
// every 256 neighbours, which brings the largest magnitude among them into [128, 256): 2^17 of range below it, and the binade
// above it free for what rounds up.  sqrt(v) and not v, because the range of v is twice that in bits.  Rounding to a code is up or
// down at random with the probability that keeps the value on average: to the nearest, v would never shrink, for a step takes
// at most 0.1 % off it (b2 = 0.999) and half a code is 6 %.  The random bits are a hash of (seed, step, tensor, element): the
// step is a function of its inputs.  A second moment that is not zero never rounds to zero (its root is a divisor).  What is not
// finite is kept as NaN in its own place and leaves its block's scale alone.
//
// Bound by HBM: 28 bytes an element for fp32 with 32-bit moments, 10 for bf16 with 8-bit ones.  One launch takes up to 48
// tensors, whose addresses travel in the kernel's arguments (nothing to copy, nothing to keep alive under a captured graph); a
// workgroup takes 4096 elements of one tensor, a wave 256 at a time - the block that shares a scale, so its largest magnitude
// is one reduction over the wave.  Measured: 33.0 M elements of fp32 in 16 tensors, moments in 32 bits 160 us (5.8 TB/s), the gradients'
// sums of squares before it 43 us; 62.7 M of bf16 in 12 tensors, moments in 8 bits 137 us (4.6 TB/s).
#include "tfc_types.h"

#include <algorithm>
#include <climits>

#pragma clang fp contract(off)

namespace {

constexpr int TENSORS = 48;   // of one launch: 48 x 72 + 49 x 4 bytes of the 4 KB of arguments
constexpr int CHUNK = 4096;   // elements of a workgroup
constexpr int QBLOCK = 256;   // elements that share a scale
constexpr int SQ_CHUNK = 16384;

struct Group {
    tfc_adamw_tensor t[TENSORS];
    int first[TENSORS + 1];  // first workgroup of each tensor
    int n;
};

struct Hyper {
    double lr, b1, b2, eps, wd;
    const float* lr_dev;
};

struct TensorStep {  // what the update needs of (hyper-parameters, step count), one record for every tensor
    float decay, step, inv_root, clip;
    uint32_t key, pad[3];
};

__device__ __forceinline__ int find_tensor(const Group& g, int block) {  // the last tensor whose first workgroup is <= block
    int lo = 0, hi = g.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (g.first[mid] <= block)
            lo = mid;
        else
            hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ uint32_t mixed(uint32_t x) {
    x = (x ^ (x >> 16)) * 0x6C8E9CF5u;
    x = (x ^ (x >> 15)) * 0x35297A4Du;
    return x ^ (x >> 16);
}

// ---- sums of squares, one double for each workgroup (products in double too: they do not overflow where fp32 gradients do not)
template <class T>
__global__ __launch_bounds__(256) void tfc_grad_sumsq_kernel(const Group g, double* __restrict__ part) {
    constexpr int V = TfcType<T>::V;
    const int k = find_tensor(g, blockIdx.x);
    const T* p = (const T*)g.t[k].g;
    const long n = g.t[k].n, base = (long)((int)blockIdx.x - g.first[k]) * SQ_CHUNK;
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < SQ_CHUNK / (256 * V); ++i) {
        const long at = base + ((long)i * 256 + threadIdx.x) * V;
        float v[V];
        tfc_load_f<T, V>(p + at, n - at, v);
#pragma unroll
        for (int j = 0; j < V; ++j) s += (double)v[j] * (double)v[j];
    }
    __shared__ double lds[256];
    lds[threadIdx.x] = s;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
        if ((int)threadIdx.x < o) lds[threadIdx.x] += lds[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) part[blockIdx.x] = lds[0];
}

// ---- start of a step: the gradients' norm from its partial sums, every tensor's step count, and what follows from both
__global__ __launch_bounds__(1024) void tfc_adamw_begin_kernel(const Group g, const Hyper h, uint32_t seed,
                                                               const double* __restrict__ part, long n_part, double max_norm,
                                                               float* __restrict__ norm_out, TensorStep* __restrict__ out) {
    __shared__ double lds[1024];
    float clip = 1.f;
    if (part) {
        double s = 0.0;
        for (long i = threadIdx.x; i < n_part; i += 1024) s += part[i];
        lds[threadIdx.x] = s;
        __syncthreads();
        for (int o = 512; o > 0; o >>= 1) {
            if ((int)threadIdx.x < o) lds[threadIdx.x] += lds[threadIdx.x + o];
            __syncthreads();
        }
        const double norm = sqrt(lds[0]);
        const double c = max_norm / (norm + 1e-6);
        clip = (float)(c > 1.0 ? 1.0 : c);  // (NaN stays NaN: a norm that is no number leaves none in the parameters)
        if (threadIdx.x == 0 && norm_out) *norm_out = (float)norm;
    }
    const int k = threadIdx.x;
    if (k >= g.n) return;
    int* count = g.t[k].step;
    const int t = *count + 1;
    *count = t;
    const double lr = h.lr_dev ? (double)*h.lr_dev : h.lr;
    TensorStep r;
    r.decay = (float)(1.0 - lr * h.wd);
    r.step = (float)(lr / (1.0 - pow(h.b1, (double)t)));
    r.inv_root = (float)(1.0 / sqrt(1.0 - pow(h.b2, (double)t)));
    r.clip = clip;
    r.key = mixed(seed + 0x9E3779B9u * (uint32_t)t + 0x632BE5ABu * (uint32_t)g.t[k].index);
    r.pad[0] = r.pad[1] = r.pad[2] = 0;
    out[k] = r;
}

// ---- e4m3 codes
constexpr uint32_t INF_BITS = 0x7F800000u;

// Largest of 64 lanes' numbers, in every lane.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#define TFC_MAX_STEP(CTRL, ROWS)                                                                             \
    {                                                                                                        \
        const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);         \
        v = v > o ? v : o;                                                                                   \
    }
    TFC_MAX_STEP(0xB1, 0xF)   // quad_perm [1,0,3,2]
    TFC_MAX_STEP(0x4E, 0xF)   // quad_perm [2,3,0,1]
    TFC_MAX_STEP(0x141, 0xF)  // row_half_mirror
    TFC_MAX_STEP(0x140, 0xF)  // row_mirror
    TFC_MAX_STEP(0x142, 0xA)  // row_bcast15 -> rows 1, 3
    TFC_MAX_STEP(0x143, 0xC)  // row_bcast31 -> rows 2, 3
#undef TFC_MAX_STEP
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

// Scale exponent (biased) of a block whose largest finite magnitude has these bits: magnitude 2^-(e - 127) in [128, 256).
__device__ __forceinline__ int scale_exponent(uint32_t top) {
    const int e = (int)(top >> 23) - 7;
    return e < 1 ? 1 : e;
}

// Four values to codes and their block's scale.  Rounding up or down at random is the conversion instruction's own: it adds the
// upper 20 of the 32 random bits to what is dropped (16 bits of randomness here, the others zero).
template <bool ROOT>
__device__ __forceinline__ uint32_t to_codes(const float (&x)[4], const uint32_t (&random)[4], int& e) {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) top = max(top, __float_as_uint(x[j]) & 0x7FFFFFFFu);
    top = wave_max(top);
    const bool odd = top >= INF_BITS;  // (the same in all lanes) something is not finite: it counts for nothing
    if (odd) {
        top = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t b = __float_as_uint(x[j]) & 0x7FFFFFFFu;
            top = max(top, b < INF_BITS ? b : 0u);
        }
        top = wave_max(top);
    }
    e = scale_exponent(top);
    const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
    int w = 0;
#define TFC_TO_CODE(J)                                                                                       \
    {                                                                                                        \
        float y = x[J] * inv;                                                                                \
        if (ROOT) y = x[J] > 0.f ? fmaxf(y, 0x1p-9f) : 0.f; /* a root that is not zero does not become zero */ \
        w = __builtin_amdgcn_cvt_sr_fp8_f32(y, random[J], w, J);                                             \
    }
    TFC_TO_CODE(0) TFC_TO_CODE(1) TFC_TO_CODE(2) TFC_TO_CODE(3)
#undef TFC_TO_CODE
    if (odd) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if ((__float_as_uint(x[j]) & INF_BITS) == INF_BITS) w = (int)(((uint32_t)w & ~(0xFFu << (8 * j))) | (0x7Fu << (8 * j)));
    }
    return (uint32_t)w;
}

__device__ __forceinline__ void from_codes(uint32_t w, float scale, float (&x)[4]) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    x[0] = lo[0] * scale, x[1] = lo[1] * scale, x[2] = hi[0] * scale, x[3] = hi[1] * scale;
}

template <class T, int BITS>
__global__ __launch_bounds__(256) void tfc_adamw_kernel(const Group g, const TensorStep* __restrict__ steps, float b1, float c1,
                                                        float b2, float c2, float eps) {
    const int k = find_tensor(g, blockIdx.x);
    const long n = g.t[k].n;
    T* p = (T*)g.t[k].p;
    const T* gr = (const T*)g.t[k].g;
    const TensorStep st = steps[k];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long base = (long)((int)blockIdx.x - g.first[k]) * CHUNK;
#pragma unroll
    for (int i = 0; i < CHUNK / (4 * QBLOCK); ++i) {
        const long blk = base + (long)(i * 4 + wave) * QBLOCK;
        if (blk >= n) break;  // (the whole wave)
        const long at = blk + lane * 4, left = n - at;
        float pv[4], gv[4], m[4], r[4], v[4];
        tfc_load_f<T, 4>(p + at, left, pv);
        tfc_load_f<T, 4>(gr + at, left, gv);
        uint8_t *mc = nullptr, *vc = nullptr;
        if constexpr (BITS == 32) {
            tfc_load_f<float, 4>((const float*)g.t[k].m + at, left, m);
            tfc_load_f<float, 4>((const float*)g.t[k].v + at, left, v);
        } else {
            mc = (uint8_t*)g.t[k].m + at;  // (whole blocks: the padding behind n holds zeros)
            vc = (uint8_t*)g.t[k].v + at;
            from_codes(*(const uint32_t*)mc, __uint_as_float((uint32_t)g.t[k].m_scale[blk / QBLOCK] << 23), m);
            from_codes(*(const uint32_t*)vc, __uint_as_float((uint32_t)g.t[k].v_scale[blk / QBLOCK] << 23), r);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = r[j] * r[j];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float gg = gv[j] * st.clip;
            m[j] = m[j] * b1 + gg * c1;
            v[j] = v[j] * b2 + gg * gg * c2;
            r[j] = sqrtf(v[j]);
            pv[j] = pv[j] * st.decay - m[j] / (r[j] * st.inv_root + eps) * st.step;
        }
        tfc_store_f<T, 4>(p + at, left, pv);
        if constexpr (BITS == 32) {
            tfc_store_f<float, 4>((float*)g.t[k].m + at, left, m);
            tfc_store_f<float, 4>((float*)g.t[k].v + at, left, v);
        } else {
            if (left < 4) {  // the padding stays zero
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j >= left) m[j] = r[j] = 0.f;
            }
            uint32_t hm[4], hv[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t h = mixed((uint32_t)(at + j) ^ st.key ^ ((uint32_t)((at + j) >> 32) * 0x2545F491u));
                hm[j] = h << 16;
                hv[j] = h & 0xFFFF0000u;
            }
            int em, ev;
            *(uint32_t*)mc = to_codes<false>(m, hm, em);
            *(uint32_t*)vc = to_codes<true>(r, hv, ev);
            if (lane == 0) {
                g.t[k].m_scale[blk / QBLOCK] = (uint8_t)em;
                g.t[k].v_scale[blk / QBLOCK] = (uint8_t)ev;
            }
        }
    }
}

int64_t fill_group(const tfc_adamw_tensor* t, int n, int64_t chunk, Group& g) {
    int64_t blocks = 0;
    g.n = n;
    for (int i = 0; i < n; ++i) {
        g.t[i] = t[i];
        g.first[i] = (int)blocks;
        blocks += (t[i].n + chunk - 1) / chunk;
        if (blocks > INT_MAX) return -1;
    }
    for (int i = n; i <= TENSORS; ++i) g.first[i] = (int)blocks;
    return blocks;
}

// The tensors are taken TENSORS at a time.
template <class F>
int by_groups(const tfc_adamw_tensor* t, int n_tensors, int64_t chunk, F&& f) {
    for (int i = 0; i < n_tensors; i += TENSORS) {
        Group g{};
        const int64_t blocks = fill_group(t + i, std::min(TENSORS, n_tensors - i), chunk, g);
        if (blocks < 0) return tfc_set_error(TFC_EINVAL, "tfc_adamw: more than 2^31 workgroups of elements in %d tensors", g.n);
        const int rc = f(g, i, blocks);
        if (rc) return rc;
    }
    return TFC_OK;
}

int check_tensors(const char* who, const tfc_adamw_tensor* t, int32_t n, int32_t dtype) {
    TFC_REQUIRE(n >= 0 && (n == 0 || t), TFC_EINVAL, "%s: bad tensor table", who);
    TFC_REQUIRE(tfc_dtype_ok(dtype), TFC_EINVAL, "%s: unknown dtype %d", who, (int)dtype);
    for (int i = 0; i < n; ++i)
        TFC_REQUIRE(t[i].n >= 0 && (t[i].n == 0 || t[i].g), TFC_EINVAL, "%s: tensor %d: bad size or null gradient", who, i);
    return TFC_OK;
}

template <class T>
int grad_sumsq(const tfc_adamw_tensor* t, int n, double* part, hipStream_t s) {
    int64_t at = 0;
    return by_groups(t, n, SQ_CHUNK, [&](const Group& g, int, int64_t blocks) {
        if (blocks == 0) return (int)TFC_OK;
        hipLaunchKernelGGL(tfc_grad_sumsq_kernel<T>, dim3((unsigned)blocks), dim3(256), 0, s, g, part + at);
        TFC_LAUNCH_CHECK("tfc_grad_sumsq");
        at += blocks;
        return (int)TFC_OK;
    });
}

template <class T>
int adamw_update(const Group& g, int64_t blocks, int bits, const tfc_adamw_hyper& h, const TensorStep* steps, hipStream_t s) {
    const float b1 = (float)h.beta1, c1 = (float)(1.0 - h.beta1), b2 = (float)h.beta2, c2 = (float)(1.0 - h.beta2);
    if (bits == 32)
        hipLaunchKernelGGL((tfc_adamw_kernel<T, 32>), dim3((unsigned)blocks), dim3(256), 0, s, g, steps, b1, c1, b2, c2, (float)h.eps);
    else
        hipLaunchKernelGGL((tfc_adamw_kernel<T, 8>), dim3((unsigned)blocks), dim3(256), 0, s, g, steps, b1, c1, b2, c2, (float)h.eps);
    TFC_LAUNCH_CHECK("tfc_adamw");
    return TFC_OK;
}

}  // namespace

extern "C" int64_t tfc_grad_sumsq_partials(const tfc_adamw_tensor* t, int32_t n_tensors) {
    int64_t blocks = 0;
    for (int i = 0; t && i < n_tensors; ++i)
        if (t[i].n > 0) blocks += (t[i].n + SQ_CHUNK - 1) / SQ_CHUNK;
    return blocks;
}

extern "C" int tfc_grad_sumsq(const tfc_adamw_tensor* t, int32_t n_tensors, int32_t dtype, double* partials, tfc_stream_t stream) {
    const int bad = check_tensors("tfc_grad_sumsq", t, n_tensors, dtype);
    if (bad) return bad;
    if (tfc_grad_sumsq_partials(t, n_tensors) == 0) return TFC_OK;
    TFC_REQUIRE(partials, TFC_EINVAL, "tfc_grad_sumsq: null output");
    TfcProfScope prof("tfc_grad_sumsq", (hipStream_t)stream);
    return TFC_BY_DTYPE(dtype, grad_sumsq, t, n_tensors, partials, (hipStream_t)stream);
}

extern "C" int64_t tfc_adamw_workspace_bytes(int32_t n_tensors) { return std::max(n_tensors, 0) * (int64_t)sizeof(TensorStep); }

extern "C" int tfc_adamw_step(const tfc_adamw_tensor* t, int32_t n_tensors, int32_t dtype, int32_t state_bits,
                              const tfc_adamw_hyper* hyper, const double* partials, int64_t n_partials, float* norm, void* workspace,
                              int64_t workspace_bytes, tfc_stream_t stream) {
    const int bad = check_tensors("tfc_adamw_step", t, n_tensors, dtype);
    if (bad) return bad;
    TFC_REQUIRE(state_bits == 32 || state_bits == 8, TFC_EINVAL, "tfc_adamw_step: moments of %d bits (32 or 8)", (int)state_bits);
    TFC_REQUIRE(hyper, TFC_EINVAL, "tfc_adamw_step: null hyper-parameters");
    TFC_REQUIRE(n_partials >= 0 && (n_partials == 0 || partials), TFC_EINVAL, "tfc_adamw_step: null partial sums");
    if (n_tensors == 0) return TFC_OK;
    for (int i = 0; i < n_tensors; ++i) {
        TFC_REQUIRE(t[i].step, TFC_EINVAL, "tfc_adamw_step: tensor %d: null step count", i);
        TFC_REQUIRE(t[i].n == 0 || (t[i].p && t[i].m && t[i].v && (state_bits == 32 || (t[i].m_scale && t[i].v_scale))), TFC_EINVAL,
                    "tfc_adamw_step: tensor %d: null pointer", i);
        TFC_REQUIRE(state_bits == 32 || t[i].n == 0 || (((uintptr_t)t[i].m | (uintptr_t)t[i].v) & 3) == 0, TFC_EINVAL,
                    "tfc_adamw_step: tensor %d: 8-bit moments must start at a multiple of 4 bytes", i);
    }
    TFC_REQUIRE(workspace && workspace_bytes >= tfc_adamw_workspace_bytes(n_tensors), TFC_EINVAL,
                "tfc_adamw_step: workspace too small");
    hipStream_t s = (hipStream_t)stream;
    TfcProfScope prof("tfc_adamw", s);
    const Hyper h{hyper->lr, hyper->beta1, hyper->beta2, hyper->eps, hyper->weight_decay, hyper->lr_device};
    TensorStep* steps = (TensorStep*)workspace;
    return by_groups(t, n_tensors, CHUNK, [&](const Group& g, int at, int64_t blocks) {
        hipLaunchKernelGGL(tfc_adamw_begin_kernel, dim3(1), dim3(1024), 0, s, g, h, hyper->seed, hyper->max_norm > 0 ? partials : nullptr,
                           (long)n_partials, hyper->max_norm, norm, steps + at);
        TFC_LAUNCH_CHECK("tfc_adamw_begin");
        if (blocks == 0) return (int)TFC_OK;
        return TFC_BY_DTYPE(dtype, adamw_update, g, blocks, state_bits, *hyper, steps + at, s);
    });
}
