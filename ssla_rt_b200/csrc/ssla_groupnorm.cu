// ssla_groupnorm.cu -- group norm with an activation, channels last
// (include/ssla_ops.h).
//
// A slab is what shares one mean and variance: the positions of one sample
// times the channels of one group.
//   - small slabs (k_gn_slab): a few lanes or one CTA hold a slab in
//     registers; one read, two-pass statistics, one write;
//   - others: k_gn_sums leaves every slab's shifted sums per slice of the
//     positions in the workspace, k_gn_apply joins them (in 64 bits) and
//     writes the outputs.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "ssla_ops.cuh"

namespace ssla {
namespace ops {
namespace {

constexpr int kGnThreads = 256;

struct GnArgs {
    const float *weight, *bias;
    long long x_sample, x_pos, y_sample, y_pos;
    int n, positions, channels, groups, width;     // width: channels of a group
    int act;
    float eps;
};

// y / (1 + e^-y); where e^-y overflows the limit is -0.  16-bit outputs take
// the fast exponential and quotient (their errors, about 2^-21 here, are far
// below half a step of the output, 2^-9 or 2^-12), 32-bit ones do not.
template <typename T> __device__ __forceinline__ float silu(float y) {
    if constexpr (sizeof(T) == 2) return __fdividef(y, 1.0f + __expf(-y));
    else return y / (1.0f + expf(-y));
}

template <typename T>
__device__ __forceinline__ float gn_finish(float x, float mean, float rstd, float w, float b, int act) {
    const float y = fmaf((x - mean) * rstd, w, b);
    return act == SSLA_ACT_SILU ? silu<T>(y) : y;
}

// ---- small slabs: LPS threads each hold EPT vectors of a slab -------------
template <int LPS> __device__ __forceinline__ float slab_sum(float v, float* red) {
#pragma unroll
    for (int m = (LPS < 32 ? LPS : 32) / 2; m; m >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, m);
    if constexpr (LPS > 32) {
        __syncthreads();
        if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < LPS / 32; ++w) v += red[w];
    }
    return v;
}

template <typename T, int VEC, int LPS, int EPT>
__global__ void __launch_bounds__(kGnThreads) k_gn_slab(GnArgs a, const T* x, T* y) {
    __shared__ float red[kGnThreads / 32];
    const int lane = threadIdx.x % LPS;
    const long long slab = static_cast<long long>(blockIdx.x) * (kGnThreads / LPS) + threadIdx.x / LPS;
    const bool on = slab < static_cast<long long>(a.n) * a.groups;
    const int n = on ? static_cast<int>(slab / a.groups) : 0, g = on ? static_cast<int>(slab % a.groups) : 0;
    const int wv = a.width / VEC, vecs = a.positions * wv;
    const T* xp = x + n * a.x_sample + g * a.width;
    float v[EPT][VEC];
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < EPT; ++e) {
        const int k = e * LPS + lane;
        if (on && k < vecs) {
            const int p = k / wv;
            load_vec<T, VEC>(xp + p * a.x_pos + (k - p * wv) * VEC, v[e]);
#pragma unroll
            for (int j = 0; j < VEC; ++j) sum += v[e][j];
        }
    }
    const float inv = 1.0f / (static_cast<float>(a.positions) * static_cast<float>(a.width));
    const float mean = slab_sum<LPS>(sum, red) * inv;
    float sq = 0.0f;
#pragma unroll
    for (int e = 0; e < EPT; ++e)
        if (on && e * LPS + lane < vecs)
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float d = v[e][j] - mean;
                sq = fmaf(d, d, sq);
            }
    const float rstd = 1.0f / sqrtf(slab_sum<LPS>(sq, red) * inv + a.eps);
    T* yp = y + n * a.y_sample + g * a.width;
#pragma unroll
    for (int e = 0; e < EPT; ++e) {
        const int k = e * LPS + lane;
        if (on && k < vecs) {
            const int p = k / wv, c = (k - p * wv) * VEC;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const int ch = g * a.width + c + j;
                v[e][j] = gn_finish<T>(v[e][j], mean, rstd, a.weight ? __ldg(a.weight + ch) : 1.0f,
                                       a.bias ? __ldg(a.bias + ch) : 0.0f, a.act);
            }
            store_vec<T, VEC>(yp + p * a.y_pos + c, v[e]);
        }
    }
}

// ---- large slabs ------------------------------------------------------------
// CTA (slice, group chunk, sample): positions [p0, p1) of `gpc` whole groups.
// Thread (tx, ty): channel vector tx (+ multiples of TX where one group is
// wider than the CTA), positions p0 + ty, p0 + ty + TY, ...
struct GnSplit {
    int splits, chunks, gpc, tx, ty;
};

__device__ __forceinline__ float gn_shift(float x) { return fabsf(x) <= 3.402823466e38f ? x : 0.0f; }

template <typename T, int VEC>
__global__ void __launch_bounds__(kGnThreads) k_gn_sums(GnArgs a, GnSplit s, const T* x, float2* part) {
    __shared__ float2 red[kGnThreads];
    const int n = blockIdx.z, g0 = blockIdx.y * s.gpc, ng = min(s.gpc, a.groups - g0);
    const int wv = a.width / VEC, cv = ng * wv;
    const int p0 = static_cast<int>(static_cast<long long>(a.positions) * blockIdx.x / s.splits);
    const int p1 = static_cast<int>(static_cast<long long>(a.positions) * (blockIdx.x + 1) / s.splits);
    const int tx = threadIdx.x % s.tx, ty = threadIdx.x / s.tx;
    const T* xn = x + n * a.x_sample + static_cast<long long>(g0) * a.width;
    float s1 = 0.0f, s2 = 0.0f;
    if (ty < s.ty)
        for (int c = tx; c < cv; c += s.tx) {
            // the first position's first channel of the group as the shift
            const float shift = gn_shift(to_f<T>(xn[c / wv * a.width]));
            const T* xp = xn + c * VEC;
#pragma unroll 4
            for (int p = p0 + ty; p < p1; p += s.ty) {
                float v[VEC];
                load_vec<T, VEC>(xp + p * a.x_pos, v);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float d = v[j] - shift;
                    s1 += d;
                    s2 = fmaf(d, d, s2);
                }
            }
        }
    red[threadIdx.x] = make_float2(s1, s2);
    __syncthreads();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    for (int g = warp; g < ng; g += kGnThreads / 32) {
        const int w = ng == 1 ? min(s.tx, wv) : wv, lo = ng == 1 ? 0 : g * wv;
        float a1 = 0.0f, a2 = 0.0f;
        for (int k = lane; k < w * s.ty; k += 32) {
            const float2 r = red[k / w * s.tx + lo + k % w];
            a1 += r.x;
            a2 += r.y;
        }
#pragma unroll
        for (int m = 16; m; m >>= 1) {
            a1 += __shfl_xor_sync(0xFFFFFFFFu, a1, m);
            a2 += __shfl_xor_sync(0xFFFFFFFFu, a2, m);
        }
        if (lane == 0) part[(static_cast<size_t>(n) * a.groups + g0 + g) * s.splits + blockIdx.x] = make_float2(a1, a2);
    }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kGnThreads) k_gn_stats(GnArgs a, int splits, const T* x, const float2* part, float2* stat) {
    // one warp per slab: joins the slices' sums in 64 bits
    const long long slab = static_cast<long long>(blockIdx.x) * (kGnThreads / 32) + threadIdx.x / 32;
    if (slab >= static_cast<long long>(a.n) * a.groups) return;
    const int lane = threadIdx.x % 32;
    double a1 = 0.0, a2 = 0.0;
    for (int k = lane; k < splits; k += 32) {
        const float2 r = part[slab * splits + k];
        a1 += r.x;
        a2 += r.y;
    }
#pragma unroll
    for (int m = 16; m; m >>= 1) {
        a1 += __shfl_xor_sync(0xFFFFFFFFu, a1, m);
        a2 += __shfl_xor_sync(0xFFFFFFFFu, a2, m);
    }
    if (lane == 0) {
        const double inv = 1.0 / (static_cast<double>(a.positions) * a.width);
        const float shift = gn_shift(to_f<T>(x[slab / a.groups * a.x_sample + slab % a.groups * a.width]));
        const double m = a1 * inv, var = a2 * inv - m * m;   // a non-finite value: NaN
        stat[slab] = make_float2(static_cast<float>(shift + m), static_cast<float>(1.0 / sqrt((var < 0.0 ? 0.0 : var) + a.eps)));
    }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kGnThreads) k_gn_apply(GnArgs a, GnSplit s, const T* x, T* y, const float2* stat) {
    const int n = blockIdx.z, g0 = blockIdx.y * s.gpc, ng = min(s.gpc, a.groups - g0);
    const int wv = a.width / VEC, cv = ng * wv;
    const int p0 = static_cast<int>(static_cast<long long>(a.positions) * blockIdx.x / s.splits);
    const int p1 = static_cast<int>(static_cast<long long>(a.positions) * (blockIdx.x + 1) / s.splits);
    const int tx = threadIdx.x % s.tx, ty = threadIdx.x / s.tx;
    if (ty >= s.ty) return;
    const int ch0 = g0 * a.width;
    for (int c = tx; c < cv; c += s.tx) {
        const float2 st = stat[static_cast<size_t>(n) * a.groups + g0 + c / wv];
        float w[VEC], b[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            w[j] = a.weight ? __ldg(a.weight + ch0 + c * VEC + j) : 1.0f;
            b[j] = a.bias ? __ldg(a.bias + ch0 + c * VEC + j) : 0.0f;
        }
        const T* xp = x + n * a.x_sample + ch0 + c * VEC;
        T* yp = y + n * a.y_sample + ch0 + c * VEC;
#pragma unroll 4
        for (int p = p0 + ty; p < p1; p += s.ty) {
            float v[VEC];
            load_vec<T, VEC>(xp + p * a.x_pos, v);
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = gn_finish<T>(v[j], st.x, st.y, w[j], b[j], a.act);
            store_vec<T, VEC>(yp + p * a.y_pos, v);
        }
    }
}

// ---- host ----------------------------------------------------------------
int check_gn(const SslaGroupNorm* a) {
    const char* who = "group norm";
    if (!a) return fail(SSLA_ERR_ARG, "%s: null argument", who);
    if (!dtype_ok(a->dtype)) return fail(SSLA_ERR_ARG, "%s: dtype %d is not an SSLA_DT_* value", who, a->dtype);
    if (a->activation != SSLA_ACT_NONE && a->activation != SSLA_ACT_SILU)
        return fail(SSLA_ERR_ARG, "%s: activation %d is not an SSLA_ACT_* value", who, a->activation);
    if (a->n < 0 || a->positions < 0 || a->channels < 0)
        return fail(SSLA_ERR_ARG, "%s: a size is negative", who);
    if (a->groups < 1 || a->channels % a->groups)
        return fail(SSLA_ERR_ARG, "%s: %d channels in %d groups", who, a->channels, a->groups);
    if (!(a->eps >= 0.0f) || !std::isfinite(a->eps)) return fail(SSLA_ERR_ARG, "%s: eps %g", who, a->eps);
    if (a->n == 0 || a->positions == 0 || a->channels == 0) return SSLA_OK;
    if (a->positions > (1LL << 40) / a->channels || a->channels > (1 << 24) || a->n > INT_MAX / a->groups)
        return fail(SSLA_ERR_ARG, "%s: too large", who);
    if (!a->x || !a->y) return fail(SSLA_ERR_ARG, "%s: null pointer", who);
    const int sz = dtype_size(a->dtype);
    if (!aligned(a->x, sz) || !aligned(a->y, sz) || !aligned(a->weight, 4) || !aligned(a->bias, 4))
        return fail(SSLA_ERR_ARG, "%s: a pointer is not aligned to its element", who);
    const long long most = LLONG_MAX / 16 / std::max(a->n, a->positions);
    for (long long s : {a->x_sample, a->x_pos, a->y_sample, a->y_pos})
        if (s < 0 || s > most) return fail(SSLA_ERR_ARG, "%s: a stride is negative or too large", who);
    const bool by_sample = (a->positions == 1 || a->y_pos >= a->channels) &&
                           (a->n == 1 || a->y_sample >= (a->positions - 1) * a->y_pos + a->channels);
    const bool by_pos = (a->n == 1 || a->y_sample >= a->channels) &&
                        (a->positions == 1 || a->y_pos >= (a->n - 1) * a->y_sample + a->channels);
    if (!by_sample && !by_pos) return fail(SSLA_ERR_ARG, "%s: y overlaps itself", who);
    auto bytes = [&](long long s, long long p) {
        return static_cast<size_t>((a->n - 1) * s + (a->positions - 1) * p + a->channels) * sz;
    };
    const size_t xn = bytes(a->x_sample, a->x_pos), yn = bytes(a->y_sample, a->y_pos), wn = 4ull * a->channels;
    const bool same = a->x == a->y && (a->n == 1 || a->x_sample == a->y_sample) &&
                      (a->positions == 1 || a->x_pos == a->y_pos);
    if (!same && overlaps(a->x, xn, a->y, yn)) return fail(SSLA_ERR_ARG, "%s: y overlaps x", who);
    if ((a->weight && overlaps(a->y, yn, a->weight, wn)) || (a->bias && overlaps(a->y, yn, a->bias, wn)))
        return fail(SSLA_ERR_ARG, "%s: y overlaps weight or bias", who);
    return SSLA_OK;
}

int gn_vec(const SslaGroupNorm* a) {
    const int sz = dtype_size(a->dtype), width = a->channels / a->groups;
    const long long all = width | (a->positions > 1 ? a->x_pos | a->y_pos : 0) | (a->n > 1 ? a->x_sample | a->y_sample : 0);
    for (int v = 16 / sz; v > 1; v >>= 1)
        if (all % v == 0 && aligned(a->x, v * sz) && aligned(a->y, v * sz)) return v;
    return 1;
}

// Threads that hold a small slab and vectors of each; false: a large slab.
bool gn_small(const SslaGroupNorm* a, int vec, int* lps, int* ept) {
    const long long vecs = static_cast<long long>(a->positions) * (a->channels / a->groups / vec);
    const int most = vec >= 8 ? 4 : 8;             // registers: 32 values a thread
    if (vecs <= 8) *lps = 8, *ept = 1;
    else if (vecs <= 16) *lps = 16, *ept = 1;
    else if (vecs <= 32) *lps = 32, *ept = 1;
    else if (vecs <= 64) *lps = 32, *ept = 2;
    else if (vecs <= 128) *lps = 32, *ept = 4;
    else if (vecs <= kGnThreads * most) *lps = kGnThreads, *ept = most;
    else return false;
    return true;
}

GnSplit gn_split(const SslaGroupNorm* a, int vec) {
    GnSplit s;
    const int wv = a->channels / a->groups / vec;
    s.gpc = std::max(1, std::min(a->groups, kGnThreads / wv));
    s.chunks = (a->groups + s.gpc - 1) / s.gpc;
    s.tx = std::min(kGnThreads, s.gpc * wv);
    s.ty = std::max(1, kGnThreads / s.tx);
    // about eight CTAs per SM in all, at least four rounds of positions each
    const long long ctas = static_cast<long long>(a->n) * s.chunks;
    const long long want = std::max<long long>(1, 148 * 8 / ctas);
    s.splits = static_cast<int>(std::max<long long>(1, std::min<long long>(want, a->positions / (4 * s.ty))));
    return s;
}

size_t gn_bytes(const SslaGroupNorm* a) {
    if (a->n == 0 || a->positions == 0 || a->channels == 0) return 0;
    const int vec = gn_vec(a);
    int lps, ept;
    if (gn_small(a, vec, &lps, &ept)) return 0;
    return static_cast<size_t>(a->n) * a->groups * (gn_split(a, vec).splits + 1) * sizeof(float2);
}

}  // namespace
}  // namespace ops
}  // namespace ssla

using namespace ssla::ops;

extern "C" {

int ssla_group_norm_workspace(const SslaGroupNorm* a, size_t* bytes) {
    if (!bytes) return fail(SSLA_ERR_ARG, "group norm: null argument");
    if (const int rc = check_gn(a); rc != SSLA_OK) return rc;
    *bytes = gn_bytes(a);
    return SSLA_OK;
}

int ssla_group_norm(const SslaGroupNorm* a, void* workspace, size_t workspace_bytes, void* stream) {
    if (const int rc = check_gn(a); rc != SSLA_OK) return rc;
    if (a->n == 0 || a->positions == 0 || a->channels == 0) return SSLA_OK;
    const size_t need = gn_bytes(a);
    if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
        return fail(SSLA_ERR_ARG, "group norm: workspace of %zu bytes, %zu needed, 16-byte aligned", workspace_bytes, need);
    OnDevice dev(a->device);
    if (dev.err != SSLA_OK) return dev.err;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    GnArgs d;
    d.weight = a->weight; d.bias = a->bias;
    d.x_sample = a->x_sample; d.x_pos = a->x_pos; d.y_sample = a->y_sample; d.y_pos = a->y_pos;
    d.n = a->n; d.positions = a->positions; d.channels = a->channels; d.groups = a->groups;
    d.width = a->channels / a->groups;
    d.act = a->activation; d.eps = a->eps;
    const int vec = gn_vec(a);
    auto run = [&](auto t, auto v) {
        using T = decltype(t);
        constexpr int V = decltype(v)::value;
        const T* x = static_cast<const T*>(a->x);
        T* y = static_cast<T*>(a->y);
        int lps, ept;
        const long long slabs = static_cast<long long>(a->n) * a->groups;
        if (gn_small(a, vec, &lps, &ept)) {
            const unsigned grid = static_cast<unsigned>((slabs + kGnThreads / lps - 1) / (kGnThreads / lps));
            auto go = [&](auto l, auto e) {
                k_gn_slab<T, V, decltype(l)::value, decltype(e)::value><<<grid, kGnThreads, 0, st>>>(d, x, y);
                return launched("k_gn_slab");
            };
            using std::integral_constant;
            if (lps == 8) return go(integral_constant<int, 8>(), integral_constant<int, 1>());
            if (lps == 16) return go(integral_constant<int, 16>(), integral_constant<int, 1>());
            if (lps == 32 && ept == 1) return go(integral_constant<int, 32>(), integral_constant<int, 1>());
            if (lps == 32 && ept == 2) return go(integral_constant<int, 32>(), integral_constant<int, 2>());
            if (lps == 32) return go(integral_constant<int, 32>(), integral_constant<int, 4>());
            return go(integral_constant<int, kGnThreads>(), integral_constant<int, (V >= 8 ? 4 : 8)>());
        }
        const GnSplit s = gn_split(a, vec);
        float2* stat = static_cast<float2*>(workspace);
        float2* part = stat + slabs;
        if (s.chunks > 65535 || a->n > 65535) {
            return fail(SSLA_ERR_ARG, "group norm: more than 65535 samples or groups of large slabs");
        }
        const dim3 grid(s.splits, s.chunks, a->n);
        k_gn_sums<T, V><<<grid, kGnThreads, 0, st>>>(d, s, x, part);
        k_gn_stats<T, V><<<static_cast<unsigned>((slabs + 7) / 8), kGnThreads, 0, st>>>(d, s.splits, x, part, stat);
        k_gn_apply<T, V><<<grid, kGnThreads, 0, st>>>(d, s, x, y, stat);
        return launched("group norm");
    };
    auto by_vec = [&](auto t) {
        using std::integral_constant;
        if constexpr (sizeof(t) == 2)
            if (vec == 8) return run(t, integral_constant<int, 8>());
        if (vec == 4) return run(t, integral_constant<int, 4>());
        if (vec == 2) return run(t, integral_constant<int, 2>());
        return run(t, integral_constant<int, 1>());
    };
    return a->dtype == SSLA_DT_F32 ? by_vec(float()) : a->dtype == SSLA_DT_BF16 ? by_vec(__nv_bfloat16())
                                                                                  : by_vec(__half());
}

}  // extern "C"
