// ssla_groupnorm.cu -- group norm with an activation, channels last
// (include/ssla_ops.h).
//
// A slab is what shares one mean and variance: the positions of one sample
// times the channels of one group.
//   - small slabs (k_gn_slab): a few lanes or one CTA hold a slab in
//     registers; one read, two-pass statistics, one write;
//   - slabs that fit the shared memory of a cluster of up to eight CTAs
//     (k_gn_cluster): one read, one write (8 x 5,120 x 96 in 8 groups, fp32: 11.4
//     us, bf16 17.2);
//   - others: k_gn_sums leaves every slab's sums per slice of the positions in
//     the workspace, k_gn_apply joins them and writes the outputs; the second
//     read mostly comes from L2 (8 x 20,000 x 120 in 3 groups, fp32: 53 us, bf16
//     34).
//
// The last two take the moments in one pass.  A thread sums the differences of
// its values, and their squares, from the mean of its own first vector in 32
// bits, and folds them into moments about zero in 64 (fold), in which they are
// joined.  The mean of k of n values is at most sqrt(n / k) of their deviation
// from the mean of all, so that the squares add up to at most 1 + n / k times
// what is left of them, whatever the values are: n / k is a thread's vectors
// between folds, at most kGnFold or a cluster's rounds.  (A shift by one value
// of the whole slab lost three digits where that value was an outlier.)
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <numeric>
#include <type_traits>

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
    int wide;                                      // weight and bias are 16-byte aligned
    int stream;                                    // x and y are too large for L2
    float eps;
    double inv;                                    // 1 / values of a slab
};

// A vector's elements two at a time (packed 32-bit arithmetic); each
// component is the ordinary operation.
template <int VEC> __device__ __forceinline__ float add_up(const float (&x)[VEC]) {
    if constexpr (VEC == 1) return x[0];
    else {
        float2 s = make_float2(x[0], x[1]);
#pragma unroll
        for (int j = 2; j < VEC; j += 2) s = __fadd2_rn(s, make_float2(x[j], x[j + 1]));
        return s.x + s.y;
    }
}
// s1 += sum of (x - shift), s2 += sum of their squares.
template <int VEC> __device__ __forceinline__ void moments(const float (&x)[VEC], float shift, float2& s1, float2& s2) {
    if constexpr (VEC == 1) {
        const float d = x[0] - shift;
        s1.x += d;
        s2.x = fmaf(d, d, s2.x);
    } else {
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
            const float2 d = __fadd2_rn(make_float2(x[j], x[j + 1]), make_float2(-shift, -shift));
            s1 = __fadd2_rn(s1, d);
            s2 = __ffma2_rn(d, d, s2);
        }
    }
}

// Adds n values, given as the sums of their differences from `shift` and of
// those' squares, to moments about zero (a mean of 2^20 deviations still
// leaves 13 bits of the variance there).
__device__ __forceinline__ void fold(double2& m, int n, float shift, float2 s1, float2 s2) {
    const double d = static_cast<double>(s1.x) + s1.y, ns = static_cast<double>(n) * shift;
    m.x += d + ns;
    m.y += (static_cast<double>(s2.x) + s2.y) + shift * (2.0 * d + ns);
}

// SiLU, y / (1 + e^-y), with the hardware's exponential and reciprocal:
// relative errors of 2^-22 each and |y| 2^-23 from rounding the exponent,
// which is below 2^-20 where the value counts and below half a step of 16-bit
// outputs everywhere.  For y < -87 the reciprocal itself is below the normal
// numbers, while y e^y, which is what is left of SiLU, is one down to -91.9.
__device__ __forceinline__ float exp2_hw(float x) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x));
    return e;
}
__device__ __forceinline__ float rcp_hw(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
constexpr float kNegLog2e = -1.44269504f, kSiluTail = 125.0f;   // the exponent from where 32-bit results go by halves
template <typename T, int VEC> __device__ __forceinline__ void silu(float (&x)[VEC]) {
    constexpr int N = (VEC + 1) / 2;
    float2 y[N];
    float most = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        y[j] = make_float2(x[2 * j], 2 * j + 1 < VEC ? x[2 * j + 1] : 0.0f);
        float2 o;
        if constexpr (std::is_same_v<T, __nv_bfloat16>) {
            // the quotient times 2^32, so that it stays normal as far as bf16 goes (the sum rounds the exponent to 2^-19)
            const float2 t = __ffma2_rn(y[j], make_float2(kNegLog2e, kNegLog2e), make_float2(-32.0f, -32.0f));
            o = __fmul2_rn(__fmul2_rn(y[j], make_float2(0x1p-32f, 0x1p-32f)),
                           make_float2(rcp_hw(0x1p-32f + exp2_hw(t.x)), rcp_hw(0x1p-32f + exp2_hw(t.y))));
        } else {                                   // (fp16 ends above all this)
            const float2 t = __fmul2_rn(y[j], make_float2(kNegLog2e, kNegLog2e));
            o = __fmul2_rn(y[j], make_float2(rcp_hw(1.0f + exp2_hw(t.x)), rcp_hw(1.0f + exp2_hw(t.y))));
            if (sizeof(T) == 4) most = fmaxf(most, fmaxf(t.x, t.y));
        }
        x[2 * j] = o.x;
        if (2 * j + 1 < VEC) x[2 * j + 1] = o.y;
    }
    if (sizeof(T) == 4 && most > kSiluTail)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float v = j % 2 ? y[j / 2].y : y[j / 2].x, t = v * kNegLog2e, h = exp2_hw(-0.5f * t);
            if (t > kSiluTail) x[j] = (v * h) * h;
        }
}

// x <- act((x - mean) * rstd * w + b)
template <typename T, int VEC>
__device__ __forceinline__ void gn_finish(float (&x)[VEC], float mean, float rstd, const float (&w)[VEC], const float (&b)[VEC],
                                          int act) {
    if constexpr (VEC == 1) {
        x[0] = fmaf((x[0] - mean) * rstd, w[0], b[0]);
        if (act == SSLA_ACT_SILU) silu<T, 1>(x);
    } else {
        const float2 m = make_float2(-mean, -mean), r = make_float2(rstd, rstd);
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
            const float2 y = __ffma2_rn(__fmul2_rn(__fadd2_rn(make_float2(x[j], x[j + 1]), m), r), make_float2(w[j], w[j + 1]),
                                        make_float2(b[j], b[j + 1]));
            x[j] = y.x;
            x[j + 1] = y.y;
        }
        if (act == SSLA_ACT_SILU) silu<T, VEC>(x);
    }
}

// VEC weights (or the given constant) from channel c on.
template <int VEC>
__device__ __forceinline__ void channel_params(const float* p, int c, float none, bool wide, float (&x)[VEC]) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[j] = none;
    if (!p) return;
    if constexpr (VEC >= 4) {
        if (wide) {
#pragma unroll
            for (int j = 0; j < VEC; j += 4) {
                const float4 f = __ldg(reinterpret_cast<const float4*>(p + c + j));
                x[j] = f.x; x[j + 1] = f.y; x[j + 2] = f.z; x[j + 3] = f.w;
            }
            return;
        }
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) x[j] = __ldg(p + c + j);
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

// Resident CTAs per SM that the forms of one or two vectors are built for.
// What bounds them is how many warps hide the loads and the exponentials:
// 16,384 rows of 16 groups of 128 (bf16, SiLU) take 39 us (3.5 TB/s) with four
// CTAs of two vectors a thread, 40 with one vector, 46 with three CTAs of twice
// the slabs, 59 where six CTAs make the registers spill.
constexpr int kGnSlabCtas = 4;

// A thread takes UNR slabs at a time, gridDim.x * (slabs of a CTA) apart:
// the launch makes that a multiple of the groups where it can, so that a
// thread's channels, and the weights it keeps, stay the same.
template <typename T, int VEC, int LPS, int EPT, int UNR>
__global__ void __launch_bounds__(kGnThreads, LPS <= 32 && EPT <= 2 ? kGnSlabCtas : 1) k_gn_slab(GnArgs a, const T* x, T* y) {
    __shared__ float red[kGnThreads / 32];
    constexpr int kPer = kGnThreads / LPS;
    const int lane = threadIdx.x % LPS;
    const unsigned slabs = static_cast<unsigned>(a.n) * a.groups, stride = gridDim.x * kPer;   // below 2^31 (check_gn)
    const int wv = a.width / VEC, vecs = a.positions * wv;
    const float inv = 1.0f / (static_cast<float>(a.positions) * static_cast<float>(a.width));
    const bool wide = VEC >= 4 && a.wide;
    float w[EPT][VEC], b[EPT][VEC];
    int kept = -1;
    // a multiple of the groups apart, a thread's slabs need no division
    const unsigned groups = a.groups, turn = stride / groups, first = blockIdx.x * kPer + threadIdx.x / LPS;
    const bool steady = turn * groups == stride;
    const unsigned n_first = first / groups, g_first = first - n_first * groups;
    unsigned round = 0;
    auto params = [&](int g) {
#pragma unroll
        for (int e = 0; e < EPT; ++e) {
            const int k = e * LPS + lane;
            if (k < vecs) {
                const int c = (a.positions == 1 ? k : k % wv) * VEC;
                channel_params<VEC>(a.weight, g * a.width + c, 1.0f, wide, w[e]);
                channel_params<VEC>(a.bias, g * a.width + c, 0.0f, wide, b[e]);
            }
        }
        kept = g;
    };
    if (first < slabs) params(g_first);             // in flight with the first values
    // all threads of a CTA run the same rounds (wide slabs meet at barriers)
    for (unsigned base = blockIdx.x * kPer; base < slabs; base += UNR * stride, round += UNR) {
        float v[UNR][EPT][VEC], mean[UNR], rstd[UNR];
        int n[UNR], g[UNR];
#pragma unroll
        for (int u = 0; u < UNR; ++u) {
            const unsigned slab = base + u * stride + threadIdx.x / LPS;
            const unsigned nn = steady ? n_first + (round + u) * turn : slab / groups;
            n[u] = slab < slabs ? static_cast<int>(nn) : -1;
            g[u] = slab < slabs ? static_cast<int>(steady ? g_first : slab - nn * groups) : 0;
            const T* xp = x + (n[u] >= 0 ? n[u] * a.x_sample + static_cast<long long>(g[u]) * a.width : 0);
#pragma unroll
            for (int e = 0; e < EPT; ++e) {
                const int k = e * LPS + lane;
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[u][e][j] = 0.0f;
                if (n[u] >= 0 && k < vecs) {
                    const int p = a.positions == 1 ? 0 : k / wv;
                    load_vec_hint<T, VEC>(xp + p * a.x_pos + (k - p * wv) * VEC, v[u][e], a.stream);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < UNR; ++u) {
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < EPT; ++e) sum += add_up<VEC>(v[u][e]);
            mean[u] = slab_sum<LPS>(sum, red) * inv;
        }
#pragma unroll
        for (int u = 0; u < UNR; ++u) {
            float2 none = make_float2(0.0f, 0.0f), sq = none;
#pragma unroll
            for (int e = 0; e < EPT; ++e)
                if (e * LPS + lane < vecs) moments<VEC>(v[u][e], mean[u], none, sq);
            const float var = slab_sum<LPS>(sq.x + sq.y, red) * inv + a.eps;
            rstd[u] = sizeof(T) == 2 ? rsqrtf(var) : 1.0f / sqrtf(var);
        }
#pragma unroll
        for (int u = 0; u < UNR; ++u) {
            if (n[u] < 0) continue;
            T* yp = y + n[u] * a.y_sample + static_cast<long long>(g[u]) * a.width;
            if (g[u] != kept) params(g[u]);
#pragma unroll
            for (int e = 0; e < EPT; ++e) {
                const int k = e * LPS + lane;
                if (k < vecs) {
                    const int p = a.positions == 1 ? 0 : k / wv, c = (k - p * wv) * VEC;
                    gn_finish<T, VEC>(v[u][e], mean[u], rstd[u], w[e], b[e], a.act);
                    store_vec_hint<T, VEC>(yp + p * a.y_pos + c, v[u][e], a.stream);
                }
            }
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

constexpr int kGnFold = 32;                       // vectors of a thread between two folds

template <typename T, int VEC>
__global__ void __launch_bounds__(kGnThreads, 8) k_gn_sums(GnArgs a, GnSplit s, const T* x, double2* part) {
    __shared__ double2 red[kGnThreads];
    const int n = blockIdx.z, g0 = blockIdx.y * s.gpc, ng = min(s.gpc, a.groups - g0);
    const int wv = a.width / VEC, cv = ng * wv;
    const int p0 = static_cast<int>(static_cast<long long>(a.positions) * blockIdx.x / s.splits);
    const int p1 = static_cast<int>(static_cast<long long>(a.positions) * (blockIdx.x + 1) / s.splits);
    const int tx = threadIdx.x % s.tx, ty = threadIdx.x / s.tx;
    const T* xn = x + n * a.x_sample + static_cast<long long>(g0) * a.width;
    red[threadIdx.x] = make_double2(0.0, 0.0);     // (here rather than in registers, which are what limits the CTAs)
    if (ty < s.ty)
        for (int c = tx; c < cv; c += s.tx) {      // (more than one: all of one group)
            const T* xp = xn + c * VEC;
            for (int p = p0 + ty; p < p1;) {
                const int end = min(p1, p + kGnFold * s.ty);
                float v[VEC];
                load_vec<T, VEC>(xp + p * a.x_pos, v);
                const float shift = add_up<VEC>(v) * (1.0f / VEC);
                const int count = ((end - p - 1) / s.ty + 1) * VEC;
                float2 s1 = make_float2(0.0f, 0.0f), s2 = s1;
#pragma unroll 4
                for (; p < end; p += s.ty) {
                    load_vec<T, VEC>(xp + p * a.x_pos, v);
                    moments<VEC>(v, shift, s1, s2);
                }
                fold(red[threadIdx.x], count, shift, s1, s2);
            }
        }
    __syncthreads();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    for (int g = warp; g < ng; g += kGnThreads / 32) {
        const int w = ng == 1 ? min(s.tx, wv) : wv, lo = ng == 1 ? 0 : g * wv;
        double a1 = 0.0, a2 = 0.0;
        for (int k = lane; k < w * s.ty; k += 32) {
            const double2 r = red[k / w * s.tx + lo + k % w];
            a1 += r.x;
            a2 += r.y;
        }
#pragma unroll
        for (int m = 16; m; m >>= 1) {
            a1 += __shfl_xor_sync(0xFFFFFFFFu, a1, m);
            a2 += __shfl_xor_sync(0xFFFFFFFFu, a2, m);
        }
        if (lane == 0)
            part[(static_cast<size_t>(n) * a.groups + g0 + g) * s.splits + blockIdx.x] = make_double2(a1, a2);
    }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kGnThreads, VEC * sizeof(T) < 16 ? 6 : VEC == 4 ? 5 : 4)
k_gn_apply(GnArgs a, GnSplit s, const T* x, T* y, const double2* part) {
    extern __shared__ float2 stat[];               // (mean, 1 / deviation) of the CTA's groups
    const int n = blockIdx.z, g0 = blockIdx.y * s.gpc, ng = min(s.gpc, a.groups - g0);
    const int wv = a.width / VEC, cv = ng * wv;
    const int p0 = static_cast<int>(static_cast<long long>(a.positions) * blockIdx.x / s.splits);
    const int p1 = static_cast<int>(static_cast<long long>(a.positions) * (blockIdx.x + 1) / s.splits);
    const int tx = threadIdx.x % s.tx, ty = threadIdx.x / s.tx;
    const int ch0 = g0 * a.width;
    const T* xn = x + n * a.x_sample + ch0;
    asm volatile("griddepcontrol.wait;" ::: "memory");   // the sums of the kernel before
    // one warp a slab joins the slices' sums
    for (int g = threadIdx.x / 32; g < ng; g += kGnThreads / 32) {
        double a1 = 0.0, a2 = 0.0;
        for (int k = threadIdx.x % 32; k < s.splits; k += 32) {
            const double2 r = part[(static_cast<size_t>(n) * a.groups + g0 + g) * s.splits + k];
            a1 += r.x;
            a2 += r.y;
        }
#pragma unroll
        for (int m = 16; m; m >>= 1) {
            a1 += __shfl_xor_sync(0xFFFFFFFFu, a1, m);
            a2 += __shfl_xor_sync(0xFFFFFFFFu, a2, m);
        }
        if (threadIdx.x % 32 == 0) {
            const double m = a1 * a.inv, var = a2 * a.inv - m * m;   // a non-finite value: NaN
            stat[g] = make_float2(static_cast<float>(m), static_cast<float>(1.0 / sqrt((var < 0.0 ? 0.0 : var) + a.eps)));
        }
    }
    __syncthreads();
    if (ty >= s.ty) return;
    for (int c = tx; c < cv; c += s.tx) {
        const float2 st = stat[c / wv];
        float w[VEC], b[VEC];
        channel_params<VEC>(a.weight, ch0 + c * VEC, 1.0f, VEC >= 4 && a.wide, w);
        channel_params<VEC>(a.bias, ch0 + c * VEC, 0.0f, VEC >= 4 && a.wide, b);
        const T* xp = xn + c * VEC;
        T* yp = y + n * a.y_sample + ch0 + c * VEC;
#pragma unroll 4
        for (int p = p0 + ty; p < p1; p += s.ty) {
            float v[VEC];
            load_vec<T, VEC>(xp + p * a.x_pos, v);
            gn_finish<T, VEC>(v, st.x, st.y, w, b, a.act);
            store_vec<T, VEC>(yp + p * a.y_pos, v);
        }
    }
}

// ---- slabs that fit the shared memory of a cluster -----------------------------
// One read: each CTA of a cluster keeps its slice of the positions (of `gpc`
// whole groups of one sample) in shared memory -- every thread its own
// vectors, in its own places --, the CTAs read one another's sums through
// distributed shared memory, and each writes its slice's outputs.
constexpr int kGnClusterThreads = 1024;
constexpr int kGnClusterBytes = 184 * 1024;    // of values
constexpr int kGnClusterSmem = 227 * 1024 - kGnClusterThreads * static_cast<int>(sizeof(double2));   // and all but the static part

struct GnCluster {
    int ctas, chunks, gpc, tx, ty, rounds;         // rounds: position steps of a thread
};

template <typename T, int VEC>
__global__ void __launch_bounds__(kGnClusterThreads) k_gn_cluster(GnArgs a, GnCluster s, const T* x, T* y) {
    extern __shared__ __align__(16) uint8_t gn_smem[];
    __shared__ double2 red[kGnClusterThreads];
    Pack<T, VEC>* tile = reinterpret_cast<Pack<T, VEC>*>(gn_smem);
    double2* sums = reinterpret_cast<double2*>(gn_smem + static_cast<size_t>(s.rounds) * kGnClusterThreads * sizeof(Pack<T, VEC>));
    double2* part = sums + s.gpc;                  // max(32, gpc)
    float2* stat = reinterpret_cast<float2*>(part + max(32, s.gpc));
    const int rank = blockIdx.x, n = blockIdx.z, g0 = blockIdx.y * s.gpc, ng = min(s.gpc, a.groups - g0);
    const int wv = a.width / VEC, cv = ng * wv;
    const int p0 = static_cast<int>(static_cast<long long>(a.positions) * rank / s.ctas);
    const int p1 = static_cast<int>(static_cast<long long>(a.positions) * (rank + 1) / s.ctas);
    const int tid = threadIdx.x, tx = tid % s.tx, ty = tid / s.tx, ch0 = g0 * a.width;
    const bool on = ty < s.ty && tx < cv;
    const int g = on ? tx / wv : 0;
    const T* xn = x + n * a.x_sample + ch0;
    float2 s1 = make_float2(0.0f, 0.0f), s2 = s1;
    double2 m = make_double2(0.0, 0.0);
    float w[VEC], b[VEC];
    if (on) {
        const T* xp = xn + tx * VEC;
        constexpr int kBatch = 8;                  // loads in flight
        float shift = 0.0f;
        int count = 0;
        for (int r0 = 0; r0 < s.rounds; r0 += kBatch) {
            Pack<T, VEC> k[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                const int p = p0 + ty + (r0 + i) * s.ty;
                if (p < p1) k[i] = *reinterpret_cast<const Pack<T, VEC>*>(xp + p * a.x_pos);
            }
            if (r0 == 0 && p0 + ty < p1) {
                float v[VEC];
                unpack_vec<T, VEC>(k[0], v);
                shift = add_up<VEC>(v) * (1.0f / VEC);
            }
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                if (p0 + ty + (r0 + i) * s.ty >= p1) break;
                tile[(r0 + i) * kGnClusterThreads + tid] = k[i];
                float v[VEC];
                unpack_vec<T, VEC>(k[i], v);
                moments<VEC>(v, shift, s1, s2);
                count += VEC;
            }
        }
        fold(m, count, shift, s1, s2);
    }
    if (on) {
        channel_params<VEC>(a.weight, ch0 + tx * VEC, 1.0f, VEC >= 4 && a.wide, w);
        channel_params<VEC>(a.bias, ch0 + tx * VEC, 0.0f, VEC >= 4 && a.wide, b);
    }
    red[tid] = m;
    __syncthreads();
    const int warp = tid / 32, lane = tid % 32;
    // group i's threads in `slices` parts, a warp each, then the parts
    const int slices = max(1, kGnClusterThreads / 32 / ng);
    for (int u = warp; u < ng * slices; u += kGnClusterThreads / 32) {
        const int i = u % ng, sl = u / ng;
        double a1 = 0.0, a2 = 0.0;
        const int t0 = wv < 32 ? lane + 32 * sl : sl, dt = wv < 32 ? 32 * slices : slices, q0 = wv < 32 ? 0 : lane, dq = wv < 32 ? 1 : 32;
        for (int t = t0; t < s.ty; t += dt)
            for (int q = q0; q < wv; q += dq) {
                const double2 r = red[t * s.tx + i * wv + q];
                a1 += r.x;
                a2 += r.y;
            }
#pragma unroll
        for (int m = 16; m; m >>= 1) {
            a1 += __shfl_xor_sync(0xFFFFFFFFu, a1, m);
            a2 += __shfl_xor_sync(0xFFFFFFFFu, a2, m);
        }
        if (lane == 0) part[u] = make_double2(a1, a2);
    }
    __syncthreads();
    for (int i = tid; i < ng; i += kGnClusterThreads) {
        double2 r = part[i];
        for (int sl = 1; sl < slices; ++sl) {
            r.x += part[i + sl * ng].x;
            r.y += part[i + sl * ng].y;
        }
        sums[i] = r;
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    for (int i = warp; i < ng; i += kGnClusterThreads / 32) {   // lane c: CTA c's sums
        double a1 = 0.0, a2 = 0.0;
        if (lane < s.ctas) {
            uint32_t there;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                         : "=r"(there) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(sums + i))), "r"(lane));
            asm volatile("ld.shared::cluster.v2.f64 {%0, %1}, [%2];" : "=d"(a1), "=d"(a2) : "r"(there) : "memory");
        }
#pragma unroll
        for (int m = 4; m; m >>= 1) {
            a1 += __shfl_xor_sync(0xFFFFFFFFu, a1, m);
            a2 += __shfl_xor_sync(0xFFFFFFFFu, a2, m);
        }
        if (lane == 0) {
            const double m = a1 * a.inv, var = a2 * a.inv - m * m;   // a non-finite value: NaN
            stat[i] = make_float2(static_cast<float>(m), 1.0f / sqrtf(static_cast<float>((var < 0.0 ? 0.0 : var) + a.eps)));
        }
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // this CTA has read its peers' sums
    __syncthreads();
    const float2 st = stat[g];
    T* yp = y + n * a.y_sample + ch0 + tx * VEC;
    if (on)
#pragma unroll 4
        for (int r = 0; r < s.rounds; ++r) {
            const int p = p0 + ty + r * s.ty;
            if (p >= p1) break;
            float v[VEC];
            unpack_vec<T, VEC>(tile[r * kGnClusterThreads + tid], v);
            gn_finish<T, VEC>(v, st.x, st.y, w, b, a.act);
            store_vec<T, VEC>(yp + p * a.y_pos, v);
        }
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");     // no CTA leaves while a peer may read it
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
    // positions and samples are stepped over in 32 bits, by a few thousand at most
    if (a->positions > std::min((1LL << 40) / a->channels, INT_MAX - 65536LL) || a->channels > (1 << 24) ||
        a->n > (INT_MAX - 65536) / a->groups)
        return fail(SSLA_ERR_ARG, "%s: %d samples of %d positions, %d channels: too large", who, a->n, a->positions, a->channels);
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
    else if (vecs <= 16) *lps = 8, *ept = 2;
    else if (vecs <= 32) *lps = 16, *ept = 2;
    else if (vecs <= 64) *lps = 32, *ept = 2;
    else if (vecs <= 128) *lps = 32, *ept = 4;
    else if (vecs <= kGnThreads * most) *lps = kGnThreads, *ept = most;
    else return false;
    return true;
}

size_t gn_cluster_bytes(const GnCluster& c, int vec, int sz) {
    return static_cast<size_t>(c.rounds) * kGnClusterThreads * vec * sz + c.gpc * (sizeof(double2) + sizeof(float2)) +
           std::max(32, c.gpc) * sizeof(double2);
}

// The smallest cluster, of whole groups of at least 64 contiguous bytes,
// whose slices fit and that gives (nearly) every SM a CTA; the widest that
// fits where none does; false: a slab does not fit.  Small clusters, because
// the GPU's parts do not all hold two of eight such CTAs: eight maps of
// 80 x 64 x 96 took two turns, 18.9 us, in 16 clusters of eight, and 12.7 us in
// 32 of four before the groups' sums were spread over all warps; 11.4 us now.
bool gn_cluster(const SslaGroupNorm* a, int vec, GnCluster* c) {
    const int wv = a->channels / a->groups / vec, sz = dtype_size(a->dtype);
    if (wv > kGnClusterThreads || a->n > 65535) return false;
    bool found = false;
    for (int ctas = 1; ctas <= 8; ctas *= 2)
        for (int parts = 1; parts <= 8; parts *= 2) {
            GnCluster k;
            k.ctas = ctas;
            k.gpc = std::min((a->groups + parts - 1) / parts, kGnClusterThreads / wv);
            if (parts > 1 && static_cast<long long>(k.gpc) * wv * vec * sz < 64) continue;
            k.chunks = (a->groups + k.gpc - 1) / k.gpc;
            if (k.chunks > 65535) continue;
            k.tx = k.gpc * wv;
            k.ty = kGnClusterThreads / k.tx;
            k.rounds = ((a->positions + ctas - 1) / ctas + k.ty - 1) / k.ty;
            if (k.rounds > kGnClusterBytes / (kGnClusterThreads * vec * sz)) continue;
            if (gn_cluster_bytes(k, vec, sz) > kGnClusterSmem) continue;
            found = true;
            *c = k;
            if (static_cast<long long>(a->n) * k.chunks * ctas >= 128 || k.rounds <= 2) return true;
        }
    return found;
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
    GnCluster c;
    if (gn_small(a, vec, &lps, &ept)) return 0;
    if (a->n > 65535) {                            // (done in parts: the first, and a smaller last one)
        SslaGroupNorm part = *a;
        part.n = 65535;
        const size_t whole = gn_bytes(&part);
        part.n = (a->n - 1) % 65535 + 1;
        return std::max(whole, gn_bytes(&part));
    }
    if (gn_cluster(a, vec, &c)) return 0;
    return static_cast<size_t>(a->n) * a->groups * gn_split(a, vec).splits * sizeof(double2);
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
    auto meets = [&](const void* p, long long s, long long q, int sz) {
        return p && overlaps(workspace, need, p, static_cast<size_t>((a->n - 1) * s + (a->positions - 1) * q + a->channels) * sz);
    };
    if (need && (meets(a->x, a->x_sample, a->x_pos, dtype_size(a->dtype)) || meets(a->y, a->y_sample, a->y_pos, dtype_size(a->dtype)) ||
                 meets(a->weight, 0, 0, 4) || meets(a->bias, 0, 0, 4)))
        return fail(SSLA_ERR_ARG, "group norm: the workspace overlaps a tensor");
    int lps, ept;
    if (a->n > 65535 && !gn_small(a, gn_vec(a), &lps, &ept)) {
        // more samples than a grid's depth: in parts, one after the other on the stream
        const int sz = dtype_size(a->dtype);
        for (int n0 = 0; n0 < a->n; n0 += 65535) {
            SslaGroupNorm part = *a;
            part.n = std::min(a->n - n0, 65535);
            part.x = static_cast<const char*>(a->x) + n0 * a->x_sample * sz;
            part.y = static_cast<char*>(a->y) + n0 * a->y_sample * sz;
            if (const int rc = ssla_group_norm(&part, workspace, workspace_bytes, stream); rc != SSLA_OK) return rc;
        }
        return SSLA_OK;
    }
    OnDevice dev(a->device);
    if (dev.err != SSLA_OK) return dev.err;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    GnArgs d;
    d.weight = a->weight; d.bias = a->bias;
    d.x_sample = a->x_sample; d.x_pos = a->x_pos; d.y_sample = a->y_sample; d.y_pos = a->y_pos;
    d.n = a->n; d.positions = a->positions; d.channels = a->channels; d.groups = a->groups;
    d.width = a->channels / a->groups;
    d.act = a->activation; d.eps = a->eps;
    d.inv = 1.0 / (static_cast<double>(a->positions) * d.width);
    d.wide = aligned(a->weight, 16) && aligned(a->bias, 16);
    d.stream = 2LL * a->n * a->positions * a->channels * dtype_size(a->dtype) > kStreamBytes;
    const int vec = gn_vec(a);
    auto run = [&](auto t, auto v) {
        using T = decltype(t);
        constexpr int V = decltype(v)::value;
        const T* x = static_cast<const T*>(a->x);
        T* y = static_cast<T*>(a->y);
        const long long slabs = static_cast<long long>(a->n) * a->groups;
        if (gn_small(a, vec, &lps, &ept)) {
            auto go = [&](auto l, auto e, auto un) {
                constexpr int LPS = decltype(l)::value, UNR = decltype(un)::value, kPer = kGnThreads / LPS;
                // the resident CTAs, a multiple of what keeps a thread's group
                const long long all = (slabs + kPer * UNR - 1) / (kPer * UNR);
                const int turn = a->groups / std::gcd(a->groups, kPer);
                long long grid = std::min<long long>(all, 148 * (LPS <= 32 ? kGnSlabCtas : 8));
                if (grid > turn) grid -= grid % turn;
                k_gn_slab<T, V, LPS, decltype(e)::value, UNR><<<static_cast<unsigned>(grid), kGnThreads, 0, st>>>(d, x, y);
                return launched("k_gn_slab");
            };
            using std::integral_constant;
            constexpr integral_constant<int, 1> one;
            constexpr integral_constant<int, 2> two;
            constexpr integral_constant<int, 4> four;
            constexpr integral_constant<int, 32> warp;
            if (lps == 8 && ept == 1) return go(integral_constant<int, 8>(), one, two);
            if (lps == 8) return go(integral_constant<int, 8>(), two, one);
            if (lps == 16) return go(integral_constant<int, 16>(), two, one);
            if (lps == 32 && ept == 2) return go(warp, two, one);
            if (lps == 32) return go(warp, four, one);
            return go(integral_constant<int, kGnThreads>(), integral_constant<int, (V >= 8 ? 4 : 8)>(), one);
        }
        GnCluster c;
        if (gn_cluster(a, vec, &c)) {
            const size_t bytes = gn_cluster_bytes(c, V, sizeof(T));
            allow_smem<k_gn_cluster<T, V>>(kGnClusterSmem);
            cudaLaunchConfig_t cfg = {};
            cudaLaunchAttribute at;
            at.id = cudaLaunchAttributeClusterDimension;
            at.val.clusterDim.x = c.ctas;
            at.val.clusterDim.y = at.val.clusterDim.z = 1;
            cfg.gridDim = dim3(c.ctas, c.chunks, a->n);
            cfg.blockDim = dim3(kGnClusterThreads);
            cfg.dynamicSmemBytes = bytes;
            cfg.stream = st;
            cfg.attrs = &at;
            cfg.numAttrs = 1;
            cudaLaunchKernelEx(&cfg, k_gn_cluster<T, V>, d, c, x, y);
            return launched("k_gn_cluster");
        }
        const GnSplit s = gn_split(a, vec);
        if (s.chunks > 65535) return fail(SSLA_ERR_ARG, "group norm: more than 65535 group chunks of large slabs");
        double2* part = static_cast<double2*>(workspace);
        const dim3 grid(s.splits, s.chunks, a->n);
        k_gn_sums<T, V><<<grid, kGnThreads, 0, st>>>(d, s, x, part);
        // the second launch's latency passes under the first kernel
        cudaLaunchConfig_t cfg = {};
        cudaLaunchAttribute at;
        at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at.val.programmaticStreamSerializationAllowed = 1;
        cfg.gridDim = grid;
        cfg.blockDim = dim3(kGnThreads);
        cfg.dynamicSmemBytes = s.gpc * sizeof(float2);
        cfg.stream = st;
        cfg.attrs = &at;
        cfg.numAttrs = 1;
        cudaLaunchKernelEx(&cfg, k_gn_apply<T, V>, d, s, x, y, static_cast<const double2*>(part));
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
