// ssla_statecache.cu -- the 8-bit cache of recurrent states
// (include/ssla_ops.h): codes of one byte with a 32-bit scale for each block
// of a row, written and read back by slot.
//
// Memory bound: one read of the values, one write of a quarter (fp32) or a
// half (16-bit types) of the bytes plus the scales.  LG lanes share a block,
// VEC values a lane and step, so that a block's maximum is a few shuffles
// and its values stay in registers between the maximum and the codes.
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>

#include "ssla_ops.cuh"

namespace ssla {
namespace ops {
namespace {

constexpr int kCacheThreads = 256;
constexpr int kMaxBlock = 256;

struct CacheArgs {
    uint8_t* codes;
    float* scales;
    const int* slots;
    long long x_state, x_row;
    int n, n_slots, rows, cols, block, blocks;     // blocks per row
};

// RN(x / s) for |x| <= about 448 s, given y = RN(1 / s) and s, y well inside
// the normal range: Markstein's correction (IBM J. Res. Dev. 34, 1990) -- one
// step makes the estimate faithful, a second one correctly rounded.
__device__ __forceinline__ float quotient(float x, float s, float y) {
    float q = x * y;
    q = fmaf(fmaf(-s, q, x), y, q);
    return fmaf(fmaf(-s, q, x), y, q);
}

template <int FMT> __device__ __forceinline__ uint8_t encode(float q) {
    if constexpr (FMT == SSLA_FMT_INT8) {
        return static_cast<uint8_t>(static_cast<int8_t>(__float2int_rn(fminf(fmaxf(q, -127.0f), 127.0f))));
    } else {
        return __nv_cvt_float_to_fp8(q, __NV_SATFINITE, __NV_E4M3);
    }
}
template <int FMT> __device__ __forceinline__ float decode(uint8_t c) {
    if constexpr (FMT == SSLA_FMT_INT8) {
        return static_cast<float>(static_cast<int8_t>(c));
    } else {
        return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
    }
}

// Block t of state i: row t / blocks, columns [c, c + width).
template <typename T, int FMT, int VEC, int LG, int EPT, bool STORE>
__global__ void __launch_bounds__(kCacheThreads) k_state_cache(CacheArgs a, T* __restrict__ x) {
    constexpr int kGroups = kCacheThreads / LG;
    const int i = blockIdx.y, tid = threadIdx.x, lane = tid % LG, group = tid / LG;
    const int slot = a.slots ? a.slots[i] : i;
    const bool valid = slot >= 0 && slot < a.n_slots;
    if constexpr (STORE) {
        if (!valid) return;
        if (a.slots) {
            int later = 0;                          // the last state naming a slot is kept
            for (int j = i + 1 + tid; j < a.n; j += kCacheThreads) later |= a.slots[j] == slot;
            if (__syncthreads_or(later)) return;
        }
    }
    const int total = a.rows * a.blocks;
    const size_t s0 = valid ? static_cast<size_t>(slot) : 0;
    uint8_t* codes = a.codes + s0 * a.rows * a.cols;
    float* scales = a.scales + s0 * total;
    for (int t0 = blockIdx.x * kGroups; t0 < total; t0 += gridDim.x * kGroups) {
        const int t = t0 + group;
        const bool on = t < total;
        const int row = on ? t / a.blocks : 0, c = on ? (t - row * a.blocks) * a.block : 0;
        const int width = on ? min(a.block, a.cols - c) : 0;
        T* xp = x + i * a.x_state + row * a.x_row + c;
        uint8_t* cp = codes + static_cast<size_t>(row) * a.cols + c;
        if constexpr (STORE) {
            float v[EPT][VEC];
            float m = 0.0f;
            bool bad = false;
#pragma unroll
            for (int e = 0; e < EPT; ++e) {
                const int k = (e * LG + lane) * VEC;
                if (k < width) {
                    load_vec<T, VEC>(xp + k, v[e]);
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        m = fmaxf(m, fabsf(v[e][j]));
                        bad |= !(fabsf(v[e][j]) <= 3.402823466e38f);
                    }
                }
            }
            if (bad) m = __int_as_float(0x7F800000);
#pragma unroll
            for (int w = LG / 2; w; w >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, w));
            const bool finite = m < __int_as_float(0x7F800000);
            const float most = FMT == SSLA_FMT_INT8 ? 127.0f : 448.0f;
            float s = finite ? __fdiv_rn(m, most) : __int_as_float(0x7FC00000);
            // a scale rounded up next to the largest float would read back as infinity
            if (s * most == __int_as_float(0x7F800000)) s = __int_as_float(__float_as_int(s) - 1);
            const bool plain = s > 1e-30f && s < 1e30f;
            const float y = plain ? __frcp_rn(s) : 0.0f;
#pragma unroll
            for (int e = 0; e < EPT; ++e) {
                const int k = (e * LG + lane) * VEC;
                if (k < width) {
                    Pack<uint8_t, VEC> o;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) {
                        const float q = plain ? quotient(v[e][j], s, y) : s > 0.0f ? __fdiv_rn(v[e][j], s) : 0.0f;
                        o.v[j] = encode<FMT>(q);
                    }
                    *reinterpret_cast<Pack<uint8_t, VEC>*>(cp + k) = o;
                }
            }
            if (on && lane == 0) scales[t] = s;
        } else {
            const float s = on && valid ? scales[t] : 0.0f;
#pragma unroll
            for (int e = 0; e < EPT; ++e) {
                const int k = (e * LG + lane) * VEC;
                if (k < width) {
                    float v[VEC] = {};
                    if (valid) {
                        const Pack<uint8_t, VEC> o = *reinterpret_cast<const Pack<uint8_t, VEC>*>(cp + k);
#pragma unroll
                        for (int j = 0; j < VEC; ++j) v[j] = decode<FMT>(o.v[j]) * s;
                    }
                    store_vec<T, VEC>(xp + k, v);
                }
            }
        }
    }
}

int check_cache(const SslaStateCache* c, const void* x, const char* who) {
    if (!c) return fail(SSLA_ERR_ARG, "%s: null argument", who);
    if (!dtype_ok(c->dtype)) return fail(SSLA_ERR_ARG, "%s: dtype %d is not an SSLA_DT_* value", who, c->dtype);
    if (c->format != SSLA_FMT_INT8 && c->format != SSLA_FMT_E4M3)
        return fail(SSLA_ERR_ARG, "%s: format %d is not an SSLA_FMT_* value", who, c->format);
    if (c->n < 0 || c->n > 65535 || c->n_slots < 0 || c->rows < 0 || c->cols < 0)
        return fail(SSLA_ERR_ARG, "%s: n %d must be 0..65535, n_slots, rows and cols at least 0", who, c->n);
    if (c->block < 1 || c->block > kMaxBlock)
        return fail(SSLA_ERR_ARG, "%s: block %d must be 1..%d", who, c->block, kMaxBlock);
    if (c->n == 0 || c->rows == 0 || c->cols == 0) return SSLA_OK;
    const long long blocks = (c->cols + c->block - 1LL) / c->block;
    if (c->rows * blocks > INT_MAX / 2) return fail(SSLA_ERR_ARG, "%s: more than 2^30 blocks in a state", who);
    if (!c->slots && c->n > c->n_slots) return fail(SSLA_ERR_ARG, "%s: %d states for %d slots", who, c->n, c->n_slots);
    if (c->n_slots == 0) return fail(SSLA_ERR_ARG, "%s: no slots", who);
    if (!x || !c->codes || !c->scales) return fail(SSLA_ERR_ARG, "%s: null pointer", who);
    if ((c->rows > 1 && c->x_row < c->cols) ||
        (c->n > 1 && c->x_state < (c->rows - 1) * c->x_row + c->cols))
        return fail(SSLA_ERR_ARG, "%s: the states of x overlap", who);
    if (c->x_row < 0 || c->x_state < 0 || c->x_row > LLONG_MAX / 8 / (c->rows + 1LL) ||
        c->x_state > LLONG_MAX / 16 / (c->n + 1LL))
        return fail(SSLA_ERR_ARG, "%s: a stride is too large", who);
    const int sz = dtype_size(c->dtype);
    if (!aligned(x, sz) || !aligned(c->scales, 4) || !aligned(c->slots, 4))
        return fail(SSLA_ERR_ARG, "%s: a pointer is not aligned to its element", who);
    const size_t xn = static_cast<size_t>((c->n - 1) * c->x_state + (c->rows - 1) * c->x_row + c->cols) * sz;
    const size_t cn = static_cast<size_t>(c->n_slots) * c->rows * c->cols;
    const size_t sn = static_cast<size_t>(c->n_slots) * c->rows * blocks * 4;
    if (overlaps(x, xn, c->codes, cn) || overlaps(x, xn, c->scales, sn) || overlaps(c->codes, cn, c->scales, sn) ||
        overlaps(c->slots, 4ull * c->n, c->codes, cn) || overlaps(c->slots, 4ull * c->n, c->scales, sn) ||
        overlaps(c->slots, 4ull * c->n, x, xn))
        return fail(SSLA_ERR_ARG, "%s: x, codes, scales and slots may not overlap", who);
    return SSLA_OK;
}

template <bool STORE> int cache_call(const SslaStateCache* c, void* x, void* stream, const char* who) {
    if (const int rc = check_cache(c, x, who); rc != SSLA_OK) return rc;
    if (c->n == 0 || c->rows == 0 || c->cols == 0) return SSLA_OK;
    OnDevice dev(c->device);
    if (dev.err != SSLA_OK) return dev.err;
    CacheArgs a;
    a.codes = static_cast<uint8_t*>(c->codes);
    a.scales = c->scales;
    a.slots = c->slots;
    a.x_state = c->x_state; a.x_row = c->x_row;
    a.n = c->n; a.n_slots = c->n_slots; a.rows = c->rows; a.cols = c->cols; a.block = c->block;
    a.blocks = (c->cols + c->block - 1) / c->block;
    const int total = a.rows * a.blocks;
    // widest step that every block's start and width allow
    const int sz = dtype_size(c->dtype);
    const long long all = static_cast<long long>(a.cols) | a.block | (a.rows > 1 ? a.x_row : 0) | (a.n > 1 ? a.x_state : 0);
    const int vec = all % 4 == 0 && aligned(x, 4 * sz) && aligned(c->codes, 4) ? 4 : 1;
    const int lanes = (std::min(a.block, a.cols) + vec - 1) / vec;
    auto go = [&](auto t, auto fmt, auto v, auto lg, auto ept) {
        using T = decltype(t);
        constexpr int LG = decltype(lg)::value;
        const int per = kCacheThreads / LG;
        const int gx = std::min((total + per - 1) / per, std::max(1, 148 * 64 / a.n));
        k_state_cache<T, decltype(fmt)::value, decltype(v)::value, LG, decltype(ept)::value, STORE>
            <<<dim3(gx, a.n), kCacheThreads, 0, static_cast<cudaStream_t>(stream)>>>(a, static_cast<T*>(x));
        return launched("k_state_cache");
    };
    auto by_lanes = [&](auto t, auto fmt, auto v) {
        using std::integral_constant;
        if (lanes <= 4) return go(t, fmt, v, integral_constant<int, 4>(), integral_constant<int, 1>());
        if (lanes <= 8) return go(t, fmt, v, integral_constant<int, 8>(), integral_constant<int, 1>());
        if (lanes <= 16) return go(t, fmt, v, integral_constant<int, 16>(), integral_constant<int, 1>());
        if (lanes <= 32) return go(t, fmt, v, integral_constant<int, 32>(), integral_constant<int, 1>());
        if (lanes <= 64) return go(t, fmt, v, integral_constant<int, 32>(), integral_constant<int, 2>());
        return go(t, fmt, v, integral_constant<int, 32>(), integral_constant<int, 8>());
    };
    auto by_vec = [&](auto t, auto fmt) {
        return vec == 4 ? by_lanes(t, fmt, std::integral_constant<int, 4>())
                        : by_lanes(t, fmt, std::integral_constant<int, 1>());
    };
    auto by_fmt = [&](auto t) {
        return c->format == SSLA_FMT_INT8 ? by_vec(t, std::integral_constant<int, SSLA_FMT_INT8>())
                                          : by_vec(t, std::integral_constant<int, SSLA_FMT_E4M3>());
    };
    return c->dtype == SSLA_DT_F32 ? by_fmt(float()) : c->dtype == SSLA_DT_BF16 ? by_fmt(__nv_bfloat16())
                                                                                  : by_fmt(__half());
}

}  // namespace
}  // namespace ops
}  // namespace ssla

extern "C" {

int ssla_state_store(const SslaStateCache* c, const void* x, void* stream) {
    return ssla::ops::cache_call<true>(c, const_cast<void*>(x), stream, "state store");
}
int ssla_state_load(const SslaStateCache* c, void* x, void* stream) {
    return ssla::ops::cache_call<false>(c, x, stream, "state load");
}

}  // extern "C"
