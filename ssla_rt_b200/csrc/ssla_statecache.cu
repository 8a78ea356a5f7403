// ssla_statecache.cu -- the 8-bit cache of recurrent states
// (include/ssla_ops.h): codes of one byte with a 32-bit scale for each block
// of a row, written and read back by slot.
//
// Memory bound: one read of the values, one write of a quarter (fp32) or a
// half (16-bit types) of the bytes plus the scales.  192 states of 2,048 x 128
// stored as e4m3: 43 us, 92% of the measured copy rate.  Four vectors of a
// block in one lane (two shuffles for a block of 64 instead of four), two
// blocks at once, and a quotient of five operations brought it there from 92 us.
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
    int stream;                                    // the states are too many for L2
};

// RN(x / s) for |x| <= about 448 s, given y = RN(1 / s) and s, y well inside
// the normal range: Markstein's correction (IBM J. Res. Dev. 34, 1990) -- one
// step makes the estimate faithful, a second one correctly rounded.
__device__ __forceinline__ float quotient(float x, float s, float y) {
    float q = x * y;
    q = fmaf(fmaf(-s, q, x), y, q);
    return fmaf(fmaf(-s, q, x), y, q);
}

// V quotients as codes (|q| below 128 / 449, so that only rounding is left).
template <int FMT, int V>
__device__ __forceinline__ void encode(const float (&q)[V], uint8_t* p) {
    if constexpr (V == 1) {
        if constexpr (FMT == SSLA_FMT_INT8) *p = static_cast<uint8_t>(__float2int_rn(q[0]));
        else *p = __nv_cvt_float_to_fp8(q[0], __NV_SATFINITE, __NV_E4M3);
    } else {
        Pack<uint32_t, V / 4> o;
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            const float* x = q + 4 * i;
            if constexpr (FMT == SSLA_FMT_INT8) {
                uint32_t hi;                        // bytes of the second pair, then of the first below them
                asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, 0;" : "=r"(hi) : "r"(__float2int_rn(x[3])), "r"(__float2int_rn(x[2])));
                asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;"
                    : "=r"(o.v[i]) : "r"(__float2int_rn(x[1])), "r"(__float2int_rn(x[0])), "r"(hi));
            } else {
                o.v[i] = __nv_cvt_float2_to_fp8x2(make_float2(x[0], x[1]), __NV_SATFINITE, __NV_E4M3) |
                         static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(make_float2(x[2], x[3]), __NV_SATFINITE, __NV_E4M3)) << 16;
            }
        }
        *reinterpret_cast<Pack<uint32_t, V / 4>*>(p) = o;
    }
}
template <int FMT> __device__ __forceinline__ float decode(uint8_t c) {
    if constexpr (FMT == SSLA_FMT_INT8) {
        return static_cast<float>(static_cast<int8_t>(c));
    } else {
        return __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
    }
}

// Store.  LG lanes share a block and hold EPT vectors of it each; a group
// takes UNR blocks at once, all their loads before the first maximum.
// Block t of state i is row t / blocks, columns [c, c + width).
template <typename T, int FMT, int VEC, int LG, int EPT, int UNR>
__global__ void __launch_bounds__(kCacheThreads) k_state_store(CacheArgs a, const T* __restrict__ x) {
    constexpr int kGroups = kCacheThreads / LG;
    const int i = blockIdx.y, tid = threadIdx.x, lane = tid % LG, group = tid / LG;
    const int slot = a.slots ? a.slots[i] : i;
    if (slot < 0 || slot >= a.n_slots) return;
    if (a.slots) {
        int later = 0;                              // the last state naming a slot is kept
        for (int j = i + 1 + tid; j < a.n; j += kCacheThreads) later |= a.slots[j] == slot;
        if (__syncthreads_or(later)) return;
    }
    const int total = a.rows * a.blocks;
    uint8_t* codes = a.codes + static_cast<size_t>(slot) * a.rows * a.cols;
    float* scales = a.scales + static_cast<size_t>(slot) * total;
    const T* xi = x + i * a.x_state;
    constexpr float most = FMT == SSLA_FMT_INT8 ? 127.0f : 448.0f;
    for (int t0 = blockIdx.x * kGroups * UNR; t0 < total; t0 += gridDim.x * kGroups * UNR) {
        float v[UNR][EPT][VEC];
        int width[UNR];
        uint8_t* cp[UNR];
#pragma unroll
        for (int u = 0; u < UNR; ++u) {
            const int t = t0 + u * kGroups + group;
            width[u] = 0;
            cp[u] = codes;
            if (t < total) {
                const int row = a.blocks == 1 ? t : t / a.blocks, c = (t - row * a.blocks) * a.block;
                width[u] = min(a.block, a.cols - c);
                const T* xp = xi + row * a.x_row + c;
                cp[u] = codes + static_cast<size_t>(row) * a.cols + c;
#pragma unroll
                for (int e = 0; e < EPT; ++e) {
                    const int k = (e * LG + lane) * VEC;
                    if (k < width[u]) load_vec_hint<T, VEC>(xp + k, v[u][e], a.stream);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < UNR; ++u) {
            // largest magnitude as its bits: NaN above infinity above the finite
            uint32_t m = 0;
#pragma unroll
            for (int e = 0; e < EPT; ++e)
                if ((e * LG + lane) * VEC < width[u])
#pragma unroll
                    for (int j = 0; j < VEC; ++j) m = max(m, __float_as_uint(v[u][e][j]) & 0x7FFFFFFFu);
#pragma unroll
            for (int w = LG / 2; w; w >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, w));
            float s = m < 0x7F800000u ? __fdiv_rn(__uint_as_float(m), most) : __int_as_float(0x7FC00000);
            // a scale rounded up next to the largest float would read back as infinity
            if (s * most == __int_as_float(0x7F800000)) s = __int_as_float(__float_as_int(s) - 1);
            if (s > 1e-30f && s < 1e30f) {
                const float y = __frcp_rn(s);
#pragma unroll
                for (int e = 0; e < EPT; ++e) {
                    const int k = (e * LG + lane) * VEC;
                    if (k < width[u]) {
#pragma unroll
                        for (int j = 0; j < VEC; ++j) v[u][e][j] = quotient(v[u][e][j], s, y);
                        encode<FMT, VEC>(v[u][e], cp[u] + k);
                    }
                }
            } else {                                // zeros, non-finite values, the ends of the exponent range
#pragma unroll
                for (int e = 0; e < EPT; ++e) {
                    const int k = (e * LG + lane) * VEC;
                    if (k < width[u]) {
#pragma unroll
                        for (int j = 0; j < VEC; ++j)
                            v[u][e][j] = s > 0.0f ? fminf(fmaxf(__fdiv_rn(v[u][e][j], s), -most), most) : 0.0f;
                        encode<FMT, VEC>(v[u][e], cp[u] + k);
                    }
                }
            }
            if (width[u] && lane == 0) scales[t0 + u * kGroups + group] = s;
        }
    }
}

// Load.  VEC consecutive values of the state a thread and step, blocks and
// rows wherever they end; `split`: a vector may span two blocks or rows.
template <typename T, int FMT, int VEC>
__global__ void __launch_bounds__(kCacheThreads) k_state_load(CacheArgs a, T* __restrict__ x, int split) {
    const int i = blockIdx.y;
    const int slot = a.slots ? a.slots[i] : i;
    const bool valid = slot >= 0 && slot < a.n_slots;
    const size_t s0 = valid ? static_cast<size_t>(slot) : 0;
    const long long size = static_cast<long long>(a.rows) * a.cols;
    const uint8_t* codes = a.codes + s0 * size;
    const float* scales = a.scales + s0 * a.rows * a.blocks;
    T* xi = x + i * a.x_state;
    const long long step = static_cast<long long>(gridDim.x) * kCacheThreads * VEC;
#pragma unroll 2
    for (long long e = (static_cast<long long>(blockIdx.x) * kCacheThreads + threadIdx.x) * VEC; e < size; e += step) {
        int row, c;
        if (size <= INT_MAX) {
            row = static_cast<unsigned>(e) / static_cast<unsigned>(a.cols);
            c = static_cast<int>(e) - row * a.cols;
        } else {
            row = static_cast<int>(e / a.cols);
            c = static_cast<int>(e - static_cast<long long>(row) * a.cols);
        }
        float v[VEC] = {};
        if (valid) {
            const Pack<uint8_t, VEC> o = *reinterpret_cast<const Pack<uint8_t, VEC>*>(codes + e);
            int b = static_cast<unsigned>(c) / static_cast<unsigned>(a.block);
            const float* sp = scales + static_cast<size_t>(row) * a.blocks + b;
            float s = *sp;
            if (VEC == 1 || !split) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[j] = decode<FMT>(o.v[j]) * s;
            } else {
                int left = min(a.block, a.cols - b * a.block) - (c - b * a.block), rest = a.cols - c;
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    if (left == 0) {                // blocks and rows follow one another in memory
                        if (rest == 0) rest = a.cols;
                        left = min(a.block, rest);
                        s = *++sp;
                    }
                    v[j] = decode<FMT>(o.v[j]) * s;
                    --left;
                    --rest;
                }
            }
        }
        store_vec_hint<T, VEC>(xi + row * a.x_row + c, v, a.stream);
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

template <typename F> int with_cache_types(const SslaStateCache* c, F&& f) {
    auto by_fmt = [&](auto t) {
        return c->format == SSLA_FMT_INT8 ? f(t, std::integral_constant<int, SSLA_FMT_INT8>())
                                          : f(t, std::integral_constant<int, SSLA_FMT_E4M3>());
    };
    return c->dtype == SSLA_DT_F32 ? by_fmt(float()) : c->dtype == SSLA_DT_BF16 ? by_fmt(__nv_bfloat16())
                                                                                  : by_fmt(__half());
}

CacheArgs cache_args(const SslaStateCache* c) {
    CacheArgs a;
    a.codes = static_cast<uint8_t*>(c->codes);
    a.scales = c->scales;
    a.slots = c->slots;
    a.x_state = c->x_state; a.x_row = c->x_row;
    a.n = c->n; a.n_slots = c->n_slots; a.rows = c->rows; a.cols = c->cols; a.block = c->block;
    a.blocks = (c->cols + c->block - 1) / c->block;
    a.stream = static_cast<long long>(c->n) * c->rows * c->cols * (dtype_size(c->dtype) + 1) > kStreamBytes;
    return a;
}

// CTAs of a state: enough for the whole call to fill the GPU several times.
unsigned cache_grid(long long ctas, int n) {
    return static_cast<unsigned>(std::min(ctas, std::max(1LL, 148LL * 64 / n)));
}

int store_call(const SslaStateCache* c, const void* x, void* stream) {
    const char* who = "state store";
    if (const int rc = check_cache(c, x, who); rc != SSLA_OK) return rc;
    if (c->n == 0 || c->rows == 0 || c->cols == 0) return SSLA_OK;
    OnDevice dev(c->device);
    if (dev.err != SSLA_OK) return dev.err;
    const CacheArgs a = cache_args(c);
    const int total = a.rows * a.blocks, sz = dtype_size(c->dtype);
    // the widest vectors that every block's start and width allow: 16 bytes of
    // values, four 16-bit values, or single ones
    const long long all = static_cast<long long>(a.cols) | a.block | (a.rows > 1 ? a.x_row : 0) | (a.n > 1 ? a.x_state : 0);
    auto fits = [&](int v) { return all % v == 0 && aligned(x, v * sz) && aligned(c->codes, v); };
    const int vec = sz == 2 && fits(8) ? 8 : fits(4) ? 4 : 1;
    const int need = (std::min(a.block, a.cols) + vec - 1) / vec;      // vectors of a block
    return with_cache_types(c, [&](auto t, auto fmt) {
        using T = decltype(t);
        auto go = [&](auto v, auto lg, auto ept, auto unr) {
            constexpr int LG = decltype(lg)::value, UNR = decltype(unr)::value;
            const int per = kCacheThreads / LG * UNR;
            k_state_store<T, decltype(fmt)::value, decltype(v)::value, LG, decltype(ept)::value, UNR>
                <<<dim3(cache_grid((total + per - 1LL) / per, a.n), a.n), kCacheThreads, 0, static_cast<cudaStream_t>(stream)>>>(
                    a, static_cast<const T*>(x));
            return launched("k_state_store");
        };
        using std::integral_constant;
        // wide vectors: four of a block in one lane (few shuffles); single
        // values: neighbouring lanes (full sectors)
        auto wide = [&](auto v) {
            constexpr integral_constant<int, 4> e;
            constexpr integral_constant<int, 2> u;
            if (need <= 4) return go(v, integral_constant<int, 1>(), e, u);
            if (need <= 8) return go(v, integral_constant<int, 2>(), e, u);
            if (need <= 16) return go(v, integral_constant<int, 4>(), e, u);
            if (need <= 32) return go(v, integral_constant<int, 8>(), e, u);
            return go(v, integral_constant<int, 16>(), e, u);
        };
        if constexpr (sizeof(T) == 2)
            if (vec == 8) return wide(integral_constant<int, 8>());
        if (vec == 4) return wide(integral_constant<int, 4>());
        constexpr integral_constant<int, 1> one;
        if (need <= 8) return go(one, integral_constant<int, 8>(), one, integral_constant<int, 4>());
        if (need <= 32) return go(one, integral_constant<int, 32>(), one, integral_constant<int, 4>());
        return go(one, integral_constant<int, 32>(), integral_constant<int, 8>(), one);
    });
}

int load_call(const SslaStateCache* c, void* x, void* stream) {
    const char* who = "state load";
    if (const int rc = check_cache(c, x, who); rc != SSLA_OK) return rc;
    if (c->n == 0 || c->rows == 0 || c->cols == 0) return SSLA_OK;
    OnDevice dev(c->device);
    if (dev.err != SSLA_OK) return dev.err;
    const CacheArgs a = cache_args(c);
    const long long size = static_cast<long long>(a.rows) * a.cols;
    const int sz = dtype_size(c->dtype);
    // a state's values follow one another: vectors need not respect its rows
    const bool flat = a.rows == 1 || a.x_row == a.cols;
    auto fits = [&](int v) {
        return flat && size % v == 0 && (a.n == 1 || a.x_state % v == 0) && aligned(x, v * sz) && aligned(c->codes, v);
    };
    const int vec = sz == 2 && fits(8) ? 8 : fits(4) ? 4 : 1;
    const int split = a.cols % vec || a.block % vec;
    return with_cache_types(c, [&](auto t, auto fmt) {
        using T = decltype(t);
        auto go = [&](auto v) {
            constexpr int V = decltype(v)::value;
            const long long per = 2LL * kCacheThreads * V;
            k_state_load<T, decltype(fmt)::value, V>
                <<<dim3(cache_grid((size + per - 1) / per, a.n), a.n), kCacheThreads, 0, static_cast<cudaStream_t>(stream)>>>(
                    a, static_cast<T*>(x), split);
            return launched("k_state_load");
        };
        if constexpr (sizeof(T) == 2)
            if (vec == 8) return go(std::integral_constant<int, 8>());
        if (vec == 4) return go(std::integral_constant<int, 4>());
        return go(std::integral_constant<int, 1>());
    });
}

}  // namespace
}  // namespace ops
}  // namespace ssla

extern "C" {

int ssla_state_store(const SslaStateCache* c, const void* x, void* stream) { return ssla::ops::store_call(c, x, stream); }
int ssla_state_load(const SslaStateCache* c, void* x, void* stream) { return ssla::ops::load_call(c, x, stream); }

}  // extern "C"
