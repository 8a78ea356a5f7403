// ssla_ops.cuh -- what the recurrent-state operators (include/ssla_ops.h)
// share: element types, error returns of their C entries, launches.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <string>

#include "ssla_b200.h"
#include "ssla_ops.h"

namespace ssla {

void set_last_error(const std::string& msg);   // ssla_engine.cu

namespace ops {

// Sets the calling thread's error text; never throws.
inline int fail(int code, const char* fmt, ...) noexcept {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    try {
        set_last_error(buf);
    } catch (...) {
    }
    return code;
}

// Makes `dev` current for the scope; `err` is SSLA_OK or the code to return.
struct OnDevice {
    int prev = -1, err = SSLA_OK;
    explicit OnDevice(int dev) noexcept {
        static const int n = [] {                  // fixed for the process
            int c = 0;
            if (cudaGetDeviceCount(&c) != cudaSuccess) cudaGetLastError(), c = 0;
            return c;
        }();
        if (n == 0) {
            err = fail(SSLA_ERR_NO_DEVICE, "no CUDA device");
            return;
        }
        if (dev < 0 || dev >= n) {
            err = fail(SSLA_ERR_ARG, "device %d of %d", dev, n);
            return;
        }
        if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
        if (prev == dev) {
            prev = -1;
        } else if (cudaError_t e = cudaSetDevice(dev); e != cudaSuccess) {
            err = fail(SSLA_ERR_CUDA, "cudaSetDevice: %s", cudaGetErrorString(e));
        }
    }
    ~OnDevice() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

inline int launched(const char* what) noexcept {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? SSLA_OK : fail(SSLA_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

// Raises a kernel's dynamic shared memory limit, once per device.
template <auto K> inline void allow_smem(int bytes) noexcept {
    static std::atomic<unsigned long long> done{0};
    int dev = 0;
    cudaGetDevice(&dev);
    const unsigned long long bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_relaxed) & bit) return;
    cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    done.fetch_or(bit, std::memory_order_relaxed);
}

inline bool dtype_ok(int dt) { return dt == SSLA_DT_F32 || dt == SSLA_DT_BF16 || dt == SSLA_DT_F16; }
inline int dtype_size(int dt) { return dt == SSLA_DT_F32 ? 4 : 2; }
inline bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// Whether byte ranges [a, a + na) and [b, b + nb) meet.
inline bool overlaps(const void* a, size_t na, const void* b, size_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return na && nb && x < y + nb && y < x + na;
}

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_f<__half>(__half x) { return __half2float(x); }

template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }

// V consecutive values at p (aligned to V * sizeof(T)) as floats, and back.
template <typename T, int V> struct alignas(sizeof(T) * V) Pack { T v[V]; };

// Two 16-bit values as floats, and back (one rounding each).
template <typename T> __device__ __forceinline__ float2 unpack16(uint32_t u);
template <> __device__ __forceinline__ float2 unpack16<__nv_bfloat16>(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
}
template <> __device__ __forceinline__ float2 unpack16<__half>(uint32_t u) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
}
template <typename T> __device__ __forceinline__ uint32_t pack16(float x, float y);
template <> __device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float x, float y) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&p);
}
template <> __device__ __forceinline__ uint32_t pack16<__half>(float x, float y) {
    const __half2 p = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&p);
}

template <typename T, int V>
__device__ __forceinline__ void unpack_vec(const Pack<T, V>& k, float (&x)[V]) {
    if constexpr (sizeof(T) == 2 && V % 2 == 0) {
        uint32_t u[V / 2];
        memcpy(u, &k, sizeof u);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            const float2 f = unpack16<T>(u[i]);
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = to_f<T>(k.v[i]);
    }
}
template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&x)[V]) {
    const Pack<T, V> k = *reinterpret_cast<const Pack<T, V>*>(p);
    unpack_vec<T, V>(k, x);
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[V]) {
    Pack<T, V> k;
    if constexpr (sizeof(T) == 2 && V % 2 == 0) {
        uint32_t u[V / 2];
#pragma unroll
        for (int i = 0; i < V / 2; ++i) u[i] = pack16<T>(x[2 * i], x[2 * i + 1]);
        memcpy(&k, u, sizeof u);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) k.v[i] = from_f<T>(x[i]);
    }
    *reinterpret_cast<Pack<T, V>*>(p) = k;
}

// What a call reads and writes once and is larger than this goes past L2
// (evict first): it would only push out what others keep there.
constexpr long long kStreamBytes = 64LL << 20;

// load_vec / store_vec of 4 to 16 bytes with the streaming hint where asked.
template <typename T, int V>
__device__ __forceinline__ void load_vec_hint(const T* p, float (&x)[V], bool stream) {
    constexpr int B = sizeof(T) * V;
    if constexpr (B == 16 || B == 8 || B == 4) {
        if (stream) {
            Pack<T, V> k;
            if constexpr (B == 16) {
                const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p));
                memcpy(&k, &u, B);
            } else if constexpr (B == 8) {
                const uint2 u = __ldcs(reinterpret_cast<const uint2*>(p));
                memcpy(&k, &u, B);
            } else {
                const uint32_t u = __ldcs(reinterpret_cast<const uint32_t*>(p));
                memcpy(&k, &u, B);
            }
            unpack_vec<T, V>(k, x);
            return;
        }
    }
    load_vec<T, V>(p, x);
}
template <typename T, int V>
__device__ __forceinline__ void store_vec_hint(T* p, const float (&x)[V], bool stream) {
    constexpr int B = sizeof(T) * V;
    if constexpr (B == 16 || B == 8 || B == 4) {
        if (stream) {
            Pack<T, V> k;
            store_vec<T, V>(k.v, x);
            if constexpr (B == 16) {
                uint4 u;
                memcpy(&u, &k, B);
                __stcs(reinterpret_cast<uint4*>(p), u);
            } else if constexpr (B == 8) {
                uint2 u;
                memcpy(&u, &k, B);
                __stcs(reinterpret_cast<uint2*>(p), u);
            } else {
                uint32_t u;
                memcpy(&u, &k, B);
                __stcs(reinterpret_cast<uint32_t*>(p), u);
            }
            return;
        }
    }
    store_vec<T, V>(p, x);
}

}  // namespace ops
}  // namespace ssla
