// Value types of the operators on sequences of tokens (embed.cu, rms_norm.cu, gated_scan.cu): storage type T, the type
// W it is computed in (float; double for double), conversions and packets of several elements.
#pragma once

#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace db2 {

template <typename T> struct WideOf {
    using type = float;
};
template <> struct WideOf<double> {
    using type = double;
};
template <typename T> using wide_t = typename WideOf<T>::type;

__device__ __forceinline__ double widen(double x) { return x; }
__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float widen(__nv_fp8_e4m3 x) { return static_cast<float>(x); }

// one rounding to nearest even
template <typename T, typename W> __device__ __forceinline__ T narrow(W x) {
    if constexpr (std::is_same_v<T, __half>) {
        if constexpr (std::is_same_v<W, double>)
            return __double2half(x);
        else
            return __float2half_rn(x);
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        if constexpr (std::is_same_v<W, double>)
            return __double2bfloat16(x);
        else
            return __float2bfloat16_rn(x);
    } else
        return static_cast<T>(x);
}

// N elements that are loaded and stored at once (N * sizeof(T) <= 16, the address a multiple of that)
template <typename T, int N> struct alignas(sizeof(T) * N) Vec {
    T v[N];
};
template <typename T, int N> __device__ __forceinline__ Vec<T, N> ld_vec(const T *p) {
    return *reinterpret_cast<const Vec<T, N> *>(p);
}
template <typename T, int N> __device__ __forceinline__ void st_vec(T *p, const Vec<T, N> &x) {
    *reinterpret_cast<Vec<T, N> *>(p) = x;
}

// the same for N values, pairs of 16-bit ones in one instruction
template <typename T, int N, typename W> __device__ __forceinline__ Vec<T, N> narrow_all(const W *x) {
    Vec<T, N> z;
    if constexpr (sizeof(T) == 2 && N % 2 == 0) {
#pragma unroll
        for (int k = 0; k < N; k += 2) {
            if constexpr (std::is_same_v<T, __half>)
                *reinterpret_cast<__half2 *>(&z.v[k]) = __floats2half2_rn(x[k], x[k + 1]);
            else
                *reinterpret_cast<__nv_bfloat162 *>(&z.v[k]) = __floats2bfloat162_rn(x[k], x[k + 1]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; k++)
            z.v[k] = narrow<T>(x[k]);
    }
    return z;
}

// ---- arithmetic on N wide values at once; floats go in pairs, two to an instruction ----
template <typename T, int N> __device__ __forceinline__ void widen_all(const Vec<T, N> &x, wide_t<T> *y) {
    if constexpr (std::is_same_v<T, __nv_bfloat16> && N % 2 == 0) {
#pragma unroll
        for (int k = 0; k < N; k += 2) { // a bfloat16 is the upper half of a float
            const uint32_t two = *reinterpret_cast<const uint32_t *>(&x.v[k]);
            y[k] = __uint_as_float(two << 16);
            y[k + 1] = __uint_as_float(two & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; k++)
            y[k] = widen(x.v[k]);
    }
}
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
    uint64_t p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
    return p;
}
__device__ __forceinline__ void pair_to(uint64_t p, float *a) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a[0]), "=f"(a[1]) : "l"(p)); }
// o = a * b + c
template <int N, typename W> __device__ __forceinline__ void fma_all(const W *a, const W *b, const W *c, W *o) {
    if constexpr (std::is_same_v<W, float> && N % 2 == 0) {
#pragma unroll
        for (int k = 0; k < N; k += 2) {
            uint64_t r;
            asm("fma.rn.f32x2 %0, %1, %2, %3;"
                : "=l"(r)
                : "l"(pair_of(a[k], a[k + 1])), "l"(pair_of(b[k], b[k + 1])), "l"(pair_of(c[k], c[k + 1])));
            pair_to(r, o + k);
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; k++)
            o[k] = a[k] * b[k] + c[k];
    }
}
// o = a * b
template <int N, typename W> __device__ __forceinline__ void mul_all(const W *a, const W *b, W *o) {
    if constexpr (std::is_same_v<W, float> && N % 2 == 0) {
#pragma unroll
        for (int k = 0; k < N; k += 2) {
            uint64_t r;
            asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair_of(a[k], a[k + 1])), "l"(pair_of(b[k], b[k + 1])));
            pair_to(r, o + k);
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; k++)
            o[k] = a[k] * b[k];
    }
}
// o = a + b
template <int N, typename W> __device__ __forceinline__ void add_all(const W *a, const W *b, W *o) {
    if constexpr (std::is_same_v<W, float> && N % 2 == 0) {
#pragma unroll
        for (int k = 0; k < N; k += 2) {
            uint64_t r;
            asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair_of(a[k], a[k + 1])), "l"(pair_of(b[k], b[k + 1])));
            pair_to(r, o + k);
        }
    } else {
#pragma unroll
        for (int k = 0; k < N; k++)
            o[k] = a[k] + b[k];
    }
}
template <int N, typename W> __device__ __forceinline__ void set_all(W *o, W x) {
#pragma unroll
    for (int k = 0; k < N; k++)
        o[k] = x;
}
// sum over k of a[k] * b[k], added to two partial sums (pairs), or to the first of them
template <int N, typename W> __device__ __forceinline__ void dot_all(const W *a, const W *b, W *sums) {
    if constexpr (N % 2 == 0) {
#pragma unroll
        for (int k = 0; k < N; k += 2)
            fma_all<2>(a + k, b + k, sums, sums);
    } else {
#pragma unroll
        for (int k = 0; k < N; k++)
            sums[0] = a[k] * b[k] + sums[0];
    }
}

// N elements from global to shared memory, asynchronously (at once where they are fewer than four bytes).  fetch_commit
// closes a group of them, fetch_wait<K> waits until all but the last K groups have arrived, for the calling thread.
template <typename T, int N> __device__ __forceinline__ void fetch(T *to, const T *from) {
    constexpr int bytes = sizeof(T) * N;
    const unsigned at = (unsigned)__cvta_generic_to_shared(to);
    if constexpr (bytes == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
    else if constexpr (bytes >= 4)
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(from), "n"(bytes) : "memory");
    else
        st_vec<T, N>(to, ld_vec<T, N>(from));
}
__device__ __forceinline__ void fetch_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int K> __device__ __forceinline__ void fetch_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(K) : "memory"); }

// A kernel that follows another one of the same call may be set up while that one still runs: launch_next starts it early,
// and wait_for_last, the first thing that all its threads do, returns when the kernel before it has finished and its
// writes are visible.  start_next, in the kernel before, says that all its CTAs are on their way.  (A call's first kernel is
// launched the ordinary way and so waits for everything in front of it.)
__device__ __forceinline__ void wait_for_last() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void start_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
template <typename... P, typename... A>
int launch_next(const char *what, void (*kernel)(P...), dim3 grid, int block, size_t smem, cudaStream_t st, A... args) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
    return after_launch(what); // takes the error of a launch that failed
}

// whether rows of ld elements of es bytes starting at p all lie on multiples of `bytes` (absent operands do)
inline bool rows_aligned(const void *p, int64_t ld, size_t es, size_t bytes) {
    return !p || (reinterpret_cast<uintptr_t>(p) % bytes == 0 && (size_t)ld * es % bytes == 0);
}

// a matrix operand of `rows` rows: the leading dimension covers the columns (one row needs none)
inline bool ld_ok(int64_t ld, int64_t rows, int64_t cols) { return ld >= cols || rows <= 1; }

} // namespace db2

// the four storage types of the sequence operators
#define DB2_DISPATCH_SEQ(dtype, T, ...)                                                                                \
    switch (dtype) {                                                                                                   \
    case DB2_F64: {                                                                                                    \
        using T = double;                                                                                              \
        __VA_ARGS__;                                                                                                   \
    } break;                                                                                                           \
    case DB2_F32: {                                                                                                    \
        using T = float;                                                                                               \
        __VA_ARGS__;                                                                                                   \
    } break;                                                                                                           \
    case DB2_F16: {                                                                                                    \
        using T = __half;                                                                                              \
        __VA_ARGS__;                                                                                                   \
    } break;                                                                                                           \
    case DB2_BF16: {                                                                                                   \
        using T = __nv_bfloat16;                                                                                       \
        __VA_ARGS__;                                                                                                   \
    } break;                                                                                                           \
    default:                                                                                                           \
        return ::db2::set_error(DB2_EUNSUPPORTED, "unsupported value type code %d", (int)(dtype));                     \
    }
