// Root-mean-square norm of the rows of a matrix, with the addition of a residual in front of it, and its gradient.
//
//   s = x + residual (rounded to the value type: what is stored is what is normalised)      s = x without a residual
//   rstd = 1 / sqrt(mean(s^2) + eps)          y = s * rstd * weight
//   8-bit result: per group of columns  scale = max|y| / 448,  q = e4m3(y / scale); see Divisor for how it is rounded
//
//   t = dy * weight       dx = rstd * (t - s * rstd^2 * mean(t * s)) + dsum       dweight = column sums of dy * s * rstd
//
// Statistics, products and sums are float (double for double).  All of it is bound by memory: a row is read once, kept
// in registers while its sum is formed, and written from there.
#include "runtime.h"
#include "seq.cuh"

namespace db2 {

namespace {

constexpr float E4M3_MAX = 448.0f;

// Sum over the `tpr` threads of a row, in one fixed order; tpr is a power of two below 32 or a multiple of 32, and the rows
// of a CTA lie side by side.  Every thread of the CTA calls it the same number of times; `red` alternates between two
// halves, so one barrier is enough.
constexpr int NORM_MAX_WARPS = 16;
template <typename W> struct RowSum {
    W *red; // 2 * NORM_MAX_WARPS
    int turn = 0;
    __device__ W operator()(W v, int tpr) {
        const int in_warp = tpr < 32 ? tpr : 32;
        for (int o = in_warp >> 1; o >= 1; o >>= 1)
            v += shfl_xor(v, o);
        if (tpr <= 32)
            return v;
        W *half = red + turn * NORM_MAX_WARPS;
        turn ^= 1;
        if (threadIdx.x % 32 == 0)
            half[threadIdx.x / 32] = v;
        __syncthreads();
        const int warps = tpr / 32, first = threadIdx.x / tpr * warps;
        W s = half[first];
        for (int k = 1; k < warps; k++)
            s += half[first + k];
        return s;
    }
};

// Rows on their way: a thread's packets of its next NORM_STAGES - 1 rows, in shared memory.  It reads nothing else
// there, so no barrier is needed.
constexpr int NORM_STAGES = 2;
extern __shared__ __align__(16) unsigned char norm_smem[];
template <typename T, int N, int PPT> struct RowRing {
    int operands, stage = 0;
    __device__ T *at(int stage, int operand, int k) const {
        return reinterpret_cast<T *>(norm_smem) + (((stage * operands + operand) * PPT + k) * (int)blockDim.x + (int)threadIdx.x) * N;
    }
    __device__ Vec<T, N> get(int operand, int k) const { return ld_vec<T, N>(at(stage, operand, k)); }
    __device__ int last() const { return stage == 0 ? NORM_STAGES - 1 : stage - 1; } // the one emptied last
    __device__ void next() { stage = stage == NORM_STAGES - 1 ? 0 : stage + 1; }
};
// A thread's two-byte elements of one row into the ring, which cannot be copied asynchronously: they are loaded all at once,
// without conditions (places without an element repeat the last one), since a load whose store to shared memory follows
// at once holds up the next one.
template <typename T, int N, int PPT>
__device__ __forceinline__ void fetch_row(const RowRing<T, N, PPT> &ring, int stage, int operand, const T *row, int tx, int tpr,
                                          int packets) {
    Vec<T, N> x[PPT];
#pragma unroll
    for (int k = 0; k < PPT; k++)
        x[k] = ld_vec<T, N>(row + (tx + k * tpr < packets ? tx + k * tpr : packets - 1) * N);
#pragma unroll
    for (int k = 0; k < PPT; k++)
        st_vec<T, N>(ring.at(stage, operand, k), x[k]);
}
size_t ring_bytes(size_t packet, int ppt, int operands, int block) {
    return (size_t)NORM_STAGES * operands * ppt * block * packet;
}

template <typename T> struct NormArgs { // x, residual and sum may be the same matrix, and res one of x and residual
    const T *x, *residual, *weight;
    T *sum;
    void *res; // T, or e4m3
    float *scales;
    wide_t<T> *rstd;
    int64_t rows, cols, x_ld, residual_ld, sum_ld, res_ld, scales_ld;
    int64_t group;  // columns per scale; 0: one scale a row
    int64_t groups; // scales per row
    wide_t<T> eps, share; // share: 1 / cols
};

template <typename T, int N>
__device__ __forceinline__ Vec<T, N> add_residual(const Vec<T, N> &x, const Vec<T, N> &r) {
    wide_t<T> a[N], b[N];
    widen_all(x, a);
    widen_all(r, b);
    add_all<N>(a, b, a);
    return narrow_all<T, N>(a);
}
template <typename T, int N> __device__ __forceinline__ void squares(const Vec<T, N> &s, wide_t<T> *sums) {
    wide_t<T> v[N];
    widen_all(s, v);
    dot_all<N>(v, v, sums);
}
// y of packet p
template <typename T, int N>
__device__ __forceinline__ void normalised(const Vec<T, N> &s, const T *weight, int64_t p, wide_t<T> rstd, wide_t<T> *y) {
    wide_t<T> r[N];
    set_all<N>(r, rstd);
    widen_all(s, y);
    mul_all<N>(y, r, y);
    if (weight) {
        widen_all(ld_vec<T, N>(weight + p * N), r);
        mul_all<N>(y, r, y);
    }
}
// max |y|, NaN if there is one, as an integer: the order of non-negative floats is that of their bits, and a NaN is above
// infinity, so that maxima over the bits do not depend on the order and keep a NaN
template <int N> __device__ __forceinline__ unsigned largest(const float *y) {
    float m = 0.0f;
#pragma unroll
    for (int k = 0; k < N; k++)
        asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(m), "f"(fabsf(y[k])));
    return __float_as_uint(m);
}
// 1 / rms is common to a row, so that y / scale = 448 * v / max|v| with v = s * weight: the quotient is formed from v, whose
// roundings are few, and rounded once.  v is taken times 7/8 and the power of two below 1 / rms, which rounds nothing
// and keeps it as large as y; in bf16 v and max|v| / 448 are then exact, and q is the nearest value to the definition's
// (a tie goes to the even one).  Rounding y and multiplying it by 1 / scale instead puts ties on either side: of 8192 x 5120
// bf16 values in groups of 128, 3968 were then a step of e4m3 off, and none are now (73.5 us then, 77.8 now).
struct RowScale {
    float by, back; // v = s * by * weight,  y = v * back
};
__device__ __forceinline__ RowScale row_scale(float rstd) {
    const unsigned bits = __float_as_uint(rstd), exponent = bits & 0x7f800000u;
    if (exponent == 0 || exponent == 0x7f800000u) // zero, infinite or NaN: as it is
        return {rstd, 8.0f / 7.0f};
    return {__uint_as_float(exponent) * 0.875f, __uint_as_float(bits - exponent + 0x3f800000u) * (8.0f / 7.0f)};
}
// What the values of a group are divided by, from the bits of their max|v|.  `by` is 0 where there is nothing to correct in
// two products by inv: a group with an infinity (its finite values give 0), and one whose scale, which never goes below
// the smallest normal number, does not follow its values.
struct Divisor {
    float scale, by, inv;
};
__device__ __forceinline__ Divisor divisor(unsigned most, float back) {
    constexpr float least = 1.17549435e-38f; // 2^-126
    if (most == 0)
        return {1.0f, 1.0f, 1.0f};
    const float by = __uint_as_float(most) / E4M3_MAX, scale = by * back;
    if (scale < least)
        return {least, 0.0f, back * 0.5f / least};
    return {scale, isinf(by) ? 0.0f : by, 1.0f / by};
}
template <int N> __device__ __forceinline__ void store_q8(void *res, int64_t at, float *y, const Divisor &d) {
    Vec<__nv_fp8_storage_t, N> q;
    float inv[N], by[N], first[N];
    set_all<N>(inv, d.inv);
    set_all<N>(by, -d.by);
    mul_all<N>(y, inv, first);
    fma_all<N>(first, by, y, y); // what the first quotient leaves, exactly
    fma_all<N>(y, inv, first, y);
    if constexpr (N == 1)
        q.v[0] = __nv_cvt_float_to_fp8(y[0], __NV_SATFINITE, __NV_E4M3);
    else {
#pragma unroll
        for (int k = 0; k < N; k += 2) {
            *reinterpret_cast<__nv_fp8x2_storage_t *>(&q.v[k]) =
                __nv_cvt_float2_to_fp8x2(make_float2(y[k], y[k + 1]), __NV_SATFINITE, __NV_E4M3);
        }
    }
    st_vec<__nv_fp8_storage_t, N>(static_cast<__nv_fp8_storage_t *>(res) + at, q);
}

// Rows of up to tpr * PPT packets: a thread holds packets tx, tx + tpr, ... of its row.  The CTA stays for many rows.
template <typename T, int N, int PPT, bool Q8>
__global__ void __launch_bounds__(NORM_MAX_WARPS * 32) norm_rows_kernel(NormArgs<T> a, int tpr) {
    using W = wide_t<T>;
    __shared__ W red[2 * NORM_MAX_WARPS];
    const int at_once = blockDim.x / tpr, tx = threadIdx.x % tpr, ty = threadIdx.x / tpr;
    const int packets = (int)(a.cols / N); // cols is a multiple of N
    RowSum<W> row_sum{red};
    RowRing<T, N, PPT> ring{a.residual ? 2 : 1};
    // rows of the CTA x groups (8-bit results whose groups span warps), behind the ring
    unsigned *group_max = reinterpret_cast<unsigned *>(ring.at(NORM_STAGES, 0, 0) - (int)threadIdx.x * N);
    const int64_t step = (int64_t)gridDim.x * at_once;
    auto load = [&](int stage, int64_t r) {
        if (r < a.rows) {
            if constexpr (sizeof(T) * N >= 4) {
#pragma unroll
                for (int k = 0; k < PPT; k++)
                    if (tx + k * tpr < packets) {
                        fetch<T, N>(ring.at(stage, 0, k), a.x + r * a.x_ld + (tx + k * tpr) * N);
                        if (a.residual)
                            fetch<T, N>(ring.at(stage, 1, k), a.residual + r * a.residual_ld + (tx + k * tpr) * N);
                    }
            } else {
                fetch_row(ring, stage, 0, a.x + r * a.x_ld, tx, tpr, packets);
                if (a.residual)
                    fetch_row(ring, stage, 1, a.residual + r * a.residual_ld, tx, tpr, packets);
            }
        }
        fetch_commit();
    };
    for (int i = 0; i < NORM_STAGES - 1; i++)
        load(i, (int64_t)blockIdx.x * at_once + ty + i * step);
    for (int64_t r0 = (int64_t)blockIdx.x * at_once; r0 < a.rows; r0 += step) {
        const int64_t r = r0 + ty;
        const bool live = r < a.rows;
        Vec<T, N> s[PPT];
        fetch_wait<NORM_STAGES - 2>();
        if (live) {
#pragma unroll
            for (int k = 0; k < PPT; k++)
                if (tx + k * tpr < packets) {
                    s[k] = ring.get(0, k);
                    if (a.residual)
                        s[k] = add_residual(s[k], ring.get(1, k));
                }
            if (a.sum) {
                T *sum = a.sum + r * a.sum_ld;
#pragma unroll
                for (int k = 0; k < PPT; k++)
                    if (tx + k * tpr < packets)
                        st_vec<T, N>(sum + (tx + k * tpr) * N, s[k]);
            }
        }
        load(ring.last(), r + (NORM_STAGES - 1) * step);
        ring.next();
        W ss[2] = {0, 0};
#pragma unroll
        for (int k = 0; k < PPT; k++)
            if (live && tx + k * tpr < packets)
                squares(s[k], ss);
        const W rstd = rsqrt(row_sum(ss[0] + ss[1], tpr) * a.share + a.eps); // every thread of a row: no divisions
        if (live && tx == 0 && a.rstd)
            a.rstd[r] = rstd;
        if constexpr (!Q8) {
            if (live) {
                T *res = static_cast<T *>(a.res) + r * a.res_ld;
#pragma unroll
                for (int k = 0; k < PPT; k++)
                    if (tx + k * tpr < packets) {
                        W y[N];
                        normalised<T, N>(s[k], a.weight, tx + k * tpr, rstd, y);
                        st_vec<T, N>(res + (tx + k * tpr) * N, narrow_all<T, N>(y));
                    }
            }
        } else {
            const RowScale by = row_scale(rstd);
            float y[PPT][N];
            unsigned most[PPT];
#pragma unroll
            for (int k = 0; k < PPT; k++) {
                most[k] = 0;
                if (live && tx + k * tpr < packets) {
                    normalised<T, N>(s[k], a.weight, tx + k * tpr, by.by, y[k]);
                    most[k] = largest<N>(y[k]);
                }
            }
            if (a.group == 0) {
#pragma unroll
                for (int k = 1; k < PPT; k++)
                    most[0] = max(most[0], most[k]);
#pragma unroll
                for (int k = 1; k < PPT; k++)
                    most[k] = most[0];
            }
            // threads that hold one group side by side, and whether a warp holds all of it
            const int64_t lanes64 = a.group == 0 ? tpr : a.group / N;
            const bool in_warp = lanes64 <= 32 && lanes64 <= tpr;
            const int lanes = (int)(in_warp ? lanes64 : (tpr < 32 ? tpr : 32));
#pragma unroll
            for (int k = 0; k < PPT; k++)
                for (int o = lanes >> 1; o >= 1; o >>= 1)
                    most[k] = max(most[k], __shfl_xor_sync(0xffffffffu, most[k], o));
            if (!in_warp) {
                unsigned *gm = group_max + ty * a.groups;
                for (int64_t g = tx; g < a.groups; g += tpr)
                    gm[g] = 0;
                __syncthreads();
#pragma unroll
                for (int k = 0; k < PPT; k++)
                    if (live && tx + k * tpr < packets && (tx & (lanes - 1)) == 0)
                        atomicMax(&gm[a.group == 0 ? 0 : (tx + k * tpr) * N / (int)a.group], most[k]);
                __syncthreads();
#pragma unroll
                for (int k = 0; k < PPT; k++)
                    if (tx + k * tpr < packets)
                        most[k] = gm[a.group == 0 ? 0 : (tx + k * tpr) * N / (int)a.group];
                __syncthreads();
            }
            if (live) {
#pragma unroll
                for (int k = 0; k < PPT; k++)
                    if (tx + k * tpr < packets) {
                        const Divisor d = divisor(most[k], by.back);
                        const int c = (tx + k * tpr) * N, group = (int)a.group;
                        if (group == 0 ? c == 0 : (c & (group - 1)) == 0)
                            a.scales[r * a.scales_ld + (group == 0 ? 0 : c / group)] = d.scale;
                        store_q8<N>(a.res, r * a.res_ld + c, y[k], d);
                    }
            }
        }
    }
}

// Rows that registers do not hold: one CTA per row, which is read again for every pass.  The sum is read back from where
// it was stored (the thread that stored a packet reads it), so x and residual may be overwritten by it.
constexpr int LONG_BLOCK = 512;
template <typename T, int N, bool Q8>
__global__ void __launch_bounds__(LONG_BLOCK) norm_long_kernel(NormArgs<T> a) {
    using W = wide_t<T>;
    __shared__ W red[2 * NORM_MAX_WARPS];
    __shared__ unsigned group_max[LONG_BLOCK * N / 16 + 1];
    const int64_t packets = a.cols / N; // cols is a multiple of N
    RowSum<W> row_sum{red};
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = a.x + r * a.x_ld, *residual = a.residual ? a.residual + r * a.residual_ld : nullptr;
        auto stream = [&](int64_t p) {
            const Vec<T, N> v = ld_vec<T, N>(x + p * N);
            return residual ? add_residual(v, ld_vec<T, N>(residual + p * N)) : v;
        };
        auto again = [&](int64_t p) {
            return a.sum ? ld_vec<T, N>(a.sum + r * a.sum_ld + p * N) : stream(p);
        };
        W ss[2] = {0, 0};
        for (int64_t p = threadIdx.x; p < packets; p += LONG_BLOCK) {
            const Vec<T, N> s = stream(p);
            if (a.sum)
                st_vec<T, N>(a.sum + r * a.sum_ld + p * N, s);
            squares(s, ss);
        }
        const W rstd = rsqrt(row_sum(ss[0] + ss[1], LONG_BLOCK) * a.share + a.eps);
        if (threadIdx.x == 0 && a.rstd)
            a.rstd[r] = rstd;
        if constexpr (!Q8) {
            for (int64_t p = threadIdx.x; p < packets; p += LONG_BLOCK) {
                W y[N];
                normalised<T, N>(again(p), a.weight, p, rstd, y);
                Vec<T, N> z;
#pragma unroll
                for (int k = 0; k < N; k++)
                    z.v[k] = narrow<T>(y[k]);
                st_vec<T, N>(static_cast<T *>(a.res) + r * a.res_ld + p * N, z);
            }
        } else {
            const RowScale by = row_scale(rstd);
            // turns of LONG_BLOCK packets, which hold whole groups (a group has at most 512 columns)
            unsigned row_most = 0;
            if (a.group == 0) {
                if (threadIdx.x == 0)
                    group_max[0] = 0;
                __syncthreads();
                for (int64_t p = threadIdx.x; p < packets; p += LONG_BLOCK) {
                    float y[N];
                    normalised<T, N>(again(p), a.weight, p, by.by, y);
                    row_most = max(row_most, largest<N>(y));
                }
                atomicMax(&group_max[0], row_most);
                __syncthreads();
                row_most = group_max[0];
                __syncthreads();
            }
            for (int64_t p0 = 0; p0 < packets; p0 += LONG_BLOCK) {
                const int64_t p = p0 + threadIdx.x;
                float y[N];
                unsigned most = row_most;
                if (p < packets)
                    normalised<T, N>(again(p), a.weight, p, by.by, y);
                if (a.group) {
                    const int g = (int)((int64_t)threadIdx.x * N / a.group);
                    for (int i = threadIdx.x; i < (int)(LONG_BLOCK * N / a.group) + 1; i += LONG_BLOCK)
                        group_max[i] = 0;
                    __syncthreads();
                    if (p < packets)
                        atomicMax(&group_max[g], largest<N>(y));
                    __syncthreads();
                    most = group_max[g];
                    __syncthreads();
                }
                if (p < packets) {
                    const Divisor d = divisor(most, by.back);
                    if (a.group == 0 ? p == 0 : p * N % a.group == 0)
                        a.scales[r * a.scales_ld + (a.group == 0 ? 0 : p * N / a.group)] = d.scale;
                    store_q8<N>(a.res, r * a.res_ld + p * N, y, d);
                }
            }
        }
    }
}

template <typename T> struct NormGradArgs { // dx may be the same matrix as grad, sum or dsum
    const T *grad, *sum, *weight, *dsum;
    const wide_t<T> *rstd;
    T *dx;
    wide_t<T> *part; // CTAs x part_ld column sums, or null
    int64_t rows, cols, grad_ld, sum_ld, dsum_ld, dx_ld, part_ld;
    wide_t<T> share; // 1 / cols
};

// dx of the rows, and the CTA's column sums of dy * s * rstd: a thread keeps the sums of its columns in registers over
// all rows that the CTA visits; the rows that a CTA holds at once are joined through shared memory in order.
template <typename T, int N, int PPT>
__global__ void __launch_bounds__(NORM_MAX_WARPS * 32) norm_grad_rows_kernel(NormGradArgs<T> a, int tpr) {
    using W = wide_t<T>;
    __shared__ W red[2 * NORM_MAX_WARPS];
    const int at_once = blockDim.x / tpr, tx = threadIdx.x % tpr, ty = threadIdx.x / tpr;
    const int packets = (int)(a.cols / N); // cols is a multiple of N
    RowSum<W> row_sum{red};
    RowRing<T, N, PPT> ring{a.dsum ? 3 : 2};
    W dw[PPT][N];
#pragma unroll
    for (int k = 0; k < PPT; k++)
#pragma unroll
        for (int j = 0; j < N; j++)
            dw[k][j] = 0;
    const int64_t step = (int64_t)gridDim.x * at_once;
    auto load = [&](int stage, int64_t r) {
        if (r < a.rows) {
            if constexpr (sizeof(T) * N >= 4) {
#pragma unroll
                for (int k = 0; k < PPT; k++)
                    if (tx + k * tpr < packets) {
                        fetch<T, N>(ring.at(stage, 0, k), a.grad + r * a.grad_ld + (tx + k * tpr) * N);
                        fetch<T, N>(ring.at(stage, 1, k), a.sum + r * a.sum_ld + (tx + k * tpr) * N);
                        if (a.dsum)
                            fetch<T, N>(ring.at(stage, 2, k), a.dsum + r * a.dsum_ld + (tx + k * tpr) * N);
                    }
            } else {
                fetch_row(ring, stage, 0, a.grad + r * a.grad_ld, tx, tpr, packets);
                fetch_row(ring, stage, 1, a.sum + r * a.sum_ld, tx, tpr, packets);
                if (a.dsum)
                    fetch_row(ring, stage, 2, a.dsum + r * a.dsum_ld, tx, tpr, packets);
            }
        }
        fetch_commit();
    };
    for (int i = 0; i < NORM_STAGES - 1; i++)
        load(i, (int64_t)blockIdx.x * at_once + ty + i * step);
    W next_rstd = (int64_t)blockIdx.x * at_once + ty < a.rows ? a.rstd[(int64_t)blockIdx.x * at_once + ty] : W(0);
    for (int64_t r0 = (int64_t)blockIdx.x * at_once; r0 < a.rows; r0 += step) {
        const int64_t r = r0 + ty;
        const bool live = r < a.rows;
        const int64_t row = r;
        const W rstd = next_rstd;
        next_rstd = r + step < a.rows ? a.rstd[r + step] : W(0);
        load(ring.last(), r + (NORM_STAGES - 1) * step);
        fetch_wait<NORM_STAGES - 1>();
        W dots[2] = {0, 0}, t[PPT][N], v[PPT][N]; // t = dy * weight, v = s
        if (live) {
#pragma unroll
            for (int k = 0; k < PPT; k++)
                if (tx + k * tpr < packets) {
                    W x[N], r[N];
                    widen_all(ring.get(0, k), t[k]);
                    widen_all(ring.get(1, k), v[k]);
                    set_all<N>(r, rstd);
                    mul_all<N>(v[k], r, x);
                    fma_all<N>(t[k], x, dw[k], dw[k]);
                    if (a.weight) {
                        widen_all(ld_vec<T, N>(a.weight + (tx + k * tpr) * N), x);
                        mul_all<N>(t[k], x, t[k]);
                    }
                    dot_all<N>(t[k], v[k], dots);
                }
        }
        const W factor = row_sum(dots[0] + dots[1], tpr) * a.share * rstd * rstd;
        if (live) {
            W f[N], r[N];
            set_all<N>(f, -factor);
            set_all<N>(r, rstd);
#pragma unroll
            for (int k = 0; k < PPT; k++)
                if (tx + k * tpr < packets) {
                    fma_all<N>(v[k], f, t[k], v[k]);
                    if (a.dsum) {
                        W d[N];
                        widen_all(ring.get(2, k), d);
                        fma_all<N>(v[k], r, d, v[k]);
                    } else
                        mul_all<N>(v[k], r, v[k]);
                    st_vec<T, N>(a.dx + row * a.dx_ld + (tx + k * tpr) * N, narrow_all<T, N>(v[k]));
                }
        }
        ring.next();
    }
    start_next(); // not earlier: CTAs that only wait take their places among those that work
    if (!a.part)
        return;
    W *part = a.part + (int64_t)blockIdx.x * a.part_ld;
    if (at_once == 1) {
#pragma unroll
        for (int k = 0; k < PPT; k++)
            if (tx + k * tpr < packets)
#pragma unroll
                for (int j = 0; j < N; j++)
                    part[(tx + k * tpr) * N + j] = dw[k][j];
        return;
    }
    fetch_wait<0>();
    W *join = reinterpret_cast<W *>(norm_smem); // over the ring
#pragma unroll
    for (int k = 0; k < PPT; k++) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < N; j++)
            join[threadIdx.x * N + j] = dw[k][j];
        __syncthreads();
        if (ty == 0 && tx + k * tpr < packets)
#pragma unroll
            for (int j = 0; j < N; j++) {
                W v = join[tx * N + j];
                for (int i = 1; i < at_once; i++)
                    v += join[(i * tpr + tx) * N + j];
                part[(tx + k * tpr) * N + j] = v;
            }
    }
}

template <typename T, int N>
__global__ void __launch_bounds__(LONG_BLOCK) norm_grad_long_kernel(NormGradArgs<T> a) {
    using W = wide_t<T>;
    __shared__ W red[2 * NORM_MAX_WARPS];
    const int64_t packets = a.cols / N; // cols is a multiple of N
    RowSum<W> row_sum{red};
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *g = a.grad + r * a.grad_ld, *s = a.sum + r * a.sum_ld;
        const W rstd = a.rstd[r];
        W dot = 0;
        for (int64_t p = threadIdx.x; p < packets; p += LONG_BLOCK) {
            const Vec<T, N> gv = ld_vec<T, N>(g + p * N), sv = ld_vec<T, N>(s + p * N);
            Vec<T, N> w;
            if (a.weight)
                w = ld_vec<T, N>(a.weight + p * N);
#pragma unroll
            for (int j = 0; j < N; j++)
                dot += (a.weight ? widen(gv.v[j]) * widen(w.v[j]) : W(widen(gv.v[j]))) * widen(sv.v[j]);
        }
        const W factor = row_sum(dot, LONG_BLOCK) * a.share * rstd * rstd;
        for (int64_t p = threadIdx.x; p < packets; p += LONG_BLOCK) {
            const Vec<T, N> gv = ld_vec<T, N>(g + p * N), sv = ld_vec<T, N>(s + p * N);
            Vec<T, N> w, d, z;
            if (a.weight)
                w = ld_vec<T, N>(a.weight + p * N);
            if (a.dsum)
                d = ld_vec<T, N>(a.dsum + r * a.dsum_ld + p * N);
#pragma unroll
            for (int j = 0; j < N; j++) {
                W v = rstd * ((a.weight ? widen(gv.v[j]) * widen(w.v[j]) : W(widen(gv.v[j]))) - widen(sv.v[j]) * factor);
                if (a.dsum)
                    v += widen(d.v[j]);
                z.v[j] = narrow<T>(v);
            }
            st_vec<T, N>(a.dx + r * a.dx_ld + p * N, z);
        }
    }
}

// column sums of dy * s * rstd for the long rows: CTA (x, y) takes 32 columns and every gridDim.y-th group of 8 rows
// (launched before dx is written, which may be the same matrix as grad or sum)
template <typename T> __global__ void __launch_bounds__(256) norm_dweight_kernel(NormGradArgs<T> a) {
    using W = wide_t<T>;
    __shared__ W sums[8][33];
    const int tx = threadIdx.x % 32, ty = threadIdx.x / 32;
    const int64_t c = (int64_t)blockIdx.x * 32 + tx;
    W v = 0;
    if (c < a.cols)
        for (int64_t r = (int64_t)blockIdx.y * 8 + ty; r < a.rows; r += (int64_t)gridDim.y * 8)
            v += widen(a.grad[r * a.grad_ld + c]) * (widen(a.sum[r * a.sum_ld + c]) * a.rstd[r]);
    sums[ty][tx] = v;
    __syncthreads();
    if (ty == 0 && c < a.cols) {
        for (int k = 1; k < 8; k++)
            v += sums[k][tx];
        a.part[(int64_t)blockIdx.y * a.part_ld + c] = v;
    }
}

// dweight[c] = sum over the parts, in order within JOIN_SHARES shares and over the shares
constexpr int JOIN_SHARES = 32;
template <typename W>
__global__ void __launch_bounds__(32 * JOIN_SHARES)
    norm_join_kernel(const W *__restrict__ part, int parts, int64_t cols, int64_t part_ld, W *__restrict__ res) {
    __shared__ W sums[JOIN_SHARES][33];
    wait_for_last();
    const int tx = threadIdx.x % 32, ty = threadIdx.x / 32;
    const int64_t c = (int64_t)blockIdx.x * 32 + tx;
    const int share = (parts + JOIN_SHARES - 1) / JOIN_SHARES, first = ty * share;
    const int last = first + share < parts ? first + share : parts;
    W v = 0;
    if (c < cols) {
#pragma unroll 16
        for (int i = first; i < last; i++)
            v += part[(int64_t)i * part_ld + c];
    }
    sums[ty][tx] = v;
    __syncthreads();
    if (ty == 0 && c < cols) {
        for (int k = 1; k < JOIN_SHARES; k++)
            v += sums[k][tx];
        res[c] = v;
    }
}

// How many threads share a row and how many packets each holds: the fewest places without a packet, and among equal ones
// the most packets a thread.  Few rows (fewer than SMs): as few packets a thread as fit, which shortens the way of the
// single row.
struct RowPlan {
    int tpr, ppt, block;
    bool fits;
};
constexpr int NORM_SMEM = 210 << 10, NORM_RING = 192 << 10; // of a CTA: all, and the ring
RowPlan row_plan(int64_t packets, int64_t rows, int first, int most, int step, int place_bytes) {
    RowPlan p{0, 0, 0, false};
    for (int ppt = first; ppt <= most; ppt += step) {
        int64_t tpr = (packets + ppt - 1) / ppt;
        tpr = tpr < 32 ? next_pow2(tpr < 8 ? 8 : tpr) : (tpr + 31) / 32 * 32;
        if (tpr > NORM_MAX_WARPS * 32 || tpr * ppt * place_bytes > NORM_RING)
            continue;
        if (!p.fits || (rows >= sm_count() && tpr * ppt <= (int64_t)p.tpr * p.ppt)) {
            p.tpr = (int)tpr;
            p.ppt = ppt;
            p.fits = true;
        }
    }
    p.block = p.fits ? p.tpr * (p.tpr < 256 ? 256 / p.tpr : 1) : 0;
    return p;
}
// packets a thread that there are kernels for: 1 to 3 (gradient: 4), or 4 smaller ones
template <typename T, int N> RowPlan row_plan(int64_t cols, int64_t rows, bool back) {
    const int place = NORM_STAGES * (back ? 3 : 2) * N * (int)sizeof(T);
    return N <= 2 && sizeof(T) * N < 16 ? row_plan(cols / N, rows, 4, 4, 1, place) : row_plan(cols / N, rows, 1, back ? 4 : 3, 1, place);
}
#define DB2_BY_PACKETS(N, BACK, ppt, LAUNCH)                                                                                 \
    if constexpr (N * sizeof(T) < 16) {                                                                                \
        LAUNCH(4)                                                                                                      \
    } else if (ppt == 1) {                                                                                             \
        LAUNCH(1)                                                                                                      \
    } else if (ppt == 2) {                                                                                             \
        LAUNCH(2)                                                                                                      \
    } else if (ppt == 3) {                                                                                             \
        LAUNCH(3)                                                                                                      \
    } else {                                                                                                           \
        if constexpr (BACK) {                                                                                          \
            LAUNCH(4)                                                                                                  \
        }                                                                                                              \
    }

// CTAs that stay on the device for all rows
template <typename K> int resident_ctas(K kernel, PerDeviceOnce &once, int block, size_t smem, int64_t most, unsigned *ctas) {
    DB2_CHECK(smem <= (size_t)NORM_SMEM, DB2_ECUDA, "rmsNorm: %zu bytes of shared memory", smem);
    if (once.need()) {
        DB2_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, NORM_SMEM));
        once.mark();
    }
    *ctas = (unsigned)most;
    if (most <= sm_count())
        return DB2_OK;
    int per_sm = 1;
    DB2_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, block, smem));
    DB2_CHECK(per_sm > 0, DB2_ECUDA, "rmsNorm: the kernel does not fit on an SM");
    // more than 1024 threads of an SM get in one another's way at the memory: 16384 x 4096 bf16 forward takes 87 us with
    // four CTAs of 256 on an SM, 101 with six
    const int most_per_sm = (1024 + block - 1) / block;
    const int64_t n = (int64_t)sm_count() * (per_sm < most_per_sm ? per_sm : most_per_sm);
    *ctas = (unsigned)(most < n ? most : n);
    return DB2_OK;
}

template <typename T, int N, bool Q8> int norm_launch(const NormArgs<T> &a, cudaStream_t st) {
    const RowPlan p = row_plan<T, N>(a.cols, a.rows, false);
    if (!p.fits) {
        const int64_t max_grid = (int64_t)1 << 30;
        norm_long_kernel<T, N, Q8><<<(unsigned)(a.rows < max_grid ? a.rows : max_grid), LONG_BLOCK, 0, st>>>(a);
        return after_launch("norm_long_kernel");
    }
    const int at_once = p.block / p.tpr;
    unsigned grid = 0;
#define DB2_NORM(PPT)                                                                                                  \
    const size_t smem = ring_bytes(sizeof(T) * N, PPT, a.residual ? 2 : 1, p.block) + (Q8 ? at_once * a.groups * 4 : 0); \
    static PerDeviceOnce once;                                                                                         \
    DB2_TRY(resident_ctas(norm_rows_kernel<T, N, PPT, Q8>, once, p.block, smem, (a.rows + at_once - 1) / at_once, &grid));   \
    norm_rows_kernel<T, N, PPT, Q8><<<grid, p.block, smem, st>>>(a, p.tpr);
    DB2_BY_PACKETS(N, false, p.ppt, DB2_NORM)
#undef DB2_NORM
    return after_launch("norm_rows_kernel");
}

// most CTAs of the gradient kernel: each keeps its own column sums
int64_t grad_ctas(int64_t rows) {
    const int64_t cap = (int64_t)sm_count() * 8;
    return rows < 1 ? 1 : (rows < cap ? rows : cap);
}

template <typename T, int N> int norm_grad_launch(NormGradArgs<T> a, wide_t<T> *dweight, cudaStream_t st) {
    const RowPlan p = row_plan<T, N>(a.cols, a.rows, true);
    const int64_t ctas = grad_ctas(a.rows);
    int parts;
    if (!p.fits) {
        parts = (int)(ctas < 16 ? ctas : 16);
        if (a.part) {
            norm_dweight_kernel<T><<<dim3((unsigned)((a.cols + 31) / 32), (unsigned)parts), 256, 0, st>>>(a);
            DB2_TRY(after_launch("norm_dweight_kernel"));
        }
        norm_grad_long_kernel<T, N><<<(unsigned)ctas, LONG_BLOCK, 0, st>>>(a);
        DB2_TRY(after_launch("norm_grad_long_kernel"));
    } else {
        const int at_once = p.block / p.tpr;
        const int64_t blocks = (a.rows + at_once - 1) / at_once;
        unsigned grid = 0;
#define DB2_NORM_GRAD(PPT)                                                                                             \
    size_t smem = ring_bytes(sizeof(T) * N, PPT, a.dsum ? 3 : 2, p.block);                                             \
    if (smem < p.block * N * sizeof(wide_t<T>)) /* where the rows of a CTA are joined */                               \
        smem = p.block * N * sizeof(wide_t<T>);                                                                        \
    static PerDeviceOnce once;                                                                                         \
    DB2_TRY(resident_ctas(norm_grad_rows_kernel<T, N, PPT>, once, p.block, smem, blocks < ctas ? blocks : ctas, &grid));     \
    norm_grad_rows_kernel<T, N, PPT><<<grid, p.block, smem, st>>>(a, p.tpr);
        DB2_BY_PACKETS(N, true, p.ppt, DB2_NORM_GRAD)
#undef DB2_NORM_GRAD
        DB2_TRY(after_launch("norm_grad_rows_kernel"));
        parts = (int)grid;
    }
    if (a.part) {
        DB2_TRY(launch_next("norm_join_kernel", norm_join_kernel<wide_t<T>>, dim3((unsigned)((a.cols + 31) / 32)),
                            32 * JOIN_SHARES, 0, st, a.part, parts, a.cols, a.part_ld, dweight));
    }
    return DB2_OK;
}
#undef DB2_BY_PACKETS

int64_t part_ld_of(int64_t cols) { return (cols + 7) / 8 * 8; }

bool seq_type(int dtype) {
    return dtype == DB2_F64 || dtype == DB2_F32 || dtype == DB2_F16 || dtype == DB2_BF16;
}

// the arguments that both forms of the norm share
int check_norm(const char *what, const void *x, int64_t rows, int64_t cols, int64_t x_ld, const void *residual,
               int64_t residual_ld, double eps, const void *sum, int64_t sum_ld, const void *res, int64_t res_ld) {
    DB2_CHECK(eps >= 0.0, DB2_EINVAL, "%s: eps must not be negative", what);
    DB2_CHECK(cols > 0, DB2_EINVAL, "%s: rows without columns have no mean", what);
    DB2_CHECK(x && res, DB2_EINVAL, "%s: null operand", what);
    DB2_CHECK(ld_ok(x_ld, rows, cols) && (!residual || ld_ok(residual_ld, rows, cols)) &&
                  (!sum || ld_ok(sum_ld, rows, cols)) && ld_ok(res_ld, rows, cols),
              DB2_EINVAL, "%s: a leading dimension is smaller than the number of columns", what);
    return DB2_OK;
}

void count(db2_context *ctx, uint64_t before) {
    std::lock_guard<std::mutex> lock(ctx->mu);
    ctx->stats.launches += g_launches.load(std::memory_order_relaxed) - before;
}

// checks of the handle forms that compare matrices with one another
int check_operands(const char *what, const db2_matrix *x, const db2_matrix *other, const char *name) {
    DB2_CHECK(!other || (other->dtype == x->dtype && other->rows == x->rows && other->cols == x->cols), DB2_EINVAL,
              "%s: %s must have the shape and value type of the first argument", what, name);
    return DB2_OK;
}
int check_weight(const char *what, const db2_matrix *x, const db2_matrix *weight) {
    DB2_CHECK(!weight || (weight->dtype == x->dtype && weight->rows == 1 && weight->cols == x->cols), DB2_EINVAL,
              "%s: weight must be a row matrix of %lld columns and of the same value type", what, (long long)x->cols);
    return DB2_OK;
}
int wide_dtype(int dtype) { return dtype == DB2_F64 ? DB2_F64 : DB2_F32; }

// rmsNorm (scales == nullptr) and rmsNormQ8 on handles
int norm_on_handles(db2_context *ctx, const char *what, db2_matrix **res, db2_matrix **scales, db2_matrix **sum,
                    db2_matrix **rstd, db2_matrix *x, db2_matrix *residual, db2_matrix *weight, double eps,
                    int64_t group) {
    DB2_CHECK(seq_type(x->dtype) && (!scales || x->dtype != DB2_F64), DB2_EUNSUPPORTED,
              "%s: unsupported value type code %d", what, x->dtype);
    DB2_CHECK(eps >= 0.0, DB2_EINVAL, "%s: eps must not be negative", what);
    DB2_CHECK(x->cols > 0 || x->rows == 0, DB2_EINVAL, "%s: rows without columns have no mean", what);
    DB2_TRY(check_operands(what, x, residual, "residual"));
    DB2_TRY(check_weight(what, x, weight));
    DB2_CHECK(!scales || group == 0 || (group >= 16 && group <= 512 && (group & (group - 1)) == 0), DB2_EINVAL,
              "%s: groups of 16, 32, 64, 128, 256 or 512 columns, or 0 for the whole row (got %lld)", what,
              (long long)group);
    bind_device(ctx);
    const uint64_t before = g_launches.load();
    Results results;
    DB2_TRY(results.add(what, res, scales ? DB2_F8E4M3 : x->dtype, x->rows, x->cols));
    DB2_TRY(results.add(what, scales, DB2_F32, x->rows, group ? (x->cols + group - 1) / group : 1));
    DB2_TRY(results.add(what, sum, x->dtype, x->rows, x->cols));
    DB2_TRY(results.add(what, rstd, wide_dtype(x->dtype), x->rows, 1));
    const DeviceOperand dx(x), dres(residual), dw(weight);
    DB2_TRY(results.apart(what, x, {res, sum}));
    DB2_TRY(results.apart(what, residual, {res, sum}));
    DB2_TRY(results.apart(what, weight));
    // (a buffer that others read as well is replaced)
    DB2_CHECK(!rstd || !*rstd || x->rows <= 1 || !(*rstd)->dev || (*rstd)->dev_ld == 1 ||
                  (!(*rstd)->is_view && (*rstd)->dev.use_count() > 1),
              DB2_EUNSUPPORTED, "%s: rstd into a strided result view", what);
    DB2_TRY(prepare_result(ctx, res, scales ? DB2_F8E4M3 : x->dtype, x->rows, x->cols));
    if (scales)
        DB2_TRY(prepare_result(ctx, scales, DB2_F32, x->rows, group ? (x->cols + group - 1) / group : 1));
    if (sum)
        DB2_TRY(prepare_result(ctx, sum, x->dtype, x->rows, x->cols));
    if (rstd)
        DB2_TRY(prepare_result(ctx, rstd, wide_dtype(x->dtype), x->rows, 1));
    if (x->rows > 0) {
        void *sp = sum ? (*sum)->dev_ptr() : nullptr, *tp = rstd ? (*rstd)->dev_ptr() : nullptr;
        const int64_t sld = sum ? (*sum)->dev_ld : 0;
        if (scales)
            DB2_TRY(db2k_rms_norm_q8(x->dtype, dx.ptr, x->rows, x->cols, dx.ld, dres.ptr, dres.ld, dw.ptr, eps, sp, sld,
                                     (*res)->dev_ptr(), (*res)->dev_ld, (*scales)->dev_ptr(), (*scales)->dev_ld, group,
                                     tp, ctx->stream));
        else
            DB2_TRY(db2k_rms_norm(x->dtype, dx.ptr, x->rows, x->cols, dx.ld, dres.ptr, dres.ld, dw.ptr, eps, sp, sld,
                                  (*res)->dev_ptr(), (*res)->dev_ld, tp, ctx->stream));
    }
    count(ctx, before);
    return results.done();
}

} // namespace
} // namespace db2

using namespace db2;

extern "C" {

int db2k_rms_norm(int dtype, const void *x, int64_t rows, int64_t cols, int64_t x_ld, const void *residual,
                  int64_t residual_ld, const void *weight, double eps, void *sum, int64_t sum_ld, void *res,
                  int64_t res_ld, void *rstd, void *stream) {
    DB2_CHECK(seq_type(dtype), DB2_EUNSUPPORTED, "rmsNorm: unsupported value type code %d", dtype);
    DB2_CHECK(rows >= 0 && cols >= 0, DB2_EINVAL, "rmsNorm: negative shape");
    if (rows == 0)
        return DB2_OK;
    DB2_TRY(check_norm("rmsNorm", x, rows, cols, x_ld, residual, residual_ld, eps, sum, sum_ld, res, res_ld));
    DB2_DISPATCH_SEQ(dtype, T, {
        constexpr int N = 16 / sizeof(T);
        NormArgs<T> a{static_cast<const T *>(x), static_cast<const T *>(residual), static_cast<const T *>(weight),
                      static_cast<T *>(sum), res, nullptr, static_cast<wide_t<T> *>(rstd), rows, cols, x_ld,
                      residual_ld, sum_ld, res_ld, 0, 0, 0, (wide_t<T>)eps, wide_t<T>(1) / wide_t<T>(cols)};
        auto packed = [&](int n) {
            const size_t b = n * sizeof(T);
            return cols % n == 0 && rows_aligned(x, x_ld, sizeof(T), b) && rows_aligned(residual, residual_ld, sizeof(T), b) &&
                   rows_aligned(weight, 0, sizeof(T), b) && rows_aligned(sum, sum_ld, sizeof(T), b) &&
                   rows_aligned(res, res_ld, sizeof(T), b);
        };
        if (packed(N))
            return norm_launch<T, N, false>(a, as_stream(stream));
        return N > 2 && packed(2) ? norm_launch<T, 2, false>(a, as_stream(stream))
                                  : norm_launch<T, 1, false>(a, as_stream(stream));
    });
    return DB2_OK;
}

int db2k_rms_norm_q8(int dtype, const void *x, int64_t rows, int64_t cols, int64_t x_ld, const void *residual,
                     int64_t residual_ld, const void *weight, double eps, void *sum, int64_t sum_ld, void *res,
                     int64_t res_ld, void *scales, int64_t scales_ld, int64_t group, void *rstd, void *stream) {
    DB2_CHECK(seq_type(dtype) && dtype != DB2_F64, DB2_EUNSUPPORTED, "rmsNormQ8: unsupported value type code %d", dtype);
    DB2_CHECK(rows >= 0 && cols >= 0, DB2_EINVAL, "rmsNormQ8: negative shape");
    DB2_CHECK(group == 0 || (group >= 16 && group <= 512 && (group & (group - 1)) == 0), DB2_EINVAL,
              "rmsNormQ8: groups of 16, 32, 64, 128, 256 or 512 columns, or 0 for the whole row (got %lld)",
              (long long)group);
    if (rows == 0)
        return DB2_OK;
    DB2_TRY(check_norm("rmsNormQ8", x, rows, cols, x_ld, residual, residual_ld, eps, sum, sum_ld, res, res_ld));
    const int64_t groups = group ? (cols + group - 1) / group : 1;
    DB2_CHECK(scales && ld_ok(scales_ld, rows, groups), DB2_EINVAL,
              "rmsNormQ8: null scales or their leading dimension smaller than the number of groups");
    auto go = [&](auto tag) {
        using T = decltype(tag);
        constexpr int N = 16 / sizeof(T);
        NormArgs<T> a{static_cast<const T *>(x), static_cast<const T *>(residual), static_cast<const T *>(weight),
                      static_cast<T *>(sum), res, static_cast<float *>(scales), static_cast<float *>(rstd), rows, cols,
                      x_ld, residual_ld, sum_ld, res_ld, scales_ld, group, groups, (float)eps, 1.0f / (float)cols};
        auto packed = [&](int n) {
            const size_t b = n * sizeof(T);
            return cols % n == 0 && rows_aligned(x, x_ld, sizeof(T), b) && rows_aligned(residual, residual_ld, sizeof(T), b) &&
                   rows_aligned(weight, 0, sizeof(T), b) && rows_aligned(sum, sum_ld, sizeof(T), b) &&
                   rows_aligned(res, res_ld, 1, n);
        };
        if (packed(N))
            return norm_launch<T, N, true>(a, as_stream(stream));
        return packed(2) ? norm_launch<T, 2, true>(a, as_stream(stream)) : norm_launch<T, 1, true>(a, as_stream(stream));
    };
    return dtype == DB2_F32 ? go(float()) : dtype == DB2_F16 ? go(__half()) : go(__nv_bfloat16());
}

size_t db2k_rms_norm_grad_scratch_bytes(int dtype, int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0)
        return 0;
    return (size_t)grad_ctas(rows) * part_ld_of(cols) * (dtype == DB2_F64 ? 8 : 4);
}

int db2k_rms_norm_grad(int dtype, const void *grad, int64_t grad_ld, int64_t rows, int64_t cols, const void *sum,
                       int64_t sum_ld, const void *weight, const void *rstd, const void *dsum, int64_t dsum_ld, void *dx,
                       int64_t dx_ld, void *dweight, void *scratch, size_t scratch_bytes, void *stream) {
    DB2_CHECK(seq_type(dtype), DB2_EUNSUPPORTED, "rmsNormGrad: unsupported value type code %d", dtype);
    DB2_CHECK(rows >= 0 && cols >= 0, DB2_EINVAL, "rmsNormGrad: negative shape");
    if (cols == 0)
        return DB2_OK;
    if (rows == 0) {
        if (dweight)
            DB2_CUDA(cudaMemsetAsync(dweight, 0, (size_t)cols * (dtype == DB2_F64 ? 8 : 4), as_stream(stream)));
        return DB2_OK;
    }
    DB2_CHECK(grad && sum && rstd && dx, DB2_EINVAL, "rmsNormGrad: null operand");
    DB2_CHECK(ld_ok(grad_ld, rows, cols) && ld_ok(sum_ld, rows, cols) && (!dsum || ld_ok(dsum_ld, rows, cols)) &&
                  ld_ok(dx_ld, rows, cols),
              DB2_EINVAL, "rmsNormGrad: a leading dimension is smaller than the number of columns");
    DB2_CHECK(!dweight || (scratch && scratch_bytes >= db2k_rms_norm_grad_scratch_bytes(dtype, rows, cols) &&
                           aligned16(scratch)),
              DB2_EINVAL, "rmsNormGrad: scratch smaller than db2k_rms_norm_grad_scratch_bytes, or not 16-byte aligned");
    DB2_DISPATCH_SEQ(dtype, T, {
        constexpr int N = 16 / sizeof(T);
        NormGradArgs<T> a{static_cast<const T *>(grad), static_cast<const T *>(sum), static_cast<const T *>(weight),
                          static_cast<const T *>(dsum), static_cast<const wide_t<T> *>(rstd), static_cast<T *>(dx),
                          dweight ? static_cast<wide_t<T> *>(scratch) : nullptr, rows, cols, grad_ld, sum_ld, dsum_ld,
                          dx_ld, part_ld_of(cols), wide_t<T>(1) / wide_t<T>(cols)};
        auto packed = [&](int n) {
            const size_t b = n * sizeof(T);
            return cols % n == 0 && rows_aligned(grad, grad_ld, sizeof(T), b) && rows_aligned(sum, sum_ld, sizeof(T), b) &&
                   rows_aligned(weight, 0, sizeof(T), b) && rows_aligned(dsum, dsum_ld, sizeof(T), b) &&
                   rows_aligned(dx, dx_ld, sizeof(T), b);
        };
        wide_t<T> *dw = static_cast<wide_t<T> *>(dweight);
        if (packed(N))
            return norm_grad_launch<T, N>(a, dw, as_stream(stream));
        return N > 2 && packed(2) ? norm_grad_launch<T, 2>(a, dw, as_stream(stream))
                                  : norm_grad_launch<T, 1>(a, dw, as_stream(stream));
    });
    return DB2_OK;
}

int db2_rmsNorm(db2_context *ctx, db2_matrix **res, db2_matrix **sum, db2_matrix **rstd, db2_matrix *x,
                db2_matrix *residual, db2_matrix *weight, double eps) {
    DB2_API_BEGIN
    DB2_CHECK(ctx && res && x, DB2_EINVAL, "null argument");
    return norm_on_handles(ctx, "rmsNorm", res, nullptr, sum, rstd, x, residual, weight, eps, 0);
    DB2_API_END
}

int db2_rmsNormQ8(db2_context *ctx, db2_matrix **res, db2_matrix **scales, db2_matrix **sum, db2_matrix **rstd,
                  db2_matrix *x, db2_matrix *residual, db2_matrix *weight, double eps, int64_t group) {
    DB2_API_BEGIN
    DB2_CHECK(ctx && res && scales && x, DB2_EINVAL, "null argument");
    return norm_on_handles(ctx, "rmsNormQ8", res, scales, sum, rstd, x, residual, weight, eps, group);
    DB2_API_END
}

int db2_rmsNormGrad(db2_context *ctx, db2_matrix **dx, db2_matrix **dweight, db2_matrix *grad, db2_matrix *sum,
                    db2_matrix *weight, db2_matrix *rstd, db2_matrix *dsum) {
    DB2_API_BEGIN
    DB2_CHECK(ctx && dx && grad && sum && rstd, DB2_EINVAL, "null argument");
    DB2_CHECK(seq_type(grad->dtype), DB2_EUNSUPPORTED, "rmsNormGrad: unsupported value type code %d", grad->dtype);
    DB2_TRY(check_operands("rmsNormGrad", grad, sum, "sum"));
    DB2_TRY(check_operands("rmsNormGrad", grad, dsum, "dsum"));
    DB2_TRY(check_weight("rmsNormGrad", grad, weight));
    DB2_CHECK(rstd->dtype == wide_dtype(grad->dtype) && rstd->rows == grad->rows && rstd->cols == 1, DB2_EINVAL,
              "rmsNormGrad: rstd must be the column matrix that rmsNorm gave");
    bind_device(ctx);
    const uint64_t before = g_launches.load();
    const DeviceOperand dg(grad), ds(sum), dw(weight), dr(rstd), dd(dsum);
    DB2_CHECK(dr.ld == 1 || grad->rows <= 1, DB2_EUNSUPPORTED, "rmsNormGrad: rstd is a strided view");
    Results results;
    DB2_TRY(results.add("rmsNormGrad", dx, grad->dtype, grad->rows, grad->cols));
    DB2_TRY(results.add("rmsNormGrad", dweight, wide_dtype(grad->dtype), 1, grad->cols));
    for (const db2_matrix *m : {grad, sum, dsum})
        DB2_TRY(results.apart("rmsNormGrad", m, {dx}));
    for (const db2_matrix *m : {weight, rstd})
        DB2_TRY(results.apart("rmsNormGrad", m));
    DB2_TRY(prepare_result(ctx, dx, grad->dtype, grad->rows, grad->cols));
    if (dweight)
        DB2_TRY(prepare_result(ctx, dweight, wide_dtype(grad->dtype), 1, grad->cols));
    const size_t sb = db2k_rms_norm_grad_scratch_bytes(grad->dtype, grad->rows, grad->cols);
    void *scratch = nullptr;
    DB2_TRY(ctx_scratch(ctx, sb, &scratch));
    DB2_TRY(db2k_rms_norm_grad(grad->dtype, dg.ptr, dg.ld, grad->rows, grad->cols, ds.ptr, ds.ld, dw.ptr, dr.ptr, dd.ptr,
                               dd.ld, (*dx)->dev_ptr(), (*dx)->dev_ld, dweight ? (*dweight)->dev_ptr() : nullptr,
                               scratch, ctx->scratch_bytes, ctx->stream));
    count(ctx, before);
    return results.done();
    DB2_API_END
}

} // extern "C"
