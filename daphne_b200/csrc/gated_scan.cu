// Gated linear recurrence down the rows of every column, over packed sequences of rows, its gradient, and its step for
// one new row per sequence.
//
//   h[t] = f[t] * h[t-1] + u[t]          DB2_GATE_DECAY:   f = g,           u = x
//                                        DB2_GATE_SIGMOID: f = sigmoid(g),  u = (1 - f) * x
//   gradient, from the last row up (c = what row t + 1 sends to row t, at first the gradient of the last state):
//     delta[t] = dh[t] + c     dg = delta * h[t-1] (SIGMOID: delta * (h[t-1] - x) * f * (1 - f))
//     c = f[t] * delta[t]      dx = delta          (SIGMOID: delta * (1 - f))                      dh0 = the last c
//
// Both are first-order recurrences v <- a * v + b, and the composition of two such steps is one again: (A, B) of a run of
// rows says all about it.  A warp holds 8 (gradient: 4) consecutive rows of 32 lanes x VEC columns in registers and forms their
// (A, B); the warps of a CTA exchange theirs through shared memory; every warp then walks its rows once more, from the
// value that really enters them.  So each operand is read once and each result written once.
//
// Bound by memory.  States, gates and products are float (double for double); the stored h is rounded once, the running
// state never.  The gradient reads h as it was stored, which is what a caller has: where a rounded h enters dg = delta *
// h[t-1], dg is off by 1.85e-3 of its size in bf16, with the state of the forward pass it would be by the 1.66e-3 that its
// own rounding costs.
#include "runtime.h"
#include "seq.cuh"

namespace db2 {

namespace {

// A lane takes 8 bytes of a row, a warp several consecutive rows at once.  More rows would spread the exchange between the
// warps over more work, but the gates and inputs of a thread's rows have to stay in its registers.
template <typename T> constexpr int widest() { return 8 / sizeof(T); }
template <bool BACK> constexpr int scan_rows() { return BACK ? 4 : 8; }
// Rows on their way lie in shared memory, so many tiles (rows of all warps) of them, copied asynchronously.
constexpr int SCAN_STAGES = 3;

template <typename T> struct ScanArgs {
    using W = wide_t<T>;
    const T *g, *x, *grad, *above; // above: the forward result h (gradient only)
    T *h, *dg, *dx;
    const W *h0, *init; // init: the state that enters (forward: h0; gradient: the gradient of the last state)
    W *last;            // the state that leaves (forward: last state; gradient: dh0)
    W *part;            // split sequences: (A, B) per block, then a copy of init (last may be written over init before
                        // the CTA of another block has read it)
    const int64_t *off;
    int64_t g_ld, x_ld, grad_ld, above_ld, h_ld, dg_ld, dx_ld, h0_ld, init_ld, last_ld, part_ld;
    int64_t rows, cols, seqs, strips;
    int blocks; // blocks that a sequence is cut into, with a pass of its own
};

// rows of sequence s; offsets outside [0, rows] or that go back give fewer rows, never others' memory
template <typename T>
__device__ __forceinline__ void sequence(const ScanArgs<T> &a, int64_t s, int64_t *begin, int64_t *end) {
    if (a.off) {
        const int64_t b = a.off[s], e = a.off[s + 1];
        *begin = b < 0 ? 0 : (b > a.rows ? a.rows : b);
        *end = e < *begin ? *begin : (e > a.rows ? a.rows : e);
    } else {
        const int64_t len = a.rows / a.seqs;
        *begin = s * len;
        *end = *begin + len;
    }
}

// f = sigmoid(g) = 1 / (1 + e) and o = 1 - f = e / (1 + e) with e = exp(-g).  In float e is the approximate base-2
// exponential of t = -g / ln 2, times 1 + (-g - t ln 2) for what t has lost by being rounded.  Measured, f and 1 - f are off
// by at most 5.3 half steps (2^-24, relative) at any g; without that factor by 31 at |g| = 40.  Forward and gradient of 8 x
// 4096 x 2048 bf16: 272 us with it, 269 without.  g is held within [-125 ln 2, 128]:
// e * f stays finite, f does not go below 2^-125, and 1 - f is zero from g = 87.4 on.  A NaN passes through.
__device__ __forceinline__ void gate_pair(float g, float *f, float *o) {
    float c, e, r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(g), "f"(-86.6433945f));
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(c), "f"(128.0f));
    const float t = c * -1.44269504f;
    // ln 2 in two parts, as in Cody and Waite's reduction of arguments
    const float lost = fmaf(t, 1.90465421e-9f, fmaf(t, -0.693147182f, -c));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    e = fmaf(e, lost, e);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    *f = r;
    *o = e * r;
}
__device__ __forceinline__ void gate_pair(double g, double *f, double *o) {
    const double e = exp(-fabs(g)), r = 1.0 / (1.0 + e), q = e * r;
    *f = g >= 0.0 ? r : q;
    *o = g >= 0.0 ? q : r;
}

// A product of gates as it is passed on: finite, so that gates above 1 whose product overflows do not turn a state of zero
// into NaN.  (A gate that is itself not finite makes the composed step's b so, too.)
__device__ __forceinline__ float finite(float a) { return fminf(fmaxf(a, -3.40282347e38f), 3.40282347e38f); }
__device__ __forceinline__ double finite(double a) { return fmin(fmax(a, -1.7976931348623157e308), 1.7976931348623157e308); }

// A composed step per channel of a strip, as it lies in shared memory.
template <typename W, int VEC> struct Steps {
    W a[32 * VEC], b[32 * VEC];
};
template <typename W, int VEC> __device__ __forceinline__ void put(Steps<W, VEC> &s, int lane, const W *A, const W *B) {
#pragma unroll
    for (int k = 0; k < VEC; k++) {
        s.a[lane * VEC + k] = finite(A[k]);
        s.b[lane * VEC + k] = B[k];
    }
}

// CTA (sequence, strip of 32 x VEC columns, block of rows).  AGGREGATE: only (A, B) of the block, into part.  Otherwise the
// results; the state that enters a block is init, advanced by part of the blocks in front of it.
// Registers: three CTAs of four warps, or one of eight, on an SM.  With 128 registers a thread, four CTAs fit, but the
// loads of a tile no longer stand together in front of their uses: 30000 x 2560 f16 in 37 sequences took 135 us instead
// of 105, 8 x 4096 x 2048 bf16 (forward and backward, eight warps) 385 instead of 266 (before the sigmoid's correction, with
// which they take 115 to 125 and 272).
template <typename T, int VEC, int WARPS, bool BACK, bool SIGMOID, bool AGGREGATE>
__global__ void __launch_bounds__(WARPS * 32, WARPS == 4 ? 3 : 1) gated_scan_kernel(ScanArgs<T> a) {
    using W = wide_t<T>;
    using V = Vec<T, VEC>;
    constexpr int R = scan_rows<BACK>(), TILE = WARPS * R, STAGES = SCAN_STAGES;
    // operands that are read, and where they stand in a stage
    constexpr bool X = !BACK || (SIGMOID && !AGGREGATE), ABOVE = BACK && !AGGREGATE;
    constexpr int AT_X = 1, AT_D = X ? 2 : 1, AT_ABOVE = AT_D + 1, OPERANDS = 1 + X + BACK + ABOVE;
    __shared__ __align__(16) Steps<W, VEC> agg[2][WARPS];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int64_t strip = blockIdx.x % a.strips, rest = blockIdx.x / a.strips;
    const int64_t blk = rest % a.blocks, seq = rest / a.blocks;
    const int64_t c = (strip * 32 + lane) * VEC;
    const bool in = c < a.cols; // cols is a multiple of VEC
    if (AGGREGATE)
        start_next();
    else
        wait_for_last();
    int64_t begin, end;
    sequence(a, seq, &begin, &end);
    // rows of the block, a multiple of the tile each: n rows from `first` on, in the direction of the recurrence
    const int64_t len = end - begin, per = ((len + a.blocks - 1) / a.blocks + TILE - 1) / TILE * TILE;
    const int64_t skip = blk * per < len ? blk * per : len, n = len - skip < per ? len - skip : per;
    const int64_t first = BACK ? end - 1 - skip : begin + skip;

    W state[VEC], prod[VEC]; // AGGREGATE: (prod, state) is the step composed so far
#pragma unroll
    for (int k = 0; k < VEC; k++) {
        prod[k] = W(1);
        state[k] = !AGGREGATE && in && a.init ? a.init[seq * a.init_ld + c + k] : W(0);
        if (AGGREGATE && in && a.init && blk == 0 && warp == 0) // the copy that the second pass reads
            a.part[(a.seqs * a.blocks * 2 + seq) * a.part_ld + c + k] = a.init[seq * a.init_ld + c + k];
    }
    if (!AGGREGATE && blk > 0) { // the blocks in front: a share for each warp, then the shares in order
        const int64_t share = (blk + WARPS - 1) / WARPS, b0 = warp * share, b1 = b0 + share < blk ? b0 + share : blk;
        const W *p = a.part + (seq * a.blocks + b0) * 2 * a.part_ld + c;
        W A[VEC], B[VEC];
#pragma unroll
        for (int k = 0; k < VEC; k++) {
            A[k] = W(1);
            B[k] = W(0);
        }
        if (in) {
#pragma unroll 16
            for (int64_t b = b0; b < b1; b++, p += 2 * a.part_ld)
#pragma unroll
                for (int k = 0; k < VEC; k++) {
                    B[k] = p[k] * B[k] + p[a.part_ld + k];
                    A[k] = finite(A[k] * p[k]);
                }
        }
        put(agg[1][warp], lane, A, B); // the first tile uses the other half
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WARPS; w++)
#pragma unroll
            for (int k = 0; k < VEC; k++)
                state[k] = agg[1][w].a[lane * VEC + k] * state[k] + agg[1][w].b[lane * VEC + k];
    }
    // Row q of the block lies q leading dimensions behind the first one, or in front of it.
    const int64_t dir = BACK ? -1 : 1, q_first = warp * R;
    const int64_t r_first = first + dir * q_first;
    const T *pg = a.g + r_first * a.g_ld + c;
    const T *px = X ? a.x + r_first * a.x_ld + c : nullptr;
    const T *pd = BACK ? a.grad + r_first * a.grad_ld + c : nullptr;
    const T *pa = ABOVE ? a.above + (r_first - 1) * a.above_ld + c : nullptr;
    // a thread reads nothing from the stages but what it fetched itself: they need no barrier
    extern __shared__ __align__(16) unsigned char stage_mem[];
    T *mine_at = reinterpret_cast<T *>(stage_mem) + (int64_t)warp * STAGES * OPERANDS * R * 32 * VEC + lane * VEC;
    auto at = [&](int stage, int operand, int i) { return mine_at + ((stage * OPERANDS + operand) * R + i) * 32 * VEC; };
    // rows that are there of the R from row q on, for this lane; all: for all lanes, and none is the sequence's first one
    auto rows_from = [&](int64_t q) { return !in || q >= n ? 0 : (n - q < R ? (int)(n - q) : R); };
    auto all_there = [&](int64_t q, int m) {
        return (bool)__all_sync(0xffffffffu, m == R && (!ABOVE || first - q - (R - 1) > begin));
    };
    auto load_row = [&](int stage, int i, bool above) {
        fetch<T, VEC>(at(stage, 0, i), pg + i * dir * a.g_ld);
        if constexpr (X)
            fetch<T, VEC>(at(stage, AT_X, i), px + i * dir * a.x_ld);
        if constexpr (BACK)
            fetch<T, VEC>(at(stage, AT_D, i), pd - i * a.grad_ld);
        if constexpr (ABOVE)
            if (above)
                fetch<T, VEC>(at(stage, AT_ABOVE, i), pa - i * a.above_ld);
    };
    auto load = [&](int stage, int64_t q) {
        const int m = rows_from(q);
        if (all_there(q, m)) {
#pragma unroll
            for (int i = 0; i < R; i++)
                load_row(stage, i, true);
        } else {
#pragma unroll
            for (int i = 0; i < R; i++)
                if (i < m)
                    load_row(stage, i, first - q - i > begin);
        }
        fetch_commit();
        pg += TILE * dir * a.g_ld;
        if constexpr (X)
            px += TILE * dir * a.x_ld;
        if constexpr (BACK)
            pd -= TILE * a.grad_ld;
        if constexpr (ABOVE)
            pa -= TILE * a.above_ld;
    };
    for (int k = 0; k < STAGES - 1; k++)
        load(k, q_first + k * TILE);
    int stage = 0;
    int turn = 0;
    for (int64_t round = 0; round < n; round += TILE, turn ^= 1) {
        const int64_t q = round + q_first;
        const int m = rows_from(q);
        const bool all = all_there(q, m);
        W f[R][VEC], o[R][VEC], b[R][VEC]; // gate, 1 - gate, u or dh
        V kx[R], ka[R];
        fetch_wait<STAGES - 2>();
        auto open = [&](int i) {
            const V rg = ld_vec<T, VEC>(at(stage, 0, i));
            V rx, rd;
            if constexpr (X)
                rx = ld_vec<T, VEC>(at(stage, AT_X, i));
            if constexpr (BACK)
                rd = ld_vec<T, VEC>(at(stage, AT_D, i));
#pragma unroll
            for (int k = 0; k < VEC; k++) {
                f[i][k] = widen(rg.v[k]);
                if constexpr (SIGMOID)
                    gate_pair(f[i][k], &f[i][k], &o[i][k]);
                if constexpr (BACK)
                    b[i][k] = widen(rd.v[k]);
                else
                    b[i][k] = SIGMOID ? o[i][k] * widen(rx.v[k]) : W(widen(rx.v[k]));
            }
            if constexpr (ABOVE) {
                if constexpr (X)
                    kx[i] = rx;
                ka[i] = ld_vec<T, VEC>(at(stage, AT_ABOVE, i));
            }
        };
        if (all) {
#pragma unroll
            for (int i = 0; i < R; i++)
                open(i);
        } else { // rows that are not there leave the state as it is
#pragma unroll
            for (int i = 0; i < R; i++) {
                if (i < m)
                    open(i);
                else
#pragma unroll
                    for (int k = 0; k < VEC; k++) {
                        f[i][k] = W(1);
                        b[i][k] = W(0);
                    }
            }
        }
        // the stage that the round before has emptied
        load(stage == 0 ? STAGES - 1 : stage - 1, q + (STAGES - 1) * TILE);
        stage = stage == STAGES - 1 ? 0 : stage + 1;
        W A[VEC], B[VEC];
#pragma unroll
        for (int k = 0; k < VEC; k++) {
            A[k] = f[0][k];
            // 0 * f: a gate that is not finite leaves its mark in B, where finite() does not reach
            B[k] = BACK ? f[0][k] * b[0][k] : f[0][k] * W(0) + b[0][k];
        }
#pragma unroll
        for (int i = 1; i < R; i++)
#pragma unroll
            for (int k = 0; k < VEC; k++) {
                B[k] = BACK ? f[i][k] * (B[k] + b[i][k]) : f[i][k] * B[k] + b[i][k];
                A[k] *= f[i][k];
            }
        put(agg[turn][warp], lane, A, B);
        __syncthreads(); // the halves of agg alternate: nobody writes this one again before the next barrier
        W v[VEC];
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            if (w == warp) {
#pragma unroll
                for (int k = 0; k < VEC; k++)
                    v[k] = state[k];
            }
#pragma unroll
            for (int k = 0; k < VEC; k++) {
                state[k] = agg[turn][w].a[lane * VEC + k] * state[k] + agg[turn][w].b[lane * VEC + k];
                if constexpr (AGGREGATE)
                    prod[k] = finite(prod[k] * agg[turn][w].a[lane * VEC + k]);
            }
        }
        if constexpr (!AGGREGATE) {
            const int64_t r = first + dir * q;
            auto close = [&](int i, bool top) {
                V y, z;
                if constexpr (!BACK) {
#pragma unroll
                    for (int k = 0; k < VEC; k++) {
                        v[k] = f[i][k] * v[k] + b[i][k];
                        y.v[k] = narrow<T>(v[k]);
                    }
                    st_vec<T, VEC>(a.h + (r + i) * a.h_ld + c, y);
                } else {
                    W above[VEC];
#pragma unroll
                    for (int k = 0; k < VEC; k++)
                        above[k] = !top ? W(widen(ka[i].v[k])) : (a.h0 ? a.h0[seq * a.h0_ld + c + k] : W(0));
#pragma unroll
                    for (int k = 0; k < VEC; k++) {
                        const W delta = b[i][k] + v[k];
                        v[k] = f[i][k] * delta;
                        if constexpr (SIGMOID) {
                            y.v[k] = narrow<T>(v[k] * ((above[k] - widen(kx[i].v[k])) * o[i][k]));
                            z.v[k] = narrow<T>(delta * o[i][k]);
                        } else {
                            y.v[k] = narrow<T>(delta * above[k]);
                            z.v[k] = narrow<T>(delta);
                        }
                    }
                    st_vec<T, VEC>(a.dg + (r - i) * a.dg_ld + c, y);
                    st_vec<T, VEC>(a.dx + (r - i) * a.dx_ld + c, z);
                }
            };
            if (all) {
#pragma unroll
                for (int i = 0; i < R; i++)
                    close(i, false);
            } else {
#pragma unroll
                for (int i = 0; i < R; i++)
                    if (i < m)
                        close(i, BACK && r - i == begin);
            }
        }
    }
    if (warp == 0 && in) {
        W *p = a.part + (seq * a.blocks + blk) * 2 * a.part_ld + c;
#pragma unroll
        for (int k = 0; k < VEC; k++) {
            if (AGGREGATE) {
                p[k] = prod[k];
                p[a.part_ld + k] = state[k];
            } else if (blk == a.blocks - 1 && a.last)
                a.last[seq * a.last_ld + c + k] = state[k];
        }
    }
}

template <typename T, bool SIGMOID>
__global__ void __launch_bounds__(256)
    gated_step_kernel(const T *g, int64_t g_ld, const T *x, int64_t x_ld, int64_t n, int64_t cols, const wide_t<T> *state,
                      int64_t state_ld, wide_t<T> *new_state, int64_t new_ld, T *h, int64_t h_ld) {
    using W = wide_t<T>;
    for (int64_t r = blockIdx.y; r < n; r += gridDim.y)
        for (int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x; c < cols; c += (int64_t)gridDim.x * 256) {
            W f = widen(g[r * g_ld + c]), u = widen(x[r * x_ld + c]), o;
            if (SIGMOID) {
                gate_pair(f, &f, &o);
                u *= o;
            }
            const W v = f * state[r * state_ld + c] + u;
            new_state[r * new_ld + c] = v;
            if (h)
                h[r * h_ld + c] = narrow<T>(v);
        }
}

// How sequences are shared out, from the shape and the number of SMs alone (both directions share the scratch).  `ctas` =
// sequences x strips of columns work independently.  Four warps each when there are more of them than SMs, eight
// otherwise.  Where they leave more than a third of the SMs without work (few columns, few sequences), sequences are cut
// into blocks: a first pass composes the blocks' steps, and the second one reads the inputs again, from L2 when they fit
// there.  (128 CTAs of eight warps reach 70 % of the memory's rate, the two passes 53 %.)
struct ScanPlan {
    int blocks, warps;
    int vec; // columns that a lane takes
};
// `vec`: the most that shapes and addresses allow.  The number of blocks does not depend on it: the scratch is asked for
// without pointers.
template <typename T> ScanPlan scan_plan(int64_t rows, int64_t cols, int64_t seqs, int vec) {
    ScanPlan p{1, 4, vec};
    const int64_t sms = sm_count();
    auto ctas = [&](int64_t v) { return (cols + 32 * v - 1) / (32 * v) * seqs; };
    const int64_t fewest = ctas(widest<T>());
    if (fewest * 3 >= sms * 2 || rows / seqs < 1024) {
        p.warps = ctas(vec) <= sms ? 8 : 4;
        return p;
    }
    // a narrow matrix leaves lanes of its last strip without columns: single elements waste fewer
    if (cols % (32 * vec) != 0)
        p.vec = 1;
    // Below 1024 rows a sequence two passes gain little or nothing.  One sequence, two passes against one: of 512 rows (in
    // blocks of 128) 19.7 and 16.6 us at 1024 columns bf16; of 1024 rows 19.5 and 27, 31 and 29 at 8192 columns; of 2048
    // rows 20 and 52, 44 and 52.  As many blocks as make three CTAs for an SM, what fits there: 16384 x 4096 bf16 takes
    // 166 us with two, 136 with three, 134 with six; 4096 x 4096 takes 52, 41 and 52.
    const int64_t want = sms * 3 / fewest, most = rows / seqs / 256;
    p.blocks = (int)(want < most ? want : most);
    return p;
}

template <typename T, int VEC, int WARPS, bool BACK, bool SIGMOID> int scan_launch(ScanArgs<T> a, cudaStream_t st) {
    a.strips = (a.cols + 32 * VEC - 1) / (32 * VEC);
    const int64_t ctas = a.strips * a.blocks * a.seqs;
    DB2_CHECK(ctas < ((int64_t)1 << 31), DB2_EUNSUPPORTED, "gatedScan: too many sequences and columns for one launch");
    constexpr size_t stage = (size_t)SCAN_STAGES * WARPS * scan_rows<BACK>() * 32 * VEC * sizeof(T);
    constexpr int operands = BACK ? (SIGMOID ? 4 : 3) : 2;
    auto whole = gated_scan_kernel<T, VEC, WARPS, BACK, SIGMOID, false>;
    auto aggregate = gated_scan_kernel<T, VEC, 4, BACK, SIGMOID, true>;
    static PerDeviceOnce once;
    if (once.need()) {
        DB2_CUDA(cudaFuncSetAttribute(whole, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(stage * operands)));
        DB2_CUDA(cudaFuncSetAttribute(aggregate, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(stage * 2)));
        once.mark();
    }
    if constexpr (WARPS == 4)
        if (a.blocks > 1) {
            aggregate<<<(unsigned)ctas, 128, stage * 2, st>>>(a);
            DB2_TRY(after_launch("gated_scan_kernel"));
            if (a.init) {
                a.init = a.part + a.seqs * a.blocks * 2 * a.part_ld;
                a.init_ld = a.part_ld;
            }
            return launch_next("gated_scan_kernel", whole, dim3((unsigned)ctas), WARPS * 32, stage * operands, st, a);
        }
    whole<<<(unsigned)ctas, WARPS * 32, stage * operands, st>>>(a);
    return after_launch("gated_scan_kernel");
}

template <typename T, bool BACK> int scan_any(ScanArgs<T> &a, int gate, int vec, cudaStream_t st) {
    constexpr int N = widest<T>();
    const ScanPlan p = scan_plan<T>(a.rows, a.cols, a.seqs, vec);
    a.blocks = p.blocks;
    const bool s = gate == DB2_GATE_SIGMOID;
#define DB2_SCAN(VEC, WARPS)                                                                                           \
    return s ? scan_launch<T, VEC, WARPS, BACK, true>(a, st) : scan_launch<T, VEC, WARPS, BACK, false>(a, st)
    if (p.vec == N) {
        if (p.warps == 8)
            DB2_SCAN(N, 8);
        DB2_SCAN(N, 4);
    }
    if (N > 2 && p.vec == 2) {
        if (p.warps == 8)
            DB2_SCAN(2, 8);
        DB2_SCAN(2, 4);
    }
    if (p.warps == 8)
        DB2_SCAN(1, 8);
    DB2_SCAN(1, 4);
#undef DB2_SCAN
}

bool seq_type(int dtype) {
    return dtype == DB2_F64 || dtype == DB2_F32 || dtype == DB2_F16 || dtype == DB2_BF16;
}
int64_t scan_part_ld(int64_t cols) { return (cols + 7) / 8 * 8; }

// what both directions check; *done: nothing to do
int check_scan(const char *what, int dtype, int gate, int64_t rows, int64_t cols, const void *off, int64_t seqs) {
    DB2_CHECK(seq_type(dtype), DB2_EUNSUPPORTED, "%s: unsupported value type code %d", what, dtype);
    DB2_CHECK(gate == DB2_GATE_DECAY || gate == DB2_GATE_SIGMOID, DB2_EINVAL, "%s: unknown gate %d", what, gate);
    DB2_CHECK(rows >= 0 && cols >= 0 && seqs >= 0, DB2_EINVAL, "%s: negative shape", what);
    DB2_CHECK(off || seqs == 0 || rows % seqs == 0, DB2_EINVAL,
              "%s: without offsets the %lld rows must be %lld equally long sequences", what, (long long)rows,
              (long long)seqs);
    return DB2_OK;
}

void count(db2_context *ctx, uint64_t before) {
    std::lock_guard<std::mutex> lock(ctx->mu);
    ctx->stats.launches += g_launches.load(std::memory_order_relaxed) - before;
}

int wide_dtype(int dtype) { return dtype == DB2_F64 ? DB2_F64 : DB2_F32; }

int check_rows(const char *what, const db2_matrix *g, const db2_matrix *m, const char *name) {
    DB2_CHECK(m->dtype == g->dtype && m->rows == g->rows && m->cols == g->cols, DB2_EINVAL,
              "%s: %s must have the shape and value type of the gates", what, name);
    return DB2_OK;
}
int check_state(const char *what, const db2_matrix *g, const db2_matrix *m, int64_t seqs, const char *name) {
    DB2_CHECK(!m || (m->dtype == wide_dtype(g->dtype) && m->rows == seqs && m->cols == g->cols), DB2_EINVAL,
              "%s: %s must have one row per sequence (%lld), %lld columns and the wide value type", what, name,
              (long long)seqs, (long long)g->cols);
    return DB2_OK;
}
// number of sequences: one, or what the offsets say; offsets that do not ascend within the rows are an error, which takes
// a look at them on the host
int sequences(db2_context *ctx, const char *what, const db2_matrix *g, db2_matrix *offsets, int64_t *seqs) {
    *seqs = 1;
    if (!offsets)
        return DB2_OK;
    DB2_CHECK(offsets->dtype == DB2_I64 && offsets->cols == 1 && offsets->rows >= 1, DB2_EINVAL,
              "%s: offsets must be a column matrix of int64 with one row more than there are sequences", what);
    *seqs = offsets->rows - 1;
    std::vector<int64_t> host((size_t)offsets->rows);
    DB2_TRY(db2_matrix_to_host(offsets, host.data(), 1));
    for (size_t i = 0; i < host.size(); i++)
        DB2_CHECK(host[i] >= (i ? host[i - 1] : 0) && host[i] <= g->rows, DB2_EDOMAIN,
                  "%s: offsets must ascend within [0, %lld], got %lld at position %lld", what, (long long)g->rows,
                  (long long)host[i], (long long)i);
    return DB2_OK;
}
// results that cover all rows: rows of no sequence keep what is there, so a fresh matrix starts as zeros
int prepare_rows(db2_context *ctx, db2_matrix **res, const db2_matrix *g, bool all_rows) {
    if (*res)
        return prepare_update(*res);
    return db2_matrix_create(ctx, g->dtype, g->rows, g->cols, all_rows ? 0 : 1, res);
}
} // namespace
} // namespace db2

using namespace db2;

extern "C" {

size_t db2k_gated_scan_scratch_bytes(int dtype, int64_t rows, int64_t cols, int64_t seqs) {
    if (rows <= 0 || cols <= 0 || seqs <= 0)
        return 0;
    const int es = (int)dtype_size(dtype);
    const int blocks = (es == 8   ? scan_plan<double>(rows, cols, seqs, 1)
                        : es == 4 ? scan_plan<float>(rows, cols, seqs, 1)
                                  : scan_plan<__half>(rows, cols, seqs, 1))
                           .blocks;
    return blocks < 2 ? 0 : (size_t)seqs * (blocks * 2 + 1) * scan_part_ld(cols) * (dtype == DB2_F64 ? 8 : 4);
}

int db2k_gated_scan(int dtype, int gate, const void *g, int64_t g_ld, const void *x, int64_t x_ld, int64_t rows,
                    int64_t cols, const int64_t *row_off, int64_t seqs, const void *h0, int64_t h0_ld, void *h,
                    int64_t h_ld, void *last, int64_t last_ld, void *scratch, size_t scratch_bytes, void *stream) {
    DB2_TRY(check_scan("gatedScan", dtype, gate, rows, cols, row_off, seqs));
    if (cols == 0 || seqs == 0)
        return DB2_OK;
    DB2_CHECK((g && x && h) || rows == 0, DB2_EINVAL, "gatedScan: null operand");
    DB2_CHECK(ld_ok(g_ld, rows, cols) && ld_ok(x_ld, rows, cols) && ld_ok(h_ld, rows, cols) &&
                  (!h0 || ld_ok(h0_ld, seqs, cols)) && (!last || ld_ok(last_ld, seqs, cols)),
              DB2_EINVAL, "gatedScan: a leading dimension is smaller than the number of columns");
    const size_t need = db2k_gated_scan_scratch_bytes(dtype, rows, cols, seqs);
    DB2_CHECK(need == 0 || (scratch && scratch_bytes >= need && aligned16(scratch)), DB2_EINVAL,
              "gatedScan: scratch smaller than db2k_gated_scan_scratch_bytes, or not 16-byte aligned");
    DB2_DISPATCH_SEQ(dtype, T, {
        using W = wide_t<T>;
        ScanArgs<T> a{};
        a.g = static_cast<const T *>(g);
        a.x = static_cast<const T *>(x);
        a.h = static_cast<T *>(h);
        a.init = static_cast<const W *>(h0);
        a.last = static_cast<W *>(last);
        a.part = static_cast<W *>(scratch);
        a.off = row_off;
        a.g_ld = g_ld;
        a.x_ld = x_ld;
        a.h_ld = h_ld;
        a.init_ld = h0_ld;
        a.last_ld = last_ld;
        a.part_ld = scan_part_ld(cols);
        a.rows = rows;
        a.cols = cols;
        a.seqs = seqs;
        auto packed = [&](int n) {
            const size_t b = n * sizeof(T);
            return cols % n == 0 && rows_aligned(g, g_ld, sizeof(T), b) && rows_aligned(x, x_ld, sizeof(T), b) &&
                   rows_aligned(h, h_ld, sizeof(T), b);
        };
        const int vec = packed(widest<T>()) ? widest<T>() : (widest<T>() > 2 && packed(2) ? 2 : 1);
        return scan_any<T, false>(a, gate, vec, as_stream(stream));
    });
    return DB2_OK;
}

int db2k_gated_scan_grad(int dtype, int gate, const void *g, int64_t g_ld, const void *x, int64_t x_ld, const void *h,
                         int64_t h_ld, const void *grad, int64_t grad_ld, int64_t rows, int64_t cols,
                         const int64_t *row_off, int64_t seqs, const void *h0, int64_t h0_ld, const void *grad_last,
                         int64_t grad_last_ld, void *dg, int64_t dg_ld, void *dx, int64_t dx_ld, void *dh0,
                         int64_t dh0_ld, void *scratch, size_t scratch_bytes, void *stream) {
    DB2_TRY(check_scan("gatedScanGrad", dtype, gate, rows, cols, row_off, seqs));
    if (cols == 0 || seqs == 0)
        return DB2_OK;
    const bool sigmoid = gate == DB2_GATE_SIGMOID;
    DB2_CHECK((g && (x || !sigmoid) && h && grad && dg && dx) || rows == 0, DB2_EINVAL, "gatedScanGrad: null operand");
    DB2_CHECK(ld_ok(g_ld, rows, cols) && (!sigmoid || ld_ok(x_ld, rows, cols)) && ld_ok(h_ld, rows, cols) &&
                  ld_ok(grad_ld, rows, cols) && ld_ok(dg_ld, rows, cols) && ld_ok(dx_ld, rows, cols) &&
                  (!h0 || ld_ok(h0_ld, seqs, cols)) && (!grad_last || ld_ok(grad_last_ld, seqs, cols)) &&
                  (!dh0 || ld_ok(dh0_ld, seqs, cols)),
              DB2_EINVAL, "gatedScanGrad: a leading dimension is smaller than the number of columns");
    const size_t need = db2k_gated_scan_scratch_bytes(dtype, rows, cols, seqs);
    DB2_CHECK(need == 0 || (scratch && scratch_bytes >= need && aligned16(scratch)), DB2_EINVAL,
              "gatedScanGrad: scratch smaller than db2k_gated_scan_scratch_bytes, or not 16-byte aligned");
    DB2_DISPATCH_SEQ(dtype, T, {
        using W = wide_t<T>;
        ScanArgs<T> a{};
        a.g = static_cast<const T *>(g);
        a.x = static_cast<const T *>(x);
        a.above = static_cast<const T *>(h);
        a.grad = static_cast<const T *>(grad);
        a.dg = static_cast<T *>(dg);
        a.dx = static_cast<T *>(dx);
        a.h0 = static_cast<const W *>(h0);
        a.init = static_cast<const W *>(grad_last);
        a.last = static_cast<W *>(dh0);
        a.part = static_cast<W *>(scratch);
        a.off = row_off;
        a.g_ld = g_ld;
        a.x_ld = x_ld;
        a.above_ld = h_ld;
        a.grad_ld = grad_ld;
        a.dg_ld = dg_ld;
        a.dx_ld = dx_ld;
        a.h0_ld = h0_ld;
        a.init_ld = grad_last_ld;
        a.last_ld = dh0_ld;
        a.part_ld = scan_part_ld(cols);
        a.rows = rows;
        a.cols = cols;
        a.seqs = seqs;
        auto packed = [&](int n) {
            const size_t b = n * sizeof(T);
            return cols % n == 0 && rows_aligned(g, g_ld, sizeof(T), b) && (!sigmoid || rows_aligned(x, x_ld, sizeof(T), b)) &&
                   rows_aligned(h, h_ld, sizeof(T), b) && rows_aligned(grad, grad_ld, sizeof(T), b) &&
                   rows_aligned(dg, dg_ld, sizeof(T), b) && rows_aligned(dx, dx_ld, sizeof(T), b);
        };
        const int vec = packed(widest<T>()) ? widest<T>() : (widest<T>() > 2 && packed(2) ? 2 : 1);
        return scan_any<T, true>(a, gate, vec, as_stream(stream));
    });
    return DB2_OK;
}

int db2k_gated_step(int dtype, int gate, const void *g, int64_t g_ld, const void *x, int64_t x_ld, int64_t n, int64_t cols,
                    const void *state, int64_t state_ld, void *new_state, int64_t new_state_ld, void *h, int64_t h_ld,
                    void *stream) {
    DB2_TRY(check_scan("gatedStep", dtype, gate, n, cols, nullptr, 1));
    if (n == 0 || cols == 0)
        return DB2_OK;
    DB2_CHECK(g && x && state && new_state, DB2_EINVAL, "gatedStep: null operand");
    DB2_CHECK(ld_ok(g_ld, n, cols) && ld_ok(x_ld, n, cols) && ld_ok(state_ld, n, cols) && ld_ok(new_state_ld, n, cols) &&
                  (!h || ld_ok(h_ld, n, cols)),
              DB2_EINVAL, "gatedStep: a leading dimension is smaller than the number of columns");
    const int64_t gx = (cols + 255) / 256;
    const dim3 grid((unsigned)(gx < 65535 ? gx : 65535), (unsigned)(n < 65535 ? n : 65535));
    DB2_DISPATCH_SEQ(dtype, T, {
        using W = wide_t<T>;
        auto kernel = gate == DB2_GATE_SIGMOID ? gated_step_kernel<T, true> : gated_step_kernel<T, false>;
        kernel<<<grid, 256, 0, as_stream(stream)>>>(static_cast<const T *>(g), g_ld, static_cast<const T *>(x), x_ld, n,
                                                    cols, static_cast<const W *>(state), state_ld,
                                                    static_cast<W *>(new_state), new_state_ld, static_cast<T *>(h), h_ld);
        return after_launch("gated_step_kernel");
    });
    return DB2_OK;
}

int db2_gatedScan(db2_context *ctx, int gate, db2_matrix **h, db2_matrix **last, db2_matrix *g, db2_matrix *x,
                  db2_matrix *offsets, db2_matrix *h0) {
    DB2_API_BEGIN
    DB2_CHECK(ctx && h && g && x, DB2_EINVAL, "null argument");
    DB2_TRY(check_scan("gatedScan", g->dtype, gate, g->rows, g->cols, nullptr, 1));
    DB2_TRY(check_rows("gatedScan", g, x, "x"));
    bind_device(ctx);
    int64_t seqs = 1;
    DB2_TRY(sequences(ctx, "gatedScan", g, offsets, &seqs));
    DB2_TRY(check_state("gatedScan", g, h0, seqs, "h0"));
    Results results;
    DB2_TRY(results.add("gatedScan", h, g->dtype, g->rows, g->cols));
    DB2_TRY(results.add("gatedScan", last, wide_dtype(g->dtype), seqs, g->cols));
    const uint64_t before = g_launches.load();
    const DeviceOperand dg(g), dx(x), doff(offsets), dh0(h0);
    DB2_CHECK(!offsets || doff.ld == 1 || seqs == 0, DB2_EUNSUPPORTED, "gatedScan: offsets are a strided view");
    DB2_TRY(results.apart("gatedScan", g, {h}));
    DB2_TRY(results.apart("gatedScan", x, {h}));
    DB2_TRY(results.apart("gatedScan", h0, {last}));
    DB2_TRY(prepare_rows(ctx, h, g, !offsets));
    if (last)
        DB2_TRY(prepare_result(ctx, last, wide_dtype(g->dtype), seqs, g->cols));
    void *scratch = nullptr;
    const size_t sb = db2k_gated_scan_scratch_bytes(g->dtype, g->rows, g->cols, seqs);
    DB2_TRY(ctx_scratch(ctx, sb, &scratch));
    DB2_TRY(db2k_gated_scan(g->dtype, gate, dg.ptr, dg.ld, dx.ptr, dx.ld, g->rows, g->cols,
                            static_cast<const int64_t *>(doff.ptr), seqs, dh0.ptr, dh0.ld, (*h)->dev_ptr(),
                            (*h)->dev_ld, last ? (*last)->dev_ptr() : nullptr, last ? (*last)->dev_ld : 0, scratch,
                            ctx->scratch_bytes, ctx->stream));
    count(ctx, before);
    return results.done();
    DB2_API_END
}

int db2_gatedScanGrad(db2_context *ctx, int gate, db2_matrix **dg, db2_matrix **dx, db2_matrix **dh0, db2_matrix *g,
                      db2_matrix *x, db2_matrix *h, db2_matrix *grad, db2_matrix *offsets, db2_matrix *h0,
                      db2_matrix *grad_last) {
    DB2_API_BEGIN
    DB2_CHECK(ctx && dg && dx && g && h && grad && (x || gate == DB2_GATE_DECAY), DB2_EINVAL, "null argument");
    DB2_TRY(check_scan("gatedScanGrad", g->dtype, gate, g->rows, g->cols, nullptr, 1));
    if (x)
        DB2_TRY(check_rows("gatedScanGrad", g, x, "x"));
    DB2_TRY(check_rows("gatedScanGrad", g, h, "h"));
    DB2_TRY(check_rows("gatedScanGrad", g, grad, "grad"));
    bind_device(ctx);
    int64_t seqs = 1;
    DB2_TRY(sequences(ctx, "gatedScanGrad", g, offsets, &seqs));
    DB2_TRY(check_state("gatedScanGrad", g, h0, seqs, "h0"));
    DB2_TRY(check_state("gatedScanGrad", g, grad_last, seqs, "grad_last"));
    Results results;
    DB2_TRY(results.add("gatedScanGrad", dg, g->dtype, g->rows, g->cols));
    DB2_TRY(results.add("gatedScanGrad", dx, g->dtype, g->rows, g->cols));
    DB2_TRY(results.add("gatedScanGrad", dh0, wide_dtype(g->dtype), seqs, g->cols));
    const uint64_t before = g_launches.load();
    const DeviceOperand og(g), ox(x), oh(h), od(grad), ooff(offsets), oh0(h0), ol(grad_last);
    DB2_CHECK(!offsets || ooff.ld == 1 || seqs == 0, DB2_EUNSUPPORTED, "gatedScanGrad: offsets are a strided view");
    for (const db2_matrix *m : {g, gate == DB2_GATE_SIGMOID ? x : nullptr, h, grad, h0, grad_last})
        DB2_TRY(results.apart("gatedScanGrad", m));
    DB2_TRY(prepare_rows(ctx, dg, g, !offsets));
    DB2_TRY(prepare_rows(ctx, dx, g, !offsets));
    if (dh0)
        DB2_TRY(prepare_result(ctx, dh0, wide_dtype(g->dtype), seqs, g->cols));
    void *scratch = nullptr;
    const size_t sb = db2k_gated_scan_scratch_bytes(g->dtype, g->rows, g->cols, seqs);
    DB2_TRY(ctx_scratch(ctx, sb, &scratch));
    DB2_TRY(db2k_gated_scan_grad(g->dtype, gate, og.ptr, og.ld, ox.ptr, ox.ld, oh.ptr, oh.ld, od.ptr, od.ld, g->rows,
                                 g->cols, static_cast<const int64_t *>(ooff.ptr), seqs, oh0.ptr, oh0.ld, ol.ptr, ol.ld,
                                 (*dg)->dev_ptr(), (*dg)->dev_ld, (*dx)->dev_ptr(), (*dx)->dev_ld,
                                 dh0 ? (*dh0)->dev_ptr() : nullptr, dh0 ? (*dh0)->dev_ld : 0, scratch,
                                 ctx->scratch_bytes, ctx->stream));
    count(ctx, before);
    return results.done();
    DB2_API_END
}

int db2_gatedStep(db2_context *ctx, int gate, db2_matrix **h, db2_matrix **new_state, db2_matrix *g, db2_matrix *x,
                  db2_matrix *state) {
    DB2_API_BEGIN
    DB2_CHECK(ctx && h && new_state && g && x && state, DB2_EINVAL, "null argument");
    DB2_TRY(check_scan("gatedStep", g->dtype, gate, g->rows, g->cols, nullptr, 1));
    DB2_TRY(check_rows("gatedStep", g, x, "x"));
    DB2_TRY(check_state("gatedStep", g, state, g->rows, "state"));
    Results results;
    DB2_TRY(results.add("gatedStep", h, g->dtype, g->rows, g->cols));
    DB2_TRY(results.add("gatedStep", new_state, wide_dtype(g->dtype), g->rows, g->cols));
    bind_device(ctx);
    const uint64_t before = g_launches.load();
    // a new state in the place of the old one is written where it is: each element is read before it is written
    const bool in_place = *new_state == state;
    const DeviceOperand dg(g), dx(x);
    DB2_TRY(ensure_device(state));
    for (const db2_matrix *m : {g, x, state}) // an element of each is read before the results' are written
        DB2_TRY(results.apart("gatedStep", m, {h, new_state}));
    if (in_place)
        DB2_TRY(prepare_update(state, true));
    const DeviceOperand ds(state); // before any result is prepared, which may name it
    DB2_TRY(prepare_result(ctx, h, g->dtype, g->rows, g->cols));
    if (!in_place)
        DB2_TRY(prepare_result(ctx, new_state, wide_dtype(g->dtype), g->rows, g->cols));
    DB2_TRY(db2k_gated_step(g->dtype, gate, dg.ptr, dg.ld, dx.ptr, dx.ld, g->rows, g->cols, ds.ptr, ds.ld,
                            (*new_state)->dev_ptr(), (*new_state)->dev_ld, (*h)->dev_ptr(), (*h)->dev_ld, ctx->stream));
    count(ctx, before);
    return results.done();
    DB2_API_END
}

} // extern "C"
