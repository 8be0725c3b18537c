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
// rows says all about it.  A warp holds SCAN_R consecutive rows of 32 lanes x VEC columns in registers and forms their
// (A, B); the warps of a CTA exchange theirs through shared memory; every warp then walks its rows once more, from the
// value that really enters them.  So each operand is read once and each result written once.
//
// Bound by memory.  States, gates and products are float (double for double); the stored h is rounded once, the running
// state never.
#include "runtime.h"
#include "seq.cuh"

namespace db2 {

namespace {

constexpr int SCAN_WARPS = 8, SCAN_R = 8, SCAN_TILE = SCAN_WARPS * SCAN_R;

template <typename T> struct ScanArgs {
    using W = wide_t<T>;
    const T *g, *x, *grad, *above; // above: the forward result h (gradient only)
    T *h, *dg, *dx;
    const W *h0, *init; // init: the state that enters (forward: h0; gradient: the gradient of the last state)
    W *last;            // the state that leaves (forward: last state; gradient: dh0)
    W *part;            // split sequences: (A, B) per block, later the state that enters the block
    const int64_t *off;
    int64_t g_ld, x_ld, grad_ld, above_ld, h_ld, dg_ld, dx_ld, h0_ld, init_ld, last_ld, part_ld;
    int64_t rows, cols, seqs, strips;
    int blocks; // blocks that a sequence is cut into
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

// f = sigmoid(g) and 1 - f, each accurate relative to itself: e = exp(-|g|) lies in [0, 1], and the two are 1 / (1 + e) and
// e / (1 + e).  In float the fast exponential and division cost a few units in the last place of f.
__device__ __forceinline__ void gate_pair(float g, float *f, float *o) {
    const float e = __expf(-fabsf(g)), r = __fdividef(1.0f, 1.0f + e), q = e * r;
    *f = g >= 0.0f ? r : q;
    *o = g >= 0.0f ? q : r;
    if (g != g)
        *f = *o = g;
}
__device__ __forceinline__ void gate_pair(double g, double *f, double *o) {
    const double e = exp(-fabs(g)), r = 1.0 / (1.0 + e), q = e * r;
    *f = g >= 0.0 ? r : q;
    *o = g >= 0.0 ? q : r;
    if (g != g)
        *f = *o = g;
}

// a * v + b for a state v and a composed step: a state of zero stays out of it, so that a product of large gates that
// overflowed does not turn it into NaN
template <typename W> __device__ __forceinline__ W step_state(W a, W v, W b) {
    return v == W(0) ? b : a * v + b;
}

// CTA (sequence, strip of columns, block of rows).  AGGREGATE: only (A, B) of the block, into part.  Otherwise the
// results; the state that enters is init, or part when sequences are cut into several blocks.
template <typename T, int VEC, bool BACK, bool SIGMOID, bool AGGREGATE>
__global__ void __launch_bounds__(SCAN_WARPS * 32) gated_scan_kernel(ScanArgs<T> a) {
    using W = wide_t<T>;
    using V = Vec<T, VEC>;
    __shared__ W agg[2][SCAN_WARPS][2][32 * VEC];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int64_t strip = blockIdx.x % a.strips, rest = blockIdx.x / a.strips;
    const int64_t blk = rest % a.blocks, seq = rest / a.blocks;
    const int64_t c = (strip * 32 + lane) * VEC;
    const bool in = c < a.cols; // cols is a multiple of VEC
    int64_t begin, end;
    sequence(a, seq, &begin, &end);
    // rows of the block, a multiple of the tile each: n rows from `first` on, in the direction of the recurrence
    const int64_t len = end - begin, per = ((len + a.blocks - 1) / a.blocks + SCAN_TILE - 1) / SCAN_TILE * SCAN_TILE;
    const int64_t skip = blk * per < len ? blk * per : len, n = len - skip < per ? len - skip : per;
    const int64_t first = BACK ? end - 1 - skip : begin + skip;
    W *my_part = a.part + (seq * a.blocks + blk) * 2 * a.part_ld;

    W state[VEC], prod[VEC]; // AGGREGATE: (prod, state) is the step composed so far
#pragma unroll
    for (int k = 0; k < VEC; k++) {
        prod[k] = W(1);
        state[k] = W(0);
        if (!AGGREGATE && in) {
            if (a.blocks > 1)
                state[k] = my_part[c + k];
            else if (a.init)
                state[k] = a.init[seq * a.init_ld + c + k];
        }
    }
    V rg[SCAN_R], rb[SCAN_R], rx[SCAN_R], ra[SCAN_R]; // g; x or grad; (gradient) x; (gradient) h of the row above
    auto row_at = [&](int64_t q) { return BACK ? first - q : first + q; };
    auto load = [&](int64_t q0) {
#pragma unroll
        for (int i = 0; i < SCAN_R; i++)
            if (in && q0 + i < n) {
                const int64_t r = row_at(q0 + i);
                rg[i] = ld_vec<T, VEC>(a.g + r * a.g_ld + c);
                rb[i] = BACK ? ld_vec<T, VEC>(a.grad + r * a.grad_ld + c) : ld_vec<T, VEC>(a.x + r * a.x_ld + c);
                if constexpr (BACK && !AGGREGATE) {
                    if constexpr (SIGMOID)
                        rx[i] = ld_vec<T, VEC>(a.x + r * a.x_ld + c);
                    if (r > begin)
                        ra[i] = ld_vec<T, VEC>(a.above + (r - 1) * a.above_ld + c);
                }
            }
    };
    load(warp * SCAN_R);
    int turn = 0;
    for (int64_t tile = 0; tile < n; tile += SCAN_TILE, turn ^= 1) {
        const int64_t q0 = tile + warp * SCAN_R;
        W f[SCAN_R][VEC], o[SCAN_R][VEC], b[SCAN_R][VEC]; // gate, 1 - gate, u or dh
        W A[VEC], B[VEC];
#pragma unroll
        for (int k = 0; k < VEC; k++) {
            A[k] = W(1);
            B[k] = W(0);
        }
#pragma unroll
        for (int i = 0; i < SCAN_R; i++)
#pragma unroll
            for (int k = 0; k < VEC; k++) {
                f[i][k] = W(1);
                o[i][k] = b[i][k] = W(0);
                if (in && q0 + i < n) {
                    const W g = widen(rg[i].v[k]);
                    if (SIGMOID)
                        gate_pair(g, &f[i][k], &o[i][k]);
                    else
                        f[i][k] = g;
                    b[i][k] = widen(rb[i].v[k]);
                    if (SIGMOID && !BACK)
                        b[i][k] *= o[i][k];
                }
                B[k] = BACK ? f[i][k] * (B[k] + b[i][k]) : f[i][k] * B[k] + b[i][k];
                A[k] *= f[i][k];
            }
        V px[SCAN_R], pa[SCAN_R];
        if constexpr (BACK && !AGGREGATE) {
#pragma unroll
            for (int i = 0; i < SCAN_R; i++) {
                px[i] = rx[i];
                pa[i] = ra[i];
            }
        }
        load(q0 + SCAN_TILE); // on its way while the warps exchange their steps
#pragma unroll
        for (int k = 0; k < VEC; k++) {
            agg[turn][warp][0][lane * VEC + k] = A[k];
            agg[turn][warp][1][lane * VEC + k] = B[k];
        }
        __syncthreads(); // the halves of agg alternate: nobody writes this one again before the next barrier
        W v[VEC];
#pragma unroll
        for (int w = 0; w < SCAN_WARPS; w++)
#pragma unroll
            for (int k = 0; k < VEC; k++) {
                const W wa = agg[turn][w][0][lane * VEC + k], wb = agg[turn][w][1][lane * VEC + k];
                if (w == warp)
                    v[k] = state[k];
                state[k] = step_state(wa, state[k], wb);
                if (AGGREGATE)
                    prod[k] *= wa;
            }
        if constexpr (!AGGREGATE) {
#pragma unroll
            for (int i = 0; i < SCAN_R; i++) {
                const bool live = in && q0 + i < n;
                const int64_t r = row_at(q0 + i);
                V y, z;
#pragma unroll
                for (int k = 0; k < VEC; k++) {
                    if constexpr (!BACK) {
                        v[k] = f[i][k] * v[k] + b[i][k];
                        y.v[k] = narrow<T>(v[k]);
                    } else {
                        const W delta = b[i][k] + v[k];
                        W above = W(0);
                        if (live && r > begin)
                            above = widen(pa[i].v[k]);
                        else if (live && a.h0)
                            above = a.h0[seq * a.h0_ld + c + k];
                        if constexpr (SIGMOID) {
                            y.v[k] = narrow<T>(delta * (above - (live ? W(widen(px[i].v[k])) : W(0))) * f[i][k] * o[i][k]);
                            z.v[k] = narrow<T>(delta * o[i][k]);
                        } else {
                            y.v[k] = narrow<T>(delta * above);
                            z.v[k] = narrow<T>(delta);
                        }
                        v[k] = f[i][k] * delta;
                    }
                }
                if (live) {
                    if constexpr (!BACK)
                        st_vec<T, VEC>(a.h + r * a.h_ld + c, y);
                    else {
                        st_vec<T, VEC>(a.dg + r * a.dg_ld + c, y);
                        st_vec<T, VEC>(a.dx + r * a.dx_ld + c, z);
                    }
                }
            }
        }
    }
    if (warp == 0 && in) {
#pragma unroll
        for (int k = 0; k < VEC; k++) {
            if (AGGREGATE) {
                my_part[c + k] = prod[k];
                my_part[a.part_ld + c + k] = state[k];
            } else if (a.blocks == 1 && a.last)
                a.last[seq * a.last_ld + c + k] = state[k];
        }
    }
}

// (A, B) of the blocks of every sequence -> the state that enters each block; the state that leaves the last one
template <typename T> __global__ void __launch_bounds__(128) gated_carry_kernel(ScanArgs<T> a) {
    using W = wide_t<T>;
    const int64_t i = (int64_t)blockIdx.x * 128 + threadIdx.x;
    if (i >= a.seqs * a.cols)
        return;
    const int64_t seq = i / a.cols, c = i % a.cols;
    W v = a.init ? a.init[seq * a.init_ld + c] : W(0);
    W *p = a.part + seq * a.blocks * 2 * a.part_ld + c;
#pragma unroll 8
    for (int b = 0; b < a.blocks; b++, p += 2 * a.part_ld) {
        const W A = p[0], B = p[a.part_ld];
        p[0] = v;
        v = step_state(A, v, B);
    }
    if (a.last)
        a.last[seq * a.last_ld + c] = v;
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

// Blocks that a sequence is cut into: one (a single pass over the data) when the sequences and strips alone keep the SMs
// busy or when a block would be shorter than four tiles.  Depends on the shape and the number of SMs alone.
template <typename T> constexpr int widest() { return sizeof(T) == 2 ? 2 : 1; }
int scan_blocks(size_t es, int64_t rows, int64_t cols, int64_t seqs) {
    if (rows <= 0 || cols <= 0 || seqs <= 0)
        return 1;
    const int64_t strips = (cols + 31) / 32 / (es == 2 ? 2 : 1) + 1, ctas = strips * seqs;
    const int64_t want = ((int64_t)sm_count() * 4 + ctas - 1) / ctas, most = rows / seqs / (4 * SCAN_TILE);
    const int64_t b = want < most ? want : most;
    return b < 2 ? 1 : (int)(b > 1024 ? 1024 : b);
}

template <typename T, int VEC, bool BACK, bool SIGMOID> int scan_launch(ScanArgs<T> a, cudaStream_t st) {
    a.strips = (a.cols + 32 * VEC - 1) / (32 * VEC);
    const int64_t ctas = a.strips * a.blocks * a.seqs;
    DB2_CHECK(ctas < ((int64_t)1 << 31), DB2_EUNSUPPORTED, "gatedScan: too many sequences and columns for one launch");
    if (a.blocks > 1) {
        gated_scan_kernel<T, VEC, BACK, SIGMOID, true><<<(unsigned)ctas, SCAN_WARPS * 32, 0, st>>>(a);
        DB2_TRY(after_launch("gated_scan_kernel"));
        gated_carry_kernel<T><<<(unsigned)((a.seqs * a.cols + 127) / 128), 128, 0, st>>>(a);
        DB2_TRY(after_launch("gated_carry_kernel"));
    }
    gated_scan_kernel<T, VEC, BACK, SIGMOID, false><<<(unsigned)ctas, SCAN_WARPS * 32, 0, st>>>(a);
    return after_launch("gated_scan_kernel");
}

template <typename T, bool BACK> int scan_any(const ScanArgs<T> &a, int gate, bool packed, cudaStream_t st) {
    constexpr int N = widest<T>();
    if (packed)
        return gate == DB2_GATE_SIGMOID ? scan_launch<T, N, BACK, true>(a, st) : scan_launch<T, N, BACK, false>(a, st);
    return gate == DB2_GATE_SIGMOID ? scan_launch<T, 1, BACK, true>(a, st) : scan_launch<T, 1, BACK, false>(a, st);
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
    if (*res) {
        DB2_CHECK((*res)->dtype == g->dtype && (*res)->rows == g->rows && (*res)->cols == g->cols, DB2_EINVAL,
                  "pre-allocated result has shape (%lld x %lld) / type %d, expected (%lld x %lld) / type %d",
                  (long long)(*res)->rows, (long long)(*res)->cols, (*res)->dtype, (long long)g->rows,
                  (long long)g->cols, g->dtype);
        return prepare_update(*res);
    }
    return db2_matrix_create(ctx, g->dtype, g->rows, g->cols, all_rows ? 0 : 1, res);
}
} // namespace
} // namespace db2

using namespace db2;

extern "C" {

size_t db2k_gated_scan_scratch_bytes(int dtype, int64_t rows, int64_t cols, int64_t seqs) {
    if (rows <= 0 || cols <= 0 || seqs <= 0)
        return 0;
    const int blocks = scan_blocks(dtype_size(dtype), rows, cols, seqs);
    return blocks < 2 ? 0 : (size_t)seqs * blocks * 2 * scan_part_ld(cols) * (dtype == DB2_F64 ? 8 : 4);
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
        a.blocks = scan_blocks(sizeof(T), rows, cols, seqs);
        constexpr size_t al = sizeof(T) * widest<T>();
        const bool packed = cols % widest<T>() == 0 && rows_aligned(g, g_ld, sizeof(T), al) &&
                            rows_aligned(x, x_ld, sizeof(T), al) && rows_aligned(h, h_ld, sizeof(T), al);
        return scan_any<T, false>(a, gate, packed, as_stream(stream));
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
        a.blocks = scan_blocks(sizeof(T), rows, cols, seqs);
        constexpr size_t al = sizeof(T) * widest<T>();
        const bool packed = cols % widest<T>() == 0 && rows_aligned(g, g_ld, sizeof(T), al) &&
                            (!sigmoid || rows_aligned(x, x_ld, sizeof(T), al)) && rows_aligned(h, h_ld, sizeof(T), al) &&
                            rows_aligned(grad, grad_ld, sizeof(T), al) && rows_aligned(dg, dg_ld, sizeof(T), al) &&
                            rows_aligned(dx, dx_ld, sizeof(T), al);
        return scan_any<T, true>(a, gate, packed, as_stream(stream));
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
    DB2_CHECK(!last || !*last || *last != *h, DB2_EINVAL, "gatedScan: two results are to go to one matrix");
    const uint64_t before = g_launches.load();
    const DeviceOperand dg(g), dx(x), doff(offsets), dh0(h0);
    DB2_CHECK(!offsets || doff.ld == 1 || seqs == 0, DB2_EUNSUPPORTED, "gatedScan: offsets are a strided view");
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
    return DB2_OK;
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
    db2_matrix *slots[3] = {*dg, *dx, dh0 ? *dh0 : nullptr};
    for (int i = 0; i < 3; i++)
        for (int j = 0; j < i; j++)
            DB2_CHECK(!slots[i] || slots[i] != slots[j], DB2_EINVAL, "gatedScanGrad: two results are to go to one matrix");
    const uint64_t before = g_launches.load();
    const DeviceOperand og(g), ox(x), oh(h), od(grad), ooff(offsets), oh0(h0), ol(grad_last);
    DB2_CHECK(!offsets || ooff.ld == 1 || seqs == 0, DB2_EUNSUPPORTED, "gatedScanGrad: offsets are a strided view");
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
    return DB2_OK;
    DB2_API_END
}

int db2_gatedStep(db2_context *ctx, int gate, db2_matrix **h, db2_matrix **new_state, db2_matrix *g, db2_matrix *x,
                  db2_matrix *state) {
    DB2_API_BEGIN
    DB2_CHECK(ctx && h && new_state && g && x && state, DB2_EINVAL, "null argument");
    DB2_TRY(check_scan("gatedStep", g->dtype, gate, g->rows, g->cols, nullptr, 1));
    DB2_TRY(check_rows("gatedStep", g, x, "x"));
    DB2_TRY(check_state("gatedStep", g, state, g->rows, "state"));
    DB2_CHECK(!*h || *h != *new_state, DB2_EINVAL, "gatedStep: two results are to go to one matrix");
    bind_device(ctx);
    const uint64_t before = g_launches.load();
    // a new state in the place of the old one is written where it is: each element is read before it is written
    const bool in_place = *new_state == state;
    const DeviceOperand dg(g), dx(x);
    DB2_TRY(prepare_result(ctx, h, g->dtype, g->rows, g->cols));
    if (in_place)
        DB2_TRY(prepare_update(state));
    const DeviceOperand ds(state);
    if (!in_place)
        DB2_TRY(prepare_result(ctx, new_state, wide_dtype(g->dtype), g->rows, g->cols));
    DB2_TRY(db2k_gated_step(g->dtype, gate, dg.ptr, dg.ld, dx.ptr, dx.ld, g->rows, g->cols, ds.ptr, ds.ld,
                            (*new_state)->dev_ptr(), (*new_state)->dev_ld, (*h)->dev_ptr(), (*h)->dev_ld, ctx->stream));
    count(ctx, before);
    return DB2_OK;
    DB2_API_END
}

} // extern "C"
