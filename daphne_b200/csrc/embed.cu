// Embedding: rows of a table picked by token and scaled, and the gradient of the table.
//
//   res[i]  = scale * table[token[i]]                               (token -1: a row of zeros)
//   dtable[v] = scale * sum over i with token[i] == v of grad[i]    (in the order of i)
//
// It is the product of the one-hot matrix of the tokens with the table, P @ E and t(P) @ dY, without P.
//
// The gradient sorts the tokens (stably, by key and position), so that equal tokens lie side by side and every sum has
// one fixed order of additions: no floating-point atomics, the same bits in every run.
#include "runtime.h"
#include "seq.cuh"

namespace db2 {

namespace {

constexpr int EMB_THREADS = 256;
constexpr int EMB_UNROLL = 4; // packets of a row in flight per thread

// tokens are int64 or int32
template <typename I> __device__ __forceinline__ int64_t token_at(const void *tokens, int64_t ld, int64_t i) {
    return (int64_t) static_cast<const I *>(tokens)[i * ld];
}

// Rows are copied by `1 << log_tpr` threads each; a CTA holds EMB_THREADS >> log_tpr rows, blockIdx.y cuts long rows.
// Bound by memory: one read and one write per element.
template <typename T, int N, typename I>
__global__ void __launch_bounds__(EMB_THREADS)
    embed_kernel(const T *__restrict__ table, int64_t vocab, int64_t cols, int64_t table_ld, const void *tokens,
                 int64_t tokens_ld, int64_t n, wide_t<T> scale, T *__restrict__ res, int64_t res_ld, int log_tpr,
                 int32_t *status) {
    const int tpr = 1 << log_tpr, tx = threadIdx.x & (tpr - 1), ty = threadIdx.x >> log_tpr;
    const int rows_per_cta = EMB_THREADS >> log_tpr;
    const int64_t packets = cols / N;
    for (int64_t r = (int64_t)blockIdx.x * rows_per_cta + ty; r < n; r += (int64_t)gridDim.x * rows_per_cta) {
        const int64_t t = token_at<I>(tokens, tokens_ld, r);
        const bool ok = t >= 0 && t < vocab;
        if (!ok && t != -1 && status && tx == 0 && blockIdx.y == 0)
            *status = 1;
        const T *src = table + (ok ? t : 0) * table_ld;
        T *dst = res + r * res_ld;
        for (int64_t p0 = (int64_t)blockIdx.y * tpr * EMB_UNROLL + tx; p0 < packets;
             p0 += (int64_t)gridDim.y * tpr * EMB_UNROLL) {
            Vec<T, N> x[EMB_UNROLL];
#pragma unroll
            for (int u = 0; u < EMB_UNROLL; u++)
                if (ok && p0 + u * tpr < packets)
                    x[u] = ld_vec<T, N>(src + (p0 + u * tpr) * N);
#pragma unroll
            for (int u = 0; u < EMB_UNROLL; u++)
                if (p0 + u * tpr < packets) {
                    Vec<T, N> y;
#pragma unroll
                    for (int k = 0; k < N; k++)
                        y.v[k] = narrow<T>(ok ? widen(x[u].v[k]) * scale : wide_t<T>(0));
                    st_vec<T, N>(dst + (p0 + u * tpr) * N, y);
                }
        }
        if (N > 1 && blockIdx.y == 0)
            for (int64_t c = packets * N + tx; c < cols; c += tpr)
                dst[c] = narrow<T>(ok ? widen(src[c]) * scale : wide_t<T>(0));
    }
}

int log2_ceil(int64_t x) {
    int b = 0;
    while (((int64_t)1 << b) < x)
        b++;
    return b;
}

template <typename T, int N, typename I>
int embed_launch(const void *table, int64_t vocab, int64_t cols, int64_t table_ld, const void *tokens,
                 int64_t tokens_ld, int64_t n, double scale, void *res, int64_t res_ld, int32_t *status,
                 cudaStream_t st) {
    // a thread takes up to EMB_UNROLL packets of a row in one go
    const int64_t packets = cols / N;
    int log_tpr = log2_ceil((packets + EMB_UNROLL - 1) / EMB_UNROLL);
    if (log_tpr > 8)
        log_tpr = 8;
    const int64_t row_groups = (n + (EMB_THREADS >> log_tpr) - 1) / (EMB_THREADS >> log_tpr);
    const int64_t span = ((int64_t)1 << log_tpr) * EMB_UNROLL;
    int64_t gy = (packets + span - 1) / span;
    const int64_t cap = (int64_t)sm_count() * 16;
    gy = gy < 1 ? 1 : (gy > 64 ? 64 : gy);
    const int64_t gx = row_groups < cap ? row_groups : cap;
    embed_kernel<T, N, I><<<dim3((unsigned)gx, (unsigned)gy), EMB_THREADS, 0, st>>>(
        static_cast<const T *>(table), vocab, cols, table_ld, tokens, tokens_ld, n, (wide_t<T>)scale,
        static_cast<T *>(res), res_ld, log_tpr, status);
    return after_launch("embed_kernel");
}

// ---- sorting the tokens ----
//
// Every sort delivers key[] (ascending) and pos[] (ascending among equal keys).  A token that names no row gets the key
// `vocab`, behind all others.

constexpr int SORT_CHUNK = 512;            // tokens that a CTA sorts by itself
// Tokens that are merged in one go: their sorted chunks lie in shared memory.  Every CTA reads all keys and searches every
// chunk, so merging grows with the square of the tokens, the radix passes hardly: 16384 tokens of 128256 take 33 us merged
// (whole gradient, 8 columns) and 63 by radix, 28672 take 58 and 65, 40960 take 71 and 69, 49152 take 82 and 67 to 70.
constexpr int MERGE_MAX = 80 * SORT_CHUNK;
constexpr int MERGE_THREADS = 512, MERGE_ROUND = MERGE_THREADS / 8; // of a CTA; tokens that eight lanes each share
// chunks lie one word apart from multiples of the 32 banks: lanes at the same step of their searches do not collide
constexpr int MERGE_PITCH = SORT_CHUNK + 1;

// The table's rows, which become zero before the sums are written: further CTAs of the kernel that sorts chunks, which keeps
// few SMs busy, do it, or a kernel in front of the radix passes.  A CTA writes 128 packets of a row at a time.
struct Zeros {
    char *at;
    int64_t rows, row_bytes, ld_bytes;
    int packet;     // 16, or the size of an element
    int64_t tail;   // bytes behind the last row, a multiple of the element's size
    int element;
};
template <int BYTES> struct alignas(BYTES) Blank {
    unsigned char b[BYTES];
};
template <int BYTES> __device__ __forceinline__ void write_zeros(const Zeros &z, int cta, int ctas) {
    const int groups = blockDim.x / 128, tx = threadIdx.x % 128;
    const int64_t packets = z.row_bytes / BYTES;
    const Blank<BYTES> zero{};
    for (int64_t r = (int64_t)cta * groups + threadIdx.x / 128; r < z.rows; r += (int64_t)ctas * groups) {
        char *row = z.at + r * z.ld_bytes;
#pragma unroll 4
        for (int64_t p = tx; p < packets; p += 128)
            *reinterpret_cast<Blank<BYTES> *>(row + p * BYTES) = zero;
    }
}
__device__ __forceinline__ void write_zeros_any(const Zeros &z, int cta, int ctas) {
    if (cta == 0 && z.tail > 0) {
        char *p = z.at + z.rows * z.ld_bytes;
        for (int64_t i = (int64_t)threadIdx.x * z.element; i < z.tail; i += (int64_t)blockDim.x * z.element)
            if (z.element == 2)
                *reinterpret_cast<uint16_t *>(p + i) = 0;
            else if (z.element == 4)
                *reinterpret_cast<uint32_t *>(p + i) = 0;
            else
                *reinterpret_cast<uint64_t *>(p + i) = 0;
    }
    switch (z.packet) {
    case 16: write_zeros<16>(z, cta, ctas); break;
    case 8: write_zeros<8>(z, cta, ctas); break;
    case 4: write_zeros<4>(z, cta, ctas); break;
    default: write_zeros<2>(z, cta, ctas); break;
    }
}
__global__ void __launch_bounds__(SORT_CHUNK) table_zero_kernel(Zeros z) { write_zeros_any(z, blockIdx.x, gridDim.x); }

template <typename I>
__device__ __forceinline__ uint32_t token_key(const void *tokens, int64_t ld, int64_t i, int64_t vocab,
                                              int32_t *status) {
    const int64_t t = token_at<I>(tokens, ld, i);
    if (t >= 0 && t < vocab)
        return (uint32_t)t;
    if (t != -1 && status)
        *status = 1;
    return (uint32_t)vocab;
}

// Tokens of a call that has nothing to compute (no table rows, no columns): they are looked at for their status only.
template <typename I>
__global__ void __launch_bounds__(EMB_THREADS)
    token_check_kernel(const void *tokens, int64_t tokens_ld, int64_t n, int64_t vocab, int32_t *status) {
    for (int64_t i = (int64_t)blockIdx.x * EMB_THREADS + threadIdx.x; i < n; i += (int64_t)gridDim.x * EMB_THREADS)
        token_key<I>(tokens, tokens_ld, i, vocab, status);
}
int check_tokens(const char *what, int index_dtype, const void *tokens, int64_t tokens_ld, int64_t n, int64_t vocab,
                 int32_t *status, cudaStream_t st) {
    if (n == 0 || !status)
        return DB2_OK;
    DB2_CHECK(tokens && ld_ok(tokens_ld, n, 1), DB2_EINVAL, "%s: null tokens or their stride too small", what);
    const int64_t want = (n + EMB_THREADS - 1) / EMB_THREADS, cap = (int64_t)sm_count() * 8;
    const unsigned grid = (unsigned)(want < cap ? want : cap);
    if (index_dtype == DB2_I64)
        token_check_kernel<int64_t><<<grid, EMB_THREADS, 0, st>>>(tokens, tokens_ld, n, vocab, status);
    else
        token_check_kernel<int32_t><<<grid, EMB_THREADS, 0, st>>>(tokens, tokens_ld, n, vocab, status);
    return after_launch("token_check_kernel");
}

// Chunks of SORT_CHUNK tokens, each sorted by (key, position): a token's place is how many keys of its chunk are smaller, or
// the same and in front of it.  A thread per token compares it with all of them, four at a time; what comes before and
// behind the warp's own 32 tokens needs one comparison each.  (A bitonic network over chunks of 1024 takes 9 us.)
template <typename I>
__global__ void __launch_bounds__(SORT_CHUNK)
    token_chunk_kernel(const void *tokens, int64_t tokens_ld, int n, int64_t vocab, uint32_t *__restrict__ key,
                       uint32_t *__restrict__ pos, int32_t *status, int chunks, Zeros z) {
    if ((int)blockIdx.x >= chunks) {
        write_zeros_any(z, blockIdx.x - chunks, gridDim.x - chunks);
        return;
    }
    start_next(); // (the CTAs above say so by their end: their stores come first)
    __shared__ uint4 quads[SORT_CHUNK / 4];
    const int base = blockIdx.x * SORT_CHUNK, t = threadIdx.x;
    // places behind the last token hold a key behind all others
    const uint32_t k = base + t < n ? token_key<I>(tokens, tokens_ld, base + t, vocab, status) : 0xffffffffu;
    reinterpret_cast<uint32_t *>(quads)[t] = k;
    __syncthreads();
    const int own = t / 32 * 8;
    int place = 0;
#pragma unroll 4
    for (int q = 0; q < own; q++) {
        const uint4 x = quads[q];
        place += (x.x <= k) + (x.y <= k) + (x.z <= k) + (x.w <= k);
    }
#pragma unroll
    for (int q = own; q < own + 8; q++) {
        const uint4 x = quads[q];
        place += (x.x < k || (x.x == k && q * 4 < t)) + (x.y < k || (x.y == k && q * 4 + 1 < t)) +
                 (x.z < k || (x.z == k && q * 4 + 2 < t)) + (x.w < k || (x.w == k && q * 4 + 3 < t));
    }
#pragma unroll 4
    for (int q = own + 8; q < SORT_CHUNK / 4; q++) {
        const uint4 x = quads[q];
        place += (x.x < k) + (x.y < k) + (x.z < k) + (x.w < k);
    }
    if (base + t < n) {
        key[base + place] = k;
        pos[base + place] = (uint32_t)(base + t);
    }
}

// Sorted chunks -> sorted tokens: the place of a token is its place within its chunk plus, for every other chunk, how many of
// its keys are smaller (or the same, in chunks in front).  8 to 32 lanes share a token, each takes every so many chunks; the
// keys of all chunks lie in shared memory, ten steps of a binary search each.
__global__ void __launch_bounds__(MERGE_THREADS)
    token_merge_kernel(const uint32_t *__restrict__ key, const uint32_t *__restrict__ pos, int n,
                       uint32_t *__restrict__ key_out, uint32_t *__restrict__ pos_out, int per_cta) {
    extern __shared__ uint32_t k[];
    wait_for_last();
    start_next();
#pragma unroll 8
    for (int i = threadIdx.x; i < n; i += MERGE_THREADS)
        k[i / SORT_CHUNK * MERGE_PITCH + i % SORT_CHUNK] = key[i];
    __syncthreads();
    const int lane = threadIdx.x % 32, chunks = (n + SORT_CHUNK - 1) / SORT_CHUNK;
    const int group = chunks <= 8 ? 8 : (chunks <= 16 ? 16 : 32); // lanes that share a token
    const int first = blockIdx.x * per_cta, part = lane % group;
    for (int i = first + threadIdx.x / group; i < first + per_cta; i += MERGE_THREADS / group) {
        const int at = i < n ? i : n - 1, own = at / SORT_CHUNK; // all lanes stay for the sum
        const uint32_t mine = k[own * MERGE_PITCH + at % SORT_CHUNK], its_pos = pos[at];
        int place = 0;
        for (int c = part; c < chunks; c += group) {
            if (c == own) {
                place += at - own * SORT_CHUNK;
                continue;
            }
            const uint32_t *chunk = k + c * MERGE_PITCH;
            const int len = n - c * SORT_CHUNK < SORT_CHUNK ? n - c * SORT_CHUNK : SORT_CHUNK;
            const uint32_t below = mine + (c < own); // keys are smaller than 2^32 - 1
            int lo = 0;
#pragma unroll
            for (int step = SORT_CHUNK / 2; step >= 1; step /= 2)
                if (lo + step <= len && chunk[lo + step - 1] < below)
                    lo += step;
            place += lo + (lo < len && chunk[lo] < below); // the steps add up to SORT_CHUNK - 1
        }
        for (int o = group / 2; o >= 1; o >>= 1)
            place += __shfl_xor_sync(0xffffffffu, place, o);
        if (part == 0 && i < n) {
            key_out[place] = mine;
            pos_out[place] = its_pos;
        }
    }
}

// Radix sort, lowest digit first, up to 9 bits a pass: tiles of RADIX_TILE tokens are counted by digit, the counts of all
// tiles are scanned (digit by digit, tile by tile), and every tile moves its tokens to their places in order.
constexpr int RADIX_THREADS = 256, RADIX_WARPS = RADIX_THREADS / 32;
constexpr int RADIX_PER_WARP = 512;
constexpr int RADIX_TILE = RADIX_WARPS * RADIX_PER_WARP;
constexpr int RADIX_BITS = 9, RADIX_BINS = 1 << RADIX_BITS;

struct RadixIn { // the tokens themselves in the first pass (key == nullptr), keys and positions later
    const void *tokens;
    int64_t tokens_ld, vocab;
    const uint32_t *key, *pos;
};
template <typename I>
__device__ __forceinline__ void radix_load(const RadixIn &in, int64_t i, uint32_t *key, uint32_t *pos,
                                           int32_t *status) {
    if (in.key) {
        *key = in.key[i];
        *pos = in.pos[i];
    } else {
        *key = token_key<I>(in.tokens, in.tokens_ld, i, in.vocab, status);
        *pos = (uint32_t)i;
    }
}

template <typename I>
__global__ void __launch_bounds__(RADIX_THREADS)
    radix_count_kernel(RadixIn in, int64_t n, int shift, int bins, uint32_t *__restrict__ counts, int32_t *status) {
    __shared__ uint32_t h[RADIX_BINS];
    for (int b = threadIdx.x; b < bins; b += RADIX_THREADS)
        h[b] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * RADIX_TILE;
    for (int i = threadIdx.x; i < RADIX_TILE && base + i < n; i += RADIX_THREADS) {
        uint32_t key, pos;
        radix_load<I>(in, base + i, &key, &pos, status);
        atomicAdd(&h[(key >> shift) & (bins - 1)], 1u); // integer counts: the order of additions does not show
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += RADIX_THREADS)
        counts[(int64_t)b * gridDim.x + blockIdx.x] = h[b];
}

// exclusive prefix over all counts, in place, by one CTA
__global__ void __launch_bounds__(1024) radix_scan_kernel(uint32_t *__restrict__ counts, int64_t m) {
    __shared__ uint32_t warp_sum[32];
    const int t = threadIdx.x, lane = t % 32, warp = t / 32;
    uint32_t carry = 0;
    for (int64_t b = 0; b < m; b += 4096) {
        uint32_t v[4], sum = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int64_t i = b + t * 4 + k;
            v[k] = i < m ? counts[i] : 0u;
            sum += v[k];
        }
        uint32_t inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o)
                inc += y;
        }
        if (lane == 31)
            warp_sum[warp] = inc;
        __syncthreads();
        uint32_t before = 0, all = 0;
        for (int w = 0; w < 32; w++) {
            before += w < warp ? warp_sum[w] : 0u;
            all += warp_sum[w];
        }
        uint32_t run = carry + before + inc - sum;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int64_t i = b + t * 4 + k;
            if (i < m)
                counts[i] = run;
            run += v[k];
        }
        carry += all;
        __syncthreads();
    }
}

// A warp owns RADIX_PER_WARP consecutive tokens of the tile and walks them 32 at a time; next[w][d] is the place of warp
// w's next token with digit d.  Lanes with the same digit take consecutive places in lane order.
template <typename I>
__global__ void __launch_bounds__(RADIX_THREADS)
    radix_move_kernel(RadixIn in, int64_t n, int shift, int bins, const uint32_t *__restrict__ offsets,
                      uint32_t *__restrict__ key_out, uint32_t *__restrict__ pos_out) {
    __shared__ uint32_t next[RADIX_WARPS][RADIX_BINS];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    for (int b = threadIdx.x; b < RADIX_WARPS * RADIX_BINS; b += RADIX_THREADS)
        (&next[0][0])[b] = 0;
    __syncthreads();
    const int64_t base = (int64_t)blockIdx.x * RADIX_TILE + warp * RADIX_PER_WARP;
    for (int i = lane; i < RADIX_PER_WARP && base + i < n; i += 32) {
        uint32_t key, pos;
        radix_load<I>(in, base + i, &key, &pos, nullptr);
        atomicAdd(&next[warp][(key >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += RADIX_THREADS) {
        uint32_t run = offsets[(int64_t)b * gridDim.x + blockIdx.x];
        for (int w = 0; w < RADIX_WARPS; w++) {
            const uint32_t c = next[w][b];
            next[w][b] = run;
            run += c;
        }
    }
    __syncthreads();
    for (int i = 0; i < RADIX_PER_WARP; i += 32) { // the same trips for all lanes
        const bool in_range = base + i + lane < n;
        uint32_t key = 0, pos = 0;
        if (in_range)
            radix_load<I>(in, base + i + lane, &key, &pos, nullptr);
        const uint32_t d = in_range ? (key >> shift) & (bins - 1) : (uint32_t)RADIX_BINS;
        const unsigned peers = __match_any_sync(0xffffffffu, d);
        const int before = __popc(peers & ((1u << lane) - 1u));
        uint32_t place = 0;
        if (in_range)
            place = next[warp][d] + before;
        __syncwarp();
        if (in_range && before == 0)
            next[warp][d] += __popc(peers);
        __syncwarp();
        if (in_range) {
            key_out[place] = key;
            pos_out[place] = pos;
        }
    }
}

// ---- sums over equal tokens ----

constexpr int SUM_THREADS = 128;
constexpr int SUM_RUN = 32;   // sorted tokens that one group of threads adds up
constexpr int SUM_AHEAD = 8;  // gradient rows in flight per thread

constexpr int SUM_MIN_LOG = 2; // at least four threads share a run

struct SumArgs {
    const uint32_t *key, *pos;
    int64_t n, cols, vocab, grad_ld, res_ld, part_ld;
    int64_t runs;     // ceil(n / SUM_RUN)
    int log_tpr;
};

// A run of SUM_RUN sorted tokens x a block of columns: rows of equal tokens are added in registers (32 bits or more);
// where the token changes, the sum is finished -- written to the table when all its rows lie in the run, to `part`
// otherwise: part[run][0] holds the sum of a token that came over from the run before, part[run][1] that of a token that
// starts in the run and goes on behind it.  Equal amounts of work whatever the tokens' frequencies.
// Bound by memory: every gradient row is read once, every row of a token that occurs written once here (and once before,
// when the table was cleared).
template <typename T, typename R, int N, bool ADD>
__global__ void __launch_bounds__(SUM_THREADS)
    embed_sum_kernel(SumArgs a, const T *__restrict__ grad, wide_t<T> scale, R *__restrict__ res,
                     wide_t<T> *__restrict__ part) {
    using W = wide_t<T>;
    // the tokens of the CTA's runs, and the one in front and behind: key k of a run stands at keys[1 + k]
    __shared__ uint32_t keys[(SUM_THREADS >> SUM_MIN_LOG) * SUM_RUN + 2], rows[(SUM_THREADS >> SUM_MIN_LOG) * SUM_RUN];
    const int tpr = 1 << a.log_tpr, tx = threadIdx.x & (tpr - 1), ty = threadIdx.x >> a.log_tpr;
    const int here = (SUM_THREADS >> a.log_tpr) * SUM_RUN;
    wait_for_last();
    start_next();
    const int64_t cta_first = (int64_t)blockIdx.x * here;
    for (int i = threadIdx.x; i < here + 2; i += SUM_THREADS) {
        const int64_t at = cta_first + i - 1;
        keys[i] = at >= 0 && at < a.n ? a.key[at] : 0xffffffffu;
        if (i < here && at + 1 < a.n)
            rows[i] = a.pos[at + 1];
    }
    __syncthreads();
    const int64_t run = (int64_t)blockIdx.x * (SUM_THREADS >> a.log_tpr) + ty;
    if (run >= a.runs)
        return;
    const int64_t b = run * SUM_RUN;
    const int len = a.n - b < SUM_RUN ? (int)(a.n - b) : SUM_RUN;
    const uint32_t *key = keys + 1 + ty * SUM_RUN, *row = rows + ty * SUM_RUN;
    const uint32_t vocab = (uint32_t)a.vocab, before = key[-1], behind = key[len];
    const int64_t packets = a.cols / N; // cols is a multiple of N
    for (int64_t p = (int64_t)blockIdx.y * tpr + tx; p < packets; p += (int64_t)gridDim.y * tpr) {
        const int64_t c = p * N;
        W acc[N];
#pragma unroll
        for (int k = 0; k < N; k++)
            acc[k] = W(0);
        uint32_t cur = key[0];
        int slot = cur == before ? 0 : -1; // -1: the sum starts in this run
        auto finish = [&](uint32_t next) {
            if (cur >= vocab)
                return;
            if (slot < 0 && next != cur) {
                R *dst = res + (int64_t)cur * a.res_ld + c;
                W y[N];
#pragma unroll
                for (int k = 0; k < N; k++)
                    y[k] = acc[k] * scale;
                if constexpr (ADD) {
                    const Vec<R, N> old = ld_vec<R, N>(dst);
#pragma unroll
                    for (int k = 0; k < N; k++)
                        y[k] += W(widen(old.v[k]));
                }
                st_vec<R, N>(dst, narrow_all<R, N>(y));
            } else {
                W *dst = part + (run * 2 + (slot < 0 ? 1 : 0)) * a.part_ld + c;
#pragma unroll
                for (int k = 0; k < N; k++)
                    dst[k] = acc[k];
            }
        };
        for (int i = 0; i < len; i += SUM_AHEAD) {
            Vec<T, N> x[SUM_AHEAD];
#pragma unroll
            for (int u = 0; u < SUM_AHEAD; u++) { // places without a row load row 0: loads under conditions go one by one
                const int64_t r = i + u < len && key[i + u] < vocab ? row[i + u] : 0;
                x[u] = ld_vec<T, N>(grad + r * a.grad_ld + c);
            }
#pragma unroll
            for (int u = 0; u < SUM_AHEAD; u++) {
                if (i + u >= len)
                    break;
                if (key[i + u] != cur) {
                    finish(key[i + u]);
                    cur = key[i + u];
                    slot = -1;
#pragma unroll
                    for (int k = 0; k < N; k++)
                        acc[k] = W(0);
                }
                if (cur < vocab) {
#pragma unroll
                    for (int k = 0; k < N; k++)
                        acc[k] += widen(x[u].v[k]);
                }
            }
        }
        finish(behind);
    }
}

// Tokens whose rows span several runs: the run in which such a token starts adds the partial sums behind it, in order.
// A CTA looks at `per` runs and 32 x JOIN_N columns; for each run that has something to join, its warps take equal shares
// of the parts, whose sums are added in the order of the shares.  Most runs have nothing to join: where they are many, a
// CTA looks at up to JOIN_RUNS of them, so that fewer CTAs are started for nothing (16 per SM).
constexpr int JOIN_Y = 8, JOIN_N = 4, JOIN_RUNS = 8;
template <typename T, typename R, bool ADD>
__global__ void __launch_bounds__(32 * JOIN_Y)
    embed_join_kernel(SumArgs a, wide_t<T> scale, R *__restrict__ res, const wide_t<T> *__restrict__ part, int per) {
    using W = wide_t<T>;
    __shared__ W sums[JOIN_Y][32 * JOIN_N];
    const int tx = threadIdx.x % 32, ty = threadIdx.x / 32;
    wait_for_last();
    __shared__ uint32_t token[JOIN_RUNS]; // the token to join, or the number of table rows
    if (threadIdx.x < per) {
        const int64_t run = (int64_t)blockIdx.x * per + threadIdx.x, b = run * SUM_RUN, e = b + SUM_RUN;
        uint32_t v = (uint32_t)a.vocab;
        if (run + 1 < a.runs) { // not the last run: e < n
            const uint32_t last = a.key[e - 1], next = a.key[e], start = a.key[b], before = b > 0 ? a.key[b - 1] : 0xffffffffu;
            if (last < v && next == last && !(start == last && before == last))
                v = last; // it goes on behind this run and starts in it
        }
        token[threadIdx.x] = v;
    }
    __syncthreads();
    for (int i = 0; i < per; i++) {
        const int64_t run = (int64_t)blockIdx.x * per + i;
        const uint32_t v = token[i];
        if (v == (uint32_t)a.vocab)
            continue; // uniform over the CTA
        // runs behind this one that hold a part: those that begin with this token
        int64_t more = 0;
        for (;;) {
            const int64_t j = run + 1 + more + tx;
            const unsigned part_of = __ballot_sync(0xffffffffu, j < a.runs && a.key[j * SUM_RUN] == v);
            more += part_of == 0xffffffffu ? 32 : __ffs(~part_of) - 1;
            if (part_of != 0xffffffffu)
                break;
        }
        const int64_t share = (more + JOIN_Y) / JOIN_Y;
        const int64_t first = ty * share, last = first + share < more + 1 ? first + share : more + 1;
        for (int64_t c0 = (int64_t)blockIdx.y * 32 * JOIN_N; c0 < a.cols; c0 += (int64_t)gridDim.y * 32 * JOIN_N) {
            W acc[JOIN_N];
#pragma unroll
            for (int k = 0; k < JOIN_N; k++)
                acc[k] = W(0);
            if (c0 + tx * JOIN_N < a.cols) { // part_ld is a multiple of JOIN_N
#pragma unroll 8
                for (int64_t j = first; j < last; j++) {
                    const W *p = part + ((run + j) * 2 + (j == 0 ? 1 : 0)) * a.part_ld + c0 + tx * JOIN_N;
#pragma unroll
                    for (int k = 0; k < JOIN_N; k += 16 / sizeof(W)) {
                        const Vec<W, 16 / sizeof(W)> x = ld_vec<W, 16 / sizeof(W)>(p + k);
#pragma unroll
                        for (int i = 0; i < (int)(16 / sizeof(W)); i++)
                            acc[k + i] += x.v[i];
                    }
                }
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < JOIN_N; k++)
                sums[ty][tx * JOIN_N + k] = acc[k];
            __syncthreads();
            for (int j = threadIdx.x; j < 32 * JOIN_N && c0 + j < a.cols; j += 32 * JOIN_Y) {
                W s = sums[0][j];
                for (int k = 1; k < JOIN_Y; k++)
                    s += sums[k][j];
                R *dst = res + (int64_t)v * a.res_ld + c0 + j;
                *dst = narrow<R>(ADD ? W(widen(*dst)) + s * scale : s * scale);
            }
        }
    }
}

struct GradPlan {
    int64_t runs, part_ld, tiles;
    int bits, passes;
    size_t key_off[2], pos_off[2], counts_off, part_off, bytes;
};
size_t take(size_t *at, size_t bytes) {
    const size_t here = *at;
    *at += (bytes + 255) / 256 * 256;
    return here;
}
GradPlan grad_plan(size_t wide_size, int64_t vocab, int64_t cols, int64_t n) {
    GradPlan p{};
    p.runs = (n + SUM_RUN - 1) / SUM_RUN;
    p.part_ld = (cols + 7) / 8 * 8;
    p.bits = log2_ceil(vocab + 1);
    p.passes = n <= MERGE_MAX ? 0 : (p.bits + RADIX_BITS - 1) / RADIX_BITS;
    p.tiles = (n + RADIX_TILE - 1) / RADIX_TILE;
    size_t at = 0;
    for (int i = 0; i < (p.passes == 1 || n <= SORT_CHUNK ? 1 : 2); i++) {
        p.key_off[i] = take(&at, (size_t)n * 4);
        p.pos_off[i] = take(&at, (size_t)n * 4);
    }
    if (p.passes)
        p.counts_off = take(&at, (size_t)p.tiles * RADIX_BINS * 4);
    p.part_off = take(&at, (size_t)p.runs * 2 * p.part_ld * wide_size);
    p.bytes = at;
    return p;
}

template <typename I>
int embed_sort(const GradPlan &p, const void *tokens, int64_t tokens_ld, int64_t n, int64_t vocab, char *scratch,
               const uint32_t **key, const uint32_t **pos, int32_t *status, Zeros z, cudaStream_t st) {
    uint32_t *k[2], *q[2];
    for (int i = 0; i < 2; i++) {
        k[i] = reinterpret_cast<uint32_t *>(scratch + p.key_off[i]);
        q[i] = reinterpret_cast<uint32_t *>(scratch + p.pos_off[i]);
    }
    // CTAs that write zeros: as many as the rows need, at most what fits on the device
    const int64_t want = (z.rows + (z.tail > 0) + 3) / 4, cap = (int64_t)sm_count() * 4;
    const unsigned zero_ctas = (unsigned)(want < cap ? want : cap);
    if (p.passes == 0) {
        // two launches, or one, where counting with 9-bit digits takes six
        const int chunks = (int)((n + SORT_CHUNK - 1) / SORT_CHUNK);
        token_chunk_kernel<I><<<chunks + zero_ctas, SORT_CHUNK, 0, st>>>(tokens, tokens_ld, (int)n, vocab, k[0], q[0],
                                                                         status, chunks, z);
        DB2_TRY(after_launch("token_chunk_kernel"));
        *key = k[0];
        *pos = q[0];
        if (chunks == 1)
            return DB2_OK;
        static PerDeviceOnce once;
        if (once.need()) {
            DB2_CUDA(cudaFuncSetAttribute(token_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          MERGE_MAX / SORT_CHUNK * MERGE_PITCH * 4));
            once.mark();
        }
        // every CTA reads all keys: no more CTAs than SMs, of whole rounds of MERGE_ROUND tokens
        const int per_cta = (int)((n + sm_count() * MERGE_ROUND - 1) / (sm_count() * MERGE_ROUND)) * MERGE_ROUND;
        DB2_TRY(launch_next("token_merge_kernel", token_merge_kernel, dim3((unsigned)((n + per_cta - 1) / per_cta)),
                            MERGE_THREADS, (size_t)chunks * MERGE_PITCH * 4, st, k[0], q[0], (int)n, k[1], q[1], per_cta));
        *key = k[1];
        *pos = q[1];
        return DB2_OK;
    }
    if (zero_ctas > 0) {
        table_zero_kernel<<<zero_ctas, SORT_CHUNK, 0, st>>>(z);
        DB2_TRY(after_launch("table_zero_kernel"));
    }
    uint32_t *counts = reinterpret_cast<uint32_t *>(scratch + p.counts_off);
    RadixIn in{tokens, tokens_ld, vocab, nullptr, nullptr};
    int shift = 0;
    for (int pass = 0; pass < p.passes; pass++) {
        const int bits = (p.bits - shift + p.passes - pass - 1) / (p.passes - pass), bins = 1 << bits;
        const int to = pass % 2;
        radix_count_kernel<I><<<(unsigned)p.tiles, RADIX_THREADS, 0, st>>>(in, n, shift, bins, counts, status);
        DB2_TRY(after_launch("radix_count_kernel"));
        radix_scan_kernel<<<1, 1024, 0, st>>>(counts, p.tiles * bins);
        DB2_TRY(after_launch("radix_scan_kernel"));
        radix_move_kernel<I><<<(unsigned)p.tiles, RADIX_THREADS, 0, st>>>(in, n, shift, bins, counts, k[to], q[to]);
        DB2_TRY(after_launch("radix_move_kernel"));
        in.key = k[to];
        in.pos = q[to];
        shift += bits;
    }
    *key = in.key;
    *pos = in.pos;
    return DB2_OK;
}

template <typename T, typename R, int N, bool ADD>
int embed_sum(SumArgs a, const void *grad, double scale, void *res, void *part, cudaStream_t st) {
    const int64_t packets = a.cols / N;
    a.log_tpr = log2_ceil(packets);
    a.log_tpr = a.log_tpr > 7 ? 7 : (a.log_tpr < SUM_MIN_LOG ? SUM_MIN_LOG : a.log_tpr);
    const int64_t groups = SUM_THREADS >> a.log_tpr;
    const int64_t gx = (a.runs + groups - 1) / groups;
    int64_t gy = (packets + (1 << a.log_tpr) - 1) >> a.log_tpr;
    gy = gy > 1024 ? 1024 : gy;
    DB2_TRY(launch_next("embed_sum_kernel", embed_sum_kernel<T, R, N, ADD>, dim3((unsigned)gx, (unsigned)gy), SUM_THREADS, 0,
                        st, a, static_cast<const T *>(grad), (wide_t<T>)scale, static_cast<R *>(res),
                        static_cast<wide_t<T> *>(part)));
    if (a.runs > 1) {
        int64_t jy = (a.cols + 32 * JOIN_N - 1) / (32 * JOIN_N);
        jy = jy > 64 ? 64 : jy;
        int64_t per = a.runs * jy / ((int64_t)sm_count() * 16);
        per = per < 1 ? 1 : (per > JOIN_RUNS ? JOIN_RUNS : per);
        const int64_t jx = (a.runs - 1 + per - 1) / per;
        DB2_TRY(launch_next("embed_join_kernel", embed_join_kernel<T, R, ADD>, dim3((unsigned)jx, (unsigned)jy), 32 * JOIN_Y, 0,
                            st, a, (wide_t<T>)scale, static_cast<R *>(res), static_cast<const wide_t<T> *>(part), (int)per));
    }
    return DB2_OK;
}

template <typename T, typename R>
int embed_sum_any(const SumArgs &a, const void *grad, double scale, void *res, void *part, int accumulate,
                  cudaStream_t st) {
    constexpr int N = 16 / (sizeof(T) > sizeof(R) ? sizeof(T) : sizeof(R)); // both sides' packets are at most 16 bytes
    auto packed = [&](int n) {
        return a.cols % n == 0 && rows_aligned(grad, a.grad_ld, sizeof(T), n * sizeof(T)) &&
               rows_aligned(res, a.res_ld, sizeof(R), n * sizeof(R));
    };
    if (packed(N))
        return accumulate ? embed_sum<T, R, N, true>(a, grad, scale, res, part, st)
                          : embed_sum<T, R, N, false>(a, grad, scale, res, part, st);
    if constexpr (N > 2)
        if (packed(2)) // pairs
            return accumulate ? embed_sum<T, R, 2, true>(a, grad, scale, res, part, st)
                              : embed_sum<T, R, 2, false>(a, grad, scale, res, part, st);
    return accumulate ? embed_sum<T, R, 1, true>(a, grad, scale, res, part, st)
                      : embed_sum<T, R, 1, false>(a, grad, scale, res, part, st);
}

bool seq_type(int dtype) {
    return dtype == DB2_F64 || dtype == DB2_F32 || dtype == DB2_F16 || dtype == DB2_BF16;
}

void count(db2_context *ctx, uint64_t before) {
    std::lock_guard<std::mutex> lock(ctx->mu);
    ctx->stats.launches += g_launches.load(std::memory_order_relaxed) - before;
}

// the status word of the token checks: its place among the context's words, cleared before the launch and read after it
constexpr int EMB_STATUS = 40;
int clear_status(db2_context *ctx) {
    DB2_CUDA(cudaMemsetAsync(ctx->dev_status + EMB_STATUS, 0, sizeof(int32_t), ctx->stream));
    return DB2_OK;
}
int check_status(db2_context *ctx, const char *what, int64_t vocab) {
    DB2_CUDA(cudaMemcpyAsync(ctx->host_status + EMB_STATUS, ctx->dev_status + EMB_STATUS, sizeof(int32_t),
                             cudaMemcpyDeviceToHost, ctx->stream));
    DB2_CUDA(cudaStreamSynchronize(ctx->stream));
    DB2_CHECK(ctx->host_status[EMB_STATUS] == 0, DB2_EDOMAIN,
              "%s: a token lies outside the %lld rows of the table (-1 marks padding)", what, (long long)vocab);
    return DB2_OK;
}

} // namespace

DeviceOperand::DeviceOperand(db2_matrix *m) {
    if (!m)
        return;
    const int rc = ensure_device(m);
    if (rc != DB2_OK)
        throw Error(rc, err_buf());
    keep = m->dev;
    ptr = m->dev_ptr();
    ld = m->dev_ld;
}

// whether two matrices have elements in common, as far as their placements on the device tell
static bool overlap(const db2_matrix *a, const db2_matrix *b) {
    if (!a || !b || !a->dev || a->dev != b->dev || a->rows * a->cols == 0 || b->rows * b->cols == 0)
        return false;
    const int64_t a_end = a->dev_off + (a->rows - 1) * a->dev_ld + a->cols, b_end = b->dev_off + (b->rows - 1) * b->dev_ld + b->cols;
    if (a_end <= b->dev_off || b_end <= a->dev_off)
        return false;
    const int64_t ld = a->dev_ld;
    if (a->esize() != b->esize() || ld != b->dev_ld || ld <= 0)
        return true;
    const int64_t ca = a->dev_off % ld, cb = b->dev_off % ld; // views of one matrix: their columns may lie side by side
    return ca + a->cols > ld || cb + b->cols > ld || (ca < cb + b->cols && cb < ca + a->cols);
}
int Results::add(const char *what, db2_matrix **slot, int dtype, int64_t rows, int64_t cols) {
    if (!slot)
        return DB2_OK;
    for (int i = 0; i < n; i++)
        DB2_CHECK(slot != slots[i] && (!*slot || (*slot != *slots[i] && !(*slots[i] && (*slot)->is_view && (*slots[i])->is_view &&
                                                                         overlap(*slot, *slots[i])))),
                  DB2_EINVAL, "%s: two results are to go to one matrix", what);
    if (*slot)
        DB2_TRY(check_result(*slot, dtype, rows, cols));
    slots[n] = slot;
    fresh[n++] = !*slot;
    return DB2_OK;
}
int Results::apart(const char *what, const db2_matrix *m, std::initializer_list<db2_matrix **> may_be) const {
    for (int i = 0; i < n; i++) {
        const db2_matrix *r = *slots[i];
        if (!r || !r->is_view || !overlap(r, m))
            continue;
        bool same = false;
        for (db2_matrix **s : may_be)
            same = same || (s == slots[i] && r->dtype == m->dtype && r->rows == m->rows && r->cols == m->cols &&
                            r->dev_off == m->dev_off && (r->dev_ld == m->dev_ld || r->rows <= 1));
        DB2_CHECK(same, DB2_EINVAL, "%s: a result is a view that overlaps an operand", what);
    }
    return DB2_OK;
}
Results::~Results() {
    for (int i = 0; i < n && !is_done; i++)
        if (fresh[i] && *slots[i]) {
            db2_matrix_decref(*slots[i]);
            *slots[i] = nullptr;
        }
}

int prepare_update(db2_matrix *m, bool lent) {
    DB2_TRY(ensure_device(m));
    const bool stays = m->is_view || (lent && !m->dev->owned);
    DB2_TRY(lazy_settle(m, stays));
    if (!stays && m->dev.use_count() > 1) {
        // other handles read the buffer: the update goes to a copy
        auto fresh = make_devbuf(m->ctx, (size_t)m->rows * m->cols * m->esize());
        if (m->rows * m->cols > 0)
            DB2_CUDA(cudaMemcpy2DAsync(fresh->ptr, (size_t)m->cols * m->esize(), m->dev_ptr(),
                                       (size_t)m->dev_ld * m->esize(), (size_t)m->cols * m->esize(), (size_t)m->rows,
                                       cudaMemcpyDeviceToDevice, m->ctx->stream));
        m->dev = fresh;
        m->dev_off = 0;
        m->dev_ld = m->cols;
    } else if (m->dev) {
        m->dev->version++;
    }
    m->is_seq = false;
    m->combined = false;
    m->host_valid = false;
    return DB2_OK;
}

} // namespace db2

using namespace db2;

extern "C" {

int db2k_embed(int dtype, const void *table, int64_t vocab, int64_t cols, int64_t table_ld, int index_dtype,
               const void *tokens, int64_t tokens_ld, int64_t n, double scale, void *res, int64_t res_ld,
               int32_t *dev_status, void *stream) {
    DB2_CHECK(seq_type(dtype), DB2_EUNSUPPORTED, "embed: unsupported value type code %d", dtype);
    DB2_CHECK(index_dtype == DB2_I64 || index_dtype == DB2_I32, DB2_EUNSUPPORTED, "embed: tokens are int64 or int32");
    DB2_CHECK(vocab >= 0 && cols >= 0 && n >= 0, DB2_EINVAL, "embed: negative shape");
    if (n == 0 || cols == 0)
        return check_tokens("embed", index_dtype, tokens, tokens_ld, n, vocab, dev_status, as_stream(stream));
    DB2_CHECK((table || vocab == 0) && tokens && res, DB2_EINVAL, "embed: null operand");
    DB2_CHECK(ld_ok(table_ld, vocab, cols) && ld_ok(res_ld, n, cols) && ld_ok(tokens_ld, n, 1), DB2_EINVAL,
              "embed: a leading dimension is smaller than the number of columns");
#define DB2_EMBED(N, I)                                                                                                \
    return embed_launch<T, N, I>(table, vocab, cols, table_ld, tokens, tokens_ld, n, scale, res, res_ld, dev_status,   \
                                 as_stream(stream))
    DB2_DISPATCH_SEQ(dtype, T, {
        constexpr int N = 16 / sizeof(T);
        if (rows_aligned(table, table_ld, sizeof(T), 16) && rows_aligned(res, res_ld, sizeof(T), 16)) {
            if (index_dtype == DB2_I64)
                DB2_EMBED(N, int64_t);
            DB2_EMBED(N, int32_t);
        }
        if (N > 2 && rows_aligned(table, table_ld, sizeof(T), 2 * sizeof(T)) && // pairs
            rows_aligned(res, res_ld, sizeof(T), 2 * sizeof(T))) {
            if (index_dtype == DB2_I64)
                DB2_EMBED(2, int64_t);
            DB2_EMBED(2, int32_t);
        }
        if (index_dtype == DB2_I64)
            DB2_EMBED(1, int64_t);
        DB2_EMBED(1, int32_t);
    });
#undef DB2_EMBED
    return DB2_OK;
}

size_t db2k_embed_grad_scratch_bytes(int dtype, int64_t vocab, int64_t cols, int64_t n) {
    if (vocab <= 0 || cols <= 0 || n <= 0)
        return 0;
    return grad_plan(dtype == DB2_F64 ? 8 : 4, vocab, cols, n).bytes;
}

int db2k_embed_grad(int dtype, const void *grad, int64_t grad_ld, int64_t n, int64_t cols, int index_dtype,
                    const void *tokens, int64_t tokens_ld, double scale, int res_dtype, void *res, int64_t vocab,
                    int64_t res_ld, int accumulate, void *scratch, size_t scratch_bytes, int32_t *dev_status,
                    void *stream) {
    DB2_CHECK(seq_type(dtype), DB2_EUNSUPPORTED, "embedGrad: unsupported value type code %d", dtype);
    DB2_CHECK(res_dtype == dtype || (res_dtype == DB2_F32 && dtype != DB2_F64), DB2_EUNSUPPORTED,
              "embedGrad: the result has the value type of the gradient, or float");
    DB2_CHECK(index_dtype == DB2_I64 || index_dtype == DB2_I32, DB2_EUNSUPPORTED,
              "embedGrad: tokens are int64 or int32");
    DB2_CHECK(vocab >= 0 && cols >= 0 && n >= 0, DB2_EINVAL, "embedGrad: negative shape");
    DB2_CHECK(n < ((int64_t)1 << 31) && vocab < ((int64_t)1 << 31) - 1, DB2_EUNSUPPORTED,
              "embedGrad: fewer than 2^31 tokens and table rows");
    if (vocab == 0 || cols == 0)
        return check_tokens("embedGrad", index_dtype, tokens, tokens_ld, n, vocab, dev_status, as_stream(stream));
    DB2_CHECK(res && ld_ok(res_ld, vocab, cols), DB2_EINVAL, "embedGrad: null result or a leading dimension too small");
    cudaStream_t st = as_stream(stream);
    if (n == 0) {
        if (!accumulate)
            DB2_CUDA(cudaMemset2DAsync(res, (size_t)(vocab > 1 ? res_ld : cols) * dtype_size(res_dtype), 0,
                                       (size_t)cols * dtype_size(res_dtype), (size_t)vocab, st));
        return DB2_OK;
    }
    const GradPlan p = grad_plan(dtype == DB2_F64 ? 8 : 4, vocab, cols, n);
    DB2_CHECK(grad && tokens && ld_ok(grad_ld, n, cols) && ld_ok(tokens_ld, n, 1), DB2_EINVAL,
              "embedGrad: null operand or a leading dimension too small");
    DB2_CHECK(scratch && scratch_bytes >= p.bytes && aligned16(scratch), DB2_EINVAL,
              "embedGrad: scratch smaller than db2k_embed_grad_scratch_bytes, or not 16-byte aligned");
    SumArgs a{};
    char *s = static_cast<char *>(scratch);
    const size_t es = dtype_size(res_dtype);
    Zeros z{static_cast<char *>(res), accumulate ? 0 : vocab, (int64_t)((size_t)cols * es), (int64_t)((size_t)res_ld * es), 0,
            0, (int)es};
    if (!accumulate && (res_ld == cols || vocab == 1) && aligned16(res)) { // one run of bytes: rows of 8 KB, and the rest
        const int64_t all = vocab * z.row_bytes;
        z.row_bytes = z.ld_bytes = 8192;
        z.rows = all / 8192;
        z.tail = all % 8192;
    }
    z.packet = rows_aligned(res, z.rows > 1 ? z.ld_bytes : 0, 1, 16) && z.row_bytes % 16 == 0 ? 16 : (int)es;
    if (index_dtype == DB2_I64)
        DB2_TRY(embed_sort<int64_t>(p, tokens, tokens_ld, n, vocab, s, &a.key, &a.pos, dev_status, z, st));
    else
        DB2_TRY(embed_sort<int32_t>(p, tokens, tokens_ld, n, vocab, s, &a.key, &a.pos, dev_status, z, st));
    a.n = n;
    a.cols = cols;
    a.vocab = vocab;
    a.grad_ld = grad_ld;
    a.res_ld = res_ld;
    a.part_ld = p.part_ld;
    a.runs = p.runs;
    if (dtype == DB2_F16 && res_dtype == DB2_F32)
        return embed_sum_any<__half, float>(a, grad, scale, res, s + p.part_off, accumulate, st);
    if (dtype == DB2_BF16 && res_dtype == DB2_F32)
        return embed_sum_any<__nv_bfloat16, float>(a, grad, scale, res, s + p.part_off, accumulate, st);
    DB2_DISPATCH_SEQ(dtype, T, return (embed_sum_any<T, T>(a, grad, scale, res, s + p.part_off, accumulate, st)));
    return DB2_OK;
}

int db2_embed(db2_context *ctx, db2_matrix **res, db2_matrix *table, db2_matrix *tokens, double scale) {
    DB2_API_BEGIN
    DB2_CHECK(ctx && res && table && tokens, DB2_EINVAL, "null argument");
    DB2_CHECK(seq_type(table->dtype), DB2_EUNSUPPORTED, "embed: unsupported value type code %d", table->dtype);
    DB2_CHECK(tokens->cols == 1, DB2_EINVAL, "embed: tokens must be a column matrix");
    DB2_CHECK(tokens->dtype == DB2_I64 || tokens->dtype == DB2_I32, DB2_EUNSUPPORTED,
              "embed: tokens are int64 or int32");
    bind_device(ctx);
    const uint64_t before = g_launches.load();
    const DeviceOperand dt(table), di(tokens);
    Results results;
    DB2_TRY(results.add("embed", res, table->dtype, tokens->rows, table->cols));
    DB2_TRY(results.apart("embed", table));
    DB2_TRY(prepare_result(ctx, res, table->dtype, tokens->rows, table->cols));
    DB2_TRY(clear_status(ctx));
    DB2_TRY(db2k_embed(table->dtype, dt.ptr, table->rows, table->cols, dt.ld, tokens->dtype, di.ptr, di.ld, tokens->rows,
                       scale, (*res)->dev_ptr(), (*res)->dev_ld, ctx->dev_status + EMB_STATUS, ctx->stream));
    count(ctx, before);
    DB2_TRY(check_status(ctx, "embed", table->rows));
    return results.done();
    DB2_API_END
}

int db2_embedGrad(db2_context *ctx, db2_matrix **res, db2_matrix *grad, db2_matrix *tokens, int64_t vocab, double scale,
                  int res_dtype, int accumulate) {
    DB2_API_BEGIN
    DB2_CHECK(ctx && res && grad && tokens, DB2_EINVAL, "null argument");
    DB2_CHECK(seq_type(grad->dtype), DB2_EUNSUPPORTED, "embedGrad: unsupported value type code %d", grad->dtype);
    DB2_CHECK(tokens->cols == 1 && tokens->rows == grad->rows, DB2_EINVAL,
              "embedGrad: tokens must be a column matrix with as many rows as grad (%lld), got (%lld x %lld)",
              (long long)grad->rows, (long long)tokens->rows, (long long)tokens->cols);
    DB2_CHECK(tokens->dtype == DB2_I64 || tokens->dtype == DB2_I32, DB2_EUNSUPPORTED,
              "embedGrad: tokens are int64 or int32");
    DB2_CHECK(res_dtype == grad->dtype || (res_dtype == DB2_F32 && grad->dtype != DB2_F64), DB2_EUNSUPPORTED,
              "embedGrad: the result has the value type of the gradient, or float");
    DB2_CHECK(vocab >= 0, DB2_EINVAL, "embedGrad: negative number of table rows");
    DB2_CHECK(*res || !accumulate, DB2_EINVAL, "embedGrad: adding needs a matrix to add to");
    bind_device(ctx);
    const uint64_t before = g_launches.load();
    const DeviceOperand dg(grad), di(tokens);
    Results results;
    if (accumulate) {
        DB2_CHECK((*res)->dtype == res_dtype && (*res)->rows == vocab && (*res)->cols == grad->cols, DB2_EINVAL,
                  "embedGrad: the matrix to add to has shape (%lld x %lld) / type %d, expected (%lld x %lld) / type %d",
                  (long long)(*res)->rows, (long long)(*res)->cols, (*res)->dtype, (long long)vocab,
                  (long long)grad->cols, res_dtype);
        DB2_TRY(results.add("embedGrad", res, res_dtype, vocab, grad->cols));
        DB2_TRY(results.apart("embedGrad", grad));
        DB2_TRY(prepare_update(*res, (*res)->dev != grad->dev)); // (its own operand is read before it is added to)
    } else {
        DB2_TRY(results.add("embedGrad", res, res_dtype, vocab, grad->cols));
        DB2_TRY(results.apart("embedGrad", grad));
        DB2_TRY(prepare_result(ctx, res, res_dtype, vocab, grad->cols));
    }
    const size_t sb = db2k_embed_grad_scratch_bytes(grad->dtype, vocab, grad->cols, grad->rows);
    void *scratch = nullptr;
    DB2_TRY(ctx_scratch(ctx, sb, &scratch));
    DB2_TRY(clear_status(ctx));
    DB2_TRY(db2k_embed_grad(grad->dtype, dg.ptr, dg.ld, grad->rows, grad->cols, tokens->dtype, di.ptr, di.ld, scale,
                            res_dtype, (*res)->dev_ptr(), vocab, (*res)->dev_ld, accumulate, scratch,
                            ctx->scratch_bytes, ctx->dev_status + EMB_STATUS, ctx->stream));
    count(ctx, before);
    DB2_TRY(check_status(ctx, "embedGrad", vocab));
    return results.done();
    DB2_API_END
}

} // extern "C"
