// Embedding lookup with scaling, and its gradient.
//
//   out[r] = s * table[tok[r]]                      dtable[v] (+)= s * sum over r with tok[r] = v of dout[r]
//
// Lookup: a group of threads per row, every thread a few vectors of the row; memory latency and bandwidth are all there is.
//
// Gradient: the rows are sorted by token (stable radix sort, so rows of one token keep their order), then summed in that order in
// fp32: no atomics on values, the same bits every time.
//   1. sort: digits of up to 9 bits; up to SMALL_SORT tokens every block does all passes for itself in shared memory and goes on with the sums,
//      otherwise two launches a pass (digit counts of every tile; ranks and scatter).  Tokens outside the table get the key `vocab` and end
//      up last.
//   2. sum: the sorted rows are cut into pieces of `piece` rows; a group of threads sums a piece column by column.  A token whose
//      rows lie inside one piece is written at once; one that crosses a border leaves a partial sum per piece ("head": it began in
//      an earlier piece; "tail": it begins here and goes on).
//   3. join: the pieces with a tail (a list, filled by atomics: its order changes no result; few pieces are all looked at) add the heads that
//      follow.
// A frequent token is thus spread over as many groups as it has pieces.  Without accumulation the rows of tokens that do not occur are
// zeroed by extra blocks of the same launches, so that the table is written once.
// Measured on a B200 (device time of a pass among passes over the same buffers; with buffers that change 3 to 14 % more): lookup of 65536 x 1024 bf16 29.6 us
// (7.5 TB/s of what it reads and writes; repeated rows come from L2), x 1023, single elements, 68 us, of 64 x 512 2 us, a launch.  Gradient of
// 32768 x 1024 bf16 in a table of 50000 rows 75 to 77 us against 42 us of bytes: the sort takes 19 us of latency (four launches of 16 blocks), the sums
// with 209 MB 38 us (5.5 TB/s), the joins 10 us of latency.  In a table of 259 rows the same batch takes 41 us against 10.5: two launches of the sort, sums into
// partial rows and joins over long runs of pieces.  1516 x 128 in 259 rows 11.3 us: the sort 4.8, the sums 2.3 and a second launch for the joins 2.5.
#include <math.h>

#include "typed.cuh"

namespace b2 {
namespace {

// ---- lookup -------------------------------------------------------------------------------------------------------------------
// Loads a thread has under way: the narrower, the more
__host__ __device__ constexpr int in_flight(int w) { return w >= 4 ? 4 : w == 2 ? 8 : 16; }
// tpr threads a row (a power of two up to 256), W elements an access
template <typename T, typename U, int W>
__global__ void __launch_bounds__(256) embedding_forward_kernel(U *__restrict__ out, long long ld_out, const T *__restrict__ table, long long ld_table, int vocab,
                                                                int dim, const int *__restrict__ tokens, long long rows, float scale, int tpr) {
    constexpr int UN = in_flight(W);
    const int lane = threadIdx.x & (tpr - 1);
    const int per_block = 256 / tpr;
    for (long long r = (long long)blockIdx.x * per_block + threadIdx.x / tpr; r < rows; r += (long long)gridDim.x * per_block) {
        const int tok = __ldg(tokens + r);
        U *to = out + r * ld_out;
        if (tok >= 0 && tok < vocab) {
            const T *from = table + (long long)tok * ld_table;
            int c = lane * W;
            for (; c + (UN - 1) * tpr * W < dim; c += UN * tpr * W) {
                float v[UN][W];
#pragma unroll
                for (int i = 0; i < UN; ++i) load_vec<T, W>(v[i], from + c + i * tpr * W);
#pragma unroll
                for (int i = 0; i < UN; ++i) {
#pragma unroll
                    for (int j = 0; j < W; ++j) v[i][j] *= scale;
                    store_vec<U, W>(to + c + i * tpr * W, v[i]);
                }
            }
            for (; c < dim; c += tpr * W) {
                float v[W];
                load_vec<T, W>(v, from + c);
#pragma unroll
                for (int j = 0; j < W; ++j) v[j] *= scale;
                store_vec<U, W>(to + c, v);
            }
        } else {
            // a padding frame is zero; a token beyond the table shows as NaN
            const float fill = tok < 0 ? 0.0f : nanf("");
            float v[W];
#pragma unroll
            for (int j = 0; j < W; ++j) v[j] = fill;
            for (int c = lane * W; c < dim; c += tpr * W) store_vec<U, W>(to + c, v);
        }
    }
}

// ---- sort ---------------------------------------------------------------------------------------------------------------------
constexpr int MAX_DIGIT_BITS = 9;
constexpr int SORT_THREADS = 512, SORT_WARPS = SORT_THREADS / 32;
constexpr int SMALL_SORT = 4096;             // tokens one block sorts in shared memory

__device__ __forceinline__ unsigned key_of(int tok, int vocab) { return (tok >= 0 && tok < vocab) ? (unsigned)tok : (unsigned)vocab; }

// the lanes, of those active, that hold the same digit as this one
__device__ __forceinline__ unsigned same_digit(unsigned active, unsigned digit) { return __match_any_sync(active, digit); }

// Exclusive prefix sum over one value a thread; all threads of the block call it.
__device__ __forceinline__ unsigned block_exclusive_scan(unsigned x, unsigned *warp_tot) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    unsigned inc = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
    }
    if (lane == 31) warp_tot[w] = inc;
    __syncthreads();
    unsigned before = inc - x;
#pragma unroll
    for (int i = 0; i < SORT_WARPS; ++i) before += i < w ? warp_tot[i] : 0;
    __syncthreads();
    return before;
}
// count[warp][digit] becomes the place of the first key of (digit, warp): digits in order, within a digit the warps in order.  before: what thread d adds for
// digit d; total: its keys in all tiles, or a negative value for those counted here.
__device__ __forceinline__ void places(unsigned *count, int digits, unsigned before, int total, unsigned *warp_tot) {
    const int d = threadIdx.x;
    unsigned c[SORT_WARPS], sum = 0;
#pragma unroll
    for (int w = 0; w < SORT_WARPS; ++w) {
        c[w] = d < digits ? count[w * digits + d] : 0;
        sum += c[w];
    }
    unsigned at = block_exclusive_scan(total < 0 ? sum : (unsigned)total, warp_tot) + before;
    if (d < digits)
#pragma unroll
        for (int w = 0; w < SORT_WARPS; ++w) { count[w * digits + d] = at; at += c[w]; }
    __syncthreads();
}

// All passes for up to SMALL_SORT tokens, in the block's shared memory: sm holds SMALL_WORDS words and the counts.  Warp w ranks the keys
// [w * seg, (w + 1) * seg) in rounds of 32, counts kept per (digit, warp), so equal digits stay in order.  *keys and *rows are the sorted ones.
constexpr int SMALL_WORDS = 3 * SMALL_SORT;
__device__ __forceinline__ void sort_in_block(unsigned *sm, const int *tokens, int n, int vocab, int passes, int bits, const unsigned **keys, const unsigned short **rows) {
    unsigned *key[2] = {sm, sm + SMALL_SORT};
    unsigned short *row[2] = {(unsigned short *)(sm + 2 * SMALL_SORT), (unsigned short *)(sm + 2 * SMALL_SORT) + SMALL_SORT};
    unsigned *count = sm + SMALL_WORDS;                    // [SORT_WARPS][digits]
    __shared__ unsigned warp_tot[SORT_WARPS];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, digits = 1 << bits;
    for (int i = threadIdx.x; i < n; i += SORT_THREADS) { key[0][i] = key_of(tokens[i], vocab); row[0][i] = (unsigned short)i; }
    __syncthreads();
    const int seg = ((n + SORT_WARPS - 1) / SORT_WARPS + 31) & ~31;
    for (int p = 0; p < passes; ++p) {
        const unsigned *kin = key[p & 1];
        const unsigned short *rin = row[p & 1];
        unsigned *kout = key[(p & 1) ^ 1];
        unsigned short *rout = row[(p & 1) ^ 1];
        for (int i = threadIdx.x; i < digits * SORT_WARPS; i += SORT_THREADS) count[i] = 0;
        __syncthreads();
        unsigned short rank[SMALL_SORT / SORT_THREADS];
#pragma unroll
        for (int k = 0; k < SMALL_SORT / SORT_THREADS; ++k) {
            const int i = w * seg + k * 32 + lane;
            const bool on = k * 32 < seg && i < n;
            const unsigned active = __ballot_sync(0xffffffffu, on);
            if (on) {
                const unsigned d = (kin[i] >> (p * bits)) & (digits - 1);
                const unsigned same = same_digit(active, d), c = count[w * digits + d];
                __syncwarp(active);
                if (lane == 31 - __clz(same)) count[w * digits + d] = c + __popc(same);
                rank[k] = (unsigned short)(c + __popc(same & ((1u << lane) - 1)));
            }
            __syncwarp();
        }
        __syncthreads();
        places(count, digits, 0, -1, warp_tot);
#pragma unroll
        for (int k = 0; k < SMALL_SORT / SORT_THREADS; ++k) {
            const int i = w * seg + k * 32 + lane;
            if (k * 32 < seg && i < n) {
                const unsigned d = (kin[i] >> (p * bits)) & (digits - 1), at = count[w * digits + d] + rank[k];
                kout[at] = kin[i];
                rout[at] = rin[i];
            }
        }
        __syncthreads();
    }
    *keys = key[passes & 1];
    *rows = row[passes & 1];
}

struct SortArgs {
    const int *tokens;                     // first pass: the keys come from here, the rows are 0, 1, 2, ...
    const unsigned *kin; const int *rin;   // later passes
    unsigned *kout; int *rout;
    unsigned *hist;                        // [tiles][digits]
    unsigned *present, *list_count;
    int n, vocab, shift, bits, tiles, tile;
};
// rows of the gradient that extra blocks of a launch zero: tokens in [v0, v1) that do not occur
struct ZeroArgs {
    void *dtable;
    long long row_bytes, ld_bytes;
    const unsigned *present;
    int v0, v1;
    int unit;                              // bytes of a store that every row starts and ends on: 16, 4 or 2
};

__device__ __forceinline__ unsigned sort_key(const SortArgs &a, int i) { return a.tokens ? key_of(a.tokens[i], a.vocab) : a.kin[i]; }

// by a warp
__device__ __forceinline__ void zero_row(const ZeroArgs &z, long long v) {
    const int lane = threadIdx.x & 31;
    char *p = (char *)z.dtable + v * z.ld_bytes;
    if (z.unit == 16)
        for (long long b = lane * 16; b < z.row_bytes; b += 512) *reinterpret_cast<uint4 *>(p + b) = make_uint4(0, 0, 0, 0);
    else if (z.unit == 4)
        for (long long b = lane * 4; b < z.row_bytes; b += 128) *reinterpret_cast<unsigned *>(p + b) = 0;
    else
        for (long long b = lane * 2; b < z.row_bytes; b += 64) *reinterpret_cast<unsigned short *>(p + b) = 0;
}
// one warp a row; block `blk` of `blks`
__device__ __forceinline__ void zero_rows(const ZeroArgs &z, int blk, int blks) {
    const int warps = blockDim.x >> 5;
    for (long long v = (long long)z.v0 + (long long)blk * warps + (threadIdx.x >> 5); v < z.v1; v += (long long)blks * warps) {
        if (z.present[v >> 5] >> (v & 31) & 1) continue;
        zero_row(z, v);
    }
}

// digit counts of every tile; the first pass also notes which tokens occur (their bits were cleared before)
__global__ void __launch_bounds__(SORT_THREADS) sort_count_kernel(const SortArgs a, const ZeroArgs z) {
    grid_wait();
    grid_release();
    if ((int)blockIdx.x >= a.tiles) { zero_rows(z, blockIdx.x - a.tiles, gridDim.x - a.tiles); return; }
    extern __shared__ unsigned sm[];
    const int digits = 1 << a.bits;
    for (int i = threadIdx.x; i < digits; i += SORT_THREADS) sm[i] = 0;
    __syncthreads();
    const int i0 = blockIdx.x * a.tile, i1 = min(a.n, i0 + a.tile);
    for (int i = i0 + threadIdx.x; i < i1; i += SORT_THREADS) {
        const unsigned k = sort_key(a, i);
        atomicAdd(sm + ((k >> a.shift) & (digits - 1)), 1u);
        // With many rows a token, nearly all of them find its bit set if they look, and do not queue for its word (65536 rows of 20 tokens: 66 us
        // without, 38 us with a look; 32768 rows of 50000 tokens: 78 and 80 us)
        if (a.tokens && k < (unsigned)a.vocab && !(a.n / 8 > a.vocab && __ldcg(a.present + (k >> 5)) >> (k & 31) & 1))
            atomicOr(a.present + (k >> 5), 1u << (k & 31));
    }
    __syncthreads();
    for (int i = threadIdx.x; i < digits; i += SORT_THREADS) a.hist[(size_t)blockIdx.x * digits + i] = sm[i];
}

// ranks of a tile's keys and scatter; every block adds up the counts before its own by itself
__global__ void __launch_bounds__(SORT_THREADS) sort_scatter_kernel(const SortArgs a, const ZeroArgs z) {
    grid_wait();
    grid_release();
    if ((int)blockIdx.x >= a.tiles) { zero_rows(z, blockIdx.x - a.tiles, gridDim.x - a.tiles); return; }
    extern __shared__ unsigned sm[];
    __shared__ unsigned warp_tot[SORT_WARPS];
    const int digits = 1 << a.bits, lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    unsigned *count = sm;                                  // [SORT_WARPS][digits]
    for (int i = threadIdx.x; i < digits * SORT_WARPS; i += SORT_THREADS) count[i] = 0;
    unsigned before = 0, total = 0;
    if ((int)threadIdx.x < digits) {
#pragma unroll 8
        for (int t = 0; t < a.tiles; ++t) {
            const unsigned h = a.hist[(size_t)t * digits + threadIdx.x];
            if (t < (int)blockIdx.x) before += h;
            total += h;
        }
    }
    __syncthreads();
    // counts of every warp's segment of the tile
    const int i0 = blockIdx.x * a.tile, i1 = min(a.n, i0 + a.tile), seg = a.tile / SORT_WARPS;
    const int s0 = i0 + w * seg, s1 = min(i1, s0 + seg);
    for (int i = s0 + lane; i < s1; i += 32) atomicAdd(count + w * digits + ((sort_key(a, i) >> a.shift) & (digits - 1)), 1u);
    __syncthreads();
    places(count, digits, before, (int)total, warp_tot);
    for (int j = s0; j < s1; j += 32) {
        const int i = j + lane;
        const bool on = i < s1;
        const unsigned active = __ballot_sync(0xffffffffu, on);
        if (on) {
            const unsigned k = sort_key(a, i), d = (k >> a.shift) & (digits - 1);
            const unsigned same = same_digit(active, d), c = count[w * digits + d];
            __syncwarp(active);
            if (lane == 31 - __clz(same)) count[w * digits + d] = c + __popc(same);
            const unsigned at = c + __popc(same & ((1u << lane) - 1));
            a.kout[at] = k;
            a.rout[at] = a.tokens ? i : a.rin[i];
        }
        __syncwarp();
    }
}

// ---- sums ---------------------------------------------------------------------------------------------------------------------
struct SumArgs {
    const unsigned *keys; const int *rows;
    float *partial;                 // [pieces][2][dim_pad]
    int *list; unsigned *list_count;
    long long ld_dout, ld_dtable;
    int n, vocab, dim, dim_pad, piece, pieces, tpr, cols, accumulate;
    float scale;
};

template <typename U, int W> __device__ __forceinline__ void put_row(U *to, const float (&s)[W], float scale, int accumulate) {
    float v[W];
    if (accumulate) {
        load_vec<U, W>(v, to);
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = fmaf(scale, s[j], v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = scale * s[j];
    }
    store_vec<U, W>(to, v);
}

constexpr int SUM_THREADS = 128, MIN_GROUP = 8, MAX_PIECE = 64;
constexpr int AHEAD = 12;                    // rows a thread has under way

// A group of a.tpr threads (a power of two, MIN_GROUP to SUM_THREADS) takes a.tpr times 16 bytes of a piece's rows: a thread the columns col0 + i * step, NV
// vectors of them, as the rows' alignment asks for.  key, row: the piece's n rows in shared memory; before, behind: the keys on either side;
// ring: AHEAD times 16 bytes for each of the block's THREADS threads.
template <typename T, int W> __host__ __device__ constexpr int sum_vectors() { return 16 / (W * (int)sizeof(T)); }
template <typename T, typename U, int W, int THREADS, typename Row>
__device__ __forceinline__ void sum_piece(U *__restrict__ dtable, const T *dout, const SumArgs &a, int p, int col0, int step, const unsigned *key, const Row *row,
                                          int n, unsigned before, unsigned behind, uint4 *ring) {
    constexpr int NV = sum_vectors<T, W>();
    constexpr bool RING = W * sizeof(T) >= 4;
    unsigned cur = key[0];
    if (cur >= (unsigned)a.vocab) return;                  // nothing but padding from here on
    bool from_before = before == cur;
    float acc[NV][W];
    const auto clear = [&]() {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) acc[i][j] = 0.0f;
    };
    clear();
    const auto save = [&](float *to) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (col0 + i * step < a.dim) store_vec<float, W>(to + col0 + i * step, acc[i]);
    };
    const auto put = [&]() {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (col0 + i * step < a.dim) put_row<U, W>(dtable + (long long)cur * a.ld_dtable + col0 + i * step, acc[i], a.scale, a.accumulate);
    };
    float *head = a.partial + (size_t)p * 2 * a.dim_pad;
    // another token, or padding: the one before is complete (what ends with the piece is seen to below)
    const auto turn = [&](unsigned k) {
        if (from_before) save(head);
        else put();
        from_before = false;
        cur = k;
        clear();
    };
    if constexpr (RING) {
        // the next AHEAD rows are on their way into the thread's own slots
        constexpr int VB = W * sizeof(T);
        const unsigned slots = (unsigned)__cvta_generic_to_shared(ring) + threadIdx.x * VB;
        const auto fetch = [&](int i, int stage) {
            if (i < n && key[i] < (unsigned)a.vocab)
#pragma unroll
                for (int v = 0; v < NV; ++v)
                    if (col0 + v * step < a.dim) cp_async<VB>(slots + (stage * NV + v) * THREADS * VB, dout + (long long)row[i] * a.ld_dout + col0 + v * step);
            cp_commit();
        };
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) fetch(i, i);
        for (int i = 0, stage = 0; i < n; ++i, stage = stage + 1 < AHEAD ? stage + 1 : 0) {
            cp_wait<AHEAD - 1>();
            const unsigned k = key[i];
            if (k != cur) turn(k);
            if (k >= (unsigned)a.vocab) break;             // padding to the end
            float x[NV][W];
#pragma unroll
            for (int v = 0; v < NV; ++v)
                load_vec<T, W>(x[v], reinterpret_cast<const T *>(reinterpret_cast<const char *>(ring) + (stage * NV + v) * THREADS * VB + threadIdx.x * VB));
            fetch(i + AHEAD, stage);
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int j = 0; j < W; ++j) acc[v][j] += x[v][j];
        }
    } else {
        constexpr int ROWS = 4;                            // 16-bit elements one by one: 32 loads under way
        for (int i = 0; i < n; i += ROWS) {
            T x[ROWS][NV];
            unsigned k[ROWS];
#pragma unroll
            for (int u = 0; u < ROWS; ++u) {
                k[u] = i + u < n ? key[i + u] : 0xffffffffu;
                if (k[u] < (unsigned)a.vocab)
#pragma unroll
                    for (int v = 0; v < NV; ++v)
                        if (col0 + v * step < a.dim) x[u][v] = dout[(long long)row[i + u] * a.ld_dout + col0 + v * step];
            }
#pragma unroll
            for (int u = 0; u < ROWS; ++u) {
                if (k[u] != cur && i + u < n && cur < (unsigned)a.vocab) turn(k[u]);
                if (k[u] < (unsigned)a.vocab)
#pragma unroll
                    for (int v = 0; v < NV; ++v) acc[v][0] += to_float(x[u][v]);
            }
        }
    }
    if (cur >= (unsigned)a.vocab) return;
    if (from_before) save(head);
    else if (behind == cur) {
        save(head + a.dim_pad);
        if (a.list && col0 == 0) a.list[atomicAdd(a.list_count, 1u)] = p;
    } else put();
}

// Every other block zeroes absent rows as long as there are any: stores that nothing waits for, beside loads that the sums wait for.
template <typename T, typename U, int W>
__global__ void __launch_bounds__(SUM_THREADS) embedding_sum_kernel(U *__restrict__ dtable, const T *dout, const SumArgs a, const ZeroArgs z, int sum_blocks,
                                                                    int zero_blocks) {
    __shared__ unsigned s_key[SUM_THREADS / MIN_GROUP * MAX_PIECE];
    __shared__ int s_row[SUM_THREADS / MIN_GROUP * MAX_PIECE];
    __shared__ uint4 ring[W * sizeof(T) >= 4 ? AHEAD * SUM_THREADS : 1];
    grid_wait();
    grid_release();
    const int both = 2 * min(sum_blocks, zero_blocks);
    int block = blockIdx.x;
    if (block < both) {
        if (block & 1) { zero_rows(z, block >> 1, zero_blocks); return; }
        block >>= 1;
    } else {
        block -= both >> 1;
        if (zero_blocks > sum_blocks) { zero_rows(z, block, zero_blocks); return; }
    }
    const int step = a.tpr * W, width = step * sum_vectors<T, W>(), tiles = (a.dim + width - 1) / width;
    const int group = threadIdx.x / a.tpr, lane = threadIdx.x & (a.tpr - 1);
    const long long unit = (long long)block * (SUM_THREADS / a.tpr) + group;
    const int p = (int)(unit / tiles), col0 = (int)(unit - (long long)p * tiles) * width + lane * W;
    // the piece's keys and rows first: then the rows themselves can all be asked for at once
    const int i0 = p < a.pieces ? p * a.piece : a.n, n = min(a.n - i0, a.piece);
    unsigned *key = s_key + group * a.piece;
    int *row = s_row + group * a.piece;
    for (int i = lane; i < n; i += a.tpr) { key[i] = a.keys[i0 + i]; row[i] = a.rows[i0 + i]; }
    const unsigned before = n > 0 && i0 > 0 ? a.keys[i0 - 1] : 0xffffffffu, behind = n > 0 && i0 + n < a.n ? a.keys[i0 + n] : 0xffffffffu;
    __syncthreads();
    if (n > 0 && col0 < a.dim) sum_piece<T, U, W, SUM_THREADS>(dtable, dout, a, p, col0, step, key, row, n, before, behind, ring);
}

// Sort and sums in one launch, for few tokens: every block sorts all of them by itself, which takes no longer than one block would, and then has its share of
// the pieces' keys and rows in its own shared memory.  Block 0 leaves the keys for the joins.
template <typename T, typename U, int W>
__global__ void __launch_bounds__(SORT_THREADS) embedding_small_kernel(U *__restrict__ dtable, const T *dout, const int *tokens, const SumArgs a,
                                                                       const ZeroArgs z, int passes, int bits, unsigned *__restrict__ keys_out) {
    extern __shared__ __align__(16) unsigned sm[];
    grid_wait();
    const unsigned *key;
    const unsigned short *row;
    sort_in_block(sm, tokens, a.n, a.vocab, passes, bits, &key, &row);
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < a.n; i += SORT_THREADS) keys_out[i] = key[i];
    // absent rows: a lane looks for each of 32 tokens among the keys
    for (long long v0 = (long long)z.v0 + ((long long)blockIdx.x * SORT_WARPS + (threadIdx.x >> 5)) * 32; v0 < z.v1; v0 += (long long)gridDim.x * SORT_WARPS * 32) {
        const unsigned v = (unsigned)v0 + (threadIdx.x & 31);
        int lo = 0, hi = a.n;                              // the first key that is not below v
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (key[mid] < v) lo = mid + 1; else hi = mid;
        }
        unsigned absent = __ballot_sync(0xffffffffu, v < (unsigned)z.v1 && (lo == a.n || key[lo] != v));
        for (; absent; absent &= absent - 1) zero_row(z, v0 + __ffs(absent) - 1);
    }
    const int step = a.tpr * W, width = step * sum_vectors<T, W>(), tiles = (a.dim + width - 1) / width, groups = SORT_THREADS / a.tpr;
    const int group = threadIdx.x / a.tpr, lane = threadIdx.x & (a.tpr - 1);
    uint4 *ring = reinterpret_cast<uint4 *>(sm + SMALL_WORDS);   // the counts are done with
    for (int unit = blockIdx.x * groups + group; unit < a.pieces * tiles; unit += gridDim.x * groups) {
        const int p = unit / tiles, col0 = (unit - p * tiles) * width + lane * W, i0 = p * a.piece, n = min(a.n - i0, a.piece);
        if (col0 < a.dim)
            sum_piece<T, U, W, SORT_THREADS>(dtable, dout, a, p, col0, step, key + i0, row + i0, n, i0 > 0 ? key[i0 - 1] : 0xffffffffu, i0 + n < a.n ? key[i0 + n] : 0xffffffffu, ring);
    }
}

// Tokens that cross pieces: tail of the first piece plus the heads of those that follow.  A block is a.cols column vectors x 256 / a.cols
// phases: a phase adds every so-many-th head, the phases' sums are added in order.
template <typename U, int W>
__global__ void __launch_bounds__(256) embedding_join_kernel(U *__restrict__ dtable, const SumArgs a) {
    constexpr int P = W < 4 ? 4 : W;                       // partial sums are aligned whatever the table is
    __shared__ __align__(16) float part[256 * P];
    grid_wait();
    const unsigned n_list = a.list ? *a.list_count : a.pieces;
    const int phases = 256 / a.cols, x = threadIdx.x & (a.cols - 1), y = threadIdx.x / a.cols, col = ((int)blockIdx.y * a.cols + x) * P;
    for (unsigned li = blockIdx.x; li < n_list; li += gridDim.x) {
        const int p = a.list ? a.list[li] : (int)li;
        if ((p + 1) * (long long)a.piece >= a.n) continue;
        const unsigned key = a.keys[(size_t)(p + 1) * a.piece], last = a.keys[(size_t)(p + 1) * a.piece - 1], before = p > 0 ? a.keys[(size_t)p * a.piece - 1] : 0xffffffffu;
        // without a list: does a token that begins in the piece go on behind it?
        if (!a.list && (key >= (unsigned)a.vocab || last != key || before == key)) continue;
        float s[P];
#pragma unroll
        for (int j = 0; j < P; ++j) s[j] = 0.0f;
        if (col < a.dim) {
            if (y == 0) load_vec<float, P>(s, a.partial + ((size_t)p * 2 + 1) * a.dim_pad + col);
            for (unsigned q = p + 1 + y; q < (unsigned)a.pieces; q += 4 * phases) {
                float v[4][P];
                unsigned k[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    // the head is fetched beside the key that tells whether it is one
                    const unsigned at = q + u * phases, in = min(at, (unsigned)a.pieces - 1);
                    k[u] = at < (unsigned)a.pieces ? a.keys[(size_t)in * a.piece] : 0xffffffffu;
                    load_vec<float, P>(v[u], a.partial + (size_t)in * 2 * a.dim_pad + col);
                }
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (k[u] == key) {
#pragma unroll
                        for (int j = 0; j < P; ++j) s[j] += v[u][j];
                    }
                if (k[3] != key) break;
            }
        }
        store_vec<float, P>(part + threadIdx.x * P, s);
        __syncthreads();
        if (y == 0 && col < a.dim) {
#pragma unroll 7
            for (int i = 1; i < phases; ++i) {
                float v[P];
                load_vec<float, P>(v, part + (i * a.cols + x) * P);
#pragma unroll
                for (int j = 0; j < P; ++j) s[j] += v[j];
            }
#pragma unroll
            for (int i = 0; i < P; i += W)
                if (col + i < a.dim) put_row<U, W>(dtable + (long long)key * a.ld_dtable + col + i, *reinterpret_cast<const float(*)[W]>(s + i), a.scale, a.accumulate);
        }
        __syncthreads();
    }
}

// ---- plan of a gradient call --------------------------------------------------------------------------------------------------
struct Plan {
    int bits, passes, tiles, tile, piece, pieces, dim_pad;
    size_t present, count, keys[2], rows[2], hist, list, partial, total;   // byte offsets in the workspace
};
size_t pad256(size_t x) { return (x + 255) & ~(size_t)255; }

Plan make_plan(long long n, int vocab, int dim) {
    Plan p;
    int bits = 1;
    while (((unsigned)vocab >> bits) != 0) ++bits;                          // keys 0 .. vocab
    p.passes = (bits + MAX_DIGIT_BITS - 1) / MAX_DIGIT_BITS;
    p.bits = (bits + p.passes - 1) / p.passes;
    // tiles: as few keys as fill the device, so that a tile's rounds are short; at least 2048
    long long tile = (n + 147) / 148;
    tile = tile < 2048 ? 2048 : (tile + SORT_THREADS - 1) / SORT_THREADS * SORT_THREADS;
    p.tile = (int)tile;
    p.tiles = (int)((n + tile - 1) / tile);
    // pieces: few rows give parallel groups, many rows few partial sums (32768 rows: 16 rows a piece 87 us, 32 77 us, 64 78 us)
    p.piece = n <= 4096 ? 8 : n <= 16384 ? 16 : n <= 262144 ? 32 : MAX_PIECE;
    p.pieces = (int)((n + p.piece - 1) / p.piece);
    p.dim_pad = (dim + 15) / 16 * 16;
    size_t at = 0;
    const auto take = [&at](size_t bytes) { const size_t o = at; at += pad256(bytes); return o; };
    p.count = take(4);
    p.present = take(((size_t)vocab + 31) / 32 * 4);
    p.keys[0] = take((size_t)n * 4); p.keys[1] = take((size_t)n * 4);
    p.rows[0] = take((size_t)n * 4); p.rows[1] = take((size_t)n * 4);
    p.hist = take((size_t)p.tiles * (1 << p.bits) * 4);
    p.list = take((size_t)p.pieces * 4);
    p.partial = take((size_t)p.pieces * 2 * p.dim_pad * 4);
    p.total = at;
    return p;
}

bool bad_sizes(const char *who, long long n, int vocab, int dim) {
    if (n < 0 || n > (1ll << 30) || vocab < 1 || vocab > (1 << 27) || dim < 1 || dim > (1 << 20)) {
        set_error("%s: %lld tokens, %d table rows of %d (at most 2^30, 2^27 and 2^20)", who, n, vocab, dim);
        return true;
    }
    return false;
}

// the widest access that dim, both leading dimensions and both addresses allow
int common_width(int most, int dim, const void *a, long long lda, int ea, const void *b, long long ldb, int eb) {
    for (int w = most; w > 1; w >>= 1) {
        const size_t ba = (size_t)w * ea < 16 ? (size_t)w * ea : 16, bb = (size_t)w * eb < 16 ? (size_t)w * eb : 16;
        if (dim % w == 0 && lda % w == 0 && ldb % w == 0 && aligned_to(a, ba) && aligned_to(b, bb)) return w;
    }
    return 1;
}

template <typename T, typename U, int W>
int forward(U *out, long long ld_out, const T *table, long long ld_table, int vocab, int dim, const int *tokens, long long n, float scale, cudaStream_t st) {
    // few rows: a thread per vector, so that all loads go out at once; many rows: as many as a thread has under way
    const unsigned vecs = (unsigned)((dim + W - 1) / W);
    const bool few = (double)n * vecs < 148.0 * 2048;
    unsigned tpr = pow2_at_least(few ? vecs : (vecs + in_flight(W) - 1) / in_flight(W));
    if (tpr > 256) tpr = 256;
    const long long per = 256 / tpr, want = (n + per - 1) / per, most = 0x7fffffff;
    embedding_forward_kernel<T, U, W><<<(unsigned)(want < most ? want : most), 256, 0, st>>>(out, ld_out, table, ld_table, vocab, dim, tokens, n, scale, (int)tpr);
    count_launch();
    B2_CUDA(cudaGetLastError());
    return B2_OK;
}

template <typename T, typename U, int W>
int sums(U *dtable, const T *dout, const SumArgs &base, const ZeroArgs &z, int zero_blocks, const int *tokens, const Plan &plan, unsigned *keys, cudaStream_t st) {
    SumArgs a = base;
    const int per_thread = 16 / (int)sizeof(T), P = W < 4 ? 4 : W;        // columns of a thread of the sums, and of the joins
    unsigned tpr = pow2_at_least((unsigned)((a.dim + per_thread - 1) / per_thread));
    tpr = tpr > SUM_THREADS ? SUM_THREADS : tpr < MIN_GROUP ? MIN_GROUP : tpr;
    a.tpr = (int)tpr;
    const unsigned cols = pow2_at_least((unsigned)((a.dim + P - 1) / P));
    a.cols = cols > 32 ? 32 : (int)cols;
    const long long tiles = (a.dim + (long long)tpr * per_thread - 1) / ((long long)tpr * per_thread), per = SUM_THREADS / tpr;
    const long long blocks = (a.pieces * tiles + per - 1) / per;
    if (a.n <= SMALL_SORT) {
        const int sort_bytes = (1 << plan.bits) * SORT_WARPS * 4, ring_bytes = W * sizeof(T) >= 4 ? AHEAD * SORT_THREADS * 16 : 0;
        const int smem = SMALL_WORDS * 4 + (sort_bytes > ring_bytes ? sort_bytes : ring_bytes);
        B2_TRY(set_max_dynamic_smem((const void *)embedding_small_kernel<T, U, W>, SMALL_WORDS * 4 + AHEAD * SORT_THREADS * 16));
        // as many blocks as have something to do, or as there are multiprocessors
        const long long units = (a.pieces * tiles * tpr + SORT_THREADS - 1) / SORT_THREADS, rows = ((long long)z.v1 - z.v0 + 4 * SORT_WARPS - 1) / (4 * SORT_WARPS);
        const long long want = units > rows ? units : rows;
        B2_TRY(launch_chained(embedding_small_kernel<T, U, W>, dim3((unsigned)(want < sm_count() ? want : sm_count())), dim3(SORT_THREADS), smem, st, dtable, dout, tokens, a, z,
                              plan.passes, plan.bits, keys));
    } else if (blocks + zero_blocks > 0x7fffffffll) { set_error("b2_embedding_backward: %lld blocks", blocks); return B2_ERR_BAD_SHAPE; }
    else B2_TRY(launch_chained(embedding_sum_kernel<T, U, W>, dim3((unsigned)(blocks + zero_blocks)), dim3(SUM_THREADS), 0, st, dtable, dout, a, z, (int)blocks, zero_blocks));
    const int join_tiles = (a.dim + a.cols * P - 1) / (a.cols * P), most = (sm_count() * 8 + join_tiles - 1) / join_tiles;
    return launch_chained(embedding_join_kernel<U, W>, dim3((unsigned)(a.pieces < most ? a.pieces : most), (unsigned)join_tiles), dim3(256), 0, st, dtable, a);
}

template <typename T, typename U>
int backward(U *dtable, long long ld_dtable, int vocab, int dim, const T *dout, long long ld_dout, const int *tokens, long long n, float scale, bool accumulate,
             char *ws, cudaStream_t st) {
    const Plan p = make_plan(n, vocab, dim);
    unsigned *present = (unsigned *)(ws + p.present), *count = (unsigned *)(ws + p.count), *keys[2] = {(unsigned *)(ws + p.keys[0]), (unsigned *)(ws + p.keys[1])};
    int *rows[2] = {(int *)(ws + p.rows[0]), (int *)(ws + p.rows[1])};
    ZeroArgs z = {dtable, (long long)dim * (long long)sizeof(U), ld_dtable * (long long)sizeof(U), present, 0, accumulate ? 0 : vocab, 16};
    while (z.unit > 2 && (z.row_bytes % z.unit || z.ld_bytes % z.unit || !aligned_to(dtable, z.unit))) z.unit = z.unit == 16 ? 4 : 2;
    int last = 0;
    if (n > SMALL_SORT) {
        B2_CUDA(cudaMemsetAsync(ws, 0, p.keys[0], st));                   // the list's length and the bits of the tokens that occur
        // rows that a launch of the sort zeroes besides: about as much as fits under its latency
        const long long share = (20ll << 20) / (z.row_bytes > 0 ? z.row_bytes : 1);
        SortArgs a = {tokens, nullptr, nullptr, nullptr, nullptr, (unsigned *)(ws + p.hist), present, count, (int)n, vocab, 0, p.bits, p.tiles, p.tile};
        const int digits = 1 << p.bits;
        const int rest = z.v1;
        for (int i = 0; i < p.passes; ++i) {
            a.shift = i * p.bits;
            a.kout = keys[i & 1]; a.rout = rows[i & 1];
            for (int half = 0; half < 2; ++half) {
                ZeroArgs zz = z;
                zz.v1 = z.v0;
                if (i || half) zz.v1 = (int)(z.v0 + share < rest ? z.v0 + share : rest);   // the first launch finds out which tokens occur
                const int zb = zz.v1 > zz.v0 ? 2 * sm_count() : 0;
                z.v0 = zz.v1;
                if (half == 0) B2_TRY(launch_chained(sort_count_kernel, dim3(p.tiles + zb), dim3(SORT_THREADS), digits * 4, st, a, zz));
                else B2_TRY(launch_chained(sort_scatter_kernel, dim3(p.tiles + zb), dim3(SORT_THREADS), digits * SORT_WARPS * 4, st, a, zz));
            }
            last = i & 1;
            a.tokens = nullptr;
            a.kin = a.kout; a.rin = a.rout;
        }
    }
    SumArgs a = {keys[last], rows[last], (float *)(ws + p.partial), n > SMALL_SORT ? (int *)(ws + p.list) : nullptr, count, ld_dout, ld_dtable, (int)n, vocab, dim, p.dim_pad, p.piece, p.pieces,
                 0, 0, accumulate ? 1 : 0, scale};
    const long long left = z.v1 - z.v0, zero_blocks = left > 0 ? (left + 3) / 4 < sm_count() * 16ll ? (left + 3) / 4 : sm_count() * 16ll : 0;
    const int w = common_width(16 / (int)sizeof(T), dim, dout, ld_dout, sizeof(T), dtable, ld_dtable, sizeof(U));
    if (w == 8) return sums<T, U, (16 / sizeof(T))>(dtable, dout, a, z, (int)zero_blocks, tokens, p, keys[0], st);
    if (w >= 4) return sums<T, U, 4>(dtable, dout, a, z, (int)zero_blocks, tokens, p, keys[0], st);
    if (w >= 2) return sums<T, U, 2>(dtable, dout, a, z, (int)zero_blocks, tokens, p, keys[0], st);
    return sums<T, U, 1>(dtable, dout, a, z, (int)zero_blocks, tokens, p, keys[0], st);
}

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" {

int b2_embedding_forward(void *out, int out_type, long long ld_out, const void *table, int table_type, long long ld_table, int vocab, int dim, const int *tokens_dev,
                         long long n, float scale, b2_stream stream) {
    if (bad_sizes("b2_embedding_forward", n, vocab, dim)) return B2_ERR_BAD_SHAPE;
    const int eo = type_size(out_type), et = type_size(table_type);
    if (!eo || !et) { set_error("b2_embedding_forward: unknown element type (output %d, table %d)", out_type, table_type); return B2_ERR_BAD_ARG; }
    if (ld_out < dim || ld_table < dim || ld_out > MAX_LD || ld_table > MAX_LD) {
        set_error("b2_embedding_forward: leading dimension too small or beyond 2^40 (output %lld, table %lld for %d columns)", ld_out, ld_table, dim);
        return B2_ERR_BAD_ARG;
    }
    if (!n) return B2_OK;
    if (!out || !table || !tokens_dev) { set_error("b2_embedding_forward: null pointer"); return B2_ERR_BAD_ARG; }
    if (!aligned_to(out, eo) || !aligned_to(table, et) || !aligned_to(tokens_dev, 4)) {
        set_error("b2_embedding_forward: an address is not aligned to its elements");
        return B2_ERR_BAD_ARG;
    }
    return with_type(table_type, [&](auto *t) {
        return with_type(out_type, [&](auto *o) {
            typedef B2_ELEM(t) T;
            typedef B2_ELEM(o) U;
            const int w = common_width(16 / (int)sizeof(T), dim, table, ld_table, et, out, ld_out, eo);
            const auto go = [&](auto width) {
                return forward<T, U, decltype(width)::value>((U *)out, ld_out, (const T *)table, ld_table, vocab, dim, tokens_dev, n, scale, (cudaStream_t)stream);
            };
            if (w == 8) return go(std::integral_constant<int, 16 / (int)sizeof(T)>());
            if (w >= 4) return go(std::integral_constant<int, 4>());
            if (w >= 2) return go(std::integral_constant<int, 2>());
            return go(std::integral_constant<int, 1>());
        });
    });
}

size_t b2_embedding_backward_workspace(long long n, int vocab, int dim) {
    if (n < 1 || bad_sizes("b2_embedding_backward_workspace", n, vocab, dim)) return 0;
    return make_plan(n, vocab, dim).total;
}

int b2_embedding_backward(void *dtable, int dtable_type, long long ld_dtable, int vocab, int dim, const void *dout, int dout_type, long long ld_dout,
                          const int *tokens_dev, long long n, float scale, int accumulate, void *workspace, size_t workspace_bytes, b2_stream stream) {
    if (bad_sizes("b2_embedding_backward", n, vocab, dim)) return B2_ERR_BAD_SHAPE;
    const int et = type_size(dtable_type), ed = type_size(dout_type);
    if (!et || !ed) { set_error("b2_embedding_backward: unknown element type (table %d, output errors %d)", dtable_type, dout_type); return B2_ERR_BAD_ARG; }
    if (ld_dtable < dim || ld_dout < dim || ld_dtable > MAX_LD || ld_dout > MAX_LD) {
        set_error("b2_embedding_backward: leading dimension too small or beyond 2^40 (table %lld, output errors %lld for %d columns)", ld_dtable, ld_dout, dim);
        return B2_ERR_BAD_ARG;
    }
    if (!dtable || !aligned_to(dtable, et)) { set_error("b2_embedding_backward: the table's gradient is missing or not aligned to its elements"); return B2_ERR_BAD_ARG; }
    if (!n) {
        if (!accumulate) B2_CUDA(cudaMemset2DAsync(dtable, (size_t)ld_dtable * et, 0, (size_t)dim * et, vocab, (cudaStream_t)stream));
        return B2_OK;
    }
    if (!dout || !tokens_dev || !workspace) { set_error("b2_embedding_backward: null pointer"); return B2_ERR_BAD_ARG; }
    if (!aligned_to(dout, ed) || !aligned_to(tokens_dev, 4) || !aligned_to(workspace, 256)) {
        set_error("b2_embedding_backward: an address is not aligned to its elements, or the workspace not to 256 bytes");
        return B2_ERR_BAD_ARG;
    }
    const size_t need = b2_embedding_backward_workspace(n, vocab, dim);
    if (workspace_bytes < need) { set_error("b2_embedding_backward: %zu bytes of workspace, %zu are needed", workspace_bytes, need); return B2_ERR_BAD_SHAPE; }
    return with_type(dout_type, [&](auto *d) {
        return with_type(dtable_type, [&](auto *t) {
            typedef B2_ELEM(d) T;
            typedef B2_ELEM(t) U;
            return backward<T, U>((U *)dtable, ld_dtable, vocab, dim, (const T *)dout, ld_dout, tokens_dev, n, scale, accumulate != 0, (char *)workspace,
                                  (cudaStream_t)stream);
        });
    });
}

}  // extern "C"
