// A step of beam search: the K best continuations of a sequence's beams over all tokens, and the beams' states by the beams that go on.
//
//   score(b, v) = score_b + z_bv - lse_b,  z = s * x where token v is allowed, -inf elsewhere;   rank = weight_b * score(b, v)
//
// Within a beam the ranks are in the order of z, so the K best of a beam are its K largest logits, and the beam's log sum is not needed to find them.
// First kernel: a block goes through a slice of a beam's row in chunks of 1024 vectors, each thread copying its own part of the next chunk into shared memory.  What the
// best lanes of every warp have reached is a bound that K entries pass, and hardly more do (16 of 8192: about 35); it is taken again after 1, 3, 7, ... chunks.  A
// vector whose largest entry reaches it is laid aside; in the end the entries that reach the bound of the whole slice are counted into their places.
// Second kernel, started while the first one drains: a block joins the sums and the lists of a sequence's beams, the ranks in 64 bits (scores of different
// beams meet, and 32 bits would make ties of what the beams' logits tell apart).
// The sums and their logarithms are fp32 ones, as everywhere here: good to 2^-22 or so, which is what decides between beams that are closer than that.
// Bound by instructions (18 an entry with a mask, 14 without, 5 of them for its exponential) and by the launches' latency.  Measured on a B200 (device time over the same buffers; in brackets a pass over
// buffers that change): 64 x 8 rows of 50001 bf16 with a mask, 16 continuations 32 us (35; the bytes' floor is 8), of that the second kernel 6 us; 4 rows of 32000 fp32 9.6 us (11.8), two launches.
// Slow are rows of one slice whose mask rules out their first tokens up to behind chunk 1 or 3: the bound stays at -inf until the next of the chunks after which it is taken again, so too many vectors are
// laid aside, and the slice is gone through once for each continuation (the same 64 x 8 rows without their first 20000 tokens 324 us).
// Reordering: 64 x 8 beams with 112 MB of states and frames 33 us for the copy there and back (6.8 TB/s).
#include <math.h>

#include <type_traits>

#include "logits.cuh"

namespace b2 {
namespace {

constexpr int MAX_BEAMS = 64, MAX_BEST = 64, MOST_VOCAB = 1 << 26;
constexpr int SLICE_THREADS = 256, SLICE_VECS = 4;        // threads of a slice, vectors of 16 bytes each has in registers
constexpr int CHUNK = SLICE_THREADS * SLICE_VECS;

typedef Sum Part;                    // of a slice

struct SelectArgs {
    const unsigned char *mask; long long ld_mask;
    const float *scores; const unsigned char *finished; const float *weights;
    long long groups, ld;
    int beams, vocab, top, end_token, slices, slice;     // slice: vectors of a slice
    float scale;
    Part *parts; Key *lists;                             // [row][slice], [row][slice][top]
    float *best; int *from, *tokens;
};
// whether beam `row` has continuations of its own (finished ones have their one without looking at the logits)
__device__ __forceinline__ bool runs(const SelectArgs &a, long long row) {
    const float s = a.scores[row], w = a.weights ? a.weights[row] : 1.0f;
    return s > neg_inf() && s < __int_as_float(0x7f800000) && w > 0.0f && w < __int_as_float(0x7f800000) && !(a.finished && a.finished[row]);
}

// bytes of x as the selector's digits tell; 8 and above: the sign of byte digit - 8, all over
template <unsigned S> __device__ __forceinline__ unsigned signs(unsigned x) { unsigned y; asm("prmt.b32 %0, %1, 0, %2;" : "=r"(y) : "r"(x), "n"(S)); return y; }
// The mask's bytes of a vector's entries, in words: as an array of bytes they would be taken apart and put together again
template <typename T> struct Flags { unsigned w[4 / sizeof(T)]; };
// -inf in the places of q whose bytes are 0
template <typename T> __device__ __forceinline__ void rule_out(uint4 &q, const Flags<T> &on) {
    unsigned w[4] = {q.x, q.y, q.z, q.w}, s[2] = {0, 0}, keep[4];      // keep: a sign all over an entry's bytes
#pragma unroll
    for (int i = 0; i < 4 / (int)sizeof(T); ++i) s[i] = ((on.w[i] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | on.w[i];     // the sign of a byte that is not 0
    if constexpr (sizeof(T) == 4) {
        keep[0] = signs<0x8888>(s[0]); keep[1] = signs<0x9999>(s[0]); keep[2] = signs<0xaaaa>(s[0]); keep[3] = signs<0xbbbb>(s[0]);
    } else {
        keep[0] = signs<0x9988>(s[0]); keep[1] = signs<0xbbaa>(s[0]); keep[2] = signs<0x9988>(s[1]); keep[3] = signs<0xbbaa>(s[1]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (w[i] & keep[i]) | (Raw<T>::NONE & ~keep[i]);
    q = make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T> __device__ __forceinline__ Flags<T> load_flags(const unsigned char *m) {
    Flags<T> f;
    if constexpr (sizeof(T) == 4) f.w[0] = *reinterpret_cast<const unsigned *>(m);
    else {
        const uint2 v = *reinterpret_cast<const uint2 *>(m);
        f.w[0] = v.x;
        f.w[1] = v.y;
    }
    return f;
}

// What the `rounds` best lanes of a warp hold at least: rounds * warps entries reach the least of it over the warps
__device__ __forceinline__ unsigned reached(unsigned best, int rounds) {
    unsigned least = 0;
    for (int i = 0; i < rounds; ++i) {
        least = __reduce_max_sync(FULL, best);
        if ((int)(threadIdx.x & 31) == __ffs(__ballot_sync(FULL, best == least)) - 1) best = 0;
    }
    return least;
}
// the least over the first `warps` of 8
__device__ __forceinline__ unsigned least_of(const unsigned *bounds, int warps) { return __reduce_min_sync(FULL, bounds[min((int)(threadIdx.x & 31), warps - 1)]); }

template <typename T, bool MASK>
__global__ void __launch_bounds__(SLICE_THREADS, 4) beam_rows_kernel(const T *logits, const SelectArgs a) {
    constexpr int THREADS = SLICE_THREADS, W = 16 / sizeof(T), U = SLICE_VECS, WARPS = THREADS / 32, CAP = 512;
    __shared__ unsigned bounds[WARPS];
    __shared__ Part parts[WARPS];
    __shared__ uint4 ring[2][U][THREADS];
    __shared__ __align__(16) T hits[CAP][W];            // vectors that hold an entry of interest
    __shared__ int hit_at[CAP];                           // where they are in the row
    __shared__ Key found[CAP], winner[WARPS];
    __shared__ int n_hits, count;
    grid_release();
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const long long row = a.slices == 1 ? blockIdx.x : blockIdx.x / (unsigned)a.slices;
    const int part = a.slices == 1 ? 0 : (int)(blockIdx.x % (unsigned)a.slices);
    const T *x = logits + row * a.ld;
    const int mis = (int)(((uintptr_t)x & 15) / sizeof(T));
    const unsigned char *mk = MASK ? a.mask + row * a.ld_mask : nullptr;
    const bool mask_vec = MASK && ((uintptr_t)(mk - mis) & (W - 1)) == 0;
    const int v0 = part * a.slice, v1 = min(v0 + a.slice, (mis + a.vocab + W - 1) / W);
    if (t == 0) n_hits = count = 0;
    // A thread copies the vectors of its next chunk into shared memory while it works on one, for itself alone; their mask's bytes wait in registers
    Flags<T> on[MASK ? U : 1], on_next[MASK ? U : 1];
    const auto whole = [&](int v) { return v < v1 && v * W >= mis && (v + 1) * W - mis <= a.vocab; };
    // most chunks lie inside their row, and need no tests
    const auto inside = [&](int from) { return from * W >= mis && (from + CHUNK) * W - mis <= a.vocab && from + CHUNK <= v1 && (!MASK || mask_vec); };
    const T *const x_here = x - mis + t * W;
    const unsigned char *const mk_here = MASK ? mk - mis + t * W : nullptr;
    const unsigned ring_here = (unsigned)__cvta_generic_to_shared(&ring[0][0][t]);
    const auto ahead = [&](int from, int to) {
        const unsigned at = ring_here + to * (U * THREADS * 16);
        if (inside(from)) {
            const T *src = x_here + from * W;
#pragma unroll
            for (int u = 0; u < U; ++u) cp_async<16>(at + u * (THREADS * 16), src + u * (THREADS * W));
            if (MASK)
#pragma unroll
                for (int u = 0; u < U; ++u) on_next[u] = load_flags<T>(mk_here + (from + u * THREADS) * W);
            cp_commit();
            return;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int v = from + t + u * THREADS;
            if (!whole(v)) continue;
            cp_async<16>(at + u * (THREADS * 16), x - mis + v * W);
            if (MASK && mask_vec) on_next[u] = load_flags<T>(mk - mis + v * W);
        }
        cp_commit();
    };
    Part sum = {neg_inf(), 0.0f};
    float best = neg_inf(), limit = neg_inf();             // the thread's largest; what an entry has to reach
    // warps full of vectors, and the lanes of each that hold `top` entries together (more than 32: too few entries for a bound)
    const int warps = min(WARPS, (v1 - v0) / 32), rounds = warps > 0 ? (a.top + warps - 1) / warps : 33;
    int renew = 0, chunk = 0;
    ahead(v0, 0);
    if (!runs(a, row)) {                                   // asked while the logits are on the way
        cp_wait<0>();
        return;
    }
    if (rounds > 32) __syncthreads();                      // n_hits is set; else the first bound's barrier comes before the first hit
    for (int from = v0; from < v1; from += THREADS * U, ++chunk) {
        if (MASK)
#pragma unroll
            for (int u = 0; u < U; ++u) on[u] = on_next[u];
        ahead(from + THREADS * U, (chunk + 1) & 1);
        cp_wait<1>();
        uint4 q[U];
        if (inside(from)) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                q[u] = ring[chunk & 1][u][t];
                if (MASK) rule_out<T>(q[u], on[u]);
            }
        } else
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int v = from + t + u * THREADS;
            if (whole(v)) {
                q[u] = ring[chunk & 1][u][t];
                if (MASK && mask_vec) rule_out<T>(q[u], on[u]);
            } else q[u] = make_uint4(Raw<T>::NONE, Raw<T>::NONE, Raw<T>::NONE, Raw<T>::NONE);
        }
        // the ends of the row, and masks whose bytes lie across the vectors: entry by entry, through this thread's place in the ring
        if ((MASK && !mask_vec) || from * W < mis || (from + THREADS * U) * W - mis > a.vocab) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int v = from + t + u * THREADS, i0 = v * W - mis;
                if (v >= v1 || (whole(v) && !(MASK && !mask_vec))) continue;
                T *const mine = reinterpret_cast<T *>(&ring[chunk & 1][u][t]);
#pragma unroll 1
                for (int j = 0; j < W; ++j) {
                    const int i = i0 + j;
                    if (i < 0 || i >= a.vocab || (MASK && !mk[i])) mine[j] = from_float<T>(neg_inf());
                    else if (!whole(v)) mine[j] = x[i];
                }
                q[u] = ring[chunk & 1][u][t];
            }
        }
        unsigned big[U];
#pragma unroll
        for (int u = 0; u < U; ++u) big[u] = larger_of<T>(q[u]);
        unsigned biggest = big[0];
#pragma unroll
        for (int u = 1; u < U; ++u) biggest = Raw<T>::larger(biggest, big[u]);
        const float mine = __fmul_rn(Raw<T>::largest(biggest), a.scale);
        best = max_nan(best, mine);
        if (chunk == renew) {
            // the bound from what was met so far, after 1, 2, 4, 8, ... chunks
            if (rounds <= 32) {
                const unsigned mine_reached = reached(ordered(best), rounds);
                if (chunk) __syncthreads();
                if (lane == 0) bounds[warp] = mine_reached;
                __syncthreads();
                limit = ordered_value(least_of(bounds, warps));
            }
            renew = 2 * renew + 1;
        }
        if (mine >= limit && mine > neg_inf())
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (__fmul_rn(Raw<T>::largest(big[u]), a.scale) >= limit) {
                    const int at = atomicAdd(&n_hits, 1);
                    if (at < CAP) {
                        *reinterpret_cast<uint4 *>(&hits[at][0]) = q[u];
                        hit_at[at] = (from + t + u * THREADS) * W - mis;
                    }
                }
        if (!(mine <= sum.m)) rise(sum, mine);
        if (sum.m != neg_inf()) {
            const Pair l2 = pair(LOG2E, LOG2E);
            Pair p = 0;
            less_of_type<T>(a.scale, sum.m, [&](const auto &less) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    float z[W];
                    Raw<T>::values(z, q[u]);
#pragma unroll
                    for (int j = 0; j < W; j += 2) {
                        const float2 d = halves(mul2(less(z[j], z[j + 1]), l2));
                        p = add2(p, pair(ex2(d.x), ex2(d.y)));
                    }
                }
            });
            const float2 h = halves(p);
            sum.s += h.x + h.y;
        }
    }
    sum = team_join<32>(sum);
    const unsigned all_reached = chunk > 1 && rounds <= 32 ? reached(ordered(best), rounds) : 0;         // the bound of the whole slice
    if (lane == 0) parts[warp] = sum;
    __syncthreads();
    if (chunk > 1 && rounds <= 32) {
        if (lane == 0) bounds[warp] = all_reached;
        __syncthreads();
        limit = ordered_value(least_of(bounds, warps));
    }
    Key *const list = a.lists + (row * a.slices + part) * a.top;
    const int h = n_hits;
    if (h <= CAP)
        for (int i = t; i < h * W; i += THREADS) {
            const float z = __fmul_rn(to_float(hits[i / W][i % W]), a.scale);
            if (z >= limit && z > neg_inf()) {
                const int at = atomicAdd(&count, 1);
                if (at < CAP) found[at] = make_key(z, hit_at[i / W] + i % W);
            }
        }
    if (warp == WARPS - 1) {
        Part all = lane < WARPS ? parts[lane] : Part{neg_inf(), 0.0f};
        all = team_join<WARPS>(all);
        if (lane == 0) a.parts[row * a.slices + part] = all;
    }
    __syncthreads();
    const int n = count;
    if (h <= CAP && n <= CAP) {
        for (int i = t; i < n; i += THREADS) {
            const Key k = found[i];
            int before = 0;
#pragma unroll 4
            for (int j = 0; j < n; ++j) before += found[j] > k;
            if (before < a.top) list[before] = k;
        }
        for (int i = n + t; i < a.top; i += THREADS) list[i] = 0;
        return;
    }
    // many that reach the bound, as in a row of equal logits: the next best in turn
    const int i0 = max(v0 * W - mis, 0), i1 = min(v1 * W - mis, a.vocab);
    Key last = ~0ull;
    for (int i = 0; i < a.top; ++i) {
        Key k = 0;
        for (int e = i0 + t; e < i1; e += THREADS) {
            const float z = __fmul_rn(to_float(x[e]), a.scale);
            if (!(z >= limit) || z == neg_inf() || (MASK && !mk[e])) continue;
            const Key c = make_key(z, e);
            if (c < last && c > k) k = c;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const Key other = __shfl_xor_sync(FULL, k, o);
            if (other > k) k = other;
        }
        if (lane == 0) winner[warp] = k;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WARPS; ++w)
            if (winner[w] > k) k = winner[w];
        if (t == 0) list[i] = k;
        last = k;
        __syncthreads();
    }
}

// A continuation in the order of ranks: the rank, then beam (lower first), logit (larger), token (lower) in one word
struct Cand { double rank; unsigned long long tie; };
__device__ __forceinline__ bool better(const Cand &a, const Cand &b) { return a.rank > b.rank || (a.rank == b.rank && a.tie > b.tie); }
__device__ __forceinline__ Cand no_cand() { return {-INFINITY, 0}; }
__device__ __forceinline__ unsigned long long tie_of(int beam, float z, int token) {
    return ((unsigned long long)(MAX_BEAMS - 1 - beam) << 58) | ((unsigned long long)ordered(z) << 26) | (unsigned)(MOST_VOCAB - 1 - token);
}
__device__ __forceinline__ int beam_of(unsigned long long tie) { return MAX_BEAMS - 1 - (int)(tie >> 58); }
__device__ __forceinline__ float logit_of(unsigned long long tie) { return ordered_value((unsigned)(tie >> 26)); }
__device__ __forceinline__ int token_of(unsigned long long tie) { return MOST_VOCAB - 1 - (int)(tie & (MOST_VOCAB - 1)); }

// One block a sequence.  A bound from the threads' best entries first, as above; where beams of different strength let too many pass, the one that the K best reach is found
// digit by digit, from the counts of the ranks' digits in 32 bits (a rounding to fewer bits keeps the order, so that whatever reaches the bound in 64 bits
// reaches it in 32).  The entries that reach it are counted into their places.
constexpr int JOIN_THREADS = 256, DIGIT_BITS = 11, DIGITS = 1 << DIGIT_BITS, MOST_FOUND = 512, MOST_ENTRIES = 64 * MAX_BEST;
__global__ void __launch_bounds__(JOIN_THREADS) beam_join_kernel(const SelectArgs a) {
    __shared__ double off[MAX_BEAMS], weight[MAX_BEAMS];
    __shared__ bool ended[MAX_BEAMS];
    __shared__ int counts[DIGITS], warp_counts[JOIN_THREADS / 32];
    __shared__ unsigned ranks[MOST_ENTRIES], bounds[JOIN_THREADS / 32];      // the entries' ranks as ordered integers, 0: none
    __shared__ Cand found[MOST_FOUND];
    __shared__ __align__(16) unsigned orders[MOST_FOUND];                        // the same entries' ranks as ordered integers
    __shared__ int digit, left, reach, count;
    __shared__ Cand winner[JOIN_THREADS / 32];
    constexpr int WARPS = JOIN_THREADS / 32, EACH = DIGITS / JOIN_THREADS;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const long long g = blockIdx.x;
    const int lists = a.beams * a.slices, entries = lists * a.top;
    const Key *const keys = a.lists + g * entries;
    grid_wait();
    const Key first = t < entries ? keys[t] : 0;             // on the way while the sums are joined
    // score_b - lse_b of the beams; NaN: no continuations
    for (int b = warp; b < a.beams; b += WARPS) {
        const long long row = g * a.beams + b;
        const float score = a.scores[row], w = a.weights ? a.weights[row] : 1.0f;
        const bool end = a.finished && a.finished[row];
        const Part mine = lane < a.slices ? a.parts[row * a.slices + lane] : Part{neg_inf(), 0.0f};      // (what stands there for a beam at its end is not used)
        const bool fit = score > neg_inf() && score < __int_as_float(0x7f800000) && w > 0.0f && w < __int_as_float(0x7f800000);
        double o = nan("");
        if (fit && end) o = (double)score;
        else if (fit) {
            float m = mine.m;
            for (int i = lane + 32; i < a.slices; i += 32) m = max_nan(m, a.parts[row * a.slices + i].m);
#pragma unroll
            for (int x = 16; x > 0; x >>= 1) m = max_nan(m, __shfl_xor_sync(FULL, m, x));
            // a slice's sum has the error of 32 bits already: the factors need no more
            double s = mine.m != neg_inf() ? (double)(mine.s * expf(mine.m - m)) : 0.0;
            for (int i = lane + 32; i < a.slices; i += 32) {
                const Part p = a.parts[row * a.slices + i];
                if (p.m != neg_inf()) s += (double)(p.s * expf(p.m - m));
            }
            s = warp_sum(s);
            o = m == neg_inf() ? nan("") : (double)score - (double)m - log(s);
        }
        if (lane == 0) { off[b] = o; weight[b] = (double)w; ended[b] = end; }
    }
    if (t == 0) { count = 0; left = a.top; }
    __syncthreads();
    // entry i, the i % top th of a list
    const unsigned per_top = a.top > 1 ? 0xffffffffu / (unsigned)a.top + 1 : 0;
    const auto cand = [&](int i, Key k) -> Cand {
        const int l = a.top > 1 ? (int)__umulhi((unsigned)i, per_top) : i, b = a.slices == 1 ? l : l / a.slices;
        const double o = off[b];
        if (o != o) return no_cand();
        if (ended[b]) return i == b * a.slices * a.top ? Cand{weight[b] * o, tie_of(b, 0.0f, a.end_token)} : no_cand();
        if (!k) return no_cand();
        const float z = key_value(k);
        return {weight[b] * (o + (double)z), tie_of(b, z, key_index(k))};
    };
    unsigned best = 0;
#pragma unroll 1
    for (int i = t; i < entries; i += JOIN_THREADS) {
        const Cand c = cand(i, i == t ? first : keys[i]);
        const unsigned k = c.tie ? ordered((float)c.rank) : 0;
        ranks[i] = k;
        best = max(best, k);
    }
    const auto for_all = [&](auto &&f) {
        for (int i = t; i < entries; i += JOIN_THREADS)
            if (ranks[i]) f(i, ranks[i]);
    };
    const int full = min(entries, JOIN_THREADS) / 32, rounds = full > 0 ? (a.top + full - 1) / full : 33;
    unsigned guess = 0;
    if (rounds <= 32) {
        const unsigned mine = reached(best, rounds);
        if (lane == 0) bounds[warp] = mine;
        __syncthreads();
        guess = least_of(bounds, full);
    }
    int passed = 0;
    for_all([&](int, unsigned k) { passed += k >= guess; });
    passed = __reduce_add_sync(FULL, passed);
    if (lane == 0) warp_counts[warp] = passed;
    __syncthreads();
    passed = __reduce_add_sync(FULL, lane < WARPS ? warp_counts[lane] : 0);
    // counting 160 entries into their places takes as long as finding two digits
    const bool enough = passed <= max(160, 2 * a.top + 32);
    unsigned bound = enough ? guess : 0;                       // or the digits found so far, and zeros
#pragma unroll 1
    for (int shift = enough ? -1 : 32 - DIGIT_BITS; shift >= 0;) {
        for (int i = t; i < DIGITS; i += JOIN_THREADS) counts[i] = 0;
        __syncthreads();
        if (t == 0) digit = -1;                              // all have taken the one before
        const int want = left;                               // before the barriers behind which it is written
        const int above = shift ? shift + DIGIT_BITS : 32 % DIGIT_BITS;      // the last digit has the bits that are left
        for_all([&](int, unsigned k) {
            if (above >= 32 || k >> above == bound >> above) atomicAdd(&counts[(k >> shift) & ((1u << (above - shift)) - 1)], 1);
        });
        __syncthreads();
        // the digits in falling order, EACH a thread: the one with which `left` entries are reached
        int mine[EACH], sum = 0;
#pragma unroll
        for (int i = 0; i < EACH; ++i) sum += mine[i] = counts[DIGITS - 1 - (t * EACH + i)];
        int before = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(FULL, before, o);
            if (lane >= o) before += x;
        }
        if (lane == 31) warp_counts[warp] = before;
        __syncthreads();
        before -= sum;
        for (int w = 0; w < warp; ++w) before += warp_counts[w];
        if (before < want && want <= before + sum) {
            int at = before;
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                if (at < want && want <= at + mine[i]) {
                    digit = DIGITS - 1 - (t * EACH + i);
                    reach = a.top - want + at + mine[i];             // all that reach the bound with this digit
                    left = want - at;
                }
                at += mine[i];
            }
        }
        __syncthreads();
        if (digit < 0) break;                                // fewer than `top` altogether: all of them
        bound |= (unsigned)digit << shift;
        if (shift == 0 || reach <= 2 * a.top) break;
        shift = max(0, shift - DIGIT_BITS);
    }
    for_all([&](int i, unsigned k) {
        if (k >= bound) {
            const int at = atomicAdd(&count, 1);
            if (at < MOST_FOUND) {
                found[at] = cand(i, keys[i]);
                orders[at] = k;
            }
        }
    });
    __syncthreads();
    const auto write = [&](int place, const Cand &c) {
        const long long i = g * a.top + place;
        const bool none = c.tie == 0;
        const int b = none ? 0 : beam_of(c.tie);
        a.best[i] = none ? neg_inf() : ended[b] ? (float)off[b] : (float)(off[b] + (double)logit_of(c.tie));
        a.from[i] = none ? -1 : b;
        a.tokens[i] = none ? -1 : token_of(c.tie);
    };
    const int n = count;
    if (n <= MOST_FOUND) {
        // in 32 bits, and in 64 where those are equal
        if (t < -n % 4 + 4 && n + t < MOST_FOUND) orders[n + t] = 0;
        __syncthreads();
        for (int i = t; i < n; i += JOIN_THREADS) {
            const unsigned mine = orders[i];
            int before = 0;
            for (int j = 0; j < n; j += 4) {
                const uint4 k = *reinterpret_cast<const uint4 *>(&orders[j]);
                before += (k.x > mine) + (k.y > mine) + (k.z > mine) + (k.w > mine);
                if (k.x == mine || k.y == mine || k.z == mine || k.w == mine)
                    for (int e = j; e < min(n, j + 4); ++e) before += orders[e] == mine && better(found[e], found[i]);
            }
            if (before < a.top) write(before, found[i]);
        }
        for (int i = n + t; i < a.top; i += JOIN_THREADS) write(i, no_cand());
        return;
    }
    // many equal ranks: the next best in turn
    Cand last = {INFINITY, ~0ull};
    for (int place = 0; place < a.top; ++place) {
        Cand top = no_cand();
        for_all([&](int i, unsigned) {
            const Cand c = cand(i, keys[i]);
            if (better(last, c) && better(c, top)) top = c;
        });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const Cand other = {__shfl_xor_sync(FULL, top.rank, o), __shfl_xor_sync(FULL, top.tie, o)};
            if (better(other, top)) top = other;
        }
        if (lane == 0) winner[warp] = top;
        __syncthreads();
        for (int w = 0; w < WARPS; ++w)
            if (better(winner[w], top)) top = winner[w];
        if (t == 0) write(place, top);
        last = top.tie != 0 ? top : no_cand();
        __syncthreads();
    }
}

int vectors_of(int vocab, int type) { const int w = 16 / type_size(type); return (vocab + w - 1) / w + 1; }   // one more: a row may start inside a vector
// Slices of a row, of whole chunks of 1024 vectors: one where the rows fill the device (bounds and lists cost a slice several chunks' time), more where they do not
// (and 64 lists for a sequence at most, which the second kernel goes through)
int slices_of(long long rows, int beams, int vocab, int type) {
    const int chunks = (vectors_of(vocab, type) + CHUNK - 1) / CHUNK;
    // blocks that run at a time: 4 on each of 148 SMs.  A number, so that the workspace has the same size wherever it is asked for
    long long most = rows && rows < 592 ? 592 / rows : 1;
    if (most > 64 / beams) most = 64 / beams;
    const int each = (int)((chunks + most - 1) / most);
    return (chunks + each - 1) / each;
}

template <typename T> int select(const T *logits, SelectArgs a, int type, cudaStream_t st) {
    const int chunks = (vectors_of(a.vocab, type) + CHUNK - 1) / CHUNK;
    a.slice = (chunks + a.slices - 1) / a.slices * CHUNK;
    const long long blocks = a.groups * a.beams * a.slices;
    if (blocks > 0x7fffffffll) { set_error("b2_beam_select: %lld rows of %d", a.groups * a.beams, a.vocab); return B2_ERR_BAD_SHAPE; }
    if (a.mask) beam_rows_kernel<T, true><<<(unsigned)blocks, SLICE_THREADS, 0, st>>>(logits, a);
    else beam_rows_kernel<T, false><<<(unsigned)blocks, SLICE_THREADS, 0, st>>>(logits, a);
    count_launch();
    B2_CUDA(cudaGetLastError());
    return launch_chained(beam_join_kernel, dim3((unsigned)a.groups), dim3(JOIN_THREADS), 0, st, a);
}

bool sizes_fit(long long groups, int beams, int vocab, int top) {
    return groups >= 0 && groups <= 0x7fffffff / MAX_BEAMS && beams >= 1 && beams <= MAX_BEAMS && vocab >= 1 && vocab <= MOST_VOCAB && top >= 1 && top <= MAX_BEST;
}

// ---- reordering -----------------------------------------------------------------------------------------------------------------------
constexpr int MAX_STATES = 32;       // of a launch; more take several
struct StateArgs {
    b2_state s[MAX_STATES];
    int n, beams;
    long long groups;
    const int *parents;
    unsigned first[MAX_STATES + 1];  // of the blocks of tensor i
};
// A thread moves a column of N bytes (of the same place in a sequence's beams) for all beams of a sequence: it alone reads and writes it, so that a state may
// be reordered in place without a barrier.  HELD beams at a time are in registers; in place all are (narrower columns then, if there are more than MOST_HELD).
template <int N> struct Bytes;
template <> struct Bytes<16> { typedef uint4 T; };
template <> struct Bytes<8> { typedef uint2 T; };
template <> struct Bytes<4> { typedef unsigned T; };
template <> struct Bytes<2> { typedef unsigned short T; };
template <> struct Bytes<1> { typedef unsigned char T; };
template <typename V> __device__ __forceinline__ V zero_of() { V v; memset(&v, 0, sizeof(V)); return v; }

constexpr int MOVE_THREADS = 128, MOST_HELD = 16;
template <int N, int HELD> __device__ __forceinline__ void move(const b2_state &s, const int *parent, int beams, long long base) {
    typedef typename Bytes<N>::T V;
    const char *in = (const char *)s.data + base;
    char *out = (char *)s.out + base;
    const bool place = s.data == s.out;
    for (int b0 = 0; b0 < beams; b0 += HELD) {
        V v[HELD];
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            if (b0 + i >= beams) break;
            const int p = parent[b0 + i];
            v[i] = p < 0 || (place && p == b0 + i) ? zero_of<V>() : *reinterpret_cast<const V *>(in + p * s.row_bytes);
        }
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            if (b0 + i >= beams) break;
            if (!(place && parent[b0 + i] == b0 + i)) *reinterpret_cast<V *>(out + (b0 + i) * s.row_bytes) = v[i];
        }
    }
}
// Narrow rows (tokens so far, say): the beams of a sequence and outer index are up to ITEMS pieces of each of `team` lanes, next to each other in memory.  A lane has its own of
// BATCH outer indices in registers before any is written.
constexpr int SMALL = 4;
template <int ITEMS> struct Batch { static constexpr int N = ITEMS == 1 ? 8 : 2; };
template <int N, int ITEMS>
__device__ __forceinline__ void move_small(const b2_state &s, const int *parent, int beams, int columns, int team, long long chunk, long long groups, unsigned group) {
    typedef typename Bytes<N>::T V;
    constexpr int BATCH = Batch<ITEMS>::N;
    const int lane = (int)threadIdx.x & (team - 1), pieces = beams * columns, step = MOVE_THREADS / team;
    const long long row = beams * s.row_bytes, first = chunk * (step * BATCH) + threadIdx.x / team;
    long long from[ITEMS];                 // where a piece comes from, -1: zeros
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int k = lane + i * team, b = min(k, pieces - 1) / columns, p = parent[b];
        from[i] = p < 0 ? -1 : p * s.row_bytes + (long long)(k - b * columns) * N;
    }
    V v[BATCH][ITEMS];
#pragma unroll
    for (int e = 0; e < BATCH; ++e) {
        const long long o = first + e * step;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            if (o < s.outer && lane + i * team < pieces)
                v[e][i] = from[i] < 0 ? zero_of<V>() : *reinterpret_cast<const V *>((const char *)s.data + (o * groups + group) * row + from[i]);
    }
    __syncwarp();
#pragma unroll
    for (int e = 0; e < BATCH; ++e) {
        const long long o = first + e * step;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
            if (o < s.outer && lane + i * team < pieces) *reinterpret_cast<V *>((char *)s.out + (o * groups + group) * row + (long long)(lane + i * team) * N) = v[e][i];
    }
}
// How a tensor is moved.  width: bytes of a column or piece, what the addresses and the rows allow, and 4 where more than MOST_HELD beams have to be in registers at once.
// team: lanes of a sequence and outer index with narrow rows, else 0; batch: outer indices of each
struct Way { int width, team, batch; };
__host__ __device__ __forceinline__ Way way_of(const b2_state &s, int beams) {
    const unsigned long long at = ((uintptr_t)s.data | (uintptr_t)s.out | (uintptr_t)s.row_bytes) & 15;
    int width = at == 0 ? 16 : at & 1 ? 1 : at & 2 ? 2 : at & 4 ? 4 : 8;
    const long long pieces = s.row_bytes / width * beams;
    if (pieces <= 32 * SMALL) {
        int team = 1;
        while (team < 32 && team < pieces) team *= 2;
        return {width, team, pieces <= team ? Batch<1>::N : Batch<SMALL>::N};
    }
    if (s.data == s.out && beams > MOST_HELD && width > 4) width = 4;
    return {width, 0, 0};
}
// a block's threads have columns of one sequence, those of all outer indices one after the other
template <int HELD> __global__ void __launch_bounds__(MOVE_THREADS) beam_reorder_kernel(const __grid_constant__ StateArgs a) {
    __shared__ int parent[MAX_BEAMS];
    int i = 0;
    while (i + 1 < a.n && blockIdx.x >= a.first[i + 1]) ++i;
    const b2_state &s = a.s[i];
    const Way way = way_of(s, a.beams);
    const int width = way.width;
    const unsigned groups = (unsigned)a.groups, k = blockIdx.x - a.first[i], group = k % groups;     // blocks of a tensor: [chunk][group]
    if ((int)threadIdx.x < a.beams) {
        const int p = a.parents[(long long)group * a.beams + threadIdx.x];
        parent[threadIdx.x] = p >= 0 && p < a.beams ? p : -1;
    }
    if (way.team) {
        const int columns = (int)(s.row_bytes / width);
        __syncthreads();
        const auto go = [&](auto bytes) {
            constexpr int N = decltype(bytes)::value;
            if (columns * a.beams <= way.team) move_small<N, 1>(s, parent, a.beams, columns, way.team, k / groups, a.groups, group);
            else move_small<N, SMALL>(s, parent, a.beams, columns, way.team, k / groups, a.groups, group);
        };
        switch (width) {
            case 16: return go(std::integral_constant<int, 16>());
            case 8: return go(std::integral_constant<int, 8>());
            case 4: return go(std::integral_constant<int, 4>());
            case 2: return go(std::integral_constant<int, 2>());
            default: return go(std::integral_constant<int, 1>());
        }
    }
    const long long columns = s.row_bytes / width, at = (long long)(k / groups) * MOVE_THREADS + threadIdx.x;
    long long o, column;
    if (columns * s.outer <= 0x7fffffff) {
        o = (unsigned)at / (unsigned)columns;
        column = (unsigned)at % (unsigned)columns;
    } else {
        o = at / columns;
        column = at % columns;
    }
    __syncthreads();
    if (o >= s.outer) return;
    const long long base = (o * a.groups + group) * a.beams * s.row_bytes + column * width;
    if (HELD <= MOST_HELD && width == 16) return move<16, HELD <= MOST_HELD ? HELD : 1>(s, parent, a.beams, base);
    if (HELD <= MOST_HELD && width == 8) return move<8, HELD <= MOST_HELD ? HELD : 1>(s, parent, a.beams, base);
    if (width == 4) return move<4, HELD>(s, parent, a.beams, base);
    if (width == 2) return move<2, HELD>(s, parent, a.beams, base);
    return move<1, HELD>(s, parent, a.beams, base);
}

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" {

size_t b2_beam_select_workspace(long long groups, int beams, int vocab, int top) {
    if (!sizes_fit(groups, beams, vocab, top)) return 0;
    const int wide = slices_of(groups * beams, beams, vocab, B2_F32), narrow = slices_of(groups * beams, beams, vocab, B2_BF16);
    const size_t slices = (size_t)(wide > narrow ? wide : narrow) * (size_t)groups * beams;      // the most of any type
    return slices * (sizeof(Part) + (size_t)top * sizeof(Key));
}

int b2_beam_select(const void *logits, int type, long long groups, int beams, int vocab, long long ld, const unsigned char *mask, long long ld_mask, float scale,
                   const float *scores, const unsigned char *finished, const float *weights, int end_token, int top, float *top_scores, int *top_beams, int *top_tokens,
                   void *workspace, size_t workspace_bytes, b2_stream stream) {
    const int e = type_size(type);
    if (!e) { set_error("b2_beam_select: unknown element type %d", type); return B2_ERR_BAD_ARG; }
    if (!sizes_fit(groups, beams, vocab, top)) {
        set_error("b2_beam_select: %lld sequences, %d beams (1 to %d), %d logits (at most 2^26), %d continuations (1 to %d)", groups, beams, MAX_BEAMS, vocab, top, MAX_BEST);
        return B2_ERR_BAD_SHAPE;
    }
    if (ld < vocab || ld > MAX_LD || (mask && ((ld_mask != 0 && ld_mask < vocab) || ld_mask > MAX_LD))) {
        set_error("b2_beam_select: leading dimension too small or beyond 2^40 (logits %lld, mask %lld for %d columns)", ld, ld_mask, vocab);
        return B2_ERR_BAD_ARG;
    }
    if (!(scale > 0.0f) || scale > 3.402823466e38f) { set_error("b2_beam_select: the scale %g is not a positive number", (double)scale); return B2_ERR_BAD_ARG; }
    if (finished && (end_token < 0 || end_token >= vocab)) { set_error("b2_beam_select: end_token %d of %d", end_token, vocab); return B2_ERR_BAD_ARG; }
    if (!groups) return B2_OK;
    if (!logits || !aligned_to(logits, e)) { set_error("b2_beam_select: the logits are missing or not aligned to their elements"); return B2_ERR_BAD_ARG; }
    if (!scores || !top_scores || !top_beams || !top_tokens || !workspace) { set_error("b2_beam_select: null pointer"); return B2_ERR_BAD_ARG; }
    if (!aligned_to(scores, 4) || !aligned_to(weights, 4) || !aligned_to(top_scores, 4) || !aligned_to(top_beams, 4) || !aligned_to(top_tokens, 4)) {
        set_error("b2_beam_select: a vector of tokens or numbers is not aligned to 4 bytes");
        return B2_ERR_BAD_ARG;
    }
    if (!aligned_to(workspace, 16)) { set_error("b2_beam_select: the workspace is not aligned to 16 bytes"); return B2_ERR_BAD_ARG; }
    const size_t need = b2_beam_select_workspace(groups, beams, vocab, top);
    if (workspace_bytes < need) { set_error("b2_beam_select: a workspace of %zu bytes, %zu are needed", workspace_bytes, need); return B2_ERR_BAD_SHAPE; }
    SelectArgs a = {};
    a.mask = mask; a.ld_mask = ld_mask; a.scores = scores; a.finished = finished; a.weights = weights;
    a.groups = groups; a.ld = ld; a.beams = beams; a.vocab = vocab; a.top = top; a.end_token = end_token; a.scale = scale;
    a.slices = slices_of(groups * beams, beams, vocab, type);
    a.lists = (Key *)workspace;
    a.parts = (Part *)(a.lists + (size_t)a.slices * (size_t)groups * beams * top);
    a.best = top_scores; a.from = top_beams; a.tokens = top_tokens;
    return with_type(type, [&](auto *t) { return select((const B2_ELEM(t) *)logits, a, type, (cudaStream_t)stream); });
}

int b2_beam_reorder(const b2_state *states, int n, const int *parents, long long groups, int beams, b2_stream stream) {
    if (n < 0 || groups < 0 || groups > 0x7fffffff / MAX_BEAMS || beams < 1 || beams > MAX_BEAMS) {
        set_error("b2_beam_reorder: %d tensors, %lld sequences of %d beams (1 to %d)", n, groups, beams, MAX_BEAMS);
        return B2_ERR_BAD_SHAPE;
    }
    if (!n || !groups) return B2_OK;
    if (!states || !parents || !aligned_to(parents, 4)) { set_error("b2_beam_reorder: null pointer, or parents that are not aligned to 4 bytes"); return B2_ERR_BAD_ARG; }
    for (int i = 0; i < n; ++i) {
        const b2_state &s = states[i];
        if (s.outer < 0 || s.row_bytes < 0 || s.outer > MAX_LD || s.row_bytes > MAX_LD) { set_error("b2_beam_reorder: tensor %d: %lld x rows of %lld bytes", i, s.outer, s.row_bytes); return B2_ERR_BAD_SHAPE; }
        const double bytes = (double)s.outer * (double)groups * beams * (double)s.row_bytes;
        if (bytes > 1e15) { set_error("b2_beam_reorder: tensor %d: %lld x rows of %lld bytes", i, s.outer, s.row_bytes); return B2_ERR_BAD_SHAPE; }
        if (!s.outer || !s.row_bytes) continue;
        if (!s.data) { set_error("b2_beam_reorder: null pointer (tensor %d)", i); return B2_ERR_BAD_ARG; }
        const char *p = (const char *)s.data, *q = (const char *)s.out, *end = p + (long long)bytes;
        if (q && q != p && q < end && p < q + (long long)bytes) { set_error("b2_beam_reorder: tensor %d and its output overlap", i); return B2_ERR_BAD_ARG; }
    }
    // in place, more than MOST_HELD beams are in registers at once, in narrow columns: a launch of their own
    for (int pass = 0; pass < 2; ++pass) {
        int i = 0;
        while (i < n) {
            StateArgs a;
            a.n = 0; a.beams = beams; a.groups = groups; a.parents = parents;
            unsigned long long blocks = 0;
            for (; i < n && a.n < MAX_STATES; ++i) {
                b2_state s = states[i];
                if (!s.outer || !s.row_bytes) continue;
                if (!s.out) s.out = s.data;
                const Way way = way_of(s, beams);
                if ((!way.team && s.out == s.data && beams > MOST_HELD) != (pass == 1)) continue;
                const double more = (double)groups * ceil((way.team ? (double)s.outer * way.team / way.batch : (double)s.outer * (double)(s.row_bytes / way.width)) / MOVE_THREADS);
                if (more > 2147483647.0) { set_error("b2_beam_reorder: tensor %d is too large", i); return B2_ERR_BAD_SHAPE; }
                if (blocks + (unsigned long long)more > 2147483647ull) break;
                a.s[a.n] = s;
                a.first[a.n++] = (unsigned)blocks;
                blocks += (unsigned long long)more;
            }
            a.first[a.n] = (unsigned)blocks;
            if (!blocks) continue;
            const auto go = [&](auto kernel) { kernel<<<(unsigned)blocks, MOVE_THREADS, 0, (cudaStream_t)stream>>>(a); };
            if (pass) go(beam_reorder_kernel<MAX_BEAMS>);
            else if (beams <= 4) go(beam_reorder_kernel<4>);
            else if (beams <= 8) go(beam_reorder_kernel<8>);
            else go(beam_reorder_kernel<MOST_HELD>);
            count_launch();
            B2_CUDA(cudaGetLastError());
        }
    }
    return B2_OK;
}

}  // extern "C"
