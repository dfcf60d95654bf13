// Divergence of rows of logits from a teacher that is known by its K most likely tokens i_k and their log probabilities t_k, and its gradient.
//
//   z = s * x,  lse = log sum_j e^z_j,  p = e^(z - lse)
//   without a rest:  q = e^t / sum e^t                          L = sum_k q_k (log q_k - log p_k)
//   with a rest:     q = e^t, q_r = 1 - sum q, p_r = sum of p off the list      L = sum_k q_k (log q_k - log p_k) + q_r (log q_r - log p_r)
//   dL/dx_j = s (p_j - q_k) at i_k, s (p_j - q_r e^(z_j - lse_r)) = s e^(z_j - lse_r) (p_r - q_r) elsewhere (without a rest s p_j)
//
// Forward: p_r is a sum of its own, over the tokens that are not listed.  As 1 - sum p_k it would lose all its digits where the listed tokens hold most
// of the mass, which is what a good student does.  A row passes through shared memory in pieces of 2 KB that each warp copies ahead for itself; a lane holds
// up to four places of the list, and when a piece is there the lanes whose tokens lie in it take their logits out and leave -inf behind.  So the sum over the
// rest needs no test at any entry, and nothing is read twice.  Narrow rows lie there whole, and as few lanes as the list has places have a row: with a warp a row the
// list's arithmetic is most of the work (65536 rows of 100 fp32: 8.9 us, a warp a row 47.7 us).
// Backward: one read, one write; a ninth warp prepares a block's list while the logits of the eight are on the way; the gradient of unlisted tokens is written
// everywhere, and then that of the listed ones over it, by the block whose segment holds them: no entry is read or written by two blocks, so that a gradient may take its logits' place.  Only one exponential an entry: the rest's probabilities given that it is the rest, times the row's
// factor p_r - q_r.
// Bound, for long rows of 16-bit logits, by memory, the exponentials and 7 issue slots an entry close behind.  Measured on a B200 (device time over the same buffers; in brackets a
// pass over buffers that change): 8192 rows of 50001 bf16, 32 listed, with a rest 126 us (147; 821 MB: 6.5 TB/s); backward 8192 rows of 32003 bf16, 64 listed 162 us (175;
// 1053 MB: 6.5 TB/s); 38400 rows of 259 fp32, 16 listed, backward 13.3 us (21).
#include <math.h>

#include "logits.cuh"

namespace b2 {
namespace {

constexpr int MAX_LIST = 128;
constexpr float LEAST_REST = 9.5367431640625e-7f;      // 2^-20

// The places of a row's list that a lane holds: place s * TEAM + lane, the lanes of a row being TEAM neighbours of a warp.  tok -1: empty, or listed further
// ahead
template <int SLOTS, int TEAM> struct List {
    static_assert(SLOTS == 1 || TEAM == 32, "a short list has a place a lane");
    int tok[SLOTS];
    float lp[SLOTS];
    static __device__ __forceinline__ unsigned lanes() { return TEAM == 32 ? FULL : ((1u << (TEAM & 31)) - 1u) << (threadIdx.x & 31 & ~(TEAM - 1)); }
    static __device__ __forceinline__ bool any_of(bool x) { return (__ballot_sync(FULL, x) & lanes()) != 0; }
    __device__ __forceinline__ void load(const int *tokens, const float *lps, long long r, int top) {
        const int lane = threadIdx.x & (TEAM - 1);
        const long long at = r * top;
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            const int k = s * 32 + lane;
            tok[s] = k < top ? tokens[at + k] : -1;
            lp[s] = k < top ? lps[at + k] : neg_inf();
        }
    }
    // empties the places whose token is negative or stands further ahead; true where a token is not below vocab or a log probability is NaN or +inf
    __device__ __forceinline__ bool settle(int vocab) {
        const int lane = threadIdx.x & 31;
        bool wrong = false, twice[SLOTS];
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            twice[s] = (__ffs(__match_any_sync(FULL, tok[s]) & lanes()) - 1) != lane;
#pragma unroll
            for (int e = 0; e < s; ++e)
#pragma unroll 8
                for (int i = 0; i < 32; ++i) twice[s] |= __shfl_sync(FULL, tok[e], i) == tok[s];
        }
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            if (twice[s]) tok[s] = -1;
            if (tok[s] < 0) { tok[s] = -1; lp[s] = neg_inf(); }
            else if (tok[s] >= vocab || !(lp[s] < __int_as_float(0x7f800000))) wrong = true;
        }
        return any_of(wrong);
    }
    __device__ __forceinline__ bool any() const {
        bool one = false;
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) one |= tok[s] >= 0;
        return any_of(one);
    }
};
// The teacher's probabilities (q of the lane's places, the rest's, what log q is less than lp); false: the row says nothing
template <int SLOTS, int TEAM, bool REST> __device__ __forceinline__ bool teacher(const List<SLOTS, TEAM> &list, float (&q)[SLOTS], float &rest, float &minus) {
    float most = neg_inf(), sum = 0.0f;
    rest = minus = 0.0f;
    if (!REST) {
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) most = fmaxf(most, list.lp[s]);
#pragma unroll
        for (int o = TEAM / 2; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(FULL, most, o));
    }
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) sum += q[s] = REST ? expf(list.lp[s]) : most == neg_inf() ? 0.0f : expf(list.lp[s] - most);
#pragma unroll
    for (int o = TEAM / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(FULL, sum, o);
    if (REST) {
        // in fp32, as the listed probabilities are: a rest of 2e-6 comes out 1.4 % off in the mean, 6 % at most; with 64 bits it would be 0.3 %, of log probabilities that are rounded themselves
        rest = 1.0f - sum;
        if (rest < LEAST_REST) rest = 0.0f;
        return list.any();
    }
    if (most == neg_inf()) return false;
    const float inv = 1.0f / sum;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) q[s] *= inv;
    minus = most + logf(sum);
    return true;
}

// ---- forward ------------------------------------------------------------------------------------------------------------------------
template <typename T, int U> __device__ __forceinline__ void add_vectors(Sum &a, const uint4 (&q)[U], float scale) {
    constexpr int W = 16 / sizeof(T);
    unsigned big = larger_of<T>(q[0]);
#pragma unroll
    for (int u = 1; u < U; ++u) big = Raw<T>::larger(big, larger_of<T>(q[u]));
    const float m = __fmul_rn(Raw<T>::largest(big), scale);
    if (!(m <= a.m)) rise(a, m);
    if (a.m == neg_inf()) return;
    const Pair l2 = pair(LOG2E, LOG2E);
    Pair s = 0;
    less_of_type<T>(scale, a.m, [&](const auto &less) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float x[W];
            Raw<T>::values(x, q[u]);
#pragma unroll
            for (int j = 0; j < W; j += 2) {
                const float2 t = halves(mul2(less(x[j], x[j + 1]), l2));
                s = add2(s, pair(ex2(t.x), ex2(t.y)));
            }
        }
    });
    const float2 v = halves(s);
    a.s += v.x + v.y;
}

struct FwdArgs {
    const int *tokens; const float *lps;
    float *loss, *lse, *lse_rest;
    long long rows, ld;
    int vocab, top;
    float scale;
};
// A row's results from its list, the listed tokens' z (-inf where a place is empty) and the sum t over the other tokens (without a rest: over all)
template <int SLOTS, int TEAM, bool REST>
__device__ __forceinline__ void finish_row(const FwdArgs &a, long long r, const List<SLOTS, TEAM> &list, const float (&z)[SLOTS], const Sum &t, bool wrong) {
    const float inf = __int_as_float(0x7f800000);
    float q[SLOTS], q_rest, minus;
    const bool known = teacher<SLOTS, TEAM, REST>(list, q, q_rest, minus);
    Sum all = t;
    if (REST) {
        Sum mine = {neg_inf(), 0.0f};
#pragma unroll
        for (int s = 0; s < SLOTS; ++s)
            if (!(z[s] <= neg_inf())) mine = join(mine, z[s] == inf ? Sum{nanf(""), 1.0f} : Sum{z[s], 1.0f});
        all = join(t, team_join<TEAM>(mine));
    }
    const float log_all = logf(all.s), log_rest = logf(t.s);
    float part = 0.0f;
    if (all.m != neg_inf()) {
#pragma unroll
        for (int s = 0; s < SLOTS; ++s)
            if (q[s] > 0.0f) part += q[s] * ((list.lp[s] - minus) - ((z[s] - all.m) - log_all));
    } else {
#pragma unroll
        for (int s = 0; s < SLOTS; ++s)
            if (q[s] > 0.0f) part = inf;
    }
#pragma unroll
    for (int o = TEAM / 2; o > 0; o >>= 1) part += __shfl_xor_sync(FULL, part, o);
    if ((threadIdx.x & (TEAM - 1)) == 0 && r < a.rows) {
        const float lse = all.m == neg_inf() ? neg_inf() : all.m + log_all;
        if (REST && q_rest > 0.0f) part += t.m == neg_inf() ? inf : q_rest * (logf(q_rest) - (((t.m - all.m) + log_rest) - log_all));
        a.loss[r] = wrong || (known && lse != lse) ? nanf("") : known ? part : 0.0f;
        a.lse[r] = lse;
        if (REST) a.lse_rest[r] = t.m == neg_inf() ? neg_inf() : t.m + log_rest;
    }
}

// Narrow rows, up to TEAM * U vectors: TEAM neighbouring lanes each, as few as the list has places.  The row lies in shared memory as it does behind a 16-byte boundary.
template <typename T, int TEAM, int U, int SLOTS, bool REST>
__global__ void __launch_bounds__(256) distill_forward_rows_kernel(const T *logits, const FwdArgs a) {
    constexpr int W = 16 / sizeof(T), EDGES = (2 * W - 2 + TEAM - 1) / TEAM;
    __shared__ uint4 rows[256 / TEAM][TEAM * U];
    const int lane = threadIdx.x & (TEAM - 1);
    const long long row = (long long)blockIdx.x * (256 / TEAM) + threadIdx.x / TEAM, r = row < a.rows ? row : a.rows - 1;      // whole warps take part in the lists
    const T *x = logits + r * a.ld;
    const int mis = (int)(((uintptr_t)x & 15) / sizeof(T));
    uint4 *const mine = rows[threadIdx.x / TEAM];
    T *const flat = reinterpret_cast<T *>(mine);                 // entry i at i + mis
    List<SLOTS, TEAM> list;
    list.load(a.tokens, a.lps, r, a.top);
    const unsigned at = (unsigned)__cvta_generic_to_shared(mine + lane);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int v = lane + TEAM * u;
        if (v * W >= mis && (v + 1) * W <= mis + a.vocab) cp_async<16>(at + u * (TEAM * 16), x - mis + v * W);
        else mine[v] = make_uint4(Raw<T>::NONE, Raw<T>::NONE, Raw<T>::NONE, Raw<T>::NONE);
    }
    cp_commit();
    const int head = min(a.vocab, (W - mis) % W), body = (a.vocab - head) / W * W;
    T edge[EDGES];
#pragma unroll
    for (int e = 0; e < EDGES; ++e) {
        const int i = lane + TEAM * e < head ? lane + TEAM * e : lane + TEAM * e + body;
        edge[e] = i < a.vocab ? x[i] : from_float<T>(0.0f);
    }
    const bool wrong = list.settle(a.vocab);
    __syncwarp();                                                // the vectors at the ends are emptied
#pragma unroll
    for (int e = 0; e < EDGES; ++e) {
        const int i = lane + TEAM * e < head ? lane + TEAM * e : lane + TEAM * e + body;
        if (i < a.vocab) flat[i + mis] = edge[e];
    }
    cp_wait<0>();
    __syncwarp();
    float z[SLOTS];
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) {
        const bool there = list.tok[s] >= 0 && list.tok[s] < a.vocab;
        z[s] = there ? __fmul_rn(to_float(flat[list.tok[s] + mis]), a.scale) : neg_inf();
        if (REST && there) flat[list.tok[s] + mis] = from_float<T>(neg_inf());
    }
    __syncwarp();
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) q[u] = mine[lane + TEAM * u];
    Sum t = {neg_inf(), 0.0f};
    add_vectors<T, U>(t, q, a.scale);
    finish_row<SLOTS, TEAM, REST>(a, row, list, z, team_join<TEAM>(t), wrong);
}

constexpr int PIECE = 128, RING = 3;      // vectors of 16 bytes in a piece (4 a lane), pieces in a warp's ring

// A row's place among the 16-byte boundaries: `head` entries before the first one, nv vectors, the rest behind
struct Row {
    int head, nv;
    template <typename T> __device__ __forceinline__ Row(const T *x, int vocab) {
        constexpr int W = 16 / sizeof(T);
        head = (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T);
        if (head > vocab) head = vocab;
        nv = (vocab - head) / W;
    }
};

// WARPS warps a row (1: a block has 8 rows under way), each with the row's pieces w, w + WARPS, ...
template <typename T, int WARPS, int SLOTS, bool REST>
__global__ void __launch_bounds__(256) distill_forward_kernel(const T *logits, const FwdArgs a) {
    constexpr int W = 16 / sizeof(T);
    extern __shared__ uint4 rings[];
    uint4 (*ring)[PIECE] = reinterpret_cast<uint4 (*)[PIECE]>(rings) + (threadIdx.x >> 5) * RING;
    __shared__ float edges[8][32], picked[WARPS > 1 ? MAX_LIST : 1];
    __shared__ Sum sums[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, w = WARPS > 1 ? warp : 0;
    const long long team = WARPS > 1 ? blockIdx.x : (long long)blockIdx.x * 8 + warp, teams = WARPS > 1 ? gridDim.x : (long long)gridDim.x * 8;

    // what is copied next: the vectors src on of row ir, `ahead_left` of which are left for this warp and those behind it
    long long ir = team;
    int slot = 0, ahead_left = 0;
    const uint4 *src = nullptr;
    const auto enter = [&]() {
        if (ir >= a.rows) return;
        const T *x = logits + ir * a.ld;
        const Row g(x, a.vocab);
        src = reinterpret_cast<const uint4 *>(x + g.head) + w * PIECE + lane;
        ahead_left = g.nv - w * PIECE;
    };
    const unsigned ring0 = (unsigned)__cvta_generic_to_shared(&ring[0][lane]);
    const auto issue = [&](int to) {
        while (ahead_left <= 0 && ir < a.rows) {
            ir += teams;
            enter();
        }
        if (ahead_left > 0) {
            const unsigned at = ring0 + to * (PIECE * 16);
            if (ahead_left >= PIECE) {
#pragma unroll
                for (int u = 0; u < PIECE / 32; ++u) cp_async<16>(at + 512 * u, src + 32 * u);
            } else {
#pragma unroll
                for (int u = 0; u < PIECE / 32; ++u)
                    if (lane + 32 * u < ahead_left) cp_async<16>(at + 512 * u, src + 32 * u);
            }
            src += WARPS * PIECE;
            ahead_left -= WARPS * PIECE;
        }
        cp_commit();
    };
    enter();
    List<SLOTS, 32> list, next;
    float edge = 0.0f;
    const auto ahead = [&](long long r) {
        if (r >= a.rows) return;
        next.load(a.tokens, a.lps, r, a.top);
        const T *x = logits + r * a.ld;
        const Row g(x, a.vocab);
        const int behind = a.vocab - g.head - g.nv * W;
        edge = w == 0 && lane < g.head + behind ? to_float(x[lane < g.head ? lane : lane + g.nv * W]) : neg_inf();
    };
    for (int i = 0; i < RING - 1; ++i) issue(i);
    ahead(team);
    for (long long r = team; r < a.rows; r += teams) {
        const T *x = logits + r * a.ld;
        const Row g(x, a.vocab);
        list = next;
        float z_edge = edge;
        ahead(r + teams);
        const bool wrong = list.settle(a.vocab);
        float z[SLOTS];
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) z[s] = neg_inf();
        Sum t = {neg_inf(), 0.0f};
        if (w == 0) {
            // the entries outside the vectors
            edges[warp][lane] = z_edge;
            __syncwarp();
#pragma unroll
            for (int s = 0; s < SLOTS; ++s) {
                const int at = list.tok[s] < g.head ? list.tok[s] : list.tok[s] >= g.head + g.nv * W ? list.tok[s] - g.nv * W : -1;
                if (at >= 0 && at < 32 && list.tok[s] < a.vocab) {
                    z[s] = __fmul_rn(edges[warp][at], a.scale);
                    if (REST) edges[warp][at] = neg_inf();
                }
            }
            __syncwarp();
            z_edge = edges[warp][lane];
            __syncwarp();
            z_edge = __fmul_rn(z_edge, a.scale);               // what the scale takes to -inf adds nothing
            if (!(z_edge <= neg_inf())) t = {z_edge, 1.0f};
            // +inf as e^(inf - inf)
            if (t.m == __int_as_float(0x7f800000)) t.m = t.s = nanf("");
        }
        int first = g.head + w * PIECE * W;
        for (int left = g.nv - w * PIECE; left > 0; left -= WARPS * PIECE, first += WARPS * PIECE * W) {
            cp_wait<RING - 2>();
            __syncwarp();
            issue(slot == 0 ? RING - 1 : slot - 1);
            T *piece = reinterpret_cast<T *>(&ring[slot][0]);
            const unsigned n = (unsigned)min(PIECE, left) * W;
#pragma unroll
            for (int s = 0; s < SLOTS; ++s)
                if ((unsigned)(list.tok[s] - first) < n) {
                    z[s] = __fmul_rn(to_float(piece[list.tok[s] - first]), a.scale);
                    if (REST) piece[list.tok[s] - first] = from_float<T>(neg_inf());
                }
            if (REST) __syncwarp();
            uint4 q[PIECE / 32];
            if (left >= PIECE) {
#pragma unroll
                for (int u = 0; u < PIECE / 32; ++u) q[u] = ring[slot][lane + 32 * u];
            } else {
#pragma unroll
                for (int u = 0; u < PIECE / 32; ++u)
                    q[u] = lane + 32 * u < left ? ring[slot][lane + 32 * u] : make_uint4(Raw<T>::NONE, Raw<T>::NONE, Raw<T>::NONE, Raw<T>::NONE);
            }
            __syncwarp();
            add_vectors<T, PIECE / 32>(t, q, a.scale);
            slot = slot == RING - 1 ? 0 : slot + 1;
        }
        t = team_join<32>(t);
        if (WARPS > 1) {
            if (lane == 0) sums[warp] = t;
#pragma unroll
            for (int s = 0; s < SLOTS; ++s)
                if (list.tok[s] >= 0 && list.tok[s] < a.vocab) {
                    const int at = list.tok[s];
                    const bool outside = at < g.head || at >= g.head + g.nv * W;
                    if (outside ? w == 0 : (at - g.head) / (PIECE * W) % WARPS == w) picked[s * 32 + lane] = z[s];
                }
            __syncthreads();
            if (w == 0) {
                t = team_join<32>(lane < WARPS ? sums[lane] : Sum{neg_inf(), 0.0f});
#pragma unroll
                for (int s = 0; s < SLOTS; ++s)
                    if (list.tok[s] >= 0 && list.tok[s] < a.vocab) z[s] = picked[s * 32 + lane];
            }
            __syncthreads();
            if (w != 0) continue;
        }
        finish_row<SLOTS, 32, REST>(a, r, list, z, t, wrong);
    }
    cp_wait<0>();
}

template <typename T, int SLOTS, bool REST> int launch_forward(const T *logits, const FwdArgs &a, cudaStream_t st) {
    constexpr int W = 16 / sizeof(T), BYTES = 8 * RING * PIECE * 16;
    const int vecs = (a.vocab + W - 1) / W + 1;                   // one more: a row may start inside a vector
    const auto rows = [&](auto kernel, long long blocks) -> int {
        if (blocks > 0x7fffffffll) { set_error("b2_distill_forward: %lld rows", a.rows); return B2_ERR_BAD_SHAPE; }
        kernel<<<(unsigned)blocks, 256, 0, st>>>(logits, a);
        count_launch();
        B2_CUDA(cudaGetLastError());
        return B2_OK;
    };
    if constexpr (SLOTS == 1) {
        if (a.top <= 8 && vecs <= 8 * 4) return rows(distill_forward_rows_kernel<T, 8, 4, 1, REST>, (a.rows + 31) / 32);
        if (a.top <= 16 && vecs <= 16 * 6) return rows(distill_forward_rows_kernel<T, 16, 6, 1, REST>, (a.rows + 15) / 16);
    }
    if (vecs <= 32 * 4) return rows(distill_forward_rows_kernel<T, 32, 4, SLOTS, REST>, (a.rows + 7) / 8);
    // A warp a row where the rows fill the device, a block a row else (bf16, 32 listed, a warp / a block: 1200 x 50000 41 / 29 us, 2000 x 50000 42 / 42, 4000 x 50000 80 / 82; rows of a few pieces would want
    // the warp earlier, 1200 x 3000 6.7 / 11.9 us); 4 blocks an SM for long rows (8192 x 50001: 126 us, with 3 137 us), 3 for shorter ones (40000 x 3000:
    // 69 us, with 4 75 us)
    const bool many = a.rows >= 16 * sm_count();
    const long long teams = many ? (a.rows + 7) / 8 : a.rows, most = (vecs >= 1024 ? 4ll : 3ll) * sm_count();
    const auto go = [&](auto kernel) -> int {
        B2_TRY(set_max_dynamic_smem((const void *)kernel, BYTES));
        kernel<<<(unsigned)(teams < most ? teams : most), 256, BYTES, st>>>(logits, a);
        count_launch();
        B2_CUDA(cudaGetLastError());
        return B2_OK;
    };
    return many ? go(distill_forward_kernel<T, 1, SLOTS, REST>) : go(distill_forward_kernel<T, 8, SLOTS, REST>);
}
template <typename T, int SLOTS> int forward_of(const T *logits, const FwdArgs &a, cudaStream_t st) {
    return a.lse_rest ? launch_forward<T, SLOTS, true>(logits, a, st) : launch_forward<T, SLOTS, false>(logits, a, st);
}
template <typename T> int forward(const T *logits, const FwdArgs &a, cudaStream_t st) {
    if (a.top <= 32) return forward_of<T, 1>(logits, a, st);
    if (a.top <= 64) return forward_of<T, 2>(logits, a, st);
    return forward_of<T, 4>(logits, a, st);
}

// ---- backward -----------------------------------------------------------------------------------------------------------------------
struct BwdArgs {
    const int *tokens; const float *lps;
    const float *lse, *lse_rest, *dloss;
    long long rows, ld, ld_out;
    int vocab, top;
    float scale;
};
struct RowGrad { float base, factor; int what; };      // what: 0 zeros, 1 gradient, 2 NaN

// A row's vectors: v holds the entries v * W - mis on; whole ones lie inside the row
template <typename T> struct Place {
    static constexpr int W = 16 / sizeof(T);
    const T *x;
    T *d;
    int mis, vocab;
    bool out_vec;
    __device__ __forceinline__ Place(T *dlogits, const T *logits, const BwdArgs &a, long long r) : x(logits + r * a.ld), d(dlogits + r * a.ld_out), vocab(a.vocab) {
        mis = (int)(((uintptr_t)x & 15) / sizeof(T));
        out_vec = (((uintptr_t)(d - mis)) & 15) == 0;
    }
    __device__ __forceinline__ bool whole(int v) const { return v * W >= mis && (v + 1) * W <= mis + vocab; }
    __device__ __forceinline__ void load(uint4 &q, int v) const {
        if (whole(v)) q = *reinterpret_cast<const uint4 *>(x - mis + (size_t)v * W);
    }
};
// the gradients off the list of the entries of vector v, whose logits are q; nothing if it is not whole
template <typename T, bool ADD> __device__ __forceinline__ void vector_grads(const Place<T> &p, const uint4 &q, int v, const RowGrad &g, float scale) {
    constexpr int W = 16 / sizeof(T);
    if (!p.whole(v)) return;
    T *const d = p.d + v * W - p.mis;
    float z[W], o[W], old[W];
    if (ADD) {
        if (p.out_vec) load_vec<T, W>(old, d);
        else
#pragma unroll
            for (int j = 0; j < W; ++j) old[j] = to_float(d[j]);
    }
    if (g.what == 1) {
        const Pair factor = pair(g.factor, g.factor);
        Raw<T>::values(z, q);
        less_of_type<T>(scale, g.base, [&](const auto &less) {
#pragma unroll
            for (int j = 0; j < W; j += 2) {
                const float2 t = halves(mul2(exp_pair<T>(less(z[j], z[j + 1])), factor));
                o[j] = ADD ? old[j] + t.x : t.x;
                o[j + 1] = ADD ? old[j + 1] + t.y : t.y;
            }
        });
    } else {
        const float none = g.what == 2 ? nanf("") : 0.0f;
#pragma unroll
        for (int j = 0; j < W; ++j) o[j] = none;
    }
    if (p.out_vec) store_vec<T, W>(d, o);
    else
#pragma unroll
        for (int j = 0; j < W; ++j) d[j] = from_float<T>(o[j]);
}
// The entries in front of the first whole vector and behind the last one, at most 2 W - 2: entry e of them
template <typename T> __device__ __forceinline__ int edge_entry(const Place<T> &p, int e) {
    constexpr int W = 16 / sizeof(T);
    const int head = min(p.vocab, (W - p.mis) % W), body = (p.vocab - head) / W * W;
    return e < head ? e : e + body;                    // not below vocab: there is none
}
template <typename T, bool ADD> __device__ __forceinline__ void edge_grad(const Place<T> &p, int i, T x, const RowGrad &g, float scale) {
    if (i >= p.vocab) return;
    const float o = g.what == 1 ? expf(__fmul_rn(to_float(x), scale) - g.base) * g.factor : g.what == 2 ? nanf("") : 0.0f;
    p.d[i] = from_float<T>(ADD ? to_float(p.d[i]) + o : o);
}

// The list of a row: the row's factors, and the gradients of the listed tokens within [lo, hi)
template <typename T, int SLOTS, int TEAM, bool REST, bool ADD> struct RowList {
    List<SLOTS, TEAM> list;
    float q[SLOTS], lse, rest, weight;
    T z[SLOTS], old[SLOTS];
    __device__ __forceinline__ void load(const BwdArgs &a, long long r) {
        list.load(a.tokens, a.lps, r, a.top);
        lse = a.lse[r];
        rest = REST ? a.lse_rest[r] : 0.0f;
        weight = a.dloss[r] * a.scale;
    }
    // what stands at the listed tokens before anything is written
    __device__ __forceinline__ void gather(const Place<T> &p, int lo, int hi) {
#pragma unroll
        for (int s = 0; s < SLOTS; ++s) {
            const bool here = list.tok[s] >= lo && list.tok[s] < hi;
            z[s] = here ? p.x[list.tok[s]] : from_float<T>(0.0f);
            if (ADD) old[s] = here ? p.d[list.tok[s]] : from_float<T>(0.0f);
        }
    }
    __device__ __forceinline__ RowGrad factors(int vocab) {
        float q_rest, minus;
        const bool wrong = list.settle(vocab), known = teacher<SLOTS, TEAM, REST>(list, q, q_rest, minus);
        RowGrad g = {0.0f, 0.0f, wrong ? 2 : known && lse != neg_inf() ? 1 : 0};
        // e^(z - base) * factor off the list; where the rest has no mass all of its logits are -inf
        const bool split = REST && rest != neg_inf();
        g.base = split ? rest : lse;
        g.factor = weight * (split ? expf(rest - lse) - q_rest : 1.0f);
        return g;
    }
    __device__ __forceinline__ void store(T *d, int lo, int hi, float scale) const {
#pragma unroll
        for (int s = 0; s < SLOTS; ++s)
            if (list.tok[s] >= lo && list.tok[s] < hi) {
                const float o = weight * (expf(__fmul_rn(to_float(z[s]), scale) - lse) - q[s]);
                d[list.tok[s]] = from_float<T>(ADD ? to_float(old[s]) + o : o);
            }
    }
};

// Narrow rows, up to TEAM * U vectors: TEAM neighbouring lanes each, as few as the list has places
template <typename T, int TEAM, int U, int SLOTS, bool REST, bool ADD>
__global__ void __launch_bounds__(256, 4) distill_backward_rows_kernel(T *dlogits, const T *logits, const BwdArgs a) {
    const int lane = threadIdx.x & (TEAM - 1);
    const long long row = (long long)blockIdx.x * (256 / TEAM) + threadIdx.x / TEAM;
    const bool real = row < a.rows;
    const long long r = real ? row : a.rows - 1;              // whole warps take part in the lists
    const Place<T> p(dlogits, logits, a, r);
    RowList<T, SLOTS, TEAM, REST, ADD> list;
    list.load(a, r);
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) p.load(q[u], lane + TEAM * u);
    constexpr int EDGES = (2 * 16 / sizeof(T) - 2 + TEAM - 1) / TEAM;
    T edge[EDGES];
#pragma unroll
    for (int e = 0; e < EDGES; ++e) edge[e] = edge_entry(p, lane + TEAM * e) < a.vocab ? p.x[edge_entry(p, lane + TEAM * e)] : from_float<T>(0.0f);
    list.gather(p, 0, a.vocab);
    const RowGrad g = list.factors(a.vocab);
    __syncwarp();
    if (!real || (g.what == 0 && ADD)) return;
#pragma unroll
    for (int u = 0; u < U; ++u) vector_grads<T, ADD>(p, q[u], lane + TEAM * u, g, a.scale);
#pragma unroll
    for (int e = 0; e < EDGES; ++e) edge_grad<T, ADD>(p, edge_entry(p, lane + TEAM * e), edge[e], g, a.scale);
    __syncwarp(List<SLOTS, TEAM>::lanes());
    if (g.what == 1) list.store(p.d, 0, a.vocab, a.scale);
}

// Wide rows in segments of 256 U vectors: eight warps have their logits on the way while a ninth takes the list in hand; it writes the gradients of the listed
// tokens over those that the eight wrote.
constexpr int STREAM = 256;
template <typename T, int U, int SLOTS, bool REST, bool ADD>
__global__ void __launch_bounds__(STREAM + 32, 3) distill_backward_kernel(T *dlogits, const T *logits, const BwdArgs a, int segs) {
    constexpr int W = 16 / sizeof(T);
    __shared__ RowGrad shared;
    const int at = threadIdx.x, seg = (int)(blockIdx.x % (unsigned)segs);
    const long long r = blockIdx.x / (unsigned)segs;
    const Place<T> p(dlogits, logits, a, r);
    if (at >= STREAM) {
        const int lo = max(0, seg * STREAM * U * W - p.mis), hi = min(a.vocab, (seg + 1) * STREAM * U * W - p.mis);
        RowList<T, SLOTS, 32, REST, ADD> list;
        list.load(a, r);
        // the entries outside the vectors are this warp's too, where they lie in its segment: no other block reads or writes what is listed there
        const int end = edge_entry(p, at - STREAM), i = end >= lo && end < hi ? end : a.vocab;
        T edge = from_float<T>(0.0f);
        if (i < a.vocab) edge = p.x[i];
        // the eight wait for the factors: what only this warp needs is not waited for before they are there (8192 x 32003: 162 us, in the other order 178 us)
        const RowGrad g = list.factors(a.vocab);
        if (at == STREAM) shared = g;
        list.gather(p, lo, hi);
        __syncthreads();
        if (g.what != 0 || !ADD) edge_grad<T, ADD>(p, i, edge, g, a.scale);
        __syncthreads();
        if (g.what == 1) list.store(p.d, lo, hi, a.scale);
        return;
    }
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) p.load(q[u], seg * STREAM * U + at + u * STREAM);
    __syncthreads();
    const RowGrad g = shared;
    if (g.what != 0 || !ADD)
#pragma unroll
        for (int u = 0; u < U; ++u) vector_grads<T, ADD>(p, q[u], seg * STREAM * U + at + u * STREAM, g, a.scale);
    __syncthreads();
}

template <typename T, int SLOTS, bool REST, bool ADD> int launch_backward(T *dlogits, const T *logits, const BwdArgs &a, cudaStream_t st) {
    constexpr int W = 16 / sizeof(T);
    const int vecs = (a.vocab + W - 1) / W + 1;               // one more: a row may start inside a vector
    const auto go = [&](auto kernel, long long blocks, int threads, auto... more) -> int {
        if (blocks > 0x7fffffffll) { set_error("b2_distill_backward: %lld rows of %d", a.rows, a.vocab); return B2_ERR_BAD_SHAPE; }
        kernel<<<(unsigned)blocks, threads, 0, st>>>(dlogits, logits, a, more...);
        count_launch();
        B2_CUDA(cudaGetLastError());
        return B2_OK;
    };
    if constexpr (SLOTS == 1) {
        if (a.top <= 8 && vecs <= 8 * 4) return go(distill_backward_rows_kernel<T, 8, 4, 1, REST, ADD>, (a.rows + 31) / 32, 256);
        if (a.top <= 16 && vecs <= 16 * 6) return go(distill_backward_rows_kernel<T, 16, 6, 1, REST, ADD>, (a.rows + 15) / 16, 256);
    }
    if (vecs <= 32 * 4) return go(distill_backward_rows_kernel<T, 32, 4, SLOTS, REST, ADD>, (a.rows + 7) / 8, 256);
    // Vectors of a thread: 2 where the rows do not fill the device (rows of 32000 bf16, 2 / 8: 30 rows 2.4 / 3.3 us, 120 3.4 / 3.7, 150 4.7 / 4.6, 600 11.4 / 10.8)
    const bool few = (double)a.rows * vecs < 4096.0 * sm_count();
    const int u = few ? 2 : 8, segs = (vecs + STREAM * u - 1) / (STREAM * u);
    if (few) return go(distill_backward_kernel<T, 2, SLOTS, REST, ADD>, a.rows * segs, STREAM + 32, segs);
    return go(distill_backward_kernel<T, 8, SLOTS, REST, ADD>, a.rows * segs, STREAM + 32, segs);
}
template <typename T, int SLOTS> int backward_of(T *dlogits, const T *logits, const BwdArgs &a, bool add, cudaStream_t st) {
    if (a.lse_rest) return add ? launch_backward<T, SLOTS, true, true>(dlogits, logits, a, st) : launch_backward<T, SLOTS, true, false>(dlogits, logits, a, st);
    return add ? launch_backward<T, SLOTS, false, true>(dlogits, logits, a, st) : launch_backward<T, SLOTS, false, false>(dlogits, logits, a, st);
}
template <typename T> int backward(T *dlogits, const T *logits, const BwdArgs &a, bool add, cudaStream_t st) {
    if (a.top <= 32) return backward_of<T, 1>(dlogits, logits, a, add, st);
    if (a.top <= 64) return backward_of<T, 2>(dlogits, logits, a, add, st);
    return backward_of<T, 4>(dlogits, logits, a, add, st);
}

int check(const char *who, const void *logits, int type, long long rows, int vocab, long long ld, float scale, const int *tokens, const float *lps, int top) {
    const int e = type_size(type);
    if (!e) { set_error("%s: unknown element type %d", who, type); return B2_ERR_BAD_ARG; }
    if (rows < 0 || vocab < 1 || vocab > (1 << 27)) { set_error("%s: %lld rows of %d logits (at most 2^27)", who, rows, vocab); return B2_ERR_BAD_SHAPE; }
    if (top < 1 || top > MAX_LIST) { set_error("%s: %d listed tokens (1 to %d)", who, top, MAX_LIST); return B2_ERR_BAD_SHAPE; }
    if (ld < vocab || ld > MAX_LD) { set_error("%s: leading dimension %lld too small or beyond 2^40 (%d columns)", who, ld, vocab); return B2_ERR_BAD_ARG; }
    if (!(scale > 0.0f) || scale > 3.402823466e38f) { set_error("%s: the scale %g is not a positive number", who, (double)scale); return B2_ERR_BAD_ARG; }
    if (rows && (!logits || !aligned_to(logits, e))) { set_error("%s: the logits are missing or not aligned to their elements", who); return B2_ERR_BAD_ARG; }
    if (rows && (!tokens || !lps || !aligned_to(tokens, 4) || !aligned_to(lps, 4))) {
        set_error("%s: the teacher's tokens or log probabilities are missing or not aligned to 4 bytes", who);
        return B2_ERR_BAD_ARG;
    }
    return B2_OK;
}

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" {

int b2_distill_forward(const void *logits, int type, long long rows, int vocab, long long ld, float scale, const int *top_tokens, const float *top_logprobs, int top,
                       float *loss, float *lse, float *lse_rest, b2_stream stream) {
    B2_TRY(check("b2_distill_forward", logits, type, rows, vocab, ld, scale, top_tokens, top_logprobs, top));
    if (!rows) return B2_OK;
    if (!loss || !lse) { set_error("b2_distill_forward: null pointer"); return B2_ERR_BAD_ARG; }
    if (!aligned_to(loss, 4) || !aligned_to(lse, 4) || !aligned_to(lse_rest, 4)) { set_error("b2_distill_forward: a vector of numbers is not aligned to 4 bytes"); return B2_ERR_BAD_ARG; }
    const FwdArgs a = {top_tokens, top_logprobs, loss, lse, lse_rest, rows, ld, vocab, top, scale};
    return with_type(type, [&](auto *t) { return forward((const B2_ELEM(t) *)logits, a, (cudaStream_t)stream); });
}

int b2_distill_backward(void *dlogits, long long ld_dlogits, const void *logits, int type, long long rows, int vocab, long long ld, float scale, const int *top_tokens,
                        const float *top_logprobs, int top, const float *lse, const float *lse_rest, const float *dloss, int accumulate, b2_stream stream) {
    B2_TRY(check("b2_distill_backward", logits, type, rows, vocab, ld, scale, top_tokens, top_logprobs, top));
    if (ld_dlogits < vocab || ld_dlogits > MAX_LD) {
        set_error("b2_distill_backward: leading dimension %lld of the gradient too small or beyond 2^40 (%d columns)", ld_dlogits, vocab);
        return B2_ERR_BAD_ARG;
    }
    if (!rows) return B2_OK;
    if (!dlogits || !aligned_to(dlogits, type_size(type))) { set_error("b2_distill_backward: the gradient is missing or not aligned to its elements"); return B2_ERR_BAD_ARG; }
    if (!lse || !dloss) { set_error("b2_distill_backward: null pointer"); return B2_ERR_BAD_ARG; }
    if (!aligned_to(lse, 4) || !aligned_to(lse_rest, 4) || !aligned_to(dloss, 4)) { set_error("b2_distill_backward: a vector of numbers is not aligned to 4 bytes"); return B2_ERR_BAD_ARG; }
    if (dlogits == logits && (ld_dlogits != ld || accumulate)) { set_error("b2_distill_backward: in place with another leading dimension, or added to the logits"); return B2_ERR_BAD_ARG; }
    const BwdArgs a = {top_tokens, top_logprobs, lse, lse_rest, dloss, rows, ld, ld_dlogits, vocab, top, scale};
    return with_type(type, [&](auto *t) {
        typedef B2_ELEM(t) T;
        return backward<T>((T *)dlogits, (const T *)logits, a, accumulate != 0, (cudaStream_t)stream);
    });
}

}  // extern "C"
