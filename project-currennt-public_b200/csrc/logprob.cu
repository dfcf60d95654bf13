// Log probabilities of given tokens under rows of logits, with the entropy of each row and its most likely tokens, and their gradient.
//
//   z_j = s * x_j where token j is allowed, -inf elsewhere;   lse = log sum_j e^z_j;   logprob = z_tok - lse
//   H = -sum_j p_j log p_j,  p_j = e^(z_j - lse);   the K largest z_j by (value, lower index first)
//   dx_j = s * (g * ([j = tok] - p_j) - h * p_j * (log p_j + H))       for gradients g of logprob and h of H
//
// Forward, one pass: every thread keeps the largest value m it has met, S = sum e^(z - m) and E = sum e^(z - m) (z - m); a new maximum
// rescales both.  Then lse = m + log S and H = log S - E / S, which needs no difference of large numbers.
// The K largest: a warp keeps its best K as a sorted list, one entry a lane; a batch of values is looked at only if its maximum
// passes the K-th entry, so that after the first batches insertions are rare (K log(n) of them for values in random order).
// Rows of up to 1024 entries stay in the registers of one warp.  Longer rows take a block, or a thread-block cluster of up to 16 blocks
// when there are few rows: its blocks hand their sums and lists to the first one through distributed shared memory, so that a row needs
// neither a second launch nor a workspace.
// Bound by memory for long rows: 4 to 5 issue slots and one ex2 an entry, against the 11 entries of 2 bytes that arrive per cycle and SM.
#include <math.h>

#include <cooperative_groups.h>

#include "typed.cuh"

namespace cg = cooperative_groups;

namespace b2 {
namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr unsigned FULL = 0xffffffffu;
constexpr int MAX_TOP = 32;

__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float max_nan(float a, float b) { float y; asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b)); return y; }
__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }

// ---- running sums -----------------------------------------------------------------------------------------------------------------
struct Sums { float m, s, e; };   // largest z, sum of e^(z - m), sum of e^(z - m) (z - m)

// The differences are taken before the factor log2(e), so that values near the type's lowest one do not become -inf on the way.
__device__ __forceinline__ void rescale(Sums &a, float m) {
    // a.m > -inf here; a NaN in either maximum makes the sums NaN
    const float d = a.m - m, r = ex2(d * LOG2E);
    a.e = r == 0.0f ? 0.0f : r * fmaf(a.s, d, a.e);
    a.s = r == 0.0f ? 0.0f : r * a.s;
    a.m = m;
}
__device__ __forceinline__ Sums merge(Sums a, Sums b) {
    const float m = max_nan(a.m, b.m);
    if (m == neg_inf()) return a;
    if (a.m != neg_inf()) rescale(a, m);
    if (b.m != neg_inf()) rescale(b, m);
    return {m, a.s + b.s, a.e + b.e};
}
__device__ __forceinline__ Sums warp_merge(Sums a) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Sums b = {__shfl_xor_sync(FULL, a.m, o), __shfl_xor_sync(FULL, a.s, o), __shfl_xor_sync(FULL, a.e, o)};
        a = merge(a, b);
    }
    return a;
}
// N values z whose maximum (NaN if one is NaN) is top
template <int N> __device__ __forceinline__ void add_values(Sums &a, const float (&z)[N], float top) {
    if (!(top <= a.m)) {
        if (a.m != neg_inf()) rescale(a, top); else a = {top, 0.0f, 0.0f};
    }
    if (a.m == neg_inf()) return;
    float s = 0.0f, e = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        // z = -inf adds nothing, and 0 * -inf must not be formed; a NaN (one value, or +inf - +inf) stays
        const float d = max_nan(z[i] - a.m, -3.402823466e38f), w = ex2(d * LOG2E);
        s += w;
        e = fmaf(w, d, e);
    }
    a.s += s;
    a.e += e;
}

// ---- the K largest ------------------------------------------------------------------------------------------------------------------
// An entry is one 64-bit key: the value as an ordered integer above, the complement of its index below; larger is better.  0 is no entry.
typedef unsigned long long Key;
__device__ __forceinline__ Key make_key(float z, int index) {
    const unsigned b = __float_as_uint(z + 0.0f);           // -0 counts as 0
    const unsigned o = z != z ? FULL : (b ^ ((b >> 31) ? FULL : 0x80000000u));
    return ((Key)o << 32) | (unsigned)~index;
}
__device__ __forceinline__ float key_value(Key k) {
    const unsigned o = (unsigned)(k >> 32);
    return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : FULL));
}
__device__ __forceinline__ int key_index(Key k) { return (int)~(unsigned)k; }

// Lane l holds the l-th best of the warp, descending.  A value is of interest if it is not below `limit` (the K-th best, or a bound known
// from elsewhere) and above `floor`: the K-th best of what came before the current vectors, whose indices are all lower, so that an
// equal value loses against it.
struct TopList {
    Key key;
    float limit, floor;
    __device__ __forceinline__ void clear() { key = 0; limit = floor = neg_inf(); }
    __device__ __forceinline__ bool wants(float z) const { return !(z < limit) && !(z <= floor); }
    __device__ __forceinline__ void insert(Key k, int K) {
        const int lane = threadIdx.x & 31;
        const int pos = __popc(__ballot_sync(FULL, key > k));
        const Key up = __shfl_up_sync(FULL, key, 1);
        if (lane >= pos) key = lane == pos ? k : up;
        const Key last = __shfl_sync(FULL, key, K - 1);
        if (last) limit = key_value(last);
    }
    __device__ __forceinline__ void settle(int K) {
        const Key last = __shfl_sync(FULL, key, K - 1);
        if (last) floor = key_value(last);
    }
};
// Offers every lane's N values of the indices at, at + step, ...
template <int N> __device__ __forceinline__ void offer(TopList &t, const float (&z)[N], int at, int step, int K) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        unsigned who = __ballot_sync(FULL, t.wants(z[i]));
        while (who) {
            const int src = __ffs(who) - 1;
            const Key k = make_key(__shfl_sync(FULL, z[i], src), __shfl_sync(FULL, at + i * step, src));
            if (k > __shfl_sync(FULL, t.key, K - 1)) t.insert(k, K);
            who &= who - 1;
            who &= __ballot_sync(FULL, t.wants(z[i]));
        }
    }
    t.settle(K);
}
// The K-th largest of the 32 lanes' values: a bound that at least K values of the warp reach.
__device__ __forceinline__ float kth_of_lanes(float v, int K) {
    const int lane = threadIdx.x & 31;
    if (v != v) v = __int_as_float(0x7f800000);
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
        for (int j = k >> 1; j > 0; j >>= 1) {
            const float o = __shfl_xor_sync(FULL, v, j);
            const bool desc = (lane & k) == 0, low = (lane & j) == 0;
            v = (desc == low) ? fmaxf(v, o) : fminf(v, o);
        }
    return __shfl_sync(FULL, v, K - 1);
}
// Lane l, if `have`, holds a list of K keys (descending, 0 behind the last): the best K of all lists, lane k the k-th.
__device__ __forceinline__ Key merge_lists(const Key *list, int K, bool have) {
    const int lane = threadIdx.x & 31;
    int at = 0;
    Key head = have ? list[0] : 0, mine = 0;
    for (int k = 0; k < K; ++k) {
        const unsigned hi = __reduce_max_sync(FULL, (unsigned)(head >> 32));
        if (!hi) break;
        const unsigned lo = __reduce_max_sync(FULL, (unsigned)(head >> 32) == hi ? (unsigned)head : 0u);
        const Key best = ((Key)hi << 32) | lo;
        if (head == best) { ++at; head = at < K ? list[at] : 0; }
        if (lane == k) mine = best;
    }
    return mine;
}

// ---- forward ----------------------------------------------------------------------------------------------------------------------
struct FwdArgs {
    const unsigned char *mask; long long ld_mask;
    const int *tokens;
    float *logprob, *lse, *entropy, *top_logprobs;
    int *top_tokens;
    long long rows, ld;
    int vocab, top;
    float scale;
};

// The row's token and its value, fetched by one thread before the row is read
struct Given { int tok; float z; };
template <typename T> __device__ __forceinline__ Given load_given(const FwdArgs &a, long long r, const T *x) {
    Given g = {-1, 0.0f};
    if (!a.logprob) return g;
    g.tok = a.tokens[r];
    if (g.tok >= 0 && g.tok < a.vocab) g.z = (!a.mask || a.mask[r * a.ld_mask + g.tok]) ? __fmul_rn(to_float(x[g.tok]), a.scale) : neg_inf();
    return g;
}
// log probabilities are (z - m) - log S: z - lse would lose log S beside a large m
__device__ __forceinline__ float log_of(float z, const Sums &t, float ls) { return (z - t.m) - ls; }
// written by one thread; returns log S
__device__ __forceinline__ float write_row(const FwdArgs &a, long long r, const Given &g, Sums t) {
    const float ls = logf(t.s);
    const bool none = t.m == neg_inf();                       // nothing allowed, or nothing above -inf
    const float lse = none ? neg_inf() : t.m + ls;
    a.lse[r] = lse;
    if (a.entropy) a.entropy[r] = none ? 0.0f : ls - t.e / t.s;
    if (a.logprob) {
        float lp = g.tok < 0 ? 0.0f : nanf("");               // padding; a token beyond the vocabulary shows as NaN
        // -inf - -inf is no number, but the token's probability is 0
        if (g.tok >= 0 && g.tok < a.vocab) lp = g.z == neg_inf() && lse == lse ? g.z : log_of(g.z, t, ls);
        a.logprob[r] = lp;
    }
    return ls;
}
__device__ __forceinline__ void write_top(const FwdArgs &a, long long r, Key k, const Sums &t, float ls) {
    const int lane = threadIdx.x & 31;
    if (lane < a.top) {
        a.top_tokens[r * a.top + lane] = k ? key_index(k) : -1;
        a.top_logprobs[r * a.top + lane] = k ? log_of(key_value(k), t, ls) : neg_inf();
    }
}

// One warp a row, NV entries a lane.
template <typename T, int NV> __global__ void __launch_bounds__(256) logprob_warp_kernel(const T *__restrict__ logits, const FwdArgs a) {
    const int lane = threadIdx.x & 31;
    const long long r = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (r >= a.rows) return;
    const T *x = logits + r * a.ld;
    float z[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) z[i] = lane + 32 * i < a.vocab ? to_float(x[lane + 32 * i]) : neg_inf();
    Given g = {-1, 0.0f};
    if (lane == 0) g = load_given(a, r, x);
    if (a.mask) {
        const unsigned char *mk = a.mask + r * a.ld_mask;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (lane + 32 * i < a.vocab && !mk[lane + 32 * i]) z[i] = neg_inf();
    }
    float top = neg_inf();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        z[i] = __fmul_rn(z[i], a.scale);
        top = max_nan(top, z[i]);
    }
    float wide = top;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) wide = max_nan(wide, __shfl_xor_sync(FULL, wide, o));
    Sums t = {neg_inf(), 0.0f, 0.0f};
    add_values<NV>(t, z, wide);
    t.s = warp_sum(t.s);
    t.e = warp_sum(t.e);
    float ls = 0.0f;
    if (lane == 0) ls = write_row(a, r, g, t);
    if (a.top) {
        ls = __shfl_sync(FULL, ls, 0);
        TopList best;
        best.clear();
        best.limit = kth_of_lanes(top, a.top);
        offer<NV>(best, z, lane, 32, a.top);
        write_top(a, r, best.key, t, ls);
    }
}

// blocks_per_row blocks a row (a thread-block cluster where there are several).  Entries are taken in vectors of W = 16 bytes from the
// 16-byte boundary at or below the row's start, U vectors a thread and batch.
template <typename T, int THREADS, bool TOP, bool MASK>
__global__ void __launch_bounds__(THREADS) logprob_row_kernel(const T *__restrict__ logits, const FwdArgs a, int blocks_per_row) {
    constexpr int W = 16 / sizeof(T), U = 4, WARPS = THREADS / 32, MOST = 16;
    __shared__ Sums sums[WARPS], all_sums[MOST];
    __shared__ Key lists[WARPS][MAX_TOP], all_lists[MOST][MAX_TOP];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const long long r = blockIdx.x / (unsigned)blocks_per_row;
    const int part = (int)(blockIdx.x % (unsigned)blocks_per_row);
    // the first block's shared memory may be written once that block runs: arrive here, wait before the write
    if (blocks_per_row > 1) cg::this_cluster().barrier_arrive();
    const T *x = logits + r * a.ld;
    const unsigned char *mk = MASK ? a.mask + r * a.ld_mask : nullptr;
    const int mis = (int)(((uintptr_t)x & 15) / sizeof(T));
    const T *base = x - mis;
    const int end = mis + a.vocab, vecs = (end + W - 1) / W; // vector v holds the entries v * W - mis ...
    const int v0 = (int)((long long)vecs * part / blocks_per_row), v1 = (int)((long long)vecs * (part + 1) / blocks_per_row);
    const bool mask_vec = MASK && ((uintptr_t)(mk - mis) & (W - 1)) == 0;
    Given g = {-1, 0.0f};
    if (part == 0 && threadIdx.x == 0) g = load_given(a, r, x);
    Sums t = {neg_inf(), 0.0f, 0.0f};
    TopList best;
    best.clear();
    for (int b = v0 + w * 32; b < v1; b += THREADS * U) {
        float z[U * W];
        const int last = b + THREADS * (U - 1) + 32;         // one behind the batch's last vector
        if ((b > 0 || mis == 0) && last <= v1 && last * W <= end) {
            float q[U][W];
#pragma unroll
            for (int u = 0; u < U; ++u) load_vec<T, W>(q[u], base + (size_t)(b + u * THREADS + lane) * W);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < W; ++j) z[u * W + j] = q[u][j];
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int v = b + u * THREADS + lane;
                float q[W];
#pragma unroll
                for (int j = 0; j < W; ++j) q[j] = neg_inf();
                if (v < v1) {
                    if (v * W >= mis && (v + 1) * W <= end) load_vec<T, W>(q, base + (size_t)v * W);
                    else
#pragma unroll
                        for (int j = 0; j < W; ++j)
                            if (v * W + j >= mis && v * W + j < end) q[j] = to_float(base[v * W + j]);
                }
#pragma unroll
                for (int j = 0; j < W; ++j) z[u * W + j] = q[j];
            }
        }
        if (MASK) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int v = b + u * THREADS + lane;
                Vec<unsigned char, W> on;
                if (v < v1 && mask_vec && v * W >= mis && (v + 1) * W <= end) on = *reinterpret_cast<const Vec<unsigned char, W> *>(mk - mis + v * W);
                else
#pragma unroll
                    for (int j = 0; j < W; ++j) on.v[j] = v < v1 && v * W + j >= mis && v * W + j < end ? mk[v * W + j - mis] : 0;
#pragma unroll
                for (int j = 0; j < W; ++j)
                    if (!on.v[j]) z[u * W + j] = neg_inf();
            }
        }
        float top = neg_inf();
#pragma unroll
        for (int i = 0; i < U * W; ++i) {
            z[i] = __fmul_rn(z[i], a.scale);
            top = max_nan(top, z[i]);
        }
        add_values<U * W>(t, z, top);
        if (TOP) {
            if (best.limit == neg_inf()) best.limit = kth_of_lanes(top, a.top);
            if (__any_sync(FULL, best.wants(top))) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    float q[W];
#pragma unroll
                    for (int j = 0; j < W; ++j) q[j] = z[u * W + j];
                    offer<W>(best, q, (b + u * THREADS + lane) * W - mis, 1, a.top);
                }
            }
        }
    }
    t = warp_merge(t);
    if (lane == 0) sums[w] = t;
    if (TOP) lists[w][lane] = best.key;
    __syncthreads();
    // the first warp joins the block's warps, then that of the first block the row's blocks
    Key k = 0;
    if (w == 0) {
        t = warp_merge(lane < WARPS ? sums[lane] : Sums{neg_inf(), 0.0f, 0.0f});
        if (TOP) k = merge_lists(lists[lane < WARPS ? lane : 0], a.top, lane < WARPS);
    }
    if (blocks_per_row > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        cluster.barrier_wait();
        if (w == 0) {
            if (lane == 0) *cluster.map_shared_rank(&all_sums[part], 0) = t;
            if (TOP) *cluster.map_shared_rank(&all_lists[part][lane], 0) = k;
        }
        cluster.sync();
        if (part != 0) return;
        if (w == 0) {
            t = warp_merge(lane < blocks_per_row ? all_sums[lane] : Sums{neg_inf(), 0.0f, 0.0f});
            if (TOP) k = merge_lists(all_lists[lane < blocks_per_row ? lane : 0], a.top, lane < blocks_per_row);
        }
    }
    if (w == 0) {
        float ls = 0.0f;
        if (lane == 0) ls = write_row(a, r, g, t);
        if (TOP) write_top(a, r, k, t, __shfl_sync(FULL, ls, 0));
    }
}

template <typename T, bool TOP, bool MASK> int launch_rows(const T *logits, const FwdArgs &a, cudaStream_t st) {
    constexpr int W = 16 / sizeof(T);
    // few rows: several blocks a row, as long as each has at least a batch of 256 threads
    int per_row = 1;
    while (per_row < 8 && a.rows * per_row * 2 <= 2 * sm_count() && (a.vocab / (per_row * 2)) >= 256 * 4 * W) per_row *= 2;
    if (a.rows * per_row > 0x7fffffffll) { set_error("b2_logprob_forward: %lld rows", a.rows); return B2_ERR_BAD_SHAPE; }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * per_row));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = per_row;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = per_row > 1 ? 1 : 0;
    count_launch();
    B2_CUDA(cudaLaunchKernelEx(&cfg, logprob_row_kernel<T, 256, TOP, MASK>, logits, a, per_row));
    return B2_OK;
}

template <typename T> int forward(const T *logits, const FwdArgs &a, cudaStream_t st) {
    if (a.vocab <= 1024) {
        const long long blocks = (a.rows + 7) / 8;
        if (blocks > 0x7fffffffll) { set_error("b2_logprob_forward: %lld rows", a.rows); return B2_ERR_BAD_SHAPE; }
        const int nv = (a.vocab + 31) / 32;
        if (nv <= 4) logprob_warp_kernel<T, 4><<<(unsigned)blocks, 256, 0, st>>>(logits, a);
        else if (nv <= 10) logprob_warp_kernel<T, 10><<<(unsigned)blocks, 256, 0, st>>>(logits, a);
        else if (nv <= 18) logprob_warp_kernel<T, 18><<<(unsigned)blocks, 256, 0, st>>>(logits, a);
        else logprob_warp_kernel<T, 32><<<(unsigned)blocks, 256, 0, st>>>(logits, a);
        count_launch();
        B2_CUDA(cudaGetLastError());
        return B2_OK;
    }
    if (a.top) return a.mask ? launch_rows<T, true, true>(logits, a, st) : launch_rows<T, true, false>(logits, a, st);
    return a.mask ? launch_rows<T, false, true>(logits, a, st) : launch_rows<T, false, false>(logits, a, st);
}

// ---- backward -----------------------------------------------------------------------------------------------------------------------
struct BwdArgs {
    const unsigned char *mask; long long ld_mask;
    const int *tokens;
    const float *lse, *dlogprob, *entropy, *dentropy;
    long long rows, ld, ld_out;
    int vocab;
    float scale;
};
// fp32 gradients with the exponential of the full accuracy, 16-bit ones with the hardware's: its error of 2^-22 is lost in their rounding
template <typename T> __device__ __forceinline__ float exp_for(float x) { return sizeof(T) == 4 ? expf(x) : ex2(x * LOG2E); }

struct RowGrad { float lse, g, h, H; int tok; };
template <typename T, bool ENT> __device__ __forceinline__ float entry_grad(const RowGrad &q, float x, float scale, bool on, int i) {
    if (!on) return 0.0f;
    const float lp = __fmul_rn(x, scale) - q.lse;
    const float p = exp_for<T>(lp);
    float d = -q.g * p;
    // p = 0 has no share in the entropy's gradient, whatever log p is; NaN stays
    if (ENT) d = p == 0.0f ? d : fmaf(-q.h * p, lp + q.H, d);
    if (i == q.tok) d += q.g;
    return d * scale;
}

// Threads go over (row, vector) pairs: tpr threads a row, each up to U vectors apart by tpr.
template <typename T, bool ENT, bool MASK>
__global__ void __launch_bounds__(256) logprob_backward_kernel(T *__restrict__ dlogits, const T *logits, const BwdArgs a, int tpr, int segs) {
    constexpr int W = 16 / sizeof(T), U = 2;
    const int per_block = 256 / tpr;
    // a row of several segments takes whole blocks (tpr = 256)
    const long long r = segs > 1 ? (long long)(blockIdx.x / (unsigned)segs) : (long long)blockIdx.x * per_block + threadIdx.x / tpr;
    const int seg = segs > 1 ? (int)(blockIdx.x % (unsigned)segs) : 0;
    if (r >= a.rows) return;
    const T *x = logits + r * a.ld;
    T *d = dlogits + r * a.ld_out;
    const int mis = (int)(((uintptr_t)x & 15) / sizeof(T));
    const bool out_vec = (((uintptr_t)(d - mis)) & 15) == 0;
    RowGrad q;
    q.tok = __ldg(a.tokens + r);
    q.lse = __ldg(a.lse + r);
    q.g = a.dlogprob ? __ldg(a.dlogprob + r) : 0.0f;
    q.h = ENT ? __ldg(a.dentropy + r) : 0.0f;
    q.H = ENT ? __ldg(a.entropy + r) : 0.0f;
    // padding, and a row that allows nothing: no gradient.  A token beyond the vocabulary shows as NaN, as its log probability does.
    const bool zero = q.tok < 0 || q.lse == neg_inf();
    const float bad = q.tok >= a.vocab ? nanf("") : 0.0f;
    const unsigned char *mk = MASK ? a.mask + r * a.ld_mask : nullptr;
    const bool mask_vec = MASK && ((uintptr_t)(mk - mis) & (W - 1)) == 0;
    const int first = seg * tpr * U + (threadIdx.x & (tpr - 1));
    float z[U][W];
    bool whole[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int v = first + u * tpr;
        whole[u] = v * W >= mis && (v + 1) * W <= mis + a.vocab;
        if (whole[u] && !zero) load_vec<T, W>(z[u], x - mis + (size_t)v * W);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int v = first + u * tpr, i0 = v * W - mis;
        if (whole[u]) {
            unsigned char on[W];
            if (MASK) {
                if (mask_vec) *reinterpret_cast<Vec<unsigned char, W> *>(on) = *reinterpret_cast<const Vec<unsigned char, W> *>(mk + i0);
                else {
#pragma unroll
                    for (int j = 0; j < W; ++j) on[j] = mk[i0 + j];
                }
            }
            float o[W];
#pragma unroll
            for (int j = 0; j < W; ++j) o[j] = zero ? 0.0f : entry_grad<T, ENT>(q, z[u][j], a.scale, !MASK || on[j], i0 + j) + bad;
            if (out_vec) store_vec<T, W>(d + i0, o);
            else {
#pragma unroll
                for (int j = 0; j < W; ++j) d[i0 + j] = from_float<T>(o[j]);
            }
        } else {
            for (int j = 0; j < W; ++j) {
                const int i = i0 + j;
                if (i < 0 || i >= a.vocab) continue;
                d[i] = from_float<T>(zero ? 0.0f : entry_grad<T, ENT>(q, to_float(x[i]), a.scale, !MASK || mk[i], i) + bad);
            }
        }
    }
}

template <typename T, bool ENT, bool MASK> int backward(T *dlogits, const T *logits, const BwdArgs &a, cudaStream_t st) {
    constexpr int W = 16 / sizeof(T), U = 2;
    const int vecs = (a.vocab + W - 1) / W + 1;               // one more: a row may start inside a vector
    unsigned tpr = pow2_at_least((unsigned)((vecs + U - 1) / U));
    if (tpr > 256) tpr = 256;
    const int segs = (vecs + (int)tpr * U - 1) / ((int)tpr * U);
    const long long per = 256 / tpr, blocks = (a.rows * segs + per - 1) / per;
    if (blocks > 0x7fffffffll) { set_error("b2_logprob_backward: %lld rows of %d", a.rows, a.vocab); return B2_ERR_BAD_SHAPE; }
    logprob_backward_kernel<T, ENT, MASK><<<(unsigned)blocks, 256, 0, st>>>(dlogits, logits, a, (int)tpr, segs);
    count_launch();
    B2_CUDA(cudaGetLastError());
    return B2_OK;
}

int check(const char *who, const void *logits, int type, long long rows, int vocab, long long ld, const unsigned char *mask, long long ld_mask, float scale) {
    const int e = type_size(type);
    if (!e) { set_error("%s: unknown element type %d", who, type); return B2_ERR_BAD_ARG; }
    if (rows < 0 || vocab < 1 || vocab > (1 << 27)) { set_error("%s: %lld rows of %d logits (at most 2^27)", who, rows, vocab); return B2_ERR_BAD_SHAPE; }
    if (ld < vocab || (mask && ld_mask != 0 && ld_mask < vocab)) {
        set_error("%s: leading dimension too small (logits %lld, mask %lld for %d columns)", who, ld, ld_mask, vocab);
        return B2_ERR_BAD_ARG;
    }
    if (!(scale > 0.0f) || scale > 3.402823466e38f) { set_error("%s: the scale %g is not a positive number", who, (double)scale); return B2_ERR_BAD_ARG; }
    if (rows && (!logits || !aligned_to(logits, e))) { set_error("%s: the logits are missing or not aligned to their elements", who); return B2_ERR_BAD_ARG; }
    return B2_OK;
}

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" {

int b2_logprob_forward(const void *logits, int type, long long rows, int vocab, long long ld, const unsigned char *mask, long long ld_mask, float scale,
                       const int *tokens_dev, float *logprob, float *lse, float *entropy, int top, int *top_tokens, float *top_logprobs, b2_stream stream) {
    B2_TRY(check("b2_logprob_forward", logits, type, rows, vocab, ld, mask, ld_mask, scale));
    if (top < 0 || top > MAX_TOP) { set_error("b2_logprob_forward: %d alternatives (at most %d)", top, MAX_TOP); return B2_ERR_BAD_SHAPE; }
    if (!rows) return B2_OK;
    if (!lse || (logprob && !tokens_dev) || (top && (!top_tokens || !top_logprobs))) { set_error("b2_logprob_forward: null pointer"); return B2_ERR_BAD_ARG; }
    const FwdArgs a = {mask, ld_mask, tokens_dev, logprob, lse, entropy, top_logprobs, top_tokens, rows, ld, vocab, top, scale};
    return with_type(type, [&](auto *t) { return forward((const B2_ELEM(t) *)logits, a, (cudaStream_t)stream); });
}

int b2_logprob_backward(void *dlogits, long long ld_dlogits, const void *logits, int type, long long rows, int vocab, long long ld, const unsigned char *mask,
                        long long ld_mask, float scale, const int *tokens_dev, const float *lse, const float *dlogprob, const float *entropy, const float *dentropy,
                        b2_stream stream) {
    B2_TRY(check("b2_logprob_backward", logits, type, rows, vocab, ld, mask, ld_mask, scale));
    if (ld_dlogits < vocab) { set_error("b2_logprob_backward: leading dimension too small (gradient %lld for %d columns)", ld_dlogits, vocab); return B2_ERR_BAD_ARG; }
    if (!rows) return B2_OK;
    if (!dlogits || !aligned_to(dlogits, type_size(type))) { set_error("b2_logprob_backward: the gradient is missing or not aligned to its elements"); return B2_ERR_BAD_ARG; }
    if (!tokens_dev || !lse || (dentropy && !entropy)) { set_error("b2_logprob_backward: null pointer"); return B2_ERR_BAD_ARG; }
    if (dlogits == logits && ld_dlogits != ld) { set_error("b2_logprob_backward: in place with another leading dimension"); return B2_ERR_BAD_ARG; }
    const BwdArgs a = {mask, ld_mask, tokens_dev, lse, dlogprob, entropy, dentropy, rows, ld, ld_dlogits, vocab, scale};
    return with_type(type, [&](auto *t) {
        typedef B2_ELEM(t) T;
        T *d = (T *)dlogits;
        const T *x = (const T *)logits;
        if (dentropy) return mask ? backward<T, true, true>(d, x, a, (cudaStream_t)stream) : backward<T, true, false>(d, x, a, (cudaStream_t)stream);
        return mask ? backward<T, false, true>(d, x, a, (cudaStream_t)stream) : backward<T, false, false>(d, x, a, (cudaStream_t)stream);
    });
}

}  // extern "C"
