// Log probabilities of given tokens under rows of logits, with the entropy of each row and its most likely tokens, and their gradient.
//
//   z_j = s * x_j where token j is allowed, -inf elsewhere;   lse = log sum_j e^z_j;   logprob = z_tok - lse
//   H = -sum_j p_j log p_j,  p_j = e^(z_j - lse);   the K largest z_j by (value, lower index first)
//   dx_j = s * (g * ([j = tok] - p_j) - h * p_j * (log p_j + H))       for gradients g of logprob and h of H
//
// z_j is the fp32 product everywhere: in the sums, for the given token, in the ranking and in the gradient.  A fused multiply-add would take the
// unrounded one in the sums, and a likely token could end above log 1 by the rounding of a large z.  So S >= 1, and no log probability is above 0.
// Forward, one pass: every thread keeps the largest value m it has met, S = sum e^(z - m) and E = sum e^(z - m) (z - m); a new maximum
// rescales both.  Then lse = m + log S and H = log S - E / S, which needs no difference of large numbers.
// The K largest: a warp keeps its best K as a sorted list, one entry a lane; a batch of values is looked at only if its maximum
// passes the K-th entry, so that after the first batches insertions are rare (K log(n) of them for values in random order).
// Rows of up to 1024 entries stay in the registers of 4 to 32 lanes.  Longer rows take a warp where the rows alone fill the device, a block of 4 or
// 8 warps where they do not, or, when there are few, a thread-block cluster of up to 8 blocks, which hand their sums and lists to the first
// one through distributed shared memory: a row needs neither a second launch nor a workspace.
// Bound, for long rows of 16-bit logits, by memory, with the exponentials close behind: 11.6 entries may arrive per cycle and SM, and the special
// function units return 16 exponentials.  Measured on a B200 (device time of a pass among passes over the same buffers; with buffers that change 3 to 8 % more,
// and cards differ by 5 %): 8192 rows of 50001 bf16 with entropy 138 us (91 % of the copy bandwidth; two bytes an entry), with four alternatives
// 165 us (the chains of the insertions, 20 a row), with 20 246 us; 38400 rows of 259 fp32 9 us (69 %); 8 rows of 131072 with a mask and eight
// alternatives 11.6 us, without alternatives 6.8 us, a launch and two trips to memory of it.  A mask makes long rows slow: 8192 rows of 32003 bf16 with a
// shared one 308 us (26 %), bytes are tested one by one and the registers spill.
// Backward: one read, one write.  8192 rows of 32003 bf16 that start anywhere 168 to 170 us (95 %), with a shared mask 281 us (57 %); 38400 of 259 fp32 18 us.
#include <math.h>

#include <cooperative_groups.h>

#include <initializer_list>

#include "typed.cuh"

namespace cg = cooperative_groups;

namespace b2 {
namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr unsigned FULL = 0xffffffffu;
constexpr int MAX_TOP = 32;

// The hardware's exponential, whatever the logits' type: its error of 2^-22 goes into a sum whose own roundings are as large (38400 rows of 259 fp32: 4.2e-8 off in
// the mean, a plain form with expf 4.1e-8).  Results below 2^-126 are 0.
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float max_nan(float a, float b) { float y; asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b)); return y; }
__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }

// z of two logits less what both subtract, z rounded.  Packed products and sums become one packed FMA in the assembler, rounding modifiers or not, and that
// subtracts from the unrounded product; one that is an FMA already, with -0 for its addend, stays as it is.  The -0 is made from the scale, where it can not be
// seen to be one.  With a scale that is a power of two the product needs no rounding, and the one FMA is right (8192 rows of 50001 with four alternatives: 180 us a pass, with
// two instructions 185 us).
struct Exact {
    Pair s, off;
    __device__ __forceinline__ Pair operator()(float x, float y) const { return fma2(pair(x, y), s, off); }
};
struct Rounded {
    Pair s, off, none;
    __device__ __forceinline__ Rounded(Pair s_, Pair off_, float scale) : s(s_), off(off_) {
        const float zero = __fmul_rn(scale, -0.0f);
        none = pair(zero, zero);
    }
    __device__ __forceinline__ Pair operator()(float x, float y) const { return add2(fma2(pair(x, y), s, none), off); }
};
// f(function of two logits), the one that the scale asks for
template <typename F> __device__ __forceinline__ void less_of(float scale, float minus, F &&f) {
    const Pair s = pair(scale, scale), off = pair(-minus, -minus);
    if ((__float_as_uint(scale) & 0x7fffffu) == 0) f(Exact{s, off});
    else f(Rounded(s, off, scale));
}

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

// ---- vectors of 16 bytes as they were loaded ------------------------------------------------------------------------------------------
template <typename T> struct Raw;
template <> struct Raw<float> {
    static constexpr unsigned NONE = 0xff800000u;      // -inf in every place of a word
    static __device__ __forceinline__ void values(float (&z)[4], const uint4 &q) {
        z[0] = __uint_as_float(q.x); z[1] = __uint_as_float(q.y); z[2] = __uint_as_float(q.z); z[3] = __uint_as_float(q.w);
    }
    static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b) { return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b))); }
    static __device__ __forceinline__ float largest(unsigned a) { return __uint_as_float(a); }
};
template <> struct Raw<__nv_bfloat16> {
    static constexpr unsigned NONE = 0xff80ff80u;
    static __device__ __forceinline__ float2 two(unsigned a) { return make_float2(__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u)); }
    static __device__ __forceinline__ void values(float (&z)[8], const uint4 &q) {
        const float2 a = two(q.x), b = two(q.y), c = two(q.z), d = two(q.w);
        z[0] = a.x; z[1] = a.y; z[2] = b.x; z[3] = b.y; z[4] = c.x; z[5] = c.y; z[6] = d.x; z[7] = d.y;
    }
    static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b) { unsigned y; asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b)); return y; }
    static __device__ __forceinline__ float largest(unsigned a) { const float2 v = two(a); return max_nan(v.x, v.y); }
};
template <> struct Raw<__half> {
    static constexpr unsigned NONE = 0xfc00fc00u;
    static __device__ __forceinline__ float2 two(unsigned a) { return __half22float2(*reinterpret_cast<const __half2 *>(&a)); }
    static __device__ __forceinline__ void values(float (&z)[8], const uint4 &q) {
        const float2 a = two(q.x), b = two(q.y), c = two(q.z), d = two(q.w);
        z[0] = a.x; z[1] = a.y; z[2] = b.x; z[3] = b.y; z[4] = c.x; z[5] = c.y; z[6] = d.x; z[7] = d.y;
    }
    static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b) { unsigned y; asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(y) : "r"(a), "r"(b)); return y; }
    static __device__ __forceinline__ float largest(unsigned a) { const float2 v = two(a); return max_nan(v.x, v.y); }
};
template <typename T> __device__ __forceinline__ unsigned larger_of(const uint4 &q) {
    typedef Raw<T> R;
    return R::larger(R::larger(q.x, q.y), R::larger(q.z, q.w));
}
// The sums over U vectors of logits x; top: their largest x (NaN if one is NaN).  A pair of entries costs two conversions, one packed maximum
// (by the caller), two packed FMAs, a packed product and sum, and two exponentials, with a scale that is no power of two a packed sum more.  Where an
// entry is -inf the sum of w * d turns NaN and is taken again with the differences held above -inf; SAFE does so at once.
template <typename T, int U, bool SAFE> __device__ __forceinline__ void add_vectors(Sums &a, const uint4 (&q)[U], float top, float scale) {
    constexpr int W = 16 / sizeof(T);
    const float m = __fmul_rn(top, scale);
    if (!(m <= a.m)) {
        if (a.m != neg_inf()) rescale(a, m); else a = {m, 0.0f, 0.0f};
    }
    if (a.m == neg_inf()) return;
    if (!SAFE) {
        const Pair l2 = pair(LOG2E, LOG2E);
        Pair s = 0, e = 0;
        less_of(scale, a.m, [&](const auto &less) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float x[W];
                Raw<T>::values(x, q[u]);
#pragma unroll
                for (int j = 0; j < W; j += 2) {
                    const Pair d = less(x[j], x[j + 1]);
                    const float2 t = halves(mul2(d, l2));
                    const Pair w = pair(ex2(t.x), ex2(t.y));
                    s = add2(s, w);
                    e = fma2(w, d, e);
                }
            }
        });
        const float2 sv = halves(s), ev = halves(e);
        const float en = ev.x + ev.y;
        if (en == en) {
            a.s += sv.x + sv.y;
            a.e += en;
            return;
        }
    }
    float s = 0.0f, e = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float x[W];
        Raw<T>::values(x, q[u]);
#pragma unroll
        for (int j = 0; j < W; ++j) {
            const float d = max_nan(__fmul_rn(x[j], scale) - a.m, -3.402823466e38f), w = ex2(d * LOG2E);
            s += w;
            e = fmaf(w, d, e);
        }
    }
    a.s += s;
    a.e += e;
}

// ---- the K largest ------------------------------------------------------------------------------------------------------------------
// An entry is one 64-bit key: the value as an ordered integer above, the complement of its index below; larger is better.  0 is no entry.
typedef unsigned long long Key;
__device__ __forceinline__ unsigned ordered(float z) {
    const unsigned b = __float_as_uint(z + 0.0f);           // -0 counts as 0
    return z != z ? FULL : (b ^ ((b >> 31) ? FULL : 0x80000000u));
}
__device__ __forceinline__ float ordered_value(unsigned o) { return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : FULL)); }
__device__ __forceinline__ Key make_key(float z, int index) { return ((Key)ordered(z) << 32) | (unsigned)~index; }
__device__ __forceinline__ float key_value(Key k) { return ordered_value((unsigned)(k >> 32)); }
__device__ __forceinline__ int key_index(Key k) { return (int)~(unsigned)k; }

// Lane l holds the l-th best of the warp, descending.  A value is of interest if it is not below `limit` (the K-th best, or a bound known
// from elsewhere) and above `floor`: the K-th best of the batches before the current one, whose indices are all lower, so that an equal
// value loses against it.
struct TopList {
    Key key, last;     // last: the K-th entry, the same in all lanes
    float limit, floor;
    __device__ __forceinline__ void clear() { key = last = 0; limit = floor = neg_inf(); }
    __device__ __forceinline__ bool wants(float z) const { return !(z < limit) && !(z <= floor); }
    __device__ __forceinline__ void insert(Key k, int K) {
        const int lane = threadIdx.x & 31;
        const int pos = __popc(__ballot_sync(FULL, key > k));
        const Key up = __shfl_up_sync(FULL, key, 1);
        if (lane >= pos) key = lane == pos ? k : up;
        last = __shfl_sync(FULL, key, K - 1);
        if (last) limit = fmaxf(limit, key_value(last));
    }
    __device__ __forceinline__ void settle() { if (last) floor = key_value(last); }
};
// Offers N values of every lane, those of value i at the indices at + i * 32 over the lanes.
template <int N> __device__ __forceinline__ void offer(TopList &t, const float (&z)[N], int at, int K) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        unsigned who = __ballot_sync(FULL, t.wants(z[i]));
        while (who) {
            const int src = __ffs(who) - 1;
            const Key k = make_key(__shfl_sync(FULL, z[i], src), at + i * 32 + src);
            if (k > t.last) t.insert(k, K);
            who &= who - 1;
            who &= __ballot_sync(FULL, t.wants(z[i]));
        }
    }
}
// Offers a batch of U vectors a lane, vector u of lane l at the indices at + (u * step + l) * W ...; top: the lane's largest logit.  A lane that
// has a candidate lays its vectors down in `spread`, and every lane looks at one entry (U * W <= 32).
template <typename T, int U>
__device__ __forceinline__ void offer_vectors(TopList &t, const uint4 (&q)[U], float top, float scale, int at, int step, uint4 *spread, int K) {
    constexpr int W = 16 / sizeof(T);
    static_assert(U * W <= 32, "an entry a lane");
    const int lane = threadIdx.x & 31;
    const float ztop = __fmul_rn(top, scale);
    unsigned who = __ballot_sync(FULL, t.wants(ztop));
    while (who) {
        const int src = __ffs(who) - 1;
        if (lane == src)
#pragma unroll
            for (int u = 0; u < U; ++u) spread[u] = q[u];
        __syncwarp();
        const float z = lane < U * W ? __fmul_rn(to_float(reinterpret_cast<const T *>(spread)[lane]), scale) : neg_inf();
        __syncwarp();
        unsigned which = __ballot_sync(FULL, t.wants(z));
        while (which) {
            const int e = __ffs(which) - 1;
            const Key k = make_key(__shfl_sync(FULL, z, e), at + (e / W * step + src) * W + e % W);
            if (k > t.last) t.insert(k, K);
            which &= which - 1;
            which &= __ballot_sync(FULL, t.wants(z));
        }
        who &= who - 1;
        who &= __ballot_sync(FULL, t.wants(ztop));
    }
    t.settle();
}
// The 32 lanes' values in descending order (NaN counts as +inf): at least k + 1 values of the warp reach that of lane k.
__device__ __forceinline__ float sort_lanes(float v) {
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
    return v;
}
// The best K of N lists, put in order into out.  Every list holds 32 keys, descending, 0 behind the last; thread (warp l, lane j) brings key j
// of list l.  A key's place is the number of larger keys, found by bisection in every list.  out holds zeros before; the caller's
// barriers stand before and behind.
template <int N> __device__ __forceinline__ void join_lists(Key *out, const Key (*lists)[MAX_TOP], Key mine, int K) {
    if (!mine) return;
    int at[N];
#pragma unroll
    for (int l = 0; l < N; ++l) at[l] = 0;
#pragma unroll
    for (int s = 16; s > 0; s >>= 1)
#pragma unroll
        for (int l = 0; l < N; ++l) at[l] += lists[l][at[l] + s - 1] > mine ? s : 0;
    int place = 0;
#pragma unroll
    for (int l = 0; l < N; ++l) place += at[l] + (lists[l][31] > mine);
    if (place < K) out[place] = mine;
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
        best.limit = __shfl_sync(FULL, sort_lanes(top), a.top - 1);
        offer<NV>(best, z, 0, a.top);
        write_top(a, r, best.key, t, ls);
    }
}

// Several rows a warp, for rows of which no alternatives are asked: G lanes a row, NV vectors a lane.  The reductions and the row's closing
// arithmetic then serve 32 / G rows at once; they are as much work as 100 entries.
template <typename T, int G, int NV> __global__ void __launch_bounds__(256) logprob_rows_kernel(const T *__restrict__ logits, const FwdArgs a) {
    constexpr int W = 16 / sizeof(T);
    const int lane = threadIdx.x & (G - 1);
    const long long at = ((long long)blockIdx.x * 256 + threadIdx.x) / G, r = at < a.rows ? at : a.rows - 1;
    const T *x = logits + r * a.ld;
    const int mis = (int)(((uintptr_t)x & 15) / sizeof(T)), end = mis + a.vocab;
    const T *base = x - mis;
    uint4 q[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int v = (lane + G * i) * W;
        q[i] = make_uint4(Raw<T>::NONE, Raw<T>::NONE, Raw<T>::NONE, Raw<T>::NONE);
        if (v >= mis && v + W <= end) q[i] = __ldg(reinterpret_cast<const uint4 *>(base + v));
    }
    // the row's first and last entries, where their vectors are shared with the neighbours
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int v = (lane + G * i) * W;
        if (v >= end || (v >= mis && v + W <= end)) continue;
        Vec<T, W> part_of = *reinterpret_cast<const Vec<T, W> *>(&q[i]);
#pragma unroll
        for (int j = 0; j < W; ++j)
            if (v + j >= mis && v + j < end) part_of.v[j] = base[v + j];
        q[i] = *reinterpret_cast<const uint4 *>(&part_of);
    }
    Given g = {-1, 0.0f};
    if (at < a.rows && lane == 0) g = load_given(a, r, x);
    if (a.mask) {
        const unsigned char *mk = a.mask + r * a.ld_mask;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            Vec<T, W> part_of = *reinterpret_cast<const Vec<T, W> *>(&q[i]);
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const int e = (lane + G * i) * W + j - mis;
                if (e >= 0 && e < a.vocab && !mk[e]) part_of.v[j] = from_float<T>(neg_inf());
            }
            q[i] = *reinterpret_cast<const uint4 *>(&part_of);
        }
    }
    unsigned most = larger_of<T>(q[0]);
#pragma unroll
    for (int i = 1; i < NV; ++i) most = Raw<T>::larger(most, larger_of<T>(q[i]));
    float top = Raw<T>::largest(most);
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(FULL, top, o));
    Sums t = {__fmul_rn(top, a.scale), 0.0f, 0.0f};
    if (t.m != neg_inf()) {
        const Rounded less(pair(a.scale, a.scale), pair(-t.m, -t.m), a.scale);
        const Pair l2 = pair(LOG2E, LOG2E);
        Pair s = 0, e = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float z[W];
            Raw<T>::values(z, q[i]);
#pragma unroll
            for (int j = 0; j < W; j += 2) {
                const float2 v = halves(less(z[j], z[j + 1]));
                const Pair d = pair(max_nan(v.x, -3.402823466e38f), max_nan(v.y, -3.402823466e38f));   // as in add_values
                const float2 y = halves(mul2(d, l2));
                const Pair w = pair(ex2(y.x), ex2(y.y));
                s = add2(s, w);
                e = fma2(w, d, e);
            }
        }
        const float2 sv = halves(s), ev = halves(e);
        t.s = sv.x + sv.y;
        t.e = ev.x + ev.y;
    }
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) {
        t.s += __shfl_xor_sync(FULL, t.s, o);
        t.e += __shfl_xor_sync(FULL, t.e, o);
    }
    if (at < a.rows && lane == 0) write_row(a, r, g, t);
}

// blocks_per_row blocks a row (a thread-block cluster where there are several).  Entries are taken in vectors of W = 16 bytes from the
// 16-byte boundary at or below the row's start, U vectors a thread and batch; the next batch is on its way while one is worked on.
template <typename T, int THREADS, bool TOP, bool MASK>
__global__ void __launch_bounds__(THREADS, 640 / THREADS) logprob_row_kernel(const T *__restrict__ logits, const FwdArgs a, int blocks_per_row) {
    constexpr int W = 16 / sizeof(T), U = 4, WARPS = THREADS / 32, MOST = 8;
    __shared__ Sums sums[WARPS], all_sums[MOST];
    __shared__ Key lists[WARPS][MAX_TOP], all_lists[MOST][MAX_TOP], joined[3][MAX_TOP];
    __shared__ uint4 spread[WARPS][U];
    __shared__ unsigned block_limit;                         // the highest limit of the block's warps, as an ordered integer
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const long long r = blockIdx.x / (unsigned)blocks_per_row;
    const int part = (int)(blockIdx.x % (unsigned)blocks_per_row);
    // the first block's shared memory may be written once that block runs: arrive here, wait before the write
    if (blocks_per_row > 1) {
        if (TOP && w < MOST) all_lists[w][lane] = 0;         // a cluster has 8 warps a block
        cg::this_cluster().barrier_arrive();
    }
    const T *x = logits + r * a.ld;
    const unsigned char *mk = MASK ? a.mask + r * a.ld_mask : nullptr;
    const int mis = (int)(((uintptr_t)x & 15) / sizeof(T));
    const T *base = x - mis;
    const int end = mis + a.vocab, vecs = (end + W - 1) / W; // vector v holds the entries v * W - mis ...
    const int v0 = (int)((long long)vecs * part / blocks_per_row), v1 = (int)((long long)vecs * (part + 1) / blocks_per_row);
    const bool mask_vec = MASK && ((uintptr_t)(mk - mis) & (W - 1)) == 0;
    typedef Vec<unsigned char, W> Allowed;
    const auto load = [&](uint4 (&q)[U], Allowed (&on)[U], int b) {
        const int last = b + THREADS * (U - 1) + 32;         // one behind the batch's last vector
        if ((b > 0 || mis == 0) && last <= v1 && last * W <= end) {
#pragma unroll
            for (int u = 0; u < U; ++u) q[u] = __ldg(reinterpret_cast<const uint4 *>(base + (size_t)(b + u * THREADS + lane) * W));
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int v = b + u * THREADS + lane;
                q[u] = make_uint4(Raw<T>::NONE, Raw<T>::NONE, Raw<T>::NONE, Raw<T>::NONE);
                if (v >= v1) continue;
                if (v * W >= mis && (v + 1) * W <= end) q[u] = __ldg(reinterpret_cast<const uint4 *>(base + (size_t)v * W));
                else {
                    Vec<T, W> part_of = *reinterpret_cast<const Vec<T, W> *>(&q[u]);
#pragma unroll
                    for (int j = 0; j < W; ++j)
                        if (v * W + j >= mis && v * W + j < end) part_of.v[j] = base[v * W + j];
                    q[u] = *reinterpret_cast<const uint4 *>(&part_of);
                }
            }
        }
        if (MASK) {
            if (mask_vec && (b > 0 || mis == 0) && last <= v1 && last * W <= end) {
#pragma unroll
                for (int u = 0; u < U; ++u) on[u] = *reinterpret_cast<const Allowed *>(mk - mis + (b + u * THREADS + lane) * W);
            } else {
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int j = 0; j < W; ++j) {
                        const int v = b + u * THREADS + lane, i = v * W + j;
                        on[u].v[j] = v < v1 && i >= mis && i < end ? mk[i - mis] : 0;
                    }
            }
        }
    };
    const auto rule_out = [&](uint4 (&q)[U], const Allowed (&on)[U]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            unsigned *word = reinterpret_cast<unsigned *>(&q[u]);
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const unsigned place = sizeof(T) == 4 ? FULL : 0xffffu << (16 * (j & 1));
                if (!on[u].v[j]) word[j * (int)sizeof(T) / 4] = (word[j * (int)sizeof(T) / 4] & ~place) | (Raw<T>::NONE & place);
            }
        }
    };
    Given g = {-1, 0.0f};
    Sums t = {neg_inf(), 0.0f, 0.0f};
    TopList best;
    best.clear();
    uint4 now[U], next[U];
    Allowed on[U], on_next[U];
    int b = v0 + w * 32;
    if (b < v1) load(now, on, b);
    if (part == 0 && threadIdx.x == 0) g = load_given(a, r, x);
    const auto largest = [&](const uint4 (&q)[U]) {
        unsigned most = larger_of<T>(q[0]);
#pragma unroll
        for (int u = 1; u < U; ++u) most = Raw<T>::larger(most, larger_of<T>(q[u]));
        return Raw<T>::largest(most);
    };
    const auto post = [&](float limit) {
        if (lane == 0 && limit > neg_inf()) atomicMax(&block_limit, ordered(limit));
    };
    if (TOP) {
        // a bound from the first batches, so that the lists do not fill up with what will not stay: the K-th largest of all lanes' maxima
        if (MASK && b < v1) rule_out(now, on);
        const float most = sort_lanes(b < v1 ? __fmul_rn(largest(now), a.scale) : neg_inf());
        if (WARPS == 1) best.limit = __shfl_sync(FULL, most, a.top - 1);
        else {
            const Key key = lane < a.top ? make_key(most, w * 32 + lane) : 0;
            lists[w][lane] = key;
            if (w < 3) joined[w][lane] = 0;
            if (threadIdx.x == 0) block_limit = 0;
            __syncthreads();
            join_lists<WARPS>(joined[0], lists, key, a.top);
            __syncthreads();
            best.limit = key_value(joined[0][a.top - 1]);
        }
    }
    for (; b < v1; b += THREADS * U) {
        if (b + THREADS * U < v1) load(next, on_next, b + THREADS * U);
        if (MASK) rule_out(now, on);
        const float top = largest(now);
        add_vectors<T, U, MASK>(t, now, top, a.scale);
        if (TOP) {
            if (WARPS > 1) {
                const unsigned known = *(volatile unsigned *)&block_limit;
                if (known) best.limit = fmaxf(best.limit, ordered_value(known));
            }
            if (__any_sync(FULL, best.wants(__fmul_rn(top, a.scale)))) {
                offer_vectors<T, U>(best, now, top, a.scale, b * W - mis, THREADS, spread[w], a.top);
                if (WARPS > 1) post(best.limit);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            now[u] = next[u];
            if (MASK) on[u] = on_next[u];
        }
    }
    t = warp_merge(t);
    Key k = best.key;
    if (WARPS > 1) {
        if (lane == 0) sums[w] = t;
        if (lane >= a.top) k = 0;
        if (TOP) lists[w][lane] = k;
        __syncthreads();
        if (w == 0) t = warp_merge(lane < WARPS ? sums[lane] : Sums{neg_inf(), 0.0f, 0.0f});
        if (TOP) {
            join_lists<WARPS>(joined[1], lists, k, a.top);
            __syncthreads();
            k = joined[1][lane];
        }
    }
    if (blocks_per_row > 1) {
        // the row's blocks hand over to the first
        cg::cluster_group cluster = cg::this_cluster();
        cluster.barrier_wait();
        if (w == 0) {
            if (lane == 0) *cluster.map_shared_rank(&all_sums[part], 0) = t;
            if (TOP) *cluster.map_shared_rank(&all_lists[part][lane], 0) = k;
        }
        cluster.sync();
        if (part != 0) return;
        if (w == 0) t = warp_merge(lane < blocks_per_row ? all_sums[lane] : Sums{neg_inf(), 0.0f, 0.0f});
        if (TOP) {
            if (w < blocks_per_row) join_lists<MOST>(joined[2], all_lists, all_lists[w][lane], a.top);
            __syncthreads();
            k = joined[2][lane];
        }
    }
    if (w == 0) {
        float ls = 0.0f;
        if (lane == 0) ls = write_row(a, r, g, t);
        if (TOP) write_top(a, r, k, t, __shfl_sync(FULL, ls, 0));
    }
}

template <typename T, int THREADS, bool TOP, bool MASK> int launch_rows(const T *logits, const FwdArgs &a, cudaStream_t st) {
    constexpr int W = 16 / sizeof(T);
    // few rows: several blocks a row, as long as each has at least a batch
    int per_row = 1;
    while (THREADS == 256 && per_row < 8 && a.rows * per_row * 2 <= 2 * sm_count() && (a.vocab / (per_row * 2)) >= THREADS * 4 * W) per_row *= 2;
    if (a.rows * per_row > 0x7fffffffll) { set_error("b2_logprob_forward: %lld rows", a.rows); return B2_ERR_BAD_SHAPE; }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * per_row));
    cfg.blockDim = dim3(THREADS);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = per_row;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = per_row > 1 ? 1 : 0;
    count_launch();
    B2_CUDA(cudaLaunchKernelEx(&cfg, logprob_row_kernel<T, THREADS, TOP, MASK>, logits, a, per_row));
    return B2_OK;
}

template <typename T> int forward(const T *logits, const FwdArgs &a, cudaStream_t st) {
    if (a.vocab <= 1024 && !a.top) {
        const auto go = [&](auto kernel, int lanes) -> int {
            const long long blocks = (a.rows * lanes + 255) / 256;
            if (blocks > 0x7fffffffll) { set_error("b2_logprob_forward: %lld rows", a.rows); return B2_ERR_BAD_SHAPE; }
            kernel<<<(unsigned)blocks, 256, 0, st>>>(logits, a);
            count_launch();
            B2_CUDA(cudaGetLastError());
            return B2_OK;
        };
        constexpr int W = 16 / sizeof(T), NV = W == 4 ? 9 : 5;
        const int vecs = (a.vocab + W - 1) / W + 1;           // one more: a row may start inside a vector
        if (vecs <= 4 * NV) return go(logprob_rows_kernel<T, 4, NV>, 4);
        if (vecs <= 8 * NV) return go(logprob_rows_kernel<T, 8, NV>, 8);
        if (vecs <= 16 * NV) return go(logprob_rows_kernel<T, 16, NV>, 16);
        return go(logprob_rows_kernel<T, 32, NV>, 32);
    }
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
    // What a warp does once a row (its first list, the joins) is the less the fewer warps a row has: one where the rows alone fill the device
    // (8192 rows of 50001, four alternatives: 165 us, with four warps 231, with eight 340), four for some rows (1200 rows of 200000: 112 us, with one warp 147, with
    // eight 133)
    const auto go = [&](auto threads) -> int {
        constexpr int N = decltype(threads)::value;
        if (a.top) return a.mask ? launch_rows<T, N, true, true>(logits, a, st) : launch_rows<T, N, true, false>(logits, a, st);
        return a.mask ? launch_rows<T, N, false, true>(logits, a, st) : launch_rows<T, N, false, false>(logits, a, st);
    };
    if (a.rows >= 16 * sm_count()) return go(std::integral_constant<int, 32>());
    if (a.rows >= 4 * sm_count()) return go(std::integral_constant<int, 128>());
    return go(std::integral_constant<int, 256>());
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
// fp32 gradients with the exponential of the full accuracy, 16-bit ones with the hardware's: its error of 2^-22 is lost in their rounding (and a probability
// below 2^-126 is 0)
template <typename T> __device__ __forceinline__ Pair exp_pair(Pair x) {
    const float2 v = halves(sizeof(T) == 4 ? x : mul2(x, pair(LOG2E, LOG2E)));
    return sizeof(T) == 4 ? pair(expf(v.x), expf(v.y)) : pair(ex2(v.x), ex2(v.y));
}
// What a row's entries share: dx = p (c0 + c1 log p) with c0 = -s (g + h H), c1 = -s h, and s g more at the token.
struct RowGrad { float lse, c0, c1, at_token; int tok; };
// N entries from index i0 on
template <typename T, int N, bool ENT> __device__ __forceinline__ void entry_grads(float (&o)[N], const float (&x)[N], const RowGrad &q, float scale, int i0) {
    const Pair c0 = pair(q.c0, q.c0), c1 = pair(q.c1, q.c1);
    less_of(scale, q.lse, [&](const auto &less) {
#pragma unroll
        for (int j = 0; j < N; j += 2) {
            Pair lp = less(x[j], x[j + 1]);
            if (ENT) {
                // below -1000 the probability is 0 whatever the logarithm is; -inf must not meet that 0
                const float2 v = halves(lp);
                lp = pair(max_nan(v.x, -1000.0f), max_nan(v.y, -1000.0f));
            }
            const float2 d = halves(mul2(exp_pair<T>(lp), ENT ? fma2(lp, c1, c0) : c0));
            o[j] = d.x;
            o[j + 1] = d.y;
        }
    });
    if ((unsigned)(q.tok - i0) < (unsigned)N)
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (i0 + j == q.tok) o[j] += q.at_token;
}

// tpr threads a row, each up to U vectors apart by tpr; a long row takes several blocks.  Bound by memory (5 to 6 issue slots an entry).
template <typename T, bool ENT, bool MASK, int U>
__global__ void __launch_bounds__(256) logprob_backward_kernel(T *dlogits, const T *logits, const BwdArgs a, int tpr, int segs) {
    constexpr int W = 16 / sizeof(T);
    const int per_block = 256 / tpr;
    // a row of several segments takes whole blocks (tpr = 256)
    const long long r = segs > 1 ? (long long)(blockIdx.x / (unsigned)segs) : (long long)blockIdx.x * per_block + threadIdx.x / tpr;
    const int seg = segs > 1 ? (int)(blockIdx.x % (unsigned)segs) : 0;
    if (r >= a.rows) return;
    const T *x = logits + r * a.ld;
    T *d = dlogits + r * a.ld_out;
    const int mis = (int)(((uintptr_t)x & 15) / sizeof(T));
    const bool out_vec = (((uintptr_t)(d - mis)) & 15) == 0;
    const int first = seg * tpr * U + (threadIdx.x & (tpr - 1));
    const auto whole = [&](int v) { return v * W >= mis && (v + 1) * W <= mis + a.vocab; };
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (whole(first + u * tpr)) raw[u] = *reinterpret_cast<const uint4 *>(x - mis + (size_t)(first + u * tpr) * W);
    RowGrad q;
    q.tok = __ldg(a.tokens + r);
    const float lse = __ldg(a.lse + r), g = a.dlogprob ? __ldg(a.dlogprob + r) : 0.0f, h = ENT ? __ldg(a.dentropy + r) : 0.0f;
    q.lse = lse;
    q.c0 = -a.scale * (ENT ? fmaf(h, __ldg(a.entropy + r), g) : g);
    q.c1 = -a.scale * h;
    q.at_token = a.scale * g;
    // padding, and a row that allows nothing: no gradient.  A token beyond the vocabulary shows as NaN, as its log probability does.
    const bool zero = q.tok < 0 || lse == neg_inf();
    if (q.tok >= a.vocab) q.c0 = nanf("");
    const unsigned char *mk = MASK ? a.mask + r * a.ld_mask : nullptr;
    const bool mask_vec = MASK && ((uintptr_t)(mk - mis) & (W - 1)) == 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int v = first + u * tpr, i0 = v * W - mis;
        if (i0 >= a.vocab) break;
        const bool inside = whole(v);
        float z[W], o[W];
        if (inside) Raw<T>::values(z, raw[u]);
        else
#pragma unroll
            for (int j = 0; j < W; ++j) z[j] = i0 + j >= 0 && i0 + j < a.vocab ? to_float(x[i0 + j]) : 0.0f;
        if (zero) {
#pragma unroll
            for (int j = 0; j < W; ++j) o[j] = 0.0f;
        } else {
            entry_grads<T, W, ENT>(o, z, q, a.scale, i0);
            if (MASK) {
                Vec<unsigned char, W> on;
                if (inside && mask_vec) on = *reinterpret_cast<const Vec<unsigned char, W> *>(mk + i0);
                else
#pragma unroll
                    for (int j = 0; j < W; ++j) on.v[j] = i0 + j >= 0 && i0 + j < a.vocab ? mk[i0 + j] : 0;
#pragma unroll
                for (int j = 0; j < W; ++j) o[j] = on.v[j] ? o[j] : 0.0f;
            }
        }
        if (inside && out_vec) store_vec<T, W>(d + i0, o);
        else
#pragma unroll
            for (int j = 0; j < W; ++j)
                if (i0 + j >= 0 && i0 + j < a.vocab) d[i0 + j] = from_float<T>(o[j]);
    }
}

template <typename T, bool ENT, bool MASK> int backward(T *dlogits, const T *logits, const BwdArgs &a, cudaStream_t st) {
    constexpr int W = 16 / sizeof(T);
    const int vecs = (a.vocab + W - 1) / W + 1;               // one more: a row may start inside a vector
    const auto go = [&](auto vectors) -> int {
        constexpr int U = decltype(vectors)::value;
        unsigned tpr = pow2_at_least((unsigned)((vecs + U - 1) / U));
        if (tpr > 256) tpr = 256;
        const int segs = (vecs + (int)tpr * U - 1) / ((int)tpr * U);
        const long long per = 256 / tpr, blocks = (a.rows * segs + per - 1) / per;
        if (blocks > 0x7fffffffll) { set_error("b2_logprob_backward: %lld rows of %d", a.rows, a.vocab); return B2_ERR_BAD_SHAPE; }
        logprob_backward_kernel<T, ENT, MASK, U><<<(unsigned)blocks, 256, 0, st>>>(dlogits, logits, a, (int)tpr, segs);
        count_launch();
        B2_CUDA(cudaGetLastError());
        return B2_OK;
    };
    // Vectors of a thread: 2 where the rows do not fill the device (16 rows of 32003: 2.5 us, with 8 3.9 us), else 8 (8192 rows: 167 us, with 4 171 us,
    // with 2 191 us), with a mask 4 (shared: 280 us, with 8 347 us, with 2 303 us; a mask a row: 310, 366, 305 us)
    if ((double)a.rows * vecs < 4096.0 * sm_count()) return go(std::integral_constant<int, 2>());
    return go(std::integral_constant<int, MASK ? 4 : 8>());
}

// vectors of 4-byte numbers, one a row
bool misaligned(const char *who, std::initializer_list<const void *> all) {
    for (const void *p : all)
        if (!aligned_to(p, 4)) { set_error("%s: a vector of tokens or numbers is not aligned to 4 bytes", who); return true; }
    return false;
}
int check(const char *who, const void *logits, int type, long long rows, int vocab, long long ld, const unsigned char *mask, long long ld_mask, float scale) {
    const int e = type_size(type);
    if (!e) { set_error("%s: unknown element type %d", who, type); return B2_ERR_BAD_ARG; }
    if (rows < 0 || vocab < 1 || vocab > (1 << 27)) { set_error("%s: %lld rows of %d logits (at most 2^27)", who, rows, vocab); return B2_ERR_BAD_SHAPE; }
    if (ld < vocab || ld > MAX_LD || (mask && ((ld_mask != 0 && ld_mask < vocab) || ld_mask > MAX_LD))) {
        set_error("%s: leading dimension too small or beyond 2^40 (logits %lld, mask %lld for %d columns)", who, ld, ld_mask, vocab);
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
    if (misaligned("b2_logprob_forward", {tokens_dev, logprob, lse, entropy, top_tokens, top_logprobs})) return B2_ERR_BAD_ARG;
    const FwdArgs a = {mask, ld_mask, tokens_dev, logprob, lse, entropy, top_logprobs, top_tokens, rows, ld, vocab, top, scale};
    return with_type(type, [&](auto *t) { return forward((const B2_ELEM(t) *)logits, a, (cudaStream_t)stream); });
}

int b2_logprob_backward(void *dlogits, long long ld_dlogits, const void *logits, int type, long long rows, int vocab, long long ld, const unsigned char *mask,
                        long long ld_mask, float scale, const int *tokens_dev, const float *lse, const float *dlogprob, const float *entropy, const float *dentropy,
                        b2_stream stream) {
    B2_TRY(check("b2_logprob_backward", logits, type, rows, vocab, ld, mask, ld_mask, scale));
    if (ld_dlogits < vocab || ld_dlogits > MAX_LD) {
        set_error("b2_logprob_backward: leading dimension too small or beyond 2^40 (gradient %lld for %d columns)", ld_dlogits, vocab);
        return B2_ERR_BAD_ARG;
    }
    if (!rows) return B2_OK;
    if (!dlogits || !aligned_to(dlogits, type_size(type))) { set_error("b2_logprob_backward: the gradient is missing or not aligned to its elements"); return B2_ERR_BAD_ARG; }
    if (!tokens_dev || !lse || (dentropy && !entropy)) { set_error("b2_logprob_backward: null pointer"); return B2_ERR_BAD_ARG; }
    if (dlogits == logits && ld_dlogits != ld) { set_error("b2_logprob_backward: in place with another leading dimension"); return B2_ERR_BAD_ARG; }
    if (misaligned("b2_logprob_backward", {tokens_dev, lse, dlogprob, entropy, dentropy})) return B2_ERR_BAD_ARG;
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
