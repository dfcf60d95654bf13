// Norms before and after a residual block, fused with the block's gate and residual scale, and their gradients.
//
//   n = w2 * norm(f) + b2        the block's output f normalised (after the block)
//   y = x + a * gate * n         gated, scaled and added to the residual stream
//   h = w1 * norm(y) + b1        normalised for the next block (before it)
//
// norm(v) = (v - mean) / sqrt(var + eps) (layer norm) or v / sqrt(mean(v^2) + eps) (RMS norm).  y is rounded to the tensors' type before the
// second norm, so that a backward pass that reads y differentiates what the forward pass computed.  The gate has gate_rows rows; frame r
// takes row r % gate_rows: one row for all frames, one for each of the parallel sequences of a time-major fraction, or one per frame.
//
// Backward, with u1 = (y - m1) r1, u2 = (f - m2) r2 and d the gradients coming in:
//   dt = dy + r1 (w1 dh - [mean(w1 dh)] - u1 mean(w1 dh u1)),   dx = dt,   dn = a gate dt,   dgate = a dt n
//   df = r2 (w2 dn - [mean(w2 dn)] - u2 mean(w2 dn u2)),   dw1 = sum dh u1, db1 = sum dh, dw2 = sum dn u2, db2 = sum dn   (over frames)
//
// Bound by memory: a row stays in registers between its loads and its stores, so every tensor is read once and written once.  A warp
// takes a row where 4 vectors a lane hold it, a block otherwise.  The backward kernel has a fixed number of workers; a worker keeps
// the same columns for all its rows, so the sums over frames stay in registers until the end, go to the workspace once, and are
// added there in a fixed order by a second launch: no atomics, the same bits every time.
#include <math.h>

#include "typed.cuh"

namespace b2 {
namespace {

constexpr int MAX_DIM = 8192;

struct NormArgs {
    const char *pat;
    const float *w1, *b1, *w2, *b2;
    const void *gate;
    float4 *stats;                    // per row: mean and 1/deviation of f, of y
    long long rows, gate_rows, ld_gate;
    int dim, layer_norm;
    float eps, a, inv_dim;
};

// Sums over the threads of a row: a warp, or all warps of the block (buffers alternate, so one barrier a sum is enough).  red holds 2 * N * 32
// floats; those of warps that are not there are zero.
template <int N> __device__ __forceinline__ void row_sums(float (&x)[N], int warps, float4 (*red)[8], int &phase) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = warp_sum(x[i]);
    if (warps == 1) return;
    float4(*buf)[8] = red + (phase & 1) * N;
    ++phase;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) reinterpret_cast<float *>(buf[i])[threadIdx.x >> 5] = x[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float4 s = buf[i][0];
        for (int k = 1; k < (warps + 3) >> 2; ++k) {
            const float4 y = buf[i][k];
            s.x += y.x; s.y += y.y; s.z += y.z; s.w += y.w;
        }
        x[i] = (s.x + s.y) + (s.z + s.w);
    }
}
__device__ __forceinline__ void clear_sums(float4 *red, int n) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) red[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    __syncthreads();
}

// columns of a thread: vector i starts at column (i * tpr + lane) * W
template <typename T, int W, int NV, bool FULL = false> struct Cols {
    static __device__ __forceinline__ void load(float (&v)[NV][W], const T *row, int tpr, int lane, int dim, float other) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * tpr + lane) * W;
            if (FULL || c < dim) load_vec<T, W>(v[i], row + c);
            else
#pragma unroll
                for (int j = 0; j < W; ++j) v[i][j] = other;
        }
    }
    static __device__ __forceinline__ void store(T *row, const float (&v)[NV][W], int tpr, int lane, int dim) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * tpr + lane) * W;
            if (FULL || c < dim) store_vec<T, W>(row + c, v[i]);
        }
    }
};

// v becomes its normalised self; columns beyond dim are zero before and stay so
template <int W, int NV>
__device__ __forceinline__ void normalise(float (&v)[NV][W], const NormArgs &a, int tpr, int lane, int warps, float4 (*red)[8], int &phase, float &mean, float &rstd) {
    float s[1] = {0.0f};
    mean = 0.0f;
    if (a.layer_norm) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) s[0] += v[i][j];
        row_sums<1>(s, warps, red, phase);
        mean = s[0] * a.inv_dim;
        s[0] = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if ((i * tpr + lane) * W < a.dim)
#pragma unroll
                for (int j = 0; j < W; ++j) v[i][j] -= mean;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) s[0] = fmaf(v[i][j], v[i][j], s[0]);
    row_sums<1>(s, warps, red, phase);
    rstd = 1.0f / sqrtf(fmaf(s[0], a.inv_dim, a.eps));
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) v[i][j] *= rstd;
}

template <int W, int NV> __device__ __forceinline__ void affine(float (&v)[NV][W], const float *w, const float *b, int tpr, int lane, int dim) {
    float q[NV][W];
    if (w) {
        Cols<float, W, NV>::load(q, w, tpr, lane, dim, 0.0f);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) v[i][j] *= q[i][j];
    }
    if (b) {
        Cols<float, W, NV>::load(q, b, tpr, lane, dim, 0.0f);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) v[i][j] += q[i][j];
    }
}

// tpr threads a row: 32 (the block holds 8 rows) or the whole block
template <typename T, int W, int NV>
__global__ void __launch_bounds__(NV == 8 ? 1024 : 512) block_norm_forward_kernel(const NormArgs a, const T *x, long long ld_x, const T *f, long long ld_f, T *y,
                                                                                  long long ld_y, T *h, long long ld_h, int tpr) {
    __shared__ float4 red[2][8];
    const int warps = tpr >> 5, lane = warps == 1 ? (threadIdx.x & 31) : threadIdx.x;
    const long long r = warps == 1 ? (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    if (r >= a.rows) return;
    if (warps > 1) clear_sums(red[0], 16);
    int phase = 0;
    typedef Cols<T, W, NV> C;
    float v[NV][W], n[NV][W];
    float4 st = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (a.pat && a.pat[r] == PAT_NONE) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) v[i][j] = 0.0f;
        if (y) C::store(y + r * ld_y, v, tpr, lane, a.dim);
        if (h) C::store(h + r * ld_h, v, tpr, lane, a.dim);
        if (a.stats && lane == 0) a.stats[r] = st;
        return;
    }
    C::load(v, x + r * ld_x, tpr, lane, a.dim, 0.0f);
    if (f) {
        float g[NV][W];
        C::load(n, f + r * ld_f, tpr, lane, a.dim, 0.0f);
        if (a.gate) C::load(g, (const T *)a.gate + (r % a.gate_rows) * a.ld_gate, tpr, lane, a.dim, 0.0f);
        normalise<W, NV>(n, a, tpr, lane, warps, red, phase, st.x, st.y);
        affine<W, NV>(n, a.w2, a.b2, tpr, lane, a.dim);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const float s = a.gate ? a.a * g[i][j] : a.a;
                v[i][j] = to_float(from_float<T>(fmaf(s, n[i][j], v[i][j])));
            }
    }
    if (y) C::store(y + r * ld_y, v, tpr, lane, a.dim);
    if (h) {
        normalise<W, NV>(v, a, tpr, lane, warps, red, phase, st.z, st.w);
        affine<W, NV>(v, a.w1, a.b1, tpr, lane, a.dim);
        C::store(h + r * ld_h, v, tpr, lane, a.dim);
    }
    if (a.stats && lane == 0) a.stats[r] = st;
}

struct BackArgs {
    unsigned ld_dx, ld_df, ld_dy, ld_dh, ld_y, ld_f, ld_dgate;
    void *dgate;
    float *partial;                   // [blocks][4][dim_pad]: dw1, db1, dw2, db2 of every block
    float *partial_gate;              // [workers][dim_pad], where several workers share a row of the gate
    int dim_pad, per_group, groups_at_once;
};

// Copies of 16 bytes (the first `bytes` of them, zeros behind) into shared memory that nobody waits for before cp_wait
__device__ __forceinline__ void cp_async(unsigned to, const void *from, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async(unsigned to, const void *from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// until at most n (0 to 2) of the newest groups are under way
__device__ __forceinline__ void cp_wait(int n) {
    if (n == 0) asm volatile("cp.async.wait_group 0;" ::: "memory");
    else if (n == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 2;" ::: "memory");
}

// The rows a worker takes, one after another: rows member, member + per_group, ... of the R frames that share a row of the gate, for every
// such group of the worker.
struct RowWalk {
    int g, m, G, R, member, per_group, groups;
    __device__ __forceinline__ bool ended() const { return g >= G; }
    __device__ __forceinline__ unsigned row() const { return (unsigned)m * (unsigned)G + (unsigned)g; }
    __device__ __forceinline__ bool last_of_group() const { return (long long)m + per_group >= R; }
    __device__ __forceinline__ void next() {
        if (last_of_group()) { m = member; g = groups < G - g ? g + groups : G; } else m += per_group;
    }
};

// Stores a thread's columns, held as pairs
template <int W, int NV, bool FULL> struct Out {
    int tpr, lane, dim;
    template <typename T> __device__ __forceinline__ void operator()(T *to, const Pair (&v)[NV * W / 2]) const {
        float q[NV][W];
#pragma unroll
        for (int n = 0; n < NV * W / 2; ++n) {
            const float2 x = halves(v[n]);
            q[2 * n / W][2 * n % W] = x.x;
            q[(2 * n + 1) / W][(2 * n + 1) % W] = x.y;
        }
        Cols<T, W, NV, FULL>::store(to, q, tpr, lane, dim);
    }
};

// A worker is a warp (tpr = 32) or a block.  per_group workers share a row of the gate (all workers, if there is one row or none), and
// groups_at_once rows of the gate are worked on side by side.  BIAS: means are subtracted or the norms have a bias (without both, sums are saved).
// FULL: dy, dh, f, dx and df are all there and the threads' columns are just the row's: a third of the instructions were tests of that.
// The next `stages` - 1 rows are on their way into shared memory while one is worked on: what a row's two sums over the threads leave idle
// would otherwise be the memory.  With whole vectors a thread copies the vectors that it will read; rows that start anywhere (W = 1) are
// copied as the 16-byte pieces that hold them, by all their threads, and read element by element, so that loads and stores stay coalesced.
template <typename T, int W, int NV, int MAXT, bool BIAS, bool FULL>
__global__ void __launch_bounds__(MAXT, MAXT <= 256 ? 2 : 1) block_norm_backward_kernel(const NormArgs a, const BackArgs k, T *dx, T *df, const T *dy, const T *dh, const T *y,
                                                                                        const T *f, int tpr, int stages) {
    constexpr int S = BIAS ? 2 : 1, N = NV * W, H = N / 2;   // a thread's columns, as pairs
    constexpr bool KEEP = MAXT <= 256 && !BIAS;         // the weights stay in registers
    __shared__ float4 red[2 * S][8];
    extern __shared__ __align__(16) char ring[];
    const int warps = tpr >> 5, lane = warps == 1 ? (threadIdx.x & 31) : threadIdx.x;
    const int worker = warps == 1 ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    const int G = a.gate_rows > 0 ? (int)a.gate_rows : 1;
    clear_sums(red[0], 2 * S * 8);
    int phase = 0;
    const auto column = [&](int i) { return (i * tpr + lane) * W; };   // of vector i
    const auto weights = [&](Pair (&v)[H], const float *w) {
        float q[NV][W];
        Cols<float, W, NV, FULL>::load(q, w, tpr, lane, a.dim, 0.0f);
#pragma unroll
        for (int n = 0; n < H; ++n) v[n] = pair(q[2 * n / W][2 * n % W], q[(2 * n + 1) / W][(2 * n + 1) % W]);
    };
    const auto fill = [](Pair (&v)[H], float x) {
#pragma unroll
        for (int n = 0; n < H; ++n) v[n] = pair(x, x);
    };
    Pair w1[H], w2[H], b2[H], s_w1[H], s_b1[H], s_w2[H], s_b2[H], s_g[H];
    fill(w1, 1.0f); fill(w2, 1.0f); fill(b2, 0.0f);
    fill(s_w1, 0.0f); fill(s_b1, 0.0f); fill(s_w2, 0.0f); fill(s_b2, 0.0f); fill(s_g, 0.0f);
    if (KEEP && a.w1) weights(w1, a.w1);
    if (KEEP && a.w2) weights(w2, a.w2);
    const int group0 = worker / k.per_group, member = worker - group0 * k.per_group;
    RowWalk now = {group0 < k.groups_at_once ? group0 : G, member, G, (int)(a.rows / G), member, k.per_group, k.groups_at_once}, ahead = now;
    // shared memory, per stage: 5 tensors x NV vectors of 16 bytes a thread, or the rows of 5 tensors for every row group; then 16 bytes a warp for
    // the statistics
    const int pitch = W > 1 ? NV * (int)blockDim.x * 16 : (int)blockDim.x / tpr * (tpr * NV * (int)sizeof(T) + 32);   // of a tensor
    const int stage_bytes = 5 * pitch + (int)(blockDim.x >> 5) * 16, stat_at = 5 * pitch + (int)(threadIdx.x >> 5) * 16;
    const unsigned ring0 = (unsigned)__cvta_generic_to_shared(ring);
    const int mine = W > 1 ? (int)threadIdx.x * 16 : (warps == 1 ? (int)(threadIdx.x >> 5) : 0) * (tpr * NV * (int)sizeof(T) + 32);
    const auto copy = [&](int stage, int what, const T *p, unsigned row, unsigned ld) {
        const T *from = p + (unsigned long long)row * ld;
        if constexpr (W > 1) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (FULL || column(i) < a.dim) cp_async(ring0 + stage + mine + what * pitch + i * (int)blockDim.x * 16, from + column(i));
        } else {
            const int mis = (int)((uintptr_t)from & 15), bytes = mis + a.dim * (int)sizeof(T);
            const unsigned to = ring0 + stage + mine + what * pitch;
            for (int at = lane * 16; at < bytes; at += tpr * 16) cp_async(to + at, (const char *)from - mis + at, bytes - at < 16 ? bytes - at : 16);
        }
    };
    // a row as it was copied; `other` beyond its end
    const auto take = [&](Pair (&v)[H], int stage, int what, const T *p, unsigned row, unsigned ld, float other) {
        float q[N];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float x[W];
#pragma unroll
            for (int j = 0; j < W; ++j) x[j] = other;
            if constexpr (W > 1) {
                if (FULL || column(i) < a.dim) load_vec<T, W>(x, reinterpret_cast<const T *>(ring + stage + mine + what * pitch + i * (int)blockDim.x * 16));
            } else {
                const int mis = (int)((uintptr_t)(p + (unsigned long long)row * ld) & 15);
                if (FULL || column(i) < a.dim) load_vec<T, W>(x, reinterpret_cast<const T *>(ring + stage + mine + what * pitch + mis) + column(i));
            }
#pragma unroll
            for (int j = 0; j < W; ++j) q[i * W + j] = x[j];
        }
#pragma unroll
        for (int n = 0; n < H; ++n) v[n] = pair(q[2 * n], q[2 * n + 1]);
    };
    const Out<W, NV, FULL> put = {tpr, lane, a.dim};
    const auto row_barrier = [&]() {
        if (W == 1 && warps > 1) __syncthreads();
        else __syncwarp();                              // the statistics come by the warp's first lane
    };
    const auto next_stage = [&](int stage) { return stage + stage_bytes < stages * stage_bytes ? stage + stage_bytes : 0; };
    unsigned on_bits = 0, on_at = 0, on_to = 0;         // which of the rows under way are no padding: bits come in at on_to, go out at on_at
    char pat_ahead = !ahead.ended() && a.pat ? __ldg(a.pat + ahead.row()) : 1;
    const auto advance = [&](int stage) {
        const bool on = !ahead.ended() && pat_ahead != PAT_NONE;
        on_bits = (on_bits & ~(1u << on_to)) | ((unsigned)on << on_to);
        on_to = (on_to + 1) & 31;
        if (on) {
            const unsigned r = ahead.row();
            if ((threadIdx.x & 31) == 0) cp_async(ring0 + stage + stat_at, a.stats + r);
            if (FULL || dh) { copy(stage, 0, dh, r, k.ld_dh); copy(stage, 1, y, r, k.ld_y); }
            if (FULL || dy) copy(stage, 2, dy, r, k.ld_dy);
            if (FULL || f) copy(stage, 3, f, r, k.ld_f);
            if ((FULL || f) && a.gate) copy(stage, 4, (const T *)a.gate, ahead.g, (unsigned)a.ld_gate);
        }
        cp_commit();
        if (ahead.ended()) return;
        ahead.next();
        if (a.pat && !ahead.ended()) pat_ahead = __ldg(a.pat + ahead.row());   // looked at when the next copies start
    };
    int at = 0, to = 0;                                 // the stage worked on, and the one that is filled next
    for (int s = 0; s + 1 < stages; ++s) { advance(to); to = next_stage(to); }
    for (; !now.ended(); at = next_stage(at), to = next_stage(to)) {
        if (stages > 1) {
            cp_wait(stages - 2);
            row_barrier();                              // the row is there for all its threads, and all have left the one before
            advance(to);
        } else {
            row_barrier();
            advance(0);
            cp_wait(0);
            row_barrier();
        }
        const unsigned r = now.row(), g = now.g;
        const bool on = on_bits >> on_at & 1, done = now.last_of_group();
        on_at = (on_at + 1) & 31;
        now.next();
        Pair d[H], u[H], t[H];
        if (!on) {
            fill(d, 0.0f);
            if (FULL || dx) put(dx + (unsigned long long)r * k.ld_dx, d);
            if (FULL || df) put(df + (unsigned long long)r * k.ld_df, d);
        } else {
            const float4 st = *reinterpret_cast<const float4 *>(ring + at + stat_at);
            // u = (v - mean) / deviation; sums of d and of d u
            const auto centre = [&](float mean, float rstd) {
                const Pair mm = pair(-mean, -mean), rr = pair(rstd, rstd);
#pragma unroll
                for (int n = 0; n < H; ++n) u[n] = mul2(BIAS ? add2(u[n], mm) : u[n], rr);
            };
            const auto joint = [&](float (&s)[S]) {
                Pair p = 0, q = 0;
#pragma unroll
                for (int n = 0; n < H; ++n) {
                    p = fma2(d[n], u[n], p);
                    if (BIAS) q = add2(q, d[n]);
                }
                const float2 x = halves(p), z = halves(q);
                s[0] = x.x + x.y;
                if (BIAS) s[S - 1] = z.x + z.y;
                row_sums<S>(s, warps, red, phase);
                s[0] = -s[0] * a.inv_dim;
                if (BIAS) s[S - 1] = a.layer_norm ? -s[S - 1] * a.inv_dim : 0.0f;
            };
            if (FULL || dh) {
                float s[S];
                take(d, at, 0, dh, r, k.ld_dh, 0.0f);
                take(u, at, 1, y, r, k.ld_y, st.z);
                if (!KEEP && a.w1) weights(w1, a.w1);
                centre(st.z, st.w);
#pragma unroll
                for (int n = 0; n < H; ++n) {
                    s_w1[n] = fma2(d[n], u[n], s_w1[n]);
                    if (BIAS) s_b1[n] = add2(s_b1[n], d[n]);
                    d[n] = mul2(d[n], w1[n]);
                }
                joint(s);
                const Pair p = pair(s[0], s[0]), q = pair(s[S - 1], s[S - 1]), rr = pair(st.w, st.w);
                if (FULL || dy) take(t, at, 2, dy, r, k.ld_dy, 0.0f);
                else fill(t, 0.0f);
#pragma unroll
                for (int n = 0; n < H; ++n) d[n] = fma2(fma2(u[n], p, BIAS ? add2(d[n], q) : d[n]), rr, t[n]);
            } else if (dy) take(d, at, 2, dy, r, k.ld_dy, 0.0f);
            if (FULL || dx) put(dx + (unsigned long long)r * k.ld_dx, d);
            if (FULL || f) {
                float s[S];
                take(u, at, 3, f, r, k.ld_f, st.x);
                if (a.gate) take(t, at, 4, (const T *)a.gate, g, (unsigned)a.ld_gate, 0.0f);
                else {
#pragma unroll
                    for (int n = 0; n < H; ++n) t[n] = pair(FULL || column(2 * n / W) < a.dim ? 1.0f : 0.0f, FULL || column((2 * n + 1) / W) < a.dim ? 1.0f : 0.0f);
                }
                if (!KEEP && a.w2) weights(w2, a.w2);
                if (BIAS && a.b2) weights(b2, a.b2);
                centre(st.x, st.y);
                const Pair aa = pair(a.a, a.a);
#pragma unroll
                for (int n = 0; n < H; ++n) {
                    d[n] = mul2(d[n], aa);
                    s_g[n] = fma2(d[n], BIAS ? fma2(u[n], w2[n], b2[n]) : mul2(u[n], w2[n]), s_g[n]);
                    d[n] = mul2(d[n], t[n]);
                    s_w2[n] = fma2(d[n], u[n], s_w2[n]);
                    if (BIAS) s_b2[n] = add2(s_b2[n], d[n]);
                    d[n] = mul2(d[n], w2[n]);
                }
                if (FULL || df) {
                    joint(s);
                    const Pair p = pair(s[0], s[0]), q = pair(s[S - 1], s[S - 1]), rr = pair(st.y, st.y);
#pragma unroll
                    for (int n = 0; n < H; ++n) d[n] = mul2(fma2(u[n], p, BIAS ? add2(d[n], q) : d[n]), rr);
                    put(df + (unsigned long long)r * k.ld_df, d);
                }
            }
        }
        if (done && k.dgate) {
            if (k.per_group == 1) put((T *)k.dgate + (unsigned long long)g * k.ld_dgate, s_g);
            else put(k.partial_gate + (size_t)worker * k.dim_pad, s_g);
            fill(s_g, 0.0f);
        }
    }
    cp_wait(0);
    if (!k.partial) return;
    float *out = k.partial + (size_t)blockIdx.x * 4 * k.dim_pad;
    if (warps > 1) {
        put(out, s_w1);
        put(out + k.dim_pad, s_b1);
        put(out + 2 * k.dim_pad, s_w2);
        put(out + 3 * k.dim_pad, s_b2);
    } else {
        float *join = reinterpret_cast<float *>(ring);
        const int w = threadIdx.x >> 5, nw = blockDim.x >> 5, width = 32 * N;
        __syncthreads();                                // the copies of all warps have arrived
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            put(join + w * width, q == 0 ? s_w1 : q == 1 ? s_b1 : q == 2 ? s_w2 : s_b2);
            __syncthreads();
            for (int c = threadIdx.x; c < a.dim; c += blockDim.x) {
                float s = 0.0f;
                for (int i = 0; i < nw; ++i) s += join[i * width + c];
                out[q * k.dim_pad + c] = s;
            }
            __syncthreads();
        }
    }
}

// Sums of the workspace over blocks (blockIdx.y < 4: one weight gradient each) or over the workers of a row of the gate.
// 32 columns x 32 phases a block; the phases are added in order.
struct ReduceArgs {
    const float *partial, *partial_gate;
    float *out[4];
    void *dgate;
    long long ld_dgate;
    int dim, dim_pad, blocks, per_group;
};
template <typename T> __global__ void __launch_bounds__(1024) block_norm_reduce_kernel(const ReduceArgs a) {
    __shared__ float part[32][33];
    grid_wait();
    const int c = blockIdx.x * 32 + threadIdx.x, y = threadIdx.y, q = blockIdx.y;
    const bool gate = q >= 4;
    if (!gate && !a.out[q]) return;
    const float *p = gate ? a.partial_gate + (size_t)(q - 4) * a.per_group * a.dim_pad : a.partial + (size_t)q * a.dim_pad;
    const size_t step = gate ? a.dim_pad : (size_t)4 * a.dim_pad;
    const int n = gate ? a.per_group : a.blocks;
    float s = 0.0f;
    if (c < a.dim)
#pragma unroll 4
        for (int i = y; i < n; i += 32) s += p[(size_t)i * step + c];
    part[y][threadIdx.x] = s;
    __syncthreads();
    if (y == 0 && c < a.dim) {
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; ++i) t += part[i][threadIdx.x];
        if (gate) ((T *)a.dgate)[(long long)(q - 4) * a.ld_dgate + c] = from_float<T>(t);
        else a.out[q][c] = t;
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------------------
// widest vectors (16 bytes) only where every row of every tensor starts and ends on them
struct Width {
    int w;
    int elem;
    void rows(const void *p, long long ld) { if (p && (ld % w || !aligned_to(p, 16))) w = 1; }
    void floats(const float *p) { if (!aligned_to(p, 16)) w = 1; }
};
Width width_of(const b2_block_norm *d) {
    Width x = {16 / type_size(d->type), type_size(d->type)};
    if (d->dim % x.w) x.w = 1;
    x.rows(d->gate, d->ld_gate);
    x.floats(d->w_pre); x.floats(d->b_pre); x.floats(d->w_post); x.floats(d->b_post);
    return x;
}

int check(const char *who, const b2_block_norm *d) {
    if (!d) { set_error("%s: null pointer", who); return B2_ERR_BAD_ARG; }
    const int e = type_size(d->type);
    if (!e) { set_error("%s: unknown element type %d", who, d->type); return B2_ERR_BAD_ARG; }
    if (d->rows < 0 || d->rows > 0x7fffffffll || d->dim < 1 || d->dim > MAX_DIM) {
        set_error("%s: %lld rows of %d (at most 2^31 - 1 and %d)", who, d->rows, d->dim, MAX_DIM);
        return B2_ERR_BAD_SHAPE;
    }
    if (!(d->eps >= 0.0f) || d->eps > 3.4e38f || d->residual_scale != d->residual_scale) {
        set_error("%s: epsilon %g, residual scale %g", who, (double)d->eps, (double)d->residual_scale);
        return B2_ERR_BAD_ARG;
    }
    if (d->gate) {
        if (d->gate_rows < 1 || (d->rows && d->rows % d->gate_rows)) {
            set_error("%s: a gate of %lld rows for %lld frames (the frames must be a multiple)", who, d->gate_rows, d->rows);
            return B2_ERR_BAD_SHAPE;
        }
        if (d->ld_gate < d->dim || d->ld_gate > 0x7fffffffll) {
            set_error("%s: leading dimension of the gate too small or beyond 2^31 (%lld for %d columns)", who, d->ld_gate, d->dim);
            return B2_ERR_BAD_ARG;
        }
        if (!aligned_to(d->gate, e)) { set_error("%s: the gate is not aligned to its elements", who); return B2_ERR_BAD_ARG; }
    }
    if (!aligned_to(d->w_pre, 4) || !aligned_to(d->b_pre, 4) || !aligned_to(d->w_post, 4) || !aligned_to(d->b_post, 4) || !aligned_to(d->stats, 16)) {
        set_error("%s: weights have to be aligned to 4 bytes, the statistics to 16", who);
        return B2_ERR_BAD_ARG;
    }
    return B2_OK;
}
int check_rows(const char *who, const char *name, const b2_block_norm *d, const void *p, long long ld) {
    if (!p) return B2_OK;
    if (ld < d->dim || ld > 0x7fffffffll) {
        set_error("%s: leading dimension of %s too small or beyond 2^31 (%lld for %d columns)", who, name, ld, d->dim);
        return B2_ERR_BAD_ARG;
    }
    if (!aligned_to(p, type_size(d->type))) { set_error("%s: %s is not aligned to its elements", who, name); return B2_ERR_BAD_ARG; }
    return B2_OK;
}
NormArgs args_of(const b2_block_norm *d) {
    return {d->pat_types, d->w_pre, d->b_pre, d->w_post, d->b_post, d->gate, (float4 *)d->stats, d->rows, d->gate ? d->gate_rows : 1, d->ld_gate, d->dim,
            d->layer_norm ? 1 : 0, d->eps, d->residual_scale, 1.0f / (float)d->dim};
}

template <typename T, int W>
int forward(const b2_block_norm *d, const T *x, long long ld_x, const T *f, long long ld_f, T *y, long long ld_y, T *h, long long ld_h, cudaStream_t st) {
    const NormArgs a = args_of(d);
    const int vecs = (d->dim + W - 1) / W;
    const auto go = [&](auto kernel, int tpr) -> int {
        const unsigned blocks = tpr == 32 ? (unsigned)((d->rows + 7) / 8) : (unsigned)d->rows;
        kernel<<<blocks, tpr == 32 ? 256 : tpr, 0, st>>>(a, x, ld_x, f, ld_f, y, ld_y, h, ld_h, tpr);
        count_launch();
        B2_CUDA(cudaGetLastError());
        return B2_OK;
    };
    if (vecs <= 32) return go(block_norm_forward_kernel<T, W, 1>, 32);
    if (vecs <= 64) return go(block_norm_forward_kernel<T, W, 2>, 32);
    if (vecs <= 128) return go(block_norm_forward_kernel<T, W, 4>, 32);
    if (vecs <= 2048) return go(block_norm_forward_kernel<T, W, 4>, (int)pow2_at_least((unsigned)(vecs + 3) / 4));
    return go(block_norm_forward_kernel<T, W, 8>, (int)pow2_at_least((unsigned)(vecs + 7) / 8));
}

// Workers of the backward pass.  tpr: threads a row, each with `per_thread` columns or two times as many; blocks: as many as 512 threads a
// multiprocessor give (their registers, and the shared memory of a deep ring)
struct BackPlan { int tpr, threads, blocks, workers, per_group, groups_at_once; };
BackPlan back_plan(long long rows, int dim, int per_thread, long long gate_rows) {
    BackPlan p;
    const unsigned t = pow2_at_least((unsigned)((dim + per_thread - 1) / per_thread));
    p.tpr = t < 32 ? 32 : t > 1024 ? 1024 : (int)t;
    p.threads = p.tpr == 32 ? 256 : p.tpr;
    const int each = p.threads / p.tpr;
    long long blocks = (long long)sm_count() * (512 > p.threads ? 512 / p.threads : 1);
    if (blocks * each > rows) blocks = (rows + each - 1) / each;
    p.blocks = (int)blocks;
    p.workers = p.blocks * each;
    const long long G = gate_rows > 0 ? gate_rows : 1;
    p.per_group = (int)(p.workers / G);
    if (p.per_group < 1) p.per_group = 1;
    if (p.per_group > rows / G) p.per_group = (int)(rows / G);
    p.groups_at_once = p.workers / p.per_group;
    return p;
}

template <typename T, int W>
int backward(const b2_block_norm *d, T *dx, long long ld_dx, T *df, long long ld_df, T *dgate, long long ld_dgate, float *const (&dw)[4], const T *dy, long long ld_dy,
             const T *dh, long long ld_dh, const T *y, long long ld_y, const T *f, long long ld_f, float *ws, cudaStream_t st) {
    const NormArgs a = args_of(d);
    const int per_thread = W > 1 ? W : 8;
    const BackPlan p = back_plan(d->rows, d->dim, per_thread, d->gate ? d->gate_rows : 0);
    BackArgs k = {(unsigned)ld_dx, (unsigned)ld_df, (unsigned)ld_dy, (unsigned)ld_dh, (unsigned)ld_y, (unsigned)ld_f, (unsigned)ld_dgate, dgate, nullptr, nullptr, (d->dim + 15) / 16 * 16, p.per_group, p.groups_at_once};
    const bool sums = dw[0] || dw[1] || dw[2] || dw[3], gate_sums = dgate && p.per_group > 1;
    if (sums) k.partial = ws;
    k.partial_gate = ws + (size_t)p.blocks * 4 * k.dim_pad;
    // the ring: up to 4 rows in what the blocks of a multiprocessor share
    const int nv = W == 1 ? 8 : d->dim > p.tpr * W ? 2 : 1, here = 512 > p.threads ? 512 / p.threads : 1;
    const int pitch = W > 1 ? nv * p.threads * 16 : p.threads / p.tpr * (p.tpr * nv * (int)sizeof(T) + 32), stage_bytes = 5 * pitch + p.threads / 32 * 16;
    const int most = 208 * 1024, join_bytes = p.tpr == 32 ? 8 * 32 * W * nv * 4 : 0;
    int stages = most / here / stage_bytes;
    stages = stages > 4 ? 4 : stages < 1 ? 1 : stages;
    const int smem = stages * stage_bytes > join_bytes ? stages * stage_bytes : join_bytes;
    const auto go = [&](auto kernel) -> int {
        B2_TRY(set_max_dynamic_smem((const void *)kernel, most));
        kernel<<<p.blocks, p.threads, smem, st>>>(a, k, dx, df, dy, dh, y, f, p.tpr, stages);
        count_launch();
        B2_CUDA(cudaGetLastError());
        return B2_OK;
    };
    const bool bias = d->layer_norm || dw[1] || dw[3] || d->b_post;
    const bool full = W > 1 && d->dim == p.tpr * W && dx && df && dy && dh && f;
    const auto pick = [&](auto b) {
        constexpr bool B = decltype(b)::value;
        constexpr int NV = W == 1 ? 8 : 1;
        if constexpr (W > 1)
            if (full) {
                if (p.threads <= 256) return go(block_norm_backward_kernel<T, W, 1, 256, B, true>);
                if (p.threads <= 512) return go(block_norm_backward_kernel<T, W, 1, 512, B, true>);
                return go(block_norm_backward_kernel<T, W, 1, 1024, B, true>);
            }
        if (p.threads <= 256) return go(block_norm_backward_kernel<T, W, NV, 256, B, false>);
        if (p.threads <= 512) return go(block_norm_backward_kernel<T, W, NV, 512, B, false>);
        if constexpr (W == 4)
            if (nv == 2) return go(block_norm_backward_kernel<T, W, 2, 1024, B, false>);
        return go(block_norm_backward_kernel<T, W, NV, 1024, B, false>);
    };
    B2_TRY(bias ? pick(std::true_type()) : pick(std::false_type()));
    if (!sums && !gate_sums) return B2_OK;
    const ReduceArgs r = {k.partial, k.partial_gate, {dw[0], dw[1], dw[2], dw[3]}, gate_sums ? dgate : nullptr, ld_dgate, d->dim, k.dim_pad, p.blocks, p.per_group};
    const unsigned groups = gate_sums ? (unsigned)(d->gate ? d->gate_rows : 1) : 0;
    return launch_chained(block_norm_reduce_kernel<T>, dim3((d->dim + 31) / 32, 4 + groups), dim3(32, 32), 0, st, r);
}

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" {

int b2_block_norm_forward(const b2_block_norm *d, const void *x, long long ld_x, const void *f, long long ld_f, void *y, long long ld_y, void *h, long long ld_h,
                          b2_stream stream) {
    const char *who = "b2_block_norm_forward";
    B2_TRY(check(who, d));
    B2_TRY(check_rows(who, "x", d, x, ld_x));
    B2_TRY(check_rows(who, "f", d, f, ld_f));
    B2_TRY(check_rows(who, "y", d, y, ld_y));
    B2_TRY(check_rows(who, "h", d, h, ld_h));
    if (!d->rows) return B2_OK;
    if (!x || (!y && !h) || (f && !y)) { set_error("%s: null pointer (x, and y where there is f, are needed; y or h is written)", who); return B2_ERR_BAD_ARG; }
    if (h == x || (f && (h == f || y == f)) || (h && h == y)) { set_error("%s: only y may take the place of x", who); return B2_ERR_BAD_ARG; }
    if (y == x && ld_y != ld_x) { set_error("%s: y takes the place of x with another leading dimension", who); return B2_ERR_BAD_ARG; }
    Width w = width_of(d);
    w.rows(x, ld_x); w.rows(f, ld_f); w.rows(y, ld_y); w.rows(h, ld_h);
    return with_type(d->type, [&](auto *t) {
        typedef B2_ELEM(t) T;
        constexpr int W = 16 / sizeof(T);
        if (w.w == W) return forward<T, W>(d, (const T *)x, ld_x, (const T *)f, ld_f, (T *)y, ld_y, (T *)h, ld_h, (cudaStream_t)stream);
        return forward<T, 1>(d, (const T *)x, ld_x, (const T *)f, ld_f, (T *)y, ld_y, (T *)h, ld_h, (cudaStream_t)stream);
    });
}

size_t b2_block_norm_backward_workspace(long long rows, int dim, long long gate_rows) {
    if (rows < 1 || rows > 0x7fffffffll || dim < 1 || dim > MAX_DIM || gate_rows < 0) return 0;
    // enough for any type and alignment
    size_t most = 0;
    for (int per_thread = 4; per_thread <= 8; per_thread *= 2) {
        const BackPlan p = back_plan(rows, dim, per_thread, gate_rows);
        const size_t n = (size_t)p.blocks * 4 + p.workers;
        if (n > most) most = n;
    }
    return most * ((dim + 15) / 16 * 16) * sizeof(float);
}

int b2_block_norm_backward(const b2_block_norm *d, void *dx, long long ld_dx, void *df, long long ld_df, void *dgate, long long ld_dgate, float *dw_pre, float *db_pre,
                           float *dw_post, float *db_post, const void *dy, long long ld_dy, const void *dh, long long ld_dh, const void *y, long long ld_y, const void *f,
                           long long ld_f, void *workspace, size_t workspace_bytes, b2_stream stream) {
    const char *who = "b2_block_norm_backward";
    B2_TRY(check(who, d));
    B2_TRY(check_rows(who, "dx", d, dx, ld_dx));
    B2_TRY(check_rows(who, "df", d, df, ld_df));
    B2_TRY(check_rows(who, "dgate", d, dgate, ld_dgate));
    B2_TRY(check_rows(who, "dy", d, dy, ld_dy));
    B2_TRY(check_rows(who, "dh", d, dh, ld_dh));
    B2_TRY(check_rows(who, "y", d, y, ld_y));
    B2_TRY(check_rows(who, "f", d, f, ld_f));
    if (!aligned_to(dw_pre, 4) || !aligned_to(db_pre, 4) || !aligned_to(dw_post, 4) || !aligned_to(db_post, 4)) {
        set_error("%s: weight gradients have to be aligned to 4 bytes", who);
        return B2_ERR_BAD_ARG;
    }
    if (dgate && !d->gate) { set_error("%s: a gradient for a gate that is not there", who); return B2_ERR_BAD_ARG; }
    if ((df || dgate || dw_post || db_post) && !f) { set_error("%s: gradients of the norm after the block need f", who); return B2_ERR_BAD_ARG; }
    if ((dw_pre || db_pre) && !dh) { set_error("%s: gradients of the norm before the block need dh", who); return B2_ERR_BAD_ARG; }
    if (!d->rows) {
        // sums over no frames
        float *w[4] = {dw_pre, db_pre, dw_post, db_post};
        for (float *p : w)
            if (p) B2_CUDA(cudaMemsetAsync(p, 0, (size_t)d->dim * sizeof(float), (cudaStream_t)stream));
        if (dgate) B2_CUDA(cudaMemset2DAsync(dgate, (size_t)ld_dgate * type_size(d->type), 0, (size_t)d->dim * type_size(d->type), (size_t)d->gate_rows, (cudaStream_t)stream));
        return B2_OK;
    }
    if (!d->stats || (!dy && !dh) || (dh && !y)) { set_error("%s: null pointer (the statistics, dy or dh, and y where there is dh, are needed)", who); return B2_ERR_BAD_ARG; }
    if (!workspace || !aligned_to(workspace, 16)) { set_error("%s: the workspace is missing or not aligned to 16 bytes", who); return B2_ERR_BAD_ARG; }
    const size_t need = b2_block_norm_backward_workspace(d->rows, d->dim, d->gate ? d->gate_rows : 0);
    if (workspace_bytes < need) { set_error("%s: %zu bytes of workspace, %zu are needed", who, workspace_bytes, need); return B2_ERR_BAD_SHAPE; }
    const void *in[4] = {dy, dh, y, f};
    const long long ld_in[4] = {ld_dy, ld_dh, ld_y, ld_f};
    for (int i = 0; i < 4; ++i)
        if ((in[i] && in[i] == dx && ld_in[i] != ld_dx) || (in[i] && in[i] == df && ld_in[i] != ld_df)) {
            set_error("%s: a gradient takes the place of an input with another leading dimension", who);
            return B2_ERR_BAD_ARG;
        }
    if (dx && dx == df) { set_error("%s: dx and df are the same", who); return B2_ERR_BAD_ARG; }
    Width w = width_of(d);
    w.rows(dx, ld_dx); w.rows(df, ld_df); w.rows(dgate, ld_dgate); w.rows(dy, ld_dy); w.rows(dh, ld_dh); w.rows(y, ld_y); w.rows(f, ld_f);
    float *const dw[4] = {dw_pre, db_pre, dw_post, db_post};
    return with_type(d->type, [&](auto *t) {
        typedef B2_ELEM(t) T;
        constexpr int W = 16 / sizeof(T);
        const auto go = [&](auto width) {
            return backward<T, decltype(width)::value>(d, (T *)dx, ld_dx, (T *)df, ld_df, (T *)dgate, ld_dgate, dw, (const T *)dy, ld_dy, (const T *)dh, ld_dh, (const T *)y,
                                                       ld_y, (const T *)f, ld_f, (float *)workspace, (cudaStream_t)stream);
        };
        return w.w == W ? go(std::integral_constant<int, W>()) : go(std::integral_constant<int, 1>());
    });
}

}  // extern "C"
