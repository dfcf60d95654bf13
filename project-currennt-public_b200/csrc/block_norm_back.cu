// The gradients of the norms around a residual block: formulas and layout at the top of block_norm.cu.
#include "block_norm.cuh"

namespace b2 {
namespace {

struct BackArgs {
    unsigned ld_dx, ld_df, ld_dy, ld_dh, ld_y, ld_f, ld_dgate;
    void *dgate;
    float *partial;                   // [blocks][4][dim_pad]: dw1, db1, dw2, db2 of every block
    float *partial_gate;              // [workers][dim_pad], where several workers share a row of the gate
    int dim_pad, per_group, groups_at_once;
};

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

// fp32 elements are copied one by one here (48256 x 405, RMS: 117 us, by row 168 us; in the forward pass by row 61 us and one by one 74 us for 38400 x 511)
template <typename T> __host__ __device__ constexpr bool by_row(int w) { return w == 1 && sizeof(T) == 2; }

// A worker is a warp (TPR = 32) or a block of TPR threads.  per_group workers share a row of the gate (all workers, if there is one row or none), and
// groups_at_once rows of the gate are worked on side by side.  BIAS: means are subtracted or the norms have a bias (without both, sums are saved).
// FULL: dy, dh, f, dx and df are all there and the threads' columns are just the row's: a third of the instructions were tests of that.
// As in the forward kernel, the next `stages` - 1 rows (up to three, as many as fit) are on their way into shared memory while one is worked on.
template <typename T, int W, int NV, int TPR, bool BIAS, bool FULL>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR, 512 / (TPR == 32 ? 256 : TPR) > 0 ? 512 / (TPR == 32 ? 256 : TPR) : 1)
    block_norm_backward_kernel(const NormArgs a, const BackArgs k, T *dx, T *df, const T *dy, const T *dh, const T *y, const T *f, int stages) {
    constexpr int S = BIAS ? 2 : 1, N = NV * W, H = N / 2;   // a thread's columns, as pairs
    // The weights stay in registers; elsewhere they are loaded again for every row, which for 2048 channels with two weights and a bias is 24 KB of fp32, as much as
    // the row itself (16384 x 2048 bf16 with layer norm and biases 137 us, without 95 us).  Above 4096 columns of 16 bits a thread has 64 registers and spills.
    constexpr bool KEEP = TPR <= 256 && !BIAS;
    __shared__ float4 red[2 * S][8];
    extern __shared__ __align__(16) char ring[];
    constexpr int tpr = TPR, warps = TPR / 32;
    const int lane = warps == 1 ? (threadIdx.x & 31) : threadIdx.x;
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
    const Ring<T, W, NV, FULL, 5, by_row<T>(W)> shared(ring, tpr, lane, a.dim, stages);
    const auto take = [&](Pair (&v)[H], int stage, int what, const T *p, unsigned row, unsigned ld, float other) {
        float q[NV][W];
        shared.take(q, stage, what, p + (unsigned long long)row * ld, other);
#pragma unroll
        for (int n = 0; n < H; ++n) v[n] = pair(q[2 * n / W][2 * n % W], q[(2 * n + 1) / W][(2 * n + 1) % W]);
    };
    const Out<W, NV, FULL> put = {tpr, lane, a.dim};
    unsigned on_bits = 0, on_at = 0, on_to = 0;         // which of the rows under way are no padding: bits come in at on_to, go out at on_at
    char pat_ahead = !ahead.ended() && a.pat ? __ldg(a.pat + ahead.row()) : 1;
    const auto advance = [&](int stage) {
        const bool on = !ahead.ended() && pat_ahead != PAT_NONE;
        on_bits = (on_bits & ~(1u << on_to)) | ((unsigned)on << on_to);
        on_to = (on_to + 1) & 31;
        if (on) {
            const unsigned r = ahead.row();
            // the statistics by the warp's first lane
            if ((threadIdx.x & 31) == 0) cp_async<16>(shared.base_addr + shared.spare(stage), a.stats + r);
            if (FULL || dh) { shared.copy(stage, 0, dh + (unsigned long long)r * k.ld_dh); shared.copy(stage, 1, y + (unsigned long long)r * k.ld_y); }
            if (FULL || dy) shared.copy(stage, 2, dy + (unsigned long long)r * k.ld_dy);
            if (FULL || f) shared.copy(stage, 3, f + (unsigned long long)r * k.ld_f);
            if ((FULL || f) && a.gate) shared.copy(stage, 4, (const T *)a.gate + (unsigned long long)ahead.g * (unsigned)a.ld_gate);
        }
        cp_commit();
        if (ahead.ended()) return;
        ahead.next();
        if (a.pat && !ahead.ended()) pat_ahead = __ldg(a.pat + ahead.row());   // looked at when the next copies start
    };
    int at = 0, to = 0;                                 // the stage worked on, and the one that is filled next
    for (int s = 0; s + 1 < stages; ++s) { advance(to); to = shared.next(to); }
    for (; !now.ended(); at = shared.next(at), to = shared.next(to)) {
        if (stages > 1) {
            cp_wait(stages - 2);
            shared.barrier();                           // the row is there for all its threads, and all have left the one before
            advance(to);
        } else {
            shared.barrier();
            advance(0);
            cp_wait(0);
            shared.barrier();
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
            const float4 st = *reinterpret_cast<const float4 *>(ring + shared.spare(at));
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
    const int per_thread = W * sizeof(T) == 16 ? W : 8;
    const BackPlan p = back_plan(d->rows, d->dim, per_thread, d->gate ? d->gate_rows : 0);
    BackArgs k = {(unsigned)ld_dx, (unsigned)ld_df, (unsigned)ld_dy, (unsigned)ld_dh, (unsigned)ld_y, (unsigned)ld_f, (unsigned)ld_dgate, dgate, nullptr, nullptr, (d->dim + 15) / 16 * 16, p.per_group, p.groups_at_once};
    const bool sums = dw[0] || dw[1] || dw[2] || dw[3], gate_sums = dgate && p.per_group > 1;
    if (sums) k.partial = ws;
    k.partial_gate = ws + (size_t)p.blocks * 4 * k.dim_pad;
    // the ring: up to 4 rows in what the blocks of a multiprocessor share
    // narrow accesses: 8 columns a thread, 4 where a warp holds the row with that (65536 x 101 bf16: 62 us, with 8 77; x 102: 41 us, with 8 53)
    const bool narrow = W * sizeof(T) != 16 && d->dim <= 128;
    const int nv = narrow ? 4 / W : W * sizeof(T) != 16 ? 8 / W : d->dim > p.tpr * W ? 2 : 1, here = 512 > p.threads ? 512 / p.threads : 1;
    const auto stage = [&](auto vectors) { return Ring<T, W, decltype(vectors)::value, false, 5, by_row<T>(W)>::bytes(p.threads, p.tpr); };
    constexpr int ONE = W * sizeof(T) == 16 ? 1 : 8 / W, NARROW = W * sizeof(T) == 16 ? 2 : 4 / W;   // of whole vectors, two only in the widest fp32 rows
    const int stage_bytes = nv == ONE ? stage(std::integral_constant<int, ONE>()) : stage(std::integral_constant<int, NARROW>());
    const int most = 208 * 1024, join_bytes = p.tpr == 32 ? 8 * 32 * W * nv * 4 : 0;
    int stages = most / here / stage_bytes;
    stages = stages > 4 ? 4 : stages < 1 ? 1 : stages;
    const int smem = stages * stage_bytes > join_bytes ? stages * stage_bytes : join_bytes;
    const auto go = [&](auto kernel) -> int {
        B2_TRY(set_max_dynamic_smem((const void *)kernel, most));
        kernel<<<p.blocks, p.threads, smem, st>>>(a, k, dx, df, dy, dh, y, f, stages);
        count_launch();
        B2_CUDA(cudaGetLastError());
        return B2_OK;
    };
    const bool bias = d->layer_norm || dw[1] || dw[3] || d->b_post;
    const bool full = W * sizeof(T) == 16 && d->dim == p.tpr * W && dx && df && dy && dh && f;
    const auto pick = [&](auto b) {
        constexpr bool B = decltype(b)::value;
        constexpr int NV = W * sizeof(T) == 16 ? 1 : 8 / W;
        const auto sized = [&](auto threads) -> int {
            constexpr int TPR = decltype(threads)::value;
            if constexpr (W * sizeof(T) == 16)
                if (full) return go(block_norm_backward_kernel<T, W, 1, TPR, B, true>);
            if constexpr (W == 4 && TPR == 1024)
                if (nv == 2) return go(block_norm_backward_kernel<T, W, 2, TPR, B, false>);
            if constexpr (W * sizeof(T) != 16 && TPR == 32)
                if (narrow) return go(block_norm_backward_kernel<T, W, 4 / W, TPR, B, false>);
            return go(block_norm_backward_kernel<T, W, NV, TPR, B, false>);
        };
        if (p.tpr == 1024) return sized(std::integral_constant<int, 1024>());
        if (p.tpr == 512) return sized(std::integral_constant<int, 512>());
        if (p.tpr == 256) return sized(std::integral_constant<int, 256>());
        if (p.tpr == 128) return sized(std::integral_constant<int, 128>());
        if (p.tpr == 64) return sized(std::integral_constant<int, 64>());
        return sized(std::integral_constant<int, 32>());
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

size_t b2_block_norm_backward_workspace(long long rows, int dim, long long gate_rows) {
    if (rows < 1 || rows > 0x7fffffffll || dim < 1 || dim > MAX_DIM || gate_rows < 0 || (gate_rows && rows % gate_rows)) return 0;
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
    if (d->gate && (dx == d->gate || df == d->gate) && (d->gate_rows != d->rows || (dx == d->gate ? ld_dx : ld_df) != d->ld_gate)) {
        set_error("%s: a gradient takes the place of the gate, which has other rows", who);
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
        if (w.w == W) return go(std::integral_constant<int, W>());
        if constexpr (W == 8)
            if (w.w == 2) return go(std::integral_constant<int, 2>());
        return go(std::integral_constant<int, 1>());
    });
}

}  // extern "C"
