// Element types of the token operators (fp32, bf16, fp16): conversions, 16-byte vectors of them, and what their launches share.
// Arithmetic is fp32 everywhere; a value is rounded to its type once, when it is stored.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace b2 {

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// N elements that are loaded and stored as one naturally aligned access (N * sizeof(T) <= 16), or as several of 16 bytes
template <typename T, int N> struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Vec { T v[N]; };
template <typename T, int N> __device__ __forceinline__ void load_vec(float (&out)[N], const T *p) {
    const Vec<T, N> x = *reinterpret_cast<const Vec<T, N> *>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = to_float(x.v[i]);
}
template <typename T, int N> __device__ __forceinline__ void store_vec(T *p, const float (&in)[N]) {
    Vec<T, N> x;
#pragma unroll
    for (int i = 0; i < N; ++i) x.v[i] = from_float<T>(in[i]);
    *reinterpret_cast<Vec<T, N> *>(p) = x;
}

constexpr long long MAX_LD = 1ll << 40;   // elements from row to row: 2^31 rows of them stay inside 64 bits
inline int type_size(int type) { return type == B2_F32 ? 4 : (type == B2_BF16 || type == B2_F16) ? 2 : 0; }
inline bool aligned_to(const void *p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) == 0; }
inline unsigned pow2_at_least(unsigned x) { unsigned p = 1; while (p < x) p <<= 1; return p; }

// calls f with a null pointer of the element type
template <typename F> int with_type(int type, F &&f) {
    switch (type) {
        case B2_F32: return f((float *)nullptr);
        case B2_BF16: return f((__nv_bfloat16 *)nullptr);
        case B2_F16: return f((__half *)nullptr);
    }
    set_error("unknown element type %d", type);
    return B2_ERR_BAD_ARG;
}
#define B2_ELEM(p) std::remove_pointer_t<decltype(p)>

// A launch that may start while the kernel before it on the stream drains; the kernel calls grid_wait() before it touches
// what that one wrote (and before it writes what that one reads).  Behind the wait it reads by plain loads: __ldg and loads through
// `const ... *__restrict__` are for memory that nobody writes while the kernel runs, and may be moved above it.
template <typename... KArgs, typename... Args>
int launch_chained(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args &&...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    count_launch();
    B2_CUDA(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...));
    return B2_OK;
}
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ---- packed arithmetic: two fp32 values an instruction ---------------------------------------------------------------------------------
typedef unsigned long long Pair;   // two fp32 values for the packed instructions
__device__ __forceinline__ Pair pair(float x, float y) { Pair p; asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(x), "f"(y)); return p; }
__device__ __forceinline__ float2 halves(Pair p) { float2 v; asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(p)); return v; }
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) { Pair d; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c)); return d; }
__device__ __forceinline__ Pair mul2(Pair a, Pair b) { Pair d; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b)); return d; }
__device__ __forceinline__ Pair add2(Pair a, Pair b) { Pair d; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b)); return d; }

// Copies of 16 bytes (the first `bytes` of them, zeros behind) into shared memory that nobody waits for before cp_wait
__device__ __forceinline__ void cp_async(unsigned to, const void *from, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
// BYTES (4, 8 or 16) of them
template <int BYTES> __device__ __forceinline__ void cp_async(unsigned to, const void *from) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// until at most N of the newest groups are under way
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// the same for n from 0 to 2
__device__ __forceinline__ void cp_wait(int n) {
    if (n == 0) asm volatile("cp.async.wait_group 0;" ::: "memory");
    else if (n == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 2;" ::: "memory");
}

// sums over a warp; every lane gets the result
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}
__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

}  // namespace b2
