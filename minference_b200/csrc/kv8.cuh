// The 8-bit key/value cache of one layer: layout and conversions shared by the kernels that fill it, read it and
// attend over it.
//
//   codes   [batch, heads, capacity, 128] one byte each, e4m3 or int8, capacity a multiple of 64
//   scales  [batch, heads, capacity / 64] fp32: value = code * scale of the token's block of 64 tokens
//   tail    [batch, heads, 64, 128] bf16: the tokens behind the last complete block, token t in row t % 64
//
// A block is quantised once, when its last token arrives, from the bf16 values of all its tokens, so a scale never
// changes and no value is rounded twice; until then its tokens are used as they came.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <utility>

#include "common.h"

namespace minf {

constexpr int kKv8Block = 64;
constexpr int kKv8Dim = 128;
constexpr float kKv8MinScale = 7.888609052210118e-31f;      // 2^-100: what a block of smaller values is scaled by

// Four e4m3 codes -> two half2 registers (exact: every e4m3 value is an f16 value, NaN stays NaN).
__device__ __forceinline__ void e4m3x4_to_half(uint32_t x, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\t"
        "mov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}\n"
        : "=r"(lo), "=r"(hi)
        : "r"(x));
}
// Four int8 codes -> two half2 registers (exact).  The byte with its sign bit flipped, under the exponent byte 0x64,
// is the half 1024 + 128 + code: one subtraction leaves the code.
__device__ __forceinline__ void int8x4_to_half(uint32_t x, uint32_t& lo, uint32_t& hi) {
    const uint32_t y = x ^ 0x80808080u;
    uint32_t a = __byte_perm(y, 0x64646464u, 0x4140), b = __byte_perm(y, 0x64646464u, 0x4342);
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(0x64806480u));
}
template <int FMT>
__device__ __forceinline__ void codes_to_half(uint32_t x, uint32_t& lo, uint32_t& hi) {
    if constexpr (FMT == MINF_KV8_E4M3) e4m3x4_to_half(x, lo, hi);
    else int8x4_to_half(x, lo, hi);
}

// Eight codes (two words) -> fp32 values of the given scale.
template <int FMT>
__device__ __forceinline__ void codes_to_values(uint2 c, float scale, float (&v)[8]) {
    uint32_t h[4];
    codes_to_half<FMT>(c.x, h[0], h[1]);
    codes_to_half<FMT>(c.y, h[2], h[3]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        v[2 * i] = f.x * scale;
        v[2 * i + 1] = f.y * scale;
    }
}

__device__ __forceinline__ void bf16x8_to_values(uint4 x, float (&v)[8]) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

// Number of tokens a sequence holds; a length outside [0, limit] is reported and clipped.
__device__ __forceinline__ int kv8_length(const int32_t* lengths, int all, int b, int limit, int32_t* status) {
    const int n = lengths ? lengths[b] : all;
    if (n < 0 || n > limit) {
        if (threadIdx.x == 0) atomicOr(status + MINF_ST_ERROR, MINF_ERR_KV8_RANGE);
        return n < 0 ? 0 : limit;
    }
    return n;
}

// A kernel that may start while the one before it in the stream ends: its launch is hidden behind that one's last CTAs.  It
// waits for the other's results itself (dependents_wait); the other says that it may be launched (dependents_launch).
template <class... Params, class... Args>
cudaError_t launch_behind(void (*kernel)(Params...), dim3 grid, int threads, size_t shared, cudaStream_t stream, Args&&... args) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = shared;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}
__device__ __forceinline__ void dependents_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void dependents_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Lets a kernel use `bytes` of dynamic shared memory, once per device (`done`: a bit for each device, one word per kernel).
template <class Kernel>
cudaError_t allow_shared(Kernel kernel, int bytes, std::atomic<unsigned long long>& done) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const unsigned long long bit = device < 64 ? 1ull << device : 0ull;
    if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// Host-side check of a cache descriptor; MINF_OK or a negative code with its message set.
int kv8_check(const minf_kv8_cache* c);

}  // namespace minf
