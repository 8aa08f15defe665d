// The paged 8-bit K/V cache: what its kernels share. Layout and rules: include/decide_cuda.h (dc_kv8_cache).
#pragma once
#include "common.cuh"

// Status-word values of the dc_kv8_* kernels (violations only the device can see; messages in ctx.cu).
enum {
    DC_STATUS_KV8_OFFSETS = 71,     // row offsets that fall, pass `rows` or exceed the given maximum or the sequence's length
    DC_STATUS_KV8_LENGTH = 72,      // a sequence longer than its row of the table, or than max_len
    DC_STATUS_KV8_PAGE = 73,        // a page id outside the pool
    DC_STATUS_KV8_POSITION = 74,    // a query position at or past the sequence's length
    DC_STATUS_KV8_SHARED = 75,      // a write to a page that is free or that several sequences hold
    DC_STATUS_KV8_POOL = 76,        // too few free pages
    DC_STATUS_KV8_SEQUENCE = 77,    // a sequence index past n_seqs, or one named twice
    DC_STATUS_KV8_REFS = 78         // a page freed more often than it was held
};

// Host-side checks of a call: DC_OK, or dc_fail with `who` in the message.
int dc_kv8_require(dc_ctx* ctx, const char* who, const dc_kv8_cache* cache);

int dc_kv8_attention_warm(dc_ctx* ctx);
int dc_kv8_attention_tc_warm(dc_ctx* ctx);

// Makes the context's device current for the scope of an entry point: the caller's current device may be another one.
struct dc_device_scope {
    int before = -1;
    explicit dc_device_scope(const dc_ctx* ctx) {
        int now = -1;
        if (cudaGetDevice(&now) == cudaSuccess && now != ctx->device && cudaSetDevice(ctx->device) == cudaSuccess) before = now;
    }
    ~dc_device_scope() {
        if (before >= 0) cudaSetDevice(before);
    }
};

// Launches a dc_kv8_* kernel. `early`: as a programmatic dependent, put on the GPU while the kernel before it in the stream still runs, so
// that its launch (about 1 us) overlaps; every kernel starts with kv8_begin(), which waits for that one to be done and its writes to
// be there. Worth it for the second kernel of a call and for small grids (one token over 603 keys 7.4 -> 6.8 us); a grid that has one
// CTA for each SM loses by it, since CTAs that came early share SMs when their turn comes (131,071 keys 51 -> 64 us).
template <typename... P, typename... A>
int dc_kv8_launch(dc_ctx* ctx, const char* what, void (*kernel)(P...), bool early, dim3 grid, uint32_t block, size_t smem, cudaStream_t stream, A... args) {
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = early ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return dc_fail(ctx, DC_CUDA_ERROR, "%s: launch failed: %s", what, cudaGetErrorString(e));
    }
    return dc_check_launch(ctx, what);
}

namespace dc {

// The first thing a kernel does, before it touches memory that another kernel writes. Kernels launched early take their inputs without
// __restrict__ and __ldg: a load that the compiler may take for one of constant memory could move ahead of the wait.
__device__ __forceinline__ void kv8_begin() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

__device__ __forceinline__ void kv8_flag(int* status, int code) { atomicCAS(status, 0, code); }

// Largest finite e4m3 magnitude is 448 = 0.875 * 2^9: the least e with 448 * 2^e >= amax is exponent(amax) - 9 in frexp's sense
// (amax = f * 2^exponent, f in [0.5, 1)), one more where f > 0.875. Read off the bits of amax, exactly. The floor of 2^-60 keeps
// 1/scale and products of scales far from fp32's limits; a page of smaller values (none in a trained model) loses bits.
constexpr int kKv8ExpMin = -60;
__device__ __forceinline__ int kv8_exponent(float amax) {
    const uint32_t b = __float_as_uint(amax);
    const int e = static_cast<int>(b >> 23) - 126 - 9 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return max(e, kKv8ExpMin);
}
__device__ __forceinline__ float kv8_exp2i(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }   // -126 <= e <= 127
// Exponent of a power of two; NaN stays NaN.
__device__ __forceinline__ float kv8_log2i(float scale) {
    return isnan(scale) ? scale : static_cast<float>(static_cast<int>((__float_as_uint(scale) >> 23) & 0xffu) - 127);
}

// Two fp32 values -> two e4m3 codes (lo in bits 0..7), round to nearest even, |x| <= 448 here.
__device__ __forceinline__ uint16_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// Two e4m3 codes -> two fp16 values, exactly.
__device__ __forceinline__ float2 e4m3x2_to_float2(uint16_t c) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(c));
    return __half22float2(*reinterpret_cast<__half2*>(&h));
}

// Pages that `tokens` tokens take.
__host__ __device__ __forceinline__ uint32_t kv8_pages(uint32_t tokens, uint32_t page_size) { return (tokens + page_size - 1) / page_size; }

}  // namespace dc
