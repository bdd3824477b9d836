// What the kernels around the paged key-value cache share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "mb_device.cuh"

namespace mb {
namespace paged {

constexpr int kMaxRows = 2048;   // requests of a table, and tokens of a step of one token a request
// Of a row of the table, and places of mb_paged_reserve: what is rounded up to a block or a grid's stride stays an int.
constexpr int kMaxTokens = 1 << 30;

struct Strides2 {
    long long token, head;   // elements
};
struct Strides3 {
    long long page, token, head;
};

struct AttentionArgs {
    int tokens, requests, heads, kv_heads, head_dim, width, pages, page_shift, zero_rest;
    float scale;
    Strides2 q, k, v;
    Strides3 kpool, vpool;
    const unsigned short *query, *key, *value;
    const unsigned short *key_pages, *value_pages;   // mb_paged_attention writes to the places of new tokens
    const int *table, *lengths, *index;
    unsigned short* out;
    int* status;
    int wait_limit_ns;
};

// Whether a phase is there, without waiting for it: try_wait suspends the thread for some time.
__device__ __forceinline__ bool mbar_test_wait(unsigned long long* bar, unsigned int parity) {
    unsigned int done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return done != 0;
}
// The wait for a phase that was not there: it ends after the limit, or when another one of the CTA did.  A limit of less than
// a millisecond is looked at all the time, without suspending.
__device__ __forceinline__ bool wait_within(unsigned long long* bar, unsigned int parity, volatile int* abort_flag, int limit_ns) {
    if (limit_ns >= 1000000) return mbar_wait_bounded(bar, parity, abort_flag, limit_ns);
    const unsigned long long start = global_timer_ns();
    while (!mbar_test_wait(bar, parity))
        if (*abort_flag || global_timer_ns() - start > static_cast<unsigned long long>(limit_ns)) return false;
    return true;
}

// Weights are 2^(log2(e) (score - highest) + shift).  fp16: up by 2^15, so that small ones keep their digits when they
// are rounded to 16 bits; bf16: down by 2^31, so that no sum over a context, which has at most 2^30 keys,
// overflows whatever the values are (fp16 values cannot).
constexpr float kLog2e = 1.4426950408889634f;
template <typename T>
constexpr float kWeightShift = 15.f;
template <>
constexpr float kWeightShift<__nv_bfloat16> = -31.f;

// Four neighbouring outputs from sums of weighted values and the sum of weights; no weight at all: zero.
template <typename T>
__device__ __forceinline__ void store_output(unsigned short* to, float4 sum, float total) {
    const float inverse = total == 0.f ? 0.f : 1.f / total;
    uint2 packed;
    if constexpr (std::is_same_v<T, __half>) {
        const __half2 a = __floats2half2_rn(sum.x * inverse, sum.y * inverse);
        const __half2 b = __floats2half2_rn(sum.z * inverse, sum.w * inverse);
        packed = make_uint2(*reinterpret_cast<const unsigned int*>(&a), *reinterpret_cast<const unsigned int*>(&b));
    } else {
        const __nv_bfloat162 a = __floats2bfloat162_rn(sum.x * inverse, sum.y * inverse);
        const __nv_bfloat162 b = __floats2bfloat162_rn(sum.z * inverse, sum.w * inverse);
        packed = make_uint2(*reinterpret_cast<const unsigned int*>(&a), *reinterpret_cast<const unsigned int*>(&b));
    }
    *reinterpret_cast<uint2*>(to) = packed;
}

// A launch that may begin while the kernel before it in the stream ends: every kernel here waits (griddepcontrol.wait)
// before it touches global memory, and then that kernel is complete.
template <typename... Params, typename... Args>
cudaError_t launch_early(void (*kernel)(Params...), dim3 grid, int threads, size_t smem, int cluster, cudaStream_t stream,
                         const Args&... args) {
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = cluster;
    attributes[1].val.clusterDim.y = 1;
    attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&config, kernel, args...);
}

// mb_paged_decode.cu
int decode_admitted(const AttentionArgs& a);
int64_t decode_workspace(const AttentionArgs& a);
int decode_attention(const AttentionArgs& a, int element, void* workspace, cudaStream_t stream);
int multiprocessors(int* device, cudaError_t* err);   // of the current device

// mb_paged_prompt.cu
int prompt_admitted(const AttentionArgs& a);
int64_t prompt_workspace(const AttentionArgs& a);
int prompt_attention(const AttentionArgs& a, int element, void* workspace, cudaStream_t stream);

}  // namespace paged
}  // namespace mb
