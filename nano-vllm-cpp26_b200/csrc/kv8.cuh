// The 8-bit paged KV cache: formats, parameters and launch interfaces shared by
// its kernels and its C ABI (kv8_abi.cu).
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "kernels.cuh"

namespace nvllm {

constexpr int kKv8MinExp = -100;  // rows below it store small codes or zeros
constexpr int kKv8MaxExp = 119;   // 448 * 2^119 is the largest value a row can hold

// An arena of one layer: base pointers and strides. Codes are bytes, so the
// strides of ArenaGeom (in elements) are byte strides; the exponents of block b,
// head h, slot s are at b * exp_block_stride + layer_off + h * block_size + s.
struct Kv8Arena {
    unsigned char* k_codes;  // at the call's layer
    unsigned char* v_codes;
    int8_t* k_exps;          // at the call's layer
    int8_t* v_exps;
    int64_t block_stride;      // codes, bytes from block to block
    int64_t row;               // codes, bytes from slot to slot (num_heads * head_dim)
    int64_t exp_block_stride;  // exponents from block to block
    int64_t num_blocks;
    int32_t block_size;
    int32_t num_heads;  // KV heads
    int32_t head_dim;
};

// Rows of key/value (write: in, read: out).
struct Kv8Rows {
    void* key;
    void* value;
    int64_t key_stride;    // elements
    int64_t value_stride;  // elements
    const int32_t* slots;
    int64_t num_tokens;
};

struct Kv8AttnParams {
    void* out;
    const void* q;
    int64_t out_stride;  // elements
    int64_t q_stride;    // elements
    Kv8Arena a;
    const int32_t* block_tables;
    const int32_t* cu_seqlens_q;
    const int32_t* context_lens;
    int32_t max_blocks;
    int32_t num_seqs;
    int32_t max_query_len;
    int32_t max_context_len;
    int32_t group;  // query heads per KV head
    int32_t window;
    int32_t sinks;
    float qk_scale_log2;  // softmax scale * log2(e)
};

// True when the sequence's metadata agree with the call's bounds.
__device__ __forceinline__ bool kv8_metadata_ok(const Kv8AttnParams& p, int q0, int qlen, int ctx) {
    return q0 >= 0 && qlen >= 0 && qlen <= ctx && qlen <= p.max_query_len &&
           ctx <= p.max_context_len && int64_t(ctx) <= int64_t(p.max_blocks) * p.a.block_size;
}

// 2^e for e in [-126, 127].
__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((e + 127) << 23); }

// Four E4M3 or INT8 codes, the lowest byte first, as fp32.
template <int kFormat>
__device__ __forceinline__ float4 kv8_codes4(uint32_t w) {
    if constexpr (kFormat == NVLLM_KV8_E4M3) {
        uint32_t lo, hi;
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
            "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo));
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        return make_float4(a.x, a.y, b.x, b.y);
    } else {
        // 2^23 + (code + 128) as fp32 bits, less 2^23 + 128: exact
        const uint32_t u = w ^ 0x80808080u;
        const float c = 8388736.0f;
        return make_float4(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440)) - c,
                           __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7441)) - c,
                           __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7442)) - c,
                           __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7443)) - c);
    }
}

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) {
    return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// vec: rows and strides 16-byte aligned.
cudaError_t launch_kv8_write(const Kv8Arena& a, const Kv8Rows& r, int32_t dtype, int32_t format,
                             bool vec, cudaStream_t stream);
cudaError_t launch_kv8_read(const Kv8Arena& a, const Kv8Rows& r, int32_t dtype, int32_t format,
                            bool vec, cudaStream_t stream);

size_t kv8_attention_workspace(int32_t num_seqs, int32_t max_query_len, int32_t max_context_len,
                               int32_t num_query_heads, const ArenaGeom& g);
cudaError_t launch_kv8_attention(const Kv8AttnParams& p, int32_t dtype, int32_t format,
                                 void* workspace, cudaStream_t stream);

}  // namespace nvllm
