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
    int32_t block_shift;  // log2 of block_size where it is a power of two, else -1
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
    uint32_t* status;        // the device status word (whole-program kernels)
    uint32_t* timeout_info;  // and the timeout record
    bool fp16;            // 16-bit rows are fp16, not bf16 (kernels that serve both)
};

// ---- work list ---------------------------------------------------------------
// A query tile is `tile_rows` consecutive packed rows of one sequence and KV head:
// packed row r is token r / group, query head kv_head * group + r % group, so that
// the heads of a group share what is read. Its visible positions, in chunks of
// `chunk` positions aligned to multiples of it, form a list: first the chunks
// that hold sink positions, then those from the window's start to the tile's
// last position. An item is a run of one tile's list; a tile that one item covers
// writes its rows, the parts of others leave (m, l, acc) partials to be merged.
struct Kv8Item {
    int32_t seq;
    int32_t row0;    // first packed row
    int32_t c0, c1;  // the run of the tile's list
    int32_t nsink;   // chunks of sinks at its start
    int32_t lo;      // chunk of its first entry after them
    int32_t slot;    // partial slot (times KV heads, plus the head), < 0: whole tile
    int32_t pad;
};
struct Kv8Merge {
    int32_t seq;
    int32_t row0;
    int32_t slot;   // of the first part
    int32_t parts;  // 0: nothing to merge
};
struct Kv8Counters {
    int32_t next;    // cursor over items x KV heads
    int32_t items;
    int32_t merges;
};
struct Kv8Work {
    Kv8Counters* counters;
    Kv8Item* items;
    Kv8Merge* merges;
    float* acc;    // [slot][tile_rows][head_dim], weights relative to 2^m
    float2* ml;    // [slot][tile_rows] (m, l)
    int32_t tile_rows;
    int32_t chunk;
    int32_t min_run;   // shortest run (chunks) a tile is cut into
    int32_t target;    // runs to aim for, over all KV heads
    int32_t round;     // items that run at once (0: not used)
    int32_t groups;    // > 0: one tile per sequence, cut into that many equal ranges (no plan)
    int32_t snap;      // ranges end where sequences do: no tile is cut
    int32_t merge_grid;  // CTAs of the merge, 0: no tile is ever cut
};

constexpr int kKv8Sms = 148;
constexpr int kKv8Sub = 16;  // positions of one MMA tile of the mma.sync kernel

// 16-position tiles per chunk: independent work between a warp's few, long
// dependences (a maximum over lanes, a rescale), as far as registers go. (At
// head_dim 128, 64 x 512-4096 positions: 240 us with two on 12 warps an SM, 234-249
// with one on 16; 4 x 32768: 85 against 99.)
constexpr int kv8_subs(int head_dim, int nq) {
    return nq > 2 || head_dim == 256 ? 1 : head_dim == 128 || nq == 2 ? 2 : 4;
}

// Its CTAs per SM, by registers and shared memory.
constexpr int kv8_resident(int head_dim, int nq) { return head_dim * nq >= 512 || head_dim == 256 ? 2 : 3; }

// Most sequences of a call without a plan (longer batches take several).
constexpr int kKv8SelfSeqs = 512;

// (The kernels start while the one before them drains, which may be writing the
// cache: their loads are plain ones, never through the read-only path.)

// Carves the workspace for a work list whose tile_rows, chunk, min_run and target
// are set (base may be NULL to learn the size, returned in bytes).
size_t kv8_work_layout(Kv8Work& w, unsigned char* base, int32_t num_seqs, int32_t max_query_len,
                       int32_t max_context_len, int32_t group, const ArenaGeom& g);
cudaError_t launch_kv8_plan(const Kv8AttnParams& p, const Kv8Work& w, cudaStream_t stream);
cudaError_t launch_kv8_merge(const Kv8AttnParams& p, const Kv8Work& w, int32_t dtype,
                             cudaStream_t stream);

// Block-table entry and slot of a position.
__device__ __forceinline__ void kv8_place(const Kv8Arena& a, int pos, int& entry, int& slot) {
    entry = a.block_shift >= 0 ? pos >> a.block_shift : pos / a.block_size;
    slot = pos - entry * a.block_size;
}

// 16 bytes from global to shared memory, or zeros where there is nothing to read.
__device__ __forceinline__ void kv8_copy16(uint32_t dst, const unsigned char* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void kv8_copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void kv8_copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Position of entry c of a tile's list, in chunks.
__device__ __forceinline__ int kv8_chunk(const Kv8Item& it, int c) {
    return c < it.nsink ? c : it.lo + c - it.nsink;
}

// True when the sequence's metadata agree with the call's bounds.
__device__ __forceinline__ bool kv8_metadata_ok(const Kv8AttnParams& p, int q0, int qlen, int ctx) {
    return q0 >= 0 && qlen >= 0 && qlen <= ctx && qlen <= p.max_query_len &&
           ctx <= p.max_context_len && int64_t(ctx) <= int64_t(p.max_blocks) * p.a.block_size;
}

// One sequence's rows and tiles; rows < 0: metadata that contradict the bounds.
struct Kv8Seq {
    int first_pos;  // position of its first new row
    int rows;       // packed rows
    int ntiles;
};
__device__ __forceinline__ Kv8Seq kv8_seq(const Kv8AttnParams& p, const Kv8Work& w, int s) {
    const int q0 = p.cu_seqlens_q[s];
    const int qlen = p.cu_seqlens_q[s + 1] - q0;
    const int ctx = p.context_lens[s];
    if (!kv8_metadata_ok(p, q0, qlen, ctx)) return {0, -1, 0};
    const int rows = qlen * p.group;
    return {ctx - qlen, rows, (rows + w.tile_rows - 1) / w.tile_rows};
}

// The list of tile t: chunks in all, of which sinks, and the first after them.
struct Kv8List {
    int n, nsink, lo;
};
__device__ __forceinline__ Kv8List kv8_list(const Kv8AttnParams& p, const Kv8Work& w,
                                            const Kv8Seq& q, int t) {
    const int r0 = t * w.tile_rows;
    const int r1 = min(r0 + w.tile_rows, q.rows) - 1;
    const int p0 = q.first_pos + r0 / p.group;
    const int p1 = q.first_pos + r1 / p.group;
    const int first = p.window > 0 ? max(0, p0 - p.window + 1) : 0;
    const int lo = first / w.chunk;
    const int nsink = min((min(p.sinks, first) + w.chunk - 1) / w.chunk, lo);
    return {nsink + p1 / w.chunk + 1 - lo, nsink, lo};
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

// The kernel for few rows per KV head (kv8_attention.cuh; fp32: else 16-bit rows).
template <int HD>
cudaError_t launch_kv8_rows(const Kv8AttnParams& p, const Kv8Work& w, bool fp32, int32_t format,
                            cudaStream_t stream);

// The kernel for many rows per KV head (kv8_attention_tc.cu).
bool kv8_tc_supported(int32_t dtype, int32_t head_dim);
Kv8Work kv8_tc_work();
cudaError_t launch_kv8_tc(const Kv8AttnParams& p, const Kv8Work& w, int32_t dtype, int32_t format,
                          cudaStream_t stream);

}  // namespace nvllm
