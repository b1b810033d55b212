// The extern "C" entry points of the 8-bit paged KV cache (declared in
// include/nvllm.h): argument checks and dispatch.
#include <cstdint>

#include "../../include/nvllm.h"
#include "kv8.cuh"

using namespace nvllm;

namespace {

bool aligned16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; }

int element_bytes(int32_t dtype) {
    switch (dtype) {
        case NVLLM_DTYPE_FP32: return 4;
        case NVLLM_DTYPE_BF16:
        case NVLLM_DTYPE_FP16: return 2;
        default: return 0;
    }
}

// Fills a from the arena handle at one layer (NVLLM_OK or the status to return).
int prepare_arena(Kv8Arena& a, const nvllm_kv8_arena* arena, int32_t layer,
                  const nvllm_kv_layout* lay) {
    if (arena == nullptr || !arena->k_codes || !arena->v_codes || !arena->k_exps || !arena->v_exps) {
        return NVLLM_ERR_INVALID;
    }
    if (arena->format != NVLLM_KV8_E4M3 && arena->format != NVLLM_KV8_INT8) return NVLLM_ERR_INVALID;
    if (!aligned16(arena->k_codes) || !aligned16(arena->v_codes)) return NVLLM_ERR_INVALID;
    const ArenaGeom g = make_geom(lay);
    const int64_t exp_layer = int64_t(g.num_heads) * g.block_size;
    a.k_codes = static_cast<unsigned char*>(arena->k_codes) + layer * g.layer_stride;
    a.v_codes = static_cast<unsigned char*>(arena->v_codes) + layer * g.layer_stride;
    a.k_exps = arena->k_exps + layer * exp_layer;
    a.v_exps = arena->v_exps + layer * exp_layer;
    a.block_stride = g.block_stride;
    a.row = g.row;
    a.exp_block_stride = g.num_layers * exp_layer;
    a.num_blocks = g.num_blocks;
    a.block_size = g.block_size;
    a.block_shift = -1;
    for (int i = 0; i < 31; ++i) {
        if (g.block_size == (1 << i)) a.block_shift = i;
    }
    a.num_heads = g.num_heads;
    a.head_dim = g.head_dim;
    return NVLLM_OK;
}

int move_rows(bool write, void* key, void* value, int32_t dtype, int64_t key_stride,
              int64_t value_stride, const nvllm_kv8_arena* arena, const int32_t* slot_mapping,
              int64_t num_tokens, int32_t layer, const nvllm_kv_layout* layout, void* stream) {
    const int lv = validate_layout(layout);
    if (lv != NVLLM_OK) return lv;
    const int size = element_bytes(dtype);
    if (size == 0 || num_tokens < 0 || layer < 0 || layer >= layout->num_layers) {
        return NVLLM_ERR_INVALID;
    }
    if (num_tokens == 0) return NVLLM_OK;
    const int64_t row = int64_t(layout->num_heads) * layout->head_dim;
    // the kernels count pieces of 16 values in 32 bits
    if (num_tokens > INT32_MAX || num_tokens > int64_t(0xFFFFFF00u) / (row / 16)) {
        return NVLLM_ERR_INVALID;
    }
    if (!key || !value || !slot_mapping || key_stride < row || value_stride < row) {
        return NVLLM_ERR_INVALID;
    }
    Kv8Arena a;
    const int rc = prepare_arena(a, arena, layer, layout);
    if (rc != NVLLM_OK) return rc;
    const Kv8Rows r{key, value, key_stride, value_stride, slot_mapping, num_tokens};
    const bool vec = aligned16(key) && aligned16(value) && key_stride * size % 16 == 0 &&
                     value_stride * size % 16 == 0;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t e = write ? launch_kv8_write(a, r, dtype, arena->format, vec, st)
                                : launch_kv8_read(a, r, dtype, arena->format, vec, st);
    return e == cudaSuccess ? NVLLM_OK : NVLLM_ERR_CUDA;
}

// The checks that the workspace query and the call share.
bool attention_sizes_ok(int32_t num_seqs, int32_t max_query_len, int32_t max_context_len,
                        int32_t num_query_heads, const nvllm_kv_layout* lay) {
    return num_seqs >= 0 && max_query_len >= 1 && max_context_len >= max_query_len &&
           num_query_heads >= lay->num_heads && num_query_heads % lay->num_heads == 0 &&
           // rows of a sequence, counted over the heads of a group, and (sequence,
           // head) pairs stay within 32 bits
           int64_t(max_query_len) * (num_query_heads / lay->num_heads) <= INT32_MAX / 2 &&
           int64_t(num_seqs) * num_query_heads <= INT32_MAX / 2 && num_seqs <= 65535;
}

}  // namespace

extern "C" {

int nvllm_kv8_write(const void* key, const void* value, int32_t dtype, int64_t key_stride,
                    int64_t value_stride, const nvllm_kv8_arena* arena,
                    const int32_t* slot_mapping, int64_t num_tokens, int32_t layer,
                    const nvllm_kv_layout* layout, void* stream) {
    return move_rows(true, const_cast<void*>(key), const_cast<void*>(value), dtype, key_stride,
                     value_stride, arena, slot_mapping, num_tokens, layer, layout, stream);
}

int nvllm_kv8_read(void* key, void* value, int32_t dtype, int64_t key_stride,
                   int64_t value_stride, const nvllm_kv8_arena* arena,
                   const int32_t* slot_mapping, int64_t num_tokens, int32_t layer,
                   const nvllm_kv_layout* layout, void* stream) {
    return move_rows(false, key, value, dtype, key_stride, value_stride, arena, slot_mapping,
                     num_tokens, layer, layout, stream);
}

size_t nvllm_kv8_attention_workspace_size(int32_t num_seqs, int32_t max_query_len,
                                          int32_t max_context_len, int32_t num_query_heads,
                                          const nvllm_kv_layout* layout) {
    if (validate_layout(layout) != NVLLM_OK ||
        !attention_sizes_ok(num_seqs, max_query_len, max_context_len, num_query_heads, layout)) {
        return 0;
    }
    return kv8_attention_workspace(num_seqs, max_query_len, max_context_len, num_query_heads,
                                   make_geom(layout));
}

int nvllm_kv8_attention(void* out, int64_t out_stride, const void* query, int64_t query_stride,
                        int32_t dtype, const nvllm_kv8_arena* arena,
                        const int32_t* block_tables, int32_t max_blocks_per_seq,
                        const int32_t* cu_seqlens_q, const int32_t* context_lens,
                        int32_t num_seqs, int32_t max_query_len, int32_t max_context_len,
                        int32_t num_query_heads, int32_t layer, float scale, int32_t window,
                        int32_t sinks, void* workspace, size_t workspace_bytes,
                        const nvllm_kv_layout* layout, void* stream) {
    const int lv = validate_layout(layout);
    if (lv != NVLLM_OK) return lv;
    const int size = element_bytes(dtype);
    if (size == 0 || layer < 0 || layer >= layout->num_layers || window < 0 || sinks < 0 ||
        !attention_sizes_ok(num_seqs, max_query_len, max_context_len, num_query_heads, layout)) {
        return NVLLM_ERR_INVALID;
    }
    if (num_seqs == 0) return NVLLM_OK;
    if (max_blocks_per_seq < 1 ||
        int64_t(max_context_len) > int64_t(max_blocks_per_seq) * layout->block_size) {
        return NVLLM_ERR_INVALID;
    }
    if (!out || !query || !block_tables || !cu_seqlens_q || !context_lens) return NVLLM_ERR_INVALID;
    const int64_t row = int64_t(num_query_heads) * layout->head_dim;
    if (out_stride < row || query_stride < row || !aligned16(out) || !aligned16(query) ||
        out_stride * size % 16 != 0 || query_stride * size % 16 != 0) {
        return NVLLM_ERR_INVALID;
    }
    if (!(scale > 0.0f) || scale > 1e30f) return NVLLM_ERR_INVALID;
    Kv8AttnParams p{};
    const int rc = prepare_arena(p.a, arena, layer, layout);
    if (rc != NVLLM_OK) return rc;
    const size_t need = kv8_attention_workspace(num_seqs, max_query_len, max_context_len,
                                                num_query_heads, make_geom(layout));
    if (workspace == nullptr || workspace_bytes < need ||
        (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) {
        return NVLLM_ERR_WORKSPACE;
    }
    p.out = out;
    p.q = query;
    p.out_stride = out_stride;
    p.q_stride = query_stride;
    p.block_tables = block_tables;
    p.cu_seqlens_q = cu_seqlens_q;
    p.context_lens = context_lens;
    p.max_blocks = max_blocks_per_seq;
    p.num_seqs = num_seqs;
    p.max_query_len = max_query_len;
    p.max_context_len = max_context_len;
    p.group = num_query_heads / layout->num_heads;
    // a window that no context outgrows is none; so bounded, the kernels' sums of
    // positions stay within 32 bits
    p.window = window >= max_context_len ? 0 : window;
    p.sinks = p.window > 0 ? (sinks < max_context_len ? sinks : max_context_len) : 0;
    p.qk_scale_log2 = scale * kLog2e;
    const cudaError_t e = launch_kv8_attention(p, dtype, arena->format, workspace,
                                               static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? NVLLM_OK : NVLLM_ERR_CUDA;
}

}  // extern "C"
