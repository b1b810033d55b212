// Attention over the 8-bit paged cache: which kernel takes a call, its work list and
// workspace. Sequences of few rows per KV head go to the mma.sync kernel
// (kv8_attention.cuh), a tile each; prompts and chunks in bf16 or fp16 at head_dim
// 64 and 128 to the tensor-memory kernel (kv8_attention_tc.cu), the rest of them
// to the mma.sync kernel, several tiles a sequence.
#include <algorithm>

#include "kv8.cuh"

namespace nvllm {

namespace {

cudaError_t launch_rows(const Kv8AttnParams& p, const Kv8Work& w, bool fp32, int32_t format,
                        cudaStream_t st) {
    switch (p.a.head_dim) {
        case 32: return launch_kv8_rows<32>(p, w, fp32, format, st);
        case 64: return launch_kv8_rows<64>(p, w, fp32, format, st);
        case 128: return launch_kv8_rows<128>(p, w, fp32, format, st);
        case 256: return launch_kv8_rows<256>(p, w, fp32, format, st);
        default: return cudaErrorInvalidValue;
    }
}

// Columns (rows of one term) of 8-column MMA tiles for this many packed rows.
int columns_for(int64_t rows, int one, int head_dim) {
    return rows <= one ? 1 : rows <= 2 * one || head_dim > 128 ? 2 : 4;
}

// Rows of one 8-column tile.
int rows_of_tile(int32_t dtype) { return dtype == NVLLM_DTYPE_FP32 ? 4 : 8; }

// The work list of a batch whose sequences are one tile each.
Kv8Work self_work(int nq, int32_t dtype, bool snap, const ArenaGeom& g) {
    Kv8Work w{};
    w.tile_rows = nq * rows_of_tile(dtype);
    w.chunk = kKv8Sub * kv8_subs(g.head_dim, nq);
    w.groups = std::max(1, kKv8Sms * kv8_resident(g.head_dim, nq) / g.num_heads);
    w.min_run = std::max(1, 256 / w.chunk);
    w.snap = snap;
    return w;
}

// Sequences that see at most this many positions are not cut: a cut costs its partials
// and the merge. Both sides measured, whole | cut, us, bf16 head_dim 128 (2048 units:
// fp32):
//   seen                          512         1024        1280        2048        4096
//   8 (sequence, KV head) units   16.4 | 40   22.5 | 40   26.6 | 41   36.9 | 38   61 | 46
//   32                            18.4 | 26   24.6 | 32   28.7 | 26   38.9 | 38   70 | 43
//   128                           20.5 | 24   30.7 | 34   34.8 | 34   49.2 | 40   84 | 54
//   256                           26.6 | 34   36.9 | 42   43.0 | 44   55.4 | 56   92 | 82
//   2048                          76 | 81     121 | 124   145 | 147   210 | 214   385 | 388
constexpr int kWholeFew = 1280;   // where the units are fewer than the SMs
constexpr int kWholeMany = 2048;

// seen: most positions that a tile sees.
Kv8Work work_for(int32_t max_query_len, int64_t seen, int64_t units, int32_t group, int32_t dtype,
                 const ArenaGeom& g) {
    const int one = rows_of_tile(dtype);
    const int64_t rows = int64_t(max_query_len) * group;
    const int nq = columns_for(rows, one, g.head_dim);
    if (rows <= nq * one) return self_work(nq, dtype, seen <= (units >= kKv8Sms ? kWholeMany : kWholeFew), g);
    if (kv8_tc_supported(dtype, g.head_dim)) return kv8_tc_work();
    Kv8Work w{};
    w.tile_rows = nq * one;
    w.chunk = kKv8Sub * kv8_subs(g.head_dim, nq);
    w.min_run = 512 / w.chunk;
    w.target = kKv8Sms * kv8_resident(g.head_dim, nq) * 5;
    return w;
}

}  // namespace

size_t kv8_attention_workspace(int32_t num_seqs, int32_t max_query_len, int32_t max_context_len,
                               int32_t num_query_heads, const ArenaGeom& g) {
    // of the call itself and of every smaller one: a workspace serves them all
    const int group = num_query_heads / g.num_heads;
    size_t n = 0;
    for (int32_t dtype : {NVLLM_DTYPE_FP32, NVLLM_DTYPE_BF16}) {
        Kv8Work w = work_for(max_query_len, max_context_len, 0, group, dtype, g);
        n = std::max(n, kv8_work_layout(w, nullptr, num_seqs, max_query_len, max_context_len, group, g));
        for (int q = 1; q <= columns_for(int64_t(max_query_len) * group, rows_of_tile(dtype), g.head_dim); q *= 2) {
            Kv8Work self = self_work(q, dtype, max_context_len <= kWholeFew, g);
            n = std::max(n, kv8_work_layout(self, nullptr, num_seqs, 1, max_context_len, 1, g));
        }
    }
    return n;
}

cudaError_t launch_kv8_attention(const Kv8AttnParams& all, int32_t dtype, int32_t format,
                                 void* workspace, cudaStream_t stream) {
    ArenaGeom g{};
    g.num_heads = all.a.num_heads;
    g.head_dim = all.a.head_dim;
    int64_t seen = all.max_context_len;
    if (all.window > 0) seen = std::min(seen, int64_t(all.window) + all.max_query_len + all.sinks);
    Kv8Work w = work_for(all.max_query_len, seen, int64_t(all.num_seqs) * g.num_heads, all.group, dtype, g);
    // without a plan a call counts at most kKv8SelfSeqs sequences itself
    const int step = w.groups > 0 ? kKv8SelfSeqs : all.num_seqs;
    for (int s = 0; s < all.num_seqs; s += step) {
        Kv8AttnParams p = all;
        p.num_seqs = std::min(step, all.num_seqs - s);
        p.block_tables += int64_t(s) * p.max_blocks;
        p.cu_seqlens_q += s;
        p.context_lens += s;
        kv8_work_layout(w, static_cast<unsigned char*>(workspace), p.num_seqs, p.max_query_len,
                        p.max_context_len, p.group, g);
        cudaError_t e = w.groups > 0 ? cudaSuccess : launch_kv8_plan(p, w, stream);
        if (e != cudaSuccess) return e;
        if (w.groups == 0 && kv8_tc_supported(dtype, g.head_dim)) {
            e = device_report(&p.status, &p.timeout_info);
            if (e != cudaSuccess) return e;
            e = launch_kv8_tc(p, w, dtype, format, stream);
        } else if (dtype == NVLLM_DTYPE_FP32) {
            e = launch_rows(p, w, true, format, stream);
        } else {
            p.fp16 = dtype == NVLLM_DTYPE_FP16;
            e = launch_rows(p, w, false, format, stream);
        }
        if (e != cudaSuccess) return e;
        if (w.merge_grid > 0) {
            e = launch_kv8_merge(p, w, dtype, stream);
            if (e != cudaSuccess) return e;
        }
    }
    return cudaSuccess;
}

}  // namespace nvllm
