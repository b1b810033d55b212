// Causal attention over the 8-bit paged cache, in its simplest form: a warp per
// (row, query head) walks the visible positions, a position's scores by a
// butterfly of shuffles, online softmax in the log2 domain, all in fp32:
//   s_j = scale q . K_j,  o = sum_j 2^(s_j - m) V_j / sum_j 2^(s_j - m)
// over j <= p, and with a window j > p - window or j < sinks.
#include "kv8.cuh"

namespace nvllm {

namespace {

constexpr int kWarps = 8;

template <typename T, int kFormat, int HD>
__global__ void __launch_bounds__(kWarps * 32) kv8_attention_kernel(const Kv8AttnParams p) {
    constexpr int PER = HD >= 128 ? HD / 32 : 4;  // dims per lane
    constexpr int LANES = HD / PER;               // lanes that hold a row
    pdl_release();
    pdl_wait();
    const int s = blockIdx.y;
    const int head = blockIdx.x;
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const bool on = lane < LANES;
    const int q0 = p.cu_seqlens_q[s];
    const int qlen = p.cu_seqlens_q[s + 1] - q0;
    const int ctx = p.context_lens[s];
    if (!kv8_metadata_ok(p, q0, qlen, ctx)) {
        if (head == 0 && threadIdx.x == 0) raise_status(kStatusMetadata);
        return;
    }
    const int kvh = head / p.group;
    const int32_t* table = p.block_tables + int64_t(s) * p.max_blocks;
    for (int i = warp; i < qlen; i += kWarps) {
        const int pos = ctx - qlen + i;
        const T* qr = static_cast<const T*>(p.q) + int64_t(q0 + i) * p.q_stride + head * HD;
        float q[PER], o[PER];
#pragma unroll
        for (int d = 0; d < PER; ++d) {
            q[d] = on ? to_float(qr[lane * PER + d]) * p.qk_scale_log2 : 0.f;
            o[d] = 0.f;
        }
        float m = -INFINITY, l = 0.f;
        const int first = p.window > 0 ? max(0, pos - p.window + 1) : 0;
        const int nsink = p.window > 0 ? min(p.sinks, first) : 0;
        const int total = nsink + pos - first + 1;
        for (int n = 0; n < total; ++n) {
            const int j = n < nsink ? n : first + n - nsink;
            const int64_t blk = table[j / p.a.block_size];
            const int in = j % p.a.block_size;
            const bool ok = blk >= 0 && blk < p.a.num_blocks;
            if (!ok && lane == 0) raise_status(kStatusBounds);
            float k[PER], v[PER];
#pragma unroll
            for (int d = 0; d < PER; ++d) k[d] = v[d] = 0.f;
            if (ok && on) {
                const int64_t at = blk * p.a.block_stride + in * p.a.row + int64_t(kvh) * HD + lane * PER;
                const int64_t ea = blk * p.a.exp_block_stride + int64_t(kvh) * p.a.block_size + in;
                const float ks = exp2_int(min(max(int(p.a.k_exps[ea]), -126), 127));
                const float vs = exp2_int(min(max(int(p.a.v_exps[ea]), -126), 127));
#pragma unroll
                for (int d = 0; d < PER; d += 4) {
                    const float4 kc = kv8_codes4<kFormat>(*reinterpret_cast<const uint32_t*>(p.a.k_codes + at + d));
                    const float4 vc = kv8_codes4<kFormat>(*reinterpret_cast<const uint32_t*>(p.a.v_codes + at + d));
                    k[d] = kc.x * ks; k[d + 1] = kc.y * ks; k[d + 2] = kc.z * ks; k[d + 3] = kc.w * ks;
                    v[d] = vc.x * vs; v[d + 1] = vc.y * vs; v[d + 2] = vc.z * vs; v[d + 3] = vc.w * vs;
                }
            }
            float sc = 0.f;
#pragma unroll
            for (int d = 0; d < PER; ++d) sc = fmaf(q[d], k[d], sc);
            sc = warp_sum_xor(sc, 32);
            const float mn = fmaxf(m, sc);
            const float alpha = exp2f(m - mn);
            const float w = exp2f(sc - mn);
            l = fmaf(l, alpha, w);
            m = mn;
#pragma unroll
            for (int d = 0; d < PER; ++d) o[d] = fmaf(o[d], alpha, w * v[d]);
        }
        T* orow = static_cast<T*>(p.out) + int64_t(q0 + i) * p.out_stride + head * HD;
#pragma unroll
        for (int d = 0; d < PER; ++d) {
            if (on) orow[lane * PER + d] = from_float<T>(o[d] / l);
        }
    }
}

template <typename T, int kFormat>
cudaError_t launch_hd(const Kv8AttnParams& p, cudaStream_t st) {
    const dim3 grid(unsigned(p.a.num_heads * p.group), unsigned(p.num_seqs));
    const dim3 block(kWarps * 32);
    switch (p.a.head_dim) {
        case 32: return launch_programmatic(kv8_attention_kernel<T, kFormat, 32>, grid, block, 0, st, p);
        case 64: return launch_programmatic(kv8_attention_kernel<T, kFormat, 64>, grid, block, 0, st, p);
        case 128: return launch_programmatic(kv8_attention_kernel<T, kFormat, 128>, grid, block, 0, st, p);
        case 256: return launch_programmatic(kv8_attention_kernel<T, kFormat, 256>, grid, block, 0, st, p);
        default: return cudaErrorInvalidValue;
    }
}

template <typename T>
cudaError_t launch_type(const Kv8AttnParams& p, int32_t format, cudaStream_t st) {
    return format == NVLLM_KV8_E4M3 ? launch_hd<T, NVLLM_KV8_E4M3>(p, st)
                                    : launch_hd<T, NVLLM_KV8_INT8>(p, st);
}

}  // namespace

size_t kv8_attention_workspace(int32_t, int32_t, int32_t, int32_t, const ArenaGeom&) { return 256; }

cudaError_t launch_kv8_attention(const Kv8AttnParams& p, int32_t dtype, int32_t format, void*,
                                 cudaStream_t stream) {
    switch (dtype) {
        case NVLLM_DTYPE_FP32: return launch_type<float>(p, format, stream);
        case NVLLM_DTYPE_BF16: return launch_type<__nv_bfloat16>(p, format, stream);
        case NVLLM_DTYPE_FP16: return launch_type<__half>(p, format, stream);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace nvllm
