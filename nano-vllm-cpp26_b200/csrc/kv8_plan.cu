// Work list of the 8-bit cache's attention, and the merge of cut tiles.
//
// The lengths live on the device, so one CTA builds the list: it counts the chunks
// of every tile, W over all KV heads, and cuts tiles into runs of at most
//   L = max(min_run, ceil(W / target)) chunks,
// as equal as they come, so that a few long sequences fill the GPU as well as many
// short ones. A tile of n > L chunks has ceil(n / L) <= 2 n / L parts, so there are
// at most 2 target partial slots over all heads, whatever the batch.
//
// Where no tile is that long (a late chunk of a long prompt: many tiles of nearly
// one length) the tiles of the last, partly filled round of CTAs are cut instead, in
// as many parts as fill it: 512 tiles of 192-256 key tiles on 148 CTAs take 3.5
// rounds in place of 4, 1213 us in place of 1332 (chunk of 4096 at 16384, 32 heads over
// 8 x 128; of 4096 at 8192 566 in place of 593). Fresh causal prompts, whose lists
// average half the longest, measured the same with and without it (8192 rows 742 us,
// 2048 rows 91 us), so it is left to lists that average three quarters. Tiles are
// counted in the order of the sequences, so that the same ones are cut every time.
#include <algorithm>

#include "kv8.cuh"

namespace nvllm {

namespace {

constexpr int kPlanThreads = 1024;

size_t align_up(size_t x) { return (x + 255) / 256 * 256; }

// kWide: a warp per sequence, its lanes over the tiles; else a thread per sequence.
template <bool kWide>
__global__ void __launch_bounds__(kPlanThreads) kv8_plan_kernel(const Kv8AttnParams p, const Kv8Work w) {
    __shared__ unsigned long long total;
    __shared__ int longest;
    __shared__ int tiles_before[kWide ? kPlanThreads : 1];  // kWide: of earlier sequences
    __shared__ int warp_tiles[kPlanThreads / 32];
    __shared__ int n_items, n_slots, n_merges;
    const int lane = threadIdx.x & 31;
    const int me = kWide ? threadIdx.x >> 5 : threadIdx.x;
    constexpr int kSeqs = kWide ? kPlanThreads / 32 : kPlanThreads;
    constexpr int kStep = kWide ? 32 : 1;
    const int t0 = kWide ? lane : 0;
    if (threadIdx.x == 0) {
        total = 0;
        longest = 0;
        n_items = n_slots = n_merges = 0;
    }
    pdl_release();
    pdl_wait();  // the metadata may come from the kernel before; the workspace is its
    __syncthreads();
    if constexpr (kWide) tiles_before[threadIdx.x] = 0;
    __syncthreads();
    long long mine = 0;
    int most = 0;
    for (int s = me; s < p.num_seqs; s += kSeqs) {
        const Kv8Seq q = kv8_seq(p, w, s);
        if (q.rows < 0 && t0 == 0) raise_status(kStatusMetadata);
        for (int t = t0; t < q.ntiles; t += kStep) {
            const int n = kv8_list(p, w, q, t).n;
            mine += n;
            most = max(most, n);
        }
        if (kWide && lane == 0 && s < kPlanThreads) tiles_before[s] = q.ntiles;
    }
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) atomicMax(&longest, most);
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane == 0 && mine) atomicAdd(&total, (unsigned long long)mine);
    __syncthreads();
    const long long all = (long long)total * p.a.num_heads;
    const int run = int(max((long long)w.min_run, (all + w.target - 1) / w.target));
    // from which tile on (in the order of the sequences) the last round's are cut
    int cut_from = INT32_MAX, cut_parts = 1;
    if constexpr (kWide) {
        int x = tiles_before[threadIdx.x];
        const int own = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) warp_tiles[threadIdx.x >> 5] = x;
        __syncthreads();
        int tiles = 0;
        x -= own;
        for (int i = 0; i < kPlanThreads / 32; ++i) {
            if (i < int(threadIdx.x >> 5)) x += warp_tiles[i];
            tiles += warp_tiles[i];
        }
        tiles_before[threadIdx.x] = x;
        __syncthreads();
        const int H = p.a.num_heads;
        const long long units = (long long)tiles * H;
        const long long rest = w.round > 0 ? units % w.round : 0;
        // lists of one length, or nearly (three quarters on average), and none cut
        if (p.num_seqs <= kPlanThreads && units > w.round && rest > 0 && run >= longest &&
            (long long)total * 4 >= (long long)longest * tiles * 3) {
            const int last = int((rest + H - 1) / H);  // tiles of the last round
            cut_parts = w.round / (last * H);
            if (cut_parts > 1) cut_from = tiles - last;
        }
    }
    // the longest lists, those of a sequence's last tiles, go out first
    for (int base = 0; base < p.num_seqs; base += kSeqs) {
        const int s = base + me;
        const Kv8Seq q = s < p.num_seqs ? kv8_seq(p, w, s) : Kv8Seq{0, 0, 0};
        for (int i = 0;; i += kStep) {
            const int t = q.ntiles - 1 - i - t0;
            if (!__any_sync(0xffffffffu, t >= 0)) break;
            const Kv8List l = t >= 0 ? kv8_list(p, w, q, t) : Kv8List{0, 0, 0};
            int parts = t < 0 ? 0 : l.n > run ? (l.n + run - 1) / run : 1;
            if (kWide && t >= 0 && cut_from != INT32_MAX && tiles_before[s] + i + t0 >= cut_from) {
                parts = max(1, min(cut_parts, l.n / (4 * w.min_run)));  // shorter ones cost what they save
            }
            const int slots = parts > 1 ? parts : 0;
            // this lane's places: an inclusive scan of both counts in one word
            long long x = ((long long)(slots) << 32) | (unsigned)parts;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long long y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            const unsigned cut = __ballot_sync(0xffffffffu, slots > 0);
            int bi = 0, bs = 0, bm = 0;
            if (lane == 31) {
                bi = atomicAdd(&n_items, int(x & 0xffffffff));
                if (cut) {
                    bs = atomicAdd(&n_slots, int(x >> 32));
                    bm = atomicAdd(&n_merges, __popc(cut));
                }
            }
            bi = __shfl_sync(0xffffffffu, bi, 31) + int(x & 0xffffffff) - parts;
            bs = __shfl_sync(0xffffffffu, bs, 31) + int(x >> 32) - slots;
            bm = __shfl_sync(0xffffffffu, bm, 31) + __popc(cut & ((1u << lane) - 1));
            // a tile in many parts is written by the warp together, the others by their lanes
            constexpr int kFew = 8;
            for (int k = 0; k < parts && parts <= kFew; ++k) {
                w.items[bi + k] = Kv8Item{s, t * w.tile_rows, int((long long)l.n * k / parts),
                                          int((long long)l.n * (k + 1) / parts), l.nsink, l.lo,
                                          parts > 1 ? bs + k : -1, 0};
            }
            if (slots > 0) w.merges[bm] = Kv8Merge{s, t * w.tile_rows, bs, parts};
            for (unsigned left = __ballot_sync(0xffffffffu, parts > kFew); left; left &= left - 1) {
                const int from = __ffs(left) - 1;
                const int n = __shfl_sync(0xffffffffu, parts, from);
                const int i0 = __shfl_sync(0xffffffffu, bi, from);
                const int s0 = __shfl_sync(0xffffffffu, bs, from);
                const long long len = __shfl_sync(0xffffffffu, l.n, from);
                Kv8Item item{__shfl_sync(0xffffffffu, s, from),
                             __shfl_sync(0xffffffffu, t, from) * w.tile_rows,
                             0,
                             0,
                             __shfl_sync(0xffffffffu, l.nsink, from),
                             __shfl_sync(0xffffffffu, l.lo, from),
                             0,
                             0};
                for (int k = lane; k < n; k += 32) {
                    item.c0 = int(len * k / n);
                    item.c1 = int(len * (k + 1) / n);
                    item.slot = s0 + k;
                    w.items[i0 + k] = item;
                }
            }
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) *w.counters = Kv8Counters{0, n_items, n_merges};
}

// out = sum_k acc_k 2^(m_k - M) / sum_k l_k 2^(m_k - M), M = max_k m_k: a warp per
// (cut tile, KV head, row), parts in order. Without a plan the list has an entry for
// every range, most of them empty, and the grid is that of the tiles: with few
// (sequence, KV head) units each warp steps through many entries, which is most of
// the call (1 x 16384 positions, one head, fp32: 126 us).
template <typename T, int HD>
__global__ void __launch_bounds__(256) kv8_merge_kernel(const Kv8AttnParams p, const Kv8Work w) {
    constexpr int PER = HD / 32;
    pdl_release();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int H = p.a.num_heads;
    // without a plan every range has an entry; a range's partials are its first
    // tile's, which began in an earlier range, then its last one's
    const long long merges = w.groups > 0 ? w.groups : w.counters->merges;
    const long long total = merges * H * w.tile_rows;
    for (long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); i < total; i += gridDim.x * 8ll) {
        const int r = int(i % w.tile_rows);
        const int h = int(i / w.tile_rows % H);
        const Kv8Merge m = w.merges[i / w.tile_rows / H];
        if (m.parts == 0) continue;
        const int q0 = p.cu_seqlens_q[m.seq];
        const int row = m.row0 + r;
        if (row >= (p.cu_seqlens_q[m.seq + 1] - q0) * p.group) continue;
        const auto at = [&](int k) { 
            const int slot = m.slot + (w.groups > 0 && k > 0 ? 2 * k - 1 : k);
            return (int64_t(slot) * H + h) * w.tile_rows + r;
        };
        float M = -INFINITY;
        for (int k = lane; k < m.parts; k += 32) M = fmaxf(M, __ldcg(&w.ml[at(k)].x));
        M = warp_max_xor(M, 32);
        float L = 0.f, o[PER];
#pragma unroll
        for (int d = 0; d < PER; ++d) o[d] = 0.f;
        // a part in which the row sees nothing has m = -inf, l = 0
        for (int k = 0; k < m.parts; k += 4) {
            float2 ml[4];
            float a[4][PER];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (k + u < m.parts) {
                    ml[u] = __ldcg(&w.ml[at(k + u)]);
#pragma unroll
                    for (int d = 0; d < PER; ++d) a[u][d] = __ldcg(w.acc + at(k + u) * HD + d * 32 + lane);
                } else {
                    ml[u] = make_float2(-INFINITY, 0.f);
#pragma unroll
                    for (int d = 0; d < PER; ++d) a[u][d] = 0.f;
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                // (a part may have all of the weight and 2^-200 of the values: the square
                // root of the factor, twice)
                const float root = ml[u].x == -INFINITY ? 0.f : exp2f(0.5f * (ml[u].x - M));
                L = fmaf(ml[u].y * root, root, L);
                const float f = root * root;
#pragma unroll
                for (int d = 0; d < PER; ++d) o[d] = fmaf(a[u][d], f, o[d]);
            }
        }
        const float inv = 1.0f / L;
        T* dst = static_cast<T*>(p.out) + int64_t(q0 + row / p.group) * p.out_stride +
                 int64_t(h * p.group + row % p.group) * HD;
#pragma unroll
        for (int d = 0; d < PER; ++d) dst[d * 32 + lane] = from_float<T>(o[d] * inv);
    }
}

template <typename T>
cudaError_t launch_merge_type(const Kv8AttnParams& p, const Kv8Work& w, cudaStream_t st) {
    const dim3 grid(unsigned(w.merge_grid)), block(256);
    switch (p.a.head_dim) {
        case 32: return launch_programmatic(kv8_merge_kernel<T, 32>, grid, block, 0, st, p, w);
        case 64: return launch_programmatic(kv8_merge_kernel<T, 64>, grid, block, 0, st, p, w);
        case 128: return launch_programmatic(kv8_merge_kernel<T, 128>, grid, block, 0, st, p, w);
        case 256: return launch_programmatic(kv8_merge_kernel<T, 256>, grid, block, 0, st, p, w);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace

size_t kv8_work_layout(Kv8Work& w, unsigned char* base, int32_t num_seqs, int32_t max_query_len,
                       int32_t max_context_len, int32_t group, const ArenaGeom& g) {
    const int64_t tiles = (int64_t(max_query_len) * group + w.tile_rows - 1) / w.tile_rows;
    const int64_t units = int64_t(num_seqs) * tiles;
    // most chunks of one tile: two more than the positions, for the sinks' and the
    // window's ragged ends
    const int64_t chunks = (int64_t(max_context_len) + w.chunk - 1) / w.chunk + 2;
    const bool cut = chunks > w.min_run;
    const int64_t parts = cut ? (chunks + w.min_run - 1) / w.min_run : 1;
    int64_t slots = cut ? std::min<int64_t>(2 * int64_t(w.target) / g.num_heads + 1, units * parts) : 0;
    int64_t merges = slots;
    if (w.groups > 0) {
        merges = w.snap ? 0 : w.groups;
        slots = 2 * merges;
    }
    size_t off = 0;
    auto take = [&](size_t bytes) {
        unsigned char* at = base + off;
        off = align_up(off + bytes);
        return at;
    };
    w.counters = reinterpret_cast<Kv8Counters*>(take(sizeof(Kv8Counters)));
    w.items = reinterpret_cast<Kv8Item*>(take(size_t(w.groups > 0 ? 0 : units + slots) * sizeof(Kv8Item)));
    w.merges = reinterpret_cast<Kv8Merge*>(take(size_t(merges) * sizeof(Kv8Merge)));
    w.ml = reinterpret_cast<float2*>(take(size_t(slots) * g.num_heads * w.tile_rows * sizeof(float2)));
    w.acc = reinterpret_cast<float*>(take(size_t(slots) * g.num_heads * w.tile_rows * g.head_dim * sizeof(float)));
    const int64_t rows = std::min<int64_t>(units, merges) * g.num_heads * w.tile_rows;
    w.merge_grid = int32_t(std::min<int64_t>((rows + 7) / 8, 148 * 4));
    return off;
}

cudaError_t launch_kv8_plan(const Kv8AttnParams& p, const Kv8Work& w, cudaStream_t stream) {
    const int64_t tiles = (int64_t(p.max_query_len) * p.group + w.tile_rows - 1) / w.tile_rows;
    // a warp per sequence pays from a few tiles on; decode batches have one
    return launch_programmatic(tiles > 4 ? kv8_plan_kernel<true> : kv8_plan_kernel<false>, dim3(1),
                               dim3(kPlanThreads), 0, stream, p, w);
}

cudaError_t launch_kv8_merge(const Kv8AttnParams& p, const Kv8Work& w, int32_t dtype,
                             cudaStream_t stream) {
    switch (dtype) {
        case NVLLM_DTYPE_FP32: return launch_merge_type<float>(p, w, stream);
        case NVLLM_DTYPE_BF16: return launch_merge_type<__nv_bfloat16>(p, w, stream);
        case NVLLM_DTYPE_FP16: return launch_merge_type<__half>(p, w, stream);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace nvllm
