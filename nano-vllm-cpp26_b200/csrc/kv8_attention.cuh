// Attention over the 8-bit paged cache for few rows per KV head (decode, short
// chunks, and every geometry the tensor-memory kernel does not take), on
// mma.sync m16n8k16 with fp32 accumulation.
//
// With q' = q scaled by a power of two to [1, 2) per row, K_j = c_j 2^(a_j) and
// V_j = d_j 2^(b_j) (codes and exponents):
//   x_j = (q' . c_j) 2^(a_j) qs      log2-domain score, qs the scale taken out
//   m   = max_j (x_j + b_j)          largest contribution's size
//   P_j = 2^(x_j + b_j - m),  acc = sum_j P_j d_j,  l = sum_j 2^(x_j - m),  o = acc / l
// Codes are exact in fp16, so the exponents never touch the products, and with m
// the size of contributions (not of weights) P is in [0, 1] and the largest one
// keeps all its bits however far apart the rows' exponents are.
// The largest weight that counts then is between 2^-119 and 2^100 (b_j is in [-100,
// 119]), which leaves no room below for smaller ones: the exponential gives 2^20
// 2^(x_j - m), and its sum is taken times 2^-20 in the instruction that adds, so that
// nothing above 2^-146 is lost. When m moves by more than fp32 spans, l must keep
// what P and acc may drop (rows of zeros have b_j = -100 and may have all of the
// weight): l is rescaled by the square root of the factor, twice. (Both at every
// step: branching to them where some b_j is large cost 1-4 % more.)
//
// Operands are fp16 terms: q' of fp32 rows as two (2^-23 of the row's largest
// element), of bf16 and fp16 rows as one (exact up to 2^-25 of the largest); P of
// fp32 rows as two terms (2^-22), of others as one (2^-11, no more than the
// output's own rounding: bf16 outputs are 1.7e-3 of their norm from 64 bits, as with
// P in fp32).
//
// The products are taken transposed, S^T = K Q^T and O^T = V^T P^T, so that
// positions and dims fill the MMA's 16 rows and the few query rows its 8 columns:
// half the MMAs and accumulators of the other order. The two terms of an fp32 row
// are columns 2r and 2r + 1, which one lane holds, and which it adds; with 4 rows
// or fewer they cost nothing. P's pairs become the next product's operand by one
// 8 x 8 transpose (movmatrix).
//
// What bounds a decode is the cache's bytes. A CTA of 4 warps takes runs of
// chunks (kv8_plan.cu, or without a plan an equal range of a decode batch, see
// SelfRange); a warp takes every fourth chunk of SUB x 16 positions and
// brings them into its own two shared-memory buffers by 16-byte asynchronous
// copies (positions that no row sees as zeros), one chunk in flight while it
// computes the other. Of K, lane (g, t) reads the pieces t, t + 4, .. of rows g
// and g + 8 (the MMA's order of the dims is permuted to match, Q's fragments are
// stored that way); of V, the piece g of rows 2t, 2t + 1, 2t + 8, 2t + 9, whose
// bytes are paired across rows as they are converted. Pieces are placed so that
// both reads are free of bank conflicts (Ring::swizzle). The warps' results are
// joined through shared memory at the end of a run.
//
// Measured on B200: 64 sequences of 512-4096 positions, 32 heads x 128, fp32 rows:
// 244-247 us, 5.0 TB/s (0.76 of the copy rate), latency-bound at 45 % issue with 12
// warps an SM; 4 x 32768 positions, 32 heads over 8, bf16 rows: 82 us, 66 of them here
// and the rest the merge. Few (sequence, KV head) units at a long context are the
// merge's (kv8_plan.cu): one sequence of 32768, 32 heads over 8, 71 us for 10 us of
// bytes; of 131072, 8 heads on one, 372 us.
// The order with query rows on the MMA's 16 rows took 518 us for the first, the
// transposed one with fragments loaded straight into registers 280.
#pragma once

#include <algorithm>

#include "kv8.cuh"

namespace nvllm {

namespace {

constexpr int kWarps = 4;
constexpr int kSub = kKv8Sub;

// Rows are fp32 (T float) or 16-bit, bf16 and fp16 in one kernel (T uint16_t): only
// Q's load and the output's store tell them apart.
template <typename T>
constexpr int terms() { return sizeof(T) == 4 ? 2 : 1; }
__device__ __forceinline__ float value_of(float x, bool) { return x; }
__device__ __forceinline__ float value_of(uint16_t x, bool fp16) {
    return fp16 ? __half2float(__ushort_as_half(x)) : __bfloat162float(__ushort_as_bfloat16(x));
}
__device__ __forceinline__ void put_value(float* dst, float x, bool) { *dst = x; }
__device__ __forceinline__ void put_value(uint16_t* dst, float x, bool fp16) {
    *dst = fp16 ? __half_as_ushort(__float2half_rn(x)) : __bfloat16_as_ushort(__float2bfloat16_rn(x));
}

// Shapes of the fragments at head_dim HD.
template <int HD>
struct Frag {
    static constexpr int KB = HD / 4 < 16 ? HD / 4 : 16;  // bytes of one K piece of a lane
    static constexpr int KP = HD / 4 / KB;                // K pieces of a lane per row
    static constexpr int VB = HD / 8 < 16 ? HD / 8 : 16;  // bytes of one V piece
    static constexpr int VP = HD / 8 / VB;                // V pieces of a lane per row
    static constexpr int KW = KB / 4;                     // words (MMA steps) per K piece
    static constexpr int VW = VB / 4;                     // words (2 MMA tiles each) per V piece
    static constexpr int KSTEPS = HD / 16;
    static constexpr int MTILES = HD / 16;                // 16-dim tiles of O^T
};

template <int BYTES>
struct Piece {
    uint32_t w[BYTES / 4];
};

template <int BYTES>
__device__ __forceinline__ Piece<BYTES> read_piece(const unsigned char* p) {
    Piece<BYTES> r;
    if constexpr (BYTES == 16) {
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w;
    } else if constexpr (BYTES == 8) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        r.w[0] = v.x; r.w[1] = v.y;
    } else {
        r.w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
    return r;
}

// Four codes -> two pairs of fp16, in order.
template <int kFormat>
__device__ __forceinline__ void to_half4(uint32_t w, uint32_t& a, uint32_t& b) {
    if constexpr (kFormat == NVLLM_KV8_E4M3) {
        asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\t"
            "cvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
            : "=r"(a), "=r"(b)
            : "r"(w));
    } else {
        // 1024 + (code + 128) as fp16 bits, less 1152: exact
        const uint32_t u = w ^ 0x80808080u;
        const __half2 c = __half2half2(__ushort_as_half(0x6480));
        uint32_t x = __byte_perm(u, 0x64646464u, 0x4140), y = __byte_perm(u, 0x64646464u, 0x4342);
        const __half2 p = __hsub2(*reinterpret_cast<__half2*>(&x), c);
        const __half2 q = __hsub2(*reinterpret_cast<__half2*>(&y), c);
        a = *reinterpret_cast<const uint32_t*>(&p);
        b = *reinterpret_cast<const uint32_t*>(&q);
    }
}

__device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 2^kUpBy times a weight is at most 2^(100 + kMargin + 2 + 20) < 2^128 (2: half a step
// of the largest scores, by which m is off). Added after m is taken off: beside a score
// beyond 2^27 it would be rounded away.
constexpr float kUpBy = 20.0f;

// a, b as fp16 in one word (a low).
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_rest(float a, float b, uint32_t h) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    return pack_half(a - f.x, b - f.y);
}

// The 8 x 8 transpose of 16-bit values held as fragments.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// O of a row is rescaled only when the largest contribution grows by more than
// this (log2): until then P <= 2^margin, and it cancels in acc / l.
constexpr float kMargin = 4.0f;

// One 16-position tile of K or V in shared memory: rows of HD bytes, the 16-byte
// pieces of a 128-byte line permuted by its rows. K's reads take 8 / (HD / 16)
// neighbouring rows' pieces at once, V's the same pieces of rows 0, 2, 4, 6: the
// permutation gives both all eight places of a line.
template <int HD>
struct Ring {
    static constexpr int TILE = kSub * HD;
    static constexpr int PIECES = HD / 16;           // of a row
    static constexpr int STEP = 32 / PIECES;         // rows that the lanes of a warp copy at once
    static constexpr int COPIES = kSub / STEP;       // per lane and tile
    __device__ static __forceinline__ int swizzle(int row) {
        if constexpr (HD >= 128) return ((row >> 1) & 3) * 2 ^ (row & 1) * 4;
        if constexpr (HD == 64) return ((row >> 1) & 3) * 2;
        return ((row >> 2) & 1) * 2;
    }
    // byte offset of byte `b` of row `row`
    __device__ static __forceinline__ int at(int row, int b) {
        return (row * HD + b) ^ (swizzle(row) * 16);
    }
};

template <typename T, int HD, int NQ>
struct Tile {
    static constexpr int ROWS = NQ * 8 / terms<T>();   // rows of a query tile
    static constexpr int Q_WORDS = NQ * (HD / 16) * 64;  // fragments of Q
    static constexpr bool Q_REGS = NQ * (HD / 16) <= 8;  // held in registers
    static constexpr int SUB = kv8_subs(HD, NQ);
    static constexpr int OROW = HD + 4;
    static constexpr size_t BUF = 2 * SUB * Ring<HD>::TILE;        // K and V of a chunk
    static constexpr size_t RING = kWarps * 2 * BUF;
    static constexpr size_t JOIN = size_t(kWarps) * ROWS * (OROW + 2) * 4;  // overlays the buffers
    static constexpr size_t EXPS = RING > JOIN ? RING : JOIN;      // factors of a chunk's positions
    static constexpr size_t Q = EXPS + kWarps * 2 * SUB * 32 * 4;
    static constexpr size_t SCALE = Q + Q_WORDS * 4;
    static constexpr size_t FIRST = SCALE + ROWS * 4;              // chunks before each sequence
    static constexpr size_t SMEM = FIRST + (kKv8SelfSeqs + 1) * 4;
    static constexpr int CTAS = kv8_resident(HD, NQ);
};

// The range of the batch that a CTA takes when there is no plan (one tile per
// sequence): the chunks of all sequences in a row, in w.groups equal ranges; a
// range's CTAs, one per KV head, walk the same positions side by side, so that
// the heads' bytes of a position, which are neighbours in memory, are read at
// about the same time.
struct SelfRange {
    int x, x1;  // chunks of this CTA, from the first of all sequences
    int s;      // sequence of x
};

// All threads: first[s] = chunks before sequence s; returns the CTA's range.
__device__ SelfRange self_range(const Kv8AttnParams& p, const Kv8Work& w, int* first, int grp, bool lead) {
    constexpr int PER = kKv8SelfSeqs / (kWarps * 32);
    __shared__ int warp_sum[kWarps];
    __shared__ int warp_some[kWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int n[PER], sum = 0, some = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int s = threadIdx.x * PER + i;
        n[i] = 0;
        if (s < p.num_seqs) {
            const Kv8Seq q = kv8_seq(p, w, s);
            if (q.rows < 0 && blockIdx.x == 0) raise_status(kStatusMetadata);
            if (q.rows > 0) n[i] = kv8_list(p, w, q, 0).n;
        }
        sum += n[i];
        some += n[i] > 0;
    }
    some = __reduce_add_sync(0xffffffffu, some);
    int x = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) {
        warp_sum[warp] = x;
        warp_some[warp] = some;
    }
    __syncthreads();
    int before = x - sum;
    int total = 0;
    some = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
        before += i < warp ? warp_sum[i] : 0;
        total += warp_sum[i];
        some += warp_some[i];
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        first[threadIdx.x * PER + i] = before;
        before += n[i];
    }
    if (threadIdx.x == 0) first[kKv8SelfSeqs] = total;
    __syncthreads();
    // a range is worth its partials from min_run chunks on, or a sequence of its own
    const int groups = min(w.groups, max(max(1, some), total / w.min_run));
    auto seq_of = [&](int at) {  // the sequence that holds chunk `at` (after empty ones)
        int lo = 0, hi = kKv8SelfSeqs;
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (first[mid] <= at) lo = mid; else hi = mid;
        }
        return lo;
    };
    auto edge = [&](int i) {
        const int at = int((long long)total * i / groups);
        if (!w.snap || i == 0 || i == groups) return at;
        const int s = seq_of(at);
        return first[s] == at ? at : first[s + 1];
    };
    SelfRange r{0, 0, 0};
    if (grp < groups) {
        r.x = edge(grp);
        r.x1 = edge(grp + 1);
        if (r.x < r.x1) r.s = seq_of(r.x);
    }
    if (!w.snap && lead && threadIdx.x == 0) {
        // the tile that starts in this range and goes on past it
        Kv8Merge m{0, 0, 2 * grp + 1, 0};
        if (r.x < r.x1 && r.x1 < total) {
            const int s = seq_of(r.x1 - 1);
            if (first[s] >= r.x && first[s + 1] > r.x1) {
                m.seq = s;
                // the range of the tile's last chunk: the first whose end is past it
                m.parts = 2;
                while (int((long long)total * (grp + m.parts) / groups) < first[s + 1]) ++m.parts;
            }
        }
        w.merges[grp] = m;
    }
    return r;
}

template <typename T, int kFormat, int HD, int NQ, bool kB16, bool kSelf>
__global__ void __launch_bounds__(kWarps * 32, Tile<T, HD, NQ>::CTAS)
kv8_attention_kernel(const Kv8AttnParams p, const Kv8Work w) {
    using F = Frag<HD>;
    using S = Tile<T, HD, NQ>;
    constexpr int NT = terms<T>();
    constexpr int RL = NT == 2 ? 1 : 2;    // rows of a lane per 8 columns
    constexpr int OL = NT == 2 ? 2 : 4;    // sums of a lane per 16 x 8 tile of O^T
    constexpr int SUB = S::SUB;
    constexpr int CHUNK = SUB * kSub;
    extern __shared__ __align__(16) unsigned char smem[];
    uint32_t* sQ = reinterpret_cast<uint32_t*>(smem + S::Q);
    float* sO = reinterpret_cast<float*>(smem);                                // [warp][row][OROW]
    float2* sML = reinterpret_cast<float2*>(sO + kWarps * S::ROWS * S::OROW);  // [warp][row]
    float* sScale = reinterpret_cast<float*>(smem + S::SCALE);
    __shared__ int s_next;

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int g = lane >> 2;
    const int t = lane & 3;
    using R = Ring<HD>;
    unsigned char* ring = smem + warp * 2 * S::BUF;  // [buffer][tile][K, V]
    float* sE = reinterpret_cast<float*>(smem + S::EXPS) + warp * 2 * SUB * 32;  // [buffer][tile][lane]
    pdl_release();
    pdl_wait();  // the work list, the rows and the cache come from the kernels before
    const int H = p.a.num_heads;
    const int total = kSelf ? 0 : w.counters->items * H;
    const int grp = int(blockIdx.x) / H;
    int* first = reinterpret_cast<int*>(smem + S::FIRST);
    SelfRange range{0, 0, 0};
    if constexpr (kSelf) range = self_range(p, w, first, grp, int(blockIdx.x) % H == 0);

    for (;;) {
        Kv8Item item;
        int h;
        if constexpr (kSelf) {
            if (range.x >= range.x1) return;
            while (first[range.s + 1] <= range.x) ++range.s;  // sequences without rows
            const Kv8List l = kv8_list(p, w, kv8_seq(p, w, range.s), 0);
            item.seq = range.s;
            item.row0 = 0;
            item.c0 = range.x - first[range.s];
            item.c1 = min(range.x1 - first[range.s], l.n);
            item.nsink = l.nsink;
            item.lo = l.lo;
            item.slot = item.c1 - item.c0 == l.n ? -1 : 2 * grp + (item.c0 == 0 ? 1 : 0);
            range.x = first[range.s] + item.c1;
            h = int(blockIdx.x) % H;
            __syncthreads();  // the buffers are free
        } else {
            __syncthreads();
            if (threadIdx.x == 0) s_next = atomicAdd(&w.counters->next, 1);
            __syncthreads();
            const int it = s_next;
            if (it >= total) return;
            item = w.items[it / H];
            h = it % H;
        }
        const int q0 = p.cu_seqlens_q[item.seq];
        const int qlen = p.cu_seqlens_q[item.seq + 1] - q0;
        const int first_pos = p.context_lens[item.seq] - qlen;
        const int nrows = min(S::ROWS, qlen * p.group - item.row0);
        const int32_t* table = p.block_tables + int64_t(item.seq) * p.max_blocks;
        const int pos_lo = first_pos + item.row0 / p.group;
        const int pos_hi = first_pos + (item.row0 + nrows - 1) / p.group;

        // ---- where the positions of a chunk live --------------------------------
        // Only positions that some row of the tile sees are looked up: blocks that
        // a window has left behind may be anyone's.
        auto seen = [&](int j) {
            return j <= pos_hi && (p.window <= 0 || j > pos_lo - p.window || j < p.sinks);
        };
        auto block_at = [&](int j, int& slot) -> int {
            int entry;
            kv8_place(p.a, j, entry, slot);
            const int b = table[entry];
            if (b >= 0 && b < p.a.num_blocks) return b;
            raise_status(kStatusBounds);
            return -1;
        };
        struct Where {
            int blk;   // kB16: of the 16 positions; else of position lane % 16. < 0: none
            int in;    // kB16: slot of the first; else of position lane % 16
            int exps;  // a_j of position lane (< 16), b_j of position lane - 16
        };
        int ahead_blk = -1, ahead_in = 0;  // kB16: of the warp's next 32 tiles of 16, one per lane
        auto base_of = [&](int c) { return kv8_chunk(item, c) * CHUNK; };
        auto locate = [&](int c, int n, int u) -> Where {  // tile u of entry c, the warp's n-th
            Where x;
            if constexpr (kB16) {
                // block_size is a multiple of 16: 16 positions lie in one block
                const int at = n * SUB + u;
                if ((at & 31) == 0) {
                    const int cc = c + (lane / SUB) * kWarps;
                    ahead_blk = -1;
                    if (cc < item.c1) {
                        const int j = base_of(cc) + lane % SUB * kSub;
                        if (j <= pos_hi && (p.window <= 0 || j + kSub - 1 > pos_lo - p.window || j < p.sinks)) {
                            ahead_blk = block_at(j, ahead_in);
                        }
                    }
                }
                x.blk = __shfl_sync(0xffffffffu, ahead_blk, at & 31);
                x.in = __shfl_sync(0xffffffffu, ahead_in, at & 31);
            } else {
                const int j = base_of(c) + u * kSub + (lane & 15);
                x.in = 0;
                x.blk = seen(j) ? block_at(j, x.in) : -1;
            }
            x.exps = kKv8MinExp;  // of a row of zeros, so that it raises no maximum
            if (x.blk >= 0) {
                const int8_t* e = lane < 16 ? p.a.k_exps : p.a.v_exps;
                x.exps = e[int64_t(x.blk) * p.a.exp_block_stride + int64_t(h) * p.a.block_size +
                           (kB16 ? x.in + (lane & 15) : x.in)];
            }
            return x;
        };
        // starts the copies of entry c into buffer b; its exponents come back
        struct Exps {
            int e[SUB];
        };
        const int64_t piece = int64_t(h) * HD + lane % R::PIECES * 16;
        const int64_t lane_row = piece + lane / R::PIECES * p.a.row;  // kB16: of the lane's first row
        const int64_t step_row = R::STEP * p.a.row;
        auto issue = [&](int c, int n, int b) -> Exps {
            Exps r;
            const int base = base_of(c);
            const bool all = base >= 0 && base + CHUNK - 1 <= pos_hi &&
                             (p.window <= 0 || base > pos_lo - p.window || base + CHUNK <= p.sinks);
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                const Where x = locate(c, n, u);
                r.e[u] = x.exps;
                const uint32_t dst = smem_addr(ring + b * S::BUF + u * 2 * R::TILE);
                const int64_t tile = int64_t(x.blk) * p.a.block_stride + int64_t(x.in) * p.a.row + lane_row;
#pragma unroll
                for (int i = 0; i < R::COPIES; ++i) {
                    const int row = lane / R::PIECES + i * R::STEP;
                    int64_t at = tile + i * step_row;
                    bool on = x.blk >= 0;
                    if constexpr (kB16) {
                        if (!all) on = on && seen(base + u * kSub + row);
                    } else {
                        const int blk = __shfl_sync(0xffffffffu, x.blk, row);
                        const int in = __shfl_sync(0xffffffffu, x.in, row);
                        on = blk >= 0;
                        at = int64_t(blk) * p.a.block_stride + int64_t(in) * p.a.row + piece;
                    }
                    at = on ? at : 0;
                    const uint32_t to = dst + R::at(row, lane % R::PIECES * 16);
                    kv8_copy16(to, p.a.k_codes + at, on);
                    kv8_copy16(to + R::TILE, p.a.v_codes + at, on);
                }
            }
            return r;
        };
        auto store_exps = [&](const Exps& x, int b) {  // 2^a_j of the 16 positions, then b_j
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                sE[(b * SUB + u) * 32 + lane] = lane < 16 ? exp2_int(min(max(x.e[u], -126), 127)) : float(x.e[u]);
            }
        };
        Exps ahead{};
        {
            const int c = item.c0 + warp;
            Exps first{};
            if (c < item.c1) first = issue(c, 0, 0);
            kv8_copy_commit();
            if (c + kWarps < item.c1) ahead = issue(c + kWarps, 1, 1);
            kv8_copy_commit();
            store_exps(first, 0);
        }

        // ---- Q: each row scaled to [1, 2), its terms stored as MMA fragments ----
        // Dim d of column n is what lane (n, t) of step (i, s) holds, d = KB (t + 4 i)
        // + 4 s + e, as half e of its two words.
        for (int r = warp; r < S::ROWS; r += kWarps) {
            constexpr int PER = HD / 32;
            float x[PER];
            float a = 0.f;
            const bool on = r < nrows;
            const int row = item.row0 + r;
            const T* src = static_cast<const T*>(p.q) + int64_t(q0 + row / p.group) * p.q_stride +
                           int64_t(h * p.group + row % p.group) * HD;
#pragma unroll
            for (int d = 0; d < PER; ++d) {
                x[d] = on ? value_of(src[d * 32 + lane], p.fp16) : 0.f;
                a = fmaxf(a, fabsf(x[d]));
            }
            a = warp_max_xor(a, 32);
            // exponent of the largest element, kept where 2^-e and 2^e are normal
            const int e = min(max(int(__float_as_uint(a) >> 23) - 127, -126), 126);
            const float inv = exp2_int(-e);
            if (lane == 0) sScale[r] = exp2_int(e) * p.qk_scale_log2;
            const int nq = r / (8 / NT), col = r % (8 / NT) * NT;
#pragma unroll
            for (int d = 0; d < PER; ++d) {
                const float v = x[d] * inv;
                const int dim = d * 32 + lane;
                const int piece = dim / F::KB, step = (piece >> 2) * F::KW + (dim % F::KB) / 4;
                __half* dst = reinterpret_cast<__half*>(
                                  sQ + ((nq * F::KSTEPS + step) * 32 + col * 4 + (piece & 3)) * 2) + (dim & 3);
                const __half hi = __float2half_rn(v);
                dst[0] = hi;
                if constexpr (NT == 2) dst[16] = __float2half_rn(v - __half2float(hi));  // the next column
            }
        }
        __syncthreads();
        uint2 qf[S::Q_REGS ? NQ : 1][S::Q_REGS ? F::KSTEPS : 1];
        if constexpr (S::Q_REGS) {
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
                for (int k = 0; k < F::KSTEPS; ++k) {
                    qf[nq][k] = *reinterpret_cast<const uint2*>(sQ + ((nq * F::KSTEPS + k) * 32 + lane) * 2);
                }
        }

        // rows of this lane: scale, position (rows past the tile see what its last
        // one sees, and their zero Q keeps them finite)
        float qs[NQ][RL], m[NQ][RL], l[NQ][RL];
        int pos[NQ][RL];
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
            for (int i = 0; i < RL; ++i) {
                const int r = nq * (8 / NT) + t * RL + i;
                qs[nq][i] = sScale[r];
                pos[nq][i] = first_pos + (item.row0 + min(r, nrows - 1)) / p.group;
                m[nq][i] = -INFINITY;
                l[nq][i] = 0.f;
            }
        float o[NQ][F::MTILES][OL];
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
            for (int k = 0; k < F::MTILES; ++k)
#pragma unroll
                for (int e = 0; e < OL; ++e) o[nq][k][e] = 0.f;

        for (int c = item.c0 + warp, n = 0; c < item.c1; c += kWarps, ++n) {
            const int buf = n & 1;
            kv8_copy_wait<1>();
            store_exps(ahead, buf ^ 1);
            __syncwarp();
            const unsigned char* sK = ring + buf * S::BUF;
            const unsigned char* sV = sK + R::TILE;
            // ---- S^T = K Q^T ----------------------------------------------------
            float s[NQ][SUB][4];
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
                for (int u = 0; u < SUB; ++u)
#pragma unroll
                    for (int k = 0; k < 4; ++k) s[nq][u][k] = 0.f;
#pragma unroll
            for (int q = 0; q < F::KP; ++q) {
                Piece<F::KB> kr[SUB][2];
#pragma unroll
                for (int u = 0; u < SUB; ++u)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        kr[u][i] = read_piece<F::KB>(sK + u * 2 * R::TILE + R::at(g + 8 * i, (t + 4 * q) * F::KB));
                    }
#pragma unroll
                for (int st = 0; st < F::KW; ++st) {
                    const int step = q * F::KW + st;
#pragma unroll
                    for (int u = 0; u < SUB; ++u) {
                        uint32_t a[4];
                        to_half4<kFormat>(kr[u][0].w[st], a[0], a[2]);
                        to_half4<kFormat>(kr[u][1].w[st], a[1], a[3]);
#pragma unroll
                        for (int nq = 0; nq < NQ; ++nq) {
                            const uint2 f = S::Q_REGS ? qf[S::Q_REGS ? nq : 0][S::Q_REGS ? step : 0]
                                                      : *reinterpret_cast<const uint2*>(
                                                            sQ + ((nq * F::KSTEPS + step) * 32 + lane) * 2);
                            mma(s[nq][u], a, f.x, f.y);
                        }
                    }
                }
            }
            // this lane's positions: base + 16 u + g + 8 k
            float ka[SUB][2], vb[SUB][2];
#pragma unroll
            for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    ka[u][k] = sE[(buf * SUB + u) * 32 + g + 8 * k];
                    vb[u][k] = sE[(buf * SUB + u) * 32 + g + 8 * k + 16];
                }

            // ---- softmax ----------------------------------------------------------
            const int base = base_of(c);
            const bool ragged = base + CHUNK - 1 > pos_lo ||
                                (p.window > 0 && base + p.window <= pos_hi && base + CHUNK > p.sinks);
            uint32_t pb[NQ][SUB][2];
            float alpha[NQ][RL];
#pragma unroll
            for (int nq = 0; nq < NQ; ++nq) {
                float pw[SUB][2][2];  // [tile][position][column]
#pragma unroll
                for (int i = 0; i < RL; ++i) {
                    float x[SUB][2], top = -INFINITY;
#pragma unroll
                    for (int u = 0; u < SUB; ++u)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const float d = NT == 2 ? s[nq][u][2 * k] + s[nq][u][2 * k + 1] : s[nq][u][2 * k + i];
                            // the factors first: a code sum times 2^a alone may leave fp32's
                            // range (large keys, small queries). Rounded before m is taken off.
                            x[u][k] = __fmul_rn(d, ka[u][k] * qs[nq][i]);
                            if (ragged) {
                                const int j = base + u * kSub + g + 8 * k;
                                const bool see = j <= pos[nq][i] &&
                                                 (p.window <= 0 || j > pos[nq][i] - p.window || j < p.sinks);
                                if (!see) x[u][k] = -INFINITY;
                            }
                            top = fmaxf(top, x[u][k] + vb[u][k]);
                        }
#pragma unroll
                    for (int q = 4; q < 32; q <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, q));
                    const float mn = top > m[nq][i] + kMargin ? top : m[nq][i];
                    const float mu = mn == -INFINITY ? 0.f : mn;  // nothing seen yet
                    const float root = ex2(0.5f * (m[nq][i] - mu));
                    alpha[nq][i] = root * root;
                    m[nq][i] = mn;
                    float sum = 0.f;
#pragma unroll
                    for (int u = 0; u < SUB; ++u)
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const float y = x[u][k] - mu;
                            sum = fmaf(ex2(y + kUpBy), 0x1p-20f, sum);
                            pw[u][k][i] = ex2(y + vb[u][k]);
                        }
                    l[nq][i] = fmaf(l[nq][i] * root, root, sum);
                }
#pragma unroll
                for (int u = 0; u < SUB; ++u)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        if constexpr (NT == 2) {
                            const float hi = __half2float(__float2half_rn(pw[u][k][0]));
                            pw[u][k][1] = pw[u][k][0] - hi;
                            pw[u][k][0] = hi;
                        }
                        pb[nq][u][k] = transpose8(pack_half(pw[u][k][0], pw[u][k][1]));
                    }
            }

            // ---- O^T += V^T P^T -----------------------------------------------------
            // fp32 rows: the products of a chunk are added in fp32 registers, since
            // the tensor core's own accumulation truncates and a long context would
            // add that up. Others accumulate in place.
            if constexpr (NT == 1) {
                bool grew = false;
#pragma unroll
                for (int nq = 0; nq < NQ; ++nq) grew |= alpha[nq][0] != 1.f || alpha[nq][1] != 1.f;
                if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                    for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
                        for (int k = 0; k < F::MTILES; ++k)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[nq][k][e] *= alpha[nq][e & 1];
                }
            }
#pragma unroll
            for (int q = 0; q < F::VP; ++q) {
                Piece<F::VB> vr[SUB][4];
#pragma unroll
                for (int u = 0; u < SUB; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        vr[u][i] = read_piece<F::VB>(sV + u * 2 * R::TILE +
                                                     R::at(2 * t + (i & 1) + 8 * (i >> 1), (g + 8 * q) * F::VB));
                    }
#pragma unroll
                for (int st = 0; st < F::VW; ++st) {
                    float d[NQ][2][4];  // fp32 rows: this chunk's products
                    if constexpr (NT == 2) {
#pragma unroll
                        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
                            for (int j = 0; j < 2; ++j)
#pragma unroll
                                for (int e = 0; e < 4; ++e) d[nq][j][e] = 0.f;
                    }
#pragma unroll
                    for (int u = 0; u < SUB; ++u) {
                        uint32_t a[2][4];  // of the 2 tiles of this word
                        const uint32_t x0 = vr[u][0].w[st], x1 = vr[u][1].w[st];
                        const uint32_t y0 = vr[u][2].w[st], y1 = vr[u][3].w[st];
                        to_half4<kFormat>(__byte_perm(x0, x1, 0x5140), a[0][0], a[0][1]);
                        to_half4<kFormat>(__byte_perm(x0, x1, 0x7362), a[1][0], a[1][1]);
                        to_half4<kFormat>(__byte_perm(y0, y1, 0x5140), a[0][2], a[0][3]);
                        to_half4<kFormat>(__byte_perm(y0, y1, 0x7362), a[1][2], a[1][3]);
#pragma unroll
                        for (int j = 0; j < 2; ++j)
#pragma unroll
                            for (int nq = 0; nq < NQ; ++nq) {
                                float* sum = NT == 2 ? d[nq][j] : o[nq][(q * F::VW + st) * 2 + j];
                                mma(sum, a[j], pb[nq][u][0], pb[nq][u][1]);
                            }
                    }
                    if constexpr (NT == 2) {
#pragma unroll
                        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                float* sum = o[nq][(q * F::VW + st) * 2 + j];
                                sum[0] = fmaf(sum[0], alpha[nq][0], d[nq][j][0] + d[nq][j][1]);
                                sum[1] = fmaf(sum[1], alpha[nq][0], d[nq][j][2] + d[nq][j][3]);
                            }
                    }
                }
            }
            __syncwarp();  // the buffer is free
            if (c + 2 * kWarps < item.c1) ahead = issue(c + 2 * kWarps, n + 2, buf);
            kv8_copy_commit();
        }

        // ---- join the warps ---------------------------------------------------------
        kv8_copy_wait<0>();
        __syncthreads();  // the buffers are read no more
        // Lane (g, t) holds dims VB g + 8 VB q + 2 k + e (tile (q, k), half e) of its rows
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
            for (int i = 0; i < RL; ++i) {
                float sum = l[nq][i];
#pragma unroll
                for (int q = 4; q < 32; q <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, q);
                const int r = nq * (8 / NT) + t * RL + i;
                if (g == 0) sML[warp * S::ROWS + r] = make_float2(m[nq][i], sum);
                float* dst = sO + (warp * S::ROWS + r) * S::OROW;
#pragma unroll
                for (int q = 0; q < F::VP; ++q)
#pragma unroll
                    for (int j = 0; j < F::VB; j += 4) {
                        const int k = (q * F::VB + j) / 2;
                        *reinterpret_cast<float4*>(dst + F::VB * g + 8 * F::VB * q + j) =
                            NT == 2 ? make_float4(o[nq][k][0], o[nq][k][1], o[nq][k + 1][0], o[nq][k + 1][1])
                                    : make_float4(o[nq][k][i], o[nq][k][OL / 2 + i], o[nq][k + 1][i],
                                                  o[nq][k + 1][OL / 2 + i]);
                    }
            }
        __syncthreads();
        for (int r = warp; r < nrows; r += kWarps) {
            float2 ml[kWarps];
            float M = -INFINITY;
#pragma unroll
            for (int k = 0; k < kWarps; ++k) {
                ml[k] = sML[k * S::ROWS + r];
                M = fmaxf(M, ml[k].x);
            }
            const float mu = M == -INFINITY ? 0.f : M;
            float L = 0.f, f[kWarps];
#pragma unroll
            for (int k = 0; k < kWarps; ++k) {
                const float root = ex2(0.5f * (ml[k].x - mu));
                f[k] = root * root;
                L = fmaf(ml[k].y * root, root, L);
            }
            const int row = item.row0 + r;
            const int64_t slot = (int64_t(item.slot) * H + h) * S::ROWS + r;
            const bool whole = item.slot < 0;
            const float inv = whole ? 1.0f / L : 1.0f;
            T* dst = static_cast<T*>(p.out) + int64_t(q0 + row / p.group) * p.out_stride +
                     int64_t(h * p.group + row % p.group) * HD;
#pragma unroll
            for (int d = lane; d < HD; d += 32) {
                float v = 0.f;
#pragma unroll
                for (int k = 0; k < kWarps; ++k) v = fmaf(sO[(k * S::ROWS + r) * S::OROW + d], f[k], v);
                if (whole) {
                    put_value(dst + d, v * inv, p.fp16);
                } else {
                    w.acc[slot * HD + d] = v;
                }
            }
            if (!whole && lane == 0) w.ml[slot] = make_float2(M, L);
        }
    }
}

template <typename T, int kFormat, int HD, int NQ, bool kB16, bool kSelf>
cudaError_t launch_kernel(const Kv8AttnParams& p, const Kv8Work& w, cudaStream_t st) {
    auto* k = kv8_attention_kernel<T, kFormat, HD, NQ, kB16, kSelf>;
    using S = Tile<T, HD, NQ>;
    static bool ready[64] = {false};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!ready[dev]) {
        e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, int(S::SMEM));
        if (e != cudaSuccess) return e;
        ready[dev] = true;
    }
    const int grid = kSelf ? w.groups * p.a.num_heads : kKv8Sms * S::CTAS;
    return launch_programmatic(k, dim3(unsigned(grid)), dim3(kWarps * 32), S::SMEM, st, p, w);
}

template <typename T, int kFormat, int HD, int NQ>
cudaError_t launch_blocks(const Kv8AttnParams& p, const Kv8Work& w, cudaStream_t st) {
    const bool b16 = p.a.block_size % kSub == 0;
    if (w.groups > 0) {
        return b16 ? launch_kernel<T, kFormat, HD, NQ, true, true>(p, w, st)
                   : launch_kernel<T, kFormat, HD, NQ, false, true>(p, w, st);
    }
    // several tiles per sequence: the largest ones, of what the tensor-memory kernel
    // does not take
    if constexpr ((NQ == 4 && (HD == 32 || sizeof(T) == 4)) || (NQ == 2 && HD == 256)) {
        return b16 ? launch_kernel<T, kFormat, HD, NQ, true, false>(p, w, st)
                   : launch_kernel<T, kFormat, HD, NQ, false, false>(p, w, st);
    }
    return cudaErrorInvalidValue;
}

template <typename T, int kFormat, int HD>
cudaError_t launch_tile(const Kv8AttnParams& p, const Kv8Work& w, cudaStream_t st) {
    switch (w.tile_rows * terms<T>() / 8) {
        case 1: return launch_blocks<T, kFormat, HD, 1>(p, w, st);
        case 2: return launch_blocks<T, kFormat, HD, 2>(p, w, st);
        case 4:
            if constexpr (HD <= 128) return launch_blocks<T, kFormat, HD, 4>(p, w, st);
            break;
    }
    return cudaErrorInvalidValue;
}

}  // namespace

template <int HD>
cudaError_t launch_kv8_rows(const Kv8AttnParams& p, const Kv8Work& w, bool fp32, int32_t format,
                            cudaStream_t st) {
    if (fp32) {
        return format == NVLLM_KV8_E4M3 ? launch_tile<float, NVLLM_KV8_E4M3, HD>(p, w, st)
                                        : launch_tile<float, NVLLM_KV8_INT8, HD>(p, w, st);
    }
    return format == NVLLM_KV8_E4M3 ? launch_tile<uint16_t, NVLLM_KV8_E4M3, HD>(p, w, st)
                                    : launch_tile<uint16_t, NVLLM_KV8_INT8, HD>(p, w, st);
}

}  // namespace nvllm
