// Attention over the 8-bit paged cache for many rows per KV head (prompts and
// chunks), on tcgen05 with accumulators in tensor memory; bf16 and fp16 rows,
// head_dim 64 and 128, any block size.
//
// A tile is 256 packed rows (kv8.cuh) of one sequence and KV head, two halves of
// 128; keys come in tiles of 64. With q' = q scaled by a power of two to [1, 2)
// per row, codes c_j, d_j and exponents a_j, b_j of K and V, and A the largest a_j
// of a key tile (U = 7 for E4M3, 5 for INT8):
//   K'_j = c_j 2^(a_j - A + U)                 in fp16
//   S = q' . K'_j,  x_j = S 2^(A - U) qs       log2-domain score
//   m = running max of x_j,  P_j = 2^(x_j - m - 16)   in bf16
//   acc += sum_j P_j V_j,  l += sum_j P_j,  o = acc / l     V_j = d_j 2^(b_j) in bf16
// The exponents cost nothing per score: they are folded into the operands while
// codes become 16-bit floats, K's against the tile's largest, which is one more
// factor of the row's scale. V is exact in bf16 whatever its exponent; K' in fp16
// is exact for rows within 2^22 of the tile's largest (2^29 for INT8) and beyond
// that off by 2^-36 of the largest: a factor below fp16's range is taken in two
// steps, of which only the last rounds. P is rounded to bf16, half a step of which is
// the output's own (outputs are 2.4e-3 of their norm from 64 bits, 1.7e-3 with P in
// fp32); for fp16 rows, whose step is finer, P is two bf16 terms.
//
// One CTA per SM, 20 warps in 5 warpgroups:
//   warps 0-3, 4-7  softmax of the tile's first and second 128 rows: a thread owns
//                   a row and its TMEM lane. Reads S, masks ragged tiles, P goes
//                   back over S as the next product's A operand; O is rescaled
//                   only when m moves by more than kMargin (rarely).
//   warps 8-15      converters: 16-byte pieces of codes to 16-bit floats, into a ring
//                   of three stages in the MMA's 128-byte swizzle.
//   warps 16, 17    MMAs of the first and second half, one lane each: O(n) += P(n)
//                   V(n), then S(n+2) in P's place, while the softmax works on
//                   S(n+1).
//   warps 18, 19    loaders of K and of V: block ids, codes by asynchronous copies
//                   into a ring of three tiles, and the rows' factors from their
//                   exponents; rows that no query of the tile sees are 0.
// The last three warpgroups give registers to the softmax.
// TMEM (512 columns): S of half i, buffer b at 128 i + 64 b, O of half i at 256 +
// 128 i.
//
// A key tile costs at least 1024 cycles of the special function units (64 x 256
// exponentials) and, at head_dim 128, as many of the tensor cores. It takes about
// 2400: MMAs on different accumulators have no order of their own, so the S that
// takes P's place waits until O is complete, and an S of N = 64 is paced by Q's
// re-reads from shared memory (66 cycles in place of 32).
// Measured on B200: 4096 rows at position 16384, 32 heads over 8 x 128, bf16: 1.21
// ms, 797 TFLOP/s; 8191 rows, window 1000, 16 heads over 4 x 64: 128 us. On the way:
// one MMA warp for both halves 1.57 ms (its own instructions paced it), four
// converter warps that also loaded 1.55, factors written a tile late 1.44, no tile
// of the last round cut 1.30. A step of 128 keys with one S per half was slower, 1.69
// against 1.44: S is then exposed behind the softmax.
//
// Every wait is bounded; on a timeout the CTA lets its MMAs finish, reports
// NVLLM_ERR_TIMEOUT with the wait's record and frees its TMEM.
#include <algorithm>
#include <type_traits>

#include "kv8.cuh"
#include "tcgen05.cuh"

namespace nvllm {

namespace {

constexpr int kHalf = 128;           // rows of a half (TMEM lanes)
constexpr int kRows = 2 * kHalf;     // rows of a tile
constexpr int kKeys = 64;            // keys of a key tile
constexpr int kStages = 3;
constexpr int kTops = 16;            // more tiles than K's loader can be ahead of the softmax (8)
constexpr int kRaw = 3;              // key tiles of codes on their way or landed
constexpr int kConvWarp0 = 8;
constexpr int kConvWarps = 8;
constexpr int kMmaWarp = 16;
constexpr int kLoadWarp = 18;  // K's loader, then V's
constexpr int kThreads = 640;
constexpr int kItemReaders = kThreads / 32 - 1;  // every warp but K's loader
// Registers a thread: 96 at launch (65536 / 640). The converters' two warpgroups
// fall to 64 and the last to 64, the two softmax warpgroups rise to 144:
// 2 x 144 + 2 x 64 + 64 = 5 x 96.
constexpr int kLaunchRegs = 96;
constexpr int kSoftmaxRegs = 144;
constexpr int kConvRegs = 64;
constexpr int kMmaRegs = 64;
static_assert(2 * kSoftmaxRegs + 2 * kConvRegs + kMmaRegs <= 5 * kLaunchRegs, "register split");
constexpr uint32_t kTmemCols = 512;
constexpr float kMargin = 8.0f;
// Weights are taken this much lower (log2; it cancels in acc / l): a weight can reach
// 2^kMargin, a value 2^127.8, and their sums have to stay within fp32. bf16 has the
// range, and 2^-16 of the smallest value, 2^-109, is a normal number still.
constexpr float kDownBy = 16.0f;
// Scores go through one multiply-add, whose exact product can exceed the rounded m by
// 2^-24 of it: 4 at this size, and infinity as a weight from 2^31 on. Beyond it
// (rows whose m is, which models' are not) scores are rounded first.
constexpr float kFarScore = 67108864.0f;  // 2^26

template <int kFormat>
constexpr int kUp = kFormat == NVLLM_KV8_E4M3 ? 7 : 5;

// Instruction descriptors for kind::f16 with fp32 accumulation: fp16 or bf16 A and B.
constexpr uint32_t idesc(int M, int N, bool bf16, bool b_mn) {
    return (1u << 4)                   // D format: f32
           | (uint32_t(bf16) << 7)     // A format
           | (uint32_t(bf16) << 10)    // B format
           | (uint32_t(b_mn) << 16)    // B major
           | (uint32_t(N >> 3) << 17)  // N / 8
           | (uint32_t(M >> 4) << 24); // M / 16
}

struct Control {
    uint64_t raw_full[2][kRaw]; // [K, V]: codes landed (32 arrivals) and factors written
    uint64_t raw_free[2][kRaw]; // and read (one arrival per converter warp)
    uint64_t kc_full[kStages];  // K' of a stage written (one arrival per converter warp)
    uint64_t vc_full[kStages];  // V of a stage written
    uint64_t k_free[kStages];   // S of the stage's key tile complete (both halves)
    uint64_t v_free[kStages];   // O of it complete (both halves)
    uint64_t top_full[kTops];   // top written
    uint64_t s_full[2][2];      // [half][buffer]: S complete
    uint64_t p_full[2][2];      // P written, O rescaled if need be (one arrival per warp)
    uint64_t o_full[2][2];      // O of that key tile complete
    uint64_t drain[2];
    uint64_t item_full[2];      // two-slot queue of work items
    uint64_t item_free[2];
    uint64_t q_full[2];         // Q of a half written, items with rows in the half counted
    int32_t top[kTops];         // A of a key tile
    int32_t small[kRaw];        // some K factor of a key tile is below fp16's range
    int32_t large[kRaw];        // some V exponent of a key tile is above 7
    uint32_t tmem_base;
    int32_t items[2];
    uint32_t abort;             // address of the barrier whose wait gave up first, or 0
};

template <int HD>
struct Shape {
    static constexpr uint32_t ATOM = kKeys * 128;           // 64 keys x 64 dims of K' or V'
    static constexpr uint32_t TILE = ATOM * (HD / 64);
    static constexpr uint32_t Q_ATOM = kHalf * 128;         // 128 rows x 64 dims
    static constexpr uint32_t Q_HALF = Q_ATOM * (HD / 64);
    static constexpr uint32_t OFF_Q = 0;
    static constexpr uint32_t OFF_K = 2 * Q_HALF;
    static constexpr uint32_t OFF_V = OFF_K + kStages * TILE;
    static constexpr uint32_t RAW = kKeys * HD;             // codes of a key tile of K or V
    static constexpr uint32_t OFF_RAW = OFF_V + kStages * TILE;
    static constexpr uint32_t OFF_FACTOR = OFF_RAW + 2 * kRaw * RAW;
    static constexpr uint32_t OFF_CTL = OFF_FACTOR + 2 * kRaw * kKeys * 8;
    static constexpr uint32_t SMEM = OFF_CTL + 1024 + 1024;  // + control block + alignment slack
    static_assert(SMEM <= 227u * 1024u, "shared memory");
    static_assert(sizeof(Control) <= 1024, "control block");
    static constexpr int PIECES = HD / 16;                     // 16-code pieces of a row
    static constexpr int STEP = kConvWarps * 32 / PIECES;      // rows converted at once
    static constexpr int COPIES = kKeys / STEP;                // pieces per thread and tensor
    static constexpr int LOAD_STEP = 32 / PIECES;              // rows that a loader copies at once
};

__device__ __forceinline__ bool wait_or_abort(uint64_t* bar, uint32_t parity, Control* ctl) {
    return mbar_wait_or_abort(bar, parity, &ctl->abort);
}

__device__ __forceinline__ float ex2_ftz(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The lowest n of 64 bits (none below 0, all from 64 on).
__device__ __forceinline__ uint64_t below(int n) {
    return n <= 0 ? 0 : n >= 64 ? ~uint64_t(0) : (uint64_t(1) << n) - 1;
}

// Two floats by one instruction, and the largest of three.
__device__ __forceinline__ uint64_t pair(float2 a) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y));
    return r;
}
__device__ __forceinline__ float2 unpair(uint64_t a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pair(a)), "l"(pair(b)), "l"(pair(c)));
    return unpair(r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair(a)), "l"(pair(b)));
    return unpair(r);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

__device__ __forceinline__ uint32_t pack_half(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// What pack_bf16 left of a and b, as bf16.
__device__ __forceinline__ uint32_t pack_rest(float a, float b, uint32_t h) {
    const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&h));
    return pack_bf16(a - f.x, b - f.y);
}

// 2^e as an fp16 pair, e <= 15 (below 2^-24, the smallest fp16: 0).
constexpr int kHalfMinExp = -24;
// Any code times 2^-15 is an exact fp16: a multiple of 2^-24.
constexpr int kCodeShift = 15;
__device__ __forceinline__ __half2 half_power(int e) {
    return __float2half2_rn(exp2_int(max(e, -30)));
}

// Four codes times f (a power of two) -> two fp16 pairs, in order.
template <int kFormat>
__device__ __forceinline__ void scaled_half4(uint32_t w, __half2 f, uint32_t& a, uint32_t& b) {
    __half2 x, y;
    if constexpr (kFormat == NVLLM_KV8_E4M3) {
        uint32_t lo, hi;
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\t"
            "cvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
        x = __hmul2(*reinterpret_cast<__half2*>(&lo), f);
        y = __hmul2(*reinterpret_cast<__half2*>(&hi), f);
    } else {
        // (1024 + u) - 1152 = code for u = code + 128: exact, then the factor
        const uint32_t u = w ^ 0x80808080u;
        const __half2 c = __half2half2(__ushort_as_half(0x6480));
        uint32_t lo = __byte_perm(u, 0x64646464u, 0x4140), hi = __byte_perm(u, 0x64646464u, 0x4342);
        x = __hmul2(__hsub2(*reinterpret_cast<__half2*>(&lo), c), f);
        y = __hmul2(__hsub2(*reinterpret_cast<__half2*>(&hi), c), f);
    }
    a = *reinterpret_cast<const uint32_t*>(&x);
    b = *reinterpret_cast<const uint32_t*>(&y);
}

// Four codes times 2^e -> the bf16 pairs (0, 2) and (1, 3): bytes that are two
// apart land in a word's halves without a byte shuffle, and the epilogue knows.
// E4M3: sign, exponent and mantissa bits moved into a bf16 are code * 2^-120 (its
// subnormals too), so f = 2^(e + 120). INT8: 128 + the low seven bits as a bf16,
// less 128, or 256 where the sign bit is set; f = 2^e.
template <int kFormat>
__device__ __forceinline__ void scaled_bf16x4(uint32_t w, __nv_bfloat162 f, uint32_t& even, uint32_t& odd) {
    __nv_bfloat162 x, y;
    if constexpr (kFormat == NVLLM_KV8_E4M3) {
        uint32_t lo = ((w & 0x007F007Fu) << 4) | ((w & 0x00800080u) << 8);
        uint32_t hi = ((w & 0x7F007F00u) >> 4) | (w & 0x80008000u);
        x = *reinterpret_cast<__nv_bfloat162*>(&lo);
        y = *reinterpret_cast<__nv_bfloat162*>(&hi);
    } else {
        const uint32_t v = w >> 8;
        uint32_t a = (w & 0x007F007Fu) | 0x43004300u, b = (w & 0x00800080u) | 0xC300C300u;
        uint32_t c = (v & 0x007F007Fu) | 0x43004300u, d = (v & 0x00800080u) | 0xC300C300u;
        x = __hadd2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
        y = __hadd2(*reinterpret_cast<__nv_bfloat162*>(&c), *reinterpret_cast<__nv_bfloat162*>(&d));
    }
    x = __hmul2(x, f);
    y = __hmul2(y, f);
    even = *reinterpret_cast<const uint32_t*>(&x);
    odd = *reinterpret_cast<const uint32_t*>(&y);
}

template <typename T, int kFormat, int HD>
__global__ void __launch_bounds__(kThreads, 1)
kv8_attention_tc_kernel(const Kv8AttnParams p, const Kv8Work w) {
    using S = Shape<HD>;
    constexpr int U = kUp<kFormat>;
    constexpr int NP = std::is_same_v<T, __half> ? 2 : 1;  // terms of P
    constexpr uint32_t kIdescS = idesc(kHalf, kKeys, false, false);
    constexpr uint32_t kIdescO = idesc(kHalf, HD, true, true);
    extern __shared__ unsigned char smem_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* sQ = base + S::OFF_Q;
    unsigned char* sK = base + S::OFF_K;
    unsigned char* sV = base + S::OFF_V;
    unsigned char* sRaw = base + S::OFF_RAW;  // [K, V][slot][row][HD]
    uint32_t* sFactor = reinterpret_cast<uint32_t*>(base + S::OFF_FACTOR);  // [K, V][slot][row][2]
    Control* ctl = reinterpret_cast<Control*>(base + S::OFF_CTL);
    const int tid = threadIdx.x;
    const int warp = tid >> 5;
    const int lane = tid & 31;

    if (tid == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&ctl->kc_full[i], kConvWarps);
            mbar_init(&ctl->vc_full[i], kConvWarps);
            mbar_init(&ctl->k_free[i], 2);
            mbar_init(&ctl->v_free[i], 2);
        }
        for (int i = 0; i < 2 * kRaw; ++i) {
            mbar_init(&ctl->raw_full[0][i], 33);
            mbar_init(&ctl->raw_free[0][i], kConvWarps);
        }
        for (int i = 0; i < kTops; ++i) mbar_init(&ctl->top_full[i], 1);
        for (int i = 0; i < 2; ++i) {
            for (int b = 0; b < 2; ++b) {
                mbar_init(&ctl->s_full[i][b], 1);
                mbar_init(&ctl->p_full[i][b], kHalf / 32);
                mbar_init(&ctl->o_full[i][b], 1);
            }
            mbar_init(&ctl->item_full[i], 1);
            mbar_init(&ctl->drain[i], 1);
            mbar_init(&ctl->q_full[i], kHalf / 32);
            mbar_init(&ctl->item_free[i], kItemReaders);
        }
        ctl->abort = 0;
    }
    fence_barrier_init();
    if (warp == kMmaWarp) {
        tc::tmem_alloc(&ctl->tmem_base, kTmemCols);
        tc::tmem_relinquish();
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = ctl->tmem_base;
    pdl_release();
    pdl_wait();  // the work list, the rows and the cache come from the kernels before

    const int H = p.a.num_heads;
    const int total = w.counters->items * H;
    uint32_t seq = 0;          // key tiles of this CTA so far, and of the first half
    uint32_t seq1 = 0;         // and of the second half
    bool issued_mma = false;   // MMA warp

    auto wait_all = [&](uint64_t* bar, uint32_t parity) -> bool {
        return __all_sync(0xffffffffu, wait_or_abort(bar, parity, ctl));
    };
    // One arrival for the warp, after all its lanes' writes (each fenced by its lane).
    auto warp_arrive = [&](uint64_t* bar) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar);
    };
    // Work items: K's loader takes each from the global cursor and
    // publishes it in queue slot j % 2; every other warp reads the items in order
    // and frees the slot. -1 ends the loop. No role waits for the others at an
    // item's end.
    auto publish = [&](uint32_t j, int it) -> bool {
        const uint32_t slot = j & 1u;
        if (j >= 2 && !wait_or_abort(&ctl->item_free[slot], ((j >> 1) - 1) & 1u, ctl)) return false;
        ctl->items[slot] = it;
        mbar_arrive(&ctl->item_full[slot]);
        return true;
    };
    auto take = [&](uint32_t j) -> int {
        const uint32_t slot = j & 1u;
        if (!wait_all(&ctl->item_full[slot], (j >> 1) & 1u)) return -1;
        const int it = *reinterpret_cast<volatile int32_t*>(&ctl->items[slot]);
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->item_free[slot]);
        return it;
    };

    auto next_item = [&](uint32_t j) -> int {
        int it = -1;
        if (warp == kLoadWarp) {
            if (lane == 0) {
                if (!*reinterpret_cast<volatile uint32_t*>(&ctl->abort)) {
                    it = atomicAdd(&w.counters->next, 1);
                    if (it >= total) it = -1;
                }
                if (!publish(j, it)) it = -1;
            }
            it = __shfl_sync(0xffffffffu, it, 0);
        } else {
            it = take(j);
        }
        return *reinterpret_cast<volatile uint32_t*>(&ctl->abort) ? -1 : it;
    };
    struct Job {
        Kv8Item item;
        int h, q0, first_pos, nrows, ntiles, halves, pos_lo, pos_hi;
    };
    auto job_of = [&](int it) -> Job {
        Job x;
        x.item = w.items[it / H];
        x.h = it % H;
        x.q0 = p.cu_seqlens_q[x.item.seq];
        const int qlen = p.cu_seqlens_q[x.item.seq + 1] - x.q0;
        x.first_pos = p.context_lens[x.item.seq] - qlen;
        x.nrows = min(kRows, qlen * p.group - x.item.row0);
        x.ntiles = x.item.c1 - x.item.c0;
        x.halves = x.nrows > kHalf ? 2 : 1;
        x.pos_lo = x.first_pos + x.item.row0 / p.group;
        x.pos_hi = x.first_pos + (x.item.row0 + x.nrows - 1) / p.group;
        return x;
    };
    auto done = [&](const Job& x) {
        seq += x.ntiles;
        if (x.halves == 2) seq1 += x.ntiles;
    };

    if (warp < kConvWarp0) {
        // ---------------------------------------------------------------- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        for (uint32_t j = 0;; ++j) {
            const int it = next_item(j);
            if (it < 0) break;
            const Job job = job_of(it);
            const Kv8Item& item = job.item;
            const int h = job.h, q0 = job.q0, first_pos = job.first_pos, nrows = job.nrows;
            const int ntiles = job.ntiles, halves = job.halves, pos_lo = job.pos_lo, pos_hi = job.pos_hi;
            const uint32_t n0 = seq;
            const int half = warp >> 2;
            const uint32_t hn0 = half ? seq1 : seq;
            const int r = tid - half * kHalf;              // row of the half, TMEM lane
            const int row = item.row0 + half * kHalf + r;  // packed row
            const bool live = half * kHalf + r < nrows;
            const uint32_t lane_off = uint32_t((warp & 3) * 32) << 16;
            const uint32_t tO = tmem + 256u + 128u * half + lane_off;
            float qs = 0.f;
            if (half < halves) {
                // Q's row as fp16, scaled to [1, 2); this half's earlier S all completed
                constexpr int N = HD / 8;  // 16-byte pieces of the row
                uint4 raw[N];
                const uint4* src = reinterpret_cast<const uint4*>(
                    static_cast<const T*>(p.q) + int64_t(q0 + row / p.group) * p.q_stride +
                    int64_t(h * p.group + row % p.group) * HD);
                float a = 0.f;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    raw[i] = make_uint4(0, 0, 0, 0);
                    if (live) raw[i] = src[i];
                    const T* v = reinterpret_cast<const T*>(&raw[i]);
#pragma unroll
                    for (int k = 0; k < 8; ++k) a = fmaxf(a, fabsf(to_float(v[k])));
                }
                const int e = min(max(int(__float_as_uint(a) >> 23) - 127, -126), 126);
                const float inv = exp2_int(-e);
                qs = exp2_int(e) * p.qk_scale_log2;
                unsigned char* dst = sQ + half * S::Q_HALF + r * 128;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const T* v = reinterpret_cast<const T*>(&raw[i]);
                    uint4 o;
                    o.x = pack_half(to_float(v[0]) * inv, to_float(v[1]) * inv);
                    o.y = pack_half(to_float(v[2]) * inv, to_float(v[3]) * inv);
                    o.z = pack_half(to_float(v[4]) * inv, to_float(v[5]) * inv);
                    o.w = pack_half(to_float(v[6]) * inv, to_float(v[7]) * inv);
                    *reinterpret_cast<uint4*>(dst + (i >> 3) * S::Q_ATOM + ((i & 7) ^ (r & 7)) * 16) = o;
                }
                tc::fence_async_smem();
                warp_arrive(&ctl->q_full[half]);
            }
            const int pos = first_pos + (item.row0 + min(half * kHalf + r, nrows - 1)) / p.group;
            float m = -INFINITY, l = 0.f;
            bool ok = true;
            for (int t = 0; half < halves && t < ntiles; ++t) {
                const uint32_t n = n0 + t;
                const uint32_t hn = hn0 + t;
                const uint32_t b = hn & 1u;
                if (!wait_all(&ctl->top_full[n % kTops], (n / kTops) & 1u) ||
                    !wait_all(&ctl->s_full[half][b], (hn >> 1) & 1u)) {
                    ok = false;
                    break;
                }
                const int A = *reinterpret_cast<const volatile int32_t*>(&ctl->top[n % kTops]);
                tc::fence_after_sync();
                const uint32_t tS = tmem + 128u * half + 64u * b + lane_off;
                float sc[kKeys];
                tc::tmem_ld32(tS, sc);
                tc::tmem_ld32(tS + 32u, sc + 32);
                tc::tmem_ld_wait();
                const int kbase = kv8_chunk(item, item.c0 + t) * kKeys;
                if (kbase + kKeys - 1 > pos_lo ||
                    (p.window > 0 && kbase + p.window <= pos_hi && kbase + kKeys > p.sinks)) {
                    // the tile's keys that the row sees, a bit each: up to its own, and from
                    // the window's start or before the sinks' end
                    uint64_t see = below(pos + 1 - kbase);
                    if (p.window > 0) see &= ~below(pos + 1 - p.window - kbase) | below(p.sinks - kbase);
                    const uint32_t see_lo = uint32_t(see), see_hi = uint32_t(see >> 32);
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        sc[k] = see_lo & (1u << k) ? sc[k] : -INFINITY;
                        sc[32 + k] = see_hi & (1u << k) ? sc[32 + k] : -INFINITY;
                    }
                }
                // a factor above 0 keeps -inf what it is for rows of zeros
                float f = fmaxf(qs * exp2_int(min(max(A - U, -126), 127)), 1.2e-38f);
                float mx[4] = {sc[0], sc[1], sc[2], sc[3]};
#pragma unroll
                for (int k = 4; k < kKeys; k += 8) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        mx[q] = k + 4 + q < kKeys ? max3(mx[q], sc[k + q], sc[k + 4 + q]) : fmaxf(mx[q], sc[k + q]);
                    }
                }
                const float top = max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]) * f;
                const float mn = top > m + kMargin ? top : m;
                const float mu = mn == -INFINITY ? 0.f : mn;  // nothing seen yet
                const float alpha = ex2_ftz(m - mu);
                m = mn;
                const bool far = fabsf(mu) > kFarScore;
                if (__any_sync(0xffffffffu, alpha != 1.0f || far)) {  // one vote: it is on every tile's path
                    if (__any_sync(0xffffffffu, far)) {
                        // (of these rows alone: the others keep their bits)
                        const float g = far ? f : 1.0f;
#pragma unroll
                        for (int k = 0; k < kKeys; ++k) sc[k] = __fmul_rn(sc[k], g);
                        f = far ? 1.0f : f;
                    }
                    if (t > 0) {
                        // O must hold the previous tile's products before it is rescaled
                        if (!wait_all(&ctl->o_full[half][b ^ 1u], ((hn - 1) >> 1) & 1u)) {
                            ok = false;
                            break;
                        }
                        tc::fence_after_sync();
#pragma unroll 1
                        for (int c = 0; c < HD / 32; ++c) {
                            float ov[32];
                            tc::tmem_ld32(tO + c * 32u, ov);
                            tc::tmem_ld_wait();
#pragma unroll
                            for (int k = 0; k < 32; ++k) ov[k] *= alpha;
                            tc::tmem_st32(tO + c * 32u, ov);
                        }
                    }
                }
                float2 ls[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                const float2 f2 = make_float2(f, f), mu2 = make_float2(-mu - kDownBy, -mu - kDownBy);
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    uint32_t pk[16], rest[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        float2 x = fma2(make_float2(sc[32 * q + 2 * k], sc[32 * q + 2 * k + 1]), f2, mu2);
                        x = make_float2(ex2_ftz(x.x), ex2_ftz(x.y));
                        ls[k & 1] = add2(ls[k & 1], x);
                        pk[k] = pack_bf16(x.x, x.y);
                        if constexpr (NP == 2) rest[k] = pack_rest(x.x, x.y, pk[k]);
                    }
                    tc::tmem_st16(tS + 16u * q, pk);
                    if constexpr (NP == 2) tc::tmem_st16(tS + 32u + 16u * q, rest);
                }
                l = fmaf(l, alpha, (ls[0].x + ls[0].y) + (ls[1].x + ls[1].y));
                tc::tmem_st_wait();
                tc::fence_before_sync();
                warp_arrive(&ctl->p_full[half][b]);
            }
            if (ok && half < halves) {
                const uint32_t hn = hn0 + ntiles - 1;
                if (wait_all(&ctl->o_full[half][hn & 1u], (hn >> 1) & 1u)) {
                    tc::fence_after_sync();
                    const bool whole = item.slot < 0;
                    const float scale = whole ? 1.0f / l : 1.0f;
                    const int64_t slot = (int64_t(item.slot) * H + h) * kRows + half * kHalf + r;
                    T* dst = static_cast<T*>(p.out) + int64_t(q0 + row / p.group) * p.out_stride +
                             int64_t(h * p.group + row % p.group) * HD;
#pragma unroll 1
                    for (int c = 0; c < HD / 32; ++c) {
                        float ov[32];
                        tc::tmem_ld32(tO + c * 32u, ov);
                        tc::tmem_ld_wait();
                        if (!live) continue;
                        // columns 4 k + (0, 1, 2, 3) are dims 4 k + (0, 2, 1, 3)
#pragma unroll
                        for (int k = 1; k < 32; k += 4) {
                            const float x = ov[k];
                            ov[k] = ov[k + 1];
                            ov[k + 1] = x;
                        }
                        if (whole) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                uint4 raw;
                                T* v = reinterpret_cast<T*>(&raw);
#pragma unroll
                                for (int q = 0; q < 8; ++q) v[q] = from_float<T>(ov[8 * k + q] * scale);
                                reinterpret_cast<uint4*>(dst + c * 32)[k] = raw;
                            }
                        } else {
                            float4* acc = reinterpret_cast<float4*>(w.acc + slot * HD + c * 32);
#pragma unroll
                            for (int k = 0; k < 8; ++k) {
                                acc[k] = make_float4(ov[4 * k] * scale, ov[4 * k + 1] * scale, ov[4 * k + 2] * scale,
                                                     ov[4 * k + 3] * scale);
                            }
                        }
                    }
                    if (live && !whole) w.ml[slot] = make_float2(m, l);
                }
            }
            tc::fence_before_sync();
            done(job);
        }
    } else if (warp < kMmaWarp) {
        // ------------------------------------------------------------- converters
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kConvRegs));
        const int ct = tid - 32 * kConvWarp0;
        const int piece = ct % S::PIECES;
        const int row0 = ct / S::PIECES;
        // Where the thread's piece goes: atom piece / 4, two 16-byte chunks swizzled by
        // the row (STEP is a multiple of 8: the same for all its rows). Pieces of the
        // second atom write theirs in the other order, so that the 8 lanes of a row
        // reach 8 places of the banks.
        const int swap = (piece >> 2) & 1;
        const uint32_t put_row = (piece >> 2) * S::ATOM + row0 * 128;
        const uint32_t put0 = put_row + (((piece & 3) * 2 + swap) ^ (row0 & 7)) * 16;
        const uint32_t put1 = put_row + (((piece & 3) * 2 + 1 - swap) ^ (row0 & 7)) * 16;
        const unsigned char* my_raw = sRaw + ct * 16;
        uint32_t slot = 0, slot_ph = 0;  // of the next tile's codes
        uint32_t st = 0, st_ph = 1;      // of the next stage, and the phase that frees it
        for (uint32_t j = 0;; ++j) {
            const int it = next_item(j);
            if (it < 0) break;
            const Job job = job_of(it);
            const int ntiles = job.ntiles;
            bool ok = true;
            for (int t = 0; ok && t < ntiles; ++t) {
                // K'
                ok = wait_all(&ctl->raw_full[0][slot], slot_ph);
                if (!ok) break;
                uint4 x[S::COPIES];
                uint2 f[S::COPIES];
#pragma unroll
                for (int i = 0; i < S::COPIES; ++i) {
                    x[i] = *reinterpret_cast<const uint4*>(my_raw + slot * S::RAW + i * S::STEP * HD);
                    f[i].x = sFactor[(slot * kKeys + row0 + S::STEP * i) * 2];
                }
                const bool small = ctl->small[slot];
                if (small) {
#pragma unroll
                    for (int i = 0; i < S::COPIES; ++i) f[i].y = sFactor[(slot * kKeys + row0 + S::STEP * i) * 2 + 1];
                }
                warp_arrive(&ctl->raw_free[0][slot]);
                // a stage's first use waits for nothing (the phase before the first)
                ok = wait_all(&ctl->k_free[st], st_ph);
                if (!ok) break;
                unsigned char* stage = sK + st * S::TILE;
#pragma unroll
                for (int i = 0; i < S::COPIES; ++i) {
                    const __half2 f2 = *reinterpret_cast<const __half2*>(&f[i].x);
                    uint32_t o[8];
                    scaled_half4<kFormat>(x[i].x, f2, o[0], o[1]);
                    scaled_half4<kFormat>(x[i].y, f2, o[2], o[3]);
                    scaled_half4<kFormat>(x[i].z, f2, o[4], o[5]);
                    scaled_half4<kFormat>(x[i].w, f2, o[6], o[7]);
                    if (small) {
                        const __half2 g = *reinterpret_cast<const __half2*>(&f[i].y);
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const __half2 y = __hmul2(*reinterpret_cast<__half2*>(&o[k]), g);
                            o[k] = *reinterpret_cast<const uint32_t*>(&y);
                        }
                    }
                    const uint4 a = make_uint4(o[0], o[1], o[2], o[3]), b = make_uint4(o[4], o[5], o[6], o[7]);
                    *reinterpret_cast<uint4*>(stage + put0 + i * S::STEP * 128) = swap ? b : a;
                    *reinterpret_cast<uint4*>(stage + put1 + i * S::STEP * 128) = swap ? a : b;
                }
                tc::fence_async_smem();
                warp_arrive(&ctl->kc_full[st]);
                // V
                ok = wait_all(&ctl->raw_full[1][slot], slot_ph);
                if (!ok) break;
#pragma unroll
                for (int i = 0; i < S::COPIES; ++i) {
                    x[i] = *reinterpret_cast<const uint4*>(my_raw + (kRaw + slot) * S::RAW + i * S::STEP * HD);
                    f[i] = *reinterpret_cast<const uint2*>(
                        sFactor + ((kRaw + slot) * kKeys + row0 + S::STEP * i) * 2);
                }
                const bool large = ctl->large[slot];
                warp_arrive(&ctl->raw_free[1][slot]);
                ok = wait_all(&ctl->v_free[st], st_ph);
                if (!ok) break;
                stage = sV + st * S::TILE;
#pragma unroll
                for (int i = 0; i < S::COPIES; ++i) {
                    const __nv_bfloat162 f2 = *reinterpret_cast<const __nv_bfloat162*>(&f[i].x);
                    uint32_t o[8];
                    scaled_bf16x4<kFormat>(x[i].x, f2, o[0], o[1]);
                    scaled_bf16x4<kFormat>(x[i].y, f2, o[2], o[3]);
                    scaled_bf16x4<kFormat>(x[i].z, f2, o[4], o[5]);
                    scaled_bf16x4<kFormat>(x[i].w, f2, o[6], o[7]);
                    if (large) {
                        const __nv_bfloat162 g = *reinterpret_cast<const __nv_bfloat162*>(&f[i].y);
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const __nv_bfloat162 y = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&o[k]), g);
                            o[k] = *reinterpret_cast<const uint32_t*>(&y);
                        }
                    }
                    const uint4 a = make_uint4(o[0], o[1], o[2], o[3]), b = make_uint4(o[4], o[5], o[6], o[7]);
                    *reinterpret_cast<uint4*>(stage + put0 + i * S::STEP * 128) = swap ? b : a;
                    *reinterpret_cast<uint4*>(stage + put1 + i * S::STEP * 128) = swap ? a : b;
                }
                tc::fence_async_smem();
                warp_arrive(&ctl->vc_full[st]);
                if (++slot == kRaw) slot = 0, slot_ph ^= 1u;
                if (++st == kStages) st = 0, st_ph ^= 1u;
            }
        }
    } else {
        // one instruction for the whole warpgroup, before its roles part
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kMmaRegs));
        if (warp >= kLoadWarp) {
            // ---------------------------------------------------------------- loaders
            const int kv = warp - kLoadWarp;  // K's or V's
            const unsigned char* codes = kv ? p.a.v_codes : p.a.k_codes;
            const int8_t* exps = kv ? p.a.v_exps : p.a.k_exps;
            const uint32_t raw_addr = smem_addr(sRaw + kv * kRaw * S::RAW) + lane * 16;
            uint32_t* factor = sFactor + kv * kRaw * kKeys * 2;
            const int row0 = lane / S::PIECES;
            uint32_t slot = 0, slot_ph = 1;  // of the next tile, and the phase that frees it
            for (uint32_t j = 0;; ++j) {
                const int it = next_item(j);
                if (it < 0) break;
                const Job job = job_of(it);
                const Kv8Item& item = job.item;
                const int h = job.h, ntiles = job.ntiles, pos_lo = job.pos_lo, pos_hi = job.pos_hi;
                const uint32_t n0 = seq;
                const int32_t* table = p.block_tables + int64_t(item.seq) * p.max_blocks;
                const int64_t column = int64_t(h) * HD + lane % S::PIECES * 16;
                const int64_t exp_head = int64_t(h) * p.a.block_size;
                // lane l finds positions l and l + 32 of a tile: the table's entry (kNone
                // where no row sees) and the slot
                constexpr int kNone = INT32_MIN;
                struct Where {
                    int blk[2], in[2];
                };
                auto find = [&](int c) -> Where {
                    Where x;
                    const int kbase = kv8_chunk(item, c) * kKeys + lane;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int pos = kbase + 32 * i;
                        x.blk[i] = kNone;
                        x.in[i] = 0;
                        if (c < item.c1 && pos <= pos_hi &&
                            (p.window <= 0 || pos > pos_lo - p.window || pos < p.sinks)) {
                            int entry;
                            kv8_place(p.a, pos, entry, x.in[i]);
                            x.blk[i] = table[entry];
                        }
                    }
                    return x;
                };
                // The factors of the lane's two positions, from their exponents (-1000:
                // nothing there): K's against the tile's largest, V's its own, in E4M3 with
                // the 2^120 that the codes lack. K's leaves fp16's range 2^31 below the
                // largest (2^29 for INT8), V's bf16's above 2^7: the rest is a second
                // factor, which almost no tile has.
                auto write_factors = [&](const int (&e)[2], uint32_t at, uint32_t n) {
                    uint32_t* dst = factor + (at * kKeys + lane) * 2;
                    if (kv == 0) {
                        const int A = max(__reduce_max_sync(0xffffffffu, max(e[0], e[1])), kKv8MinExp);
                        const int lowest = U - A + min(e[0] < kKv8MinExp ? A : e[0], e[1] < kKv8MinExp ? A : e[1]);
                        const bool small = __any_sync(0xffffffffu, lowest < kHalfMinExp);
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int g = e[i] - A + U;
                            const __half2 f = half_power(small ? max(g, -kCodeShift) : g);
                            const __half2 rest = half_power(min(g + kCodeShift, 0));
                            dst[64 * i] = *reinterpret_cast<const uint32_t*>(&f);
                            dst[64 * i + 1] = *reinterpret_cast<const uint32_t*>(&rest);
                        }
                        __syncwarp();
                        if (lane == 0) {
                            ctl->small[at] = small;
                            ctl->top[n % kTops] = A;
                            mbar_arrive(&ctl->top_full[n % kTops]);
                            mbar_arrive(&ctl->raw_full[0][at]);
                        }
                    } else {
                        constexpr int kBias = kFormat == NVLLM_KV8_E4M3 ? 120 : 0;
                        const bool large = kBias > 0 && __any_sync(0xffffffffu, max(e[0], e[1]) > 7);
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const __nv_bfloat162 f =
                                __float2bfloat162_rn(exp2_int(min(max(e[i], -126) + kBias, 127)));
                            const __nv_bfloat162 g = __float2bfloat162_rn(exp2_int(max(e[i] - 7, 0)));
                            dst[64 * i] = *reinterpret_cast<const uint32_t*>(&f);
                            dst[64 * i + 1] = *reinterpret_cast<const uint32_t*>(&g);
                        }
                        __syncwarp();
                        if (lane == 0) {
                            ctl->large[at] = large;
                            mbar_arrive(&ctl->raw_full[1][at]);
                        }
                    }
                };
                auto check = [&](Where& x) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (x.blk[i] != kNone && (x.blk[i] < 0 || x.blk[i] >= p.a.num_blocks)) {
                            atomicOr(p.status, kStatusBounds);
                            x.blk[i] = kNone;
                        }
                    }
                };
                auto load_exps = [&](const Where& x, int (&e)[2]) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        e[i] = -1000;
                        if (x.blk[i] >= 0) {
                            e[i] = exps[int64_t(x.blk[i]) * p.a.exp_block_stride + exp_head + x.in[i]];
                        }
                    }
                };
                // block ids two tiles ahead, exponents one
                Where x = find(item.c0), next = find(item.c0 + 1);
                check(x);
                int e[2];
                load_exps(x, e);
                for (int t = 0; t < ntiles; ++t) {
                    if (!wait_all(&ctl->raw_free[kv][slot], slot_ph)) break;
                    int64_t off[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        off[i] = x.blk[i] < 0 ? -1 : int64_t(x.blk[i]) * p.a.block_stride + int64_t(x.in[i]) * p.a.row;
                    }
                    const uint32_t dst = raw_addr + slot * S::RAW;
#pragma unroll
                    for (int i = 0; i < kKeys / S::LOAD_STEP; ++i) {
                        // row r's finder is lane r % 32, element r / 32, which depends on i alone
                        const int64_t at = __shfl_sync(0xffffffffu, off[S::LOAD_STEP * i / 32],
                                                       (row0 + S::LOAD_STEP * i) & 31);
                        kv8_copy16(dst + i * 512, codes + (at < 0 ? 0 : at + column), at >= 0);
                    }
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(
                                     smem_addr(&ctl->raw_full[kv][slot]))
                                 : "memory");
                    write_factors(e, slot, n0 + t);
                    x = next;
                    check(x);
                    load_exps(x, e);
                    next = find(item.c0 + t + 2);
                    if (++slot == kRaw) slot = 0, slot_ph ^= 1u;
                }
                done(job);
            }
            kv8_copy_commit();
            kv8_copy_wait<0>();
        } else {
            // ------------------------------------------------------------------- MMAs
            // One warp issues a half's MMAs. Its own instructions pace it (a few dependent
            // ones cost as much as an MMA), so what they need is built once and stepped:
            // descriptors, barrier addresses, and stage and phase of the next O and S. All
            // of it is warp-uniform and lives in uniform registers, where the
            // instructions take it from.
            auto uniform = [](uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); };
            const uint32_t i = uniform(warp - kMmaWarp);
            const uint64_t q_desc = tc::sw128_desc(uniform(smem_addr(sQ)) + i * S::Q_HALF, 16, 1024);
            const uint64_t k_desc = tc::sw128_desc(uniform(smem_addr(sK)), 16, 1024);
            const uint64_t v_desc = tc::sw128_desc(uniform(smem_addr(sV)), S::ATOM, 1024);
            const uint32_t tS = uniform(tmem) + 128u * i;
            const uint32_t tO = uniform(tmem) + 256u + 128u * i;
            auto both = [&](uint64_t* x, uint32_t px, uint64_t* y, uint32_t py) -> bool {
                return __all_sync(0xffffffffu, wait_or_abort(x, px, ctl) && wait_or_abort(y, py, ctl));
            };
            uint32_t k_st = 0, k_ph = 0, v_st = 0, v_ph = 0;  // stage and phase of the next S and O
            uint32_t s_n = 0, o_n = 0;                        // S and O of this half so far
            uint32_t q_n = 0;                                 // items with rows in this half so far
            for (uint32_t j = 0;; ++j) {
                const int it = next_item(j);
                if (it < 0) break;
                const Job job = job_of(it);
                const int ntiles = int(uniform(uint32_t(job.ntiles)));
                const bool on = uniform(uint32_t(job.halves)) > i;
                // q_full counts only items with rows in this half, on both sides: over the
                // others this warp and the half's softmax each run ahead of the other by up
                // to two items, and a phase per item would be mistaken for another's. The
                // softmax cannot leave an item of its half without this warp's S, so neither
                // is ever two counted phases from the other.
                bool ok = !on || wait_all(&ctl->q_full[i], q_n & 1u);
                q_n += on;
                // t < 0: the first two S. Then O(t) and the S that takes its P's place; the
                // softmax works on S(t + 1) meanwhile.
                for (int t = -2; ok && t < ntiles; ++t) {
                    if (t >= 0) {
                        const uint32_t b = o_n & 1u;
                        ok = on ? both(&ctl->vc_full[v_st], v_ph, &ctl->p_full[i][b], (o_n >> 1) & 1u)
                                : wait_all(&ctl->vc_full[v_st], v_ph);
                        if (!ok) break;
                        if (tc::elect_one()) {
                            if (on) {
                                tc::fence_after_sync();
                                const uint64_t vd = v_desc + v_st * (S::TILE >> 4);
                                const uint32_t pb = tS + 64u * b;
#pragma unroll
                                for (int k = 0; k < kKeys / 16; ++k) {
                                    const uint64_t v = vd + k * (2048 >> 4);
                                    tc::mma_f16_ts(tO, pb + 8u * k, v, kIdescO, k > 0 || t > 0);
                                    if constexpr (NP == 2) tc::mma_f16_ts(tO, pb + 32u + 8u * k, v, kIdescO, true);
                                }
                                tc::commit(&ctl->o_full[i][b]);
                                tc::commit(&ctl->v_free[v_st]);
                            } else {
                                mbar_arrive(&ctl->v_free[v_st]);
                            }
                        }
                        __syncwarp();
                        if (++v_st == kStages) v_st = 0, v_ph ^= 1u;
                        o_n += on;
                    }
                    if (t + 2 < ntiles) {
                        const uint32_t b = s_n & 1u;
                        // the P in this S's place is read once O(t) completes
                        ok = on && t >= 0 ? both(&ctl->kc_full[k_st], k_ph, &ctl->o_full[i][b], ((s_n - 2) >> 1) & 1u)
                                          : wait_all(&ctl->kc_full[k_st], k_ph);
                        if (!ok) break;
                        if (tc::elect_one()) {
                            if (on) {
                                tc::fence_after_sync();
                                const uint64_t kd = k_desc + k_st * (S::TILE >> 4);
                                const uint32_t d = tS + 64u * b;
#pragma unroll
                                for (int k = 0; k < HD / 16; ++k) {
                                    tc::mma_f16(d, q_desc + ((k >> 2) * (S::Q_ATOM >> 4) + (k & 3) * 2),
                                                kd + ((k >> 2) * (S::ATOM >> 4) + (k & 3) * 2), kIdescS, k > 0);
                                }
                                tc::commit(&ctl->s_full[i][b]);
                                tc::commit(&ctl->k_free[k_st]);
                            } else {
                                mbar_arrive(&ctl->k_free[k_st]);
                            }
                        }
                        issued_mma = true;
                        __syncwarp();
                        if (++k_st == kStages) k_st = 0, k_ph ^= 1u;
                        s_n += on;
                    }
                }
            }
        }
    }

    // Teardown: on an abort, let this CTA's MMAs finish (bounded) before its
    // shared memory and TMEM are released.
    if (issued_mma && tc::elect_one()) {
        tc::commit(&ctl->drain[warp - kMmaWarp]);
        const uint64_t t0 = global_ns();
        while (!mbar_try_wait(&ctl->drain[warp - kMmaWarp], 0) && global_ns() - t0 < kWaitLimitNs) {
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    if (tid == 0 && ctl->abort != 0) {
        // the record's code: the barrier's place in the control block
        report_abort(p.status, p.timeout_info, kStatusInKv8Tc, ctl->abort, reinterpret_cast<uint64_t*>(ctl));
    }
    if (warp == kMmaWarp) {
        tc::fence_after_sync();
        tc::tmem_dealloc(tmem, kTmemCols);
    }
}

template <typename T, int kFormat, int HD>
cudaError_t launch_kernel(const Kv8AttnParams& p, const Kv8Work& w, cudaStream_t st) {
    auto* k = kv8_attention_tc_kernel<T, kFormat, HD>;
    static bool ready[64] = {false};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (!ready[dev]) {
        // the split counts on what the block is launched with: with fewer registers
        // the softmax warps would wait for theirs for good
        cudaFuncAttributes attr{};
        e = cudaFuncGetAttributes(&attr, k);
        if (e != cudaSuccess) return e;
        if (attr.numRegs < kLaunchRegs) return cudaErrorInvalidConfiguration;
        e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, int(Shape<HD>::SMEM));
        if (e != cudaSuccess) return e;
        ready[dev] = true;
    }
    return launch_programmatic(k, dim3(kKv8Sms), dim3(kThreads), Shape<HD>::SMEM, st, p, w);
}

template <typename T, int kFormat>
cudaError_t launch_hd(const Kv8AttnParams& p, const Kv8Work& w, cudaStream_t st) {
    return p.a.head_dim == 64 ? launch_kernel<T, kFormat, 64>(p, w, st) : launch_kernel<T, kFormat, 128>(p, w, st);
}

template <typename T>
cudaError_t launch_type(const Kv8AttnParams& p, const Kv8Work& w, int32_t format, cudaStream_t st) {
    return format == NVLLM_KV8_E4M3 ? launch_hd<T, NVLLM_KV8_E4M3>(p, w, st)
                                    : launch_hd<T, NVLLM_KV8_INT8>(p, w, st);
}

}  // namespace

bool kv8_tc_supported(int32_t dtype, int32_t head_dim) {
    return dtype != NVLLM_DTYPE_FP32 && (head_dim == 64 || head_dim == 128);
}

Kv8Work kv8_tc_work() {
    Kv8Work w{};
    w.tile_rows = kRows;
    w.chunk = kKeys;
    w.min_run = 8;
    w.target = kKv8Sms;
    w.round = kKv8Sms;
    return w;
}

cudaError_t launch_kv8_tc(const Kv8AttnParams& p, const Kv8Work& w, int32_t dtype, int32_t format,
                          cudaStream_t stream) {
    return dtype == NVLLM_DTYPE_BF16 ? launch_type<__nv_bfloat16>(p, w, format, stream)
                                     : launch_type<__half>(p, w, format, stream);
}

}  // namespace nvllm
