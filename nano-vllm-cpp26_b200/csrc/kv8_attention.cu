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
// keeps all its bits however far apart the rows' exponents are; 2^(x_j - m) <=
// 2^100 since b_j >= -100.
//
// Operands are fp16 terms: q' of fp32 rows as two (2^-23 of the row's largest
// element), of bf16 and fp16 rows as one (exact up to 2^-25 of the largest); P of
// fp32 rows as two terms (2^-23), of others as one (2^-12, less than the output's
// own rounding). The two terms of a row are rows g and g + 8 of the same
// 16-row tile, so that a tile of fp32 rows holds 8 rows and one MMA computes both
// terms: at the few rows of a decode they cost nothing, and a lane adds its two
// halves itself.
//
// What bounds a decode is the cache's bytes. A CTA of 4 warps takes runs of
// chunks (kv8_plan.cu); a warp takes every fourth chunk of 16 positions and
// loads its fragments straight from the arenas: of K, lane (g, t) the 16-byte
// pieces t, t + 4, .. of rows g and g + 8 (the MMA's order of the dims is
// permuted to match, Q's fragments are stored that way); of V, the pieces of
// dims g of rows 2t, 2t + 1, 2t + 8, 2t + 9, whose bytes are paired across rows
// as they are converted. No shared memory and no bank conflicts on the way; K of
// the next chunk is in flight through the softmax and P V, V through Q K. The
// warps' results are joined through shared memory at the end of a run.
#include <algorithm>

#include "kv8.cuh"

namespace nvllm {

namespace {

constexpr int kWarps = 4;
constexpr int kChunk = 16;

template <typename T>
constexpr int terms() { return sizeof(T) == 4 ? 2 : 1; }

// Shapes of the fragments at head_dim HD.
template <int HD>
struct Frag {
    static constexpr int KB = HD / 4 < 16 ? HD / 4 : 16;  // bytes of one K piece of a lane
    static constexpr int KP = HD / 4 / KB;                // K pieces of a lane per row
    static constexpr int VB = HD / 8 < 16 ? HD / 8 : 16;  // bytes of one V piece
    static constexpr int VP = HD / 8 / VB;                // V pieces of a lane per row
    static constexpr int KW = KB / 4;                     // words (MMA steps) per K piece
    static constexpr int VW = VB / 4;                     // words (4 MMA tiles each) per V piece
    static constexpr int KSTEPS = HD / 16;
    static constexpr int NTILES = HD / 8;
};

template <int BYTES>
struct Piece {
    uint32_t w[BYTES / 4];
};

// Read once by this tile: do not keep it in L1.
template <int BYTES>
__device__ __forceinline__ Piece<BYTES> load_piece(const unsigned char* p) {
    Piece<BYTES> r;
    if constexpr (BYTES == 16) {
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3])
                     : "l"(p));
    } else if constexpr (BYTES == 8) {
        asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(r.w[0]), "=r"(r.w[1]) : "l"(p));
    } else {
        asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(r.w[0]) : "l"(p));
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

// a, b as fp16 in one word (a low).
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack_rest(float a, float b, uint32_t h) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    return pack_half(a - f.x, b - f.y);
}

// O of a row is rescaled only when the largest contribution grows by more than
// this (log2): until then P <= 2^margin, and it cancels in acc / l.
constexpr float kMargin = 4.0f;

template <typename T, int HD, int MT>
struct Tile {
    static constexpr int ROWS = MT * 16 / terms<T>();  // rows of a query tile
    static constexpr int Q_WORDS = MT * (HD / 16) * 128;  // fragments of Q
    static constexpr int OROW = HD + 4;
    // the warps' results overlay Q's fragments
    static constexpr size_t JOIN = size_t(kWarps) * ROWS * (OROW + 2) * 4;
    static constexpr size_t SMEM = (Q_WORDS * 4 > JOIN ? Q_WORDS * 4 : JOIN) + ROWS * 4;
};

template <typename T, int kFormat, int HD, int MT, bool kB16>
__global__ void __launch_bounds__(kWarps * 32, HD * MT >= 256 ? 2 : 3)
kv8_attention_kernel(const Kv8AttnParams p, const Kv8Work w) {
    using F = Frag<HD>;
    using S = Tile<T, HD, MT>;
    constexpr int NT = terms<T>();
    constexpr int RL = NT == 2 ? 1 : 2;  // rows of a lane per 16-row tile
    extern __shared__ __align__(16) unsigned char smem[];
    uint32_t* sQ = reinterpret_cast<uint32_t*>(smem);
    float* sO = reinterpret_cast<float*>(smem);                       // [warp][row][OROW]
    float2* sML = reinterpret_cast<float2*>(sO + kWarps * S::ROWS * S::OROW);  // [warp][row]
    float* sScale = reinterpret_cast<float*>(smem + S::SMEM) - S::ROWS;
    __shared__ int s_next;

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int g = lane >> 2;
    const int t = lane & 3;
    pdl_release();
    pdl_wait();  // the work list, the rows and the cache come from the kernels before
    const int H = p.a.num_heads;
    const int total = w.counters->items * H;

    for (;;) {
        __syncthreads();
        if (threadIdx.x == 0) s_next = atomicAdd(&w.counters->next, 1);
        __syncthreads();
        const int it = s_next;
        if (it >= total) return;
        const Kv8Item item = w.items[it / H];
        const int h = it % H;
        const int q0 = p.cu_seqlens_q[item.seq];
        const int qlen = p.cu_seqlens_q[item.seq + 1] - q0;
        const int first_pos = p.context_lens[item.seq] - qlen;
        const int nrows = min(S::ROWS, qlen * p.group - item.row0);
        const int32_t* table = p.block_tables + int64_t(item.seq) * p.max_blocks;

        // ---- Q: each row scaled to [1, 2), its terms stored as MMA fragments ----
        // A warp takes a row at a time; element d of a lane's row goes where lane
        // (g, t) of step (i, s) finds it: d = KB (t + 4 i) + 4 s + e, words e / 2 of
        // the two row halves.
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
                x[d] = on ? to_float(src[d * 32 + lane]) : 0.f;
                a = fmaxf(a, fabsf(x[d]));
            }
            a = warp_max_xor(a, 32);
            // exponent of the largest element, kept where 2^-e and 2^e are normal
            const int e = min(max(int(__float_as_uint(a) >> 23) - 127, -126), 126);
            const float inv = exp2_int(-e);
            if (lane == 0) sScale[r] = exp2_int(e) * p.qk_scale_log2;
            const int mt = r / (16 / NT), rr = r % (16 / NT);
#pragma unroll
            for (int d = 0; d < PER; ++d) {
                const float v = x[d] * inv;
                const int dim = d * 32 + lane;
                const int piece = dim / F::KB, step = (piece >> 2) * F::KW + (dim % F::KB) / 4;
                const int e4 = dim & 3;
                // word (row half) + 2 (e4 / 2) of lane (rr % 8) * 4 + piece % 4
                __half* dst = reinterpret_cast<__half*>(
                    sQ + ((mt * F::KSTEPS + step) * 32 + (rr & 7) * 4 + (piece & 3)) * 4);
                const __half hi = __float2half_rn(v);
                dst[(e4 >> 1) * 4 + (NT == 2 ? 0 : rr >> 3) * 2 + (e4 & 1)] = hi;
                if constexpr (NT == 2) {
                    dst[(e4 >> 1) * 4 + 2 + (e4 & 1)] = __float2half_rn(v - __half2float(hi));
                }
            }
        }
        __syncthreads();

        // rows of this lane: scale, position (rows past the tile see nothing, and
        // their zero Q keeps them finite)
        float qs[MT][RL];
        int pos[MT][RL];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < RL; ++i) {
                const int r = mt * 8 * RL + i * 8 + g;
                qs[mt][i] = sScale[r];
                pos[mt][i] = first_pos + (item.row0 + min(r, nrows - 1)) / p.group;
            }
        const int pos_lo = first_pos + item.row0 / p.group;
        const int pos_hi = first_pos + (item.row0 + nrows - 1) / p.group;

        float m[MT][RL], l[MT][RL];
        float o[MT][F::NTILES][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int i = 0; i < RL; ++i) {
                m[mt][i] = -INFINITY;
                l[mt][i] = 0.f;
            }
#pragma unroll
            for (int n = 0; n < F::NTILES; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[mt][n][c] = 0.f;
        }

        // ---- where the positions of a chunk live --------------------------------
        // Lane l holds, for position l % 16 of its chunk, block and slot (block < 0:
        // a position past the tile's last one, or a block outside the arena).
        int blk_ahead = 0;  // kB16: block of the warp's 32 next chunks, one per lane
        auto block_at = [&](int j) -> int {  // block of position j
            if (j > pos_hi) return -1;
            const int b = table[j / p.a.block_size];
            if (b < 0 || b >= p.a.num_blocks) {
                raise_status(kStatusBounds);
                return -1;
            }
            return b;
        };
        struct Where {
            int blk, in;  // of position lane % 16
            int exps;     // kB16 or not: a_j of position lane (< 16), b_j of lane - 16
            int base;     // first position
        };
        auto locate = [&](int c, int n) -> Where {  // entry c of the list, the warp's n-th
            Where x;
            x.base = kv8_chunk(item, c) * kChunk;
            const int j = x.base + (lane & 15);
            if constexpr (kB16) {
                if ((n & 31) == 0) {
                    const int cc = c + lane * kWarps;
                    blk_ahead = cc < item.c1 ? block_at(kv8_chunk(item, cc) * kChunk) : -1;
                }
                x.blk = __shfl_sync(0xffffffffu, blk_ahead, n & 31);
                x.in = j % p.a.block_size;
                if (j > pos_hi) x.blk = -1;
            } else {
                x.blk = block_at(j);
                x.in = j % p.a.block_size;
            }
            const int8_t* e = lane < 16 ? p.a.k_exps : p.a.v_exps;
            x.exps = 0;
            if (x.blk >= 0) x.exps = e[int64_t(x.blk) * p.a.exp_block_stride + int64_t(h) * p.a.block_size + x.in];
            return x;
        };
        auto row_of = [&](const Where& x, int key, int& blk) -> int64_t {  // byte offset of the row
            blk = __shfl_sync(0xffffffffu, x.blk, key);
            const int in = __shfl_sync(0xffffffffu, x.in, key);
            return int64_t(blk) * p.a.block_stride + int64_t(in) * p.a.row + int64_t(h) * HD;
        };
        Piece<F::KB> kr[2][F::KP];
        Piece<F::VB> vr[4][F::VP];
        auto load_k = [&](const Where& x) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                int blk;
                const int64_t at = row_of(x, g + 8 * i, blk);
#pragma unroll
                for (int q = 0; q < F::KP; ++q) {
                    if (blk >= 0) {
                        kr[i][q] = load_piece<F::KB>(p.a.k_codes + at + (t + 4 * q) * F::KB);
                    } else {
#pragma unroll
                        for (int s = 0; s < F::KW; ++s) kr[i][q].w[s] = 0;
                    }
                }
            }
        };
        auto load_v = [&](const Where& x) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                int blk;
                const int64_t at = row_of(x, 2 * t + (i & 1) + 8 * (i >> 1), blk);
#pragma unroll
                for (int q = 0; q < F::VP; ++q) {
                    if (blk >= 0) {
                        vr[i][q] = load_piece<F::VB>(p.a.v_codes + at + (g + 8 * q) * F::VB);
                    } else {
#pragma unroll
                        for (int s = 0; s < F::VW; ++s) vr[i][q].w[s] = 0;
                    }
                }
            }
        };

        int c = item.c0 + warp, n = 0;
        Where cur{};
        if (c < item.c1) {
            cur = locate(c, n);
            load_k(cur);
            load_v(cur);
        }
        for (; c < item.c1; c += kWarps, ++n) {
            // ---- S = Q K^T ------------------------------------------------------
            float s[MT][2][4];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int k = 0; k < 4; ++k) s[mt][i][k] = 0.f;
#pragma unroll
            for (int q = 0; q < F::KP; ++q)
#pragma unroll
                for (int st = 0; st < F::KW; ++st) {
                    uint32_t b[2][2];
                    to_half4<kFormat>(kr[0][q].w[st], b[0][0], b[0][1]);
                    to_half4<kFormat>(kr[1][q].w[st], b[1][0], b[1][1]);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        const uint4 a = *reinterpret_cast<const uint4*>(
                            sQ + ((mt * F::KSTEPS + q * F::KW + st) * 32 + lane) * 4);
                        // words: (row g, dims 0 1), (row g + 8, 0 1), (g, 2 3), (g + 8, 2 3)
                        const uint32_t f[4] = {a.x, a.y, a.z, a.w};
                        mma(s[mt][0], f, b[0][0], b[0][1]);
                        mma(s[mt][1], f, b[1][0], b[1][1]);
                    }
                }
            // the next chunk's K flies from here on
            const Where now = cur;
            const bool more = c + kWarps < item.c1;
            if (more) {
                cur = locate(c + kWarps, n + 1);
                load_k(cur);
            }

            // ---- softmax ----------------------------------------------------------
            // this lane's positions: base + 8 i + 2 t + e
            float ka[2][2], vb[2][2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int key = 8 * i + 2 * t + e;
                    ka[i][e] = exp2_int(min(max(__shfl_sync(0xffffffffu, now.exps, key), -126), 127));
                    vb[i][e] = float(__shfl_sync(0xffffffffu, now.exps, key + 16));
                }
            const bool ragged = now.base + kChunk - 1 > pos_lo ||
                                (p.window > 0 && now.base + p.window <= pos_hi && now.base + kChunk > p.sinks);
            uint32_t pa[MT][4];
            float alpha[MT][RL];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                for (int i = 0; i < RL; ++i) {
                    float x[2][2];
                    float top = -INFINITY;
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float d = NT == 2 ? s[mt][k][e] + s[mt][k][e + 2] : s[mt][k][2 * i + e];
                            x[k][e] = (d * ka[k][e]) * qs[mt][i];
                            if (ragged) {
                                const int j = now.base + 8 * k + 2 * t + e;
                                const bool see = j <= pos[mt][i] &&
                                                 (p.window <= 0 || j > pos[mt][i] - p.window || j < p.sinks);
                                if (!see) x[k][e] = -INFINITY;
                            }
                            top = fmaxf(top, x[k][e] + vb[k][e]);
                        }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const float mn = top > m[mt][i] + kMargin ? top : m[mt][i];
                    const float mu = mn == -INFINITY ? 0.f : mn;  // nothing seen yet
                    alpha[mt][i] = ex2(m[mt][i] - mu);
                    m[mt][i] = mn;
                    float sum = 0.f;
                    float w2[2][2];
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float y = x[k][e] - mu;
                            sum += ex2(y);
                            w2[k][e] = ex2(y + vb[k][e]);
                        }
                    l[mt][i] = fmaf(l[mt][i], alpha[mt][i], sum);
                    if constexpr (NT == 2) {
                        pa[mt][0] = pack_half(w2[0][0], w2[0][1]);
                        pa[mt][2] = pack_half(w2[1][0], w2[1][1]);
                        pa[mt][1] = pack_rest(w2[0][0], w2[0][1], pa[mt][0]);
                        pa[mt][3] = pack_rest(w2[1][0], w2[1][1], pa[mt][2]);
                    } else {
                        pa[mt][i] = pack_half(w2[0][0], w2[0][1]);
                        pa[mt][2 + i] = pack_half(w2[1][0], w2[1][1]);
                    }
                }
            }

            // ---- O += P V -----------------------------------------------------------
            // fp32 rows: the products of a chunk are added in fp32 registers, since
            // the tensor core's own accumulation truncates and a long context would
            // add that up. Others accumulate in place.
            if constexpr (NT == 1) {
                bool grew = false;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) grew |= alpha[mt][0] != 1.f || alpha[mt][1] != 1.f;
                if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int q = 0; q < F::NTILES; ++q)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[mt][q][e] *= alpha[mt][e >> 1];
                }
            }
#pragma unroll
            for (int q = 0; q < F::VP; ++q)
#pragma unroll
                for (int st = 0; st < F::VW; ++st) {
                    uint32_t b0[4], b1[4];  // of the 4 tiles of this word
                    const uint32_t x0 = vr[0][q].w[st], x1 = vr[1][q].w[st];
                    const uint32_t y0 = vr[2][q].w[st], y1 = vr[3][q].w[st];
                    to_half4<kFormat>(__byte_perm(x0, x1, 0x5140), b0[0], b0[1]);
                    to_half4<kFormat>(__byte_perm(x0, x1, 0x7362), b0[2], b0[3]);
                    to_half4<kFormat>(__byte_perm(y0, y1, 0x5140), b1[0], b1[1]);
                    to_half4<kFormat>(__byte_perm(y0, y1, 0x7362), b1[2], b1[3]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int tile = (q * F::VW + st) * 4 + j;
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            if constexpr (NT == 2) {
                                float d[4] = {0.f, 0.f, 0.f, 0.f};
                                mma(d, pa[mt], b0[j], b1[j]);
                                o[mt][tile][0] = fmaf(o[mt][tile][0], alpha[mt][0], d[0] + d[2]);
                                o[mt][tile][1] = fmaf(o[mt][tile][1], alpha[mt][0], d[1] + d[3]);
                            } else {
                                mma(o[mt][tile], pa[mt], b0[j], b1[j]);
                            }
                        }
                    }
                }
            if (more) load_v(cur);
        }

        // ---- join the warps ---------------------------------------------------------
        __syncthreads();  // Q's fragments are read no more
        // Lane (g, t) holds, of tile (q, j), dims VB (2t + e) + 8 VB q + j of rows g (+ 8)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < RL; ++i) {
                float sum = l[mt][i];
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                const int r = mt * 8 * RL + i * 8 + g;
                if (t == 0) sML[warp * S::ROWS + r] = make_float2(m[mt][i], sum);
                float* dst = sO + (warp * S::ROWS + r) * S::OROW;
#pragma unroll
                for (int q = 0; q < F::VP; ++q)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int j = 0; j < F::VB; j += 4) {
                            const int tile = q * F::VB + j;
                            const int k = NT == 2 ? e : 2 * i + e;
                            *reinterpret_cast<float4*>(dst + F::VB * (2 * t + e) + 8 * F::VB * q + j) =
                                make_float4(o[mt][tile][k], o[mt][tile + 1][k], o[mt][tile + 2][k],
                                            o[mt][tile + 3][k]);
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
                f[k] = ex2(ml[k].x - mu);
                L = fmaf(ml[k].y, f[k], L);
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
                    dst[d] = from_float<T>(v * inv);
                } else {
                    w.acc[slot * HD + d] = v;
                }
            }
            if (!whole && lane == 0) w.ml[slot] = make_float2(M, L);
        }
    }
}

template <typename T, int kFormat, int HD, int MT, bool kB16>
cudaError_t launch_kernel(const Kv8AttnParams& p, const Kv8Work& w, cudaStream_t st) {
    auto* k = kv8_attention_kernel<T, kFormat, HD, MT, kB16>;
    constexpr size_t smem = Tile<T, HD, MT>::SMEM;
    static int grid_per_device[64] = {0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    if (grid_per_device[dev] == 0) {
        e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
        if (e != cudaSuccess) return e;
        int sms = 0, per_sm = 0;
        e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
        if (e != cudaSuccess) return e;
        e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, k, kWarps * 32, smem);
        if (e != cudaSuccess) return e;
        grid_per_device[dev] = sms * std::max(per_sm, 1);
    }
    return launch_programmatic(k, dim3(unsigned(grid_per_device[dev])), dim3(kWarps * 32), smem, st, p, w);
}

template <typename T, int kFormat, int HD>
cudaError_t launch_tile(const Kv8AttnParams& p, const Kv8Work& w, cudaStream_t st) {
    const bool b16 = p.a.block_size % kChunk == 0;
    if constexpr (HD <= 128) {
        if (w.tile_rows > 16 / terms<T>()) {
            return b16 ? launch_kernel<T, kFormat, HD, 2, true>(p, w, st)
                       : launch_kernel<T, kFormat, HD, 2, false>(p, w, st);
        }
    }
    return b16 ? launch_kernel<T, kFormat, HD, 1, true>(p, w, st)
               : launch_kernel<T, kFormat, HD, 1, false>(p, w, st);
}

template <typename T, int kFormat>
cudaError_t launch_hd(const Kv8AttnParams& p, const Kv8Work& w, cudaStream_t st) {
    switch (p.a.head_dim) {
        case 32: return launch_tile<T, kFormat, 32>(p, w, st);
        case 64: return launch_tile<T, kFormat, 64>(p, w, st);
        case 128: return launch_tile<T, kFormat, 128>(p, w, st);
        case 256: return launch_tile<T, kFormat, 256>(p, w, st);
        default: return cudaErrorInvalidValue;
    }
}

template <typename T>
cudaError_t launch_type(const Kv8AttnParams& p, const Kv8Work& w, int32_t format, cudaStream_t st) {
    return format == NVLLM_KV8_E4M3 ? launch_hd<T, NVLLM_KV8_E4M3>(p, w, st)
                                    : launch_hd<T, NVLLM_KV8_INT8>(p, w, st);
}

// The work list's shape for these rows.
Kv8Work work_for(int32_t max_query_len, int32_t group, int32_t dtype, int32_t head_dim) {
    Kv8Work w{};
    const int one = dtype == NVLLM_DTYPE_FP32 ? 8 : 16;  // rows of one 16-row MMA tile
    const bool two = head_dim <= 128 && int64_t(max_query_len) * group > one;
    w.tile_rows = two ? 2 * one : one;
    w.chunk = kChunk;
    w.min_run = 32;
    w.target = 148 * 3 * 5;
    return w;
}

}  // namespace

size_t kv8_attention_workspace(int32_t num_seqs, int32_t max_query_len, int32_t max_context_len,
                               int32_t num_query_heads, const ArenaGeom& g) {
    const int group = num_query_heads / g.num_heads;
    size_t n = 0;
    for (int32_t dtype : {NVLLM_DTYPE_FP32, NVLLM_DTYPE_BF16}) {
        Kv8Work w = work_for(max_query_len, group, dtype, g.head_dim);
        n = std::max(n, kv8_work_layout(w, nullptr, num_seqs, max_query_len, max_context_len, group, g));
    }
    return n;
}

cudaError_t launch_kv8_attention(const Kv8AttnParams& p, int32_t dtype, int32_t format,
                                 void* workspace, cudaStream_t stream) {
    Kv8Work w = work_for(p.max_query_len, p.group, dtype, p.a.head_dim);
    ArenaGeom g{};
    g.num_heads = p.a.num_heads;
    g.head_dim = p.a.head_dim;
    kv8_work_layout(w, static_cast<unsigned char*>(workspace), p.num_seqs, p.max_query_len,
                    p.max_context_len, p.group, g);
    cudaError_t e = launch_kv8_plan(p, w, stream);
    if (e != cudaSuccess) return e;
    switch (dtype) {
        case NVLLM_DTYPE_FP32: e = launch_type<float>(p, w, format, stream); break;
        case NVLLM_DTYPE_BF16: e = launch_type<__nv_bfloat16>(p, w, format, stream); break;
        case NVLLM_DTYPE_FP16: e = launch_type<__half>(p, w, format, stream); break;
        default: return cudaErrorInvalidValue;
    }
    if (e != cudaSuccess || w.merge_grid == 0) return e;
    return launch_kv8_merge(p, w, dtype, stream);
}

}  // namespace nvllm
