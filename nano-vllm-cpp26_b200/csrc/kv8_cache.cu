// The quantising write into the 8-bit paged arenas, and the read back.
//
// A row of one (token, KV head) is head_dim values x. With M the largest code
// (448 for E4M3, 127 for INT8):
//   x' = 0 for NaN, else x clamped to +-M 2^119
//   e  = the smallest integer >= -100 with max|x'| <= M 2^e
//   code = x' 2^-e rounded to the nearest code, ties to even
// e comes from the bits of max|x'|: max = f 2^b with 1 <= f < 2, and M = 1.75 * 2^8
// or 1.984375 * 2^6, so e = b - 8 (or 6), plus one where f exceeds M's fraction. x' 2^-e
// is exact (a power of two) wherever it is not far below the smallest code.
// The read is code 2^e, exact in fp32 and bf16.
//
// Both move bytes and nothing else: 2 * head_dim * (sizeof(T) + 1) + 2 per (token,
// KV head), the floor being that at the copy rate. In the write a thread owns 16
// values of K and the same 16 of V (one 16-byte store of codes each), hd / 16
// neighbouring lanes share a row and find its maximum by shuffles; all of a
// thread's loads are in flight before the first is used. Measured on B200, 10229
// tokens of 32 x 128 fp32: 71 us, 5.9 TB/s (0.90 of the copy rate); 65536 of 8 x 128
// bf16: 90-98 us, 4.1-4.5 TB/s.
#include "kv8.cuh"

namespace nvllm {

namespace {

constexpr int kThreads = 256;
constexpr int kPiece = 16;  // values per thread and tensor

// 16 consecutive values as fp32.
template <typename T, bool kVec>
__device__ __forceinline__ void load_piece(const T* src, float* x) {
    if constexpr (kVec) {
        constexpr int N = 16 / int(sizeof(T));  // values in 16 bytes
        uint4 raw[kPiece / N];
#pragma unroll
        for (int i = 0; i < kPiece / N; ++i) raw[i] = __ldcs(reinterpret_cast<const uint4*>(src) + i);
#pragma unroll
        for (int i = 0; i < kPiece / N; ++i) {
            const T* v = reinterpret_cast<const T*>(&raw[i]);
#pragma unroll
            for (int j = 0; j < N; ++j) x[i * N + j] = to_float(v[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kPiece; ++i) x[i] = to_float(src[i]);
    }
}

template <int kFormat>
struct Format;
template <>
struct Format<NVLLM_KV8_E4M3> {
    static constexpr uint32_t kFraction = 0x600000u;  // 448 = 1.75 * 2^8
    static constexpr int kBits = 8;
    static constexpr float kMax = 448.0f;
};
template <>
struct Format<NVLLM_KV8_INT8> {
    static constexpr uint32_t kFraction = 0x7E0000u;  // 127 = 1.984375 * 2^6
    static constexpr int kBits = 6;
    static constexpr float kMax = 127.0f;
};

template <int kFormat>
__device__ __forceinline__ int row_exponent(float a) {
    using F = Format<kFormat>;
    const uint32_t b = __float_as_uint(a);
    const int e = int(b >> 23) - 127 - F::kBits + ((b & 0x7FFFFFu) > F::kFraction ? 1 : 0);
    return max(e, kKv8MinExp);
}

// Four values, already scaled by 2^-e, as codes.
template <int kFormat>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
    if constexpr (kFormat == NVLLM_KV8_E4M3) {
        uint32_t w;
        asm("{\n\t.reg .b16 lo, hi;\n\t"
            "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
            "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
            "mov.b32 %0, {lo, hi};\n\t}"
            : "=r"(w)
            : "f"(a), "f"(b), "f"(c), "f"(d));
        return w;
    } else {
        // |x| <= 127: adding 1.5 * 2^23 rounds to the nearest integer, ties to
        // even, into the low bits
        const float c0 = 12582912.0f;
        const uint32_t ab = __byte_perm(__float_as_uint(a + c0), __float_as_uint(b + c0), 0x0040);
        const uint32_t cd = __byte_perm(__float_as_uint(c + c0), __float_as_uint(d + c0), 0x0040);
        return __byte_perm(ab, cd, 0x5410);
    }
}

// Clamps, finds the row's exponent with the hd / 16 lanes of the row, and
// encodes this thread's 16 values.
template <int kFormat, int HD>
__device__ __forceinline__ int encode_piece(float* x, uint4& codes) {
    constexpr float kTop = Format<kFormat>::kMax * 0x1p119f;
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < kPiece; ++i) {
        x[i] = x[i] == x[i] ? fminf(fmaxf(x[i], -kTop), kTop) : 0.f;
        a = fmaxf(a, fabsf(x[i]));
    }
#pragma unroll
    for (int o = 1; o < HD / kPiece; o <<= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
    const int e = row_exponent<kFormat>(a);
    const float inv = exp2_int(-e);
#pragma unroll
    for (int i = 0; i < kPiece; ++i) x[i] *= inv;
    codes = make_uint4(encode4<kFormat>(x[0], x[1], x[2], x[3]), encode4<kFormat>(x[4], x[5], x[6], x[7]),
                       encode4<kFormat>(x[8], x[9], x[10], x[11]),
                       encode4<kFormat>(x[12], x[13], x[14], x[15]));
    return e;
}

// Where piece `piece` of slot `slot` lives.
struct Place {
    int64_t codes;
    int64_t exp;
};
template <int HD>
__device__ __forceinline__ Place place_of(const Kv8Arena& a, int32_t slot, uint32_t piece) {
    const int32_t blk = slot / a.block_size;
    const int32_t in = slot % a.block_size;
    const uint32_t head = piece / (HD / kPiece);
    return {blk * a.block_stride + in * a.row + int64_t(piece) * kPiece,
            blk * a.exp_block_stride + int64_t(head) * a.block_size + in};
}

template <typename T, int kFormat, int HD, bool kVec>
__global__ void __launch_bounds__(kThreads)
kv8_write_kernel(const Kv8Arena a, const Kv8Rows r) {
    pdl_release();
    pdl_wait();  // the rows and the slot mapping may come from the kernel before
    const uint32_t per_token = uint32_t(a.row / kPiece);
    const uint32_t idx = blockIdx.x * kThreads + threadIdx.x;
    const uint32_t t = idx / per_token;
    const uint32_t piece = idx % per_token;
    // the lanes of a row agree on all of this; they stay for the shuffles
    int32_t slot = t < r.num_tokens ? r.slots[t] : -1;
    if (slot >= 0 && slot / a.block_size >= a.num_blocks) {
        if (piece == 0) raise_status(kStatusBounds);
        slot = -1;
    }
    float k[kPiece], v[kPiece];
    if (slot >= 0) {
        load_piece<T, kVec>(static_cast<const T*>(r.key) + t * r.key_stride + piece * kPiece, k);
        load_piece<T, kVec>(static_cast<const T*>(r.value) + t * r.value_stride + piece * kPiece, v);
    } else {
#pragma unroll
        for (int i = 0; i < kPiece; ++i) k[i] = v[i] = 0.f;
    }
    uint4 kc, vc;
    const int ke = encode_piece<kFormat, HD>(k, kc);
    const int ve = encode_piece<kFormat, HD>(v, vc);
    if (slot < 0) return;
    const Place at = place_of<HD>(a, slot, piece);
    *reinterpret_cast<uint4*>(a.k_codes + at.codes) = kc;
    *reinterpret_cast<uint4*>(a.v_codes + at.codes) = vc;
    if (piece % (HD / kPiece) == 0) {
        a.k_exps[at.exp] = int8_t(ke);
        a.v_exps[at.exp] = int8_t(ve);
    }
}

// The read's pieces are 16 bytes of output (4 or 8 values), so that a warp's stores
// are whole lines; a thread takes kReads of them, kThreads apart, of K and of V.
// Measured on B200, 32768 rows of 32 x 128 to fp32: 261 us, 5.1 TB/s (four pieces a
// thread 274; the write's pieces, four strided 16-byte stores of fp32, 288); 65536 of
// 8 x 128 to bf16: 84 us, 4.8 TB/s.
constexpr int kReads = 2;

template <typename T, int kFormat, bool kVec>
__device__ __forceinline__ void store_values(T* dst, const uint32_t* codes, int e) {
    constexpr int N = 16 / int(sizeof(T));
    // a row that the write made has e in [-100, 119]
    const float scale = exp2_int(min(max(e, -126), 127));
    T x[N];
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        const float4 c = kv8_codes4<kFormat>(codes[i]);
        x[4 * i] = from_float<T>(c.x * scale);
        x[4 * i + 1] = from_float<T>(c.y * scale);
        x[4 * i + 2] = from_float<T>(c.z * scale);
        x[4 * i + 3] = from_float<T>(c.w * scale);
    }
    if constexpr (kVec) {
        uint4 raw;
        T* v = reinterpret_cast<T*>(&raw);
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = x[j];
        __stcs(reinterpret_cast<uint4*>(dst), raw);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) dst[i] = x[i];
    }
}

template <typename T, int kFormat, int HD, bool kVec>
__global__ void __launch_bounds__(kThreads) kv8_read_kernel(const Kv8Arena a, const Kv8Rows r) {
    constexpr int N = 16 / int(sizeof(T));  // values of a piece
    pdl_release();
    pdl_wait();
    const uint32_t per_token = uint32_t(a.row / N);
    const uint64_t total = uint64_t(r.num_tokens) * per_token;
    const uint64_t first = uint64_t(blockIdx.x) * (kThreads * kReads) + threadIdx.x;
    uint32_t t[kReads], piece[kReads], kc[kReads][N / 4], vc[kReads][N / 4];
    int ke[kReads], ve[kReads];
    bool on[kReads];
#pragma unroll
    for (int i = 0; i < kReads; ++i) {
        const uint64_t idx = first + uint64_t(i) * kThreads;
        on[i] = idx < total;
        // (both fit 32 bits: the pieces of 16 values of a call do)
        t[i] = on[i] ? uint32_t(idx / per_token) : 0;
        piece[i] = uint32_t(idx - uint64_t(t[i]) * per_token);
        const int32_t slot = on[i] ? r.slots[t[i]] : -1;
        on[i] = slot >= 0;
        if (on[i] && slot / a.block_size >= a.num_blocks) {
            if (piece[i] == 0) raise_status(kStatusBounds);
            on[i] = false;
        }
        if (!on[i]) continue;
        const int32_t blk = slot / a.block_size;
        const int32_t in = slot % a.block_size;
        const int64_t at = blk * a.block_stride + in * a.row + int64_t(piece[i]) * N;
        const int64_t ea = blk * a.exp_block_stride + int64_t(piece[i] / (HD / N)) * a.block_size + in;
        if constexpr (N == 4) {
            kc[i][0] = __ldcs(reinterpret_cast<const uint32_t*>(a.k_codes + at));
            vc[i][0] = __ldcs(reinterpret_cast<const uint32_t*>(a.v_codes + at));
        } else {
            const uint2 x = __ldcs(reinterpret_cast<const uint2*>(a.k_codes + at));
            const uint2 y = __ldcs(reinterpret_cast<const uint2*>(a.v_codes + at));
            kc[i][0] = x.x, kc[i][1] = x.y, vc[i][0] = y.x, vc[i][1] = y.y;
        }
        ke[i] = a.k_exps[ea];
        ve[i] = a.v_exps[ea];
    }
#pragma unroll
    for (int i = 0; i < kReads; ++i) {
        if (!on[i]) continue;
        const int64_t c = int64_t(piece[i]) * N;
        store_values<T, kFormat, kVec>(static_cast<T*>(r.key) + t[i] * r.key_stride + c, kc[i], ke[i]);
        store_values<T, kFormat, kVec>(static_cast<T*>(r.value) + t[i] * r.value_stride + c, vc[i], ve[i]);
    }
}

template <typename T, int kFormat, int HD>
cudaError_t launch_hd(bool write, const Kv8Arena& a, const Kv8Rows& r, bool vec, cudaStream_t st) {
    const uint64_t per_cta = write ? uint64_t(kThreads) * kPiece
                                   : uint64_t(kThreads) * kReads * (16 / sizeof(T));
    const dim3 grid(unsigned((uint64_t(r.num_tokens) * uint64_t(a.row) + per_cta - 1) / per_cta));
    auto* k = write ? (vec ? kv8_write_kernel<T, kFormat, HD, true> : kv8_write_kernel<T, kFormat, HD, false>)
                    : (vec ? kv8_read_kernel<T, kFormat, HD, true> : kv8_read_kernel<T, kFormat, HD, false>);
    return launch_programmatic(k, grid, dim3(kThreads), 0, st, a, r);
}

template <typename T, int kFormat>
cudaError_t launch_format(bool write, const Kv8Arena& a, const Kv8Rows& r, bool vec, cudaStream_t st) {
    switch (a.head_dim) {
        case 32: return launch_hd<T, kFormat, 32>(write, a, r, vec, st);
        case 64: return launch_hd<T, kFormat, 64>(write, a, r, vec, st);
        case 128: return launch_hd<T, kFormat, 128>(write, a, r, vec, st);
        case 256: return launch_hd<T, kFormat, 256>(write, a, r, vec, st);
        default: return cudaErrorInvalidValue;
    }
}

template <typename T>
cudaError_t launch_type(bool write, const Kv8Arena& a, const Kv8Rows& r, int32_t format, bool vec,
                        cudaStream_t st) {
    return format == NVLLM_KV8_E4M3 ? launch_format<T, NVLLM_KV8_E4M3>(write, a, r, vec, st)
                                    : launch_format<T, NVLLM_KV8_INT8>(write, a, r, vec, st);
}

cudaError_t launch(bool write, const Kv8Arena& a, const Kv8Rows& r, int32_t dtype, int32_t format,
                   bool vec, cudaStream_t st) {
    switch (dtype) {
        case NVLLM_DTYPE_FP32: return launch_type<float>(write, a, r, format, vec, st);
        case NVLLM_DTYPE_BF16: return launch_type<__nv_bfloat16>(write, a, r, format, vec, st);
        case NVLLM_DTYPE_FP16: return launch_type<__half>(write, a, r, format, vec, st);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace

cudaError_t launch_kv8_write(const Kv8Arena& a, const Kv8Rows& r, int32_t dtype, int32_t format,
                             bool vec, cudaStream_t stream) {
    return launch(true, a, r, dtype, format, vec, stream);
}

cudaError_t launch_kv8_read(const Kv8Arena& a, const Kv8Rows& r, int32_t dtype, int32_t format,
                            bool vec, cudaStream_t stream) {
    return launch(false, a, r, dtype, format, vec, stream);
}

}  // namespace nvllm
