// The 8-bit paged cache: addressing, codes and their conversions, shared by the kernels over it.
//
//   K codes [blocks][layers][kv heads][16 tokens][D]      a token's head dims are contiguous
//   V codes [blocks][layers][kv heads][D][16 tokens]      a head dim's tokens are contiguous
//   scales  [layers][kv heads][blocks][K, V]              biased exponents, one byte each
//
// A code stands for code * 2^(scale - 127).  Scales are powers of two, so that applying one is exact: a code's
// value is an fp16 / bf16 number, e4m3 codes change their scale without another rounding (but for codes that fall
// among its subnormals), and every kernel may apply the scale where that is cheapest: K's to the scores, V's in the
// conversion or to the probabilities.  Within a block V lies
// transposed because that is the operand order of the second product: a lane's 16 bytes are the 16 tokens
// of one head dim, and no transpose stands between memory and the matrix cores.  The scales lie apart from the
// codes, by layer and head: a layer's attention reads one dense array, not one byte out of every cache line.
#pragma once

#include "common.h"

namespace mkv {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef unsigned uint4v __attribute__((ext_vector_type(4)));

static constexpr int kBlk = 16;                   // tokens per block
static constexpr float kLog2E = 1.442695040888963f;
static constexpr float kFar = -1.0e30f;           // a finite "minus infinity": differences of two stay finite

// element types of q, k, v, o
struct F16 {
    typedef _Float16 elem;
    typedef half8 vec8;
    // rows are clamped to the largest value whose code cannot stand for an infinity of the type
    static constexpr float kMost = 61440.f;       // 1.875 * 2^15
    static __device__ __forceinline__ float4v mfma(vec8 a, vec8 b, float4v c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};
struct BF16 {
    typedef __bf16 elem;
    typedef bf8 vec8;
    static constexpr float kMost = 0x1.ep127f;    // 1.875 * 2^127
    static __device__ __forceinline__ float4v mfma(vec8 a, vec8 b, float4v c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};

__device__ __forceinline__ float pow2_of(unsigned biased) { return __builtin_bit_cast(float, biased << 23); }

// Code types.  exponent(): the least biased exponent e >= 1 with amax <= largest code * 2^(e - 127), read off the
// float's own bits.  encode4(): four values (already scaled into range) to four codes.  raw(): eight codes to the
// element type, unscaled; scaled(): times 2^(e - 127).
struct E4M3 {
    static constexpr bool kHasNaN = true;
    static __device__ __forceinline__ unsigned exponent(float amax) {       // 448 = 1.75 * 2^8
        const unsigned u = __builtin_bit_cast(unsigned, amax);
        const int e = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u);
        return e < 1 ? 1u : (unsigned)e;
    }
    static __device__ __forceinline__ unsigned encode4(float a, float b, float c, float d) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    }
    static __device__ __forceinline__ void decode4(unsigned w, float (&x)[4]) {
        x[0] = __builtin_amdgcn_cvt_f32_fp8(w, 0);
        x[1] = __builtin_amdgcn_cvt_f32_fp8(w, 1);
        x[2] = __builtin_amdgcn_cvt_f32_fp8(w, 2);
        x[3] = __builtin_amdgcn_cvt_f32_fp8(w, 3);
    }
    static __device__ __forceinline__ half8 scaled(F16, unsigned w0, unsigned w1, unsigned e) {
        const float s = pow2_of(e);
        const half2v a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, s, false);
        const half2v b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, s, true);
        const half2v c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, s, false);
        const half2v d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, s, true);
        return (half8){a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
    }
    static __device__ __forceinline__ bf8 scaled(BF16, unsigned w0, unsigned w1, unsigned e) {
        const float s = pow2_of(e);
        const bf2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s, false);
        const bf2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, s, true);
        const bf2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s, false);
        const bf2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, s, true);
        return (bf8){a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
    }
    template <class T>
    static __device__ __forceinline__ typename T::vec8 raw(T t, unsigned w0, unsigned w1) { return scaled(t, w0, w1, 127u); }
};

struct Int8 {
    static constexpr bool kHasNaN = false;
    static __device__ __forceinline__ unsigned exponent(float amax) {       // 127 = 1.984375 * 2^6
        const unsigned u = __builtin_bit_cast(unsigned, amax);
        const int e = (int)(u >> 23) - 6 + ((u & 0x7fffffu) > 0x7e0000u);
        return e < 1 ? 1u : (unsigned)e;
    }
    static __device__ __forceinline__ unsigned byte_of(float x) {           // nearest, ties to even; NaN has no code: 0
        return (unsigned)(int)(x == x ? __builtin_rintf(x) : 0.f) & 0xffu;
    }
    static __device__ __forceinline__ unsigned encode4(float a, float b, float c, float d) {
        return byte_of(a) | (byte_of(b) << 8) | (byte_of(c) << 16) | (byte_of(d) << 24);
    }
    static __device__ __forceinline__ void decode4(unsigned w, float (&x)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = (float)(int)(signed char)(w >> (8 * j));
    }
    // 0x6400 | u is the fp16 number 1024 + u: with u = code + 128, subtracting 1152 leaves the code
    static __device__ __forceinline__ half8 raw(F16, unsigned w0, unsigned w1) {
        const unsigned u[2] = {w0 ^ 0x80808080u, w1 ^ 0x80808080u};
        const half2v off = (half2v){(_Float16)1152.f, (_Float16)1152.f};
        half2v h[4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            h[2 * j] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, u[j], 0x04010400u)) - off;
            h[2 * j + 1] = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, u[j], 0x04030402u)) - off;
        }
        return (half8){h[0].x, h[0].y, h[1].x, h[1].y, h[2].x, h[2].y, h[3].x, h[3].y};
    }
    // The scale in two factors: 2^-30, which a block of V's smallest fp16 numbers has, is no fp16 number.  A code times the
    // first, 2^-14 at least, is exact; the second is fp16 down to its subnormals, 2^-24, and the product rounds once.
    static __device__ __forceinline__ half8 scaled(F16 t, unsigned w0, unsigned w1, unsigned e) {
        const int x = min((int)e - 127, 15);
        const int x0 = max(x, -14);
        const _Float16 f0 = __builtin_bit_cast(_Float16, (unsigned short)((x0 + 15) << 10));
        const _Float16 f1 = (_Float16)pow2_of((unsigned)(x - x0 + 127));
        return raw(t, w0, w1) * f0 * f1;
    }
    static __device__ __forceinline__ bf8 scaled(BF16, unsigned w0, unsigned w1, unsigned e) {
        const float s = pow2_of(e);
        float a[4], b[4];
        decode4(w0, a);
        decode4(w1, b);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            a[j] *= s;
            b[j] *= s;
        }
        return (bf8){(__bf16)a[0], (__bf16)a[1], (__bf16)a[2], (__bf16)a[3],
                     (__bf16)b[0], (__bf16)b[1], (__bf16)b[2], (__bf16)b[3]};
    }
    static __device__ __forceinline__ bf8 raw(BF16, unsigned w0, unsigned w1) {
        float a[4], b[4];
        decode4(w0, a);
        decode4(w1, b);
        return (bf8){(__bf16)a[0], (__bf16)a[1], (__bf16)a[2], (__bf16)a[3],
                     (__bf16)b[0], (__bf16)b[1], (__bf16)b[2], (__bf16)b[3]};
    }
};

// Bytes of one block in either code tensor, and of one (layer, head) slab in it.
__host__ __device__ __forceinline__ int64_t block_bytes8(const mkv_pool8& p) {
    return (int64_t)p.num_layers * p.num_kv_heads * kBlk * p.head_dim;
}
__host__ __device__ __forceinline__ int64_t slab_offset8(const mkv_pool8& p, int layer, int kvh) {
    return ((int64_t)layer * p.num_kv_heads + kvh) * kBlk * p.head_dim;
}
// The (K, V) exponent pair of block 0 for one layer and head; block b's is b pairs further.
__host__ __device__ __forceinline__ uint16_t* scale_row8(const mkv_pool8& p, int layer, int kvh) {
    return (uint16_t*)p.scales + ((int64_t)layer * p.num_kv_heads + kvh) * p.num_blocks;
}

// max over the four lanes {l, l^16, l^32, l^48}: swap 16-lane rows, then 32-lane halves
__device__ __forceinline__ float max_over_quarters(float x) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    x = fmaxf(__builtin_bit_cast(float, (unsigned)a[0]), __builtin_bit_cast(float, (unsigned)a[1]));
    const unsigned w = __builtin_bit_cast(unsigned, x);
    auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return fmaxf(__builtin_bit_cast(float, (unsigned)b[0]), __builtin_bit_cast(float, (unsigned)b[1]));
}
__device__ __forceinline__ float sum_over_quarters(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

int check_pool8(const mkv_pool8* p);
int check_batch8(const mkv_batch* b);

// The prefill chunks of a batch, as the kernels trust them: a chunk's rows end where the host's bounds do.
struct Chunks8 {
    const int32_t* start_locs;
    const int32_t* lens;
    int32_t max_len, num_tokens;
};
__device__ __forceinline__ int chunk_rows(const Chunks8& c, int b, int64_t start) {
    return start < 0 ? 0 : (int)max((int64_t)0, min((int64_t)min(c.lens[b], c.max_len), c.num_tokens - start));
}
__host__ __device__ __forceinline__ Chunks8 chunks_of(const mkv_batch& b) {
    return Chunks8{b.prefill_start_locs, b.prefill_lens, b.max_prefill_len, b.num_prefill_tokens};
}

// Joins the partials of output rows cut into `splits` (mid_o normalised, mid_lse = log2 of the sum of exponentials,
// kFar where a split held nothing) and writes the rows to o.  `rows`: q heads x tokens, of the longest chunk where the rows
// are those of chunks.
int launch_merge8(int dtype, int head_dim, const float* mid_o, const float* mid_lse, void* o, int64_t o_stride,
                  int32_t num_q_heads, int32_t rows, int32_t chunk_count, int32_t splits, const Chunks8& chunks, hipStream_t s);

}  // namespace mkv
