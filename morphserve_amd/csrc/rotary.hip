// Rotary position embedding from positions: half or interleaved pairs, part of the head, fp32 tables.
//
//   (x0, x1) -> (x0 c - x1 s, x0 s + x1 c)        products and sums in 32 bits, one rounding at the end
//
// Nothing is reused but a token's table row (by its heads), so memory bounds it: every element of q and k is read
// and written once.  A thread takes eight pairs of one head (16 bytes of each member of the pair) or, where the
// output is another tensor, eight of the dims behind the rotated ones.  The tokens' units are numbered
// through, so that a workgroup is full whatever the number of heads; a token's table row is read by its heads from
// the caches.  16385 tokens of 32 + 8 heads x 128, half of each head rotated, into other tensors: 73.2 us for 340 MB, 4.6 TB/s; 64 tokens
// 3.9 us, the launch.
#include "kv8.h"

namespace mkv {

static constexpr int kVec = 8;       // pairs, or kept dims, per thread: 16 bytes of each member of the pair

struct RotaryArgs {
    const void *q, *k;
    void *q_out, *k_out;
    int64_t q_stride, k_stride, q_out_stride, k_out_stride;    // elements
    const int32_t* positions;
    const float *cos_t, *sin_t;
    int64_t num_positions;
    int32_t num_tokens, num_q_heads, num_heads, head_dim, rotary_dim;
    int32_t units, rot_units;        // units per head row; the first rot_units of them rotate
};

// The pair (x0, x1) turned by the angle of (c, s): no contraction, so that every path rounds alike.
__device__ __forceinline__ void turn(float x0, float x1, float c, float s, float& y0, float& y1) {
#pragma clang fp contract(off)
    const float p0 = x0 * c, p1 = x1 * s, p2 = x0 * s, p3 = x1 * c;
    y0 = p0 - p1;
    y1 = p2 + p3;
}

// A vector from or to an address of any alignment that its elements have.
template <bool LOOSE, class V, class E>
__device__ __forceinline__ V wide_load(const E* p) {
    if constexpr (!LOOSE) return *(const V*)p;
    V v;
    __builtin_memcpy(&v, p, sizeof(V));
    return v;
}
template <bool LOOSE, class V, class E>
__device__ __forceinline__ void wide_store(E* p, V v) {
    if constexpr (!LOOSE) *(V*)p = v;
    else __builtin_memcpy(p, &v, sizeof(V));
}

// LOOSE: the number of pairs or of kept dims is no multiple of kVec, or an address or stride not aligned for it.  The accesses
// are as wide, at whatever address, and a head's last thread takes its last kVec pairs, some of which are its neighbour's too:
// written twice, alike, or, in place, left to the neighbour.
template <class T, bool INTERLEAVED, bool LOOSE>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryArgs a) {
    typedef typename T::elem E;
    typedef E vec __attribute__((ext_vector_type(kVec)));
    typedef float fvec __attribute__((ext_vector_type(kVec)));
    const uint32_t per_token = (uint32_t)a.num_heads * a.units;
    const uint32_t idx = blockIdx.x * 256u + threadIdx.x;          // the launcher keeps this below 2^31
    const uint32_t t = idx / per_token;
    if (t >= (uint32_t)a.num_tokens) return;
    const uint32_t r = idx - t * per_token;
    const uint32_t head = r / (uint32_t)a.units;
    const int u = (int)(r - head * a.units);
    const bool is_k = (int)head >= a.num_q_heads;
    const int64_t h = is_k ? (int)head - a.num_q_heads : (int)head;
    const E* src = (const E*)(is_k ? a.k : a.q) + (int64_t)t * (is_k ? a.k_stride : a.q_stride) + h * a.head_dim;
    E* dst = (E*)(is_k ? a.k_out : a.q_out) + (int64_t)t * (is_k ? a.k_out_stride : a.q_out_stride) + h * a.head_dim;
    if (u >= a.rot_units) {
        int d = a.rotary_dim + (u - a.rot_units) * kVec;
        if (LOOSE && d + kVec > a.head_dim) {
            if (a.head_dim - a.rotary_dim < kVec) {
                for (int e = d; e < a.head_dim; ++e) dst[e] = src[e];
                return;
            }
            d = a.head_dim - kVec;
        }
        wide_store<LOOSE>(dst + d, wide_load<LOOSE, vec>(src + d));
        return;
    }
    const int half = a.rotary_dim >> 1;
    const int64_t pos = a.positions[t];
    const bool known = pos >= 0 && pos < a.num_positions;
    const int first = LOOSE && half >= kVec ? min(u * kVec, half - kVec) : u * kVec;      // of the thread's pairs
    const int64_t row = known ? pos * half + first : 0;
    const int d0 = INTERLEAVED ? 2 * first : first;
    if (LOOSE && half < kVec) {
        for (int j = 0; j < half; ++j) {
            const int e0 = d0 + (INTERLEAVED ? 2 * j : j), e1 = INTERLEAVED ? e0 + 1 : e0 + half;
            const float c = known ? a.cos_t[row + j] : __builtin_nanf(""), s = known ? a.sin_t[row + j] : __builtin_nanf("");
            float y0, y1;
            turn((float)src[e0], (float)src[e1], c, s, y0, y1);
            dst[e0] = (E)y0;
            dst[e1] = (E)y1;
        }
        return;
    }
    const int d1 = INTERLEAVED ? d0 + kVec : d0 + half;
    const vec a0 = wide_load<LOOSE, vec>(src + d0), a1 = wide_load<LOOSE, vec>(src + d1);
    fvec c, s;
    if (known) {
        c = wide_load<LOOSE, fvec>(a.cos_t + row);
        s = wide_load<LOOSE, fvec>(a.sin_t + row);
    } else {
        c = s = (fvec)__builtin_nanf("");
    }
    vec o0, o1;
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
        // the j-th pair: in the interleaved layout elements 2j, 2j + 1 of the 2 kVec read
        const int e0 = 2 * j, e1 = 2 * j + 1;
        const float x0 = (float)(INTERLEAVED ? (e0 < kVec ? a0[e0 % kVec] : a1[e0 % kVec]) : a0[j]);
        const float x1 = (float)(INTERLEAVED ? (e1 < kVec ? a0[e1 % kVec] : a1[e1 % kVec]) : a1[j]);
        float y0, y1;
        turn(x0, x1, c[j], s[j], y0, y1);
        if (INTERLEAVED) {
            if (e0 < kVec) o0[e0 % kVec] = (E)y0; else o1[e0 % kVec] = (E)y0;
            if (e1 < kVec) o0[e1 % kVec] = (E)y1; else o1[e1 % kVec] = (E)y1;
        } else {
            o0[j] = (E)y0;
            o1[j] = (E)y1;
        }
    }
    if (LOOSE && first != u * kVec && src == dst) {
        const int own = INTERLEAVED ? 2 * (u * kVec - first) : u * kVec - first;       // elements in front of the thread's own
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
            if (e >= own) dst[d0 + e] = o0[e];
            if (e + (INTERLEAVED ? kVec : 0) >= own) dst[d1 + e] = o1[e];
        }
        return;
    }
    wide_store<LOOSE>(dst + d0, o0);
    wide_store<LOOSE>(dst + d1, o1);
}

template <class T, bool LOOSE>
static void launch_rotary(int layout, dim3 grid, hipStream_t s, const RotaryArgs& a) {
    if (layout == MKV_ROPE_HALF)
        hipLaunchKernelGGL((rotary_kernel<T, false, LOOSE>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((rotary_kernel<T, true, LOOSE>), grid, dim3(256), 0, s, a);
}

}  // namespace mkv

extern "C" int mkv_rope_positions(int32_t dtype, int32_t layout, const void* q, const void* k, void* q_out, void* k_out,
                                  int64_t q_stride, int64_t k_stride, int64_t q_out_stride, int64_t k_out_stride,
                                  const int32_t* positions, const float* cos_table, const float* sin_table,
                                  int64_t num_positions, int64_t num_tokens, int32_t num_q_heads,
                                  int32_t num_kv_heads, int32_t head_dim, int32_t rotary_dim, void* stream) {
    MKV_REQUIRE(dtype == MKV_F16 || dtype == MKV_BF16, "dtype %d is neither MKV_F16 nor MKV_BF16", dtype);
    MKV_REQUIRE(layout == MKV_ROPE_HALF || layout == MKV_ROPE_INTERLEAVED, "unknown rotary layout %d", layout);
    MKV_REQUIRE(num_tokens >= 0 && num_tokens <= 0x7fffffff, "num_tokens %lld outside [0, 2^31)", (long long)num_tokens);
    MKV_REQUIRE(num_q_heads > 0 && num_kv_heads >= 0 && num_q_heads <= 65535 && num_kv_heads <= 65535,
                "head counts %d, %d outside the supported range", num_q_heads, num_kv_heads);
    MKV_REQUIRE(head_dim > 0 && head_dim <= 65535 && rotary_dim > 0 && rotary_dim <= head_dim && rotary_dim % 2 == 0,
                "rotary_dim %d must be even and within head_dim %d", rotary_dim, head_dim);
    if (num_tokens == 0) return MKV_OK;
    MKV_REQUIRE(q && q_out && positions && cos_table && sin_table && (num_kv_heads == 0 || (k && k_out)), "NULL argument");
    MKV_REQUIRE(num_positions >= 0, "num_positions must be >= 0");
    const int64_t q_row = (int64_t)num_q_heads * head_dim, k_row = (int64_t)num_kv_heads * head_dim;
    MKV_REQUIRE(num_tokens == 1 || (q_stride >= q_row && q_out_stride >= q_row && k_stride >= k_row && k_out_stride >= k_row),
                "rows overlap: a stride is shorter than its row");
    MKV_REQUIRE(num_tokens == 1 || ((q != q_out || q_stride == q_out_stride) && (!k || k != k_out || k_stride == k_out_stride)),
                "in place, input and output have one stride");
    // 16385 tokens of 32 + 8 heads x 128, 104 dims half-split: aligned accesses of four pairs 95 us, loose ones of eight 77; 70
    // dims, where not even two divide the pairs: one pair a thread 278 us, loose 95, interleaved 251 and 81.
    const uintptr_t at = (uintptr_t)q | (uintptr_t)q_out | (uintptr_t)k | (uintptr_t)k_out | (uintptr_t)cos_table | (uintptr_t)sin_table;
    int64_t strides = q_stride | q_out_stride;
    if (num_kv_heads) strides |= k_stride | k_out_stride;
    const bool loose = (rotary_dim / 2) % mkv::kVec != 0 || head_dim % mkv::kVec != 0 || strides % mkv::kVec != 0 || at % 16 != 0;
    mkv::RotaryArgs a = {};
    a.num_q_heads = num_q_heads;
    a.num_heads = num_q_heads + num_kv_heads;
    a.head_dim = head_dim;
    a.rotary_dim = rotary_dim;
    a.rot_units = mkv::cdiv(rotary_dim / 2, mkv::kVec);
    const bool in_place = q == q_out && (num_kv_heads == 0 || k == k_out);
    a.units = a.rot_units + (in_place ? 0 : mkv::cdiv(head_dim - rotary_dim, mkv::kVec));
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.q_out_stride = q_out_stride;
    a.k_out_stride = k_out_stride;
    a.cos_t = cos_table;
    a.sin_t = sin_table;
    a.num_positions = num_positions;
    hipStream_t s = (hipStream_t)stream;
    // thread numbers are 32-bit: very long batches go out in parts
    const int64_t per_token = (int64_t)a.num_heads * a.units;
    const int64_t most = ((int64_t)1 << 30) / per_token > 0 ? ((int64_t)1 << 30) / per_token : 1;
    MKV_REQUIRE(per_token < ((int64_t)1 << 30), "a row of %lld units is too long", (long long)per_token);
    for (int64_t t0 = 0; t0 < num_tokens; t0 += most) {
        const int64_t n = num_tokens - t0 < most ? num_tokens - t0 : most;
        a.q = (const char*)q + t0 * q_stride * 2;
        a.q_out = (char*)q_out + t0 * q_out_stride * 2;
        a.k = num_kv_heads ? (const char*)k + t0 * k_stride * 2 : nullptr;
        a.k_out = num_kv_heads ? (char*)k_out + t0 * k_out_stride * 2 : nullptr;
        a.positions = positions + t0;
        a.num_tokens = (int32_t)n;
        const dim3 grid((unsigned)((n * per_token + 255) / 256));
        if (dtype == MKV_F16) {
            if (loose) mkv::launch_rotary<mkv::F16, true>(layout, grid, s, a);
            else mkv::launch_rotary<mkv::F16, false>(layout, grid, s, a);
        } else {
            if (loose) mkv::launch_rotary<mkv::BF16, true>(layout, grid, s, a);
            else mkv::launch_rotary<mkv::BF16, false>(layout, grid, s, a);
        }
        MKV_HIP(hipGetLastError());
    }
    return MKV_OK;
}
