// Append to the 8-bit paged cache, alone or with the rotary embedding of q and k in the same launch.
//
// A unit of work is what one block receives in one head: rows [a, b) of K, of V or (rotary) of a q head.  One wave
// takes one unit: the maximum that decides the scale needs every row of the block at once, and up to sixteen rows
// of one head fit the wave's registers, so the new values are read once and nothing is staged.  Memory bounds a
// prefill batch (2 bytes in and 1 out an element) and the launch a decode batch.
//
//   K, q: a lane holds eight consecutive head dims of a row, 64 such pieces a step; the members of a rotary pair
//         that lie in another piece are read a second time (from the cache line just fetched) rather than exchanged.
//   V:    stored transposed, so a lane holds one or two head dims of all sixteen rows and writes their codes as
//         16 consecutive bytes.
//
// The rows a block already held are read again only where a larger scale makes their codes change (K), or where a
// lane's 16 bytes hold codes that have to survive (V).
#include "kv8.h"

namespace mkv {

struct Store8Args {
    mkv_pool8 pool;
    mkv_batch batch;
    const char *k, *v, *q;
    char* q_out;
    int64_t k_stride, v_stride, q_stride, q_out_stride;     // elements
    const float *cos_t, *sin_t;
    int64_t num_positions;
    int32_t layer, num_q_heads, rotary_dim, interleaved;
    int32_t blocks_per_seq;                                 // grid cells per prefill sequence
};

// What one grid cell covers: rows [a, b) of block `pid` (its first row is batch row `row`, position 16 j + a).
struct Cell {
    int64_t pid;          // -1: the rows have no place in the cache
    int64_t row;
    int64_t pos0;         // position of the block's row 0
    int a, b;             // rows of the cell
    int b_known;          // rows [a, b_known) lie inside the rotary tables
};

template <bool ROPE>
__device__ __forceinline__ bool find_cell(const Store8Args& g, Cell& c) {
    const mkv_batch& m = g.batch;
    const int prefill_cells = m.num_prefill_seqs * g.blocks_per_seq;
    int64_t seq_slot;
    int64_t blk;
    if ((int)blockIdx.x < prefill_cells) {
        const int s = (int)blockIdx.x / g.blocks_per_seq;
        const int j = (int)blockIdx.x - s * g.blocks_per_seq;
        const int64_t start = m.prefill_start_locs[s];
        const int64_t len = chunk_rows(chunks_of(m), s, start);
        const int64_t prefix = m.prefix_lens ? m.prefix_lens[s] : 0;
        if (len <= 0 || prefix < 0) return false;
        blk = prefix / kBlk + j;
        const int64_t first = max(prefix, blk * kBlk), end = min(prefix + len, (blk + 1) * kBlk);
        if (first >= end) return false;
        c.a = (int)(first - blk * kBlk);
        c.b = (int)(end - blk * kBlk);
        c.row = start + (first - prefix);
        seq_slot = s;
    } else {
        const int i = (int)blockIdx.x - prefill_cells;
        const int64_t pos = (int64_t)m.decoding_lens[i] - 1;
        c.row = (int64_t)m.num_prefill_tokens + i;
        blk = pos >= 0 ? pos / kBlk : 0;
        c.a = pos >= 0 ? (int)(pos - blk * kBlk) : 0;
        c.b = c.a + 1;
        seq_slot = (int64_t)m.num_prefill_seqs + i;
        if (pos < 0) {                                      // no position: no place in the cache, q is not known
            c.pid = -1;
            c.pos0 = 0;
            c.b_known = c.a;
            return ROPE;
        }
    }
    c.pos0 = blk * kBlk;
    const int64_t seq = m.seq_ids[seq_slot];
    c.pid = -1;
    if (seq >= 0 && seq < m.table_rows && blk < m.max_blocks_per_seq) {
        const int64_t pid = m.block_table[seq * m.max_blocks_per_seq + blk];
        if (pid >= 0 && pid < g.pool.num_blocks) c.pid = pid;
    }
    c.b_known = ROPE ? (int)max((int64_t)c.a, min((int64_t)c.b, g.num_positions - c.pos0)) : c.b;
    return true;
}

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) x = fmaxf(x, __shfl_xor(x, s));
    return x;
}

// the largest finite value of the cache instead of what lies beyond it; NaN stays
template <class T>
__device__ __forceinline__ float clamped(float x) {
    return __builtin_fabsf(x) > T::kMost ? __builtin_copysignf(T::kMost, x) : x;
}

// Eight consecutive head dims [8 ch, 8 ch + 8) of a row, rotated by the table row of `pos`.
template <class T, bool ROPE>
__device__ __forceinline__ void load_piece(const typename T::elem* row, int ch, int64_t pos, const Store8Args& g,
                                           float (&x)[8]) {
    typedef typename T::vec8 vec8;
    const vec8 own = *(const vec8*)(row + 8 * ch);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)own[e];
    if constexpr (ROPE) {
#pragma clang fp contract(off)
        const int R = g.rotary_dim, half = R >> 1;
        if (8 * ch >= R) return;
        if (g.interleaved) {
            const float4v c = *(const float4v*)(g.cos_t + pos * half + 4 * ch);
            const float4v s = *(const float4v*)(g.sin_t + pos * half + 4 * ch);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float x0 = x[2 * j], x1 = x[2 * j + 1];
                const float p0 = x0 * c[j], p1 = x1 * s[j], p2 = x0 * s[j], p3 = x1 * c[j];
                x[2 * j] = p0 - p1;
                x[2 * j + 1] = p2 + p3;
            }
        } else {
            const bool upper = 8 * ch >= half;                       // half is a multiple of 8
            const int d = 8 * ch - (upper ? half : 0);
            const vec8 other = *(const vec8*)(row + (upper ? d : d + half));
            float c[8], s[8];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float4v cv = *(const float4v*)(g.cos_t + pos * half + d + 4 * j);
                const float4v sv = *(const float4v*)(g.sin_t + pos * half + d + 4 * j);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    c[4 * j + e] = cv[e];
                    s[4 * j + e] = sv[e];
                }
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float y = (float)other[e];
                const float p = x[e] * c[e], r = y * s[e];           // the piece is x0 below half, x1 above
                x[e] = upper ? r + p : p - r;
            }
        }
    }
}

template <class T, int D>
__device__ __forceinline__ void rotate_q(const Store8Args& g, const Cell& c, int head, int lane) {
    typedef typename T::elem E;
    constexpr int kPieces = D / 8;
#pragma unroll
    for (int i = 0; i < kBlk * kPieces / 64; ++i) {
        const int id = lane + 64 * i;
        const int r = id / kPieces, ch = id % kPieces;
        // a row's pieces are read by the lanes of one step before any of them is written: q_out may be q
        if (r < c.a || r >= c.b) continue;
        const int64_t row = c.row + (r - c.a);
        const E* src = (const E*)g.q + row * g.q_stride + (int64_t)head * D;
        float x[8];
        if (r < c.b_known) {
            load_piece<T, true>(src, ch, c.pos0 + r, g, x);
        } else {
            load_piece<T, false>(src, ch, 0, g, x);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (8 * ch < g.rotary_dim) x[e] = __builtin_nanf("");
        }
        typename T::vec8 o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = (E)x[e];
        *(typename T::vec8*)((E*)g.q_out + row * g.q_out_stride + (int64_t)head * D + 8 * ch) = o;
    }
}

// The block's exponent once rows with this maximum have joined it, and the one its older codes have.
template <class C>
__device__ __forceinline__ unsigned joined_exponent(float amax, bool fresh, unsigned had) {
    const unsigned e = C::exponent(amax);
    return fresh ? e : max(e, had);
}

template <class T, class C, int D, bool ROPE>
__device__ __forceinline__ void store_k(const Store8Args& g, const Cell& c, int kvh, int lane) {
    typedef typename T::elem E;
    constexpr int kPieces = D / 8, kSteps = kBlk * kPieces / 64;
    float x[kSteps][8];
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const int id = lane + 64 * i;
        const int r = id / kPieces, ch = id % kPieces;
        if (r >= c.a && r < c.b_known) {
            const E* src = (const E*)g.k + (c.row + (r - c.a)) * g.k_stride + (int64_t)kvh * D;
            load_piece<T, ROPE>(src, ch, c.pos0 + r, g, x[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[i][e] = clamped<T>(x[i][e]);
                amax = fmaxf(amax, __builtin_fabsf(x[i][e]));        // a NaN does not enter
            }
        }
    }
    amax = wave_max(amax);
    uint8_t* scale = (uint8_t*)(scale_row8(g.pool, g.layer, kvh) + c.pid);
    const unsigned had = scale[0];
    const unsigned e8 = joined_exponent<C>(amax, c.a == 0, had);
    const float inv = pow2_of(254u - min(e8, 253u));
    const float again = pow2_of(had) * inv;                          // older codes to the new scale
    uint8_t* slab = (uint8_t*)g.pool.k + c.pid * block_bytes8(g.pool) + slab_offset8(g.pool, g.layer, kvh);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const int id = lane + 64 * i;
        const int r = id / kPieces, ch = id % kPieces;
        uint2* at = (uint2*)(slab + r * D + 8 * ch);
        if (r >= c.a && r < c.b_known) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = x[i][e] * inv;
            *at = make_uint2(C::encode4(y[0], y[1], y[2], y[3]), C::encode4(y[4], y[5], y[6], y[7]));
        } else if (r < c.a && e8 != had) {
            const uint2 old = *at;
            float y[4], z[4];
            C::decode4(old.x, y);
            C::decode4(old.y, z);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                y[e] *= again;
                z[e] *= again;
            }
            *at = make_uint2(C::encode4(y[0], y[1], y[2], y[3]), C::encode4(z[0], z[1], z[2], z[3]));
        }
    }
    if (lane == 0) scale[0] = (uint8_t)e8;
}

template <class T, class C, int D>
__device__ __forceinline__ void store_v(const Store8Args& g, const Cell& c, int kvh, int lane) {
    typedef typename T::elem E;
    constexpr int kDims = D / 64;                                    // head dims per lane
    typedef E vecd __attribute__((ext_vector_type(kDims)));
    float x[kDims][kBlk];
    float amax = 0.f;
    const E* src = (const E*)g.v + (int64_t)kvh * D + lane * kDims;
#pragma unroll
    for (int r = 0; r < kBlk; ++r) {
#pragma unroll
        for (int d = 0; d < kDims; ++d) x[d][r] = 0.f;
        if (r >= c.a && r < c.b_known) {                             // the same for the whole wave
            const vecd y = *(const vecd*)(src + (c.row + (r - c.a)) * g.v_stride);
#pragma unroll
            for (int d = 0; d < kDims; ++d) {
                x[d][r] = clamped<T>((float)y[d]);
                amax = fmaxf(amax, __builtin_fabsf(x[d][r]));
            }
        }
    }
    amax = wave_max(amax);
    uint8_t* scale = (uint8_t*)(scale_row8(g.pool, g.layer, kvh) + c.pid) + 1;
    const unsigned had = *scale;
    const unsigned e8 = joined_exponent<C>(amax, c.a == 0, had);
    const float inv = pow2_of(254u - min(e8, 253u));
    const float again = pow2_of(had) * inv;
    uint4v* at = (uint4v*)((uint8_t*)g.pool.v + c.pid * block_bytes8(g.pool) + slab_offset8(g.pool, g.layer, kvh)) + lane * kDims;
    const bool whole = c.a == 0 && c.b_known == kBlk;
#pragma unroll
    for (int d = 0; d < kDims; ++d) {
        uint4v w = {0u, 0u, 0u, 0u};
        if (!whole) w = at[d];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const unsigned fresh = C::encode4(x[d][4 * n] * inv, x[d][4 * n + 1] * inv, x[d][4 * n + 2] * inv, x[d][4 * n + 3] * inv);
            unsigned kept = w[n];
            if (!whole && 4 * n < c.a && e8 != had) {
                float y[4];
                C::decode4(kept, y);
                const unsigned moved = C::encode4(y[0] * again, y[1] * again, y[2] * again, y[3] * again);
                // rows below a take their moved codes; what lies behind the cell's rows stays
                const int below = min(c.a - 4 * n, 4);
                const unsigned mask = below >= 4 ? ~0u : (1u << (8 * below)) - 1u;
                kept = (kept & ~mask) | (moved & mask);
            }
            const int lo = min(max(c.a - 4 * n, 0), 4), hi = min(max(c.b_known - 4 * n, 0), 4);
            const unsigned to_hi = hi >= 4 ? ~0u : (1u << (8 * hi)) - 1u;
            const unsigned to_lo = lo >= 4 ? ~0u : (1u << (8 * lo)) - 1u;
            const unsigned mask = to_hi & ~to_lo;
            w[n] = (kept & ~mask) | (fresh & mask);
        }
        at[d] = w;
    }
    if (lane == 0) *scale = (uint8_t)e8;
}

template <class T, class C, int D, bool ROPE>
__global__ __launch_bounds__(256) void store8_kernel(const Store8Args g) {
    const int lane = threadIdx.x & 63;
    // unit: K heads, V heads, then q heads
    int unit = __builtin_amdgcn_readfirstlane((int)blockIdx.y * 4 + (int)(threadIdx.x >> 6));
    const int Hkv = g.pool.num_kv_heads;
    Cell c;
    if (!find_cell<ROPE>(g, c)) return;
    if (unit < 2 * Hkv) {
        if (c.pid < 0 || c.b_known <= c.a) return;
        if (unit < Hkv) store_k<T, C, D, ROPE>(g, c, unit, lane);
        else store_v<T, C, D>(g, c, unit - Hkv, lane);
    } else if (ROPE && unit < 2 * Hkv + g.num_q_heads) {
        rotate_q<T, D>(g, c, unit - 2 * Hkv, lane);
    }
}

int check_pool8(const mkv_pool8* p) {
    MKV_REQUIRE(p != nullptr, "pool is NULL");
    MKV_REQUIRE(p->k && p->v && p->scales, "pool pointers are NULL");
    MKV_REQUIRE(p->num_layers > 0 && p->num_kv_heads > 0 && p->num_kv_heads <= 65535, "pool dims must be positive (L=%d Hkv=%d)",
                p->num_layers, p->num_kv_heads);
    MKV_REQUIRE(p->block_size == kBlk, "the 8-bit cache supports block_size 16 only (got %d)", p->block_size);
    MKV_REQUIRE(p->head_dim == 64 || p->head_dim == 128, "the 8-bit cache supports head_dim 64 and 128 (got %d)", p->head_dim);
    MKV_REQUIRE(p->kind == MKV_KV8_E4M3 || p->kind == MKV_KV8_INT8, "unknown kind %d of 8-bit codes", p->kind);
    MKV_REQUIRE(p->num_blocks >= 1 && p->num_blocks <= 0x7fffffff, "the pool must hold 1 to 2^31 - 1 blocks (got %lld)",
                (long long)p->num_blocks);
    MKV_REQUIRE(((uintptr_t)p->k & 15) == 0 && ((uintptr_t)p->v & 15) == 0 && ((uintptr_t)p->scales & 1) == 0,
                "pool bases must be 16-byte aligned, scales 2-byte aligned");
    return MKV_OK;
}

int check_batch8(const mkv_batch* b) {
    MKV_REQUIRE(b != nullptr, "batch is NULL");
    MKV_REQUIRE(b->num_prefill_seqs >= 0 && b->num_prefill_tokens >= 0 && b->max_prefill_len >= 0 && b->num_decoding_seqs >= 0,
                "negative count");
    if (b->num_prefill_seqs == 0 && b->num_decoding_seqs == 0) return MKV_OK;
    MKV_REQUIRE(b->block_table && b->seq_ids, "NULL argument");
    MKV_REQUIRE(b->max_blocks_per_seq >= 0 && b->max_blocks_per_seq <= ((int64_t)1 << 26) && b->table_rows >= 0,
                "a block table of %lld x %lld is not supported", (long long)b->table_rows, (long long)b->max_blocks_per_seq);
    MKV_REQUIRE(b->num_prefill_seqs == 0 || (b->prefill_start_locs && b->prefill_lens), "prefill rows without their tables");
    MKV_REQUIRE(b->num_decoding_seqs == 0 || b->decoding_lens, "decode rows without their lengths");
    return MKV_OK;
}

template <class T, class C>
static void launch_store8(int head_dim, bool rope, dim3 grid, hipStream_t s, const Store8Args& g) {
    if (head_dim == 128 && rope) hipLaunchKernelGGL((store8_kernel<T, C, 128, true>), grid, dim3(256), 0, s, g);
    else if (head_dim == 128) hipLaunchKernelGGL((store8_kernel<T, C, 128, false>), grid, dim3(256), 0, s, g);
    else if (rope) hipLaunchKernelGGL((store8_kernel<T, C, 64, true>), grid, dim3(256), 0, s, g);
    else hipLaunchKernelGGL((store8_kernel<T, C, 64, false>), grid, dim3(256), 0, s, g);
}

}  // namespace mkv

extern "C" {

int mkv_sizeof_pool8(void) { return (int)sizeof(mkv_pool8); }

int mkv_sizeof_batch(void) { return (int)sizeof(mkv_batch); }

int mkv_store8(const mkv_pool8* pool, const mkv_batch* batch, int32_t dtype, const void* k, const void* v,
               int64_t k_stride, int64_t v_stride, int32_t layer, int32_t rope, const void* q, void* q_out,
               int64_t q_stride, int64_t q_out_stride, int32_t num_q_heads, const float* cos_table,
               const float* sin_table, int64_t num_positions, int32_t rotary_dim, void* stream) {
    int rc = mkv::check_pool8(pool);
    if (rc) return rc;
    rc = mkv::check_batch8(batch);
    if (rc) return rc;
    MKV_REQUIRE(dtype == MKV_F16 || dtype == MKV_BF16, "dtype %d is neither MKV_F16 nor MKV_BF16", dtype);
    MKV_REQUIRE(layer >= 0 && layer < pool->num_layers, "layer %d outside [0, %d)", layer, pool->num_layers);
    MKV_REQUIRE(rope == MKV_ROPE_NONE || rope == MKV_ROPE_HALF || rope == MKV_ROPE_INTERLEAVED, "unknown rotary layout %d", rope);
    const bool prefill = batch->num_prefill_seqs > 0 && batch->max_prefill_len > 0;
    if (!prefill && batch->num_decoding_seqs == 0) return MKV_OK;
    MKV_REQUIRE(k && v, "NULL argument");
    MKV_REQUIRE((((uintptr_t)k | (uintptr_t)v) & 15) == 0 && ((k_stride | v_stride) & 7) == 0,
                "k/v rows must be 16-byte aligned");
    mkv::Store8Args g = {};
    g.pool = *pool;
    g.batch = *batch;
    g.k = (const char*)k;
    g.v = (const char*)v;
    g.k_stride = k_stride;
    g.v_stride = v_stride;
    g.layer = layer;
    int units = 2 * pool->num_kv_heads;
    if (rope != MKV_ROPE_NONE) {
        MKV_REQUIRE(q && q_out && cos_table && sin_table, "NULL argument");
        MKV_REQUIRE(num_q_heads > 0 && num_q_heads <= 65535, "num_q_heads %d outside the supported range", num_q_heads);
        MKV_REQUIRE(rotary_dim > 0 && rotary_dim <= pool->head_dim && rotary_dim % 16 == 0,
                    "rotary_dim %d must be a multiple of 16 within head_dim %d", rotary_dim, pool->head_dim);
        MKV_REQUIRE(num_positions >= 0, "num_positions must be >= 0");
        MKV_REQUIRE((((uintptr_t)q | (uintptr_t)q_out | (uintptr_t)cos_table | (uintptr_t)sin_table) & 15) == 0 &&
                        ((q_stride | q_out_stride) & 7) == 0,
                    "q rows and the rotary tables must be 16-byte aligned");
        MKV_REQUIRE(q != q_out || q_stride == q_out_stride, "in place, q and q_out have one stride");
        g.q = (const char*)q;
        g.q_out = (char*)q_out;
        g.q_stride = q_stride;
        g.q_out_stride = q_out_stride;
        g.num_q_heads = num_q_heads;
        g.cos_t = cos_table;
        g.sin_t = sin_table;
        g.num_positions = num_positions;
        g.rotary_dim = rotary_dim;
        g.interleaved = rope == MKV_ROPE_INTERLEAVED;
        units += num_q_heads;
    }
    // a chunk behind a prefix may begin inside a block: one cell more
    g.blocks_per_seq = prefill ? mkv::cdiv(batch->max_prefill_len, mkv::kBlk) + (batch->prefix_lens ? 1 : 0) : 0;
    const int64_t cells = (int64_t)batch->num_prefill_seqs * g.blocks_per_seq + batch->num_decoding_seqs;
    MKV_REQUIRE(cells <= 0x7fffffff, "too many rows in one call");
    const dim3 grid((unsigned)cells, (unsigned)mkv::cdiv(units, 4));
    hipStream_t s = (hipStream_t)stream;
    const bool rot = rope != MKV_ROPE_NONE;
    if (dtype == MKV_F16) {
        if (pool->kind == MKV_KV8_E4M3) mkv::launch_store8<mkv::F16, mkv::E4M3>(pool->head_dim, rot, grid, s, g);
        else mkv::launch_store8<mkv::F16, mkv::Int8>(pool->head_dim, rot, grid, s, g);
    } else {
        if (pool->kind == MKV_KV8_E4M3) mkv::launch_store8<mkv::BF16, mkv::E4M3>(pool->head_dim, rot, grid, s, g);
        else mkv::launch_store8<mkv::BF16, mkv::Int8>(pool->head_dim, rot, grid, s, g);
    }
    MKV_HIP(hipGetLastError());
    return MKV_OK;
}

}  // extern "C"
