// Append to the 8-bit paged cache, alone or with the rotary embedding of q and k in the same launch.
//
// A unit of work is what one block receives in one head: rows [a, b) of K, of V or (rotary) of a q head.  One wave
// takes one unit: the maximum that decides the scale needs every row of the block at once, and up to sixteen rows
// of one head fit the wave's registers, so the new values are read once and nothing is staged.  Memory bounds a
// prefill batch (2 bytes in and 1 out an element) and the launch a decode batch.
//
//   K, q: a lane holds sixteen head dims of a row -- both members of eight rotary pairs, so that a row and its angles are
//         read once -- and 64 such pieces make a step.
//   V:    stored transposed, so a lane holds one or two head dims of all sixteen rows and writes their codes as
//         16 consecutive bytes.
//
// All of a unit's loads go out before anything waits for one: lanes and steps without a row of their own read one that
// the unit has, rather than branch.  The rows a block already held are read again only where a larger scale makes their
// codes change (K), or where a lane's 16 bytes hold codes that have to survive (V).
//
// With the rotary embedding, eight prompts of 512 tokens, 32 + 32 heads x 128: 36.5 us for 170 MB, 4.65 TB/s, what a copy
// reaches (4.7); five ragged chunks and 57 decode rows of 64 + 8 heads 16 us for 66 MB, 4.1 TB/s; 64 decode rows of 32 + 8 heads
// 4.6 us, the launch.  Before a unit's loads went out together the prompts took 50 us.
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
    int32_t blocks_per_seq;                                 // cells per prefill sequence
    int32_t unit_groups;                                    // workgroups per cell, four units each
};

// What one cell (decode rows first, then the prefill sequences' blocks) covers: rows [a, b) of block `pid` (its first row is batch row `row`, position 16 j + a).
struct Cell {
    int64_t pid;          // -1: the rows have no place in the cache
    int64_t row;
    int64_t pos0;         // position of the block's row 0
    int a, b;             // rows of the cell
    int b_known;          // rows [a, b_known) lie inside the rotary tables
};

template <bool ROPE>
__device__ __forceinline__ bool find_cell(const Store8Args& g, int cell, Cell& c) {
    const mkv_batch& m = g.batch;
    int64_t seq_slot;
    int64_t blk;
    if (cell >= m.num_decoding_seqs) {
        const int s = (cell - m.num_decoding_seqs) / g.blocks_per_seq;
        const int j = cell - m.num_decoding_seqs - s * g.blocks_per_seq;
        const int64_t start = m.prefill_start_locs[s];
        const int64_t len = chunk_rows(chunks_of(m), s, start);
        const int64_t prefix = m.prefix_lens ? max(m.prefix_lens[s], 0) : 0;
        if (len <= 0) return false;
        blk = prefix / kBlk + j;
        const int64_t first = max(prefix, blk * kBlk), end = min(prefix + len, (blk + 1) * kBlk);
        if (first >= end) return false;
        c.a = (int)(first - blk * kBlk);
        c.b = (int)(end - blk * kBlk);
        c.row = start + (first - prefix);
        seq_slot = s;
    } else {
        const int i = cell;
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

// Where the lane's sixteen dims of a row lie: two runs of eight.
struct Piece {
    int lo, hi;           // first dims of the runs
    int table;            // first of the eight table columns; -1: not rotated
};

template <bool ROPE>
__device__ __forceinline__ Piece piece_at(const Store8Args& g, int i) {
    Piece p = {16 * i, 16 * i + 8, -1};
    if (ROPE && 16 * i < g.rotary_dim) {                             // rotary_dim is a multiple of 16
        p.table = 8 * i;
        if (!g.interleaved) {
            p.lo = 8 * i;
            p.hi = 8 * i + (g.rotary_dim >> 1);
        }
    }
    return p;
}

// The piece of one row, rotated by the table row of `pos`: x[0 .. 8) from dim lo, x[8 .. 16) from dim hi.
template <class T, bool ROPE>
__device__ __forceinline__ void load_piece(const typename T::elem* row, const Piece& p, int64_t pos, const Store8Args& g,
                                           float (&x)[16]) {
    typedef typename T::vec8 vec8;
    const vec8 lo = *(const vec8*)(row + p.lo), hi = *(const vec8*)(row + p.hi);
    float c[8], s[8];
    if constexpr (ROPE) {
        const int64_t at = pos * (g.rotary_dim >> 1) + max(p.table, 0);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float4v cv = *(const float4v*)(g.cos_t + at + 4 * j), sv = *(const float4v*)(g.sin_t + at + 4 * j);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                c[4 * j + e] = cv[e];
                s[4 * j + e] = sv[e];
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        x[e] = (float)lo[e];
        x[8 + e] = (float)hi[e];
    }
    if constexpr (ROPE) {
#pragma clang fp contract(off)
        if (p.table < 0) return;
        const bool side = g.interleaved;                             // pairs side by side, or eight apart in x
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (side) {
                const float x0 = x[2 * e], x1 = x[2 * e + 1];
                const float p0 = x0 * c[e], p1 = x1 * s[e], p2 = x0 * s[e], p3 = x1 * c[e];
                x[2 * e] = p0 - p1;
                x[2 * e + 1] = p2 + p3;
            } else {
                const float x0 = x[e], x1 = x[8 + e];
                const float p0 = x0 * c[e], p1 = x1 * s[e], p2 = x0 * s[e], p3 = x1 * c[e];
                x[e] = p0 - p1;
                x[8 + e] = p2 + p3;
            }
        }
    }
}

// Rows of the steps.  ONE: the unit has a single row (a decode step's), which the first lanes take in one step.
template <bool ONE, int PIECES>
struct Steps {
    static constexpr int count = ONE ? 1 : kBlk * PIECES / 64;
    static __device__ __forceinline__ int row(const Cell& c, int lane, int i) { return ONE ? c.a : (lane + 64 * i) / PIECES; }
    static __device__ __forceinline__ bool mine(int lane) { return !ONE || lane < PIECES; }
};

template <class T, int D, bool ONE>
__device__ __forceinline__ void rotate_q(const Store8Args& g, const Cell& c, int head, int lane) {
    typedef typename T::elem E;
    typedef typename T::vec8 vec8;
    typedef Steps<ONE, D / 16> S;
    const Piece p = piece_at<true>(g, lane % (D / 16));
    float x[S::count][16];
    // every row is read before any is written: q_out may be q
#pragma unroll
    for (int i = 0; i < S::count; ++i) {
        const int r = min(max(S::row(c, lane, i), c.a), c.b - 1);
        const int64_t pos = r < c.b_known ? c.pos0 + r : 0;
        load_piece<T, true>((const E*)g.q + (c.row + (r - c.a)) * g.q_stride + (int64_t)head * D, p, pos, g, x[i]);
    }
#pragma unroll
    for (int i = 0; i < S::count; ++i) {
        const int r = S::row(c, lane, i);
        if (!S::mine(lane) || r < c.a || r >= c.b) continue;
        const bool lost = r >= c.b_known && p.table >= 0;            // no angle for this row
        vec8 lo, hi;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            lo[e] = (E)(lost ? __builtin_nanf("") : x[i][e]);
            hi[e] = (E)(lost ? __builtin_nanf("") : x[i][8 + e]);
        }
        E* dst = (E*)g.q_out + (c.row + (r - c.a)) * g.q_out_stride + (int64_t)head * D;
        *(vec8*)(dst + p.lo) = lo;
        *(vec8*)(dst + p.hi) = hi;
    }
}

// The block's exponent once rows with this maximum have joined it, and the one its older codes have.
template <class C>
__device__ __forceinline__ unsigned joined_exponent(float amax, bool fresh, unsigned had) {
    const unsigned e = C::exponent(amax);
    return fresh ? e : max(e, had);
}

// Four codes of an older scale at the new one.
template <class C>
__device__ __forceinline__ unsigned moved4(unsigned w, float again) {
    float y[4];
    C::decode4(w, y);
    return C::encode4(y[0] * again, y[1] * again, y[2] * again, y[3] * again);
}

template <class T, class C, int D, bool ROPE, bool ONE>
__device__ __forceinline__ void store_k(const Store8Args& g, const Cell& c, int kvh, int lane) {
    typedef typename T::elem E;
    typedef Steps<ONE, D / 16> S;
    const Piece p = piece_at<ROPE>(g, lane % (D / 16));
    uint8_t* scale = (uint8_t*)(scale_row8(g.pool, g.layer, kvh) + c.pid);
    const unsigned had = scale[0];
    float x[S::count][16];
    float amax = 0.f;
    // a row outside the unit's is read as its nearest one, which the maximum does not mind
#pragma unroll
    for (int i = 0; i < S::count; ++i) {
        const int r = min(max(S::row(c, lane, i), c.a), c.b_known - 1);
        load_piece<T, ROPE>((const E*)g.k + (c.row + (r - c.a)) * g.k_stride + (int64_t)kvh * D, p, c.pos0 + r, g, x[i]);
    }
#pragma unroll
    for (int i = 0; i < S::count; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            x[i][e] = clamped<T>(x[i][e]);
            amax = fmaxf(amax, __builtin_fabsf(x[i][e]));            // a NaN does not enter
        }
    amax = wave_max(amax);
    const unsigned e8 = joined_exponent<C>(amax, c.a == 0, had);
    const float inv = pow2_of(254u - min(e8, 253u));
    uint8_t* slab = (uint8_t*)g.pool.k + c.pid * block_bytes8(g.pool) + slab_offset8(g.pool, g.layer, kvh);
#pragma unroll
    for (int i = 0; i < S::count; ++i) {
        const int r = S::row(c, lane, i);
        if (!S::mine(lane) || r < c.a || r >= c.b_known) continue;
        float y[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) y[e] = x[i][e] * inv;
        *(uint2*)(slab + r * D + p.lo) = make_uint2(C::encode4(y[0], y[1], y[2], y[3]), C::encode4(y[4], y[5], y[6], y[7]));
        *(uint2*)(slab + r * D + p.hi) = make_uint2(C::encode4(y[8], y[9], y[10], y[11]), C::encode4(y[12], y[13], y[14], y[15]));
    }
    if (c.a > 0 && e8 != had) {                                      // the same for the wave
        const float again = pow2_of(had) * inv;                      // older codes to the new scale
        for (int u = lane; u < c.a * (D / 16); u += 64) {
            uint4* at = (uint4*)slab + u;
            const uint4 w = *at;
            *at = make_uint4(moved4<C>(w.x, again), moved4<C>(w.y, again), moved4<C>(w.z, again), moved4<C>(w.w, again));
        }
    }
    if (lane == 0) scale[0] = (uint8_t)e8;
}

template <class T, class C, int D, bool ONE>
__device__ __forceinline__ void store_v(const Store8Args& g, const Cell& c, int kvh, int lane) {
    typedef typename T::elem E;
    constexpr int kDims = D / 64;                                    // head dims per lane
    constexpr int kN = ONE ? 1 : kBlk;                               // rows read
    typedef E vecd __attribute__((ext_vector_type(kDims)));
    const E* src = (const E*)g.v + (int64_t)kvh * D + lane * kDims;
    uint8_t* scale = (uint8_t*)(scale_row8(g.pool, g.layer, kvh) + c.pid) + 1;
    const unsigned had = *scale;
    uint4* at = (uint4*)((uint8_t*)g.pool.v + c.pid * block_bytes8(g.pool) + slab_offset8(g.pool, g.layer, kvh)) + lane * kDims;
    const bool whole = !ONE && c.a == 0 && c.b_known == kBlk;
    vecd y[kN];
#pragma unroll
    for (int r = 0; r < kN; ++r) {
        const int rr = ONE ? c.a : min(max(r, c.a), c.b_known - 1);
        y[r] = *(const vecd*)(src + (c.row + (rr - c.a)) * g.v_stride);
    }
    uint4 held[kDims];
#pragma unroll
    for (int d = 0; d < kDims; ++d) held[d] = whole ? make_uint4(0u, 0u, 0u, 0u) : at[d];
    float x[kDims][kN];
    float amax = 0.f;
#pragma unroll
    for (int r = 0; r < kN; ++r)
#pragma unroll
        for (int d = 0; d < kDims; ++d) {
            x[d][r] = clamped<T>((float)y[r][d]);
            amax = fmaxf(amax, __builtin_fabsf(x[d][r]));
        }
    amax = wave_max(amax);
    const unsigned e8 = joined_exponent<C>(amax, c.a == 0, had);
    const float inv = pow2_of(254u - min(e8, 253u));
    const float again = pow2_of(had) * inv;
    const bool moves = c.a > 0 && e8 != had;
    // of each word's four rows: those below a take their moved codes, [a, b) the new ones, those behind stay
    auto word = [&](unsigned w, unsigned fresh, int n) {
        auto below = [n](int r) {
            const int in = min(max(r - 4 * n, 0), 4);
            return in >= 4 ? ~0u : (1u << (8 * in)) - 1u;
        };
        const unsigned old = below(c.a), upto = below(c.b_known);
        if (moves) w = (w & ~old) | (moved4<C>(w, again) & old);
        return (w & ~(upto & ~old)) | (fresh & upto & ~old);
    };
#pragma unroll
    for (int d = 0; d < kDims; ++d) {
        unsigned fresh[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            if (ONE) fresh[n] = n ? fresh[0] : C::encode4(x[d][0] * inv, x[d][0] * inv, x[d][0] * inv, x[d][0] * inv);
            else fresh[n] = C::encode4(x[d][(4 * n) % kN] * inv, x[d][(4 * n + 1) % kN] * inv, x[d][(4 * n + 2) % kN] * inv, x[d][(4 * n + 3) % kN] * inv);
        }
        if (whole) at[d] = make_uint4(fresh[0], fresh[1], fresh[2], fresh[3]);
        else at[d] = make_uint4(word(held[d].x, fresh[0], 0), word(held[d].y, fresh[1], 1), word(held[d].z, fresh[2], 2), word(held[d].w, fresh[3], 3));
    }
    if (lane == 0) *scale = (uint8_t)e8;
}

template <class T, class C, int D, bool ROPE>
__global__ __launch_bounds__(256) void store8_kernel(const Store8Args g) {
    const int lane = threadIdx.x & 63;
    // unit: K heads, V heads, then q heads.  The heads of a cell are consecutive workgroups: together they read whole rows.
    const int cell = (int)(blockIdx.x / (unsigned)g.unit_groups);
    const int unit = __builtin_amdgcn_readfirstlane(((int)blockIdx.x - cell * g.unit_groups) * 4 + (int)(threadIdx.x >> 6));
    const int Hkv = g.pool.num_kv_heads;
    Cell c;
    if (!find_cell<ROPE>(g, cell, c)) return;
    if (unit < 2 * Hkv) {
        if (c.pid < 0 || c.b_known <= c.a) return;
        const bool one = c.b_known - c.a == 1;
        if (unit < Hkv && one) store_k<T, C, D, ROPE, true>(g, c, unit, lane);
        else if (unit < Hkv) store_k<T, C, D, ROPE, false>(g, c, unit, lane);
        else if (one) store_v<T, C, D, true>(g, c, unit - Hkv, lane);
        else store_v<T, C, D, false>(g, c, unit - Hkv, lane);
    } else if (ROPE && unit < 2 * Hkv + g.num_q_heads) {
        if (c.b - c.a == 1) rotate_q<T, D, true>(g, c, unit - 2 * Hkv, lane);
        else rotate_q<T, D, false>(g, c, unit - 2 * Hkv, lane);
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
        MKV_REQUIRE(num_positions > 0, "the rotary tables hold no position");
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
    g.unit_groups = mkv::cdiv(units, 4);
    MKV_REQUIRE(cells * g.unit_groups * 256 <= 0xffffffffll, "too many rows in one call");      // threads of a launch
    const dim3 grid((unsigned)(cells * g.unit_groups));
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
