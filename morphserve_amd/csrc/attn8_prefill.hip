// Chunked prefill attention over the 8-bit paged cache.
//
// The rows of one kv head -- chunk positions times the q heads that share it, position-major -- are cut into tiles
// of 128, one workgroup of four waves each; a wave owns two 16-row column tiles.  Keys come 64 at a time (four
// blocks): their codes are converted once, on the way into LDS, and every wave reads the converted tile from there,
//
//   S^T[key, row] = K . Q^T        v_mfma_f32_16x16x32
//   O^T[dim, row] += V^T . P^T     v_mfma_f32_16x16x32
//
// while the next tile's codes are on their way from memory and the tile after that lends its block ids.  As in the
// decode kernel the keys are numbered so that lane group c scores block c in order, which makes K's scale one factor
// per lane and the scores, exponentiated, the operand of the second product.  V arrives transposed from the cache,
// so that both products read LDS in rows.  Where few rows meet many keys, the keys are cut into splits.
#include "kv8.h"

namespace mkv {

static constexpr int kRows = 128;             // rows per workgroup
static constexpr int kCols = 2;               // 16-row column tiles per wave
static constexpr float kLazyP = 8.f;

struct Prefill8Args {
    mkv_pool8 pool;
    mkv_batch batch;
    const char* q;
    char* o;
    int64_t q_stride, o_stride;               // elements
    float *mid_o, *mid_lse;
    int32_t group, layer, tiles_per_split, max_splits;
    int32_t num_row_tiles;                    // of the longest chunk
    float scale2;
};

// LDS rows: K has one row a key, V one a head dim.  16 bytes behind a row, and 64 more behind a block's keys, put
// the sixteen rows that the first product's operand takes (four of each block) on different banks; V's rows of 144
// bytes do the same for the second's.
template <int D>
struct Lds8 {
    static constexpr int kKRow = 2 * D + 16;
    static constexpr int kKBlock = kBlk * kKRow + 64;
    static constexpr int kK = 4 * kKBlock;
    static constexpr int kVRow = 2 * 64 + 16;
    static constexpr int kV = D * kVRow;
};

template <class T, class C, int D>
__global__ __launch_bounds__(256, 2) void attn8_prefill_kernel(const Prefill8Args g) {
    typedef typename T::elem E;
    typedef typename T::vec8 vec8;
    typedef E vec4 __attribute__((ext_vector_type(4)));
    typedef Lds8<D> L;
    constexpr int kX = D / 32, kT = D / 16, kU = D / 64;      // steps, dim tiles, 16-byte units a thread stages
    __shared__ __attribute__((aligned(16))) char k_lds[2][L::kK];
    __shared__ __attribute__((aligned(16))) char v_lds[2][L::kV];

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15;
    const int c = lane >> 4;
    // Consecutive workgroups go to the eight XCDs in turn: the low three bits pick the (sequence, kv head) residue,
    // so that all row tiles and splits of a pair share one L2.  Row tiles with most keys come first.
    const int Hkv = g.pool.num_kv_heads;
    const int pairs = Hkv * g.batch.num_prefill_seqs;
    const int pairs_x = (pairs + 7) >> 3;
    const int slot = (int)(blockIdx.x >> 3);
    const int job = slot / pairs_x;
    const int pair = (slot - job * pairs_x) * 8 + (int)(blockIdx.x & 7);
    if (pair >= pairs) return;
    const int rank = job / g.max_splits;
    const int split = job - rank * g.max_splits;
    const int kvh = pair % Hkv;
    const int b = pair / Hkv;

    const int G = g.group;
    const int Hq = Hkv * G;
    const int64_t start = g.batch.prefill_start_locs[b];
    const int len = chunk_rows(chunks_of(g.batch), b, start);
    const int rows = len * G;
    const int tiles = (rows + kRows - 1) / kRows;             // of this chunk
    if (rank >= tiles) return;
    const int row0 = (tiles - 1 - rank) * kRows;
    const int64_t seq = g.batch.seq_ids[b];
    const bool has_row = seq >= 0 && seq < g.batch.table_rows;
    const int64_t prefix = g.batch.prefix_lens ? max(g.batch.prefix_lens[b], 0) : 0;
    const int64_t room = has_row ? g.batch.max_blocks_per_seq * kBlk : 0;   // positions the table row can hold
    const int last_pos = (min(row0 + kRows, rows) - 1) / G;   // of the workgroup's rows, within the chunk
    const int kv_len = (int)min(prefix + last_pos + 1, room);
    const int nblk = (kv_len + kBlk - 1) / kBlk;
    const int num_tiles = (kv_len + 63) >> 6;
    const int tile_begin = min(split * g.tiles_per_split, num_tiles);
    const int tile_end = split == g.max_splits - 1 ? num_tiles : min(tile_begin + g.tiles_per_split, num_tiles);
    const int32_t* table = g.batch.block_table + (has_row ? seq * g.batch.max_blocks_per_seq : 0);
    const int num_blocks = (int)g.pool.num_blocks;

    // this wave's rows and Q^T: lane (row n, group c) holds dims 32 x + 8 c .. + 8 for step x
    const int r0 = row0 + wave * 16 * kCols;
    vec8 qb[kCols][kX];
    int last_key[kCols];                                      // a row sees keys 0 .. its own position
#pragma unroll
    for (int u = 0; u < kCols; ++u) {
        const int r = r0 + 16 * u + n;
        const int t = r / G;
        const E* qrow = (const E*)g.q + (start + t) * g.q_stride + ((int64_t)kvh * G + (r - t * G)) * D;
        last_key[u] = r < rows ? (int)min(prefix + t, room - 1) : -1;
#pragma unroll
        for (int x = 0; x < kX; ++x) {
            if (r < rows) qb[u][x] = *(const vec8*)(qrow + 32 * x + 8 * c);
            else qb[u][x] = (vec8)(E)0.f;
        }
    }
    const int wave_first = r0 < rows ? (int)min(prefix + r0 / G, room - 1) : -1;                      // first row's last key
    const int wave_last = r0 < rows ? (int)min(prefix + (min(r0 + 16 * kCols, rows) - 1) / G, room - 1) : -1;

    float4v acc[kCols][kT];
    float m_run[kCols], l_run[kCols];
#pragma unroll
    for (int u = 0; u < kCols; ++u) {
        m_run[u] = kFar;
        l_run[u] = 0.f;
#pragma unroll
        for (int t = 0; t < kT; ++t) acc[u][t] = (float4v){0.f, 0.f, 0.f, 0.f};
    }

    const int64_t block_bytes = block_bytes8(g.pool);
    const int64_t slab = slab_offset8(g.pool, g.layer, kvh);
    const uint8_t* k_base = (const uint8_t*)g.pool.k + slab;
    const uint8_t* v_base = (const uint8_t*)g.pool.v + slab;
    const uint16_t* scales = scale_row8(g.pool, g.layer, kvh);

    // ---- staging: a tile's slabs are 4 D units of 16 bytes each for K and V; unit w belongs to block w / D ----------
    auto id_of = [&](int blk) {
        const int pid = blk < nblk ? table[blk] : -1;
        return pid >= 0 && pid < num_blocks ? pid : -1;
    };
    uint4v kreg[kU], vreg[kU];
    unsigned ereg[kU];                                        // exponents of the staged units' blocks
    int st_pid[kU];                                           // their ids, one tile ahead
    int my_pid, my_pid_next;                                  // ids of block c of the current / staged tile
    unsigned my_ex, my_ex_next;
    auto load_ids = [&](int tile) {
#pragma unroll
        for (int u = 0; u < kU; ++u) st_pid[u] = id_of(4 * tile + (tid + 256 * u) / D);
        my_pid_next = id_of(4 * tile + c);
    };
    auto fetch = [&]() {
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int64_t at = (int64_t)max(st_pid[u], 0) * block_bytes + 16 * ((tid + 256 * u) % D);
            kreg[u] = *(const uint4v*)(k_base + at);
            vreg[u] = *(const uint4v*)(v_base + at);
            ereg[u] = st_pid[u] >= 0 ? scales[st_pid[u]] : 0x7f7fu;
        }
        my_ex_next = my_pid_next >= 0 ? scales[my_pid_next] : 0x7f7fu;
    };
    auto stage = [&](int buf, int tile) {
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int w = tid + 256 * u;
            const int blk = w / D, o = w % D;
            // K: 16 dims of a key
            char* kd = k_lds[buf] + blk * L::kKBlock + (o * 16 / D) * L::kKRow + (o * 16 % D) * 2;
            *(vec8*)kd = C::raw(T{}, kreg[u][0], kreg[u][1]);
            *(vec8*)(kd + 16) = C::raw(T{}, kreg[u][2], kreg[u][3]);
            // V: 16 keys of a dim; codes behind the last key, and of a block that is not there, count as 0
            const int valid = st_pid[u] >= 0 ? min(max(kv_len - (4 * tile + blk) * kBlk, 0), kBlk) : 0;
            unsigned keep[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int in = min(max(valid - 4 * j, 0), 4);
                keep[j] = in >= 4 ? ~0u : (1u << (8 * in)) - 1u;
            }
            char* vd = v_lds[buf] + o * L::kVRow + blk * 32;
            *(vec8*)vd = v_operand<T, C>(vreg[u][0] & keep[0], vreg[u][1] & keep[1], ereg[u] >> 8);
            *(vec8*)(vd + 16) = v_operand<T, C>(vreg[u][2] & keep[2], vreg[u][3] & keep[3], ereg[u] >> 8);
        }
    };

    const int k_rd = (n >> 2) * L::kKBlock + (n & 3) * L::kKRow + 16 * c;      // + 4 j rows, + 64 x bytes
    const int v_rd = n * L::kVRow + 32 * c;                                    // + 16 t rows, + 16 z bytes

    auto consume = [&](int buf, int tile) {
        const bool here = my_pid >= 0;
        const bool careful = __ballot(!here) != 0 || tile * 64 + 63 > wave_first;      // the same for the wave
        const float f = g.scale2 * pow2_of(my_ex & 0xffu);
        const int key0 = (4 * tile + c) * kBlk;
        float4v st[kCols][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int u = 0; u < kCols; ++u) st[u][j] = (float4v){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int x = 0; x < kX; ++x) {
                const vec8 ka = *(const vec8*)(k_lds[buf] + k_rd + 4 * j * L::kKRow + 64 * x);
#pragma unroll
                for (int u = 0; u < kCols; ++u) st[u][j] = T::mfma(ka, qb[u][x], st[u][j]);
            }
        }
        vec8 pb[kCols][2];
#pragma unroll
        for (int u = 0; u < kCols; ++u) {
            float s[16], mx = kFar;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[e] = st[u][e >> 2][e & 3] * f;
                if (careful && !(here && key0 + e <= last_key[u])) s[e] = kFar;
                mx = fmaxf(mx, s[e]);
            }
            if (__ballot(mx - m_run[u] > kLazyP) != 0) {
                const float m_new = fmaxf(m_run[u], max_over_quarters(mx));
                const float alpha = __builtin_amdgcn_exp2f(m_run[u] - m_new);
                l_run[u] *= alpha;
#pragma unroll
                for (int t = 0; t < kT; ++t) acc[u][t] *= alpha;
                m_run[u] = m_new;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[e] = __builtin_amdgcn_exp2f(s[e] - m_run[u]);
                if (careful && !(here && key0 + e <= last_key[u])) s[e] = 0.f;
            }
#pragma unroll
            for (int e = 0; e < 16; e += 4) l_run[u] += (s[e] + s[e + 1]) + (s[e + 2] + s[e + 3]);
            if constexpr (!T::kScaleV) {
                const float fv = pow2_of(my_ex >> 8);
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] *= fv;
            }
#pragma unroll
            for (int z = 0; z < 2; ++z)
                pb[u][z] = (vec8){(E)s[8 * z], (E)s[8 * z + 1], (E)s[8 * z + 2], (E)s[8 * z + 3],
                                  (E)s[8 * z + 4], (E)s[8 * z + 5], (E)s[8 * z + 6], (E)s[8 * z + 7]};
        }
#pragma unroll
        for (int t = 0; t < kT; ++t)
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                const vec8 va = *(const vec8*)(v_lds[buf] + v_rd + 16 * t * L::kVRow + 16 * z);
#pragma unroll
                for (int u = 0; u < kCols; ++u) acc[u][t] = T::mfma(va, pb[u][z], acc[u][t]);
            }
    };

    if (tile_begin < tile_end) {
        load_ids(tile_begin);
        fetch();
        stage(0, tile_begin);
        my_pid = my_pid_next;
        my_ex = my_ex_next;
        load_ids(tile_begin + 1);                             // past the end: no block
    }
    for (int tile = tile_begin; tile < tile_end; ++tile) {
        const int buf = (tile - tile_begin) & 1;
        const bool more = tile + 1 < tile_end;
        __syncthreads();                                      // this tile is staged; the other buffer is free
        if (more) fetch();
        if (tile * 64 <= wave_last) consume(buf, tile);
        if (more) {
            stage(buf ^ 1, tile + 1);
            my_pid = my_pid_next;
            my_ex = my_ex_next;
            load_ids(tile + 2);
        }
    }

    // ---- output: a lane holds, of row n of a column tile, dims 16 t + 4 c .. + 4 -------------------------------------
#pragma unroll
    for (int u = 0; u < kCols; ++u) {
        const float l = sum_over_quarters(l_run[u]);
        const int r = r0 + 16 * u + n;
        if (r >= rows) continue;
        const float inv = l == 0.f ? 0.f : 1.f / l;           // a row with nothing to attend to: zeros
        const int t = r / G;
        const int64_t head = (int64_t)kvh * G + (r - t * G);
        if (g.max_splits == 1) {
            E* orow = (E*)g.o + (start + t) * g.o_stride + head * D;
#pragma unroll
            for (int d = 0; d < kT; ++d)
                *(vec4*)(orow + 16 * d + 4 * c) = (vec4){(E)(acc[u][d][0] * inv), (E)(acc[u][d][1] * inv),
                                                         (E)(acc[u][d][2] * inv), (E)(acc[u][d][3] * inv)};
        } else {
            const int64_t at = ((start + t) * Hq + head) * g.max_splits + split;
#pragma unroll
            for (int d = 0; d < kT; ++d) *(float4v*)(g.mid_o + at * D + 16 * d + 4 * c) = acc[u][d] * inv;
            if (c == 0) g.mid_lse[at] = l == 0.f ? kFar : __builtin_amdgcn_logf(l) + m_run[u];
        }
    }
}

template <class T, class C>
static void launch_prefill8(int head_dim, dim3 grid, hipStream_t s, const Prefill8Args& g) {
    if (head_dim == 128) hipLaunchKernelGGL((attn8_prefill_kernel<T, C, 128>), grid, dim3(256), 0, s, g);
    else hipLaunchKernelGGL((attn8_prefill_kernel<T, C, 64>), grid, dim3(256), 0, s, g);
}

}  // namespace mkv

extern "C" int mkv_attn8_prefill(const mkv_pool8* pool, const mkv_batch* batch, int32_t dtype, const void* q, void* o,
                                 int64_t q_stride, int64_t o_stride, int32_t num_q_heads, float softmax_scale,
                                 int32_t layer, int32_t tokens_per_split, int32_t max_splits, void* mid_o,
                                 void* mid_lse, void* stream) {
    int rc = mkv::check_pool8(pool);
    if (rc) return rc;
    rc = mkv::check_batch8(batch);
    if (rc) return rc;
    MKV_REQUIRE(dtype == MKV_F16 || dtype == MKV_BF16, "dtype %d is neither MKV_F16 nor MKV_BF16", dtype);
    MKV_REQUIRE(layer >= 0 && layer < pool->num_layers, "layer %d outside [0, %d)", layer, pool->num_layers);
    if (batch->num_prefill_seqs == 0 || batch->max_prefill_len == 0) return MKV_OK;
    MKV_REQUIRE(q && o, "NULL argument");
    MKV_REQUIRE(num_q_heads > 0 && num_q_heads % pool->num_kv_heads == 0 && num_q_heads / pool->num_kv_heads <= 16,
                "num_q_heads %d must be 1 to 16 times num_kv_heads %d", num_q_heads, pool->num_kv_heads);
    MKV_REQUIRE(tokens_per_split > 0 && tokens_per_split % 64 == 0, "tokens_per_split %d must be a positive multiple of 64",
                tokens_per_split);
    MKV_REQUIRE(max_splits >= 1, "max_splits must be >= 1");
    MKV_REQUIRE(max_splits == 1 || (mid_o && mid_lse), "scratch buffers are NULL");
    MKV_REQUIRE(((uintptr_t)mid_o & 15) == 0 && ((uintptr_t)mid_lse & 3) == 0, "mid_o must be 16-byte aligned, mid_lse 4-byte aligned");
    MKV_REQUIRE((((uintptr_t)q | (uintptr_t)o) & 15) == 0 && ((q_stride | o_stride) & 7) == 0, "q and o rows must be 16-byte aligned");
    const int group = num_q_heads / pool->num_kv_heads;
    MKV_REQUIRE((int64_t)batch->max_prefill_len * num_q_heads <= 0x7fffff00 && batch->num_prefill_seqs <= 65535,
                "too many rows in one call");
    mkv::Prefill8Args g = {};
    g.pool = *pool;
    g.batch = *batch;
    g.q = (const char*)q;
    g.o = (char*)o;
    g.q_stride = q_stride;
    g.o_stride = o_stride;
    g.mid_o = (float*)mid_o;
    g.mid_lse = (float*)mid_lse;
    g.group = group;
    g.layer = layer;
    g.tiles_per_split = tokens_per_split / 64;
    g.max_splits = max_splits;
    g.num_row_tiles = mkv::cdiv((int64_t)batch->max_prefill_len * group, mkv::kRows);
    g.scale2 = softmax_scale * mkv::kLog2E;
    const int64_t pairs_x = ((int64_t)pool->num_kv_heads * batch->num_prefill_seqs + 7) / 8;
    const int64_t cells = pairs_x * 8 * g.num_row_tiles * max_splits;
    MKV_REQUIRE(cells <= 0x7fffffff, "too many rows in one call");
    const dim3 grid((unsigned)cells);
    hipStream_t s = (hipStream_t)stream;
    if (dtype == MKV_F16) {
        if (pool->kind == MKV_KV8_E4M3) mkv::launch_prefill8<mkv::F16, mkv::E4M3>(pool->head_dim, grid, s, g);
        else mkv::launch_prefill8<mkv::F16, mkv::Int8>(pool->head_dim, grid, s, g);
    } else {
        if (pool->kind == MKV_KV8_E4M3) mkv::launch_prefill8<mkv::BF16, mkv::E4M3>(pool->head_dim, grid, s, g);
        else mkv::launch_prefill8<mkv::BF16, mkv::Int8>(pool->head_dim, grid, s, g);
    }
    MKV_HIP(hipGetLastError());
    if (max_splits > 1)
        return mkv::launch_merge8(dtype, pool->head_dim, (const float*)mid_o, (const float*)mid_lse, o, o_stride,
                                  num_q_heads, dim3((unsigned)(batch->max_prefill_len * num_q_heads), (unsigned)batch->num_prefill_seqs),
                                  max_splits, mkv::chunks_of(*batch), s);
    return MKV_OK;
}
