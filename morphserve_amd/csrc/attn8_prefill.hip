// Chunked prefill attention over the 8-bit paged cache.
//
// The rows of one kv head -- chunk positions times the q heads that share it, position-major -- are cut into tiles of 64
// to 256, one workgroup of four or eight waves each; a wave owns one or two 16-row column tiles.  Keys come 64 at a time
// (four blocks): their codes are converted once, on the way into LDS, and every wave reads the converted tile from there,
//
//   S^T[key, row] = K . Q^T        v_mfma_f32_16x16x32
//   O^T[dim, row] += V^T . P^T     v_mfma_f32_16x16x32
//
// while the next tile's codes are on their way from memory and the tile after that lends its block ids.  As in the
// decode kernel the keys are numbered so that lane group c scores block c in order, which makes K's scale one factor
// per lane and the scores, exponentiated, the operand of the second product.  V arrives transposed from the cache,
// so that both products read LDS in rows.  Where few rows meet many keys, the keys are cut into splits.
//
// Bound: the matrix cores where rows are many -- 2048 tokens of 32 q heads after 8192 cached ones take 365 to 380 us, 815 to
// 850 TFLOP/s of the two products, whole prompts of 8192 tokens 605 to 650 us (830 to 900) -- less what the softmax leaves
// them idle: the two waves of a SIMD alternate between products and exponentials.  A wave reads its operands from LDS four
// ahead of the products, during the last of K's already V's first, and nothing is loaded under a condition, since waits where
// two paths meet take the worse one.
#include <type_traits>

#include "kv8.h"

namespace mkv {

static constexpr int kAhead = 4;              // operands requested from LDS ahead of their products, K's and then V's
static constexpr float kLazyP = 8.f;

// The larger of two numbers as the median of them and infinity: one instruction, where fmaxf first makes its operands
// canonical -- and one that the compiler knows to read a matrix product's result.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_amdgcn_fmed3f(a, b, __builtin_inff()); }

struct Prefill8Args {
    mkv_pool8 pool;
    mkv_batch batch;
    const char* q;
    char* o;
    int64_t q_stride, o_stride;               // elements
    float *mid_o, *mid_lse;
    int32_t group, layer, tiles_per_split, max_splits;
    int32_t sorted, key_tiles;                // row tiles by length; about the most key tiles that one sees
    int32_t paired;                           // a workgroup takes a chunk's i-th longest row tile and its i-th shortest
    float scale2;
};

// LDS rows: K has one row a key, V one a head dim.  A 16-byte read of a wave is served in groups of sixteen lanes, eight
// consecutive ones and eight of the opposite half of the next lane group, measured with feeding products: 5.1 cycles a
// read without conflicts and 8.0 with any.  Row distances of two 16-byte slots modulo sixteen (ten serve as well),
// eight between blocks, with the lane group one slot further, keep every such group on sixteen different slots:
// slot 2 n + c for K (10 n + c for the shorter rows of 64 dims) and 10 n + c for V.
template <int D>
struct Lds8 {
    static constexpr int kKRow = D == 64 ? 160 : 288;
    static constexpr int kKBlock = kBlk * kKRow + 128;
    static constexpr int kK = 4 * kKBlock;
    static constexpr int kVRow = 160;            // keys 0 .. 7 of the four blocks, then keys 8 .. 15
    static constexpr int kV = D * kVRow;
};

// A row does not see every key of its last tiles, and a NaN there must not reach it through a weight of 0: where such tiles
// are staged, V's NaN are taken out and noted, a bit for each key and dim, and put into the rows that see their keys.  Costs
// 2 % on long prompts (e4m3; int8 has no NaN).
template <int D>
struct NaN8 {
    uint64_t keys[2][D];                      // of the staged tiles: dim's keys 0 .. 63 with a NaN
    union {
        uint8_t wave[2][8];                   // has the wave met one among the units that it staged
        uint64_t any[2];
    };
};

// Which row tile is the job-th longest of the batch?  A launch that does not fit the chip at once is as long as its last
// workgroups make it, so the row tiles with most keys go first, whatever chunk they belong to.  A chunk's tiles with at
// least t key tiles are its last ones and their number has a closed form; the t that the job falls on is found by
// bisection, a lane counting for a chunk (or for every 64th).  False: there are not so many row tiles.
__device__ __forceinline__ int wave_sum(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);      // row_shr 1, 2, 4, 8: sums within rows of 16
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);     // row 0's to row 1, row 2's to row 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);     // row 1's to rows 2 and 3
    return __builtin_amdgcn_readlane(x, 63);
}

struct ChunkTiles {
    int rows, tiles, group, per;      // rows and row tiles of a chunk, rows per position, rows per tile
    int prefix;
    // row tiles that see at least t key tiles: those with a position p, prefix + p + 1 > 64 (t - 1)
    __device__ __forceinline__ int at_least(int t) const {
        const int64_t p = max((int64_t)64 * (t - 1) - prefix, (int64_t)0) * group;
        return p >= rows ? 0 : tiles - (int)(p / per);
    }
};

__device__ __forceinline__ ChunkTiles chunk_tiles(const Prefill8Args& g, int per, int b) {
    ChunkTiles c = {0, 0, g.group, per, 0};
    if (b < g.batch.num_prefill_seqs) {
        c.rows = chunk_rows(chunks_of(g.batch), b, g.batch.prefill_start_locs[b]) * g.group;
        c.tiles = (c.rows + per - 1) / per;
        c.prefix = g.batch.prefix_lens ? max(g.batch.prefix_lens[b], 0) : 0;
    }
    return c;
}

__device__ __forceinline__ bool nth_longest(const Prefill8Args& g, int per, int job, int lane, int& b, int& rank) {
    const int seqs = g.batch.num_prefill_seqs;
    const ChunkTiles mine = chunk_tiles(g, per, lane);
    auto count = [&](int t) {
        int n = mine.at_least(t);
        for (int s = lane + 64; s < seqs; s += 64) n += chunk_tiles(g, per, s).at_least(t);
        return wave_sum(n);
    };
    if (job >= count(0)) return false;
    int lo = 0, hi = g.key_tiles + 1;                         // count(lo) > job >= count(hi)
    while (count(hi) > job) hi *= 2;                          // the host's bound may be too low
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (count(mid) > job) lo = mid;
        else hi = mid;
    }
    int left = job - count(hi);                               // among the tiles with exactly lo key tiles, by chunk
    for (int s0 = 0; s0 < seqs; s0 += 64) {
        const ChunkTiles c = s0 ? chunk_tiles(g, per, s0 + lane) : mine;
        const int longer = c.at_least(hi), own = c.at_least(lo) - longer;
        int upto = own;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const int x = __shfl_up(upto, s);
            if (lane >= s) upto += x;
        }
        const uint64_t past = __ballot(upto > left);
        if (past) {
            const int at = __ffsll((unsigned long long)past) - 1;
            b = s0 + at;
            rank = __shfl(longer, at) + left - (__shfl(upto, at) - __shfl(own, at));
            b = __builtin_amdgcn_readfirstlane(b);
            rank = __builtin_amdgcn_readfirstlane(rank);
            return true;
        }
        left -= __shfl(upto, 63);
    }
    return false;
}

// A workgroup's row tile against its range of the keys: rows row0 .. of the `rows` of chunk b, starting at batch row `start`;
// then, where `second` is not -1, the tile that begins there: an earlier one, with the whole keys as its range.
template <class T, class C, int D, int WAVES, int COLS>
__device__ __forceinline__ void attend_tile(const Prefill8Args& g, char (*k_lds)[Lds8<D>::kK], char (*v_lds)[Lds8<D>::kV], NaN8<D>& nans, int b,
                                            int split, int kvh, int64_t start, int rows, int row0, int second) {
    typedef typename T::elem E;
    typedef typename T::vec8 vec8;
    typedef E vec4 __attribute__((ext_vector_type(4)));
    typedef Lds8<D> L;
    constexpr int kThreads = 64 * WAVES;
    constexpr int kRows = 16 * COLS * WAVES;                  // rows of the tile
    constexpr int kX = D / 32, kT = D / 16;                   // steps of the first product, dim tiles of the second
    constexpr int kUnits = 4 * D;                             // 16-byte units of a tile's K (and V) slabs
    static_assert(kUnits % kThreads == 0, "every thread takes as many units");
    constexpr int kU = kUnits / kThreads;
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15;
    const int c = lane >> 4;
    const int G = g.group;
    const int Hq = g.pool.num_kv_heads * G;
    const int64_t seq = g.batch.seq_ids[b];
    const bool has_row = seq >= 0 && seq < g.batch.table_rows;
    const int64_t prefix = g.batch.prefix_lens ? max(g.batch.prefix_lens[b], 0) : 0;
    const int64_t room = has_row ? g.batch.max_blocks_per_seq * kBlk : 0;   // positions the table row can hold
    const int last_pos = (min(row0 + kRows, rows) - 1) / G;   // of the workgroup's rows, within the chunk
    const int kv_len = (int)min(prefix + last_pos + 1, room);
    const int nblk = (kv_len + kBlk - 1) / kBlk;
    const int num_tiles = (kv_len + 63) >> 6;
    const int tile_begin = min(split * g.tiles_per_split, num_tiles);
    int tile_end = split == g.max_splits - 1 ? num_tiles : min(tile_begin + g.tiles_per_split, num_tiles);
    const int32_t* table = g.batch.block_table + (has_row ? seq * g.batch.max_blocks_per_seq : 0);
    const int num_blocks = (int)g.pool.num_blocks;

    // this wave's rows and Q^T: lane (row n, group c) holds dims 32 x + 8 c .. + 8 for step x
    vec8 qb[COLS][kX];
    int r0, last_key[COLS], wave_last;                       // a row sees keys 0 .. its own position
    auto take_rows = [&](int from) {
        r0 = from + wave * 16 * COLS;
#pragma unroll
        for (int u = 0; u < COLS; ++u) {
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
        wave_last = r0 < rows ? (int)min(prefix + (min(r0 + 16 * COLS, rows) - 1) / G, room - 1) : -1;
    };
    take_rows(row0);

    // Row sums come out of the matrix cores too: a V^T row of ones makes every register of lsum the row's sum of
    // the rounded probabilities, the ones the numerator is built from.
    float4v acc[COLS][kT], lsum[COLS];
    float m_run[COLS];
    const vec8 ones = (vec8)(E)1.f;
    auto clear = [&] {
#pragma unroll
        for (int u = 0; u < COLS; ++u) {
            m_run[u] = kFar;
            lsum[u] = (float4v){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < kT; ++t) acc[u][t] = (float4v){0.f, 0.f, 0.f, 0.f};
        }
    };
    clear();

    const int64_t block_bytes = block_bytes8(g.pool);
    const int64_t slab = slab_offset8(g.pool, g.layer, kvh);
    const uint8_t* k_base = (const uint8_t*)g.pool.k + slab;
    const uint8_t* v_base = (const uint8_t*)g.pool.v + slab;
    const uint16_t* scales = scale_row8(g.pool, g.layer, kvh);

    // ---- staging: unit w of a tile's slabs belongs to block w / D; a thread takes units tid, tid + kThreads, ... ---------
    // below kUnits as it is; with the bound in sight the compiler's order of the loop is 2 % faster for few rows (52.3 us, 53.3)
    auto unit = [&](int u) { return (tid + kThreads * u) % kUnits; };
    // Ids are kept as the table holds them and looked at when they are used, a tile later: loads complete in order, and a
    // glance at an id that was just asked for would wait for the codes asked for before it.
    auto ask_id = [&](int blk) { return table[min(blk, nblk - 1)]; };
    auto known_id = [&](int blk, int id) { return blk < nblk && id >= 0 && id < num_blocks ? id : -1; };
    uint4v kreg[kU], vreg[kU];
    int valid[kU];                                            // keys of the units' blocks that count
    unsigned ereg[kU];                                        // the blocks' exponents
    int ids[kU], id_c;                                        // of the tile after the fetched one: units' blocks, block c
    bool here = false, here_next = false;                     // block c of the current / fetched tile
    unsigned ex = 0, ex_next = 0;
    auto ask_ids = [&](int tile) {
#pragma unroll
        for (int u = 0; u < kU; ++u) ids[u] = ask_id(4 * tile + unit(u) / D);
        id_c = ask_id(4 * tile + c);
    };
    // behind a row tile's last key tile comes the second one's first (or, of no use, the first again)
    auto after = [&](int tile) { return tile + 1 < tile_end ? tile + 1 : tile_begin; };
    // requests the codes of `tile` and the ids of the one after it
    auto fetch = [&](int tile) {
        const int own = known_id(4 * tile + c, id_c);
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int blk = 4 * tile + unit(u) / D;
            const int id = known_id(blk, ids[u]);
            const int64_t at = (int64_t)max(id, 0) * block_bytes + 16 * (unit(u) % D);
            kreg[u] = *(const uint4v*)(k_base + at);
            vreg[u] = *(const uint4v*)(v_base + at);
            ereg[u] = scales[max(id, 0)];
            valid[u] = id >= 0 ? min(max(kv_len - blk * kBlk, 0), kBlk) : 0;
        }
        ex_next = scales[max(own, 0)];
        here_next = own >= 0;
        ask_ids(after(tile));
    };
    // The tiles that every row of a row tile sees whole end here.
    auto whole_until = [&](int from, int end) { return max(tile_begin, min(end, (int)((min(prefix + from / G, room - 1) + 1) >> 6))); };
    int full_end = whole_until(row0, tile_end);
    constexpr bool kOverflows = !C::kHasNaN && std::is_same<T, F16>::value;
    auto mask_of = [](int keys, unsigned (&keep)[4]) {        // the bytes of a block's first keys
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int in = min(max(keys - 4 * j, 0), 4);
            keep[j] = in >= 4 ? ~0u : (1u << (8 * in)) - 1u;
        }
    };
    auto stage = [&](int buf, bool cut) {                     // cut: some row does not see the whole tile
        unsigned found = 0;
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int w = unit(u);
            const int blk = w / D, o = w % D;
            // K: 16 dims of a key; a block that is not there is one of zeros
            const unsigned there = valid[u] > 0 ? ~0u : 0u;
            char* kd = k_lds[buf] + blk * L::kKBlock + (o * 16 / D) * L::kKRow + (o * 16 % D) * 2;
            *(vec8*)kd = C::raw(T{}, kreg[u][0] & there, kreg[u][1] & there);
            *(vec8*)(kd + 16) = C::raw(T{}, kreg[u][2] & there, kreg[u][3] & there);
            // V: 16 keys of a dim; codes behind the last key have no weight, but a NaN among them would count
            unsigned keep[4] = {~0u, ~0u, ~0u, ~0u};
            if (C::kHasNaN) mask_of(valid[u], keep);
            if (C::kHasNaN && cut) {
                unsigned keys = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    // a byte's top bit where its code is a NaN: all seven bits below are set
                    const unsigned at = (((vreg[u][j] & keep[j] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
                    keep[j] &= ~(at * 0xffu);
                    keys |= ((at * 0x01020408u) >> 24 & 0xfu) << (4 * j);
                }
                ((uint16_t*)&nans.keys[buf][o])[blk] = (uint16_t)keys;
                found |= keys;
            }
            const unsigned ev = valid[u] > 0 ? ereg[u] >> 8 : 127u;
            char* vd = v_lds[buf] + o * L::kVRow + blk * 16;
            *(vec8*)vd = C::scaled(T{}, vreg[u][0] & keep[0], vreg[u][1] & keep[1], ev);
            *(vec8*)(vd + 64) = C::scaled(T{}, vreg[u][2] & keep[2], vreg[u][3] & keep[3], ev);
        }
        // Int8's -128, which the append does not write but which may lie behind the last key, overflows at fp16's largest scale
        // (bf16's would be beyond what the sums hold): blocks that end inside are written once more without what lies there.
        // Apart from the loop above, where masks cost int8 chunks 2 to 10 %; so, eight prompts of 512 tokens of 32 heads take
        // 37.5 us instead of 36.5, and four ragged chunks over 1000 to 8192 tokens the same 525.
        if (kOverflows) {
            int least = valid[0];
#pragma unroll
            for (int u = 1; u < kU; ++u) least = min(least, valid[u]);
            if (__ballot(least < kBlk) != 0) {
#pragma unroll
                for (int u = 0; u < kU; ++u) {
                    unsigned keep[4];
                    mask_of(valid[u], keep);
                    const unsigned ev = valid[u] > 0 ? ereg[u] >> 8 : 127u;
                    char* vd = v_lds[buf] + unit(u) % D * L::kVRow + unit(u) / D * 16;
                    *(vec8*)vd = C::scaled(T{}, vreg[u][0] & keep[0], vreg[u][1] & keep[1], ev);
                    *(vec8*)(vd + 64) = C::scaled(T{}, vreg[u][2] & keep[2], vreg[u][3] & keep[3], ev);
                }
            }
        }
        if (C::kHasNaN && cut) {
            const bool some = __ballot(found != 0) != 0;
            nans.wave[buf][wave] = some;
        }
    };

    const int k_rd = (n >> 2) * L::kKBlock + (n & 3) * L::kKRow + 16 * c;      // + 4 j rows, + 64 x bytes
    const int v_rd = n * L::kVRow + 16 * c;                                    // + 16 t rows, + 64 z bytes

    // One tile against the wave's rows.  MASKED: a row may not see all of its keys.
    auto consume = [&](auto masked_tag, int buf, int tile) {
        constexpr bool MASKED = decltype(masked_tag)::value;
        const char* kl = k_lds[buf] + k_rd;
        const char* vl = v_lds[buf] + v_rd;
        // the matrix phases run at raised priority: the SIMD's other wave fills the gaps with its softmax
        __builtin_amdgcn_s_setprio(2);
        float4v st[COLS][4];
        constexpr int kNK = 4 * kX;
        vec8 ka[kAhead];
        auto k_operand = [&](int e) { return *(const vec8*)(kl + 4 * (e / kX) * L::kKRow + 64 * (e % kX)); };
        auto v_operand = [&](int e) { return *(const vec8*)(vl + 16 * (e >> 1) * L::kVRow + 64 * (e & 1)); };
#pragma unroll
        for (int e = 0; e < kAhead; ++e) ka[e] = k_operand(e);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = 0; e < kNK; ++e) {
            const int j = e / kX, x = e % kX;
#pragma unroll
            for (int u = 0; u < COLS; ++u)
                st[u][j] = T::mfma(ka[e % kAhead], qb[u][x], x ? st[u][j] : (float4v){0.f, 0.f, 0.f, 0.f});
            ka[e % kAhead] = e + kAhead < kNK ? k_operand(e + kAhead) : v_operand(e + kAhead - kNK);
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(0);
        const float f = g.scale2 * pow2_of(here ? ex & 0xffu : 127u);    // > 0: keeps the order of the scores
        vec8 pb[COLS][2];
#pragma unroll
        for (int u = 0; u < COLS; ++u) {
            const int seen = MASKED ? (here ? last_key[u] - (4 * tile + c) * kBlk + 1 : 0) : kBlk;   // of the lane's sixteen keys
            float s[16], mx;
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = st[u][e >> 2][e & 3];
            if (MASKED) {
                mx = kFar;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    s[e] = e < seen ? s[e] * f : 2 * kFar;            // so far below that it weighs 0 whatever the maximum
                    mx = fmaxf(mx, s[e]);
                }
            } else {
                mx = s[0];
#pragma unroll
                for (int e = 1; e < 16; ++e) mx = larger(mx, s[e]);
                mx *= f;
                mx = here ? mx : kFar;
            }
            if (__ballot(mx - m_run[u] > kLazyP) != 0) {
                const float m_new = fmaxf(m_run[u], max_over_quarters(mx));
                const float alpha = __builtin_amdgcn_exp2f(m_run[u] - m_new);
                lsum[u] *= alpha;
#pragma unroll
                for (int t = 0; t < kT; ++t) acc[u][t] *= alpha;
                m_run[u] = m_new;
            }
            const float off = here ? -m_run[u] : kFar;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                if (MASKED) s[e] = __builtin_amdgcn_exp2f(s[e] - m_run[u]);
                else s[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], f, off));
            }
#pragma unroll
            for (int z = 0; z < 2; ++z)
                pb[u][z] = (vec8){(E)s[8 * z], (E)s[8 * z + 1], (E)s[8 * z + 2], (E)s[8 * z + 3],
                                  (E)s[8 * z + 4], (E)s[8 * z + 5], (E)s[8 * z + 6], (E)s[8 * z + 7]};
        }
        __builtin_amdgcn_s_setprio(2);
#pragma unroll
        for (int u = 0; u < COLS; ++u) {
            lsum[u] = T::mfma(ones, pb[u][0], lsum[u]);
            lsum[u] = T::mfma(ones, pb[u][1], lsum[u]);
        }
#pragma unroll
        for (int e = 0; e < 2 * kT; ++e) {
#pragma unroll
            for (int u = 0; u < COLS; ++u) acc[u][e >> 1] = T::mfma(ka[e % kAhead], pb[u][e & 1], acc[u][e >> 1]);
            if (e + kAhead < 2 * kT)
                ka[e % kAhead] = v_operand(e + kAhead);
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        const auto any = WAVES == 8 ? nans.any[buf] : (uint64_t)*(const uint32_t*)nans.wave[buf];
        if (C::kHasNaN && MASKED && __ballot(any != 0) != 0) {
#pragma unroll
            for (int u = 0; u < COLS; ++u) {
                const int upto = last_key[u] - 64 * tile + 1;
                const uint64_t seen = upto <= 0 ? 0 : upto >= 64 ? ~0ull : (1ull << upto) - 1;
#pragma unroll
                for (int t = 0; t < kT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {                    // a NaN or 0 is added
                        const uint64_t hit = nans.keys[buf][16 * t + 4 * c + e] & seen;
                        acc[u][t][e] += __builtin_bit_cast(float, min((unsigned)hit | (unsigned)(hit >> 32), 1u) * 0x7fc00000u);
                    }
            }
        }
    };

    if (tile_begin < tile_end) {
        ask_ids(tile_begin);
        fetch(tile_begin);
        stage(0, tile_begin >= full_end);
        here = here_next;
        ex = ex_next;
    }
    int buf = 0;
    int next_full = 0;                                        // full_end of the row tile after this one
    auto iterate = [&](auto masked_tag, int from, int to) {
        for (int tile = from; tile < to; ++tile) {
            const int next = after(tile);
            __syncthreads();                                  // this tile is staged; the other buffer is free
            fetch(next);
            if (tile * 64 <= wave_last) consume(masked_tag, buf, tile);
            buf ^= 1;
            stage(buf, next >= (tile + 1 < tile_end ? full_end : next_full));
            here = here_next;
            ex = ex_next;
        }
    };
    const int second_end = second < 0 ? 0 : (int)((min(prefix + (second + kRows - 1) / G + 1, room) + 63) >> 6);
    if (second >= 0) next_full = whole_until(second, second_end);
    for (;;) {
        // The tiles that every row of the workgroup sees whole, then those that hold some row's last key.  Two loops, not two
        // bodies in one: the accumulators would be copied where the bodies meet, and the registers do not suffice for that.
        iterate(std::false_type{}, tile_begin, full_end);
        iterate(std::true_type{}, full_end, tile_end);
        const int done = r0;
        const bool more = second >= 0;
        if (more) {                                               // q is on its way while the first tile's rows are written
            take_rows(second);
            tile_end = second_end;
            full_end = next_full;
            second = -1;
        }

        // ---- output: a lane holds, of row n of a column tile, dims 16 t + 4 c .. + 4 -------------------------------------
#pragma unroll
        for (int u = 0; u < COLS; ++u) {
            const float l = lsum[u][0];
            const int r = done + 16 * u + n;
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
        if (!more) break;
        clear();
    }
}

// Two waves per SIMD at 128 head dims, by the accumulators; three at 64, of three workgroups a unit, where the softmax, as long
// for half the products, has more to hide behind: twelve ragged prompts of 64 q heads 98 us with two, 77 with three.
template <class T, class C, int D, int WAVES, int COLS>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(D == 64 ? 3 : 2, D == 64 ? 3 : 2))) void attn8_prefill_kernel(const Prefill8Args g) {
    constexpr int kRows = 16 * COLS * WAVES;                  // rows per workgroup
    __shared__ __attribute__((aligned(16))) char k_lds[2][Lds8<D>::kK];
    __shared__ __attribute__((aligned(16))) char v_lds[2][Lds8<D>::kV];
    __shared__ NaN8<D> nans;
    const int lane = threadIdx.x & 63;
    // Workgroups are numbered (row tile, split, kv head), the head fastest: consecutive ones go to the eight XCDs in
    // turn, so that with eight kv heads or a multiple a head's row tiles share one L2.
    const int Hkv = g.pool.num_kv_heads;
    const int cell = (int)(blockIdx.x / (unsigned)Hkv);
    const int kvh = (int)blockIdx.x - cell * Hkv;
    const int job = cell / g.max_splits;
    const int split = cell - job * g.max_splits;
    int b, rank;                                              // rank: the row tile, counted from the chunk's last
    if (g.sorted) {
        if (!nth_longest(g, kRows, job, lane, b, rank)) return;
    } else {
        rank = job / g.batch.num_prefill_seqs;
        b = job - rank * g.batch.num_prefill_seqs;
    }
    const int64_t start = g.batch.prefill_start_locs[b];
    const int len = chunk_rows(chunks_of(g.batch), b, start);
    const int rows = len * g.group;
    const int tiles = (rows + kRows - 1) / kRows;             // of this chunk
    if (g.paired ? 2 * rank >= tiles : rank >= tiles) return;
    const int last = tiles - 1 - rank;
    const int row0 = last * kRows;
    const int second = g.paired && rank < last ? rank * kRows : -1;      // the row tile as far from the chunk's other end
    // A tile that is at most half full: one column tile a wave, on all of them, instead of two on half.  Six chunks of 1 to
    // 16 tokens of 64 q heads over 8000 to 16000 cached ones: 70 us -> 55.
    if (COLS == 2 && second < 0 && rows - row0 <= kRows / 2)
        attend_tile<T, C, D, WAVES, 1>(g, k_lds, v_lds, nans, b, split, kvh, start, rows, row0, -1);
    else
        attend_tile<T, C, D, WAVES, COLS>(g, k_lds, v_lds, nans, b, split, kvh, start, rows, row0, second);
}

template <class T, class C, int D>
static void launch_prefill8(int shape, dim3 grid, hipStream_t s, const Prefill8Args& g) {
    if constexpr (D == 128) {
        if (shape == 256) {
            hipLaunchKernelGGL((attn8_prefill_kernel<T, C, D, 8, 2>), grid, dim3(512), 0, s, g);
            return;
        }
    }
    if (shape == 128) hipLaunchKernelGGL((attn8_prefill_kernel<T, C, D, 4, 2>), grid, dim3(256), 0, s, g);
    else hipLaunchKernelGGL((attn8_prefill_kernel<T, C, D, 4, 1>), grid, dim3(256), 0, s, g);
}

template <class T>
static void launch_prefill8(const mkv_pool8& p, int shape, dim3 grid, hipStream_t s, const Prefill8Args& g) {
    if (p.kind == MKV_KV8_E4M3 && p.head_dim == 128) launch_prefill8<T, E4M3, 128>(shape, grid, s, g);
    else if (p.kind == MKV_KV8_E4M3) launch_prefill8<T, E4M3, 64>(shape, grid, s, g);
    else if (p.head_dim == 128) launch_prefill8<T, Int8, 128>(shape, grid, s, g);
    else launch_prefill8<T, Int8, 64>(shape, grid, s, g);
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
    // tile and block numbers, those behind the last key included, are 32-bit
    MKV_REQUIRE((int64_t)tokens_per_split * max_splits <= (int64_t)1 << 33, "%d ranges of %d tokens are too long", max_splits, tokens_per_split);
    MKV_REQUIRE(max_splits == 1 || (mid_o && mid_lse), "scratch buffers are NULL");
    MKV_REQUIRE(((uintptr_t)mid_o & 15) == 0 && ((uintptr_t)mid_lse & 3) == 0, "mid_o must be 16-byte aligned, mid_lse 4-byte aligned");
    MKV_REQUIRE((((uintptr_t)q | (uintptr_t)o) & 15) == 0 && ((q_stride | o_stride) & 7) == 0, "q and o rows must be 16-byte aligned");
    MKV_REQUIRE(softmax_scale > 0.f, "softmax_scale must be positive");
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
    g.scale2 = softmax_scale * mkv::kLog2E;
    const int64_t rows = (int64_t)batch->max_prefill_len * group;
    const int64_t columns = (int64_t)pool->num_kv_heads * max_splits * batch->num_prefill_seqs;
    // Rows per workgroup: 64 where a chunk has no more; 256 (one workgroup of eight waves per CU, the conversions of a
    // tile shared by more rows) for long chunks that fill the chip with them -- 2048 x 4 rows over 8192 cached tokens
    // 370 us against 407 with 128, whole prompts of 8192 tokens 637 against 707, but eight of 512 tokens 46 against 42.
    const int shape = rows <= 64 ? 64 : pool->head_dim == 128 && rows > 512 && columns * mkv::cdiv(rows, 256) >= mkv::num_cus() ? 256 : 128;
    int64_t cells = columns * mkv::cdiv(rows, shape);
    // a launch holds fewer than 2^32 threads, the joining one up to 256 for every row
    MKV_REQUIRE(cells * 512 <= 0xffffffffll && (max_splits == 1 || rows * pool->num_kv_heads * 256 <= 0xffffffffll), "too many rows in one call");
    // Finding a workgroup's place in the order costs a few microseconds: 8 x 512 tokens 42 us, sorted 48; four ragged
    // chunks over up to 7473 cached tokens 992 us, sorted 605.
    g.key_tiles = mkv::cdiv((int64_t)tokens_per_split * max_splits, 64);
    g.sorted = batch->num_prefill_seqs > 1 && cells > 2 * mkv::num_cus() && g.key_tiles >= 32;
    // Row tiles in pairs, a chunk's longest with its shortest, where the pairs still fill the chip: work of one size, and a
    // start less for two tiles, since the second's first keys are fetched under the first's last.  16 x 512 tokens of 32 q and 8
    // kv heads 72 us, single 82; 8 x 512 of 32 heads each 40.5, single 42; 8 x 256 (half the workgroups needed) 19.3 and 19.0.
    g.paired = max_splits == 1 && !g.sorted && cells >= (shape == 256 ? 2 : pool->head_dim == 128 ? 4 : 6) * mkv::num_cus();
    if (g.paired) cells = columns * mkv::cdiv(mkv::cdiv(rows, shape), 2);
    const dim3 grid((unsigned)cells);
    hipStream_t s = (hipStream_t)stream;
    if (dtype == MKV_F16) mkv::launch_prefill8<mkv::F16>(*pool, shape, grid, s, g);
    else mkv::launch_prefill8<mkv::BF16>(*pool, shape, grid, s, g);
    MKV_HIP(hipGetLastError());
    if (max_splits > 1)
        return mkv::launch_merge8(dtype, pool->head_dim, (const float*)mid_o, (const float*)mid_lse, o, o_stride,
                                  num_q_heads, batch->max_prefill_len * num_q_heads, batch->num_prefill_seqs, max_splits, mkv::chunks_of(*batch), s);
    return MKV_OK;
}
