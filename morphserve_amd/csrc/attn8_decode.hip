// Decode attention over the 8-bit paged cache, and the join of split partials.
//
// One workgroup of four waves per (split, kv head, sequence); all q heads of the kv head ride along as the columns
// of the matrix products, so a code is read from memory once.  A wave takes 64 tokens (four blocks) at a time and
// nothing passes through LDS on the way: codes go from memory to registers, are converted there and feed
//
//   S^T[token, head] = K . Q^T        v_mfma_f32_16x16x32, 32 head dims a step
//   O^T[dim, head]  += V^T . P^T      v_mfma_f32_16x16x32, 32 tokens a step
//
// Which token is which row of the first product is free, and it is chosen so that the second needs no exchange:
// lane group c = lane / 16 owns block c of the four.  Row 4c + i of score tile j is token 4j + i of block c, so the
// accumulators of a lane are the sixteen scores of ONE block in token order -- K's scale is one factor per lane --
// and, rounded, they are the second product's operand in the order in which V's sixteen bytes per head dim lie.
// The running maximum moves only when some score has outgrown it by kLazy octaves.
//
// Bound: reading the codes.  64 rows of 1024 to 1536 tokens, 8 kv heads x 128: 31.2 us, 5.4 TB/s; the same loads without any
// work 27.9 us.  128 rows and 64 q heads (int8, bf16) 59.7 us, 5.7 TB/s; 5 rows of up to 60000 tokens 96.2 us, 5.3 TB/s with
// the join.  Codes of a wave's next tile are asked for as soon as their registers are free, K's between the two products and
// V's behind the second, and are waited for one by one.  A third wave per SIMD, loads in pieces as single registers become free,
// and loads that the caches keep were no faster.
#include <type_traits>

#include "kv8.h"

namespace mkv {

static constexpr float kLazy = 8.f;        // probabilities stay below 2^8, well inside fp16

struct Attn8Args {
    mkv_pool8 pool;
    mkv_batch batch;
    const char* q;
    char* o;
    int64_t q_stride, o_stride;            // elements
    float *mid_o, *mid_lse;
    int32_t group;                         // q heads per kv head, at most 16
    int32_t layer, tiles_per_split, max_splits;
    float scale2;                          // softmax scale * log2(e)
};

template <int D>
struct Tile8 {                             // the codes of 64 tokens of one head, as the lanes hold them
    uint4v k[4][D / 64];                   // [score tile][64 head dims]
    uint4v v[D / 16];                      // [16 head dims]: the lane's dim, sixteen tokens of its block
};

template <class T, class C, int D>
__global__ __launch_bounds__(256) void attn8_decode_kernel(const Attn8Args g) {
    typedef typename T::elem E;
    typedef typename T::vec8 vec8;
    constexpr int kY = D / 64, kX = D / 32, kT = D / 16;
    // V's scale is part of the conversion, but for int8 to bf16: there the conversion would take a product a code, and
    // bf16's exponent has the range for a probability times a scale, 16 products a lane instead of 128
    constexpr bool kScaleP = std::is_same<T, BF16>::value && std::is_same<C, Int8>::value;
    __shared__ float sm_acc[4][16][D];
    __shared__ float sm_m[4][16], sm_l[4][16];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int n = lane & 15;               // column: q head of the group; row of an operand
    const int c = lane >> 4;               // lane group
    const int split = blockIdx.x;
    const int kvh = blockIdx.y;
    const int i = blockIdx.z;
    const int G = g.group;
    const int Hq = g.pool.num_kv_heads * G;

    const int64_t seq = g.batch.seq_ids[g.batch.num_prefill_seqs + i];
    const int known_len = max(g.batch.decoding_lens[i], 0);      // asked for with the sequence, not behind it
    const bool has_row = seq >= 0 && seq < g.batch.table_rows;
    const int len = has_row ? (int)min((int64_t)known_len, g.batch.max_blocks_per_seq * kBlk) : 0;
    const int32_t* table = g.batch.block_table + (has_row ? seq * g.batch.max_blocks_per_seq : 0);
    const int nblk = (len + kBlk - 1) / kBlk;
    const int num_tiles = (len + 63) >> 6;
    const int tile_begin = split * g.tiles_per_split;
    // the last split takes whatever lies behind it: a max_splits that is too small costs balance, never tokens
    const int tile_end = split == (int)gridDim.x - 1 ? num_tiles : min(tile_begin + g.tiles_per_split, num_tiles);

    // Q^T: lane (head n, group c) holds, for step x, dims 64 (x / 2) + 16 c + 8 (x % 2) .. + 8 -- the order in which
    // the 16-byte loads of K hand the dims to the lanes
    vec8 qb[kX];
    const E* qrow = (const E*)g.q + (int64_t)i * g.q_stride + ((int64_t)kvh * G + n) * D;
#pragma unroll
    for (int x = 0; x < kX; ++x) {
        if (n < G) qb[x] = *(const vec8*)(qrow + 64 * (x >> 1) + 16 * c + 8 * (x & 1));
        else qb[x] = (vec8)(E)0.f;
    }

    float4v acc[kT];
#pragma unroll
    for (int t = 0; t < kT; ++t) acc[t] = (float4v){0.f, 0.f, 0.f, 0.f};
    float m_run = kFar, l_run = 0.f;       // of head n; l_run is this lane's share

    const int64_t block_bytes = block_bytes8(g.pool);
    const int64_t slab = slab_offset8(g.pool, g.layer, kvh);
    const uint8_t* k_at = (const uint8_t*)g.pool.k + slab + (n & 3) * D + 16 * c;       // + block, 4j rows, 64y
    const uint8_t* v_at = (const uint8_t*)g.pool.v + slab + n * kBlk;                   // + block, 256 t
    const uint16_t* scales = scale_row8(g.pool, g.layer, kvh);
    const int num_blocks = (int)g.pool.num_blocks;

    // K: lane's row n belongs to block n / 4 of the tile; V and the scores: lane's block is c.  A block that is not
    // there is read from block 0 (inside the pool) and masked.
    auto load_k = [&](Tile8<D>& x, int pid) {
        const uint8_t* p = k_at + (int64_t)max(pid, 0) * block_bytes;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int y = 0; y < kY; ++y) x.k[j][y] = __builtin_nontemporal_load((const uint4v*)(p + 4 * j * D + 64 * y));
    };
    auto load_v = [&](Tile8<D>& x, int pid) {
        const uint8_t* p = v_at + (int64_t)max(pid, 0) * block_bytes;
#pragma unroll
        for (int t = 0; t < kT; ++t) x.v[t] = __builtin_nontemporal_load((const uint4v*)(p + 256 * t));
    };

    Tile8<D> x;
    // One tile.  WHOLE: its four blocks are in the pool and every token counts; otherwise tokens that do not are given
    // no probability, and their V codes, which may be anything (NaN too), are taken as 0.
    auto consume = [&](auto whole_tag, int tile, bool here, unsigned ex, auto after_k, auto after_v) {
        constexpr bool WHOLE = decltype(whole_tag)::value;
        float4v st[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            st[j] = (float4v){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int y = 0; y < kY; ++y) {
                st[j] = T::mfma(C::raw(T{}, x.k[j][y][0], x.k[j][y][1]), qb[2 * y], st[j]);
                st[j] = T::mfma(C::raw(T{}, x.k[j][y][2], x.k[j][y][3]), qb[2 * y + 1], st[j]);
            }
        }
        after_k();
        const int valid = WHOLE ? kBlk : here ? min(len - (4 * tile + c) * kBlk, kBlk) : 0;
        const float f = g.scale2 * pow2_of(ex & 0xffu);
        float s[16];
        float mx = kFar;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            s[e] = st[e >> 2][e & 3] * f;
            if (!WHOLE) s[e] = e < valid ? s[e] : kFar;
            mx = fmaxf(mx, s[e]);
        }
        if (__ballot(mx - m_run > kLazy) != 0) {
            const float m_new = fmaxf(m_run, max_over_quarters(mx));
            const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
            l_run *= alpha;
#pragma unroll
            for (int t = 0; t < kT; ++t) acc[t] *= alpha;
            m_run = m_new;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            s[e] = __builtin_amdgcn_exp2f(s[e] - m_run);
            if (!WHOLE) s[e] = e < valid ? s[e] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 16; e += 4) l_run += (s[e] + s[e + 1]) + (s[e + 2] + s[e + 3]);
        if constexpr (kScaleP) {
            const float fv = pow2_of(ex >> 8);
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] *= fv;
        }
        vec8 pb[2];
#pragma unroll
        for (int z = 0; z < 2; ++z)
            pb[z] = (vec8){(E)s[8 * z], (E)s[8 * z + 1], (E)s[8 * z + 2], (E)s[8 * z + 3],
                           (E)s[8 * z + 4], (E)s[8 * z + 5], (E)s[8 * z + 6], (E)s[8 * z + 7]};
        unsigned keep[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const int in = min(max(valid - 4 * w, 0), 4);
            keep[w] = WHOLE || in >= 4 ? ~0u : (1u << (8 * in)) - 1u;
        }
        auto values = [&](unsigned w0, unsigned w1) {
            if constexpr (kScaleP) return C::raw(T{}, w0, w1);
            else return C::scaled(T{}, w0, w1, ex >> 8);
        };
#pragma unroll
        for (int t = 0; t < kT; ++t) {
            acc[t] = T::mfma(values(x.v[t][0] & keep[0], x.v[t][1] & keep[1]), pb[0], acc[t]);
            acc[t] = T::mfma(values(x.v[t][2] & keep[2], x.v[t][3] & keep[3]), pb[1], acc[t]);
        }
        after_v();
    };

    // The wave's tiles are tile_begin + wave + 4 k.  Loads complete in order, and where two paths meet the compiler waits for
    // what either may have left: so a tile's block ids are asked for a tile ahead, before that tile's K, and looked at only
    // when they are used, and nothing is loaded under a condition.
    const int first = tile_begin + wave;
    const int count = first < tile_end ? (tile_end - first + 3) >> 2 : 0;
    int id_k = 0, id_v = 0, pid = -1;
    unsigned ex = 0;
    auto ask_ids = [&](int k) {
        const int blk = 4 * (first + 4 * k);
        id_k = table[min(blk + (n >> 2), nblk - 1)];
        id_v = table[min(blk + c, nblk - 1)];
    };
    auto request_k = [&](int k) {
        const int limit = k < count ? nblk - 4 * (first + 4 * k) : 0;      // blocks from the tile's first on
        const int pk = n >> 2 < limit && id_k >= 0 && id_k < num_blocks ? id_k : -1;
        pid = c < limit && id_v >= 0 && id_v < num_blocks ? id_v : -1;
        __builtin_amdgcn_sched_barrier(0);                   // the order of the loads is the one written here
        ask_ids(k + 1);
        ex = scales[max(pid, 0)];
        __builtin_amdgcn_sched_barrier(0);
        load_k(x, pk);
        __builtin_amdgcn_sched_barrier(0);
    };
    int k = 0;
    auto step = [&](auto whole_tag) {
        const bool here = pid >= 0;
        consume(whole_tag, first + 4 * k, here, here ? ex : 0x7f7fu,
                [&] {
                    __builtin_amdgcn_sched_barrier(0);
                    request_k(k + 1);
                },
                [&] {
                    __builtin_amdgcn_sched_barrier(0);
                    load_v(x, pid);
                    __builtin_amdgcn_sched_barrier(0);
                });
    };
    if (count > 0) {
        ask_ids(0);
        request_k(0);
        load_v(x, pid);
        // q has arrived (its loads are older than the ids'), which the compiler would otherwise doubt in the loops: not
        // knowing, it waits for all that is in flight
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int y = 0; y < kX; ++y) asm volatile("" : "+v"(qb[y]));
        // Whole tiles, then, from the first that is not, the careful body, which also takes the wave's last tile, behind
        // which nothing is asked for.  Loops apart, not two bodies in one: the accumulators would be copied where the bodies meet.
        for (; k + 1 < count && __ballot(pid < 0) == 0 && (first + 4 * k + 1) * 64 <= len; ++k) step(std::true_type{});
        for (; k + 1 < count; ++k) step(std::false_type{});
        const bool here = pid >= 0;
        consume(std::false_type{}, first + 4 * k, here, here ? ex : 0x7f7fu, [] {}, [] {});
    }

    // ---- the four waves' states meet in LDS --------------------------------------------------------
    const float l_all = sum_over_quarters(l_run);
    if (n < G) {
#pragma unroll
        for (int t = 0; t < kT; ++t) *(float4v*)&sm_acc[wave][n][16 * t + 4 * c] = acc[t];
        if (c == 0) {
            sm_m[wave][n] = m_run;
            sm_l[wave][n] = l_all;
        }
    }
    __syncthreads();
    const bool direct = gridDim.x == 1;
    for (int idx = threadIdx.x; idx < G * D; idx += 256) {
        const int h = idx / D, d = idx % D;
        const float m_tot = fmaxf(fmaxf(sm_m[0][h], sm_m[1][h]), fmaxf(sm_m[2][h], sm_m[3][h]));
        float l_tot = 0.f, a_tot = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = __builtin_amdgcn_exp2f(sm_m[w][h] - m_tot);
            l_tot += sm_l[w][h] * f;
            a_tot += sm_acc[w][h][d] * f;
        }
        const float val = l_tot == 0.f ? 0.f : a_tot / l_tot;      // nothing to attend to: zeros
        const int64_t hq = (int64_t)kvh * G + h;
        if (direct) {
            ((E*)g.o)[(int64_t)i * g.o_stride + hq * D + d] = (E)val;
        } else {
            const int64_t slot = ((int64_t)i * Hq + hq) * g.max_splits + split;
            g.mid_o[slot * D + d] = val;
            if (d == 0) g.mid_lse[slot] = l_tot == 0.f ? kFar : __builtin_amdgcn_logf(l_tot) + m_tot;
        }
    }
}

// One workgroup per output row -- of a prefill chunk (blockIdx.y) or, without start_locs, of the decode batch; wave w
// takes the partials w, w + 4, ... of the row.  A partial that holds nothing (its log sum at kFar) weighs nothing; one whose sum is a NaN counts.
template <class T, int D>
__global__ __launch_bounds__(256) void merge8_kernel(const float* __restrict__ mid_o, const float* __restrict__ mid_lse,
                                                     char* __restrict__ o, int64_t o_stride, int32_t num_q_heads,
                                                     int32_t splits, const Chunks8 chunks) {
    typedef typename T::elem E;
    constexpr int kDims = D / 64;
    typedef float vecd __attribute__((ext_vector_type(kDims)));
    __shared__ float part[4][D];
    __shared__ float part_l[4];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    int64_t t = blockIdx.x / (unsigned)num_q_heads;
    const int64_t h = blockIdx.x - t * num_q_heads;
    if (chunks.start_locs) {
        const int64_t start = chunks.start_locs[blockIdx.y];
        if (t >= chunk_rows(chunks, blockIdx.y, start)) return;
        t += start;
    }
    const int64_t base = (t * num_q_heads + h) * splits;
    float m = kFar;
    for (int s = lane; s < splits; s += 64) m = fmaxf(m, mid_lse[base + s]);
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) m = fmaxf(m, __shfl_xor(m, s));
    float l = 0.f;
    vecd a = (vecd)0.f;
    for (int s0 = wave; s0 < splits; s0 += 16) {
        vecd v[4];
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t slot = base + min(s0 + 4 * e, splits - 1);
            w[e] = mid_lse[slot];
            v[e] = *(const vecd*)(mid_o + slot * D + lane * kDims);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (s0 + 4 * e < splits && !(w[e] <= 0.5f * kFar)) {
                const float f = __builtin_amdgcn_exp2f(w[e] - m);
                l += f;
                a += f * v[e];
            }
        }
    }
#pragma unroll
    for (int d = 0; d < kDims; ++d) part[wave][lane * kDims + d] = a[d];
    if (lane == 0) part_l[wave] = l;
    __syncthreads();
    if (threadIdx.x < D) {
        const int d = threadIdx.x;
        const float sum = (part[0][d] + part[1][d]) + (part[2][d] + part[3][d]);
        const float all = (part_l[0] + part_l[1]) + (part_l[2] + part_l[3]);
        ((E*)o)[t * o_stride + h * D + d] = (E)(all == 0.f ? 0.f : sum / all);
    }
}

static constexpr int kFewSplits = 8;

// The same for a few splits: a wave per row, its partials requested together.
template <class T, int D>
__global__ __launch_bounds__(256) void merge8_few_kernel(const float* __restrict__ mid_o, const float* __restrict__ mid_lse,
                                                         char* __restrict__ o, int64_t o_stride, int32_t num_q_heads,
                                                         int32_t rows, int32_t splits, const Chunks8 chunks) {
    typedef typename T::elem E;
    constexpr int kDims = D / 64;
    typedef float vecd __attribute__((ext_vector_type(kDims)));
    const int lane = threadIdx.x & 63;
    const int row = (int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if (row >= rows) return;
    int64_t t = row / (unsigned)num_q_heads;
    const int64_t h = row - t * num_q_heads;
    if (chunks.start_locs) {
        const int64_t start = chunks.start_locs[blockIdx.y];
        if (t >= chunk_rows(chunks, blockIdx.y, start)) return;
        t += start;
    }
    const int64_t base = (t * num_q_heads + h) * splits;
    vecd v[kFewSplits];
    float w[kFewSplits];
#pragma unroll
    for (int s = 0; s < kFewSplits; ++s) {
        const int64_t slot = base + min(s, splits - 1);
        w[s] = mid_lse[slot];
        v[s] = *(const vecd*)(mid_o + slot * D + lane * kDims);
    }
    float m = kFar;
#pragma unroll
    for (int s = 0; s < kFewSplits; ++s) m = fmaxf(m, w[s]);
    float l = 0.f;
    vecd a = (vecd)0.f;
#pragma unroll
    for (int s = 0; s < kFewSplits; ++s) {
        if (s < splits && !(w[s] <= 0.5f * kFar)) {
            const float f = __builtin_amdgcn_exp2f(w[s] - m);
            l += f;
            a += f * v[s];
        }
    }
    a *= l == 0.f ? 0.f : 1.f / l;
    E* out = (E*)o + t * o_stride + h * D + lane * kDims;
#pragma unroll
    for (int d = 0; d < kDims; ++d) out[d] = (E)a[d];
}

int launch_merge8(int dtype, int head_dim, const float* mid_o, const float* mid_lse, void* o, int64_t o_stride,
                  int32_t num_q_heads, int32_t rows, int32_t chunk_count, int32_t splits, const Chunks8& chunks, hipStream_t s) {
    // A wave per row where there are few partials: 512 tokens of 32 q heads in four ranges 58 us with the attention, with a
    // workgroup per row 72.  With more than four and rows that do not fill the chip the partials of a row are better shared by
    // four waves: one row of 32 q heads in eight ranges 9.2 us, by a wave 10.5; 4096 rows in eight 34, by a wave 26.
    const bool few = splits <= (rows < 2048 ? kFewSplits / 2 : kFewSplits);
    const dim3 grid(few ? (unsigned)cdiv(rows, 4) : (unsigned)rows, (unsigned)chunk_count);
#define MKV_MERGE(T, D)                                                                                                         \
    do {                                                                                                                        \
        if (few)                                                                                                                \
            hipLaunchKernelGGL((merge8_few_kernel<T, D>), grid, dim3(256), 0, s, mid_o, mid_lse, (char*)o, o_stride,           \
                               num_q_heads, rows, splits, chunks);                                                              \
        else                                                                                                                    \
            hipLaunchKernelGGL((merge8_kernel<T, D>), grid, dim3(256), 0, s, mid_o, mid_lse, (char*)o, o_stride, num_q_heads,   \
                               splits, chunks);                                                                                 \
    } while (0)
    if (dtype == MKV_F16 && head_dim == 128) MKV_MERGE(F16, 128);
    else if (dtype == MKV_F16) MKV_MERGE(F16, 64);
    else if (head_dim == 128) MKV_MERGE(BF16, 128);
    else MKV_MERGE(BF16, 64);
#undef MKV_MERGE
    MKV_HIP(hipGetLastError());
    return MKV_OK;
}

template <class T, class C>
static void launch_decode8(int head_dim, dim3 grid, hipStream_t s, const Attn8Args& g) {
    if (head_dim == 128) hipLaunchKernelGGL((attn8_decode_kernel<T, C, 128>), grid, dim3(256), 0, s, g);
    else hipLaunchKernelGGL((attn8_decode_kernel<T, C, 64>), grid, dim3(256), 0, s, g);
}

}  // namespace mkv

extern "C" int mkv_attn8_decode(const mkv_pool8* pool, const mkv_batch* batch, int32_t dtype, const void* q, void* o,
                                int64_t q_stride, int64_t o_stride, int32_t num_q_heads, float softmax_scale,
                                int32_t layer, int32_t tokens_per_split, int32_t max_splits, void* mid_o,
                                void* mid_lse, void* stream) {
    int rc = mkv::check_pool8(pool);
    if (rc) return rc;
    rc = mkv::check_batch8(batch);
    if (rc) return rc;
    MKV_REQUIRE(dtype == MKV_F16 || dtype == MKV_BF16, "dtype %d is neither MKV_F16 nor MKV_BF16", dtype);
    MKV_REQUIRE(layer >= 0 && layer < pool->num_layers, "layer %d outside [0, %d)", layer, pool->num_layers);
    const int n = batch->num_decoding_seqs;
    if (n == 0) return MKV_OK;
    MKV_REQUIRE(q && o, "NULL argument");
    MKV_REQUIRE(num_q_heads > 0 && num_q_heads % pool->num_kv_heads == 0 && num_q_heads / pool->num_kv_heads <= 16,
                "num_q_heads %d must be 1 to 16 times num_kv_heads %d", num_q_heads, pool->num_kv_heads);
    MKV_REQUIRE(tokens_per_split > 0 && tokens_per_split % 64 == 0, "tokens_per_split %d must be a positive multiple of 64",
                tokens_per_split);
    MKV_REQUIRE(max_splits >= 1, "max_splits must be >= 1");
    // tile and block numbers, those behind the last key included, are 32-bit
    MKV_REQUIRE((int64_t)tokens_per_split * max_splits <= (int64_t)1 << 33, "%d ranges of %d tokens are too long", max_splits, tokens_per_split);
    MKV_REQUIRE((int64_t)max_splits * 256 <= 0xffffffffll, "%d ranges are too many", max_splits);        // threads of the launch
    MKV_REQUIRE(max_splits == 1 || (mid_o && mid_lse), "scratch buffers are NULL");
    MKV_REQUIRE(((uintptr_t)mid_o & 15) == 0 && ((uintptr_t)mid_lse & 3) == 0, "mid_o must be 16-byte aligned, mid_lse 4-byte aligned");
    MKV_REQUIRE(((uintptr_t)q & 15) == 0 && (q_stride & 7) == 0, "q rows must be 16-byte aligned");
    MKV_REQUIRE(n <= 65535, "at most 65535 decode rows per call");
    MKV_REQUIRE((int64_t)n * num_q_heads * 256 <= 0xffffffffll, "too many rows in one call");     // threads of the joining launch
    mkv::Attn8Args g = {};
    g.pool = *pool;
    g.batch = *batch;
    g.q = (const char*)q;
    g.o = (char*)o;
    g.q_stride = q_stride;
    g.o_stride = o_stride;
    g.mid_o = (float*)mid_o;
    g.mid_lse = (float*)mid_lse;
    g.group = num_q_heads / pool->num_kv_heads;
    g.layer = layer;
    g.tiles_per_split = tokens_per_split / 64;
    g.max_splits = max_splits;
    g.scale2 = softmax_scale * mkv::kLog2E;
    const dim3 grid((unsigned)max_splits, (unsigned)pool->num_kv_heads, (unsigned)n);
    hipStream_t s = (hipStream_t)stream;
    if (dtype == MKV_F16) {
        if (pool->kind == MKV_KV8_E4M3) mkv::launch_decode8<mkv::F16, mkv::E4M3>(pool->head_dim, grid, s, g);
        else mkv::launch_decode8<mkv::F16, mkv::Int8>(pool->head_dim, grid, s, g);
    } else {
        if (pool->kind == MKV_KV8_E4M3) mkv::launch_decode8<mkv::BF16, mkv::E4M3>(pool->head_dim, grid, s, g);
        else mkv::launch_decode8<mkv::BF16, mkv::Int8>(pool->head_dim, grid, s, g);
    }
    MKV_HIP(hipGetLastError());
    if (max_splits > 1)
        return mkv::launch_merge8(dtype, pool->head_dim, (const float*)mid_o, (const float*)mid_lse, o, o_stride,
                                  num_q_heads, n * num_q_heads, 1, max_splits, mkv::Chunks8{}, s);
    return MKV_OK;
}
