// Attention of a chunk of new tokens per row over a paged cache that holds them already (speculative tokens, portions of
// prompts, whole prompts), on the 5th-generation tensor cores.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^((q . k_j) scale log2(e) - m),   j in [max(0, L + t - window), L + t]
//
// for query t < n of a row with L keys before its n new ones.  Running maximum and sum in fp32, one pass over the keys; P is
// rounded to bf16 (2^-8 of a term of the sum at most, the type of V) because the tensor core takes it beside V in that type.
//
// A tile is CH_M = 128 query rows of one (row, kv head): the G query heads of the group at 128 / G consecutive tokens, row = token * G +
// head, so keys and values are read once for the whole group.  It walks over its keys in tiles of 64, cut at multiples of 64.  Pages
// hold a multiple of 48 tokens, so a tile lies in one page or in two, at a multiple of 16: it is copied in one box or two, by maps of boxes of
// 16, 32, 48 and 64 keys.
// The pipeline is that of the dense kernel (prefill_attn.cu): two persistent CTAs per SM, a copying thread, a thread that issues S = Q K^T two
// tiles ahead and O += P V, and one softmax thread per query row that takes its scores out of tensor memory and puts P back over them.
//
// What a CTA works through, found from the rows' lengths by all of its threads before the first tile:
//   stretches: the sequence of all key tiles of all tiles of queries, (row, kv head) by (row, kv head), is cut into equal stretches, one per
//     CTA; tiles of queries that lie in several leave partial sums.  Balanced to a key tile whatever the lengths.  Where tiles of queries share
//     keys (more than one per row) and the keys are more than L2 holds, up to CH_PHASES groups of pairs are cut one after the other.
//   a deal: where tiles of queries are many or alike enough to fill the CTAs' rounds they go to the CTAs uncut, back and forth: of rows of like
//     lengths longest first as in the dense kernel, of others row by row, empty ones left out, a last round of few long tiles cut into stretches.  A CTA's threads write its list; the copying thread reads an entry ahead.
//   clusters: few pairs of short rows, one tile of queries each, are bound by launches and round trips.  A cluster takes a pair, each CTA a part of its
//     keys, and the parts meet in shared memory: no sums over the rows ahead of the work, no launch behind it.
// chunk_finish_kernel adds up partial sums in the order of the keys: results don't depend on timing.
//
// Bounds and figures.  Many new tokens: the tensor pipe and the softmax chain.  A key tile takes the pipe 640 cycles (S 8 products of 48 with both operands
// in shared memory, O 4 of 64) and the exponentials 512.  By the SMs' own counters the two CTAs of an SM get through one each in 1850 cycles, taken over a whole
// pass of long rows (within a piece 1680), in 2500 where pieces have 17 (whole prompts of 2048: hand-over, masked tiles and tail besides).
// 2011 tokens behind 62 000 keys, 16 + 4 heads: 1050 to 1100 us = 950 TFLOP/s, the clock at 1.42 GHz under the power limit; 8 prompts of 2048, 12 heads: 125 us =
// 825 by themselves, 147 in a long run (1.50 GHz).  Few new tokens: the keys' bytes.  2 x 8 tokens, 12 heads, 457 MB of keys and values: 80 us = 5.7 TB/s, 562 MB:
// 95 = 5.9; 48 x 5 tokens behind about 2048, 16 + 4 heads: 46 us for 210 MB, 52 for 229 = 4.4 to 4.5 TB/s, of which about 14 us are launches,
// lengths, the first tiles' latency and the sums of parts, whatever the keys.  4 x 4 tokens of short rows: 7.5 us, launch and round trips.
// Tried and slower: two threads per query row (147 us for the prompts), a warp of its own that cleans edge tiles (155), half or a quarter of the exponentials
// as polynomials on the FMA pipe (131, 127), a maximum taken from the tile before, scores asked for before the stores of P are waited for (126).
//
// Every barrier wait is bounded; one that runs out sets NCKV_ST_TIMEOUT, the CTA stops issuing work, waits for its copies, frees its
// tensor memory and returns.
#include <math.h>

#include "nckv_common.cuh"
#include "tc05.cuh"

namespace nckv {

constexpr int CH_M = 128, CH_N = 64;
constexpr int CH_STAGES = 2, CH_VSTAGES = 3;  // of K and of V
constexpr int CH_THREADS = CH_M + 64;         // softmax threads, the issuing warp, the copying warp
constexpr int CH_KV_BYTES = CH_N * NCKV_D * 2;
constexpr int CH_TMEM_COLS = 256;  // S / P buffers [0, 64), [64, 128); O [128, 256)
constexpr int CH_PHASES = 4;       // most groups of pairs that are cut one after the other
constexpr int CH_MIN_TILES = 1;    // shortest stretch of a CTA
constexpr int CH_ROWS = 4096;      // most rows of a launch: 48 KB of shared memory that the keys come to later
constexpr int CH_RING = 8;         // pieces of work that the copying thread can be ahead with: it is four at most (five stages, pieces of one tile)
constexpr int CH_PITCH = NCKV_D + 4;  // floats of a row where a cluster's parts meet
constexpr long long CH_PART_BYTES = 160LL << 20, CH_PHASE_BYTES = 48LL << 20;

struct ChunkMaps {
    CUtensorMap q, k[4], v[4];  // k, v: boxes of 16, 32, 48 and 64 keys of 64 channels
};

struct alignas(16) ChunkPlan {  // a CTA's stretch of a phase: its first key tile (-1: none), how far into which tile of queries that is, and the whole tile's key tiles
    int at, off, count, b, hkv, t0, begin, each;  // the phase begins at `begin` and is cut every `each`
    int n, none[3];                               // new tokens of the row
};

struct alignas(16) ChunkDeal {  // a tile of queries: row (-1: nothing), kv head + Hkv * number of the tile, the row's lengths; the part of its key tiles
    int b, local, L, n;
    int off, n_tiles, slot, none;  // n_tiles 0: all of them
};

struct ChunkParams {
    const int32_t *table, *seqlens, *new_tokens;  // new_tokens may be null: T for every row
    const __nv_bfloat16 *v_pool;
    __nv_bfloat16 *out;
    ChunkPlan *plan;    // (phases, CTAs): how the stretches were cut
    ChunkDeal *deals;   // (CTAs, deal_room): what was dealt
    int deal_room;
    float *part_ml;  // (slots, part_rows, 2): maximum and sum
    float *part_o;   // (slots, part_rows, 128), not divided by the sum
    int32_t *status;
    int B, T, Hq, Hkv, G, tile_tokens, n_qtiles;
    int page_tokens, max_pages, n_pages, capacity;
    int64_t page_stride, token_stride;
    int window_left;
    int phases, part_rows;        // phases 0: nothing is cut
    int phase_pairs;              // (row, kv head) pairs of a phase
    int group_pairs, n_groups;    // of a deal
    float scale_log2;
};

// A row's lengths; n = 0 for one that can't be (its outputs are zeros).
struct ChunkRow {
    int L, n;
};
__device__ __forceinline__ ChunkRow chunk_row(const ChunkParams &p, int b) {
    ChunkRow r;
    r.L = __ldg(p.seqlens + b);
    r.n = p.new_tokens ? min(max(__ldg(p.new_tokens + b), 0), p.T) : p.T;
    if (r.L < 0 || (long long)r.L + r.n > p.capacity) r.L = r.n = 0;
    return r;
}

// Key tiles [first, first + count) that any of the tokens [t0, t0 + tile_tokens) of a row sees.
struct ChunkSpan {
    int kv_lo, kv_hi, first, count;
};
__device__ __forceinline__ ChunkSpan chunk_span(const ChunkParams &p, const ChunkRow &r, int t0) {
    ChunkSpan s;
    s.kv_lo = p.window_left >= 0 ? max(0, r.L + t0 - p.window_left) : 0;
    s.kv_hi = r.L + min(t0 + p.tile_tokens, r.n);
    s.first = s.kv_lo / CH_N;
    s.count = t0 < r.n ? (s.kv_hi + CH_N - 1) / CH_N - s.first : 0;
    return s;
}

// A CTA's piece of work: key tiles [tile0, tile0 + n_tiles) of one tile of queries.
struct ChunkUnit {
    int b, hkv, t0, L, n;
    int kv_lo, kv_hi, tile0, n_tiles;
    int slot;  // where the partial sums go; -1: all keys, the output is written
};

// Where a CTA's stretch of a phase lies: [at, end) in the sequence of key tiles, beginning at key tile `off` of a tile of queries.
struct ChunkStretch {
    int at, end, b, hkv, qt, off;
};

// Walks over a CTA's pieces of work.
struct ChunkCursor {
    ChunkUnit u;
    int t;    // key tile inside the piece
    int seq;  // number of the piece among the CTA's
    bool valid;
    int phase;  // -1: dealt
    int at;     // next key tile of the stretch, or next round of the deal
    int begin, end, qt, off;
    ChunkSpan span;
    // Looked up ahead of need: a row's lengths, or an entry of the deal, take longer than a key tile.
    ChunkRow next_row;
    ChunkDeal next_deal;

    __device__ __forceinline__ void item(const ChunkParams &p) {
        u.t0 = qt * p.tile_tokens;
        span = chunk_span(p, ChunkRow{u.L, u.n}, u.t0);
    }
    __device__ __forceinline__ void row(const ChunkParams &p, int b, const ChunkRow &r) {
        u.b = b;
        u.L = r.L;
        u.n = r.n;
        next_row = chunk_row(p, min(b + 1, p.B - 1));
    }
    __device__ __forceinline__ bool enter(const ChunkParams &p, const ChunkStretch *stretches) {  // the next phase with something in it
        for (; phase < p.phases; ++phase) {
            const ChunkStretch s = stretches[phase];
            if (s.at >= s.end) continue;
            at = begin = s.at;
            end = s.end;
            row(p, s.b, chunk_row(p, s.b));
            u.hkv = s.hkv;
            qt = s.qt;
            off = s.off;
            item(p);
            return true;
        }
        return false;
    }
    // `deals`: rounds that were dealt to this CTA, -1: stretches
    __device__ __forceinline__ void start(const ChunkParams &p, const ChunkStretch *stretches, int deals) {
        seq = -1;
        at = begin = 0;
        end = deals;
        phase = deals < 0 ? 0 : -1;
        valid = true;
        if (deals < 0) valid = enter(p, stretches);
        else if (deals > 0) next_deal = p.deals[(long long)blockIdx.x * p.deal_room];
        if (valid) load(p, stretches);
    }
    __device__ __forceinline__ void load(const ChunkParams &p, const ChunkStretch *stretches) {
        t = 0;
        ++seq;
        if (phase >= 0) {
            if (at >= end) {
                ++phase;
                valid = enter(p, stretches);
                if (!valid) return;
            } else {
                while (off >= span.count) {  // ends: there are tiles behind `at`
                    off = 0;
                    if ((++qt) * p.tile_tokens >= u.n) {
                        qt = 0;
                        if (++u.hkv == p.Hkv) {
                            u.hkv = 0;
                            do row(p, u.b + 1, next_row);
                            while (u.n == 0);
                        }
                    }
                    item(p);
                }
            }
            u.kv_lo = span.kv_lo;
            u.kv_hi = span.kv_hi;
            u.n_tiles = min(span.count - off, end - at);
            u.tile0 = span.first + off;
            u.slot = u.n_tiles == span.count ? -1 : (phase * (int)gridDim.x + (int)blockIdx.x) * 2 + (at != begin);
            off += u.n_tiles;
            at += u.n_tiles;
            return;
        }
        for (;;) {
            if (at >= end) {
                valid = false;
                return;
            }
            const ChunkDeal d = next_deal;
            if (++at < end) next_deal = p.deals[(long long)blockIdx.x * p.deal_room + at];
            if (d.b < 0) continue;
            u.b = d.b;
            u.L = d.L;
            u.n = d.n;
            qt = d.local / p.Hkv;
            u.hkv = d.local - qt * p.Hkv;
            item(p);
            u.kv_lo = span.kv_lo;
            u.kv_hi = span.kv_hi;
            u.n_tiles = d.n_tiles ? d.n_tiles : span.count;
            u.tile0 = span.first + d.off;
            u.slot = d.slot;
            return;
        }
    }
    __device__ __forceinline__ void advance(const ChunkParams &p, const ChunkStretch *stretches) {
        if (++t >= u.n_tiles) load(p, stretches);
    }
    __device__ __forceinline__ bool last_of_unit() const { return t == u.n_tiles - 1; }
};

// Whether uncut tiles dealt to the CTAs take less than stretches (0): 1 in the order of like rows, 2 row by row, 3 row by row with the last round, if it
// is short, cut into stretches of at least CH_REST key tiles (3: 61 us where 6 and 12 take 57, window 512).  Rows' key tiles per kv head lie
// between `least` and `most`; `items` tiles of queries have `tiles` key tiles altogether.  A piece costs some 2 tiles, a phase of stretches
// CH_CUT for the partial sums that it leaves (twice 64 KB per CTA, written and read) and the launch that adds them up.  us as stretches / like
// rows / row by row, window -1: 8 x 2048 tokens, 12 + 12 heads, no context 215 / 126 / 170; 2 x 1722, 10 + 1 heads 52 / 37 / 40; 8 x 862, 10 + 1, contexts of
// 0 to 114 67 / 38 / 47; 2011 behind 60000, 16 + 4 1088 / 1139 / 1147; up to 1931 new tokens in 5 rows, 6 + 6 50 / 45 / 39; 24 x up to 384, 16 + 4, window 1024
// 113 / 103 / 85; 21 x up to 220 behind up to 3019, 12 + 12 91 / 100 / 99.  A last round of few tiles runs faster than the others, so it is cut only where it
// saves CH_REST_CUT: 24 x up to 384 behind up to 8192, 16 + 4 heads, row by row / with the last round cut, window 2048 132 / 122, window 1024 82 / 85.
constexpr float CH_CUT = 25.f;
constexpr int CH_REST = 6, CH_REST_TILES = 2;  // tiles of queries of a last round to a thread
constexpr float CH_REST_CUT = 16.f;
__device__ __forceinline__ int chunk_dealt(const ChunkParams &p, int least, int most, long long tiles, int items, int longest, int grid) {
    if (p.phases == 0) return 1;
    if (p.n_qtiles == 1 || items == 0) return 0;
    const float each = (float)tiles / items, per_cta = (float)tiles / grid, rounds = (float)items / grid;
    const bool like_rows = !p.new_tokens && most - least <= most / 3;
    const bool alike = longest < 1.5f * each;  // then rounds are whole, else the short tiles fill them up, longest first or not
    const float deal = alike ? ceilf(rounds) * (each + 2.f) : like_rows ? fmaxf(per_cta * 1.05f, (float)longest) + 2.f * rounds : per_cta + longest + 2.f * rounds;
    if (!like_rows && alike && items > grid && grid <= CH_REST_TILES * CH_THREADS) {
        const float full = floorf(rounds), rest = full * (each + 2.f) + fmaxf((rounds - full) * each, (float)CH_REST) + CH_REST_CUT;
        if (rest < fminf(deal, per_cta + 2.f * rounds + CH_CUT * p.phases)) return 3;
    }
    return deal <= per_cta + 2.f * rounds + CH_CUT * p.phases ? 2 - like_rows : 0;
}

__device__ __forceinline__ bool not_finite2(uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; }

// What values that are not finite add to a query row: they were taken out of the shared tiles that some rows don't see all of (zero
// times infinity would reach those rows).  Rare, so it reads the pages again.
__device__ __noinline__ float chunk_not_finite(const ChunkParams &p, const ChunkUnit u, int pos, int channel) {
    float sum = 0.f;
    const int hi = min(pos + 1, u.kv_hi), lo = p.window_left >= 0 ? max(pos - p.window_left, 0) : 0;
    const int first_pos = u.L + u.t0, last_pos = u.L + min(u.t0 + p.tile_tokens, u.n) - 1;
    for (int t = 0; t < u.n_tiles; ++t) {
        const int key0 = (u.tile0 + t) * CH_N;
        if (!(key0 + CH_N - 1 > first_pos || (p.window_left >= 0 && key0 < last_pos - p.window_left))) continue;
        for (int j = max(lo, key0); j < min(hi, key0 + CH_N); ++j) {
            const int idx = j / p.page_tokens, page = p.table[(long long)u.b * p.max_pages + idx];
            if (page < 0 || page >= p.n_pages) continue;
            const float v = __bfloat162float(p.v_pool[page * p.page_stride + (long long)(j - idx * p.page_tokens) * p.token_stride + u.hkv * NCKV_D + channel]);
            if (!(fabsf(v) <= 3.4e38f)) sum += v;
        }
    }
    return sum;
}

__host__ __device__ constexpr uint32_t chunk_q_half(int rows) { return (rows <= 32 ? 32 : rows <= 64 ? 64 : 128) * 128; }

template <bool CLUSTER>
__global__ void __launch_bounds__(CH_THREADS, 2)
chunk_attn_kernel(const __grid_constant__ ChunkMaps maps, const __grid_constant__ ChunkParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    if ((smem_u32(smem) & 1023u) != 0) {  // uniform; checked rather than assumed
        if (threadIdx.x == 0) atomicOr(p.status, (int)NCKV_ST_TIMEOUT);
        return;
    }
    // Q in one buffer of two halves of 128 rows, or two buffers where a piece has at most 64 or 32 rows (the product reads 128 all the same:
    // what it finds behind them only reaches rows that nobody looks at)
    const uint32_t q_bufs = p.part_rows <= CH_M / 2 ? 2 : 1, q_half = chunk_q_half(p.part_rows);
    uint8_t *sQ = smem, *sK = sQ + 2 * q_bufs * q_half, *sV = sK + CH_STAGES * CH_KV_BYTES;
    // Barriers of key tiles are indexed by the tile's number g in the CTA's stream: stage g % 2 or g % 3, buffer g & 1, and the phase
    // follows from g as well.  (What each of them says: prefill_attn.cu.)
    uint64_t *bars = reinterpret_cast<uint64_t *>(sV + CH_VSTAGES * CH_KV_BYTES);
    uint64_t *bar_q = bars, *bar_k = bars + 2, *bar_v = bars + 4, *bar_s = bars + 7, *bar_o = bars + 9, *bar_p = bars + 11;
    uint64_t *bar_u = bars + 13;  // [CH_RING] piece posted
    ChunkUnit *ring = reinterpret_cast<ChunkUnit *>(bars + 13 + CH_RING);            // piece u of the CTA at u % CH_RING; n_tiles 0: no more
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(ring + CH_RING);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    volatile int *s_poison = reinterpret_cast<volatile int *>(tmem_slot + 2);        // [4]: piece seq (seq & 3) had values that are not finite
    ChunkStretch *s_stretch = reinterpret_cast<ChunkStretch *>(tmem_slot + 6);       // [CH_PHASES]
    int *s_sum = reinterpret_cast<int *>(ring);                                      // [6][6], before there are pieces

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        prefetch_tensormap(&maps.q);
        prefetch_tensormap(&maps.k[3]);
        prefetch_tensormap(&maps.v[3]);
        for (int i = 0; i < CH_RING; ++i) mbar_init(&bar_u[i], 1);
        for (int s = 0; s < CH_STAGES; ++s) mbar_init(&bar_k[s], 1);
        for (int s = 0; s < CH_VSTAGES; ++s) mbar_init(&bar_v[s], 1);
        for (int s = 0; s < 2; ++s) {
            mbar_init(&bar_q[s], 1);
            mbar_init(&bar_s[s], 1);
            mbar_init(&bar_o[s], 1);
            mbar_init(&bar_p[s], CH_M / 32);
        }
        *abort_flag = 0;
        for (int i = 0; i < 4; ++i) s_poison[i] = -1;
        for (int i = 0; i < CH_PHASES; ++i) s_stretch[i].at = s_stretch[i].end = 0;
        fence_mbar_init();
    }
    if (warp == 0) {
        tmem_alloc(tmem_slot, CH_TMEM_COLS);
        tmem_relinquish();
    }
    pdl_wait_prior_grids();  // lengths and tables may come from the grid before
    int dealt = 0, deals = -1;
    bool any_idle = false;
    [[maybe_unused]] ChunkUnit mine;
    // where a cluster's parts meet: where K and V have been
    [[maybe_unused]] float *s_part = reinterpret_cast<float *>(sK);
    [[maybe_unused]] float2 *s_part_ml = reinterpret_cast<float2 *>(s_part + CH_M * CH_PITCH);
    if constexpr (CLUSTER) {
    const int ctas = (int)cluster_ctas(), rank = (int)cluster_rank(), pair = (int)blockIdx.x / ctas;
    mine.b = pair / p.Hkv;
    mine.hkv = pair - mine.b * p.Hkv;
    mine.t0 = 0;
    const ChunkRow r = chunk_row(p, mine.b);
    const ChunkSpan sp = chunk_span(p, r, 0);
    const int lo = sp.count * rank / ctas;
    mine.L = r.L;
    mine.n = r.n;
    mine.kv_lo = sp.kv_lo;
    mine.kv_hi = sp.kv_hi;
    mine.tile0 = sp.first + lo;
    mine.n_tiles = sp.count * (rank + 1) / ctas - lo;
    mine.slot = 0;
    if (tid == 0 && rank == 0 && mine.hkv == 0) {  // lengths out of range: reported once
        const int L = p.seqlens[mine.b], n = p.new_tokens ? p.new_tokens[mine.b] : p.T;
        if (L < 0 || n < 0) atomicOr(p.status, (int)NCKV_ST_BAD_SEQLEN);
        else if (n > p.T || (long long)L + n > p.capacity) atomicOr(p.status, (int)NCKV_ST_OVERFLOW);
    }
    for (int t = r.n + rank; t < p.T; t += ctas)  // slots without a token
        for (int i = tid; i < p.G * 16; i += CH_THREADS)
            reinterpret_cast<uint4 *>(p.out + (((long long)mine.b * p.T + t) * p.Hq + mine.hkv * p.G) * NCKV_D)[i] = make_uint4(0, 0, 0, 0);
    if (mine.n_tiles == 0 && tid < CH_M) s_part_ml[tid] = make_float2(-INFINITY, 0.f);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    } else {
    // ---- lengths: `width` lanes to a row -----------------------------------------------------------------
    // s_tiles[b]: key tiles of row b's tiles of queries, per kv head; s_place[b]: key tiles before row b; s_items[b]: tiles of queries, in all heads,
    // then those before row b.  They lie where K and V come later.
    int *s_tiles = reinterpret_cast<int *>(sK), *s_place = s_tiles + CH_ROWS, *s_items = s_place + CH_ROWS;
    int width = 1;
    while (width < 32 && width < p.n_qtiles) width *= 2;
    const int member = tid & (width - 1), groups = CH_THREADS / width;
    int items = 0, longest = 0, least = 0x7fffffff, most = 0;
    bool idle = false;  // a row has slots without a token, or can't be
    for (int b = tid / width; b < p.B; b += groups) {  // (whole groups of lanes)
        const ChunkRow r = chunk_row(p, b);
        idle |= r.n < p.T;
        if (blockIdx.x == 0 && member == 0) {  // lengths out of range: reported once
            const int L = p.seqlens[b], n = p.new_tokens ? p.new_tokens[b] : p.T;
            if (L < 0 || n < 0) atomicOr(p.status, (int)NCKV_ST_BAD_SEQLEN);
            else if (n > p.T || (long long)L + n > p.capacity) atomicOr(p.status, (int)NCKV_ST_OVERFLOW);
        }
        int n = 0;
        for (int qt = member; qt * p.tile_tokens < r.n; qt += width) {
            const int c = chunk_span(p, r, qt * p.tile_tokens).count;
            n += c;
            longest = max(longest, c);
        }
        const uint32_t mask = width == 32 ? 0xffffffffu : ((1u << width) - 1) << (lane & ~(width - 1));
        for (int off = 1; off < width; off <<= 1) n += __shfl_xor_sync(mask, n, off);
        if (member == 0) {
            s_tiles[b] = n;
            s_items[b] = (r.n + p.tile_tokens - 1) / p.tile_tokens * p.Hkv;
            items += s_items[b];
            least = min(least, n);
            most = max(most, n);
        }
    }
    __syncwarp();
    items = __reduce_add_sync(0xffffffffu, items);
    longest = __reduce_max_sync(0xffffffffu, longest);
    least = __reduce_min_sync(0xffffffffu, least);
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) {
        s_sum[warp] = items;
        s_sum[6 + warp] = longest;
        s_sum[12 + warp] = least;
        s_sum[18 + warp] = most;
    }
    tc_fence_before();
    any_idle = __syncthreads_or(idle);
    tc_fence_after();
    items = 0;
    for (int w = 0; w < CH_THREADS / 32; ++w) {
        items += s_sum[w];
        longest = max(longest, s_sum[6 + w]);
        least = min(least, s_sum[12 + w]);
        most = max(most, s_sum[18 + w]);
    }
    int all = 0, all_items = 0;  // key tiles and tiles of queries before a chunk of rows, then of all
    for (int b0 = 0; b0 < p.B; b0 += CH_THREADS) {
        const int mine = b0 + tid < p.B ? s_tiles[b0 + tid] * p.Hkv : 0, my_items = b0 + tid < p.B ? s_items[b0 + tid] : 0;
        int before = mine, items_before = my_items;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, before, off), w = __shfl_up_sync(0xffffffffu, items_before, off);
            if (lane >= off) {
                before += v;
                items_before += w;
            }
        }
        if (b0) __syncthreads();  // the sums of the chunk before have been read
        if (lane == 31) {
            s_sum[24 + warp] = before;
            s_sum[30 + warp] = items_before;
        }
        __syncthreads();
        before += all - mine;
        items_before += all_items - my_items;
        for (int w = 0; w < CH_THREADS / 32; ++w) {
            if (w < warp) {
                before += s_sum[24 + w];
                items_before += s_sum[30 + w];
            }
            all += s_sum[24 + w];
            all_items += s_sum[30 + w];
        }
        if (b0 + tid < p.B) {
            s_place[b0 + tid] = before;
            s_items[b0 + tid] = items_before;
        }
    }
    dealt = chunk_dealt(p, least, most, all, items, longest, (int)gridDim.x);
    if (tid < p.phases) p.plan[tid * gridDim.x + blockIdx.x].at = -1;
    __syncthreads();
    if (dealt) {
        // a thread to a round; dealt back and forth
        const int pairs = p.B * p.Hkv, per_group = p.group_pairs * p.n_qtiles, grid = (int)gridDim.x, c = (int)blockIdx.x;
        const int limit = dealt == 1 ? pairs * p.n_qtiles : dealt == 2 ? items : items / grid * grid;
        ChunkDeal *mine = p.deals + (long long)c * p.deal_room;
        auto row_by_row = [&](int idx) {
            int lo = 0, hi = p.B - 1;  // the first row with tiles behind idx
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                if (s_items[mid + 1] > idx) hi = mid;
                else lo = mid + 1;
            }
            const ChunkRow r = chunk_row(p, lo);
            const int in_row = idx - s_items[lo], qt = (r.n + p.tile_tokens - 1) / p.tile_tokens - 1 - in_row / p.Hkv;  // longest first
            return ChunkDeal{lo, qt * p.Hkv + in_row % p.Hkv, r.L, r.n, 0, 0, -1, 0};
        };
        deals = limit / grid;
        deals += ((deals & 1) ? grid - 1 - c : c) < limit - deals * grid;
        for (int i = tid; i < deals; i += CH_THREADS) {
            const int idx = i * grid + ((i & 1) ? grid - 1 - c : c);
            if (dealt == 1) {
                const int grp = min(idx / per_group, p.n_groups - 1), in_grp = idx - grp * per_group;
                const int grp_pairs = grp == p.n_groups - 1 ? pairs - grp * p.group_pairs : p.group_pairs;
                const int pair = grp * p.group_pairs + in_grp % grp_pairs, qt = p.n_qtiles - 1 - in_grp / grp_pairs;  // all pairs' longest tiles first
                const ChunkRow r = chunk_row(p, pair / p.Hkv);
                mine[i] = ChunkDeal{qt * p.tile_tokens < r.n ? pair / p.Hkv : -1, qt * p.Hkv + pair % p.Hkv, r.L, r.n, 0, 0, -1, 0};
            } else mine[i] = row_by_row(idx);
        }
        if (dealt == 3) {  // the last round's key tiles one behind the other, CH_REST_TILES of its tiles of queries to a thread
            ChunkDeal d[CH_REST_TILES];
            int count[CH_REST_TILES], before = 0, sum = 0;
#pragma unroll
            for (int j = 0; j < CH_REST_TILES; ++j) {
                const int idx = limit + tid * CH_REST_TILES + j;
                count[j] = 0;
                if (idx < items) {
                    d[j] = row_by_row(idx);
                    count[j] = chunk_span(p, ChunkRow{d[j].L, d[j].n}, d[j].local / p.Hkv * p.tile_tokens).count;
                }
                sum += count[j];
            }
            before = sum;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, before, off);
                if (lane >= off) before += v;
            }
            if (lane == 31) s_sum[warp] = before;
            __syncthreads();
            before -= sum;
            int total = 0;
            for (int w = 0; w < CH_THREADS / 32; ++w) {
                if (w < warp) before += s_sum[w];
                total += s_sum[w];
            }
            const int each = max((total + grid - 1) / grid, CH_REST), from = (int)min((long long)c * each, (long long)total), end = min(from + each, total);
#pragma unroll
            for (int j = 0; j < CH_REST_TILES; ++j) {
                const int upto = before + count[j], number = tid * CH_REST_TILES + j;
                if (from < end && from >= before && from < upto) {
                    s_sum[8] = number;
                    const int hkv = d[j].local % p.Hkv, t0 = d[j].local / p.Hkv * p.tile_tokens;
                    p.plan[c] = ChunkPlan{from, from - before, count[j], d[j].b, hkv, t0, 0, each, d[j].n, {0, 0, 0}};
                }
                if (from < end && end > before && end <= upto) s_sum[9] = number;
                before = upto;
            }
            __syncthreads();
            if (from < end) {
                const int first = s_sum[8];
                before -= sum;
#pragma unroll
                for (int j = 0; j < CH_REST_TILES; ++j) {
                    const int lo = max(from, before), hi = min(end, before + count[j]);
                    if (lo < hi) {
                        d[j].off = lo - before;
                        d[j].n_tiles = hi - lo;
                        d[j].slot = hi - lo == count[j] ? -1 : c * 2 + (lo != from);
                        mine[deals + tid * CH_REST_TILES + j - first] = d[j];
                    }
                    before += count[j];
                }
                deals += s_sum[9] - first + 1;
            }
        }
    }
    // A warp to a phase: its stretch of this CTA.
    if (!dealt && warp < p.phases) {
        auto place = [&](int pair) {  // key tiles before a (row, kv head)
            const int b = pair / p.Hkv;
            return b < p.B ? s_place[b] + (pair - b * p.Hkv) * s_tiles[b] : all;
        };
        const int lo = place(warp * p.phase_pairs), hi = place(min((warp + 1) * p.phase_pairs, p.B * p.Hkv));
        const int each = max((hi - lo + (int)gridDim.x - 1) / (int)gridDim.x, CH_MIN_TILES);
        const int from = (int)min(lo + (long long)each * blockIdx.x, (long long)hi);
        if (from < hi) {
            int row = -1;
            for (int b0 = 0; row < 0; b0 += 32) {  // the row that holds key tile `from`
                const int b = b0 + lane;
                const unsigned votes = __ballot_sync(0xffffffffu, b < p.B && s_place[b] <= from && from < s_place[b] + s_tiles[b] * p.Hkv);
                if (votes) row = b0 + __ffs(votes) - 1;
            }
            const ChunkRow r = chunk_row(p, row);
            ChunkStretch st;
            st.at = from;
            st.end = min(from + each, hi);
            st.b = row;
            const int rel = from - s_place[row];
            st.hkv = rel / s_tiles[row];
            int off = rel - st.hkv * s_tiles[row], count = 0;
            for (int qt0 = 0;; qt0 += 32) {  // and the tile of queries
                count = chunk_span(p, r, (qt0 + lane) * p.tile_tokens).count;
                int upto = count;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, upto, d);
                    if (lane >= d) upto += v;
                }
                const unsigned votes = __ballot_sync(0xffffffffu, off < upto);
                if (votes) {
                    const int l = __ffs(votes) - 1;
                    off -= __shfl_sync(0xffffffffu, upto - count, l);
                    count = __shfl_sync(0xffffffffu, count, l);
                    st.qt = qt0 + l;
                    break;
                }
                off -= __shfl_sync(0xffffffffu, upto, 31);
            }
            st.off = off;
            if (lane == 0) {
                s_stretch[warp] = st;
                p.plan[warp * gridDim.x + blockIdx.x] = ChunkPlan{st.at, off, count, row, st.hkv, st.qt * p.tile_tokens, lo, each, r.n, {0, 0, 0}};
            }
        }
    }
    fence_proxy_async_smem();  // the sums' place is K's from here on
    __syncthreads();
    }
    pdl_launch_dependents();  // the sums of parts: their CTAs wait where there is room for them
    const uint32_t tmem_base = *tmem_slot;
    const uint32_t tmem_s = tmem_base, tmem_o = tmem_base + 128;
    const uint32_t lane_sel = (uint32_t)((warp & 3) * 32) << 16;  // a warp reaches TMEM lanes 32*(warp % 4) ..

    constexpr uint32_t IDESC_S = umma_idesc(CH_M, CH_N, 0, 0);
    constexpr uint32_t IDESC_O = umma_idesc(CH_M, NCKV_D, 0, 1);
    auto timed_out = [&]() {
        *abort_flag = 1;
        atomicOr(p.status, (int)NCKV_ST_TIMEOUT);
    };
    auto par2 = [](uint32_t g) -> uint32_t { return (g >> 1) & 1u; };

    if (warp == CH_M / 32 + 1) {
        // =============== one lane moves the tiles ===================================================
        if (elect_one()) {
            ChunkCursor kc;  // next K tile
            if constexpr (CLUSTER) {
                kc.u = mine;
                kc.t = 0;
                kc.valid = mine.n_tiles > 0;
            } else {
                kc.start(p, s_stretch, deals);
            }
            uint32_t gk = 0, gv = 0, nu = 0, nq = 0;  // copies issued; pieces posted, their Q tiles asked for
            auto post = [&](bool more) {
                ChunkUnit &u = ring[nu % CH_RING];
                u = kc.u;
                if (!more) u.n_tiles = 0;
                mbar_arrive(&bar_u[nu % CH_RING]);
                ++nu;
            };
            // Where a tile lies, looked up a tile ahead of its copies: `keys` of it in one page, the rest at the next one's front.  Parts outside
            // [kv_lo, kv_hi) need no page: they read as zeros, as pages outside the pool do.
            struct Places {
                int idx, tok;  // page of the row, and token in it at which the tile begins
                int page[2], need, keys;
            };
            auto look_up = [&](Places &pl, const ChunkUnit &u, int t) {
                const int key0 = (u.tile0 + t) * CH_N;
                if (t == 0) {
                    pl.idx = key0 / p.page_tokens;
                    pl.tok = key0 - pl.idx * p.page_tokens;
                } else {
                    pl.tok += CH_N;
                    if (pl.tok >= p.page_tokens) {
                        pl.tok -= p.page_tokens;
                        ++pl.idx;
                    }
                    if (pl.tok >= p.page_tokens) {  // pages of 48
                        pl.tok -= p.page_tokens;
                        ++pl.idx;
                    }
                }
                pl.keys = min(CH_N, p.page_tokens - pl.tok);
                const int32_t *row = p.table + (long long)u.b * p.max_pages + pl.idx;
                pl.need = 0;
                if (key0 + pl.keys > u.kv_lo) {  // key0 < kv_hi for every tile
                    pl.page[0] = __ldg(row);
                    pl.need = 1;
                }
                if (pl.keys < CH_N && key0 + pl.keys < u.kv_hi) {  // and its last key is one of the piece's or behind them
                    pl.page[1] = __ldg(row + 1);
                    pl.need |= 2;
                }
            };
            auto load_tile = [&](uint8_t *dst, const CUtensorMap *map, uint64_t *bar, const Places &pl, int hkv) {
                mbar_arrive_expect_tx(bar, CH_KV_BYTES);
                int page0 = p.n_pages, page1 = p.n_pages;
                if (pl.need & 1) page0 = pl.page[0];
                if (pl.need & 2) page1 = pl.page[1];
                if (((pl.need & 1) && (unsigned)page0 >= (unsigned)p.n_pages) || ((pl.need & 2) && (unsigned)page1 >= (unsigned)p.n_pages)) {
                    atomicOr(p.status, (int)NCKV_ST_BAD_PAGE);
                    page0 = min((unsigned)page0, (unsigned)p.n_pages);
                    page1 = min((unsigned)page1, (unsigned)p.n_pages);
                }
                const CUtensorMap *m = map + (pl.keys / 16 - 1);
                tma_load_4d(dst, m, bar, 0, hkv, pl.tok, page0);
                tma_load_4d(dst + CH_KV_BYTES / 2, m, bar, 64, hkv, pl.tok, page0);
                if (pl.keys < CH_N) {
                    m = map + (CH_N - pl.keys) / 16 - 1;
                    dst += pl.keys * 128;
                    tma_load_4d(dst, m, bar, 0, hkv, 0, page1);
                    tma_load_4d(dst + CH_KV_BYTES / 2, m, bar, 64, hkv, 0, page1);
                }
            };
            Places kp, vp;
            uint32_t vu = 0;  // piece and key tile of the next V tile
            int vt = 0;
            bool v_known = true;  // its places
            auto load_k = [&]() {
                const int stage = (int)(gk % CH_STAGES);
                load_tile(sK + stage * CH_KV_BYTES, maps.k, &bar_k[stage], kp, kc.u.hkv);
                const bool ends = kc.last_of_unit();
                if constexpr (CLUSTER) kc.valid = ++kc.t < mine.n_tiles;
                else kc.advance(p, s_stretch);
                ++gk;
                if (ends) post(kc.valid);
                if (kc.valid) look_up(kp, kc.u, kc.t);
            };
            auto load_v = [&]() {
                const int stage = (int)(gv % CH_VSTAGES);
                const ChunkUnit &u = ring[vu % CH_RING];
                if (!v_known) look_up(vp, u, vt);
                load_tile(sV + stage * CH_KV_BYTES, maps.v, &bar_v[stage], vp, u.hkv);
                ++gv;
                if (++vt == u.n_tiles) {
                    vt = 0;
                    ++vu;
                }
                v_known = gv < gk;  // V follows K: its piece is posted
                if (v_known) look_up(vp, ring[vu % CH_RING], vt);
            };
            auto load_q = [&]() {
                const ChunkUnit &u = ring[nq % CH_RING];
                const uint32_t buf = nq % q_bufs;
                uint8_t *dst = sQ + 2 * buf * q_half;
                mbar_arrive_expect_tx(&bar_q[buf], (uint32_t)(p.tile_tokens * p.G * NCKV_D * 2));
                tma_load_4d(dst, &maps.q, &bar_q[buf], 0, u.hkv * p.G, u.t0, u.b);
                tma_load_4d(dst + q_half, &maps.q, &bar_q[buf], 64, u.hkv * p.G, u.t0, u.b);
                ++nq;
            };
            bool ok = true;
            post(kc.valid);
            if (kc.valid) {
                load_q();
                look_up(kp, kc.u, 0);
                look_up(vp, kc.u, 0);
                // V behind K, whose pieces it takes
                while (gk < CH_STAGES && kc.valid) load_k();
                while (gv < CH_VSTAGES && gv < gk) load_v();
                uint32_t wu = 0;  // piece of the tile whose score product is awaited
                int left = ring[0].n_tiles;
                for (uint32_t g = 0;; ++g) {
                    // Q of a piece ahead where there is room for it
                    while (nq < wu + q_bufs && nq < nu && ring[nq % CH_RING].n_tiles) load_q();
                    // what S(g)'s completion releases: a Q buffer if g ends its piece, K(g)'s stage for
                    // K(g+2) and, P V(g-2) being complete too, V(g-2)'s stage for V(g+1)
                    ok = mbar_wait_bounded(&bar_s[g & 1], par2(g));
                    if (!ok) break;
                    if (--left == 0) {  // the next piece was posted behind the copy of this one's last keys
                        left = ring[++wu % CH_RING].n_tiles;
                        if (left == 0) break;
                    }
                    if (kc.valid) load_k();
                    while (gv < gk && gv <= (g ? g + 1 : CH_VSTAGES - 1)) load_v();
                }
            }
            if (!ok) timed_out();
            if (*abort_flag) {  // the last copies may still be under way
                for (uint32_t s = 0; s < q_bufs && s < nq; ++s) mbar_wait_bounded(&bar_q[(nq - 1 - s) % q_bufs], ((nq - 1 - s) / q_bufs) & 1u);
                for (uint32_t s = 0; s < CH_STAGES && s < gk; ++s) mbar_wait_bounded(&bar_k[(gk - 1 - s) % CH_STAGES], ((gk - 1 - s) / CH_STAGES) & 1u);
                for (uint32_t s = 0; s < CH_VSTAGES && s < gv; ++s) mbar_wait_bounded(&bar_v[(gv - 1 - s) % CH_VSTAGES], ((gv - 1 - s) / CH_VSTAGES) & 1u);
            }
        }
        __syncwarp();
    } else if (warp == CH_M / 32) {
        // =============== one thread feeds the tensor core ==========================================
        if (elect_one()) {
            const uint64_t desc_q = smem_desc_sw128(smem_u32(sQ), 16, 1024);
            const uint64_t desc_k = smem_desc_sw128(smem_u32(sK), 16, 1024);
            const uint64_t desc_v = smem_desc_sw128(smem_u32(sV), CH_KV_BYTES / 2, 1024);
            uint32_t gs = 0, gp = 0, su = 0, pu = 0;  // tiles and pieces of the next score product and of the next P V product
            int s_n = 0, s_t = 0, p_t = 0;            // key tiles of the piece; tile inside it
            auto next_piece = [&]() -> bool {
                if (!mbar_wait_bounded(&bar_u[su % CH_RING], (su / CH_RING) & 1u)) return false;
                s_n = ring[su % CH_RING].n_tiles;
                return true;
            };
            auto issue_s = [&]() -> bool {
                const uint32_t stage = gs % CH_STAGES;
                const uint32_t buf = su % q_bufs;
                if (s_t == 0 && !mbar_wait_bounded(&bar_q[buf], (su / q_bufs) & 1u)) return false;  // first tile of a piece: its Q
                if (!mbar_wait_bounded(&bar_k[stage], (gs / CH_STAGES) & 1u)) return false;
                tc_fence_after();
                const uint64_t dk = desc_k + (uint64_t)((stage * CH_KV_BYTES) >> 4);
                const uint32_t ds = tmem_s + (gs & 1u) * CH_N;
#pragma unroll
                for (int kk = 0; kk < NCKV_D / 16; ++kk) {
                    const uint32_t off = (uint32_t)(kk & 3) * 32;
                    const uint64_t da = desc_q + (uint64_t)(((2 * buf + (kk >> 2)) * q_half + off) >> 4);
                    const uint64_t db = dk + (uint64_t)(((kk >> 2) * (CH_KV_BYTES / 2) + off) >> 4);
                    umma_bf16(ds, da, db, IDESC_S, kk > 0 ? 1u : 0u);
                }
                umma_commit(&bar_s[gs & 1u]);
                ++gs;
                if (++s_t < s_n) return true;
                s_t = 0;
                ++su;
                return next_piece();
            };
            bool ok = next_piece();
            if (ok && s_n) ok = issue_s();
            if (ok && s_n) ok = issue_s();
            while (gp < gs && ok) {
                // P(gp) is in TMEM, S(gp) has been read, O carries the scale P was made with
                const uint32_t vstage = gp % CH_VSTAGES;
                ok = mbar_wait_bounded(&bar_p[gp & 1u], par2(gp)) && mbar_wait_bounded(&bar_v[vstage], (gp / CH_VSTAGES) & 1u);
                if (!ok) break;
                tc_fence_after();
                const uint64_t dv = desc_v + (uint64_t)((vstage * CH_KV_BYTES) >> 4);
                const uint32_t pbase = tmem_s + (gp & 1u) * CH_N;
#pragma unroll
                for (int ks = 0; ks < CH_N / 16; ++ks) {
                    const uint64_t db = dv + (uint64_t)((ks * 16 * 128) >> 4);
                    umma_bf16_a_tmem(tmem_o, pbase + (uint32_t)ks * 8, db, IDESC_O, (p_t > 0 || ks > 0) ? 1u : 0u);
                }
                const int from_end = ring[pu % CH_RING].n_tiles - 1 - p_t;
                if (from_end < 2) umma_commit(&bar_o[from_end]);
                if (s_n) ok = issue_s();
                ++p_t;
                if (from_end == 0) {
                    p_t = 0;
                    ++pu;
                }
                ++gp;
            }
            if (!ok) timed_out();
        }
        __syncwarp();
    } else {
        // =============== softmax threads: one per query row =========================================
        const int row = tid, tok = row / p.G, head = row - tok * p.G;
        if (any_idle) {  // zeros, a share of the slots per CTA
            for (int b = 0; b < p.B; ++b) {
                const int n = chunk_row(p, b).n;
                if (n == p.T) continue;
                const long long words = (long long)(p.T - n) * p.Hq * (NCKV_D / 8);
                uint4 *dst = reinterpret_cast<uint4 *>(p.out + ((long long)b * p.T + n) * p.Hq * NCKV_D);
                for (long long i = (long long)blockIdx.x * CH_M + tid; i < words; i += (long long)gridDim.x * CH_M) dst[i] = make_uint4(0, 0, 0, 0);
            }
        }
        bool aborted = false;
        uint32_t g = 0;               // number of the current piece's tile 0 in the stream
        uint32_t n_o0 = 0, n_o1 = 0;  // phases of bar_o[0] / bar_o[1] used up by the pieces before this one
        auto warp_wait = [&](uint64_t *bar, uint32_t parity) -> bool {
            if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
            int ok = *abort_flag == 0;
            if (lane == 0 && ok) ok = mbar_wait_bounded(bar, parity) ? 1 : 0;
            ok = __shfl_sync(0xffffffffu, ok, 0);
            __syncwarp();  // orders the lanes' later reads of the tile behind lane 0's observation
            return ok != 0;
        };
        for (uint32_t seq = 0; !aborted; ++seq) {
            if (!warp_wait(&bar_u[seq % CH_RING], (seq / CH_RING) & 1u)) {
                aborted = true;
                break;
            }
            const ChunkUnit it = ring[seq % CH_RING];
            if (it.n_tiles == 0) break;
            const int n_tiles = it.n_tiles, first_pos = it.L + it.t0, tokens = min(p.tile_tokens, it.n - it.t0);
            const int pos = first_pos + tok;  // absolute position of this row's token
            const bool live = tok < tokens;
            const bool warp_live = warp * 32 < tokens * p.G;  // the other warps only keep the barriers going
            auto pv_done = [&](int t) -> bool {
                const int from_end = n_tiles - 1 - t;
                const uint32_t x = g + (uint32_t)t;
                return from_end >= 2 ? warp_wait(&bar_s[(x + 2) & 1u], par2(x + 2)) : warp_wait(&bar_o[from_end], (from_end == 0 ? n_o0 : n_o1) & 1u);
            };
            // P is scaled by m_used, which follows the running maximum lazily: it is only raised (and the O row in TMEM
            // rescaled) when the maximum has grown by more than 2^8
            float m_used = -INFINITY, l_run = 0.f;
            for (int t = 0; t < n_tiles; ++t) {
                const uint32_t gt = g + (uint32_t)t;
                const int key0 = (it.tile0 + t) * CH_N;
                const uint32_t tmem_s_it = tmem_s + (uint32_t)(gt & 1) * CH_N;
                if (!warp_wait(&bar_s[gt & 1u], par2(gt))) {  // uniform over the warp
                    aborted = true;
                    break;
                }
                tc_fence_after();
                // tiles that some row of the piece doesn't see all of (uniform over the CTA)
                const bool edge = key0 + CH_N - 1 > first_pos || key0 < it.kv_lo ||
                                  (p.window_left >= 0 && key0 < first_pos + tokens - 1 - p.window_left);
                if (warp_live) {
                    float s_val[CH_N];
                    tmem_ld64(tmem_s_it + lane_sel, s_val);
                    if (edge) {
                        // this row sees columns [c_lo, c_hi) of the tile
                            const int c_hi = min(max(min(pos, it.kv_hi - 1) - key0 + 1, 0), CH_N);
                            const int c_lo = p.window_left >= 0 ? min(max(pos - p.window_left - key0, 0), CH_N) : 0;
                            const unsigned long long seen = (c_hi == CH_N ? ~0ull : (1ull << c_hi) - 1) & (c_lo == CH_N ? 0ull : ~0ull << c_lo);
                            const uint32_t seen0 = (uint32_t)seen, seen1 = (uint32_t)(seen >> 32);
#pragma unroll
                            for (int c = 0; c < CH_N; ++c) s_val[c] = ((c < 32 ? seen0 : seen1) >> (c & 31) & 1u) ? s_val[c] : -INFINITY;
                    }
                    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int c = 0; c < CH_N; c += 8) {
                        mx4[0] = fmax3(mx4[0], s_val[c], s_val[c + 1]);
                        mx4[1] = fmax3(mx4[1], s_val[c + 2], s_val[c + 3]);
                        mx4[2] = fmax3(mx4[2], s_val[c + 4], s_val[c + 5]);
                        mx4[3] = fmax3(mx4[3], s_val[c + 6], s_val[c + 7]);
                    }
                    const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * p.scale_log2;
                    const bool raise = mx > m_used + 8.f;  // also the first tile that shows this row a key (m_used = -inf)
                    const float alpha = raise ? ex2_approx(m_used - mx) : 1.f;
                    if (raise) {
                        l_run *= alpha;
                        m_used = mx;
                    }
                    const float m_use = m_used == -INFINITY ? 0.f : m_used;  // a row that has seen no key yet
                    float2 rs01 = make_float2(0.f, 0.f), rs23 = make_float2(0.f, 0.f);
                    const float2 scale2 = make_float2(p.scale_log2, p.scale_log2), neg_m2 = make_float2(-m_use, -m_use);
                    uint32_t pk[CH_N / 2];
#pragma unroll
                    for (int c = 0; c < CH_N; c += 4) {
                        const float2 x01 = ffma2(make_float2(s_val[c], s_val[c + 1]), scale2, neg_m2);
                        const float2 x23 = ffma2(make_float2(s_val[c + 2], s_val[c + 3]), scale2, neg_m2);
                        const float2 p01 = make_float2(ex2_approx(x01.x), ex2_approx(x01.y));
                        const float2 p23 = make_float2(ex2_approx(x23.x), ex2_approx(x23.y));
                        rs01 = fadd2(rs01, p01);
                        rs23 = fadd2(rs23, p23);
                        pk[c / 2] = pack_bf16x2(p01.x, p01.y);
                        pk[c / 2 + 1] = pack_bf16x2(p23.x, p23.y);
                    }
                    l_run += (rs01.x + rs01.y) + (rs23.x + rs23.y);
                    tmem_st_words(tmem_s_it + lane_sel, pk);
                    if (t > 0 && __any_sync(0xffffffffu, raise)) {
                        if (!pv_done(t - 1)) {
                            timed_out();
                            aborted = true;
                            break;
                        }
                        tc_fence_after();
#pragma unroll
                        for (int ch = 0; ch < NCKV_D / 32; ++ch) {
                            float c[32];
                            tmem_ld32(tmem_o + lane_sel + ch * 32, c);
#pragma unroll
                            for (int i = 0; i < 32; ++i) c[i] *= alpha;
                            tmem_st32(tmem_o + lane_sel + ch * 32, c);
                        }
                    }
                }
                if (edge) {
                    // Keys that nobody of the piece sees may hold anything, keys that only some rows see may hold values that are not
                    // finite: a probability of zero must meet neither.
                    const int stage = (int)(gt % CH_VSTAGES), lo = it.kv_lo - key0, hi = it.kv_hi - key0;
                    uint8_t *vd = sV + stage * CH_KV_BYTES;
                    if (warp_wait(&bar_v[stage], (gt / CH_VSTAGES) & 1u)) {
#pragma unroll 2
                        for (int i = tid; i < CH_N * 16; i += CH_M) {
                            const int r = i >> 4, ch = i & 15;
                            uint4 *w = reinterpret_cast<uint4 *>(vd + (ch >> 3) * (CH_KV_BYTES / 2) + r * 128 + ((ch & 7) << 4));
                            if (r < lo || r >= hi) {
                                *w = make_uint4(0, 0, 0, 0);
                                continue;
                            }
                            uint4 x = *w;
                            if (not_finite2(x.x) | not_finite2(x.y) | not_finite2(x.z) | not_finite2(x.w)) {
                                uint16_t *e = reinterpret_cast<uint16_t *>(w);
                                for (int k = 0; k < 8; ++k)
                                    if ((e[k] & 0x7f80u) == 0x7f80u) e[k] = 0;
                                s_poison[seq & 3] = (int)seq;
                            }
                        }
                    }
                    fence_proxy_async_smem();  // the cleared values must be visible to the tensor core
                }
                tc_fence_before();  // orders this thread's TMEM loads/stores before the next MMAs
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar_p[gt & 1]);  // one arrival per warp
            }
            if (aborted) break;

            // ---- the piece's end ---------------------------------------------------------------------
            if (!pv_done(n_tiles - 1)) {
                timed_out();
                aborted = true;
                break;
            }
            tc_fence_after();
            if (warp_live) {
                const bool poison = s_poison[seq & 3] == (int)seq;
                const float inv = it.slot >= 0 ? 1.f : (l_run > 0.f ? 1.f / l_run : (l_run == l_run ? 0.f : l_run));
                const long long part = (long long)it.slot * p.part_rows + row;
                uint4 *dst = reinterpret_cast<uint4 *>(p.out + (((long long)it.b * p.T + it.t0 + tok) * p.Hq + it.hkv * p.G + head) * NCKV_D);
                if (it.slot >= 0 && live) (CLUSTER ? s_part_ml + row : reinterpret_cast<float2 *>(p.part_ml) + part)[0] = make_float2(m_used, l_run);
#pragma unroll
                for (int ch = 0; ch < NCKV_D / 32; ++ch) {
                    float c[32];
                    __syncwarp();
                    tmem_ld32(tmem_o + lane_sel + ch * 32, c);
                    if (live) {
                        if (poison) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) c[i] += chunk_not_finite(p, it, pos, ch * 32 + i);
                        }
                        if constexpr (CLUSTER) {
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                *reinterpret_cast<float4 *>(s_part + row * CH_PITCH + ch * 32 + i * 4) = make_float4(c[4 * i], c[4 * i + 1], c[4 * i + 2], c[4 * i + 3]);
                        } else if (it.slot >= 0) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                uint32_t w[8];
#pragma unroll
                                for (int e = 0; e < 8; ++e) w[e] = __float_as_uint(c[8 * i + e]);
                                st_global_v8(p.part_o + part * NCKV_D + ch * 32 + i * 8, w);
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < 2; ++i) {  // 32 bytes per store: whole sectors
                                uint32_t w[8];
#pragma unroll
                                for (int e = 0; e < 8; ++e) w[e] = pack_bf16x2(c[16 * i + 2 * e] * inv, c[16 * i + 2 * e + 1] * inv);
                                st_global_v8(dst + (ch * 2 + i) * 2, w);
                            }
                        }
                    }
                }
                __syncwarp();
            }
            // O is read: order those loads before the first P V of the next piece, which overwrites it and
            // is only issued after this thread's next arrival on bar_p
            tc_fence_before();
            g += (uint32_t)n_tiles;
            n_o0 += 1;
            n_o1 += n_tiles >= 2;
        }
        if (aborted && *abort_flag == 0) timed_out();  // a wait ran out in this warp
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem_base, CH_TMEM_COLS);
    if constexpr (CLUSTER) {  // rows rank, rank + ctas, ...: the parts in the order of the keys, as in chunk_finish_kernel
        const int ctas = (int)cluster_ctas(), rank = (int)cluster_rank(), rows = min(p.tile_tokens, mine.n) * p.G;
        cluster_sync();
        for (int row = rank + ctas * warp; row < rows; row += ctas * (CH_THREADS / 32)) {
            float2 ml[8];
            float4 x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {  // all of them on their way at once
                ml[i] = make_float2(-INFINITY, 0.f);
                x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i < ctas) {
                    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(ml[i].x), "=f"(ml[i].y) : "r"(smem_of_rank(s_part_ml + row, (uint32_t)i)) : "memory");
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                 : "=f"(x[i].x), "=f"(x[i].y), "=f"(x[i].z), "=f"(x[i].w)
                                 : "r"(smem_of_rank(s_part + row * CH_PITCH + lane * 4, (uint32_t)i))
                                 : "memory");
                }
            }
            float m = -INFINITY, l = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, ml[i].x);
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (ml[i].x == -INFINITY && ml[i].y == 0.f) continue;  // this row sees none of the part's keys; what lies there is nothing
                const float w = exp2f(ml[i].x - m);
                l += w * ml[i].y;
                o.x += w * x[i].x;
                o.y += w * x[i].y;
                o.z += w * x[i].z;
                o.w += w * x[i].w;
            }
            const int tok = row / p.G, head = mine.hkv * p.G + row - tok * p.G;
            const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
            reinterpret_cast<uint2 *>(p.out + (((long long)mine.b * p.T + tok) * p.Hq + head) * NCKV_D)[lane] =
                make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
        }
        __syncwarp();
        cluster_sync();  // the others may still be reading
    }
}

// Adds up the parts of a tile of queries whose keys were cut: O = sum 2^(m_s - M) O_s / sum 2^(m_s - M) l_s.  Block (CTA, rows, phase) looks at
// the cut where that CTA's stretch begins and takes the tile's rows if it is the tile's first cut; WARPS warps to a row, EACH rows
// one after the other.
template <int WARPS, int EACH>
__global__ void __launch_bounds__(256) chunk_finish_kernel(const __grid_constant__ ChunkParams p) {
    pdl_wait_prior_grids();
    __shared__ float4 s_o[WARPS > 1 ? 8 : 1][32];
    __shared__ float s_l[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, mine = warp % WARPS;
    const int c = (int)blockIdx.x, grid = (int)gridDim.x, phase = (int)blockIdx.z;
    const ChunkPlan cut = p.plan[phase * grid + c];
    if (cut.at < 0 || cut.off == 0) return;
    const int from = cut.at - cut.off - cut.begin, first = from / cut.each, last = (from + cut.count - 1) / cut.each, parts = last - first + 1;
    if (c != first + 1) return;
    const int rows = min(p.tile_tokens, cut.n - cut.t0) * p.G;
    const long long slot0 = ((long long)phase * grid + first) * 2;
    const bool second = first * cut.each < from;  // the first part is not the first piece of its stretch
    auto part_of = [&](int i, int row) -> long long { return (slot0 + 2 * i + (i == 0 && second)) * p.part_rows + row; };
    constexpr int STEP = 8 / WARPS;
    const int row0 = (int)blockIdx.y * STEP * EACH + warp / WARPS;
#pragma unroll 1
    for (int k = 0; k < EACH; ++k) {
        const int row = row0 + k * STEP;
        if (row >= rows) return;  // uniform over the warps of a row
        // this warp's first two parts are asked for beside all parts' maxima
        constexpr int AHEAD = 2;
        float2 ml[AHEAD];
        float4 x[AHEAD];
#pragma unroll
        for (int k2 = 0; k2 < AHEAD; ++k2) {
            const int i = mine + k2 * WARPS;
            ml[k2] = make_float2(-INFINITY, 0.f);
            x[k2] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (i < parts) {
                ml[k2] = *reinterpret_cast<const float2 *>(p.part_ml + part_of(i, row) * 2);
                x[k2] = reinterpret_cast<const float4 *>(p.part_o + part_of(i, row) * NCKV_D)[lane];
            }
        }
        float m = -INFINITY, l = 0.f;
        for (int i = lane; i < parts; i += 32) m = fmaxf(m, p.part_ml[part_of(i, row) * 2]);
#pragma unroll
        for (int off = 16; off; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](float2 part, float4 v) {
            if (part.x == -INFINITY && part.y == 0.f) return;  // this row sees none of the part's keys
            const float w = exp2f(part.x - m);
            l += w * part.y;
            o.x += w * v.x;
            o.y += w * v.y;
            o.z += w * v.z;
            o.w += w * v.w;
        };
#pragma unroll
        for (int k2 = 0; k2 < AHEAD; ++k2) add(ml[k2], x[k2]);
#pragma unroll 4
        for (int i = mine + AHEAD * WARPS; i < parts; i += WARPS)
            add(*reinterpret_cast<const float2 *>(p.part_ml + part_of(i, row) * 2), reinterpret_cast<const float4 *>(p.part_o + part_of(i, row) * NCKV_D)[lane]);
        if constexpr (WARPS > 1) {
            s_o[warp][lane] = o;
            if (lane == 0) s_l[warp] = l;
            __syncthreads();
            if (mine) return;
#pragma unroll
            for (int w = 1; w < WARPS; ++w) {
                const float4 x = s_o[warp + w][lane];
                l += s_l[warp + w];
                o.x += x.x;
                o.y += x.y;
                o.z += x.z;
                o.w += x.w;
            }
        }
        const int tok = row / p.G, head = cut.hkv * p.G + row - tok * p.G;
        const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
        reinterpret_cast<uint2 *>(p.out + (((long long)cut.b * p.T + cut.t0 + tok) * p.Hq + head) * NCKV_D)[lane] =
            make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
    }
}

static size_t chunk_smem_bytes(int part_rows) {
    return 2 * (part_rows <= CH_M / 2 ? 2 : 1) * chunk_q_half(part_rows) + (CH_STAGES + CH_VSTAGES) * CH_KV_BYTES + (13 + CH_RING) * sizeof(uint64_t) + CH_RING * sizeof(ChunkUnit) + 6 * 4 +
           CH_PHASES * sizeof(ChunkStretch);
}
static_assert(CH_RING * sizeof(ChunkUnit) >= 36 * 4, "the sums over the rows lie where the pieces come later");

// How a launch of these sizes is cut: what of it doesn't depend on the rows' lengths.
struct ChunkShape {
    int G, tile_tokens, n_qtiles, grid, phases, phase_pairs, part_rows;
    int ctas;  // of a cluster; 0: no clusters
    long long n_items;
    int deal_room;
    size_t plan_bytes, deal_bytes;
};
// CTAs to a pair (0: stretches) where rows have one tile of queries: as many as the chip has room for at once (two per SM, some lost between
// clusters of 4 and 8), if a CTA's key tiles are then few and not many more than a stretch would have.  Lengths aren't known here, a full table is
// taken for them.  us as stretches / clusters of 2 / 4 / 8, 6 + 6 heads, 4 tokens: 4 rows of up to 500 keys 11.8 / 9.3 / 9.0 / 8.6, 8 12.8 / 10.2 / 9.5 / 16.4,
// 24 18.8 / 11.4 / 22.6 / 39.3; 4 rows of 4000 20.6 / 35.2 / 22.5 / 17.7, 2 of 8000 19.7 / 58.4 / 34.9 / 23.0; 16 rows of 4000, 16 + 4 heads 38.5 / 36.1 / 27.7 /
// 36.6.  With 128 query rows stretches leave much larger partial sums: 4 x 32 tokens behind 8000, 16 + 4 heads 37.6 / 60.9 / 37.9 / 29.2.
constexpr int CH_SHARE = 16;
static int chunk_cluster(long long pairs, long long key_tiles, int part_rows) {
    const long long room = 2LL * sm_count(), stretch = pairs * key_tiles / room;
    for (int ctas = 8; ctas >= 1; ctas /= 2) {
        if (pairs * ctas > (ctas > 2 ? room * 9 / 10 : room)) continue;
        const long long share = (key_tiles + ctas - 1) / ctas;
        return share <= CH_SHARE && share <= stretch + (part_rows <= 32 ? 8 : 20) ? ctas : 0;
    }
    return 0;
}
static ChunkShape chunk_shape(int B, int T, int Hq, int Hkv, long long capacity, long long window_left) {
    ChunkShape s;
    s.G = Hq / Hkv;
    s.tile_tokens = CH_M / s.G < T ? CH_M / s.G : T;
    s.n_qtiles = (T + s.tile_tokens - 1) / s.tile_tokens;
    s.n_items = (long long)B * Hkv * s.n_qtiles;
    s.part_rows = s.tile_tokens * s.G;
    const int most = 2 * sm_count();  // two CTAs per SM
    const long long key_tiles = (capacity + CH_N - 1) / CH_N, pairs = (long long)B * Hkv;
    s.grid = (int)(s.n_items * key_tiles < most ? s.n_items * key_tiles : most);
    long long keys = window_left >= 0 && window_left + T < capacity ? window_left + T : capacity;
    s.phases = 1;
    if (s.n_qtiles > 1) {
        long long n = (pairs * keys * 512 + CH_PHASE_BYTES - 1) / CH_PHASE_BYTES;
        const long long room = CH_PART_BYTES / ((long long)2 * s.grid * s.part_rows * (NCKV_D + 2) * 4);
        n = n < room ? n : room;
        n = n < pairs ? n : pairs;
        s.phases = (int)(n < 1 ? 1 : n < CH_PHASES ? n : CH_PHASES);
    }
    s.phase_pairs = (int)((pairs + s.phases - 1) / s.phases);
    s.phases = (int)((pairs + s.phase_pairs - 1) / s.phase_pairs);
    if (s.grid == 1) s.phases = 0;
    s.ctas = s.n_qtiles == 1 && s.grid > 1 ? chunk_cluster(pairs, (keys + CH_N - 1) / CH_N, s.part_rows) : 0;
    if (s.ctas) {
        s.grid = (int)pairs * s.ctas;
        s.phases = 0;
    }
    s.plan_bytes = ((size_t)s.phases * s.grid * sizeof(ChunkPlan) + 255) / 256 * 256;
    s.deal_room = (int)(s.n_items / s.grid + 1) + s.grid;  // (a last round that is cut: fewer parts than it has tiles)
    // (rows of one tile of queries are never dealt, but for the one CTA of a grid of one)
    s.deal_bytes = s.ctas || (s.n_qtiles == 1 && s.grid > 1) ? 0 : ((size_t)s.grid * s.deal_room * sizeof(ChunkDeal) + 255) / 256 * 256;
    return s;
}
static size_t chunk_workspace(const ChunkShape &s) {
    return s.deal_bytes + (s.phases ? s.plan_bytes + (size_t)s.phases * 2 * s.grid * s.part_rows * (NCKV_D + 2) * 4 : 0);
}
static int chunk_check_sizes(const char *name, int B, int T, int Hq, int Hkv, int page_tokens, int max_pages) {
    if (B <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || page_tokens <= 0 || max_pages <= 0) {
        set_error("%s: non-positive size (B=%d T=%d Hq=%d Hkv=%d page_tokens=%d max_pages=%d)", name, B, T, Hq, Hkv, page_tokens, max_pages);
        return NCKV_E_ARG;
    }
    if (B > CH_ROWS) {
        set_error("%s: B=%d rows, at most %d", name, B, CH_ROWS);
        return NCKV_E_UNSUPPORTED;
    }
    if (Hq % Hkv != 0 || Hq / Hkv > CH_M) {
        set_error("%s: Hq=%d must be a multiple of Hkv=%d, at most %d times it", name, Hq, Hkv, CH_M);
        return NCKV_E_UNSUPPORTED;
    }
    if (page_tokens % nckv_paged_tile_tokens() != 0) {
        set_error("%s: page_tokens=%d must be a multiple of %d", name, page_tokens, nckv_paged_tile_tokens());
        return NCKV_E_ARG;
    }
    const long long capacity = (long long)page_tokens * max_pages;
    const long long key_tiles = (capacity + CH_N - 1) / CH_N, pairs = (long long)B * Hkv;
    if (capacity > 0x3fffffffLL || pairs > 0x3fffffffLL || pairs * T > 0x3fffffffLL ||
        pairs * ((T + CH_M / (Hq / Hkv) - 1) / (CH_M / (Hq / Hkv))) > 0x3fffffffLL / key_tiles) {
        set_error("%s: B=%d T=%d Hkv=%d with %lld tokens of capacity is too large for one launch", name, B, T, Hkv, capacity);
        return NCKV_E_UNSUPPORTED;
    }
    return NCKV_OK;
}

}  // namespace nckv

extern "C" size_t nckv_prefill_attn_paged_workspace_bytes(int B, int T, int Hq, int Hkv, int page_tokens, int max_pages, int window_left) {
    using namespace nckv;
    if (chunk_check_sizes("prefill_attn_paged_workspace_bytes", B, T, Hq, Hkv, page_tokens, max_pages) != NCKV_OK) return 0;
    return chunk_workspace(chunk_shape(B, T, Hq, Hkv, (long long)page_tokens * max_pages, window_left));
}

extern "C" int nckv_prefill_attn_paged(const void *q, const void *k_pool, const void *v_pool, const int32_t *block_table,
                                       const int32_t *cache_seqlens, const int32_t *new_tokens, void *out, int B, int T, int Hq, int Hkv,
                                       int D, int page_tokens, int max_pages, int n_pages, int64_t page_stride, int64_t token_stride,
                                       int window_left, void *workspace, size_t workspace_bytes, int32_t *status, void *stream) {
    using namespace nckv;
    const char *name = "prefill_attn_paged";
    if (!q || !k_pool || !v_pool || !block_table || !cache_seqlens || !out || !status) {
        set_error("%s: null pointer argument", name);
        return NCKV_E_ARG;
    }
    if (D != NCKV_D) {
        set_error("%s: head_dim %d unsupported (kernels are built for 128)", name, D);
        return NCKV_E_UNSUPPORTED;
    }
    int rc = chunk_check_sizes(name, B, T, Hq, Hkv, page_tokens, max_pages);
    if (rc != NCKV_OK) return rc;
    if (n_pages <= 0 || page_stride < 0) {
        set_error("%s: n_pages=%d must be positive", name, n_pages);
        return NCKV_E_ARG;
    }
    if (((uintptr_t)q & 15) || ((uintptr_t)out & 31)) {
        set_error("%s: q must be 16-byte and out 32-byte aligned", name);
        return NCKV_E_ARG;
    }
    const ChunkShape s = chunk_shape(B, T, Hq, Hkv, (long long)page_tokens * max_pages, window_left);
    const size_t need = chunk_workspace(s);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255))) {
        set_error("%s: needs %zu bytes of workspace, 256-byte aligned", name, need);
        return workspace && workspace_bytes < need ? NCKV_E_CAPACITY : NCKV_E_ARG;
    }
    ChunkMaps maps;
    const int64_t dims[4] = {D, Hq, T, B}, strides[3] = {D, (int64_t)Hq * D, (int64_t)T * Hq * D};
    const int q_box[4] = {64, s.G, s.tile_tokens, 1};
    rc = make_tensor_map(&maps.q, q, 4, dims, strides, q_box);
    for (int i = 0; i < 4 && rc == NCKV_OK; ++i) {
        if (i < 3 && page_tokens % CH_N == 0) continue;  // tiles lie in one page
        rc = make_kv_tensor_map(&maps.k[i], k_pool, n_pages, page_tokens, Hkv, page_stride, token_stride, 16 * (i + 1));
        if (rc == NCKV_OK) rc = make_kv_tensor_map(&maps.v[i], v_pool, n_pages, page_tokens, Hkv, page_stride, token_stride, 16 * (i + 1));
    }
    if (rc != NCKV_OK) return rc;

    ChunkParams p;
    p.table = block_table;
    p.seqlens = cache_seqlens;
    p.new_tokens = new_tokens;
    p.v_pool = static_cast<const __nv_bfloat16 *>(v_pool);
    p.out = static_cast<__nv_bfloat16 *>(out);
    p.deals = static_cast<ChunkDeal *>(workspace);
    p.deal_room = s.deal_room;
    char *const rest = static_cast<char *>(workspace) + s.deal_bytes;
    p.plan = reinterpret_cast<ChunkPlan *>(rest);
    p.part_o = p.part_ml = nullptr;
    if (s.phases) {
        p.part_o = reinterpret_cast<float *>(rest + s.plan_bytes);
        p.part_ml = p.part_o + (size_t)s.phases * 2 * s.grid * s.part_rows * NCKV_D;
    }
    p.status = status;
    p.B = B; p.T = T; p.Hq = Hq; p.Hkv = Hkv; p.G = s.G; p.tile_tokens = s.tile_tokens; p.n_qtiles = s.n_qtiles;
    p.page_tokens = page_tokens; p.max_pages = max_pages; p.n_pages = n_pages; p.capacity = page_tokens * max_pages;
    p.page_stride = page_stride; p.token_stride = token_stride;
    p.window_left = window_left;
    p.phases = s.phases; p.phase_pairs = s.phase_pairs; p.part_rows = s.part_rows;
    p.scale_log2 = (float)(1.4426950408889634 / sqrt((double)D));
    {
        // Pairs per group: all of them while their keys and values fit a third of L2, else as many as do, rounded down to a
        // number whose tiles are a multiple of two rounds of the CTAs (dealt back and forth, every CTA then gets the same mix).
        const long long keys = window_left >= 0 && (long long)window_left + CH_M < p.capacity ? window_left + CH_M : p.capacity;
        const long long pairs = (long long)B * Hkv, bytes_per_pair = keys * 512 + 1;
        long long g = pairs;
        if (pairs * bytes_per_pair > (40LL << 20)) {
            g = (40LL << 20) / bytes_per_pair;
            long long a = 2LL * s.grid, b = s.n_qtiles;
            while (b) { const long long t = a % b; a = b; b = t; }
            const long long unit = 2LL * s.grid / a;  // pairs
            if (g >= unit) g -= g % unit;
            if (g < 1) g = 1;
            if (g > pairs) g = pairs;
        }
        p.n_groups = (int)(pairs / g);  // the last group also takes the remainder
        p.group_pairs = (int)g;
    }
    const size_t smem = chunk_smem_bytes(s.part_rows);
    const int ctas = s.ctas;
    static bool attr_set[64] = {false};
    int dev = 0;
    NCKV_CUDA_CHECK(cudaGetDevice(&dev));
    if (dev >= 64 || !attr_set[dev]) {
        NCKV_CUDA_CHECK(cudaFuncSetAttribute(chunk_attn_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)chunk_smem_bytes(CH_M)));
        NCKV_CUDA_CHECK(cudaFuncSetAttribute(chunk_attn_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)chunk_smem_bytes(CH_M)));
        if (dev < 64) attr_set[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)s.grid);
    cfg.blockDim = dim3(CH_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)ctas;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctas ? 2 : 1;
    if (ctas) {
        NCKV_CUDA_CHECK(cudaLaunchKernelEx(&cfg, chunk_attn_kernel<true>, maps, p));
        return NCKV_OK;
    }
    NCKV_CUDA_CHECK(cudaLaunchKernelEx(&cfg, chunk_attn_kernel<false>, maps, p));
    if (s.phases) {
        // few rows: all of a block's warps to one, over the parts
        const bool wide = s.part_rows <= 16;
        const int step = wide ? 1 : s.part_rows <= 64 ? 8 : 16;
        cfg.gridDim = dim3((unsigned)s.grid, (unsigned)((s.part_rows + step - 1) / step), (unsigned)s.phases);
        cfg.blockDim = dim3(256);
        cfg.dynamicSmemBytes = 0;
        NCKV_CUDA_CHECK(cudaLaunchKernelEx(&cfg, wide ? chunk_finish_kernel<8, 1> : step == 8 ? chunk_finish_kernel<1, 1> : chunk_finish_kernel<1, 2>, p));
    }
    return NCKV_OK;
}
