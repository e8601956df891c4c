// Low-rank adapters of many requests beside a projection that all of them share: for row r of request b with slot s = slots[b],
//   out_r = bf16(y_r + scale_s up_s (down_s x_r)),   out_r = y_r where s is negative,
// down (S, R, K), up (S, N, R), R at most 128.  Sums are fp32; between the products t = down x is split into two bf16 terms (16 bits), so that
// nothing but the result is rounded to the activations' type.
//
// Requests of few tokens (decode, drafted tokens; many: adapters_tc.cu): memory-bound, on the adapters' bytes.  8 rows of one slot make a unit,
// T tokens of a request or requests of the same slot together, so that an adapter is read once for all of them; which requests a unit has
// every CTA finds from the slots.  A cluster of CTAs takes a unit in one launch: each CTA multiplies its part of the channels, the parts of t
// meet through distributed shared memory in the order of the ranks, and each CTA adds its part of the outputs to y.  Every warp streams its own
// part of the weights through a ring of its own by TMA, `up` right behind `down`, so that the first outputs' weights arrive while t is still on
// its way: boxes of 64 channels of 32 ranks, then 32 outputs by up to 64 ranks.  (By 16-byte asynchronous copies, whose addresses the lanes
// work out, 256 requests at rank 64 took 32 us where this form of copies took 21; straight from global memory to registers 34.)
// 256 rows over 48 adapters of rank 64, 2048 -> 8192 (72 MB): 19.1 us = 3.8 TB/s, 1.5 of them until a CTA knows its rows, 4.6 for its part of t, 2 until the
// parts have met and 7.4 for its part of the outputs; 64 rows of as many adapters, 2048 -> 2048 at rank 16: 6.7; 4 rows of 768 channels: 4.5 (latency).
// mma.sync with the weights as the 16 rows and the tokens as the 8 columns (tensor memory would want 128 rows): with the tokens as rows the
// instruction's rate was the limit.  Up to four tokens have both terms of t in one product.
#include "adapters.cuh"
#include "tc05.cuh"

namespace nckv {

constexpr int AD_THREADS = 256, AD_ROWS = 8, AD_AHEAD = 4;  // AD_AHEAD: groups of outputs whose y is on its way (1: 256 rows, 8192 outputs at rank 64 take 0.4 us more)
constexpr int AD_TABLE = 256;  // slots up to which requests are counted warp by warp: 2 KB
constexpr int AD_BOX = 32, AD_BOX_BYTES = AD_BOX * 128, AD_STAGES = 3;  // of a warp's ring

struct AdapterRows : AdapterParams {
    int chunks;       // units of AD_ROWS tokens per request
    int per_unit;     // requests of one slot that share a unit (1 where a request has several units)
    int k_each, n_each;  // channels and outputs of a CTA
};

// How a unit's rows are found: its number says so; requests compared within a warp; counted warp by warp; counted.  One kernel each: with all of them in
// one, code that isn't run cost 0.3 of 9 us.
enum AdapterFind { AD_OWN, AD_WARP, AD_CTA, AD_ANY };
static AdapterFind adapter_find(int per_unit, int B, int S) {
    return per_unit == 1 ? AD_OWN : B <= 32 ? AD_WARP : B <= AD_THREADS && S < AD_TABLE ? AD_CTA : AD_ANY;
}
// Words of shared memory that requests are counted in.
__host__ __device__ constexpr int adapter_counts(AdapterFind find, int S) { return find == AD_CTA ? 2 * (S + 1) : find == AD_ANY ? S + 1 : 0; }

// Rows of a unit: row numbers in s_row (-1: none), and its slot (-1: no adapter).  False: there is no such unit.
template <AdapterFind FIND>
__device__ __forceinline__ bool adapter_unit(const AdapterRows &p, int unit, int *s_row, int *s_count, int &slot, int &rows) {
    // s_count: requests of each slot, then of none
    __shared__ int s_warp[AD_THREADS / 32], s_which[2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid < AD_ROWS) s_row[tid] = -1;
    if constexpr (FIND == AD_OWN) {
        const int b = unit / p.chunks, chunk = unit - b * p.chunks;
        slot = p.slots[b];
        if (slot >= p.S) slot = -1;
        rows = min(AD_ROWS, p.T - chunk * AD_ROWS);
        __syncthreads();
        if (tid < rows) s_row[tid] = b * p.T + chunk * AD_ROWS + tid;
        __syncthreads();
        return true;
    }
    if constexpr (FIND == AD_WARP) {  // every warp: a lane to a request; the first of every per_unit ones of a slot stands for the unit
        const int s0 = lane < p.B ? p.slots[lane] : -2, s = lane >= p.B ? -2 : s0 < 0 || s0 >= p.S ? -1 : s0;
        const unsigned same = __match_any_sync(0xffffffffu, s), below = (1u << lane) - 1;
        const int rank = __popc(same & below);
        unsigned firsts = __ballot_sync(0xffffffffu, lane < p.B && rank % p.per_unit == 0);
        if (unit >= __popc(firsts)) return false;
        for (int i = 0; i < unit; ++i) firsts &= firsts - 1;
        const int first = __ffs(firsts) - 1, rank0 = __shfl_sync(0xffffffffu, rank, first);
        slot = __shfl_sync(0xffffffffu, s, first);
        const unsigned members = __ballot_sync(0xffffffffu, s == slot && rank >= rank0 && rank < rank0 + p.per_unit);
        rows = __popc(members) * p.T;
        __syncthreads();
        if (warp == 0 && (members >> lane & 1))
            for (int t = 0; t < p.T; ++t) s_row[(rank - rank0) * p.T + t] = lane * p.T + t;
        __syncthreads();
        return true;
    }
    auto slot_of = [&](int i) {
        const int s = p.slots[i];
        return s < 0 || s >= p.S ? p.S : s;
    };
    if constexpr (FIND == AD_CTA) {  // a thread to a request, then to a slot
        unsigned long long *s_table = reinterpret_cast<unsigned long long *>(s_count);  // (zero) requests of each slot, a byte to a warp
        auto sum = [](unsigned long long c) { return (int)__dp4a((unsigned)c, 0x01010101u, __dp4a((unsigned)(c >> 32), 0x01010101u, 0u)); };
        const int s = tid < p.B ? slot_of(tid) : -1;
        const unsigned same = __match_any_sync(0xffffffffu, s), below = same & ((1u << lane) - 1);
        if (s >= 0 && !below) reinterpret_cast<uint8_t *>(s_table + s)[warp] = (uint8_t)__popc(same);
        __syncthreads();
        // requests of the slot ahead of this one; units of this thread's slot
        const int rank = __popc(below) + (s >= 0 ? sum(s_table[s] & ((1ull << (8 * warp)) - 1)) : 0);
        const int units = tid <= p.S ? (sum(s_table[tid]) + p.per_unit - 1) / p.per_unit : 0;
        int before = units;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, before, off);
            if (lane >= off) before += v;
        }
        if (lane == 31) s_warp[warp] = before;
        __syncthreads();
        before -= units;
        int all = 0;
        for (int w = 0; w < AD_THREADS / 32; ++w) {
            if (w < warp) before += s_warp[w];
            all += s_warp[w];
        }
        if (unit >= all) return false;
        if (unit >= before && unit < before + units) {
            s_which[0] = tid;
            s_which[1] = (unit - before) * p.per_unit;
        }
        __syncthreads();
        const int which = s_which[0], first = s_which[1];
        slot = which < p.S ? which : -1;
        const bool member = s == which && rank >= first && rank < first + p.per_unit;
        if (member)
            for (int t = 0; t < p.T; ++t) s_row[(rank - first) * p.T + t] = tid * p.T + t;
        rows = __syncthreads_count(member) * p.T;
        return true;
    }
    if constexpr (FIND == AD_ANY) {
        int mine0 = -1;  // the slot of request tid
        for (int i = tid; i < p.B; i += AD_THREADS) {  // (the counts are zero)
            const int s = slot_of(i);
            if (i == tid) mine0 = s;
            atomicAdd(&s_count[s], 1);
        }
        __syncthreads();
        // units before each thread's run of slots
        const int run = (p.S + AD_THREADS) / AD_THREADS, lo = min(tid * run, p.S + 1), hi = min(lo + run, p.S + 1);
        int mine = 0;
        for (int i = lo; i < hi; ++i) mine += (s_count[i] + p.per_unit - 1) / p.per_unit;
        int before = mine;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, before, off);
            if (lane >= off) before += v;
        }
        if (lane == 31) s_warp[warp] = before;
        __syncthreads();
        int all = 0;
        before -= mine;
        for (int w = 0; w < AD_THREADS / 32; ++w) {
            if (w < warp) before += s_warp[w];
            all += s_warp[w];
        }
        if (unit >= all) return false;
        if (unit >= before && unit < before + mine) {
            int i = lo;
            for (;; ++i) {
                const int n = (s_count[i] + p.per_unit - 1) / p.per_unit;
                if (unit < before + n) break;
                before += n;
            }
            s_which[0] = i;
            s_which[1] = unit - before;
        }
        __syncthreads();
        const int which = s_which[0], first = s_which[1] * p.per_unit;
        slot = which < p.S ? which : -1;
        rows = min(s_count[which] - first, p.per_unit) * p.T;
        // its members: the requests of the slot from the first-th on, in order
        int found = 0;
        for (int i0 = 0; i0 < p.B && found < first + p.per_unit; i0 += AD_THREADS) {
            const int i = i0 + tid;
            const bool member = i < p.B && (i0 ? slot_of(i) : mine0) == which;
            const unsigned votes = __ballot_sync(0xffffffffu, member);
            __syncthreads();
            if (lane == 0) s_warp[warp] = __popc(votes);
            __syncthreads();
            int at = found - first + __popc(votes & ((1u << lane) - 1));
            for (int w = 0; w < AD_THREADS / 32; ++w) {
                if (w < warp) at += s_warp[w];
                found += s_warp[w];
            }
            if (member && at >= 0 && at < p.per_unit)
                for (int t = 0; t < p.T; ++t) s_row[at * p.T + t] = i * p.T + t;
        }
        __syncthreads();
        return true;
    }
}

// What the second term of t holds; nothing beside an infinity, whose rest would be NaN.
__device__ __forceinline__ float adapter_rest(float t, float hi) { return fabsf(hi) <= 3.4e38f ? t - hi : 0.f; }

// Down: a warp takes every eighth step of 64 channels.  Up: a warp takes every eighth group of 32 outputs; row i of product j is output
// j * 16 + i % 8 * 2 + i / 8 of the 32, so that a lane holds 2 consecutive ones of a token.
template <int STEPS, AdapterFind FIND>  // steps of 16 ranks
__global__ void __launch_bounds__(AD_THREADS, 2)
adapter_rows_kernel(const __grid_constant__ CUtensorMap map_down, const __grid_constant__ CUtensorMap map_up, const __grid_constant__ AdapterRows p) {
    constexpr int RANKS = 16 * STEPS, PITCH = RANKS + 4, WARPS = AD_THREADS / 32;
    constexpr int GROUPS = (RANKS + AD_BOX - 1) / AD_BOX, UP_BOXES = (RANKS + 63) / 64;  // boxes of a step of channels, of a group of outputs
    constexpr int AT_ONCE = STEPS <= 2 ? 8 : 32 / STEPS / 2;                             // warps whose sums meet at once: 9 KB at most
    extern __shared__ __align__(1024) uint8_t smem[];
    float(*s_t)[PITCH] = reinterpret_cast<float(*)[PITCH]>(smem + WARPS * AD_STAGES * AD_BOX_BYTES);
    float(*s_sum)[AD_ROWS][PITCH] = reinterpret_cast<float(*)[AD_ROWS][PITCH]>(s_t + AD_ROWS);
    uint64_t *bars = reinterpret_cast<uint64_t *>(s_sum + AT_ONCE);
    int *s_count = reinterpret_cast<int *>(bars + WARPS * AD_STAGES);
    __shared__ int s_row[AD_ROWS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane & 3, line = lane >> 2;
    uint8_t *ring = smem + warp * AD_STAGES * AD_BOX_BYTES;
    uint64_t *bar = bars + warp * AD_STAGES;
    if (lane == 0) {
        prefetch_tensormap(&map_down);
        prefetch_tensormap(&map_up);
        for (int i = 0; i < AD_STAGES; ++i) mbar_init(&bar[i], 1);
        fence_mbar_init();
    }
    __syncwarp();
    for (int i = threadIdx.x; i < adapter_counts(FIND, p.S); i += AD_THREADS) s_count[i] = 0;
    __syncthreads();
    pdl_wait_prior_grids();
    pdl_launch_dependents();  // behind the wait: what a next grid reads ahead of its own is older than this one's operands
    const int ctas = (int)cluster_ctas(), rank = (int)cluster_rank();
    int slot, rows;
    if (!adapter_unit<FIND>(p, blockIdx.x / ctas, s_row, s_count, slot, rows)) return;  // all of the cluster's CTAs
    const int n_lo = rank * p.n_each, n_hi = min(n_lo + p.n_each, p.N);
    if (slot < 0 || (smem_u32(smem) & 1023u) != 0) {
        if (slot >= 0 && threadIdx.x == 0) atomicOr(p.status, (int)NCKV_ST_TIMEOUT);  // checked rather than assumed
        if (rank == 0 && slot < 0 && (int)threadIdx.x < rows && p.slots[s_row[threadIdx.x] / p.T] >= p.S) atomicOr(p.status, (int)NCKV_ST_BAD_ADAPTER);
        const int vecs = (n_hi - n_lo) / 8;
        if (p.out != p.y)
            for (int i = threadIdx.x; i < rows * vecs; i += AD_THREADS) {
                const int row = s_row[i / vecs], n = n_lo + i % vecs * 8;
                *reinterpret_cast<uint4 *>(p.out + row * p.out_stride + n) = *reinterpret_cast<const uint4 *>(p.y + row * p.y_stride + n);
            }
        return;
    }
    // ---- this warp's stream of boxes: (step of channels, 32 ranks), then (32 outputs, 64 ranks) ---------
    const int k_lo = rank * p.k_each, k_hi = min(k_lo + p.k_each, p.K);
    const int k_steps = max(0, (k_hi - k_lo - warp * 64 + 64 * WARPS - 1) / (64 * WARPS)), n_steps = max(0, (n_hi - n_lo - warp * AD_BOX + AD_BOX * WARPS - 1) / (AD_BOX * WARPS));
    const int down_boxes = k_steps * GROUPS, boxes = down_boxes + n_steps * UP_BOXES;
    int fetched = 0;
    auto fetch = [&](int i) {  // lane 0
        const int s = i % AD_STAGES;
        const bool first = i < down_boxes;
        const int j = first ? i : i - down_boxes;
        const int c0 = first ? k_lo + (j / GROUPS * WARPS + warp) * 64 : j % UP_BOXES * 64;
        const int c1 = first ? j % GROUPS * AD_BOX : n_lo + (j / UP_BOXES * WARPS + warp) * AD_BOX;
        mbar_arrive_expect_tx(&bar[s], AD_BOX_BYTES);
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                smem_u32(ring + s * AD_BOX_BYTES)),
            "l"(first ? &map_down : &map_up), "r"(c0), "r"(c1), "r"(slot), "r"(smem_u32(&bar[s]))
            : "memory");
        fetched = i + 1;
    };
    bool ok = true;
    auto landed = [&](int i) -> uint32_t {  // box i is in shared memory
        const int s = i % AD_STAGES;
        const uint32_t parity = (i / AD_STAGES) & 1;
        if (!__all_sync(0xffffffffu, mbar_try_wait(&bar[s], parity))) {
            const int done = lane == 0 ? mbar_wait_bounded(&bar[s], parity) : 1;
            ok = __shfl_sync(0xffffffffu, done, 0) && ok;
            __syncwarp();
        }
        return smem_u32(ring + s * AD_BOX_BYTES);
    };
    auto next = [&](int i) {  // box i has been read: its place is for the one AD_STAGES later
        __syncwarp();
        if (ok && lane == 0 && i + AD_STAGES < boxes) fetch(i + AD_STAGES);
    };
    if (lane == 0)
        for (int i = 0; i < AD_STAGES && i < boxes; ++i) fetch(i);
    // a 16 x 16 operand comes as four matrices of 8 x 8: rows 0-7 and 8-15 of the first half of the columns, then of the second
    const int m_low = lane >> 3 & 1, m_half = lane >> 4, m_row = lane & 7;
    const int my_row = s_row[line];  // the token that this lane holds the channels and ranks of
    int box = 0;
    // ---- down ---------------------------------------------------------------------------------------
    float d[STEPS][4];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) d[i][0] = d[i][1] = d[i][2] = d[i][3] = 0.f;
    for (int step = 0; step < k_steps && ok; ++step) {
        const int k0 = k_lo + (step * WARPS + warp) * 64;
        uint32_t x[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int k = k0 + i * 16 + e * 8 + quad * 2;
                x[i][e] = 0;
                if (my_row >= 0 && k < k_hi) x[i][e] = *reinterpret_cast<const uint32_t *>(p.x + my_row * p.x_stride + k);
            }
#pragma unroll
        for (int group = 0; group < GROUPS; ++group, ++box) {
            const uint32_t at = landed(box);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if (group * 2 + j >= STEPS) break;
                float(&a)[4] = d[group * 2 + j];
                const int row = j * 16 + m_low * 8 + m_row;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t w0, w1, w2, w3;
                    ldmatrix_x4(w0, w1, w2, w3, at + row * 128 + (((i * 2 + m_half) ^ (row & 7)) << 4));
                    mma_bf16_16816(a[0], a[1], a[2], a[3], w0, w1, w2, w3, x[i][0], x[i][1]);
                }
            }
            next(box);
        }
    }
    // y of AD_AHEAD groups of outputs, of the two tokens whose results this lane holds
    const int t0 = s_row[quad * 2], t1 = s_row[quad * 2 + 1];
    uint32_t y_ring[AD_AHEAD][2][2];
    auto load_y = [&](uint32_t (&y)[2][2], int step) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int n = n_lo + (step * WARPS + warp) * AD_BOX + j * 16 + line * 2;
            y[j][0] = y[j][1] = 0;
            if (n < n_hi && t0 >= 0) y[j][0] = *reinterpret_cast<const uint32_t *>(p.y + t0 * p.y_stride + n);
            if (n < n_hi && t1 >= 0) y[j][1] = *reinterpret_cast<const uint32_t *>(p.y + t1 * p.y_stride + n);
        }
    };
#pragma unroll
    for (int i = 0; i < AD_AHEAD; ++i)
        if (i < n_steps) load_y(y_ring[i], i);
    // ---- the warps' sums, then the CTAs', in a fixed order ---------------------------------------------
    for (int w0 = 0; w0 < WARPS; w0 += AT_ONCE) {
        if (w0) __syncthreads();
        if (warp >= w0 && warp < w0 + AT_ONCE)
#pragma unroll
            for (int i = 0; i < STEPS; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) s_sum[warp - w0][quad * 2 + (e & 1)][i * 16 + line + (e >> 1) * 8] = d[i][e];
        __syncthreads();
        for (int i = threadIdx.x; i < AD_ROWS * RANKS / 4; i += AD_THREADS) {
            const int row = i / (RANKS / 4), r = i % (RANKS / 4) * 4;
            float4 sum = w0 ? *reinterpret_cast<float4 *>(&s_t[row][r]) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) {
                const float4 v = *reinterpret_cast<const float4 *>(&s_sum[k][row][r]);
                sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
            }
            *reinterpret_cast<float4 *>(&s_t[row][r]) = sum;
        }
    }
    float(*t)[PITCH] = s_t;
    if (ctas > 1) {
        cluster_sync();
        t = s_sum[0];
        for (int i = threadIdx.x; i < AD_ROWS * RANKS / 4; i += AD_THREADS) {
            const int row = i / (RANKS / 4), r = i % (RANKS / 4) * 4;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
            for (int c = 0; c < ctas; ++c) {
                float4 v;
                asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                             : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                             : "r"(smem_of_rank(&s_t[row][r], (uint32_t)c))
                             : "memory");
                sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
            }
            *reinterpret_cast<float4 *>(&t[row][r]) = sum;
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // this CTA has read the others' sums
    }
    __syncthreads();
    // ---- up -----------------------------------------------------------------------------------------
    // t as two bf16 terms: of this lane's token, or, with up to four tokens, the first term of tokens 0-3 in lines 0-3 and the second in 4-7
    const bool both = rows <= AD_ROWS / 2;
    uint32_t hi[STEPS][2], lo[STEPS][2];
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float2 v = *reinterpret_cast<const float2 *>(&t[both ? line & 3 : line][i * 16 + e * 8 + quad * 2]);
            hi[i][e] = pack_bf16x2(v.x, v.y);
            lo[i][e] = pack_bf16x2(adapter_rest(v.x, bf16lo(hi[i][e])), adapter_rest(v.y, bf16hi(hi[i][e])));
            if (both && line >= 4) hi[i][e] = lo[i][e];
        }
    const float scale = p.scales[slot];
    for (int step0 = 0; step0 < n_steps && ok; step0 += AD_AHEAD)
#pragma unroll
        for (int ahead = 0; ahead < AD_AHEAD; ++ahead) {
            const int step = step0 + ahead;
            if (step >= n_steps) break;
            uint32_t(&y)[2][2] = y_ring[ahead];
            float o[2][4];
#pragma unroll
            for (int j = 0; j < 2; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
#pragma unroll
            for (int part = 0; part < UP_BOXES; ++part, ++box) {
                const uint32_t at = landed(box);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int row = j * 16 + m_row * 2 + m_low;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (part * 4 + i >= STEPS) break;
                        uint32_t w0, w1, w2, w3;
                        ldmatrix_x4(w0, w1, w2, w3, at + row * 128 + (((i * 2 + m_half) ^ (row & 7)) << 4));
                        mma_bf16_16816(o[j][0], o[j][1], o[j][2], o[j][3], w0, w1, w2, w3, hi[part * 4 + i][0], hi[part * 4 + i][1]);
                        if (!both) mma_bf16_16816(o[j][0], o[j][1], o[j][2], o[j][3], w0, w1, w2, w3, lo[part * 4 + i][0], lo[part * 4 + i][1]);
                    }
                }
                next(box);
            }
            if (!ok) break;
            if (both)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[j][e] += __shfl_xor_sync(0xffffffffu, o[j][e], 2);  // quads 0 and 1: the tokens' first terms
            uint32_t out[2][2];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) out[j][e] = pack_bf16x2(bf16lo(y[j][e]) + scale * o[j][e], bf16hi(y[j][e]) + scale * o[j][2 + e]);
            if (step + AD_AHEAD < n_steps) load_y(y, step + AD_AHEAD);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int n = n_lo + (step * WARPS + warp) * AD_BOX + j * 16 + line * 2;
                if (n < n_hi && t0 >= 0) *reinterpret_cast<uint32_t *>(p.out + t0 * p.out_stride + n) = out[j][0];
                if (n < n_hi && t1 >= 0) *reinterpret_cast<uint32_t *>(p.out + t1 * p.out_stride + n) = out[j][1];
            }
        }
    if (!ok && lane == 0) {  // a copy did not land in time: the ones behind it may still be under way
        atomicOr(p.status, (int)NCKV_ST_TIMEOUT);
        for (int i = max(fetched - AD_STAGES, 0); i < fetched; ++i) mbar_wait_bounded(&bar[i % AD_STAGES], (i / AD_STAGES) & 1);
    }
    __syncwarp();
    if (ctas > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // the others have read this one's
}

using AdapterKernel = void (*)(CUtensorMap, CUtensorMap, AdapterRows);
template <int STEPS>
static AdapterKernel adapter_kernel(AdapterFind find) {
    return find == AD_OWN ? adapter_rows_kernel<STEPS, AD_OWN> : find == AD_WARP ? adapter_rows_kernel<STEPS, AD_WARP>
         : find == AD_CTA ? adapter_rows_kernel<STEPS, AD_CTA> : adapter_rows_kernel<STEPS, AD_ANY>;
}

// Units at most: the requests are known here, their slots aren't.
static long long adapter_units(int B, int T, int S, int *per_unit, int *chunks) {
    *chunks = (T + AD_ROWS - 1) / AD_ROWS;
    *per_unit = T < AD_ROWS ? AD_ROWS / T : 1;
    if (*per_unit == 1) return (long long)B * *chunks;
    const long long most = (long long)S + 1 + B / *per_unit;
    return most < B ? most : B;
}

static int adapter_check_sizes(const char *name, int B, int T, int K, int N, int R, int S) {
    if (B <= 0 || T <= 0 || K <= 0 || N <= 0 || R <= 0 || S <= 0) {
        set_error("%s: non-positive size (B=%d T=%d K=%d N=%d R=%d S=%d)", name, B, T, K, N, R, S);
        return NCKV_E_ARG;
    }
    if (R > AD_MAX_RANK || R % 8 || K % 8 || N % 8) {
        set_error("%s: rank %d must be at most %d, and it, K=%d and N=%d multiples of 8", name, R, AD_MAX_RANK, K, N);
        return NCKV_E_UNSUPPORTED;
    }
    if (S > 8192) {
        set_error("%s: %d adapters are more than 8192", name, S);
        return NCKV_E_UNSUPPORTED;
    }
    if ((long long)B * T > 0x3fffffffLL) {
        set_error("%s: B=%d requests of T=%d tokens are too many for one launch", name, B, T);
        return NCKV_E_UNSUPPORTED;
    }
    return NCKV_OK;
}

// Whether rows of `cols` elements `stride` apart lie on any of other ones.  At one distance rows may lie between each other (column slices of one
// tensor); at two they have to be apart altogether.
static bool adapter_rows_meet(const void *a, int64_t a_stride, int a_cols, const void *b, int64_t b_stride, int b_cols, long long rows) {
    const long long lo_a = (long long)((uintptr_t)a / 2), lo_b = (long long)((uintptr_t)b / 2);
    if (lo_a + (rows - 1) * a_stride + a_cols <= lo_b || lo_b + (rows - 1) * b_stride + b_cols <= lo_a) return false;
    if (rows == 1 || a_stride != b_stride) return true;
    const long long off = ((lo_b - lo_a) % a_stride + a_stride) % a_stride;
    return off < a_cols || off + b_cols > a_stride;
}

}  // namespace nckv

extern "C" size_t nckv_adapters_workspace_bytes(int B, int T, int K, int N, int R, int S) {
    using namespace nckv;
    if (adapter_check_sizes("adapters_workspace_bytes", B, T, K, N, R, S) != NCKV_OK) return 0;
    if (adapters_tiled(B, T)) return adapters_tc_bytes(B, T, R);
    return 0;
}

extern "C" int nckv_adapters(const void *y, int64_t y_stride, const void *x, int64_t x_stride, const void *down, const void *up,
                             const int32_t *slots, const float *scales, void *out, int64_t out_stride, int B, int T, int K, int N, int R,
                             int S, void *workspace, size_t workspace_bytes, int32_t *status, void *stream) {
    using namespace nckv;
    const char *name = "adapters";
    if (!y || !x || !down || !up || !slots || !scales || !out || !status) {
        set_error("%s: null pointer argument", name);
        return NCKV_E_ARG;
    }
    int rc = adapter_check_sizes(name, B, T, K, N, R, S);
    if (rc != NCKV_OK) return rc;
    if (x_stride < K || y_stride < N || out_stride < N || (x_stride | y_stride | out_stride) % 8) {
        set_error("%s: row strides must be multiples of 8 elements and span a row", name);
        return NCKV_E_ARG;
    }
    if (((uintptr_t)y | (uintptr_t)x | (uintptr_t)down | (uintptr_t)up | (uintptr_t)out | (uintptr_t)workspace) & 15) {
        set_error("%s: tensors must be 16-byte aligned", name);
        return NCKV_E_ARG;
    }
    const long long all = (long long)B * T;
    if (adapter_rows_meet(out, out_stride, N, x, x_stride, K, all)) {
        set_error("%s: the result and x share memory", name);
        return NCKV_E_ARG;
    }
    if ((out != y || out_stride != y_stride) && adapter_rows_meet(out, out_stride, N, y, y_stride, N, all)) {
        set_error("%s: the result is neither y nor beside it: they share memory", name);
        return NCKV_E_ARG;
    }
    if (workspace_bytes < nckv_adapters_workspace_bytes(B, T, K, N, R, S) || (workspace_bytes && !workspace)) {
        set_error("%s: needs %zu bytes of workspace", name, nckv_adapters_workspace_bytes(B, T, K, N, R, S));
        return NCKV_E_CAPACITY;
    }
    AdapterRows p;
    p.y = static_cast<const __nv_bfloat16 *>(y);
    p.x = static_cast<const __nv_bfloat16 *>(x);
    p.down = static_cast<const __nv_bfloat16 *>(down);
    p.up = static_cast<const __nv_bfloat16 *>(up);
    p.out = static_cast<__nv_bfloat16 *>(out);
    p.slots = slots;
    p.scales = scales;
    p.t = workspace;
    p.status = status;
    p.y_stride = y_stride; p.x_stride = x_stride; p.out_stride = out_stride;
    p.B = B; p.T = T; p.K = K; p.N = N; p.R = R; p.S = S;
    if (adapters_tiled(B, T)) return adapters_tc(p, static_cast<cudaStream_t>(stream));
    const long long units = adapter_units(B, T, S, &p.per_unit, &p.chunks);
    // A cluster's CTAs: about what the chip holds at once, two per SM.  us with 8 / 4 / 2 / 1, 2048 channels and outputs at rank 16: 16 units 5.4 / 5.7 /
    // 7.4 / 9.7, 32 6.1 / 6.3 / 7.6 / 9.9, 64 12.1 / 7.6 / 8.2 / 10.5; 1536 x 4608 at rank 32: 64 16.0 / 10.2 / 11.7 / 17.9, 128 30.9 / 20.1 / 16.5 /
    // 20.1; 2048 x 8192 at rank 64: at most 81 (the slots decide) 27.9 / 19.5 / 26.7 / 34.8, 256 118 / 76 / 65 / 58.
    const int sms = sm_count(), most = K > N ? K / 64 : N / AD_BOX;
    int ctas = units <= sms / 4 ? 8 : units <= sms * 2 / 3 ? 4 : units <= sms ? 2 : 1;
    while (ctas > 1 && ctas * 4 > most) ctas /= 2;
    p.k_each = ((K + ctas - 1) / ctas + 63) / 64 * 64;
    p.n_each = ((N + ctas - 1) / ctas + AD_BOX - 1) / AD_BOX * AD_BOX;
    CUtensorMap map_down, map_up;
    const int box[3] = {64, AD_BOX, 1};
    const int64_t down_dims[3] = {K, R, S}, down_strides[2] = {K, (int64_t)R * K}, up_dims[3] = {R, N, S}, up_strides[2] = {R, (int64_t)N * R};
    rc = make_tensor_map(&map_down, down, 3, down_dims, down_strides, box);
    if (rc == NCKV_OK) rc = make_tensor_map(&map_up, up, 3, up_dims, up_strides, box);
    if (rc != NCKV_OK) return rc;
    const AdapterFind find = adapter_find(p.per_unit, B, S);
    const int steps = R <= 16 ? 1 : R <= 32 ? 2 : R <= 64 ? 4 : 8, at_once = steps <= 2 ? 8 : 16 / steps, warps = AD_THREADS / 32;
    const size_t smem = (size_t)warps * AD_STAGES * AD_BOX_BYTES + (size_t)(1 + at_once) * AD_ROWS * (16 * steps + 4) * 4 + warps * AD_STAGES * 8 +
                        (size_t)adapter_counts(find, S) * 4;
    const auto kernel = steps == 1 ? adapter_kernel<1>(find) : steps == 2 ? adapter_kernel<2>(find) : steps == 4 ? adapter_kernel<4>(find) : adapter_kernel<8>(find);
    static bool attr_set[64][9][4] = {};
    int dev = 0;
    NCKV_CUDA_CHECK(cudaGetDevice(&dev));
    if (dev >= 64 || !attr_set[dev][steps][find]) {
        NCKV_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
        if (dev < 64) attr_set[dev][steps][find] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(units * ctas));
    cfg.blockDim = dim3(AD_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)ctas;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    NCKV_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, map_down, map_up, p));
    return NCKV_OK;
}
