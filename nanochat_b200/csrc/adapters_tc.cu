// Low-rank adapters beside a shared projection for requests of many tokens (adapters.cu: few): both launches on the tensor cores
// (tcgen05, accumulators in tensor memory), bound by the activations' bytes: x read once, y read and written once.
// 6 x 1531 tokens, 6144 -> 1536 at rank 32 (173 MB): 40 us = 4.3 TB/s; 8 x 2048, 2048 -> 8192 at rank 64 (607 MB): 118 us = 5.1.
//
// A tile is 128 tokens of one request.  All operands come by TMA with the 128-byte swizzle over maps of three dimensions (channels, tokens,
// requests), which clip a request's last tile and fill ranks and channels up with zeros.
//   adapter_tile_down   t = down x.  A cluster of CTAs shares a tile's channels (so that few tiles still fill the chip), adds the parts up through
//                       distributed shared memory in the order of the ranks and writes t as two bf16 terms side by side, hi and lo.
//   adapter_tile_up     out = y + scale up t: persistent CTAs, one per SM, over equal runs of (tile, 64 outputs).  t's two terms stay in
//                       shared memory for a tile; y and up come through a ring, whose y part the rows' warps turn into the
//                       result in place, from where every warp stores its 32 rows by TMA.  y and up are asked for ahead of the wait
//                       for the launch before.
// Every wait on an mbarrier is bounded; one that runs out sets NCKV_ST_TIMEOUT, the CTA waits for its copies, frees its tensor memory and
// returns.
#include "adapters.cuh"
#include "tc05.cuh"

namespace nckv {

constexpr int AT_M = 128, AT_K = 64, AT_N = 64;
constexpr int AT_THREADS = 192;             // copies, products, four warps for the accumulator's rows
constexpr int AT_UP_THREADS = 64 + 2 * 128;  // two groups of four take steps in turn
constexpr int AT_ACCS = 4;                   // accumulators of adapter_tile_up
constexpr int AT_X_BYTES = AT_M * AT_K * 2;
constexpr int AT_DOWN_STAGES = 6, AT_MAX_CLUSTER = 8;

struct AdapterTile {
    AdapterParams a;
    int RP;      // rank rounded up to 16
    int tiles;   // of 128 tokens per request
    int stages;  // of adapter_tile_up
    bool in_place;
};

__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, uint64_t *bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap *map, const void *src, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map), "r"(c0), "r"(c1), "r"(c2),
                 "r"(smem_u32(src))
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
template <int LEFT> __device__ __forceinline__ void tma_stores_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(LEFT) : "memory"); }
__device__ __forceinline__ void tma_stores_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

__device__ __forceinline__ int adapter_slot(const AdapterParams &p, int b) {
    const int s = p.slots[b];
    return s < p.S ? s : -1;
}

__global__ void __launch_bounds__(AT_THREADS, 1)
adapter_tile_down(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_down, const __grid_constant__ AdapterTile q) {
    extern __shared__ __align__(1024) uint8_t smem[];
    const AdapterParams &p = q.a;
    pdl_wait_prior_grids();
    const int ctas = (int)cluster_ctas(), rank = (int)cluster_rank(), tile = (int)blockIdx.x / ctas;
    const int b = tile / q.tiles, t0 = (tile - b * q.tiles) * AT_M, slot = adapter_slot(p, b);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (slot < 0) {  // all of the cluster's CTAs
        if (tid == 0 && rank == 0 && p.slots[b] >= p.S) atomicOr(p.status, (int)NCKV_ST_BAD_ADAPTER);
        return;
    }
    const int stage_bytes = AT_X_BYTES + q.RP * AT_K * 2;
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + AT_DOWN_STAGES * stage_bytes);
    uint64_t *bar_full = bars, *bar_free = bars + AT_DOWN_STAGES, *bar_acc = bars + 2 * AT_DOWN_STAGES;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * AT_DOWN_STAGES + 1);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const uint32_t columns = q.RP <= 32 ? 32 : q.RP <= 64 ? 64 : 128;
    if (warp == 0) {
        tmem_alloc(tmem_slot, columns);
        tmem_relinquish();
    } else if (tid == 32) {
        prefetch_tensormap(&map_x);
        prefetch_tensormap(&map_down);
        for (int i = 0; i < AT_DOWN_STAGES; ++i) {
            mbar_init(&bar_full[i], 1);
            mbar_init(&bar_free[i], 1);
        }
        mbar_init(bar_acc, 1);
        *abort_flag = (smem_u32(smem) & 1023u) != 0;  // checked rather than assumed
        fence_mbar_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // Behind the wait: the next grid reads slots, y and weights ahead of its own.  Behind the allocation: its CTAs hold tensor memory while
    // they wait for this grid.
    pdl_launch_dependents();
    const uint32_t tmem = *tmem_slot;
    auto timed_out = [&]() {
        *abort_flag = 1;
        atomicOr(p.status, (int)NCKV_ST_TIMEOUT);
    };
    // every ctas-th step: the cluster reads a row's channels side by side (n > 0: at most as many CTAs as steps)
    const int steps = (p.K + AT_K - 1) / AT_K, n = (steps - rank + ctas - 1) / ctas;
    if (*abort_flag) {
        if (tid == 0) timed_out();
    } else if (warp == 0) {
        if (elect_one()) {
            bool ok = true;
            int issued = 0;
            for (int i = 0; i < n && ok; ++i) {
                const int s = i % AT_DOWN_STAGES;
                if (i >= AT_DOWN_STAGES) ok = mbar_wait_bounded(&bar_free[s], (i / AT_DOWN_STAGES + 1) & 1);
                if (!ok) break;
                uint8_t *at = smem + s * stage_bytes;
                mbar_arrive_expect_tx(&bar_full[s], stage_bytes);
                tma_load_3d(at, &map_x, &bar_full[s], (i * ctas + rank) * AT_K, t0, b);
                tma_load_3d(at + AT_X_BYTES, &map_down, &bar_full[s], (i * ctas + rank) * AT_K, 0, slot);
                ++issued;
            }
            if (!ok) timed_out();
            if (*abort_flag)
                for (int i = max(issued - AT_DOWN_STAGES, 0); i < issued; ++i) mbar_wait_bounded(&bar_full[i % AT_DOWN_STAGES], (i / AT_DOWN_STAGES) & 1);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (elect_one()) {
            const uint32_t idesc = umma_idesc(AT_M, q.RP, 0, 0);
            bool ok = true;
            for (int i = 0; i < n && ok; ++i) {
                const int s = i % AT_DOWN_STAGES;
                ok = mbar_wait_bounded(&bar_full[s], (i / AT_DOWN_STAGES) & 1);
                if (!ok) break;
                tc_fence_after();
                const uint32_t at = smem_u32(smem + s * stage_bytes);
                const uint64_t da = smem_desc_sw128(at, 16, 1024), db = smem_desc_sw128(at + AT_X_BYTES, 16, 1024);
#pragma unroll
                for (int k = 0; k < AT_K / 16; ++k) umma_bf16(tmem, da + (uint64_t)(k * 32 >> 4), db + (uint64_t)(k * 32 >> 4), idesc, i > 0 || k > 0);
                umma_commit(&bar_free[s]);
            }
            if (ok) umma_commit(bar_acc);
            else timed_out();
        }
        __syncwarp();
    }
    // this CTA's sums into its shared memory (the operands have been read), row by row
    const int pitch = q.RP + 4;
    float *sums = reinterpret_cast<float *>(smem);
    if (warp >= 2 && !*abort_flag) {
        int ok = lane == 0 ? mbar_wait_bounded(bar_acc, 0) : 1;
        ok = __shfl_sync(0xffffffffu, ok, 0);
        __syncwarp();
        if (!ok) {
            if (lane == 0) timed_out();
        } else {
            tc_fence_after();
            const int row = (warp & 3) * 32 + lane;
            for (int c = 0; c < q.RP; c += 16) {
                uint32_t r[16];
                asm volatile(
                    "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
                    "tcgen05.wait::ld.sync.aligned;"
                    : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                      "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                    : "r"(tmem + ((uint32_t)((warp & 3) * 32) << 16) + c)
                    : "memory");
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<uint4 *>(sums + row * pitch + c + 4 * i) = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
            }
            tc_fence_before();
        }
    }
    cluster_sync();
    // rows rank, rank + ctas, ...: the CTAs' sums in the order of their ranks, as two bf16 terms
    const int quads = q.RP / 4;
    __nv_bfloat16 *t = static_cast<__nv_bfloat16 *>(p.t);
    for (int i = tid; i < AT_M / ctas * quads; i += AT_THREADS) {
        const int row = i / quads * ctas + rank, c = i % quads * 4;
        if (t0 + row >= p.T) continue;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int r = 0; r < ctas; ++r) {
            float4 v;
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                         : "r"(smem_of_rank(sums + row * pitch + c, (uint32_t)r))
                         : "memory");
            sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
        }
        auto rest = [](float v, float hi) { return fabsf(hi) <= 3.4e38f ? v - hi : 0.f; };  // nothing beside an infinity
        uint2 hi = make_uint2(pack_bf16x2(sum.x, sum.y), pack_bf16x2(sum.z, sum.w)), lo;
        lo.x = pack_bf16x2(rest(sum.x, bf16lo(hi.x)), rest(sum.y, bf16hi(hi.x)));
        lo.y = pack_bf16x2(rest(sum.z, bf16lo(hi.y)), rest(sum.w, bf16hi(hi.y)));
        __nv_bfloat16 *dst = t + ((long long)b * p.T + t0 + row) * 2 * q.RP + c;
        *reinterpret_cast<uint2 *>(dst) = hi;
        *reinterpret_cast<uint2 *>(dst + q.RP) = lo;
    }
    cluster_sync();  // the others may still be reading
    if (warp == 0) tmem_dealloc(tmem, columns);
}

__global__ void __launch_bounds__(AT_UP_THREADS, 1)
adapter_tile_up(const __grid_constant__ CUtensorMap map_t, const __grid_constant__ CUtensorMap map_up, const __grid_constant__ CUtensorMap map_y,
                const __grid_constant__ CUtensorMap map_out, const __grid_constant__ AdapterTile q) {
    extern __shared__ __align__(1024) uint8_t smem[];
    const AdapterParams &p = q.a;
    const int t_boxes = (2 * q.RP + 63) / 64, up_boxes = (p.R + 63) / 64;
    const int t_bytes = t_boxes * AT_M * 128, y_bytes = AT_M * 128, up_bytes = up_boxes * AT_N * 128, stage_bytes = y_bytes + up_bytes;
    uint8_t *s_t = smem, *ring = smem + t_bytes;
    uint64_t *bars = reinterpret_cast<uint64_t *>(ring + q.stages * stage_bytes);
    uint64_t *bar_full = bars, *bar_free = bars + q.stages;
    uint64_t *bar_acc = bars + 2 * q.stages, *bar_read = bar_acc + AT_ACCS, *bar_t = bar_acc + 2 * AT_ACCS, *bar_t_read = bar_t + 1;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bar_t + 2);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (warp == 0) {
        tmem_alloc(tmem_slot, AT_ACCS * AT_N);
        tmem_relinquish();
    } else if (tid == 32) {
        prefetch_tensormap(&map_t);
        prefetch_tensormap(&map_up);
        prefetch_tensormap(&map_y);
        prefetch_tensormap(&map_out);
        for (int i = 0; i < q.stages; ++i) {
            mbar_init(&bar_full[i], 1);
            mbar_init(&bar_free[i], 4);
        }
        for (int i = 0; i < AT_ACCS; ++i) {
            mbar_init(&bar_acc[i], 1);
            mbar_init(&bar_read[i], 4);
        }
        mbar_init(bar_t, 1);
        mbar_init(bar_t_read, 1);
        *abort_flag = (smem_u32(smem) & 1023u) != 0;  // checked rather than assumed
        fence_mbar_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    auto timed_out = [&]() {
        *abort_flag = 1;
        atomicOr(p.status, (int)NCKV_ST_TIMEOUT);
    };
    // this CTA's run of steps: (tile, 64 outputs), outputs fastest
    const int n_steps = (p.N + AT_N - 1) / AT_N;
    const long long total = (long long)p.B * q.tiles * n_steps;
    const long long lo = total * blockIdx.x / gridDim.x, hi = total * (blockIdx.x + 1) / gridDim.x;
    // calls f(first step of a tile, its number of steps, request, first token, slot) for the tiles of the run that there is something to do for
    auto for_tiles = [&](auto &&f) {
        for (long long at = lo; at < hi;) {
            const int tile = (int)(at / n_steps), from = (int)(at - (long long)tile * n_steps), n = (int)min((long long)(n_steps - from), hi - at);
            const int b = tile / q.tiles, slot = adapter_slot(p, b);
            at += n;
            if (slot < 0 && q.in_place) continue;
            if (!f(from, n, b, (tile - b * q.tiles) * AT_M, slot)) return;
        }
    };
    if (*abort_flag) {
        if (tid == 0) timed_out();
    } else if (warp == 0) {
        // =============== copies ==============================================================================
        if (elect_one()) {
            uint32_t g = 0, n_t = 0;
            bool ok = true, waited = false;
            for_tiles([&](int from, int n, int b, int t0, int slot) {
                for (int i = 0; i < n; ++i, ++g) {
                    const uint32_t s = g % q.stages;
                    if (g >= (uint32_t)q.stages) ok = mbar_wait_bounded(&bar_free[s], (g / q.stages + 1) & 1);
                    if (!ok) return false;
                    uint8_t *at = ring + s * stage_bytes;
                    const int n0 = (from + i) * AT_N;
                    mbar_arrive_expect_tx(&bar_full[s], slot >= 0 ? stage_bytes : y_bytes);
                    tma_load_3d(at, &map_y, &bar_full[s], n0, t0, b);
                    if (slot >= 0)
                        for (int k = 0; k < up_boxes; ++k) tma_load_3d(at + y_bytes + k * AT_N * 128, &map_up, &bar_full[s], k * 64, n0, slot);
                    // t behind as much of the ring as doesn't need this tile's steps done (a stage is free two steps behind its own)
                    if (slot >= 0 && i == min(n, q.stages - 2) - 1) {
                        if (!waited) pdl_wait_prior_grids();
                        waited = true;
                        if (n_t) ok = mbar_wait_bounded(bar_t_read, (n_t + 1) & 1);
                        if (!ok) return false;
                        mbar_arrive_expect_tx(bar_t, t_bytes);
                        for (int k = 0; k < t_boxes; ++k) tma_load_3d(s_t + k * AT_M * 128, &map_t, bar_t, k * 64, t0, b);
                        ++n_t;
                    }
                }
                return true;
            });
            if (!waited) pdl_wait_prior_grids();
            if (!ok) timed_out();
            if (*abort_flag) {
                if (n_t) mbar_wait_bounded(bar_t, (n_t - 1) & 1);
                for (uint32_t i = g > (uint32_t)q.stages ? g - q.stages : 0; i < g; ++i) mbar_wait_bounded(&bar_full[i % q.stages], (i / q.stages) & 1);
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // =============== products ============================================================================
        if (elect_one()) {
            constexpr uint32_t IDESC = umma_idesc(AT_M, AT_N, 0, 0);
            const uint64_t desc_t = smem_desc_sw128(smem_u32(s_t), 16, 1024);
            uint32_t g = 0, m = 0, n_t = 0;  // steps, steps with products, tiles with them
            bool ok = true;
            for_tiles([&](int, int n, int, int, int slot) {
                if (slot < 0) {
                    g += n;
                    return true;
                }
                ok = mbar_wait_bounded(bar_t, n_t & 1);
                for (int i = 0; i < n && ok; ++i, ++g, ++m) {
                    const uint32_t s = g % q.stages;
                    ok = mbar_wait_bounded(&bar_full[s], (g / q.stages) & 1) && (m < AT_ACCS || mbar_wait_bounded(&bar_read[m % AT_ACCS], (m / AT_ACCS + 1) & 1));
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t desc_up = smem_desc_sw128(smem_u32(ring + s * stage_bytes + y_bytes), 16, 1024);
                    for (int k = 0; k < q.RP / 8; ++k) {  // hi, then lo
                        const int rank = k * 16 % q.RP, col = k * 16;
                        umma_bf16(tmem + (m % AT_ACCS) * AT_N, desc_t + (uint64_t)((col / 64 * AT_M * 128 + col % 64 * 2) >> 4),
                                  desc_up + (uint64_t)((rank / 64 * AT_N * 128 + rank % 64 * 2) >> 4), IDESC, k > 0);
                    }
                    umma_commit(&bar_acc[m % AT_ACCS]);
                }
                if (ok) umma_commit(bar_t_read);
                ++n_t;
                return ok;
            });
            if (!ok) timed_out();
        }
        __syncwarp();
    } else {
        // =============== rows: y in the ring becomes the result ==============================================
        const int part = warp & 3, row = part * 32 + lane, group = (warp - 2) / 4;
        auto warp_wait = [&](uint64_t *bar, uint32_t parity) -> bool {
            if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
            int ok = *abort_flag == 0;
            if (lane == 0 && ok) ok = mbar_wait_bounded(bar, parity) ? 1 : 0;
            ok = __shfl_sync(0xffffffffu, ok, 0);
            __syncwarp();
            return ok != 0;
        };
        uint32_t g = 0, m = 0;
        int last = -1;  // stage of this warp's store before
        bool ok = true;
        for_tiles([&](int from, int n, int b, int t0, int slot) {
            const float scale = slot >= 0 ? p.scales[slot] : 0.f;
            for (int i = 0; i < n; ++i, ++g, m += slot >= 0) {
                if ((int)(g & 1) != group) continue;
                const uint32_t s = g % q.stages;
                uint8_t *y = ring + s * stage_bytes;
                ok = warp_wait(&bar_full[s], (g / q.stages) & 1);
                if (!ok) return false;
                if (slot >= 0) {
                    ok = warp_wait(&bar_acc[m % AT_ACCS], (m / AT_ACCS) & 1);
                    if (!ok) return false;
                    tc_fence_after();
                    float d[AT_N];
                    tmem_ld64(tmem + (m % AT_ACCS) * AT_N + ((uint32_t)(part * 32) << 16), d);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&bar_read[m % AT_ACCS]);
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        uint4 *at = reinterpret_cast<uint4 *>(y + row * 128 + ((c ^ (row & 7)) << 4));
                        uint4 v = *at;
                        v.x = pack_bf16x2(bf16lo(v.x) + scale * d[8 * c], bf16hi(v.x) + scale * d[8 * c + 1]);
                        v.y = pack_bf16x2(bf16lo(v.y) + scale * d[8 * c + 2], bf16hi(v.y) + scale * d[8 * c + 3]);
                        v.z = pack_bf16x2(bf16lo(v.z) + scale * d[8 * c + 4], bf16hi(v.z) + scale * d[8 * c + 5]);
                        v.w = pack_bf16x2(bf16lo(v.w) + scale * d[8 * c + 6], bf16hi(v.w) + scale * d[8 * c + 7]);
                        *at = v;
                    }
                    fence_proxy_async_smem();  // the results must be visible to the store
                }
                __syncwarp();
                if (lane == 0) {
                    if (t0 + part * 32 < p.T) tma_store_3d(&map_out, y + part * 32 * 128, (from + i) * AT_N, t0 + part * 32, b);
                    else asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    if (last >= 0) {  // the store before has read its stage
                        tma_stores_read<1>();
                        mbar_arrive(&bar_free[last]);
                    }
                    last = (int)s;
                }
            }
            return true;
        });
        if (lane == 0) tma_stores_done();
        if (!ok && *abort_flag == 0) timed_out();
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem, AT_ACCS * AT_N);
}

static int rank_pad(int R) { return (R + 15) / 16 * 16; }
size_t adapters_tc_bytes(int B, int T, int R) { return (size_t)B * T * 2 * rank_pad(R) * 2; }

static size_t adapter_down_smem(int RP) { return AT_DOWN_STAGES * (size_t)(AT_X_BYTES + RP * AT_K * 2) + (2 * AT_DOWN_STAGES + 1) * 8 + 16; }
static size_t adapter_up_smem(int RP, int R, int stages) {
    return (size_t)(2 * RP + 63) / 64 * AT_M * 128 + (size_t)stages * (AT_M * 128 + (R + 63) / 64 * AT_N * 128) + (2 * stages + 2 * AT_ACCS + 2) * 8 + 16;
}

int adapters_tc(const AdapterParams &a, cudaStream_t stream) {
    AdapterTile q;
    q.a = a;
    q.RP = rank_pad(a.R);
    q.tiles = (a.T + AT_M - 1) / AT_M;
    q.in_place = a.out == a.y;
    CUtensorMap map_x, map_down, map_t, map_up, map_y, map_out;
    auto map3 = [](CUtensorMap *m, const void *base, int64_t d0, int64_t d1, int64_t d2, int64_t stride, int rows) {
        const int64_t dims[3] = {d0, d1, d2}, strides[2] = {stride, d1 * stride};
        const int box[3] = {64, rows, 1};
        return make_tensor_map(m, base, 3, dims, strides, box);
    };
    int rc = map3(&map_x, a.x, a.K, a.T, a.B, a.x_stride, AT_M);
    if (!rc) rc = map3(&map_down, a.down, a.K, a.R, a.S, a.K, q.RP);
    if (!rc) rc = map3(&map_t, a.t, 2 * q.RP, a.T, a.B, 2 * q.RP, AT_M);
    if (!rc) rc = map3(&map_up, a.up, a.R, a.N, a.S, a.R, AT_N);
    if (!rc) rc = map3(&map_y, a.y, a.N, a.T, a.B, a.y_stride, AT_M);
    if (!rc) rc = map3(&map_out, a.out, a.N, a.T, a.B, a.out_stride, 32);
    if (rc != NCKV_OK) return rc;
    const int sms = sm_count();
    const long long tiles = (long long)a.B * q.tiles, n_steps = (a.N + AT_N - 1) / AT_N;
    if (tiles > 0x7fffffffLL / AT_MAX_CLUSTER) {
        set_error("adapters: B=%d requests of T=%d tokens are too many for one launch", a.B, a.T);
        return NCKV_E_UNSUPPORTED;
    }
    int ctas = 1;  // of a cluster: a power of two that a tile's rows and channels can be shared by
    while (ctas < AT_MAX_CLUSTER && 2 * ctas * tiles <= sms && 2 * ctas <= (a.K + AT_K - 1) / AT_K) ctas *= 2;  // (two to an SM: a third were on it at a time)
    q.stages = 8;
    while (q.stages > 4 && adapter_up_smem(q.RP, a.R, q.stages) > 220 * 1024) --q.stages;
    const size_t down_smem = adapter_down_smem(q.RP), up_smem = adapter_up_smem(q.RP, a.R, q.stages);
    static bool attr_set[64] = {false};
    int dev = 0;
    NCKV_CUDA_CHECK(cudaGetDevice(&dev));
    if (dev >= 64 || !attr_set[dev]) {
        NCKV_CUDA_CHECK(cudaFuncSetAttribute(adapter_tile_down, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024));
        NCKV_CUDA_CHECK(cudaFuncSetAttribute(adapter_tile_up, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024));
        if (dev < 64) attr_set[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(AT_THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)ctas;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cfg.gridDim = dim3((unsigned)(tiles * ctas));
    cfg.dynamicSmemBytes = down_smem;
    NCKV_CUDA_CHECK(cudaLaunchKernelEx(&cfg, adapter_tile_down, map_x, map_down, q));
    cfg.numAttrs = 1;
    cfg.blockDim = dim3(AT_UP_THREADS);
    cfg.gridDim = dim3((unsigned)(tiles * n_steps < sms ? tiles * n_steps : sms));
    cfg.dynamicSmemBytes = up_smem;
    NCKV_CUDA_CHECK(cudaLaunchKernelEx(&cfg, adapter_tile_up, map_t, map_up, map_y, map_out, q));
    return NCKV_OK;
}

// Tiles pay where many units of 8 rows would read the same adapters again and a tile is filled enough.  us in tiles / by rows, 1536 x 4608 at rank 16,
// an adapter to every request: 1 request of 128 tokens 7.9 / 7.0, 4 of 64 10.0 / 9.2, 4 of 128 10.5 / 9.2, 16 of 32 15.4 / 9.2, 16 of 64 16.1 / 14.4,
// 16 of 128 18.5 / 24.1, 64 of 32 32.0 / 24.5, 64 of 48 32.6 / 43.8, 64 of 128 42.2 / 86.5; rank 64 likewise.
bool adapters_tiled(int B, int T) { return T > 32 && (long long)B * ((T + 7) / 8) > 128; }

}  // namespace nckv
