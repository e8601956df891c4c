// Low-rank adapters of many requests beside a projection that all of them share: for row r of request b with slot s = slots[b],
//   out_r = bf16(y_r + scale_s up_s (down_s x_r)),   out_r = y_r where s is negative,
// down (S, R, K), up (S, N, R), R at most 128.  Two launches: t = down x into fp32 scratch, then up t onto y.  Sums are fp32; between the
// products t is split into two bf16 terms (16 bits), so that nothing but the result is rounded to the activations' type.
//
// Few rows per adapter (decode, drafted tokens): memory-bound, on the adapters' bytes.  16 rows of one slot make a unit, T tokens of a request
// or requests of the same slot together, so that an adapter is read once for all of them.  Which requests a unit has every CTA finds from
// the slots (counts per slot, then the members in order; under the launch before it).  mma.sync, operands straight from global memory in
// 8- and 16-byte loads: the order of the channels inside a product is free, so a lane's consecutive ones stand for the two pairs that
// the instruction wants from it.
#include "adapters.cuh"

namespace nckv {

constexpr int AD_THREADS = 256, AD_ROWS = 16;

struct AdapterRows : AdapterParams {
    int chunks;       // units of AD_ROWS tokens per request
    int per_unit;     // requests of one slot that share a unit (1 where a request has several units)
    int splits, k_each, n_each;  // parts of the channels and outputs of a CTA
};

// Rows of a unit: row numbers in s_row (-1: none), and its slot (-1: no adapter).  False: there is no such unit.
__device__ __forceinline__ bool adapter_unit(const AdapterRows &p, int unit, int *s_row, int &slot, int &rows) {
    extern __shared__ int s_count[];  // requests of each slot, then of none
    __shared__ int s_warp[AD_THREADS / 32], s_which[2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid < AD_ROWS) s_row[tid] = -1;
    if (p.per_unit == 1) {
        const int b = unit / p.chunks, chunk = unit - b * p.chunks;
        slot = p.slots[b];
        if (slot >= p.S) slot = -1;
        rows = min(AD_ROWS, p.T - chunk * AD_ROWS);
        __syncthreads();
        if (tid < rows) s_row[tid] = b * p.T + chunk * AD_ROWS + tid;
        __syncthreads();
        return true;
    }
    for (int i = tid; i <= p.S; i += AD_THREADS) s_count[i] = 0;
    __syncthreads();
    for (int i = tid; i < p.B; i += AD_THREADS) {
        const int s = p.slots[i];
        atomicAdd(&s_count[s < 0 || s >= p.S ? p.S : s], 1);
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
        const int s = i < p.B ? p.slots[i] : -2;
        const bool member = i < p.B && (s < 0 || s >= p.S ? p.S : s) == which;
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

// t[part][row] = down x over a part of the channels: a warp takes every eighth step of 32 channels, the warps' sums meet in shared memory.
template <int TILES>  // of 8 ranks
__global__ void __launch_bounds__(AD_THREADS) adapter_down_kernel(const __grid_constant__ AdapterRows p) {
    __shared__ int s_row[AD_ROWS];
    __shared__ float s_t[AD_ROWS][TILES * 8 + 1];
    pdl_wait_prior_grids();
    pdl_launch_dependents();  // behind the wait: the next grid looks at the slots ahead of its own
    int slot, rows;
    if (!adapter_unit(p, blockIdx.x, s_row, slot, rows)) return;
    if (slot < 0) {
        if (blockIdx.y == 0 && (int)threadIdx.x < rows && p.slots[s_row[threadIdx.x] / p.T] >= p.S) atomicOr(p.status, (int)NCKV_ST_BAD_ADAPTER);
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane & 3, line = lane >> 2;
    const int k_lo = blockIdx.y * p.k_each, k_hi = min(k_lo + p.k_each, p.K);
    const int r0 = s_row[line], r1 = s_row[line + 8];
    const uint4 zero = make_uint4(0, 0, 0, 0);
    const __nv_bfloat16 *down = p.down + (long long)slot * p.R * p.K;
    float d[TILES][4];
#pragma unroll
    for (int i = 0; i < TILES; ++i) d[i][0] = d[i][1] = d[i][2] = d[i][3] = 0.f;
    for (int k = k_lo + warp * 32 + quad * 8; k - quad * 8 < k_hi; k += AD_THREADS) {
        const bool in = k < k_hi;
        uint4 a0 = zero, a1 = zero, b[TILES];
        if (in && r0 >= 0) a0 = *reinterpret_cast<const uint4 *>(p.x + r0 * p.x_stride + k);
        if (in && r1 >= 0) a1 = *reinterpret_cast<const uint4 *>(p.x + r1 * p.x_stride + k);
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            b[i] = zero;
            if (in && i * 8 + line < p.R) b[i] = *reinterpret_cast<const uint4 *>(down + (long long)(i * 8 + line) * p.K + k);
        }
#pragma unroll
        for (int i = 0; i < TILES; ++i) {
            mma_bf16_16816(d[i][0], d[i][1], d[i][2], d[i][3], a0.x, a1.x, a0.y, a1.y, b[i].x, b[i].y);
            mma_bf16_16816(d[i][0], d[i][1], d[i][2], d[i][3], a0.z, a1.z, a0.w, a1.w, b[i].z, b[i].w);
        }
    }
    // the warps' sums, one after the other: the order is fixed
    for (int w = 0; w < AD_THREADS / 32; ++w) {
        if (warp == w) {
#pragma unroll
            for (int i = 0; i < TILES; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float &s = s_t[line + (e >> 1) * 8][i * 8 + quad * 2 + (e & 1)];
                    s = w ? s + d[i][e] : d[i][e];
                }
        }
        __syncthreads();
    }
    float *t = static_cast<float *>(p.t) + (long long)blockIdx.y * p.B * p.T * p.R;
    for (int i = threadIdx.x; i < rows * p.R; i += AD_THREADS) {
        const int row = i / p.R, r = i - row * p.R;
        t[(long long)s_row[row] * p.R + r] = s_t[row][r];
    }
}

// What the second term of t holds; nothing beside an infinity, whose rest would be NaN.
__device__ __forceinline__ float adapter_rest(float t, float hi) { return fabsf(hi) <= 3.4e38f ? t - hi : 0.f; }

// out = y + scale up t over a part of the outputs: a warp takes 32 outputs at a time.  Output column of (product j, column c) is
// c / 2 * 8 + j * 2 + c % 2 of the 32, so that a lane holds 8 consecutive ones of a row.
template <int STEPS>  // of 16 ranks
__global__ void __launch_bounds__(AD_THREADS) adapter_up_kernel(const __grid_constant__ AdapterRows p) {
    __shared__ int s_row[AD_ROWS];
    __shared__ __align__(16) float s_t[AD_ROWS][STEPS * 16 + 4];
    int slot, rows;
    const bool any = adapter_unit(p, blockIdx.x, s_row, slot, rows);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane & 3, line = lane >> 2;
    const int n_lo = blockIdx.y * p.n_each, n_hi = min(n_lo + p.n_each, p.N);
    const int r0 = any ? s_row[line] : -1, r1 = any ? s_row[line + 8] : -1;
    const __nv_bfloat16 *up = p.up + (long long)(any && slot >= 0 ? slot : 0) * p.N * p.R;
    uint4 y0, y1;
    uint2 w[STEPS][4];
    auto load = [&](int n0) {  // what 32 outputs need
        const int n = n0 + quad * 8;
        y0 = y1 = make_uint4(0, 0, 0, 0);
        if (n < n_hi && r0 >= 0) y0 = *reinterpret_cast<const uint4 *>(p.y + r0 * p.y_stride + n);
        if (n < n_hi && r1 >= 0) y1 = *reinterpret_cast<const uint4 *>(p.y + r1 * p.y_stride + n);
        if (slot < 0) return;
#pragma unroll
        for (int i = 0; i < STEPS; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int at = n0 + line / 2 * 8 + j * 2 + (line & 1), r = i * 16 + quad * 4;
                w[i][j] = make_uint2(0, 0);
                if (at < n_hi && r < p.R) w[i][j] = *reinterpret_cast<const uint2 *>(up + (long long)at * p.R + r);
            }
    };
    int n0 = n_lo + warp * 32;
    if (any && n0 < n_hi && !(slot < 0 && p.out == p.y)) load(n0);  // neither y nor the adapters come from the launch before
    pdl_wait_prior_grids();
    if (!any || (slot < 0 && p.out == p.y)) return;
    uint32_t hi[STEPS][4], lo[STEPS][4];
    if (slot >= 0) {
        // t of the unit's rows, summed over the parts of the channels
        const float *t = static_cast<const float *>(p.t);
        const long long part = (long long)p.B * p.T * p.R;
        const int quads = STEPS * 4;
        for (int i = threadIdx.x; i < AD_ROWS * quads; i += AD_THREADS) {
            const int row = i / quads, r = i % quads * 4, at = s_row[row];
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
            if (at >= 0 && r < p.R) {
                const float *src = t + (long long)at * p.R + r;
#pragma unroll 4
                for (int s = 0; s < p.splits; ++s) {
                    const float4 v = *reinterpret_cast<const float4 *>(src + s * part);
                    sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
                }
            }
            *reinterpret_cast<float4 *>(&s_t[row][r]) = sum;
        }
        __syncthreads();
        // as two bf16 terms
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            const float4 t0 = *reinterpret_cast<const float4 *>(&s_t[line][i * 16 + quad * 4]), t1 = *reinterpret_cast<const float4 *>(&s_t[line + 8][i * 16 + quad * 4]);
            const float v[4][2] = {{t0.x, t0.y}, {t1.x, t1.y}, {t0.z, t0.w}, {t1.z, t1.w}};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                hi[i][e] = pack_bf16x2(v[e][0], v[e][1]);
                lo[i][e] = pack_bf16x2(adapter_rest(v[e][0], bf16lo(hi[i][e])), adapter_rest(v[e][1], bf16hi(hi[i][e])));
            }
        }
    }
    const float scale = slot >= 0 ? p.scales[slot] : 0.f;
    for (; n0 < n_hi;) {
        const int n = n0 + quad * 8;
        uint4 o0 = y0, o1 = y1;
        if (slot >= 0) {
            float d[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) d[j][0] = d[j][1] = d[j][2] = d[j][3] = 0.f;
#pragma unroll
            for (int i = 0; i < STEPS; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    mma_bf16_16816(d[j][0], d[j][1], d[j][2], d[j][3], hi[i][0], hi[i][1], hi[i][2], hi[i][3], w[i][j].x, w[i][j].y);
                    mma_bf16_16816(d[j][0], d[j][1], d[j][2], d[j][3], lo[i][0], lo[i][1], lo[i][2], lo[i][3], w[i][j].x, w[i][j].y);
                }
            auto add = [&](uint4 y, int e) {
                uint4 o;
                o.x = pack_bf16x2(bf16lo(y.x) + scale * d[0][e], bf16hi(y.x) + scale * d[0][e + 1]);
                o.y = pack_bf16x2(bf16lo(y.y) + scale * d[1][e], bf16hi(y.y) + scale * d[1][e + 1]);
                o.z = pack_bf16x2(bf16lo(y.z) + scale * d[2][e], bf16hi(y.z) + scale * d[2][e + 1]);
                o.w = pack_bf16x2(bf16lo(y.w) + scale * d[3][e], bf16hi(y.w) + scale * d[3][e + 1]);
                return o;
            };
            o0 = add(y0, 0);
            o1 = add(y1, 2);
        }
        n0 += AD_THREADS;
        if (n0 < n_hi) load(n0);
        if (n < n_hi && r0 >= 0) *reinterpret_cast<uint4 *>(p.out + r0 * p.out_stride + n) = o0;
        if (n < n_hi && r1 >= 0) *reinterpret_cast<uint4 *>(p.out + r1 * p.out_stride + n) = o1;
    }
}

// Units at most: known requests, unknown slots.  And in how many parts their channels go, so that there are enough CTAs for the chip, each
// with a step for all of its warps.
static long long adapter_units(int B, int T, int S, int *per_unit, int *chunks) {
    *chunks = (T + AD_ROWS - 1) / AD_ROWS;
    *per_unit = T < AD_ROWS ? AD_ROWS / T : 1;
    if (*per_unit == 1) return (long long)B * *chunks;
    const long long most = (long long)S + 1 + B / *per_unit;
    return most < B ? most : B;
}
static int adapter_parts(long long units, int channels, int ctas_per_sm, int least) {
    const long long want = (long long)ctas_per_sm * sm_count() / units, most = (channels + least - 1) / least;
    const long long n = want < most ? want : most;
    return (int)(n < 1 ? 1 : n);
}
constexpr int AD_MAX_SPLITS = 16;
static int adapter_splits(long long units, int K) {
    const int n = adapter_parts(units, K, 4, AD_THREADS);
    return n < AD_MAX_SPLITS ? n : AD_MAX_SPLITS;
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

}  // namespace nckv

extern "C" size_t nckv_adapters_workspace_bytes(int B, int T, int K, int N, int R, int S) {
    using namespace nckv;
    if (adapter_check_sizes("adapters_workspace_bytes", B, T, K, N, R, S) != NCKV_OK) return 0;
    if (adapters_tiled(T)) return adapters_tc_bytes(B, T, R);
    int per_unit, chunks;
    const long long units = adapter_units(B, T, S, &per_unit, &chunks);
    return (size_t)adapter_splits(units, K) * B * T * R * 4;
}

extern "C" int nckv_adapters(const void *y, int64_t y_stride, const void *x, int64_t x_stride, const void *down, const void *up,
                             const int32_t *slots, const float *scales, void *out, int64_t out_stride, int B, int T, int K, int N, int R,
                             int S, void *workspace, size_t workspace_bytes, int32_t *status, void *stream) {
    using namespace nckv;
    const char *name = "adapters";
    if (!y || !x || !down || !up || !slots || !scales || !out || !workspace || !status) {
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
    if (workspace_bytes < nckv_adapters_workspace_bytes(B, T, K, N, R, S)) {
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
    if (adapters_tiled(T)) return adapters_tc(p, static_cast<cudaStream_t>(stream));
    const long long units = adapter_units(B, T, S, &p.per_unit, &p.chunks);
    p.splits = adapter_splits(units, K);
    p.k_each = ((K + p.splits - 1) / p.splits + 31) / 32 * 32;
    const int n_parts = adapter_parts(units, N, 4, AD_THREADS);
    p.n_each = ((N + n_parts - 1) / n_parts + 31) / 32 * 32;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(AD_THREADS);
    cfg.dynamicSmemBytes = p.per_unit > 1 ? (size_t)(S + 1) * 4 : 0;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cfg.gridDim = dim3((unsigned)units, (unsigned)((K + p.k_each - 1) / p.k_each));
    p.splits = (int)cfg.gridDim.y;
    const int tiles = (R + 7) / 8;
    NCKV_CUDA_CHECK(cudaLaunchKernelEx(&cfg, tiles <= 1 ? adapter_down_kernel<1> : tiles <= 2 ? adapter_down_kernel<2> :
                                       tiles <= 4 ? adapter_down_kernel<4> : tiles <= 8 ? adapter_down_kernel<8> : adapter_down_kernel<16>, p));
    cfg.gridDim = dim3((unsigned)units, (unsigned)((N + p.n_each - 1) / p.n_each));
    NCKV_CUDA_CHECK(cudaLaunchKernelEx(&cfg, tiles <= 2 ? adapter_up_kernel<1> : tiles <= 4 ? adapter_up_kernel<2> : tiles <= 8 ? adapter_up_kernel<4> :
                                       adapter_up_kernel<8>, p));
    return NCKV_OK;
}
