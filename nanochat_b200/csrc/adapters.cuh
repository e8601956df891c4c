// What the two forms of the adapters' launches share (adapters.cu, adapters_tc.cu).
#pragma once

#include "nckv_common.cuh"

namespace nckv {

constexpr int AD_MAX_RANK = 128;

struct AdapterParams {
    const __nv_bfloat16 *y, *x, *down, *up;
    __nv_bfloat16 *out;
    const int32_t *slots;
    const float *scales;
    void *t;  // scratch: down x
    int32_t *status;
    int64_t y_stride, x_stride, out_stride;
    int B, T, K, N, R, S;
};

// The form on the tensor cores: many tokens per request.
bool adapters_tiled(int B, int T);
size_t adapters_tc_bytes(int B, int T, int R);
int adapters_tc(const AdapterParams &p, cudaStream_t stream);

}  // namespace nckv
