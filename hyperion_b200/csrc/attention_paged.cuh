// What the two kernels of the shared-prefix attention have in common (attention_paged.cu:
// tiles of 16 rows and the merge; attention_paged_tc.cu: tiles of 128 rows).
#pragma once

#include "kernels.h"

namespace hyb {

constexpr float kSharedLog2e = 1.4426950408889634f;
constexpr int kTcRows = 128;

__device__ __forceinline__ float shared_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// How a call's rows and keys are split; the same on the host for the scratch size and the
// grids, and on the device. Parts of a row, in this order: those of the 128-row kernel, the
// prefix's and the request's own ones of the 16-row kernel.
struct SharedPlan {
    int tc_splits = 0;       // parts of the 128-row kernel (0: not launched)
    int tc_tiles = 0;        // 128-row tiles over all rows, or of one request
    int tc_per_request = 0;  // tiles hold one request's rows and cover prefix and own keys
    int tiles_p = 0, split_p = 0;  // 16-row tiles over all rows; parts of the prefix
    int tiles_o = 0, split_o = 0;  // 16-row tiles of one request; parts of its own keys
    int chunk_o = 0;               // own keys of one part
    __host__ __device__ int splits() const { return tc_splits + split_p + split_o; }
};

// Scratch: fp32 partial outputs [T][n_heads][n][hd], then (m, l) pairs [T][n_heads][n]; m in
// powers of two. A part with l = 0 has no output written.
struct SharedParts {
    float* o;
    float2* ml;
    int n;
};

void launch_shared_attn_tc(const SharedAttnParams& p, const SharedPlan& pl, const SharedParts& parts, cudaStream_t stream);

}  // namespace hyb
