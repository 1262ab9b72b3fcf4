// What the two kernels of the shared-prefix attention have in common (attention_paged.cu:
// tiles of 16 rows and the merge; attention_paged_tc.cu: tiles of 128 rows).
#pragma once

#include "kernels.h"
#include "tma.cuh"

#include <utility>

namespace hyb {

constexpr float kSharedLog2e = 1.4426950408889634f;
constexpr int kTcRows = 128;
constexpr float kSharedLazy = 40.f;  // log2 of how far a row's maximum may outgrow its reference

__device__ __forceinline__ float shared_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ bool shared_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done)
                 : "r"(bar), "r"(parity)
                 : "memory");
    return done != 0;
}
__device__ __forceinline__ uint64_t shared_now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
__device__ __forceinline__ uint32_t shared_pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// Waits for the phase of this parity, for half a second at most. A thread that gave up once
// (ok is false) waits no more, so a launch whose copies never land ends after about that.
__device__ __forceinline__ void shared_wait(bool& ok, uint32_t bar, uint32_t parity, int* timeouts) {
    if (!ok || shared_try_wait(bar, parity)) return;
    const uint64_t t0 = shared_now_ns();
    do {
        if (shared_try_wait(bar, parity)) return;
    } while (shared_now_ns() - t0 < 500000000ull);
    atomicAdd(timeouts, 1);
    ok = false;
}

// The same by a whole warp, which goes on as one.
__device__ __forceinline__ void shared_warp_wait(bool& ok, uint32_t bar, uint32_t parity, int* timeouts) {
    if (!ok || __all_sync(0xffffffffu, shared_try_wait(bar, parity))) return;
    const uint64_t t0 = shared_now_ns();
    do {
        if (__all_sync(0xffffffffu, shared_try_wait(bar, parity))) return;
    } while (__all_sync(0xffffffffu, shared_now_ns() - t0 < 500000000ull));
    if ((threadIdx.x & 31) == 0) atomicAdd(timeouts, 1);
    ok = false;
}

// Issued by the lane whose `leader` is set, of a warp that goes on as one: a copy issued lane by
// lane with lane-dependent coordinates takes over 100 cycles.
__device__ __forceinline__ void shared_tma_load_if(uint32_t dst, const void* map, int c0, int c1, int c2, uint32_t bar, uint32_t leader) {
    asm volatile(
        "{\n .reg .pred q;\n setp.ne.u32 q, %6, 0;\n"
        " @q cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n}\n" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar), "r"(leader)
        : "memory");
}
// How a call's rows and keys are split; the same on the host for the scratch size and the
// grids, and on the device.
struct SharedPlan {
    int tc_splits = 0;       // parts of the 128-row kernel (0: not launched)
    int tc_tiles = 0;        // 128-row tiles over all rows, or of one request
    int tc_per_request = 0;  // tiles hold one request's rows and cover prefix and own keys
    int prefix_unit = 0;     // 16-row kernel: one tile of all rows against the prefix
    int tiles_o = 0;         // 16-row tiles of one request (0: not launched)
    int o_prefix = 0;        // they cover the prefix too
    int unit_req = 0, unit_rows = 0;  // how units are numbered, see unit_of
    int one_part = 0;        // a CTA takes a whole unit and writes the output
    int shares = 0;          // otherwise: shares of every KV head's slices, a warp each
    // The number of a 16-row unit: tile `tile` of request `req`, whose rows start at token t0. By request
    // (tiles_o numbers each) where all have tiles_o tiles or nearly so. Where one is much longer than the
    // others (a prefill chunk beside single rows) that would count every request as the longest, so there
    // t0 * G / 16 + req + tile for G rows a token: a request of n rows begins at a number at least
    // ceil(n / 16) below the next one's, as floor(x + y) + 1 >= floor(x) + ceil(y), and all stay below
    // T * G / 16 + n_req.
    __host__ __device__ int unit_of(int req, int t0, int tile) const {
        return prefix_unit + tile + req * unit_req + static_cast<int>(static_cast<unsigned long long>(t0) * unit_rows / 16);
    }
    // nothing has to be joined
    __host__ __device__ bool direct() const { return one_part != 0 || (tc_per_request != 0 && tc_splits == 1); }
};

// Scratch of the parts that shared_merge_kernel joins; m in powers of two, and a part with l = 0 has
// no output written.
struct SharedParts {
    // of the 128-row kernel: [T][n_heads][n][hd] outputs and [T][n_heads][n] (m, l)
    float* o;
    float2* ml;
    int n;
    int direct;  // no scratch and no merge
    // of the 16-row kernel: share w's piece of unit u has place w + u (unique: each piece after a
    // share's first, and each share after the first, raises one of the two): [places][n_kv][16][hd]
    // and [places][n_kv][16]; of every unit the first share that has a piece, and how many do
    float* po;
    float2* pml;
    int2* unit;
};

// Rows of request `req` at or past max_q (no tile holds them): NaN, in the heads of one KV head.
// For calls without a merge, by one CTA of the request.
__device__ __forceinline__ void shared_fill_unserved(const SharedAttnParams& p, int req, int hk, int t0, int threads) {
    const int t1 = min(p.row_start[req + 1], p.T), G = p.n_heads / p.n_kv;
    for (int t = max(t0, t0 + min(p.max_q, p.T)); t < t1; ++t) {
        if (p.row_pos[t] < 0) continue;
        uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + (static_cast<size_t>(t) * p.n_heads + hk * G) * p.hd);
        for (int i = threadIdx.x; i < G * p.hd / 2; i += threads) dst[i] = 0x7fff7fffu;
    }
}

// Launch with an optional programmatic dependency on the kernel before it in the stream.
template <typename... P, typename... A>
void shared_launch(void (*kern)(P...), unsigned grid, unsigned threads, size_t smem, cudaStream_t stream, bool pdl, A&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    HYB_CUDA(cudaLaunchKernelEx(&cfg, kern, std::forward<A>(args)...));
}

void launch_shared_attn_tc(const SharedAttnParams& p, const SharedPlan& pl, const SharedParts& parts, cudaStream_t stream);
int64_t read_shared_attn_tc_wait_timeouts();

// Tensor maps of the pools: boxes of 64 head_dim columns of one KV head x `box_slots` slots.
void shared_pool_maps(const SharedAttnParams& p, int box_slots, CUtensorMap* tk, CUtensorMap* tv);

}  // namespace hyb
