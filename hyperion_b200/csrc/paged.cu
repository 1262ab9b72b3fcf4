// Paged KV cache of a batch: block tables, slot map and row tables from the requests'
// lengths (paged_plan_kernel), and the QK-norm + RoPE + cache write through the slot map
// (qkv_post_paged_kernel).
//
// A pool is [n_pages][page_size][n_kv][hd]; token j of a request lives in slot
// table[j / page_size] * page_size + j % page_size of the pool.
#include "kernels.h"

#include <algorithm>
#include <climits>
#include <mutex>
#include <set>
#include <utility>

namespace hyb {

void allow_smem(const void* kernel, size_t bytes) {
    static std::mutex mu;
    static std::set<std::pair<const void*, int>> done;
    int dev = 0;
    HYB_CUDA(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lk(mu);
    if (done.count({kernel, dev})) return;
    HYB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
    done.insert({kernel, dev});
}

namespace {

// ------------------------------------------------------------------------------ plan
// Request b holds c cached tokens and adds n. Its rows are the exclusive prefix sum of n;
// its new pages, ceil((c + n) / P) - ceil(c / P) of them, are the next entries of the free
// list in request order (a second exclusive prefix sum). Two scans of a few thousand
// integers are latency, not work, so every CTA repeats them over all requests (the lengths
// come from L2 after the first) instead of paying a second launch, and then fills its share
// of the rows: row r finds its request by binary search in the row starts, in shared memory.
// 64 requests of one token: 8.5 us; 512 requests of 1 to 1023 tokens (6.4 MB): 12.6 us.
constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;

__device__ __forceinline__ long long block_scan_ll(long long v, long long* total, long long* red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long n = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += n;
    }
    if (lane == 31) red[warp] = inc;
    __syncthreads();
    if (warp == 0) {
        long long t = red[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long n = __shfl_up_sync(0xffffffffu, t, o);
            if (lane >= o) t += n;
        }
        red[lane] = t;
    }
    __syncthreads();
    const long long before = warp ? red[warp - 1] : 0;
    *total = red[kPlanWarps - 1];
    __syncthreads();
    return before + inc - v;
}

// Pages that hold c >= 0 tokens; c + P - 1 may pass 2^31.
__device__ __forceinline__ int pages_of(int c, int P) { return c == 0 ? 0 : (c - 1) / P + 1; }

// The last index i in [0, n) with a[i] <= v (a ascending, a[0] <= v).
__device__ __forceinline__ int last_le(const int* a, int n, int v) {
    int lo = 0, hi = n;  // a[lo] <= v, a[hi] > v or hi == n
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= v) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(const PagedPlanParams p) {
    extern __shared__ int sm_plan[];
    __shared__ long long red[kPlanWarps];
    int* s_row = sm_plan;               // [n] first row
    int* s_page = s_row + p.n_req;      // [n] first free-list entry
    int* s_cached = s_page + p.n_req;   // [n] cached tokens; ~cached where the request is refused
    const int n = p.n_req, P = p.page_size;
    const int per = (n + kPlanThreads - 1) / kPlanThreads;
    const int b0 = min(n, static_cast<int>(threadIdx.x) * per), b1 = min(n, b0 + per);
    const long long table_tokens = static_cast<long long>(p.max_blocks) * P;

    long long rows = 0;
    for (int b = b0; b < b1; ++b) {
        const int c = p.cached[b], a = p.added[b];
        if (c >= 0 && a > 0) rows += a;
        s_cached[b] = c;
        s_page[b] = a;  // the added tokens until the second scan
    }
    long long total_rows = 0;
    long long r0 = block_scan_ll(rows, &total_rows, red);
    long long need = 0;
    for (int b = b0; b < b1; ++b) {
        const int c = s_cached[b], a = s_page[b];
        const bool sane = c >= 0 && a >= 0;
        const long long len = static_cast<long long>(c) + a;
        const long long r1 = r0 + (sane ? a : 0);
        s_row[b] = static_cast<int>(min(r0, static_cast<long long>(p.max_rows)));
        const bool fits = sane && len <= table_tokens && r1 <= p.max_rows;
        if (fits) need += (len + P - 1) / P - (c + static_cast<long long>(P) - 1) / P;
        r0 = r1;
    }
    long long total_need = 0;
    long long q0 = block_scan_ll(need, &total_need, red);
    // granted requests that need pages are a prefix of those that need some: the first one
    // the free list cannot serve leaves every later one past its end
    int refused = 0;
    long long taken = 0;
    for (int b = b0; b < b1; ++b) {
        const int c = s_cached[b], a = s_page[b];
        const bool sane = c >= 0 && a >= 0;
        const long long len = static_cast<long long>(c) + a;
        const long long r1 = (sane ? a : 0) + static_cast<long long>(s_row[b]);
        const bool fits = sane && len <= table_tokens && r1 <= p.max_rows;
        const long long nb = fits ? (len + P - 1) / P - (c + static_cast<long long>(P) - 1) / P : 0;
        const bool granted = fits && (nb == 0 || q0 + nb <= p.n_free);
        if (granted && nb > 0) taken = q0 + nb;
        refused += granted ? 0 : 1;
        s_page[b] = static_cast<int>(min(q0, static_cast<long long>(INT_MAX)));
        s_cached[b] = granted ? c : (c < 0 ? -1 : ~c);
        if (blockIdx.x == 0) {
            p.row_start[b] = s_row[b];
            p.total_lens[b] = granted ? static_cast<int>(len) : max(c, 0);
        }
        q0 += nb;
    }
    // block totals of `taken` (maximum) and `refused` (sum)
    long long tmax = taken;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        tmax = max(tmax, __shfl_xor_sync(0xffffffffu, tmax, o));
        refused += __shfl_xor_sync(0xffffffffu, refused, o);
    }
    __shared__ int s_refused;
    if (threadIdx.x == 0) s_refused = 0;
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = tmax;
    __syncthreads();
    if ((threadIdx.x & 31) == 0 && refused) atomicAdd(&s_refused, refused);
    long long pages = 0;
#pragma unroll 4
    for (int w = 0; w < kPlanWarps; ++w) pages = max(pages, red[w]);
    const int n_rows = static_cast<int>(min(total_rows, static_cast<long long>(p.max_rows)));
    __syncthreads();

    // ---- the pages taken, entered in their requests' tables
    const unsigned nthreads = gridDim.x * kPlanThreads, me = blockIdx.x * kPlanThreads + threadIdx.x;
    for (long long j = me; j < pages; j += nthreads) {
        const int b = last_le(s_page, n, static_cast<int>(j));
        const int held = pages_of(s_cached[b], P);
        p.table[static_cast<size_t>(b) * p.max_blocks + held + (j - s_page[b])] = p.free_pages[j];
    }
    // ---- rows; a row's page is an old entry of the table (which nobody writes here) or an
    // entry of the free list
    for (unsigned at_row = me; at_row < static_cast<unsigned>(p.max_rows); at_row += nthreads) {  // signed, the last step could pass 2^31
        const int r = static_cast<int>(at_row);
        int req = -1, pos = -1, slot = -1;
        if (r < n_rows) {
            req = last_le(s_row, n, r);
            const int sc = s_cached[req], c = sc < 0 ? ~sc : sc;
            const long long at = static_cast<long long>(c) + (r - s_row[req]);
            pos = static_cast<int>(min(p.pos0 + at, static_cast<long long>(INT_MAX)));
            if (sc >= 0) {
                const int local = static_cast<int>(at);  // inside the table
                const int blk = local / P, held = pages_of(c, P);
                const int page = blk < held ? p.table[static_cast<size_t>(req) * p.max_blocks + blk]
                                            : p.free_pages[s_page[req] + blk - held];
                if (page >= 0 && page < p.n_pages) slot = page * P + local % P;
            }
        }
        p.row_req[r] = req;
        p.row_pos[r] = pos;
        p.slot_map[r] = slot;
    }
    if (blockIdx.x == 0) {
        int bad = 0;
        // pages outside the pool: those taken, and the partly filled ones that are continued
        for (long long j = threadIdx.x; j < pages; j += kPlanThreads) {
            const int page = p.free_pages[j];
            bad += page < 0 || page >= p.n_pages;
        }
        for (int b = b0; b < b1; ++b) {
            const int c = s_cached[b];
            if (c <= 0 || c % P == 0 || p.added[b] == 0) continue;
            const int page = p.table[static_cast<size_t>(b) * p.max_blocks + c / P];
            bad += page < 0 || page >= p.n_pages;
        }
        __shared__ int s_bad;
        if (threadIdx.x == 0) s_bad = 0;
        __syncthreads();
        if (bad) atomicAdd(&s_bad, bad);
        __syncthreads();
        if (threadIdx.x == 0) {
            p.row_start[n] = n_rows;
            p.status[0] = static_cast<int>(pages);
            p.status[1] = n_rows;
            p.status[2] = s_refused;
            p.status[3] = s_bad;
        }
    }
}

// ------------------------------------------------------------------------------ append
// y = x * rsqrt(mean(x^2) + eps) * w (v: without w); RoPE turns the pair (e, e + hd/2) of q
// and k by pos * inv_freq[e]; everything in fp32, rounded to bf16 once. Each projection row is
// read once and written once; what bounds it is a row's chain (position, angles in double, a
// barrier, load, reduction, store) with nothing of the next row in flight. A group of hd/16 lanes owns one head and
// each lane 8 neighbouring elements of either half (two 16-byte accesses, and both ends of
// a pair in one lane), so a warp handles 512/hd heads at once; the row's hd/2 sines and
// cosines are computed once in shared memory for all its heads. Angles are reduced in
// double: pos * inv_freq in fp32 would be off by 2^-24 * pos radians (0.008 at 131072).
// 2048 rows of 16 query and 8 KV heads of 256 (67 MB): 22.5 us from HBM (3.0 TB/s; the bytes alone
// 10.2), 15.0 with the data in L2; 64 rows of 32 + 16 heads of 128: 5.2 us.
constexpr int kPostThreads = 256;

template <int HD>
__global__ void __launch_bounds__(kPostThreads) qkv_post_paged_kernel(const QkvPostPagedParams p) {
    constexpr int HALF = HD / 2, LANES = HALF / 8, GROUPS = kPostThreads / LANES;
    __shared__ float s_cos[HALF], s_sin[HALF];
    const int row = blockIdx.x;
    const int pos = p.row_pos[row];
    if (pos < 0) return;  // padding row: nothing is written
    const int slot = p.slot_map[row];
    const bool cached = slot >= 0 && slot < p.n_slots;
    for (int e = threadIdx.x; e < HALF; e += kPostThreads) {
        double turns = static_cast<double>(pos) * static_cast<double>(p.inv_freq[e]) * 0.31830988618379067154;
        turns -= 2.0 * rint(0.5 * turns);  // half turns in [-1, 1]
        sincospif(static_cast<float>(turns), &s_sin[e], &s_cos[e]);
    }
    __syncthreads();
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const unsigned mask = LANES == 32 ? 0xffffffffu : (((1u << LANES) - 1) << ((threadIdx.x & 31) / LANES * LANES));
    const int units = p.n_heads + (p.v_from_k ? 1 : 2) * p.n_kv;
    const bf16* src_row = p.qkv + static_cast<size_t>(row) * p.ld;
    for (int u = group; u < units; u += GROUPS) {
        const bf16* src = src_row + static_cast<size_t>(u) * HD + lane * 8;
        const uint4 lo = *reinterpret_cast<const uint4*>(src), hi = *reinterpret_cast<const uint4*>(src + HALF);
        float a[8], b[8];
        const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a[2 * i] = __uint_as_float(wl[i] << 16);
            a[2 * i + 1] = __uint_as_float(wl[i] & 0xffff0000u);
            b[2 * i] = __uint_as_float(wh[i] << 16);
            b[2 * i + 1] = __uint_as_float(wh[i] & 0xffff0000u);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += a[i] * a[i] + b[i] * b[i];
#pragma unroll
        for (int o = LANES / 2; o; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
        const float inv = rsqrtf(ss * (1.0f / HD) + p.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            a[i] *= inv;
            b[i] *= inv;
        }
        auto store = [&](bf16* dst, const float (&x)[8], const float (&y)[8]) {
            uint32_t ox[4], oy[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                ox[i] = pack_bf2(f2bf(x[2 * i]), f2bf(x[2 * i + 1]));
                oy[i] = pack_bf2(f2bf(y[2 * i]), f2bf(y[2 * i + 1]));
            }
            *reinterpret_cast<uint4*>(dst + lane * 8) = make_uint4(ox[0], ox[1], ox[2], ox[3]);
            *reinterpret_cast<uint4*>(dst + HALF + lane * 8) = make_uint4(oy[0], oy[1], oy[2], oy[3]);
        };
        const bool is_q = u < p.n_heads, is_k = !is_q && u < p.n_heads + p.n_kv;
        const size_t cell = static_cast<size_t>(cached ? slot : 0) * p.n_kv;
        if (!is_q && !cached) continue;
        if (!is_q && (!is_k || p.v_from_k)) {
            const int h = is_k ? u - p.n_heads : u - p.n_heads - p.n_kv;
            store(p.v_pool + (cell + h) * HD, a, b);
            if (!is_k) continue;
        }
        const bf16* w = (is_q ? p.q_norm : p.k_norm) + lane * 8;
        const uint4 ul = *reinterpret_cast<const uint4*>(w), uh = *reinterpret_cast<const uint4*>(w + HALF);
        const uint32_t vl[4] = {ul.x, ul.y, ul.z, ul.w}, vh[4] = {uh.x, uh.y, uh.z, uh.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int e = lane * 8 + i;
            const float x = a[i] * bf2f(static_cast<uint16_t>(vl[i / 2] >> (16 * (i & 1))));
            const float y = b[i] * bf2f(static_cast<uint16_t>(vh[i / 2] >> (16 * (i & 1))));
            a[i] = x * s_cos[e] - y * s_sin[e];
            b[i] = x * s_sin[e] + y * s_cos[e];
        }
        if (is_q) store(p.q_out + (static_cast<size_t>(row) * p.n_heads + u) * HD, a, b);
        else store(p.k_pool + (cell + u - p.n_heads) * HD, a, b);
    }
}

}  // namespace

void launch_paged_plan(const PagedPlanParams& p, cudaStream_t stream) {
    const size_t smem = static_cast<size_t>(p.n_req) * 3 * sizeof(int);
    allow_smem(reinterpret_cast<const void*>(paged_plan_kernel), kMaxPlanRequests * 3 * sizeof(int));
    // one row a thread until every SM has a CTA
    const int blocks = std::max(1, std::min((p.max_rows - 1) / kPlanThreads + 1, num_sms()));
    paged_plan_kernel<<<blocks, kPlanThreads, smem, stream>>>(p);
    HYB_LAUNCH_CHECK("paged_plan_kernel");
}

void launch_qkv_post_paged(const QkvPostPagedParams& p, cudaStream_t stream) {
    switch (p.hd) {
        case 64: qkv_post_paged_kernel<64><<<p.T, kPostThreads, 0, stream>>>(p); break;
        case 128: qkv_post_paged_kernel<128><<<p.T, kPostThreads, 0, stream>>>(p); break;
        case 256: qkv_post_paged_kernel<256><<<p.T, kPostThreads, 0, stream>>>(p); break;
        default: throw ArgError("qkv_post_paged: head_dim must be 64, 128 or 256");
    }
    HYB_LAUNCH_CHECK("qkv_post_paged_kernel");
}

}  // namespace hyb
