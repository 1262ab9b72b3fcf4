// Attention of a batch of rows over a prefix that all requests share and over each
// request's own pages of a paged KV cache.
//
// Row t (of request b, at absolute position pos) sees the prefix keys at positions
// [0, prefix_len) and the request's own keys j < own_len at positions prefix_len + j, both
// only up to pos and, with a window, after pos - window. With s = scale * q.k (soft-capped
// when asked) the output is sum_j exp(s_j) v_j / sum_j exp(s_j). A softmax over a set of
// keys is joined exactly from its parts: a part keeps m = max s, l = sum exp(s - m) and
// o = sum exp(s - m) v, and the whole is sum_i exp(m_i - M) o_i / sum_i exp(m_i - M) l_i.
// So the prefix is one part for the batch (its keys are read once, with the rows of all
// requests as one matrix), each request's pages are others, long parts are split over the
// SMs, and shared_merge_kernel joins them.
//
// Statistics and accumulators are fp32. The probabilities are rounded to bf16 for the
// tensor cores, as unnormalised exp(s - m) <= 1, and l sums the rounded ones, so that the
// rounding cancels where all weights round alike.
#include "attention_paged.cuh"
#include "tma.cuh"

#include <algorithm>
#include <climits>

namespace hyb {

namespace {

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(a), "=r"(b), "=r"(c), "=r"(d)
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(a), "=r"(b), "=r"(c), "=r"(d)
                 : "r"(addr)
                 : "memory");
}
// 16 bytes global -> shared, or 16 zero bytes (nothing is read) when !take.
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool take) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

constexpr int kTileRows = 16;
constexpr int kWarps = 4;
constexpr int kSlice = 16;             // keys of one warp step
constexpr int kTargetCtas = 2 * 148;   // two waves of one CTA on every SM of a B200

SharedPlan plan_shared(int T, int n_req, int max_q, int max_own, int prefix_len, int n_heads, int n_kv) {
    SharedPlan s;
    const int G = n_heads / n_kv;
    max_q = std::min(max_q, T);
    const long long all_rows = static_cast<long long>(T) * G, req_rows = static_cast<long long>(max_q) * G;
    auto tiles = [](long long rows, int tile) { return static_cast<int>((rows + tile - 1) / tile); };
    // Tiles of one request's rows when they fill 128-row tiles about as well as the whole
    // batch's rows do: then prefix and own keys are one pass.
    const bool per_request = req_rows > kTileRows && 4ll * n_req * tiles(req_rows, kTcRows) <= 5ll * tiles(all_rows, kTcRows);
    if (per_request) {
        s.tc_per_request = 1;
        s.tc_tiles = tiles(req_rows, kTcRows);
    } else if (prefix_len > 0 && all_rows > kTileRows) {
        s.tc_tiles = tiles(all_rows, kTcRows);
    }
    if (s.tc_tiles > 0) {
        const long long units = static_cast<long long>(s.tc_tiles) * n_kv * (per_request ? n_req : 1);
        const long long blocks = (prefix_len + (per_request ? max_own : 0) + 63) / 64;
        s.tc_splits = static_cast<int>(std::max<long long>(1, std::min<long long>((blocks + 1) / 2, 148 / units)));
        if (per_request) return s;
    } else if (prefix_len > 0) {
        s.tiles_p = tiles(all_rows, kTileRows);
        const long long units = static_cast<long long>(s.tiles_p) * n_kv;
        s.split_p = static_cast<int>(std::max<long long>(1, std::min<long long>((prefix_len + 63) / 64, kTargetCtas / units)));
    }
    if (max_own > 0) {
        s.tiles_o = tiles(req_rows, kTileRows);
        const long long units = static_cast<long long>(s.tiles_o) * n_kv * n_req;
        const long long want = std::max<long long>(1, std::min<long long>((max_own + 63) / 64, 2 * kTargetCtas / units));
        s.chunk_o = static_cast<int>(((max_own + want - 1) / want + 63) / 64 * 64);
        s.split_o = (max_own + s.chunk_o - 1) / s.chunk_o;
    }
    return s;
}

template <int HD>
struct SmallPlan {
    static constexpr int kStages = 3;
    static constexpr int kHalf = kSlice * HD * 2;          // K or V of one slice
    static constexpr int kStage = 2 * kHalf;
    static constexpr int kRing = kWarps * kStages * kStage;
    static constexpr int kMerge = kWarps * kTileRows * HD * 4;
    static constexpr int kSmem = kRing > kMerge ? kRing : kMerge;
};

// One CTA: up to 16 rows (row m of a tile = token m / G, head m % G of the KV head's group)
// against one part of the prefix or of one request's keys. Each warp takes every fourth
// 16-key slice of the part on its own: cp.async into its own 3-stage ring (zero fill of keys
// that no row of the tile sees, so whatever the pool holds there cannot reach a product),
// QK^T and PV on mma.sync m16n8k16, online softmax; the four warps' results are joined at
// the end. Rows share every byte of K and V that is loaded, so up to 16 rows cost the same
// traffic as one: HBM bound.
template <int HD>
__global__ void __launch_bounds__(kWarps * 32) shared_attn_small_kernel(const SharedAttnParams p, const SharedPlan pl,
                                                                        SharedParts parts) {
    using SP = SmallPlan<HD>;
    constexpr int KS = HD / 16, CH = HD / 8;
    extern __shared__ __align__(128) unsigned char sm[];
    __shared__ float s_m[kWarps][kTileRows], s_l[kWarps][kTileRows];
    __shared__ int s_pos[kTileRows];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = p.n_heads / p.n_kv;

    // ---- which part
    long long id = blockIdx.x;
    const long long n_prefix = static_cast<long long>(pl.tiles_p) * p.n_kv * pl.split_p;
    const bool prefix = id < n_prefix;
    int split, hk, tile, req = 0;
    if (prefix) {
        split = static_cast<int>(id % pl.split_p);
        id /= pl.split_p;
        hk = static_cast<int>(id % p.n_kv);
        tile = static_cast<int>(id / p.n_kv);
    } else {
        id -= n_prefix;
        hk = static_cast<int>(id % p.n_kv);
        id /= p.n_kv;
        split = static_cast<int>(id % pl.split_o);
        id /= pl.split_o;
        tile = static_cast<int>(id % pl.tiles_o);
        req = static_cast<int>(id / pl.tiles_o);
    }
    // ---- its rows: m in [m0, m0 + rows) of the (token, head) pairs from token t0 on
    int t0 = 0, n_tok = p.T;
    if (!prefix) {
        t0 = min(max(p.row_start[req], 0), p.T);
        n_tok = min(min(p.row_start[req + 1], p.T) - t0, p.max_q);
    }
    const long long m0 = static_cast<long long>(tile) * kTileRows;
    const int rows = static_cast<int>(max(0ll, min(static_cast<long long>(kTileRows), static_cast<long long>(n_tok) * G - m0)));
    if (rows <= 0) return;
    if (threadIdx.x < kTileRows)
        s_pos[threadIdx.x] = threadIdx.x < rows ? p.row_pos[t0 + (m0 + threadIdx.x) / G] : -1;
    __syncthreads();
    int pmin = INT_MAX, pmax = -1;
#pragma unroll
    for (int m = 0; m < kTileRows; ++m)
        if (s_pos[m] >= 0) {
            pmin = min(pmin, s_pos[m]);
            pmax = max(pmax, s_pos[m]);
        }
    // ---- its keys: [lo, hi) are seen by some row, [k0, k1) are this part's
    const int base = prefix ? 0 : p.prefix_len;
    const long long table_keys = static_cast<long long>(p.max_blocks) * p.page_size;
    const int len = prefix ? p.prefix_len
                           : static_cast<int>(min(static_cast<long long>(max(0, min(p.own_lens[req], p.max_own))), table_keys));
    const int hi = min(len, max(0, pmax + 1 - base));
    const int lo = p.window > 0 && pmax >= 0
                       ? static_cast<int>(min(static_cast<long long>(hi), max(0ll, static_cast<long long>(pmin) - p.window + 1 - base)))
                       : 0;
    const int first = lo & ~(kSlice - 1);  // parts start on slice borders
    const int per = prefix ? ((hi - first + pl.split_p - 1) / pl.split_p + 63) & ~63 : pl.chunk_o;
    const long long from = first + static_cast<long long>(split) * per;
    const int k0 = static_cast<int>(min(from, static_cast<long long>(hi))), k1 = static_cast<int>(min(from + per, static_cast<long long>(hi)));
    const int* table = prefix ? p.prefix_table : p.table + static_cast<size_t>(req) * p.max_blocks;
    const int n_slices = k1 > k0 ? (k1 - k0 + kSlice - 1) / kSlice : 0;
    const int mine = n_slices > warp ? (n_slices - warp + kWarps - 1) / kWarps : 0;

    // ---- queries into fragments
    uint32_t qf[KS][4];
    const int g = lane >> 2, c2 = 2 * (lane & 3);
    {
        const int mA = g, mB = g + 8;
        const long long pa = m0 + min(mA, rows - 1), pb = m0 + min(mB, rows - 1);
        const bf16* qa = p.q + ((t0 + pa / G) * p.n_heads + hk * G + pa % G) * HD;
        const bf16* qb = p.q + ((t0 + pb / G) * p.n_heads + hk * G + pb % G) * HD;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            qf[k][0] = *reinterpret_cast<const uint32_t*>(qa + 16 * k + c2);
            qf[k][1] = *reinterpret_cast<const uint32_t*>(qb + 16 * k + c2);
            qf[k][2] = *reinterpret_cast<const uint32_t*>(qa + 16 * k + 8 + c2);
            qf[k][3] = *reinterpret_cast<const uint32_t*>(qb + 16 * k + 8 + c2);
        }
    }
    const int posA = s_pos[g], posB = s_pos[g + 8];
    float o[HD / 8][4];
#pragma unroll
    for (int i = 0; i < HD / 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
    float mA = -INFINITY, mB = -INFINITY, lA = 0.f, lB = 0.f;
    bool bad = false;

    const uint32_t ring = smem_u32(sm) + warp * SP::kStages * SP::kStage;
    int pages = 0;  // lane i: the page of this warp's slice i of the current 32
    auto load_pages = [&](int from) {
        const int i = from + lane;
        const int key = k0 + (warp + i * kWarps) * kSlice;
        pages = i < mine ? table[key / p.page_size] : 0;
        if (pages < 0 || pages >= p.n_pages) {
            bad = true;
            pages = -1;
        }
    };
    auto fetch = [&](int i) {  // this warp's slice i into stage i % kStages
        if (i < mine) {
            if ((i & 31) == 0) load_pages(i);
            const int page = __shfl_sync(0xffffffffu, pages, i & 31);
            const int key0 = k0 + (warp + i * kWarps) * kSlice;
            const size_t cell = (static_cast<size_t>(max(page, 0)) * p.page_size + key0 % p.page_size) * p.n_kv + hk;
            const bf16* kg = p.k_pool + cell * HD;
            const bf16* vg = p.v_pool + cell * HD;
            const uint32_t dst = ring + (i % SP::kStages) * SP::kStage;
            const size_t step = static_cast<size_t>(p.n_kv) * HD;
#pragma unroll
            for (int j = 0; j < kSlice * CH / 32; ++j) {
                const int idx = lane + 32 * j, key = idx / CH, ch = idx % CH;
                const bool take = page >= 0 && key0 + key >= lo && key0 + key < hi;
                const uint32_t at = dst + key * (HD * 2) + ((ch ^ (key & 7)) << 4);
                cp16(at, kg + (take ? key * step + ch * 8 : 0), take);
                cp16(at + SP::kHalf, vg + (take ? key * step + ch * 8 : 0), take);
            }
        }
        cp_commit();
    };
#pragma unroll
    for (int i = 0; i < SP::kStages - 1; ++i) fetch(i);
    const float scale2 = p.scale * kSharedLog2e;
    for (int i = 0; i < mine; ++i) {
        fetch(i + SP::kStages - 1);
        cp_wait<SP::kStages - 1>();
        __syncwarp();
        const uint32_t kb = ring + (i % SP::kStages) * SP::kStage, vb = kb + SP::kHalf;
        const int key0 = k0 + (warp + i * kWarps) * kSlice;
        // scores of 16 rows x 16 keys: this lane's rows g, g + 8 and keys c2, c2 + 1 (+ 8)
        float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
        {
            const int key = (lane & 7) + ((lane >> 4) << 3), half = (lane >> 3) & 1;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint32_t b0, b1, b2, b3;
                ldsm_x4(kb + key * (HD * 2) + (((2 * k + half) ^ (key & 7)) << 4), b0, b1, b2, b3);
                mma_bf16_16816(s0, qf[k][0], qf[k][1], qf[k][2], qf[k][3], b0, b1);
                mma_bf16_16816(s1, qf[k][0], qf[k][1], qf[k][2], qf[k][3], b2, b3);
            }
        }
        auto shape = [&](float dot, int key, int pos) {
            float s = p.softcap > 0.f ? p.softcap * kSharedLog2e * tanhf(dot * p.scale / p.softcap) : dot * scale2;
            const int kp = base + key;
            const bool see = key >= lo && key < hi && kp <= pos && (p.window == 0 || kp > pos - p.window);
            return see ? s : -INFINITY;
        };
        float v[8];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            v[j] = shape(s0[j], key0 + c2 + j, posA);
            v[2 + j] = shape(s1[j], key0 + 8 + c2 + j, posA);
            v[4 + j] = shape(s0[2 + j], key0 + c2 + j, posB);
            v[6 + j] = shape(s1[2 + j], key0 + 8 + c2 + j, posB);
        }
        float xA = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), xB = fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7]));
#pragma unroll
        for (int w = 1; w <= 2; w <<= 1) {
            xA = fmaxf(xA, __shfl_xor_sync(0xffffffffu, xA, w));
            xB = fmaxf(xB, __shfl_xor_sync(0xffffffffu, xB, w));
        }
        const float nA = fmaxf(mA, xA), nB = fmaxf(mB, xB);
        // a row that has seen no key keeps m = -inf; 0 stands in so that no inf - inf appears
        const float zA = nA == -INFINITY ? 0.f : nA, zB = nB == -INFINITY ? 0.f : nB;
        if (__any_sync(0xffffffffu, nA != mA || nB != mB)) {
            const float aA = shared_ex2(mA - zA), aB = shared_ex2(mB - zB);
            lA *= aA;
            lB *= aB;
#pragma unroll
            for (int d = 0; d < HD / 8; ++d) {
                o[d][0] *= aA;
                o[d][1] *= aA;
                o[d][2] *= aB;
                o[d][3] *= aB;
            }
            mA = nA;
            mB = nB;
        }
        uint32_t pf[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float z = j < 2 ? zA : zB;
            pf[j] = pack_bf2(f2bf(shared_ex2(v[2 * j] - z)), f2bf(shared_ex2(v[2 * j + 1] - z)));
            const float sum = __uint_as_float(pf[j] << 16) + __uint_as_float(pf[j] & 0xffff0000u);
            if (j < 2) lA += sum;
            else lB += sum;
        }
        {
            const int key = lane & 15, half = lane >> 4;
#pragma unroll
            for (int d = 0; d < HD / 16; ++d) {
                uint32_t b0, b1, b2, b3;
                ldsm_x4_t(vb + key * (HD * 2) + (((2 * d + half) ^ (key & 7)) << 4), b0, b1, b2, b3);
                mma_bf16_16816(o[2 * d], pf[0], pf[2], pf[1], pf[3], b0, b1);
                mma_bf16_16816(o[2 * d + 1], pf[0], pf[2], pf[1], pf[3], b2, b3);
            }
        }
        __syncwarp();  // every lane has read the stage that the next fetch refills
    }
    cp_wait<0>();
#pragma unroll
    for (int w = 1; w <= 2; w <<= 1) {
        lA += __shfl_xor_sync(0xffffffffu, lA, w);
        lB += __shfl_xor_sync(0xffffffffu, lB, w);
    }
    // a page outside the pool: the rows of the tile come out as NaN, not as a silent subset
    if (__any_sync(0xffffffffu, bad)) {
        lA = lB = __int_as_float(0x7fffffff);
        mA = mB = 0.f;
    }
    if ((lane & 3) == 0) {
        s_m[warp][g] = mA;
        s_m[warp][g + 8] = mB;
        s_l[warp][g] = lA;
        s_l[warp][g + 8] = lB;
    }
    __syncthreads();  // statistics written; every warp is done with its ring
    float* so = reinterpret_cast<float*>(sm) + warp * kTileRows * HD;
#pragma unroll
    for (int d = 0; d < HD / 8; ++d) {
        *reinterpret_cast<float2*>(so + g * HD + 8 * d + c2) = make_float2(o[d][0], o[d][1]);
        *reinterpret_cast<float2*>(so + (g + 8) * HD + 8 * d + c2) = make_float2(o[d][2], o[d][3]);
    }
    __syncthreads();
    const int at = pl.tc_splits + (prefix ? split : pl.split_p + split);
    for (int idx = threadIdx.x; idx < rows * (HD / 4); idx += kWarps * 32) {
        const int m = idx / (HD / 4), d = 4 * (idx % (HD / 4));
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_m[w][m]);
        const float z = M == -INFINITY ? 0.f : M;
        float L = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float f = shared_ex2(s_m[w][m] - z);
            const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(sm) + (w * kTileRows + m) * HD + d);
            L += f * s_l[w][m];
            acc.x += f * x.x;
            acc.y += f * x.y;
            acc.z += f * x.z;
            acc.w += f * x.w;
        }
        const long long pr = m0 + m;
        const size_t row = static_cast<size_t>(t0 + pr / G) * p.n_heads + hk * G + pr % G;
        if (L != 0.f) *reinterpret_cast<float4*>(parts.o + (row * parts.n + at) * HD + d) = acc;
        if (d == 0) parts.ml[row * parts.n + at] = make_float2(M, L);
    }
}

// One warp per (row, head): joins the parts. Rows before row_start[0] or from
// row_start[n_req] on belong to no request and are left as they were; a row whose request
// breaks the bounds the caller gave (more rows than max_q, more keys than max_own or its
// table) has parts that were not computed and becomes NaN.
template <int HD>
__global__ void __launch_bounds__(256) shared_merge_kernel(const SharedAttnParams p, SharedParts parts) {
    const int lane = threadIdx.x & 31;
    const long long unit = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) >> 5;
    if (unit >= static_cast<long long>(p.T) * p.n_heads) return;
    const int t = static_cast<int>(unit / p.n_heads);
    if (t < p.row_start[0] || t >= p.row_start[p.n_req] || p.row_pos[t] < 0) return;
    int lo = 0, hi = p.n_req;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (p.row_start[mid] <= t) lo = mid;
        else hi = mid;
    }
    const int own = p.own_lens[lo];
    const bool broken = t - p.row_start[lo] >= p.max_q || own > p.max_own ||
                        own > static_cast<long long>(p.max_blocks) * p.page_size;
    const int splits = parts.n;
    const float2* ml = parts.ml + unit * splits;
    const float* src = parts.o + unit * splits * HD;
    float M = -INFINITY;
    for (int s = lane; s < splits; s += 32) M = fmaxf(M, ml[s].x);
    M = warp_max(M);
    const float z = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    constexpr int PER = HD / 32;
    float acc[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] = 0.f;
    for (int s = 0; s < splits; ++s) {
        const float2 v = ml[s];
        if (v.y == 0.f) continue;  // no key of the part is seen
        const float f = shared_ex2(v.x - z);
        L += f * v.y;
#pragma unroll
        for (int i = 0; i < PER; ++i) acc[i] += f * src[static_cast<size_t>(s) * HD + lane * PER + i];
    }
    float inv = L > 0.f ? 1.0f / L : (L == 0.f ? 0.f : L);  // no key seen: zeros; NaN stays
    if (broken) inv = __int_as_float(0x7fffffff);
    uint32_t w[PER / 2];
#pragma unroll
    for (int i = 0; i < PER / 2; ++i) w[i] = pack_bf2(f2bf(acc[2 * i] * inv), f2bf(acc[2 * i + 1] * inv));
    uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + unit * HD + lane * PER);
#pragma unroll
    for (int i = 0; i < PER / 2; ++i) dst[i] = w[i];
}

template <int HD>
void launch_shared_t(const SharedAttnParams& p, const SharedPlan& pl, SharedParts parts, cudaStream_t stream) {
    using SP = SmallPlan<HD>;
    const long long n_prefix = static_cast<long long>(pl.tiles_p) * p.n_kv * pl.split_p;
    const long long n_own = static_cast<long long>(pl.tiles_o) * p.n_kv * pl.split_o * p.n_req;
    if (pl.tc_splits > 0) launch_shared_attn_tc(p, pl, parts, stream);
    if (n_prefix + n_own > INT_MAX) throw ArgError("sdpa_shared_prefix: too many parts");
    if (n_prefix + n_own > 0) {
        allow_smem(reinterpret_cast<const void*>(shared_attn_small_kernel<HD>), SP::kSmem);
        shared_attn_small_kernel<HD><<<static_cast<unsigned>(n_prefix + n_own), kWarps * 32, SP::kSmem, stream>>>(p, pl, parts);
        HYB_LAUNCH_CHECK("shared_attn_small_kernel");
    }
    const long long warps = static_cast<long long>(p.T) * p.n_heads;
    shared_merge_kernel<HD><<<static_cast<unsigned>((warps + 7) / 8), 256, 0, stream>>>(p, parts);
    HYB_LAUNCH_CHECK("shared_merge_kernel");
}

}  // namespace

size_t shared_attn_scratch_bytes(int T, int n_req, int max_q, int max_own, int prefix_len, int n_heads, int n_kv,
                                 int hd) {
    const SharedPlan s = plan_shared(T, n_req, max_q, max_own, prefix_len, n_heads, n_kv);
    const size_t units = static_cast<size_t>(T) * n_heads * s.splits();
    return units * hd * sizeof(float) + units * sizeof(float2) + 16;
}

void launch_shared_attn(const SharedAttnParams& p, cudaStream_t stream) {
    const SharedPlan pl = plan_shared(p.T, p.n_req, p.max_q, p.max_own, p.prefix_len, p.n_heads, p.n_kv);
    const size_t units = static_cast<size_t>(p.T) * p.n_heads * pl.splits();
    if (p.scratch_bytes < shared_attn_scratch_bytes(p.T, p.n_req, p.max_q, p.max_own, p.prefix_len, p.n_heads, p.n_kv, p.hd))
        throw ArgError("sdpa_shared_prefix: scratch too small");
    SharedParts parts;
    parts.o = static_cast<float*>(p.scratch);
    parts.ml = reinterpret_cast<float2*>(parts.o + units * p.hd);
    parts.n = pl.splits();
    switch (p.hd) {
        case 64: launch_shared_t<64>(p, pl, parts, stream); break;
        case 128: launch_shared_t<128>(p, pl, parts, stream); break;
        case 256: launch_shared_t<256>(p, pl, parts, stream); break;
        default: throw ArgError("sdpa_shared_prefix: head_dim must be 64, 128 or 256");
    }
}

}  // namespace hyb
