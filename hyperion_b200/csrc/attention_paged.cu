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

__device__ int g_shared_small_wait_timeouts = 0;

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
constexpr int kTileRows = 16;
constexpr int kWarps = 4;
constexpr int kSlice = 16;  // keys of one warp step

SharedPlan plan_shared(int T, int n_req, int max_q, int max_own, int prefix_len, int n_heads, int n_kv, int hd) {
    SharedPlan s;
    const int G = n_heads / n_kv;
    max_q = std::min(max_q, T);
    const long long all_rows = static_cast<long long>(T) * G, req_rows = static_cast<long long>(max_q) * G;
    auto tiles = [](long long rows, int tile) { return static_cast<int>((rows + tile - 1) / tile); };
    // Tiles of one request's rows when they fill 128-row tiles about as well as the whole
    // batch's rows do: then prefix and own keys are one pass.
    if (req_rows > kTileRows && 4ll * n_req * tiles(req_rows, kTcRows) <= 5ll * tiles(all_rows, kTcRows)) {
        s.tc_per_request = 1;
        s.tc_tiles = tiles(req_rows, kTcRows);
    } else if (prefix_len > 128 && all_rows > kTileRows) {
        s.tc_tiles = tiles(all_rows, kTcRows);
    }
    if (s.tc_tiles > 0) {
        const long long units = static_cast<long long>(s.tc_tiles) * n_kv * (s.tc_per_request ? n_req : 1);
        const long long blocks = (static_cast<long long>(prefix_len) + (s.tc_per_request ? max_own : 0) + 63) / 64;
        s.tc_splits = static_cast<int>(std::max<long long>(1, std::min<long long>((blocks + 1) / 2, 148 / units)));
        if (s.tc_per_request) return s;
    }
    // A single request shares with nobody, and a short prefix costs less to read again than
    // to treat apart.
    s.o_prefix = s.tc_tiles == 0 && prefix_len > 0 && (n_req == 1 || prefix_len <= 128);
    const bool prefix_items = s.tc_tiles == 0 && prefix_len > 0 && !s.o_prefix;
    const long long keys_o = static_cast<long long>(max_own) + (s.o_prefix ? prefix_len : 0);
    s.tiles_o = keys_o > 0 ? tiles(req_rows, kTileRows) : 0;
    s.tiles_p = prefix_items ? tiles(all_rows, kTileRows) : 0;
    // Parts of about the same length: as many as two CTAs on every SM take at once, of 64 keys
    // (a shorter part is all latency) to 256 KB of K and V (the SMs finish within one part of each
    // other). Half of max_own stands for the requests' mean.
    const long long units_o = static_cast<long long>(s.tiles_o) * n_kv * n_req, units_p = static_cast<long long>(s.tiles_p) * n_kv;
    const long long work = units_o * (s.o_prefix ? prefix_len + max_own / 2 : max_own / 2) + units_p * prefix_len;
    const long long part = std::min<long long>(1024, std::max<long long>(64, (work / 296 + 63) / 64 * 64));
    if (s.tiles_p > 0) s.split_p = static_cast<int>((prefix_len + part - 1) / part);
    if (s.tiles_o > 0) {
        s.chunk_o = static_cast<int>(part / kSlice);
        s.split_o = static_cast<int>(((prefix_len * (s.o_prefix ? 1ll : 0ll) + kSlice - 1) / kSlice + (max_own + kSlice - 1) / kSlice + s.chunk_o - 1) / s.chunk_o);
    }
    return s;
}

// The keys of one segment (prefix or own) for a tile of rows: those in [lo, hi) are seen by some
// row, its slices start at key `first`.
struct Keys {
    const int* table;
    int base, lo, hi, first, slices;
};
__device__ __forceinline__ Keys keys_of(const int* table, int base, int len, int pmin, int pmax, int window) {
    Keys k;
    k.table = table;
    k.base = base;
    k.hi = static_cast<int>(min(static_cast<long long>(len), max(0ll, static_cast<long long>(pmax) + 1 - base)));
    k.lo = 0;
    if (window > 0) k.lo = static_cast<int>(min(static_cast<long long>(k.hi), max(0ll, static_cast<long long>(pmin) - window + 1 - base)));
    k.first = k.lo & ~(kSlice - 1);
    // without a window the slices depend on the length alone, so that their pages can be looked
    // up before the rows' positions are known
    k.slices = window > 0 ? (k.hi > k.lo ? (k.hi - k.first + kSlice - 1) / kSlice : 0) : (len + kSlice - 1) / kSlice;
    return k;
}

template <int HD>
struct SmallPlan {
    // K or V of one slice is one stage, head_dim / 64 boxes of [16 keys][128 bytes]; 24 KB a warp,
    // so that two CTAs share an SM and one streams while the other starts or ends
    static constexpr int kHalf = kSlice * HD * 2;
    static constexpr int kStages = 24 * 1024 / kHalf;
    static constexpr int kRing = kWarps * kStages * kHalf;
    static constexpr int kMerge = kWarps * kTileRows * HD * 4;
    static constexpr int kBars = kRing > kMerge ? kRing : kMerge;
    static constexpr int kSmem = kBars + kWarps * kStages * 8 + 1024;  // + alignment slack
};

// One CTA: up to 16 rows (row m of a tile = token m / G, head m % G of the KV head's group)
// against one part of the prefix, or of one request's keys. Each warp takes every fourth
// 16-key slice of the part on its own: tensor-map copies into its own ring, QK^T and PV on
// mma.sync m16n8k16, online softmax; the four warps' results are joined at the end. V rows
// of keys that no row of the tile sees are cleared before the product (0 * NaN). Rows
// share every byte of K and V that is loaded, so up to 16 rows cost the same traffic as one:
// HBM bound, if the eight warps of an SM get through a slice in 1.5 us at head_dim 128; so
// copies are issued for a whole slice at once (per-lane 16-byte copies took half of 660
// instructions a slice), and masks and rescaling sit behind warp-uniform branches.
// The chain in front of the first copy is three loads deep: lengths, row starts and pages;
// positions; keys.
template <int HD>
__global__ void __launch_bounds__(kWarps * 32, 2)
    shared_attn_small_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                             const SharedAttnParams p, const SharedPlan pl, SharedParts parts, int after_tc) {
    using SP = SmallPlan<HD>;
    constexpr int KS = HD / 16, SUB = HD / 64, ST = SP::kStages;
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* sm = smem_dyn + ((1024 - (smem_u32(smem_dyn) & 1023)) & 1023);
    __shared__ float s_m[kWarps][kTileRows], s_l[kWarps][kTileRows];
    __shared__ int s_row[kTileRows];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = p.n_heads / p.n_kv;
    const uint32_t leader = lane == 0;
    const uint32_t ring = smem_u32(sm) + warp * ST * SP::kHalf, full = smem_u32(sm) + SP::kBars + warp * ST * 8;
    pdl_launch_dependents();
    if (lane < ST) mbar_init(full + 8 * lane, 1);
    mbar_init_fence();
    __syncwarp();

    // ---- which part
    int id = blockIdx.x;
    const int n_prefix = pl.tiles_p * p.n_kv * pl.split_p;
    const bool prefix = id < n_prefix;
    int split, hk, tile, req = 0;
    if (prefix) {
        split = id % pl.split_p;
        id /= pl.split_p;
        hk = id % p.n_kv;
        tile = id / p.n_kv;
    } else {
        id -= n_prefix;
        hk = id % p.n_kv;
        id /= p.n_kv;
        split = id % pl.split_o;
        id /= pl.split_o;
        tile = id % pl.tiles_o;
        req = id / pl.tiles_o;
    }
    // ---- lengths, row starts
    int t0 = 0, n_tok = p.T, own = 0;
    const long long most = min(static_cast<long long>(p.max_own), static_cast<long long>(p.max_blocks) * p.page_size);
    bool broken = false;
    if (!prefix) {
        const int a = p.row_start[req], b = p.row_start[req + 1], len = p.own_lens[req];
        t0 = min(max(a, 0), p.T);
        n_tok = min(min(b, p.T) - t0, p.max_q);
        own = static_cast<int>(min(static_cast<long long>(max(0, len)), most));
        broken = len > most;
    }
    const int len_p = prefix || pl.o_prefix ? p.prefix_len : 0;
    const int per = prefix ? 0 : pl.chunk_o;
    const int* own_table = p.table + static_cast<size_t>(req) * p.max_blocks;
    // ---- the pages of this warp's first 32 slices, one a lane, while no window moves the slices
    int pages = 0;
    const int slices_p = (len_p + kSlice - 1) / kSlice;
    // a prefix item splits the prefix evenly, in steps of 64 keys
    const int per_p = prefix ? (((p.prefix_len + pl.split_p - 1) / pl.split_p + 63) & ~63) / kSlice : 0;
    if (p.window == 0) {
        const int s = split * (prefix ? per_p : per) + warp + lane * kWarps;
        if (s < slices_p) pages = p.prefix_table[s * kSlice / p.page_size];
        else if (!prefix && s - slices_p < (own + kSlice - 1) / kSlice) pages = own_table[(s - slices_p) * kSlice / p.page_size];
    }
    if (parts.direct && tile == pl.tiles_o - 1 && split == 0) shared_fill_unserved(p, req, hk, t0, kWarps * 32);
    // ---- rows m0 .. m0 + rows of the (token, head) pairs from token t0 on
    const int m0 = tile * kTileRows;
    const int rows = static_cast<int>(max(0ll, min(static_cast<long long>(kTileRows), static_cast<long long>(n_tok) * G - m0)));
    if (rows <= 0) {
        if (after_tc) pdl_wait();
        return;
    }
    // lane m (and m + 16): row m's position and place
    const int mm = m0 + min(lane & 15, rows - 1), tok = mm / G;
    const int my_pos = (lane & 15) < rows ? p.row_pos[t0 + tok] : -1;
    const int my_row = (t0 + tok) * p.n_heads + hk * G + (mm - tok * G);
    const int g = lane >> 2, c2 = 2 * (lane & 3);
    uint32_t qf[KS][4];
    {
        const bf16* qa = p.q + static_cast<size_t>(__shfl_sync(0xffffffffu, my_row, g)) * HD;
        const bf16* qb = p.q + static_cast<size_t>(__shfl_sync(0xffffffffu, my_row, g + 8)) * HD;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            qf[k][0] = *reinterpret_cast<const uint32_t*>(qa + 16 * k + c2);
            qf[k][1] = *reinterpret_cast<const uint32_t*>(qb + 16 * k + c2);
            qf[k][2] = *reinterpret_cast<const uint32_t*>(qa + 16 * k + 8 + c2);
            qf[k][3] = *reinterpret_cast<const uint32_t*>(qb + 16 * k + 8 + c2);
        }
    }
    if (warp == 0 && lane < kTileRows) s_row[lane] = my_row | (my_pos < 0 ? 0x80000000 : 0);
    const int pmin = __reduce_min_sync(0xffffffffu, my_pos < 0 ? INT_MAX : my_pos);
    const int pmax = __reduce_max_sync(0xffffffffu, my_pos);
    const int posA = __shfl_sync(0xffffffffu, my_pos, g), posB = __shfl_sync(0xffffffffu, my_pos, g + 8);
    // ---- its keys: slices [s0, s1) of the prefix's, then the request's own
    const Keys ka = keys_of(p.prefix_table, 0, len_p, pmin, pmax, p.window);
    const Keys kb = keys_of(own_table, p.prefix_len, own, pmin, pmax, p.window);
    const int total = ka.slices + kb.slices;
    const int step = !prefix ? per : (p.window == 0 ? per_p : (ka.slices + pl.split_p - 1) / pl.split_p);
    const int s0 = static_cast<int>(min(static_cast<long long>(total), static_cast<long long>(split) * step));
    const int s1 = min(total, s0 + step);
    const int mine = s1 - s0 > warp ? (s1 - s0 - warp + kWarps - 1) / kWarps : 0;

    float o[HD / 8][4];
#pragma unroll
    for (int i = 0; i < HD / 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
    float mA = -INFINITY, mB = -INFINITY, lA = 0.f, lB = 0.f;
    bool bad = false;

    bool ok = true;
    const int page_shift = __ffs(p.page_size) - 1, in_page = p.page_size - 1;
    auto load_pages = [&](int from) {  // of this warp's slices from .. from + 31, as first slots
        const int i = from + lane, s = s0 + warp + i * kWarps;
        const bool a = s < ka.slices;
        const int key = a ? ka.first + s * kSlice : kb.first + (s - ka.slices) * kSlice;
        if ((from > 0 || p.window > 0) && i < mine) pages = (a ? ka.table : kb.table)[key >> page_shift];
        const bool there = pages >= 0 && pages < p.n_pages;
        if (i < mine && !there) bad = true;
        // slices without a visible key, and bad pages: a box past the pool, which reads as zeros
        pages = i < mine && there && key < (a ? ka.hi : kb.hi) ? (pages << page_shift) + (key & in_page) : p.n_pages << page_shift;
    };
    int f_slot = 0;
    auto fetch = [&](int j) {  // K (even) or V (odd) of this warp's slice j / 2
        const int i = j >> 1;
        if (i < mine) {
            if ((j & 63) == 0) load_pages(i);
            const int at = __shfl_sync(0xffffffffu, pages, i & 31);
            const uint32_t bar = full + 8 * f_slot, dst = ring + f_slot * SP::kHalf;
            if (lane == 0) mbar_expect_tx(bar, SP::kHalf);
            __syncwarp();
#pragma unroll
            for (int d = 0; d < SUB; ++d)
                shared_tma_load_if(dst + d * (kSlice * 128), (j & 1) ? &tm_v : &tm_k, 64 * d, hk, at, bar, leader);
        }
        f_slot = f_slot + 1 == ST ? 0 : f_slot + 1;
    };
#pragma unroll
    for (int j = 0; j < ST - 1; ++j) fetch(j);
    const bool plain = p.softcap <= 0.f && p.scale > 0.f;  // the maximum is taken over the raw products
    const float s2 = plain ? p.scale * kSharedLog2e : 1.f;
    // ldmatrix offsets of this lane in a [16 keys][128 bytes] box, for the four 32-byte columns
    uint32_t k_off[4], v_off[4];
    {
        const int kk = (lane & 7) + ((lane >> 4) << 3), kh = (lane >> 3) & 1, vk = lane & 15, vh = lane >> 4;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            k_off[c] = kk * 128 + (((2 * c + kh) ^ (kk & 7)) << 4);
            v_off[c] = vk * 128 + (((2 * c + vh) ^ (vk & 7)) << 4);
        }
    }
    int slot = 0, phase = 0;
    for (int i = 0; i < mine; ++i) {
        fetch(2 * i + ST - 1);
        const int s = s0 + warp + i * kWarps;
        const bool in_a = s < ka.slices;
        const int key0 = in_a ? ka.first + s * kSlice : kb.first + (s - ka.slices) * kSlice;
        const int lo = in_a ? ka.lo : kb.lo, hi = in_a ? ka.hi : kb.hi, base = in_a ? 0 : p.prefix_len;
        // scores of 16 rows x 16 keys: this lane's rows g, g + 8 and keys c2, c2 + 1 (+ 8)
        float v[8];
        {
            shared_warp_wait(ok, full + 8 * slot, phase, &g_shared_small_wait_timeouts);
            const uint32_t kt = ring + slot * SP::kHalf;
            float s0v[4] = {0.f, 0.f, 0.f, 0.f}, s1v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                uint32_t b0, b1, b2, b3;
                ldsm_x4(kt + (k >> 2) * (kSlice * 128) + k_off[k & 3], b0, b1, b2, b3);
                mma_bf16_16816(s0v, qf[k][0], qf[k][1], qf[k][2], qf[k][3], b0, b1);
                mma_bf16_16816(s1v, qf[k][0], qf[k][1], qf[k][2], qf[k][3], b2, b3);
            }
            v[0] = s0v[0], v[1] = s0v[1], v[2] = s1v[0], v[3] = s1v[1];
            v[4] = s0v[2], v[5] = s0v[3], v[6] = s1v[2], v[7] = s1v[3];
            if (++slot == ST) slot = 0, phase ^= 1;
        }
        if (!plain) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                v[j] = kSharedLog2e * (p.softcap > 0.f ? p.softcap * tanhf(v[j] * p.scale / p.softcap) : v[j] * p.scale);
        }
        const bool inside = key0 >= lo && key0 + kSlice <= hi;
        if (!(inside && base + key0 + kSlice - 1 <= pmin && (p.window == 0 || base + key0 > pmax - p.window))) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int key = key0 + c2 + (j & 1) + ((j & 2) << 2), kp = base + key, pos = j < 4 ? posA : posB;
                if (!(key >= lo && key < hi && kp <= pos && (p.window == 0 || kp > pos - p.window))) v[j] = -INFINITY;
            }
        }
        float xA = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), xB = fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7]));
#pragma unroll
        for (int w = 1; w <= 2; w <<= 1) {
            xA = fmaxf(xA, __shfl_xor_sync(0xffffffffu, xA, w));
            xB = fmaxf(xB, __shfl_xor_sync(0xffffffffu, xB, w));
        }
        xA *= s2;
        xB *= s2;
        // the reference of a row: its first maximum, moved when outgrown by 2^40 (fp32's exponent
        // range carries the rest). A row that has seen no key keeps -inf; 0 stands in below, so that
        // no inf - inf appears.
        const bool upA = xA > mA + kSharedLazy || (mA == -INFINITY && xA > -INFINITY);
        const bool upB = xB > mB + kSharedLazy || (mB == -INFINITY && xB > -INFINITY);
        if (__any_sync(0xffffffffu, upA || upB)) {
            const float nA = upA ? xA : mA, nB = upB ? xB : mB;
            const float aA = upA ? shared_ex2(mA - nA) : 1.f, aB = upB ? shared_ex2(mB - nB) : 1.f;
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
        const float zA = mA == -INFINITY ? 0.f : mA, zB = mB == -INFINITY ? 0.f : mB;
        uint32_t pf[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float z = j < 2 ? zA : zB;
            pf[j] = shared_pack(shared_ex2(fmaf(v[2 * j], s2, -z)), shared_ex2(fmaf(v[2 * j + 1], s2, -z)));
            const float sum = __uint_as_float(pf[j] << 16) + __uint_as_float(pf[j] & 0xffff0000u);
            if (j < 2) lA += sum;
            else lB += sum;
        }
        __syncwarp();  // every lane has read the K stage that the next copy refills
        fetch(2 * i + ST);
        {
            shared_warp_wait(ok, full + 8 * slot, phase, &g_shared_small_wait_timeouts);
            const uint32_t vt = ring + slot * SP::kHalf;
            if (!inside) {
                const int head = min(kSlice, max(0, lo - key0)), tail = max(0, min(kSlice, hi - key0));  // rows before, from
                const int n = tail <= head ? kSlice : head + kSlice - tail;
                for (int j = lane; j < n * SUB * 8; j += 32) {
                    const int r = j / (SUB * 8), key = tail <= head || r < head ? r : tail + r - head, ch = j % (SUB * 8);
                    asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(vt + (ch >> 3) * (kSlice * 128) + key * 128 + (ch & 7) * 16),
                                 "r"(0)
                                 : "memory");
                }
                fence_proxy_async();  // before a later copy into the stage
                __syncwarp();
            }
#pragma unroll
            for (int d = 0; d < HD / 16; ++d) {
                uint32_t b0, b1, b2, b3;
                ldsm_x4_t(vt + (d >> 2) * (kSlice * 128) + v_off[d & 3], b0, b1, b2, b3);
                mma_bf16_16816(o[2 * d], pf[0], pf[2], pf[1], pf[3], b0, b1);
                mma_bf16_16816(o[2 * d + 1], pf[0], pf[2], pf[1], pf[3], b2, b3);
            }
            if (++slot == ST) slot = 0, phase ^= 1;
        }
        __syncwarp();  // and the V stage
    }
    if (!ok) {
        // a wait gave up: give copies that may still be in flight the same time again
        const uint64_t from = shared_now_ns();
        while (shared_now_ns() - from < 500000000ull) __nanosleep(1000);
    }
#pragma unroll
    for (int w = 1; w <= 2; w <<= 1) {
        lA += __shfl_xor_sync(0xffffffffu, lA, w);
        lB += __shfl_xor_sync(0xffffffffu, lB, w);
    }
    // a page outside the pool: the rows of the tile come out as NaN, not as a silent subset
    if (__any_sync(0xffffffffu, bad) || (broken && parts.direct)) {
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
        const size_t row = static_cast<size_t>(s_row[m] & 0x7fffffff);
        if (!parts.direct) {
            if (L != 0.f) *reinterpret_cast<float4*>(parts.o + (row * parts.n + at) * HD + d) = acc;
            if (d == 0) parts.ml[row * parts.n + at] = make_float2(M, L);
        } else if (s_row[m] >= 0) {  // the only part of its rows: the output itself
            const float inv = L > 0.f ? 1.0f / L : L;
            *reinterpret_cast<uint2*>(p.out + row * HD + d) =
                make_uint2(pack_bf2(f2bf(acc.x * inv), f2bf(acc.y * inv)), pack_bf2(f2bf(acc.z * inv), f2bf(acc.w * inv)));
        }
    }
    // this grid may start under the 128-row kernel's last CTAs; it ends after them, so that the
    // merge, which waits for this grid, waits for both
    if (after_tc) pdl_wait();
}

// W warps per (row, head) join its parts, each every W-th. Rows before row_start[0] or from
// row_start[n_req] on belong to no request and are left as they were; a row whose request
// breaks the bounds the caller gave (more rows than max_q, more keys than max_own or its
// table) has parts that were not computed and becomes NaN.
template <int HD>
__global__ void __launch_bounds__(256) shared_merge_kernel(const SharedAttnParams p, SharedParts parts, int W) {
    constexpr int PER = HD / 32;
    __shared__ float s_o[8][HD];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp % W;
    const long long unit = (static_cast<long long>(blockIdx.x) * 8 + warp) / W;
    const int t = static_cast<int>(min(unit / p.n_heads, static_cast<long long>(p.T)));
    bool live = t < p.T, broken = false;
    if (live) {
        live = t >= p.row_start[0] && t < p.row_start[p.n_req] && p.row_pos[t] >= 0;
        if (live) {
            int lo = 0, hi = p.n_req;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (p.row_start[mid] <= t) lo = mid;
                else hi = mid;
            }
            const int own = p.own_lens[lo];
            broken = t - p.row_start[lo] >= p.max_q || own > p.max_own ||
                     own > static_cast<long long>(p.max_blocks) * p.page_size;
        }
    }
    pdl_wait();
    float L = 0.f, acc[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] = 0.f;
    if (live) {
        const float2* ml = parts.ml + static_cast<size_t>(unit) * parts.n;
        const float* src = parts.o + static_cast<size_t>(unit) * parts.n * HD + lane * PER;
        float M = -INFINITY;
        for (int s = lane; s < parts.n; s += 32) M = fmaxf(M, ml[s].x);
        M = warp_max(M);
        const float z = M == -INFINITY ? 0.f : M;
        for (int s0 = 0; s0 < parts.n; s0 += 32) {
            float f = 0.f, fl = 0.f;
            if (s0 + lane < parts.n) {
                const float2 v = ml[s0 + lane];
                f = v.y == 0.f ? 0.f : shared_ex2(v.x - z);  // l = 0: no key of the part is seen, no output written
                fl = f * v.y;
            }
            L += warp_sum(fl);
            const int n = min(32, parts.n - s0);
#pragma unroll 4
            for (int s = sub; s < n; s += W) {
                const float fs = __shfl_sync(0xffffffffu, f, s);
                if (fs == 0.f) continue;
                const float* at = src + static_cast<size_t>(s0 + s) * HD;
                if constexpr (PER == 2) {
                    const float2 x = *reinterpret_cast<const float2*>(at);
                    acc[0] += fs * x.x;
                    acc[1] += fs * x.y;
                } else {
#pragma unroll
                    for (int i = 0; i < PER; i += 4) {
                        const float4 x = *reinterpret_cast<const float4*>(at + i);
                        acc[i] += fs * x.x;
                        acc[i + 1] += fs * x.y;
                        acc[i + 2] += fs * x.z;
                        acc[i + 3] += fs * x.w;
                    }
                }
            }
        }
    }
    if (W > 1) {
#pragma unroll
        for (int i = 0; i < PER; ++i) s_o[warp][lane * PER + i] = acc[i];
        __syncthreads();
        if (sub != 0) return;
        for (int w = 1; w < W; ++w)
#pragma unroll
            for (int i = 0; i < PER; ++i) acc[i] += s_o[warp + w][lane * PER + i];
    }
    if (!live) return;
    float inv = L > 0.f ? 1.0f / L : (L == 0.f ? 0.f : L);  // no key seen: zeros; NaN stays
    if (broken) inv = __int_as_float(0x7fffffff);
    uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + static_cast<size_t>(unit) * HD + lane * PER);
#pragma unroll
    for (int i = 0; i < PER / 2; ++i) dst[i] = pack_bf2(f2bf(acc[2 * i] * inv), f2bf(acc[2 * i + 1] * inv));
}

template <int HD>
void launch_shared_t(const SharedAttnParams& p, const SharedPlan& pl, const SharedParts& parts, cudaStream_t stream) {
    using SP = SmallPlan<HD>;
    const long long n_prefix = static_cast<long long>(pl.tiles_p) * p.n_kv * pl.split_p;
    const long long n_req = static_cast<long long>(pl.tiles_o) * p.n_kv * pl.split_o * p.n_req;
    const long long warps = static_cast<long long>(p.T) * p.n_heads;
    if (n_prefix + n_req > INT_MAX || warps > INT_MAX - 8) throw ArgError("sdpa_shared_prefix: too many parts");
    if (pl.tc_splits > 0) launch_shared_attn_tc(p, pl, parts, stream);
    if (n_prefix + n_req > 0) {
        allow_smem(reinterpret_cast<const void*>(shared_attn_small_kernel<HD>), SP::kSmem);
        CUtensorMap tk, tv;
        shared_pool_maps(p, kSlice, &tk, &tv);
        shared_launch(shared_attn_small_kernel<HD>, static_cast<unsigned>(n_prefix + n_req), kWarps * 32, SP::kSmem, stream,
                      pl.tc_splits > 0, tk, tv, p, pl, parts, pl.tc_splits > 0 ? 1 : 0);
    }
    if (parts.direct) return;  // the only part wrote the output
    // one warp joins a few parts as fast as several: the loads of four are in flight at once
    const int W = parts.n >= 16 ? 8 : (parts.n >= 8 ? 4 : (parts.n >= 4 ? 2 : 1));
    shared_launch(shared_merge_kernel<HD>, static_cast<unsigned>((warps * W + 7) / 8), 256, 0, stream, parts.n > 0, p, parts, W);
}

}  // namespace

size_t shared_attn_scratch_bytes(int T, int n_req, int max_q, int max_own, int prefix_len, int n_heads, int n_kv,
                                 int hd) {
    const SharedPlan s = plan_shared(T, n_req, max_q, max_own, prefix_len, n_heads, n_kv, hd);
    const size_t units = s.direct() ? 0 : static_cast<size_t>(T) * n_heads * s.splits();
    return units * hd * sizeof(float) + units * sizeof(float2) + 512;
}

void launch_shared_attn(const SharedAttnParams& p, cudaStream_t stream) {
    const SharedPlan pl = plan_shared(p.T, p.n_req, p.max_q, p.max_own, p.prefix_len, p.n_heads, p.n_kv, p.hd);
    const size_t units = static_cast<size_t>(p.T) * p.n_heads * pl.splits();
    if (p.scratch_bytes < shared_attn_scratch_bytes(p.T, p.n_req, p.max_q, p.max_own, p.prefix_len, p.n_heads, p.n_kv, p.hd))
        throw ArgError("sdpa_shared_prefix: scratch too small");
    SharedParts parts;
    parts.o = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(p.scratch) + 255) & ~static_cast<uintptr_t>(255));
    parts.ml = reinterpret_cast<float2*>(parts.o + units * p.hd);
    parts.n = pl.splits();
    parts.direct = pl.direct();
    switch (p.hd) {
        case 64: launch_shared_t<64>(p, pl, parts, stream); break;
        case 128: launch_shared_t<128>(p, pl, parts, stream); break;
        case 256: launch_shared_t<256>(p, pl, parts, stream); break;
        default: throw ArgError("sdpa_shared_prefix: head_dim must be 64, 128 or 256");
    }
}

int64_t read_shared_attn_wait_timeouts() {
    int a = 0;
    HYB_CUDA(cudaMemcpyFromSymbol(&a, g_shared_small_wait_timeouts, sizeof(int)));
    return a + read_shared_attn_tc_wait_timeouts();
}

}  // namespace hyb
