// Shared-prefix attention for many rows on the 5th-generation tensor cores: the part of
// attention_paged.cu's work whose rows fill a 128-row tile.
//
// One CTA: 128 (token, head) rows of one KV head against a run of 64-key blocks. The rows are
// those of the whole batch against the prefix (decode), or those of one request against the
// prefix and then its own keys (prefill). One pass over the keys with a running maximum:
//   S = Q K^T (tcgen05.mma, fp32 in TMEM, two buffers), p = exp2(s - m) into a bf16 operand
//   in shared memory, O += P V (fp32 in TMEM).
// The reference maximum m of a row moves only when the running one has outgrown it by more
// than 2^8: p then stays below 256, which costs neither bf16 nor the fp32 sums any
// precision, and the 128 x head_dim accumulator is rescaled a few times per row instead of
// once a block.
//
// Warps 0..7: softmax. Warp w reads TMEM lanes 32 (w % 4).. (one row a thread) and 32 of the
//   block's 64 key columns; the two warps of a row exchange their block maxima through shared
//   memory (one 64-thread barrier a block).
// Warp 8: producer. Looks the pages up (32 table entries at a time, one a lane) and issues
//   the tensor-map copies of the K and V blocks, one box a lane: 64 head_dim columns of
//   min(page_size, 64) slots, 128-byte swizzled.
// Warp 9: allocates TMEM and issues the MMAs from one lane, S(c + 1) before P V(c), so that
//   the softmax of a block runs under the products of its neighbours. In the few blocks that
//   stick out of the visible keys it first clears the V rows outside: what a pool holds there
//   may be NaN, and 0 * NaN would reach the sums.
// Every mbarrier wait is bounded; TMEM is freed before the CTA exits.
#include "attention_paged.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

#include <climits>

namespace hyb {

__device__ int g_shared_attn_wait_timeouts = 0;

namespace {

constexpr int kRows = kTcRows;  // 128
constexpr int kKeys = 64;
constexpr int kSoftWarps = 8;
constexpr int kSoftThreads = kSoftWarps * 32;
constexpr int kTmaWarp = kSoftWarps, kMmaWarp = kSoftWarps + 1;
constexpr int kThreads = kSoftThreads + 64;
constexpr float kLazy = 8.f;  // log2 of how far a row's maximum may outgrow its reference

template <int HD>
struct TcShared {
    static constexpr uint32_t kTmemCols = HD > 128 ? 512 : 256;  // S 2 x 64 + O HD
    static constexpr int kSub = HD / 64;
    static constexpr int kSlots = HD == 256 ? 4 : 8;
    static constexpr int kPBufs = HD == 256 ? 1 : 2;  // a second one does not fit beside head_dim 256
    static constexpr int kQBytes = kRows * HD * 2;
    static constexpr int kTileBytes = kKeys * HD * 2;
    static constexpr int kPBytes = kRows * kKeys * 2;
    static constexpr int kOffSlots = kQBytes;
    static constexpr int kOffP = kOffSlots + kSlots * kTileBytes;
    static constexpr int kOffMax = kOffP + kPBufs * kPBytes;     // float [2][2][kRows]
    static constexpr int kOffPos = kOffMax + 4 * kRows * 4;      // int [kRows]
    static constexpr int kOffBars = kOffPos + kRows * 4;
    static constexpr int kSmem = kOffBars + 256 + 1024;          // + alignment slack
};

__device__ __forceinline__ bool wait_b(uint32_t bar, uint32_t parity) {
    if (mbar_wait_bounded(bar, parity)) return true;
    atomicAdd(&g_shared_attn_wait_timeouts, 1);
    return false;
}

// Instruction descriptor: bf16 A and B, f32 D; B MN-major when b_mn.
__host__ __device__ constexpr uint32_t idesc_bf16(int M, int N, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn ? (1u << 16) : 0u) | (static_cast<uint32_t>(N >> 3) << 17) |
           (static_cast<uint32_t>(M >> 4) << 24);
}

// MN-major 128-byte-swizzle descriptor: rows are keys, 64 head_dim values per 128-byte row;
// 64-wide groups `lbo` bytes apart, 8-key groups 1024 bytes apart.
__device__ __forceinline__ uint64_t mn_desc(uint32_t smem_addr, uint32_t lbo) {
    return static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4) | static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16 |
           static_cast<uint64_t>(1024 >> 4) << 32 | static_cast<uint64_t>(1) << 46 | static_cast<uint64_t>(2) << 61;
}

// Thread l writes TMEM lane (lane field of taddr) + l, 32 consecutive columns.
__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pair_sync(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }

// The keys of one segment (prefix or own) that a tile of rows sees: [lo, hi), in 64-key blocks.
struct Segment {
    const int* table;
    int base, lo, hi, blocks;
    __device__ int first() const { return lo & ~(kKeys - 1); }
};
__device__ __forceinline__ Segment segment(const int* table, int base, int len, int pmin, int pmax, int window) {
    Segment s;
    s.table = table;
    s.base = base;
    s.hi = static_cast<int>(min(static_cast<long long>(len), max(0ll, static_cast<long long>(pmax) + 1 - base)));
    s.lo = window > 0 && pmax >= 0
               ? static_cast<int>(min(static_cast<long long>(s.hi), max(0ll, static_cast<long long>(pmin) - window + 1 - base)))
               : 0;
    s.blocks = s.hi > s.lo ? (s.hi - s.first() + kKeys - 1) / kKeys : 0;
    return s;
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
    shared_attn_tc_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                          const SharedAttnParams p, const SharedPlan pl, SharedParts parts) {
    using S = TcShared<HD>;
    constexpr int SUB = S::kSub, SLOTS = S::kSlots, PB = S::kPBufs;
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* sm = smem_dyn + ((1024 - (smem_u32(smem_dyn) & 1023)) & 1023);
    const uint32_t sbase = smem_u32(sm);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = p.n_heads / p.n_kv;

    // ---- which rows and which part of the keys
    int id = blockIdx.x;
    const int split = id % pl.tc_splits;
    id /= pl.tc_splits;
    const int hk = id % p.n_kv;
    id /= p.n_kv;
    const bool per_request = pl.tc_per_request != 0;
    const int tile = per_request ? id % pl.tc_tiles : id, req = per_request ? id / pl.tc_tiles : 0;
    int t0 = 0, n_tok = p.T;
    if (per_request) {
        t0 = min(max(p.row_start[req], 0), p.T);
        n_tok = min(min(p.row_start[req + 1], p.T) - t0, p.max_q);
    }
    const long long m0 = static_cast<long long>(tile) * kRows;
    const int rows = static_cast<int>(max(0ll, min(static_cast<long long>(kRows), static_cast<long long>(n_tok) * G - m0)));
    if (rows <= 0) return;

    int* s_pos = reinterpret_cast<int*>(sm + S::kOffPos);
    float* s_max = reinterpret_cast<float*>(sm + S::kOffMax);
    const uint32_t slot_full = sbase + S::kOffBars;
    const uint32_t slot_empty = slot_full + 8 * SLOTS;
    const uint32_t s_full = slot_empty + 8 * SLOTS;  // [2]
    const uint32_t s_empty = s_full + 16;            // [2]
    const uint32_t p_full = s_empty + 16;            // [PB]
    const uint32_t p_empty = p_full + 16;            // [PB]
    const uint32_t o_full = p_empty + 16;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + S::kOffBars + 8 * (2 * SLOTS + 9));
    volatile int* s_bad = reinterpret_cast<volatile int*>(tmem_slot + 1);
    static_assert(8 * (2 * SLOTS + 9) + 8 <= 256, "barriers fit");

    if (threadIdx.x == 0) {
        for (int s = 0; s < SLOTS; ++s) {
            mbar_init(slot_full + 8 * s, 1);
            mbar_init(slot_empty + 8 * s, 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(s_full + 8 * s, 1);
            mbar_init(s_empty + 8 * s, kSoftWarps);
        }
        for (int s = 0; s < PB; ++s) {
            mbar_init(p_full + 8 * s, kSoftWarps);
            mbar_init(p_empty + 8 * s, 1);
        }
        mbar_init(o_full, 1);
        mbar_init_fence();
        *s_bad = 0;
    }
    if (warp == kMmaWarp) {
        tmem_alloc(smem_u32(tmem_slot), S::kTmemCols);
        tmem_relinquish();
    }
    if (threadIdx.x < kRows) s_pos[threadIdx.x] = threadIdx.x < rows ? p.row_pos[t0 + (m0 + threadIdx.x) / G] : -1;
    // queries: row r of the tile, 16-byte chunk ch of sub-tile d, in the K-major swizzled layout
    for (int i = threadIdx.x; i < kRows * (HD / 8); i += kThreads) {
        const int r = i / (HD / 8), ch = i % (HD / 8);
        uint4 v = make_uint4(0, 0, 0, 0);
        if (r < rows) {
            const long long pr = m0 + r;
            v = *reinterpret_cast<const uint4*>(p.q + ((t0 + pr / G) * p.n_heads + hk * G + pr % G) * HD + 8 * ch);
        }
        *reinterpret_cast<uint4*>(sm + (ch >> 3) * (kRows * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = v;
    }
    fence_proxy_async();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t tmem_s = tmem, tmem_o = tmem + 128;

    int pmin = INT_MAX, pmax = -1;
    for (int i = lane; i < kRows; i += 32)
        if (s_pos[i] >= 0) {
            pmin = min(pmin, s_pos[i]);
            pmax = max(pmax, s_pos[i]);
        }
    pmin = __reduce_min_sync(0xffffffffu, pmin);
    pmax = __reduce_max_sync(0xffffffffu, pmax);
    const Segment sp = segment(p.prefix_table, 0, p.prefix_len, pmin, pmax, p.window);
    Segment so = {nullptr, p.prefix_len, 0, 0, 0};
    if (per_request) {
        const long long most = min(static_cast<long long>(p.max_own), static_cast<long long>(p.max_blocks) * p.page_size);
        const int own = static_cast<int>(min(static_cast<long long>(max(0, p.own_lens[req])), most));
        so = segment(p.table + static_cast<size_t>(req) * p.max_blocks, p.prefix_len, own, pmin, pmax, p.window);
    }
    const int all = sp.blocks + so.blocks;
    const int c0 = static_cast<int>(static_cast<long long>(all) * split / pl.tc_splits);
    const int nb = static_cast<int>(static_cast<long long>(all) * (split + 1) / pl.tc_splits) - c0;
    // the segment and first key of this part's block c
    auto block = [&](int c, int& key0) -> const Segment& {
        const int b = c0 + c;
        const bool own = b >= sp.blocks;
        const Segment& s = own ? so : sp;
        key0 = s.first() + (own ? b - sp.blocks : b) * kKeys;
        return s;
    };
    bool ok = true;

    if (warp == kTmaWarp) {
        const int piece = min(p.page_size, kKeys);  // slots of one box
        const int pieces = kKeys / piece, boxes = SUB * pieces;
        const int per_load = pieces == 1 ? 32 : 32 / pieces;  // blocks whose pages 32 lanes hold
        int page = 0;
        for (int c = 0; c < nb; ++c) {
            int key0;
            if (c % per_load == 0) {
                // lane i: the page of piece i % pieces of block c + i / pieces; -1 past the visible keys
                page = -1;
                if (c + lane / pieces < nb) {
                    const Segment& s = block(c + lane / pieces, key0);
                    const int key = key0 + (lane % pieces) * piece;
                    if (key < s.hi && key + piece > s.lo) {
                        page = s.table[key / p.page_size];
                        if (page < 0 || page >= p.n_pages) {
                            *s_bad = 1;
                            page = -1;
                        }
                    }
                }
            }
            block(c, key0);
            const int src = (c % per_load) * pieces;
            const int mine = __shfl_sync(0xffffffffu, page, src + lane % pieces);
            // a page that nobody sees (or none): a box past the pool, which reads as zeros
            const int at = mine >= 0 ? mine * p.page_size + (key0 + (lane % pieces) * piece) % p.page_size : p.n_pages * p.page_size;
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                const int i = 2 * c + kv, slot = i % SLOTS;
                if (i >= SLOTS) ok &= wait_b(slot_empty + 8 * slot, ((i / SLOTS) - 1) & 1);
                if (lane == 0) mbar_expect_tx(slot_full + 8 * slot, S::kTileBytes);
                __syncwarp();
                if (lane < boxes) {
                    const int d = lane / pieces;
                    tma_load_3d(sbase + S::kOffSlots + slot * S::kTileBytes + d * (kKeys * 128) + (lane % pieces) * piece * 128,
                                kv ? &tm_v : &tm_k, 64 * d, hk, at, slot_full + 8 * slot);
                }
            }
        }
    } else if (warp == kMmaWarp) {
        constexpr uint32_t id_s = idesc_bf16(kRows, kKeys, false);
        constexpr uint32_t id_o = idesc_bf16(kRows, HD, true);
        auto issue_s = [&](int c) {
            const int i = 2 * c, slot = i % SLOTS, sb = c & 1;
            ok &= wait_b(slot_full + 8 * slot, (i / SLOTS) & 1);
            if (c >= 2) ok &= wait_b(s_empty + 8 * sb, ((c >> 1) - 1) & 1);
            tc_fence_after();
            if (lane == 0) {
                const uint32_t kbase = sbase + S::kOffSlots + slot * S::kTileBytes;
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk) {
                    const uint64_t ad = sw128_kmajor_desc(sbase + (kk >> 2) * (kRows * 128)) + 2 * (kk & 3);
                    const uint64_t bd = sw128_kmajor_desc(kbase + (kk >> 2) * (kKeys * 128)) + 2 * (kk & 3);
                    tc_mma_f16(tmem_s + 64 * sb, ad, bd, id_s, kk > 0 ? 1u : 0u);
                }
                tc_commit(s_full + 8 * sb);
                tc_commit(slot_empty + 8 * slot);
            }
            __syncwarp();
        };
        auto issue_pv = [&](int c) {
            const int i = 2 * c + 1, slot = i % SLOTS, pb = c % PB;
            ok &= wait_b(slot_full + 8 * slot, (i / SLOTS) & 1);
            int key0;
            const Segment& s = block(c, key0);
            if (key0 < s.lo || key0 + kKeys > s.hi) {
                unsigned char* vt = sm + S::kOffSlots + slot * S::kTileBytes;
                for (int j = lane; j < kKeys * SUB * 8; j += 32) {
                    const int key = (j >> 3) % kKeys, d = (j >> 3) / kKeys;
                    if (key0 + key < s.lo || key0 + key >= s.hi)
                        *reinterpret_cast<uint4*>(vt + d * (kKeys * 128) + key * 128 + (j & 7) * 16) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async();
                __syncwarp();
            }
            ok &= wait_b(p_full + 8 * pb, (c / PB) & 1);
            tc_fence_after();
            if (lane == 0) {
                const uint32_t vbase = sbase + S::kOffSlots + slot * S::kTileBytes;
#pragma unroll
                for (int kk = 0; kk < kKeys / 16; ++kk) {
                    const uint64_t ad = sw128_kmajor_desc(sbase + S::kOffP + pb * S::kPBytes) + 2 * kk;
                    const uint64_t bd = mn_desc(vbase + kk * 2048, kKeys * 128);
                    tc_mma_f16(tmem_o, ad, bd, id_o, (c > 0 || kk > 0) ? 1u : 0u);
                }
                tc_commit(p_empty + 8 * pb);
                tc_commit(slot_empty + 8 * slot);
            }
            __syncwarp();
        };
        if (nb > 0) {
            issue_s(0);
            for (int c = 0; c < nb; ++c) {
                if (c + 1 < nb) issue_s(c + 1);
                issue_pv(c);
            }
            if (lane == 0) tc_commit(o_full);
        }
    } else {
        const int grp = warp & 3, half = warp >> 2;
        const int r = 32 * grp + lane;
        const int pos = s_pos[r];
        const uint32_t lane_off = static_cast<uint32_t>(32 * grp) << 16;
        const float scale2 = p.scale * kSharedLog2e;
        float m = -INFINITY, l = 0.f;
        for (int c = 0; c < nb; ++c) {
            const int sb = c & 1, pb = c % PB;
            int key0;
            const Segment& s = block(c, key0);
            ok &= wait_b(s_full + 8 * sb, (c >> 1) & 1);
            tc_fence_after();
            uint32_t v[32];
            tmem_ld_32x32b_x32(tmem_s + lane_off + 64 * sb + 32 * half, v);
            tmem_ld_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(s_empty + 8 * sb);
            float x[32];
            if (p.softcap > 0.f) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    x[i] = p.softcap * kSharedLog2e * tanhf(__uint_as_float(v[i]) * p.scale / p.softcap);
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(v[i]) * scale2;
            }
            // blocks wholly inside every row's view skip the per-key mask
            const bool full = key0 >= s.lo && key0 + kKeys <= s.hi && s.base + key0 + kKeys - 1 <= pmin &&
                              (p.window == 0 || s.base + key0 > pmax - p.window);
            if (!full) {
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const int key = key0 + 32 * half + i, kp = s.base + key;
                    const bool see = key >= s.lo && key < s.hi && kp <= pos && (p.window == 0 || kp > pos - p.window);
                    if (!see) x[i] = -INFINITY;
                }
            }
            float mx = x[0];
#pragma unroll
            for (int i = 1; i < 32; ++i) mx = fmaxf(mx, x[i]);
            float* ex = s_max + (c & 1) * 2 * kRows;
            ex[half * kRows + r] = mx;
            pair_sync(1 + grp);
            mx = fmaxf(mx, ex[(half ^ 1) * kRows + r]);
            // both warps of the row see the same numbers and decide alike
            const bool move = mx > m + kLazy || (m == -INFINITY && mx > -INFINITY);
            if (__any_sync(0xffffffffu, move)) {
                const float nm = move ? mx : m;
                if (c > 0) {
                    const float f = move ? shared_ex2(m - nm) : 1.f;
                    l *= f;
                    ok &= wait_b(p_empty + 8 * ((c - 1) % PB), ((c - 1) / PB) & 1);  // P V(c - 1) is done
                    tc_fence_after();
#pragma unroll 1
                    for (int col = half * (HD / 2); col < (half + 1) * (HD / 2); col += 32) {
                        uint32_t o[32];
                        tmem_ld_32x32b_x32(tmem_o + lane_off + col, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        tmem_st_32x32b_x32(tmem_o + lane_off + col, o);
                        tmem_st_wait();
                    }
                    tc_fence_before();
                }
                m = nm;
            }
            const float z = m == -INFINITY ? 0.f : m;
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                w[i] = pack_bf2(f2bf(shared_ex2(x[2 * i] - z)), f2bf(shared_ex2(x[2 * i + 1] - z)));
                l += __uint_as_float(w[i] << 16) + __uint_as_float(w[i] & 0xffff0000u);
            }
            if (c >= PB) ok &= wait_b(p_empty + 8 * pb, ((c / PB) - 1) & 1);
            unsigned char* prow = sm + S::kOffP + pb * S::kPBytes + r * 128;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<uint4*>(prow + (((4 * half + i) ^ (r & 7)) << 4)) =
                    make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
            fence_proxy_async();  // generic-proxy writes -> the MMA's async-proxy reads
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 8 * pb);
        }
        // ---- the row's sum over both halves, then its accumulator
        float* ex = s_max + (nb & 1) * 2 * kRows;
        ex[half * kRows + r] = l;
        pair_sync(1 + grp);
        l += ex[(half ^ 1) * kRows + r];
        if (nb > 0) {
            ok &= wait_b(o_full, 0);
            tc_fence_after();
        }
        if (*s_bad) {
            m = 0.f;
            l = __int_as_float(0x7fffffff);
        }
        const long long pr = m0 + r;
        const size_t row = static_cast<size_t>(t0 + pr / G) * p.n_heads + hk * G + pr % G;
        if (r < rows && half == 0) parts.ml[row * parts.n + split] = make_float2(m, l);
        if (nb > 0) {
#pragma unroll 1
            for (int col = half * (HD / 2); col < (half + 1) * (HD / 2); col += 32) {
                uint32_t o[32];
                tmem_ld_32x32b_x32(tmem_o + lane_off + col, o);
                tmem_ld_wait();
                if (r < rows) {
                    float* dst = parts.o + (row * parts.n + split) * HD + col;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        *reinterpret_cast<uint4*>(dst + 4 * i) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                }
            }
        }
    }
    if (!ok && lane == 0) {
        // a wait gave up: wait (bounded) for copies and MMAs that may still be in flight
        const int n = 2 * nb;
        for (int s = 0; s < SLOTS && s < n; ++s) mbar_wait_bounded(slot_full + 8 * s, ((n - 1 - s) / SLOTS) & 1);
        mbar_wait_bounded(o_full, 0);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, S::kTmemCols);
    }
}

template <int HD>
void launch_t(const SharedAttnParams& p, const SharedPlan& pl, const SharedParts& parts, cudaStream_t stream) {
    using S = TcShared<HD>;
    CUtensorMap tk, tv;
    const uint64_t dims[3] = {HD, static_cast<uint64_t>(p.n_kv), static_cast<uint64_t>(p.n_pages) * p.page_size};
    const uint64_t strides[2] = {HD * 2, static_cast<uint64_t>(p.n_kv) * HD * 2};
    const uint32_t box[3] = {64, 1, static_cast<uint32_t>(p.page_size < kKeys ? p.page_size : kKeys)};
    encode_tma(&tk, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, p.k_pool, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    encode_tma(&tv, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, p.v_pool, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    allow_smem(reinterpret_cast<const void*>(shared_attn_tc_kernel<HD>), S::kSmem);
    const long long ctas = static_cast<long long>(pl.tc_tiles) * (pl.tc_per_request ? p.n_req : 1) * p.n_kv * pl.tc_splits;
    if (ctas > INT_MAX) throw ArgError("sdpa_shared_prefix: too many parts");
    shared_attn_tc_kernel<HD><<<static_cast<unsigned>(ctas), kThreads, S::kSmem, stream>>>(tk, tv, p, pl, parts);
    HYB_LAUNCH_CHECK("shared_attn_tc_kernel");
}

}  // namespace

void launch_shared_attn_tc(const SharedAttnParams& p, const SharedPlan& pl, const SharedParts& parts, cudaStream_t stream) {
    switch (p.hd) {
        case 64: launch_t<64>(p, pl, parts, stream); break;
        case 128: launch_t<128>(p, pl, parts, stream); break;
        default: launch_t<256>(p, pl, parts, stream); break;
    }
}

int64_t read_shared_attn_wait_timeouts() {
    int a = 0;
    HYB_CUDA(cudaMemcpyFromSymbol(&a, g_shared_attn_wait_timeouts, sizeof(int)));
    return a;
}

}  // namespace hyb
