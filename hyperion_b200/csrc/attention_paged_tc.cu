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
// Warps 0..3 and 4..7: two softmax groups that take the blocks in turn, one row a thread, so
//   that the exponentials of one block run under the loads, maxima and stores of the next (a
//   single group leaves its own latency, some 3000 cycles a block, in the chain). A group
//   hands the rows' references on to the other before it starts its exponentials.
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
constexpr int kGroupWarps = 4;
constexpr int kTmaWarp = kSoftWarps, kMmaWarp = kSoftWarps + 1;
constexpr int kThreads = kSoftWarps * 32 + 64;
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
    static constexpr int kOffRef = kOffP + kPBufs * kPBytes;  // float [kRows]: the rows' references
    static constexpr int kOffSum = kOffRef + kRows * 4;       // float [kRows]: the second group's sums
    static constexpr int kOffPos = kOffSum + kRows * 4;       // int [kRows]: positions
    static constexpr int kOffRow = kOffPos + kRows * 4;       // int [kRows]: token * n_heads + head
    static constexpr int kOffBars = kOffRow + kRows * 4;
    static constexpr int kSmem = kOffBars + 256 + 1024;          // + alignment slack
};

__device__ __forceinline__ bool try_wait(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(done)
                 : "r"(bar), "r"(parity)
                 : "memory");
    return done != 0;
}
__device__ __forceinline__ uint64_t now_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
// Waits for the phase of this parity, for half a second at most. A thread that gave up once
// (ok is false) waits no more, so a launch whose copies never land ends after about that.
__device__ __forceinline__ void wait_b(bool& ok, uint32_t bar, uint32_t parity) {
    if (!ok || try_wait(bar, parity)) return;
    const uint64_t t0 = now_ns();
    do {
        if (try_wait(bar, parity)) return;
    } while (now_ns() - t0 < 500000000ull);
    atomicAdd(&g_shared_attn_wait_timeouts, 1);
    ok = false;
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
// Hand-over between warp w of one softmax group and warp w of the other.
__device__ __forceinline__ void hand_on(int id) { asm volatile("bar.arrive %0, 64;" ::"r"(id) : "memory"); }
__device__ __forceinline__ void take_over(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }
// 32 bytes to global memory (a whole sector).
__device__ __forceinline__ void st_v8(float* p, const uint32_t* r) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
                 "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ uint32_t pack_rn(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

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
    pdl_launch_dependents();
    if (parts.direct && tile == pl.tc_tiles - 1 && split == 0) shared_fill_unserved(p, req, hk, t0, kThreads);
    if (rows <= 0) return;

    int* s_pos = reinterpret_cast<int*>(sm + S::kOffPos);
    int* s_row = reinterpret_cast<int*>(sm + S::kOffRow);
    float* s_ref = reinterpret_cast<float*>(sm + S::kOffRef);
    float* s_sum = reinterpret_cast<float*>(sm + S::kOffSum);
    const uint32_t slot_full = sbase + S::kOffBars;
    const uint32_t slot_empty = slot_full + 8 * SLOTS;
    const uint32_t s_full = slot_empty + 8 * SLOTS;  // [2]
    const uint32_t s_empty = s_full + 16;            // [2]
    const uint32_t p_full = s_empty + 16;            // [2]: P of even and odd blocks is written
    const uint32_t pv_done = p_full + 16;            // [2]: P V of even and odd blocks is done
    const uint32_t o_full = pv_done + 16;
    const uint32_t q_full = o_full + 8;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sm + S::kOffBars + 8 * (2 * SLOTS + 10));
    volatile int* s_bad = reinterpret_cast<volatile int*>(tmem_slot + 1);
    static_assert(8 * (2 * SLOTS + 10) + 8 <= 256, "barriers fit");

    if (threadIdx.x == 0) {
        for (int s = 0; s < SLOTS; ++s) {
            mbar_init(slot_full + 8 * s, 1);
            mbar_init(slot_empty + 8 * s, 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(s_full + 8 * s, 1);
            mbar_init(s_empty + 8 * s, kGroupWarps);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(p_full + 8 * s, kGroupWarps);
            mbar_init(pv_done + 8 * s, 1);
        }
        mbar_init(o_full, 1);
        mbar_init(q_full, kSoftWarps);
        mbar_init_fence();
        *s_bad = 0;
    }
    if (warp == kMmaWarp) {
        tmem_alloc(smem_u32(tmem_slot), S::kTmemCols);
        tmem_relinquish();
    }
    if (threadIdx.x < kRows) {
        const int pr = static_cast<int>(m0) + min(static_cast<int>(threadIdx.x), rows - 1), tok = pr / G;
        s_pos[threadIdx.x] = static_cast<int>(threadIdx.x) < rows ? p.row_pos[t0 + tok] : -1;
        s_row[threadIdx.x] = (t0 + tok) * p.n_heads + hk * G + (pr - tok * G);
    }
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
    bool broken = false;
    if (per_request) {
        const long long most = min(static_cast<long long>(p.max_own), static_cast<long long>(p.max_blocks) * p.page_size);
        const int own = static_cast<int>(min(static_cast<long long>(max(0, p.own_lens[req])), most));
        broken = p.own_lens[req] > most;  // with several parts the merge says so
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
                if (i >= SLOTS) wait_b(ok, slot_empty + 8 * slot, ((i / SLOTS) - 1) & 1);
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
            wait_b(ok, slot_full + 8 * slot, (i / SLOTS) & 1);
            if (c >= 2) wait_b(ok, s_empty + 8 * sb, ((c >> 1) - 1) & 1);
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
            wait_b(ok, slot_full + 8 * slot, (i / SLOTS) & 1);
            int key0;
            const Segment& s = block(c, key0);
            if (key0 < s.lo || key0 + kKeys > s.hi) {
                unsigned char* vt = sm + S::kOffSlots + slot * S::kTileBytes;
                const int head = min(kKeys, max(0, s.lo - key0)), tail = min(kKeys, s.hi - key0);  // rows before, from
                for (int j = lane; j < (head + kKeys - tail) * SUB * 8; j += 32) {
                    const int n = j / (SUB * 8), key = n < head ? n : tail + n - head, ch = j % (SUB * 8);
                    *reinterpret_cast<uint4*>(vt + (ch >> 3) * (kKeys * 128) + key * 128 + (ch & 7) * 16) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async();
                __syncwarp();
            }
            wait_b(ok, p_full + 8 * (c & 1), (c >> 1) & 1);
            tc_fence_after();
            if (lane == 0) {
                const uint32_t vbase = sbase + S::kOffSlots + slot * S::kTileBytes;
#pragma unroll
                for (int kk = 0; kk < kKeys / 16; ++kk) {
                    const uint64_t ad = sw128_kmajor_desc(sbase + S::kOffP + pb * S::kPBytes) + 2 * kk;
                    const uint64_t bd = mn_desc(vbase + kk * 2048, kKeys * 128);
                    tc_mma_f16(tmem_o, ad, bd, id_o, (c > 0 || kk > 0) ? 1u : 0u);
                }
                tc_commit(pv_done + 8 * (c & 1));
                tc_commit(slot_empty + 8 * slot);
            }
            __syncwarp();
        };
        if (nb > 0) {
            wait_b(ok, q_full, 0);
            issue_s(0);
            for (int c = 0; c < nb; ++c) {
                if (c + 1 < nb) issue_s(c + 1);
                issue_pv(c);
            }
            if (lane == 0) tc_commit(o_full);
        }
    } else {
        // queries: row r of the tile, 16-byte chunk ch, in the K-major swizzled layout
#pragma unroll 8
        for (int i = threadIdx.x; i < kRows * (HD / 8); i += kSoftWarps * 32) {
            const int r = i / (HD / 8), ch = i % (HD / 8);
            const uint4 v = r < rows ? *reinterpret_cast<const uint4*>(p.q + static_cast<size_t>(s_row[r]) * HD + 8 * ch)
                                     : make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(sm + (ch >> 3) * (kRows * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4)) = v;
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);

        const int quad = warp & 3, group = warp >> 2;
        const int r = 32 * quad + lane;
        const int pos = s_pos[r];
        const uint32_t lane_off = static_cast<uint32_t>(32 * quad) << 16;
        const int mine = 1 + 2 * quad + group, other = 1 + 2 * quad + (group ^ 1);  // hand-over barriers
        // with a plain positive scale the maximum is taken over the raw products
        const bool plain = p.softcap <= 0.f && p.scale > 0.f;
        const float s2 = plain ? p.scale * kSharedLog2e : 1.f;
        float m = -INFINITY;  // the reference that l is held at
        float l = 0.f;
        for (int c = group; c < nb; c += 2) {
            const int pb = c % PB;
            int key0;
            const Segment& s = block(c, key0);
            wait_b(ok, s_full + 8 * group, (c >> 1) & 1);
            tc_fence_after();
            uint32_t v[2][32];
            tmem_ld_32x32b_x32(tmem_s + lane_off + 64 * group, v[0]);
            tmem_ld_32x32b_x32(tmem_s + lane_off + 64 * group + 32, v[1]);
            tmem_ld_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(s_empty + 8 * group);
            float x[64];
#pragma unroll
            for (int i = 0; i < 64; ++i) x[i] = __uint_as_float(v[i >> 5][i & 31]);
            if (!plain) {
#pragma unroll
                for (int i = 0; i < 64; ++i)
                    x[i] = kSharedLog2e * (p.softcap > 0.f ? p.softcap * tanhf(x[i] * p.scale / p.softcap) : x[i] * p.scale);
            }
            // blocks wholly inside every row's view skip the per-key mask
            const bool full = key0 >= s.lo && key0 + kKeys <= s.hi && s.base + key0 + kKeys - 1 <= pmin &&
                              (p.window == 0 || s.base + key0 > pmax - p.window);
            if (!full) {
                const long long wlo = p.window > 0 ? static_cast<long long>(pos) - p.window + 1 - s.base : 0;
                const int from = static_cast<int>(min(max(wlo, static_cast<long long>(s.lo)), static_cast<long long>(s.hi))) - key0;
                const int to = min(s.hi - 1, pos - s.base) + 1 - key0;
#pragma unroll
                for (int i = 0; i < 64; ++i)
                    if (i < from || i >= to) x[i] = -INFINITY;
            }
            float mx4[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
            for (int i = 4; i < 64; ++i) mx4[i & 3] = fmaxf(mx4[i & 3], x[i]);
            const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * s2;
            // the reference after block c - 1, moved if this block outgrows it, for block c + 1
            float ref = -INFINITY;
            if (c > 0) {
                take_over(other);
                ref = s_ref[r];
            }
            const bool move = mx > ref + kLazy || (ref == -INFINITY && mx > -INFINITY);
            const float now = move ? mx : ref;
            if (c + 1 < nb) {
                s_ref[r] = now;
                hand_on(mine);
            }
            // P V(c - 2) used this group's barrier last; the next use is P V(c), which needs this
            // group's P(c), so the barrier is one phase ahead at most and the parity is enough. With
            // P V(c - 2) done the same holds for the other group's barrier and P V(c - 1).
            if (c >= 2) wait_b(ok, pv_done + 8 * group, ((c - 2) >> 1) & 1);
            if (c > 0 && __any_sync(0xffffffffu, move)) {
                const float f = move ? shared_ex2(ref - now) : 1.f;
                wait_b(ok, pv_done + 8 * (group ^ 1), ((c - 1) >> 1) & 1);  // P V(c - 1) is done
                tc_fence_after();
#pragma unroll 1
                for (int col = 0; col < HD; col += 32) {
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
            const float z = now == -INFINITY ? 0.f : now;
            if (now != m) {
                l *= shared_ex2(m - z);  // 0 * 0 where nothing was seen yet
                m = now;
            }
            uint32_t w[32];
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                w[i] = pack_rn(shared_ex2(fmaf(x[2 * i], s2, -z)), shared_ex2(fmaf(x[2 * i + 1], s2, -z)));
                sum[(2 * i) & 3] += __uint_as_float(w[i] << 16);
                sum[(2 * i + 1) & 3] += __uint_as_float(w[i] & 0xffff0000u);
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            if (PB == 1 && c > 0) wait_b(ok, pv_done + 8 * (group ^ 1), ((c - 1) >> 1) & 1);  // the only buffer
            unsigned char* prow = sm + S::kOffP + pb * S::kPBytes + r * 128;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                *reinterpret_cast<uint4*>(prow + ((i ^ (r & 7)) << 4)) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
            fence_proxy_async();  // generic-proxy writes -> the MMA's async-proxy reads
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 8 * group);
        }
        // ---- the row's sum over both groups at the last reference, then its accumulator: the
        // group that took the last block holds that reference
        const int last = nb > 0 ? (nb - 1) & 1 : 0;
        if (group != last) {
            s_sum[r] = l;
            s_ref[r] = m;  // what it handed on last, if anything
            hand_on(9 + quad);
        } else {
            take_over(9 + quad);
            const float om = s_ref[r], z = m == -INFINITY ? 0.f : m;
            l += s_sum[r] * shared_ex2(om - z);
        }
        if (nb > 0) {
            wait_b(ok, o_full, 0);
            tc_fence_after();
        }
        if (*s_bad || (broken && parts.direct)) {
            m = 0.f;
            l = __int_as_float(0x7fffffff);
        }
        if (!parts.direct) {
            if (group == last && r < rows) parts.ml[static_cast<size_t>(s_row[r]) * parts.n + split] = make_float2(m, l);
            if (nb > 0) {
                float* dst = parts.o + (static_cast<size_t>(s_row[r]) * parts.n + split) * HD;
#pragma unroll 1
                for (int col = group * (HD / 2); col < (group + 1) * (HD / 2); col += 32) {
                    uint32_t o[32];
                    tmem_ld_32x32b_x32(tmem_o + lane_off + col, o);
                    tmem_ld_wait();
                    if (r < rows) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) st_v8(dst + col + 8 * i, o + 8 * i);
                    }
                }
            }
        } else {
            // the only part of its rows: the output itself
            if (group == last) s_sum[r] = l;
            asm volatile("bar.sync 13, 256;" ::: "memory");  // the softmax warps
            l = s_sum[r];
            const float inv = l > 0.f ? 1.0f / l : l;  // no key seen: 0 (nothing was accumulated); NaN stays
            uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + static_cast<size_t>(s_row[r]) * HD);
#pragma unroll 1
            for (int col = group * (HD / 2); col < (group + 1) * (HD / 2); col += 32) {
                uint32_t o[32];
                if (nb > 0) {
                    tmem_ld_32x32b_x32(tmem_o + lane_off + col, o);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0u;
                }
                if (r < rows && pos >= 0) {
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) w[i] = pack_rn(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
                    st_v8(reinterpret_cast<float*>(dst + col / 2), w);
                    st_v8(reinterpret_cast<float*>(dst + col / 2 + 8), w + 8);
                }
            }
        }
    }
    if (!ok) {
        // a wait gave up: give copies and MMAs that may still be in flight the same time again
        const uint64_t t0 = now_ns();
        while (now_ns() - t0 < 500000000ull) __nanosleep(1000);
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
