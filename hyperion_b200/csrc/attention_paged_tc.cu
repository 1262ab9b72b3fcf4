// Shared-prefix attention for many rows on the 5th-generation tensor cores: the part of
// attention_paged.cu's work whose rows fill a 128-row tile.
//
// One CTA: 128 (token, head) rows of one KV head against a run of key blocks (of 128 keys; of 64
// at head_dim 256). The rows are those of the whole batch against the prefix (decode), or those
// of one request against the prefix and then its own keys (prefill). One pass over the keys with
// a running maximum:
//   S = Q K^T (tcgen05.mma, fp32 in TMEM, two buffers), p = exp2(s - m) as a bf16 operand,
//   O += P V (fp32 in TMEM).
// The reference m of a row (its first block's maximum) moves only when the running maximum
// has outgrown it by more than 2^40. p and the sums have fp32's exponent range, so larger
// values cost no precision (2^40 times 2^31 keys is far from overflow), and the 128 x head_dim
// accumulator is next to never rescaled; a threshold of 2^8 rescaled in 12% of a warp's blocks.
//
// Warps 0..3 and 4..7: two softmax groups that take the blocks in turn, one row a thread, so
//   that the exponentials of one block run under the loads, maxima and stores of the next (a
//   single group leaves its own latency, some 3000 cycles a block, in the chain). A group
//   hands the rows' references on to the other before it starts its exponentials.
// Warps 8 and 9: producers of the K and of the V blocks. They look the pages up (32 table
//   entries at a time, one a lane, a batch ahead) and issue the tensor-map copies: boxes of 64
//   head_dim columns of min(page_size, block) slots, 128-byte swizzled.
// Warp 10: allocates TMEM and issues the MMAs from one lane, S(c + 2) next to P V(c), so that
//   the softmax of a block runs under the products of its neighbours.
// In the few blocks that stick out of the visible keys the softmax group clears the V rows
// outside before it hands P over: what a pool holds there may be NaN, and 0 * NaN would reach
// the sums.
// Every mbarrier wait is bounded; TMEM is freed before the CTA exits.
//
// Measured on a B200. head_dim 256, 16 query and 8 KV heads, 8 requests of 200 to 300 rows on a
// prefix of 8192 and up to 600 own tokens: 324 us, 846 TFLOP/s (332 to 347 us once the clock gives way
// under load), half of what a large dense product reaches. A 64-key block takes some 2100 cycles, its products alone 1270 of them (a
// product of 128 x 64 x 16 takes 47, of 128 x 128 x 16 64, of 128 x 256 x 16 128); the rest is the chain
// softmax(c) -> P V(c) -> S(c + 2) of the two blocks in flight, and the waits and commits of the issuing
// warp between its products (a wait on a complete barrier 109 cycles, a commit 40). Copies of the
// kernel without the exponentials, and without the copies of K and V, took as long. Tried: S of
// 128 columns with the queries in shared memory (310 us, but few rows with a window 32 -> 35 us),
// that with S and P V issued by a warp each or with the scores held in registers (the same), and
// with loops of 32 keys (327 us).
// head_dim 128, 32 query and 16 KV heads, 64 rows on a 16384-token prefix: 35 us for 134 MB of
// keys and values and 17.2 GFLOP (3.8 TB/s, 490 TFLOP/s).
#include "attention_paged.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

#include <climits>

namespace hyb {

__device__ int g_shared_attn_wait_timeouts = 0;

namespace {

constexpr int kRows = kTcRows;  // 128
constexpr int kSoftWarps = 8;
constexpr int kGroupWarps = 4;
constexpr int kTmaWarp = kSoftWarps, kMmaWarp = kSoftWarps + 2;  // two producers: K, V
constexpr int kThreads = kSoftWarps * 32 + 96;

// Shared memory: the ring of K and V blocks and two P blocks. The queries are in TMEM: as a
// shared-memory operand they would be read again for every block and take the ring's room (64 KB
// at head_dim 256).
template <int HD>
struct TcShared {
    // keys of a block: 128 where TMEM holds two such S beside O (a block's waits, commits and hand-overs
    // cost the same whatever its length: 1780 cycles for 64 keys of head_dim 128)
    static constexpr int kKeys = HD == 256 ? 64 : 128;
    static constexpr uint32_t kTmemCols = 512;  // S 2 x kKeys, O HD, Q HD / 2
    static constexpr int kSub = HD / 64;
    // P: at head_dim 256 in TMEM, over the S it comes from; S(c + 2) then has to follow P V(c). 348 -> 324 us
    // in the case above: less shared-memory traffic, and 32 KB more for the ring. Otherwise in shared
    // memory, and S(c + 2) goes first
    static constexpr bool kPTmem = HD == 256;
    static constexpr int kSlots = HD == 256 ? 7 : (HD == 128 ? 5 : 8);
    static constexpr int kTileBytes = kKeys * HD * 2;
    static constexpr int kPBytes = kPTmem ? 0 : kRows * kKeys * 2;  // kKeys / 64 sub-tiles of [128 rows][128 bytes]
    static constexpr int kOffP = kSlots * kTileBytes;
    static constexpr int kOffSum = kOffP - kRows * 4;        // float [kRows], once the ring is no longer read
    static constexpr int kOffRef = kOffP + 2 * kPBytes;      // float [kRows]: the rows' references
    static constexpr int kOffPos = kOffRef + kRows * 4;      // int [kRows]: positions
    static constexpr int kOffBars = kOffPos + kRows * 4;
    static constexpr int kSmem = kOffBars + 384 + 1024;      // + alignment slack
};

__device__ __forceinline__ void wait_b(bool& ok, uint32_t bar, uint32_t parity) {
    shared_wait(ok, bar, parity, &g_shared_attn_wait_timeouts);
}
__device__ __forceinline__ void warp_wait(bool& ok, uint32_t bar, uint32_t parity) {
    shared_warp_wait(ok, bar, parity, &g_shared_attn_wait_timeouts);
}

// Instruction descriptor: bf16 A and B, f32 D; B MN-major when b_mn.
__host__ __device__ constexpr uint32_t idesc_bf16(int M, int N, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn ? (1u << 16) : 0u) | (static_cast<uint32_t>(N >> 3) << 17) |
           (static_cast<uint32_t>(M >> 4) << 24);
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
// Descriptors are passed as their lower words (address, leading offset); the upper one says
// 1024 bytes between 8-row groups, version 1 and the 128-byte swizzle.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
// D[tmem] = A * B^T (+ D when accumulate), issued by the lane whose `leader` is set: A in TMEM
// (16 bf16 of a row in 8 columns) ...
__device__ __forceinline__ void mma_tmem_a(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, bool accumulate,
                                           uint32_t leader) {
    asm volatile(
        "{\n .reg .pred p, q;\n .reg .b64 b;\n setp.ne.u32 p, %4, 0;\n setp.ne.u32 q, %5, 0;\n mov.b64 b, {%2, %6};\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n}\n" ::"r"(d_tmem),
        "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(accumulate ? 1u : 0u), "r"(leader), "r"(kDescHi)
        : "memory");
}
// ... or in shared memory.
__device__ __forceinline__ void mma_smem_a(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, bool accumulate,
                                           uint32_t leader) {
    asm volatile(
        "{\n .reg .pred p, q;\n .reg .b64 a, b;\n setp.ne.u32 p, %4, 0;\n setp.ne.u32 q, %5, 0;\n mov.b64 a, {%1, %6};\n"
        " mov.b64 b, {%2, %6};\n @q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n}\n" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate ? 1u : 0u), "r"(leader), "r"(kDescHi)
        : "memory");
}
__device__ __forceinline__ void commit_if(uint32_t bar, uint32_t leader) {
    asm volatile(
        "{\n .reg .pred q;\n setp.ne.u32 q, %1, 0;\n"
        " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(bar),
        "r"(leader)
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Hand-over between warp w of one softmax group and warp w of the other.
__device__ __forceinline__ void hand_on(int id) { asm volatile("bar.arrive %0, 64;" ::"r"(id) : "memory"); }
__device__ __forceinline__ void take_over(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }
// The keys of one segment (prefix or own) that a tile of rows sees: [lo, hi), in blocks from `first` on.
struct Segment {
    const int* table;
    int base, lo, hi, first, blocks;
};
template <int kKeys>
__device__ __forceinline__ Segment segment(const int* table, int base, int len, int pmin, int pmax, int window) {
    Segment s;
    s.table = table;
    s.base = base;
    s.hi = static_cast<int>(min(static_cast<long long>(len), max(0ll, static_cast<long long>(pmax) + 1 - base)));
    s.lo = window > 0 && pmax >= 0
               ? static_cast<int>(min(static_cast<long long>(s.hi), max(0ll, static_cast<long long>(pmin) - window + 1 - base)))
               : 0;
    s.first = s.lo & ~(kKeys - 1);
    s.blocks = s.hi > s.lo ? (s.hi - s.first + kKeys - 1) / kKeys : 0;
    return s;
}

// PLAIN: no soft-cap and a positive scale, so that a row's maximum is that of its raw products.
template <int HD, bool PLAIN>
__global__ void __launch_bounds__(kThreads, 1)
    shared_attn_tc_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                          const SharedAttnParams p, const SharedPlan pl, SharedParts parts) {
    using S = TcShared<HD>;
    constexpr int SUB = S::kSub, SLOTS = S::kSlots, kKeys = S::kKeys, HALVES = kKeys / 64;
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
    int t0 = 0, n_tok = p.T, own = 0, begin = 0, end = INT_MAX;
    bool broken = false;
    if (!per_request) {
        // rows of no request see nothing, whatever their positions say: they would widen the window of the others
        begin = p.row_start[0];
        end = p.row_start[p.n_req];
    } else {
        const int first = p.row_start[req], next = p.row_start[req + 1], len = p.own_lens[req];
        const long long most = min(static_cast<long long>(p.max_own), static_cast<long long>(p.max_blocks) * p.page_size);
        t0 = min(max(first, 0), p.T);
        n_tok = min(min(next, p.T) - t0, p.max_q);
        own = static_cast<int>(min(static_cast<long long>(max(0, len)), most));
        broken = len > most;  // with several parts the merge says so
    }
    const long long m0 = static_cast<long long>(tile) * kRows;
    const int rows = static_cast<int>(max(0ll, min(static_cast<long long>(kRows), static_cast<long long>(n_tok) * G - m0)));
    pdl_launch_dependents();
    if (parts.direct && tile == pl.tc_tiles - 1 && split == 0) shared_fill_unserved(p, req, hk, t0, kThreads);
    if (rows <= 0) return;

    int* s_pos = reinterpret_cast<int*>(sm + S::kOffPos);
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
    static_assert(8 * (2 * SLOTS + 10) + 8 <= 384, "barriers fit");

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
    // softmax threads: row r of the tile is (token, head) pair m0 + r; its place, position and
    // share of the query row (the groups take 64 elements in turn), on their way before the barrier
    const int quad = warp & 3, group = warp >> 2, r = 32 * quad + lane;
    constexpr int kQ = HD == 256 ? 2 : 1;
    uint32_t qw[kQ][32];
    int row = 0, pos = -1;
    if (warp < kSoftWarps) {
        const int pr = static_cast<int>(m0) + min(r, rows - 1), tok = pr / G;
        row = (t0 + tok) * p.n_heads + hk * G + (pr - tok * G);
        if (r < rows) {
            pos = p.row_pos[t0 + tok];
            if (t0 + tok < begin || t0 + tok >= end) pos = -1;
        }
        const uint4* src = reinterpret_cast<const uint4*>(p.q + static_cast<size_t>(row) * HD);
#pragma unroll
        for (int j = 0; j < kQ; ++j)
            if (HD > 64 || group == 0) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint4 v = r < rows ? src[8 * (2 * j + (HD > 64 ? group : 0)) + i] : make_uint4(0, 0, 0, 0);
                    qw[j][4 * i] = v.x;
                    qw[j][4 * i + 1] = v.y;
                    qw[j][4 * i + 2] = v.z;
                    qw[j][4 * i + 3] = v.w;
                }
            }
        if (group == 0) s_pos[r] = pos;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __reduce_max_sync(0xffffffffu, *tmem_slot);
    const uint32_t tmem_s = tmem, tmem_o = tmem + 2 * kKeys, tmem_q = tmem_o + HD;

    int pmin = INT_MAX, pmax = -1;
    for (int i = lane; i < kRows; i += 32)
        if (s_pos[i] >= 0) {
            pmin = min(pmin, s_pos[i]);
            pmax = max(pmax, s_pos[i]);
        }
    pmin = __reduce_min_sync(0xffffffffu, pmin);
    pmax = __reduce_max_sync(0xffffffffu, pmax);
    const Segment sp = segment<kKeys>(p.prefix_table, 0, p.prefix_len, pmin, pmax, p.window);
    Segment so = {nullptr, p.prefix_len, 0, 0, 0, 0};
    if (per_request) so = segment<kKeys>(p.table + static_cast<size_t>(req) * p.max_blocks, p.prefix_len, own, pmin, pmax, p.window);
    const int all = sp.blocks + so.blocks;
    const int c0 = static_cast<int>(static_cast<long long>(all) * split / pl.tc_splits);
    const int nb = __reduce_max_sync(0xffffffffu, static_cast<int>(static_cast<long long>(all) * (split + 1) / pl.tc_splits) - c0);
    // the segment and first key of this part's block c
    auto block = [&](int c, int& key0) -> const Segment& {
        const int b = c0 + c;
        const bool own = b >= sp.blocks;
        const Segment& s = own ? so : sp;
        key0 = s.first + (own ? b - sp.blocks : b) * kKeys;
        return s;
    };
    bool ok = true;
    if (warp == kTmaWarp || warp == kTmaWarp + 1) {
        const bool is_v = warp != kTmaWarp;
        const CUtensorMap* map = is_v ? &tm_v : &tm_k;
        const int piece = min(p.page_size, kKeys), shift = __ffs(piece) - 1;  // slots of one box
        const int pieces = kKeys >> shift, in_page = p.page_size - 1;
        const int per_load = pieces == 1 ? 32 : 32 / pieces;  // blocks whose pages 32 lanes hold
        const int page_shift = __ffs(p.page_size) - 1;
        const uint32_t leader = lane == 0;
        // lane i: piece i % pieces of block c + i / pieces; whether some row sees a key of it
        auto piece_of = [&](int c, int& key, const int*& table) {
            c += lane / pieces;
            if (c >= nb) return false;
            const Segment& s = block(c, key);
            key += (lane % pieces) << shift;
            table = s.table;
            return key < s.hi && key + piece > s.lo;
        };
        auto look_up = [&](int c) {
            int key;
            const int* table;
            return piece_of(c, key, table) ? table[key >> page_shift] : 0;
        };
        int next = look_up(0), at = 0;  // the pages one batch ahead of their use; lane i's first slot
        for (int c = 0; c < nb; ++c) {
            if (c % per_load == 0) {
                int key;
                const int* table;
                const bool seen = piece_of(c, key, table), there = next >= 0 && next < p.n_pages;
                if (seen && !there) *s_bad = 1;
                // pieces that nobody sees (and bad pages): a box past the pool, which reads as zeros
                at = seen && there ? (next << page_shift) + (key & in_page) : p.n_pages << page_shift;
                next = look_up(c + per_load);
            }
            // the ring's items in the order of the products: K 0, K 1, V 0, K 2, V 1, .., K nb-1, V nb-2, V nb-1
            const int i = is_v ? (c + 1 < nb ? 2 * c + 2 : 2 * nb - 1) : (c == 0 ? 0 : 2 * c - 1), slot = i % SLOTS;
            if (i >= SLOTS) warp_wait(ok, slot_empty + 8 * slot, ((i / SLOTS) - 1) & 1);
            if (lane == 0) mbar_expect_tx(slot_full + 8 * slot, S::kTileBytes);
            __syncwarp();
            const uint32_t dst = sbase + slot * S::kTileBytes;
            for (int q = 0; q < pieces; ++q) {
                const int row = __shfl_sync(0xffffffffu, at, (c % per_load) * pieces + q);
#pragma unroll
                for (int d = 0; d < SUB; ++d)
                    shared_tma_load_if(dst + d * (kKeys * 128) + ((q << shift) << 7), map, 64 * d, hk, row, slot_full + 8 * slot, leader);
            }
        }
    } else if (warp == kMmaWarp) {
        // The whole warp runs the loop with warp-uniform values and lane 0 alone issues, by a
        // predicate: descriptors then stay in uniform registers. With the issue in a one-lane branch
        // an MMA took some 65 cycles to issue, twice what the tensor cores need for it.
        constexpr uint32_t id_s = idesc_bf16(kRows, kKeys, false);
        constexpr uint32_t id_o = idesc_bf16(kRows, HD, true);
        const uint32_t leader = lane == 0;
        const uint32_t ring = sbase >> 4, p_lo = ((sbase + S::kOffP) >> 4) | (1u << 16);
        auto issue_s = [&](int sb, int slot) {
            tc_fence_after();
            const uint32_t lo = (ring + slot * (S::kTileBytes >> 4)) | (1u << 16);
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk)
                mma_tmem_a(tmem_s + kKeys * sb, tmem_q + 8 * kk, lo + (kk >> 2) * (kKeys * 128 >> 4) + 2 * (kk & 3), id_s, kk > 0, leader);
            commit_if(s_full + 8 * sb, leader);
            commit_if(slot_empty + 8 * slot, leader);
        };
        if (nb > 0) {
            warp_wait(ok, q_full, 0);
            warp_wait(ok, slot_full, 0);
            issue_s(0, 0);
            int ks = 1, kph = 0, vs = nb > 1 ? 2 : 1, vph = 0;  // ring places of the next K and V, their phases
            if (nb > 1) {
                warp_wait(ok, slot_full + 8 * ks, kph);
                issue_s(1, ks);
            }
            // S(c + 2) goes before P V(c): its buffer is free as soon as the softmax of block c has
            // read it, and the group finds it ready when it is through with block c
            auto next_s = [&]() {
                ks += 2;
                if (ks >= SLOTS) {
                    ks -= SLOTS;
                    kph ^= 1;
                }
            };
            for (int c = 0; c < nb; ++c) {
                const int sb = c & 1;
                const bool v_here = shared_try_wait(slot_full + 8 * vs, vph);  // asked for ahead of its use
                bool k_here = true;
                if (c + 2 < nb) {
                    next_s();
                    k_here = shared_try_wait(slot_full + 8 * ks, kph);
                    if constexpr (!S::kPTmem) {
                        warp_wait(ok, s_empty + 8 * sb, (c >> 1) & 1);
                        if (!__all_sync(0xffffffffu, k_here)) warp_wait(ok, slot_full + 8 * ks, kph);
                        issue_s(sb, ks);
                    }
                }
                if (!__all_sync(0xffffffffu, v_here)) warp_wait(ok, slot_full + 8 * vs, vph);
                warp_wait(ok, p_full + 8 * sb, (c >> 1) & 1);
                tc_fence_after();
                const uint32_t vlo = (ring + vs * (S::kTileBytes >> 4)) | (((kKeys * 128 >> 4) & 0x3FFFu) << 16);
#pragma unroll
                for (int kk = 0; kk < kKeys / 16; ++kk) {
                    if constexpr (S::kPTmem)
                        mma_tmem_a(tmem_o, tmem_s + kKeys * sb + 8 * kk, vlo + kk * (2048 >> 4), id_o, c > 0 || kk > 0, leader);
                    else
                        mma_smem_a(tmem_o, p_lo + sb * (S::kPBytes >> 4) + (kk >> 2) * (kRows * 128 >> 4) + 2 * (kk & 3),
                                   vlo + kk * (2048 >> 4), id_o, c > 0 || kk > 0, leader);
                }
                commit_if(pv_done + 8 * sb, leader);
                commit_if(slot_empty + 8 * vs, leader);
                if constexpr (S::kPTmem) {
                    // MMAs run in order: S(c + 2) overwrites P(c) once P V(c) has read it
                    if (c + 2 < nb) {
                        if (!__all_sync(0xffffffffu, k_here)) warp_wait(ok, slot_full + 8 * ks, kph);
                        issue_s(sb, ks);
                    }
                }
                vs += c + 2 < nb ? 2 : 1;
                if (vs >= SLOTS) {
                    vs -= SLOTS;
                    vph ^= 1;
                }
            }
            commit_if(o_full, leader);
        }
    } else {
        const uint32_t lane_off = static_cast<uint32_t>(32 * quad) << 16;
        // queries into TMEM: lane r, two bf16 a column
        if (HD > 64 || group == 0) {
#pragma unroll
            for (int j = 0; j < kQ; ++j) tmem_st_32x32b_x32(tmem_q + lane_off + 32 * (2 * j + (HD > 64 ? group : 0)), qw[j]);
            tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
        const int mine = 1 + 2 * quad + group, other = 1 + 2 * quad + (group ^ 1);  // hand-over barriers
        const float s2 = PLAIN ? p.scale * kSharedLog2e : 1.f;
        float m = -INFINITY;  // the reference that l is held at
        float l = 0.f;
        for (int c = group; c < nb; c += 2) {
            int key0;
            const Segment& s = block(c, key0);
            wait_b(ok, s_full + 8 * group, (c >> 1) & 1);
            tc_fence_after();
            // blocks wholly inside every row's view skip the per-key mask
            const bool full = key0 >= s.lo && key0 + kKeys <= s.hi && s.base + key0 + kKeys - 1 <= pmin &&
                              (p.window == 0 || s.base + key0 > pmax - p.window);
            const long long wlo = p.window > 0 ? static_cast<long long>(pos) - p.window + 1 - s.base : 0;
            const int from = static_cast<int>(min(max(wlo, static_cast<long long>(s.lo)), static_cast<long long>(s.hi))) - key0;
            const int to = min(s.hi - 1, pos - s.base) + 1 - key0;
            float x[64];
            auto load = [&](int h) {  // the scores of the block's keys 64 h .. 64 h + 63
                uint32_t v[2][32];
                tmem_ld_32x32b_x32(tmem_s + lane_off + kKeys * group + 64 * h, v[0]);
                tmem_ld_32x32b_x32(tmem_s + lane_off + kKeys * group + 64 * h + 32, v[1]);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 64; ++i) x[i] = __uint_as_float(v[i >> 5][i & 31]);
                if constexpr (!PLAIN) {
#pragma unroll
                    for (int i = 0; i < 64; ++i)
                        x[i] = kSharedLog2e * (p.softcap > 0.f ? p.softcap * tanhf(x[i] * p.scale / p.softcap) : x[i] * p.scale);
                }
                if (!full) {
#pragma unroll
                    for (int i = 0; i < 64; ++i)
                        if (64 * h + i < from || 64 * h + i >= to) x[i] = -INFINITY;
                }
            };
            auto read = [&]() {  // S is free for block c + 2
                if constexpr (!S::kPTmem) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(s_empty + 8 * group);
                }
            };
            float mx = -INFINITY;
#pragma unroll 1
            for (int h = 0; h < HALVES; ++h) {
                load(h);
                if (HALVES == 1) read();
                float mx4[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
                for (int i = 4; i < 64; ++i) mx4[i & 3] = fmaxf(mx4[i & 3], x[i]);
                mx = fmaxf(mx, fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * s2);
            }
            // the reference after block c - 1, moved if this block outgrows it, for block c + 1
            float ref = -INFINITY;
            if (c > 0) {
                take_over(other);
                ref = s_ref[r];
            }
            const bool move = mx > ref + kSharedLazy || (ref == -INFINITY && mx > -INFINITY);
            const float now = move ? mx : ref;
            if (c + 1 < nb) {
                s_ref[r] = now;
                hand_on(mine);
            }
            if (c > 0 && __any_sync(0xffffffffu, move)) {
                const float f = move ? shared_ex2(ref - now) : 1.f;
                // P V(c - 1) is done. Its barrier's phase is told by parity: with P V(c - 2) done it is
                // at most one phase behind, and P V(c + 1), the next use, cannot be through before
                // P V(c), which needs this group's P(c).
                if (c >= 2) wait_b(ok, pv_done + 8 * group, ((c - 2) >> 1) & 1);
                wait_b(ok, pv_done + 8 * (group ^ 1), ((c - 1) >> 1) & 1);
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
            // one half is still in registers; of two, both are read again (keeping one spills)
#pragma unroll 1
            for (int h = 0; h < HALVES; ++h) {
                if (HALVES > 1) {
                    load(h);
                    if (h + 1 == HALVES) read();
                }
                uint32_t w[32];
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    w[i] = shared_pack(shared_ex2(fmaf(x[2 * i], s2, -z)), shared_ex2(fmaf(x[2 * i + 1], s2, -z)));
                    sum[(2 * i) & 3] += __uint_as_float(w[i] << 16);
                    sum[(2 * i + 1) & 3] += __uint_as_float(w[i] & 0xffff0000u);
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                if constexpr (S::kPTmem) {
                    tmem_st_32x32b_x32(tmem_s + lane_off + kKeys * group, w);
                    tmem_st_wait();
                    tc_fence_before();
                } else {
                    if (h == 0 && c >= 2) wait_b(ok, pv_done + 8 * group, ((c - 2) >> 1) & 1);  // the buffer's last reader
                    unsigned char* prow = sm + S::kOffP + group * S::kPBytes + h * (kRows * 128) + r * 128;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        *reinterpret_cast<uint4*>(prow + ((i ^ (r & 7)) << 4)) =
                            make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                }
            }
            if (key0 < s.lo || key0 + kKeys > s.hi) {
                // V rows that no row of the tile sees; the block's V has its place in the ring to
                // itself until P V(c), and what held the place before was used up by a product
                // issued ahead of S(c)
                const int i = c + 1 < nb ? 2 * c + 2 : 2 * nb - 1, slot = i % SLOTS;
                wait_b(ok, slot_full + 8 * slot, (i / SLOTS) & 1);
                unsigned char* vt = sm + slot * S::kTileBytes;
                const int head = min(kKeys, max(0, s.lo - key0)), tail = min(kKeys, s.hi - key0);  // rows before, from
                for (int j = r; j < (head + kKeys - tail) * SUB * 8; j += kRows) {
                    const int n = j / (SUB * 8), key = n < head ? n : tail + n - head, ch = j % (SUB * 8);
                    *reinterpret_cast<uint4*>(vt + (ch >> 3) * (kKeys * 128) + key * 128 + (ch & 7) * 16) = make_uint4(0, 0, 0, 0);
                }
            }
            if (!S::kPTmem || key0 < s.lo || key0 + kKeys > s.hi)
                fence_proxy_async();  // generic-proxy writes -> the MMA's async-proxy reads
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 8 * group);
        }
        // ---- the row's sum over both groups at the last reference, then its accumulator: the
        // group that took the last block holds that reference
        if (nb > 0) {
            wait_b(ok, o_full, 0);
            tc_fence_after();
        }
        const int last = nb > 0 ? (nb - 1) & 1 : 0;
        if (group != last) {
            s_sum[r] = l;  // at the end of the ring: every product is done
            s_ref[r] = m;  // what it handed on last, if anything
            hand_on(9 + quad);
        } else {
            take_over(9 + quad);
            const float om = s_ref[r], z = m == -INFINITY ? 0.f : m;
            l += s_sum[r] * shared_ex2(om - z);
        }
        if (*s_bad || (broken && parts.direct)) {
            m = 0.f;
            l = __int_as_float(0x7fffffff);
        }
        if (!parts.direct) {
            if (group == last && r < rows) parts.ml[static_cast<size_t>(row) * parts.n + split] = make_float2(m, l);
            if (nb > 0) {
                // Through the ring, whose copies and products are done, so that a warp writes whole
                // rows: stored from the registers, a row a lane, they took three times as long.
                constexpr int kPitch = HD * 4 + 16;  // lanes' rows start in different banks
                static_assert(kRows * kPitch <= S::kOffSum, "the output fits where the ring was");
#pragma unroll 1
                for (int col = group * (HD / 2); col < (group + 1) * (HD / 2); col += 32) {
                    uint32_t o[32];
                    tmem_ld_32x32b_x32(tmem_o + lane_off + col, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        *reinterpret_cast<uint4*>(sm + r * kPitch + col * 4 + 16 * i) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                }
                if (group == 0) s_pos[r] = row;  // positions are no longer read
                asm volatile("bar.sync 13, 256;" ::: "memory");  // the softmax warps
                constexpr int kLanes = HD / 4 < 32 ? HD / 4 : 32, kAt = 32 / kLanes;  // lanes of a row, rows at once
                for (int q = warp * kAt + lane / kLanes; q < rows; q += kSoftWarps * kAt) {
                    float* dst = parts.o + (static_cast<size_t>(s_pos[q]) * parts.n + split) * HD;
#pragma unroll
                    for (int i = 0; i < HD / 4 / kLanes; ++i) {
                        const int at = (lane % kLanes + i * kLanes) * 4;
                        *reinterpret_cast<uint4*>(dst + at) = *reinterpret_cast<const uint4*>(sm + q * kPitch + at * 4);
                    }
                }
            }
        } else {
            // the only part of its rows: the output itself
            if (group == last) s_sum[r] = l;
            asm volatile("bar.sync 13, 256;" ::: "memory");  // the softmax warps
            l = s_sum[r];
            const float inv = l > 0.f ? 1.0f / l : l;  // no key seen: 0 (nothing was accumulated); NaN stays
            uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + static_cast<size_t>(row) * HD);
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
                    for (int i = 0; i < 16; ++i) w[i] = shared_pack(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
#pragma unroll
                    for (int i = 0; i < 4; ++i)  // 16 bytes at a time: rows start at no wider boundary
                        *reinterpret_cast<uint4*>(dst + col / 2 + 4 * i) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                }
            }
        }
    }
    if (!ok) {
        // a wait gave up: give copies and MMAs that may still be in flight the same time again
        const uint64_t t0 = shared_now_ns();
        while (shared_now_ns() - t0 < 500000000ull) __nanosleep(1000);
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
    shared_pool_maps(p, p.page_size < S::kKeys ? p.page_size : S::kKeys, &tk, &tv);
    auto kern = p.softcap <= 0.f && p.scale > 0.f ? shared_attn_tc_kernel<HD, true> : shared_attn_tc_kernel<HD, false>;
    allow_smem(reinterpret_cast<const void*>(kern), S::kSmem);
    const long long ctas = static_cast<long long>(pl.tc_tiles) * (pl.tc_per_request ? p.n_req : 1) * p.n_kv * pl.tc_splits;
    if (ctas > INT_MAX) throw ArgError("sdpa_shared_prefix: too many parts");
    kern<<<static_cast<unsigned>(ctas), kThreads, S::kSmem, stream>>>(tk, tv, p, pl, parts);
    HYB_LAUNCH_CHECK("shared_attn_tc_kernel");
}

}  // namespace

void shared_pool_maps(const SharedAttnParams& p, int box_slots, CUtensorMap* tk, CUtensorMap* tv) {
    const uint64_t hd = static_cast<uint64_t>(p.hd), dims[3] = {hd, static_cast<uint64_t>(p.n_kv), static_cast<uint64_t>(p.n_pages) * p.page_size};
    const uint64_t strides[2] = {hd * 2, static_cast<uint64_t>(p.n_kv) * hd * 2};
    const uint32_t box[3] = {64, 1, static_cast<uint32_t>(box_slots)};
    encode_tma(tk, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, p.k_pool, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    encode_tma(tv, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, p.v_pool, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

void launch_shared_attn_tc(const SharedAttnParams& p, const SharedPlan& pl, const SharedParts& parts, cudaStream_t stream) {
    switch (p.hd) {
        case 64: launch_t<64>(p, pl, parts, stream); break;
        case 128: launch_t<128>(p, pl, parts, stream); break;
        default: launch_t<256>(p, pl, parts, stream); break;
    }
}

int64_t read_shared_attn_tc_wait_timeouts() {
    int a = 0;
    HYB_CUDA(cudaMemcpyFromSymbol(&a, g_shared_attn_wait_timeouts, sizeof(int)));
    return a;
}

}  // namespace hyb
