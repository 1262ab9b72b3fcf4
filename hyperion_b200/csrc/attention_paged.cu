// Attention of a batch of rows over a prefix that all requests share and over each
// request's own pages of a paged KV cache.
//
// Row t (of request b, at absolute position pos) sees the prefix keys at positions
// [0, prefix_len) and the request's own keys j < own_len at positions prefix_len + j, both
// only up to pos and, with a window, after pos - window. With s = scale * q.k (soft-capped
// when asked) the output is sum_j exp(s_j) v_j / sum_j exp(s_j). A softmax over a set of
// keys is joined exactly from its parts: a part keeps a reference m, l = sum exp(s - m) and
// o = sum exp(s - m) v, and the whole is sum_i exp(m_i - M) o_i / sum_i exp(m_i - M) l_i with
// M = max m_i, whatever the references. m is a maximum that the part met and moves only when the
// scores outgrow it by a factor of 2^40 (kSharedLazy).
// So the prefix is one part for the batch (its keys are read once, with the rows of all
// requests as one matrix), each request's pages are others, long parts are split over the
// SMs, and shared_merge_kernel joins them.
//
// Statistics and accumulators are fp32. The probabilities are rounded to bf16 for the
// tensor cores, as unnormalised exp(s - m), and l sums the rounded ones, so that the rounding
// cancels where all weights round alike. They reach 2^40 and not only 1; bf16 has fp32's
// exponents, so that costs no precision, and sums over 2^31 keys stay finite for |v| below 2^56.
// l is at least 1 for a row that sees a key, and the factors exp(m_i - M) are at most 1.
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

constexpr int kMinSlices = 4;     // of a warp's share: a shorter one is all latency
constexpr int kCtas = 2 * 148;    // two on every SM of a B200

// The sizes of a call that the plan goes by.
struct Sizes {
    int T, n_req, max_q, max_own, prefix_len, n_heads, n_kv, hd;
    long long all_rows, req_rows;  // (token, head) pairs of a KV head: of all rows, of a request's
    int tiles_o, tc_tiles, tc_tiles_o;
    Sizes(int T_, int n_req_, int max_q_, int max_own_, int prefix_len_, int n_heads_, int n_kv_, int hd_)
        : T(T_), n_req(n_req_), max_q(std::min(max_q_, T_)), max_own(max_own_), prefix_len(prefix_len_), n_heads(n_heads_),
          n_kv(n_kv_), hd(hd_) {
        const int G = n_heads / n_kv;
        auto tiles = [](long long rows, int tile) { return static_cast<int>((rows + tile - 1) / tile); };
        all_rows = static_cast<long long>(T) * G;
        req_rows = static_cast<long long>(max_q) * G;
        tiles_o = tiles(req_rows, kTileRows);
        tc_tiles = tiles(all_rows, kTcRows);
        tc_tiles_o = tiles(req_rows, kTcRows);
    }
    // keys of the prefix, and 64-key blocks of prefix and own keys, that one row sees at most
    long long seen(int window) const { return window > 0 ? std::min(prefix_len, window) : prefix_len; }
    long long blocks(int window) const {
        const long long all = static_cast<long long>(prefix_len) + max_own;
        return ((window > 0 ? std::min<long long>(all, static_cast<long long>(window) + max_q) : all) + 63) / 64;
    }
};

// The ways to go through a call's keys.
enum class Way {
    kApart,       // the prefix by tiles of all rows, the requests' own keys by the 16-row kernel
    kPerRequest,  // 128-row tiles of one request's rows over prefix and own keys
    kTogether,    // the 16-row kernel over both
};

// The only sensible one, where there is one.
bool only_way(const Sizes& z, Way* way) {
    // up to 16 rows in all: one 16-row tile of them against the prefix, unless there is nobody to share with
    if (z.all_rows <= kTileRows) *way = z.prefix_len > 128 && z.n_req > 1 ? Way::kApart : Way::kTogether;
    // tiles of one request's rows that are filled about as well as those of all rows
    else if (z.req_rows > kTileRows && 4ll * z.n_req * z.tc_tiles_o <= 5ll * z.tc_tiles) *way = Way::kPerRequest;
    else if (z.prefix_len == 0) *way = Way::kTogether;
    else return false;
    return true;
}

// Otherwise by what they take, in microseconds. The constants are measured without a soft-cap, for
// requests of equal rows and about one tile an SM. They count one start for all the tiles that an SM
// takes in turn, no soft-cap and every request as long as max_q: many requests with short keys, the
// more so with a soft-cap, and ragged batches can go a slower way than they had to.
Way way_of(const Sizes& z, int window) {
    Way way;
    if (only_way(z, &way)) return way;
    // 128-row kernel: 8 to start and end and a block on an SM 0.8, with head_dim 256 1.2; 16-row kernel: 5, and
    // slices of head_dim 256 at 400 in a microsecond from HBM, 650 when read again (L2); joining: 6; the two
    // kernels one after the other: 8. Half of max_own stands for the requests' mean.
    const double wide = z.hd / 256., block = 0.4 + 0.8 * wide;
    const double units_o = static_cast<double>(z.n_req) * z.tiles_o * z.n_kv, own = units_o * z.max_own / 2 / kSlice * wide / 400;
    const long long units_tc = static_cast<long long>(z.n_req) * z.tc_tiles_o * z.n_kv, seen = z.seen(window);
    const double per_request = 8 + static_cast<double>((units_tc + 147) / 148 * z.blocks(window)) * block;
    const double together = 11 + own + units_o * static_cast<double>(seen / kSlice) * wide / 650;
    const double apart = 27 + own + std::max(1., static_cast<double>(z.tc_tiles * z.n_kv * ((seen + 63) / 64)) / 148) * block;
    if (per_request < together && per_request < apart) return Way::kPerRequest;
    return together < apart ? Way::kTogether : Way::kApart;
}

// Whether the kernel's 32-bit numbers of slices could overflow (some room left for tiles that begin
// inside a slice). Requests' rows are disjoint, so that the tiles are at most those of all rows and
// one more each.
bool too_many_slices(const Sizes& z, const SharedPlan& s) {
    if (s.shares == 0) return false;
    auto slices = [](long long keys) { return (keys + kSlice - 1) / kSlice; };
    const long long tiles = std::min(static_cast<long long>(z.n_req) * s.tiles_o, z.all_rows / kTileRows + z.n_req);
    const double all = static_cast<double>(tiles) * static_cast<double>(slices(z.max_own) + (s.o_prefix ? slices(z.prefix_len) : 0));
    return all + static_cast<double>(slices(z.prefix_len)) >= 2147483648.;
}

SharedPlan plan_of(const Sizes& z, Way way, int window) {
    SharedPlan s;
    if (way == Way::kPerRequest) {
        const long long units = static_cast<long long>(z.n_req) * z.tc_tiles_o * z.n_kv;
        s.tc_per_request = 1;
        s.tc_tiles = z.tc_tiles_o;
        s.tc_splits = static_cast<int>(std::max<long long>(1, std::min<long long>((z.blocks(window) + 1) / 2, 148 / units)));
        return s;
    }
    if (way == Way::kApart && z.all_rows > kTileRows) {
        const long long units = static_cast<long long>(z.tc_tiles) * z.n_kv;
        s.tc_tiles = z.tc_tiles;
        s.tc_splits = static_cast<int>(std::max<long long>(1, std::min<long long>((z.seen(window) + 127) / 128, 148 / units)));
    }
    s.prefix_unit = way == Way::kApart && z.all_rows <= kTileRows;
    s.o_prefix = way == Way::kTogether && z.prefix_len > 0;
    const long long prefix_slices = (z.prefix_len + kSlice - 1) / kSlice;
    const long long unit_slices = (z.max_own + kSlice - 1) / kSlice + (s.o_prefix ? prefix_slices : 0);
    if (unit_slices > 0) s.tiles_o = z.tiles_o;
    const bool by_rows = static_cast<long long>(z.n_req) * s.tiles_o > z.all_rows / kTileRows + z.n_req;
    s.unit_req = by_rows ? 1 : s.tiles_o;
    s.unit_rows = by_rows ? z.n_heads / z.n_kv : 0;
    if (way == Way::kTogether && unit_slices > 0 && unit_slices <= kWarps * kMinSlices) {
        s.one_part = 1;
        return s;
    }
    // as many shares of every KV head's slices as fill two CTAs an SM
    const long long slices = static_cast<long long>(z.n_req) * s.tiles_o * unit_slices + (s.prefix_unit ? prefix_slices : 0);
    if (slices > 0) s.shares = static_cast<int>(std::max<long long>(1, std::min<long long>(kCtas * kWarps / z.n_kv, slices / kMinSlices)));
    return s;
}

// The keys of one segment (prefix or own) for some rows: those in [lo, hi) are seen by one of
// them (for rows at neighbouring positions), the slices start at key `first`.
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
    // without a window the slices depend on the length alone, so that shares can be cut and pages
    // looked up before the rows' positions are known
    k.slices = window > 0 ? (k.hi > k.lo ? (k.hi - k.first + kSlice - 1) / kSlice : 0) : (len + kSlice - 1) / kSlice;
    return k;
}

// The rows of request `req` (-1: all), its own keys within the bounds, and whether it breaks them.
struct Request {
    int t0, n_tok, own;
    bool broken;
};
__device__ __forceinline__ Request request_of(const SharedAttnParams& p, int req) {
    Request r = {0, p.T, 0, false};
    if (req >= 0) {
        const int a = p.row_start[req], b = p.row_start[req + 1], len = p.own_lens[req];
        const long long most = min(static_cast<long long>(p.max_own), static_cast<long long>(p.max_blocks) * p.page_size);
        r.t0 = min(max(a, 0), p.T);
        r.n_tok = max(0, min(min(b, p.T) - r.t0, p.max_q));
        r.own = static_cast<int>(min(static_cast<long long>(max(0, len)), most));
        r.broken = len > most;
    }
    return r;
}

// The position of row t of that request (-1: of all rows, of which those of no request see nothing,
// whatever their positions say: they would widen the window of the others' tile).
__device__ __forceinline__ int pos_of(const SharedAttnParams& p, int req, int t) {
    const int pos = p.row_pos[t];
    return req < 0 && (t < p.row_start[0] || t >= p.row_start[p.n_req]) ? -1 : pos;
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
    static constexpr int kStart = kBars + kWarps * kStages * 8;  // per request: first slice, slices of a unit
    static constexpr int kSmem = kStart + 2 * kMaxSharedRequests * 4 + 1024;  // + alignment slack
};

// Up to 16 rows (row m of a tile = token m / G, head m % G of the KV head's group) against 16-key
// slices, on mma.sync m16n8k16 with an online softmax, each warp on its own: tensor-map copies
// into its own ring, V rows of keys that no row of the request sees cleared before the product
// (0 * NaN). Rows share every byte of K and V that is loaded, so up to 16 rows cost the same
// traffic as one: HBM bound, if the eight warps of an SM get through a slice in 1.5 us at
// head_dim 128; so copies are issued for a whole slice at once (per-lane 16-byte copies took half
// of 660 instructions a slice), and masks and rescaling sit behind warp-uniform branches.
//
// A unit is a tile of rows with the keys it has to see: the batch's rows with the prefix, or one
// request's with its own keys (o_prefix: the prefix in front). All units' slices in a row are cut
// into equal shares, whatever the requests' lengths (each CTA adds the lengths up itself); a warp
// takes a share for one KV head, writes what it has for a unit (a piece) and goes on with the next.
// Neighbouring warps take the same share for neighbouring heads, whose keys are neighbours in
// memory: with the heads one after the other in the row of slices the same kernel reached half
// the bandwidth. ONE: short units, a CTA takes a whole one, joins its four warps and writes
// the output itself. PLAIN: no soft-cap and a positive scale, so that a row's maximum is that of its
// raw products.
// 64 requests of up to 1024 own tokens, 32 query and 16 KV heads of 128 (269 MB): 54 us behind the prefix
// kernel, 4.9 TB/s. ONE, a request of 50 keys: 6.7 us, 4 of them the kernel.
template <int HD, bool ONE, bool PLAIN>
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

    // this warp's share [r0, r1) of the slices, for head my_hk
    unsigned* s_start = reinterpret_cast<unsigned*>(sm + SP::kStart);
    int* s_slices = reinterpret_cast<int*>(s_start + kMaxSharedRequests);
    unsigned r0 = 0, r1 = 0, prefix_slices = 0;
    const int my_warp = blockIdx.x * kWarps + warp, my_share = my_warp / p.n_kv, my_hk = my_warp % p.n_kv;
    if constexpr (!ONE) {
        // positions matter for the number of slices only where a window cuts the keys
        auto span = [&](int req, const Request& r, int& lo, int& hi) {
            lo = INT_MAX;
            hi = -1;
            for (int t = 0; p.window > 0 && t < r.n_tok; ++t) {
                const int pos = pos_of(p, req, r.t0 + t);
                if (pos >= 0) {
                    lo = min(lo, pos);
                    hi = max(hi, pos);
                }
            }
        };
        int lo, hi;
        if (pl.prefix_unit) {
            span(-1, request_of(p, -1), lo, hi);
            prefix_slices = keys_of(nullptr, 0, p.prefix_len, lo, hi, p.window).slices;
        }
        const int per = (p.n_req + kWarps * 32 - 1) / (kWarps * 32);
        const int b0 = min(p.n_req, static_cast<int>(threadIdx.x) * per), b1 = min(p.n_req, b0 + per);
        unsigned sum = 0;
        for (int b = b0; b < b1 && pl.tiles_o > 0; ++b) {
            const Request r = request_of(p, b);
            span(b, r, lo, hi);
            const int n = keys_of(nullptr, p.prefix_len, r.own, lo, hi, p.window).slices +
                          (pl.o_prefix ? keys_of(nullptr, 0, p.prefix_len, lo, hi, p.window).slices : 0);
            s_slices[b] = n;
            s_start[b] = sum;
            sum += static_cast<unsigned>(n) * ((r.n_tok * G + kTileRows - 1) / kTileRows);
        }
        unsigned before = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned x = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += x;
        }
        if (lane == 31) s_row[warp] = static_cast<int>(before);
        __syncthreads();
        before -= sum;
        unsigned total = prefix_slices;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += s_row[w];
            total += s_row[w];
        }
        for (int b = b0; b < b1; ++b) s_start[b] += prefix_slices + before;
        __syncthreads();
        if (pl.tiles_o == 0) {
            for (int b = b0; b < b1; ++b) s_slices[b] = 0;
            __syncthreads();
        }
        const unsigned shares = min(static_cast<unsigned>(pl.shares), max(1u, total / kMinSlices));
        if (my_share < static_cast<int>(shares)) {
            r0 = static_cast<unsigned>(static_cast<uint64_t>(my_share) * total / shares);
            r1 = static_cast<unsigned>(static_cast<uint64_t>(my_share + 1) * total / shares);
        }
        // which shares have a piece of a unit: for the merge, every unit by one CTA
        auto pieces = [&](unsigned a, int n) {
            if (total == 0 || n == 0) return make_int2(0, 0);
            auto share_of = [&](uint64_t end) { return min(static_cast<unsigned>((end * shares - 1) / total), shares - 1); };
            const unsigned w0 = share_of(static_cast<uint64_t>(a) + 1), w1 = max(w0, share_of(static_cast<uint64_t>(a) + n));
            return make_int2(static_cast<int>(w0), static_cast<int>(w1 - w0 + 1));
        };
        if (blockIdx.x == 0 && threadIdx.x == 0 && pl.prefix_unit) parts.unit[0] = pieces(0, prefix_slices);
        if (pl.unit_rows == 0) {
            for (int i = blockIdx.x * kWarps * 32 + threadIdx.x; i < p.n_req * pl.tiles_o; i += gridDim.x * kWarps * 32) {
                const int b = i / pl.tiles_o;
                parts.unit[pl.prefix_unit + i] = pieces(s_start[b] + (i - b * pl.tiles_o) * s_slices[b], s_slices[b]);
            }
        } else {
            for (int b = blockIdx.x * kWarps + warp; b < p.n_req; b += gridDim.x * kWarps) {
                const Request r = request_of(p, b);
                const int tiles = min(pl.tiles_o, static_cast<int>((static_cast<long long>(r.n_tok) * G + kTileRows - 1) / kTileRows));
                for (int i = lane; i < tiles; i += 32) parts.unit[pl.unit_of(b, r.t0, i)] = pieces(s_start[b] + i * s_slices[b], s_slices[b]);
            }
        }
    }

    int slot = 0, phase = 0;  // the ring's next stage
    bool ok = true;
#pragma unroll 1
    for (bool more = true; more;) {
    // ---- which unit, and which of its slices: i-th one s0 + i * stride
    int req, tile, hk, s0, mine;
    constexpr int stride = ONE ? kWarps : 1;
    if constexpr (ONE) {
        hk = blockIdx.x % p.n_kv;
        const int unit = blockIdx.x / p.n_kv;
        tile = unit % pl.tiles_o;
        req = unit / pl.tiles_o;
        s0 = warp;
        mine = 0;
        more = false;
    } else {
        if (r0 >= r1) break;
        int n;
        hk = my_hk;
        if (r0 < prefix_slices) {
            tile = 0;
            req = -1;
            n = prefix_slices;
            s0 = r0;
        } else {
            int lo = 0, hi = p.n_req;  // the last request that starts at or before r0 (it has slices)
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (s_start[mid] <= r0) lo = mid;
                else hi = mid;
            }
            req = lo;
            n = s_slices[req];
            const unsigned rel = r0 - s_start[req];
            tile = min(static_cast<int>(rel / n), pl.tiles_o - 1);
            s0 = static_cast<int>(rel % n);
        }
        mine = min(static_cast<int>(r1 - r0), n - s0);
        r0 += mine;
    }
    const Request rq = request_of(p, req);
    const int t0 = rq.t0, len_p = req < 0 || pl.o_prefix ? p.prefix_len : 0;
    const int* own_table = p.table + static_cast<size_t>(max(req, 0)) * p.max_blocks;
    // ---- the pages of this warp's first 32 slices, one a lane, while no window moves the slices
    int pages = 0;
    const int slices_p = (len_p + kSlice - 1) / kSlice;
    if (p.window == 0) {
        const int s = s0 + lane * stride;
        if (s < slices_p) pages = p.prefix_table[s * kSlice / p.page_size];
        else if (s - slices_p < (rq.own + kSlice - 1) / kSlice) pages = own_table[(s - slices_p) * kSlice / p.page_size];
    }
    if (ONE && tile == pl.tiles_o - 1) shared_fill_unserved(p, req, hk, t0, kWarps * 32);
    // ---- rows m0 .. m0 + rows of the (token, head) pairs from token t0 on
    const int m0 = tile * kTileRows;
    const int rows = static_cast<int>(max(0ll, min(static_cast<long long>(kTileRows), static_cast<long long>(rq.n_tok) * G - m0)));
    if (ONE && rows <= 0) return;
    // lane m (and m + 16): row m's position and place
    const int mm = m0 + min(lane & 15, rows - 1), tok = mm / G;
    const int my_pos = (lane & 15) < rows ? pos_of(p, req, t0 + tok) : -1;
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
    if (ONE && warp == 0 && lane < kTileRows) s_row[lane] = my_row | (my_pos < 0 ? 0x80000000 : 0);
    // the span of the tile's positions; of the request's where a window cuts the keys by it
    int pmin = my_pos < 0 ? INT_MAX : my_pos, pmax = my_pos;
    if (!ONE && p.window > 0)
        for (int t = lane; t < rq.n_tok; t += 32) {
            const int pos = pos_of(p, req, t0 + t);
            if (pos >= 0) pmin = min(pmin, pos);
            pmax = max(pmax, pos);
        }
    pmin = __reduce_min_sync(0xffffffffu, pmin);
    pmax = __reduce_max_sync(0xffffffffu, pmax);
    const int posA = __shfl_sync(0xffffffffu, my_pos, g), posB = __shfl_sync(0xffffffffu, my_pos, g + 8);
    // ---- its keys: the prefix's slices, then the request's own
    const Keys ka = keys_of(p.prefix_table, 0, len_p, pmin, pmax, p.window);
    const Keys kb = keys_of(own_table, p.prefix_len, rq.own, pmin, pmax, p.window);
    if (ONE) mine = ka.slices + kb.slices > warp ? (ka.slices + kb.slices - warp + kWarps - 1) / kWarps : 0;

    float o[HD / 8][4];
#pragma unroll
    for (int i = 0; i < HD / 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
    float mA = -INFINITY, mB = -INFINITY, lA = 0.f, lB = 0.f;
    bool bad = false;

    const int page_shift = __ffs(p.page_size) - 1, in_page = p.page_size - 1;
    auto load_pages = [&](int from) {  // of this warp's slices from .. from + 31, as first slots
        const int i = from + lane, s = s0 + i * stride;
        const bool a = s < ka.slices;
        const int key = a ? ka.first + s * kSlice : kb.first + (s - ka.slices) * kSlice;
        if ((from > 0 || p.window > 0) && i < mine) pages = (a ? ka.table : kb.table)[key >> page_shift];
        const bool there = pages >= 0 && pages < p.n_pages;
        const bool seen = i < mine && key < (a ? ka.hi : kb.hi);
        if (seen && !there) bad = true;
        // slices without a visible key, and bad pages: a box past the pool, which reads as zeros
        pages = seen && there ? (pages << page_shift) + (key & in_page) : p.n_pages << page_shift;
    };
    int f_slot = slot;
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
    const float s2 = PLAIN ? p.scale * kSharedLog2e : 1.f;
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
    for (int i = 0; i < mine; ++i) {
        fetch(2 * i + ST - 1);
        const int s = s0 + i * stride;
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
        if constexpr (!PLAIN) {
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
#pragma unroll
    for (int w = 1; w <= 2; w <<= 1) {
        lA += __shfl_xor_sync(0xffffffffu, lA, w);
        lB += __shfl_xor_sync(0xffffffffu, lB, w);
    }
    // a page outside the pool: the rows of the tile come out as NaN, not as a silent subset
    if (__any_sync(0xffffffffu, bad) || (ONE && rq.broken)) {
        lA = lB = __int_as_float(0x7fffffff);
        mA = mB = 0.f;
    }
    if constexpr (!ONE) {
        const int unit = req < 0 ? 0 : pl.unit_of(req, t0, tile);
        const size_t place = (static_cast<size_t>(my_share + unit) * p.n_kv + hk) * kTileRows;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int m = g + 8 * half;
            const float l = half ? lB : lA;
            if (m >= rows) continue;
            if ((lane & 3) == 0) parts.pml[place + m] = make_float2(half ? mB : mA, l);
            if (l == 0.f) continue;
            float* dst = parts.po + (place + m) * HD + c2;
#pragma unroll
            for (int d = 0; d < HD / 8; ++d) *reinterpret_cast<float2*>(dst + 8 * d) = make_float2(o[d][2 * half], o[d][2 * half + 1]);
        }
    } else {
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
            if (s_row[m] < 0) continue;
            const float inv = L > 0.f ? 1.0f / L : L;
            *reinterpret_cast<uint2*>(p.out + static_cast<size_t>(s_row[m]) * HD + d) =
                make_uint2(pack_bf2(f2bf(acc.x * inv), f2bf(acc.y * inv)), pack_bf2(f2bf(acc.z * inv), f2bf(acc.w * inv)));
        }
    }
    }
    if (!ok) {
        // a wait gave up: give copies that may still be in flight the same time again
        const uint64_t from = shared_now_ns();
        while (shared_now_ns() - from < 500000000ull) __nanosleep(1000);
    }
    // this grid may start under the 128-row kernel's last CTAs; it ends after them, so that the
    // merge, which waits for this grid, waits for both
    if (after_tc) pdl_wait();
}

// W warps per (row, head) join its parts, each every W-th: those of the 128-row kernel, the pieces of
// its prefix unit, the pieces of its request's unit. Rows before row_start[0] or from
// row_start[n_req] on belong to no request and are left as they were; a row whose request
// breaks the bounds the caller gave (more rows than max_q, more keys than max_own or its
// table) has parts that were not computed and becomes NaN. After the step above: 6 us, latency.
template <int HD>
__global__ void __launch_bounds__(256) shared_merge_kernel(const SharedAttnParams p, const SharedPlan pl, SharedParts parts, int W) {
    constexpr int PER = HD / 32;
    __shared__ float s_o[8][HD];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp % W;
    const long long row = (static_cast<long long>(blockIdx.x) * 8 + warp) / W;
    const int t = static_cast<int>(min(row / p.n_heads, static_cast<long long>(p.T)));
    bool live = t < p.T, broken = false;
    // the last request that starts at or before t: 32 starts a step, by the whole warp
    int req = 0, first = 0;
    {
        const int step = (p.n_req + 31) / 32, end = p.row_start[p.n_req], pos = live ? p.row_pos[t] : -1;
        int v = lane * step < p.n_req ? p.row_start[lane * step] : INT_MAX;
        const int begin = __shfl_sync(0xffffffffu, v, 0);
        req = max(0, __popc(__ballot_sync(0xffffffffu, v <= t)) - 1) * step;
        first = __shfl_sync(0xffffffffu, v, req / step);
        if (step > 1) {
            v = lane < step && req + lane < p.n_req ? p.row_start[req + lane] : INT_MAX;
            const int more = max(0, __popc(__ballot_sync(0xffffffffu, v <= t)) - 1);
            req += more;
            first = __shfl_sync(0xffffffffu, v, more);
        }
        live = live && t >= begin && t < end && pos >= 0;
        first = max(first, 0);
        if (live) {
            const int own = p.own_lens[req];
            broken = t - first >= p.max_q || own > p.max_own || own > static_cast<long long>(p.max_blocks) * p.page_size;
        }
    }
    pdl_wait();
    float L = 0.f, acc[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] = 0.f;
    if (live && !broken) {
        const int G = p.n_heads / p.n_kv, h = static_cast<int>(row % p.n_heads), hk = h / G, g = h - hk * G;
        // its pieces: n0 of the prefix's unit from place a0 on, at row m0; n1 of its request's, at row m1
        long long a0 = 0, a1 = 0;
        int n0 = 0, n1 = 0, m0 = 0, m1 = 0;
        if (pl.prefix_unit) {
            const int2 u = parts.unit[0];  // one tile
            a0 = u.x;
            n0 = u.y;
            m0 = t * G + g;
        }
        if (pl.tiles_o > 0) {
            const int m = (t - first) * G + g, unit = pl.unit_of(req, first, m / kTileRows);
            const int2 u = parts.unit[unit];
            a1 = u.x + unit;
            n1 = u.y;
            m1 = m % kTileRows;
        }
        const int n = parts.n + n0 + n1;
        auto place = [&](int s) {  // of part s - parts.n, in rows
            s -= parts.n;
            return (((s < n0 ? a0 + s : a1 + s - n0) * p.n_kv + hk) * kTileRows) + (s < n0 ? m0 : m1);
        };
        auto stat = [&](int s) { return s < parts.n ? parts.ml[row * parts.n + s] : parts.pml[place(s)]; };
        const float2 v0 = lane < n ? stat(lane) : make_float2(-INFINITY, 0.f);  // mostly all there is
        float M = v0.x;
        for (int s = 32 + lane; s < n; s += 32) M = fmaxf(M, stat(s).x);
        M = warp_max(M);
        const float z = M == -INFINITY ? 0.f : M;
        for (int s0 = 0; s0 < n; s0 += 32) {
            const float2 v = s0 == 0 ? v0 : (s0 + lane < n ? stat(s0 + lane) : make_float2(-INFINITY, 0.f));
            const float f = v.y == 0.f ? 0.f : shared_ex2(v.x - z);  // l = 0: no key of the part is seen, no output written
            L += warp_sum(f * v.y);
            const int e = min(32, n - s0);
            constexpr int U = 4;  // parts whose loads are in flight together
            for (int s1 = sub; s1 < e; s1 += U * W) {
                float x[U][PER], fs[U];
#pragma unroll
                for (int q = 0; q < U; ++q) {
                    const int s = s1 + q * W;
                    fs[q] = __shfl_sync(0xffffffffu, f, s & 31);
                    if (s >= e) fs[q] = 0.f;
#pragma unroll
                    for (int i = 0; i < PER; ++i) x[q][i] = 0.f;
                    if (fs[q] == 0.f) continue;
                    const float* at = (s0 + s < parts.n ? parts.o + (row * parts.n + s0 + s) * HD : parts.po + place(s0 + s) * HD) + lane * PER;
                    if constexpr (PER == 2) {
                        *reinterpret_cast<float2*>(x[q]) = *reinterpret_cast<const float2*>(at);
                    } else {
#pragma unroll
                        for (int i = 0; i < PER; i += 4) *reinterpret_cast<float4*>(x[q] + i) = *reinterpret_cast<const float4*>(at + i);
                    }
                }
#pragma unroll
                for (int q = 0; q < U; ++q)
#pragma unroll
                    for (int i = 0; i < PER; ++i) acc[i] += fs[q] * x[q][i];
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
    uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + row * HD + lane * PER);
#pragma unroll
    for (int i = 0; i < PER / 2; ++i) dst[i] = pack_bf2(f2bf(acc[2 * i] * inv), f2bf(acc[2 * i + 1] * inv));
}

// Where the parts lie in the scratch.
struct Layout {
    long long rows, units, places;
    size_t o, ml, po, pml, unit, bytes;
    Layout(const SharedPlan& s, int T, int n_req, int n_heads, int n_kv, int hd) {
        rows = s.direct() ? 0 : static_cast<long long>(T) * n_heads * s.tc_splits;
        units = s.direct() ? 0 : s.prefix_unit + (s.unit_rows > 0 ? static_cast<long long>(T) * (n_heads / n_kv) / kTileRows + n_req
                                                                  : static_cast<long long>(n_req) * s.tiles_o);
        places = s.shares > 0 && !s.direct() ? (units + s.shares) * n_kv : 0;
        o = 0;
        ml = o + rows * hd * sizeof(float);
        po = (ml + rows * sizeof(float2) + 255) & ~static_cast<size_t>(255);
        pml = po + places * kTileRows * hd * sizeof(float);
        unit = pml + places * kTileRows * sizeof(float2);
        bytes = unit + units * sizeof(int2);
    }
};

template <int HD>
void launch_shared_t(const SharedAttnParams& p, const SharedPlan& pl, const SharedParts& parts, cudaStream_t stream) {
    using SP = SmallPlan<HD>;
    const long long warps = static_cast<long long>(p.T) * p.n_heads;
    if (pl.tc_splits > 0) launch_shared_attn_tc(p, pl, parts, stream);
    if (pl.one_part || pl.shares > 0) {
        const long long ctas = pl.one_part ? static_cast<long long>(p.n_req) * pl.tiles_o * p.n_kv
                                           : (static_cast<long long>(pl.shares) * p.n_kv + kWarps - 1) / kWarps;
        if (ctas > INT_MAX / kTileRows) throw ArgError("sdpa_shared_prefix: too many rows");
        CUtensorMap tk, tv;
        shared_pool_maps(p, kSlice, &tk, &tv);
        const bool plain = p.softcap <= 0.f && p.scale > 0.f;
        auto kern = pl.one_part ? (plain ? shared_attn_small_kernel<HD, true, true> : shared_attn_small_kernel<HD, true, false>)
                                : (plain ? shared_attn_small_kernel<HD, false, true> : shared_attn_small_kernel<HD, false, false>);
        allow_smem(reinterpret_cast<const void*>(kern), SP::kSmem);
        shared_launch(kern, static_cast<unsigned>(ctas), kWarps * 32, SP::kSmem, stream,
                      pl.tc_splits > 0, tk, tv, p, pl, parts, pl.tc_splits > 0 ? 1 : 0);
    }
    if (parts.direct) return;  // the only part wrote the output
    // several warps a row while all of them run at once
    const int W = warps <= 592 ? 8 : (warps <= 1184 ? 4 : (warps <= 2368 ? 2 : 1));
    shared_launch(shared_merge_kernel<HD>, static_cast<unsigned>((warps * W + 7) / 8), 256, 0, stream,
                  pl.tc_splits > 0 || pl.shares > 0, p, pl, parts, W);
}

}  // namespace

size_t shared_attn_scratch_bytes(int T, int n_req, int max_q, int max_own, int prefix_len, int n_heads, int n_kv,
                                 int hd) {
    // For any window: the most that a way takes, which is without one (the most keys, so the most parts).
    const Sizes z(T, n_req, max_q, max_own, prefix_len, n_heads, n_kv, hd);
    auto bytes = [&](Way way) { return Layout(plan_of(z, way, 0), T, n_req, n_heads, n_kv, hd).bytes; };
    Way way;
    const size_t most = only_way(z, &way) ? bytes(way) : std::max({bytes(Way::kApart), bytes(Way::kPerRequest), bytes(Way::kTogether)});
    return most + 512;
}

void launch_shared_attn(const SharedAttnParams& p, cudaStream_t stream) {
    const Sizes z(p.T, p.n_req, p.max_q, p.max_own, p.prefix_len, p.n_heads, p.n_kv, p.hd);
    const SharedPlan pl = plan_of(z, way_of(z, p.window), p.window);
    if (too_many_slices(z, pl)) throw ArgError("sdpa_shared_prefix: 2^31 or more steps of 16 keys");
    const Layout at(pl, p.T, p.n_req, p.n_heads, p.n_kv, p.hd);
    if (p.scratch_bytes < at.bytes + 512) throw ArgError("sdpa_shared_prefix: scratch too small");
    unsigned char* base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(p.scratch) + 255) & ~static_cast<uintptr_t>(255));
    SharedParts parts;
    parts.o = reinterpret_cast<float*>(base + at.o);
    parts.ml = reinterpret_cast<float2*>(base + at.ml);
    parts.n = pl.tc_splits;
    parts.direct = pl.direct();
    parts.po = reinterpret_cast<float*>(base + at.po);
    parts.pml = reinterpret_cast<float2*>(base + at.pml);
    parts.unit = reinterpret_cast<int2*>(base + at.unit);
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
