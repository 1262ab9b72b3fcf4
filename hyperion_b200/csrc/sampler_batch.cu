// Sampling of a batch of logit rows from given uniforms, every row with its own temperature,
// top-k, top-p and min-p.
//
// Row of logits x (NaN counts as -inf), M = max x, weights w = exp((x - M) / T). The tokens
// are ordered by (logit descending, index ascending); each filter keeps a prefix of that
// order: top-k the first k, top-p the shortest whose weight reaches top_p * sum(w), min-p
// those with w >= min_p. The kept set is the shortest of the three. The token is the first
// index, in index order, at which the running sum of the kept weights exceeds u * their sum.
// T <= 0 takes the first maximum.
//
// Exactness. Sums decide which token is drawn, so they must not depend on the order of the
// additions: weights are integers in units of 2^-44 of the largest, each within some 2^-27 of its
// value (Weight below), and their 64-bit sums are exact in any order (vocabulary <= 2^19). Where a
// weight alone decides, in min-p, logits are compared instead (min_p_floor).
//
// One thread-block cluster per row; CTA c of the cluster owns a contiguous slice of the row.
//
// bf16 logits (sample_hist_kernel): a bf16 value is one of 65536, so one pass over the row
// counts every value in shared memory (16-bit counters, 128 KB, indexed by the raw bits: one
// native shared atomic an element; every 2^15 logits full counters are folded into a list) and everything but the position of the token follows
// exactly from the counts: the weight of the row, the cut of the three filters, the kept
// weight and the draw's target. A second pass over the row (from L2) then looks for the
// target in index order; it compares eight logits at a time with the cut and evaluates weights
// only for kept ones. HBM sees the row once. 64 rows of 262144 logits: 50 us, of
// which the counting pass' shared atomics take 16.5 and the second pass 16.8; one row over eight CTAs:
// 23 us, a chain of short phases (counting 5.5, gathering 1.5, group weights 1.4, cut 2.3, second pass
// 2.3, token 3) and six cluster barriers of 0.4 to 1.3 us between them.
//
// fp32 logits (sample_radix_kernel): the slice is held in shared memory, and the cut of
// top-k / top-p is found by radix selection on an order-preserving 32-bit key, 11 bits a level:
// each CTA fills a histogram of counts and weights (three 16-bit limbs, so that the shared
// atomics stay native 32-bit ones), the bins that are not empty are added up in the cluster's
// first CTA over distributed shared memory, which finds the bin in which the cut lies. With 22 bits
// known there is mostly one token left in it, and the last level is one look for it. 16 rows of
// 32003 logits: 25 us (38 with the first CTA reading all histograms, and three levels), latency: two
// levels of 5 us with two cluster barriers each, the look 1, the kept weights 2, the token 4.
#include "kernels.h"
#include "tma.cuh"

#include <algorithm>
#include <cstddef>
#include <utility>

namespace hyb {

namespace {

constexpr int kThreads = 512;
constexpr int kWarpsS = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kFrac = 44;
constexpr int kMaxCluster = 8;
constexpr int kTableCopies = 16;  // of the table of powers: the lanes of a half-warp read 16 bank pairs
constexpr int kSliceBytes = 128 * 1024;  // the largest slice held in shared memory
// A slice has at most 2^19 / 8 = 65536 logits, so its limb sums fit 32 bits: 65535 * 65536 < 2^32.

typedef unsigned long long u64;

struct Hist {
    uint32_t cnt[kBins], l0[kBins], l1[kBins], l2[kBins];
};

struct Merged {  // of all slices, in the cluster's first CTA
    u64 mass[kBins];
    uint32_t cnt[kBins];
};

struct Cut {       // where a level's cut lies
    uint32_t bin;
    uint32_t cnt;  // tokens above the bin
    uint32_t in_bin;
    u64 mass;      // their weight
    u64 total;     // weight of the whole row (level 0)
};

struct Share {  // read by the other CTAs of the cluster
    u64 best;       // (key of the maximum, ~index)
    Cut cut, got;   // found by the first CTA; as it sent it
    uint32_t single;  // the only key left in the bin
    u64 sum;        // kept weight above the cut key
    uint32_t cnt;   // kept tokens above it
    uint32_t ties;  // tokens equal to it
    u64 wsum[kWarpsS];
    uint32_t wties[kWarpsS];
    u64 red[kWarpsS];
    uint32_t red32[kWarpsS];
    u64 table[32 * kTableCopies];
};

__device__ __forceinline__ void cl_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ uint32_t cl_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cl_map(const void* p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ uint32_t cl_ld32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ u64 cl_ld64(uint32_t a) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
    return v;
}
// NaN -> -inf, -0 -> +0.
__device__ __forceinline__ float canon(float x) { return x != x ? -INFINITY : x + 0.0f; }
// Order-preserving key.
__device__ __forceinline__ uint32_t key_of(float f) {
    const uint32_t u = __float_as_uint(f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}

// 2^44 * exp((x - M) / T) as an integer, without a branch on x, in fp32 pairs and integers (in
// double the same steps take over twice as long: an SM has a quarter as many lanes for it).
// d = (x - M) log2(e) / T as a pair: x - M exactly as s + e, the factor as c + cl, the product's error
// by a fused multiply-add. d = n/32 + r; 2^(n/32) is a 44-bit table entry shifted, and the entry's
// (2^r - 1) share, |r| <= 1/64, is an fp32 polynomial's, added in units of 2^17. Off by at most
// some 2^-27 of the weight, at random; far below what moves a draw between two tokens (the sums
// of thousands of weights average it further).
struct Weight {
    float M, c, cl;
    uint32_t table;  // of this lane
    bool inf;        // the maximum is +inf: its tokens share all the weight
    __device__ __forceinline__ Weight(float max, float temperature, const u64* t) : M(max), inf(max == INFINITY) {
        const double f = 1.4426950408889634074 / static_cast<double>(temperature);
        c = static_cast<float>(fmin(f, 3e38));
        cl = f < 3e38 ? static_cast<float>(f - static_cast<double>(c)) : 0.f;
        table = smem_u32(t) + (threadIdx.x & (kTableCopies - 1)) * 8;
    }
    // thread t < 32 fills its entry
    static __device__ __forceinline__ void fill(u64* t) {
        const u64 v = static_cast<u64>(rint(exp2(threadIdx.x * (1.0 / 32.0)) * 17592186044416.0));
        for (int i = 0; i < kTableCopies; ++i) t[threadIdx.x * kTableCopies + i] = v;
    }
    __device__ __forceinline__ u64 operator()(float x) const {
        if (inf) return x == INFINITY ? 1ull << kFrac : 0;
        const float s = x - M, bb = s - x, e = (x - (s - bb)) - (M + bb);  // two-sum of x and -M
        float d = s * c;
        float dl = fmaf(s, c, -d);
        dl = fmaf(s, cl, dl);
        dl = fmaf(e, c, dl);
        const bool some = d > -60.f;  // below, at -inf and for NaN the weight is 0
        d = some ? d : -60.f;
        constexpr float kMagic = 12582912.f;  // 1.5 * 2^23
        const float t = fmaf(d, 32.f, kMagic);
        const int n = __float_as_int(t) - __float_as_int(kMagic);
        const float r = fmaf(t - kMagic, -1.f / 32.f, d) + (some ? dl : 0.f);
        float q = fmaf(r, 9.6181291e-3f, 5.5504109e-2f);
        q = fmaf(q, r, 0.24022651f);
        q = fmaf(q, r, 0.69314718f);
        q *= r;  // 2^r - 1
        u64 v;
        asm("ld.shared.u64 %0, [%1];" : "=l"(v) : "r"(table + (n & 31) * (kTableCopies * 8)));
        // v 2^-17 as a float by its upper bits: 2^44 <= v < 2^45
        const float vf = __uint_as_float(0x4d000000u | (static_cast<uint32_t>(v >> 21) & 0x7fffffu));
        const int add = __float_as_int(fmaf(vf, q, kMagic)) - __float_as_int(kMagic);  // |add| < 2^22
        v += static_cast<long long>(add) * 131072;
        const int k = -(n >> 5);
        return some ? (v + ((1ull << k) >> 1)) >> k : 0;
    }
};

// The least logit that min-p keeps: exp((x - M) / T) >= min_p where x >= M + T ln(min_p). Compared
// in logits and not in weights, whose roundings (2^-27, and 2^-44 of the largest) would put close
// logits on the wrong side and lose all settings below 2^-45. Formed in double, with exp taken as
// rounded to it (half a step below 1 is 2^-54), and rounded up, so that a float is at least this
// one just when it is at least the double. min_p above 1 counts as 1.
__device__ __forceinline__ float min_p_floor(float M, float temperature, float min_p) {
    if (M == INFINITY) return M;
    const double lg = log(static_cast<double>(fminf(min_p, 1.f))) - 5.5511151231257827e-17;
    const float least = __double2float_ru(static_cast<double>(M) + static_cast<double>(temperature) * lg);
    return fmaxf(least, -3.402823466e38f);  // never -inf, whose weight is 0
}

// Inclusive block scan in thread order; *total is the block's sum.
template <typename V>
__device__ __forceinline__ V block_incl(V v, V* red, V* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V n = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += n;
    }
    __syncthreads();
    if (lane == 31) red[warp] = v;
    __syncthreads();
    V before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWarpsS; ++w) {
        const V x = red[w];
        before += w < warp ? x : V(0);
        all += x;
    }
    *total = all;
    return before + v;
}

__global__ void __launch_bounds__(kThreads) sample_radix_kernel(const SampleBatchParams p, int slice, int resident) {
    extern __shared__ __align__(16) unsigned char dyn[];
    __shared__ Share sh;
    Hist& h = *reinterpret_cast<Hist*>(dyn);
    Merged& merged = *reinterpret_cast<Merged*>(dyn + sizeof(Hist));
    float* buf = reinterpret_cast<float*>(dyn + sizeof(Hist) + sizeof(Merged));
    uint32_t nc;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(nc));
    const uint32_t rank = cl_rank();
    const int row = blockIdx.x / nc, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int lo = min(p.vocab, static_cast<int>(rank) * slice), n = min(p.vocab, lo + slice) - lo;
    const float* gx = static_cast<const float*>(p.logits) + row * p.ld + lo;

    const float temp = p.temperature ? p.temperature[row] : 1.f;
    const bool greedy = !(temp > 0.f);
    int k = p.top_k ? p.top_k[row] : 0;
    float tp = p.top_p ? p.top_p[row] : 0.f, mp = p.min_p ? p.min_p[row] : 0.f;
    const bool use_k = k > 0 && k < p.vocab, use_p = tp > 0.f && tp < 1.f, use_m = mp > 0.f;
    if (tid < 32) Weight::fill(sh.table);
    if (rank == 0)
        for (int i = tid; i < kBins; i += kThreads) {
            merged.cnt[i] = 0;
            merged.mass[i] = 0;
        }

    // ---- the slice into shared memory, its maximum (first index)
    u64 best = 0;
    {
        float bx = -INFINITY;
        int bi = -1;
        constexpr int VEC = 4;
        const bool vec = (reinterpret_cast<uintptr_t>(gx) & 15) == 0;
        const int nv = vec ? n / VEC : 0;
        for (int i = tid; i < nv; i += kThreads) {
            const uint4 v = reinterpret_cast<const uint4*>(gx)[i];
            if (resident) reinterpret_cast<uint4*>(buf)[i] = v;
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float x = canon(__uint_as_float(w[j]));
                if (bi < 0 || x > bx) {
                    bx = x;
                    bi = i * VEC + j;
                }
            }
        }
        for (int i = nv * VEC + tid; i < n; i += kThreads) {
            const float x = canon(gx[i]);
            if (resident) buf[i] = x;
            if (bi < 0 || x > bx) {
                bx = x;
                bi = i;
            }
        }
        if (bi >= 0) best = (static_cast<u64>(key_of(bx)) << 32) | static_cast<uint32_t>(~(lo + bi));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) sh.red[warp] = best;
    __syncthreads();
    if (tid == 0) {
        u64 b = 0;
        for (int w = 0; w < kWarpsS; ++w) b = max(b, sh.red[w]);
        sh.best = b;
    }
    cl_sync();
    best = lane < static_cast<int>(nc) ? cl_ld64(cl_map(&sh.best, lane)) : 0;
#pragma unroll
    for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    const uint32_t arg = ~static_cast<uint32_t>(best);
    const float M = value_of(static_cast<uint32_t>(best >> 32));
    const float* x = resident ? buf : gx;
    const Weight weight(M, temp, sh.table);
    const bool empty = M == -INFINITY;
    if (greedy || empty) {
        if (rank == 0 && tid == 0) {
            p.token[row] = empty ? -1 : static_cast<int>(arg);
            if (p.kept) p.kept[row] = empty ? 0 : 1;
            if (p.prob) p.prob[row] = empty ? 0.f : 1.f;
        }
        cl_sync();  // no CTA leaves while another may read its shared memory
        return;
    }

    // ---- the cut of top-k and top-p
    uint32_t cut_key = 0, ties_kept = 0;
    const bool cut = use_k || use_p;
    if (cut) {
        uint32_t above = 0;
        u64 mass_above = 0, target = 0;
        uint32_t in_bin = 0;
#pragma unroll 1
        for (int level = 0; level < 3; ++level) {
            const int shift = level == 0 ? 21 : (level == 1 ? 10 : 0);
            const uint32_t width = level == 2 ? 10 : 11;
            auto outside = [&](uint32_t key) { return level && (key >> (shift + width)) != (cut_key >> (shift + width)); };
            if (level == 2 && in_bin == 1) {
                // one token is left, as with 22 bits known there mostly is: whoever holds it says which
                for (int i = tid; i < n; i += kThreads) {
                    const uint32_t key = key_of(canon(x[i]));
                    if (!outside(key))
                        for (uint32_t r = 0; r < nc; ++r)
                            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cl_map(&sh.single, r)), "r"(key) : "memory");
                }
                cl_sync();
                cut_key = sh.single;
                break;
            }
            for (int i = tid; i < 4 * kBins; i += kThreads) (&h.cnt[0])[i] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += kThreads) {
                const float xi = canon(x[i]);
                const uint32_t key = key_of(xi);
                if (outside(key)) continue;
                const uint32_t bin = (key >> shift) & ((1u << width) - 1);
                atomicAdd(&h.cnt[bin], 1u);
                if (use_p) {
                    const u64 w = weight(xi);
                    if (w) {
                        atomicAdd(&h.l0[bin], static_cast<uint32_t>(w) & 0xffffu);
                        if (w >> 16) atomicAdd(&h.l1[bin], static_cast<uint32_t>(w >> 16) & 0xffffu);
                        if (w >> 32) atomicAdd(&h.l2[bin], static_cast<uint32_t>(w >> 32));
                    }
                }
            }
            __syncthreads();
            // the few hundred bins that are not empty go to the first CTA
            const uint32_t to_cnt = cl_map(merged.cnt, 0), to_mass = cl_map(merged.mass, 0);
            for (int i = tid; i < kBins; i += kThreads) {
                const uint32_t cn = h.cnt[i];
                if (!cn) continue;
                asm volatile("red.shared::cluster.add.u32 [%0], %1;" ::"r"(to_cnt + 4 * i), "r"(cn) : "memory");
                const u64 m = h.l0[i] + (static_cast<u64>(h.l1[i]) << 16) + (static_cast<u64>(h.l2[i]) << 32);
                if (m) asm volatile("red.shared::cluster.add.u64 [%0], %1;" ::"r"(to_mass + 8 * i), "l"(m) : "memory");
            }
            cl_sync();
            if (rank == 0) {
                // thread t takes bins from the top: 2047 - 4t - i
                uint32_t bc[4];
                u64 bm[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    bc[i] = merged.cnt[kBins - 1 - 4 * tid - i];
                    bm[i] = merged.mass[kBins - 1 - 4 * tid - i];
                    merged.cnt[kBins - 1 - 4 * tid - i] = 0;  // for the next level
                    merged.mass[kBins - 1 - 4 * tid - i] = 0;
                }
                uint32_t ct;
                u64 mt;
                const uint32_t cmine = bc[0] + bc[1] + bc[2] + bc[3];
                const u64 mmine = bm[0] + bm[1] + bm[2] + bm[3];
                uint32_t cum = block_incl<uint32_t>(cmine, sh.red32, &ct) - cmine + above;
                u64 cmass = block_incl<u64>(mmine, sh.red, &mt) - mmine + mass_above;
                // the smallest prefix whose weight reaches top_p of all: an integer >= top_p * Z
                if (level == 0) target = max(1ull, static_cast<u64>(ceil(static_cast<double>(tp) * static_cast<double>(mt))));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool before = (use_k && cum >= static_cast<uint32_t>(k)) || (use_p && cmass >= target);
                    const bool after = (use_k && cum + bc[i] >= static_cast<uint32_t>(k)) ||
                                       (use_p && cmass + bm[i] >= target);
                    if (!before && after) sh.cut = {static_cast<uint32_t>(kBins - 1 - 4 * tid - i), cum, bc[i], cmass, target};
                    cum += bc[i];
                    cmass += bm[i];
                }
                __syncthreads();
                if (tid < static_cast<int>(nc)) {
                    const uint32_t at = cl_map(&sh.got, tid);
                    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at + static_cast<uint32_t>(offsetof(Cut, bin))), "r"(sh.cut.bin) : "memory");
                    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at + static_cast<uint32_t>(offsetof(Cut, cnt))), "r"(sh.cut.cnt) : "memory");
                    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at + static_cast<uint32_t>(offsetof(Cut, in_bin))), "r"(sh.cut.in_bin) : "memory");
                    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at + static_cast<uint32_t>(offsetof(Cut, mass))), "l"(sh.cut.mass) : "memory");
                    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at + static_cast<uint32_t>(offsetof(Cut, total))), "l"(sh.cut.total) : "memory");
                }
            }
            cl_sync();
            cut_key |= sh.got.bin << shift;
            above = sh.got.cnt;
            in_bin = sh.got.in_bin;
            mass_above = sh.got.mass;
            target = sh.got.total;
            // the first CTA's next write of it lies behind the next level's first cluster barrier
        }
        // all tokens of the last bin are equal: as many of them as the cut needs
        uint32_t take = in_bin;
        if (use_k) take = min(take, static_cast<uint32_t>(k) - above);
        if (use_p) {
            const u64 w = weight(value_of(cut_key));
            if (w) take = static_cast<uint32_t>(min(static_cast<u64>(take), (target - mass_above + w - 1) / w));
        }
        ties_kept = take;
    }

    // ---- kept weights: warp w of the CTA owns a contiguous run of its slice
    const float least = use_m ? min_p_floor(M, temp, mp) : -INFINITY;
    const int run = ((slice + kWarpsS - 1) / kWarpsS + 31) & ~31;
    {
        const int from = warp * run, to = min(n, from + run);
        u64 sum = 0;
        uint32_t cnt = 0, ties = 0;
        for (int i = from + lane; i < to; i += 32) {
            const float xi = canon(x[i]);
            const uint32_t key = key_of(xi);
            if (cut && key <= cut_key) {
                ties += key == cut_key;
                continue;
            }
            if (xi >= least) {
                sum += weight(xi);
                ++cnt;
            }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
            cnt += __shfl_xor_sync(0xffffffffu, cnt, o);
            ties += __shfl_xor_sync(0xffffffffu, ties, o);
        }
        if (lane == 0) {
            sh.wsum[warp] = sum;
            sh.wties[warp] = ties;
            sh.red32[warp] = cnt;
        }
        __syncthreads();
        if (tid == 0) {
            u64 s = 0;
            uint32_t t = 0, q = 0;
            for (int w = 0; w < kWarpsS; ++w) {
                s += sh.wsum[w];
                t += sh.wties[w];
                q += sh.red32[w];
            }
            sh.sum = s;
            sh.ties = t;
            sh.cnt = q;
        }
    }
    cl_sync();
    u64 tie_w = cut ? weight(value_of(cut_key)) : 0;
    if (cut && value_of(cut_key) < least) {
        tie_w = 0;
        ties_kept = 0;
    }
    u64 total = 0, before = 0;          // kept weight of the row, and in front of this CTA
    uint32_t kept = 0, tie_before = 0;  // kept tokens; ties in front of this CTA
    {
        uint32_t seen = 0;
        for (uint32_t r = 0; r < nc; ++r) {
            const u64 s = cl_ld64(cl_map(&sh.sum, r));
            const uint32_t t = cl_ld32(cl_map(&sh.ties, r));
            if (r == rank) {
                before = total;
                tie_before = seen;
            }
            kept += cl_ld32(cl_map(&sh.cnt, r));
            total += s + tie_w * (min(ties_kept, seen + t) - min(ties_kept, seen));
            seen += t;
        }
        kept += ties_kept;
    }
    cl_sync();  // the cluster is done with this CTA's shared memory
    const double uw = static_cast<double>(p.u[row]) * static_cast<double>(total);
    const u64 want = uw >= 0.0 ? min(total - 1, static_cast<u64>(uw)) : 0;  // running sum > want
    // ---- the warp's run that holds it, then the token in it
    int w0 = -1;
    u64 at = before;
    uint32_t tb = tie_before;
    for (int w = 0; w < kWarpsS; ++w) {
        const u64 s = sh.wsum[w] + tie_w * (min(ties_kept, tb + sh.wties[w]) - min(ties_kept, tb));
        if (want >= at && want < at + s) {
            w0 = w;
            break;
        }
        at += s;
        tb += sh.wties[w];
    }
    if (w0 < 0) return;  // another CTA's
    const int from = w0 * run, to = min(n, from + run);
    const int per = (run + kThreads - 1) / kThreads;
    const int i0 = min(to, from + tid * per), i1 = min(to, i0 + per);
    u64 sum = 0;
    uint32_t ties = 0;
    auto kept_weight = [&](int i, bool& tie) -> u64 {
        const float xi = canon(x[i]);
        const uint32_t key = key_of(xi);
        tie = cut && key == cut_key;
        if ((cut && key <= cut_key) || xi < least) return 0;
        return weight(xi);
    };
    for (int i = i0; i < i1; ++i) {
        bool tie;
        sum += kept_weight(i, tie);
        ties += tie;
    }
    uint32_t all_ties;
    u64 all;
    const uint32_t tie_at = tb + block_incl<uint32_t>(ties, sh.red32, &all_ties) - ties;
    sum += tie_w * (min(ties_kept, tie_at + ties) - min(ties_kept, tie_at));
    u64 acc = at + block_incl<u64>(sum, sh.red, &all) - sum;
    if (want >= acc && want < acc + sum) {
        uint32_t tr = tie_at;
        for (int i = i0; i < i1; ++i) {
            bool tie;
            u64 w = kept_weight(i, tie);
            if (tie) w = tr++ < ties_kept ? tie_w : 0;
            if (want < acc + w) {
                p.token[row] = lo + i;
                if (p.kept) p.kept[row] = static_cast<int>(kept);
                if (p.prob) p.prob[row] = static_cast<float>(static_cast<double>(w) / static_cast<double>(total));
                break;
            }
            acc += w;
        }
    }
}

// ------------------------------------------------------------------------------ bf16
constexpr int kHThreads = 1024;
constexpr int kHWarps = kHThreads / 32;
constexpr int kGroups = 2048;          // ordered groups of 32 neighbouring values
constexpr int kHistBytes = 65536 * 2;
constexpr int kHSlice = 131072;
constexpr int kFold = 32768;           // logits between two folds of the counters
constexpr int kMaxBig = kHSlice / kFold;
constexpr int kBinades = 16;           // of the table of weights by value, either sign
constexpr int kHalfTab = kBinades * 128;
constexpr uint32_t kManyKept = 1024;   // kept tokens from which the table pays

// Values in descending order: place o in [0, 65536) <-> raw bits. Positive ones (NaNs above +inf
// first, whose counts are moved to -inf), then negative ones; -0 (0x8000) has the place after +0.
__device__ __forceinline__ uint32_t raw_of(uint32_t o) { return o < 32768u ? 32767u - o : o; }
__device__ __forceinline__ uint32_t place_of(uint32_t raw) { return raw < 32768u ? 32767u - raw : raw; }
constexpr uint32_t kPlaceNegInf = 0xff80u, kPlaceZero = 32767u, kPlaceNegZero = 0x8000u;
__device__ __forceinline__ bool is_nan_place(uint32_t o) { return (raw_of(o) & 0x7fffu) > 0x7f80u; }
__device__ __forceinline__ float value_at(uint32_t o) { return __uint_as_float(raw_of(o) << 16); }

struct HShare {
    u64 table[32 * kTableCopies];
    union {
        u64 mass[kGroups];       // (first CTA) weight of a group
        u64 by_value[2 * kHalfTab];  // later: the weights of the values in the upper binades
    };
    uint32_t cnt[kGroups];   // (first CTA) its count
    u64 red[kHWarps];
    uint32_t red32[kHWarps];
    float maxv;              // of this CTA's slice
    uint32_t n_big;          // counters that reached 2^15 at a fold ..
    uint32_t big[kMaxBig];   // .. each stands for 2^15 logits of this value more
    uint32_t map[kGroups / 32];  // groups with a count
    uint32_t n_list;
    float row_max;
    uint32_t bigs;           // folded counters of all CTAs
    uint16_t list[kGroups];      // the groups in which some CTA has a count
    uint32_t cut, ties;      // (first CTA) the last kept value's place, how many of it are kept
    uint32_t kept;
    u64 total;               // kept weight
    u64 sum;                 // of this CTA: kept weight above the cut
    uint32_t tied;           // logits at the cut
    u64 wsum[kHWarps];
    uint32_t wties[kHWarps];
};

template <typename V>
__device__ __forceinline__ V h_scan(V v, V* red, V* total) {  // inclusive, in thread order
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V n = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += n;
    }
    __syncthreads();
    if (lane == 31) red[warp] = v;
    __syncthreads();
    V before = lane < kHWarps ? red[lane] : V(0);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V n = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += n;
    }
    *total = __shfl_sync(0xffffffffu, before, 31);
    before = __shfl_sync(0xffffffffu, before, (warp + 31) & 31);
    return (warp ? before : V(0)) + v;
}

template <int NC>
__global__ void __launch_bounds__(kHThreads, 1) sample_hist_kernel(const SampleBatchParams p, int slice) {
    extern __shared__ __align__(16) unsigned char dyn[];
    uint32_t* hist = reinterpret_cast<uint32_t*>(dyn);
    HShare& sh = *reinterpret_cast<HShare*>(dyn + kHistBytes);
    const uint32_t rank = cl_rank();
    const int row = blockIdx.x / NC, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int lo = min(p.vocab, static_cast<int>(rank) * slice), n = min(p.vocab, lo + slice) - lo;
    const bf16* gx = static_cast<const bf16*>(p.logits) + row * p.ld + lo;
    const uint16_t* raw16 = reinterpret_cast<const uint16_t*>(gx);
    // 16-byte vectors from the first aligned logit on; `head` logits stand before it
    const int head = min(n, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(gx) & 15)) & 15) / 2);
    const int nv = (n - head) / 8, tail = head + 8 * nv;
    const uint4* vec = reinterpret_cast<const uint4*>(gx + head);

    const float temp = p.temperature ? p.temperature[row] : 1.f;
    const bool greedy = !(temp > 0.f);
    const int k = p.top_k ? p.top_k[row] : 0;
    const float tp = p.top_p ? p.top_p[row] : 0.f, mp = p.min_p ? p.min_p[row] : 0.f, u = p.u[row];
    const bool use_k = k > 0 && k < p.vocab, use_p = tp > 0.f && tp < 1.f, use_m = mp > 0.f;

    for (int i = tid; i < kHistBytes / 16; i += kHThreads) reinterpret_cast<uint4*>(hist)[i] = make_uint4(0, 0, 0, 0);
    if (tid < 32) Weight::fill(sh.table);
    if (tid == 0) sh.n_big = 0;
    __syncthreads();

    // ---- count the slice's values; its maximum
    {
        // two values share a word: the even one's count is the lower half
        const uint32_t hist_at = smem_u32(hist);
        auto add = [&](uint32_t at, uint32_t inc) { asm volatile("red.shared.add.u32 [%0], %1;" ::"r"(hist_at + at), "r"(inc) : "memory"); };
        __nv_bfloat162 mx = __halves2bfloat162(__ushort_as_bfloat16(0xff80), __ushort_as_bfloat16(0xff80));
        auto word = [&](uint32_t w) {
            mx = __hmax2(mx, *reinterpret_cast<const __nv_bfloat162*>(&w));  // a NaN loses
            if (!greedy) {  // the first maximum needs no counts
                add((w << 1) & 0x1fffcu, (w & 1u) * 65535u + 1u);
                add((w >> 15) & 0x1fffcu, ((w >> 16) & 1u) * 65535u + 1u);
            }
        };
        constexpr int U = 4;
        // vectors between two folds; the up to 14 logits beside the vectors come on top of the last
        const int chunk = n > 65535 ? kFold / 8 - 2 : nv;
        for (int c0 = 0; c0 < nv; c0 += chunk) {
            const int c1 = min(nv, c0 + chunk);
            if (c0 > 0 && !greedy) {
                // a counter holds less than 2^15 after a fold, so the logits up to the next cannot overflow it
                __syncthreads();
                for (int i = tid; i < kHistBytes / 16; i += kHThreads) {
                    uint4 v = reinterpret_cast<uint4*>(hist)[i];
                    if ((v.x | v.y | v.z | v.w) & 0x80008000u) {
                        uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int h = 0; h < 2; ++h)
                                if (x[j] & (0x8000u << (16 * h))) {
                                    x[j] &= ~(0x8000u << (16 * h));
                                    sh.big[atomicAdd(&sh.n_big, 1u) & (kMaxBig - 1)] = 8 * i + 2 * j + h;
                                }
                        reinterpret_cast<uint4*>(hist)[i] = make_uint4(x[0], x[1], x[2], x[3]);
                    }
                }
                __syncthreads();
            }
            for (int i0 = c0 + tid; i0 < c1; i0 += U * kHThreads) {
                uint4 v[U];
#pragma unroll
                for (int q = 0; q < U; ++q)
                    if (i0 + q * kHThreads < c1) v[q] = vec[i0 + q * kHThreads];
#pragma unroll
                for (int q = 0; q < U; ++q) {
                    if (i0 + q * kHThreads >= c1) break;
                    word(v[q].x);
                    word(v[q].y);
                    word(v[q].z);
                    word(v[q].w);
                }
            }
        }
        for (int i = tid; i < n - 8 * nv; i += kHThreads) {  // the up to 14 that the vectors leave at both ends
            const uint32_t raw = raw16[i < head ? i : tail + i - head];
            const uint32_t w = raw | raw << 16;
            mx = __hmax2(mx, *reinterpret_cast<const __nv_bfloat162*>(&w));
            if (!greedy) add((raw << 1) & 0x1fffcu, (raw & 1u) * 65535u + 1u);
        }
        float m = fmaxf(__low2float(mx), __high2float(mx));
        m = warp_max(m);
        if (lane == 0) sh.red32[warp] = __float_as_uint(m);
        __syncthreads();
        if (warp == 0) {
            m = warp_max(__uint_as_float(sh.red32[lane]));
            if (lane == 0) sh.maxv = m;
        }
        // groups with a count: a warp looks at eight at a time
        if (!greedy)
            for (int i = warp; i < kGroups / 8; i += kHWarps) {
                const uint4 v = reinterpret_cast<const uint4*>(hist)[32 * i + lane];
                uint32_t any = __ballot_sync(0xffffffffu, (v.x | v.y | v.z | v.w) != 0);
                any |= any >> 1;
                any |= any >> 2;  // bit 4 j: lanes 4 j .. 4 j + 3, the 32 values from 256 i + 32 j on
                uint32_t bits = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) bits |= ((any >> (4 * j)) & 1u) << j;
                if (lane == 0) reinterpret_cast<uint8_t*>(sh.map)[i] = static_cast<uint8_t>(bits);
            }
    }
    cl_sync();
    // ---- the first warp gathers what the others found (a few remote loads, each once a CTA): the
    // row's maximum, the folded counters and the groups in which some CTA has a count
    if (warp == 0) {
        float m = lane < NC ? __uint_as_float(cl_ld32(cl_map(&sh.maxv, lane))) : -INFINITY;
        m = warp_max(m) + 0.f;  // -0 counts as +0
        uint32_t big = lane < NC ? cl_ld32(cl_map(&sh.n_big, lane)) : 0;
        const uint32_t bigs = __reduce_add_sync(0xffffffffu, big);
        if (!greedy) {
            uint32_t g2[2] = {0, 0}, w[2][NC];
#pragma unroll
            for (int r = 0; r < NC; ++r) {
                w[0][r] = cl_ld32(cl_map(&sh.map[2 * lane], r));
                w[1][r] = cl_ld32(cl_map(&sh.map[2 * lane + 1], r));
            }
#pragma unroll
            for (int r = 0; r < NC; ++r) {
                g2[0] |= w[0][r];
                g2[1] |= w[1][r];
            }
            if (bigs)
                for (int r = 0; r < NC; ++r)
                    for (uint32_t b = 0; b < __shfl_sync(0xffffffffu, big, r); ++b) {
                        // a fold may have emptied the counter's group
                        const uint32_t g = cl_ld32(cl_map(&sh.big[b], r)) >> 5;
                        if (g >> 6 == static_cast<uint32_t>(lane)) g2[(g >> 5) & 1] |= 1u << (g & 31);
                    }
            // -0 (raw 0x8000, group 1024, word 32) counts at +0's place (group 0)
            const uint32_t neg = __shfl_sync(0xffffffffu, g2[0], 16) & 1u;
            if (lane == 0) g2[0] |= neg;
            uint32_t at = 0;
#pragma unroll
            for (int h = 0; h < 2; ++h)
                for (uint32_t left = __ballot_sync(0xffffffffu, g2[h] != 0); left; left &= left - 1) {
                    const int src = __ffs(left) - 1;
                    const uint32_t bits = __shfl_sync(0xffffffffu, g2[h], src);
                    const uint32_t g = 32 * (2 * src + h) + lane;
                    if (bits >> lane & 1u)  // 32 neighbouring raw values are 32 neighbouring places
                        sh.list[at + __popc(bits & ((1u << lane) - 1))] = static_cast<uint16_t>(place_of(32 * g) >> 5);
                    at += __popc(bits);
                }
            if (lane == 0) sh.n_list = at;
        }
        if (lane == 0) {
            sh.row_max = m;
            sh.bigs = bigs;
        }
    } else if (rank == 0) {
        for (int g = tid - 32; g < kGroups; g += kHThreads - 32) {
            sh.mass[g] = 0;
            sh.cnt[g] = 0;
        }
    }
    cl_sync();  // the first CTA's sums are cleared
    const float M = sh.row_max;
    if (M == -INFINITY) {
        if (rank == 0 && tid == 0) {
            p.token[row] = -1;
            if (p.kept) p.kept[row] = 0;
            if (p.prob) p.prob[row] = 0.f;
        }
        return;  // no CTA reads another's shared memory from here on
    }
    const Weight weight(M, greedy ? 1.f : temp, sh.table);
    uint32_t cut = place_of(__float_as_uint(M) >> 16), ties_kept = 1, kept = 1;
    u64 total = 1ull << kFrac;
    if (!greedy) {
        // ---- weight and count of every listed group of 32 ordered values; the cluster's CTAs take them in
        // turn
        uint32_t remote[NC];
#pragma unroll
        for (int r = 0; r < NC; ++r) remote[r] = cl_map(hist, r);
        const uint32_t bigs = sh.bigs;
        auto count_at = [&](uint32_t raw) {
            uint32_t w[NC], s = 0;
#pragma unroll
            for (int r = 0; r < NC; ++r) w[r] = cl_ld32(remote[r] + ((raw << 1) & 0x1fffcu));
#pragma unroll
            for (int r = 0; r < NC; ++r) s += raw & 1u ? w[r] >> 16 : w[r] & 0xffffu;
            if (bigs)
                for (int r = 0; r < NC; ++r)
                    for (uint32_t b = 0; b < cl_ld32(cl_map(&sh.n_big, r)); ++b)
                        if (cl_ld32(cl_map(&sh.big[b], r)) == raw) s += kFold;
            return s;
        };
        // the count of place o; NaN and -inf have no weight and count as 0 here, -0 is part of +0
        auto place_count = [&](uint32_t o) -> uint32_t {
            if (is_nan_place(o) || o == kPlaceNegZero || o == kPlaceNegInf) return 0;
            return count_at(raw_of(o)) + (o == kPlaceZero ? count_at(0x8000u) : 0u);
        };
        const uint32_t mass_at = cl_map(sh.mass, 0), cnt_at = cl_map(sh.cnt, 0);
        for (uint32_t i = rank + NC * warp; i < sh.n_list; i += NC * kHWarps) {
            const uint32_t g = sh.list[i], o = 32 * g + lane;
            uint32_t cn = place_count(o);
            u64 ms = cn ? cn * weight(value_at(o)) : 0;
            cn = __reduce_add_sync(0xffffffffu, cn);
#pragma unroll
            for (int q = 16; q; q >>= 1) ms += __shfl_xor_sync(0xffffffffu, ms, q);
            if (lane == 0) {
                asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(mass_at + 8 * g), "l"(ms) : "memory");
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cnt_at + 4 * g), "r"(cn) : "memory");
            }
        }
        cl_sync();
        if (rank == 0) {
            // two groups a thread, in order; then the group that holds the cut, a value a lane
            const uint32_t c0 = sh.cnt[2 * tid], c1 = sh.cnt[2 * tid + 1];
            const u64 m0 = sh.mass[2 * tid], m1 = sh.mass[2 * tid + 1];
            uint32_t cfin;
            u64 z;
            uint32_t cb = h_scan<uint32_t>(c0 + c1, sh.red32, &cfin) - c0 - c1;
            u64 mb = h_scan<u64>(m0 + m1, sh.red, &z) - m0 - m1;
            // the kept prefix ends at: the k-th token; the first at which the weight reaches top_p of
            // all (an integer >= top_p * Z); the last with a weight of min_p
            const u64 target = use_p ? max(1ull, static_cast<u64>(ceil(static_cast<double>(tp) * static_cast<double>(z)))) : ~0ull;
            const u64 most = use_k ? static_cast<u64>(k) : ~0ull;
            auto reached = [&](uint32_t cc, u64 mm) { return cc >= most || mm >= target; };
            const bool any_cut = reached(cfin, z);
            if (tid == 0) {
                sh.cut = 65536u;  // nothing is cut: all tokens are kept, the -inf ones (weight 0) included
                sh.ties = 0;
                sh.kept = static_cast<uint32_t>(p.vocab);
                sh.total = z;
                if (use_k && !any_cut) sh.kept = static_cast<uint32_t>(k);  // the cut lies among the -inf ones
            }
            __syncthreads();
            if (any_cut && !reached(cb, mb) && reached(cb + c0 + c1, mb + m0 + m1)) {
                const bool second = !reached(cb + c0, mb + m0);
                sh.red32[0] = 2 * tid + second;
                sh.red32[1] = second ? cb + c0 : cb;
                sh.red[0] = second ? mb + m0 : mb;
            }
            __syncthreads();
            if (any_cut && warp == 0) {
                const uint32_t o = 32 * sh.red32[0] + lane;
                const uint32_t cn = place_count(o);
                const u64 w = cn ? weight(value_at(o)) : 0, ms = cn * w;
                uint32_t ci = cn;
                u64 mi = ms;
#pragma unroll
                for (int q = 1; q < 32; q <<= 1) {
                    const uint32_t a = __shfl_up_sync(0xffffffffu, ci, q);
                    const u64 b = __shfl_up_sync(0xffffffffu, mi, q);
                    if (lane >= q) {
                        ci += a;
                        mi += b;
                    }
                }
                ci += sh.red32[1];
                mi += sh.red[0];
                if (!reached(ci - cn, mi - ms) && reached(ci, mi)) {
                    u64 take = cn;
                    if (use_k) take = min(take, most - (ci - cn));
                    if (use_p && w) take = min(take, (target - (mi - ms) + w - 1) / w);
                    sh.cut = o;
                    sh.ties = static_cast<uint32_t>(take);
                    sh.kept = ci - cn + static_cast<uint32_t>(take);
                    sh.total = mi - ms + take * w;
                }
            }
            __syncthreads();
            if (use_m) {
                // min-p: the places down to that of the least bf16 at or above the floor; where the cut
                // lies among them nothing changes
                const uint32_t f = __float_as_uint(min_p_floor(M, temp, mp) + 0.f);
                uint32_t end = place_of((f & 0x80000000u ? f : f + 0xffffu) >> 16) + 1;
                if (end == kPlaceNegZero) ++end;  // both zeros or none
                if (sh.cut >= end) {
                    const uint32_t ge = end >> 5;
                    __syncthreads();
                    if (2 * tid <= ge && ge <= 2 * tid + 1) {
                        const bool second = ge == 2u * tid + 1;
                        sh.red32[1] = second ? cb + c0 : cb;
                        sh.red[0] = second ? mb + m0 : mb;
                    }
                    __syncthreads();
                    if (warp == 0) {
                        uint32_t cn = 0;
                        u64 ms = 0;
                        const uint32_t o = 32 * ge + lane;
                        if (o < end) {
                            cn = place_count(o);
                            ms = cn ? cn * weight(value_at(o)) : 0;
                        }
#pragma unroll
                        for (int q = 16; q; q >>= 1) {
                            cn += __shfl_xor_sync(0xffffffffu, cn, q);
                            ms += __shfl_xor_sync(0xffffffffu, ms, q);
                        }
                        if (lane == 0) {
                            sh.cut = end;  // places before it are kept, none of it
                            sh.ties = 0;
                            sh.kept = sh.red32[1] + cn;
                            sh.total = sh.red[0] + ms;
                        }
                    }
                }
            }
        }
        cl_sync();
        cut = cl_ld32(cl_map(&sh.cut, 0));
        ties_kept = cl_ld32(cl_map(&sh.ties, 0));
        kept = cl_ld32(cl_map(&sh.kept, 0));
        total = cl_ld64(cl_map(&sh.total, 0));
    }
    const double uw = static_cast<double>(u) * static_cast<double>(total);
    const u64 want = greedy || !(uw >= 0.0) ? 0 : min(total - 1, static_cast<u64>(uw));  // running sum > want

    // ---- second pass: kept weight of every warp's run of the slice, in index order
    const float cut_v = cut < 65536u ? (is_nan_place(cut) ? (cut < 32768u ? INFINITY : -INFINITY) : value_at(cut) + 0.f) : -INFINITY;
    const u64 tie_w = ties_kept ? weight(cut_v) : 0;
    // above: places before the cut. Without a cut everything above -inf is (weight 0 below).
    auto look = [&](float x, bool& tie) -> u64 {
        tie = ties_kept && x == cut_v;
        return x > cut_v ? weight(x) : 0;
    };
    const int run = ((slice + kHWarps - 1) / kHWarps + 255) & ~255;  // whole warp-wide vectors
    // with many tokens kept, the weights of all values in 16 binades below the largest magnitude that
    // has a weight are tabulated (four a thread) and looked up
    const bool many = kept > kManyKept && !weight.inf;
    uint32_t tab_base = 0;
    if (many) {
        const float far = fmaxf(fabsf(M), fabsf(M - 42.f * temp));  // exp(-42) is below 2^-60
        tab_base = static_cast<uint32_t>(max(0, static_cast<int>(min(__float_as_uint(far) >> 23, 254u)) - kBinades + 1)) << 7;
        for (int i = tid; i < 2 * kHalfTab; i += kHThreads) {
            const float x = canon(__uint_as_float((tab_base + (i & (kHalfTab - 1)) | (i >= kHalfTab ? 0x8000u : 0u)) << 16));
            bool tie;
            const u64 w = look(x, tie);
            sh.by_value[i] = tie ? 1ull << 52 : w;
        }
        __syncthreads();
    }
    {
        const int from = warp * run, to = min(n, from + run);  // vectors and ends, counted from `head` on
        u64 sum = 0;
        uint32_t ties = 0;
        const __nv_bfloat162 cut2 = __float2bfloat162_rn(cut_v);
        // positions from..to - 1 of the slice: logit at position i
        auto one = [&](int i) {
            bool tie;
            const float x = canon(bf2f(raw16[i]));
            sum += look(x, tie);
            ties += tie;
        };
        // vectors that lie wholly inside [from, to)
        const int v0 = max(0, (from - head + 7) / 8), v1 = max(v0, (to - head) >= 0 ? (to - head) / 8 : 0);
        if (from < to) {
            const int a_end = min(to, head + 8 * v0), b_start = max(a_end, head + 8 * v1);
            for (int i = from + lane; i < a_end; i += 32) one(i);
            for (int i = b_start + lane; i < to; i += 32) one(i);
            if (many) {
                // every logit by one lookup; entry 2^52 stands for a logit at the cut (a thread's weights
                // stay below 2^52)
                u64 both = 0;
                auto add = [&](uint32_t raw) {
                    const uint32_t at = (raw & 0x7fffu) - tab_base;
                    if (at < static_cast<uint32_t>(kHalfTab)) {
                        both += sh.by_value[at + (raw >> 15) * kHalfTab];
                    } else {
                        const float x = canon(__uint_as_float(raw << 16));
                        if (x >= cut_v) {
                            bool tie;
                            sum += look(x, tie);
                            ties += tie;
                        }
                    }
                };
                uint4 v = v0 + lane < v1 ? vec[v0 + lane] : make_uint4(0, 0, 0, 0);
                for (int i0 = v0 + lane; i0 < v1; i0 += 32) {
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
                    if (i0 + 32 < v1) v = vec[i0 + 32];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        add(w[j] & 0xffffu);
                        add(w[j] >> 16);
                    }
                }
                sum += both & ((1ull << 52) - 1);
                ties += static_cast<uint32_t>(both >> 52);
            } else {
                for (int i0 = v0 + lane; i0 < v1; i0 += 4 * 32) {
                    uint4 v[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (i0 + 32 * q < v1) v[q] = vec[i0 + 32 * q];
                    // vectors with a logit that does not lie below the cut
                    uint32_t take = 0;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const uint32_t w[4] = {v[q].x, v[q].y, v[q].z, v[q].w};
                        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(w);
                        const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
                        if (i0 + 32 * q < v1 && !__hblt2(m, cut2)) take |= 1u << q;
                    }
                    for (; take; take &= take - 1) {
                        const int at = head + 8 * (i0 + 32 * (__ffs(take) - 1));
#pragma unroll 1
                        for (int j = 0; j < 8; ++j) one(at + j);
                    }
                }
            }
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        ties = __reduce_add_sync(0xffffffffu, ties);
        if (lane == 0) {
            sh.wsum[warp] = sum;
            sh.wties[warp] = ties;
        }
        __syncthreads();
        if (warp == 0) {
            u64 s = sh.wsum[lane];
#pragma unroll
            for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            const uint32_t t = __reduce_add_sync(0xffffffffu, sh.wties[lane]);
            if (lane == 0) {
                sh.sum = s;
                sh.tied = t;
            }
        }
    }
    cl_sync();
    u64 at = 0;          // kept weight in front of this CTA
    uint32_t tb = 0;     // logits at the cut in front of it
    for (uint32_t r = 0; r < rank; ++r) {
        const u64 s = cl_ld64(cl_map(&sh.sum, r));
        const uint32_t t = cl_ld32(cl_map(&sh.tied, r));
        at += s + tie_w * (min(ties_kept, tb + t) - min(ties_kept, tb));
        tb += t;
    }
    cl_sync();  // the cluster is done with this CTA's shared memory
    // ---- the warp's run that holds the target, then the token in it
    int w0 = -1;
    for (int w = 0; w < kHWarps; ++w) {
        const u64 s = sh.wsum[w] + tie_w * (min(ties_kept, tb + sh.wties[w]) - min(ties_kept, tb));
        if (want >= at && want < at + s) {
            w0 = w;
            break;
        }
        at += s;
        tb += sh.wties[w];
    }
    if (w0 < 0) return;  // another CTA's
    const int from = w0 * run, to = min(n, from + run), per = (run + kHThreads - 1) / kHThreads;
    const int i0 = min(to, from + tid * per), i1 = min(to, i0 + per);
    u64 sum = 0;
    uint32_t ties = 0;
    for (int i = i0; i < i1; ++i) {
        bool tie;
        sum += look(canon(bf2f(raw16[i])), tie);
        ties += tie;
    }
    uint32_t all_ties;
    u64 all;
    const uint32_t tie_at = tb + h_scan<uint32_t>(ties, sh.red32, &all_ties) - ties;
    sum += tie_w * (min(ties_kept, tie_at + ties) - min(ties_kept, tie_at));
    u64 acc = at + h_scan<u64>(sum, sh.red, &all) - sum;
    if (want >= acc && want < acc + sum) {
        uint32_t tr = tie_at;
        for (int i = i0; i < i1; ++i) {
            bool tie;
            u64 w = look(canon(bf2f(raw16[i])), tie);
            if (tie) w = tr++ < ties_kept ? tie_w : 0;
            if (want < acc + w) {
                p.token[row] = lo + i;
                if (p.kept) p.kept[row] = static_cast<int>(kept);
                if (p.prob) p.prob[row] = static_cast<float>(static_cast<double>(w) / static_cast<double>(total));
                break;
            }
            acc += w;
        }
    }
}

template <typename... P, typename... A>
void launch_cluster(void (*kern)(P...), int rows, int nc, int threads, size_t smem, cudaStream_t stream, A&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(rows) * nc);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = nc;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    HYB_CUDA(cudaLaunchKernelEx(&cfg, kern, std::forward<A>(args)...));
    HYB_LAUNCH_CHECK("sample_batch kernel");
}

template <int NC>
void launch_hist_t(const SampleBatchParams& p, cudaStream_t stream) {
    const int slice = ((p.vocab + NC - 1) / NC + 7) & ~7;
    allow_smem(reinterpret_cast<const void*>(sample_hist_kernel<NC>), kHistBytes + sizeof(HShare));
    launch_cluster(sample_hist_kernel<NC>, p.rows, NC, kHThreads, kHistBytes + sizeof(HShare), stream, p, slice);
}

void launch_hist(const SampleBatchParams& p, cudaStream_t stream) {
    // the fewest CTAs a row whose slices fit; more while all rows stay resident at once (one CTA an
    // SM) and a slice is worth one
    int nc = 1;
    while (nc < kMaxCluster && (p.vocab + nc - 1) / nc > kHSlice) nc *= 2;
    while (nc < kMaxCluster && p.rows * nc * 2 <= num_sms() && p.vocab / nc >= 8192) nc *= 2;
    switch (nc) {
        case 1: launch_hist_t<1>(p, stream); break;
        case 2: launch_hist_t<2>(p, stream); break;
        case 4: launch_hist_t<4>(p, stream); break;
        default: launch_hist_t<8>(p, stream); break;
    }
}

void launch_f32(const SampleBatchParams& p, cudaStream_t stream) {
    const int most = kSliceBytes / 4;
    int nc = 1;
    while (nc < kMaxCluster && (p.vocab + nc - 1) / nc > most) nc *= 2;
    // more CTAs a row while the rows alone leave SMs idle and a slice is worth one
    while (nc < kMaxCluster && p.rows * nc * 2 <= num_sms() && p.vocab / nc >= 4096) nc *= 2;
    const int slice = ((p.vocab + nc - 1) / nc + 7) & ~7;
    const int resident = slice <= most ? 1 : 0;  // above 2^18 logits the slice stays in L2
    allow_smem(reinterpret_cast<const void*>(sample_radix_kernel), sizeof(Hist) + sizeof(Merged) + kSliceBytes);
    launch_cluster(sample_radix_kernel, p.rows, nc, kThreads, sizeof(Hist) + sizeof(Merged) + (resident ? slice * 4 : 0), stream, p, slice, resident);
}

}  // namespace

void launch_sample_batch(const SampleBatchParams& p, cudaStream_t stream) {
    if (p.f32) launch_f32(p, stream);
    else launch_hist(p, stream);
}

}  // namespace hyb
