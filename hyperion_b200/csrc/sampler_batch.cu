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
// additions: weights are integers, w = rint(exp(..) * 2^44), and their 64-bit sums are exact
// in any order (vocabulary <= 2^19). exp is evaluated in double as 2^d, d = (x - M) log2(e) / T:
// d = n/32 + r with |r| <= 1/64, 2^r by its Taylor polynomial of degree 5 in r ln 2 (the next
// term is below (ln 2 / 64)^6 / 720 = 2e-15), 2^(j/32) from a 32-entry table.
//
// One thread-block cluster per row; CTA c of the cluster owns a contiguous slice of the row,
// loaded once into its shared memory, so the row's bytes cross HBM once and every later pass
// runs from shared memory. The cut of top-k / top-p is found by radix selection on an
// order-preserving 32-bit key, 11 bits a level: each CTA fills a histogram of counts and
// weights (three 16-bit limbs, so that the shared atomics stay native 32-bit ones), the
// cluster's first CTA adds the histograms up over distributed shared memory and finds the bin
// in which the cut lies. bf16 logits have 16-bit keys and need two levels, fp32 ones three.
#include "kernels.h"
#include "tma.cuh"

#include <algorithm>
#include <cstddef>
#include <type_traits>

namespace hyb {

namespace {

constexpr int kThreads = 512;
constexpr int kWarpsS = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kFrac = 44;
constexpr int kMaxCluster = 8;
constexpr int kSliceBytes = 128 * 1024;  // the largest slice held in shared memory
constexpr int kMaxSlice = 65536;         // limb sums of a slice fit 32 bits: 65535 * 65536 < 2^32

typedef unsigned long long u64;

struct Hist {
    uint32_t cnt[kBins], l0[kBins], l1[kBins], l2[kBins];
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
    Cut cut;
    u64 sum;        // kept weight above the cut key
    uint32_t cnt;   // kept tokens above it
    uint32_t ties;  // tokens equal to it
    u64 wsum[kWarpsS];
    uint32_t wties[kWarpsS];
    u64 red[kWarpsS];
    uint32_t red32[kWarpsS];
    double table[32];
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
__device__ __forceinline__ uint4 cl_ld128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(a)
                 : "memory");
    return v;
}

// NaN -> -inf, -0 -> +0.
__device__ __forceinline__ float canon(float x) { return x != x ? -INFINITY : x + 0.0f; }
__device__ __forceinline__ float load_x(const bf16* x, int i) { return canon(bf2f(x[i])); }
__device__ __forceinline__ float load_x(const float* x, int i) { return canon(x[i]); }
// Order-preserving key; a bf16 value's lies in the upper 16 bits, the rest zero.
template <bool F32>
__device__ __forceinline__ uint32_t key_of(float f) {
    const uint32_t u = __float_as_uint(f);
    const uint32_t k = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return F32 ? k : k & 0xffff0000u;
}
__device__ __forceinline__ float value_of(uint32_t key, bool f32) {
    if (key & 0x80000000u) return __uint_as_float(key & 0x7fffffffu);
    const uint32_t u = ~key;
    return __uint_as_float(f32 ? u : u & 0xffff0000u);
}

// rint(2^44 * exp((x - M) / T)), c = log2(e) / T.
__device__ __forceinline__ u64 weight(float x, float M, double c, const double* table) {
    if (x == M) return 1ull << kFrac;
    const double d = (static_cast<double>(x) - static_cast<double>(M)) * c;
    if (!(d > -(kFrac + 2.0))) return 0;
    constexpr double kMagic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are the rounded integer
    const double t = fma(d, 32.0, kMagic);
    const int n = __double2loint(t);
    const double r = fma(t - kMagic, -1.0 / 32.0, d) * 0.69314718055994530942;
    double q = fma(r, 1.0 / 120.0, 1.0 / 24.0);
    q = fma(q, r, 1.0 / 6.0);
    q = fma(q, r, 0.5);
    q = fma(q, r, 1.0);
    q = fma(q, r, 1.0);
    const double v = q * table[n & 31];
    // times 2^(n >> 5) 2^44 by the exponent field (results from 2^-2 up), then rounded to an integer
    const double s = __hiloint2double(__double2hiint(v) + ((n >> 5) + kFrac) * (1 << 20), __double2loint(v));
    return static_cast<u64>(__double_as_longlong(s + 4503599627370496.0)) & 0xFFFFFFFFFFFFFull;
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

template <bool F32>
__global__ void __launch_bounds__(kThreads) sample_batch_kernel(const SampleBatchParams p, int slice, int resident) {
    using T = typename std::conditional<F32, float, bf16>::type;
    extern __shared__ __align__(16) unsigned char dyn[];
    __shared__ Share sh;
    Hist& h = *reinterpret_cast<Hist*>(dyn);
    T* buf = reinterpret_cast<T*>(dyn + sizeof(Hist));
    uint32_t nc;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(nc));
    const uint32_t rank = cl_rank();
    const int row = blockIdx.x / nc, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int lo = min(p.vocab, static_cast<int>(rank) * slice), n = min(p.vocab, lo + slice) - lo;
    const T* gx = static_cast<const T*>(p.logits) + row * p.ld + lo;

    const float temp = p.temperature ? p.temperature[row] : 1.f;
    const bool greedy = !(temp > 0.f);
    int k = p.top_k ? p.top_k[row] : 0;
    float tp = p.top_p ? p.top_p[row] : 0.f, mp = p.min_p ? p.min_p[row] : 0.f;
    const bool use_k = k > 0 && k < p.vocab, use_p = tp > 0.f && tp < 1.f, use_m = mp > 0.f;
    const double c = 1.4426950408889634074 / static_cast<double>(temp);
    if (tid < 32) sh.table[tid] = exp2(tid * (1.0 / 32.0));

    // ---- the slice into shared memory, its maximum (first index)
    u64 best = 0;
    {
        float bx = -INFINITY;
        int bi = -1;
        constexpr int VEC = 16 / sizeof(T);
        const bool vec = (reinterpret_cast<uintptr_t>(gx) & 15) == 0;
        const int nv = vec ? n / VEC : 0;
        for (int i = tid; i < nv; i += kThreads) {
            const uint4 v = reinterpret_cast<const uint4*>(gx)[i];
            if (resident) reinterpret_cast<uint4*>(buf)[i] = v;
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                float x;
                if constexpr (F32) x = canon(__uint_as_float(w[j]));
                else x = canon(__uint_as_float((j & 1) ? w[j / 2] & 0xffff0000u : w[j / 2] << 16));
                if (bi < 0 || x > bx) {
                    bx = x;
                    bi = i * VEC + j;
                }
            }
        }
        for (int i = nv * VEC + tid; i < n; i += kThreads) {
            const T v = gx[i];
            if (resident) buf[i] = v;
            const float x = load_x(&v, 0);
            if (bi < 0 || x > bx) {
                bx = x;
                bi = i;
            }
        }
        if (bi >= 0) best = (static_cast<u64>(key_of<F32>(bx)) << 32) | static_cast<uint32_t>(~(lo + bi));
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
    for (uint32_t r = 0; r < nc; ++r) best = max(best, cl_ld64(cl_map(&sh.best, r)));
    const uint32_t arg = ~static_cast<uint32_t>(best);
    const float M = value_of(static_cast<uint32_t>(best >> 32), F32);
    const T* x = resident ? buf : gx;
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
        constexpr int LEVELS = F32 ? 3 : 2;
#pragma unroll 1
        for (int level = 0; level < LEVELS; ++level) {
            const int shift = level == 0 ? 21 : (level == 1 ? 10 : 0);
            const uint32_t width = level == 2 ? 10 : 11;
            for (int i = tid; i < 4 * kBins; i += kThreads) (&h.cnt[0])[i] = 0;
            __syncthreads();
            for (int i = tid; i < n; i += kThreads) {
                const float xi = load_x(x, i);
                const uint32_t key = key_of<F32>(xi);
                if (level && (key >> (shift + width)) != (cut_key >> (shift + width))) continue;
                const uint32_t bin = (key >> shift) & ((1u << width) - 1);
                atomicAdd(&h.cnt[bin], 1u);
                if (use_p) {
                    const u64 w = weight(xi, M, c, sh.table);
                    if (w) {
                        atomicAdd(&h.l0[bin], static_cast<uint32_t>(w) & 0xffffu);
                        if (w >> 16) atomicAdd(&h.l1[bin], static_cast<uint32_t>(w >> 16) & 0xffffu);
                        if (w >> 32) atomicAdd(&h.l2[bin], static_cast<uint32_t>(w >> 32));
                    }
                }
            }
            cl_sync();
            if (rank == 0) {
                // thread t takes bins from the top: 2047 - 4t - i
                uint32_t bc[4] = {0, 0, 0, 0};
                u64 bm[4] = {0, 0, 0, 0};
                const int b0 = kBins - 4 - 4 * tid;
                for (uint32_t r = 0; r < nc; ++r) {
                    const uint4 a = cl_ld128(cl_map(&h.cnt[b0], r));
                    const uint4 m0 = cl_ld128(cl_map(&h.l0[b0], r)), m1 = cl_ld128(cl_map(&h.l1[b0], r)),
                                m2 = cl_ld128(cl_map(&h.l2[b0], r));
                    const uint32_t av[4] = {a.w, a.z, a.y, a.x}, v0[4] = {m0.w, m0.z, m0.y, m0.x},
                                   v1[4] = {m1.w, m1.z, m1.y, m1.x}, v2[4] = {m2.w, m2.z, m2.y, m2.x};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        bc[i] += av[i];
                        bm[i] += v0[i] + (static_cast<u64>(v1[i]) << 16) + (static_cast<u64>(v2[i]) << 32);
                    }
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
            }
            cl_sync();
            const uint32_t a = cl_map(&sh.cut, 0);
            cut_key |= cl_ld32(a + offsetof(Cut, bin)) << shift;
            above = cl_ld32(a + offsetof(Cut, cnt));
            in_bin = cl_ld32(a + offsetof(Cut, in_bin));
            mass_above = cl_ld64(a + offsetof(Cut, mass));
            target = cl_ld64(a + offsetof(Cut, total));
            // the first CTA's next write of the cut lies behind the next level's first cluster barrier
        }
        // all tokens of the last bin are equal: as many of them as the cut needs
        uint32_t take = in_bin;
        if (use_k) take = min(take, static_cast<uint32_t>(k) - above);
        if (use_p) {
            const u64 w = weight(value_of(cut_key, F32), M, c, sh.table);
            if (w) take = static_cast<uint32_t>(min(static_cast<u64>(take), (target - mass_above + w - 1) / w));
        }
        ties_kept = take;
    }

    // ---- kept weights: warp w of the CTA owns a contiguous run of its slice
    const double mpd = static_cast<double>(fminf(mp, 1.f)) * 17592186044416.0;  // min_p in units of 2^-44
    auto passes = [&](u64 w) { return !use_m || static_cast<double>(w) >= mpd; };
    const int run = ((slice + kWarpsS - 1) / kWarpsS + 31) & ~31;
    {
        const int from = warp * run, to = min(n, from + run);
        u64 sum = 0;
        uint32_t cnt = 0, ties = 0;
        for (int i = from + lane; i < to; i += 32) {
            const float xi = load_x(x, i);
            const uint32_t key = key_of<F32>(xi);
            if (cut && key <= cut_key) {
                ties += key == cut_key;
                continue;
            }
            const u64 w = weight(xi, M, c, sh.table);
            if (passes(w)) {
                sum += w;
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
    u64 tie_w = cut ? weight(value_of(cut_key, F32), M, c, sh.table) : 0;
    if (cut && !passes(tie_w)) {
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
        const float xi = load_x(x, i);
        const uint32_t key = key_of<F32>(xi);
        tie = cut && key == cut_key;
        if (cut && key <= cut_key) return 0;
        const u64 w = weight(xi, M, c, sh.table);
        return passes(w) ? w : 0;
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

template <bool F32>
void launch_t(const SampleBatchParams& p, cudaStream_t stream) {
    const size_t elem = F32 ? 4 : 2;
    const int most = std::min<int>(kMaxSlice, kSliceBytes / static_cast<int>(elem));
    int nc = 1;
    while (nc < kMaxCluster && (p.vocab + nc - 1) / nc > most) nc *= 2;
    // more CTAs a row while the rows alone leave SMs idle and a slice is worth one
    while (nc < kMaxCluster && p.rows * nc * 2 <= num_sms() && p.vocab / nc >= 4096) nc *= 2;
    const int slice = ((p.vocab + nc - 1) / nc + 7) & ~7;
    const int resident = slice <= most ? 1 : 0;
    const size_t smem = sizeof(Hist) + (resident ? slice * elem : 0);
    auto kern = sample_batch_kernel<F32>;
    allow_smem(reinterpret_cast<const void*>(kern), sizeof(Hist) + kSliceBytes + 16);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(p.rows) * nc);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = nc;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    HYB_CUDA(cudaLaunchKernelEx(&cfg, kern, p, slice, resident));
    HYB_LAUNCH_CHECK("sample_batch_kernel");
}

}  // namespace

void launch_sample_batch(const SampleBatchParams& p, cudaStream_t stream) {
    if (p.f32) launch_t<true>(p, stream);
    else launch_t<false>(p, stream);
}

}  // namespace hyb
