// Drawing the next token of each row from its logits, with temperature, top-k, top-p and min-p, by one given uniform number.
//
//   w_i = e^{(l_i - max) / T}; kept: the tokens in the order of falling logit (equal ones: rising index) while fewer than k come before, w >= min_p,
//   and the mass before is below top_p times the mass of what the other two leave; token: the first, in the order of the indices, at which
//   the kept mass exceeds u times the whole.  T = 0: the largest logit's lowest index.  logprob = l_token - log sum e^l, without filters.
//
// A row is read from HBM once, and that (size of a logit * vocabulary) is its floor.  A cluster of 1 to 8 blocks holds the row in its shared
// memory; the passes over it (maximum; weights; the cuts; the draw) stay on the chip, the blocks exchange a few words after each.
//
// * The result is a token, not a number that may be a little off, so masses are integers: weights as multiples of 2^-44 of the largest one
//   (exponentials in fp64, relative error below 2^-44; smaller weights than 2^-45 count as nothing), whose sums do not depend on the order.
// * Cuts need no sort: tokens are counted (and their mass summed) in 1024 bins over the logits, the bin in which the cut falls is found by a
//   scan, and only its tokens are ranked against one another; a bin with too many is divided again, equal logits are counted by index.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "launch_limits.h"
#include "sampling.h"

namespace cg = cooperative_groups;

namespace sg {

namespace {

using u64 = unsigned long long;
constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = 1024, kList = 512, kMaxCluster = 8;
constexpr int kFrac = 44;                     // weights are multiples of 2^-44
constexpr float kRange = 46.f;                // log2 of the smallest weight that is looked at: what lies below is 0 as a multiple
constexpr double kLog2eD = 1.4426950408889634074;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }

// fp32 as an unsigned number of the same order (-0 as +0); 0 is below all that occur
__device__ __forceinline__ uint32_t order_key(float l) {
    const uint32_t b = __float_as_uint(l + 0.f);
    return (b >> 31) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k); }
// larger: earlier in the order (logit falling, index rising)
__device__ __forceinline__ u64 pack(float l, int index) { return (static_cast<u64>(order_key(l)) << 32) | (0xffffffffu - static_cast<uint32_t>(index)); }

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ u64 warp_scan(u64 v, int lane) {   // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 x = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += x;
    }
    return v;
}

struct Shared {
    double table[64];                 // 2^(j / 64)
    u64 mass[kBins];
    u64 list[kList], all[kList], all_q[kList];
    uint32_t count[kBins];
    u64 warp_q[kWarps];
    float warp_z[kWarps];
    // what other blocks of the cluster read
    u64 x_best, x_sum, x_cut;
    float x_z;
    uint32_t x_min, x_max, x_listed;
    // results of one thread for its block
    u64 b_before, b_total;
    uint32_t b_bin, b_count;
};

template <typename T, bool RESIDENT>
struct Row {
    cg::cluster_group cluster = cg::this_cluster();
    Shared& sh;
    const T* x;                       // this block's part of the row: shared memory, or where it lies
    int n, first, seg;                // its size, the index of its first token, tokens a warp
    int blocks, rank, warp, lane;
    float lmax;
    double to_log2;                   // log2(e) / T
    double least;                     // log2 of the smallest eligible weight
    float bin_scale, least_lo, least_hi;
    u64 cut = 0;                      // kept: pack() >= cut

    __device__ Row(Shared& s) : sh(s) {}

    __device__ __forceinline__ float at(int i) const { return to_f(x[i]); }
    __device__ __forceinline__ double log2_weight(float l) const {
        return l == lmax ? 0. : (static_cast<double>(l) - static_cast<double>(lmax)) * to_log2;
    }
    // Coarse log2 of a weight in fp32: never increases as l falls
    __device__ __forceinline__ float coarse(float l) const { return l == lmax ? 0.f : (l - lmax) * bin_scale; }
    __device__ __forceinline__ bool eligible(float l) const {
        const float t = coarse(l);
        if (t > least_hi) return true;
        if (!(t >= least_lo)) return false;                       // NaN and -inf as well
        return log2_weight(l) >= least;
    }
    // 2^t as a multiple of 2^-44, t <= 0: t = i / 64 + r, 2^r by its series to the fourth power (|r| <= 2^-7: 4e-14)
    __device__ __forceinline__ u64 weight(float l) const {
        const double t = log2_weight(l);
        if (!(t >= -45.)) return 0;
        const double big = 6755399441055744. / 64.;               // 1.5 * 2^52 / 64: adding it rounds to multiples of 1 / 64
        const double m = t + big;
        const int i = static_cast<int>(__double_as_longlong(m) & 0xffffffff);
        const double r = t - (m - big);
        double y = fma(r, 9.618129107628477e-3, 5.550410866482158e-2);   // ln2^4 / 24, ln2^3 / 6, ln2^2 / 2, ln2
        y = fma(r, y, 2.402265069591007e-1);
        y = fma(r, y, 6.931471805599453e-1);
        const double e = sh.table[i & 63];
        const double v = fma(e * r, y, e);                        // 2^(t - floor(i / 64)), in [0.99, 2.01)
        const long long bits = __double_as_longlong(v);
        const int shift = 52 - kFrac - static_cast<int>((bits >> 52) - 1023) - (i >> 6);   // 1 .. 54
        const u64 mant = (static_cast<u64>(bits) & 0xfffffffffffffull) | 0x10000000000000ull;
        return (mant + (1ull << (shift - 1))) >> shift;
    }

    template <typename F> __device__ __forceinline__ void each(F f) const {                      // all tokens of the block
        for (int i = threadIdx.x; i < n; i += kThreads) f(i, at(i));
    }

    // Sum over the block of one number a thread, and the sum before each warp's, in sh.warp_q; every thread gets the block's
    __device__ u64 block_sums(u64 v) {
        v = warp_sum(v);
        __syncthreads();
        if (lane == 0) sh.warp_q[warp] = v;
        __syncthreads();
        u64 total = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) total += sh.warp_q[w];
        return total;
    }

    // The token (index in the row) at which the sum of q(i, l) over the tokens of the row, in the order of the indices, first exceeds what `aim` makes
    // of the whole sum; `mine` is the warp's own sum.  Given to the one warp that holds it by `found(index, logit)`.
    template <typename Q, typename A, typename F> __device__ void locate(Q q, u64 mine, A aim, F found) {
        const u64 own = block_sums(mine);
        if (threadIdx.x == 0) sh.x_sum = own;
        cluster.sync();
        u64 before = 0, total = 0;
        for (int r = 0; r < blocks; ++r) {
            const u64 v = *cluster.map_shared_rank(&sh.x_sum, r);
            if (r < rank) before += v;
            total += v;
        }
        const u64 target = aim(total);
        for (int w = 0; w < warp; ++w) before += sh.warp_q[w];
        if (before <= target && target < before + sh.warp_q[warp]) {       // one warp of the cluster
            const int a = warp * seg, b = min(n, a + seg), sub = (b - a + 31) / 32;
            const int la = min(b, a + lane * sub), lb = min(b, la + sub);
            u64 s = 0;
            for (int i = la; i < lb; ++i) s += q(i, at(i));
            const u64 upto = before + warp_scan(s, lane);
            const int who = __ffs(__ballot_sync(0xffffffffu, upto > target)) - 1;
            before = __shfl_sync(0xffffffffu, upto - s, who);
            const int wa = min(b, a + who * sub), wb = min(b, wa + sub);
            for (int base = wa; base < wb; base += 32) {
                const int i = base + lane;
                const float l = i < wb ? at(i) : 0.f;
                const u64 v = i < wb ? q(i, l) : 0;
                const u64 through = before + warp_scan(v, lane);
                const unsigned hit = __ballot_sync(0xffffffffu, through > target);
                if (hit) {
                    if (lane == __ffs(hit) - 1) found(i, l);
                    break;
                }
                before = __shfl_sync(0xffffffffu, through, 31);
            }
        }
    }
    template <typename Q> __device__ __forceinline__ u64 warp_part(Q q) const {   // sum of q over the warp's own tokens
        u64 s = 0;
        const int a = warp * seg, b = min(n, a + seg);
        for (int i = a + lane; i < b; i += 32) s += q(i, at(i));
        return s;
    }

    __device__ void clear_bins() {
        for (int i = threadIdx.x; i < kBins; i += kThreads) { sh.count[i] = 0; sh.mass[i] = 0; }
        __syncthreads();
    }
    // Adds up all blocks' bins; finds the one in which the target falls (before < target <= before + bin).  With `fraction` the target is that
    // share of the whole.  False: the whole is less than the target.  Leaves the bin, what comes before it and its tokens in b_*.
    template <bool MASS> __device__ bool find_bin(double fraction, u64 base, u64& target) {
        __syncthreads();
        cluster.sync();
        constexpr int PER = kBins / kThreads;
        u64 q[PER];
        uint32_t cnt[PER];
        u64 s = 0;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            q[k] = 0;
            cnt[k] = 0;
            for (int r = 0; r < blocks; ++r) {
                const int bin = threadIdx.x * PER + k;
                cnt[k] += cluster.map_shared_rank(sh.count, r)[bin];
                if (MASS) q[k] += cluster.map_shared_rank(sh.mass, r)[bin];
            }
            if (!MASS) q[k] = cnt[k];
            s += q[k];
        }
        const u64 upto = warp_scan(s, lane);
        if (lane == 31) sh.warp_q[warp] = upto;
        __syncthreads();
        u64 before = base + upto - s, total = base;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += sh.warp_q[w];
            total += sh.warp_q[w];
        }
        if (fraction >= 0.) target = max(1ull, min(total, static_cast<u64>(ceil(fraction * static_cast<double>(total)))));
        const bool inside = total >= target;
        if (inside) {
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                if (before < target && target <= before + q[k]) { sh.b_bin = threadIdx.x * PER + k; sh.b_before = before; sh.b_count = cnt[k]; }
                before += q[k];
            }
        }
        __syncthreads();
        cluster.sync();                                            // nobody reads these bins any more
        return inside;
    }

    // Ranks the tokens for which `in` holds (at most kList in the cluster) against one another; sets the cut.
    template <bool MASS, typename In> __device__ void cut_in_list(In in, u64 base, u64 target) {
        if (threadIdx.x == 0) sh.x_listed = 0;
        __syncthreads();
        each([&](int i, float l) {
            if (in(i, l)) sh.list[min(atomicAdd(&sh.x_listed, 1u), static_cast<uint32_t>(kList - 1))] = pack(l, first + i);
        });
        __syncthreads();
        cluster.sync();
        int total = 0;
        for (int r = 0; r < blocks; ++r) {
            const int c = min(static_cast<int>(*cluster.map_shared_rank(&sh.x_listed, r)), kList - total);
            const u64* from = cluster.map_shared_rank(sh.list, r);
            for (int i = threadIdx.x; i < c; i += kThreads) {
                const u64 v = from[i];
                sh.all[total + i] = v;
                sh.all_q[total + i] = MASS ? weight(key_value(static_cast<uint32_t>(v >> 32))) : 1;
            }
            total += c;
        }
        __syncthreads();
        for (int i = rank * kWarps + warp; i < total; i += blocks * kWarps) {
            const u64 me = sh.all[i];
            u64 s = 0;
            for (int j = lane; j < total; j += 32)
                if (sh.all[j] > me) s += sh.all_q[j];
            s = base + warp_sum(s);
            if (s < target && target <= s + sh.all_q[i] && lane < blocks) *cluster.map_shared_rank(&sh.x_cut, lane) = me;
        }
        cluster.sync();
        cut = sh.x_cut;
    }

    // Keeps the tokens, in the order of falling logit, before which less than `target` has come: tokens, or mass (a share of the whole).  The bins of
    // the first division are in sh already.
    template <bool MASS> __device__ void find_cut(double fraction, u64 target) {
        if (!find_bin<MASS>(fraction, 0, target)) return;          // fewer tokens than that: all stay
        u64 base = sh.b_before;
        uint32_t bin = sh.b_bin, cnt = sh.b_count;
        const u64 old = cut;
        auto stays = [&](int i, float l) { return pack(l, first + i) >= old; };
        auto in_bin = [&](int i, float l) { return bin_of(l) == static_cast<int>(bin) && eligible(l) && stays(i, l); };
        if (cnt <= kList) return cut_in_list<MASS>(in_bin, base, target);
        // a crowded bin: divide the interval of its logits' keys
        if (threadIdx.x == 0) { sh.x_min = 0xffffffffu; sh.x_max = 0; }
        __syncthreads();
        uint32_t lo = 0xffffffffu, hi = 0;
        each([&](int i, float l) {
            if (in_bin(i, l)) { lo = min(lo, order_key(l)); hi = max(hi, order_key(l)); }
        });
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        if (lane == 0) { atomicMin(&sh.x_min, lo); atomicMax(&sh.x_max, hi); }
        __syncthreads();
        cluster.sync();
        lo = 0xffffffffu;
        hi = 0;
        for (int r = 0; r < blocks; ++r) {
            lo = min(lo, *cluster.map_shared_rank(&sh.x_min, r));
            hi = max(hi, *cluster.map_shared_rank(&sh.x_max, r));
        }
        while (lo < hi) {
            const int shift = max(0, 32 - __clz(hi - lo) - 10);
            auto within = [&](int i, float l) {
                const uint32_t k = order_key(l);
                return l == l && k >= lo && k <= hi && eligible(l) && stays(i, l);
            };
            clear_bins();
            each([&](int i, float l) {
                if (!within(i, l)) return;
                const uint32_t b = (hi - order_key(l)) >> shift;
                atomicAdd(&sh.count[b], 1u);
                if (MASS) atomicAdd(&sh.mass[b], weight(l));
            });
            find_bin<MASS>(-1., base, target);
            base = sh.b_before;
            bin = sh.b_bin;
            cnt = sh.b_count;
            const uint32_t top = hi - (bin << shift);
            lo = max(lo, top - min(top, (1u << shift) - 1));
            hi = top;
            if (cnt <= kList) {
                // (`within` reads lo and hi: the new interval)
                return cut_in_list<MASS>(within, base, target);
            }
        }
        // equal logits: the lowest indices, as many as it takes
        const uint32_t key = lo;
        const u64 one = MASS ? weight(key_value(key)) : 1, need = (target - base + one - 1) / one;
        auto same = [&](int i, float l) -> u64 { return l == l && order_key(l) == key && stays(i, l); };
        locate(same, warp_part(same), [&](u64) { return need - 1; }, [&](int i, float l) {
            for (int r = 0; r < blocks; ++r) *cluster.map_shared_rank(&sh.x_cut, r) = pack(l, first + i);
        });
        cluster.sync();
        cut = sh.x_cut;
    }
    __device__ __forceinline__ int bin_of(float l) const { return min(kBins - 1, static_cast<int>(-coarse(l) * (kBins / kRange))); }
};

template <typename T, bool RESIDENT>
__global__ void __launch_bounds__(kThreads) sample_tokens_kernel(SampleTokens p, int slice) {
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ Shared sh;
    Row<T, RESIDENT> row(sh);
    row.blocks = static_cast<int>(row.cluster.num_blocks());
    row.rank = static_cast<int>(row.cluster.block_rank());
    row.warp = threadIdx.x >> 5;
    row.lane = threadIdx.x & 31;
    const int b = blockIdx.x / row.blocks;
    row.first = row.rank * slice;
    row.n = max(0, min(p.V, row.first + slice) - row.first);
    row.seg = (row.n + kWarps - 1) / kWarps;
    const float temp = p.temperature ? p.temperature[b] : p.temperature_all;
    const int k = p.top_k ? p.top_k[b] : p.top_k_all;
    const float top_p = p.top_p ? p.top_p[b] : p.top_p_all, min_p = p.min_p ? p.min_p[b] : p.min_p_all, u = p.u[b];
    if (threadIdx.x < 64) sh.table[threadIdx.x] = exp2(threadIdx.x / 64.);

    // the row's part, and its largest logit (lowest index); shared memory keeps the offset from a 16-byte boundary
    const T* src = static_cast<const T*>(p.logits) + b * p.row_stride + row.first;
    constexpr int VE = 16 / sizeof(T);
    const int off = static_cast<int>((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));
    T* keep = reinterpret_cast<T*>(dyn) + off;
    row.x = RESIDENT ? keep : src;
    const int head = min(row.n, off ? VE - off : 0), nv = (row.n - head) / VE, tail = head + nv * VE;
    float best = -INFINITY;
    int best_i = -1;
    auto look = [&](int i, float l) {
        if (l > best) { best = l; best_i = i; }                    // a thread's tokens come in the order of their indices; NaN never wins
    };
    if (static_cast<int>(threadIdx.x) < head) {
        const T v = src[threadIdx.x];
        if (RESIDENT) keep[threadIdx.x] = v;
        look(threadIdx.x, to_f(v));
    }
    constexpr int DEPTH = 4;
    for (int base = threadIdx.x; base < nv; base += kThreads * DEPTH) {
        uint4 v[DEPTH];
#pragma unroll
        for (int d = 0; d < DEPTH; ++d)
            if (base + d * kThreads < nv) v[d] = __ldg(reinterpret_cast<const uint4*>(src + head) + base + d * kThreads);
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            const int i = base + d * kThreads;
            if (i >= nv) break;
            if (RESIDENT) reinterpret_cast<uint4*>(keep + head)[i] = v[d];
            const T* e = reinterpret_cast<const T*>(&v[d]);
#pragma unroll
            for (int j = 0; j < VE; ++j) look(head + i * VE + j, to_f(e[j]));
        }
    }
    if (tail + static_cast<int>(threadIdx.x) < row.n) {
        const int i = tail + threadIdx.x;
        const T v = src[i];
        if (RESIDENT) keep[i] = v;
        look(i, to_f(v));
    }
    u64 top = best_i >= 0 ? pack(best, row.first + best_i) : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (row.lane == 0) sh.warp_q[row.warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = max(top, sh.warp_q[w]);
    if (threadIdx.x == 0) sh.x_best = top;
    row.clear_bins();
    row.cluster.sync();
    for (int r = 0; r < row.blocks; ++r) top = max(top, *row.cluster.map_shared_rank(&sh.x_best, r));
    if (top == 0) {                                                // nothing above -inf: nothing to draw
        if (row.rank == 0 && threadIdx.x == 0) { p.token[b] = -1; p.logprob[b] = -INFINITY; }
        row.cluster.sync();
        return;
    }
    row.lmax = key_value(static_cast<uint32_t>(top >> 32));
    const int imax = static_cast<int>(0xffffffffu - static_cast<uint32_t>(top));
    const bool greedy = !(temp > 0.f), use_k = !greedy && k > 0 && k < p.V, use_p = !greedy && top_p < 1.f;
    row.to_log2 = greedy ? 0. : kLog2eD / static_cast<double>(temp);
    row.bin_scale = static_cast<float>(row.to_log2);
    row.least = !greedy && min_p > 0.f ? max(-45., log2(static_cast<double>(fminf(min_p, 1.f)))) : -45.;
    row.least_lo = static_cast<float>(row.least) * 1.0001f - 1e-6f;
    row.least_hi = static_cast<float>(row.least) * 0.9999f + 1e-6f;

    // the sum for the log-probability, and with it what the first cut (or the draw) needs
    float z = 0.f;
    auto add_z = [&](float l) { z += l == row.lmax ? 1.f : exp2f((l - row.lmax) * static_cast<float>(kLog2eD)); };
    u64 drawn = 0;
    auto kept_weight = [&](int i, float l) -> u64 { return row.eligible(l) && pack(l, row.first + i) >= row.cut ? row.weight(l) : 0; };
    if (greedy) {
        row.each([&](int, float l) { if (l == l) add_z(l); });
    } else if (!use_k && !use_p) {
        const int a = row.warp * row.seg, e = min(row.n, a + row.seg);
        for (int i = a + row.lane; i < e; i += 32) {
            const float l = row.at(i);
            if (l != l) continue;
            add_z(l);
            drawn += kept_weight(i, l);
        }
    } else {
        row.each([&](int, float l) {
            if (l != l) return;
            add_z(l);
            if (!row.eligible(l)) return;
            const int bin = row.bin_of(l);
            atomicAdd(&sh.count[bin], 1u);
            if (!use_k) atomicAdd(&sh.mass[bin], row.weight(l));
        });
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
    if (row.lane == 0) sh.warp_z[row.warp] = z;
    __syncthreads();
    if (threadIdx.x == 0) {
        float s = 0.f;
        for (int w = 0; w < kWarps; ++w) s += sh.warp_z[w];
        sh.x_z = s;
    }
    row.cluster.sync();
    z = 0.f;
    for (int r = 0; r < row.blocks; ++r) z += *row.cluster.map_shared_rank(&sh.x_z, r);

    if (greedy) {
        if (row.rank == 0 && threadIdx.x == 0) { p.token[b] = imax; p.logprob[b] = -logf(z); }
        row.cluster.sync();
        return;
    }
    if (use_k) row.template find_cut<false>(-1., static_cast<u64>(k));
    if (use_p) {
        if (use_k) {
            row.clear_bins();
            row.each([&](int i, float l) {
                if (l != l || !row.eligible(l) || pack(l, row.first + i) < row.cut) return;
                atomicAdd(&sh.count[row.bin_of(l)], 1u);
                atomicAdd(&sh.mass[row.bin_of(l)], row.weight(l));
            });
        }
        row.template find_cut<true>(fmaxf(top_p, 0.f), 0);
    }
    if (use_k || use_p) drawn = row.warp_part(kept_weight);
    row.locate(kept_weight, drawn,
               [&](u64 total) {
                   const double t = static_cast<double>(u > 0.f ? u : 0.f) * static_cast<double>(total);
                   return min(total - 1, static_cast<u64>(t));
               },
               [&](int i, float l) { p.token[b] = row.first + i; p.logprob[b] = (l == row.lmax ? 0.f : l - row.lmax) - logf(z); });
    row.cluster.sync();
}

template <typename T, bool RESIDENT>
const char* launch(const SampleTokens& p, int blocks, int slice, int smem, cudaStream_t s) {
    static std::atomic<uint64_t> raised{0};
    auto k = sample_tokens_kernel<T, RESIDENT>;
    if (RESIDENT && !raise_smem_limit(reinterpret_cast<const void*>(k), 200 * 1024, raised)) return "sample_tokens: the shared-memory limit could not be raised";
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = blocks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(p.B) * blocks);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaError_t e = cudaLaunchKernelEx(&cfg, k, p, slice); e != cudaSuccess) {
        cudaGetLastError();
        return cudaGetErrorString(e);
    }
    return nullptr;
}

template <typename T>
const char* launch_type(const SampleTokens& p, int num_sms, cudaStream_t s) {
    // Blocks a row: enough that two blocks fit an SM (80 KB of the row each), more of them while the rows alone would leave SMs idle.
    constexpr int64_t kFit = 80 * 1024, kMost = 190 * 1024;
    int blocks = 1;
    while (blocks < kMaxCluster && (static_cast<int64_t>(p.V) * sizeof(T) > kFit * blocks || (static_cast<int64_t>(p.B) * blocks * 2 <= num_sms && p.V > 2048 * blocks))) blocks *= 2;
    const int slice = ((p.V + blocks - 1) / blocks + 15) / 16 * 16;
    const int64_t bytes = static_cast<int64_t>(slice) * sizeof(T) + 16;
    if (bytes <= kMost) return launch<T, true>(p, blocks, slice, static_cast<int>(bytes), s);
    return launch<T, false>(p, blocks, slice, 0, s);               // a vocabulary beyond 8 x 190 KB is read again in every pass
}

}  // namespace

const char* sample_tokens(const SampleTokens& p, int num_sms, cudaStream_t s) {
    if (p.B <= 0) return nullptr;
    if (p.type == 0) return launch_type<__nv_bfloat16>(p, num_sms, s);
    if (p.type == 1) return launch_type<__half>(p, num_sms, s);
    return launch_type<float>(p, num_sms, s);
}

}  // namespace sg
