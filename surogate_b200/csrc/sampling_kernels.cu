// Drawing the next token of each row from its logits, with temperature, top-k, top-p and min-p, by one given uniform number.
//
//   w_i = e^{(l_i - max) / T}; kept: the tokens in the order of falling logit (equal ones: rising index) while fewer than k come before, w >= min_p,
//   and the mass before is below top_p times the mass of what the other two leave; token: the first, in the order of the indices, at which
//   the kept mass exceeds u times the whole.  T = 0: the largest logit's lowest index.  logprob = l_token - log sum e^l, without filters.
//
// A row is read from HBM once, and that (size of a logit * vocabulary) is its floor.  A cluster of 1 to 8 blocks holds the row in its shared
// memory; the passes over it (maximum; sums; the candidates) stay on the chip, and the blocks exchange a few words after each.
//
// * The result is a token, not a number that may be a little off, so masses are integers: weights as multiples of 2^-44 of the largest one
//   (exponentials in fp64 by a table of 2^(j/64) and three terms of the series: relative error below 2^-34), whose sums do not depend on the order.
//   A wrong token takes a u within that of a boundary.
// * Cuts need no sort.  Bounds leave a few candidates: the k largest logits are not below the k-th of the threads' own maxima.  Up to 512 candidates
//   are ranked against one another by one block.  More (large k) are counted, with their mass, in 1024 bins over the logits; the bin in which
//   the cut falls is found by a scan and only its tokens are ranked; a bin with too many is divided again, equal logits are counted by index.
// * Top-p alone, where flat rows leave tens of thousands of candidates, estimates masses first and proves the cut after (estimated_cut).
//
// Measured in graphs (B200; fp32, vocabulary 151 936, 608 KB a row; one row, then 256 rows, which a copy would read in 24 us): greedy 7 and 69 us; T 1
// without filters 14 and 128; top-k 40 14 and 117; top-p 0.9 28 and 290; min-p 0.05 12 and 103; T 0.7, top-k 20, top-p 0.8, min-p 0.01 12 and 111.  One row is
// latency: launch, loading, four or five exchanges in the cluster.  Many rows are bound by instructions (the fp64 weights, one to two passes) and by the
// exchanges, with two blocks an SM to fill each other's pauses.  Bf16, 64 rows of 128 256: 23 us without filters, 49 with top-p.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>
#include <utility>

#include "launch_limits.h"
#include "sampling.h"

namespace cg = cooperative_groups;

namespace sg {

namespace {

using u64 = unsigned long long;
constexpr int kThreads = 512, kWarps = kThreads / 32, kBins = 1024, kList = 512, kMaxCluster = 8;
constexpr int kOwn = 64;                      // candidates a warp can note down
constexpr int kFrac = 44;                     // weights are multiples of 2^-44
constexpr float kRange = 46.f;                // minus log2 of the smallest weight that is looked at: what lies below is 0 as a multiple
constexpr int kTable = 64, kCopies = 16;      // 2^(j / 64), a copy for each of 16 lanes so that none meet in a bank
constexpr int kMost = 190 * 1024;             // bytes of a row that a block holds at most, beside 34 KB of its own
constexpr float kLowest = -3.402823466e38f;
constexpr double kLog2eD = 1.4426950408889634074, kLn2D = 0.69314718055994530942;

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
    double table[kTable * kCopies];
    union {
        struct { alignas(16) uint32_t mass[2 * kBins]; uint32_t count[kBins]; };   // (a mass: lower word, upper word)
        struct { u64 list[kList], all[kList], all_q[kList]; };   // a block's candidates for a cut, and all blocks'
        alignas(16) uint32_t estimate[4 * kBins];
    };
    float own_l[kWarps * kOwn];       // the warps' candidates: logit, place
    int own_i[kWarps * kOwn];
    u64 warp_q[kWarps];
    float warp_z[kWarps];
    uint32_t warp_top[kWarps], warp_at[kWarps];
    int warp_n[kWarps];               // candidates of each warp
    // what other blocks of the cluster read
    u64 x_sum, x_cut, x_bins, x_above;
    float x_z;
    int x_first;                      // index of place 0
    uint32_t x_best, x_index, x_kth, x_min, x_max, x_listed, x_noted;
    // the bin found, told to all blocks
    u64 b_before;
    uint32_t b_bin, b_last;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// e^s for s <= 0, to 2^-22 (the exponential's own error: the rounding of s log2(e) is put right); 0 below -150, and for NaN
__device__ __forceinline__ float exp_below(float s) {
    constexpr float k2e = static_cast<float>(kLog2eD), ln2 = static_cast<float>(kLn2D);
    s = fmaxf(s, -150.f);
    const float t = __fmul_rn(s, k2e), left = fmaf(s, k2e, -t);
    const float r = ex2(t);
    return fmaf(r, left * ln2, r);
}
__device__ __forceinline__ float min_or_nan(float a, float b) {
    float y;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// 16 bytes of logits as fp32
template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void get(const uint4& v, float (&f)[4]) {
        f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
    }
};
template <> struct Vec<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void get(const uint4& v, float (&f)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    }
};
template <> struct Vec<__half> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void get(const uint4& v, float (&f)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w[i])); f[2 * i] = x.x; f[2 * i + 1] = x.y; }
    }
};

// One block's part of a row.  Places count its logits from the 16-byte boundary at or before its first one; places that hold none read as -inf.
template <typename T, bool RESIDENT>
struct Row {
    static constexpr int N = Vec<T>::N;
    cg::cluster_group cluster = cg::this_cluster();
    Shared& sh;
    const uint4* x;                   // the boundary: in shared memory, or where the row lies
    int off, end, nvec, seg;          // places [off, end) hold logits; vectors; vectors a warp
    int first;                        // index of place 0
    int blocks, rank, warp, lane;
    float lmax;
    double to_log2;                   // log2(e) / T
    bool steep;                       // weights need care: very low or high temperatures, infinite logits
    double least;                     // log2 of the smallest weight that min-p lets stay
    bool by_min_p;
    float bin_scale;
    float floor_l;                    // what is not below this is looked at
    // The candidates have been noted down: passes run over them.  Each warp's own, list_step apart.
    bool listed = false;
    const float* list_l;
    const int* list_i;
    int list_step, list_all;          // (list_all: how many, if they lie one behind the other)
    bool alone = false;               // one block goes on with all of them, the others have left
    u64 cut = 0;                      // kept: pack() >= cut

    __device__ Row(Shared& s) : sh(s) {}

    __device__ __forceinline__ int list_n(int w) const { return alone ? max(0, min(list_step, list_all - w * list_step)) : sh.warp_n[w]; }
    __device__ __forceinline__ void sync() const {
        if (alone) __syncthreads();
        else cluster.sync();
    }

    // the vector `v` in global memory: whole where all of it belongs to the row's part
    __device__ __forceinline__ uint4 from_global(const uint4* base, int v) const {
        if (v * N >= off && v * N + N <= end) return __ldg(base + v);
        alignas(16) T e[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int i = v * N + j;
            e[j] = i >= off && i < end ? reinterpret_cast<const T*>(base)[i] : static_cast<T>(-INFINITY);
        }
        return *reinterpret_cast<const uint4*>(e);
    }
    __device__ __forceinline__ uint4 vec(int v) const { return RESIDENT ? x[v] : from_global(x, v); }

    __device__ __forceinline__ double log2_weight(float l) const { return l == lmax ? 0. : (static_cast<double>(l) - static_cast<double>(lmax)) * to_log2; }
    // Coarse log2 of a weight in fp32: never increases as l falls
    __device__ __forceinline__ float coarse(float l) const { return l == lmax ? 0.f : (l - lmax) * bin_scale; }
    __device__ __forceinline__ int bin_of(float l) const { return static_cast<int>(fminf(fmaxf(-coarse(l) * (kBins / kRange), 0.f), kBins - 1.f)); }
    __device__ __forceinline__ bool eligible(float l) const { return !by_min_p || log2_weight(l) >= least; }
    // A logit that surely is not above one with this log2 of its weight
    __device__ __forceinline__ float logit_below(double log2_w) const {
        const double l = static_cast<double>(lmax) + log2_w * 1.000001 / to_log2;
        return fmaxf(__double2float_rd(l - fabs(l) * 1e-6), kLowest);        // (-inf never counts; NaN, from infinities: the lowest number)
    }
    // and one that surely is not below
    __device__ __forceinline__ float logit_above(double log2_w) const {
        const double l = static_cast<double>(lmax) + log2_w * 0.999999 / to_log2;
        return __double2float_ru(l + fabs(l) * 1e-6);
    }
    // 2^log2_weight as a multiple of 2^-44 plus kBias, for logits that are not below the lowest floor (whose own is 0): t = i / 64 + r, 2^r by its series
    // to the third power (|r| <= 2^-7: 3e-11).  Adding 256 to it as an fp64 leaves the multiple in the lowest bits.
    static constexpr u64 kBias = 0x4070000000000000ull;
    __device__ __forceinline__ u64 biased_weight(float l) const {
        const double d = static_cast<double>(l) - static_cast<double>(lmax);
        const double big = 6755399441055744. / kTable;            // 1.5 * 2^52 / 64: adding it rounds to multiples of 1 / 64
        const double m = fma(d, to_log2, big);
        const int i = __double2loint(m);
        const double r = fma(d, to_log2, big - m);
        const double e = sh.table[(i & (kTable - 1)) * kCopies + (lane & (kCopies - 1))];
        const double y = fma(r, fma(r, kLn2D * kLn2D * kLn2D / 6, kLn2D * kLn2D / 2), kLn2D);
        const double v = fma(e * r, y, e);
        const double w = __hiloint2double(__double2hiint(v) + (i & -kTable) * ((1 << 20) / kTable), __double2loint(v));
        return static_cast<u64>(__double_as_longlong(w + 256.));
    }
    __device__ __forceinline__ u64 fast_weight(float l) const { return biased_weight(l) - kBias; }
    __device__ __forceinline__ u64 weight(float l) const {
        if (steep) {
            if (l == lmax) return 1ull << kFrac;
            if (!((static_cast<double>(l) - static_cast<double>(lmax)) * to_log2 >= -60.)) return 0;
        }
        return fast_weight(l);
    }
    // weights of a vector's logits, 0 below `least_l` (which is not below the lowest floor): side by side, without a branch for each
    __device__ __forceinline__ void weights(const float (&l)[N], float least_l, u64 (&w)[N]) const {
        if (!steep) {
#pragma unroll
            for (int j = 0; j < N; ++j) w[j] = fast_weight(fmaxf(l[j], least_l));
#pragma unroll
            for (int j = 0; j < N; ++j) w[j] = l[j] >= least_l ? w[j] : 0;
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) w[j] = l[j] >= least_l ? weight(l[j]) : 0;
        }
    }
    // A word of each block of the cluster: lane r has that of block r, the lanes behind the last block zero
    template <typename V> __device__ __forceinline__ V of_rank(V* own) const { return lane < blocks ? *cluster.map_shared_rank(own, lane) : V{}; }
    __device__ __forceinline__ u64 sum_ranks(u64 v) const {
#pragma unroll
        for (int o = 1; o < kMaxCluster; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return __shfl_sync(0xffffffffu, v, 0);
    }

    // f(place, logit, weight if WEIGH) for the tokens that are not below floor_l, each warp its own in the order of their indices, lanes apart
    template <bool WEIGH, typename F> __device__ __forceinline__ void each(F f) const {
        if (listed) {
            const int n = list_n(warp), at = warp * list_step;
            for (int i = lane; i < n; i += 32) {
                const float l = list_l[at + i];
                if (l >= floor_l) f(list_i[at + i], l, WEIGH ? weight(l) : 0);
            }
            return;
        }
        const int b = min(nvec, (warp + 1) * seg);
        for (int v = warp * seg + lane; v < b; v += 32) {
            float l[N], most;
            Vec<T>::get(vec(v), l);
            most = l[0];
#pragma unroll
            for (int j = 1; j < N; ++j) most = fmaxf(most, l[j]);
            if (!(most >= floor_l)) continue;
            u64 w[N];
            if (WEIGH) weights(l, floor_l, w);
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (l[j] >= floor_l) f(v * N + j, l[j], WEIGH ? w[j] : 0);
        }
    }
    __device__ __forceinline__ u64 order(int place, float l) const { return pack(l, first + place); }

    // Not below the cut, whose logit is floor_l once there is one
    __device__ __forceinline__ bool stays(int place, float l) const { return l > floor_l || cut == 0 || order(place, l) >= cut; }
    __device__ __forceinline__ bool kept(int place, float l) const { return eligible(l) && stays(place, l); }

    // Sum over the block of one number a lane (a thread's share), the warps' own sums in sh.warp_q; every thread gets the block's
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
    // The thread of the block in whose share the running sum first exceeds `target`: given the sum before its share by hit(before)
    template <typename F> __device__ void block_find(u64 v, u64 target, F hit) {
        const u64 upto = warp_scan(v, lane);
        __syncthreads();
        if (lane == 31) sh.warp_q[warp] = upto;
        __syncthreads();
        u64 before = upto - v;
        for (int w = 0; w < warp; ++w) before += sh.warp_q[w];
        if (before <= target && target < before + v) hit(before);
    }

    // The token at which the sum of q(place, logit) over the tokens of the row, in the order of the indices, first exceeds what `aim` makes of
    // the whole sum; `mine` is this lane's part of its warp's sum.  One thread of the cluster gets it by found(place, logit).
    template <typename Q, typename A, typename F> __device__ void locate(Q q, u64 mine, A aim, F found) {
        const u64 own = block_sums(mine);
        if (threadIdx.x == 0) sh.x_sum = own;
        sync();
        locate_in(q, of_rank(&sh.x_sum), own, aim, found);
    }
    // the same, with the blocks' sums known: lane r has that of block r; the warps' are in sh.warp_q
    template <typename Q, typename A, typename F> __device__ void locate_in(Q q, u64 of_blocks, u64 own, A aim, F found) {
        u64 target = aim(sum_ranks(of_blocks));
        const u64 before = __shfl_sync(0xffffffffu, warp_scan(of_blocks, lane) - of_blocks, rank);
        if (target < before || target >= before + own) return;            // another block's
        target -= before;
        int w = 0;
        while (target >= sh.warp_q[w]) target -= sh.warp_q[w++];            // the warp's tokens, over the whole block
        const int a = w * seg, m = listed ? list_n(w) : min(nvec, a + seg) - a, per = (m + kThreads - 1) / kThreads;   // entries, or vectors
        const int va = min(m, static_cast<int>(threadIdx.x) * per), vb = min(m, va + per);
        auto share = [&](auto f) {
            if (listed) {
                for (int v = va; v < vb; ++v)
                    if (list_l[w * list_step + v] >= floor_l) f(list_i[w * list_step + v], list_l[w * list_step + v]);
                return;
            }
            for (int v = a + va; v < a + vb; ++v) {
                float l[N];
                Vec<T>::get(vec(v), l);
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (l[j] >= floor_l) f(v * N + j, l[j]);
            }
        };
        u64 s = 0;
        share([&](int i, float l) { s += q(i, l); });
        block_find(s, target, [&](u64 upto) {
            bool done = false;
            share([&](int i, float l) {
                upto += q(i, l);
                if (!done && upto > target) { done = true; found(i, l); }
            });
        });
    }

    // Notes down the candidates; true if all warps of the cluster have room for theirs.  `total`: all of them.
    __device__ bool note_down(int& total) {
        int n = 0;
        const int b = min(nvec, (warp + 1) * seg);
        for (int base = warp * seg; base < b && n <= kOwn; base += 32) {
            float l[N], most = -INFINITY;
            if (base + lane < b) {
                Vec<T>::get(vec(base + lane), l);
#pragma unroll
                for (int j = 0; j < N; ++j) most = fmaxf(most, l[j]);
            }
            if (!__any_sync(0xffffffffu, most >= floor_l)) continue;
            const bool some = most >= floor_l;
            int at = n, mine = 0;                                  // before this lane's: all of the lanes before it
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const bool in = some && l[j] >= floor_l;
                const unsigned all = __ballot_sync(0xffffffffu, in);
                at += __popc(all & ((1u << lane) - 1));
                n += __popc(all);
                mine |= in << j;
            }
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (mine >> j & 1) {
                    if (at < kOwn) { sh.own_l[warp * kOwn + at] = l[j]; sh.own_i[warp * kOwn + at] = (base + lane) * N + j; }
                    ++at;
                }
        }
        if (lane == 0) sh.warp_n[warp] = n;
        __syncthreads();
        if (warp == 0) {
            const int c = lane < kWarps ? sh.warp_n[lane] : 0;
            const uint32_t sum = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(min(c, kOwn)));
            if (lane == 0) sh.x_noted = sum;
            if (__any_sync(0xffffffffu, c > kOwn) && lane == 0) sh.x_noted = 0x10000000u;
        }
        sync();
        const u64 sum = sum_ranks(of_rank(&sh.x_noted));
        total = static_cast<int>(min(sum, u64{0x10000000u}));
        return sum < 0x10000000u;
    }

    __device__ void clear_bins() {
        for (int i = threadIdx.x; i < kBins; i += kThreads) sh.count[i] = sh.mass[2 * i] = sh.mass[2 * i + 1] = 0;
        __syncthreads();
    }
    // 64-bit sums of two words each, so that a native 32-bit atomic does it
    __device__ __forceinline__ void add_mass(int bin, u64 w) {
        const uint32_t lo = static_cast<uint32_t>(w), old = atomicAdd(&sh.mass[2 * bin], lo);
        const uint32_t hi = static_cast<uint32_t>(w >> 32) + (old + lo < old);
        if (hi) atomicAdd(&sh.mass[2 * bin + 1], hi);
    }
    // Adds up all blocks' bins; finds the one in which the target falls (before < target <= before + bin).  With `fraction` the target is that
    // share of the whole.  False: the whole is less than the target.  Leaves the bin and what comes before it in b_*.
    template <bool MASS> __device__ bool find_bin(double fraction, u64 base, u64& target) {
        __syncthreads();
        sync();
        // A block adds up its share of the bins (words of other blocks are slow to get, so each is fetched once); their sums are exchanged, and the
        // block in whose share the target falls tells the others the bin.
        constexpr int PER = kBins / kThreads;                      // (at one block a row; with more of them some threads have none)
        const int share = kBins / blocks, bin = rank * share + threadIdx.x * PER;
        u64 q[PER], mine = 0;
#pragma unroll
        for (int k = 0; k < PER; ++k) q[k] = 0;
        if (static_cast<int>(threadIdx.x) * PER < share) {
#pragma unroll
            for (int r = 0; r < kMaxCluster; ++r) {
                if (r >= blocks) break;
                const Shared* from = cluster.map_shared_rank(&sh, r);
                static_assert(PER == 2, "two bins are fetched at once");
                if (MASS) {
                    const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(from->mass + 2 * bin);
                    q[0] += two.x;
                    q[1] += two.y;
                } else {
                    const uint2 two = *reinterpret_cast<const uint2*>(from->count + bin);
                    q[0] += two.x;
                    q[1] += two.y;
                }
            }
#pragma unroll
            for (int k = 0; k < PER; ++k) mine += q[k];
        }
        const u64 upto = warp_scan(mine, lane);
        if (lane == 31) sh.warp_q[warp] = upto;
        __syncthreads();
        u64 before = upto - mine, own = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += sh.warp_q[w];
            own += sh.warp_q[w];
        }
        if (threadIdx.x == 0) sh.x_bins = own;
        sync();
        const u64 of_blocks = of_rank(&sh.x_bins), total = base + sum_ranks(of_blocks);
        if (fraction >= 0.) target = share_of(fraction, total);
        if (total < target) return false;                          // (the same in all blocks)
        before += base + __shfl_sync(0xffffffffu, warp_scan(of_blocks, lane) - of_blocks, rank);
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            if (before < target && target <= before + q[k]) {
                for (int r = 0; r < blocks; ++r) {
                    Shared* to = cluster.map_shared_rank(&sh, r);
                    to->b_bin = bin + k;
                    to->b_before = before;
                }
            }
            before += q[k];
        }
        sync();                                            // b_* is there, and nobody reads these bins any more
        return true;
    }
    // The least mass that a prefix must reach to be `fraction` of the whole
    static __device__ __forceinline__ u64 share_of(double fraction, u64 total) {
        return max(1ull, min(total, static_cast<u64>(ceil(fraction * static_cast<double>(total)))));
    }

    // Ranks the tokens for which `in` holds against one another and sets the cut, if they are at most kList in the cluster.
    template <bool MASS, typename In> __device__ bool cut_in_list(In in, u64 base, u64 target) {
        if (threadIdx.x == 0) sh.x_listed = 0;                     // (the bins are done with: the lists take their place)
        __syncthreads();
        each<false>([&](int i, float l, u64) {
            if (!in(i, l)) return;
            const uint32_t at = atomicAdd(&sh.x_listed, 1u);
            if (at < kList) sh.list[at] = order(i, l);
        });
        __syncthreads();
        sync();
        return rank_lists<MASS>(base, target);
    }
    // the same with the tokens in the blocks' lists (and known to be there)
    template <bool MASS> __device__ bool rank_lists(u64 base, u64 target) {
        const uint32_t of_block = of_rank(&sh.x_listed), total = static_cast<uint32_t>(sum_ranks(of_block));
        const bool fits = total <= kList;
        if (fits) {                                                // all lists come to each block, whose warps take every blocks-th token
            const uint32_t upto = static_cast<uint32_t>(warp_scan(of_block, lane));
            int r = 0;
            uint32_t first_of = 0;
#pragma unroll
            for (int x = 0; x < kMaxCluster - 1; ++x) {
                const uint32_t y = __shfl_sync(0xffffffffu, upto, x);
                if (threadIdx.x >= y && x + 1 < blocks) { r = x + 1; first_of = y; }
            }
            if (threadIdx.x < total) {
                const u64 v = cluster.map_shared_rank(sh.list, r)[threadIdx.x - first_of];
                sh.all[threadIdx.x] = v;
                sh.all_q[threadIdx.x] = MASS ? weight(key_value(static_cast<uint32_t>(v >> 32))) : 1;
            }
            __syncthreads();
            for (uint32_t i = warp * blocks + rank; i < total; i += kWarps * blocks) {
                const u64 me = sh.all[i];
                u64 s = 0;
                for (uint32_t j = lane; j < total; j += 32)
                    if (sh.all[j] > me) s += sh.all_q[j];
                s = base + warp_sum(s);
                if (s < target && target <= s + sh.all_q[i] && lane < blocks) *cluster.map_shared_rank(&sh.x_cut, lane) = me;
            }
        }
        sync();
        if (fits) set_cut(sh.x_cut);
        return fits;
    }

    // The cut of top-p where it is thought to be: lists the tokens in [lower, upper], and adds up exactly what lies above and the whole.  Which proves the
    // cut, or refuses it (not there, or too many tokens: false; the whole is known then, and nothing else).  `above`: this lane's part of its
    // warp's kept mass.
    __device__ bool proved_cut(double share, float lower, float upper, u64& above, u64& whole) {
        u64 mass = 0;
        above = 0;
        __syncthreads();
        if (threadIdx.x == 0) { sh.x_listed = 0; sh.x_cut = 0; }
        __syncthreads();
        const int e = min(nvec, (warp + 1) * seg);
        for (int v = warp * seg + lane; v < e; v += 32) {
            float l[N], most;
            Vec<T>::get(vec(v), l);
            most = l[0];
#pragma unroll
            for (int j = 1; j < N; ++j) most = fmaxf(most, l[j]);
            if (!(most >= floor_l)) continue;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const u64 w = fast_weight(fmaxf(l[j], floor_l));
                mass += w;
                if (l[j] > upper) above += w;
            }
            if (!(most >= lower)) continue;
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (l[j] >= lower && l[j] <= upper) {
                    const uint32_t at = atomicAdd(&sh.x_listed, 1u);
                    if (at < kList) sh.list[at] = order(v * N + j, l[j]);
                }
        }
        const u64 own_mass = block_sums(mass), own_above = block_sums(above);
        if (threadIdx.x == 0) { sh.x_sum = own_mass; sh.x_above = own_above; }
        __syncthreads();
        cluster.sync();
        whole = sum_ranks(of_rank(&sh.x_sum));
        const u64 base = sum_ranks(of_rank(&sh.x_above)), target = share_of(share, whole);
        if (base >= target || !rank_lists<true>(base, target) || cut == 0) return false;   // (the same in all blocks)
        const int listed_here = static_cast<int>(sh.x_listed);
        for (int i = lane; i < listed_here; i += 32) {
            const u64 token = sh.list[i];
            const int place = static_cast<int>(0xffffffffu - static_cast<uint32_t>(token)) - first;
            if (token >= cut && place / N / seg == warp) above += weight(key_value(static_cast<uint32_t>(token >> 32)));
        }
        return true;
    }

    // The cut of top-p, from an estimate of the masses: weights in fp32 and in units of 2^-14 of their bin's heaviest, added up in bins over the logits, with
    // native 32-bit atomics.  Tokens lighter than (1 - share) / vocabulary of the whole need no bin and only count in the whole, which `z` is at T = 1 and
    // not below z at higher ones.  A mass estimated so
    // is off by less than 2^-14 of itself, so the cut lies within 2^-13 of the share.
    __device__ bool estimated_cut(double share, int vocabulary, float z, float temp, u64& above, u64& whole) {
        constexpr int UNIT = 14;                                   // (sums stay below 2^32: a block has at most 2^17 tokens, V / 8, of 2^14)
        const int bins = blocks == 1 ? 2 * kBins : 4 * kBins;
        const float depth = fminf(kRange, fmaxf(static_cast<float>(log2(vocabulary / ((1. - share) * (temp >= 1.f ? z : 1.f)))), 0.f) + 0.1f), scale = bins / depth, inv_scale = depth / bins;
        for (int i = threadIdx.x; i < bins; i += kThreads) sh.estimate[i] = 0;
        if (threadIdx.x == 0) sh.b_bin = sh.b_last = 0xffffffffu;
        __syncthreads();
        const bool count_light = temp != 1.f;
        const float deepest = count_light ? floor_l : fmaxf(floor_l, logit_below(-depth));
        float light = 0.f;
        const int e = min(nvec, (warp + 1) * seg);
        for (int v = warp * seg + lane; v < e; v += 32) {
            float l[N], most;
            Vec<T>::get(vec(v), l);
            most = l[0];
#pragma unroll
            for (int j = 1; j < N; ++j) most = fmaxf(most, l[j]);
            if (!(most >= deepest)) continue;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if (!(l[j] >= deepest)) continue;
                const float c = coarse(l[j]), at = -c * scale;
                if (at < bins) {
                    const int bin = static_cast<int>(at);
                    atomicAdd(&sh.estimate[bin], __float2uint_rn(ex2(UNIT - (at - bin) * inv_scale)));
                } else if (count_light) {
                    light += ex2(c);
                }
            }
        }
        if (count_light) {
            const u64 own_light = block_sums(static_cast<u64>(light * 0x1p32f));   // (estimates are multiples of 2^-32)
            if (threadIdx.x == 0) sh.x_sum = own_light;
        }
        __syncthreads();
        cluster.sync();
        constexpr int PER = 4;
        const int part = bins / blocks, bin = rank * part + threadIdx.x * PER;
        u64 q[PER], mine = 0;
#pragma unroll
        for (int k = 0; k < PER; ++k) q[k] = 0;
        if (static_cast<int>(threadIdx.x) * PER < part) {
#pragma unroll
            for (int r = 0; r < kMaxCluster; ++r) {
                if (r >= blocks) break;
                const uint4 four = *reinterpret_cast<const uint4*>(cluster.map_shared_rank(sh.estimate, r) + bin);
                q[0] += four.x; q[1] += four.y; q[2] += four.z; q[3] += four.w;
            }
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                q[k] = static_cast<u64>(static_cast<double>(q[k]) * static_cast<double>(ex2(32 - UNIT - (bin + k) * inv_scale)));
                mine += q[k];
            }
        }
        const u64 upto = warp_scan(mine, lane);
        __syncthreads();
        if (lane == 31) sh.warp_q[warp] = upto;
        __syncthreads();
        u64 before = upto - mine, own = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += sh.warp_q[w];
            own += sh.warp_q[w];
        }
        if (threadIdx.x == 0) sh.x_bins = own;
        cluster.sync();
        const u64 of_blocks = of_rank(&sh.x_bins);
        const double aim = share * (count_light ? static_cast<double>(sum_ranks(of_blocks) + sum_ranks(of_rank(&sh.x_sum))) : static_cast<double>(z) * 0x1p32);
        const u64 from = max(1ull, static_cast<u64>(aim * (1. - 0x1p-13))), to = max(1ull, static_cast<u64>(aim * (1. + 0x1p-13)));
        before += __shfl_sync(0xffffffffu, warp_scan(of_blocks, lane) - of_blocks, rank);
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const u64 after = before + q[k];
            if (before < from && from <= after)
                for (int r = 0; r < blocks; ++r) cluster.map_shared_rank(&sh, r)->b_bin = bin + k;
            if (before < to && to <= after)
                for (int r = 0; r < blocks; ++r) cluster.map_shared_rank(&sh, r)->b_last = bin + k;
            before = after;
        }
        cluster.sync();
        const uint32_t bin_a = sh.b_bin, bin_b = min(sh.b_last, static_cast<uint32_t>(bins) - 1);   // (none: behind all bins)
        const float upper = bin_a == 0 ? INFINITY : bin_a < static_cast<uint32_t>(bins) ? logit_above(-(bin_a - 0.001) * inv_scale) : kLowest;
        return proved_cut(share, fmaxf(floor_l, logit_below(-(bin_b + 1.001) * inv_scale)), upper, above, whole);
    }
    __device__ __forceinline__ void set_cut(u64 c) {
        cut = c;
        floor_l = fmaxf(floor_l, key_value(static_cast<uint32_t>(c >> 32)));
    }

    // Keeps the tokens, in the order of falling logit, before which less than `target` has come: tokens, or mass (a share of the whole).
    template <bool MASS> __device__ void find_cut(double fraction, u64 target) {
        clear_bins();
        each<MASS>([&](int i, float l, u64 w) {
            if (!kept(i, l)) return;
            if (MASS) add_mass(bin_of(l), w);
            else atomicAdd(&sh.count[bin_of(l)], 1u);
        });
        if (!find_bin<MASS>(fraction, 0, target)) return;          // fewer tokens than that: all stay
        u64 base = sh.b_before;
        uint32_t bin = sh.b_bin;
        // (What lies below the bin is out, and is not looked at any more.)
        const float upper = bin ? logit_above(-(bin - 0.001) * (kRange / kBins)) : INFINITY;
        auto in_bin = [&](int i, float l) { return l <= upper && bin_of(l) == static_cast<int>(bin) && kept(i, l); };
        floor_l = fmaxf(floor_l, logit_below(-(bin + 1.001) * (kRange / kBins)));
        if (cut_in_list<MASS>(in_bin, base, target)) return;
        // a crowded bin: divide the interval of its logits' keys
        if (threadIdx.x == 0) { sh.x_min = 0xffffffffu; sh.x_max = 0; }
        __syncthreads();
        uint32_t lo = 0xffffffffu, hi = 0;
        each<false>([&](int i, float l, u64) {
            if (in_bin(i, l)) { lo = min(lo, order_key(l)); hi = max(hi, order_key(l)); }
        });
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        if (lane == 0) { atomicMin(&sh.x_min, lo); atomicMax(&sh.x_max, hi); }
        __syncthreads();
        sync();
        lo = __reduce_min_sync(0xffffffffu, lane < blocks ? *cluster.map_shared_rank(&sh.x_min, lane) : 0xffffffffu);
        hi = __reduce_max_sync(0xffffffffu, of_rank(&sh.x_max));
        auto within = [&](int i, float l) {
            const uint32_t k = order_key(l);
            return k >= lo && k <= hi && kept(i, l);
        };
        while (lo < hi) {
            const int shift = max(0, 32 - __clz(hi - lo) - 10);
            clear_bins();
            each<MASS>([&](int i, float l, u64 w) {
                if (!within(i, l)) return;
                const uint32_t b = (hi - order_key(l)) >> shift;
                if (MASS) add_mass(b, w);
                else atomicAdd(&sh.count[b], 1u);
            });
            find_bin<MASS>(-1., base, target);
            base = sh.b_before;
            bin = sh.b_bin;
            const uint32_t top = hi - (bin << shift);
            lo = max(lo, top - min(top, (1u << shift) - 1));
            hi = top;
            if (cut_in_list<MASS>(within, base, target)) return;
        }
        // equal logits: the lowest indices, as many as it takes
        const uint32_t key = lo;
        const u64 one = MASS ? weight(key_value(key)) : 1, need = (target - base + one - 1) / one;
        auto same = [&](int i, float l) -> u64 { return order_key(l) == key && stays(i, l); };
        u64 mine = 0;
        each<false>([&](int i, float l, u64) { mine += same(i, l); });
        locate(same, mine, [&](u64) { return need - 1; }, [&](int i, float l) {
            for (int r = 0; r < blocks; ++r) *cluster.map_shared_rank(&sh.x_cut, r) = order(i, l);
        });
        sync();
        set_cut(sh.x_cut);
    }
};

template <typename T, bool RESIDENT>
__global__ void __launch_bounds__(kThreads, 2) sample_tokens_kernel(SampleTokens p, int slice, int ahead) {
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ Shared sh;
    Row<T, RESIDENT> row(sh);
    constexpr int N = Vec<T>::N;
    row.blocks = static_cast<int>(row.cluster.num_blocks());
    row.rank = static_cast<int>(row.cluster.block_rank());
    row.warp = threadIdx.x >> 5;
    row.lane = threadIdx.x & 31;
    const int b = blockIdx.x / row.blocks, begin = row.rank * slice;
    const T* src = static_cast<const T*>(p.logits) + b * p.row_stride + begin;
    row.off = static_cast<int>((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));
    row.end = row.off + max(0, min(p.V - begin, slice));
    row.first = begin - row.off;
    row.nvec = (row.end + N - 1) / N;
    row.seg = (row.nvec + kWarps - 1) / kWarps;
    const uint4* gx = reinterpret_cast<const uint4*>(src - row.off);
    row.x = RESIDENT ? reinterpret_cast<const uint4*>(dyn) : gx;

    const float temp = p.temperature ? p.temperature[b] : p.temperature_all;
    const int k = p.top_k ? p.top_k[b] : p.top_k_all;
    const float top_p = p.top_p ? p.top_p[b] : p.top_p_all, min_p = p.min_p ? p.min_p[b] : p.min_p_all, u = p.u[b];
    // (& and not &&: with branches here, the device compiler of CUDA 12.9 gave up the test of k on the path without top_p)
    const bool drawing = temp > 0.f, greedy = !drawing, use_k = drawing & (k > 0) & (k < p.V), use_p = drawing & (top_p < 1.f), use_m = drawing & (min_p > 0.f);
    const bool z_is_mass = drawing & (temp == 1.f) & !use_k & !use_m & !use_p;   // the sum for the log-probability is the mass of all tokens

    // The row's part into shared memory, and on the way, for each thread, the largest logit that it meets (NaN never is), the vector that held it first,
    // and the sum of e^(l - that) over its other logits.  The largest itself stays out of the sum, there and where sums meet, so that the
    // log-probability of a token that is almost sure, -log(1 + z), keeps the accuracy of what is left.  Weights are 2^(l log2(e) - c) with one rounding of
    // the exponent; c's own is put right at the end.
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.count[i] = 0;
    constexpr float k2e = static_cast<float>(kLog2eD);
    float best = kLowest, z = 0.f, c = 0.f;
    int best_v = 0;
    constexpr int DEPTH = 5;
    for (int base = threadIdx.x; base < max(row.nvec, kTable); base += kThreads * DEPTH) {
        uint4 v[DEPTH];
#pragma unroll
        for (int d = 0; d < DEPTH; ++d)
            if (base + d * kThreads < row.nvec) v[d] = row.from_global(gx, base + d * kThreads);
        if (base < kTable && drawing) {                            // while the first ones are on their way
            const double e = exp2(base * (1. / kTable));
#pragma unroll
            for (int i = 0; i < kCopies; ++i) sh.table[base * kCopies + (i + base) % kCopies] = e;
        }
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            if (base + d * kThreads >= row.nvec) break;
            if (RESIDENT) reinterpret_cast<uint4*>(dyn)[base + d * kThreads] = v[d];
            float l[N];
            Vec<T>::get(v[d], l);
#pragma unroll
            for (int w = N / 2; w > 0; w /= 2)                     // the largest to l[0], the others behind it (where one is NaN, NaN)
#pragma unroll
                for (int j = 0; j < w; ++j) {
                    const float less = min_or_nan(l[j], l[j + w]);
                    l[j] = fmaxf(l[j], l[j + w]);
                    l[j + w] = less;
                }
            if (l[0] > best) {
                const float most = l[0], to = most * k2e;
                z *= ex2(c - to);
                c = to;
                l[0] = best;
                best = most;
                best_v = base + d * kThreads;
            }
            if (!z_is_mass) {
#pragma unroll
                for (int j = 0; j < N; ++j) z += ex2(fmaf(l[j], k2e, -c));
            }
        }
    }
    z = fmaf(z, fmaf(-best, k2e, c) * static_cast<float>(kLn2D), z);
    // The row that comes when this one is done, as far as that can be known, into L2: HBM would be idle while this one is worked on.
    if (RESIDENT && threadIdx.x == 0 && b + ahead < p.B) {
        const uintptr_t from = reinterpret_cast<uintptr_t>(src + ahead * p.row_stride), to = from + static_cast<uintptr_t>(max(0, row.end - row.off)) * sizeof(T);
        const uintptr_t lo = (from + 15) & ~uintptr_t{15}, hi = to & ~uintptr_t{15};
        if (lo < hi) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(lo), "r"(static_cast<uint32_t>(hi - lo)) : "memory");
    }
    bool some = true;                                              // a logit above -inf
    if (!(z >= 0.f) || best == INFINITY || best == kLowest) {      // NaN, or infinities, or nothing above the lowest number: once more, with care
        z = 0.f;
        some = false;
        best_v = 0x7fffffff;
        for (int v = threadIdx.x; v < row.nvec; v += kThreads) {
            float l[N];
            Vec<T>::get(row.vec(v), l);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if (l[j] == best && best_v > v) best_v = v;
                z += l[j] == best ? static_cast<float>(some) : l[j] < best ? exp_below(l[j] - best) : 0.f;
                some = some || l[j] == best;
            }
        }
    }
    // the block's, from its warps'
    const uint32_t key = some ? order_key(best) : 0u;
    uint32_t top = __reduce_max_sync(0xffffffffu, key), at = 0xffffffffu;
    if (top && key == top) {                                       // the first place that holds it
        float l[N];
        Vec<T>::get(row.vec(best_v), l);
#pragma unroll
        for (int j = N - 1; j >= 0; --j)
            if (l[j] == best) at = static_cast<uint32_t>(row.first + best_v * N + j);
    }
    at = __reduce_min_sync(0xffffffffu, at);
    // The lanes' sums with what stayed out of them, `from`, as one without the largest, `to`
    auto joined = [](float sum, uint32_t from, uint32_t to) {
        if (from != to) sum = from ? (sum + 1.f) * exp_below(key_value(from) - key_value(to)) : 0.f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        return to ? sum + static_cast<float>(__popc(__ballot_sync(0xffffffffu, from == to)) - 1) : 0.f;
    };
    z = joined(z, key, top);
    if (row.lane == 0) { sh.warp_top[row.warp] = top; sh.warp_z[row.warp] = z; sh.warp_at[row.warp] = at; }
    __syncthreads();
    const uint32_t of_warp = row.lane < kWarps ? sh.warp_top[row.lane] : 0;
    top = __reduce_max_sync(0xffffffffu, of_warp);
    row.lmax = top ? key_value(top) : 0.f;                         // the block's, for now
    row.to_log2 = kLog2eD / static_cast<double>(temp);
    row.bin_scale = static_cast<float>(row.to_log2);
    // The k largest logits of a row are not below the smallest of the blocks' (k / blocks)-th largest of their threads' maxima, nor below the lower
    // edge of a bin that holds it.
    const int k_each = (k + row.blocks - 1) / row.blocks;
    const bool by_maxima = use_k & (k_each <= kThreads * 3 / 4);     // (then about 1.4 times as many logits are not below)
    if (by_maxima) {
        const float t = row.coarse(best);
        if (key && t > -kRange) atomicAdd(&sh.count[row.bin_of(best)], 1u);
        __syncthreads();
        const uint32_t c0 = sh.count[2 * threadIdx.x], c1 = sh.count[2 * threadIdx.x + 1];
        const uint32_t upto = static_cast<uint32_t>(warp_scan(c0 + c1, row.lane));
        if (row.lane == 31) sh.warp_q[row.warp] = upto;
        if (threadIdx.x == 0) sh.x_kth = 0;
        __syncthreads();
        uint32_t before = upto - c0 - c1;
        for (int w = 0; w < row.warp; ++w) before += static_cast<uint32_t>(sh.warp_q[w]);
        if (before < static_cast<uint32_t>(k_each) && static_cast<uint32_t>(k_each) <= before + c0 + c1) {
            const int bin = 2 * threadIdx.x + (before + c0 < static_cast<uint32_t>(k_each));
            sh.x_kth = order_key(row.logit_below(-(bin + 1.001) * (kRange / kBins)));
        }
    }
    if (row.warp == 0) {
        z = joined(row.lane < kWarps ? sh.warp_z[row.lane] : 0.f, of_warp, top);
        at = __reduce_min_sync(0xffffffffu, row.lane < kWarps && of_warp == top ? sh.warp_at[row.lane] : 0xffffffffu);
        if (row.lane == 0) { sh.x_best = top; sh.x_z = z; sh.x_index = at; sh.x_first = row.first; }
    }
    __syncthreads();
    row.cluster.sync();
    const uint32_t of_block = row.of_rank(&sh.x_best);
    top = __reduce_max_sync(0xffffffffu, of_block);
    z = joined(row.of_rank(&sh.x_z), of_block, top);
    float log_z = log1pf(z);
    if (greedy || top == 0) {                                      // top == 0: nothing above -inf, nothing to draw
        if (row.rank == 0 && row.warp == 0) {
            at = __reduce_min_sync(0xffffffffu, of_block == top && top ? row.of_rank(&sh.x_index) : 0xffffffffu);
            if (row.lane == 0) { p.token[b] = static_cast<int>(at); p.logprob[b] = top ? -log_z : -INFINITY; }
        }
        row.cluster.sync();
        return;
    }
    row.lmax = key_value(top);
    row.steep = !(fabs(static_cast<double>(row.lmax)) * row.to_log2 < 1e8) || row.to_log2 < 1e-30;   // (what is not below the floor may be lighter than 2^-1000, or -inf heavy)
    row.by_min_p = use_m;
    row.least = use_m ? log2(static_cast<double>(fminf(min_p, 1.f))) : -kRange;
    row.floor_l = row.logit_below(fmax(row.least, -static_cast<double>(kRange)));

    // the mass for the draw, or for the bound of top-p's candidates
    u64 mass = 0;
    const bool by_estimate = use_p & !use_k & !use_m & !row.steep;
    if (!use_k & !by_estimate) {
        const int e = min(row.nvec, (row.warp + 1) * row.seg);
        for (int v = row.warp * row.seg + row.lane; v < e; v += 32) {
            float l[N], most;
            Vec<T>::get(row.vec(v), l);
            most = l[0];
#pragma unroll
            for (int j = 1; j < N; ++j) most = fmaxf(most, l[j]);
            if (!(most >= row.floor_l)) continue;
            if (use_m || row.steep) {
                u64 w[N];
                row.weights(l, row.floor_l, w);
#pragma unroll
                for (int j = 0; j < N; ++j) mass += use_m && !row.eligible(l[j]) ? 0 : w[j];
                continue;
            }
#pragma unroll                                                     // what lies below the floor weighs nothing, like the floor itself
            for (int j = 0; j < N; ++j) mass += row.biased_weight(fmaxf(l[j], row.floor_l));
            mass -= N * row.kBias;
        }
    }
    auto kept_weight = [&](int i, float l) -> u64 { return row.kept(i, l) ? row.weight(l) : 0; };
    auto aim = [&](u64 total) {
        const double t = static_cast<double>(u > 0.f ? u : 0.f) * static_cast<double>(total);
        return min(total - 1, static_cast<u64>(t));
    };
    auto found = [&](int i, float l) {
        p.token[b] = row.first + i;
        p.logprob[b] = (l == row.lmax ? 0.f : l - row.lmax) - log_z;
    };
    u64 whole = 0;
    if (use_k) {
        if (by_maxima) {
            const uint32_t kth = __reduce_min_sync(0xffffffffu, row.lane < row.blocks ? *row.cluster.map_shared_rank(&sh.x_kth, row.lane) : 0xffffffffu);
            if (kth) row.floor_l = fmaxf(row.floor_l, key_value(kth));
        }
    } else if (!by_estimate) {
        const u64 own_mass = row.block_sums(mass);
        if (threadIdx.x == 0) sh.x_sum = own_mass;
        __syncthreads();
        row.cluster.sync();
        const u64 of_blocks = row.of_rank(&sh.x_sum);
        whole = row.sum_ranks(of_blocks);
        if (z_is_mass) log_z = log1pf(static_cast<float>(static_cast<double>(whole - (1ull << kFrac)) * (1. / (1ull << kFrac))));   // (the largest weighs 2^kFrac)
        if (!use_p) {
            auto here = row.cluster.barrier_arrive();              // nothing of this block is read by others after they have got here
            row.locate_in(kept_weight, of_blocks, own_mass, aim, found);
            row.cluster.barrier_wait(std::move(here));
            return;
        }
    }
    const double share = fmax(static_cast<double>(top_p), 0.);
    if (by_estimate) {
        if (row.estimated_cut(share, p.V, 1.f + z, temp, mass, whole)) {
            row.locate(kept_weight, mass, aim, found);
            row.sync();
            return;
        }
    }
    if (use_p && !use_k) {
        // Tokens lighter than this make up less than 1 - top_p together.  (.999: their multiples of 2^-44 are rounded, each by half a multiple at most)
        const double light = (1. - share) * 0.999 * static_cast<double>(whole) / p.V;
        if (light > 1000.) row.floor_l = fmaxf(row.floor_l, row.logit_below(fmin(log2(light) - kFrac, 0.)));
    }
    int total = 0;
    const bool noted = row.note_down(total);
    // One block takes them all, if they fit: up to kList are ranked at once, one a thread; more go where its part of the row was, and the other
    // blocks leave.
    const bool at_once = noted && total <= kList, collected = noted && RESIDENT && !at_once && row.blocks > 1 && total * 8 <= slice * static_cast<int>(sizeof(T));
    float* all_l = reinterpret_cast<float*>(dyn);
    int* all_i = reinterpret_cast<int*>(dyn) + total;
    u64 me = 0;
    if ((at_once || collected) && row.rank == 0) {
        uint32_t* upto = sh.count;                                 // candidates through each warp of the cluster
        if (row.warp == 0) {
            constexpr int PER = kMaxCluster * kWarps / 32;
            uint32_t c[PER], sum = 0;
#pragma unroll
            for (int x = 0; x < PER; ++x) {
                const int w = row.lane * PER + x, r = w / kWarps;
                c[x] = r < row.blocks ? *row.cluster.map_shared_rank(&sh.warp_n[w % kWarps], r) : 0;
                sum += c[x];
            }
            uint32_t through = static_cast<uint32_t>(warp_scan(sum, row.lane)) - sum;
#pragma unroll
            for (int x = 0; x < PER; ++x) upto[row.lane * PER + x] = through += c[x];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < total; i += kThreads) {
            int w = 0;                                             // the first warp through which there are more than i
#pragma unroll
            for (int half = kMaxCluster * kWarps / 2; half > 0; half >>= 1)
                if (upto[w + half - 1] <= static_cast<uint32_t>(i)) w += half;
            const Shared* from = row.cluster.map_shared_rank(&sh, w / kWarps);
            const int at_i = w % kWarps * kOwn + i - static_cast<int>(w ? upto[w - 1] : 0);
            const float l = from->own_l[at_i];
            const int index = from->own_i[at_i] + from->x_first;
            if (at_once) {
                if (row.eligible(l)) me = pack(l, index);
            } else {
                all_l[i] = l;
                all_i[i] = index;
            }
        }
    }
    if (at_once) {
        const int i = threadIdx.x;
        row.cluster.sync();                                        // the other blocks are done
        if (row.rank != 0) return;
        const float l = key_value(static_cast<uint32_t>(me >> 32));
        const u64 w = me ? row.weight(l) : 0;
        sh.all[i] = me;
        sh.all_q[i] = w;
        __syncthreads();
        int ahead = 0;
        u64 before = 0;
        for (int j = 0; j < total; ++j)
            if (sh.all[j] > me) { ++ahead; before += sh.all_q[j]; }
        bool keep = me != 0 && (!use_k || ahead < k);
        if (use_p) {
            const u64 target = row.share_of(share, use_k ? row.block_sums(keep ? w : 0) : whole);
            keep = keep && before < target;
        }
        const u64 mine = keep ? w : 0, target = aim(row.block_sums(mine));
        row.block_find(mine, target, [&](u64) {
            p.token[b] = static_cast<int>(0xffffffffu - static_cast<uint32_t>(me));
            p.logprob[b] = (l == row.lmax ? 0.f : l - row.lmax) - log_z;
        });
        return;
    }
    row.listed = noted;
    row.list_l = sh.own_l;
    row.list_i = sh.own_i;
    row.list_step = kOwn;
    if (collected) {
        row.cluster.sync();                                        // the other blocks are done
        if (row.rank != 0) return;
        row.alone = true;
        row.blocks = 1;
        row.first = 0;
        row.list_l = all_l;
        row.list_i = all_i;
        row.list_all = total;
        row.list_step = (total + kWarps - 1) / kWarps;
    }
    if (use_k) row.template find_cut<false>(-1., static_cast<u64>(k));
    if (use_p) row.template find_cut<true>(use_k ? share : -1., row.share_of(share, whole));   // without top-k the share is one of the whole row
    u64 drawn = 0;
    row.template each<true>([&](int i, float l, u64 w) { drawn += row.kept(i, l) ? w : 0; });
    row.locate(kept_weight, drawn, aim, found);
    row.sync();
}

template <typename T, bool RESIDENT>
const char* launch(const SampleTokens& p, int blocks, int slice, int smem, int num_sms, cudaStream_t s) {
    static std::atomic<uint64_t> raised{0};
    auto k = sample_tokens_kernel<T, RESIDENT>;
    if (RESIDENT && !raise_smem_limit(reinterpret_cast<const void*>(k), kMost, raised)) return "sample_tokens: the shared-memory limit could not be raised";
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
    if (cudaError_t e = cudaLaunchKernelEx(&cfg, k, p, slice, max(1, 2 * num_sms / blocks)); e != cudaSuccess) {
        cudaGetLastError();
        return cudaGetErrorString(e);
    }
    return nullptr;
}

template <typename T>
const char* launch_type(const SampleTokens& p, int num_sms, cudaStream_t s) {
    // Blocks a row: enough that two blocks fit an SM (80 KB of the row each), more of them while the rows alone would leave SMs idle.
    constexpr int64_t kFit = 80 * 1024;
    int blocks = 1;
    while (blocks < kMaxCluster && (static_cast<int64_t>(p.V) * sizeof(T) > kFit * blocks || (static_cast<int64_t>(p.B) * blocks * 2 <= num_sms && p.V > 2048 * blocks))) blocks *= 2;
    const int slice = ((p.V + blocks - 1) / blocks + 15) / 16 * 16;
    const int64_t bytes = static_cast<int64_t>(slice) * sizeof(T) + 32;    // (a part begins up to 15 bytes behind a 16-byte boundary)
    if (bytes <= kMost) return launch<T, true>(p, blocks, slice, static_cast<int>(bytes), num_sms, s);
    return launch<T, false>(p, blocks, slice, 0, num_sms, s);               // a vocabulary beyond 8 x 190 KB is read again in every pass
}

}  // namespace

const char* sample_tokens(const SampleTokens& p, int num_sms, cudaStream_t s) {
    if (p.B <= 0) return nullptr;
    if (p.type == 0) return launch_type<__nv_bfloat16>(p, num_sms, s);
    if (p.type == 1) return launch_type<__half>(p, num_sms, s);
    return launch_type<float>(p, num_sms, s);
}

}  // namespace sg
