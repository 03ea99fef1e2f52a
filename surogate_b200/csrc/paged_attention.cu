// Attention of one new token a sequence over a paged key/value cache.
//
//   s_j = scale * q . k_j  (capped: c * tanh(s / c)),  o = sum_j e^{s_j} v_j / (sum_j e^{s_j} [+ e^{sink}]),  j in [max(0, n - window), n)
//
// Every key and value is read once for the query heads that share it: 4 * (query heads per key head) operations for each 2 or 4 bytes, so HBM
// bounds it, and all the rest is arranged around reading without a pause.
//
// * A block of four warps takes tiles of 64 keys of one row and key head (eight warps and 128 keys where rows are short and few); a warp has 16 of
//   them, which lie in one page (a page holds a multiple of 16 tokens).  Each warp has a ring of such steps in shared memory, filled by TMA (one box
//   of 16 places by 128 bytes for each 128 bytes of the head) and waited for on its own mbarriers: warps do not wait for one another.
// * Both products are m16n8k16 with the keys, or the values' elements, on the 16 rows and eight query heads on the columns: the few query heads
//   that share a key head fill a column group, and scores, weights and outputs of a head stay in the same lanes' columns.  tcgen05 would want 128
//   rows of queries for its M; here there are 1 to 16, and HBM is the bound (mma.sync runs at a quarter of its rate: 23 % of the tensor pipe with 16 heads).
// * The sums of a product may run over the head's elements in any order.  So a lane reads whole 16-byte pieces of key rows: the piece is, word
//   for word, its share of the left operand, with the query laid out to match.  For the values it reads pieces of four keys and pairs their
//   elements by byte permutes.  The weights turn from accumulator to right operand by a transposition of 8 x 8 matrices in registers.
// * A running maximum that moves only when a score exceeds it by 2^8 (see `top`): most steps need neither a maximum over lanes nor a rescaling.
//   The warps of a block have their own and meet at the end of the piece; pieces of a row in different blocks are joined by a second, small kernel.
// * Weights are split into two bf16 (or fp16) terms before they meet the values, hi + lo, which keeps 16 (22) bits: tensor cores have time to
//   spare here, and the output's own rounding stays the only one that counts.  With e4m3 values weight times scale is one fp16 term: 2^-12 of
//   itself down to 2^-21 of the largest one met, 2^-32 of the largest below; both are less than the values' own 2^-4 takes (of an element, or, where
//   it is far below its row's largest, 2^-10 of the row's scale).  That holds for scales that say how large values are; rows of zeros are found by looking.
// * e4m3: keys and values become fp16 exactly; the query as fp16 is scaled by a power of two to below 2 for each row (what it loses lies 2^-25
//   below its largest element).  The scale of a key multiplies its score; that of a value goes into its weight, and its log2 into the comparison
//   with the running maximum, which then bounds weight times scale.
//
// Measured (B200, a copy runs at 6.55 TB/s): see kStart and paged_attention_plan; 2 rows of 100 001 to 131 072 keys, 64 over 8 heads of 128, bf16
// 167 us, 6.1 TB/s; 128 rows of 2000 to 16 384 keys, 32 over 4 heads, e4m3 202 us, 6.2 TB/s; one row of 300 keys 6.6 us, which is latency:
// launch, length, page number, keys, one after the other.  A next piece requested before the warps meet, with places of their own to meet at, cost more in
// instructions than it hid (e4m3 61 -> 71 us): three blocks an SM hide one another's starts.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>

#include "launch_limits.h"
#include "paged_kv.h"
#include "sm100_ptx.cuh"

namespace sg {

namespace {

constexpr int kTile = 64, kStep = 16;   // keys of a tile that blocks share, keys of a warp and step
constexpr int kSharing = 4;              // warps of a block that shares rows with others
constexpr int RING_BYTES = 16384;   // of a warp, where two steps fit
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f, kLowest = -3.402823466e38f;

__device__ __forceinline__ uint4 lds16(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ float lds4(uint32_t a) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void prefetch_l1(const void* p) { asm volatile("prefetch.global.L1 [%0];" ::"l"(p)); }
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// tanh(y) to some 2^-21 of itself: below 0.8 Lambert's continued fraction y / (1 + y^2 / (3 + y^2 / (5 + y^2 / (7 + y^2 / 9)))) as one quotient (its
// next term is 2^-26 there), above it (e^2y - 1) / (e^2y + 1), which would cancel for small y, and with a cap of 50 cost small scores 2^-16
// of themselves and more.  NaN stays.
__device__ __forceinline__ float tanh_ratio(float y) {
    const float a = fabsf(y), q = y * y;
    const bool small = a < 0.8f;
    const float e = ex2((a > 12.f ? 12.f : a) * (2.f * kLog2e));   // (tanh 12 = 1 - 2^-34)
    const float num = small ? a * fmaf(q, q + 105.f, 945.f) : e - 1.f, den = small ? fmaf(q, fmaf(q, 15.f, 420.f), 945.f) : e + 1.f;
    return copysignf(__fdividef(num, den), y);
}
// d[16 x 8] += a[16 x 16] b[16 x 8]
template <bool BF16>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// An 8 x 8 matrix of 16-bit elements, two of a row in each lane, transposed
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
template <bool BF16> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    if (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <bool BF16> __device__ __forceinline__ float2 unpack2(uint32_t v) {
    if (BF16) return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
// two e4m3 values (the lower 16 bits) as two fp16
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t v) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
    return r;
}

// Compile-time layout of one variant.
template <int KT, int D, int ROWS, bool DEEP> struct Shape {
    static constexpr int ES = KT == kKvE4m3 ? 1 : 2;               // bytes of a cached element
    static constexpr bool BF16 = KT == kKvBf16;                    // operand type of the products: bf16, else fp16
    static constexpr int HT = ROWS / 8;                            // groups of eight query heads
    static constexpr int KCH = D * ES / 64;                        // 16-byte pieces of a key row for each of the four lanes that share it
    static constexpr int VB = D * ES >= 128 ? 16 : 8;              // bytes of a piece of a value row, shared by eight lanes
    static constexpr int VCH = D * ES / (8 * VB);
    static constexpr int E = VB / ES;                              // elements of that piece
    static constexpr int ROWB = D * ES;                            // bytes of a row
    static constexpr int PITCH = ROWB < 128 ? ROWB : 128;          // of a row in shared memory: wider ones are copied 128 bytes at a time
    static constexpr int BOXES = ROWB / PITCH, BOXEL = PITCH / ES, BOXBYTES = kStep * PITCH;
    static constexpr int KBYTES = kStep * ROWB;                    // a warp's keys of one step; its values take as much
    static constexpr int STAGE = 2 * KBYTES + (KT == kKvE4m3 ? 1024 : 0);   // swizzled tiles begin on 1024 bytes
    // Where blocks fill the GPU, four warps have 16 KB each under way, three blocks an SM.  Where there are fewer short rows than SMs, a block has eight,
    // each with up to three steps requested at once, since nothing else hides its waits (heads of 256: four, for their shared memory).
    static constexpr int WARPS = DEEP && D <= 128 ? 8 : 4, TILE = WARPS * kStep;
    static constexpr int FITS = (DEEP ? 24576 : RING_BYTES) / STAGE, MOST_STAGES = DEEP ? 3 : 8;
    static constexpr int STAGES = FITS > MOST_STAGES ? MOST_STAGES : FITS < 2 ? 2 : FITS;
    static constexpr int RING = STAGE * STAGES;                    // of one warp
    static constexpr int MT = D / 16;                              // tiles of 16 outputs
    static constexpr int SMEM = 1024 + WARPS * RING;
    static_assert(RING >= ROWS * D * 4, "a warp's ring holds its outputs when the warps meet");
    static constexpr int FIT = 230000 / (SMEM + 2048);             // blocks that an SM's shared memory holds
    static constexpr int MOST = D <= 128 ? 3 : 2;     // of 168 registers a thread, or 255
    static constexpr int PER_SM = FIT < MOST ? FIT : MOST;
};

struct Ring {            // a warp's copies under way
    const CUtensorMap* map;
    uint32_t base, bars;  // shared memory: all warps' rings, one barrier for each slot
    float* meet;          // the same memory, when the copies are done and the warps' outputs meet
    volatile int* abort_flag;
    int slot;             // the next step's
    uint32_t parity;
};

struct Cut {             // where the pieces of a shared problem go
    float* part_o;       // [2 * blocks][ROWS][D]
    float2* part_ml;     // [2 * blocks][ROWS]: maximum (base 2), sum
    long long* prefix;   // [B + 2]: first unit of each row, all units, units a block
    int blocks, min_units;
};

__device__ __forceinline__ int row_keys(const PagedAttention& p, int b) {
    const int n = p.lengths[b];
    const int64_t room = static_cast<int64_t>(p.table_width) * p.kv.page_size;
    if (n < 0 || n > room) {
        atomicExch(p.error_flag, kErrBadPage);
        return n < 0 ? 0 : static_cast<int>(room);
    }
    return n;
}
__device__ __forceinline__ int first_key(const PagedAttention& p, int n) { return p.window > 0 ? max(0, n - p.window) : 0; }
template <int TILE> __device__ __forceinline__ int row_tiles(const PagedAttention& p, int n) { return (n + TILE - 1) / TILE - first_key(p, n) / TILE; }

template <typename QT> __device__ __forceinline__ QT from_float(float x);
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* m, int c0, int c1, int c2, int c3, int c4, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(m)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(bar)
        : "memory");
}

template <int KT, typename QT, int D, int ROWS, bool DEEP>
struct Piece {
    using S = Shape<KT, D, ROWS, DEEP>;
    // weights are carried as 2^7 times themselves where they become fp16, whose smallest step is 2^-24; they are below 2^(kSlack) before
    static constexpr float kShift = S::BF16 ? 0.f : 7.f, kSlack = 8.f;
    // log2 of the least scale that counts in a maximum: a key may then weigh 2^88 and the slack in the sum of weights, and 2^30 of them fit fp32
    static constexpr float kLeastScale = -88.f;

    static __device__ Ring begin(const CUtensorMap* map, uint8_t* smem, unsigned long long* bars, int* abort_flag) {
        uint8_t* at = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem) + 1023) & ~uintptr_t{1023});
        if (threadIdx.x == 0) {
            *abort_flag = 0;
            tma_prefetch_desc(map);
        }
        if (threadIdx.x < S::WARPS * S::STAGES) mbar_init(smem_u32(bars + threadIdx.x), 1);
        fence_barrier_init();
        __syncthreads();
        return Ring{map, smem_u32(at), smem_u32(bars), reinterpret_cast<float*>(at), abort_flag, 0, 0};
    }
    static __device__ void end(const PagedAttention& p, const int* abort_flag) {
        if (threadIdx.x == 0 && *abort_flag) atomicExch(p.error_flag, 1);
    }

    // Tiles [tb, te) of row b (tile numbers of the row's positions) and head group vh.  slot < 0: the whole row; its result is written.  Else the piece is.
    // False (for the whole block) when a wait gave up: the block must stop.
    static __device__ bool run(const PagedAttention& p, const Cut& cut, int b, int vh, int n, int tb, int te, int groups, int slot, Ring& rg, float2 (*sh_ml)[16]) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
        const int G = p.Hq / p.kv.heads, kvh = vh / groups, h0 = kvh * G + (vh - kvh * groups) * ROWS, nrows = min(ROWS, kvh * G + G - h0);
        const int lo = first_key(p, n), steps = te - tb;
        const uint32_t ring = rg.base + warp * S::RING, bars = rg.bars + warp * S::STAGES * 8;
        const int* table = p.table + b * p.table_stride;
        // Row r of a product's 16 keys is key r, or r ^ 4 where r is odd.  With the order in which the copies swizzle a row's 16-byte pieces (piece ^ row % 8),
        // neither the lanes that read keys (row g) nor those that read values (rows 2c, 2c + 1) then meet in a bank.
        const int k0 = (g & 1) ? g ^ 4 : g;                        // this lane's first key; its second is 8 further on
        const int v0 = 2 * c, v1 = (2 * c ^ 4) + 1;                // rows 2c and 2c + 1, whose values it pairs; then the same 8 further on
        uint32_t k_off[2], v_off[2];
        if (S::ROWB >= 128) {
            k_off[0] = k0 * 128 + ((c ^ (k0 & 7)) << 4);
            k_off[1] = k_off[0] ^ 64;
            v_off[0] = S::KBYTES + v0 * 128 + ((g ^ (v0 & 7)) << 4);
            v_off[1] = S::KBYTES + v1 * 128 + ((g ^ (v1 & 7)) << 4);
        } else {                                                   // rows of 64 bytes: piece ^ row / 2 % 4
            k_off[0] = k_off[1] = k0 * 64 + ((c ^ ((k0 >> 1) & 3)) << 4);
            v_off[0] = S::KBYTES + v0 * 64 + (((g >> 1) ^ ((v0 >> 1) & 3)) << 4) + (g & 1) * 8;
            v_off[1] = S::KBYTES + v1 * 64 + (((g >> 1) ^ ((v1 >> 1) & 3)) << 4) + (g & 1) * 8;
        }

        // page of the warp's keys in step base + lane; -1: none of them counts
        auto load_pages = [&](int base) {
            const int64_t t = static_cast<int64_t>(tb + base + lane) * S::TILE + warp * kStep;
            if (base + lane >= steps || t >= n || t + kStep <= lo) return -1;
            int page = table[t / p.kv.page_size];
            if (page < 0 || page >= p.kv.num_pages) {
                atomicExch(p.error_flag, kErrBadPage);
                page = -1;
            }
            return page;
        };
        int pages = load_pages(0), pages_next = load_pages(32);
        unsigned have = 0;            // bit i % 32: step i has a page
        bool seen = false;            // a key that counts has been met
        int next_i = 0, next_place = (tb * S::TILE + warp * kStep) % p.kv.page_size;   // the step that is requested next
        const int place_step = S::TILE % p.kv.page_size;

        // Request the next step into slot `to`.  A step without a page has coordinates outside the cache: zeros, and nothing is read.
        auto issue = [&](int to) {
            if ((next_i & 31) == 0 && next_i > 0) {
                pages = pages_next;
                pages_next = load_pages(next_i + 32);
            }
            const int page = __shfl_sync(0xffffffffu, pages, next_i & 31);
            have = (have & ~(1u << (next_i & 31))) | (page >= 0 ? 1u << (next_i & 31) : 0u);
            if (lane == 0) {
                const uint32_t dst = ring + to * S::STAGE, bar = bars + to * 8;
                const bool scaled = KT == kKvE4m3 && page >= 0;
                mbar_expect_tx(bar, 2 * S::KBYTES + (scaled ? 128 : 0));
#pragma unroll
                for (int x = 0; x < S::BOXES; ++x) tma_load_5d(dst + x * S::BOXBYTES, rg.map, x * S::BOXEL, next_place, kvh, 0, page, bar);
#pragma unroll
                for (int x = 0; x < S::BOXES; ++x) tma_load_5d(dst + S::KBYTES + x * S::BOXBYTES, rg.map, x * S::BOXEL, next_place, kvh, 1, page, bar);
                if (scaled) {
                    const float* sp = p.kv.scales + page * p.kv.s_page_stride + kvh * p.kv.s_head_stride + next_place;
                    bulk_load(dst + 2 * S::KBYTES, sp, 64, bar);
                    bulk_load(dst + 2 * S::KBYTES + 64, sp + p.kv.s_kv_stride, 64, bar);
                }
            }
            ++next_i;
            next_place += place_step;
            if (next_place >= p.kv.page_size) next_place -= p.kv.page_size;
        };
        // all slots are free here: the step that this piece begins with goes to rg.slot
#pragma unroll
        for (int i = 0; i < S::STAGES; ++i)
            if (i < steps) issue(rg.slot + i < S::STAGES ? rg.slot + i : rg.slot + i - S::STAGES);

        // the query, piece by piece as the keys lie: head g (+ 8)
        constexpr int QW = KT == kKvE4m3 ? 8 : 4;                  // words of one head for one 16-byte piece of keys
        uint32_t q[S::HT][S::KCH][QW];
        float mult[S::HT][2];                                      // what turns a product with head 2c, 2c + 1 into a score
#pragma unroll
        for (int r = 0; r < S::HT; ++r) {
            const int row = g + 8 * r;
            const QT* src = static_cast<const QT*>(p.q) + b * p.q_b_stride + (h0 + (row < nrows ? row : 0)) * p.q_h_stride;
            constexpr int EL = 16 / S::ES;                         // elements of a piece
#pragma unroll
            for (int j = 0; j < S::KCH; ++j) {
#pragma unroll
                for (int w = 0; w < QW; w += 4) {
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (row < nrows) v = *reinterpret_cast<const uint4*>(src + (j * 4 + c) * EL + w * 2);
                    q[r][j][w] = v.x; q[r][j][w + 1] = v.y; q[r][j][w + 2] = v.z; q[r][j][w + 3] = v.w;
                }
            }
            float own = p.scale;
            if (KT == kKvE4m3 && std::is_same<QT, __nv_bfloat16>::value) {   // bf16 -> fp16 of the same value over a power of two
                float amax = 0.f;
#pragma unroll
                for (int j = 0; j < S::KCH; ++j)
#pragma unroll
                    for (int w = 0; w < QW; ++w) {
                        const float2 f = unpack2<true>(q[r][j][w]);
                        amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
                    }
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                const int e = min(max(static_cast<int>(__float_as_uint(amax) >> 23) - 127, -100), 100);
                const float down = __uint_as_float((127 - e) << 23);
                own *= __uint_as_float((127 + e) << 23);
#pragma unroll
                for (int j = 0; j < S::KCH; ++j)
#pragma unroll
                    for (int w = 0; w < QW; ++w) {
                        const float2 f = unpack2<true>(q[r][j][w]);
                        q[r][j][w] = pack2<false>(f.x * down, f.y * down);
                    }
            }
            if (p.softcap == 0.f) own *= kLog2e;
            mult[r][0] = __shfl_sync(0xffffffffu, own, 8 * c);     // lane 4 * head holds that head's
            mult[r][1] = __shfl_sync(0xffffffffu, own, 8 * c + 4);
        }
        const float cap = p.softcap, inv_cap = cap != 0.f ? 1.f / cap : 0.f, cap2 = cap * kLog2e;

        // o[m][r]: outputs of two elements of the head and of heads 8 r + 2c, + 1: [0], [1] the first element's, [2], [3] the second's
        float o[S::MT][S::HT][4];
        // Weights are relative to 2^top, which follows the scores' maximum only when they exceed it by kSlack: most steps need no maximum over lanes.
        // (top: 0 until then; limit: what a score, or score plus log2 of a value's scale, may be without that.)
        float top[S::HT][2], limit[S::HT][2], l[S::HT][2];
#pragma unroll
        for (int i = 0; i < S::MT; ++i)
#pragma unroll
            for (int r = 0; r < S::HT; ++r)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[i][r][k] = 0.f;
#pragma unroll
        for (int r = 0; r < S::HT; ++r)
#pragma unroll
            for (int k = 0; k < 2; ++k) { top[r][k] = 0.f; limit[r][k] = -INFINITY; l[r][k] = 0.f; }

        // One step: 16 keys in the slot at `at`.  Only the first and last of a row hold keys that do not count (FULL: none does).
        auto compute = [&](auto full_tag, uint32_t at, int t0) {
            constexpr bool FULL = decltype(full_tag)::value;
            // scores of 16 keys: s[r][0], [1] are key k0 with heads 8 r + 2c, + 1, s[r][2], [3] key k0 + 8
            float s[S::HT][4], s2[S::HT][4];                       // two sums, so that products do not wait for one another
#pragma unroll
            for (int r = 0; r < S::HT; ++r)
#pragma unroll
                for (int k = 0; k < 4; ++k) s[r][k] = s2[r][k] = 0.f;
#pragma unroll
            for (int j = 0; j < S::KCH; ++j) {
                const uint32_t kp = at + k_off[j & 1] + (j >> 1) * S::BOXBYTES;
                const uint4 ka = lds16(kp), kb = lds16(kp + 8 * S::PITCH);
                if (KT != kKvE4m3) {
#pragma unroll
                    for (int r = 0; r < S::HT; ++r) {
                        mma<S::BF16>(s[r], ka.x, kb.x, ka.y, kb.y, q[r][j][0], q[r][j][1]);
                        mma<S::BF16>(s2[r], ka.z, kb.z, ka.w, kb.w, q[r][j][2], q[r][j][3]);
                    }
                } else {
                    const uint32_t wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t a0 = e4m3x2_to_f16x2(static_cast<uint16_t>(wa[w])), a2 = e4m3x2_to_f16x2(static_cast<uint16_t>(wa[w] >> 16));
                        const uint32_t a1 = e4m3x2_to_f16x2(static_cast<uint16_t>(wb[w])), a3 = e4m3x2_to_f16x2(static_cast<uint16_t>(wb[w] >> 16));
#pragma unroll
                        for (int r = 0; r < S::HT; ++r) mma<false>((w & 1) ? s2[r] : s[r], a0, a1, a2, a3, q[r][j][(2 * w) % QW], q[r][j][(2 * w + 1) % QW]);
                    }
                }
            }
            float lv[2] = {0.f, 0.f}, vs[2];                       // e4m3: the two keys' value scales, and log2 of them
            if (KT == kKvE4m3) {
                const uint32_t sa = at + 2 * S::KBYTES + k0 * 4;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const float ks = lds4(sa + t * 32);
#pragma unroll
                    for (int r = 0; r < S::HT; ++r)
#pragma unroll
                        for (int h = 0; h < 2; ++h) s[r][2 * t + h] = (s[r][2 * t + h] + s2[r][2 * t + h]) * ks;
                    vs[t] = lds4(sa + 64 + t * 32);
                    vs[t] = vs[t] < 0x1p-100f ? 0x1p-100f : vs[t];   // (a NaN stays)
                    lv[t] = vs[t] < INFINITY ? fmaxf(__log2f(vs[t]), kLeastScale) : 0.f;   // (not finite: outputs become NaN, whatever the bound)
                }
            }
            if (!FULL && KT == kKvE4m3) {
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    if (t0 + k0 + 8 * t < lo || t0 + k0 + 8 * t >= n) { lv[t] = 0.f; vs[t] = 1.f; }   // not there: its scale may be anything
            }
            bool above = false;
            float most[S::HT][2];
#pragma unroll
            for (int r = 0; r < S::HT; ++r) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float x = (KT == kKvE4m3 ? s[r][k] : s[r][k] + s2[r][k]) * mult[r][k & 1];
                    if (cap != 0.f) x = cap2 * tanh_ratio(x * inv_cap);
                    if (!FULL) {
                        const int key = t0 + k0 + 4 * (k & 2);
                        if (key < lo || key >= n) x = -INFINITY;
                    }
                    s[r][k] = x;
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    most[r][h] = KT == kKvE4m3 ? fmaxf(s[r][h] + lv[0], s[r][2 + h] + lv[1]) : fmaxf(s[r][h], s[r][2 + h]);
                    above |= most[r][h] > limit[r][h];
                }
            }
            if (__any_sync(0xffffffffu, above)) {
                // A row of zeros has the scale 1, thousands of times its neighbours', and adds nothing: with that in the maximum their weights would be lost
                // among fp16's subnormals.  So such rows get the least scale.  (One that does not exceed the limit does no harm.)
                if (KT == kKvE4m3) {
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        uint32_t some = 0;                         // the four lanes of a key look at its values together
                        const uint32_t row = at + S::KBYTES + (k0 + 8 * t) * S::PITCH + c * 16;
#pragma unroll
                        for (int x = 0; x < S::BOXES; ++x)
#pragma unroll
                            for (int y = 0; y < S::PITCH; y += 64) {
                                const uint4 v = lds16(row + x * S::BOXBYTES + y);
                                some |= (v.x | v.y | v.z | v.w) & 0x7f7f7f7fu;
                            }
                        some |= __shfl_xor_sync(0xffffffffu, some, 1);
                        some |= __shfl_xor_sync(0xffffffffu, some, 2);
                        if (some == 0 && vs[t] < INFINITY) {
                            lv[t] = kLeastScale;
                            vs[t] = 0x1p-88f;
                        }
                    }
#pragma unroll
                    for (int r = 0; r < S::HT; ++r)
#pragma unroll
                        for (int h = 0; h < 2; ++h) most[r][h] = fmaxf(s[r][h] + lv[0], s[r][2 + h] + lv[1]);
                }
#pragma unroll
                for (int r = 0; r < S::HT; ++r)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float mx = most[r][h];
#pragma unroll
                        for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
                        if (mx > (limit[r][h] == -INFINITY ? -INFINITY : top[r][h])) {
                            const float f = limit[r][h] == -INFINITY ? 0.f : ex2(top[r][h] - mx);
                            top[r][h] = mx;
                            limit[r][h] = mx + kSlack;
                            l[r][h] *= f;
#pragma unroll
                            for (int m = 0; m < S::MT; ++m) { o[m][r][h] *= f; o[m][r][2 + h] *= f; }
                        }
                    }
            }
            // weights, transposed to the right operand of the second product: rows of eight keys
            uint32_t ph[S::HT][2], pl[S::HT][2];
#pragma unroll
            for (int r = 0; r < S::HT; ++r)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const float e0 = ex2(s[r][2 * t] - top[r][0]), e1 = ex2(s[r][2 * t + 1] - top[r][1]);
                    l[r][0] += e0;
                    l[r][1] += e1;
                    float w0 = e0, w1 = e1;
                    if (KT == kKvE4m3) {
                        const float f = vs[t] * 128.f;
                        w0 *= f;
                        w1 *= f;
                    } else if (kShift != 0.f) {
                        w0 *= 128.f;
                        w1 *= 128.f;
                    }
                    ph[r][t] = pack2<S::BF16>(w0, w1);
                    if (KT != kKvE4m3) {
                        const float2 back = unpack2<S::BF16>(ph[r][t]);
                        pl[r][t] = transpose8(pack2<S::BF16>(w0 - back.x, w1 - back.y));
                    }
                    ph[r][t] = transpose8(ph[r][t]);
                }
            // o += values . weights; a lane's piece of the value rows is row g (and g + 8: the next element) of E / 2 tiles
#pragma unroll
            for (int j = 0; j < S::VCH; ++j) {
                uint32_t v[4][S::VB / 4];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const uint32_t vp = at + v_off[t & 1] + (t >> 1) * 8 * S::PITCH + j * S::BOXBYTES;
                    if (S::VB == 16) {
                        const uint4 x = lds16(vp);
                        v[t][0] = x.x; v[t][1] = x.y; v[t][2 % (S::VB / 4)] = x.z; v[t][3 % (S::VB / 4)] = x.w;
                    } else {
                        const uint2 x = lds8(vp);
                        v[t][0] = x.x; v[t][1] = x.y;
                    }
                    if (!FULL) {                                   // what lies behind the row's end or before its window may be anything
                        const int key = t0 + (t & 1 ? v1 : v0) + (t >> 1) * 8;
                        if (key < lo || key >= n) {
#pragma unroll
                            for (int w = 0; w < S::VB / 4; ++w) v[t][w] = 0;
                        }
                    }
                }
#pragma unroll
                for (int w = 0; w < S::VB / 4; ++w) {
                    if (KT != kKvE4m3) {
                        const uint32_t a0 = __byte_perm(v[0][w], v[1][w], 0x5410), a1 = __byte_perm(v[0][w], v[1][w], 0x7632);
                        const uint32_t a2 = __byte_perm(v[2][w], v[3][w], 0x5410), a3 = __byte_perm(v[2][w], v[3][w], 0x7632);
#pragma unroll
                        for (int r = 0; r < S::HT; ++r) {
                            mma<S::BF16>(o[j * S::E / 2 + w][r], a0, a1, a2, a3, ph[r][0], ph[r][1]);
                            mma<S::BF16>(o[j * S::E / 2 + w][r], a0, a1, a2, a3, pl[r][0], pl[r][1]);
                        }
                    } else {
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const uint32_t sel = x ? 0x7362 : 0x5140;
                            const uint32_t u = __byte_perm(v[0][w], v[1][w], sel), y = __byte_perm(v[2][w], v[3][w], sel);
                            const uint32_t a0 = e4m3x2_to_f16x2(static_cast<uint16_t>(u)), a1 = e4m3x2_to_f16x2(static_cast<uint16_t>(u >> 16));
                            const uint32_t a2 = e4m3x2_to_f16x2(static_cast<uint16_t>(y)), a3 = e4m3x2_to_f16x2(static_cast<uint16_t>(y >> 16));
#pragma unroll
                            for (int r = 0; r < S::HT; ++r) mma<false>(o[j * S::E / 2 + 2 * w + x][r], a0, a1, a2, a3, ph[r][0], ph[r][1]);
                        }
                    }
                }
            }
        };

        int t0 = tb * S::TILE + warp * kStep;
        int i = 0;
        for (; i < steps; ++i, t0 += S::TILE) {
            if (!__all_sync(0xffffffffu, mbar_wait(bars + rg.slot * 8, rg.parity, rg.abort_flag))) break;   // a wait that gave up
            const uint32_t at = ring + rg.slot * S::STAGE;
            if ((have >> (i & 31)) & 1) {
                seen = true;
                if (t0 >= lo && t0 + kStep <= n) compute(std::true_type{}, at, t0);
                else compute(std::false_type{}, at, t0);
            }
            __syncwarp();                                          // every lane has read the slot
            if (next_i < steps) issue(rg.slot);
            if (++rg.slot == S::STAGES) { rg.slot = 0; rg.parity ^= 1; }
        }

        const bool gave_up = i < steps;
        for (; i < next_i; ++i) {                                  // only then: what this warp asked for, with a limit again
            int never = 0;
            mbar_wait(bars + rg.slot * 8, rg.parity, &never);
            if (++rg.slot == S::STAGES) { rg.slot = 0; rg.parity ^= 1; }
        }

        // The warps meet.  A warp without keys has the maximum -inf; one whose keys had no score above -inf (all of them -inf or NaN: sums are 0 or NaN) has
        // the lowest number, so that its NaN stay, and a row of nothing but such keys is not taken for an empty one.
#pragma unroll
        for (int r = 0; r < S::HT; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l[r][h] += __shfl_xor_sync(0xffffffffu, l[r][h], x);
                if (limit[r][h] == -INFINITY) top[r][h] = seen ? kLowest : -INFINITY;
                if (g == 0) sh_ml[warp][8 * r + 2 * c + h] = make_float2(top[r][h], l[r][h]);
            }
        __syncthreads();
        float* mine = rg.meet + warp * (ROWS * D);
#pragma unroll
        for (int r = 0; r < S::HT; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int head = 8 * r + 2 * c + h;
                float mm = -INFINITY;
#pragma unroll
                for (int w = 0; w < S::WARPS; ++w) mm = fmaxf(mm, sh_ml[w][head].x);
                const float f = top[r][h] == -INFINITY ? 0.f : ex2(top[r][h] - mm);
#pragma unroll
                for (int j = 0; j < S::VCH; ++j)
#pragma unroll
                    for (int e = 0; e < S::E; e += 2) {
                        const float (&acc)[4] = o[(j * S::E + e) / 2][r];
                        *reinterpret_cast<float2*>(mine + head * D + (j * 8 + g) * S::E + e) = make_float2(acc[h] * f, acc[2 + h] * f);
                    }
            }
        __syncthreads();
        for (int x = threadIdx.x * 4; x < nrows * D; x += S::WARPS * 128) {
            const int row = x / D, d = x - row * D;
            float mm = -INFINITY, ll = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < S::WARPS; ++w) mm = fmaxf(mm, sh_ml[w][row].x);
#pragma unroll
            for (int w = 0; w < S::WARPS; ++w) {
                const float2 v = sh_ml[w][row];
                const float4 a = *reinterpret_cast<const float4*>(rg.meet + w * (ROWS * D) + x);
                if (v.x != -INFINITY) ll += v.y * ex2(v.x - mm);
                acc.x += a.x; acc.y += a.y; acc.z += a.z; acc.w += a.w;
            }
            if (slot >= 0) {
                *reinterpret_cast<float4*>(cut.part_o + (static_cast<int64_t>(slot) * ROWS + row) * D + d) = acc;
                if (d == 0) cut.part_ml[slot * ROWS + row] = make_float2(mm, ll);
            } else {
                finish(p, b, h0 + row, d, mm, ll, acc);
            }
        }
        fence_proxy_async();                                       // the rings are written by copies again
        return __syncthreads_or(gave_up) == 0;
    }

    // elements d to d + 3 of one output.  mm == -inf: no key counts.  Keys without a score above -inf leave 0 / 0, or 0 / sink.
    static __device__ __forceinline__ void finish(const PagedAttention& p, int b, int h, int d, float mm, float ll, float4 acc) {
        const int64_t at = static_cast<int64_t>(b) * p.Hq + h;
        float total = ll;
        if (p.sinks) total += ex2(p.sinks[h] * kLog2e - mm);       // infinite where the sink outweighs all keys by 2^128: the output is 0
        const float f = S::BF16 ? 1.f : 0x1p-7f;
        QT y[4];
        y[0] = from_float<QT>(mm == -INFINITY ? 0.f : acc.x * f / total);
        y[1] = from_float<QT>(mm == -INFINITY ? 0.f : acc.y * f / total);
        y[2] = from_float<QT>(mm == -INFINITY ? 0.f : acc.z * f / total);
        y[3] = from_float<QT>(mm == -INFINITY ? 0.f : acc.w * f / total);
        *reinterpret_cast<uint2*>(static_cast<QT*>(p.out) + at * D + d) = *reinterpret_cast<const uint2*>(y);
        if (d == 0 && p.lse) p.lse[at] = fabsf(mm) == INFINITY ? mm : mm * kLn2 + logf(ll);   // (infinite scores: their weights are NaN)
    }
};

// Short rows: a block takes whole ones, one row and head group after the other.
template <int KT, typename QT, int D, int ROWS, bool DEEP>
__global__ void __launch_bounds__((Shape<KT, D, ROWS, DEEP>::WARPS * 32), (DEEP ? 1 : Shape<KT, D, ROWS, DEEP>::PER_SM))
paged_attention_whole_kernel(const __grid_constant__ CUtensorMap map, PagedAttention p, int groups) {
    using S = Shape<KT, D, ROWS, DEEP>;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ float2 sh_ml[S::WARPS][16];
    __shared__ unsigned long long sh_bars[S::WARPS * 8];
    __shared__ int sh_abort;
    const int vhs = p.kv.heads * groups, pairs = p.B * vhs;
    Ring rg = Piece<KT, QT, D, ROWS, DEEP>::begin(&map, smem, sh_bars, &sh_abort);
    for (int pair = blockIdx.x; pair < pairs; pair += gridDim.x) {
        const int b = pair / vhs, vh = pair - b * vhs;
        // the row's page numbers and queries are on their way while its length is
        if (static_cast<int>(threadIdx.x) * 32 < p.table_width) prefetch_l1(p.table + b * p.table_stride + threadIdx.x * 32);
        if (threadIdx.x >= 32 && threadIdx.x < 32 + ROWS) {
            const int G = p.Hq / p.kv.heads, kvh = vh / groups, h = min(kvh * G + (vh - kvh * groups) * ROWS + static_cast<int>(threadIdx.x) - 32, p.Hq - 1);
            prefetch_l1(static_cast<const QT*>(p.q) + b * p.q_b_stride + h * p.q_h_stride);
        }
        const int n = row_keys(p, b), tb = first_key(p, n) / S::TILE;
        if (!Piece<KT, QT, D, ROWS, DEEP>::run(p, Cut{}, b, vh, n, tb, tb + row_tiles<S::TILE>(p, n), groups, -1, rg, sh_ml)) break;
    }
    Piece<KT, QT, D, ROWS, DEEP>::end(p, &sh_abort);
}

// All tiles of all rows and head groups, in that order, shared evenly by the blocks: nothing on the host knows the lengths.  Each row and head group
// counts kStart tiles more than it has (at its beginning), for the instructions that a block spends on starting and ending a piece; without, blocks
// with many short rows end late.  64 rows of 100 to 4096 keys, 32 over 8 heads of 128, with 0 / 1 / 2 / 4 / 6 (before the ends were made shorter):
// bf16 103 / 101 / 100 / 98 / 99 us, e4m3 82 / 76 / 66 / 61 / 60; 128 over 8 heads, bf16 - / 147 / 136 / 123 / 120.  Rows of one length gain 1 to 2 %.
// A block's first and last piece may be part of a row; each goes to a slot of its own.
constexpr int kStart = 4;
__device__ __forceinline__ long long row_units(const PagedAttention& p, int b, int vhs) {
    const int tiles = row_tiles<kTile>(p, row_keys(p, b));
    return tiles ? static_cast<long long>(tiles + kStart) * vhs : 0;
}
template <int KT, typename QT, int D, int ROWS>
__global__ void __launch_bounds__(kSharing * 32, (Shape<KT, D, ROWS, false>::PER_SM)) paged_attention_shared_kernel(const __grid_constant__ CUtensorMap map, PagedAttention p, Cut cut, int groups) {
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ float2 sh_ml[kSharing][16];
    __shared__ unsigned long long sh_bars[kSharing * 8];
    __shared__ int sh_abort;
    __shared__ long long sh_sum[kSharing];
    __shared__ int sh_b;
    __shared__ long long sh_rest;
    const int vhs = p.kv.heads * groups, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // units (tiles of one head group) before each row: a thread adds up its share of the rows, the block scans the sums
    const int each = (p.B + kSharing * 32 - 1) / (kSharing * 32), r0 = min(p.B, static_cast<int>(threadIdx.x) * each), r1 = min(p.B, r0 + each);
    long long mine = 0;
    for (int b = r0; b < r1; ++b) mine += row_units(p, b, vhs);
    long long scan = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += v;
    }
    if (lane == 31) sh_sum[warp] = scan;
    if (threadIdx.x == 0) sh_b = p.B;
    __syncthreads();
    long long before = scan - mine, total = 0;
#pragma unroll
    for (int w = 0; w < kSharing; ++w) {
        if (w < warp) before += sh_sum[w];
        total += sh_sum[w];
    }
    const long long per = max(static_cast<long long>(cut.min_units), (total + cut.blocks - 1) / cut.blocks);
    const long long begin = per * blockIdx.x, end = min(total, begin + per);
    if (blockIdx.x == 0) {                                          // what the joining kernel needs
        long long u = before;
        for (int b = r0; b < r1; ++b) {
            cut.prefix[b] = u;
            u += row_units(p, b, vhs);
        }
        if (threadIdx.x == 0) { cut.prefix[p.B] = total; cut.prefix[p.B + 1] = per; }
    }
    if (begin >= total) return;
    if (begin >= before && begin < before + mine) {                 // exactly one thread
        long long u = before;
        for (int b = r0; b < r1; ++b) {
            const long long k = row_units(p, b, vhs);
            if (begin < u + k) { sh_b = b; sh_rest = begin - u; break; }
            u += k;
        }
    }
    Ring rg = Piece<KT, QT, D, ROWS, false>::begin(&map, smem, sh_bars, &sh_abort);   // (a barrier of the block)
    int b = sh_b;
    long long rest = sh_rest, left = end - begin;                   // units into the row, units still to do
    bool first = true;
    while (left > 0 && b < p.B) {
        const int n = row_keys(p, b), tiles = row_tiles<kTile>(p, n), units = tiles + kStart;
        if (tiles == 0 || rest >= static_cast<long long>(units) * vhs) { ++b; rest = 0; continue; }   // an empty row, or this one is done
        const int vh = static_cast<int>(rest / units), u = static_cast<int>(rest - static_cast<long long>(vh) * units);
        const int k = static_cast<int>(min(static_cast<long long>(units - u), left)), t = max(0, u - kStart), m = u + k - kStart - t;   // tiles [t, t + m)
        if (m > 0) {
            const int tb = first_key(p, n) / kTile + t;
            const int slot = m == tiles ? -1 : 2 * static_cast<int>(blockIdx.x) + (first ? 0 : 1);
            if (!Piece<KT, QT, D, ROWS, false>::run(p, cut, b, vh, n, tb, tb + m, groups, slot, rg, sh_ml)) break;
            first = false;
        }
        rest += k;
        left -= k;
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the joining kernel may take its place (it waits for this one's end)
    Piece<KT, QT, D, ROWS, false>::end(p, &sh_abort);
}

// Joins the pieces of one row and query head, and writes the outputs of empty rows.  The pieces of a row come in the order of their blocks, so
// the sums do not depend on which block ended first.
template <int KT, typename QT, int D, int ROWS>
__global__ void __launch_bounds__(D / 4) paged_attention_join_kernel(PagedAttention p, Cut cut, int groups) {
    __shared__ float sh_f[D / 4];
    const int d = 4 * threadIdx.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");             // until all blocks of the kernel before are done and what they wrote is there
    const int G = p.Hq / p.kv.heads, b = blockIdx.y, h = blockIdx.x, kvh = h / G, vhs = p.kv.heads * groups, vh = kvh * groups + (h - kvh * G) / ROWS, row = (h - kvh * G) % ROWS;
    const long long u = cut.prefix[b], units = (cut.prefix[b + 1] - u) / vhs, per = cut.prefix[p.B + 1], u0 = u + vh * units;
    if (units == 0) {
        Piece<KT, QT, D, ROWS, false>::finish(p, b, h, d, -INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f));
        return;
    }
    const int c0 = static_cast<int>((u0 + kStart) / per), c1 = static_cast<int>((u0 + units - 1) / per);   // blocks of its first and last tile
    if (c0 == c1) return;
    auto slot = [&](int c) { return static_cast<int64_t>(2 * c + (c == c0 && c0 * per < u0 ? 1 : 0)); };
    float mm = -INFINITY, ll = 0.f;
    for (int c = c0; c <= c1; ++c) mm = fmaxf(mm, cut.part_ml[slot(c) * ROWS + row].x);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int base = c0; base <= c1; base += D / 4) {
        __syncthreads();
        const int c = base + threadIdx.x;
        if (c <= c1) {
            const float2 v = cut.part_ml[slot(c) * ROWS + row];
            sh_f[threadIdx.x] = v.x == -INFINITY ? 0.f : ex2(v.x - mm);
        }
        __syncthreads();
        const int cnt = min(D / 4, c1 + 1 - base);
        for (int i = 0; i < cnt; ++i) {
            const float f = sh_f[i];
            const float4 o = *reinterpret_cast<const float4*>(cut.part_o + (slot(base + i) * ROWS + row) * D + d);
            ll += f * cut.part_ml[slot(base + i) * ROWS + row].y;
            acc.x += f * o.x; acc.y += f * o.y; acc.z += f * o.z; acc.w += f * o.w;
        }
    }
    Piece<KT, QT, D, ROWS, false>::finish(p, b, h, d, mm, ll, acc);
}

// The pages as a tensor of five dimensions (element, place, head, key / value, page), copied in boxes of 16 places.  Strides may come in any order.
const char* page_map(CUtensorMap* map, const KvPages& kv, int box_elements, int pitch) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static Encode encode = [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) return static_cast<Encode>(nullptr);
        return reinterpret_cast<Encode>(ptr);
    }();
    if (!encode) return "paged_attention: cuTensorMapEncodeTiled is not available";
    const uint64_t es = kv.type == kKvE4m3 ? 1 : 2;
    const cuuint64_t dims[5] = {static_cast<cuuint64_t>(kv.dim), static_cast<cuuint64_t>(kv.page_size), static_cast<cuuint64_t>(kv.heads), 2, static_cast<cuuint64_t>(kv.num_pages)};
    // a dimension of one entry may have any stride; the map wants a multiple of 16 bytes
    const int64_t given[4] = {kv.tok_stride, kv.head_stride, kv.kv_stride, kv.page_stride};
    cuuint64_t strides[4];
    for (int i = 0; i < 4; ++i) strides[i] = dims[i + 1] == 1 ? kv.dim * es : given[i] * es;
    const cuuint32_t box[5] = {static_cast<cuuint32_t>(box_elements), kStep, 1, 1, 1}, one[5] = {1, 1, 1, 1, 1};
    const CUresult r = encode(map, es == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 5, kv.data, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              pitch == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? nullptr : "paged_attention: the cache's strides do not make a tensor map";
}

int64_t prefix_floats(int B) { return 4 * ((static_cast<int64_t>(B) + 3) / 2); }   // of Cut::prefix; what follows starts on 16 bytes

template <int KT, typename QT, int D, int ROWS>
const char* launch(const PagedAttention& p, const PagedAttentionPlan& plan, float* ws, cudaStream_t s) {
    using S = Shape<KT, D, ROWS, false>;
    using W = Shape<KT, D, ROWS, true>;
    static std::atomic<uint64_t> raised_deep{0}, raised_whole{0}, raised_shared{0};
    CUtensorMap map;
    if (const char* e = page_map(&map, p.kv, S::BOXEL, S::PITCH)) return e;
    if (plan.whole && plan.deep) {
        auto k = paged_attention_whole_kernel<KT, QT, D, ROWS, true>;
        if (!raise_smem_limit(reinterpret_cast<const void*>(k), W::SMEM, raised_deep)) return "paged_attention: the shared-memory limit could not be raised";
        k<<<plan.blocks, W::WARPS * 32, W::SMEM, s>>>(map, p, plan.head_groups);
    } else if (plan.whole) {
        auto k = paged_attention_whole_kernel<KT, QT, D, ROWS, false>;
        if (!raise_smem_limit(reinterpret_cast<const void*>(k), S::SMEM, raised_whole)) return "paged_attention: the shared-memory limit could not be raised";
        k<<<plan.blocks, S::WARPS * 32, S::SMEM, s>>>(map, p, plan.head_groups);
    } else {
        auto k = paged_attention_shared_kernel<KT, QT, D, ROWS>;
        if (!raise_smem_limit(reinterpret_cast<const void*>(k), S::SMEM, raised_shared)) return "paged_attention: the shared-memory limit could not be raised";
        Cut cut;
        cut.blocks = plan.blocks;
        cut.min_units = 4;
        cut.prefix = reinterpret_cast<long long*>(ws);
        cut.part_ml = reinterpret_cast<float2*>(ws + prefix_floats(p.B));
        cut.part_o = reinterpret_cast<float*>(cut.part_ml + 2 * static_cast<int64_t>(plan.blocks) * ROWS);
        k<<<plan.blocks, kSharing * 32, S::SMEM, s>>>(map, p, cut, plan.head_groups);
        if (cudaError_t e = cudaGetLastError(); e != cudaSuccess) return cudaGetErrorString(e);
        cudaLaunchConfig_t cfg{};
        cudaLaunchAttribute early[1];
        early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // launched while the kernel before runs: saves the launch's own time
        early[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.gridDim = dim3(p.Hq, p.B);
        cfg.blockDim = dim3(D / 4);
        cfg.stream = s;
        cfg.attrs = early;
        cfg.numAttrs = 1;
        if (cudaError_t e = cudaLaunchKernelEx(&cfg, paged_attention_join_kernel<KT, QT, D, ROWS>, p, cut, plan.head_groups); e != cudaSuccess) {
            cudaGetLastError();
            return cudaGetErrorString(e);
        }
    }
    if (cudaError_t e = cudaGetLastError(); e != cudaSuccess) return cudaGetErrorString(e);
    return nullptr;
}

template <int KT, typename QT>
const char* launch_dim(const PagedAttention& p, const PagedAttentionPlan& plan, float* ws, cudaStream_t s) {
    if (p.kv.dim == 64) return plan.rows == 16 ? launch<KT, QT, 64, 16>(p, plan, ws, s) : launch<KT, QT, 64, 8>(p, plan, ws, s);
    if (p.kv.dim == 128) return plan.rows == 16 ? launch<KT, QT, 128, 16>(p, plan, ws, s) : launch<KT, QT, 128, 8>(p, plan, ws, s);
    return launch<KT, QT, 256, 8>(p, plan, ws, s);
}

}  // namespace

namespace {
template <int KT> int blocks_per_sm(int dim, int rows) {
    if (dim == 64) return rows == 16 ? Shape<KT, 64, 16, false>::PER_SM : Shape<KT, 64, 8, false>::PER_SM;
    if (dim == 128) return rows == 16 ? Shape<KT, 128, 16, false>::PER_SM : Shape<KT, 128, 8, false>::PER_SM;
    return Shape<KT, 256, 8, false>::PER_SM;
}
}  // namespace

PagedAttentionPlan paged_attention_plan(int B, int Hq, int Hkv, int dim, int kv_type, int64_t max_keys, int num_sms) {
    PagedAttentionPlan plan{};
    const int G = Hq / Hkv;
    // Eight rows of a product suffice up to eight query heads a key head.  Heads of 256 stay with eight: sixteen rows of 256 outputs and queries
    // would not fit a thread's registers.  With more query heads the cache is read once for each eight: 64 over 4 heads of 256, 64 rows of 100 to 4096
    // keys, bf16, 178 us where 8 over 4 take 94.
    plan.rows = G > 8 && dim <= 128 ? 16 : 8;
    plan.head_groups = (G + plan.rows - 1) / plan.rows;
    const int64_t pairs = static_cast<int64_t>(B) * Hkv * plan.head_groups, tiles = (max_keys + kTile - 1) / kTile;
    const int most = num_sms * (kv_type == kKvE4m3 ? blocks_per_sm<kKvE4m3>(dim, plan.rows) : blocks_per_sm<kKvBf16>(dim, plan.rows));
    // Rows that cannot hold more than 1024 keys (the table's width; nothing here knows their lengths) are not split.  32 query heads over 8 key heads of
    // 128, bf16, us whole / split:
    //     rows      50 to 1000 keys   512 keys      1000 keys
    //        1       10.3 / 10.2      7.3 / 10.0    10.6 / 10.2
    //        8       10.3 / 12.3      7.5 / 11.5    10.7 / 12.8
    //       32       16.4 / 17.5     11.1 / 15.9    24.9 / 29.9
    //       64       37.6 / 32.0     29.0 / 30.2    50.6 / 50.3
    //      128       55.4 / 53.5     49.1 / 52.2    85.6 / 90.3
    //      256       95.1 / 97.3     87.1 / 94.9   157.6 / 171.3
    // The split wins where rows of uneven length are one or two for each block.  Longer rows differ more in length, which only the split evens out.
    plan.whole = tiles <= 16;
    plan.deep = plan.whole && pairs <= num_sms;
    const int64_t work = plan.whole ? pairs : pairs * tiles;
    plan.blocks = static_cast<int>(work < most ? (work > 0 ? work : 1) : most);
    plan.workspace_floats = plan.whole ? 0 : prefix_floats(B) + static_cast<int64_t>(plan.blocks) * 2 * plan.rows * (dim + 2);
    return plan;
}

const char* paged_attention(const PagedAttention& p, const PagedAttentionPlan& plan, float* ws, cudaStream_t s) {
    if (p.B <= 0) return nullptr;
    const bool qb = p.q_type == kKvBf16;
    if (p.kv.type == kKvBf16) return launch_dim<kKvBf16, __nv_bfloat16>(p, plan, ws, s);
    if (p.kv.type == kKvFp16) return launch_dim<kKvFp16, __half>(p, plan, ws, s);
    return qb ? launch_dim<kKvE4m3, __nv_bfloat16>(p, plan, ws, s) : launch_dim<kKvE4m3, __half>(p, plan, ws, s);
}

}  // namespace sg
