// Writing new tokens into a paged key/value cache, and copying pages through all of its layers.
//
// Both only move data, so HBM bounds them: an appended token is read once and written once (2 * 2 * heads * dim elements), a copied page
// likewise, and nothing else is touched.  Every access is a 16-byte vector, four of them under way in each thread.
//
// Measured (B200, a copy runs at 6.55 TB/s): prompts of 21 300 tokens in all, 8 heads of 128, bf16, 31 us in a graph, 5.6 TB/s; 64 single tokens 2.5 us,
// which is a launch; 128 pages of 256 KB through 36 layers 404 us, 6.0 TB/s; a fork of 7 pages of 64 KB through 28 layers 5.9 us, where its
// dependent look-ups (two page numbers, all pairs, then the page) take half of the time.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "paged_kv.h"

namespace sg {

namespace {

// Page and place of new token t of row b.  False: the token is padding, or its place does not exist (reported).
__device__ __forceinline__ bool locate_token(const KvAppend& p, int b, int t, int& page, int& place) {
    const int count = p.count ? min(p.count[b], p.T) : p.T;
    if (t >= count) return false;
    const int64_t pos = static_cast<int64_t>(p.start[b]) + t;
    if (pos < 0 || pos >= static_cast<int64_t>(p.table_width) * p.kv.page_size) {   // (at most 2^30)
        atomicExch(p.error_flag, kErrBadPage);
        return false;
    }
    const unsigned slot = static_cast<unsigned>(pos) / static_cast<unsigned>(p.kv.page_size);
    page = p.table[b * p.table_stride + slot];
    place = static_cast<int>(pos) - static_cast<int>(slot) * p.kv.page_size;
    if (page < 0 || page >= p.kv.num_pages) {
        atomicExch(p.error_flag, kErrBadPage);
        return false;
    }
    return true;
}

// ------------------------------------------------------------------------------------------ same type: 16-byte copies
// A block takes kTokens tokens of one row (blockIdx.y): it looks up where they go once, in shared memory, while the first vectors are on their
// way, then its threads copy the tokens' 16-byte vectors (key heads, then value heads of each), kPerThread in flight each.
constexpr int kAppendThreads = 256, kAppendPerThread = 4;

template <int kTokens>
__global__ void __launch_bounds__(kAppendThreads) kv_append_copy_kernel(KvAppend p, int vec_per_head, int elem_bytes) {
    __shared__ int64_t sh_to[kTokens];                             // byte offset of the token's first key head, or -1: not written
    const int b = blockIdx.y, t0 = blockIdx.x * kTokens;
    const int count = p.count ? min(p.count[b], p.T) : p.T;
    if (t0 >= count) return;
    const int per_token = 2 * p.kv.heads * vec_per_head, tokens = min(kTokens, count - t0), total = tokens * per_token;
    const char* from[2];
    int64_t h_bytes[2], t_bytes[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        from[w] = static_cast<const char*>(p.src[w]) + (b * p.b_stride[w] + t0 * p.t_stride[w]) * elem_bytes;
        h_bytes[w] = p.h_stride[w] * elem_bytes;
        t_bytes[w] = p.t_stride[w] * elem_bytes;
    }
    if (static_cast<int>(threadIdx.x) < tokens) {
        int page, place;
        sh_to[threadIdx.x] = locate_token(p, b, t0 + threadIdx.x, page, place) ? (page * p.kv.page_stride + place * p.kv.tok_stride) * elem_bytes : -1;
    }
    char* base = static_cast<char*>(p.kv.data);
    bool located = false;
    for (int first = threadIdx.x; first - static_cast<int>(threadIdx.x) < total; first += kAppendThreads * kAppendPerThread) {
        uint4 v[kAppendPerThread];
        int token[kAppendPerThread];
        int64_t off[kAppendPerThread];
#pragma unroll
        for (int i = 0; i < kAppendPerThread; ++i) {
            const int item = first + i * kAppendThreads;
            token[i] = -1;
            if (item >= total) continue;
            token[i] = static_cast<unsigned>(item) / static_cast<unsigned>(per_token);
            const int r = item - token[i] * per_token, row = static_cast<unsigned>(r) / static_cast<unsigned>(vec_per_head), vec = r - row * vec_per_head;
            const int w = row >= p.kv.heads, h = row - w * p.kv.heads;
            v[i] = *reinterpret_cast<const uint4*>(from[w] + token[i] * t_bytes[w] + h * h_bytes[w] + vec * 16);
            off[i] = (w * p.kv.kv_stride + h * p.kv.head_stride) * elem_bytes + vec * 16;
        }
        if (!located) {                                            // (all threads come here the same number of times)
            __syncthreads();
            located = true;
        }
#pragma unroll
        for (int i = 0; i < kAppendPerThread; ++i)
            if (token[i] >= 0 && sh_to[token[i]] >= 0) *reinterpret_cast<uint4*>(base + sh_to[token[i]] + off[i]) = v[i];
    }
}

// ------------------------------------------------------------------------------------------ to e4m3, one scale a token and head
template <typename T> __device__ __forceinline__ void load8(const T* p, float (&f)[8]);
template <> __device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&f)[8]) {
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    const __nv_bfloat162* t = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 x = __bfloat1622float2(t[i]); f[2 * i] = x.x; f[2 * i + 1] = x.y; }
}
template <> __device__ __forceinline__ void load8<__half>(const __half* p, float (&f)[8]) {
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    const __half2* t = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 x = __half22float2(t[i]); f[2 * i] = x.x; f[2 * i + 1] = x.y; }
}
template <> __device__ __forceinline__ void load8<float>(const float* p, float (&f)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

// LANES lanes hold one head's row, sixteen elements each (lanes behind the row's end hold zeros): s = max |x| / 448 (at least 2^-100, so that
// 1/s and log2 s stay finite; 1 for a row of zeros), q = e4m3(x / s).  The one rounding is the cache's own type, at most 2^-4 of a value.
// A block takes kTokens tokens of one row, like the copy above, and looks up their places once; a thread has kE4m3PerThread heads under way.
// Instructions bound it, not HBM: sixteen elements a lane, so that addresses, exchanges and divisions serve more of them, took 68 us where eight
// took 83 (32768 tokens, 8 heads of 128 from bf16: 3.0 TB/s), four heads under way instead of two 89.
constexpr int kE4m3PerThread = 2;

// x / s by r = 1 / s, with one correction of the remainder (Markstein's method): within 2^-46 of the quotient before its rounding to fp32.  (With
// divisions 32768 tokens with 8 heads of 128 took 91 us, at eight elements a lane, and 83 with this.)
__device__ __forceinline__ float quotient(float x, float s, float r) {
    const float q = __fmul_rn(x, r);
    return copysignf(fmaf(fmaf(-q, s, x), r, q), x);               // (the sign of a zero, too)
}

template <typename T, int LANES, int kTokens>
__global__ void __launch_bounds__(kAppendThreads) kv_append_e4m3_kernel(KvAppend p) {
    __shared__ int sh_page[kTokens], sh_place[kTokens];            // page -1: not written
    const int b = blockIdx.y, t0 = blockIdx.x * kTokens;
    const int count = p.count ? min(p.count[b], p.T) : p.T;
    if (t0 >= count) return;
    const int tokens = min(kTokens, count - t0), heads2 = 2 * p.kv.heads, total = tokens * heads2;
    constexpr int GROUPS = kAppendThreads / LANES;
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const unsigned mask = ((1u << LANES) - 1) << (threadIdx.x % 32 / LANES * LANES);
    const bool inside = lane * 16 < p.kv.dim;
    if (static_cast<int>(threadIdx.x) < tokens) {
        int page, place;
        const bool there = locate_token(p, b, t0 + threadIdx.x, page, place);
        sh_page[threadIdx.x] = there ? page : -1;
        sh_place[threadIdx.x] = there ? place : 0;
    }
    bool located = false;
    for (int first = 0; first < total; first += GROUPS * kE4m3PerThread) {
        float f[kE4m3PerThread][16];
        int token[kE4m3PerThread], head[kE4m3PerThread];
#pragma unroll
        for (int k = 0; k < kE4m3PerThread; ++k) {
            const int item = first + k * GROUPS + group;
            token[k] = -1;
            if (item >= total) continue;
            token[k] = static_cast<unsigned>(item) / static_cast<unsigned>(heads2);
            head[k] = item - token[k] * heads2;
            const int which = head[k] >= p.kv.heads, h = head[k] - which * p.kv.heads;
            const T* from = static_cast<const T*>(p.src[which]) + b * p.b_stride[which] + (t0 + token[k]) * p.t_stride[which] + h * p.h_stride[which] + lane * 16;
            if (inside) {
                load8<T>(from, *reinterpret_cast<float(*)[8]>(f[k]));
                load8<T>(from + 8, *reinterpret_cast<float(*)[8]>(f[k] + 8));
            }
        }
        if (!located) {                                            // (all threads come here the same number of times)
            __syncthreads();
            located = true;
        }
#pragma unroll
        for (int k = 0; k < kE4m3PerThread; ++k) {
            float amax = 0.f;
            if (inside && token[k] >= 0) {
#pragma unroll
                for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(f[k][i]));
            }
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(mask, amax, o));
            if (token[k] < 0 || sh_page[token[k]] < 0) continue;
            const float s = amax > 0.f ? fmaxf(amax / 448.f, 0x1p-100f) : 1.f, r = 1.f / s;
            const float divisor = fminf(s, 1e37f);                 // an infinite row: its finite elements become zeros, the others NaN
            const int which = head[k] >= p.kv.heads, h = head[k] - which * p.kv.heads;
            const int64_t page = sh_page[token[k]];
            const int place = sh_place[token[k]];
            if (inside) {
                uint4 q;
                __nv_fp8x2_storage_t* q2 = reinterpret_cast<__nv_fp8x2_storage_t*>(&q);
#pragma unroll
                for (int i = 0; i < 8; ++i) q2[i] = __nv_cvt_float2_to_fp8x2(make_float2(quotient(f[k][2 * i], divisor, r), quotient(f[k][2 * i + 1], divisor, r)), __NV_SATFINITE, __NV_E4M3);
                *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.kv.data) + page * p.kv.page_stride + which * p.kv.kv_stride + h * p.kv.head_stride + place * p.kv.tok_stride + lane * 16) = q;
            }
            if (lane == 0) p.kv.scales[page * p.kv.s_page_stride + which * p.kv.s_kv_stride + h * p.kv.s_head_stride + place] = s;
        }
    }
}

template <typename T, int LANES>
void launch_e4m3_lanes(const KvAppend& p, cudaStream_t s) {
    if (p.T < 8) kv_append_e4m3_kernel<T, LANES, 1><<<dim3(p.T, p.B), kAppendThreads, 0, s>>>(p);
    else kv_append_e4m3_kernel<T, LANES, 8><<<dim3((p.T + 7) / 8, p.B), kAppendThreads, 0, s>>>(p);
}
template <typename T>
void launch_e4m3(const KvAppend& p, cudaStream_t s) {
    const int need = p.kv.dim / 16;                                // (16-byte vectors: a multiple of 16)
    if (need <= 4) launch_e4m3_lanes<T, 4>(p, s);
    else if (need <= 8) launch_e4m3_lanes<T, 8>(p, s);
    else launch_e4m3_lanes<T, 16>(p, s);
}

}  // namespace

void kv_append(const KvAppend& p, cudaStream_t s) {
    if (p.B <= 0 || p.T <= 0) return;
    if (p.kv.type != kKvE4m3) {
        const int es = p.kv.type == kKvFp32 ? 4 : 2;
        const int vec = p.kv.dim * es / 16;
        // one token a block for single tokens, whose rows are what there is to spread; eight for prompts, whose look-ups they share
        if (p.T < 8) kv_append_copy_kernel<1><<<dim3(p.T, p.B), kAppendThreads, 0, s>>>(p, vec, es);
        else kv_append_copy_kernel<8><<<dim3((p.T + 7) / 8, p.B), kAppendThreads, 0, s>>>(p, vec, es);
    } else if (p.src_type == kKvBf16) launch_e4m3<__nv_bfloat16>(p, s);
    else if (p.src_type == kKvFp16) launch_e4m3<__half>(p, s);
    else launch_e4m3<float>(p, s);
}

// ------------------------------------------------------------------------------------------ pages
// blockIdx.y: pair of pages, blockIdx.z: group of layers, blockIdx.x: 16 KB piece of a page (the pages' pieces first, then the scales').
// The pairs of one call run in any order, so no page may be written that another pair reads or writes: every block looks its target up among
// all sources and targets and leaves a pair that breaks this (or lies outside the cache) undone, with the error word set.
constexpr int kCopyThreads = 256, kCopyPerThread = 4, kCopyPiece = kCopyThreads * kCopyPerThread * 16;

__global__ void __launch_bounds__(kCopyThreads) kv_copy_pages_kernel(KvCopy p, int pieces0, int layers_per_block) {
    const int pair = blockIdx.y;
    const int from = p.src[pair], to = p.dst[pair];
    const bool outside = from < 0 || from >= p.num_pages || to < 0 || to >= p.num_pages;
    int clash = 0;
    for (int j = threadIdx.x; j < p.n; j += kCopyThreads) clash |= j != pair && (p.dst[j] == to || (p.src[j] == to && from != to));
    clash = __syncthreads_or(clash);
    if (outside || clash) {
        if (threadIdx.x == 0) atomicExch(p.error_flag, outside ? kErrBadPage : kErrPageOverlap);
        return;
    }
    if (from == to) return;                                        // stays as it is, and others may read it
    const int part = static_cast<int>(blockIdx.x) >= pieces0;
    const int64_t off = static_cast<int64_t>(part ? blockIdx.x - pieces0 : blockIdx.x) * kCopyPiece;
    const int64_t left = p.page_bytes[part] - off;
    const int l0 = blockIdx.z * layers_per_block, l1 = min(p.layers, l0 + layers_per_block);
    for (int l = l0; l < l1; ++l) {
        const uint8_t* a = p.base[part] + l * p.layer_bytes[part] + from * p.page_stride_bytes[part] + off;
        uint8_t* b = p.base[part] + l * p.layer_bytes[part] + to * p.page_stride_bytes[part] + off;
        uint4 v[kCopyPerThread];
#pragma unroll
        for (int i = 0; i < kCopyPerThread; ++i) {
            const int x = (i * kCopyThreads + threadIdx.x) * 16;
            if (x < left) v[i] = *reinterpret_cast<const uint4*>(a + x);
        }
#pragma unroll
        for (int i = 0; i < kCopyPerThread; ++i) {
            const int x = (i * kCopyThreads + threadIdx.x) * 16;
            if (x < left) *reinterpret_cast<uint4*>(b + x) = v[i];
        }
    }
}

void kv_copy_pages(const KvCopy& p, int num_sms, cudaStream_t s) {
    if (p.n <= 0 || p.layers <= 0) return;
    const int pieces0 = static_cast<int>((p.page_bytes[0] + kCopyPiece - 1) / kCopyPiece);
    const int pieces1 = p.base[1] ? static_cast<int>((p.page_bytes[1] + kCopyPiece - 1) / kCopyPiece) : 0;
    // one layer a block while that is what fills the GPU (eight blocks an SM); beyond it a block takes several, and looks its pair up once
    const int64_t per_layer = static_cast<int64_t>(pieces0 + pieces1) * p.n;
    int groups = static_cast<int>((static_cast<int64_t>(num_sms) * 8 * 4 + per_layer - 1) / per_layer);
    groups = groups < 1 ? 1 : groups > p.layers ? p.layers : groups;
    const int layers_per_block = (p.layers + groups - 1) / groups;
    groups = (p.layers + layers_per_block - 1) / layers_per_block;
    kv_copy_pages_kernel<<<dim3(pieces0 + pieces1, p.n, groups), kCopyThreads, 0, s>>>(p, pieces0, layers_per_block);
}

}  // namespace sg
