// Paged key/value cache: writing new tokens, copying pages, attention of one new token a sequence.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace sg {

enum KvType { kKvBf16 = 0, kKvFp16 = 1, kKvE4m3 = 2, kKvFp32 = 3 };

// One layer's pages, [page, key / value, head, place in the page, element]: strides in elements, elements contiguous, rows 16-byte aligned.
// An e4m3 cache has one fp32 scale for each page, key / value, head and place (places contiguous).
struct KvPages {
    void* data;
    float* scales;
    int64_t page_stride, kv_stride, head_stride, tok_stride;
    int64_t s_page_stride, s_kv_stride, s_head_stride;
    int num_pages, heads, page_size, dim, type;
};

struct KvAppend {
    KvPages kv;
    const void* src[2];                              // keys, values: [B, T, heads, dim], elements contiguous, rows 16-byte aligned
    int64_t b_stride[2], t_stride[2], h_stride[2];   // in elements
    int src_type;                                    // the cache's type, or any but e4m3 for an e4m3 cache
    const int* table;                                // [B, table_width] page numbers
    int64_t table_stride;
    int table_width;
    const int* start;                                // [B] position of a row's first new token
    const int* count;                                // [B] new tokens of a row, or null: T
    int B, T;
    int* error_flag;
};
void kv_append(const KvAppend& p, cudaStream_t s);

struct KvCopy {
    uint8_t* base[2];                                // pages, scales (or null)
    int64_t layer_bytes[2], page_stride_bytes[2], page_bytes[2];
    const int* src;
    const int* dst;
    int n, layers, num_pages;
    int* error_flag;
};
void kv_copy_pages(const KvCopy& p, int num_sms, cudaStream_t s);

struct PagedAttention {
    KvPages kv;
    const void* q;                                   // [B, Hq, dim], elements contiguous, rows 16-byte aligned; the cache's type, or bf16 / fp16 with an e4m3 cache
    int64_t q_b_stride, q_h_stride;                  // in elements
    int q_type;
    const int* table;
    int64_t table_stride;
    int table_width;
    const int* lengths;                              // [B] keys of each row, the new token's own among them
    const float* sinks;                              // [Hq] or null
    void* out;                                       // [B, Hq, dim] of q's type
    float* lse;                                      // [B, Hq] or null
    int B, Hq, window;
    float scale, softcap;
    int* error_flag;
};
// How a problem is cut: `blocks` blocks take whole rows and heads, one after the other (`whole`; `deep`: with more warps, few rows), or share all tiles of
// 64 keys evenly, and a second kernel joins the pieces.
struct PagedAttentionPlan {
    bool whole, deep;
    int rows, blocks, head_groups;
    int64_t workspace_floats;
};
PagedAttentionPlan paged_attention_plan(int B, int Hq, int Hkv, int dim, int kv_type, int64_t max_keys, int num_sms);
const char* paged_attention(const PagedAttention& p, const PagedAttentionPlan& plan, float* workspace, cudaStream_t s);

constexpr int kErrBadPage = 8;      // a page number, position or length outside the cache
constexpr int kErrPageOverlap = 9;  // a page copied onto one that is read or written by another pair of the same call

}  // namespace sg
