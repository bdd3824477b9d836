// What the kernels around the paged key-value cache share.
#pragma once

#include <cuda_runtime.h>

namespace mb {
namespace paged {

struct Strides2 {
    long long token, head;   // elements
};
struct Strides3 {
    long long page, token, head;
};

struct AttentionArgs {
    int tokens, requests, heads, kv_heads, head_dim, width, pages, page_shift, zero_rest;
    float scale;
    Strides2 q, k, v;
    Strides3 kpool, vpool;
    const unsigned short *query, *key, *value;
    const unsigned short *key_pages, *value_pages;   // mb_paged_attention writes to the places of new tokens
    const int *table, *lengths, *index;
    unsigned short* out;
    int* status;
};

}  // namespace paged
}  // namespace mb
