// kv8_args.h -- arguments of the attention kernels over the 8-bit pool.
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

namespace msgl {
// An item that several CTAs share: CTAs first .. last; query row of out, kv head, rows x heads of the group.
struct Kv8Shared {
    int first, last;
    int64_t q_row;
    int h, rows;
};

struct Kv8AttnArgs {
    const __nv_bfloat16* q;
    const uint8_t *kv8, *scales;
    int64_t num_pages;
    const int* page_table;
    int max_pages, max_len;
    const int *seq_lens, *q_indptr;
    int num_reqs, total_q, max_q_len, hq, hkv;
    float sl2e;  // scale * log2(e)
    __nv_bfloat16* out;
    float *ws_o, *ws_ml;
    struct Kv8Shared* ws_shared;  // by CTA: the item that it goes on with from the CTA before
    int min_units;   // of a CTA, at least
    int* err;
};
}  // namespace msgl
