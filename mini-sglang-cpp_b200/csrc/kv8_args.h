// kv8_args.h -- arguments of the attention kernels over the 8-bit pool.
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

namespace msgl {
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
    int* ws_count;
    int row_blocks;  // of a request, at most
    int min_units;   // of a CTA, at least
    int* err;
};
}  // namespace msgl
