// paged.h -- what the kernels over many sequences share (paged_rows.cuh: rotary positions and appending; paged_attn.cuh: attention):
// the batch as the kernels see it, and how a row finds its sequence and a token its place in the pages.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/lmrs_b200.h"

namespace lmrs {
int set_error(const std::string& m);   // what lmrs_b200_last_error returns; gives 1

namespace paged {

#define PG_DEVINL __device__ __forceinline__

PG_DEVINL float to_f(float v) { return v; }
PG_DEVINL float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
PG_DEVINL float to_f(__half v) { return __half2float(v); }
template <typename T> PG_DEVINL T from_f(float v);
template <> PG_DEVINL float from_f<float>(float v) { return v; }
template <> PG_DEVINL __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> PG_DEVINL __half from_f<__half>(float v) { return __float2half_rn(v); }

// lmrs_b200_batch_t with the number of rows in the call's arrays and the bounds of the pool
struct Batch {
    const int *lens, *rows, *tables, *prefix;
    int64_t table_stride;
    int seqs, table_len, prefix_len, pages, page_size;
    int64_t n_rows;
};
// Everything that comes from device memory is held against the arrays' bounds where it is read: rows of sequence b, and what it holds
struct Span { int64_t first; int count, len; };
PG_DEVINL Span span_of(const Batch& s, int b) {
    Span r;
    if (s.rows) {
        const int64_t lo = s.rows[b], hi = s.rows[b + 1];
        r.first = lo < 0 ? 0 : lo > s.n_rows ? s.n_rows : lo;
        const int64_t end = hi < r.first ? r.first : hi > s.n_rows ? s.n_rows : hi;
        r.count = (int)(end - r.first);
    } else {
        r.first = b;
        r.count = 1;
    }
    r.len = s.lens[b];
    return r;
}
// the slot (page * page_size + place in it) of token x of a list of pages, -1 where there is none
PG_DEVINL int64_t slot_of(const int* table, int table_len, int page_size, int pages, int x) {
    if (x < 0) return -1;
    const int p = x / page_size;
    if (p >= table_len) return -1;
    const int page = table[p];
    return page < 0 || page >= pages ? -1 : (int64_t)page * page_size + (x - p * page_size);
}

}  // namespace paged
}  // namespace lmrs
