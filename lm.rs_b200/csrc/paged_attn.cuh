// paged_attn.cuh -- attention of the rows of many sequences over their pages and over a prefix that all of them share.
#pragma once
#include "paged.h"
#include "paged_rows.cuh"

namespace lmrs {
namespace paged {

template <typename T> struct AttnParams {
    Batch batch;
    Rows<const T> q;
    Rows<T> out;
    const T *k, *v;
    int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;
    int kv_heads, q_heads, head_size;
    float scale, softcap;
    float* lse;
};

// CTA = a row and a head, its keys 128 at a time with the running maximum and sum: the plainest form
template <typename T>
__global__ void __launch_bounds__(128) paged_attention_kernel(const __grid_constant__ AttnParams<T> p) {
    __shared__ int found;
    __shared__ float q[256], w[128], red[4];
    __shared__ int64_t at[128];
    const int64_t r = blockIdx.x;
    const int h = blockIdx.y, g = h / (p.q_heads / p.kv_heads), D = p.head_size, t = threadIdx.x;
    const int b = seq_of_row(p.batch, r, &found);
    if (b < 0) return;
    const Span s = span_of(p.batch, b);
    const int64_t index = (int64_t)s.len - s.count + (r - s.first);
    const int prefix = index < 0 ? 0 : p.batch.prefix_len;
    const int64_t n_own = index < 0 ? 0 : min((int64_t)p.batch.table_len * p.batch.page_size, index + 1);
    const int ps = p.batch.page_size, prefix_pages = (p.batch.prefix_len + ps - 1) / ps;
    for (int e = t; e < D; e += 128) q[e] = to_f(p.q.data[r * p.q.row + h * p.q.head + e]);
    float m = -INFINITY, l = 0.0f, acc[2] = {0.0f, 0.0f};
    bool any = false;
    for (int64_t x0 = 0; x0 < prefix + n_own; x0 += 128) {
        __syncthreads();
        const int64_t x = x0 + t;
        const int64_t slot = x < prefix            ? slot_of(p.batch.prefix, prefix_pages, ps, p.batch.pages, (int)x)
                             : x < prefix + n_own ? slot_of(p.batch.tables + b * p.batch.table_stride, p.batch.table_len, ps, p.batch.pages, (int)(x - prefix))
                                                  : -1;
        const int64_t page = slot / ps, place = slot - page * ps;
        float a = -INFINITY;
        if (slot >= 0) {
            const T* k = p.k + page * p.k_page + place * p.k_slot + g * p.k_head;
            a = 0.0f;
            for (int e = 0; e < D; e++) a = fmaf(q[e], to_f(k[e]), a);
            a *= p.scale;
            if (p.softcap > 0.0f) a = p.softcap * tanhf(a / p.softcap);
        }
        at[t] = slot < 0 ? -1 : page * p.v_page + place * p.v_slot + g * p.v_head;
        any |= slot >= 0;
        float top = a;
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
        if ((t & 31) == 0) red[t >> 5] = top;
        __syncthreads();
        const float mn = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m), base = mn == -INFINITY ? 0.0f : mn;
        const float corr = expf(m - base);   // (m -infinity: 0)
        w[t] = slot < 0 ? 0.0f : expf(a - base);
        m = mn;
        __syncthreads();
        l *= corr;
        for (int i = 0; i < 128; i++) l += w[i];
        for (int c = 0; c < 2; c++)
            if (t + 128 * c < D) {
                acc[c] *= corr;
                for (int i = 0; i < 128; i++)
                    if (at[i] >= 0) acc[c] = fmaf(w[i], to_f(p.v[at[i] + t + 128 * c]), acc[c]);
            }
    }
    any = __syncthreads_or(any);
    for (int c = 0; c < 2; c++)
        if (t + 128 * c < D) p.out.data[r * p.out.row + h * p.out.head + t + 128 * c] = from_f<T>(any ? acc[c] / l : 0.0f);
    if (t == 0 && p.lse) p.lse[r * p.q_heads + h] = any ? logf(l) + (m == -INFINITY ? 0.0f : m) : -INFINITY;
}

}  // namespace paged
}  // namespace lmrs
