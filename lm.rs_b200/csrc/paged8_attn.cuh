// paged8_attn.cuh -- attention of the rows of many sequences over pages of 8-bit codes and over a prefix that all of them share.
#pragma once
#include "paged8.h"
#include "paged_attn.cuh"

namespace lmrs {
namespace paged {

template <typename T> struct Attn8Params : AttnParams<T> {   // (k, v and their strides there stay empty)
    Pages8 c;
};

// where a key's codes and their scales are
template <typename T> PG_DEVINL const uint8_t* key_codes(const Attn8Params<T>& p, Place at, int head) { return p.c.k + at.page * p.c.k_page + at.place * p.c.k_slot + head * p.c.k_head; }
template <typename T> PG_DEVINL const uint8_t* value_codes(const Attn8Params<T>& p, Place at, int head) { return p.c.v + at.page * p.c.v_page + at.place * p.c.v_slot + head * p.c.v_head; }
template <typename T> PG_DEVINL float key_scale(const Attn8Params<T>& p, Place at, int head) { return p.c.ks[at.page * p.c.ks_page + at.place / p.c.block * p.c.ks_block + head * p.c.ks_head]; }
template <typename T> PG_DEVINL float value_scale(const Attn8Params<T>& p, Place at, int head) { return p.c.vs[at.page * p.c.vs_page + at.place / p.c.block * p.c.vs_block + head * p.c.vs_head]; }

// The simplest form: a CTA a row and head, a thread a key, then a thread a column or two
template <typename T, int FORM>
__global__ void __launch_bounds__(128) row8_kernel(const __grid_constant__ Attn8Params<T> p) {
    __shared__ float weight[128], most[4];
    __shared__ int64_t from[128];
    const int t = threadIdx.x, D = p.head_size;
    const int64_t row = blockIdx.x / p.q_heads;
    const int head = (int)(blockIdx.x - row * p.q_heads), g = head / p.group, b = seq_of_row_warp(p.batch, row);
    if (b < 0) return;
    Walk w = {};
    w.s = span_of(p.batch, b);
    const int64_t index = (int64_t)w.s.len - w.s.count + (row - w.s.first);
    const T* q = p.q.data + row * p.q.row + head * p.q.head;
    float m = -INFINITY, l = 0.0f, acc[2] = {0.0f, 0.0f};
    bool any = false;
    for (int part = index < 0 ? 2 : 0; part < 2; part++) {
        w.b = part ? b : -1;
        w.keys = part ? keys_upto(p, index) : p.batch.prefix_len;
        for (int x0 = 0; x0 < w.keys; x0 += 128) {
            const Place at = unit_place(p, w, x0 + t);
            const bool there = at.page >= 0;
            float a = -INFINITY;
            if (there) {
                const uint8_t* k = key_codes(p, at, g);
                a = 0.0f;
                for (int e = 0; e < D; e++) a = fmaf(to_f(q[e]), open_code<FORM>(k[e]), a);
                a = score2(p, a * key_scale(p, at, g));
            }
            float top = a;
            for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
            __syncthreads();
            if ((t & 31) == 0) most[t >> 5] = top;
            any = __syncthreads_or(there) || any;
            const float now = fmaxf(fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])), m), base = now == -INFINITY ? 0.0f : now, corr = ex2(m - base);
            weight[t] = there ? ex2(a - base) : 0.0f;
            from[t] = there ? value_codes(p, at, g) - p.c.v : -1;
            m = now;
            __syncthreads();
            l *= corr;
            acc[0] *= corr;
            acc[1] *= corr;
            for (int i = 0; i < 128; i++) l += weight[i];
            __shared__ float scale[128];
            scale[t] = there ? value_scale(p, at, g) : 0.0f;
            __syncthreads();
            for (int i = 0; i < 128; i++)
                for (int c = 0; c < 2; c++)
                    if (from[i] >= 0 && t + 128 * c < D) acc[c] = fmaf(weight[i] * scale[i], open_code<FORM>(p.c.v[from[i] + t + 128 * c]), acc[c]);
        }
    }
    for (int c = 0; c < 2; c++)
        if (t + 128 * c < D) p.out.data[row * p.out.row + head * p.out.head + t + 128 * c] = from_f<T>(any ? acc[c] / l : 0.0f);
    if (t == 0 && p.lse) p.lse[row * p.q_heads + head] = any ? lse_of(m, l) : -INFINITY;
}

}  // namespace paged
}  // namespace lmrs
