// paged_rows.cuh -- rotary positions with several axes, and appending keys and values to pages with the rotation on the way.
//
// Pair j of a head turns by t = position[axis j] * freq j.  An angle is wanted modulo a turn, and position * freq in f32 has lost it at
// positions of some thousands; here freq / 2 pi is a 64-bit fraction of a turn (made once on the host) and the product wraps modulo 2^64, which is
// modulo a turn, exactly: the angle is off by at most position * 2^-65 turns.  What is left after taking quarter turns off goes through f32.
#pragma once
#include "paged.h"

namespace lmrs {
namespace paged {

// cosine and sine of position * turns / 2^64 turns
PG_DEVINL void cos_sin(int position, uint64_t turns, float& c, float& s) {
    const int64_t t = (int64_t)((uint64_t)(int64_t)position * turns);
    const int64_t quarter = (t >> 62) + ((t >> 61) & 1);   // nearest quarter turn; the rest is within an eighth of a turn
    const float rest = (float)(t - (int64_t)((uint64_t)quarter << 62)) * 0x1p-63f;   // in half turns
    float c0, s0;
    sincospif(rest, &s0, &c0);
    const float a = quarter & 1 ? s0 : c0, b = quarter & 1 ? c0 : s0;
    c = (quarter + 1) & 2 ? -a : a;
    s = quarter & 2 ? -b : b;
}

template <typename T> struct Rows {
    T* data;
    int64_t row, head;
};
struct Positions {
    const int* data;   // null: the same on every axis, known to the caller
    int64_t axis, row;
};

// one element of a row of heads, turned: element e of x (a head's elements)
template <typename T> PG_DEVINL T turned(const lmrs_b200_rope_t& rope, const T* x, int e, const Positions& pos, int64_t r, int same) {
    const int pairs = rope.pairs;
    if (e >= 2 * pairs) return x[e];
    const int j = rope.layout ? e >> 1 : e % pairs, second = rope.layout ? e & 1 : e >= pairs;
    float c, s;
    cos_sin(pos.data ? pos.data[rope.axis[j] * pos.axis + r * pos.row] : same, rope.turns[j], c, s);
    const float a = to_f(x[rope.layout ? 2 * j : j]), b = to_f(x[rope.layout ? 2 * j + 1 : j + pairs]);
    return from_f<T>(second ? fmaf(b, c, a * s) : fmaf(a, c, -(b * s)));
}

// CTA = a row; a thread takes whole pairs (elements of a head that nothing turns come one at a time), so that out may be x
template <typename T> PG_DEVINL void turn_row(const lmrs_b200_rope_t& rope, const T* x, int64_t x_head, T* out, int64_t out_head, int heads, int head_size, const Positions& pos,
                                              int64_t r, int same) {
    const int pairs = rope.pairs, items = head_size - pairs;   // pairs, then single elements
    for (int i = threadIdx.x; i < heads * items; i += blockDim.x) {
        const int h = i / items, j = i - h * items;
        const T* from = x + h * x_head;
        T* to = out + h * out_head;
        if (j < pairs) {
            const int e0 = rope.layout ? 2 * j : j, e1 = rope.layout ? 2 * j + 1 : j + pairs;
            const T a = turned(rope, from, e0, pos, r, same), b = turned(rope, from, e1, pos, r, same);
            to[e0] = a;
            to[e1] = b;
        } else {
            to[j + pairs] = from[j + pairs];
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) rope_axes_kernel(const __grid_constant__ lmrs_b200_rope_t rope, const Rows<const T> x, const Rows<T> out, int64_t n_rows, int heads, int head_size,
                                                        const Positions pos) {
    for (int64_t r = blockIdx.x; r < n_rows; r += gridDim.x) turn_row(rope, x.data + r * x.row, x.head, out.data + r * out.row, out.head, heads, head_size, pos, r, 0);
}

template <typename T> struct AppendParams {
    lmrs_b200_rope_t rope;   // pairs 0: nothing turns
    Batch batch;
    Positions pos;
    Rows<const T> k, v, q;
    Rows<T> q_out;           // null data: no queries
    T *k_pages, *v_pages;
    int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;
    int kv_heads, q_heads, head_size;
};

template <typename T>
__global__ void __launch_bounds__(256) paged_append_kernel(const __grid_constant__ AppendParams<T> p) {
    __shared__ int found;
    for (int64_t r = blockIdx.x; r < p.batch.n_rows; r += gridDim.x) {
        const int b = seq_of_row(p.batch, r, &found);
        if (b < 0) continue;
        const Span s = span_of(p.batch, b);
        const int64_t index = (int64_t)s.len - s.count + (r - s.first);
        const int same = (int)(p.batch.prefix_len + index);
        if (p.q_out.data) turn_row(p.rope, p.q.data + r * p.q.row, p.q.head, p.q_out.data + r * p.q_out.row, p.q_out.head, p.q_heads, p.head_size, p.pos, r, same);
        const int64_t slot = slot_of(p.batch.tables + b * p.batch.table_stride, p.batch.table_len, p.batch.page_size, p.batch.pages, index < 0 ? -1 : (int)index);
        if (slot < 0) continue;
        const int64_t page = slot / p.batch.page_size, place = slot - page * p.batch.page_size;
        turn_row(p.rope, p.k.data + r * p.k.row, p.k.head, p.k_pages + page * p.k_page + place * p.k_slot, p.k_head, p.kv_heads, p.head_size, p.pos, r, same);
        const T* v = p.v.data + r * p.v.row;
        T* to = p.v_pages + page * p.v_page + place * p.v_slot;
        for (int i = threadIdx.x; i < p.kv_heads * p.head_size; i += blockDim.x) {
            const int h = i / p.head_size, e = i - h * p.head_size;
            to[h * p.v_head + e] = v[h * p.v.head + e];
        }
    }
}

}  // namespace paged
}  // namespace lmrs
