// paged8_rows.cuh -- norms of heads with rotary positions in one pass; keys and values quantised into 8-bit pages as they are appended, and read back.
#pragma once
#include "paged8.h"
#include "paged_rows.cuh"

namespace lmrs {
namespace paged {

// ---- norms and rotation ----------------------------------------------------------------------------------------------------------------------
// y = x / sqrt(mean x^2 + eps) * weight of a head, then its pairs turned; float32 inside, rounded once.  A head is taken by 2^group neighbouring lanes of a warp, each with ROUNDS of the pieces
// that paged_rows.cuh cuts heads into, so that it is read once: the sum of its squares is done in the lanes' registers and a few exchanges.
struct HeadNorm {
    const float* weight;   // null: 1
    int64_t head;          // from one head's weights to the next's (0: all heads share them)
    float eps;
    int on;                // 0: no norm
};
template <int VEC> PG_DEVINL void load_weights(const float* w, float (&to)[VEC]) {
    if constexpr (VEC >= 4) {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
            const float4 v = *reinterpret_cast<const float4*>(w + i);
            to[i] = v.x; to[i + 1] = v.y; to[i + 2] = v.z; to[i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i++) to[i] = w[i];
    }
}
// heads from .. to - 1 of a row, by a warp.  from and to may be the same array
template <typename T, int VEC, int ROUNDS>
PG_DEVINL void norm_row(const Cut& cut, const HeadNorm& norm, int group, int D, const T* x, int64_t x_head, T* out, int64_t out_head, int from, int to, const float2* angles) {
    using P = Piece<T, VEC>;
    const int lane = threadIdx.x & 31, width = 1 << group, mine = lane & (width - 1), n = cut.turning + cut.passing, step = cut.layout ? VEC : cut.pairs;
    for (int h0 = from; h0 < to; h0 += 32 >> group) {
        const int h = h0 + (lane >> group);
        const bool is = h < to;
        P a[ROUNDS], b[ROUNDS];
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < ROUNDS; u++) {
            const int c = mine + u * width;
            if (!is || c >= n) continue;
            const bool turns = c < cut.turning;
            const T* p = x + h * x_head + (turns ? (cut.layout ? 2 * VEC : VEC) * c : 2 * cut.pairs + VEC * (c - cut.turning));
            a[u] = *reinterpret_cast<const P*>(p);
            if (turns) b[u] = *reinterpret_cast<const P*>(p + step);
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float f = to_f(a[u].v[i]), g = turns ? to_f(b[u].v[i]) : 0.0f;
                sum = fmaf(f, f, fmaf(g, g, sum));
            }
        }
        float by = 1.0f;
        if (norm.on) {
            for (int d = width >> 1; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
            by = 1.0f / sqrtf(sum / (float)D + norm.eps);
        }
#pragma unroll
        for (int u = 0; u < ROUNDS; u++) {
            const int c = mine + u * width;
            if (!is || c >= n) continue;
            const bool turns = c < cut.turning;
            const int e = turns ? (cut.layout ? 2 * VEC : VEC) * c : 2 * cut.pairs + VEC * (c - cut.turning);
            float f[VEC], g[VEC];
#pragma unroll
            for (int i = 0; i < VEC; i++) { f[i] = to_f(a[u].v[i]) * by; g[i] = turns ? to_f(b[u].v[i]) * by : 0.0f; }
            if (norm.weight) {
                float w[VEC];
                load_weights<VEC>(norm.weight + h * norm.head + e, w);
#pragma unroll
                for (int i = 0; i < VEC; i++) f[i] *= w[i];
                if (turns) {
                    load_weights<VEC>(norm.weight + h * norm.head + e + step, w);
#pragma unroll
                    for (int i = 0; i < VEC; i++) g[i] *= w[i];
                }
            }
            if (turns) {
                const float2* t = angles + VEC * c;
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    if (VEC > 1 && cut.layout) {   // neighbours: pairs 0 .. VEC / 2 - 1 of the piece are in f, the others in g
                        if (i & 1) continue;
                        turn_pair(f[i], f[i + 1 < VEC ? i + 1 : i], t[i / 2].x, t[i / 2].y);
                        turn_pair(g[i], g[i + 1 < VEC ? i + 1 : i], t[VEC / 2 + i / 2].x, t[VEC / 2 + i / 2].y);
                    } else {
                        turn_pair(f[i], g[i], t[i].x, t[i].y);
                    }
                }
            }
            P o;
            T* to_p = out + h * out_head + e;
#pragma unroll
            for (int i = 0; i < VEC; i++) o.v[i] = from_f<T>(f[i]);
            *reinterpret_cast<P*>(to_p) = o;
            if (turns) {
#pragma unroll
                for (int i = 0; i < VEC; i++) o.v[i] = from_f<T>(g[i]);
                *reinterpret_cast<P*>(to_p + step) = o;
            }
        }
    }
}

// parts: how many warps share a row; rope.pairs 0: nothing turns
template <typename T, int VEC, int ROUNDS>
__global__ void __launch_bounds__(32 * ROW_WARPS) norm_rope_kernel(const __grid_constant__ lmrs_b200_rope_t rope, const Rows<const T> x, const Rows<T> out, int64_t n_rows, int heads, int D, const Cut cut,
                                                                   const HeadNorm norm, const Positions pos, int parts, int group) {
    __shared__ alignas(16) float2 angles[ROW_WARPS][128];
    float2* mine = angles[threadIdx.x >> 5];
    const int each = (heads + parts - 1) / parts;
    for (int64_t w = (int64_t)blockIdx.x * ROW_WARPS + (threadIdx.x >> 5); w < n_rows * parts; w += (int64_t)gridDim.x * ROW_WARPS) {
        const int64_t r = w / parts;
        const int from = (int)(w - r * parts) * each;
        row_angles(rope, pos, r, 0, mine);
        norm_row<T, VEC, ROUNDS>(cut, norm, group, D, x.data + r * x.row, x.head, out.data + r * out.row, out.head, from, min(heads, from + each), mine);
    }
}

// ---- appending -------------------------------------------------------------------------------------------------------------------------------
// A CTA takes one block of tokens that share a scale: it is led by the row that is the call's first in the block, and CTAs of other rows leave at once.  First the largest size of every head
// among the block's new tokens, then the scales (and the codes that the block held before, where its scale grows), then the new codes; keys are normed and turned again for
// that, which is cheaper than keeping them.  All that a rounding to 8 bits depends on is computed in 64 bits, so that a code is the nearest one of the value that the formulas give, but for
// values within some 2^-45 of a border: in 32 bits one of ten thousand codes would be its neighbour, by 1/127 of the block's largest value.
constexpr int PUT_WARPS = 8, PUT_HEADS = 8, PUT_TOKENS = 16;   // heads a CTA takes, tokens whose angles it holds at a time

template <typename T> struct PutParams {
    lmrs_b200_rope_t rope;   // pairs 0: nothing turns
    Batch batch;
    Positions pos;
    Rows<const T> k, v, q;
    Rows<T> q_out;           // null data: no queries
    Pages8 pages;
    HeadNorm k_norm, q_norm;
    Cut turn;                // of the queries
    int q_heads, parts, group, put_ctas, head_ctas;   // CTAs that quantise: put_ctas rows times head_ctas groups of heads; the others take the queries
};

// cosine and sine of position * turns / 2^64 turns, in 64 bits
PG_DEVINL double2 cos_sin64(int position, uint64_t turns) {
    const int64_t t = (int64_t)((uint64_t)(int64_t)position * turns);
    const int64_t quarter = (t >> 62) + ((t >> 61) & 1);
    double s0, c0;
    sincospi((double)(t - (int64_t)((uint64_t)quarter << 62)) * 0x1p-63, &s0, &c0);
    const double a = quarter & 1 ? s0 : c0, b = quarter & 1 ? c0 : s0;
    return make_double2((quarter + 1) & 2 ? -a : a, quarter & 2 ? -b : b);
}

// A head of one row in a warp's registers: lane's elements are first(i), second(i) of slots lane + 32 i; a slot is a pair that turns, or two neighbours that do not
struct HeadSlots {
    int pairs, layout, D;
    PG_DEVINL int count() const { return (D + 1) / 2; }
    PG_DEVINL int first(int s) const { return s < pairs ? (layout ? 2 * s : s) : 2 * s; }
    PG_DEVINL int second(int s) const { return s < pairs ? (layout ? 2 * s + 1 : s + pairs) : 2 * s + 1; }   // (D: there is none)
};
constexpr int MOST_SLOTS = 4;   // 256 elements

template <typename T> PG_DEVINL void load_head(const HeadSlots& at, const T* x, double (&y)[MOST_SLOTS][2]) {
#pragma unroll
    for (int i = 0; i < MOST_SLOTS; i++) {
        const int s = (threadIdx.x & 31) + 32 * i;
        y[i][0] = s < at.count() ? (double)to_f(x[at.first(s)]) : 0.0;
        y[i][1] = s < at.count() && at.second(s) < at.D ? (double)to_f(x[at.second(s)]) : 0.0;
    }
}
PG_DEVINL void norm_head(const HeadSlots& at, const HeadNorm& norm, int h, double (&y)[MOST_SLOTS][2]) {
    if (!norm.on) return;
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < MOST_SLOTS; i++) sum = fma(y[i][0], y[i][0], fma(y[i][1], y[i][1], sum));
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
    const double by = 1.0 / sqrt(sum / at.D + (double)norm.eps);
#pragma unroll
    for (int i = 0; i < MOST_SLOTS; i++) {
        const int s = (threadIdx.x & 31) + 32 * i;
        if (s >= at.count()) continue;
        y[i][0] *= by;
        y[i][1] *= by;
        if (norm.weight) {
            const float* w = norm.weight + h * norm.head;
            y[i][0] *= (double)w[at.first(s)];
            if (at.second(s) < at.D) y[i][1] *= (double)w[at.second(s)];
        }
    }
}
PG_DEVINL void turn_head(const HeadSlots& at, const double2* angles, double (&y)[MOST_SLOTS][2]) {
#pragma unroll
    for (int i = 0; i < MOST_SLOTS; i++) {
        const int s = (threadIdx.x & 31) + 32 * i;
        if (s >= at.pairs) continue;
        const double2 t = angles[s];
        const double a = y[i][0], b = y[i][1];
        y[i][0] = a * t.x - b * t.y;
        y[i][1] = b * t.x + a * t.y;
    }
}
// the largest size of this lane's elements, as bits without the sign: they rise with the size, and NaN lies above all
PG_DEVINL unsigned long long size_of_head(const double (&y)[MOST_SLOTS][2]) {
    unsigned long long a = 0;
#pragma unroll
    for (int i = 0; i < MOST_SLOTS; i++)
#pragma unroll
        for (int k = 0; k < 2; k++) a = max(a, (unsigned long long)__double_as_longlong(y[i][k]) & 0x7fffffffffffffffull);
    return a;
}

template <typename T, int FORM, int VEC, int ROUNDS>
__global__ void __launch_bounds__(32 * PUT_WARPS) paged8_append_kernel(const __grid_constant__ PutParams<T> p) {
    __shared__ alignas(16) double2 angles[PUT_TOKENS][128];
    __shared__ unsigned long long most[2][PUT_HEADS];
    __shared__ float scales[2][PUT_HEADS], before[2][PUT_HEADS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = p.pages.head_size;
    const int puts = p.put_ctas * p.head_ctas;
    if ((int)blockIdx.x >= puts) {   // the queries
        float2* mine = reinterpret_cast<float2*>(angles) + 128 * warp;
        const int each = (p.q_heads + p.parts - 1) / p.parts;
        for (int64_t w = (int64_t)(blockIdx.x - puts) * PUT_WARPS + warp; w < p.batch.n_rows * p.parts; w += (int64_t)(gridDim.x - puts) * PUT_WARPS) {
            const int64_t r = w / p.parts;
            const int from = (int)(w - r * p.parts) * each, b = seq_of_row_warp(p.batch, r);
            if (b < 0) continue;
            const Span s = span_of(p.batch, b);
            row_angles(p.rope, p.pos, r, (int)(p.batch.prefix_len + (int64_t)s.len - s.count + (r - s.first)), mine);
            norm_row<T, VEC, ROUNDS>(p.turn, p.q_norm, p.group, D, p.q.data + r * p.q.row, p.q.head, p.q_out.data + r * p.q_out.row, p.q_out.head, from, min(p.q_heads, from + each), mine);
        }
        return;
    }
    const int head_cta = (int)blockIdx.x % p.head_ctas, head0 = head_cta * PUT_HEADS, heads = min(PUT_HEADS, p.pages.kv_heads - head0);
    for (int64_t r = blockIdx.x / p.head_ctas; r < p.batch.n_rows; r += p.put_ctas) {
        const int b = seq_of_row_warp(p.batch, r);
        if (b < 0) continue;
        const Span s = span_of(p.batch, b);
        const int64_t first_new = (int64_t)s.len - s.count, index64 = first_new + (r - s.first);
        if (index64 < 0) continue;
        const int index = (int)index64, start = index / p.pages.block * p.pages.block;
        if (index != start && r != s.first && index64 - 1 >= 0) continue;   // (the row before it leads)
        const int64_t slot = slot_of(p.batch.tables + b * p.batch.table_stride, p.batch.table_len, p.batch.page_size, p.batch.pages, index);
        if (slot < 0) continue;
        const int64_t page = slot / p.batch.page_size;
        const int place = (int)(slot - page * p.batch.page_size), tokens = (int)min((int64_t)(start + p.pages.block - index), (int64_t)s.len - index), older = index - start;
        const int64_t in_page = place / p.pages.block;
        const HeadSlots key_at = {p.rope.pairs, p.rope.layout, D}, value_at = {0, 0, D};
        __syncthreads();   // (the block before is done with)
        if (threadIdx.x < 2 * PUT_HEADS) most[threadIdx.x / PUT_HEADS][threadIdx.x % PUT_HEADS] = 0;
        double y[MOST_SLOTS][2];
        int64_t kept = -1;   // the item that y holds
        for (int pass = 0; pass < 2; pass++) {
            for (int t0 = 0; t0 < tokens; t0 += PUT_TOKENS) {
                const int now = min(PUT_TOKENS, tokens - t0);
                if (pass == 0 || tokens > PUT_TOKENS) {
                    __syncthreads();
                    for (int i = threadIdx.x; i < now * p.rope.pairs; i += 32 * PUT_WARPS) {
                        const int t = i / p.rope.pairs, j = i - t * p.rope.pairs;
                        const int64_t row = r + t0 + t;
                        const int position = p.pos.data ? p.pos.data[p.rope.axis[j] * p.pos.axis + row * p.pos.row] : (int)(p.batch.prefix_len + index + t0 + t);
                        angles[t][j] = cos_sin64(position, p.rope.turns[j]);
                    }
                    __syncthreads();
                }
                for (int item = warp; item < 2 * heads * now; item += PUT_WARPS) {
                    const int t = item / (2 * heads), which = (item - t * 2 * heads) / heads, h = item - t * 2 * heads - which * heads;
                    const int64_t row = r + t0 + t, number = (int64_t)t0 * 2 * heads + item;
                    const HeadSlots& at = which ? value_at : key_at;
                    if (number != kept) {
                        load_head(at, which ? p.v.data + row * p.v.row + (head0 + h) * p.v.head : p.k.data + row * p.k.row + (head0 + h) * p.k.head, y);
                        if (!which) {
                            norm_head(at, p.k_norm, head0 + h, y);
                            turn_head(at, angles[t], y);
                        }
                        kept = number;
                    }
                    if (pass == 0) {
                        unsigned long long a = size_of_head(y);
                        for (int d = 16; d; d >>= 1) a = max(a, __shfl_xor_sync(~0u, a, d));
                        if (lane == 0) atomicMax(&most[which][h], a);   // (a largest: the order does not matter)
                    } else {
                        const double scale = scales[which][h], by = 1.0 / scale;
                        uint8_t* to = which ? p.pages.v + page * p.pages.v_page + (place + t0 + t) * p.pages.v_slot + (head0 + h) * p.pages.v_head
                                            : p.pages.k + page * p.pages.k_page + (place + t0 + t) * p.pages.k_slot + (head0 + h) * p.pages.k_head;
#pragma unroll
                        for (int i = 0; i < MOST_SLOTS; i++) {
                            const int sl = lane + 32 * i;
                            if (sl >= at.count()) continue;
                            to[at.first(sl)] = close_code<FORM>(y[i][0], scale, by);
                            if (at.second(sl) < D) to[at.second(sl)] = close_code<FORM>(y[i][1], scale, by);
                        }
                    }
                }
            }
            if (pass) break;
            __syncthreads();
            if (threadIdx.x < 2 * heads) {
                const int which = threadIdx.x / heads, h = threadIdx.x - which * heads;
                float* at = which ? p.pages.vs + page * p.pages.vs_page + in_page * p.pages.vs_block + (head0 + h) * p.pages.vs_head
                                  : p.pages.ks + page * p.pages.ks_page + in_page * p.pages.ks_block + (head0 + h) * p.pages.ks_head;
                float scale = scale_for<FORM>(__longlong_as_double((long long)most[which][h]));
                const float old = older ? *at : scale;
                if (older && !(scale >= old)) scale = scale == scale ? old : scale;   // (NaN stays, old or new)
                scales[which][h] = scale;
                before[which][h] = old;
                *at = scale;
            }
            __syncthreads();
            // the codes that the block held, where its scale has grown
            for (int item = warp; item < 2 * heads * older; item += PUT_WARPS) {
                const int t = item / (2 * heads), which = (item - t * 2 * heads) / heads, h = item - t * 2 * heads - which * heads;
                const double old = before[which][h], scale = scales[which][h], by = 1.0 / scale;
                if (!(scale > old)) continue;
                uint8_t* at = which ? p.pages.v + page * p.pages.v_page + (place - older + t) * p.pages.v_slot + (head0 + h) * p.pages.v_head
                                    : p.pages.k + page * p.pages.k_page + (place - older + t) * p.pages.k_slot + (head0 + h) * p.pages.k_head;
                for (int e = lane; e < D; e += 32) at[e] = close_code<FORM>((double)open_code<FORM>(at[e]) * old, scale, by);
            }
        }
    }
}

// ---- reading back ----------------------------------------------------------------------------------------------------------------------------
// code * scale in float32 (exact to half a step), rounded to the type.  A warp a row; its lanes take 16 codes each (one, where something does not lie on 16-byte boundaries).
template <typename T> struct ReadParams {
    Batch batch;
    Pages8 pages;
    Rows<T> k, v;
};
template <typename T, int FORM, int VEC>
__global__ void __launch_bounds__(32 * ROW_WARPS) paged8_read_kernel(const __grid_constant__ ReadParams<T> p) {
    const int lane = threadIdx.x & 31, each = p.pages.head_size / VEC, total = 2 * p.pages.kv_heads * each;
    for (int64_t r = (int64_t)blockIdx.x * ROW_WARPS + (threadIdx.x >> 5); r < p.batch.n_rows; r += (int64_t)gridDim.x * ROW_WARPS) {
        const int b = seq_of_row_warp(p.batch, r);
        if (b < 0) continue;
        const Span s = span_of(p.batch, b);
        const int64_t index = (int64_t)s.len - s.count + (r - s.first);
        const int64_t slot = slot_of(p.batch.tables + b * p.batch.table_stride, p.batch.table_len, p.batch.page_size, p.batch.pages, index < 0 ? -1 : (int)index);
        const int64_t page = slot / p.batch.page_size, place = slot - page * p.batch.page_size, block = place / p.pages.block;
        for (int i = lane; i < total; i += 32) {
            const int head = i / each, e = (i - head * each) * VEC;   // values' heads behind the keys'
            const bool value = head >= p.pages.kv_heads;
            const int h = value ? head - p.pages.kv_heads : head;
            T* out = value ? p.v.data + r * p.v.row + h * p.v.head + e : p.k.data + r * p.k.row + h * p.k.head + e;
            const uint8_t* c = value ? p.pages.v + page * p.pages.v_page + place * p.pages.v_slot + h * p.pages.v_head + e : p.pages.k + page * p.pages.k_page + place * p.pages.k_slot + h * p.pages.k_head + e;
            const float* at = value ? p.pages.vs + page * p.pages.vs_page + block * p.pages.vs_block + h * p.pages.vs_head
                                    : p.pages.ks + page * p.pages.ks_page + block * p.pages.ks_block + h * p.pages.ks_head;
            if constexpr (VEC == 16) {
                const uint4 w = slot < 0 ? make_uint4(0, 0, 0, 0) : *reinterpret_cast<const uint4*>(c);
                const float scale = slot < 0 ? 0.0f : *at;
                const uint32_t words[4] = {w.x, w.y, w.z, w.w};
                constexpr int PER = 16 / sizeof(T);
                Piece<T, PER> o[sizeof(T)];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    float4 f = open_codes<FORM>(words[k]);
                    f = make_float4(f.x * scale, f.y * scale, f.z * scale, f.w * scale);
                    const float g[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
                    for (int j = 0; j < 4; j++) o[(4 * k + j) / PER].v[(4 * k + j) % PER] = from_f<T>(g[j]);
                }
#pragma unroll
                for (int k = 0; k < (int)sizeof(T); k++) *reinterpret_cast<Piece<T, PER>*>(out + k * PER) = o[k];
            } else {
                *out = from_f<T>(slot < 0 ? 0.0f : open_code<FORM>(*c) * *at);
            }
        }
    }
}

}  // namespace paged
}  // namespace lmrs
