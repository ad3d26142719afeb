// paged_rows.cuh -- rotary positions with several axes, and appending keys and values to pages with the rotation on the way.
//
// Pair j of a head turns by t = position[axis j] * freq j.  An angle is wanted modulo a turn, and position * freq in f32 has lost it at
// positions of some thousands; here freq / 2 pi is a 64-bit fraction of a turn (made once on the host) and the product wraps modulo 2^64, which is
// modulo a turn, exactly: the angle is off by at most position * (2^-65 + |freq| 2^-129) turns, which is what the host rounds (turns_of).  What is left after taking quarter turns off goes
// through f32.
//
// Both kernels are bound by the bytes of the rows (an angle serves every head of its row), or by one launch's latency where there are few.  A warp takes a row, or
// some of its heads where rows are few: its lanes compute the row's cosines and sines once into the warp's part of shared memory, then walk the row in pieces.
// A piece is the 2 x 16 bytes of VEC pairs (VEC = 16 bytes of elements): elements c and c + pairs in halves, neighbouring ones in pairs; behind them come
// pieces of 16 bytes that only pass.  Where an array does not lie on 16-byte boundaries, or pairs are no multiple of VEC, the same walk runs with VEC = 1.
// Two pieces a lane are loaded before the first is stored, with 32 warps on an SM.  (Four pieces and 16 warps: 4099 rows of 32 bf16 heads of 128 in 21.6 us
// instead of 18.1, 11,000 appended rows in 105 instead of 86, both before conversions went two elements at a time; more warps a row, which compute its angles
// again: 16.3 and 81 instead of 14.1 and 66.)
// Measured (B200): 4099 rows of 32 bf16 heads of 128, 67 MB: 14.1 us, 4770 GB/s; 11,000 rows of 32 query and 8 KV heads appended, 290 MB: 66 us, 4390 GB/s; one row of
// 40 heads 2.2 us, appended 3.6: launch and a chain of dependent loads (length, table, row).
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

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Piece { T v[VEC]; };

constexpr int ROW_WARPS = 4, ROW_AHEAD = 2, ROW_CTAS = 8;   // (8 CTAs an SM: 64 registers a thread)

// what a warp's pieces look like: `turning` of them turn a head's first 2 * pairs elements, `passing` carry the others (or all of a head that does not turn)
struct Cut {
    int pairs, layout, turning, passing;
    uint32_t reciprocal;   // of turning + passing: ceil(2^32 / n) divides numbers below 2^32 / n exactly
};
inline Cut cut_of(int pairs, int layout, int head_size, int vec) {
    Cut c = {pairs, layout, pairs / vec, (head_size - 2 * pairs) / vec, 0};
    const uint64_t n = (uint64_t)(c.turning + c.passing);
    c.reciprocal = (uint32_t)(((1ull << 32) + n - 1) / n);   // (n = 1: 0, and handled as such)
    return c;
}
constexpr int MAX_HEADS = 65535;   // heads * pieces a head stays below 2^32 / pieces

// the row's cosines and sines, by its warp
PG_DEVINL void row_angles(const lmrs_b200_rope_t& rope, const Positions& pos, int64_t r, int same, float2* angles) {
    // lanes read 32 different entries: through the kernel parameters' constant bank one after the other, so the address is hidden from the compiler and the
    // loads are ordinary ones (16.1 us -> 14.1 for 4099 rows of 32 heads of 128)
    const lmrs_b200_rope_t* t = &rope;
    asm("" : "+l"(t));
    __syncwarp();
    for (int j = threadIdx.x & 31; j < rope.pairs; j += 32) {
        float c, s;
        cos_sin(pos.data ? pos.data[t->axis[j] * pos.axis + r * pos.row] : same, t->turns[j], c, s);
        angles[j] = make_float2(c, s);
    }
    __syncwarp();
}

PG_DEVINL void turn_pair(float& a, float& b, float c, float s) {
    const float y = a;
    a = fmaf(y, c, -(b * s));
    b = fmaf(b, c, y * s);
}
// a 32-bit word of elements as floats and back (16-bit types: two of them, the first one low)
PG_DEVINL float2 open_word(uint32_t w, __nv_bfloat16) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
PG_DEVINL float2 open_word(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
PG_DEVINL uint32_t close_word(float2 v, __nv_bfloat16) { const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y); return *reinterpret_cast<const uint32_t*>(&h); }
PG_DEVINL uint32_t close_word(float2 v, __half) { const __half2 h = __floats2half2_rn(v.x, v.y); return *reinterpret_cast<const uint32_t*>(&h); }

// the pairs of a piece's two parts; t: their cosines and sines
template <typename T> PG_DEVINL void turn_piece(Piece<T, 1>& a, Piece<T, 1>& b, const float2* t, int) {
    float x = to_f(a.v[0]), y = to_f(b.v[0]);
    turn_pair(x, y, t->x, t->y);
    a.v[0] = from_f<T>(x);
    b.v[0] = from_f<T>(y);
}
PG_DEVINL void turn_piece(Piece<float, 4>& a, Piece<float, 4>& b, const float2* t, int layout) {
    const float4 t0 = *reinterpret_cast<const float4*>(t), t1 = *reinterpret_cast<const float4*>(t + 2);
    if (layout) {
        turn_pair(a.v[0], a.v[1], t0.x, t0.y);
        turn_pair(a.v[2], a.v[3], t0.z, t0.w);
        turn_pair(b.v[0], b.v[1], t1.x, t1.y);
        turn_pair(b.v[2], b.v[3], t1.z, t1.w);
    } else {
        turn_pair(a.v[0], b.v[0], t0.x, t0.y);
        turn_pair(a.v[1], b.v[1], t0.z, t0.w);
        turn_pair(a.v[2], b.v[2], t1.x, t1.y);
        turn_pair(a.v[3], b.v[3], t1.z, t1.w);
    }
}
template <typename T> PG_DEVINL void turn_piece(Piece<T, 8>& pa, Piece<T, 8>& pb, const float2* t, int layout) {
    uint32_t* a = reinterpret_cast<uint32_t*>(&pa);
    uint32_t* b = reinterpret_cast<uint32_t*>(&pb);
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if (layout) {   // a word is a pair
            const float2 t0 = t[k], t1 = t[4 + k];
            float2 x = open_word(a[k], T()), y = open_word(b[k], T());
            turn_pair(x.x, x.y, t0.x, t0.y);
            turn_pair(y.x, y.y, t1.x, t1.y);
            a[k] = close_word(x, T());
            b[k] = close_word(y, T());
        } else {
            const float4 c = *reinterpret_cast<const float4*>(t + 2 * k);
            float2 x = open_word(a[k], T()), y = open_word(b[k], T());
            turn_pair(x.x, y.x, c.x, c.y);
            turn_pair(x.y, y.y, c.z, c.w);
            a[k] = close_word(x, T());
            b[k] = close_word(y, T());
        }
    }
}

// pieces from .. to - 1 of a row (counted over its heads), by a warp.  from and to may be the same array: a piece is read before it is written
template <typename T, int VEC>
PG_DEVINL void walk_row(const Cut& cut, const T* x, int64_t x_head, T* out, int64_t out_head, int from, int to, const float2* angles) {
    using P = Piece<T, VEC>;
    const int n = cut.turning + cut.passing, step = cut.layout ? VEC : cut.pairs;   // from a piece's first 16 bytes to its second
    for (int i0 = from + (threadIdx.x & 31); i0 < to; i0 += 32 * ROW_AHEAD) {
        P a[ROW_AHEAD], b[ROW_AHEAD];
        int64_t at[ROW_AHEAD];
        int c[ROW_AHEAD];
#pragma unroll
        for (int u = 0; u < ROW_AHEAD; u++) {
            const int i = i0 + 32 * u;
            if (i >= to) break;
            const int h = n == 1 ? i : (int)__umulhi((uint32_t)i, cut.reciprocal);
            c[u] = i - h * n;
            const bool turns = c[u] < cut.turning;
            const int e = turns ? (cut.layout ? 2 * VEC : VEC) * c[u] : 2 * cut.pairs + VEC * (c[u] - cut.turning);
            const T* p = x + h * x_head + e;
            a[u] = *reinterpret_cast<const P*>(p);
            if (turns) b[u] = *reinterpret_cast<const P*>(p + step);
            at[u] = h * out_head + e;
        }
#pragma unroll
        for (int u = 0; u < ROW_AHEAD; u++) {
            const int i = i0 + 32 * u;
            if (i >= to) break;
            P* p = reinterpret_cast<P*>(out + at[u]);
            if (c[u] >= cut.turning) { *p = a[u]; continue; }
            turn_piece(a[u], b[u], angles + VEC * c[u], cut.layout);
            *p = a[u];
            *reinterpret_cast<P*>(out + at[u] + step) = b[u];
        }
    }
}

// parts: how many warps share a row
template <typename T, int VEC>
__global__ void __launch_bounds__(32 * ROW_WARPS, ROW_CTAS) rope_axes_kernel(const __grid_constant__ lmrs_b200_rope_t rope, const Rows<const T> x, const Rows<T> out, int64_t n_rows, int heads, const Cut cut,
                                                                   const Positions pos, int parts) {
    __shared__ alignas(16) float2 angles[ROW_WARPS][128];
    float2* mine = angles[threadIdx.x >> 5];
    const int total = heads * (cut.turning + cut.passing), each = (total + parts - 1) / parts;
    for (int64_t w = (int64_t)blockIdx.x * ROW_WARPS + (threadIdx.x >> 5); w < n_rows * parts; w += (int64_t)gridDim.x * ROW_WARPS) {
        const int64_t r = w / parts;
        const int from = (int)(w - r * parts) * each;
        row_angles(rope, pos, r, 0, mine);
        walk_row<T, VEC>(cut, x.data + r * x.row, x.head, out.data + r * out.row, out.head, from, min(total, from + each), mine);
    }
}

template <typename T> struct AppendParams {
    lmrs_b200_rope_t rope;   // pairs 0: nothing turns
    Batch batch;
    Positions pos;
    Rows<const T> k, v, q;
    Rows<T> q_out;           // null data: no queries
    T *k_pages, *v_pages;
    int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;
    int kv_heads, q_heads, parts;
    Cut turn, pass;          // of queries and keys, of values
};

// the sequence of row r, by a warp: the last one that begins at or before it (32 are looked at a time); -1: r lies behind the last sequence's rows
PG_DEVINL int seq_of_row_warp(const Batch& s, int64_t r) {
    if (!s.rows) return r < s.seqs ? (int)r : -1;
    const int lane = threadIdx.x & 31;
    int lo = 0, n = s.seqs;   // of sequences lo .. lo + n - 1
    while (n > 1) {
        const int step = (n + 31) / 32, b = lo + lane * step;
        const unsigned begun = __ballot_sync(~0u, b < lo + n && s.rows[b] <= r);
        const int last = begun ? 31 - __clz(begun) : 0;
        n = min(step, n - last * step);
        lo += last * step;
    }
    return s.rows[lo] <= r && r < s.rows[lo + 1] ? lo : -1;
}

template <typename T, int VEC>
__global__ void __launch_bounds__(32 * ROW_WARPS, ROW_CTAS) paged_append_kernel(const __grid_constant__ AppendParams<T> p) {
    __shared__ alignas(16) float2 angles[ROW_WARPS][128];
    float2* mine = angles[threadIdx.x >> 5];
    // a row's pieces: keys, values, queries
    const int nt = p.turn.turning + p.turn.passing, nk = p.kv_heads * nt, nv = p.kv_heads * p.pass.passing, total = nk + nv + (p.q_out.data ? p.q_heads * nt : 0);
    const int each = (total + p.parts - 1) / p.parts;
    for (int64_t w = (int64_t)blockIdx.x * ROW_WARPS + (threadIdx.x >> 5); w < p.batch.n_rows * p.parts; w += (int64_t)gridDim.x * ROW_WARPS) {
        const int64_t r = w / p.parts;
        const int from = (int)(w - r * p.parts) * each, to = min(total, from + each);
        const int b = seq_of_row_warp(p.batch, r);
        if (b < 0) continue;
        const Span s = span_of(p.batch, b);
        const int64_t index = (int64_t)s.len - s.count + (r - s.first);
        row_angles(p.rope, p.pos, r, (int)(p.batch.prefix_len + index), mine);
        const int64_t slot = slot_of(p.batch.tables + b * p.batch.table_stride, p.batch.table_len, p.batch.page_size, p.batch.pages, index < 0 ? -1 : (int)index);
        const int64_t page = slot / p.batch.page_size, place = slot - page * p.batch.page_size;
#pragma unroll 1
        for (int part = slot < 0 ? 2 : 0; part < 3; part++) {   // (one copy of the walk: three of them took 255 registers a thread, and twice the time)
            const int before = part == 0 ? 0 : part == 1 ? nk : nk + nv, here = part == 0 ? nk : part == 1 ? nv : total - nk - nv;
            const int f = max(0, from - before), t = min(here, to - before);
            if (f >= t) continue;
            const Rows<const T>& x = part == 0 ? p.k : part == 1 ? p.v : p.q;
            T* out = part == 0   ? p.k_pages + page * p.k_page + place * p.k_slot
                     : part == 1 ? p.v_pages + page * p.v_page + place * p.v_slot
                                 : p.q_out.data + r * p.q_out.row;
            walk_row<T, VEC>(part == 1 ? p.pass : p.turn, x.data + r * x.row, x.head, out, part == 0 ? p.k_head : part == 1 ? p.v_head : p.q_out.head, f, t, mine);
        }
    }
}

}  // namespace paged
}  // namespace lmrs
