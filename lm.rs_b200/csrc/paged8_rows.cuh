// paged8_rows.cuh -- norms of heads with rotary positions in one pass; keys and values quantised into 8-bit pages as they are appended, and read back.
#pragma once
#include "paged8.h"
#include "paged_rows.cuh"

namespace lmrs {
namespace paged {

// ---- norms and rotation ----------------------------------------------------------------------------------------------------------------------
// y = x / sqrt(mean x^2 + eps) * weight of a head, then its pairs turned; float32 inside, rounded once.  A head is read once: it lies in the registers of neighbouring lanes of a warp, eight elements each, and
// the sum of its squares takes a few exchanges.  Eight elements are four pairs that turn (two times four neighbours in halves, eight in pairs) or eight that do not, so that all lanes have the same to do.
// Where arrays do not lie on the boundaries that this wants, or sizes are no multiples of eight, a general walk takes the elements of a head one at a time, 32 apart.
// Two elements an instruction (f32x2) wherever there is one for it: instructions bound these kernels next to the bytes.
// Measured (B200): 4099 rows of 40 bf16 heads of 128 with weights of their own, 84 MB: 21.4 us, 3920 GB/s, 2.6 instructions a cycle of 4 (21.0 where
// lanes that do not turn multiply all the same; by pieces of 16 bytes and with a root and a quotient 28.6; two heads ahead instead of four 26.3); one row 2.6 us.
struct HeadNorm {
    const float* weight;   // null: 1
    int64_t head;          // from one head's weights to the next's (0: all heads share them)
    float eps;
    int on;                // 0: no norm
};
PG_DEVINL uint64_t two(float a, float b) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
PG_DEVINL float2 apart(uint64_t v) { float2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v)); return r; }
PG_DEVINL uint64_t mul2(uint64_t a, uint64_t b) { uint64_t r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
PG_DEVINL uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) { uint64_t r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }

// A row's angles as the fast walks read them: cosines and sines of 128 pairs, 1 and 0 from the last one on
struct Turns { float c[128], s[128]; };
// eight elements of a head, and where: lane c of its lanes has elements first .. first + 3 and second .. second + 3
struct Eight { uint64_t v[4]; };
struct EightAt {
    int first, second;
    bool zipped;   // a pair is neighbours (layout 1); else it is first + i and second + i
    bool turns;    // or the elements pass
    PG_DEVINL EightAt(int c, int pairs, int layout) {
        const bool halves = layout == 0 && 4 * c < pairs;
        first = halves ? 4 * c : 8 * c;
        second = halves ? first + pairs : first + 4;
        zipped = layout != 0;
        turns = 4 * c < pairs;
    }
};
template <typename T> struct Quad;   // four elements in memory
template <> struct Quad<float> { typedef float4 type; };
template <> struct Quad<__nv_bfloat16> { typedef uint2 type; };
template <> struct Quad<__half> { typedef uint2 type; };
PG_DEVINL void open_quad(float4 q, uint64_t& a, uint64_t& b, float) { a = two(q.x, q.y); b = two(q.z, q.w); }
template <typename T> PG_DEVINL void open_quad(uint2 q, uint64_t& a, uint64_t& b, T) {
    const float2 x = open_word(q.x, T()), y = open_word(q.y, T());
    a = two(x.x, x.y);
    b = two(y.x, y.y);
}
PG_DEVINL float4 close_quad(uint64_t a, uint64_t b, float) { const float2 x = apart(a), y = apart(b); return make_float4(x.x, x.y, y.x, y.y); }
template <typename T> PG_DEVINL uint2 close_quad(uint64_t a, uint64_t b, T) { return make_uint2(close_word(apart(a), T()), close_word(apart(b), T())); }
PG_DEVINL float squares8(const Eight& x) {
    const float2 s = apart(fma2(x.v[0], x.v[0], fma2(x.v[1], x.v[1], fma2(x.v[2], x.v[2], mul2(x.v[3], x.v[3])))));
    return s.x + s.y;
}
PG_DEVINL void scale8(Eight& x, float f) {
#pragma unroll
    for (int i = 0; i < 4; i++) x.v[i] = mul2(x.v[i], two(f, f));
}
PG_DEVINL void load_weights8(const float* w, const EightAt& at, Eight& to) {
    const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(w + at.first), b = *reinterpret_cast<const ulonglong2*>(w + at.second);
    to.v[0] = a.x; to.v[1] = a.y; to.v[2] = b.x; to.v[3] = b.y;
}
// (With the cosine of 1 and the sine of 0 that a lane has which does not turn, an infinity makes NaN of the element beside it)
PG_DEVINL void turn8(Eight& x, const Turns& t, int c, bool zipped) {
    const ulonglong2 cs = *reinterpret_cast<const ulonglong2*>(t.c + 4 * c), sn = *reinterpret_cast<const ulonglong2*>(t.s + 4 * c);
    const uint64_t minus = 0x8000000080000000ull;
    if (zipped) {
        const float2 p0 = apart(x.v[0]), p1 = apart(x.v[1]), p2 = apart(x.v[2]), p3 = apart(x.v[3]);
        const uint64_t a0 = two(p0.x, p1.x), b0 = two(p0.y, p1.y), a1 = two(p2.x, p3.x), b1 = two(p2.y, p3.y);
        const float2 y0 = apart(fma2(b0, sn.x ^ minus, mul2(a0, cs.x))), z0 = apart(fma2(b0, cs.x, mul2(a0, sn.x)));
        const float2 y1 = apart(fma2(b1, sn.y ^ minus, mul2(a1, cs.y))), z1 = apart(fma2(b1, cs.y, mul2(a1, sn.y)));
        x.v[0] = two(y0.x, z0.x); x.v[1] = two(y0.y, z0.y); x.v[2] = two(y1.x, z1.x); x.v[3] = two(y1.y, z1.y);
    } else {
        const uint64_t a0 = x.v[0], a1 = x.v[1], b0 = x.v[2], b1 = x.v[3];
        x.v[0] = fma2(b0, sn.x ^ minus, mul2(a0, cs.x));
        x.v[1] = fma2(b1, sn.y ^ minus, mul2(a1, cs.y));
        x.v[2] = fma2(b0, cs.x, mul2(a0, sn.x));
        x.v[3] = fma2(b1, cs.y, mul2(a1, sn.y));
    }
}
// the row's angles, by its warp
PG_DEVINL void row_turns(const lmrs_b200_rope_t& rope, const Positions& pos, int64_t r, int same, Turns& t) {
    const lmrs_b200_rope_t* at = &rope;   // (ordinary loads, as in row_angles)
    asm("" : "+l"(at));
    __syncwarp();
    for (int j = threadIdx.x & 31; j < 128; j += 32) {
        float c = 1.0f, s = 0.0f;
        if (j < rope.pairs) cos_sin(pos.data ? pos.data[at->axis[j] * pos.axis + r * pos.row] : same, at->turns[j], c, s);
        t.c[j] = c;
        t.s[j] = s;
    }
    __syncwarp();
}
// heads from .. to - 1 of a row, by a warp, LANES lanes a head, NORM_AHEAD times as many heads loaded before the first is stored.  x and out may be the same array
template <typename T> constexpr int NORM_AHEAD = sizeof(T) == 2 ? 4 : 2;
// 1 / sqrt(sum / D + eps), off by 4 u (u = 2^-24) for the root's approximation and 2 u for what it is taken of
PG_DEVINL float norm_factor(float sum, float over_D, float eps) { return rsqrtf(fmaf(sum, over_D, eps)); }
template <typename T, int LANES>
PG_DEVINL void norm_row8(int pairs, int layout, const HeadNorm& norm, int D, const T* x, int64_t x_head, T* out, int64_t out_head, int from, int to, const Turns& turns) {
    using Q = typename Quad<T>::type;
    constexpr int HEADS = 32 / LANES;
    const int lane = threadIdx.x & 31, c = lane & (LANES - 1);
    const EightAt at(c, pairs, layout);
    const bool mine = 8 * c < D;
    constexpr int AHEAD = NORM_AHEAD<T>;
    const float over_D = 1.0f / (float)D;
    Eight w;
    if (norm.weight && norm.head == 0 && mine) load_weights8(norm.weight, at, w);
    for (int h0 = from + lane / LANES; h0 < to + lane / LANES; h0 += HEADS * AHEAD) {   // (the same for all lanes)
        Q a[AHEAD], b[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            const int h = h0 + HEADS * u;
            if (h >= to || !mine) { a[u] = Q{}; b[u] = Q{}; continue; }
            const T* p = x + h * x_head;
            a[u] = *reinterpret_cast<const Q*>(p + at.first);
            b[u] = *reinterpret_cast<const Q*>(p + at.second);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            const int h = h0 + HEADS * u;
            if (h0 - lane / LANES + HEADS * u >= to) break;   // (all lanes)
            const bool is = h < to && mine;
            if (norm.weight && norm.head && is) load_weights8(norm.weight + h * norm.head, at, w);
            Eight y;
            open_quad(a[u], y.v[0], y.v[1], T());
            open_quad(b[u], y.v[2], y.v[3], T());
            if (norm.on) {
                float sum = squares8(y);
#pragma unroll
                for (int d = LANES >> 1; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
                scale8(y, norm_factor(sum, over_D, norm.eps));
            }
            if (!is) continue;
            if (norm.weight) {
#pragma unroll
                for (int i = 0; i < 4; i++) y.v[i] = mul2(y.v[i], w.v[i]);
            }
            if (at.turns) turn8(y, turns, c, at.zipped);
            T* p = out + h * out_head;
            *reinterpret_cast<Q*>(p + at.first) = close_quad(y.v[0], y.v[1], T());
            *reinterpret_cast<Q*>(p + at.second) = close_quad(y.v[2], y.v[3], T());
        }
    }
}
// the same for any size and place: a warp a head, elements first(s), second(s) of slots s = lane + 32 i; a slot is a pair that turns, or two neighbours that do not
struct HeadSlots {
    int pairs, layout, D;
    PG_DEVINL int count() const { return (D + 1) / 2; }
    PG_DEVINL int first(int s) const { return s < pairs ? (layout ? 2 * s : s) : 2 * s; }
    PG_DEVINL int second(int s) const { return s < pairs ? (layout ? 2 * s + 1 : s + pairs) : 2 * s + 1; }   // (D: there is none)
};
template <typename T>
PG_DEVINL void norm_row1(int pairs, int layout, const HeadNorm& norm, int D, const T* x, int64_t x_head, T* out, int64_t out_head, int from, int to, const Turns& turns) {
    const HeadSlots at = {pairs, layout, D};
    const int lane = threadIdx.x & 31;
    for (int h = from; h < to; h++) {
        float y[4][2], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int s = lane + 32 * i;
            y[i][0] = s < at.count() ? to_f(x[h * x_head + at.first(s)]) : 0.0f;
            y[i][1] = s < at.count() && at.second(s) < D ? to_f(x[h * x_head + at.second(s)]) : 0.0f;
            sum = fmaf(y[i][0], y[i][0], fmaf(y[i][1], y[i][1], sum));
        }
        float by = 1.0f;
        if (norm.on) {
            for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
            by = norm_factor(sum, 1.0f / (float)D, norm.eps);
        }
        __syncwarp();   // (all of the head has been read)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int s = lane + 32 * i;
            if (s >= at.count()) continue;
            const int e = at.first(s), f = at.second(s);
            float a = y[i][0] * by, b = y[i][1] * by;
            if (norm.weight) {
                a *= norm.weight[h * norm.head + e];
                if (f < D) b *= norm.weight[h * norm.head + f];
            }
            if (s < pairs) turn_pair(a, b, turns.c[s], turns.s[s]);
            out[h * out_head + e] = from_f<T>(a);
            if (f < D) out[h * out_head + f] = from_f<T>(b);
        }
    }
}
// LANES 0: the general walk
template <typename T, int LANES>
PG_DEVINL void norm_row(int pairs, int layout, const HeadNorm& norm, int D, const T* x, int64_t x_head, T* out, int64_t out_head, int from, int to, const Turns& turns) {
    if constexpr (LANES == 0) norm_row1(pairs, layout, norm, D, x, x_head, out, out_head, from, to, turns);
    else norm_row8<T, LANES>(pairs, layout, norm, D, x, x_head, out, out_head, from, to, turns);
}

// parts: how many warps share a row; rope.pairs 0: nothing turns
template <typename T, int LANES>
__global__ void __launch_bounds__(32 * ROW_WARPS) norm_rope_kernel(const __grid_constant__ lmrs_b200_rope_t rope, const Rows<const T> x, const Rows<T> out, int64_t n_rows, int heads, int D,
                                                                   const HeadNorm norm, const Positions pos, int parts) {
    __shared__ alignas(16) Turns turns[ROW_WARPS];
    Turns& mine = turns[threadIdx.x >> 5];
    const int each = (heads + parts - 1) / parts;
    for (int64_t w = (int64_t)blockIdx.x * ROW_WARPS + (threadIdx.x >> 5); w < n_rows * parts; w += (int64_t)gridDim.x * ROW_WARPS) {
        const int64_t r = w / parts;
        const int from = (int)(w - r * parts) * each;
        if (rope.pairs) row_turns(rope, pos, r, 0, mine);
        norm_row<T, LANES>(rope.pairs, rope.layout, norm, D, x.data + r * x.row, x.head, out.data + r * out.row, out.head, from, min(heads, from + each), mine);
    }
}

// ---- appending -------------------------------------------------------------------------------------------------------------------------------
// A warp takes one head of the keys or of the values for a block of tokens that share a scale: the largest size among the block's new tokens, the scale (and the codes that the block held before,
// where its scale grows), the new codes.  Up to PUT_HOLD tokens stay in registers all the while; longer blocks go through the input twice.  A CTA's warps share the angles of a block's tokens.
//
// A code is the nearest one of the value that the formulas give, and a scale their largest value's, to within some 2^-45 of a border: in 32 bits alone one of ten thousand codes would be its neighbour, by 1/127 of
// the block's largest value.  But 64 bits are needed where 32 cannot tell only.  With u = 2^-24, an element after its norm is off by 14 u of itself (squares: 13 u of their sum,
// mean 2 u, halved by the root; the root's approximation 4 u; two products), after its rotation by 19 u (|a| + |b|) of its pair (cosines 3 u, two products and a sum), which is 27 u of the turned pair's sizes, and by 5 u (7 u) without a norm; PUT_OFF is 32 u, PUT_OFF_TURN
// 10 u.  An element so near to a border between two codes is computed again in
// 64 bits (head64; one head of eight has one), and so are the tokens whose largest element is within 2^-17 of the block's largest.  Inputs that 32 bits would overflow on go that way altogether.
// What bounds it: the chain row - sequence - length - table - input of a block, with 16 warps on an SM (128 registers: 16 tokens of a head), the instructions of what is near a border, and fetching them (of some 9 cycles
// that a warp waits for an instruction, 3.7 go by until it has been fetched; 1.3 a cycle of 4).  Measured (B200): 11,805
// rows of 24 prompts, 32 query and 8 KV heads of 128, norms, half the columns turned, a scale for 16 tokens, 290 MB with the queries: int8 185 us (keys and values alone 125, without norm and rotation 72), e4m3 213
// (155, 81); a scale for each token 341; one row of 32 and 8 heads of 64 7.4 us, one of each of 64 sequences 10.  All of it in 64 bits, a warp a token and head: 391.
// Spills: the kernels for few tokens, with 64 registers, put 148 to 268 bytes a thread away; those of longer blocks for heads beyond 64, with 128, 776 to 916 in float32 and 200 to 284 in 16 bits.
constexpr int PUT_WARPS = 8, PUT_TOKENS = 16;   // warps of a CTA, tokens whose angles it holds at a time
constexpr float PUT_OFF = 0x1p-19f, PUT_OFF_TURN = 10.0f * 0x1p-24f;

template <typename T> struct PutParams {
    lmrs_b200_rope_t rope;   // pairs 0: nothing turns
    Batch batch;
    Positions pos;
    Rows<const T> k, v, q;
    Rows<T> q_out;           // null data: no queries
    Pages8 pages;
    HeadNorm k_norm, q_norm;
    int q_heads, parts;
    int window, windows, heads, head_ctas, put_ctas, ctas;   // CTAs that quantise: a window of rows (whose leaders they take) and `heads` heads each; the others take the queries
};

// Cosine and sine of position * turns / 2^64 turns, in 64 bits: quarter turns off, then the Taylor series on an eighth of a turn either way (their next terms are 2^-63 and 2^-66 there)
PG_DEVINL double2 cos_sin64(int position, uint64_t turns) {
    const int64_t t = (int64_t)((uint64_t)(int64_t)position * turns);
    const int64_t quarter = (t >> 62) + ((t >> 61) & 1);
    const double x = (double)(t - (int64_t)((uint64_t)quarter << 62)) * (3.14159265358979323846 * 0x1p-63), y = x * x;
    double s0 = 1.0 / 355687428096000.0, c0 = -1.0 / 6402373705728000.0;   // 1 / 17!, -1 / 18!
    s0 = fma(y, s0, -1.0 / 1307674368000.0);  c0 = fma(y, c0, 1.0 / 20922789888000.0);
    s0 = fma(y, s0, 1.0 / 6227020800.0);      c0 = fma(y, c0, -1.0 / 87178291200.0);
    s0 = fma(y, s0, -1.0 / 39916800.0);       c0 = fma(y, c0, 1.0 / 479001600.0);
    s0 = fma(y, s0, 1.0 / 362880.0);          c0 = fma(y, c0, -1.0 / 3628800.0);
    s0 = fma(y, s0, -1.0 / 5040.0);           c0 = fma(y, c0, 1.0 / 40320.0);
    s0 = fma(y, s0, 1.0 / 120.0);             c0 = fma(y, c0, -1.0 / 720.0);
    s0 = fma(y, s0, -1.0 / 6.0);              c0 = fma(y, c0, 1.0 / 24.0);
    s0 = fma(y * s0, x, x);                   c0 = fma(y, fma(y, c0, -0.5), 1.0);
    const double a = quarter & 1 ? s0 : c0, b = quarter & 1 ? c0 : s0;
    return make_double2((quarter + 1) & 2 ? -a : a, quarter & 2 ? -b : b);
}
// 1 / x and 1 / sqrt(x) by Newton's steps, off by some 2^-52 (x within float32's range; others by the functions)
PG_DEVINL double over64(double x) {
    const float f = (float)x;
    if (!(fabsf(f) > 0x1p-100f && fabsf(f) < 0x1p100f)) return 1.0 / x;
    double r = (double)(1.0f / f);
    r = fma(fma(-x, r, 1.0), r, r);
    return fma(fma(-x, r, 1.0), r, r);
}
PG_DEVINL double over_sqrt64(double x) {
    const float f = (float)x;
    if (!(f > 0x1p-100f && f < 0x1p100f)) return 1.0 / sqrt(x);
    double r = (double)rsqrtf(f);
    r = fma(fma(-x * r, r, 1.0), 0.5 * r, r);
    r = fma(fma(-x * r, r, 1.0), 0.5 * r, r);
    return fma(fma(-x * r, r, 1.0), 0.5 * r, r);
}

template <typename T> PG_DEVINL int put_position(const PutParams<T>& p, int64_t row, int index, int j) {
    return p.pos.data ? p.pos.data[p.rope.axis[j] * p.pos.axis + row * p.pos.row] : (int)(p.batch.prefix_len + index);
}
// key head h of a row in 64 bits, by a warp: elements as HeadSlots has them
template <typename T>
static __device__ __noinline__ void head64(const PutParams<T>& p, int64_t row, int index, int h, double (&y)[4][2]) {
    const HeadSlots at = {p.rope.pairs, p.rope.layout, p.pages.head_size};
    const T* x = p.k.data + row * p.k.row + h * p.k.head;
    const int lane = threadIdx.x & 31;
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int s = lane + 32 * i;
        y[i][0] = s < at.count() ? (double)to_f(x[at.first(s)]) : 0.0;
        y[i][1] = s < at.count() && at.second(s) < at.D ? (double)to_f(x[at.second(s)]) : 0.0;
        sum = fma(y[i][0], y[i][0], fma(y[i][1], y[i][1], sum));
    }
    if (p.k_norm.on) {
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
        const double by = over_sqrt64(fma(sum, over64(at.D), (double)p.k_norm.eps));
        const float* w = p.k_norm.weight + h * p.k_norm.head;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int s = lane + 32 * i;
            if (s >= at.count()) continue;
            y[i][0] *= by * (double)w[at.first(s)];
            if (at.second(s) < at.D) y[i][1] *= by * (double)w[at.second(s)];
        }
    }
#pragma unroll 1
    for (int i = 0; i < 4; i++) {
        const int s = lane + 32 * i;
        if (s >= at.pairs) continue;
        const double2 t = cos_sin64(put_position(p, row, index, s), p.rope.turns[s]);
        const double a = y[i][0], b = y[i][1];
        y[i][0] = a * t.x - b * t.y;
        y[i][1] = b * t.x + a * t.y;
    }
}
PG_DEVINL unsigned long long size_bits(double a) { return (unsigned long long)__double_as_longlong(a) & 0x7fffffffffffffffull; }   // (rise with the size, and NaN lies above all)

// y times by (1 / scale), off by `off` at most, as a code: its bits; unsure: a border lies too near
template <int FORM> PG_DEVINL uint32_t quick_code(float y, float by, float off, bool& unsure) {
    const float r = y * by;
    const float slack = fmaf(fabsf(r), 0x1p-22f, off * fabsf(by));
    if (FORM == FORM_INT8) {
        const float n = rintf(r);
        unsure = !(0.5f - fabsf(r - n) > slack);
        return (uint32_t)(int)fminf(fmaxf(n, -127.0f), 127.0f) & 0xff;
    }
    const int e = max((int)(__float_as_uint(r) >> 23 & 0xff) - 127, -6) - 3;
    const float up = __uint_as_float((uint32_t)(127 - e) << 23), t = r * up;   // (what lies above 448 is cut off: e is 125 at most)
    unsure = !(0.5f - fabsf(t - rintf(t)) > slack * up);
    uint16_t c;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %1;" : "=h"(c) : "f"(r));
    return c & 0xff;
}

// An input by itself, x / scale as the nearest code: exactly, in 32 bits, always.  (Half of all tokens of 16-bit rows have an element in the middle of two codes but for the scale's rounding, since it and the
// largest have 8 or 11 bits.)  With n steps the nearest to x by, x - n step scale is off by nothing near the middle: it is a multiple of half the last place of scale, or of x's where that is more, and
// no more than 2^24 of it; so it tells which side of the middle x lies on.
template <int FORM> PG_DEVINL uint32_t settled_code(float x, float scale, float by) {
    const float size = fabsf(x);
    const float r = __fmul_rn(size, by);   // (not to be joined with the sum below, which two things are made of)
    const uint32_t sign = __float_as_uint(x) >> 31, e = FORM == FORM_INT8 ? 130u << 23 : max(__float_as_uint(r) & 0x7f800000u, 121u << 23);   // (a step is 2^(e - 3): 1 for whole numbers)
    const float far = __uint_as_float(e + (20u << 23) + 0x400000u), half_step = __uint_as_float(e - (4u << 23));
    const float sum = __fadd_rn(r, far);   // (n in its lower bits)
    const float rest = fmaf(__fsub_rn(far, sum), scale, size), half = __fmul_rn(half_step, scale);
    uint32_t n = __float_as_uint(sum) & (FORM == FORM_INT8 ? 255 : 31);
    if (fabsf(rest) > half || (fabsf(rest) == half && (n & 1))) n += rest > 0.0f ? 1 : -1;
    if (FORM == FORM_INT8) {
        n = min(n, 127u);
        return (sign ? 0u - n : n) & 0xff;
    }
    return min(((e - (121u << 23)) >> 20) + n, 0x7eu) | sign << 7;
}

// PUT_HOLD: tokens in registers; SLOTS: slots of a lane
template <int SLOTS> constexpr int PUT_HOLD = SLOTS == 4 ? 8 : 16;
template <typename T, int SLOTS> struct HeldHeads {
    float y[PUT_HOLD<SLOTS>][SLOTS][2];
    unsigned slow;   // bit t: token t goes by 64 bits (the same for all lanes)
};
// n tokens (rows from `row` on) of a head
template <typename T, int SLOTS>
PG_DEVINL void hold_heads(const PutParams<T>& p, bool value, int64_t row, int h, int n, const Turns* turns, HeldHeads<T, SLOTS>& z) {
    const HeadSlots at = value ? HeadSlots{0, 0, p.pages.head_size} : HeadSlots{p.rope.pairs, p.rope.layout, p.pages.head_size};
    const Rows<const T>& from = value ? p.v : p.k;
    const T* x = from.data + row * from.row + h * from.head;
    const int lane = threadIdx.x & 31;
    constexpr int HOLD = PUT_HOLD<SLOTS>;
#pragma unroll
    for (int t = 0; t < HOLD; t++)
#pragma unroll
        for (int i = 0; i < SLOTS; i++) {
            const int s = lane + 32 * i;
            z.y[t][i][0] = t < n && s < at.count() ? to_f(x[t * from.row + at.first(s)]) : 0.0f;
            z.y[t][i][1] = t < n && s < at.count() && at.second(s) < at.D ? to_f(x[t * from.row + at.second(s)]) : 0.0f;
        }
    z.slow = 0;
    if (value || (!p.k_norm.on && p.rope.pairs == 0)) return;   // (the inputs themselves)
    unsigned odd = 0;
    if (p.k_norm.on) {
        float mine = 0.0f;   // lane t: the sum of token t's squares
#pragma unroll
        for (int t = 0; t < HOLD; t++) {
            if (t >= n) break;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < SLOTS; i++) sum = fmaf(z.y[t][i][0], z.y[t][i][0], fmaf(z.y[t][i][1], z.y[t][i][1], sum));
            for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
            if (lane == t) mine = sum;
        }
        const float mean = fmaf(mine, 1.0f / (float)at.D, p.k_norm.eps), by = rsqrtf(mean);
        odd = lane < n && !(mean > 0x1p-100f && mean < 0x1p100f && mine < 0x1p100f) ? 1u << lane : 0;
        const float* w = p.k_norm.weight + h * p.k_norm.head;
        float weight[SLOTS][2];
#pragma unroll
        for (int i = 0; i < SLOTS; i++) {
            const int s = lane + 32 * i;
            weight[i][0] = s < at.count() ? w[at.first(s)] : 0.0f;
            weight[i][1] = s < at.count() && at.second(s) < at.D ? w[at.second(s)] : 0.0f;
        }
#pragma unroll
        for (int t = 0; t < HOLD; t++) {
            const float f = __shfl_sync(~0u, by, t);
#pragma unroll
            for (int i = 0; i < SLOTS; i++) {
                z.y[t][i][0] *= f * weight[i][0];
                z.y[t][i][1] *= f * weight[i][1];
            }
        }
    }
#pragma unroll
    for (int t = 0; t < HOLD; t++) {
        if (t >= n) break;
#pragma unroll
        for (int i = 0; i < SLOTS; i++) {
            if (!(fabsf(z.y[t][i][0]) + fabsf(z.y[t][i][1]) < 0x1p100f)) odd |= 1u << t;
            const int s = lane + 32 * i;
            if (s < at.pairs) {
                turn_pair(z.y[t][i][0], z.y[t][i][1], turns[t].c[s], turns[t].s[s]);
            }
        }
    }
    z.slow = __reduce_or_sync(~0u, odd);
}

// What a warp does with a block's tokens is one of two, with the same steps: HeldHeads, elements one at a time, and HeldEights, eight a lane
template <typename T, int FORM, int SLOTS> struct PutOne {
    static constexpr int HOLD = PUT_HOLD<SLOTS>, LANES = 0, CTAS = 2;
    HeldHeads<T, SLOTS> z;
    PG_DEVINL void hold(const PutParams<T>& p, bool value, int64_t row, int h, int n, const Turns* turns) { hold_heads<T, SLOTS>(p, value, row, h, n, turns, z); }
    PG_DEVINL uint32_t largest(int n) const {   // of this lane's elements of tokens that are not slow, as bits
        uint32_t a = 0;
#pragma unroll
        for (int t = 0; t < HOLD; t++)
#pragma unroll
            for (int i = 0; i < SLOTS; i++)
                if (t < n && !(z.slow >> t & 1)) a = max(a, max(__float_as_uint(z.y[t][i][0]) & 0x7fffffffu, __float_as_uint(z.y[t][i][1]) & 0x7fffffffu));
        return a;
    }
    PG_DEVINL unsigned tokens_from(int n, float near) const {   // tokens that have an element of size `near` or more
        unsigned with = 0;
#pragma unroll
        for (int t = 0; t < HOLD; t++)
#pragma unroll
            for (int i = 0; i < SLOTS; i++)
                if (t < n && fmaxf(fabsf(z.y[t][i][0]), fabsf(z.y[t][i][1])) >= near) with |= 1u << t;
        return with;
    }
    // stores the codes; returns the tokens that have unsure ones
    PG_DEVINL unsigned close(const HeadSlots& at, bool plain, float off_by, int n, float scale, uint8_t* c, int64_t step) const {
        const float by = 1.0f / scale;
        const int lane = threadIdx.x & 31;
        unsigned again = 0;
#pragma unroll
        for (int t = 0; t < HOLD; t++) {
            if (t >= n) break;
#pragma unroll
            for (int i = 0; i < SLOTS; i++) {
                const int sl = lane + 32 * i;
                if (sl >= at.count()) continue;
                const float off = plain ? 0.0f : (fabsf(z.y[t][i][0]) + fabsf(z.y[t][i][1])) * off_by;
                bool unsure[2];
                uint32_t code[2] = {quick_code<FORM>(z.y[t][i][0], by, off, unsure[0]), quick_code<FORM>(z.y[t][i][1], by, off, unsure[1])};
                if (plain) {
                    if (unsure[0]) code[0] = settled_code<FORM>(z.y[t][i][0], scale, by);
                    if (unsure[1]) code[1] = settled_code<FORM>(z.y[t][i][1], scale, by);
                } else if (unsure[0] || unsure[1]) {
                    again |= 1u << t;
                }
                c[t * step + at.first(sl)] = (uint8_t)code[0];
                if (at.second(sl) < at.D) c[t * step + at.second(sl)] = (uint8_t)code[1];
            }
        }
        return again;
    }
};

// r, off by `off` and 2^-22 of itself, as a code.  Codes are n steps of 2^(e - 3), e the exponent of r or -6: r + 1.5 2^23 steps has n in its lower bits (conversions by cvt, two for two elements, were slower:
// 10,900 rows of 8 heads as they are 131 us, and 74 in int8)
PG_DEVINL uint32_t e4m3_code(float r, float off, bool& unsure) {
    const float size = fabsf(r);
    const uint32_t e = max(__float_as_uint(size) & 0x7f800000u, 121u << 23);
    const float far = __uint_as_float(e + (20u << 23) + 0x400000u), sum = __fadd_rn(size, far);
    const float rest = __fsub_rn(size, __fsub_rn(sum, far)), half_step = __uint_as_float(e - (4u << 23));
    unsure = unsure || !(fabsf(rest) + fmaf(size, 0x1p-22f, off) < half_step);
    return min(((e - (121u << 23)) >> 20) + (__float_as_uint(sum) & 31), 0x7eu) | (__float_as_uint(r) >> 24 & 0x80);
}

// LANE lanes a token, 32 / LANE tokens at a time
template <typename T, int FORM, int LANE, int TIMES_> struct PutEight {
    static constexpr int LANES = LANE, AT_ONCE = 32 / LANE, TIMES = TIMES_, HOLD = AT_ONCE * TIMES, CTAS = TIMES == 1 ? 4 : 2;   // CTAS: on an SM
    Eight z[TIMES];
    unsigned slow;
    PG_DEVINL int token(int u) const { return u * AT_ONCE + (threadIdx.x & 31) / LANE; }
    // FULL: n is HOLD, and nothing is asked for each token (with the questions, loads do not go ahead of one another: 10,900 rows of 8 heads in 141 us instead of 107)
    template <bool FULL> PG_DEVINL void hold_as(const PutParams<T>& p, bool value, int64_t row, int h, int n, const Turns* turns) {
        using Q = typename Quad<T>::type;
        const int lane = threadIdx.x & 31, c = lane & (LANE - 1), D = p.pages.head_size;
        const EightAt at(c, value ? 0 : p.rope.pairs, value ? 0 : p.rope.layout);
        const Rows<const T>& from = value ? p.v : p.k;
        const T* x = from.data + row * from.row + h * from.head;
        const bool mine = 8 * c < D;
        Q a[TIMES], b[TIMES];
#pragma unroll
        for (int u = 0; u < TIMES; u++) {
            const int t = token(u);
            if ((!FULL && t >= n) || !mine) { a[u] = Q{}; b[u] = Q{}; continue; }
            a[u] = *reinterpret_cast<const Q*>(x + t * from.row + at.first);
            b[u] = *reinterpret_cast<const Q*>(x + t * from.row + at.second);
        }
        const bool norm = !value && p.k_norm.on, turn = !value && p.rope.pairs;
        const float over_D = 1.0f / (float)D;
        Eight w = {};
        if (norm && mine) load_weights8(p.k_norm.weight + h * p.k_norm.head, at, w);
        unsigned odd = 0;
#pragma unroll
        for (int u = 0; u < TIMES; u++) {
            if (!FULL && u * AT_ONCE >= n) break;
            Eight& y = z[u];
            open_quad(a[u], y.v[0], y.v[1], T());
            open_quad(b[u], y.v[2], y.v[3], T());
            if (!norm && !turn) continue;
            const int t = token(u);
            float sum = squares8(y);
            if (norm) {
#pragma unroll
                for (int d = LANE >> 1; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
                const float mean = fmaf(sum, over_D, p.k_norm.eps);
                if ((FULL || t < n) && !(mean > 0x1p-100f && mean < 0x1p100f)) odd |= 1u << t;
                scale8(y, rsqrtf(mean));
#pragma unroll
                for (int i = 0; i < 4; i++) y.v[i] = mul2(y.v[i], w.v[i]);
                sum = squares8(y);
            }
            if ((FULL || t < n) && !(sum < 0x1p120f)) odd |= 1u << t;   // (elements of this lane's pairs below 2^60, and none NaN)
            if (turn) turn8(y, turns[t], c, at.zipped);   // (lanes that do not turn as well: what is not finite makes its block's scale NaN in any case)
        }
        slow = __reduce_or_sync(~0u, odd);
    }
    PG_DEVINL void hold(const PutParams<T>& p, bool value, int64_t row, int h, int n, const Turns* turns) {
        if (n == HOLD) hold_as<true>(p, value, row, h, n, turns);
        else hold_as<false>(p, value, row, h, n, turns);
    }
    PG_DEVINL static uint32_t size8(const Eight& y) {
        uint32_t a = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = apart(y.v[i]);
            a = max(a, max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
        }
        return a;
    }
    PG_DEVINL uint32_t largest(int n) const {
        uint32_t a = 0;
#pragma unroll
        for (int u = 0; u < TIMES; u++)
            if (token(u) < n && !(slow >> token(u) & 1)) a = max(a, size8(z[u]));
        return a;
    }
    PG_DEVINL unsigned tokens_from(int n, float near) const {
        unsigned with = 0;
#pragma unroll
        for (int u = 0; u < TIMES; u++)
            if (token(u) < n && __uint_as_float(size8(z[u])) >= near) with |= 1u << token(u);
        return with;
    }
    template <bool FULL> PG_DEVINL unsigned close_as(const HeadSlots& slots, bool plain, float off_by, int n, float scale, uint8_t* codes, int64_t step) const {
        const float by = 1.0f / scale;
        const int c = threadIdx.x & (LANE - 1);
        const EightAt at(c, slots.pairs, slots.layout);
        if (8 * c >= slots.D) return 0;
        unsigned again = 0;
#pragma unroll
        for (int u = 0; u < TIMES; u++) {
            const int t = token(u);
            if (!FULL && t >= n) break;
            const Eight& y = z[u];
            // sizes of pairs: (first + i, second + i), or neighbours
            const float2 f0 = apart(y.v[0]), f1 = apart(y.v[1]), f2 = apart(y.v[2]), f3 = apart(y.v[3]);
            const float each = off_by * by;
            const float off[4] = {each * (at.zipped ? fabsf(f0.x) + fabsf(f0.y) : fabsf(f0.x) + fabsf(f2.x)), each * (at.zipped ? fabsf(f1.x) + fabsf(f1.y) : fabsf(f0.y) + fabsf(f2.y)),
                                  each * (at.zipped ? fabsf(f2.x) + fabsf(f2.y) : fabsf(f1.x) + fabsf(f3.x)), each * (at.zipped ? fabsf(f3.x) + fabsf(f3.y) : fabsf(f1.y) + fabsf(f3.y))};
            uint32_t n8[8];
            bool unsure = false;
            if (plain) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float2 f = apart(y.v[i]);
                    n8[2 * i] = settled_code<FORM>(f.x, scale, by);
                    n8[2 * i + 1] = settled_code<FORM>(f.y, scale, by);
                }
            } else if (FORM == FORM_INT8) {
                // y by + 1.5 2^23 has the nearest whole number in its lower bits; what is left tells how far the border is
                const float limit = 0.5f - 127.0f * 0x1p-22f - fmaxf(fmaxf(off[0], off[1]), fmaxf(off[2], off[3]));
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint64_t b2 = two(by, by), r = fma2(y.v[i], b2, two(12582912.0f, 12582912.0f));
                    const float2 rest = apart(fma2(y.v[i], b2, fma2(r, two(-1.0f, -1.0f), two(12582912.0f, 12582912.0f)))), whole = apart(r);
                    unsure = unsure || !(fmaxf(fabsf(rest.x), fabsf(rest.y)) < limit);
                    n8[2 * i] = __float_as_uint(whole.x);
                    n8[2 * i + 1] = __float_as_uint(whole.y);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float2 r = apart(mul2(y.v[i], two(by, by)));
                    n8[2 * i] = e4m3_code(r.x, at.zipped ? off[i] : off[2 * (i & 1)], unsure);
                    n8[2 * i + 1] = e4m3_code(r.y, at.zipped ? off[i] : off[2 * (i & 1) + 1], unsure);
                }
            }
            if (unsure) again |= 1u << t;
            uint32_t word[2];
#pragma unroll
            for (int i = 0; i < 2; i++) word[i] = __byte_perm(__byte_perm(n8[4 * i], n8[4 * i + 1], 0x0040), __byte_perm(n8[4 * i + 2], n8[4 * i + 3], 0x0040), 0x5410);
            *reinterpret_cast<uint32_t*>(codes + t * step + at.first) = word[0];
            *reinterpret_cast<uint32_t*>(codes + t * step + at.second) = word[1];
        }
        return again;
    }
    PG_DEVINL unsigned close(const HeadSlots& slots, bool plain, float off_by, int n, float scale, uint8_t* codes, int64_t step) const {
        return n == HOLD ? close_as<true>(slots, plain, off_by, n, scale, codes, step) : close_as<false>(slots, plain, off_by, n, scale, codes, step);
    }
};
template <typename T, int FORM, int SLOTS> PG_DEVINL unsigned slow_tokens(const PutOne<T, FORM, SLOTS>& x) { return x.z.slow; }
template <typename T, int FORM, int LANE, int TIMES> PG_DEVINL unsigned slow_tokens(const PutEight<T, FORM, LANE, TIMES>& x) { return x.slow; }

// the queries of a call, by warps w, w + step, ... of all
template <typename T, int LANES> PG_DEVINL void put_queries(const PutParams<T>& p, int64_t w, int64_t step, Turns& turns) {
    const int each = (p.q_heads + p.parts - 1) / p.parts;
    for (; w < p.batch.n_rows * p.parts; w += step) {
        const int64_t r = w / p.parts;
        const int from = (int)(w - r * p.parts) * each, b = seq_of_row_warp(p.batch, r);
        if (b < 0) continue;
        const Span s = span_of(p.batch, b);
        if (p.rope.pairs) row_turns(p.rope, p.pos, r, (int)(p.batch.prefix_len + (int64_t)s.len - s.count + (r - s.first)), turns);
        norm_row<T, LANES>(p.rope.pairs, p.rope.layout, p.q_norm, p.pages.head_size, p.q.data + r * p.q.row, p.q.head, p.q_out.data + r * p.q_out.row, p.q_out.head, from, min(p.q_heads, from + each), turns);
    }
}
// By themselves, launched before paged8_append_kernel, which may start while this runs and needs nothing of it: half the warps that fit an SM, so that the other kernel's arithmetic has room beside these copies
constexpr int QUERY_CTAS = ROW_CTAS / 2;
template <typename T, int LANES>
__global__ void __launch_bounds__(32 * ROW_WARPS, ROW_CTAS) put_queries_kernel(const __grid_constant__ PutParams<T> p) {
    __shared__ alignas(16) Turns turns[ROW_WARPS];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    put_queries<T, LANES>(p, (int64_t)blockIdx.x * ROW_WARPS + (threadIdx.x >> 5), (int64_t)gridDim.x * ROW_WARPS, turns[threadIdx.x >> 5]);
}

template <typename T, int FORM, typename Put>
__global__ void __launch_bounds__(32 * PUT_WARPS, Put::CTAS) paged8_append_kernel(const __grid_constant__ PutParams<T> p) {
    __shared__ alignas(16) Turns turns[PUT_TOKENS];
    constexpr int HOLD = Put::HOLD;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = p.pages.head_size;
    const bool last_cta = blockIdx.x == gridDim.x - 1;   // (ends after put_queries_kernel, where there is one, so that whoever waits for this kernel waits for both)
    // CTAs of both kinds take turns
    const int put = (int)((int64_t)blockIdx.x * p.put_ctas / p.ctas);
    if ((int)((int64_t)(blockIdx.x + 1) * p.put_ctas / p.ctas) == put) {   // the queries
        put_queries<T, Put::LANES>(p, (int64_t)(blockIdx.x - put) * PUT_WARPS + warp, (int64_t)(p.ctas - p.put_ctas) * PUT_WARPS, turns[warp]);
        if (last_cta) asm volatile("griddepcontrol.wait;" ::: "memory");
        return;
    }
    const lmrs_b200_rope_t* rope = &p.rope;   // (lanes read different entries: ordinary loads, as in row_turns)
    asm("" : "+l"(rope));
    const int window = put / p.head_ctas, head0 = (put - window * p.head_ctas) * p.heads, heads = min(p.heads, p.pages.kv_heads - head0);
    int64_t r = (int64_t)window * p.window;
    const int64_t r_end = min(r + p.window, p.batch.n_rows);
    // Leaders of the window: rows that are their call's first in a block.  From a row on, the next one is the first of the next block or of the next sequence
    while (r < r_end) {
        const int b = seq_of_row_warp(p.batch, r);
        if (b < 0) {   // (of no sequence: rows between two of them, or behind the last)
            r++;
            continue;
        }
        const Span s = span_of(p.batch, b);
        const int64_t first_new = (int64_t)s.len - s.count, index64 = first_new + (r - s.first);
        if (index64 < 0) {   // padding
            r = max(r + 1, s.first + min((int64_t)s.count, -first_new));   // (onwards, whatever is written into the batch meanwhile)
            continue;
        }
        const int index = (int)index64, start = index / p.pages.block * p.pages.block;
        const int tokens = (int)min((int64_t)(start + p.pages.block - index), (int64_t)s.len - index);
        const int64_t row = r;
        r += max(tokens, 1);
        if (index != start && row != s.first && index64 - 1 >= 0) continue;   // (the row before it leads)
        const int64_t slot = slot_of(p.batch.tables + b * p.batch.table_stride, p.batch.table_len, p.batch.page_size, p.batch.pages, index);
        if (slot < 0) continue;
        const int64_t page = slot / p.batch.page_size;
        const int place = (int)(slot - page * p.batch.page_size), older = index - start;
        const int64_t in_page = place / p.pages.block;
        auto share_turns = [&](int t0, int n) {
            __syncthreads();
            for (int i = threadIdx.x; i < n * 128; i += 32 * PUT_WARPS) {
                const int t = i >> 7, j = i & 127;
                float c = 1.0f, sn = 0.0f;
                if (j < p.rope.pairs) cos_sin(p.pos.data ? p.pos.data[rope->axis[j] * p.pos.axis + (row + t0 + t) * p.pos.row] : (int)(p.batch.prefix_len + index + t0 + t), rope->turns[j], c, sn);
                turns[t].c[j] = c;
                turns[t].s[j] = sn;
            }
            __syncthreads();
        };
        const bool one_go = tokens <= HOLD;
        // Tasks of the warp: heads of keys and of values.  Where a block takes several goes, all warps go through its tokens together, since they share the angles
        for (int task0 = 0; task0 < 2 * heads; task0 += PUT_WARPS) {
            const int task = task0 + warp, value = task >= heads, h = head0 + (value ? task - heads : task);
            const bool is = task < 2 * heads;
            Put z;
            const HeadSlots at = value ? HeadSlots{0, 0, D} : HeadSlots{p.rope.pairs, p.rope.layout, D};
            const bool plain = value || (!p.k_norm.on && p.rope.pairs == 0);   // (the inputs themselves)
            float* scale_at = value ? p.pages.vs + page * p.pages.vs_page + in_page * p.pages.vs_block + h * p.pages.vs_head : p.pages.ks + page * p.pages.ks_page + in_page * p.pages.ks_block + h * p.pages.ks_head;
            float old = 0.0f;
            if (is && older) old = *scale_at;
            unsigned long long most = 0;   // the largest size, as its bits
            for (int t0 = 0; t0 < tokens; t0 += HOLD) {
                const int n = min(HOLD, tokens - t0);
                if (p.rope.pairs && (!one_go || task0 == 0)) share_turns(t0, n);
                if (!is) continue;
                z.hold(p, value, row + t0, h, n, turns);
                const uint32_t a = __reduce_max_sync(~0u, z.largest(n));
                if (plain) {
                    most = max(most, size_bits((double)__uint_as_float(a)));
                } else {
                    const float near = fmaxf(__uint_as_float(a), (float)__longlong_as_double((long long)most)) * (1.0f - 0x1p-17f);
                    unsigned long long top = 0;
                    for (unsigned left = __reduce_or_sync(~0u, z.tokens_from(n, near)) | slow_tokens(z); left; left &= left - 1) {   // (one, mostly)
                        const int t = __ffs(left) - 1;
                        double y[4][2];
                        head64(p, row + t0 + t, index + t0 + t, h, y);
#pragma unroll
                        for (int i = 0; i < 4; i++) top = max(top, max(size_bits(y[i][0]), size_bits(y[i][1])));
                    }
                    for (int d = 16; d; d >>= 1) top = max(top, __shfl_xor_sync(~0u, top, d));
                    most = max(most, top);
                }
            }
            float scale = 0.0f;
            if (is) {
                scale = scale_for<FORM>(__longlong_as_double((long long)most));
                if (older && !(scale >= old)) scale = scale == scale ? old : scale;   // (NaN stays, old or new)
                if (lane == 0) *scale_at = scale;
                // the codes that the block held, where its scale has grown
                if (older && scale > old) {
                    uint8_t* c = value ? p.pages.v + page * p.pages.v_page + (place - older) * p.pages.v_slot + h * p.pages.v_head : p.pages.k + page * p.pages.k_page + (place - older) * p.pages.k_slot + h * p.pages.k_head;
                    const int64_t step = value ? p.pages.v_slot : p.pages.k_slot;
                    const float by = 1.0f / scale;
                    for (int t = 0; t < older; t++, c += step)
                        for (int e = lane; e < D; e += 32) {
                            const float x = open_code<FORM>(c[e]);
                            bool unsure;   // (x old is off by u of itself)
                            uint32_t code = quick_code<FORM>(x * old, by, fabsf(x * old) * 0x1p-23f, unsure);
                            if (unsure) code = close_code<FORM>((double)x * old, scale, over64((double)scale));
                            c[e] = (uint8_t)code;
                        }
                }
            }
            // the new codes
            for (int t0 = 0; t0 < tokens; t0 += HOLD) {
                const int n = min(HOLD, tokens - t0);
                if (!one_go) {
                    if (p.rope.pairs) share_turns(t0, n);
                    if (is) z.hold(p, value, row + t0, h, n, turns);
                }
                if (!is) continue;
                uint8_t* c = value ? p.pages.v + page * p.pages.v_page + (place + t0) * p.pages.v_slot + h * p.pages.v_head : p.pages.k + page * p.pages.k_page + (place + t0) * p.pages.k_slot + h * p.pages.k_head;
                const int64_t step = value ? p.pages.v_slot : p.pages.k_slot;
                // (at the largest scale elements may lie beyond the largest code, and with one that is NaN they all are: both go by 64 bits)
                const unsigned all = (1u << n) - 1;
                const unsigned again = scale < SCALE_MOST ? __reduce_or_sync(~0u, z.close(at, plain, p.k_norm.on ? PUT_OFF : PUT_OFF_TURN, n, scale, c, step)) | slow_tokens(z) : all;
                __syncwarp();   // (the lanes that write a head again are others)
                for (unsigned left = again; left; left &= left - 1) {
                    const int t = __ffs(left) - 1;
                    double y[4][2];
                    if (plain) {
                        const Rows<const T>& from = value ? p.v : p.k;
                        const T* x = from.data + (row + t0 + t) * from.row + h * from.head;
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int sl = lane + 32 * i;
                            y[i][0] = sl < at.count() ? (double)to_f(x[at.first(sl)]) : 0.0;
                            y[i][1] = sl < at.count() && at.second(sl) < D ? (double)to_f(x[at.second(sl)]) : 0.0;
                        }
                    } else {
                        head64(p, row + t0 + t, index + t0 + t, h, y);
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int sl = lane + 32 * i;
                        if (sl >= at.count()) continue;
                        c[t * step + at.first(sl)] = close_code<FORM>(y[i][0], scale, over64((double)scale));
                        if (at.second(sl) < D) c[t * step + at.second(sl)] = close_code<FORM>(y[i][1], scale, over64((double)scale));
                    }
                }
            }
        }
        if (p.rope.pairs) __syncthreads();   // (the angles are used by all until here)
    }
    if (last_cta) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ---- reading back ----------------------------------------------------------------------------------------------------------------------------
// code * scale in float32 (exact to half a step), rounded to the type.  A warp a row; its lanes take 16 codes each (one, where something does not lie on 16-byte boundaries).
// 74,000 tokens of 8 heads of 128 in e4m3 to bf16, 560 MB: 115 us, 4830 GB/s (B200).  What bounds it is latency: a lane has one piece on its way at a time, and of 11 cycles that a warp waits for an instruction 7.7 are for
// memory (2.3 instructions a cycle of 4).
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
