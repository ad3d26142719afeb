// paged8_attn.cuh -- attention of the rows of many sequences over pages of 8-bit codes and over a prefix that all of them share.  The line of tiles, its units and parts, and their joining are
// those of paged_attn.cuh; what differs is how a tile's products are made.
//
// For one row: out = sum_j e^(s_j) v_j c_j / sum_j e^(s_j), s_j = scale * k_j (q . kc_j), where kc_j and c_j are codes and k_j and v_j their scales.  Codes are float16 numbers, so
//     scores     are tensor-core products of the queries in float16 and the codes as they are, times k_j in float32
//     weights    are w_j = 2^(s_j log2 e + log2 v_j - m): the values' scales go into the weights' exponents, m is the largest exponent (less 7), and the codes are multiplied as they are
//     the sum    of e^(s_j) is that of w_j / v_j, in float32
// The queries' types: float16 as it is; bfloat16, whose 8 bits of mantissa float16 has, times a power of two for each row that brings its largest element to between 2^14 and 2^15 (float16's steps end at 2^-24: what
// is below 2^-31 of that element loses bits, 2^-39 of it at most); float32 the same way in three pieces of 11 bits each (24 bits whole down to 2^-15 of the largest element, below that off by 2^-39 of it at most).  Weights in float16: a row's largest 2^7 to 2^15, rounded by 2^-11 of each and 2^-32 of the largest; float32: in three pieces.
#pragma once
#include <float.h>

#include "paged8.h"
#include "paged_attn.cuh"
#include "paged_tensor.cuh"

namespace lmrs {
namespace paged {

template <typename T> struct Attn8Params : AttnParams<T> {   // (k, v and their strides there stay empty)
    Pages8 c;
    int block_shift;   // log2 of the tokens that share a scale, -1 if that is no power of two
};

// one of the pool's scales: a word to shared memory, 0 where there is nothing to copy
PG_DEVINL void copy4(uint32_t to, const void* from, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(there ? 4 : 0));
}

// Codes of a register as two registers of float16 pairs.  int8: a code plus 128 in the lower bits of 1024's mantissa is 1152 more than the code.
// FOLD 0: codes 0, 1 and 2, 3 (neighbouring columns of a key); 1: codes 0, 2 and 1, 3 (the same column of two keys)
template <int FORM, int FOLD> PG_DEVINL void codes_to_halves(uint32_t w, uint32_t& a, uint32_t& b) {
    if constexpr (FORM == FORM_INT8) {
        const uint32_t u = w ^ 0x80808080u, less = 0x64806480u;
        a = __byte_perm(u, 0x64646464u, FOLD ? 0x4240 : 0x4140);
        b = __byte_perm(u, 0x64646464u, FOLD ? 0x4341 : 0x4342);
        const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&less)), y = __hsub2(*reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&less));
        a = *reinterpret_cast<const uint32_t*>(&x);
        b = *reinterpret_cast<const uint32_t*>(&y);
    } else {
        if (FOLD) w = __byte_perm(w, 0, 0x3120);
        asm("{.reg .b16 l, h; mov.b32 {l, h}, %2; cvt.rn.f16x2.e4m3x2 %0, l; cvt.rn.f16x2.e4m3x2 %1, h;}" : "=r"(a), "=r"(b) : "r"(w));
    }
}
PG_DEVINL uint32_t to_halves(float x, float y) { const __half2 h = __floats2half2_rn(x, y); return *reinterpret_cast<const uint32_t*>(&h); }
// a pair of floats in N pieces of float16, each the rounding of what those before it leave
template <int N> PG_DEVINL void split_halves(float x, float y, uint32_t (&to)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        to[i] = to_halves(x, y);
        if (i + 1 < N) {
            const float2 f = half_pair(to[i]);
            x -= f.x;
            y -= f.y;
        }
    }
}
// What a row is multiplied by so that its largest element (of size `most`) lies from 2^14 to 2^15, a power of two, and back.  (Ends of the range: 2^126 at most.)
PG_DEVINL float2 row_factor(float most) {
    const int e = min(253, 268 - (int)(__float_as_uint(most) >> 23));
    return make_float2(__uint_as_float((uint32_t)e << 23), __uint_as_float((uint32_t)(254 - e) << 23));
}
constexpr float SHIFT8 = 7.0f;   // m is so much less than the largest exponent when it is set
// the exponent and the reciprocal of a scale of values (a scale that is NaN leaves a finite reciprocal: it reaches whoever has the weight)
PG_DEVINL float2 value_terms(float v) {
    const float c = fminf(fmaxf(v, SCALE_LEAST), SCALE_MOST);
    float lg, by;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(lg) : "f"(c));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(by) : "f"(c));
    return make_float2(v == v ? lg : v, by);
}

// What bounds it: where the keys are many, latency: 5.0 TB/s of 6.5 from memory and 2.0 instructions a cycle of 4 with 12 warps on an SM (a warp spends some 800 instructions on 32 keys of 128 in int8, a third of them
// on making float16 of codes, and takes turns between waiting for the codes, 1.2 cycles an instruction, and for what it computes, 1.3); where they are few, the chain length - table - codes - scores - join.  Measured (B200): four sequences of up to 100,000 keys (520 MB of codes, 32/8 heads of 128, float16 rows, int8, a scale for each
// token) 112 us, 4620 GB/s, and 105 with a scale for 32 tokens; one sequence of 1000 keys, heads of 64: 10.8 us with the join; float32 rows, 15 sequences behind a prefix of 4096, heads of 64: 28 us.
// Steps, us for the first: tiles of 128 keys copied by all threads 16 bytes at a time 184; a warp its own keys by TMA 167; 8 rows as the products' columns (16 as their rows before) 136; boxes that ask the L2 for
// no more than their own 128 bytes of each 1024 (of 256 before: the heads' codes lie side by side) 112.
// CTA = 4 warps that share a tile's keys: a warp copies its own WARP_KEYS of them to its own slots, a tile or two ahead, and works on them by itself; the warps meet only where parts begin and end.  Codes
// come by TMA, a piece of a page at a time (spills: with 16 rows 220 to 240 bytes a thread for 16-bit heads of 128, 150 to 165 for 256), where all of a warp's keys are within the unit's (else, and where strides or pages take no tensor map, 16 bytes a lane, zeros for what is not there); scales 4 bytes a lane.
template <typename T, int DP, int ROW_TILES> struct TileShape8 {
    static constexpr int PIECES = sizeof(T) == 4 ? 3 : 1;   // of queries and weights
    static constexpr int ROWS = 8 * ROW_TILES, WARPS = 4, THREADS = 32 * WARPS, CHUNKS = DP / 16, WARP_KEYS = DP <= 128 ? 32 : 16, KEYS = WARPS * WARP_KEYS, STAGES = 2;
    static constexpr int KEY_TILES = WARP_KEYS / 16;        // products take 16 keys and 8 rows
    static constexpr int BOX = DP < 128 ? DP : 128;         // columns of a box: the bytes of a row of codes in shared memory
    static constexpr int KV = WARP_KEYS * DP, SLOT = 2 * KV, Q_ROW = DP * (int)sizeof(T), Q = ROWS * Q_ROW;
    static constexpr int SCALES = 2 * WARP_KEYS;            // floats of a slot: the keys', the values' (their logarithms, later); and a warp's WARP_KEYS reciprocals of values'
    static constexpr int SMEM = 1024 + WARPS * STAGES * SLOT + Q + WARPS * (STAGES * SCALES + WARP_KEYS) * 4;
    static constexpr int CTAS = ROW_TILES == 1 ? (DP <= 64 ? 4 : sizeof(T) == 4 && DP > 64 ? 2 : 3) : sizeof(T) == 4 ? (DP <= 64 ? 3 : 2) : DP <= 64 ? 4 : DP <= 128 ? 3 : 2;
    static constexpr int COLS = DP < 128 ? DP : 128;        // columns at a time where the warps' rows meet
    static_assert(ROWS * COLS * 4 <= SLOT, "a warp's rows fit where its keys and values were");
    static_assert(CTAS * (SMEM + 2560) <= 233472, "they fit an SM");
};
// a row's 16-byte pieces, rotated as TMA does (SWIZZLE_128B, and SWIZZLE_64B for rows of 64 bytes)
template <typename S> PG_DEVINL uint32_t code_at(int row, int piece) {
    if constexpr (S::BOX == 64) return (uint32_t)(row * 64 + ((piece ^ (row >> 1 & 3)) << 4));
    else return (uint32_t)((piece >> 3) * (S::WARP_KEYS * 128) + row * 128 + (((piece & 7) ^ (row & 7)) << 4));
}
template <int COLS> PG_DEVINL int sum8_at(int r, int c) { return r * COLS + (c ^ ((r >> 1 & 3) << 3)); }

// How codes come by TMA: `rows` keys of a page at a time (0: never); the maps' dimensions as in paged_tensor.cuh
struct Boxes8 {
    CUtensorMap k, v;
    int rows, k_place, k_head, v_place, v_head;
};

PG_DEVINL uint32_t transpose8(uint32_t v) {   // 8 x 8 elements of 16 bits, a row four lanes
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// The products of one warp: mma.sync with 16 keys as the first operand's rows, 16 columns, and 8 rows of the unit as the second operand's columns: what there is to do for a row - scores, weights, sums - takes no
// more registers and instructions than the unit's rows, and codes are converted once.  lane = 4 g + t
template <typename T, int FORM, int DP, int ROW_TILES> struct WarpTile8 {
    using S = TileShape8<T, DP, ROW_TILES>;
    static constexpr int N = S::PIECES;
    uint32_t q[N == 1 ? S::CHUNKS : 1][ROW_TILES][2];   // columns 16c + 4t .. of row 8n + g (float32: cut into pieces again for each tile, since they do not fit the registers)
    float o[S::CHUNKS][ROW_TILES][4];                   // columns 16c + 2g of rows 8n + 2t and 8n + 2t + 1, then 16c + 2g + 1
    float m[ROW_TILES][2], l[ROW_TILES][2], up[ROW_TILES], down[ROW_TILES][2];   // of rows 2t, 2t + 1, but up: what row g's queries are multiplied by; down: the dot products (times the scale, where there is no cap)
    int limit[ROW_TILES][2];                            // keys of the unit that the rows see
    bool seen[ROW_TILES][2];
    // four elements of row r, columns 16c + 4t ..
    PG_DEVINL static float4 load_q(uint32_t q_at, int r, int c) {
        const int t = threadIdx.x & 3;
        if constexpr (sizeof(T) == 4) {
            float4 v;
            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(q_at + piece_at(r, 4 * c + t, S::Q_ROW)));
            return v;
        } else {
            uint32_t a, b;
            asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(a), "=r"(b) : "r"(q_at + piece_at(r, 2 * c + (t >> 1), S::Q_ROW) + 8 * (t & 1)));
            const float2 x = open_word(a, T()), y = open_word(b, T());
            return make_float4(x.x, x.y, y.x, y.y);
        }
    }
    PG_DEVINL void begin(const Attn8Params<T>& p, uint32_t q_at) {
        const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
        __syncwarp();
#pragma unroll
        for (int n = 0; n < ROW_TILES; n++) {
            float2 f = make_float2(1.0f, 1.0f);
            if constexpr (!std::is_same<T, __half>::value) {
                float most = 0.0f;
#pragma unroll
                for (int c = 0; c < S::CHUNKS; c++) {
                    const float4 v = load_q(q_at, 8 * n + g, c);
                    most = fmaxf(fmaxf(fmaxf(most, fabsf(v.x)), fmaxf(fabsf(v.y), fabsf(v.z))), fabsf(v.w));
                }
                most = fmaxf(most, __shfl_xor_sync(~0u, most, 1));
                most = fmaxf(most, __shfl_xor_sync(~0u, most, 2));
                f = row_factor(most);
            }
            up[n] = f.x;
            if constexpr (N == 1) {
#pragma unroll
                for (int c = 0; c < S::CHUNKS; c++) {
                    const float4 v = load_q(q_at, 8 * n + g, c);
                    q[c][n][0] = to_halves(v.x * f.x, v.y * f.x);
                    q[c][n][1] = to_halves(v.z * f.x, v.w * f.x);
                }
            }
            if (!(p.softcap > 0.0f)) f.y = fminf(fmaxf(f.y * p.scale2, -FLT_MAX), FLT_MAX);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                down[n][i] = __shfl_sync(~0u, f.y, 8 * t + 4 * i);
                m[n][i] = -INFINITY;
                l[n][i] = 0.0f;
                seen[n][i] = false;
            }
        }
#pragma unroll
        for (int c = 0; c < S::CHUNKS; c++)
#pragma unroll
            for (int n = 0; n < ROW_TILES; n++)
#pragma unroll
                for (int k = 0; k < 4; k++) o[c][n][k] = 0.0f;
    }
    // there: bit j: key j of the warp's is there; first: number of its first key; scales: of the warp's keys and values in shared memory; by: room for the values' reciprocals
    PG_DEVINL void tile(const Attn8Params<T>& p, uint32_t q_at, uint32_t k_at, uint32_t v_at, uint32_t there, int first, float* scales, float* by) {
        const int lane = threadIdx.x & 31, g = lane >> 2;
        float *ks = scales, *vs = scales + S::WARP_KEYS;
        float s[S::KEY_TILES][ROW_TILES][4] = {};   // keys 16j + g of rows 2t and 2t + 1, then keys 16j + g + 8
        if (lane < S::WARP_KEYS) {   // (in their places)
            const float2 v = value_terms(vs[lane]);
            vs[lane] = v.x;
            by[lane] = v.y;
        }
        __syncwarp();   // (ldmatrix and mma are for a warp in step)
        // keys: a matrix is 8 keys of 16 columns; a lane gets columns 4t .. 4t + 3 of key g, which stand for columns 2t, 2t + 1, 2t + 8 and 2t + 9 of the product, as the queries' do
#pragma unroll
        for (int c = 0; c < S::CHUNKS; c += 2 / S::KEY_TILES) {
            uint32_t w[4];
            if constexpr (S::KEY_TILES == 2) ldmatrix4(w, k_at + code_at<S>(lane, c));
            else ldmatrix4(w, k_at + code_at<S>(lane & 15, c + (lane >> 4)));
#pragma unroll
            for (int d = 0; d < 2 / S::KEY_TILES; d++) {
                uint32_t b[N][ROW_TILES][2];
#pragma unroll
                for (int n = 0; n < ROW_TILES; n++) {
                    if constexpr (N == 1) {
                        b[0][n][0] = q[c + d][n][0];
                        b[0][n][1] = q[c + d][n][1];
                    } else {
                        const float4 v = load_q(q_at, 8 * n + g, c + d);
                        uint32_t x[N], y[N];
                        split_halves<N>(v.x * up[n], v.y * up[n], x);
                        split_halves<N>(v.z * up[n], v.w * up[n], y);
#pragma unroll
                        for (int k = 0; k < N; k++) { b[k][n][0] = x[k]; b[k][n][1] = y[k]; }
                    }
                }
#pragma unroll
                for (int j = 0; j < S::KEY_TILES; j++) {
                    uint32_t a[4];
                    codes_to_halves<FORM, 0>(w[2 * (S::KEY_TILES * d + j)], a[0], a[2]);
                    codes_to_halves<FORM, 0>(w[2 * (S::KEY_TILES * d + j) + 1], a[1], a[3]);
#pragma unroll
                    for (int n = 0; n < ROW_TILES; n++)
#pragma unroll
                        for (int k = N - 1; k >= 0; k--) mma16816(s[j][n], a, b[k][n][0], b[k][n][1], __half());
                }
            }
        }
        // scores, in powers of two, and the values' scales
#pragma unroll
        for (int j = 0; j < S::KEY_TILES; j++) {
            const float k[2] = {ks[16 * j + g], ks[16 * j + g + 8]}, v[2] = {vs[16 * j + g], vs[16 * j + g + 8]};
            if (p.softcap > 0.0f) {
                float flat[4 * ROW_TILES];
#pragma unroll
                for (int i = 0; i < 4 * ROW_TILES; i++) flat[i] = s[j][i >> 2][i & 3] * down[i >> 2][i & 1] * k[i >> 1 & 1];
                cap_scores(p, flat);
#pragma unroll
                for (int i = 0; i < 4 * ROW_TILES; i++) s[j][i >> 2][i & 3] = flat[i] + v[i >> 1 & 1];
            } else {
#pragma unroll
                for (int i = 0; i < 4 * ROW_TILES; i++) s[j][i >> 2][i & 3] = fmaf(s[j][i >> 2][i & 3] * k[i >> 1 & 1], down[i >> 2][i & 1], v[i >> 1 & 1]);
            }
        }
        constexpr uint32_t ALL = S::WARP_KEYS == 32 ? ~0u : (1u << S::WARP_KEYS % 32) - 1;
        int least = limit[0][0];
#pragma unroll
        for (int i = 1; i < 2 * ROW_TILES; i++) least = min(least, limit[i >> 1][i & 1]);
        if (!__all_sync(~0u, there == ALL && least - first >= S::WARP_KEYS)) {
#pragma unroll
            for (int n = 0; n < ROW_TILES; n++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int left = limit[n][i] - first;
                    const uint32_t sees = there & (left >= S::WARP_KEYS ? ALL : left <= 0 ? 0u : (1u << left) - 1);
                    seen[n][i] = seen[n][i] || sees;
#pragma unroll
                    for (int k = 0; k < 2 * S::KEY_TILES; k++)
                        if (!(sees >> (8 * k + g) & 1)) s[k >> 1][n][2 * (k & 1) + i] = -INFINITY;
                }
        } else {
#pragma unroll
            for (int n = 0; n < ROW_TILES; n++) seen[n][0] = seen[n][1] = true;
        }
        float now[ROW_TILES][2];
        bool grows = false;
#pragma unroll
        for (int n = 0; n < ROW_TILES; n++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                now[n][i] = fmaxf(s[0][n][i], s[0][n][2 + i]);
                if (S::KEY_TILES == 2) now[n][i] = fmaxf(now[n][i], fmaxf(s[S::KEY_TILES - 1][n][i], s[S::KEY_TILES - 1][n][2 + i]));
                grows = grows || now[n][i] > m[n][i] + (SHIFT8 + 8.0f);
            }
        // m is raised when an exponent is 8 above it, which is rare after the first tiles: weights stay below 2^15
        if (__any_sync(~0u, grows)) {
#pragma unroll
            for (int n = 0; n < ROW_TILES; n++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
#pragma unroll
                    for (int d = 4; d < 32; d *= 2) now[n][i] = fmaxf(now[n][i], __shfl_xor_sync(~0u, now[n][i], d));
                    const float top = fmaxf(m[n][i], now[n][i] - SHIFT8), corr = ex2(m[n][i] - (top == -INFINITY ? 0.0f : top));
                    m[n][i] = top;
                    l[n][i] *= corr;
#pragma unroll
                    for (int c = 0; c < S::CHUNKS; c++) { o[c][n][i] *= corr; o[c][n][2 + i] *= corr; }
                }
        }
        // weights, as the second operand: 16 keys a step
        uint32_t b[S::KEY_TILES][N][ROW_TILES][2];
#pragma unroll
        for (int n = 0; n < ROW_TILES; n++) {
            const float base[2] = {m[n][0] == -INFINITY ? 0.0f : m[n][0], m[n][1] == -INFINITY ? 0.0f : m[n][1]};
#pragma unroll
            for (int k = 0; k < 2 * S::KEY_TILES; k++) {
                const float f = by[8 * k + g], x = ex2(s[k >> 1][n][2 * (k & 1)] - base[0]), y = ex2(s[k >> 1][n][2 * (k & 1) + 1] - base[1]);
                l[n][0] = fmaf(x, f, l[n][0]);   // (of this lane's keys: the eight lanes of a row meet at the end)
                l[n][1] = fmaf(y, f, l[n][1]);
                uint32_t w[N];
                split_halves<N>(x, y, w);
#pragma unroll
                for (int i = 0; i < N; i++) b[k >> 1][i][n][k & 1] = transpose8(w[i]);
            }
        }
        // values: a matrix is 8 keys of 16 columns, transposed in pairs of columns: a lane gets columns 2g and 2g + 1 of keys 2t and 2t + 1; rows g and g + 8 of the product stand for them
#pragma unroll
        for (int c = 0; c < S::CHUNKS; c += 2 / S::KEY_TILES) {
            uint32_t w[4];
            if constexpr (S::KEY_TILES == 2) ldmatrix4t(w, v_at + code_at<S>(lane, c));
            else ldmatrix4t(w, v_at + code_at<S>(lane & 15, c + (lane >> 4)));
#pragma unroll
            for (int d = 0; d < 2 / S::KEY_TILES; d++)
#pragma unroll
                for (int j = 0; j < S::KEY_TILES; j++) {
                    uint32_t a[4];
                    codes_to_halves<FORM, 1>(w[2 * (S::KEY_TILES * d + j)], a[0], a[1]);
                    codes_to_halves<FORM, 1>(w[2 * (S::KEY_TILES * d + j) + 1], a[2], a[3]);
#pragma unroll
                    for (int n = 0; n < ROW_TILES; n++)
#pragma unroll
                        for (int k = N - 1; k >= 0; k--) mma16816(o[c + d][n], a, b[j][k][n][0], b[j][k][n][1], __half());
                }
        }
    }
    PG_DEVINL void put_ml(float2* ml) {   // [ROWS]
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int n = 0; n < ROW_TILES; n++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const bool any = __shfl_sync(~0u, (int)seen[n][i], lane & 3);   // (the same for the lanes of a row)
#pragma unroll
                for (int d = 4; d < 32; d *= 2) l[n][i] += __shfl_xor_sync(~0u, l[n][i], d);
                if (lane < 4) ml[8 * n + 2 * lane + i] = make_float2(m[n][i], any ? l[n][i] : -1.0f);
            }
    }
    // [ROWS][COLS] as sum8_at has them, columns from COLS * pass on, times the rows' factors (lane r has row r's)
    PG_DEVINL void put_o(float* to, float factor, int pass) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int n = 0; n < ROW_TILES; n++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int r = 8 * n + 2 * t + i;
                const float f = __shfl_sync(~0u, factor, r);
#pragma unroll
                for (int c = 0; c < S::CHUNKS; c++)
                    if (c / (S::COLS / 16) == pass)
                        *reinterpret_cast<float2*>(to + sum8_at<S::COLS>(r, 16 * (c % (S::COLS / 16)) + 2 * g)) = make_float2(o[c][n][i] * f, o[c][n][2 + i] * f);
            }
    }
};

template <typename T, int FORM, int DP, int ROW_TILES>
__global__ void __launch_bounds__(TileShape8<T, DP, ROW_TILES>::THREADS, TileShape8<T, DP, ROW_TILES>::CTAS) rows8_kernel(const __grid_constant__ Attn8Params<T> p, const __grid_constant__ Line l, const __grid_constant__ Boxes8 boxes) {
    using S = TileShape8<T, DP, ROW_TILES>;
    extern __shared__ uint8_t raw[];
    __shared__ Walk walks[S::WARPS][S::STAGES];   // a warp's: of the units that its copies have got to, by their number in this CTA modulo STAGES
    __shared__ uint64_t full[S::WARPS][S::STAGES];
    __shared__ float2 ml[S::WARPS][S::ROWS];
    __shared__ int gave_up_at;
    const int t = threadIdx.x, lane = t & 31, warp = __shfl_sync(~0u, t >> 5, 0), D = p.head_size;
    uint8_t* smem = raw + (((smem_at(raw) + 1023u) & ~1023u) - smem_at(raw));
    uint8_t *slots = smem + warp * (S::STAGES * S::SLOT), *queries = smem + S::WARPS * S::STAGES * S::SLOT;
    float* scales = reinterpret_cast<float*>(queries + S::Q) + warp * (S::STAGES * S::SCALES + S::WARP_KEYS);
    volatile int* gave_up = &gave_up_at;
    if (t < S::WARPS * S::STAGES) mbar_init(&full[0][0] + t, 1);
    if (t == 0) gave_up_at = 0;
    fence_barrier_init();

    Walk ahead;   // where copies are
    int64_t from, to;
    walk_begin<T, S::THREADS>(p, l, ahead, from, to);   // (synchronises the CTA)
    grid_launch();
    // The kernel before may still run.  The last CTA ends after it, so that whoever waits for this kernel waits for both; the others leave their SM to the next ones
    const bool last_cta = blockIdx.x == gridDim.x - 1;
    if (from >= to) { if (last_cta) grid_wait(); return; }

    const int n_tiles = (int)(to - from), whole = D / 16;
    int copied = 0, slot_to = 0, set_to = 0;    // tiles copied, the slot and the unit's set that the next goes to
    bool first = true, ok = true;
    uint32_t there[S::STAGES], by_tma = 0, written = 0, rounds = 0;   // a bit a slot: a tile is on its way by TMA, its bytes were last written otherwise, the phase that its barrier is in
    int page = -1, at_page = 0;   // of this lane's key in the tile that is copied next: what its table says (looked at when the copies are asked for, so that nothing waits for it), and its place there
    auto copy_queries = [&](const Walk& w) {   // by all threads
        constexpr int PIECES = S::Q_ROW / 16, VEC = 16 / sizeof(T);
        for (int e = t; e < S::ROWS * PIECES; e += S::THREADS) {
            const int x = e / PIECES, c = e % PIECES;
            const UnitRow r = unit_row(p, l, w, x);
            const bool in = r.row >= 0 && c * VEC < D;
            const T* q = in ? p.q.data + r.row * p.q.row + r.head * p.q.head + c * VEC : p.q.data;
            uint8_t* to_q = queries + piece_at(x, c, S::Q_ROW);
            if (p.q_wide) {
                copy16(smem_at(to_q), q, in);
            } else {
                Piece<T, VEC> v;
#pragma unroll
                for (int i = 0; i < VEC; i++) v.v[i] = in ? q[i] : from_f<T>(0.0f);
                *reinterpret_cast<Piece<T, VEC>*>(to_q) = v;
            }
        }
        copy_commit();
    };
    auto look = [&]() {   // (as unit_place)
        const int x = ahead.tile * S::KEYS + warp * S::WARP_KEYS + (lane & (S::WARP_KEYS - 1));
        page = -1;
        if (x < ahead.keys) {
            const int i = p.page_shift >= 0 ? x >> p.page_shift : x / p.batch.page_size;
            page = (ahead.b < 0 ? p.batch.prefix : p.batch.tables + ahead.b * p.batch.table_stride)[i];
            at_page = x - i * p.batch.page_size;
        }
    };
    // boxes of a lane: keys or values, rows, columns
    constexpr int COL_BOXES = DP / S::BOX;
    const int box_rows = boxes.rows, groups = box_rows ? S::WARP_KEYS / box_rows : 0, box = lane % max(1, 2 * COL_BOXES * groups), box_value = box & 1, box_col = (box >> 1) % COL_BOXES, box_group = (box >> 1) / COL_BOXES;
    auto copy_tile = [&]() {   // the warp's part of the tile that `ahead` stands at, whose places are known; then on to the next one.  A warp that gave up copies nothing, but walks on: all warps go by the units that warp 0 writes down
        if (copied < n_tiles) {
            if (ok) {
                const bool is = page >= 0 && page < p.batch.pages;
                const uint32_t to_codes = smem_at(slots) + slot_to * S::SLOT, bits = __ballot_sync(~0u, is) & (S::WARP_KEYS == 32 ? ~0u : (1u << S::WARP_KEYS % 32) - 1);
#pragma unroll
                for (int i = 0; i < S::STAGES; i++)
                    if (i == slot_to) there[i] = bits;
                const int page_or_0 = is ? page : 0, at = is ? at_page : 0;
                if (box_rows && ahead.tile * S::KEYS + (warp + 1) * S::WARP_KEYS <= ahead.keys) {
                    if (written >> slot_to & 1) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_expect_tx(&full[warp][slot_to], S::SLOT);
                    int of = __shfl_sync(~0u, is ? page : -1, box_group * box_rows & 31), from_row = __shfl_sync(~0u, at, box_group * box_rows & 31);
                    if (of < 0) { of = p.batch.pages; from_row = 0; }   // (outside the map: zeros)
                    __syncwarp();
                    if (lane < 2 * COL_BOXES * groups)
                        tma_box(to_codes + box_value * S::KV + box_col * (S::WARP_KEYS * S::BOX) + box_group * box_rows * S::BOX, box_value ? &boxes.v : &boxes.k, S::BOX * box_col, from_row, ahead.head, of,
                                box_value ? boxes.v_place : boxes.k_place, box_value ? boxes.v_head : boxes.k_head, &full[warp][slot_to]);
                    __syncwarp();
                    by_tma |= 1u << slot_to;
                    written &= ~(1u << slot_to);
                } else {
                    by_tma &= ~(1u << slot_to);
                    written |= 1u << slot_to;
                    const int64_t k_from = is ? page_or_0 * p.c.k_page + at * p.c.k_slot + ahead.head * p.c.k_head : -1, v_from = is ? page_or_0 * p.c.v_page + at * p.c.v_slot + ahead.head * p.c.v_head : -1;
                    constexpr int LANES = S::CHUNKS < 8 ? S::CHUNKS : 8, AT_ONCE = 32 / LANES;   // lanes a row, rows at a time
#pragma unroll 2
                    for (int r0 = 0; r0 < S::WARP_KEYS; r0 += AT_ONCE) {
                        const int row = r0 + lane / LANES;
                        const int64_t k = __shfl_sync(~0u, k_from, row), v = __shfl_sync(~0u, v_from, row);
#pragma unroll
                        for (int c = 0; c < S::CHUNKS; c += LANES) {
                            const int piece = c + lane % LANES;
                            const bool in = k >= 0 && piece < whole;
                            copy16(to_codes + code_at<S>(row, piece), in ? p.c.k + k + 16 * piece : p.c.k, in);
                            copy16(to_codes + S::KV + code_at<S>(row, piece), in ? p.c.v + v + 16 * piece : p.c.v, in);
                        }
                    }
                }
                if (lane < S::WARP_KEYS) {
                    const int block = p.block_shift >= 0 ? at >> p.block_shift : at / p.c.block;
                    const uint32_t to_scale = smem_at(scales + slot_to * S::SCALES) + 4 * lane;
                    copy4(to_scale, p.c.ks + page_or_0 * p.c.ks_page + block * p.c.ks_block + ahead.head * p.c.ks_head, is);
                    copy4(to_scale + 4 * S::WARP_KEYS, p.c.vs + page_or_0 * p.c.vs_page + block * p.c.vs_block + ahead.head * p.c.vs_head, is);
                }
            }
            if (first) {
                if (lane == 0) walks[warp][set_to] = ahead;
                first = false;
            }
            slot_to = slot_to + 1 == S::STAGES ? 0 : slot_to + 1;
            if (++copied < n_tiles) {
                if (++ahead.tile == ahead.tiles) {
                    walk_next_unit(p, l, ahead);
                    set_to = set_to + 1 == S::STAGES ? 0 : set_to + 1;
                    first = true;
                }
                look();
            }
        }
        copy_commit();
    };
    look();
#pragma unroll 1
    for (int i = 0; i < S::STAGES - 1; i++) copy_tile();

    WarpTile8<T, FORM, DP, ROW_TILES> tile;
    int set = S::STAGES - 1, slot = S::STAGES - 1, begun = 0, now = 0, tiles = 0;   // now: the tile of the unit that is worked on
    bool start = true;
#pragma unroll 1
    for (int at = 0; at < n_tiles; at++) {
        slot = slot + 1 == S::STAGES ? 0 : slot + 1;
        if (start) {
            set = set + 1 == S::STAGES ? 0 : set + 1;
            __syncwarp();
            copy_queries(walks[warp][set]);
            copy_wait<0>();
            __syncthreads();          // the other warps' parts of them
            tile.begin(p, smem_at(queries));
            const Walk& w = walks[0][set];   // (one for all warps, which meet as often as it says: lengths that change under the kernel may part the others)
            begun = now = w.tile;
            tiles = w.tiles;
#pragma unroll
            for (int i = 0; i < 2 * ROW_TILES; i++) tile.limit[i >> 1][i & 1] = unit_row(p, l, w, 8 * (i >> 1) + 2 * (lane & 3) + (i & 1)).keys;
            start = false;
        } else {
            copy_wait<S::STAGES - 2>();   // (of the scales, and what does not come by TMA)
        }
        __syncwarp();
        copy_tile();                  // (into the slot of the tile before, which this warp has worked on)
        if (ok && (by_tma >> slot & 1)) {
            ok = __all_sync(~0u, dense::mbar_wait_bounded(&full[warp][slot], rounds >> slot & 1, gave_up, dense::TG_ROWS8 + dense::TG_FULL));
            if (ok) {
                rounds ^= 1u << slot;
                by_tma &= ~(1u << slot);
            }
        }
        __syncwarp();
        if (ok) {
            uint32_t bits = there[0];
#pragma unroll
            for (int i = 1; i < S::STAGES; i++)
                if (i == slot) bits = there[i];
            tile.tile(p, smem_at(queries), smem_at(slots) + slot * S::SLOT, smem_at(slots) + slot * S::SLOT + S::KV, bits, now * S::KEYS + warp * S::WARP_KEYS, scales + slot * S::SCALES, scales + S::STAGES * S::SCALES);
        } else {   // gave up: what this warp still had to do comes out as NaN
#pragma unroll
            for (int i = 0; i < 2 * ROW_TILES; i++) {
                tile.l[i >> 1][i & 1] = NAN;
                tile.seen[i >> 1][i & 1] = true;
            }
        }
        now++;
        if (now == tiles || at + 1 == n_tiles) {   // the part ends: the warps' rows meet in their slots
            const Walk& w = walks[0][set];
            tile.put_ml(ml[warp]);
            __syncthreads();
            // lane r: row r's largest exponent, what this warp's sums are multiplied by, the sum of the weights
            float m = -INFINITY, sum = 0.0f, mine = 0.0f;
            bool any = false;
#pragma unroll
            for (int i = 0; i < S::WARPS; i++)
                if (!(ml[i][lane & (S::ROWS - 1)].y < 0.0f)) { m = fmaxf(m, ml[i][lane & (S::ROWS - 1)].x); any = true; }
            const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int i = 0; i < S::WARPS; i++) {
                const bool has = !(ml[i][lane & (S::ROWS - 1)].y < 0.0f);
                const float f = has ? ex2(ml[i][lane & (S::ROWS - 1)].x - base) : 0.0f;
                if (has) sum += ml[i][lane & (S::ROWS - 1)].y * f;
                if (i == warp) mine = f;
            }
            if (!any) sum = -1.0f;
            const int used = w.b < 0 ? (int)min((int64_t)S::ROWS, p.batch.n_rows * p.group - (int64_t)w.row_tile * S::ROWS) : min(S::ROWS, w.s.count * p.group - w.row_tile * S::ROWS);
            const float* rows = reinterpret_cast<const float*>(smem + slot * S::SLOT);
            const bool whole_part = whole_unit(p, w, begun, now - 1);
            const int64_t slot_of_part = w.unit + blockIdx.x;
#pragma unroll
            for (int pass = 0; pass < DP / S::COLS; pass++) {
                if (pass) __syncthreads();
                __syncwarp();
                tile.put_o(reinterpret_cast<float*>(slots + slot * S::SLOT), mine, pass);
                __syncthreads();
                const int quads = min(S::COLS, D - pass * S::COLS) / 4;
                for (int x = warp; x < used; x += S::WARPS) {   // a warp a row, a lane four columns
                    const float row_m = __shfl_sync(~0u, m, x), row_sum = __shfl_sync(~0u, sum, x);
                    if (lane < quads) {
                        const int c = 4 * lane, column = pass * S::COLS + c;
                        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        if (!(row_sum < 0.0f)) {
#pragma unroll
                            for (int i = 0; i < S::WARPS; i++) {
                                const float4 a = *reinterpret_cast<const float4*>(rows + i * (S::STAGES * S::SLOT / 4) + sum8_at<S::COLS>(x, c));
                                v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
                            }
                        }
                        if (whole_part) {
                            const UnitRow r = unit_row(p, l, w, x);
                            if (!(row_sum < 0.0f)) { v.x /= row_sum; v.y /= row_sum; v.z /= row_sum; v.w /= row_sum; }
                            store_row(p, r, column, v);
                            if (column == 0 && p.lse) p.lse[r.row * p.q_heads + r.head] = row_sum < 0.0f ? -INFINITY : lse_of(row_m, row_sum);
                        } else if (slot_of_part < l.slots) {
                            *reinterpret_cast<float4*>(part_at(l, D, slot_of_part, x, column)) = v;
                            if (column == 0) l.ml[slot_of_part * S::ROWS + x] = make_float2(row_m, row_sum);
                        }
                    }
                    __syncwarp();
                }
            }
            written |= 1u << slot;
            start = true;
            __syncthreads();   // (before the slots are copied to again)
        }
    }
    copy_wait<0>();
    if (!ok) {   // what TMA was asked for lands before shared memory goes away
        for (int i = 0; i < S::STAGES; i++)
            if (by_tma >> i & 1) dense::mbar_wait_for(&full[warp][i], rounds >> i & 1, nullptr);
        if (lane == 0 && p.err) *p.err = *gave_up;
    }
    if (last_cta) grid_wait();
}

}  // namespace paged
}  // namespace lmrs
