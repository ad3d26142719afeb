// paged8_attn.cuh -- attention of the rows of many sequences over pages of 8-bit codes and over a prefix that all of them share.  The line of tiles, its units and parts, and their joining are
// those of paged_attn.cuh; what differs is how a tile's products are made.
//
// For one row: out = sum_j e^(s_j) v_j c_j / sum_j e^(s_j), s_j = scale * k_j (q . kc_j), where kc_j and c_j are codes and k_j and v_j their scales.  Codes are float16 numbers, so
//     scores     are tensor-core products of the queries in float16 and the codes as they are, times k_j in float32
//     weights    are w_j = 2^(s_j log2 e + log2 v_j - m): the values' scales go into the weights' exponents, m is the largest exponent (less 7), and the codes are multiplied as they are
//     the sum    of e^(s_j) is that of w_j / v_j, in float32
// The queries' types: float16 as it is; bfloat16, whose 8 bits of mantissa float16 has, times a power of two for each row that brings its largest element to 2^14 (what is below 2^-38 of that loses
// bits: 2^-40 of the largest element at most); float32 the same way in three pieces of 11 bits each.  Weights in float16: up to 2^7, rounded by 2^-11 of each and 2^-32 of the largest; float32: in three pieces.
#pragma once
#include "paged8.h"
#include "paged_attn.cuh"

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
constexpr float SHIFT8 = 7.0f;   // m is so much less than the largest exponent
// the exponent and the reciprocal of a scale of values (a scale that is NaN leaves a finite reciprocal: it reaches whoever has the weight)
PG_DEVINL float2 value_terms(float v) {
    const float c = fminf(fmaxf(v, SCALE_LEAST), SCALE_MOST);
    float lg, by;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(lg) : "f"(c));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(by) : "f"(c));
    return make_float2(v == v ? lg : v, by);
}

// CTA = 4 warps that share a tile's keys, as in rows16_kernel.  What bounds it is the bytes of the pages, and next to them the conversions: 16 codes a lane take 4 to 6 instructions for each 4.
template <typename T, int DP> struct TileShape8 {
    static constexpr int PIECES = sizeof(T) == 4 ? 3 : 1;   // of queries and weights
    static constexpr int ROWS = 16, THREADS = 128, ROW = DP, CHUNKS = DP / 16, KEYS = DP <= 128 ? 128 : 64, STAGES = DP > 128 || (sizeof(T) == 4 && DP > 64) ? 2 : 3;
    static constexpr int WARP_KEYS = KEYS / 4, COPY_KEYS = KEYS / 32, TILES = WARP_KEYS / 8;   // keys a warp works on; keys a thread copies a quarter of; 8 keys' scores
    static constexpr int Q_ROW = DP * (int)sizeof(T), Q = ROWS * Q_ROW, KV = KEYS * ROW, STAGE = 2 * KV + 8 * KEYS, SMEM = STAGES * (STAGE + Q);
    static constexpr int CTAS = DP <= 64 ? 3 : 2;
    static constexpr int COLS = DP < 128 ? DP : 128;        // columns at a time where the warps' rows meet
    static_assert(4 * ROWS * COLS * 4 <= 2 * KV, "the four warps' rows fit where a tile's keys and values were");
};
// rows of 64 bytes: two of them make a line of the banks
template <int ROW> PG_DEVINL uint32_t code_at(int row, int piece) { return (uint32_t)(row * ROW + ((piece ^ (ROW == 64 ? row >> 1 & 3 : row & 7)) << 4)); }
template <int COLS> PG_DEVINL int sum8_at(int r, int c) { return r * COLS + (c ^ ((r & 1) << 4)); }

template <typename T, int FORM, int DP> struct WarpTile8 {
    using S = TileShape8<T, DP>;
    static constexpr int N = S::PIECES;
    uint32_t q[N == 1 ? S::CHUNKS : 1][4];   // (float32: cut into pieces again for each tile, since they do not fit the registers)
    float o[S::CHUNKS][2][4];                // columns 16c + 4t + {0, 2} and {1, 3} of rows lane / 4 and lane / 4 + 8, t = lane % 4
    float m[2], l[2], up[2], down[2];        // up: what the queries are multiplied by
    bool seen[2];
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
    PG_DEVINL void begin(uint32_t q_at) {
        const int g = (threadIdx.x & 31) >> 2;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 2; i++) {
            float most = 0.0f;
            if constexpr (!std::is_same<T, __half>::value) {
#pragma unroll
                for (int c = 0; c < S::CHUNKS; c++) {
                    const float4 v = load_q(q_at, g + 8 * i, c);
                    most = fmaxf(fmaxf(fmaxf(most, fabsf(v.x)), fmaxf(fabsf(v.y), fabsf(v.z))), fabsf(v.w));
                }
                most = fmaxf(most, __shfl_xor_sync(~0u, most, 1));
                most = fmaxf(most, __shfl_xor_sync(~0u, most, 2));
                const float2 f = row_factor(most);
                up[i] = f.x;
                down[i] = f.y;
            } else {
                up[i] = down[i] = 1.0f;
            }
            if constexpr (N == 1) {
#pragma unroll
                for (int c = 0; c < S::CHUNKS; c++) {
                    const float4 v = load_q(q_at, g + 8 * i, c);
                    q[c][i] = to_halves(v.x * up[i], v.y * up[i]);
                    q[c][2 + i] = to_halves(v.z * up[i], v.w * up[i]);
                }
            }
            m[i] = -INFINITY;
            l[i] = 0.0f;
            seen[i] = false;
        }
#pragma unroll
        for (int c = 0; c < S::CHUNKS; c++)
#pragma unroll
            for (int k = 0; k < 4; k++) o[c][0][k] = o[c][1][k] = 0.0f;
    }
    // there: bit j: key j of the warp's is there; first: number of its first key; row_keys: how many keys each row sees; ks, vs: the warp's keys' scales in shared memory, by: room for as many floats
    PG_DEVINL void tile(const Attn8Params<T>& p, uint32_t q_at, uint32_t k_at, uint32_t v_at, uint32_t there, int first, const int* row_keys, float* ks, float* vs, float* by) {
        const int lane = threadIdx.x & 31, t = lane & 3, key0 = S::WARP_KEYS * (threadIdx.x >> 5);
        float s[S::TILES][4] = {};
        if (lane < S::WARP_KEYS) {   // (in their places)
            const float2 v = value_terms(vs[lane]);
            vs[lane] = v.x;
            by[lane] = v.y;
        }
        __syncwarp();   // (ldmatrix and mma are for a warp in step)
        // keys: a matrix is 8 keys of 16 columns; a lane gets columns 4t .. 4t + 3 of key lane / 4, which stand for rows 2t, 2t + 1, 2t + 8 and 2t + 9 of the product's second operand, as the queries' do for
        // columns of the first
#pragma unroll
        for (int c = 0; c < S::CHUNKS; c += 4 / S::TILES) {
            uint32_t w[4];
            if constexpr (S::TILES == 4) ldmatrix4(w, k_at + code_at<S::ROW>(key0 + lane, c));
            else ldmatrix4(w, k_at + code_at<S::ROW>(key0 + (lane & 15), c + (lane >> 4)));
#pragma unroll
            for (int d = 0; d < 4 / S::TILES; d++) {
                uint32_t a[N][4];
                if constexpr (N == 1) {
#pragma unroll
                    for (int k = 0; k < 4; k++) a[0][k] = q[c + d][k];
                } else {
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const float4 v = load_q(q_at, lane / 4 + 8 * i, c + d);
                        uint32_t x[N], y[N];
                        split_halves<N>(v.x * up[i], v.y * up[i], x);
                        split_halves<N>(v.z * up[i], v.w * up[i], y);
#pragma unroll
                        for (int k = 0; k < N; k++) { a[k][i] = x[k]; a[k][2 + i] = y[k]; }
                    }
                }
#pragma unroll
                for (int n = 0; n < S::TILES; n++) {
                    uint32_t b0, b1;
                    codes_to_halves<FORM, 0>(w[S::TILES * d + n], b0, b1);
#pragma unroll
                    for (int k = N - 1; k >= 0; k--) mma16816(s[n], a[k], b0, b1, __half());
                }
            }
        }
        // scores
#pragma unroll
        for (int n = 0; n < S::TILES; n++) {
            const float2 k = *reinterpret_cast<const float2*>(ks + 8 * n + 2 * t);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                s[n][2 * i] *= down[i] * k.x;
                s[n][2 * i + 1] *= down[i] * k.y;
            }
        }
        if (p.softcap > 0.0f) {
            float flat[4 * S::TILES];
#pragma unroll
            for (int i = 0; i < 4 * S::TILES; i++) flat[i] = s[i >> 2][i & 3];
            cap_scores(p, flat);
#pragma unroll
            for (int i = 0; i < 4 * S::TILES; i++) s[i >> 2][i & 3] = flat[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4 * S::TILES; i++) s[i >> 2][i & 3] *= p.scale2;
        }
#pragma unroll
        for (int n = 0; n < S::TILES; n++) {
            const float2 v = *reinterpret_cast<const float2*>(vs + 8 * n + 2 * t);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                s[n][2 * i] += v.x;
                s[n][2 * i + 1] += v.y;
            }
        }
        constexpr uint32_t ALL = S::WARP_KEYS == 32 ? ~0u : (1u << S::WARP_KEYS % 32) - 1;
        const int limit[2] = {row_keys[lane / 4] - first, row_keys[lane / 4 + 8] - first};
        if (!__all_sync(~0u, there == ALL && limit[0] >= S::WARP_KEYS && limit[1] >= S::WARP_KEYS)) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint32_t sees = there & (limit[i] >= S::WARP_KEYS ? ALL : limit[i] <= 0 ? 0u : (1u << limit[i]) - 1);
                seen[i] = seen[i] || sees;
#pragma unroll
                for (int n = 0; n < S::TILES; n++)
#pragma unroll
                    for (int c = 0; c < 2; c++)
                        if (!(sees >> (8 * n + 2 * t + c) & 1)) s[n][2 * i + c] = -INFINITY;
            }
        } else {
            seen[0] = seen[1] = true;
        }
        float now[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int n = 0; n < S::TILES; n++) now[i] = fmaxf(now[i], fmaxf(s[n][2 * i], s[n][2 * i + 1]));
#pragma unroll
        for (int d = 1; d < 4; d *= 2)
#pragma unroll
            for (int i = 0; i < 2; i++) now[i] = fmaxf(now[i], __shfl_xor_sync(~0u, now[i], d));
        if (__any_sync(~0u, now[0] - SHIFT8 > m[0] || now[1] - SHIFT8 > m[1])) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float top = fmaxf(m[i], now[i] - SHIFT8), corr = ex2(m[i] - (top == -INFINITY ? 0.0f : top));
                m[i] = top;
                l[i] *= corr;
#pragma unroll
                for (int c = 0; c < S::CHUNKS; c++)
#pragma unroll
                    for (int h = 0; h < 2; h++) { o[c][h][2 * i] *= corr; o[c][h][2 * i + 1] *= corr; }
            }
        }
        // weights, as the first operand: 16 keys a step
        uint32_t a[S::TILES / 2][N][4];
        const float base[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
#pragma unroll
        for (int n = 0; n < S::TILES; n++) {
            const float2 f = *reinterpret_cast<const float2*>(by + 8 * n + 2 * t);
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float x = ex2(s[n][2 * i] - base[i]), y = ex2(s[n][2 * i + 1] - base[i]);
                l[i] = fmaf(x, f.x, fmaf(y, f.y, l[i]));   // (of this lane's keys: the four lanes of a row meet at the end)
                uint32_t w[N];
                split_halves<N>(x, y, w);
#pragma unroll
                for (int k = 0; k < N; k++) a[n >> 1][k][2 * (n & 1) + i] = w[k];
            }
        }
        // values: a matrix is 8 keys of 16 columns, transposed in pairs of columns: a lane gets columns 2 (lane / 4) and the next of keys 2t and 2t + 1, so even and odd columns are products of their own
#pragma unroll
        for (int c = 0; c < S::CHUNKS; c += 4 / S::TILES) {
            uint32_t w[4];
            if constexpr (S::TILES == 4) ldmatrix4t(w, v_at + code_at<S::ROW>(key0 + lane, c));
            else ldmatrix4t(w, v_at + code_at<S::ROW>(key0 + (lane & 15), c + (lane >> 4)));
#pragma unroll
            for (int d = 0; d < 4 / S::TILES; d++)
#pragma unroll
                for (int j = 0; j < S::TILES / 2; j++) {
                    uint32_t even[2], odd[2];
                    codes_to_halves<FORM, 1>(w[S::TILES * d + 2 * j], even[0], odd[0]);
                    codes_to_halves<FORM, 1>(w[S::TILES * d + 2 * j + 1], even[1], odd[1]);
#pragma unroll
                    for (int k = N - 1; k >= 0; k--) {
                        mma16816(o[c + d][0], a[j][k], even[0], even[1], __half());
                        mma16816(o[c + d][1], a[j][k], odd[0], odd[1], __half());
                    }
                }
        }
    }
    PG_DEVINL void put_ml(float2* ml) {   // [16]
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            l[i] += __shfl_xor_sync(~0u, l[i], 1);
            l[i] += __shfl_xor_sync(~0u, l[i], 2);
            if ((lane & 3) == 0) ml[lane / 4 + 8 * i] = make_float2(m[i], seen[i] ? l[i] : -1.0f);
        }
    }
    // [16][COLS] as sum8_at has them, columns from COLS * pass on, times the rows' factors (lane r has row r's)
    PG_DEVINL void put_o(float* to, float factor, int pass) {
        const int lane = threadIdx.x & 31, t = lane & 3;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int r = lane / 4 + 8 * i;
            const float f = __shfl_sync(~0u, factor, r);
#pragma unroll
            for (int c = 0; c < S::CHUNKS; c++)
                if (c / (S::COLS / 16) == pass)
                    *reinterpret_cast<float4*>(to + sum8_at<S::COLS>(r, 16 * (c % (S::COLS / 16)) + 4 * t)) =
                        make_float4(o[c][0][2 * i] * f, o[c][1][2 * i] * f, o[c][0][2 * i + 1] * f, o[c][1][2 * i + 1] * f);
        }
    }
};

template <typename T, int FORM, int DP>
__global__ void __launch_bounds__(TileShape8<T, DP>::THREADS, TileShape8<T, DP>::CTAS) rows16_codes_kernel(const __grid_constant__ Attn8Params<T> p, const __grid_constant__ Line l) {
    using S = TileShape8<T, DP>;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ Walk walks[S::STAGES];             // of the units that copies have got to, by their number in this CTA modulo STAGES
    __shared__ int row_keys[S::STAGES][S::ROWS];
    __shared__ __align__(16) uint8_t there[S::STAGES][S::KEYS / 8];
    __shared__ float2 ml[4][S::ROWS];
    __shared__ float2 joined[S::ROWS];
    __shared__ __align__(16) float by[S::KEYS];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, D = p.head_size;
    const uint32_t kv = smem_at(smem), queries = kv + S::STAGES * S::STAGE;

    Walk ahead;   // where copies are
    int64_t from, to;
    walk_begin<T, S::THREADS>(p, l, ahead, from, to);
    grid_launch();
    // The kernel before may still run.  The last CTA ends after it, so that whoever waits for this kernel waits for both; the others leave their SM to the next ones
    const bool last_cta = blockIdx.x == gridDim.x - 1;
    if (from >= to) { if (last_cta) grid_wait(); return; }

    // copies of a thread: keys t / 4, t / 4 + 32, ... of the tile, every fourth 16 bytes; past the end of a head zeros, so that the products need not know where it is; the first and second of four
    // neighbours also copy the keys' and the values' scales
    Place place[S::COPY_KEYS];
    const int n_tiles = (int)(to - from), whole = D / 16;
    int copied = 0, stage_to = 0, set_to = 0;   // tiles copied, the stage and the unit's set that the next goes to
    bool first = true;
    auto look = [&]() {
#pragma unroll
        for (int i = 0; i < S::COPY_KEYS; i++) place[i] = unit_place(p, ahead, ahead.tile * S::KEYS + t / 4 + 32 * i);
    };
    auto copy_tile = [&]() {   // the tile that `ahead` stands at, whose places are known; then on to the next one
        if (copied < n_tiles) {
            const uint32_t stage = kv + stage_to * S::STAGE;
#pragma unroll
            for (int i = 0; i < S::COPY_KEYS; i++) {
                const bool is = place[i].page >= 0;
                const int page = is ? place[i].page : 0, row = t / 4 + 32 * i;
                const uint8_t* k = p.c.k + page * p.c.k_page + place[i].place * p.c.k_slot + ahead.head * p.c.k_head;
                const uint8_t* v = p.c.v + page * p.c.v_page + place[i].place * p.c.v_slot + ahead.head * p.c.v_head;
#pragma unroll
                for (int c = 0; c < S::CHUNKS; c += 4) {
                    const int piece = c + (t & 3);
                    const bool in = is && (S::CHUNKS == whole || piece < whole);
                    copy16(stage + code_at<S::ROW>(row, piece), in ? k + 16 * piece : p.c.k, in);
                    copy16(stage + S::KV + code_at<S::ROW>(row, piece), in ? v + 16 * piece : p.c.v, in);
                }
                if ((t & 3) < 2) {
                    const int block = p.block_shift >= 0 ? place[i].place >> p.block_shift : place[i].place / p.c.block;
                    const float* scale = (t & 3) ? p.c.vs + page * p.c.vs_page + block * p.c.vs_block + ahead.head * p.c.vs_head : p.c.ks + page * p.c.ks_page + block * p.c.ks_block + ahead.head * p.c.ks_head;
                    copy4(stage + 2 * S::KV + 4 * (row + (t & 3) * S::KEYS), is ? scale : p.c.ks, is);
                }
                const unsigned bits = __ballot_sync(~0u, __shfl_sync(~0u, is, (4 * lane) & 31)) & 0xff;
                if (lane == 0) there[stage_to][warp + 4 * i] = (uint8_t)bits;
            }
            if (first) {
                if (t == 0) walks[set_to] = ahead;
                if (t < S::ROWS) row_keys[set_to][t] = unit_row(p, l, ahead, t).keys;
                const uint32_t q_at = queries + set_to * S::Q;
                constexpr int PIECES = S::Q_ROW / 16, VEC = 16 / sizeof(T);
                for (int e = t; e < S::ROWS * PIECES; e += S::THREADS) {
                    const int x = e / PIECES, c = e % PIECES;
                    const UnitRow r = unit_row(p, l, ahead, x);
                    const bool in = r.row >= 0 && c * VEC < D;
                    const T* q = in ? p.q.data + r.row * p.q.row + r.head * p.q.head + c * VEC : p.q.data;
                    const uint32_t at = q_at + piece_at(x, c, S::Q_ROW);
                    if (p.q_wide) {
                        copy16(at, q, in);
                    } else {
                        Piece<T, VEC> v;
#pragma unroll
                        for (int i = 0; i < VEC; i++) v.v[i] = in ? q[i] : from_f<T>(0.0f);
                        *reinterpret_cast<Piece<T, VEC>*>(smem + (at - kv)) = v;
                    }
                }
                first = false;
            }
            stage_to = stage_to + 1 == S::STAGES ? 0 : stage_to + 1;
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

    WarpTile8<T, FORM, DP> tile;
    Walk w;
    int set = S::STAGES - 1, stage = S::STAGES - 1, begun = 0, used = 0;
    bool start = true;
#pragma unroll 1
    for (int at = 0; at < n_tiles; at++) {
        copy_wait<S::STAGES - 2>();
        __syncthreads();   // the tile has landed for all threads, and the one before has been worked on by all
        copy_tile();
        stage = stage + 1 == S::STAGES ? 0 : stage + 1;
        const uint32_t k_at = kv + stage * S::STAGE, v_at = k_at + S::KV;
        if (start) {
            set = set + 1 == S::STAGES ? 0 : set + 1;
            w = walks[set];
            begun = w.tile;
            tile.begin(queries + set * S::Q);
            used = w.b < 0 ? (int)min((int64_t)S::ROWS, p.batch.n_rows * p.group - (int64_t)w.row_tile * S::ROWS) : min(S::ROWS, w.s.count * p.group - w.row_tile * S::ROWS);
            start = false;
        }
        const uint32_t bits = S::WARP_KEYS == 32 ? *reinterpret_cast<const uint32_t*>(&there[stage][4 * warp]) : *reinterpret_cast<const uint16_t*>(&there[stage][2 * warp]);
        float* scales = reinterpret_cast<float*>(smem + stage * S::STAGE + 2 * S::KV) + S::WARP_KEYS * warp;
        tile.tile(p, queries + set * S::Q, k_at, v_at, bits, w.tile * S::KEYS + warp * S::WARP_KEYS, row_keys[set], scales, scales + S::KEYS, by + S::WARP_KEYS * warp);
        const bool last = w.tile + 1 == w.tiles;
        if (last || at + 1 == n_tiles) {   // the part ends: the warps' rows meet in the tile's place
            tile.put_ml(ml[warp]);
            __syncthreads();
            // lane r: row r's largest exponent, what this warp's sums are multiplied by, the sum of the weights
            float m = -INFINITY, sum = 0.0f, mine = 0.0f;
            bool any = false;
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (!(ml[i][lane & 15].y < 0.0f)) { m = fmaxf(m, ml[i][lane & 15].x); any = true; }
            const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const bool has = !(ml[i][lane & 15].y < 0.0f);
                const float f = has ? ex2(ml[i][lane & 15].x - base) : 0.0f;
                if (has) sum += ml[i][lane & 15].y * f;
                if (i == warp) mine = f;
            }
            if (t < S::ROWS) joined[t] = make_float2(m, any ? sum : -1.0f);
            float* rows = reinterpret_cast<float*>(smem + stage * S::STAGE);
            const bool whole_part = whole_unit(p, w, begun, w.tile);
            const int64_t slot = w.unit + blockIdx.x;
#pragma unroll
            for (int pass = 0; pass < DP / S::COLS; pass++) {
                if (pass) __syncthreads();
                __syncwarp();
                tile.put_o(rows + warp * S::ROWS * S::COLS, mine, pass);
                __syncthreads();
                const int quads = min(S::COLS, D - pass * S::COLS) / 4;
                for (int e = t; e < used * quads; e += S::THREADS) {
                    const int x = e / quads, c = 4 * (e - x * quads), column = pass * S::COLS + c;
                    const float2 sums = joined[x];
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (!(sums.y < 0.0f)) {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const float4 a = *reinterpret_cast<const float4*>(rows + i * S::ROWS * S::COLS + sum8_at<S::COLS>(x, c));
                            v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
                        }
                    }
                    if (whole_part) {
                        const UnitRow r = unit_row(p, l, w, x);
                        if (!(sums.y < 0.0f)) { v.x /= sums.y; v.y /= sums.y; v.z /= sums.y; v.w /= sums.y; }
                        store_row(p, r, column, v);
                        if (column == 0 && p.lse) p.lse[r.row * p.q_heads + r.head] = sums.y < 0.0f ? -INFINITY : lse_of(sums.x, sums.y);
                    } else if (slot < l.slots) {
                        *reinterpret_cast<float4*>(part_at(l, D, slot, x, column)) = v;
                        if (column == 0) l.ml[slot * S::ROWS + x] = sums;
                    }
                }
            }
        }
        w.tile++;
        start = last;
    }
    copy_wait<0>();
    if (last_cta) grid_wait();
}

}  // namespace paged
}  // namespace lmrs
