// paged_attn.cuh -- attention of the rows of many sequences over their pages and over a prefix that all of them share.
//
// For one row: out = sum_j e^(s_j) v_j / sum_j e^(s_j) over the keys that it sees.  The keys are cut into parts that are worked on apart; a part leaves
// (m, l, o): the largest score, l = sum e^(s_j - m), o = sum e^(s_j - m) v_j, and parts are joined by rescaling to the largest m.  Scores are kept in
// powers of two (s log2 e).  What is cut, and how, is the same for all kernels here:
//   unit    16 (TILE_ROWS) rows of one KV head against one list of keys: the rows of one sequence, a row being a token and one of the query heads that share the
//           KV head, against the sequence's own tokens; or any rows of the call against the prefix, which is so read once for 16 rows, whoever they belong to
//   tile    TILE_KEYS keys of a unit
//   part    the tiles of a unit that one CTA takes.  All tiles of all units stand in one line, and CTA i of n takes those from T i / n to T (i + 1) / n,
//           whatever the sequences' lengths, which are read on the device: one long sequence spreads over the whole GPU, many short ones are packed.
// A unit that one CTA takes whole, with no prefix to join, is finished where it is computed; for the others join_kernel reads the parts from the workspace, in
// the order of their keys, so that a result depends on nothing but the call.
#pragma once
#include "paged.h"
#include "paged_rows.cuh"

namespace lmrs {
namespace paged {

PG_DEVINL uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
PG_DEVINL float ex2(float v) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
// 16 bytes to shared memory, zeros where there is nothing to copy.  (No memory clobber: commits and waits have it, and what computes the next address may move ahead)
PG_DEVINL void copy16(uint32_t to, const void* from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0));
}
PG_DEVINL void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> PG_DEVINL void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
PG_DEVINL void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
PG_DEVINL void grid_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

struct Plan {          // of sequence b, in the workspace: what stands before it in the line
    int64_t tiles;
    int64_t units;
};
template <typename T> struct AttnParams {
    Batch batch;
    Rows<const T> q;
    Rows<T> out;
    const T *k, *v;
    int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;
    int kv_heads, q_heads, head_size, group;   // group: query heads that share a KV head
    float scale2, softcap, cap_in;             // scores: scale2 = scale * log2 e; or softcap * log2 e * tanh(dot * cap_in), cap_in = scale / softcap
    float* lse;
    bool q_wide, out_wide;                     // rows on 16-byte boundaries
    int page_shift;                            // log2 of page_size, -1 if it is no power of two
    bool whole;                                // no prefix: a unit that one CTA takes is finished there
    int* err;                                  // mapped host word: set when a kernel gave up
};
// What one kernel goes through: units of the prefix (if it takes them), then those of the sequences (if it takes them)
struct Line {
    int tile_rows, tile_keys, ctas;            // (tile_rows and tile_keys: powers of two)
    int row_shift, key_shift;                  // their logarithms
    int seqs, front_tiles;                     // 0: not this kernel's; front_tiles: tiles of every unit of the prefix
    int64_t front_units;                       // kv_heads * tiles of rows
    // workspace
    Plan* plan;        // [seqs + 1]
    float2* ml;        // [slots][tile_rows]
    float* o;          // [slots][head_size / 8][tile_rows][8]: whole sectors for kernels whose threads hold rows, and for those whose lanes lie along them
    int64_t slots;     // part of unit u by CTA c: u + c (each step along the line goes on to another unit, another CTA or both)
};
PG_DEVINL float* part_at(const Line& l, int head_size, int64_t slot, int row, int c) { return l.o + ((slot * (head_size >> 3) + (c >> 3)) * l.tile_rows + row) * 8 + (c & 7); }

// (no more CTAs than tiles, so that each that takes part has some, and the parts of a unit are those of neighbours)
PG_DEVINL int64_t cta_begin(int64_t total, int ctas, int i) {
    const int64_t n = min((int64_t)ctas, total);
    if (i >= n) return total;
    const int64_t over = total * i;
    return over >> 32 ? over / n : (int64_t)((uint32_t)over / (uint32_t)n);   // (a 64-bit division takes a hundred instructions)
}
PG_DEVINL int cta_of(int64_t total, int ctas, int64_t tile) {
    const int64_t over = min((int64_t)ctas, total) * (tile + 1) + total - 1;
    return (over >> 32 ? (int)(over / total) : (int)((uint32_t)over / (uint32_t)total)) - 1;
}

// rows of a sequence's unit and the keys it goes through
// (a call's rows times the group stay below 2^31)
PG_DEVINL int unit_rows(const Span& s, int group, const Line& l) { return (s.count * group + l.tile_rows - 1) >> l.row_shift; }
template <typename T> PG_DEVINL int keys_upto(const AttnParams<T>& p, int64_t index) {   // keys of its own that a row of this index sees
    const int64_t most = (int64_t)p.batch.table_len * p.batch.page_size, n = index + 1;
    return n <= 0 ? 0 : (int)(n < most ? n : most);
}
template <typename T> PG_DEVINL int unit_keys(const AttnParams<T>& p, const Line& l, const Span& s, int tile) {
    const int rows = s.count * p.group, end = (tile + 1) << l.row_shift;
    return keys_upto(p, rows <= end ? (int64_t)s.len - 1 : (int64_t)s.len - s.count + (end - 1) / p.group);   // (of the last row)
}
template <typename T> PG_DEVINL int unit_tiles(const AttnParams<T>& p, const Line& l, const Span& s, int tile) { return (unit_keys(p, l, s, tile) + l.tile_keys - 1) >> l.key_shift; }
template <typename T> PG_DEVINL int64_t seq_tiles(const AttnParams<T>& p, const Line& l, const Span& s) {
    int64_t n = 0;
    for (int t = unit_rows(s, p.group, l) - 1; t >= 0; t--) n += unit_tiles(p, l, s, t);
    return n * p.kv_heads;
}

// Where a CTA is in the line
struct Walk {
    int64_t unit;              // number of the unit
    int b, head, row_tile;     // sequence (-1: the prefix), KV head, tile of rows
    int tile, tiles, keys;     // tile of keys, how many the unit has, its keys
    Span s;
};
template <typename T> PG_DEVINL void walk_unit(const AttnParams<T>& p, const Line& l, Walk& w) {   // fills in the keys of the unit that b, head and row_tile name
    w.keys = w.b < 0 ? p.batch.prefix_len : unit_keys(p, l, w.s, w.row_tile);
    w.tiles = (w.keys + l.tile_keys - 1) >> l.key_shift;
}
// the next unit that has tiles; KV heads lie innermost
template <typename T> PG_DEVINL void walk_next_unit(const AttnParams<T>& p, const Line& l, Walk& w) {
    do {
        w.unit++;
        if (++w.head == p.kv_heads) {
            w.head = 0;
            w.row_tile++;
            if (w.b < 0 ? w.unit >= l.front_units : w.row_tile >= unit_rows(w.s, p.group, l)) {
                w.row_tile = 0;
                do {
                    w.b++;
                    if (w.b >= l.seqs) { w.tiles = w.keys = 0; return; }   // the end of the line
                    w.s = span_of(p.batch, w.b);
                } while (w.s.count == 0);
            }
        }
        walk_unit(p, l, w);
    } while (w.tiles == 0);
    w.tile = 0;
}
// All threads: the whole line's length, and the CTA's place where it begins (`from` is that tile's number).  CTA 0 leaves the plan for join_kernel
template <typename T, int THREADS>
PG_DEVINL int64_t walk_begin(const AttnParams<T>& p, const Line& l, Walk& w, int64_t& from, int64_t& to) {
    __shared__ int64_t warp_tiles[THREADS / 32], warp_units[THREADS / 32], found[3];
    const int t = threadIdx.x, lane = t & 31, each = (l.seqs + THREADS - 1) / THREADS, b0 = min(l.seqs, t * each), b1 = min(l.seqs, b0 + each);
    int64_t tiles = 0, units = 0;
    for (int b = b0; b < b1; b++) {
        const Span s = span_of(p.batch, b);
        tiles += seq_tiles(p, l, s);
        units += (int64_t)unit_rows(s, p.group, l) * p.kv_heads;
    }
    int64_t tiles_to = tiles, units_to = units;   // up to and with this thread's
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t a = __shfl_up_sync(~0u, tiles_to, o), c = __shfl_up_sync(~0u, units_to, o);
        if (lane >= o) { tiles_to += a; units_to += c; }
    }
    if (lane == 31) { warp_tiles[t >> 5] = tiles_to; warp_units[t >> 5] = units_to; }
    if (t == 0) found[0] = found[1] = found[2] = 0;
    __syncthreads();
    const int64_t front = l.front_units * l.front_tiles;
    int64_t total = front;
    tiles_to += front;
    units_to += l.front_units;
    for (int i = 0; i < THREADS / 32; i++) {
        if (i < t >> 5) { tiles_to += warp_tiles[i]; units_to += warp_units[i]; }
        total += warp_tiles[i];
    }
    from = cta_begin(total, l.ctas, blockIdx.x);
    to = cta_begin(total, l.ctas, blockIdx.x + 1);
    if (blockIdx.x == 0) {
        int64_t at = tiles_to - tiles, u = units_to - units;
        for (int b = b0; b < b1; b++) {
            const Span s = span_of(p.batch, b);
            l.plan[b] = Plan{at, u};
            at += seq_tiles(p, l, s);
            u += (int64_t)unit_rows(s, p.group, l) * p.kv_heads;
        }
        if (t == 0) l.plan[l.seqs] = Plan{total, 0};
    }
    if (from >= front && from < to && tiles_to - tiles <= from && from < tiles_to) {   // one thread's sequences hold it
        int64_t at = tiles_to - tiles, u = units_to - units;
        for (int b = b0; b < b1; b++) {
            const Span s = span_of(p.batch, b);
            const int64_t n = seq_tiles(p, l, s);
            if (from < at + n) {
                found[0] = b;
                found[1] = at;
                found[2] = u;
                break;
            }
            at += n;
            u += (int64_t)unit_rows(s, p.group, l) * p.kv_heads;
        }
    }
    __syncthreads();
    if (from >= to) return total;
    if (from < front) {
        w.unit = from / l.front_tiles;
        w.b = -1;
        w.row_tile = (int)(w.unit / p.kv_heads);
        w.head = (int)(w.unit - (int64_t)w.row_tile * p.kv_heads);
        w.tile = (int)(from - w.unit * l.front_tiles);
    } else {
        w.b = (int)found[0];
        w.s = span_of(p.batch, w.b);
        int64_t left = from - found[1];
        int n = unit_tiles(p, l, w.s, 0);
        w.row_tile = 0;
        for (const int rows = unit_rows(w.s, p.group, l); w.row_tile + 1 < rows && left >= (int64_t)n * p.kv_heads; n = unit_tiles(p, l, w.s, ++w.row_tile)) left -= (int64_t)n * p.kv_heads;
        n = max(n, 1);   // (it is; lengths that change under the kernel may make it otherwise)
        w.head = min((int)(left / n), p.kv_heads - 1);
        w.tile = (int)(left - (int64_t)w.head * n);
        w.unit = found[2] + (int64_t)w.row_tile * p.kv_heads + w.head;
    }
    walk_unit(p, l, w);
    return total;
}

// What row `x` of a unit is: its row of the call's arrays (-1: none), its query head, and how many of the unit's keys it sees
struct UnitRow { int64_t row; int head, keys; };
template <typename T> PG_DEVINL UnitRow unit_row(const AttnParams<T>& p, const Line& l, const Walk& w, int x) {
    const int i = w.row_tile * l.tile_rows + x, token = i / p.group;
    UnitRow r = {-1, w.head * p.group + (i - token * p.group), w.keys};   // (rows that are not there see all, so that they need no mask)
    if (w.b < 0) {
        if (token < p.batch.n_rows) r.row = token;
    } else if (token < w.s.count) {
        r.row = w.s.first + token;
        r.keys = min(w.keys, keys_upto(p, (int64_t)w.s.len - w.s.count + token));
    }
    return r;
}
// where key x of a unit lies: page (-1: nowhere) and place in it
struct Place { int page, place; };
template <typename T> PG_DEVINL Place unit_place(const AttnParams<T>& p, const Walk& w, int x) {
    Place r = {-1, 0};
    if (x < w.keys) {   // (so the table reaches it)
        const int i = p.page_shift >= 0 ? x >> p.page_shift : x / p.batch.page_size, page = (w.b < 0 ? p.batch.prefix : p.batch.tables + w.b * p.batch.table_stride)[i];
        r.page = page < 0 || page >= p.batch.pages ? -1 : page;
        r.place = x - i * p.batch.page_size;
    }
    return r;
}
// A dot product as a score, in powers of two.  With a cap c: c tanh(x), x = dot scale / c.  What a weight is off by goes with the score's absolute error: from |x| = 1/2 on
// 1 - 2 / (e^2x + 1) (two units of the last place of 1), below it the Taylor series up to x^13 (its next term is 4.4e-8 at 1/2), which leaves the special-function units alone.
PG_DEVINL float tanh_far(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(ex2(x * (2.0f * LOG2E)) + 1.0f));   // (of infinity: 0)
    return fmaf(-2.0f, r, 1.0f);
}
PG_DEVINL float tanh_near(float x) {
    const float y = x * x;
    float s = fmaf(y, 21844.0f / 6081075.0f, -1382.0f / 155925.0f);
    s = fmaf(y, s, 62.0f / 2835.0f);
    s = fmaf(y, s, -17.0f / 315.0f);
    s = fmaf(y, s, 2.0f / 15.0f);
    s = fmaf(y, s, -1.0f / 3.0f);
    return fmaf(y * s, x, x);
}
template <typename T> PG_DEVINL float score2(const AttnParams<T>& p, float dot) {
    if (!(p.softcap > 0.0f)) return dot * p.scale2;
    const float x = dot * p.cap_in;
    return p.softcap * LOG2E * (fabsf(x) <= 0.5f ? tanh_near(x) : tanh_far(x));
}
// N dots of a lane, capped (all lanes of the warp: the near form where it serves all of them)
template <typename T, int N> PG_DEVINL void cap_scores(const AttnParams<T>& p, float (&s)[N]) {
    const float cap2 = p.softcap * LOG2E;
    float far = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        s[i] *= p.cap_in;
        far = fmaxf(far, fabsf(s[i]));
    }
    if (__all_sync(~0u, far <= 0.5f)) {   // (NaN comes out as NaN either way)
#pragma unroll
        for (int i = 0; i < N; i++) s[i] = cap2 * tanh_near(s[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) s[i] = cap2 * (fabsf(s[i]) <= 0.5f ? tanh_near(s[i]) : tanh_far(s[i]));
    }
}

template <typename T> PG_DEVINL void store_row(const AttnParams<T>& p, const UnitRow& r, int e, float4 v) {   // 4 elements of a result
    T* to = p.out.data + r.row * p.out.row + r.head * p.out.head + e;
    if (p.out_wide) {
        Piece<T, 4> x;
        x.v[0] = from_f<T>(v.x); x.v[1] = from_f<T>(v.y); x.v[2] = from_f<T>(v.z); x.v[3] = from_f<T>(v.w);
        *reinterpret_cast<Piece<T, 4>*>(to) = x;
    } else {
        to[0] = from_f<T>(v.x); to[1] = from_f<T>(v.y); to[2] = from_f<T>(v.z); to[3] = from_f<T>(v.w);
    }
}

// A row of a unit once more, keys `from` to `to` - 1 of the unit, by 128 threads that share a named barrier: only keys that the row sees are touched.  In the matrix products a
// value that is not finite spoils, through its weight 0, also the rows of the tile that do not see it.  acc[i]: column threadIdx.x % 128 + 128 i, unnormalised.
// Rows that come out finite never come here.
constexpr int AGAIN = 128;
struct AgainScratch { float weight[AGAIN], most[AGAIN / 32]; int64_t at[AGAIN]; };
PG_DEVINL void again_sync(int barrier) { __syncwarp(); asm volatile("bar.sync %0, %1;" ::"r"(barrier), "n"(AGAIN) : "memory"); }
template <typename T>
static __device__ __noinline__ void row_again(const AttnParams<T>& p, const Walk& w, const UnitRow& r, int from, int to, AgainScratch& sc, int barrier, float& m, float& l, float (&acc)[2]) {
    const int t = threadIdx.x & (AGAIN - 1), D = p.head_size;
    const T* q = p.q.data + r.row * p.q.row + r.head * p.q.head;
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; i++) acc[i] = 0.0f;
    to = min(to, r.keys);
    for (int x0 = from; x0 < to; x0 += AGAIN) {
        Place at_x = {-1, 0};
        if (x0 + t < to) at_x = unit_place(p, w, x0 + t);
        const bool there = at_x.page >= 0;
        float a = -INFINITY;
        if (there) {
            const T* k = p.k + at_x.page * p.k_page + at_x.place * p.k_slot + w.head * p.k_head;
            a = 0.0f;
            for (int e = 0; e < D; e++) a = fmaf(to_f(q[e]), to_f(k[e]), a);
            a = score2(p, a);
        }
        float top = a;
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
        again_sync(barrier);
        sc.at[t] = there ? at_x.page * p.v_page + at_x.place * p.v_slot + w.head * p.v_head : -1;
        if ((t & 31) == 0) sc.most[t >> 5] = top;
        again_sync(barrier);
        float now = m;
        for (int i = 0; i < AGAIN / 32; i++) now = fmaxf(now, sc.most[i]);
        const float base = now == -INFINITY ? 0.0f : now, corr = ex2(m - base);
        sc.weight[t] = there ? ex2(a - base) : 0.0f;
        m = now;
        again_sync(barrier);
        l *= corr;
        for (int i = 0; i < AGAIN; i++) l += sc.weight[i];
#pragma unroll
        for (int c = 0; c < 2; c++)
            if (t + c * AGAIN < D) {
                acc[c] *= corr;
                for (int i = 0; i < AGAIN; i++)
                    if (sc.at[i] >= 0) acc[c] = fmaf(sc.weight[i], to_f(p.v[sc.at[i] + t + c * AGAIN]), acc[c]);
            }
    }
    again_sync(barrier);
}

// A part's row leaves as (m, l) and o in the workspace, or as a result.  l = -1: the part holds no key that the row sees
PG_DEVINL float lse_of(float m, float l) { return ((m == -INFINITY ? 0.0f : m) + log2f(l)) * LN2; }
template <typename T> PG_DEVINL bool whole_unit(const AttnParams<T>& p, const Walk& w, int first, int last) { return w.b >= 0 && p.whole && first == 0 && last == w.tiles - 1; }

// ---- 16 rows a unit ------------------------------------------------------------------------------------------------------------------------
// CTA = 4 warps that share a tile's keys, each with the running (m, l, o) of all 16 rows over its keys; they meet when a part ends.  What bounds it is the
// bytes of the pages.  Copies to shared memory (16 bytes a thread, zeros for keys that are not there) run STAGES - 1 tiles ahead of the products, on into
// the units that follow, with the places of the keys one tile further ahead; rows are 16-byte pieces rotated by the row's number, which keeps all reads
// free of bank conflicts.  A page may end anywhere in a tile.
// Measured (B200, 32/8 heads): 4 sequences of 60000 keys, fp16, heads of 128: 125 us, 5300 GB/s of 6450 that a copy reaches; 128 sequences of up to 600 keys, bf16, heads of 128: 58 us, 5.4 TB/s; one of
// 1000 keys, heads of 64: 10 us with the join (launches and the chain length - table - keys).  float32, 15 sequences behind a prefix of 4096, heads of 64: 57 us; multiply-adds
// fed from shared memory bound that.  Four more warps for the copies: 127 / 138 us for the first, 58 / 61 for the last; taken back.
template <typename T, int DP> struct TileShape {
    static constexpr int ROWS = 16, THREADS = 128, ROW = DP * (int)sizeof(T), PIECES = ROW / 16, KEYS = sizeof(T) == 4 && DP > 64 ? 32 : 64, STAGES = sizeof(T) == 4 ? 2 : 3;
    static constexpr int WARP_KEYS = KEYS / 4, COPY_KEYS = KEYS / 32;   // keys a warp works on; keys a thread copies a quarter of
    static constexpr int KV = KEYS * ROW, Q = ROWS * ROW, SMEM = STAGES * (2 * KV + Q);   // (queries: one set for each unit that copies can have got to)
    static constexpr int CTAS = ROW <= 128 ? 3 : ROW <= (sizeof(T) == 4 ? 512 : 256) ? 2 : 1;
    static_assert(4 * ROWS * DP * 4 <= 2 * KV, "the four warps' rows fit where a tile's keys and values were");
};
PG_DEVINL uint32_t piece_at(int row, int piece, int row_bytes) { return (uint32_t)(row * row_bytes + ((piece ^ (row & 7)) << 4)); }

// where the warps' sums meet: float c of row r, rotated so that the rows that a store touches lie in different banks
template <int DP> PG_DEVINL int sum_at(int r, int c) { return r * DP + (c ^ ((r & 3) << 3)); }

PG_DEVINL void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
PG_DEVINL void ldmatrix4t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
PG_DEVINL void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
PG_DEVINL void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Weights are rounded to the type of the values for the products, since the tensor cores take one type for both: each by half a step at most, 2^-8 of it in bf16 and 2^-11 in fp16, either way, so
// that a result is off by that fraction of its weighted sizes where all of them go one way (measured against 64 bits: 0.0023 of a bf16 result, where rounding the result alone makes 0.0017). The sums that
// they are divided by are of the unrounded ones. Here weights are at most 1; rows128_kernel, whose m may lag by RESCALE_AT, has up to 2^8. float16 keeps fewer small numbers: its weights are 2^7 times
// as large (m is 7 less; up to 2^7 here, 2^15 there), so that what a weight loses below 2^-14 is 2^-32 of the largest at most.
template <typename T> constexpr float WEIGHT_SHIFT = 0.0f;
template <> constexpr float WEIGHT_SHIFT<__half> = 7.0f;

// the products of one warp, 16-bit types: mma.sync, 16 rows x 16 keys at a time
template <typename T, int DP> struct WarpTile {
    using S = TileShape<T, DP>;
    uint32_t q[DP / 16][4];
    float o[DP / 8][4], m[2], l[2];   // rows lane / 4 and lane / 4 + 8
    bool seen[2];
    PG_DEVINL void begin(uint32_t q_at) {
        const int lane = threadIdx.x & 31;
        __syncwarp();
#pragma unroll
        for (int k = 0; k < DP / 16; k++) ldmatrix4(q[k], q_at + piece_at(lane & 15, 2 * k + (lane >> 4), S::ROW));
#pragma unroll
        for (int n = 0; n < DP / 8; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.0f;
        seen[0] = seen[1] = false;
    }
    // there: bit j: key j of the warp's is there; first: number of its first key; row_keys: how many keys each row sees
    PG_DEVINL void tile(const AttnParams<T>& p, uint32_t, uint32_t k_at, uint32_t v_at, uint32_t there, int first, const int* row_keys, int, float*) {
        const int lane = threadIdx.x & 31, key0 = 16 * (threadIdx.x >> 5);
        float s[2][4] = {};
        __syncwarp();   // (ldmatrix and mma are for a warp in step)
        const uint32_t k_row = k_at + (uint32_t)(key0 + (lane & 7) + ((lane >> 4) << 3)) * S::ROW, k_turn = (uint32_t)(((lane >> 3) & 1) ^ (lane & 7)) << 4;
#pragma unroll
        for (int k = 0; k < DP / 16; k++) {
            uint32_t b[4];
            ldmatrix4(b, k_row + (k_turn ^ (32 * k)));   // (piece 2k or 2k + 1, rotated by the row)
            mma16816(s[0], q[k], b[0], b[1], T());
            mma16816(s[1], q[k], b[2], b[3], T());
        }
        if (p.softcap > 0.0f) {
            float flat[8];
#pragma unroll
            for (int i = 0; i < 8; i++) flat[i] = s[i >> 2][i & 3];
            cap_scores(p, flat);
#pragma unroll
            for (int i = 0; i < 8; i++) s[i >> 2][i & 3] = flat[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) s[i >> 2][i & 3] *= p.scale2;
        }
        const int limit[2] = {row_keys[lane / 4] - first, row_keys[lane / 4 + 8] - first};
        if (!__all_sync(~0u, there == 0xffffu && limit[0] >= 16 && limit[1] >= 16)) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const uint32_t sees = there & (limit[i] >= 16 ? 0xffffu : limit[i] <= 0 ? 0u : (1u << limit[i]) - 1);
                seen[i] = seen[i] || sees;
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int c = 0; c < 2; c++)
                        if (!(sees >> (8 * h + 2 * (lane & 3) + c) & 1)) s[h][2 * i + c] = -INFINITY;
            }
        } else {
            seen[0] = seen[1] = true;
        }
        float now[2];
#pragma unroll
        for (int i = 0; i < 2; i++) now[i] = fmaxf(fmaxf(s[0][2 * i], s[0][2 * i + 1]), fmaxf(s[1][2 * i], s[1][2 * i + 1]));
#pragma unroll
        for (int d = 1; d < 4; d *= 2)
#pragma unroll
            for (int i = 0; i < 2; i++) now[i] = fmaxf(now[i], __shfl_xor_sync(~0u, now[i], d));
        const bool grows = now[0] - WEIGHT_SHIFT<T> > m[0] || now[1] - WEIGHT_SHIFT<T> > m[1];
        if (__any_sync(~0u, grows)) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float top = fmaxf(m[i], now[i] - WEIGHT_SHIFT<T>), corr = ex2(m[i] - (top == -INFINITY ? 0.0f : top));
                m[i] = top;
                l[i] *= corr;
#pragma unroll
                for (int n = 0; n < DP / 8; n++) { o[n][2 * i] *= corr; o[n][2 * i + 1] *= corr; }
            }
        }
        uint32_t a[4];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float base = m[i] == -INFINITY ? 0.0f : m[i];
            float w[4];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                w[2 * h] = ex2(s[h][2 * i] - base);
                w[2 * h + 1] = ex2(s[h][2 * i + 1] - base);
                a[2 * h + i] = close_word(make_float2(w[2 * h], w[2 * h + 1]), T());
            }
            l[i] += (w[0] + w[1]) + (w[2] + w[3]);   // (of this lane's keys: the four lanes of a row meet at the end)
        }
        const uint32_t v_row = v_at + (uint32_t)(key0 + (lane & 15)) * S::ROW, v_turn = (uint32_t)((lane >> 4) ^ (lane & 7)) << 4;
#pragma unroll
        for (int n = 0; n < DP / 16; n++) {
            uint32_t b[4];
            ldmatrix4t(b, v_row + (v_turn ^ (32 * n)));
            mma16816(o[2 * n], a, b[0], b[1], T());
            mma16816(o[2 * n + 1], a, b[2], b[3], T());
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
    PG_DEVINL void put_o(float* to, float factor) {   // [16][DP] as sum_at has them, times the rows' factors (lane r has row r's)
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int r = lane / 4 + 8 * i;
            const float f = __shfl_sync(~0u, factor, r);
#pragma unroll
            for (int n = 0; n < DP / 8; n++) *reinterpret_cast<float2*>(to + sum_at<DP>(r, 8 * n + 2 * (lane & 3))) = make_float2(o[n][2 * i] * f, o[n][2 * i + 1] * f);
        }
    }
};

// the same in float32: multiply-adds.  Scores: a lane takes one of the warp's keys and some of the rows; values: all rows, DP / 32 columns.  Rows that the unit
// does not have (it has `used`) cost nothing.
template <int DP> struct WarpTile<float, DP> {
    using S = TileShape<float, DP>;
    static constexpr int KEYS = S::WARP_KEYS, TEAMS = 32 / KEYS, SHARE = 16 / TEAMS, COLS = DP / 32;   // lanes KEYS * i .. are team i: rows i, i + TEAMS, ...
    float o[16][COLS], m[SHARE], l[SHARE];
    bool seen[SHARE];
    PG_DEVINL void begin(uint32_t) {
#pragma unroll
        for (int r = 0; r < 16; r++)
#pragma unroll
            for (int c = 0; c < COLS; c++) o[r][c] = 0.0f;
#pragma unroll
        for (int i = 0; i < SHARE; i++) { m[i] = -INFINITY; l[i] = 0.0f; seen[i] = false; }
    }
    PG_DEVINL static float4 load4(uint32_t at) {
        float4 v;
        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at));
        return v;
    }
    PG_DEVINL static float2 load2(uint32_t at) {
        float2 v;
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at));
        return v;
    }
    // scratch: the warp's own [KEYS + 1][16] floats: weights, and what the rows' sums are rescaled by
    PG_DEVINL void tile(const AttnParams<float>& p, uint32_t q_at, uint32_t k_at, uint32_t v_at, uint32_t there, int first, const int* row_keys, int used, float* scratch) {
        if (used <= 4) rows<4>(p, q_at, k_at, v_at, there, first, row_keys, scratch);
        else if (used <= 8) rows<8>(p, q_at, k_at, v_at, there, first, row_keys, scratch);
        else rows<16>(p, q_at, k_at, v_at, there, first, row_keys, scratch);
    }
    template <int ROWS> PG_DEVINL void rows(const AttnParams<float>& p, uint32_t q_at, uint32_t k_at, uint32_t v_at, uint32_t there, int first, const int* row_keys, float* scratch) {
        constexpr int MINE = ROWS / TEAMS;
        const int lane = threadIdx.x & 31, key0 = KEYS * (threadIdx.x >> 5), key = lane % KEYS, team = lane / KEYS;
        float s[MINE] = {};
        const uint32_t k_row = k_at + (key0 + key) * S::ROW, k_turn = (uint32_t)(key & 7) << 4;
#pragma unroll
        for (int c = 0; c < DP / 4; c++) {   // (past the end of a head there are zeros)
            const float4 k = load4(k_row + (k_turn ^ (16 * c)));
#pragma unroll
            for (int i = 0; i < MINE; i++) {
                const float4 q = load4(q_at + piece_at(i * TEAMS + team, c, S::ROW));
                s[i] = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, fmaf(q.w, k.w, s[i]))));
            }
        }
        __syncwarp();   // (the weights of the tile before have been read)
        float now[MINE];
        bool sees[MINE];
#pragma unroll
        for (int i = 0; i < MINE; i++) {
            sees[i] = (there >> key & 1) && first + key < row_keys[i * TEAMS + team];
            s[i] = now[i] = sees[i] ? score2(p, s[i]) : -INFINITY;
        }
#pragma unroll
        for (int d = KEYS / 2; d; d >>= 1)
#pragma unroll
            for (int i = 0; i < MINE; i++) now[i] = fmaxf(now[i], __shfl_xor_sync(~0u, now[i], d));
        bool grows = false;
#pragma unroll
        for (int i = 0; i < MINE; i++) grows = grows || now[i] > m[i];
        const bool rescale = __any_sync(~0u, grows);
#pragma unroll
        for (int i = 0; i < MINE; i++) {
            const float top = fmaxf(m[i], now[i]), base = top == -INFINITY ? 0.0f : top, corr = ex2(m[i] - base), w = ex2(s[i] - base);
            if (rescale) {
                m[i] = top;
                l[i] *= corr;
                if (key == 0) scratch[KEYS * 16 + i * TEAMS + team] = corr;
            }
            l[i] += w;   // (this lane's keys)
            seen[i] = seen[i] || sees[i];
            scratch[key * 16 + i * TEAMS + team] = w;
        }
        __syncwarp();
        if (rescale) {
#pragma unroll
            for (int r = 0; r < ROWS; r++) {
                const float corr = scratch[KEYS * 16 + r];
#pragma unroll
                for (int c = 0; c < COLS; c++) o[r][c] *= corr;
            }
        }
        const uint32_t v_row = v_at + key0 * S::ROW;
#pragma unroll
        for (int j = 0; j < KEYS; j++) {
            float v[COLS];
            if constexpr (COLS == 2) {
                const float2 x = load2(v_row + piece_at(j, lane >> 1, S::ROW) + 8 * (lane & 1));
                v[0] = x.x; v[1] = x.y;
            } else {
#pragma unroll
                for (int c = 0; c < COLS; c += 4) {
                    const float4 x = load4(v_row + piece_at(j, lane + 8 * c, S::ROW));
                    v[c] = x.x; v[c + 1] = x.y; v[c + 2] = x.z; v[c + 3] = x.w;
                }
            }
#pragma unroll
            for (int r = 0; r < ROWS; r += 4) {
                const float4 w = *reinterpret_cast<const float4*>(scratch + j * 16 + r);
#pragma unroll
                for (int c = 0; c < COLS; c++) {
                    o[r][c] = fmaf(w.x, v[c], o[r][c]);
                    o[r + 1][c] = fmaf(w.y, v[c], o[r + 1][c]);
                    o[r + 2][c] = fmaf(w.z, v[c], o[r + 2][c]);
                    o[r + 3][c] = fmaf(w.w, v[c], o[r + 3][c]);
                }
            }
        }
    }
    PG_DEVINL void put_ml(float2* ml) {
        const int lane = threadIdx.x & 31, team = lane / KEYS;
#pragma unroll
        for (int i = 0; i < SHARE; i++) {
            const unsigned any = __ballot_sync(~0u, seen[i]);
#pragma unroll
            for (int d = KEYS / 2; d; d >>= 1) l[i] += __shfl_xor_sync(~0u, l[i], d);
            if (lane % KEYS == 0) ml[i * TEAMS + team] = make_float2(m[i], any >> (KEYS * team) & (KEYS == 16 ? 0xffffu : 0xffu) ? l[i] : -1.0f);
        }
    }
    PG_DEVINL void put_o(float* to, float factor) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int r = 0; r < 16; r++) {
            const float f = __shfl_sync(~0u, factor, r);
            if constexpr (COLS == 2) {
                *reinterpret_cast<float2*>(to + sum_at<DP>(r, 2 * lane)) = make_float2(o[r][0] * f, o[r][1] * f);
            } else {
#pragma unroll
                for (int c = 0; c < COLS; c += 4)
                    *reinterpret_cast<float4*>(to + sum_at<DP>(r, 4 * lane + 32 * c)) = make_float4(o[r][c] * f, o[r][c + 1] * f, o[r][c + 2] * f, o[r][c + 3] * f);
            }
        }
    }
};

template <typename T, int DP>
__global__ void __launch_bounds__(TileShape<T, DP>::THREADS, TileShape<T, DP>::CTAS) rows16_kernel(const __grid_constant__ AttnParams<T> p, const __grid_constant__ Line l) {
    using S = TileShape<T, DP>;
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ Walk walks[S::STAGES];             // of the units that copies have got to, by their number in this CTA modulo STAGES
    __shared__ int row_keys[S::STAGES][S::ROWS];
    __shared__ __align__(8) uint8_t there[S::STAGES][S::KEYS / 8];
    __shared__ float2 ml[4][S::ROWS];
    __shared__ float2 joined[S::ROWS];
    __shared__ __align__(16) float weights[sizeof(T) == 4 ? 4 : 1][sizeof(T) == 4 ? (S::WARP_KEYS + 1) * 16 : 1];
    __shared__ unsigned again;
    __shared__ AgainScratch scratch;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, D = p.head_size;
    const uint32_t kv = smem_at(smem), queries = kv + S::STAGES * 2 * S::KV;

    Walk ahead;   // where copies are
    int64_t from, to;
    walk_begin<T, S::THREADS>(p, l, ahead, from, to);
    grid_launch();
    // The kernel before may still run.  The last CTA ends after it, so that whoever waits for this kernel waits for both; the others leave their SM to the next ones
    const bool last_cta = blockIdx.x == gridDim.x - 1;
    if (from >= to) { if (last_cta) grid_wait(); return; }

    // copies of a thread: keys t / 4 (and t / 4 + 32) of the tile, every fourth 16 bytes; past the end of a head zeros, so that the products need not know where it is
    Place place[S::COPY_KEYS];
    const int n_tiles = (int)(to - from), whole = D * (int)sizeof(T) / 16;
    int copied = 0, stage_to = 0, set_to = 0;   // tiles copied, the stage and the unit's set that the next goes to
    bool first = true;
    auto look = [&]() {
#pragma unroll
        for (int i = 0; i < S::COPY_KEYS; i++) place[i] = unit_place(p, ahead, ahead.tile * S::KEYS + t / 4 + 32 * i);
    };
    auto copy_tile = [&]() {   // the tile that `ahead` stands at, whose places are known; then on to the next one
        if (copied < n_tiles) {
            const uint32_t k_at = kv + stage_to * 2 * S::KV + (t / 4) * S::ROW, turn = (uint32_t)((t & 3) ^ (t / 4 & 7)) << 4;
#pragma unroll
            for (int i = 0; i < S::COPY_KEYS; i++) {
                const bool is = place[i].page >= 0;
                const int page = is ? place[i].page : 0;
                const char* k = reinterpret_cast<const char*>(p.k + page * p.k_page + place[i].place * p.k_slot + ahead.head * p.k_head) + 16 * (t & 3);
                const char* v = reinterpret_cast<const char*>(p.v + page * p.v_page + place[i].place * p.v_slot + ahead.head * p.v_head) + 16 * (t & 3);
                if (whole == S::PIECES) {
#pragma unroll
                    for (int c = 0; c < S::PIECES; c += 4) {
                        copy16(k_at + 32 * i * S::ROW + (turn ^ (16 * c)), k + 16 * c, is);
                        copy16(k_at + S::KV + 32 * i * S::ROW + (turn ^ (16 * c)), v + 16 * c, is);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < S::PIECES; c += 4) {
                        const bool in = is && c + (t & 3) < whole;
                        copy16(k_at + 32 * i * S::ROW + (turn ^ (16 * c)), in ? k + 16 * c : reinterpret_cast<const char*>(p.k), in);
                        copy16(k_at + S::KV + 32 * i * S::ROW + (turn ^ (16 * c)), in ? v + 16 * c : reinterpret_cast<const char*>(p.v), in);
                    }
                }
                const unsigned bits = __ballot_sync(~0u, __shfl_sync(~0u, is, (4 * lane) & 31)) & 0xff;
                if (lane == 0) there[stage_to][warp + 4 * i] = (uint8_t)bits;
            }
            if (first) {
                if (t == 0) walks[set_to] = ahead;
                if (t < S::ROWS) row_keys[set_to][t] = unit_row(p, l, ahead, t).keys;
                const uint32_t q_at = queries + set_to * S::Q;
                for (int e = t; e < S::ROWS * S::PIECES; e += S::THREADS) {
                    const int x = e / S::PIECES, c = e % S::PIECES;
                    const UnitRow r = unit_row(p, l, ahead, x);
                    const bool in = r.row >= 0 && c < whole;
                    const T* q = in ? p.q.data + r.row * p.q.row + r.head * p.q.head + c * (16 / sizeof(T)) : p.q.data;
                    const uint32_t at = q_at + piece_at(x, c, S::ROW);
                    if (p.q_wide) {
                        copy16(at, q, in);
                    } else {
                        Piece<T, 16 / sizeof(T)> v;
#pragma unroll
                        for (int i = 0; i < 16 / (int)sizeof(T); i++) v.v[i] = in ? q[i] : from_f<T>(0.0f);
                        *reinterpret_cast<Piece<T, 16 / sizeof(T)>*>(smem + (at - kv)) = v;
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

    WarpTile<T, DP> tile;
    Walk w;
    int set = S::STAGES - 1, stage = S::STAGES - 1, begun = 0, used = 0;
    bool start = true;
#pragma unroll 1
    for (int at = 0; at < n_tiles; at++) {
        copy_wait<S::STAGES - 2>();
        __syncthreads();   // the tile has landed for all threads, and the one before has been worked on by all
        copy_tile();
        stage = stage + 1 == S::STAGES ? 0 : stage + 1;
        const uint32_t k_at = kv + stage * 2 * S::KV, v_at = k_at + S::KV;
        if (start) {
            set = set + 1 == S::STAGES ? 0 : set + 1;
            w = walks[set];
            begun = w.tile;
            tile.begin(queries + set * S::Q);
            used = w.b < 0 ? (int)min((int64_t)S::ROWS, p.batch.n_rows * p.group - (int64_t)w.row_tile * S::ROWS) : min(S::ROWS, w.s.count * p.group - w.row_tile * S::ROWS);
            start = false;
        }
        const uint32_t bits = S::WARP_KEYS == 16 ? *reinterpret_cast<const uint16_t*>(&there[stage][2 * warp]) : there[stage][warp];
        tile.tile(p, queries + set * S::Q, k_at, v_at, bits, w.tile * S::KEYS + warp * S::WARP_KEYS, row_keys[set], used, weights[sizeof(T) == 4 ? warp : 0]);
        const bool last = w.tile + 1 == w.tiles;
        if (last || at + 1 == n_tiles) {   // the part ends: the warps' rows meet in the tile's place
            const bool mixed = w.b >= 0 && w.s.count > 1;   // (rows that see different keys)
            tile.put_ml(ml[warp]);
            if (t == 0) again = 0;
            __syncthreads();
            {   // lane r: row r's largest score, what this warp's sums are multiplied by, the sum of the weights
                float m = -INFINITY, sum = 0.0f, mine = 0.0f;
                bool any = false;
                const int r = lane & 15;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (!(ml[i][r].y < 0.0f)) { m = fmaxf(m, ml[i][r].x); any = true; }
                const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const bool has = !(ml[i][r].y < 0.0f);
                    const float f = has ? ex2(ml[i][r].x - base) : 0.0f;
                    if (has) sum += ml[i][r].y * f;
                    if (i == warp) mine = f;
                }
                if (t < S::ROWS) joined[t] = make_float2(m, any ? sum : -1.0f);
                __syncwarp();
                tile.put_o(reinterpret_cast<float*>(smem + stage * 2 * S::KV) + warp * S::ROWS * DP, mine);
            }
            __syncthreads();
            float* rows = reinterpret_cast<float*>(smem + stage * 2 * S::KV);
            const bool whole = whole_unit(p, w, begun, w.tile);
            const int64_t slot = w.unit + blockIdx.x;
            const int quads = D / 4;
            for (int e = t; e < used * quads; e += S::THREADS) {
                const int x = e / quads, c = 4 * (e - x * quads);
                const float2 s = joined[x];
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (!(s.y < 0.0f)) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float4 a = *reinterpret_cast<const float4*>(rows + sum_at<DP>(i * S::ROWS + x, c));
                        v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
                    }
                }
                if (mixed && !isfinite(v.x + v.y + v.z + v.w)) atomicOr(&again, 1u << x);
                if (whole) {
                    const UnitRow r = unit_row(p, l, w, x);
                    if (!(s.y < 0.0f)) { v.x /= s.y; v.y /= s.y; v.z /= s.y; v.w /= s.y; }
                    store_row(p, r, c, v);
                    if (c == 0 && p.lse) p.lse[r.row * p.q_heads + r.head] = s.y < 0.0f ? -INFINITY : lse_of(s.x, s.y);
                } else if (slot < l.slots) {
                    *reinterpret_cast<float4*>(part_at(l, D, slot, x, c)) = v;
                    if (c == 0) l.ml[slot * S::ROWS + x] = s;
                }
            }
            if (mixed) __syncthreads();
            for (unsigned left = mixed ? again : 0; left; left &= left - 1) {   // (the same for all threads)
                const int x = __ffs(left) - 1;
                const UnitRow r = unit_row(p, l, w, x);
                if (joined[x].y < 0.0f) continue;
                float m, sum, acc[2];
                row_again(p, w, r, begun * S::KEYS, (w.tile + 1) * S::KEYS, scratch, 0, m, sum, acc);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int c = t + AGAIN * i;
                    if (c >= D) continue;
                    if (whole) p.out.data[r.row * p.out.row + r.head * p.out.head + c] = from_f<T>(acc[i] / sum);
                    else if (slot < l.slots) *part_at(l, D, slot, x, c) = acc[i];
                }
                if (t == 0) {
                    if (whole) { if (p.lse) p.lse[r.row * p.q_heads + r.head] = lse_of(m, sum); }
                    else if (slot < l.slots) l.ml[slot * S::ROWS + x] = make_float2(m, sum);
                }
            }
        }
        w.tile++;
        start = last;
    }
    copy_wait<0>();
    if (last_cta) grid_wait();
}

// ---- joining parts ---------------------------------------------------------------------------------------------------------------------------
// WARPS warps a row and head, their lanes its columns in fours: they take parts in turn, each with a running (m, l, o), and they meet in shared memory.  8 where
// rows are few and may have many parts, 1 otherwise (then a CTA has 8 rows or heads).  A chain of dependent reads (sequence, plan, (m, l), columns) bounds it: 11 us
// for 128 rows of 32 heads of 128 with 10 parts each (B200), 43 for 1600 rows of 16 heads of 256.
template <typename T, int WARPS, int COLS>   // COLS: 128 columns each
__global__ void __launch_bounds__(256, COLS == 1 ? 4 : 3) join_kernel(const __grid_constant__ AttnParams<T> p, const __grid_constant__ Line lf, const __grid_constant__ Line lo) {
    constexpr int ITEMS = 8 / WARPS, EACH = WARPS == 1 ? 32 : 4;   // parts a warp takes at a time
    __shared__ float2 ml[8];
    __shared__ float4 sums[8][64];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quads = p.head_size / 4, mine = warp % WARPS;
    grid_wait();
    const int items = (int)p.batch.n_rows * p.q_heads;   // (below 2^31)
    for (int64_t i0 = (int64_t)blockIdx.x * ITEMS; i0 < items; i0 += (int64_t)gridDim.x * ITEMS) {
        const int item = (int)min(i0 + warp / WARPS, (int64_t)items);
        bool out = item < items;
        const int r = out ? item / p.q_heads : 0;
        const int head = item - r * p.q_heads, b = seq_of_row_warp(p.batch, r);
        out = out && b >= 0;
        float m = -INFINITY, l = 0.0f;
        float4 o[COLS] = {};
        bool any = false;
        const int g = head / p.group, gi = head - g * p.group;
        if (out) {
            const Span s = span_of(p.batch, b);
            const int i = (int)(r - s.first), x = i * p.group + gi, row_tile = x >> lo.row_shift, tiles = unit_tiles(p, lo, s, row_tile);
            const int64_t index = (int64_t)s.len - s.count + i;
            // the parts of its own unit: those of CTAs c0 .. c1 (none: c1 < c0)
            int64_t before = 0;
            for (int t = lane; t < row_tile; t += 32) before += unit_tiles(p, lo, s, t);
            for (int d = 16; d; d >>= 1) before += __shfl_xor_sync(~0u, before, d);
            const Plan plan = lo.plan[b];
            const int64_t total = lo.plan[lo.seqs].tiles, tile0 = plan.tiles + before * p.kv_heads + (int64_t)g * tiles, unit = plan.units + (int64_t)row_tile * p.kv_heads + g;
            const int c0 = tiles ? cta_of(total, lo.ctas, tile0) : 0, c1 = tiles ? cta_of(total, lo.ctas, tile0 + tiles - 1) : -1;
            // and of the prefix'
            int f0 = 0, f1 = -1;
            const int y = r * p.group + gi;
            const int64_t f_unit = (int64_t)(y >> lf.row_shift) * p.kv_heads + g;
            if (lf.front_tiles && index >= 0) {
                const int64_t all = lf.seqs ? lf.plan[lf.seqs].tiles : lf.front_units * lf.front_tiles;
                f0 = cta_of(all, lf.ctas, f_unit * lf.front_tiles);
                f1 = cta_of(all, lf.ctas, (f_unit + 1) * lf.front_tiles - 1);
            }
            out = !p.whole || c0 != c1;   // (else it was finished where it was computed)
            if (out) {
                // EACH parts at a time: a lane reads the (m, l) of one, then all lanes sum the columns, four parts' loads ahead of their use
                const int n_front = f1 - f0 + 1, n = n_front + (c1 - c0 + 1), y_row = y & (lf.tile_rows - 1), x_row = x & (lo.tile_rows - 1);
                for (int k0 = EACH * mine; k0 < n; k0 += EACH * WARPS) {
                    const int k = lane < EACH ? k0 + lane : n;
                    const bool front = k < n_front;
                    const int64_t slot = front ? f_unit + f0 + k : unit + c0 + (k - n_front);
                    float2 part = make_float2(-INFINITY, -1.0f);
                    if (k < n && slot >= 0 && slot < (front ? lf.slots : lo.slots)) part = front ? lf.ml[slot * lf.tile_rows + y_row] : lo.ml[slot * lo.tile_rows + x_row];
                    const float* from = front ? part_at(lf, p.head_size, slot, y_row, 0) : part_at(lo, p.head_size, slot, x_row, 0);
                    const bool has = !(part.y < 0.0f);
                    unsigned left = __ballot_sync(~0u, has);
                    if (!left) continue;
                    float now = has ? part.x : -INFINITY;
                    for (int d = 16; d; d >>= 1) now = fmaxf(now, __shfl_xor_sync(~0u, now, d));
                    now = fmaxf(m, now);
                    const float base = now == -INFINITY ? 0.0f : now, f = ex2(m - base), w = has ? ex2(part.x - base) : 0.0f;
                    float sum = has ? part.y * w : 0.0f;
                    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
                    m = now;
                    l = l * f + sum;
                    any = true;
#pragma unroll
                    for (int c = 0; c < COLS; c++) { o[c].x *= f; o[c].y *= f; o[c].z *= f; o[c].w *= f; }
                    while (left) {
                        float4 v[4][COLS];
                        float wk[4];
#pragma unroll
                        for (int u = 0; u < 4; u++) {
                            const int i = left ? __ffs(left) - 1 : 0;
                            wk[u] = left ? __shfl_sync(~0u, w, i) : 0.0f;
                            const bool in_front = k0 + i < n_front;
                            const float* at = reinterpret_cast<const float*>(__shfl_sync(~0u, reinterpret_cast<unsigned long long>(from), i));
                            const int64_t step = (int64_t)(in_front ? lf.tile_rows : lo.tile_rows) * 8;   // from 8 columns to the next
#pragma unroll
                            for (int c = 0; c < COLS; c++)
                                if (lane + 32 * c < quads) v[u][c] = left ? *reinterpret_cast<const float4*>(at + (lane + 32 * c >> 1) * step + 4 * (lane & 1)) : make_float4(0, 0, 0, 0);
                            left &= left - 1;
                        }
#pragma unroll
                        for (int u = 0; u < 4; u++)
#pragma unroll
                            for (int c = 0; c < COLS; c++)
                                if (lane + 32 * c < quads) {
                                    o[c].x = fmaf(v[u][c].x, wk[u], o[c].x); o[c].y = fmaf(v[u][c].y, wk[u], o[c].y);
                                    o[c].z = fmaf(v[u][c].z, wk[u], o[c].z); o[c].w = fmaf(v[u][c].w, wk[u], o[c].w);
                                }
                    }
                }
            }
        }
        if (WARPS > 1) {   // (one item a CTA: the same branch for all)
            __syncthreads();
            if (lane == 0) ml[warp] = make_float2(m, any ? l : -1.0f);
#pragma unroll
            for (int c = 0; c < COLS; c++)
                if (lane + 32 * c < quads) sums[warp][lane + 32 * c] = o[c];
            __syncthreads();
            if (warp) continue;
            for (int i = 1; i < WARPS; i++) {
                const float2 part = ml[i];
                if (part.y < 0.0f) continue;
                const float now = fmaxf(m, part.x), base = now == -INFINITY ? 0.0f : now, f = ex2(m - base), w = ex2(part.x - base);
                m = now;
                l = l * f + part.y * w;
                any = true;
#pragma unroll
                for (int c = 0; c < COLS; c++)
                    if (lane + 32 * c < quads) {
                        const float4 v = sums[i][lane + 32 * c];
                        o[c].x = fmaf(o[c].x, f, v.x * w); o[c].y = fmaf(o[c].y, f, v.y * w);
                        o[c].z = fmaf(o[c].z, f, v.z * w); o[c].w = fmaf(o[c].w, f, v.w * w);
                    }
            }
        }
        if (!out) continue;
        const UnitRow row = {(int64_t)r, head, 0};
#pragma unroll
        for (int c = 0; c < COLS; c++)
            if (lane + 32 * c < quads)
                store_row(p, row, 4 * (lane + 32 * c), any ? make_float4(o[c].x / l, o[c].y / l, o[c].z / l, o[c].w / l) : make_float4(0.0f, 0.0f, 0.0f, 0.0f));
        if (lane == 0 && p.lse) p.lse[item] = any ? lse_of(m, l) : -INFINITY;
    }
}

}  // namespace paged
}  // namespace lmrs
