// paged8_tensor.cuh -- attention over 8-bit pages for many rows that see the same keys (the prefix, portions of prompts), on the 5th-generation tensor cores.  Rows of 16-bit types.
//
// The line, its units and parts, the order of the work and TMEM are rows128_kernel's (paged_tensor.cuh), the mathematics that of paged8_attn.cuh: both products take float16, and codes are converted on
// the way into the operands' ring:
//   warps 0-3, 4-7   the rows of the first and the second block, a thread a row.  They also bring the queries in: float16, times a power of two for each row of bfloat16
//   warps 8, 9       the keys, and the values: codes by TMA (or 16 bytes a lane) into slots of their own, two operands ahead; from there, 16 codes a lane at a time, as float16 into the ring.  Heads beyond 128: one block
//                    of rows only, and warps 4-7 take both, 16 keys each
//   warp 10          the products
// A thread's score of a key is its dot product times the key's scale; its weight carries the value's scale; both scales come from shared memory, four keys a load.
// Measured on a B200, us: 244 rows of a KV head behind 8200 keys, 8 KV heads of 128, e4m3: 39 (and 80 with the own keys and the join); 12 prompts behind 2050, heads of 256, capped: 306, and 42 for the join.
// What bounds it: of the 1.7 us that a tile of 64 keys and 256 rows takes, 1.05 go by between a copying warp's conversions (0.7 of them on places, scales and boxes of the next operand: dependent instructions of
// one warp), 0.65 for one; the rows' warps need 0.95, the products 0.3 (the tensor pipe is active for 11 % of the prefix' time, 16 % of the prompts').  A part costs some 5 us besides: its queries, its first tile, its sums.
// Steps, us for the prompts without / with a cap: all rows' queries a row a thread 399 / 492; four copying warps for heads of 256 363 / 454; queries eight lanes a row 314 / 469; caps and masks in loops
// (unrolled, their code pushes the other roles' out of the instruction cache) 314 / 348.  13 warps, so that keys and values have two each: 128 registers a thread, no faster; taken back.
#pragma once
#include "paged8_attn.cuh"
#include "paged_tensor.cuh"

namespace lmrs {
namespace paged {

template <int DP> struct TensorShape8 {
    static constexpr int THREADS = 384, BLOCK = 128, BLOCKS = DP <= 128 ? 2 : 1, ROWS = BLOCK * BLOCKS, KEYS = 64;
    // copying warps: for heads of up to 128 one for the keys and one for the values, all 64 of a tile; beyond that (one block of rows, so that warps 4-7 are free) four for both, 16 keys each
    static constexpr bool SPLIT = DP <= 128;
    static constexpr int COPIERS = SPLIT ? 2 : 4, COPIER = SPLIT ? 8 : 4, PRODUCTS = 10, WARP_KEYS = SPLIT ? 64 : 16, EACH = SPLIT ? 2 : 1;   // (their number, the first of them; keys of a lane)
    static constexpr int COL_BOXES = DP / 64;                               // 64 columns of an operand in float16: rows of 128 bytes, their 16-byte pieces rotated (SWIZZLE_128B)
    static constexpr int SLOT = COL_BOXES * KEYS * 128, SLOTS = DP <= 64 ? 8 : DP <= 128 ? 6 : 3, Q_BLOCK = COL_BOXES * BLOCK * 128;
    static constexpr int BOX = DP < 128 ? DP : 128, KV = WARP_KEYS * DP;    // codes of a copying warp: columns of a TMA box, bytes of an operand
    static constexpr int STAGES = 3;                                        // its slots for them
    static constexpr int RING = 16;                                         // tiles whose keys' places and scales are known
    static constexpr int O_AT = 256;                                        // TMEM columns: two sets of scores for each block, then o of each block
    static constexpr int SMEM = 1024 + SLOTS * SLOT + BLOCKS * Q_BLOCK + COPIERS * STAGES * KV;
    static_assert(O_AT + BLOCKS * DP <= 512 && 2 * 2 * KEYS <= O_AT, "TMEM");
};
struct KeyAt { int page, place, head, boxed; };   // (page -1: nowhere)
template <int DP> struct TensorShared8 {
    using S = TensorShape8<DP>;
    uint64_t full[S::SLOTS], empty[S::SLOTS];   // slots of the ring
    uint64_t staged[S::COPIERS][S::STAGES];     // slots of codes, where they come by TMA
    uint64_t known[S::RING];                    // which of a tile's keys are there, and their scales, are written
    uint64_t scores[4], weights[4];             // sets of scores (two for each block): written by the products, replaced by weights
    uint64_t summed[4];                         // o of a block: the products of a tile have ended, even tiles and odd ones
    uint64_t read[2];                           // the part's o of a block has been read
    uint64_t queries;                           // the part's queries are there
    uint64_t parted;                            // both groups have ended the part
    alignas(16) float key_scale[S::RING][S::KEYS], value_log[S::RING][S::KEYS], value_by[S::RING][S::KEYS];
    KeyAt places[S::SPLIT ? 1 : S::COPIERS][4][16];   // (of warps that take both) of the last four tiles whose keys were asked for
    int part_tiles[S::COPIERS][4];              // of the last four parts
    uint32_t there[S::RING][2];
    uint32_t tmem;
    int gave_up;
};
PG_DEVINL uint64_t mul_pair(uint64_t a, uint64_t b) { uint64_t r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
PG_DEVINL uint64_t same_pair(float a) { return pair_of(__float_as_uint(a), __float_as_uint(a)); }

// 16 dot products (times their keys' scales) of a lane, capped, as cap_scores does
template <typename T> PG_DEVINL void cap_pairs(const AttnParams<T>& p, uint64_t (&s)[8]) {
    const uint64_t in = same_pair(p.cap_in), out = same_pair(p.softcap * LOG2E);
    float far = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        s[i] = mul_pair(s[i], in);
        const float2 x = pair_open(s[i]);
        far = fmaxf(far, fmaxf(fabsf(x.x), fabsf(x.y)));
    }
    if (__all_sync(~0u, far <= 0.5f)) {   // (tanh_near, two at a time)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint64_t y = mul_pair(s[i], s[i]);
            uint64_t t = fma_pair(y, same_pair(21844.0f / 6081075.0f), same_pair(-1382.0f / 155925.0f));
            t = fma_pair(y, t, same_pair(62.0f / 2835.0f));
            t = fma_pair(y, t, same_pair(-17.0f / 315.0f));
            t = fma_pair(y, t, same_pair(2.0f / 15.0f));
            t = fma_pair(y, t, same_pair(-1.0f / 3.0f));
            s[i] = mul_pair(fma_pair(mul_pair(y, t), s[i], s[i]), out);
        }
    } else {
        const float cap2 = p.softcap * LOG2E;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float2 x = pair_open(s[i]);
            s[i] = pair_of(__float_as_uint(cap2 * (fabsf(x.x) <= 0.5f ? tanh_near(x.x) : tanh_far(x.x))), __float_as_uint(cap2 * (fabsf(x.y) <= 0.5f ? tanh_near(x.y) : tanh_far(x.y))));
        }
    }
}

template <typename T, int FORM, int DP>
__global__ void __launch_bounds__(TensorShape8<DP>::THREADS, 1) codes128_kernel(const __grid_constant__ Attn8Params<T> p, const __grid_constant__ Line l, const __grid_constant__ Boxes8 boxes) {
    using S = TensorShape8<DP>;
    extern __shared__ uint8_t raw[];
    __shared__ TensorShared8<DP> sh;
    uint8_t* ring = raw + (((smem_at(raw) + 1023u) & ~1023u) - smem_at(raw));
    uint8_t *queries = ring + S::SLOTS * S::SLOT, *codes = queries + S::BLOCKS * S::Q_BLOCK;
    const int warp = __shfl_sync(~0u, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31, D = p.head_size;
    volatile int* gave_up = &sh.gave_up;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S::SLOTS; i++) { mbar_init(&sh.full[i], S::KEYS / S::WARP_KEYS); mbar_init(&sh.empty[i], 1); }
        for (int i = 0; i < S::COPIERS * S::STAGES; i++) mbar_init(&sh.staged[0][0] + i, 1);
        for (int i = 0; i < S::RING; i++) mbar_init(&sh.known[i], S::COPIERS);
        for (int i = 0; i < 4; i++) { mbar_init(&sh.scores[i], 1); mbar_init(&sh.weights[i], 128); mbar_init(&sh.summed[i], 1); }
        for (int i = 0; i < 2; i++) mbar_init(&sh.read[i], 128);
        mbar_init(&sh.queries, S::ROWS);
        mbar_init(&sh.parted, S::ROWS);
        sh.gave_up = 0;
        fence_barrier_init();
    }
    Walk w;
    int64_t from, to;
    walk_begin<T, S::THREADS>(p, l, w, from, to);   // (synchronises the CTA)
    if (from >= to) { grid_launch(); return; }
    if (warp == S::PRODUCTS) {
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_at(&sh.tmem)), "n"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tmem_before();
    __syncthreads();
    tmem_after();
    const uint32_t tmem = sh.tmem;
    grid_launch();
    // Parts of the CTA, one after the other: `tiles` of unit w from w.tile on, `blocks` of its rows.  Every role walks along by itself.
    int left = (int)(to - from), tiles = 0, blocks = 0, used = 0;
    auto enter = [&]() {
        tiles = min(left, w.tiles - w.tile);
        used = w.b < 0 ? (int)min((int64_t)S::ROWS, p.batch.n_rows * p.group - (int64_t)w.row_tile * S::ROWS) : min(S::ROWS, w.s.count * p.group - w.row_tile * S::ROWS);
        blocks = used > S::BLOCK ? 2 : 1;
    };
    auto leave = [&]() {   // false: that was the last one
        left -= tiles;
        if (left <= 0) return false;
        walk_next_unit(p, l, w);
        if (w.tiles == 0) { left = 0; return false; }   // (the line ended early: lengths changed under the kernel)
        return true;
    };
    if (warp >= 4 * S::BLOCKS) {
        if (const int copier = warp - S::COPIER; copier < S::COPIERS) {
            // ---- keys and values: asked for as codes STAGES - 1 operands ahead, then converted.  Operands of a part lie in the ring as K0 K1 V0 K2 V1 ... ----
            const bool takes_keys = !S::SPLIT || copier == 0, takes_values = !S::SPLIT || copier == 1;
            const int mine = S::SPLIT ? 0 : copier, whole = D / 16, key = lane & (S::SPLIT ? 31 : S::WARP_KEYS - 1);   // (of 16 keys, two lanes each; of 64, a lane has this one and the one 32 on)
            const bool first_lanes = S::SPLIT || lane < S::WARP_KEYS;
            uint8_t* stage = codes + copier * (S::STAGES * S::KV);
            uint64_t* staged = sh.staged[copier];
            const int box_rows = boxes.rows, groups = box_rows ? S::WARP_KEYS / box_rows : 0;
            constexpr int COL_BOXES = DP / S::BOX;
            const int box_col = lane % COL_BOXES, box_group = lane / COL_BOXES;
            // what is asked for next: of part w, whose places are looked up a tile ahead
            int keys_asked = 0, values_asked = 0, key_tiles = 0, value_tiles = 0, parts = 0, asked = 0, ask_slot = 0;   // of the part; of all parts; operands
            int page[S::EACH], place[S::EACH], boxed = 0, ahead_tiles = 0;   // ahead_tiles: of the part that w is in (w goes on to it when the last places of this one have been taken)
            bool more = true, ok = true;
            uint32_t by_tma = 0, written = 0, rounds = 0;   // a bit a slot: codes are on their way by TMA, its bytes were last written otherwise, the phase that its barrier is in
            uint32_t bits_of[3][S::EACH] = {};               // (of keys by themselves) which of a slot's are there
            static_assert(S::STAGES == 3, "bits_of");
            const int* table = nullptr;
            auto look = [&](int j) {
                const int first = (w.tile + j) * S::KEYS + mine * S::WARP_KEYS;
                if (j == 0) table = w.b < 0 ? p.batch.prefix : p.batch.tables + w.b * p.batch.table_stride;
                boxed = box_rows && first + S::WARP_KEYS <= w.keys;
#pragma unroll
                for (int e = 0; e < S::EACH; e++) {
                    const int x = first + key + 32 * e;
                    page[e] = -1;
                    place[e] = 0;
                    if (x < w.keys) {
                        const int i = p.page_shift >= 0 ? x >> p.page_shift : x / p.batch.page_size;
                        page[e] = table[i];
                        place[e] = x - i * p.batch.page_size;
                    }
                }
            };
            auto ask = [&]() {   // the next operand's codes, if there is one
                if (more) {
                    const bool values = S::SPLIT ? takes_values : !(keys_asked < tiles && keys_asked - values_asked < 2);
                    KeyAt k[S::EACH];
                    if (S::SPLIT || !values) {   // whose places have been looked up
#pragma unroll
                        for (int e = 0; e < S::EACH; e++) {
                            const bool is = page[e] >= 0 && page[e] < p.batch.pages;
                            k[e] = KeyAt{is ? page[e] : -1, place[e], w.head, boxed};
                            if (S::SPLIT) {
                                const uint32_t bits = __ballot_sync(~0u, is);
#pragma unroll
                                for (int i = 0; i < 3; i++)
                                    if (i == ask_slot) bits_of[i][e] = bits;
                            }
                            const int page_or_0 = is ? page[e] : 0, at = is ? place[e] : 0, block = p.block_shift >= 0 ? at >> p.block_shift : at / p.c.block;
                            const int set = (takes_keys ? key_tiles : value_tiles) % S::RING, x = mine * S::WARP_KEYS + key + 32 * e;
                            if (first_lanes) {
                                if (takes_keys) copy4(smem_at(&sh.key_scale[set][x]), p.c.ks + page_or_0 * p.c.ks_page + block * p.c.ks_block + w.head * p.c.ks_head, is);
                                if (takes_values) copy4(smem_at(&sh.value_log[set][x]), p.c.vs + page_or_0 * p.c.vs_page + block * p.c.vs_block + w.head * p.c.vs_head, is);
                            }
                        }
                        if (!S::SPLIT && first_lanes) sh.places[mine][key_tiles & 3][key] = k[0];
                    } else {
                        k[0] = sh.places[mine][value_tiles & 3][key];
                    }
                    const uint32_t to_codes = smem_at(stage) + ask_slot * S::KV;
                    __syncwarp();
                    if (k[0].boxed) {   // (the same for all lanes)
                        if (written >> ask_slot & 1) {
                            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                            __syncwarp();
                        }
                        if (lane == 0) mbar_expect_tx(&staged[ask_slot], S::KV);
                        const int of_key = box_group * box_rows & (S::WARP_KEYS - 1);
                        int of = __shfl_sync(~0u, k[0].page, of_key & 31), from_row = __shfl_sync(~0u, k[0].place, of_key & 31);
                        if (S::EACH == 2) {
                            const int other = __shfl_sync(~0u, k[S::EACH - 1].page, of_key & 31), other_row = __shfl_sync(~0u, k[S::EACH - 1].place, of_key & 31);
                            if (of_key >= 32) { of = other; from_row = other_row; }
                        }
                        if (of < 0) { of = p.batch.pages; from_row = 0; }   // (outside the map: zeros)
                        __syncwarp();
                        if (box_group < groups)
                            tma_box(to_codes + box_col * (S::WARP_KEYS * S::BOX) + box_group * box_rows * S::BOX, values ? &boxes.v : &boxes.k, S::BOX * box_col, from_row, k[0].head, of,
                                    values ? boxes.v_place : boxes.k_place, values ? boxes.v_head : boxes.k_head, &staged[ask_slot]);
                        __syncwarp();
                        by_tma |= 1u << ask_slot;
                        written &= ~(1u << ask_slot);
                    } else {
                        written |= 1u << ask_slot;
                        const uint8_t* base = values ? p.c.v : p.c.k;
                        int64_t start[S::EACH];
#pragma unroll
                        for (int e = 0; e < S::EACH; e++)
                            start[e] = k[e].page < 0 ? -1 : values ? k[e].page * p.c.v_page + k[e].place * p.c.v_slot + k[e].head * p.c.v_head : k[e].page * p.c.k_page + k[e].place * p.c.k_slot + k[e].head * p.c.k_head;
                        constexpr int CHUNKS = DP / 16, LANES = CHUNKS < 8 ? CHUNKS : 8, AT_ONCE = 32 / LANES;   // lanes a row, rows at a time
#pragma unroll 2
                        for (int r0 = 0; r0 < S::WARP_KEYS; r0 += AT_ONCE) {
                            const int row = r0 + lane / LANES;
                            int64_t row_start = __shfl_sync(~0u, start[0], row & 31);
                            if (S::EACH == 2 && r0 >= 32) row_start = __shfl_sync(~0u, start[S::EACH - 1], row & 31);
#pragma unroll
                            for (int c = 0; c < CHUNKS; c += LANES) {
                                const int piece = c + lane % LANES;
                                const bool in = row_start >= 0 && piece < whole;
                                copy16(to_codes + code_at<S>(row, piece), in ? base + row_start + 16 * piece : base, in);
                            }
                        }
                    }
                    asked++;
                    ask_slot = ask_slot + 1 == S::STAGES ? 0 : ask_slot + 1;
                    if (values) { value_tiles++; values_asked++; }
                    else { key_tiles++; keys_asked++; }
                    if (S::SPLIT || !values) {   // its places are taken: look for the next ones
                        const int taken = takes_keys ? keys_asked : values_asked;
                        if (taken < tiles) look(taken);
                        else {
                            left -= tiles;
                            ahead_tiles = 0;
                            if (left > 0) {
                                walk_next_unit(p, l, w);
                                if (w.tiles > 0) {
                                    ahead_tiles = min(left, w.tiles - w.tile);
                                    if (lane == 0) sh.part_tiles[copier][parts & 3] = ahead_tiles;
                                    parts++;
                                    look(0);
                                }
                            }
                            if (!ahead_tiles) left = 0;
                        }
                    }
                    if ((takes_values ? values_asked : keys_asked) == tiles) {   // the part's last operand: w has gone on
                        keys_asked = values_asked = 0;
                        tiles = ahead_tiles;
                        more = tiles > 0;
                    }
                }
                copy_commit();
            };
            enter();
            if (lane == 0) sh.part_tiles[copier][0] = tiles;
            parts = 1;
            __syncwarp();
            look(0);
            for (int i = 0; i < S::STAGES - 1; i++) ask();
            // conversion: keys and values of the part that is converted, its first place in the ring, and what has been in all
            int part = 0, k_done = 0, v_done = 0, all = 0, base = 0, done = 0, from_slot = 0, part_has = tiles;
            __syncwarp();
            part_has = sh.part_tiles[copier][0];
            while (ok && done < asked) {
                ask();
                copy_wait<S::STAGES - 1>();
                const bool values = S::SPLIT ? takes_values : !(k_done < part_has && k_done - v_done < 2);
                const int at = base + (values ? (v_done + 1 < part_has ? 2 * v_done + 2 : 2 * part_has - 1) : k_done ? 2 * k_done - 1 : 0), slot = at % S::SLOTS;   // the operand's number in the ring
                if (by_tma >> from_slot & 1) {
                    ok = __all_sync(~0u, dense::mbar_wait_bounded(&staged[from_slot], rounds >> from_slot & 1, gave_up, dense::TG_CODES128 + dense::TG_FULL));
                    if (!ok) break;
                    rounds ^= 1u << from_slot;
                    by_tma &= ~(1u << from_slot);
                }
                __syncwarp();
                if (S::SPLIT || !values) {
                    const int set = all % S::RING;
                    if (takes_values && first_lanes) {
#pragma unroll
                        for (int e = 0; e < S::EACH; e++) {
                            const int x = mine * S::WARP_KEYS + key + 32 * e;
                            const float2 v = value_terms(sh.value_log[set][x]);
                            sh.value_log[set][x] = v.x;
                            sh.value_by[set][x] = v.y;
                        }
                    }
                    if (takes_keys) {
                        if (S::SPLIT) {
#pragma unroll
                            for (int e = 0; e < S::EACH; e++)
                                if (lane == 0) sh.there[set][e] = from_slot == 0 ? bits_of[0][e] : from_slot == 1 ? bits_of[1][e] : bits_of[2][e];
                        } else {
                            const unsigned bits = __ballot_sync(~0u, sh.places[S::SPLIT ? 0 : mine][all & 3][key].page >= 0);
                            if (lane == 0) reinterpret_cast<uint16_t*>(sh.there[set])[mine] = (uint16_t)bits;
                        }
                    }
                    __syncwarp();
                    if (lane == 0) arrive(&sh.known[set]);
                    all++;
                }
                ok = wait_warp(&sh.empty[slot], at / S::SLOTS + 1, gave_up, dense::TG_CODES128 + dense::TG_FREE - dense::TG_PAGED);
                if (!ok) break;
                constexpr int BATCH = 4;
#pragma unroll 1
                for (int e = 0; e < S::EACH; e++) {
                    const int row = key + 32 * e;
                    uint8_t* to_row = ring + slot * S::SLOT + (mine * S::WARP_KEYS + row) * 128;
#pragma unroll 1
                    for (int c0 = S::SPLIT ? 0 : BATCH * (lane / S::WARP_KEYS); c0 < whole; c0 += S::SPLIT ? BATCH : 2 * BATCH) {   // (past the end of a head: zeros, or what an earlier tile left; the products do not read it)
                        uint4 u[BATCH];
#pragma unroll
                        for (int i = 0; i < BATCH; i++) u[i] = *reinterpret_cast<const uint4*>(stage + from_slot * S::KV + code_at<S>(row, c0 + i));
#pragma unroll
                        for (int i = 0; i < BATCH; i++) {
                            const uint32_t words[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
                            uint32_t h[8];
#pragma unroll
                            for (int k = 0; k < 4; k++) codes_to_halves<FORM, 0>(words[k], h[2 * k], h[2 * k + 1]);
                            uint8_t* to = to_row + (c0 >> 2) * (S::KEYS * 128);
                            *reinterpret_cast<uint4*>(to + ((2 * i ^ (row & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
                            *reinterpret_cast<uint4*>(to + (((2 * i + 1) ^ (row & 7)) << 4)) = make_uint4(h[4], h[5], h[6], h[7]);
                        }
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) arrive(&sh.full[slot]);
                done++;
                from_slot = from_slot + 1 == S::STAGES ? 0 : from_slot + 1;
                if (values) v_done++;
                else k_done++;
                if ((takes_values ? v_done : k_done) == part_has) {
                    base += 2 * part_has;
                    k_done = v_done = 0;
                    part++;
                    if (part < parts) part_has = sh.part_tiles[copier][part & 3];
                }
            }
            copy_wait<0>();
            if (!ok)   // gave up: what TMA was asked for lands before shared memory goes away
                for (int i = 0; i < S::STAGES; i++)
                    if (by_tma >> i & 1) dense::mbar_wait_for(&staged[i], rounds >> i & 1, nullptr);
        } else if (warp == S::PRODUCTS) {
            // ---- products ----
            constexpr int WHO = dense::TG_CODES128 - dense::TG_PAGED;
            const uint32_t one = dense::elect_one();
            const uint32_t form = (1u << 4) | ((uint32_t)(S::BLOCK >> 4) << 24);   // f32 += f16 x f16, 128 rows
            const uint32_t score_form = form | ((uint32_t)(S::KEYS >> 3) << 17), sum_form = form | (1u << 16) | ((uint32_t)(D >> 3) << 17);   // (values are MN-major)
            const uint32_t ring_lo = (uint32_t)dense::tg_desc_sw128(ring), q_lo = (uint32_t)dense::tg_desc_sw128(queries);
            const int steps = D / 16;
            uint32_t n = 0, round = 0;           // slot of the next operand tile, rounds of the ring before it
            int w_count[4] = {0, 0, 0, 0}, part = 0;   // sets of weights taken
            bool ok = true;
            auto take = [&]() {
                ok = ok && wait_warp(&sh.full[n], (int)round, gave_up, WHO + dense::TG_FULL);
                tmem_after();
                const uint32_t slot = n;
                if (++n == S::SLOTS) { n = 0; round++; }
                return slot;
            };
            // (unrolled, so that descriptors are sums of constants in uniform registers)
            auto scores = [&](int block, int j, uint32_t slot) {
                const int set = 2 * block + (j & 1);
                const uint32_t d = tmem + (uint32_t)set * S::KEYS, a = q_lo + (uint32_t)block * (S::Q_BLOCK >> 4), b = ring_lo + slot * (S::SLOT >> 4);
#pragma unroll
                for (int k = 0; k < DP / 16; k++)
                    if (k < steps)
                        dense::tg_mma_ss1(one, d, a + (uint32_t)(k >> 2) * (S::BLOCK * 128 >> 4) + (k & 3) * 2, b + (uint32_t)(k >> 2) * (S::KEYS * 128 >> 4) + (k & 3) * 2, score_form, k > 0);
                dense::tg_commit1(one, &sh.scores[set]);
            };
            auto sums = [&](int block, int j, uint32_t slot) {
                const int set = 2 * block + (j & 1);
                if (j == 0 && part > 0) ok = ok && wait_warp(&sh.read[block], part - 1, gave_up, WHO + dense::TG_VALUES_READ);
                ok = ok && wait_warp(&sh.weights[set], w_count[set]++, gave_up, WHO + dense::TG_WEIGHTS);
                if (!ok) return;
                tmem_after();
                // 16 keys a step: two groups of 8 rows of 128 bytes; from 64 columns to the next: a box
                const uint32_t d = tmem + S::O_AT + (uint32_t)block * DP, a = tmem + (uint32_t)set * S::KEYS;
                const uint32_t b = (ring_lo & 0xffffu) + slot * (S::SLOT >> 4) + ((uint32_t)(S::KEYS * 128 >> 4) << 16), more = j > 0;
#pragma unroll
                for (int k = 0; k < S::KEYS / 16; k++) dense::tg_mma_ts1(one, d, a + k * 8, b + k * (2048 >> 4), sum_form, k > 0 ? 1u : more);
                dense::tg_commit1(one, &sh.summed[set]);
            };
            do {   // the scores of tile j + 2 follow the sums of tile j into the same set
                enter();
                ok = ok && wait_warp(&sh.queries, part, gave_up, WHO + dense::TG_QUERIES);
                tmem_after();
                for (int j = 0; j < 2 && j < tiles; j++) {
                    const uint32_t keys = take();
                    if (!ok) break;
                    for (int g = 0; g < blocks; g++) scores(g, j, keys);
                    dense::tg_commit1(one, &sh.empty[keys]);
                }
                for (int j = 0; j < tiles && ok; j++) {
                    const uint32_t values = take();
                    uint32_t keys = 0;
                    for (int g = 0; g < blocks && ok; g++) {
                        sums(g, j, values);
                        if (ok && g == blocks - 1) dense::tg_commit1(one, &sh.empty[values]);
                        if (j + 2 < tiles) {
                            if (g == 0) keys = take();
                            if (ok) scores(g, j + 2, keys);
                        }
                    }
                    if (ok && j + 2 < tiles) dense::tg_commit1(one, &sh.empty[keys]);
                }
                part++;
            } while (ok && leave());
            // the last commit is that of the last values' slot: none may arrive after the CTA has ended
            if (ok) ok = wait_warp(&sh.empty[n == 0 ? S::SLOTS - 1 : n - 1], (int)(n == 0 ? round - 1 : round), gave_up, WHO + dense::TG_FREE);
            if (!ok)   // gave up: products already issued may still run; they get a millisecond to end before shared memory and TMEM go away
                for (int i = 0; i < 1000; i++) __nanosleep(1000);
        }
        __syncwarp();
    } else {
        // ---- rows ----
        constexpr int WHO = dense::TG_CODES128 - dense::TG_PAGED;
        const int group = warp >> 2, row = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;   // this warp's 32 TMEM lanes
        int s_count[2] = {0, 0}, k_count = 0, part = 0;   // phases of earlier parts: this group's even and odd tiles, all tiles, parts
        bool ok = true;
        do {
            enter();
            const bool mine = group < blocks;
            const int x = group * S::BLOCK + row;
            if (mine) {
                const UnitRow r = unit_row(p, l, w, x);
                // The queries of the warp's rows, as float16: all products that read the last ones have ended, since their sums have been waited for.  Eight lanes a row, four rows at a time
                float2 factor = make_float2(1.0f, 1.0f);
                {
                    const int c = lane & 7, whole = D / 8, row0 = (warp & 3) * 32;
                    const uint32_t q_at = smem_at(queries) + group * S::Q_BLOCK;
                    constexpr int AT_ONCE = DP <= 128 ? 4 : 2;   // fours of rows whose loads are under way together
#pragma unroll 1
                    for (int i0 = 0; i0 < 8; i0 += AT_ONCE) {
                        Piece<T, 8> v[AT_ONCE][S::COL_BOXES];
#pragma unroll
                        for (int u = 0; u < AT_ONCE; u++) {
                            const int at = group * S::BLOCK + row0 + 4 * (i0 + u) + (lane >> 3);
                            const UnitRow of = unit_row(p, l, w, at);
                            const bool is = at < used;
                            const T* q = is ? p.q.data + of.row * p.q.row + of.head * p.q.head + 8 * c : p.q.data;
#pragma unroll
                            for (int k = 0; k < S::COL_BOXES; k++) {
                                const bool in = is && 8 * k + c < whole;
                                if (p.q_wide) {
                                    if (in) v[u][k] = *reinterpret_cast<const Piece<T, 8>*>(q + 64 * k);
                                } else {
#pragma unroll
                                    for (int e = 0; e < 8; e++)
                                        if (in) v[u][k].v[e] = q[64 * k + e];
                                }
                                if (!in)
#pragma unroll
                                    for (int e = 0; e < 8; e++) v[u][k].v[e] = from_f<T>(0.0f);
                            }
                        }
#pragma unroll
                        for (int u = 0; u < AT_ONCE; u++) {
                            float2 f = make_float2(1.0f, 1.0f);
                            if constexpr (!std::is_same<T, __half>::value) {
                                float most = 0.0f;
#pragma unroll
                                for (int k = 0; k < S::COL_BOXES; k++)
#pragma unroll
                                    for (int e = 0; e < 8; e++) most = fmaxf(most, fabsf(to_f(v[u][k].v[e])));
#pragma unroll
                                for (int d = 1; d < 8; d *= 2) most = fmaxf(most, __shfl_xor_sync(~0u, most, d));
                                f = row_factor(most);
                                const float mine_up = __shfl_sync(~0u, f.x, 8 * (lane & 3)), mine_down = __shfl_sync(~0u, f.y, 8 * (lane & 3));
                                if (lane >> 2 == i0 + u) factor = make_float2(mine_up, mine_down);
                            }
                            const int to = row0 + 4 * (i0 + u) + (lane >> 3);
#pragma unroll
                            for (int k = 0; k < S::COL_BOXES; k++) {
                                uint32_t h[4];
#pragma unroll
                                for (int e = 0; e < 4; e++) h[e] = to_halves(to_f(v[u][k].v[2 * e]) * f.x, to_f(v[u][k].v[2 * e + 1]) * f.x);
                                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(q_at + k * (S::BLOCK * 128) + to * 128 + ((c ^ (to & 7)) << 4)), "r"(h[0]), "r"(h[1]), "r"(h[2]), "r"(h[3]) : "memory");
                            }
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    arrive(&sh.queries);
                }
                const float down = p.softcap > 0.0f ? factor.y : fminf(fmaxf(factor.y * p.scale2, -FLT_MAX), FLT_MAX);
                float m = -INFINITY, sum = 0.0f;
                bool seen = false;
                const int least = w.b < 0 ? w.keys : unit_row(p, l, w, group * S::BLOCK).keys;   // (rows that come later see more)
                for (int j = 0; j < tiles && ok; j++) {
                    const int set = 2 * group + (j & 1), key0 = (w.tile + j) * S::KEYS, known = (k_count + j) % S::RING;
                    ok = wait_warp(&sh.known[known], (k_count + j) / S::RING, gave_up, WHO + dense::TG_PLACES) && wait_warp(&sh.scores[set], s_count[j & 1] + (j >> 1), gave_up, WHO + dense::TG_SCORES);
                    if (!ok) break;
                    tmem_after();
                    const uint32_t at = tmem + lanes + (uint32_t)set * S::KEYS;
                    const bool all = key0 + S::KEYS <= least && sh.there[known][0] == ~0u && sh.there[known][1] == ~0u;
                    const float *ks = sh.key_scale[known], *vl = sh.value_log[known], *vb = sh.value_by[known];
                    // Exponents.  Tiles that need neither a mask nor a cap are straight-line code on 64 of them in registers; the others go 16 at a time, in loops, to keep that code small (the warps of all
                    // roles wait for instructions otherwise), and leave the exponents where the scores were
                    uint32_t v[64];
                    float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    const bool plain = all && !(p.softcap > 0.0f);
                    auto sees = [&](int c) {   // bit i: the row sees key 32 c + i of the tile
                        const int limit = r.keys - key0 - 32 * c;
                        return sh.there[known][c] & (limit >= 32 ? ~0u : limit <= 0 ? 0u : (1u << limit) - 1);
                    };
                    if (plain) {
                        tmem_load64(at, v);
                        const uint64_t by = same_pair(down);
#pragma unroll
                        for (int i = 0; i < 64; i += 4) {
                            const ulonglong2 k = *reinterpret_cast<const ulonglong2*>(ks + i), a = *reinterpret_cast<const ulonglong2*>(vl + i);
                            const float2 e = pair_open(fma_pair(mul_pair(pair_of(v[i], v[i + 1]), k.x), by, a.x)), f = pair_open(fma_pair(mul_pair(pair_of(v[i + 2], v[i + 3]), k.y), by, a.y));
                            v[i] = __float_as_uint(e.x); v[i + 1] = __float_as_uint(e.y); v[i + 2] = __float_as_uint(f.x); v[i + 3] = __float_as_uint(f.y);
                        }
#pragma unroll
                        for (int i = 0; i < 64; i += 2) tops[i >> 1 & 3] = fmaxf(fmaxf(tops[i >> 1 & 3], __uint_as_float(v[i])), __uint_as_float(v[i + 1]));
                        seen = true;
                    } else {
#pragma unroll 1
                        for (int c = 0; c < 64; c += 16) {
                            uint32_t u[16], half[8];
                            tmem_load16(at + c, u);
                            uint64_t e[8];
#pragma unroll
                            for (int i = 0; i < 8; i++) e[i] = mul_pair(mul_pair(pair_of(u[2 * i], u[2 * i + 1]), *reinterpret_cast<const uint64_t*>(ks + c + 2 * i)), same_pair(down));
                            if (p.softcap > 0.0f) cap_pairs(p, e);
                            const uint32_t mask = sees(c >> 5) >> (c & 16);
                            seen = seen || (mask & 0xffff);
#pragma unroll
                            for (int h = 0; h < 8; h += 4) {
#pragma unroll
                                for (int i = 0; i < 4; i++) {
                                    float2 x = pair_open(add_pair(e[h + i], *reinterpret_cast<const uint64_t*>(vl + c + 2 * (h + i))));
                                    if (!(mask >> (2 * (h + i)) & 1)) x.x = -INFINITY;
                                    if (!(mask >> (2 * (h + i) + 1) & 1)) x.y = -INFINITY;
                                    tops[i] = fmaxf(tops[i], fmaxf(x.x, x.y));
                                    half[2 * i] = __float_as_uint(x.x);
                                    half[2 * i + 1] = __float_as_uint(x.y);
                                }
                                tmem_store8(at + c + 2 * h, half);
                            }
                        }
                        tmem_stored();
                    }
                    const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) - SHIFT8;
                    if (__any_sync(~0u, top > m + RESCALE_AT || (m == -INFINITY && top > m))) {
                        const float now = fmaxf(m, top), corr = ex2(m - (now == -INFINITY ? 0.0f : now));
                        if (j > 0) {
                            ok = wait_warp(&sh.summed[2 * group + ((j - 1) & 1)], s_count[(j - 1) & 1] + ((j - 1) >> 1), gave_up, WHO + dense::TG_VALUES);
                            if (!ok) break;
                            tmem_after();
#pragma unroll 1
                            for (int c = 0; c < D; c += 16) {
                                uint32_t o[16];
                                const uint32_t o_at = tmem + lanes + S::O_AT + (uint32_t)group * DP + c;
                                tmem_load16(o_at, o);
                                uint32_t a[8];
#pragma unroll
                                for (int h = 0; h < 16; h += 8) {
#pragma unroll
                                    for (int i = 0; i < 8; i++) a[i] = __float_as_uint(__uint_as_float(o[h + i]) * corr);
                                    tmem_store8(o_at + h, a);
                                }
                            }
                            tmem_stored();
                        }
                        sum *= corr;
                        m = now;
                    }
                    const float base = m == -INFINITY ? 0.0f : m;
                    const uint64_t less = same_pair(-base);
                    uint64_t total[2] = {0, 0};
                    auto weigh = [&](const uint32_t (&x)[4], const float* reciprocals, uint32_t& a, uint32_t& b) {   // four exponents to weights
                        const ulonglong2 by = *reinterpret_cast<const ulonglong2*>(reciprocals);
                        float2 e = pair_open(add_pair(pair_of(x[0], x[1]), less)), f = pair_open(add_pair(pair_of(x[2], x[3]), less));
                        e.x = ex2(e.x); e.y = ex2(e.y); f.x = ex2(f.x); f.y = ex2(f.y);
                        total[0] = fma_pair(pair_of(__float_as_uint(e.x), __float_as_uint(e.y)), by.x, total[0]);
                        total[1] = fma_pair(pair_of(__float_as_uint(f.x), __float_as_uint(f.y)), by.y, total[1]);
                        a = to_halves(e.x, e.y);
                        b = to_halves(f.x, f.y);
                    };
                    if (plain) {
                        uint32_t a[32];
#pragma unroll
                        for (int i = 0; i < 64; i += 4) {
                            const uint32_t x[4] = {v[i], v[i + 1], v[i + 2], v[i + 3]};
                            weigh(x, vb + i, a[i >> 1], a[(i >> 1) + 1]);
                        }
                        tmem_store32(at, a);   // (over scores that have been read)
                    } else {
#pragma unroll 1
                        for (int c = 0; c < 64; c += 16) {
                            uint32_t u[16], a[8];
                            tmem_load16(at + c, u);
#pragma unroll
                            for (int i = 0; i < 16; i += 4) {
                                const uint32_t x[4] = {u[i], u[i + 1], u[i + 2], u[i + 3]};
                                weigh(x, vb + c + i, a[i >> 1], a[(i >> 1) + 1]);
                            }
                            tmem_store8(at + (c >> 1), a);   // (columns c / 2 .. c / 2 + 7, all of them below c + 16: read)
                        }
                    }
                    const float2 both = pair_open(add_pair(total[0], total[1]));
                    sum += both.x + both.y;
                    tmem_stored();
                    tmem_before();
                    arrive(&sh.weights[set]);
                }
                // the part's rows
                const int64_t slot = w.unit + blockIdx.x;
                const bool whole = whole_unit(p, w, w.tile, w.tile + tiles - 1), is = x < used;
                ok = ok && wait_warp(&sh.summed[2 * group + ((tiles - 1) & 1)], s_count[(tiles - 1) & 1] + ((tiles - 1) >> 1), gave_up, WHO + dense::TG_VALUES);
                if (ok) {
                    tmem_after();
                    if (!seen) sum = -1.0f;
                    float* to_part = whole ? nullptr : part_at(l, D, slot, x, 0);
                    const bool store = is && (whole || slot < l.slots);
                    const float by = seen ? 1.0f / sum : 1.0f;
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        uint32_t o[32];
                        tmem_load32(tmem + lanes + S::O_AT + (uint32_t)group * DP + c, o);
                        if (!store) continue;
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            if (c + i >= D) break;   // (D is a multiple of 16)
                            float4 f = make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]), __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
                            float4 g = make_float4(__uint_as_float(o[i + 4]), __uint_as_float(o[i + 5]), __uint_as_float(o[i + 6]), __uint_as_float(o[i + 7]));
                            if (!seen) f = g = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            if (whole) {
                                f.x *= by; f.y *= by; f.z *= by; f.w *= by;
                                g.x *= by; g.y *= by; g.z *= by; g.w *= by;
                                store_row(p, r, c + i, f);
                                store_row(p, r, c + i + 4, g);
                            } else {
                                float4* at8 = reinterpret_cast<float4*>(to_part + (int64_t)((c + i) >> 3) * (S::ROWS * 8));
                                at8[0] = f;
                                at8[1] = g;
                            }
                        }
                    }
                    if (is) {
                        if (whole) { if (p.lse) p.lse[r.row * p.q_heads + r.head] = seen ? lse_of(m, sum) : -INFINITY; }
                        else if (slot < l.slots) l.ml[slot * S::ROWS + x] = make_float2(m, sum);
                    }
                    tmem_before();
                    arrive(&sh.read[group]);
                } else if (is) {   // gave up: NaN
                    if (whole) {
                        for (int c = 0; c < D; c++) p.out.data[r.row * p.out.row + r.head * p.out.head + c] = from_f<T>(NAN);
                        if (p.lse) p.lse[r.row * p.q_heads + r.head] = NAN;
                    } else if (slot < l.slots) {
                        l.ml[slot * S::ROWS + x] = make_float2(NAN, NAN);
                    }
                }
                s_count[0] += (tiles + 1) >> 1;
                s_count[1] += tiles >> 1;
            } else {   // a part without a second block: its turns pass
                arrive(&sh.queries);
                arrive(&sh.read[1]);
            }
            k_count += tiles;
            arrive(&sh.parted);
            ok = ok && wait_part(&sh.parted, part++, &sh.known[0], gave_up);
        } while (leave());
    }
    tmem_before();
    __syncthreads();
    if (warp == S::PRODUCTS) {
        __syncwarp();
        tmem_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
    }
    if (threadIdx.x == 0 && *gave_up && p.err) *p.err = *gave_up;
}

}  // namespace paged
}  // namespace lmrs
