// paged_tensor.cuh -- the same attention for many rows that see the same keys (the prefix, which all rows of a call share; portions of prompts), on the 5th-generation
// tensor cores.  16-bit types; the line, its units and the parts are those of paged_attn.cuh, with 128 or 256 rows a unit.
//
// CTA = 16 warps, one CTA an SM.  The rows of a unit are one or two blocks of 128, a TMEM lane each; a step of the work is one block against one tile of keys:
//     scores = Q . K^T            tcgen05.mma, both operands in shared memory, 128 x KEYS sums in TMEM (two sets, taken in turn)
//     weights = 2^(scores - m)    a thread a row: the scores from TMEM, the weights rounded to the type and back to TMEM over the scores
//     o += weights . V            tcgen05.mma, the weights from TMEM, the values in shared memory as they lie in the pages (keys x columns: MN-major)
//   warps 0-3, 4-7   the rows.  Two blocks: a group each, steps in turn, so that one's exponentials run under the other's products.  One block: the first group, and the
//                    scores of the next tile are computed meanwhile.
//   warps 8-11       copies of keys and values (16 bytes a thread, zeros for what is not there) into a ring of slots, one operand tile each, in the order K0 K1 V0 K2 V1 ...
//                    The places of a tile's keys are looked up by a thread each; pages of any size and order cost the same.
//   warp 12          the products
// o stays in TMEM for a whole part.  m is the largest score when it was last set; it is set anew, and o rescaled, only when a row's largest score has grown by
// more than 2^8 (weights stay below 2^8 and sums are f32, so that nothing is lost), which is rare after the first tile.
// Every wait on an mbarrier is bounded in time, as in dense_gemm.cuh.  Of a CTA that gives up, the rows that it still had to do come out as NaN.
#pragma once
#include "dense_gemm.cuh"
#include "paged_attn.cuh"

namespace lmrs {
namespace paged {

template <typename T, int DP> struct TensorShape {
    static constexpr int THREADS = 512, BLOCK = 128, BLOCKS = DP <= 128 ? 2 : 1, ROWS = BLOCK * BLOCKS, KEYS = DP <= 128 ? 128 : 64;
    static constexpr int BOXES = DP / 64;                                   // 64 columns of an operand: rows of 128 bytes, their 16-byte pieces rotated (SWIZZLE_128B)
    static constexpr int SLOT = BOXES * KEYS * 128, SLOTS = DP <= 64 ? 6 : 4, Q_BLOCK = BOXES * BLOCK * 128;
    static constexpr int RING = 8;                                          // tiles whose keys' places are known
    static constexpr int O_AT = DP <= 128 ? 256 : 256, S_WIDTH = 128;       // TMEM columns: two sets of scores, then o of each block
    static constexpr int SMEM = 1024 + SLOTS * SLOT + BLOCKS * Q_BLOCK;
    static_assert(O_AT + BLOCKS * DP <= 512 && 2 * S_WIDTH <= O_AT, "TMEM");
};
constexpr float RESCALE_AT = 8.0f;
constexpr int PAGED_WAIT = 5 << 8;   // (what a wait was for is not reported: any number that is not 0)

// A warp waits until phase number `count` of the barrier has ended (false: gave up).  One lane looks (9 warps of 32 looking lanes each filled the queue that copies to shared memory
// go through, and every one of those took ten times as long), under a predicate and not in a branch of its own: what follows a wait - accesses to TMEM, products,
// operands in uniform registers - is for a warp in step, and lanes that part here need not have met again by then.
PG_DEVINL bool wait_warp(uint64_t* bar, int count, volatile int* gave_up) {
    const uint32_t looks = (threadIdx.x & 31) == 0, at = smem_at(bar), parity = (uint32_t)count & 1;
    uint32_t from = 0;
    for (uint32_t i = 0;; i++) {
        uint32_t state;   // 1: ended, 2: give up
        asm volatile(
            "{\n\t.reg .pred p, l;\n\t"
            "setp.ne.b32 l, %3, 0;\n\t"
            "mov.u32 %0, 0;\n\t"
            "@l mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "@l selp.u32 %0, 1, 0, p;\n\t}"
            : "=&r"(state)
            : "r"(at), "r"(parity), "r"(looks)
            : "memory");
        const uint32_t now = dense::now_ns();
        if (i < dense::TG_LEAST_TRIES) from = now;
        if (state == 0 && (*gave_up || now - from > dense::TG_WAIT_NS)) state = 2;
        state = __shfl_sync(~0u, state, 0);
        if (state == 2) *gave_up = PAGED_WAIT;
        if (state) {
            __syncwarp();
            return state == 1;
        }
    }
}
PG_DEVINL void arrive(uint64_t* bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_at(bar)) : "memory"); }
PG_DEVINL void tmem_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
PG_DEVINL void tmem_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Loads and stores of TMEM are for a whole warp in step: where lanes may have gone different ways before (rows that are not there store nothing), they meet first.
// Loads are waited for in the same statement, so that no copy or spill of a register can come between.
PG_DEVINL void tmem_load32(uint32_t at, uint32_t (&v)[32]) {
    __syncwarp();
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
        "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]),
          "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]),
          "=r"(v[30]), "=r"(v[31])
        : "r"(at)
        : "memory");
}
PG_DEVINL void tmem_store32(uint32_t at, const uint32_t (&v)[32]) {
    __syncwarp();
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
        "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]),
        "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31]), "r"(at)
        : "memory");
}
PG_DEVINL void tmem_store16(uint32_t at, const uint32_t (&v)[16]) {
    __syncwarp();
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                 "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(at)
                 : "memory");
}
PG_DEVINL void tmem_stored() { __syncwarp(); asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// shared memory besides the operands
template <typename T, int DP> struct TensorShared {
    using S = TensorShape<T, DP>;
    uint64_t full[S::SLOTS], empty[S::SLOTS];   // slots
    uint64_t known[S::RING];                    // which of a tile's keys are there is written
    uint64_t scores[2], weights[2];             // sets of scores: written by the products, replaced by weights
    uint64_t summed[2], read[2];                // o of a block: the last product has ended; the part's o has been read
    uint64_t queries;                           // the part's queries are there
    uint64_t queries_read;                      // the last product that reads the part's queries has ended
    uint64_t parted;                            // both groups have ended the part (neither runs ahead: phases are told apart by their parity alone)
    uint32_t there[S::RING][S::KEYS / 32];
    int64_t starts[4][S::KEYS];                 // a copying warp's: where the keys' rows begin (elements; -1: nowhere)
    uint32_t tmem;
    int gave_up;
    AgainScratch again[2];
};

template <typename T, int DP>
__global__ void __launch_bounds__(512, 1) rows128_kernel(const __grid_constant__ AttnParams<T> p, const __grid_constant__ Line l) {
    using S = TensorShape<T, DP>;
    extern __shared__ uint8_t raw[];
    __shared__ TensorShared<T, DP> sh;
    uint8_t* ring = raw + (((smem_at(raw) + 1023u) & ~1023u) - smem_at(raw));   // (values of heads of up to 64 lie in one box: the next one's stride is never used)
    uint8_t* queries = ring + S::SLOTS * S::SLOT;
    const int warp = __shfl_sync(~0u, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31, D = p.head_size;
    volatile int* gave_up = &sh.gave_up;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S::SLOTS; i++) { mbar_init(&sh.full[i], 1); mbar_init(&sh.empty[i], 1); }
        for (int i = 0; i < S::RING; i++) mbar_init(&sh.known[i], 1);
        for (int i = 0; i < 2; i++) { mbar_init(&sh.scores[i], 1); mbar_init(&sh.weights[i], 128); mbar_init(&sh.summed[i], 1); mbar_init(&sh.read[i], 128); }
        mbar_init(&sh.queries, 128);
        mbar_init(&sh.queries_read, 1);
        mbar_init(&sh.parted, 256);
        sh.gave_up = 0;
        fence_barrier_init();
    }
    Walk w;
    int64_t from, to;
    walk_begin<T, S::THREADS>(p, l, w, from, to);   // (synchronises the CTA)
    if (from >= to) { grid_launch(); return; }
    if (warp == 12) {
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
    // (Every thread keeps its 128 registers.  Moved from the copying warps to the rows by setmaxnreg they were not safe: the compiler gave code of the copying warps
    // more than was left to them)
    if (warp >= 8) {
        if (warp < 12) {
            // ---- copies: operand tile n is warp n % 4's, which waits for its slot, copies, and reports it when it has landed; the other warps are at theirs ----
            const int mine = warp - 8, t = threadIdx.x - 256, pieces = (D + 15) / 16 * 2, whole = D / 8;
            int64_t* starts = sh.starts[mine];
            uint32_t n = 0;       // operand tiles of the CTA so far
            int looked = 0, part = 0;
            bool ok = true;
            bool asked = false;   // queries are on their way
            auto landed = [&]() {
                copy_wait<0>();
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                if (asked) arrive(&sh.queries);
                asked = false;
            };
            auto operand = [&](const T* base, bool values, int j) {   // tile j of the part; looked: its number in the CTA
                const uint32_t slot = n % S::SLOTS, round = n / S::SLOTS;
                if ((n++ & 3) != (uint32_t)mine || !ok) return;
                // the places of its keys, four a lane
                const int set = looked % S::RING;
                __syncwarp();
#pragma unroll
                for (int i = 0; i < S::KEYS / 32; i++) {
                    const Place at = unit_place(p, w, (w.tile + j) * S::KEYS + 32 * i + lane);
                    starts[32 * i + lane] = at.page < 0 ? -1
                                            : values    ? at.page * p.v_page + at.place * p.v_slot + w.head * p.v_head
                                                        : at.page * p.k_page + at.place * p.k_slot + w.head * p.k_head;
                    if (!values) {
                        const unsigned bits = __ballot_sync(~0u, at.page >= 0);
                        if (lane == 0) sh.there[set][i] = bits;
                    }
                }
                __syncwarp();
                if (!values && lane == 0) arrive(&sh.known[set]);
                ok = wait_warp(&sh.empty[slot], (int)round + 1, gave_up);
                if (!ok) return;
                const uint32_t at = smem_at(ring) + slot * S::SLOT;
                const int c = lane & 7;
#pragma unroll 1
                for (int r0 = lane >> 3; r0 < S::KEYS; r0 += 16) {   // (four rows' places are read before their copies are asked for)
                    const T* row[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int64_t start = starts[r0 + 4 * i];
                        row[i] = start < 0 ? nullptr : base + start + 8 * c;
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int r = r0 + 4 * i;
                        const uint32_t to_row = at + r * 128 + ((c ^ (r & 7)) << 4);
#pragma unroll
                        for (int b = 0; b < S::BOXES; b++)
                            if (8 * b + c < pieces) {
                                const bool in = row[i] && 8 * b + c < whole;
                                copy16(to_row + b * S::KEYS * 128, in ? row[i] + 64 * b : base, in);
                            }
                    }
                }
                copy_commit();
                landed();
                __syncwarp();
                if (lane == 0) arrive(&sh.full[slot]);
            };
            do {
                enter();
                if (part > 0) ok = ok && wait_warp(&sh.queries_read, part - 1, gave_up);
                if (ok) {   // the queries: eight threads a row; they are reported with the operand tile that follows
                    const int c = t & 7;
#pragma unroll 2
                    for (int x = t >> 3; x < blocks * S::BLOCK; x += 16) {
                        const UnitRow r = unit_row(p, l, w, x);
                        const T* q = r.row >= 0 ? p.q.data + r.row * p.q.row + r.head * p.q.head + 8 * c : p.q.data;
                        uint8_t* to_q = queries + (x >> 7) * S::Q_BLOCK + (x & 127) * 128 + ((c ^ (x & 7)) << 4);
#pragma unroll
                        for (int b = 0; b < S::BOXES; b++) {
                            if (8 * b + c >= pieces) continue;
                            const bool in = r.row >= 0 && 8 * b + c < whole;
                            if (p.q_wide) {
                                copy16(smem_at(to_q + b * (S::BLOCK * 128)), in ? q + 64 * b : p.q.data, in);
                            } else {
                                Piece<T, 8> v;
#pragma unroll
                                for (int i = 0; i < 8; i++) v.v[i] = in ? q[64 * b + i] : from_f<T>(0.0f);
                                *reinterpret_cast<Piece<T, 8>*>(to_q + b * (S::BLOCK * 128)) = v;
                            }
                        }
                    }
                    copy_commit();
                    asked = true;
                }
                const int first = looked;
                auto keys = [&](int j) { looked = first + j; operand(p.k, false, j); };
                keys(0);
                for (int j = 0; j < tiles; j++) {
                    if (j + 1 < tiles) keys(j + 1);
                    operand(p.v, true, j);
                }
                looked = first + tiles;
                if (asked) landed();   // (a warp that no operand tile fell to)
                part++;
            } while (leave());
        } else if (warp == 12) {
            // ---- products ----
            const uint32_t one = dense::elect_one(), type = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
            const uint32_t form = (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)(S::BLOCK >> 4) << 24);   // f32 += T x T, 128 rows
            const uint32_t score_form = form | ((uint32_t)(S::KEYS >> 3) << 17), sum_form = form | (1u << 16) | ((uint32_t)((D + 15) / 16 * 2) << 17);   // (values are MN-major)
            const uint32_t ring_lo = (uint32_t)dense::tg_desc_sw128(ring), q_lo = (uint32_t)dense::tg_desc_sw128(queries);
            const int steps = (D + 15) / 16;
            uint32_t n = 0, round = 0;           // slot of the next operand tile, rounds of the ring before it
            int w_count[2] = {0, 0}, part = 0;   // sets of weights taken
            bool ok = true;
            auto take = [&]() {
                ok = ok && wait_warp(&sh.full[n], (int)round, gave_up);
                tmem_after();
                const uint32_t slot = n;
                if (++n == S::SLOTS) { n = 0; round++; }
                return slot;
            };
            // (unrolled, so that descriptors are sums of constants in uniform registers: as a loop over k an issue took 96 cycles, three times the product)
            auto scores = [&](int block, int set, uint32_t slot) {
                const uint32_t d = tmem + (uint32_t)set * S::S_WIDTH, a = q_lo + (uint32_t)block * (S::Q_BLOCK >> 4), b = ring_lo + slot * (S::SLOT >> 4);
#pragma unroll
                for (int k = 0; k < DP / 16; k++)
                    if (k < steps)
                        dense::tg_mma_ss1(one, d, a + (uint32_t)(k >> 2) * (S::BLOCK * 128 >> 4) + (k & 3) * 2, b + (uint32_t)(k >> 2) * (S::KEYS * 128 >> 4) + (k & 3) * 2, score_form, k > 0);
                dense::tg_commit1(one, &sh.scores[set]);
            };
            auto sums = [&](int block, int set, int j, uint32_t slot) {
                if (j == 0 && part > 0) ok = ok && wait_warp(&sh.read[block], part - 1, gave_up);
                ok = ok && wait_warp(&sh.weights[set], w_count[set]++, gave_up);
                if (!ok) return;
                tmem_after();
                // 16 keys a step: two groups of 8 rows of 128 bytes; from 64 columns to the next: a box
                const uint32_t d = tmem + S::O_AT + (uint32_t)block * DP, a = tmem + (uint32_t)set * S::S_WIDTH;
                const uint32_t b = (ring_lo & 0xffffu) + slot * (S::SLOT >> 4) + ((uint32_t)(S::KEYS * 128 >> 4) << 16), more = j > 0;
#pragma unroll
                for (int k = 0; k < S::KEYS / 16; k++) dense::tg_mma_ts1(one, d, a + k * 8, b + k * (2048 >> 4), sum_form, k > 0 ? 1u : more);
                dense::tg_commit1(one, &sh.summed[block]);
            };
            do {   // operand tiles come as K0 K1 V0 K2 V1 ...
                enter();
                ok = ok && wait_warp(&sh.queries, part, gave_up);
                uint32_t slot = take();
                if (ok) {
                    scores(0, 0, slot);
                    if (blocks == 2) scores(1, 1, slot);
                    dense::tg_commit1(one, &sh.empty[slot]);
                }
                uint32_t next = tiles > 1 ? take() : 0;
                if (ok && blocks == 1 && tiles > 1) {
                    scores(0, 1, next);
                    dense::tg_commit1(one, &sh.empty[next]);
                }
                if (ok && (tiles == 1 || (blocks == 1 && tiles == 2))) dense::tg_commit1(one, &sh.queries_read);
                for (int j = 0; j < tiles && ok; j++) {
                    // one block: sums of tile j, then the scores of tile j + 2 into the same set; two: sums of a block, then its scores of tile j + 1
                    const uint32_t values = take();
                    if (!ok) break;
                    if (blocks == 1) {
                        sums(0, j & 1, j, values);
                        if (ok) dense::tg_commit1(one, &sh.empty[values]);
                        if (j + 2 < tiles) {
                            next = take();
                            if (ok) {
                                scores(0, j & 1, next);
                                dense::tg_commit1(one, &sh.empty[next]);
                                if (j + 3 == tiles) dense::tg_commit1(one, &sh.queries_read);
                            }
                        }
                    } else {
                        sums(0, 0, j, values);
                        if (ok && j + 1 < tiles) scores(0, 0, next);
                        sums(1, 1, j, values);
                        if (!ok) break;
                        dense::tg_commit1(one, &sh.empty[values]);
                        if (j + 1 < tiles) {
                            scores(1, 1, next);
                            dense::tg_commit1(one, &sh.empty[next]);
                            if (j + 2 == tiles) dense::tg_commit1(one, &sh.queries_read);
                        }
                        if (j + 2 < tiles) next = take();
                    }
                }
                part++;
            } while (ok && leave());
            // the last commit is that of the last values' slot: none may arrive after the CTA has ended
            if (ok) ok = wait_warp(&sh.empty[n == 0 ? S::SLOTS - 1 : n - 1], (int)(n == 0 ? round - 1 : round), gave_up);
            if (!ok)   // gave up: products already issued may still run; they get a millisecond to end before shared memory and TMEM go away
                for (int i = 0; i < 1000; i++) __nanosleep(1000);
        }
        __syncwarp();
    } else {
        // ---- rows ----
        const int group = warp >> 2, row = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;   // this warp's 32 TMEM lanes
        int s_count[2] = {0, 0}, k_count = 0, o_count = 0, part = 0;   // phases of earlier parts: sets of scores, tiles, sums of o, parts
        bool ok = true;
        do {
            enter();
            const bool mine = group < blocks;
            const int x = group * S::BLOCK + row;
            if (mine) {
                const UnitRow r = unit_row(p, l, w, x);
                float m = -INFINITY, sum = 0.0f;
                bool seen = false;
                const int least = w.b < 0 ? w.keys : unit_row(p, l, w, group * S::BLOCK).keys;   // (rows that come later see more)
                for (int j = 0; j < tiles && ok; j++) {
                    const int set = blocks == 2 ? group : j & 1, key0 = (w.tile + j) * S::KEYS, known = (k_count + j) % S::RING;
                    ok = wait_warp(&sh.known[known], (k_count + j) / S::RING, gave_up) && wait_warp(&sh.scores[set], s_count[set] + (blocks == 2 ? j : j >> 1), gave_up);
                    if (!ok) break;
                    tmem_after();
                    const uint32_t at = tmem + lanes + (uint32_t)set * S::S_WIDTH;
                    bool all = key0 + S::KEYS <= least;
#pragma unroll
                    for (int c = 0; c < S::KEYS / 32; c++) all = all && sh.there[known][c] == ~0u;
                    auto sees = [&](int c) {   // bit i: the row sees key 32 c + i of the tile
                        const int limit = r.keys - key0 - 32 * c;
                        return sh.there[known][c] & (limit >= 32 ? ~0u : limit <= 0 ? 0u : (1u << limit) - 1);
                    };
                    // The scores are read twice, for the largest and for the weights: 128 of them in registers leave no room for anything else (700 bytes of spills).  A score
                    // rises with its dot (falls, with a negative factor): the largest dot makes the largest score
                    float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int c = 0; c < S::KEYS / 32; c++) {
                        uint32_t v[32];
                        tmem_load32(at + 32 * c, v);
                        if (p.scale2 < 0.0f) {
#pragma unroll
                            for (int i = 0; i < 32; i++) v[i] ^= 0x80000000u;
                        }
                        if (!all) {
                            const uint32_t mask = sees(c);
                            seen = seen || mask;
#pragma unroll
                            for (int i = 0; i < 32; i++)
                                if (!(mask >> i & 1)) v[i] = 0xff800000u;
                        }
#pragma unroll
                        for (int i = 0; i < 32; i += 2) tops[i >> 1 & 3] = fmaxf(fmaxf(tops[i >> 1 & 3], __uint_as_float(v[i])), __uint_as_float(v[i + 1]));
                    }
                    seen = seen || all;
                    float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                    if (top != -INFINITY) top = score2(p, p.scale2 < 0.0f ? -top : top);
                    top -= WEIGHT_SHIFT<T>;
                    if (__any_sync(~0u, top > m + RESCALE_AT || (m == -INFINITY && top > m))) {
                        const float now = fmaxf(m, top), corr = ex2(m - (now == -INFINITY ? 0.0f : now));
                        if (j > 0) {
                            ok = wait_warp(&sh.summed[group], o_count + j - 1, gave_up);
                            if (!ok) break;
                            tmem_after();
#pragma unroll 1
                            for (int c = 0; c < D; c += 32) {
                                uint32_t o[32];
                                const uint32_t o_at = tmem + lanes + S::O_AT + (uint32_t)group * DP + c;
                                tmem_load32(o_at, o);
#pragma unroll
                                for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
                                tmem_store32(o_at, o);
                            }
                            tmem_stored();
                        }
                        sum *= corr;
                        m = now;
                    }
                    const float base = m == -INFINITY ? 0.0f : m;
                    float2 part_sums[2] = {};
#pragma unroll
                    for (int c = 0; c < S::KEYS / 32; c++) {
                        uint32_t v[32], a[16];
                        tmem_load32(at + 32 * c, v);
                        float e[32];
                        if (p.softcap > 0.0f) {
#pragma unroll
                            for (int i = 0; i < 32; i++) e[i] = __uint_as_float(v[i]);
                            cap_scores(p, e);
#pragma unroll
                            for (int i = 0; i < 32; i++) e[i] = ex2(e[i] - base);
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; i++) e[i] = ex2(fmaf(__uint_as_float(v[i]), p.scale2, -base));
                        }
                        if (!all) {
                            const uint32_t mask = sees(c);
#pragma unroll
                            for (int i = 0; i < 32; i++)
                                if (!(mask >> i & 1)) e[i] = 0.0f;
                        }
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            part_sums[i & 1].x += e[2 * i];
                            part_sums[i & 1].y += e[2 * i + 1];
                            a[i] = close_word(make_float2(e[2 * i], e[2 * i + 1]), T());
                        }
                        tmem_store16(at + 16 * c, a);   // (over scores that have been read: these 16 columns hold those of tile columns below 32 c + 32)
                    }
                    sum += (part_sums[0].x + part_sums[0].y) + (part_sums[1].x + part_sums[1].y);
                    tmem_stored();
                    tmem_before();
                    arrive(&sh.weights[set]);
                }
                // the part's rows
                const int64_t slot = w.unit + blockIdx.x;
                const bool whole = whole_unit(p, w, w.tile, w.tile + tiles - 1), is = x < used;
                ok = ok && wait_warp(&sh.summed[group], o_count + tiles - 1, gave_up);
                bool again = false;
                if (ok) {
                    tmem_after();
                    if (!seen) sum = -1.0f;
                    bool finite = true;
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        uint32_t o[32];
                        tmem_load32(tmem + lanes + S::O_AT + (uint32_t)group * DP + c, o);
                        if (!seen) {
#pragma unroll
                            for (int i = 0; i < 32; i++) o[i] = 0;
                        }
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            if (c + i >= D) continue;
                            float4 f = make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]), __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
                            finite = finite && isfinite(f.x + f.y + f.z + f.w);
                            if (!is) continue;
                            if (whole) {
                                if (seen) { f.x /= sum; f.y /= sum; f.z /= sum; f.w /= sum; }
                                store_row(p, r, c + i, f);
                            } else if (slot < l.slots) {
                                *reinterpret_cast<float4*>(part_at(l, D, slot, x, c + i)) = f;
                            }
                        }
                    }
                    if (is) {
                        if (whole) { if (p.lse) p.lse[r.row * p.q_heads + r.head] = seen ? lse_of(m, sum) : -INFINITY; }
                        else if (slot < l.slots) l.ml[slot * S::ROWS + x] = make_float2(m, sum);
                    }
                    tmem_before();
                    arrive(&sh.read[group]);
                    again = is && seen && !finite && w.b >= 0 && w.s.count > 1;   // other rows' keys may have spoiled it
                } else if (is) {   // gave up: NaN
                    if (whole) {
                        for (int c = 0; c < D; c++) p.out.data[r.row * p.out.row + r.head * p.out.head + c] = from_f<T>(NAN);
                        if (p.lse) p.lse[r.row * p.q_heads + r.head] = NAN;
                    } else if (slot < l.slots) {
                        l.ml[slot * S::ROWS + x] = make_float2(NAN, NAN);
                    }
                }
                int* flags = reinterpret_cast<int*>(sh.again[group].weight);
                again_sync(1 + group);
                flags[row] = again;
                again_sync(1 + group);
                unsigned todo[4], any = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) any |= todo[i] = __ballot_sync(~0u, flags[32 * i + lane]);
                if (any) {
                    again_sync(1 + group);   // (the flags' place is used below)
#pragma unroll 1
                    for (int i = 0; i < S::BLOCK; i++) {
                        if (!((i < 32 ? todo[0] : i < 64 ? todo[1] : i < 96 ? todo[2] : todo[3]) >> (i & 31) & 1)) continue;
                        const UnitRow r2 = unit_row(p, l, w, group * S::BLOCK + i);
                        float m2, l2, acc[2];
                        row_again(p, w, r2, w.tile * S::KEYS, (w.tile + tiles) * S::KEYS, sh.again[group], 1 + group, m2, l2, acc);
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            const int c = row + AGAIN * k;
                            if (c >= D) continue;
                            if (whole) p.out.data[r2.row * p.out.row + r2.head * p.out.head + c] = from_f<T>(acc[k] / l2);
                            else if (slot < l.slots) *part_at(l, D, slot, group * S::BLOCK + i, c) = acc[k];
                        }
                        if (row == 0) {
                            if (whole) { if (p.lse) p.lse[r2.row * p.q_heads + r2.head] = lse_of(m2, l2); }
                            else if (slot < l.slots) l.ml[slot * S::ROWS + group * S::BLOCK + i] = make_float2(m2, l2);
                        }
                    }
                }
                o_count += tiles;
            } else {
                arrive(&sh.read[1]);   // (a part without a second block: its turn passes)
            }
            k_count += tiles;
            s_count[0] += blocks == 2 ? tiles : (tiles + 1) >> 1;
            s_count[1] += blocks == 2 ? tiles : tiles >> 1;
            arrive(&sh.parted);
            ok = ok && wait_warp(&sh.parted, part++, gave_up);
        } while (leave());
    }
    tmem_before();
    __syncthreads();
    if (warp == 12) {
        __syncwarp();
        tmem_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
    }
}

}  // namespace paged
}  // namespace lmrs
