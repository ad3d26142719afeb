// paged_tensor.cuh -- the same attention for many rows that see the same keys (the prefix, which all rows of a call share; portions of prompts), on the 5th-generation
// tensor cores.  16-bit types; the line, its units and the parts are those of paged_attn.cuh, with 128 or 256 rows a unit.
//
// CTA = 12 warps of 168 registers, one CTA an SM.  The rows of a unit are one or two blocks of 128, a TMEM lane each; a step of the work is one block against one tile of keys:
//     scores = Q . K^T            tcgen05.mma, both operands in shared memory, 128 x 64 sums in TMEM (two sets for each block, taken in turn)
//     weights = 2^(scores - m)    a thread a row: the scores from TMEM, the weights rounded to the type and back to TMEM over the scores
//     o += weights . V            tcgen05.mma, the weights from TMEM, the values in shared memory as they lie in the pages (keys x columns: MN-major)
//   warps 0-3, 4-7   the rows of the first and the second block.  The scores of the next tile are computed under the exponentials of this one.
//   warps 8-9        copies of keys and values into a ring of slots, one operand tile each, in the order K0 K1 V0 K2 V1 ...  By TMA, a piece of a page at a time; a unit's last tile, and all
//                    where pages have odd sizes, 16 bytes a thread with zeros for what is not there.  The places of a tile's keys are looked up by a thread each.
//   warp 10          the products
// o stays in TMEM for a whole part.  m is the largest score when it was last set; it is set anew, and o rescaled, only when a row's largest score has grown by
// more than 2^8 (weights stay below 2^8, fp16's below 2^15, and sums are f32, so that nothing is lost), which is rare after the first tile.
// Measured on a B200, us: 512 rows of a KV head behind 32768 keys, 8 KV heads of 128, bf16: 110 (620 TFLOP/s; a library product reaches 1690).  256 rows behind
// 8200, heads of 64: 28.  Rows of 12 prompts behind 2050, heads of 256, capped: 270 (the cap's tanh and one block of rows only).  What bounds it: no unit is half busy (tensor
// cores 39 %, powers of two 29 %, issue slots 28 %, DRAM 16 %); it is the chain scores - TMEM - maximum - powers - TMEM - sums of a tile, two tiles of each block under way.
// 64 keys a tile with two sets of scores: the scores of the next tile under the powers of this one.  (128 keys with one set / this, when it was changed:
// 215 / 213 for 128 sequences behind 32768 with their own keys, 538 / 431 for the capped prompts.)
// Keys by TMA boxes and by cp.async: 174 / 292, 67 / 87 and 312 / 515 for the three with their own keys.
// Every wait on an mbarrier is bounded in time, as in dense_gemm.cuh.  Of a CTA that gives up, the rows that it still had to do come out as NaN, and the next call says so (GaveUpWord).
#pragma once
#include <atomic>
#include <mutex>

#include "dense_gemm.cuh"
#include "paged_attn.cuh"

namespace lmrs {
namespace paged {

template <typename T, int DP> struct TensorShape {
    static constexpr int THREADS = 384, COPIERS = 2, BLOCK = 128, BLOCKS = DP <= 128 ? 2 : 1, ROWS = BLOCK * BLOCKS, KEYS = 64;
    static constexpr int BOXES = DP / 64;                                   // 64 columns of an operand: rows of 128 bytes, their 16-byte pieces rotated (SWIZZLE_128B)
    static constexpr int SLOT = BOXES * KEYS * 128, SLOTS = DP <= 128 ? 8 : 4, Q_BLOCK = BOXES * BLOCK * 128;
    static constexpr int RING = 8;                                          // tiles whose keys' places are known
    static constexpr int O_AT = 256;                                        // TMEM columns: two sets of scores for each block, then o of each block
    static constexpr int SMEM = 1024 + SLOTS * SLOT + BLOCKS * Q_BLOCK;
    static_assert(O_AT + BLOCKS * DP <= 512 && 2 * 2 * KEYS <= O_AT, "TMEM");
};
constexpr float RESCALE_AT = 8.0f;

// A warp waits until phase number `count` of the barrier has ended (false: gave up).  All lanes look: a look suspends whoever looks, so that a lane which looks for the
// others parts from them, and what follows a wait - accesses to TMEM, products, operands in uniform registers - is for a warp in step.
PG_DEVINL bool wait_warp(uint64_t* bar, int count, volatile int* gave_up, int what) {
    const bool ok = __all_sync(~0u, dense::mbar_wait_bounded(bar, (uint32_t)count & 1, gave_up, dense::TG_PAGED + what));
    __syncwarp();
    return ok;
}
// The same for what comes once a part, however long the part is: the limit begins anew whenever `flips`, a barrier that goes on with the part's tiles, is seen in another phase
PG_DEVINL bool wait_part_lane(uint64_t* bar, uint32_t parity, uint64_t* flips, volatile int* gave_up) {
    uint32_t from = dense::now_ns();
    bool phase = dense::mbar_test(flips, 0);
    for (uint32_t i = 0;; i++) {   // (each try suspends for a while)
        if (mbar_try_wait(bar, parity)) return true;
        if (*gave_up) return false;
        const bool now = dense::mbar_test(flips, 0);
        if (now != phase) { phase = now; from = dense::now_ns(); i = 0; }
        else if (i >= dense::TG_LEAST_TRIES && dense::now_ns() - from >= dense::TG_WAIT_NS) break;
    }
    if (!*gave_up) *gave_up = dense::TG_PAGED + dense::TG_PART;
    return false;
}
PG_DEVINL bool wait_part(uint64_t* bar, int count, uint64_t* flips, volatile int* gave_up) {
    const bool ok = __all_sync(~0u, wait_part_lane(bar, (uint32_t)count & 1, flips, gave_up));
    __syncwarp();
    return ok;
}
// has the phase ended?
PG_DEVINL bool looks_free(uint64_t* bar, int count) { return __all_sync(~0u, dense::mbar_test(bar, (uint32_t)count & 1)); }
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
PG_DEVINL void tmem_load64(uint32_t at, uint32_t (&v)[64]) {
    __syncwarp();
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
        "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%64];\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
        "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
        "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%65];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]),
          "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]),
          "=r"(v[30]), "=r"(v[31]), "=r"(v[32]), "=r"(v[33]), "=r"(v[34]), "=r"(v[35]), "=r"(v[36]), "=r"(v[37]), "=r"(v[38]), "=r"(v[39]),
          "=r"(v[40]), "=r"(v[41]), "=r"(v[42]), "=r"(v[43]), "=r"(v[44]), "=r"(v[45]), "=r"(v[46]), "=r"(v[47]), "=r"(v[48]), "=r"(v[49]),
          "=r"(v[50]), "=r"(v[51]), "=r"(v[52]), "=r"(v[53]), "=r"(v[54]), "=r"(v[55]), "=r"(v[56]), "=r"(v[57]), "=r"(v[58]), "=r"(v[59]),
          "=r"(v[60]), "=r"(v[61]), "=r"(v[62]), "=r"(v[63])
        : "r"(at), "r"(at + 32)
        : "memory");
}
PG_DEVINL void tmem_load16(uint32_t at, uint32_t (&v)[16]) {
    __syncwarp();
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
          "=r"(v[14]), "=r"(v[15])
        : "r"(at)
        : "memory");
}
PG_DEVINL void tmem_store8(uint32_t at, const uint32_t (&v)[8]) {
    __syncwarp();
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]),
                 "r"(v[7]), "r"(at)
                 : "memory");
}
// two floats in one register pair
PG_DEVINL uint64_t pair_of(uint32_t a, uint32_t b) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(a), "r"(b)); return r; }
PG_DEVINL float2 pair_open(uint64_t v) { float2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v)); return r; }
PG_DEVINL uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) { uint64_t r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
PG_DEVINL uint64_t add_pair(uint64_t a, uint64_t b) { uint64_t r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
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
PG_DEVINL void tmem_stored() { __syncwarp(); asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Where a kernel that gave up says so: a word of the process in mapped host memory, which the next call reads
struct GaveUpWord {
    std::atomic<int*> at{nullptr};
    std::mutex making;
    int* get() {   // null: there is no memory for it
        if (int* p = at.load(std::memory_order_acquire)) return p;
        std::lock_guard<std::mutex> hold(making);
        if (int* p = at.load(std::memory_order_acquire)) return p;
        void* p = nullptr;
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;   // (the call may be captured; this is not part of it)
        cudaThreadExchangeStreamCaptureMode(&mode);
        const cudaError_t e = cudaHostAlloc(&p, sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped);   // (the same address on every device)
        cudaThreadExchangeStreamCaptureMode(&mode);
        if (e != cudaSuccess) { cudaGetLastError(); return nullptr; }
        *(int*)p = 0;
        at.store((int*)p, std::memory_order_release);
        return (int*)p;
    }
    int take() {   // what a kernel has written, once
        int* p = at.load(std::memory_order_acquire);
        return p && *(volatile int*)p ? __atomic_exchange_n(p, 0, __ATOMIC_ACQ_REL) : 0;
    }
};
inline GaveUpWord gave_up_word;   // (one for the process)

// shared memory besides the operands
template <typename T, int DP> struct TensorShared {
    using S = TensorShape<T, DP>;
    uint64_t full[S::SLOTS], empty[S::SLOTS];   // slots
    uint64_t known[S::RING];                    // which of a tile's keys are there is written
    uint64_t scores[4], weights[4];             // sets of scores (two for each block): written by the products, replaced by weights
    uint64_t summed[4];                         // o of a block: the products of a tile have ended, even tiles and odd ones (rows may be two tiles ahead of the products, and a phase
                                                // is told from the one before it only)
    uint64_t read[2];                           // the part's o of a block has been read
    uint64_t queries;                           // the part's queries are there
    uint64_t queries_read;                      // the last product that reads the part's queries has ended
    uint64_t parted;                            // both groups have ended the part (neither runs ahead: phases are told apart by their parity alone)
    uint32_t there[S::RING][S::KEYS / 32];
    int64_t starts[S::COPIERS][S::KEYS / S::COPIERS];             // a copying warp's: where the rows that it copies begin (bytes; -1: nowhere)
    uint32_t tmem;
    int gave_up;
    bool spoiled;                               // some row of some part is not finite where other rows' keys may be why
    Walk start;                                 // where the CTA begins, and how many tiles it has
    int tiles;
    AgainScratch again[2];
};

// How the copies of whole tiles go: `rows` keys of a page at a time by TMA (0: never; pages of odd sizes, or strides that no tensor map takes).  The maps' dimensions are a
// row's bytes and then, by falling nearness in memory, places, heads and pages: which of the three is which
struct Boxes {
    CUtensorMap k, v, q;
    int rows, k_place, k_head, v_place, v_head;   // dimension (0, 1, 2) of the place and the head; the page has the third
    int q_tokens;                                 // the same for queries: tokens that make up a block's rows (0: the group of a KV head does not divide them)
};
PG_DEVINL void tma_box(uint32_t to, const CUtensorMap* map, int x, int place, int head, int page, int place_at, int head_at, uint64_t* bar) {
    const int a = place_at == 0 ? place : head_at == 0 ? head : page, b = place_at == 1 ? place : head_at == 1 ? head : page, c = place_at == 2 ? place : head_at == 2 ? head : page;
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(to), "l"(map), "r"(x), "r"(a), "r"(b), "r"(c),
                 "r"(smem_at(bar))
                 : "memory");
}

template <typename T, int DP>
__global__ void __launch_bounds__(384, 1) rows128_kernel(const __grid_constant__ AttnParams<T> p, const __grid_constant__ Line l, const __grid_constant__ Boxes boxes) {
    using S = TensorShape<T, DP>;
    extern __shared__ uint8_t raw[];
    __shared__ TensorShared<T, DP> sh;
    uint8_t* ring = raw + (((smem_at(raw) + 1023u) & ~1023u) - smem_at(raw));   // (values of heads of up to 64 lie in one box: the next one's stride is never used)
    uint8_t* queries = ring + S::SLOTS * S::SLOT;
    const int warp = __shfl_sync(~0u, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31, D = p.head_size;
    constexpr int PRODUCTS = 8 + S::COPIERS;   // the warp that issues them
    volatile int* gave_up = &sh.gave_up;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S::SLOTS; i++) { mbar_init(&sh.full[i], S::COPIERS); mbar_init(&sh.empty[i], 1); }
        for (int i = 0; i < S::RING; i++) mbar_init(&sh.known[i], S::COPIERS);
        for (int i = 0; i < 4; i++) { mbar_init(&sh.scores[i], 1); mbar_init(&sh.weights[i], 128); mbar_init(&sh.summed[i], 1); }
        for (int i = 0; i < 2; i++) mbar_init(&sh.read[i], 128);
        mbar_init(&sh.queries, boxes.q_tokens ? 1 : 32 * S::COPIERS);
        mbar_init(&sh.queries_read, 1);
        mbar_init(&sh.parted, 256);
        sh.gave_up = 0;
        sh.spoiled = false;
        fence_barrier_init();
    }
    Walk w;
    int64_t from, to;
    walk_begin<T, S::THREADS>(p, l, w, from, to);   // (synchronises the CTA)
    if (from >= to) { grid_launch(); return; }
    if (threadIdx.x == 0) { sh.start = w; sh.tiles = (int)(to - from); }
    if (warp == PRODUCTS) {
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
    // (Every thread keeps its registers.  Versions that moved some from the copying warps to the rows by setmaxnreg faulted, and had other faults as well; nothing shows that the compiler keeps code
    // that follows below the number that is left, so it stays out)
    if (warp >= 8) {
        if (warp < 8 + S::COPIERS) {
            // ---- copies: each of the two warps half of every operand tile's rows, as far ahead as slots are free ----
            constexpr int SHARE = S::KEYS / S::COPIERS, EACH = SHARE / 32;   // rows a warp copies, a lane looks up
            const int mine = warp - 8, t = threadIdx.x - 256, pieces = (D + 15) / 16 * 2, whole = D / 8, c = lane & 7;
            int64_t* starts = sh.starts[mine];
            // a box a lane: piece of a page x 64 columns (one lane for all of them, with the places passed to it: 189 us instead of 176 for 128 sequences behind 32768 tokens)
            static_assert(EACH == 1, "a lane has the place of its row");
            const int wide = (D + 63) / 64, box_row = boxes.rows ? lane / wide * boxes.rows : SHARE, box_col = lane % wide;
            const uint32_t box_to = smem_at(ring) + mine * SHARE * 128 + box_col * S::KEYS * 128 + box_row * 128;
            uint32_t n = 0, slot = 0, round = 0, reported = 0, report_slot = 0;   // operand tiles asked for, the next one's slot and round of the ring; those reported, and the next of these
            int looked = 0, part = 0;
            bool ok = true, asked = false;   // asked: queries are on their way
            auto report = [&](uint32_t upto) {   // (they have landed)
                if (upto == reported) return;   // (a fence costs a thousand cycles)
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                if (asked && upto > reported) { arrive(&sh.queries); asked = false; }
                __syncwarp();
                for (; reported < upto; reported++) {
                    if (lane == 0) arrive(&sh.full[report_slot]);
                    report_slot = report_slot + 1 == S::SLOTS ? 0 : report_slot + 1;
                }
            };
            auto next_slot = [&]() {
                n++;
                if (++slot == S::SLOTS) { slot = 0; round++; }
            };
            // an operand tile: lane's rows lane, lane + 32 of the warp's lie at `place`.  boxed: all of the tile's keys are within the unit's
            auto operand = [&](bool values, const Place (&place)[EACH], bool boxed) {
                if (!ok) return;
                if (!looks_free(&sh.empty[slot], (int)round + 1)) {   // (nothing that has landed waits for a slot to come free)
                    copy_wait<0>();
                    report(n);
                    ok = wait_warp(&sh.empty[slot], (int)round + 1, gave_up, dense::TG_FREE);
                    if (!ok) return;
                }
                if (boxed) {
                    // (tiles by TMA report themselves; no other one is on its way)
                    if (lane == 0) mbar_expect_tx(&sh.full[slot], (uint32_t)(SHARE * 128 * ((D + 63) / 64)));
                    int page = __shfl_sync(~0u, place[0].page, box_row & 31), at_place = __shfl_sync(~0u, place[0].place, box_row & 31);
                    if (page < 0) { page = p.batch.pages; at_place = 0; }   // (outside the map: zeros)
                    if (box_row < SHARE)
                        tma_box(box_to + slot * S::SLOT, values ? &boxes.v : &boxes.k, 128 * box_col, at_place, w.head, page, values ? boxes.v_place : boxes.k_place,
                                values ? boxes.v_head : boxes.k_head, &sh.full[slot]);
                    __syncwarp();
                    next_slot();
                    reported = n;
                    report_slot = slot;
                    if (asked) {   // (the queries' copies are the only ones of the other kind)
                        copy_wait<0>();
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        arrive(&sh.queries);
                        asked = false;
                    }
                    return;
                }
                const T* base = values ? p.v : p.k;
                int64_t start[EACH];
#pragma unroll
                for (int i = 0; i < EACH; i++)
                    start[i] = place[i].page < 0 ? -1
                                                 : (values ? place[i].page * p.v_page + place[i].place * p.v_slot + w.head * p.v_head
                                                           : place[i].page * p.k_page + place[i].place * p.k_slot + w.head * p.k_head) * (int64_t)sizeof(T);
                __syncwarp();
#pragma unroll
                for (int i = 0; i < EACH; i++) starts[32 * i + lane] = start[i];
                __syncwarp();
                const uint32_t at = smem_at(ring) + slot * S::SLOT + (mine * SHARE + (lane >> 3)) * 128;
                const char* from = reinterpret_cast<const char*>(base) + 16 * c;
#pragma unroll 1
                for (int i0 = 0; i0 < SHARE / 4; i0 += 8) {   // (eight rows a lane: their places are read before their copies are asked for)
                    int64_t rows[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) rows[i] = starts[4 * (i0 + i) + (lane >> 3)];
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const uint32_t to_row = at + (i0 + i) * 512 + ((c ^ ((4 * i + (lane >> 3)) & 7)) << 4);
                        if (whole == DP / 8) {
                            const char* row = from + (rows[i] < 0 ? 0 : rows[i]);
#pragma unroll
                            for (int b = 0; b < S::BOXES; b++) copy16(to_row + b * S::KEYS * 128, row + 128 * b, rows[i] >= 0);
                        } else {
#pragma unroll
                            for (int b = 0; b < S::BOXES; b++)
                                if (8 * b + c < pieces) {
                                    const bool in = rows[i] >= 0 && 8 * b + c < whole;
                                    copy16(to_row + b * S::KEYS * 128, in ? from + rows[i] + 128 * b : reinterpret_cast<const char*>(base), in);
                                }
                        }
                    }
                }
                copy_commit();
                next_slot();
                if (boxes.rows) {   // (a unit's last tile)
                    copy_wait<0>();
                    report(n);
                } else {
                    copy_wait<2>();
                    if (n > 2) report(n - 2);
                }
            };
            do {
                enter();
                if (part > 0) ok = ok && wait_warp(&sh.queries_read, part - 1, gave_up, dense::TG_QUERIES_READ);
                if (ok && boxes.q_tokens) {   // the queries: rows are tokens x the heads of a group, which one box holds (rows behind the unit's own are some others', or zeros)
                    if (mine == 0 && lane == 0) {
                        const int token = (int)(w.b < 0 ? 0 : w.s.first) + w.row_tile * S::ROWS / p.group;
                        mbar_expect_tx(&sh.queries, (uint32_t)(blocks * S::BLOCK * 128 * ((D + 63) / 64)));
                        for (int block = 0; block < blocks; block++)
                            for (int b = 0; 64 * b < D; b++)
                                asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                                                 smem_at(queries) + block * S::Q_BLOCK + b * (S::BLOCK * 128)),
                                             "l"(&boxes.q), "r"(128 * b), "r"(w.head * p.group), "r"(token + block * boxes.q_tokens), "r"(smem_at(&sh.queries))
                                             : "memory");
                    }
                    __syncwarp();
                } else if (ok) {   // eight threads a row; they are reported with the operand tile that follows
                    constexpr int AT_ONCE = 4 * S::COPIERS;
                    const int x0 = t >> 3, i0 = w.row_tile * S::ROWS + x0, step = AT_ONCE / p.group, more = AT_ONCE - step * p.group;
                    int token = i0 / p.group, g = i0 - token * p.group;
#pragma unroll 4
                    for (int x = x0; x < blocks * S::BLOCK; x += AT_ONCE) {
                        const bool is = x < used;
                        const T* q = is ? p.q.data + ((w.b < 0 ? 0 : w.s.first) + token) * p.q.row + (w.head * p.group + g) * p.q.head + 8 * c : p.q.data;
                        token += step;
                        g += more;
                        if (g >= p.group) { g -= p.group; token++; }
                        uint8_t* to_q = queries + (x >> 7) * S::Q_BLOCK + (x & 127) * 128 + ((c ^ (x & 7)) << 4);
#pragma unroll
                        for (int b = 0; b < S::BOXES; b++) {
                            if (8 * b + c >= pieces) continue;
                            const bool in = is && 8 * b + c < whole;
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
                    copy_commit();   // a group of their own: the wait for them may come before any operand tile by cp.async has made one
                    __syncwarp();
                    asked = true;
                }
                Place at[EACH], next[EACH];   // of the keys of tiles j and j + 1
                auto whole_tile = [&](int j) { return boxes.rows > 0 && (w.tile + j + 1) * S::KEYS <= w.keys; };
                auto keys = [&](int j) {   // tile j of the part: where its keys and values lie, and which are there; then the keys
                    const int set = looked++ % S::RING;
#pragma unroll
                    for (int i = 0; i < EACH; i++) {
                        next[i] = unit_place(p, w, (w.tile + j) * S::KEYS + mine * SHARE + 32 * i + lane);
                        const unsigned bits = __ballot_sync(~0u, next[i].page >= 0);
                        if (lane == 0) sh.there[set][mine * EACH + i] = bits;
                    }
                    if (lane == 0 && ok) arrive(&sh.known[set]);
                    operand(false, next, whole_tile(j));
                };
                keys(0);
                for (int j = 0; j < tiles; j++) {
#pragma unroll
                    for (int i = 0; i < EACH; i++) at[i] = next[i];
                    if (j + 1 < tiles) keys(j + 1);
                    operand(true, at, whole_tile(j));
                }
                copy_wait<0>();   // (the next part waits for the queries' last reader, which needs all of this one)
                report(n);
                part++;
            } while (leave());
            if (!ok && boxes.q_tokens) dense::mbar_wait_for(&sh.queries, (part - 1) & 1, nullptr);
            if (!ok)   // gave up: what TMA was asked for lands before shared memory goes away
                for (uint32_t i = n > S::SLOTS ? n - S::SLOTS : 0; i < n; i++) dense::mbar_wait_for(&sh.full[i % S::SLOTS], (i / S::SLOTS) & 1, nullptr);
        } else if (warp == PRODUCTS) {
            // ---- products ----
            const uint32_t one = dense::elect_one(), type = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
            const uint32_t form = (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)(S::BLOCK >> 4) << 24);   // f32 += T x T, 128 rows
            const uint32_t score_form = form | ((uint32_t)(S::KEYS >> 3) << 17), sum_form = form | (1u << 16) | ((uint32_t)((D + 15) / 16 * 2) << 17);   // (values are MN-major)
            const uint32_t ring_lo = (uint32_t)dense::tg_desc_sw128(ring), q_lo = (uint32_t)dense::tg_desc_sw128(queries);
            const int steps = (D + 15) / 16;
            uint32_t n = 0, round = 0;           // slot of the next operand tile, rounds of the ring before it
            int w_count[4] = {0, 0, 0, 0}, part = 0;   // sets of weights taken
            bool ok = true;
            auto take = [&]() {
                ok = ok && wait_warp(&sh.full[n], (int)round, gave_up, dense::TG_FULL);
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
                if (j == 0 && part > 0) ok = ok && wait_warp(&sh.read[block], part - 1, gave_up, dense::TG_VALUES_READ);
                ok = ok && wait_warp(&sh.weights[set], w_count[set]++, gave_up, dense::TG_WEIGHTS);
                if (!ok) return;
                tmem_after();
                // 16 keys a step: two groups of 8 rows of 128 bytes; from 64 columns to the next: a box
                const uint32_t d = tmem + S::O_AT + (uint32_t)block * DP, a = tmem + (uint32_t)set * S::KEYS;
                const uint32_t b = (ring_lo & 0xffffu) + slot * (S::SLOT >> 4) + ((uint32_t)(S::KEYS * 128 >> 4) << 16), more = j > 0;
#pragma unroll
                for (int k = 0; k < S::KEYS / 16; k++) dense::tg_mma_ts1(one, d, a + k * 8, b + k * (2048 >> 4), sum_form, k > 0 ? 1u : more);
                dense::tg_commit1(one, &sh.summed[set]);
            };
            do {   // operand tiles come as K0 K1 V0 K2 V1 ...: the scores of tile j + 2 follow the sums of tile j into the same set
                enter();
                ok = ok && wait_warp(&sh.queries, part, gave_up, dense::TG_QUERIES);
                for (int j = 0; j < 2 && j < tiles; j++) {
                    const uint32_t keys = take();
                    if (!ok) break;
                    for (int g = 0; g < blocks; g++) scores(g, j, keys);
                    dense::tg_commit1(one, &sh.empty[keys]);
                }
                if (ok && tiles <= 2) dense::tg_commit1(one, &sh.queries_read);
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
                    if (ok && j + 2 < tiles) {
                        dense::tg_commit1(one, &sh.empty[keys]);
                        if (j + 3 == tiles) dense::tg_commit1(one, &sh.queries_read);
                    }
                }
                part++;
            } while (ok && leave());
            // the last commit is that of the last values' slot: none may arrive after the CTA has ended
            if (ok) ok = wait_warp(&sh.empty[n == 0 ? S::SLOTS - 1 : n - 1], (int)(n == 0 ? round - 1 : round), gave_up, dense::TG_FREE);
            if (!ok)   // gave up: products already issued may still run; they get a millisecond to end before shared memory and TMEM go away
                for (int i = 0; i < 1000; i++) __nanosleep(1000);
        }
        __syncwarp();
    } else {
        // ---- rows ----
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
                float m = -INFINITY, sum = 0.0f;
                bool seen = false;
                const int least = w.b < 0 ? w.keys : unit_row(p, l, w, group * S::BLOCK).keys;   // (rows that come later see more)
                for (int j = 0; j < tiles && ok; j++) {
                    const int set = 2 * group + (j & 1), key0 = (w.tile + j) * S::KEYS, known = (k_count + j) % S::RING;
                    ok = wait_warp(&sh.known[known], (k_count + j) / S::RING, gave_up, dense::TG_PLACES) && wait_warp(&sh.scores[set], s_count[j & 1] + (j >> 1), gave_up, dense::TG_SCORES);
                    if (!ok) break;
                    tmem_after();
                    const uint32_t at = tmem + lanes + (uint32_t)set * S::KEYS;
                    bool all = key0 + S::KEYS <= least;
#pragma unroll
                    for (int c = 0; c < S::KEYS / 32; c++) all = all && sh.there[known][c] == ~0u;
                    auto sees = [&](int c) {   // bit i: the row sees key 32 c + i of the tile
                        const int limit = r.keys - key0 - 32 * c;
                        return sh.there[known][c] & (limit >= 32 ? ~0u : limit <= 0 ? 0u : (1u << limit) - 1);
                    };
                    // A score rises with its dot (falls, with a negative factor): the largest dot makes the largest score.  Tiles that need no mask are straight-line code on 64 scores
                    // in registers; the others, and capped weights, go 16 at a time, in loops, to keep that code small (with all forms unrolled the rows' warps waited for
                    // instructions a fifth of their time)
                    uint32_t v[64];
                    float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    const bool plain = all && p.scale2 > 0.0f;
                    if (plain) {
                        tmem_load64(at, v);
#pragma unroll
                        for (int i = 0; i < 64; i += 2) tops[i >> 1 & 3] = fmaxf(fmaxf(tops[i >> 1 & 3], __uint_as_float(v[i])), __uint_as_float(v[i + 1]));
                    } else {
                        const uint32_t sign = p.scale2 < 0.0f ? 0x80000000u : 0u;
#pragma unroll 1
                        for (int c = 0; c < 64; c += 16) {
                            const uint32_t mask = sees(c >> 5) >> (c & 16);
                            uint32_t u[16];
                            tmem_load16(at + c, u);
                            seen = seen || (mask & 0xffff);
#pragma unroll
                            for (int i = 0; i < 16; i++)
                                if (mask >> i & 1) tops[i & 3] = fmaxf(tops[i & 3], __uint_as_float(u[i] ^ sign));
                        }
                    }
                    seen = seen || all;
                    float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                    if (top != -INFINITY) top = score2(p, p.scale2 < 0.0f ? -top : top);
                    top -= WEIGHT_SHIFT<T>;
                    if (__any_sync(~0u, top > m + RESCALE_AT || (m == -INFINITY && top > m))) {
                        const float now = fmaxf(m, top), corr = ex2(m - (now == -INFINITY ? 0.0f : now));
                        if (j > 0) {
                            ok = wait_warp(&sh.summed[2 * group + ((j - 1) & 1)], s_count[(j - 1) & 1] + ((j - 1) >> 1), gave_up, dense::TG_VALUES);
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
                    if (plain && !(p.softcap > 0.0f)) {
                        const uint64_t factor = pair_of(__float_as_uint(p.scale2), __float_as_uint(p.scale2)), less = pair_of(__float_as_uint(-base), __float_as_uint(-base));
                        uint64_t total[2] = {0, 0};
                        uint32_t a[32];
#pragma unroll
                        for (int i = 0; i < 32; i++) {
                            float2 e = pair_open(fma_pair(pair_of(v[2 * i], v[2 * i + 1]), factor, less));
                            e.x = ex2(e.x);
                            e.y = ex2(e.y);
                            total[i & 1] = add_pair(total[i & 1], pair_of(__float_as_uint(e.x), __float_as_uint(e.y)));
                            a[i] = close_word(e, T());
                        }
                        const float2 t = pair_open(add_pair(total[0], total[1]));
                        sum += t.x + t.y;
                        tmem_store32(at, a);   // (over scores that have been read)
                    } else {
                        float t0 = 0.0f, t1 = 0.0f;
#pragma unroll 1
                        for (int c = 0; c < 64; c += 16) {
                            const uint32_t mask = sees(c >> 5) >> (c & 16);
                            uint32_t u[16], a[8];
                            float e[16];
                            tmem_load16(at + c, u);
#pragma unroll
                            for (int i = 0; i < 16; i++) e[i] = __uint_as_float(u[i]);
                            if (p.softcap > 0.0f) {
                                cap_scores(p, e);
#pragma unroll
                                for (int i = 0; i < 16; i++) e[i] = ex2(e[i] - base);
                            } else {
#pragma unroll
                                for (int i = 0; i < 16; i++) e[i] = ex2(fmaf(e[i], p.scale2, -base));
                            }
#pragma unroll
                            for (int i = 0; i < 16; i++)
                                if (!(mask >> i & 1)) e[i] = 0.0f;
#pragma unroll
                            for (int i = 0; i < 8; i++) {
                                t0 += e[2 * i];
                                t1 += e[2 * i + 1];
                                a[i] = close_word(make_float2(e[2 * i], e[2 * i + 1]), T());
                            }
                            tmem_store8(at + (c >> 1), a);   // (columns c / 2 .. c / 2 + 7, all of them below c + 16: read)
                        }
                        sum += t0 + t1;
                    }
                    tmem_stored();
                    tmem_before();
                    arrive(&sh.weights[set]);
                }
                // the part's rows
                const int64_t slot = w.unit + blockIdx.x;
                const bool whole = whole_unit(p, w, w.tile, w.tile + tiles - 1), is = x < used;
                ok = ok && wait_warp(&sh.summed[2 * group + ((tiles - 1) & 1)], s_count[(tiles - 1) & 1] + ((tiles - 1) >> 1), gave_up, dense::TG_VALUES);
                if (ok) {
                    tmem_after();
                    if (!seen) sum = -1.0f;
                    float odd = 0.0f;   // becomes NaN if a sum is not finite
                    float* to = whole ? nullptr : part_at(l, D, slot, x, 0);
                    const bool store = is && (whole || slot < l.slots);
                    const float by = seen ? 1.0f / sum : 1.0f;   // (0: 1 / 0 * 0 is NaN, as 0 / 0 is)
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        uint32_t o[32];
                        tmem_load32(tmem + lanes + S::O_AT + (uint32_t)group * DP + c, o);
                        if (!seen) {
#pragma unroll
                            for (int i = 0; i < 32; i++) o[i] = 0;
                        }
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            if (c + i >= D) break;   // (D is a multiple of 8)
                            float4 f = make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]), __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
                            float4 g = make_float4(__uint_as_float(o[i + 4]), __uint_as_float(o[i + 5]), __uint_as_float(o[i + 6]), __uint_as_float(o[i + 7]));
                            odd = fmaf(f.x, 0.0f, fmaf(f.y, 0.0f, fmaf(f.z, 0.0f, fmaf(f.w, 0.0f, odd))));
                            odd = fmaf(g.x, 0.0f, fmaf(g.y, 0.0f, fmaf(g.z, 0.0f, fmaf(g.w, 0.0f, odd))));
                            if (!store) continue;
                            if (whole) {
                                f.x *= by; f.y *= by; f.z *= by; f.w *= by;
                                g.x *= by; g.y *= by; g.z *= by; g.w *= by;
                                store_row(p, r, c + i, f);
                                store_row(p, r, c + i + 4, g);
                            } else {
                                float4* at8 = reinterpret_cast<float4*>(to + (int64_t)((c + i) >> 3) * (S::ROWS * 8));
                                at8[0] = f;
                                at8[1] = g;
                            }
                        }
                    }
                    const bool finite = odd == 0.0f;
                    if (is) {
                        if (whole) { if (p.lse) p.lse[r.row * p.q_heads + r.head] = seen ? lse_of(m, sum) : -INFINITY; }
                        else if (slot < l.slots) l.ml[slot * S::ROWS + x] = make_float2(m, sum);
                    }
                    tmem_before();
                    arrive(&sh.read[group]);
                    if (is && seen && !finite && w.b >= 0 && w.s.count > 1) sh.spoiled = true;   // other rows' keys may have spoiled it
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
            } else {
                arrive(&sh.read[1]);   // (a part without a second block: its turn passes)
            }
            k_count += tiles;
            arrive(&sh.parted);
            ok = ok && wait_part(&sh.parted, part++, &sh.known[0], gave_up);
        } while (leave());
    }
    tmem_before();
    __syncthreads();
    if (warp == PRODUCTS) {
        __syncwarp();
        tmem_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
    }
    if (threadIdx.x == 0 && *gave_up && p.err) *p.err = *gave_up;
    // Rows to be summed again, all parts once more: behind the last wait of the CTA, since this takes as long as it takes (128 rows of 64 columns over 150 thousand keys: seconds)
    if (warp >= 8 || !sh.spoiled || *gave_up) return;
    const int group = warp >> 2, row = threadIdx.x & 127;
    int* flags = reinterpret_cast<int*>(sh.again[group].weight);
    w = sh.start;
    left = sh.tiles;
    do {
        enter();
        if (w.b < 0 || w.s.count <= 1 || group >= blocks) continue;
        const int64_t slot = w.unit + blockIdx.x;
        const bool whole = whole_unit(p, w, w.tile, w.tile + tiles - 1);
        if (!whole && slot >= l.slots) continue;
        const int x = group * S::BLOCK + row;
        bool again = false;
        if (x < used) {   // (what this thread has stored)
            const UnitRow r = unit_row(p, l, w, x);
            float odd = 0.0f;   // becomes NaN if the row is not finite
            if (whole)
                for (int c = 0; c < D; c++) odd = fmaf(to_f(p.out.data[r.row * p.out.row + r.head * p.out.head + c]), 0.0f, odd);
            else if (!(l.ml[slot * S::ROWS + x].y < 0.0f))
                for (int c = 0; c < D; c++) odd = fmaf(*part_at(l, D, slot, x, c), 0.0f, odd);
            again = odd != 0.0f;
        }
        again_sync(1 + group);
        flags[row] = again;
        again_sync(1 + group);
        unsigned todo[4], any = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) any |= todo[i] = __ballot_sync(~0u, flags[32 * i + lane]);
        if (!any) continue;
        again_sync(1 + group);   // (the flags' place is used below)
#pragma unroll 1
        for (int i = 0; i < S::BLOCK; i++) {
            if (!((i < 32 ? todo[0] : i < 64 ? todo[1] : i < 96 ? todo[2] : todo[3]) >> (i & 31) & 1)) continue;
            const UnitRow r = unit_row(p, l, w, group * S::BLOCK + i);
            float m, sum, acc[2];
            row_again(p, w, r, w.tile * S::KEYS, (w.tile + tiles) * S::KEYS, sh.again[group], 1 + group, m, sum, acc);
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int c = row + AGAIN * k;
                if (c >= D) continue;
                if (whole) p.out.data[r.row * p.out.row + r.head * p.out.head + c] = from_f<T>(acc[k] / sum);
                else *part_at(l, D, slot, group * S::BLOCK + i, c) = acc[k];
            }
            if (row == 0) {
                if (whole) { if (p.lse) p.lse[r.row * p.q_heads + r.head] = lse_of(m, sum); }
                else l.ml[slot * S::ROWS + group * S::BLOCK + i] = make_float2(m, sum);
            }
        }
    } while (leave());
}

}  // namespace paged
}  // namespace lmrs
