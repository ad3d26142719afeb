// paged.cu -- entry points of include/lmrs_b200.h for many sequences at once: checks of the arguments, choice of the kernels, launches.
// Device pointers, the caller's stream; nothing here allocates, synchronises or remembers anything from one call to the next.
#include <float.h>
#include <math.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "paged_attn.cuh"
#include "paged_checks.h"
#include "paged_rows.cuh"
#include "paged_tensor.cuh"

using namespace lmrs;
using namespace lmrs::paged;

namespace {

// freq / 2 pi modulo 1, in 2^-64, to the nearest: off by at most 1/2 + |freq| 2^-65 of that.  freq = m 2^e with 53 bits in m, times 1 / 2 pi in 2^-128 (rounded; arctangents of 1/5 and
// 1/239 give its digits, as the tests do), is a whole number of 192 bits in 2^(e - 128); what is wanted are its 64 bits below the point.
uint64_t turns_of(double freq) {
    constexpr uint64_t HIGH = 0x28be60db9391054aull, LOW = 0x7f09d5f47d4d3770ull;
    int e = 0;
    const uint64_t m = (uint64_t)ldexp(frexp(fabs(freq), &e), 53);
    e -= 53;
    const unsigned __int128 low = (unsigned __int128)m * LOW, high = (unsigned __int128)m * HIGH + (uint64_t)(low >> 64);
    const uint64_t words[3] = {(uint64_t)low, (uint64_t)high, (uint64_t)(high >> 64)};
    auto bits = [&](int from) {   // 64 bits of the product from bit `from` on
        uint64_t r = 0;
        for (int i = 0; i < 3; i++) {
            const int at = 64 * i - from;
            if (at > -64 && at < 64) r |= at < 0 ? words[i] >> -at : words[i] << at;
        }
        return r;
    };
    const int from = 64 - e;
    const uint64_t t = bits(from) + (from > 0 ? bits(from - 1) & 1 : 0);   // (a whole turn is none)
    return freq < 0 ? 0 - t : t;
}

}  // namespace

extern "C" int lmrs_b200_rope_init(lmrs_b200_rope_t* out, const double* freq, const uint8_t* axis, int pairs, int layout) {
    return guarded("rope_init", [&]() -> int {
        if (!out || !freq) return refuse("rope_init", "null argument");
        if (pairs < 1 || pairs > 128) return refuse("rope_init", "pairs must be 1 .. 128");
        if (layout != 0 && layout != 1) return refuse("rope_init", "layout must be 0 (halves) or 1 (neighbours)");
        lmrs_b200_rope_t r = {};
        r.pairs = pairs;
        r.layout = layout;
        for (int j = 0; j < pairs; j++) {
            if (!isfinite(freq[j])) return refuse("rope_init", "a frequency is not finite");
            r.turns[j] = turns_of(freq[j]);
            r.axis[j] = axis ? axis[j] : 0;
            if (r.axis[j] >= r.axes) r.axes = r.axis[j] + 1;
        }
        *out = r;
        return 0;
    });
}

extern "C" int lmrs_b200_rope_axes(const lmrs_b200_rope_t* rope, int dtype, const lmrs_b200_rows_t* x, const lmrs_b200_rows_t* out, int64_t n_rows, int heads,
                                   int head_size, const lmrs_b200_positions_t* pos, void* stream) {
    static const char* me = "rope_axes";
    return guarded(me, [&]() -> int {
        if (!rope || !x || !out || !pos) return refuse(me, "null argument");
        std::string why = bad_dtype(dtype);
        if (!why.empty()) return refuse(me, why);
        if (n_rows < 0 || n_rows > 0x7fffffff || heads < 0 || heads > MAX_HEADS || head_size < 1 || head_size > 256)
            return refuse(me, "n_rows must be 0 .. 2^31 - 1, heads 0 .. 65535, head_size 1 .. 256");
        why = bad_rope(rope, head_size);
        if (why.empty() && !same(x, out, n_rows, heads) && meet(x, heads, out, heads, n_rows, head_size, dtype)) why = "out lies over x without being x itself";
        if (!why.empty()) return refuse(me, why);
        int device = 0;
        const int sms = device_sms(me, &device);
        if (!sms) return 1;
        if (n_rows == 0 || heads == 0) return 0;
        why = bad_rows(x, "x", dtype, device);
        if (why.empty()) why = bad_rows(out, "out", dtype, device);
        if (why.empty()) why = !pos->data ? "null positions" : bad_ints(pos->data, "positions", device);
        if (!why.empty()) return refuse(me, why);
        return by_type(dtype, [&](auto t) {
            using T = decltype(t);
            constexpr int VEC = 16 / sizeof(T);
            const bool wide = vectors(x, dtype) && vectors(out, dtype) && rope->pairs % VEC == 0 && head_size % VEC == 0;
            const Cut cut = cut_of(rope->pairs, rope->layout, head_size, wide ? VEC : 1);
            const int parts = parts_of(n_rows, (int64_t)heads * (cut.turning + cut.passing), sms);
            (wide ? rope_axes_kernel<T, VEC> : rope_axes_kernel<T, 1>)<<<warps_grid(n_rows * parts, sms), 32 * ROW_WARPS, 0, (cudaStream_t)stream>>>(
                *rope, rows_as<const T>(x), rows_as<T>(out), n_rows, heads, cut, pos_as(pos), parts);
            return launched(me);
        });
    });
}

extern "C" int lmrs_b200_paged_append(const lmrs_b200_pages_t* pages, const lmrs_b200_batch_t* batch, int64_t n_rows, const lmrs_b200_rows_t* k, const lmrs_b200_rows_t* v,
                                      const lmrs_b200_rope_t* rope, const lmrs_b200_positions_t* pos, const lmrs_b200_rows_t* q, const lmrs_b200_rows_t* q_out, int q_heads,
                                      void* stream) {
    static const char* me = "paged_append";
    return guarded(me, [&]() -> int {
        std::string why = bad_pages(pages);
        if (why.empty()) why = bad_batch(batch, n_rows, pages->page_size);
        if (why.empty() && (q || q_out) && (!q || !q_out)) why = "q and q_out come together";
        if (why.empty() && q && !rope) why = "q without rope";
        if (why.empty() && q && (q_heads < 1 || q_heads > MAX_HEADS)) why = "q_heads must be 1 .. 65535";
        if (why.empty() && rope) why = bad_rope(rope, pages->head_size);
        if (why.empty() && q && !same(q, q_out, n_rows, q_heads) && meet(q, q_heads, q_out, q_heads, n_rows, pages->head_size, pages->dtype)) why = "q_out lies over q without being q itself";
        if (why.empty() && q && k && v && (meet(k, pages->kv_heads, q_out, q_heads, n_rows, pages->head_size, pages->dtype) || meet(v, pages->kv_heads, q_out, q_heads, n_rows, pages->head_size, pages->dtype)))
            why = "q_out lies over k or v";
        if (!why.empty()) return refuse(me, why);
        int device = 0;
        const int sms = device_sms(me, &device);
        if (!sms) return 1;
        if (n_rows == 0 || batch->seqs == 0) return 0;
        const int dtype = pages->dtype;
        why = bad_batch_memory(batch, device);
        if (why.empty()) why = bad_rows(k, "k", dtype, device);
        if (why.empty()) why = bad_rows(v, "v", dtype, device);
        if (why.empty() && q) why = bad_rows(q, "q", dtype, device);
        if (why.empty() && q) why = bad_rows(q_out, "q_out", dtype, device);
        if (why.empty() && pos) why = !pos->data ? "null positions" : bad_ints(pos->data, "positions", device);
        if (why.empty() && (!on_device(pages->k, device) || !on_device(pages->v, device))) why = "the pages are not memory of the current device";
        if (!why.empty()) return refuse(me, why);
        return by_type(dtype, [&](auto t) {
            using T = decltype(t);
            AppendParams<T> p = {};
            if (rope) p.rope = *rope;
            p.batch = batch_as(batch, pages, n_rows);
            p.pos = pos_as(rope ? pos : nullptr);
            p.k = rows_as<const T>(k);
            p.v = rows_as<const T>(v);
            if (q) { p.q = rows_as<const T>(q); p.q_out = rows_as<T>(q_out); p.q_heads = q_heads; }
            p.k_pages = (T*)pages->k; p.v_pages = (T*)pages->v;
            p.k_page = pages->k_page; p.k_slot = pages->k_slot; p.k_head = pages->k_head;
            p.v_page = pages->v_page; p.v_slot = pages->v_slot; p.v_head = pages->v_head;
            p.kv_heads = pages->kv_heads;
            constexpr int VEC = 16 / sizeof(T);
            const int pairs = rope ? rope->pairs : 0, size = pages->head_size;
            const bool wide = vectors(k, dtype) && vectors(v, dtype) && (!q || (vectors(q, dtype) && vectors(q_out, dtype))) && vectors(pages->k, pages->k_page, pages->k_head, dtype) &&
                              vectors(pages->v, pages->v_page, pages->v_head, dtype) && pages->k_slot % VEC == 0 && pages->v_slot % VEC == 0 && pairs % VEC == 0 && size % VEC == 0;
            p.turn = cut_of(pairs, rope ? rope->layout : 0, size, wide ? VEC : 1);
            p.pass = cut_of(0, 0, size, wide ? VEC : 1);
            p.parts = parts_of(n_rows, (int64_t)(p.kv_heads + p.q_heads) * (p.turn.turning + p.turn.passing) + (int64_t)p.kv_heads * p.pass.passing, sms);
            (wide ? paged_append_kernel<T, VEC> : paged_append_kernel<T, 1>)<<<warps_grid(n_rows * p.parts, sms), 32 * ROW_WARPS, 0, (cudaStream_t)stream>>>(p);
            return launched(me);
        });
    });
}

static std::string bad_attention(const lmrs_b200_pages_t* pages, const lmrs_b200_batch_t* batch, int64_t n_rows, int q_heads) {
    std::string why = bad_pages(pages);
    if (why.empty()) why = bad_batch(batch, n_rows, pages->page_size);
    if (!why.empty()) return why;
    const int64_t vec = 16 / (int64_t)size_of(pages->dtype);
    if (pages->head_size % 8) return "head_size must be a multiple of 8";
    if ((int64_t)batch->table_len * pages->page_size + batch->prefix_len > 0x7fffffff - AGAIN) return "prefix_len + table_len * page_size is beyond 2^31 - 129";   // (numbers of keys go up to the end of a tile)
    if (q_heads < 1 || q_heads > MAX_HEADS || q_heads % pages->kv_heads) return "q_heads must be a positive multiple of kv_heads, at most 65535";
    if (n_rows * q_heads > 0x40000000) return "n_rows * q_heads is beyond 2^30";
    if (!aligned(pages->k, 16) || !aligned(pages->v, 16) || pages->k_page % vec || pages->k_slot % vec || pages->k_head % vec || pages->v_page % vec || pages->v_slot % vec ||
        pages->v_head % vec)
        return "the pages' rows must lie on 16-byte boundaries";
    return "";
}

namespace {

// How a call is cut, from what the host knows of it
struct Cutting {
    Line own, front;   // the kernel's that takes the sequences' units, and that takes the prefix' (the same where one takes both)
    bool own_tensor, front_tensor;
    size_t bytes;
};
// Which kernel takes what.  float32: rows16_kernel.  16-bit types: it depends on how often the keys would be read again.  rows16_kernel reads them once per 16
// rows of a KV head and, with little to do, starts some 8 us sooner; rows128_kernel reads them once per 128 or 256 rows.  Measured on a B200 with rows16_kernel / rows128_kernel,
// us a call, 8 KV heads:
//   a sequence's own keys, 16 sequences behind up to 4000 keys (the others behind 1000 or more, with a third of the rows or more), rows of the longest sequence and a KV head:
//     head 64:  32: 45 / 64   64: 80 / 76   128: 139 / 79      128:  32: 71 / 72   64: 130 / 84   128: 239 / 87      256:  8: 143 / 93   16: 148 / 96   32: 243 / 97
//     (one sequence alone: 64: 22 / 23 at head 64, 28 / 26 at 128;  16: 31 / 32 and 8: 27 / 31 at 256)
//   the prefix, rows of all sequences and a KV head behind a prefix of 512, 2048, 8192, 32768 keys:
//     head 64:   16: 11 / 18, 13 / 23, 20 / 27, 39 / 47   32: 11 / 18, 16 / 23, 24 / 28, 63 / 47   128: 17 / 23, 28 / 27, 67 / 32, 220 / 53
//     head 128:  16: 12 / 19, 16 / 24, 25 / 30, 56 / 60   32: 13 / 19, 18 / 25, 35 / 31, 96 / 60   128: 21 / 27, 36 / 33, 102 / 34, 359 / 65
//     head 256:   8: 15 / 21, 23 / 30, 60 / 38, 162 / 83  32: 25 / 22, 35 / 31, 106 / 39, 385 / 83 128: 46 / 39, 114 / 42, 399 / 61, 1503 / 100
// So the own keys by the rows, and the prefix by the rows times keys times KV heads that rows16_kernel would have to go through; with 16 rows or fewer it reads the keys once
// and loses nothing, but for heads of 256, where only one of its CTAs fits an SM and the bytes in flight do not fill the memory.
template <int DP> struct TensorRule {
    static constexpr int OWN_ROWS = DP <= 128 ? 64 : 16, FRONT_ROWS = DP <= 128 ? 17 : 1;
    static constexpr int64_t FRONT_WORK = DP <= 128 ? 1 << 21 : 1 << 19;
};
template <typename T, int DP> Cutting cutting(const lmrs_b200_pages_t* pages, const lmrs_b200_batch_t* batch, int64_t n_rows, int q_heads, char* base) {
    const int64_t group = q_heads / pages->kv_heads, rows = n_rows * group;
    Cutting c = {};
    auto line = [&](Line& l, bool tensor, bool own, bool front) {
        int tile_rows = TileShape<T, DP>::ROWS, tile_keys = TileShape<T, DP>::KEYS, ctas = SMS * TileShape<T, DP>::CTAS;
        if constexpr (sizeof(T) == 2)
            if (tensor) { tile_rows = TensorShape<T, DP>::ROWS; tile_keys = TensorShape<T, DP>::KEYS; ctas = SMS; }
        l.tile_rows = tile_rows;
        l.tile_keys = tile_keys;
        while (1 << l.row_shift < tile_rows) l.row_shift++;
        while (1 << l.key_shift < tile_keys) l.key_shift++;
        l.seqs = own ? batch->seqs : 0;
        l.front_tiles = front ? (int)(((int64_t)batch->prefix_len + tile_keys - 1) / tile_keys) : 0;
        l.front_units = l.front_tiles ? (rows + tile_rows - 1) / tile_rows * pages->kv_heads : 0;
        // The prefix by itself: as many CTAs for each unit, where that leaves few SMs out, so that none has a part of two units (rows16_kernel's first CTAs take the SMs left out).
        // 148 / 144 CTAs, 8 or 16 units, with the own keys: 64 sequences behind 8200 keys 71 / 67 us, 128 behind 32768 175 / 171, behind 8192 113 / 109, 32 behind 32768 79 / 77, 100
        // behind 4096 59 / 54.  (Fewer still, so that the own keys' reads overlap the prefix' products, are better or worse by the lengths, which the host does not know: 96 CTAs
        // 66, 156, 114, 71, 53; 64 CTAs 61, 208, 110, 93, 45.)
        if (tensor && !own && l.front_units > 0 && l.front_units <= SMS) {
            const int even = SMS / (int)l.front_units * (int)l.front_units;
            if (even * 16 >= SMS * 15) ctas = even;
        }
        l.ctas = ctas;
        place_line(l, rows, pages->kv_heads, pages->head_size, base, c.bytes);
    };
    using R = TensorRule<DP>;
    c.own_tensor = sizeof(T) == 2 && std::min<int64_t>(batch->max_rows, n_rows) * group >= R::OWN_ROWS;
    c.front_tensor = c.own_tensor || (sizeof(T) == 2 && rows >= R::FRONT_ROWS && rows * pages->kv_heads * batch->prefix_len >= R::FRONT_WORK);
    line(c.own, c.own_tensor, true, c.own_tensor == c.front_tensor);
    if (c.own_tensor == c.front_tensor) c.front = c.own;
    else line(c.front, true, false, true);
    return c;
}
template <typename F> int by_shape(const lmrs_b200_pages_t* pages, F f) {
    return by_type(pages->dtype, [&](auto t) {
        using T = decltype(t);
        return pages->head_size <= 64 ? f(T(), std::integral_constant<int, 64>()) : pages->head_size <= 128 ? f(T(), std::integral_constant<int, 128>()) : f(T(), std::integral_constant<int, 256>());
    });
}
// Tensor maps of the pages for tiles of TensorShape X, if there are any (boxes.rows stays 0 otherwise): rows of a box are the most that divide a page and a copying warp's share
template <typename X> void box_maps(const lmrs_b200_pages_t* pages, const lmrs_b200_rows_t* q, int64_t n_rows, int q_heads, bool q_wide, Boxes& boxes) {
    typedef CUresult (*Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                               CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess ? (Encode)f : nullptr;
    }();
    if (!encode) return;
    const size_t size = size_of(pages->dtype);
    const int group = q_heads / pages->kv_heads;
    if (q_wide && X::BLOCK % group == 0 && q->row > 0 && q->head > 0) {
        const cuuint64_t dims[3] = {pages->head_size * size, (cuuint64_t)q_heads, (cuuint64_t)n_rows}, strides[2] = {q->head * size, q->row * size};
        const cuuint32_t box[3] = {128, (cuuint32_t)group, (cuuint32_t)(X::BLOCK / group)}, step[3] = {1, 1, 1};
        if (strides[0] < (1ull << 40) && strides[1] < (1ull << 40) &&
            encode(&boxes.q, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, q->data, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS)
            boxes.q_tokens = X::BLOCK / group;
    }
    int rows = X::KEYS / X::COPIERS;
    while (rows >= 8 && pages->page_size % rows) rows /= 2;
    if (rows < 8) return;
    auto map = [&](CUtensorMap* m, void* base, int64_t page, int64_t slot, int64_t head, int& place_at, int& head_at) {
        struct { int64_t stride; cuuint64_t n; cuuint32_t box; int what; } d[3] = {{slot, (cuuint64_t)pages->page_size, (cuuint32_t)rows, 0}, {head, (cuuint64_t)pages->kv_heads, 1, 1},
                                                                              {page, (cuuint64_t)pages->pages, 1, 2}};
        std::sort(d, d + 3, [](const auto& a, const auto& b) { return a.stride < b.stride; });
        const cuuint64_t dims[4] = {pages->head_size * size, d[0].n, d[1].n, d[2].n};
        const cuuint64_t strides[3] = {d[0].stride * size, d[1].stride * size, d[2].stride * size};
        const cuuint32_t box[4] = {128, d[0].box, d[1].box, d[2].box}, step[4] = {1, 1, 1, 1};
        for (int i = 0; i < 3; i++) {
            if (d[i].what == 0) place_at = i;
            if (d[i].what == 1) head_at = i;
            if (strides[i] == 0 || strides[i] % 16 || strides[i] >= (1ull << 40)) return false;
        }
        return encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, base, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    };
    if (map(&boxes.k, pages->k, pages->k_page, pages->k_slot, pages->k_head, boxes.k_place, boxes.k_head) &&
        map(&boxes.v, pages->v, pages->v_page, pages->v_slot, pages->v_head, boxes.v_place, boxes.v_head))
        boxes.rows = rows;
}

}  // namespace

extern "C" int lmrs_b200_paged_attention_workspace(const lmrs_b200_pages_t* pages, const lmrs_b200_batch_t* batch, int64_t n_rows, int q_heads, size_t* bytes) {
    static const char* me = "paged_attention_workspace";
    return guarded(me, [&]() -> int {
        if (!bytes) return refuse(me, "null argument");
        const std::string why = bad_attention(pages, batch, n_rows, q_heads);
        if (!why.empty()) return refuse(me, why);
        *bytes = 0;
        if (n_rows == 0 || batch->seqs == 0) return 0;
        return by_shape(pages, [&](auto t, auto d) {
            *bytes = cutting<decltype(t), decltype(d)::value>(pages, batch, n_rows, q_heads, nullptr).bytes;
            return 0;
        });
    });
}

extern "C" int lmrs_b200_paged_attention(const lmrs_b200_pages_t* pages, const lmrs_b200_batch_t* batch, int64_t n_rows, const lmrs_b200_rows_t* q, const lmrs_b200_rows_t* out,
                                         int q_heads, float scale, float softcap, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    static const char* me = "paged_attention";
    return guarded(me, [&]() -> int {
        std::string why = bad_attention(pages, batch, n_rows, q_heads);
        if (why.empty() && !isfinite(scale)) why = "scale is not finite";
        if (why.empty() && !(softcap >= 0.0f && isfinite(softcap))) why = "softcap must be 0 (none) or positive";
        if (!why.empty()) return refuse(me, why);
        const bool over = q && out && meet(q, q_heads, out, q_heads, n_rows, pages->head_size, pages->dtype);
        int device = 0;
        if (!(over && q->data != out->data) && !device_sms(me, &device)) return 1;   // (a call without a device says so, before it says that it is one in place)
        if (over) return refuse(me, "out lies where q does, which is read until the call has ended");
        if (n_rows == 0 || batch->seqs == 0) return 0;
        const int dtype = pages->dtype;
        why = bad_batch_memory(batch, device);
        if (why.empty()) why = bad_rows(q, "q", dtype, device);
        if (why.empty()) why = bad_rows(out, "out", dtype, device);
        if (why.empty() && lse && (!aligned(lse, 4) || !on_device(lse, device))) why = "lse is not memory of the current device";
        if (why.empty() && (!on_device(pages->k, device) || !on_device(pages->v, device))) why = "the pages are not memory of the current device";
        if (why.empty() && (!workspace || !aligned(workspace, 256) || !on_device(workspace, device))) why = "workspace is not memory of the current device on a 256-byte boundary";
        if (!why.empty()) return refuse(me, why);
        if (const int status = gave_up_word.take()) return refuse(me, "results of an earlier call are NaN: " + dense::tg_gave_up(status));
        return by_shape(pages, [&](auto t, auto d) {
            using T = decltype(t);
            using S = TileShape<T, decltype(d)::value>;
            const Cutting c = cutting<T, decltype(d)::value>(pages, batch, n_rows, q_heads, (char*)workspace);
            if (workspace_bytes < c.bytes) return refuse(me, "workspace has " + std::to_string(workspace_bytes) + " bytes, the call needs " + std::to_string(c.bytes));
            AttnParams<T> p = {};
            p.batch = batch_as(batch, pages, n_rows);
            p.q = rows_as<const T>(q);
            p.out = rows_as<T>(out);
            p.k = (const T*)pages->k; p.v = (const T*)pages->v;
            p.k_page = pages->k_page; p.k_slot = pages->k_slot; p.k_head = pages->k_head;
            p.v_page = pages->v_page; p.v_slot = pages->v_slot; p.v_head = pages->v_head;
            p.kv_heads = pages->kv_heads; p.q_heads = q_heads; p.head_size = pages->head_size; p.group = q_heads / pages->kv_heads;
            // At the ends of float32: a cap beyond 2^100 is one of 2^100 (scores of up to 2^88 are not moved by either, and its product with log2 e is finite), and no score is 0 times infinity
            const float cap = std::min(softcap, 0x1p100f);
            p.scale2 = std::max(-FLT_MAX, std::min(FLT_MAX, scale * LOG2E)); p.softcap = cap; p.cap_in = cap > 0.0f ? std::max(-FLT_MAX, std::min(FLT_MAX, scale / cap)) : 0.0f; p.lse = lse;
            p.q_wide = vectors(q, dtype);
            p.out_wide = aligned(out->data, 4 * sizeof(T)) && out->row % 4 == 0 && out->head % 4 == 0;
            p.whole = batch->prefix_len == 0;
            p.page_shift = -1;
            for (int i = 0; i < 31; i++)
                if (pages->page_size == 1 << i) p.page_shift = i;
            static std::atomic<uint64_t> allowed{0}, allowed_tensor{0};
            cudaError_t e = cudaSuccess;
            if constexpr (sizeof(T) == 2)
                if (c.front_tensor) {
                    auto kernel = rows128_kernel<T, decltype(d)::value>;
                    using X = TensorShape<T, decltype(d)::value>;
                    if ((e = allow_smem(kernel, device, X::SMEM, allowed_tensor)) != cudaSuccess) return refuse(me, cudaGetErrorString(e));
                    if (!(p.err = gave_up_word.get())) return refuse(me, "out of host memory");
                    Boxes boxes = {};
                    box_maps<X>(pages, q, n_rows, q_heads, p.q_wide, boxes);
                    kernel<<<(unsigned)c.front.ctas, X::THREADS, X::SMEM, (cudaStream_t)stream>>>(p, c.front, boxes);
                    if (launched(me)) return 1;
                }
            if (!c.own_tensor) {
                auto kernel = rows16_kernel<T, decltype(d)::value>;
                if ((e = allow_smem(kernel, device, S::SMEM, allowed)) != cudaSuccess) return refuse(me, cudaGetErrorString(e));
                if (c.front_tensor) e = launch_after(kernel, (unsigned)c.own.ctas, S::THREADS, S::SMEM, (cudaStream_t)stream, p, c.own);
                else kernel<<<(unsigned)c.own.ctas, S::THREADS, S::SMEM, (cudaStream_t)stream>>>(p, c.own);
                if (e != cudaSuccess) return refuse(me, std::string("launch failed: ") + cudaGetErrorString(e));
                if (launched(me)) return 1;
            }
            // A warp a row and head, or 8 where that leaves most of the GPU's warps idle, since there the parts are many.  One warp / 8, us a call: 32 rows and heads behind
            // 30000 keys 46 / 39; behind 4000 keys 128: 22.4 / 19.7, 512: 46.0 / 45.1, 640: 54.2 / 56.3, 1024: 77.5 / 80.6; behind 200 keys 512: 13.2 / 12.4, 1024: 19.6 / 22.0
            const int64_t items = n_rows * q_heads;
            constexpr int COLS = decltype(d)::value <= 128 ? 1 : 2;
            e = items <= SMS * 4 ? launch_after(join_kernel<T, 8, COLS>, (unsigned)items, 256, 0, (cudaStream_t)stream, p, c.front, c.own)
                                 : launch_after(join_kernel<T, 1, COLS>, (unsigned)std::min<int64_t>((items + 7) / 8, SMS * 16), 256, 0, (cudaStream_t)stream, p, c.front, c.own);
            return e == cudaSuccess ? 0 : refuse(me, std::string("launch failed: ") + cudaGetErrorString(e));
        });
    });
}
