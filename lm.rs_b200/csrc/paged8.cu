// paged8.cu -- entry points of include/lmrs_b200.h for attention over pages of 8-bit codes: checks of the arguments, choice of the kernels, launches.
// Device pointers, the caller's stream; nothing here allocates, synchronises or remembers anything from one call to the next.
#include <float.h>
#include <math.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "paged8_attn.cuh"
#include "paged8_tensor.cuh"
#include "paged8_checks.h"

using namespace lmrs;
using namespace lmrs::paged;

static std::string bad_attention8(const lmrs_b200_pages8_t* pages, const lmrs_b200_batch_t* batch, int dtype, int64_t n_rows, int q_heads) {
    std::string why = bad_pages8(pages);
    if (why.empty()) why = bad_dtype(dtype);
    if (why.empty()) why = bad_batch(batch, n_rows, pages->page_size);
    if (!why.empty()) return why;
    if ((int64_t)batch->table_len * pages->page_size + batch->prefix_len > 0x7fffffff - AGAIN) return "prefix_len + table_len * page_size is beyond 2^31 - 129";   // (numbers of keys go up to the end of a tile)
    if (q_heads < 1 || q_heads > MAX_HEADS || q_heads % pages->kv_heads) return "q_heads must be a positive multiple of kv_heads, at most 65535";
    if (n_rows * q_heads > 0x40000000) return "n_rows * q_heads is beyond 2^30";
    if (!wide_codes(pages)) return "head_size must be a multiple of 16, and the pages' rows lie on 16-byte boundaries";
    return "";
}

namespace {

// How a call is cut, from what the host knows of it (as in paged.cu)
struct Cutting8 {
    Line own, front;   // the kernel's that takes the sequences' units, and that takes the prefix' (the same where one takes both)
    bool own_tensor, front_tensor;
    size_t bytes;
};
// Which kernel takes what.  float32: rows8_kernel.  16-bit types: by how often the keys would be read, and converted, again, as in paged.cu: rows8_kernel does so for every 16 rows of a KV head (8 where no unit has more),
// codes128_kernel for every 128 or 256, and starts some 10 us later.  Measured on a B200 with rows8_kernel / codes128_kernel, us a call, 8 KV heads, int8, a scale for 16 tokens:
//   a sequence's own keys, 16 sequences behind up to 4000 keys, rows of the longest sequence and a KV head:
//     head 64:  32: 41 / 81   64: 64 / 89   128: 106 / 94      128:  32: 68 / 104   64: 120 / 115   128: 206 / 126      256:  16: 80 / 140   32: 120 / 141   64: 220 / 158
//     (one sequence alone, 64 rows: 22 / 27 at head 64, 32 / 31 at 128, 50 / 43 at 256)
//   the prefix, rows of all sequences and a KV head behind a prefix of 512, 2048, 8192, 32768 keys:
//     head 64:   16: 14 / 18, 14 / 25, 23 / 33, 35 / 62    32: 14 / 19, 16 / 26, 27 / 34, 55 / 64    64: 21 / 23, 23 / 27, 38 / 34, 91 / 65     128: 28 / 31, 33 / 36, 61 / 43, 172 / 74
//     head 128:  16: 16 / 20, 17 / 28, 29 / 37, 53 / 74    32: 17 / 24, 25 / 29, 36 / 38, 90 / 76    64: 27 / 29, 34 / 34, 58 / 43, 166 / 80    128: 37 / 41, 53 / 53, 106 / 61, 322 / 100
//     head 256:   8: 14 / 22, 18 / 33, 31 / 45, 71 / 101   16: 18 / 23, 26 / 33, 44 / 46, 129 / 116  32: 27 / 27, 34 / 36, 72 / 48, 238 / 118   128: 58 / 51, 97 / 67, 260 / 81, 906 / 155
struct Which8 { bool own_tensor, front_tensor; int row_tiles; };   // row_tiles: rows of a unit of rows8_kernel, in eights
template <int DP> struct TensorRule8 {
    static constexpr int OWN_ROWS = DP <= 64 ? 128 : DP <= 128 ? 64 : 48, FRONT_ROWS = DP <= 64 ? 33 : DP <= 128 ? 17 : 9;
    static constexpr int64_t FRONT_WORK = DP <= 64 ? 1 << 22 : DP <= 128 ? 1 << 21 : 1 << 20;
};
template <int DP> Which8 which8(const lmrs_b200_pages8_t* pages, const lmrs_b200_batch_t* batch, int dtype, int64_t n_rows, int q_heads) {
    using R = TensorRule8<DP>;
    const int64_t group = q_heads / pages->kv_heads, rows = n_rows * group, most = std::min<int64_t>(batch->max_rows, n_rows) * group;
    Which8 w = {};
    w.own_tensor = dtype != 1 && most >= R::OWN_ROWS;
    w.front_tensor = batch->prefix_len > 0 && (w.own_tensor || (dtype != 1 && rows >= R::FRONT_ROWS && rows * pages->kv_heads * batch->prefix_len >= R::FRONT_WORK));
    w.row_tiles = (batch->prefix_len && !w.front_tensor ? rows : most) <= 8 ? 1 : 2;
    return w;
}
template <typename T, int DP, int ROW_TILES> Cutting8 cutting8(const lmrs_b200_pages8_t* pages, const lmrs_b200_batch_t* batch, int64_t n_rows, int q_heads, const Which8& which, char* base) {
    const int64_t group = q_heads / pages->kv_heads, rows = n_rows * group;
    Cutting8 c = {};
    auto line = [&](Line& l, bool tensor, bool own, bool front) {
        using S = TileShape8<T, DP, ROW_TILES>;
        using X = TensorShape8<DP>;
        l.tile_rows = tensor ? X::ROWS : S::ROWS;
        l.tile_keys = tensor ? X::KEYS : S::KEYS;
        l.ctas = tensor ? SMS : SMS * S::CTAS;
        while (1 << l.row_shift < l.tile_rows) l.row_shift++;
        while (1 << l.key_shift < l.tile_keys) l.key_shift++;
        l.seqs = own ? batch->seqs : 0;
        l.front_tiles = front ? (int)(((int64_t)batch->prefix_len + l.tile_keys - 1) / l.tile_keys) : 0;
        l.front_units = l.front_tiles ? (rows + l.tile_rows - 1) / l.tile_rows * pages->kv_heads : 0;
        if (tensor && !own && l.front_units > 0 && l.front_units <= SMS) {   // (as many CTAs for each unit, as in paged.cu)
            const int even = SMS / (int)l.front_units * (int)l.front_units;
            if (even * 16 >= SMS * 15) l.ctas = even;
        }
        place_line(l, rows, pages->kv_heads, pages->head_size, base, c.bytes);
    };
    const bool one = batch->prefix_len == 0 || which.own_tensor == which.front_tensor;
    line(c.own, which.own_tensor, true, one);
    if (one) c.front = c.own;
    else line(c.front, true, false, true);
    return c;
}
// Tensor maps of the codes for boxes of S::BOX columns, if there are any (boxes.rows stays 0 otherwise): rows of a box are the most that divide a page and a warp's keys
template <typename S> void box_maps8(const lmrs_b200_pages8_t* pages, Boxes8& boxes) {
    typedef CUresult (*Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                               CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess ? (Encode)f : nullptr;
    }();
    int rows = S::WARP_KEYS;
    while (rows > 1 && pages->page_size % rows) rows /= 2;
    if (!encode || 2 * (S::WARP_KEYS / rows) * (S::KV / S::WARP_KEYS / S::BOX) > 32) return;   // (a box a lane)
    auto map = [&](CUtensorMap* m, void* base, int64_t page, int64_t slot, int64_t head, int& place_at, int& head_at) {
        struct { int64_t stride; cuuint64_t n; cuuint32_t box; int what; } d[3] = {{slot, (cuuint64_t)pages->page_size, (cuuint32_t)rows, 0}, {head, (cuuint64_t)pages->kv_heads, 1, 1},
                                                                              {page, (cuuint64_t)pages->pages, 1, 2}};
        std::sort(d, d + 3, [](const auto& a, const auto& b) { return a.stride < b.stride; });
        const cuuint64_t dims[4] = {(cuuint64_t)pages->head_size, d[0].n, d[1].n, d[2].n};
        const cuuint64_t strides[3] = {(cuuint64_t)d[0].stride, (cuuint64_t)d[1].stride, (cuuint64_t)d[2].stride};
        const cuuint32_t box[4] = {(cuuint32_t)S::BOX, d[0].box, d[1].box, d[2].box}, step[4] = {1, 1, 1, 1};
        for (int i = 0; i < 3; i++) {
            if (d[i].what == 0) place_at = i;
            if (d[i].what == 1) head_at = i;
            if (strides[i] == 0 || strides[i] % 16 || strides[i] >= (1ull << 40)) return false;
        }
        return encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, base, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, S::BOX == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                      CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    };
    if (map(&boxes.k, pages->k, pages->k_page, pages->k_slot, pages->k_head, boxes.k_place, boxes.k_head) &&
        map(&boxes.v, pages->v, pages->v_page, pages->v_slot, pages->v_head, boxes.v_place, boxes.v_head))
        boxes.rows = rows;
}
// f(type, form, padded head size, rows of a unit in eights, which kernels)
template <typename F> int by_shape8(const lmrs_b200_pages8_t* pages, const lmrs_b200_batch_t* batch, int dtype, int64_t n_rows, int q_heads, F f) {
    return by_type(dtype, [&](auto t) {
        return by_form(pages->form, [&](auto form) {
            auto by_tiles = [&](auto d) {
                const Which8 w = which8<decltype(d)::value>(pages, batch, dtype, n_rows, q_heads);
                return w.row_tiles == 1 ? f(t, form, d, std::integral_constant<int, 1>(), w) : f(t, form, d, std::integral_constant<int, 2>(), w);
            };
            return pages->head_size <= 64 ? by_tiles(std::integral_constant<int, 64>()) : pages->head_size <= 128 ? by_tiles(std::integral_constant<int, 128>()) : by_tiles(std::integral_constant<int, 256>());
        });
    });
}

}  // namespace

extern "C" int lmrs_b200_paged8_attention_workspace(const lmrs_b200_pages8_t* pages, const lmrs_b200_batch_t* batch, int dtype, int64_t n_rows, int q_heads, size_t* bytes) {
    static const char* me = "paged8_attention_workspace";
    return guarded(me, [&]() -> int {
        if (!bytes) return refuse(me, "null argument");
        const std::string why = bad_attention8(pages, batch, dtype, n_rows, q_heads);
        if (!why.empty()) return refuse(me, why);
        *bytes = 0;
        if (n_rows == 0 || batch->seqs == 0) return 0;
        return by_shape8(pages, batch, dtype, n_rows, q_heads, [&](auto t, auto, auto d, auto tiles, const Which8& which) {
            *bytes = cutting8<decltype(t), decltype(d)::value, decltype(tiles)::value>(pages, batch, n_rows, q_heads, which, nullptr).bytes;
            return 0;
        });
    });
}

extern "C" int lmrs_b200_paged8_attention(const lmrs_b200_pages8_t* pages, const lmrs_b200_batch_t* batch, int dtype, int64_t n_rows, const lmrs_b200_rows_t* q, const lmrs_b200_rows_t* out,
                                          int q_heads, float scale, float softcap, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
    static const char* me = "paged8_attention";
    return guarded(me, [&]() -> int {
        std::string why = bad_attention8(pages, batch, dtype, n_rows, q_heads);
        if (why.empty() && !isfinite(scale)) why = "scale is not finite";
        if (why.empty() && !(softcap >= 0.0f && isfinite(softcap))) why = "softcap must be 0 (none) or positive";
        if (why.empty() && q && out && meet(q, q_heads, out, q_heads, n_rows, pages->head_size, dtype)) why = "out lies where q does, which is read until the call has ended";
        if (!why.empty()) return refuse(me, why);
        int device = 0;
        if (!device_sms(me, &device)) return 1;
        if (n_rows == 0 || batch->seqs == 0) return 0;
        why = bad_batch_memory(batch, device);
        if (why.empty()) why = bad_rows(q, "q", dtype, device);
        if (why.empty()) why = bad_rows(out, "out", dtype, device);
        if (why.empty() && lse && (!aligned(lse, 4) || !on_device(lse, device))) why = "lse is not memory of the current device";
        if (why.empty()) why = bad_pages8_memory(pages, device);
        if (why.empty() && (!workspace || !aligned(workspace, 256) || !on_device(workspace, device))) why = "workspace is not memory of the current device on a 256-byte boundary";
        if (!why.empty()) return refuse(me, why);
        if (const int status = gave_up_word.take()) return refuse(me, "results of an earlier call are NaN: " + dense::tg_gave_up(status));
        return by_shape8(pages, batch, dtype, n_rows, q_heads, [&](auto t, auto form, auto d, auto tiles, const Which8& which) {
            using T = decltype(t);
            constexpr int FORM = decltype(form)::value, DP = decltype(d)::value, ROW_TILES = decltype(tiles)::value;
            using S = TileShape8<T, DP, ROW_TILES>;
            const Cutting8 c = cutting8<T, DP, ROW_TILES>(pages, batch, n_rows, q_heads, which, (char*)workspace);
            if (workspace_bytes < c.bytes) return refuse(me, "workspace has " + std::to_string(workspace_bytes) + " bytes, the call needs " + std::to_string(c.bytes));
            Attn8Params<T> p = {};
            p.batch = batch8_as(batch, pages, n_rows);
            p.q = rows_as<const T>(q);
            p.out = rows_as<T>(out);
            p.c = pages8_as(pages);
            p.kv_heads = pages->kv_heads; p.q_heads = q_heads; p.head_size = pages->head_size; p.group = q_heads / pages->kv_heads;
            // At the ends of float32: a cap beyond 2^100 is one of 2^100 (scores of up to 2^88 are not moved by either, and its product with log2 e is finite), and no score is 0 times infinity
            const float cap = std::min(softcap, 0x1p100f);
            p.scale2 = std::max(-FLT_MAX, std::min(FLT_MAX, scale * LOG2E)); p.softcap = cap; p.cap_in = cap > 0.0f ? std::max(-FLT_MAX, std::min(FLT_MAX, scale / cap)) : 0.0f; p.lse = lse;
            p.q_wide = vectors(q, dtype);
            p.out_wide = aligned(out->data, 4 * sizeof(T)) && out->row % 4 == 0 && out->head % 4 == 0;
            p.whole = batch->prefix_len == 0;
            p.page_shift = p.block_shift = -1;
            for (int i = 0; i < 31; i++) {
                if (pages->page_size == 1 << i) p.page_shift = i;
                if (pages->block == 1 << i) p.block_shift = i;
            }
            if (!(p.err = gave_up_word.get())) return refuse(me, "out of host memory");
            static std::atomic<uint64_t> allowed{0}, allowed_tensor{0};
            cudaError_t e = cudaSuccess;
            const bool tensor = which.own_tensor || which.front_tensor;
            if constexpr (sizeof(T) == 2)
                if (tensor) {
                    auto kernel = codes128_kernel<T, FORM, DP>;
                    using X = TensorShape8<DP>;
                    if ((e = allow_smem(kernel, device, X::SMEM, allowed_tensor)) != cudaSuccess) return refuse(me, cudaGetErrorString(e));
                    Boxes8 boxes = {};
                    box_maps8<X>(pages, boxes);
                    const Line& line = which.own_tensor ? c.own : c.front;
                    kernel<<<(unsigned)line.ctas, X::THREADS, X::SMEM, (cudaStream_t)stream>>>(p, line, boxes);
                    if (launched(me)) return 1;
                }
            if (!which.own_tensor) {
                auto kernel = rows8_kernel<T, FORM, DP, ROW_TILES>;
                if ((e = allow_smem(kernel, device, S::SMEM, allowed)) != cudaSuccess) return refuse(me, cudaGetErrorString(e));
                Boxes8 boxes = {};
                box_maps8<S>(pages, boxes);
                if (tensor) e = launch_after(kernel, (unsigned)c.own.ctas, S::THREADS, S::SMEM, (cudaStream_t)stream, p, c.own, boxes);
                else kernel<<<(unsigned)c.own.ctas, S::THREADS, S::SMEM, (cudaStream_t)stream>>>(p, c.own, boxes);
                if (e != cudaSuccess) return refuse(me, std::string("launch failed: ") + cudaGetErrorString(e));
                if (launched(me)) return 1;
            }
            // (which join, as in paged.cu)
            const int64_t items = n_rows * q_heads;
            constexpr int COLS = DP <= 128 ? 1 : 2;
            const AttnParams<T>& rows = p;
            e = items <= SMS * 4 ? launch_after(join_kernel<T, 8, COLS>, (unsigned)items, 256, 0, (cudaStream_t)stream, rows, c.front, c.own)
                                 : launch_after(join_kernel<T, 1, COLS>, (unsigned)std::min<int64_t>((items + 7) / 8, SMS * 16), 256, 0, (cudaStream_t)stream, rows, c.front, c.own);
            return e == cudaSuccess ? 0 : refuse(me, std::string("launch failed: ") + cudaGetErrorString(e));
        });
    });
}
