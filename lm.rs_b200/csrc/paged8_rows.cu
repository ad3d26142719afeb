// paged8_rows.cu -- entry points of include/lmrs_b200.h for norms with rotary positions, and for writing pages of 8-bit codes and reading them back: checks of the arguments, choice of the kernels, launches.
// Device pointers, the caller's stream; nothing here allocates, synchronises or remembers anything from one call to the next.
#include <math.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "paged8_checks.h"
#include "paged8_rows.cuh"

using namespace lmrs;
using namespace lmrs::paged;

namespace {

std::string bad_weight(const float* w, int64_t head, const char* name, int device) {
    if (!w) return "";
    if (!aligned(w, 4)) return std::string(name) + " does not lie on a boundary of its elements";
    if (head < 0) return std::string("negative stride of ") + name;
    return on_device(w, device) ? "" : std::string(name) + " is not memory of the current device";
}
bool wide_weight(const HeadNorm& n) { return !n.weight || (aligned(n.weight, 16) && n.head % 4 == 0); }
// do the rows r lie over any of n bytes from p on?
bool over(const lmrs_b200_rows_t* r, int64_t n_rows, int64_t heads, int64_t head_size, int dtype, const void* p, int64_t bytes) {
    if (!p || !r || n_rows < 1 || heads < 1) return false;
    typedef __int128 wide;
    const wide a = (wide)(uintptr_t)r->data, b = (wide)(uintptr_t)p, end = a + ((wide)(n_rows - 1) * r->row + (wide)(heads - 1) * r->head + head_size) * (wide)size_of(dtype);
    return a < b + bytes && b < end;
}
// Eight elements a lane: sizes in eights, pairs in fours, and rows on boundaries of four elements
bool fours(const void* p, int64_t row, int64_t head, int64_t size) { return aligned(p, 4 * size) && row % 4 == 0 && head % 4 == 0; }
bool fours(const lmrs_b200_rows_t* r, int dtype) { return fours(r->data, r->row, r->head, (int64_t)size_of(dtype)); }
bool eights(int head_size, int pairs) { return head_size % 8 == 0 && pairs % 4 == 0; }
template <typename K> struct Kind { typedef K type; };
// lanes that a head takes: f(8, 16 or 32)
template <typename F> int by_lanes(int head_size, F f) {
    return head_size <= 64 ? f(std::integral_constant<int, 8>()) : head_size <= 128 ? f(std::integral_constant<int, 16>()) : f(std::integral_constant<int, 32>());
}
int lanes_of(int head_size) { return head_size <= 64 ? 8 : head_size <= 128 ? 16 : 32; }
// warps that share a row's heads: one, or more where rows alone would not give every SM's schedulers a few each
int norm_parts(int64_t n_rows, int heads, int at_once, int sms) {
    return (int)std::max<int64_t>(1, std::min<int64_t>(((int64_t)sms * 16 + n_rows - 1) / n_rows, (heads + at_once - 1) / at_once));
}

}  // namespace

extern "C" int lmrs_b200_norm_rope(const lmrs_b200_rope_t* rope, int dtype, const lmrs_b200_rows_t* x, const lmrs_b200_rows_t* out, int64_t n_rows, int heads, int head_size, const float* weight,
                                   int64_t weight_head, float eps, const lmrs_b200_positions_t* pos, void* stream) {
    static const char* me = "norm_rope";
    return guarded(me, [&]() -> int {
        if (!x || !out) return refuse(me, "null argument");
        std::string why = bad_dtype(dtype);
        if (!why.empty()) return refuse(me, why);
        if (n_rows < 0 || n_rows > 0x7fffffff || heads < 0 || heads > MAX_HEADS || head_size < 1 || head_size > 256)
            return refuse(me, "n_rows must be 0 .. 2^31 - 1, heads 0 .. 65535, head_size 1 .. 256");
        if (rope) why = bad_rope(rope, head_size);
        if (why.empty() && (rope != nullptr) != (pos != nullptr)) why = "rope and positions come together";
        if (why.empty() && !(eps >= 0.0f && isfinite(eps))) why = "eps must be 0 or positive";
        if (why.empty() && !same(x, out, n_rows, heads) && meet(x, heads, out, heads, n_rows, head_size, dtype)) why = "out lies over x without being x itself";
        if (why.empty() && over(out, n_rows, heads, head_size, dtype, weight, 4 * ((int64_t)(heads - 1) * std::max<int64_t>(weight_head, 0) + head_size))) why = "out lies over the weights";
        if (!why.empty()) return refuse(me, why);
        int device = 0;
        const int sms = device_sms(me, &device);
        if (!sms) return 1;
        if (n_rows == 0 || heads == 0) return 0;
        why = bad_rows(x, "x", dtype, device);
        if (why.empty()) why = bad_rows(out, "out", dtype, device);
        if (why.empty()) why = bad_weight(weight, weight_head, "weight", device);
        if (why.empty() && pos) why = !pos->data ? "null positions" : bad_ints(pos->data, "positions", device);
        if (!why.empty()) return refuse(me, why);
        const HeadNorm norm = {weight, weight_head, eps, 1};
        const lmrs_b200_rope_t none = {};
        return by_type(dtype, [&](auto t) {
            using T = decltype(t);
            const int pairs = rope ? rope->pairs : 0;
            const bool wide = fours(x, dtype) && fours(out, dtype) && wide_weight(norm) && eights(head_size, pairs);
            const int parts = norm_parts(n_rows, heads, wide ? 32 / lanes_of(head_size) : 1, sms);
            auto go = [&](auto lanes) {
                norm_rope_kernel<T, decltype(lanes)::value><<<warps_grid(n_rows * parts, sms), 32 * ROW_WARPS, 0, (cudaStream_t)stream>>>(
                    rope ? *rope : none, rows_as<const T>(x), rows_as<T>(out), n_rows, heads, head_size, norm, pos_as(pos), parts);
                return launched(me);
            };
            return wide ? by_lanes(head_size, go) : go(std::integral_constant<int, 0>());
        });
    });
}

extern "C" int lmrs_b200_paged8_append(const lmrs_b200_pages8_t* pages, const lmrs_b200_batch_t* batch, int dtype, int64_t n_rows, const lmrs_b200_rows_t* k, const lmrs_b200_rows_t* v,
                                       const lmrs_b200_rope_t* rope, const lmrs_b200_positions_t* pos, const lmrs_b200_rows_t* q, const lmrs_b200_rows_t* q_out, int q_heads,
                                       const lmrs_b200_norms_t* norms, void* stream) {
    static const char* me = "paged8_append";
    return guarded(me, [&]() -> int {
        std::string why = bad_pages8(pages);
        if (why.empty()) why = bad_dtype(dtype);
        if (why.empty()) why = bad_batch(batch, n_rows, pages->page_size);
        if (why.empty() && (q || q_out) && (!q || !q_out)) why = "q and q_out come together";
        if (why.empty() && q && !rope && !(norms && norms->q)) why = "q without rope or a norm";
        if (why.empty() && q && (q_heads < 1 || q_heads > MAX_HEADS)) why = "q_heads must be 1 .. 65535";
        if (why.empty() && rope) why = bad_rope(rope, pages->head_size);
        if (why.empty() && norms && !(norms->eps >= 0.0f && isfinite(norms->eps))) why = "eps must be 0 or positive";
        const int size = why.empty() ? pages->head_size : 0;
        if (why.empty() && q && !same(q, q_out, n_rows, q_heads) && meet(q, q_heads, q_out, q_heads, n_rows, size, dtype)) why = "q_out lies over q without being q itself";
        if (why.empty() && q && k && v && (meet(k, pages->kv_heads, q_out, q_heads, n_rows, size, dtype) || meet(v, pages->kv_heads, q_out, q_heads, n_rows, size, dtype)))
            why = "q_out lies over k or v";
        if (why.empty() && q && norms && (over(q_out, n_rows, q_heads, size, dtype, norms->q, 4 * ((int64_t)(q_heads - 1) * std::max<int64_t>(norms->q_head, 0) + size)) ||
                                          over(q_out, n_rows, q_heads, size, dtype, norms->k, 4 * ((int64_t)(pages->kv_heads - 1) * std::max<int64_t>(norms->k_head, 0) + size))))
            why = "q_out lies over the weights";
        if (!why.empty()) return refuse(me, why);
        int device = 0;
        const int sms = device_sms(me, &device);
        if (!sms) return 1;
        if (n_rows == 0 || batch->seqs == 0) return 0;
        why = bad_batch_memory(batch, device);
        if (why.empty()) why = bad_rows(k, "k", dtype, device);
        if (why.empty()) why = bad_rows(v, "v", dtype, device);
        if (why.empty() && q) why = bad_rows(q, "q", dtype, device);
        if (why.empty() && q) why = bad_rows(q_out, "q_out", dtype, device);
        if (why.empty() && pos) why = !pos->data ? "null positions" : bad_ints(pos->data, "positions", device);
        if (why.empty() && norms) why = bad_weight(norms->k, norms->k_head, "the keys' weight", device);
        if (why.empty() && norms) why = bad_weight(norms->q, norms->q_head, "the queries' weight", device);
        if (why.empty()) why = bad_pages8_memory(pages, device);
        if (!why.empty()) return refuse(me, why);
        return by_type(dtype, [&](auto t) {
            using T = decltype(t);
            return by_form(pages->form, [&](auto form) {
                PutParams<T> p = {};
                if (rope) p.rope = *rope;
                p.batch = batch8_as(batch, pages, n_rows);
                p.pos = pos_as(rope ? pos : nullptr);
                p.k = rows_as<const T>(k);
                p.v = rows_as<const T>(v);
                if (q) { p.q = rows_as<const T>(q); p.q_out = rows_as<T>(q_out); p.q_heads = q_heads; }
                p.pages = pages8_as(pages);
                if (norms) {
                    p.k_norm = HeadNorm{norms->k, norms->k_head, norms->eps, norms->k != nullptr};
                    p.q_norm = HeadNorm{norms->q, norms->q_head, norms->eps, norms->q != nullptr};
                }
                const int pairs = rope ? rope->pairs : 0;
                const bool wide = eights(size, pairs) && fours(k, dtype) && fours(v, dtype) && (!q || (fours(q, dtype) && fours(q_out, dtype))) && wide_weight(p.k_norm) && wide_weight(p.q_norm) &&
                                  fours(pages->k, pages->k_page | pages->k_slot, pages->k_head, 1) && fours(pages->v, pages->v_page | pages->v_slot, pages->v_head, 1);
                p.parts = norm_parts(n_rows, q_heads, wide ? 32 / lanes_of(size) : 1, sms);
                // A CTA takes as many rows as a block has where that leaves a few CTAs for each SM (there is about one leader among them), and half as many heads where rows are few
                p.window = (int)std::max<int64_t>(1, std::min<int64_t>(pages->block, n_rows / ((int64_t)sms * 4)));
                p.windows = (int)((n_rows + p.window - 1) / p.window);
                p.heads = std::min(pages->kv_heads, (int64_t)p.windows * ((pages->kv_heads + PUT_WARPS - 1) / PUT_WARPS) < 2 * sms ? PUT_WARPS / 2 : PUT_WARPS);
                p.head_ctas = (pages->kv_heads + p.heads - 1) / p.heads;
                if ((int64_t)p.windows * p.head_ctas > 0x3fffffff) return refuse(me, "n_rows * kv_heads is too large");
                p.put_ctas = p.windows * p.head_ctas;
                // Queries in the same kernel where there are few: a second launch takes longer than they do
                const bool apart = q && n_rows * q_heads > 1 << 14;
                const int q_ctas = q && !apart ? (int)std::min<int64_t>((n_rows * p.parts + PUT_WARPS - 1) / PUT_WARPS, (int64_t)sms * 16) : 0;
                p.ctas = p.put_ctas + q_ctas;
                constexpr int FORM = decltype(form)::value;
                auto launch = [&](auto put) {
                    using Put = typename decltype(put)::type;
                    cudaError_t e = cudaSuccess;
                    if (apart) {
                        put_queries_kernel<T, Put::LANES><<<(unsigned)std::min<int64_t>((n_rows * p.parts + ROW_WARPS - 1) / ROW_WARPS, (int64_t)sms * QUERY_CTAS), 32 * ROW_WARPS, 0, (cudaStream_t)stream>>>(p);
                        if (launched(me)) return 1;
                        e = launch_after(paged8_append_kernel<T, FORM, Put>, (unsigned)p.ctas, 32 * PUT_WARPS, 0, (cudaStream_t)stream, p);
                    } else {
                        paged8_append_kernel<T, FORM, Put><<<(unsigned)p.ctas, 32 * PUT_WARPS, 0, (cudaStream_t)stream>>>(p);
                        e = cudaGetLastError();
                    }
                    return e == cudaSuccess ? 0 : refuse(me, std::string("launch failed: ") + cudaGetErrorString(e));
                };
                // Few tokens of a block in a call: as many as a warp's lanes take at once, with half the registers
                const int64_t together = std::min<int64_t>(std::min<int64_t>(batch->max_rows, n_rows), pages->block);
                if (wide) return by_lanes(size, [&](auto lanes) {
                    constexpr int L = decltype(lanes)::value;
                    return together <= 32 / L ? launch(Kind<PutEight<T, FORM, L, 1>>()) : launch(Kind<PutEight<T, FORM, L, L == 8 ? 4 : 8>>());
                });
                return size <= 64 ? launch(Kind<PutOne<T, FORM, 1>>()) : size <= 128 ? launch(Kind<PutOne<T, FORM, 2>>()) : launch(Kind<PutOne<T, FORM, 4>>());
            });
        });
    });
}

extern "C" int lmrs_b200_paged8_read(const lmrs_b200_pages8_t* pages, const lmrs_b200_batch_t* batch, int dtype, int64_t n_rows, const lmrs_b200_rows_t* k, const lmrs_b200_rows_t* v, void* stream) {
    static const char* me = "paged8_read";
    return guarded(me, [&]() -> int {
        std::string why = bad_pages8(pages);
        if (why.empty()) why = bad_dtype(dtype);
        if (why.empty()) why = bad_batch(batch, n_rows, pages->page_size);
        if (why.empty() && (!k || !v)) why = "null argument";
        if (why.empty() && meet(k, pages->kv_heads, v, pages->kv_heads, n_rows, pages->head_size, dtype)) why = "k lies over v";
        if (!why.empty()) return refuse(me, why);
        int device = 0;
        const int sms = device_sms(me, &device);
        if (!sms) return 1;
        if (n_rows == 0 || batch->seqs == 0) return 0;
        why = bad_batch_memory(batch, device);
        if (why.empty()) why = bad_rows(k, "k", dtype, device);
        if (why.empty()) why = bad_rows(v, "v", dtype, device);
        if (why.empty()) why = bad_pages8_memory(pages, device);
        if (!why.empty()) return refuse(me, why);
        return by_type(dtype, [&](auto t) {
            using T = decltype(t);
            return by_form(pages->form, [&](auto form) {
                ReadParams<T> p = {batch8_as(batch, pages, n_rows), pages8_as(pages), rows_as<T>(k), rows_as<T>(v)};
                const bool wide = wide_codes(pages) && vectors(k, dtype) && vectors(v, dtype);
                (wide ? paged8_read_kernel<T, decltype(form)::value, 16> : paged8_read_kernel<T, decltype(form)::value, 1>)<<<warps_grid(n_rows, sms), 32 * ROW_WARPS, 0, (cudaStream_t)stream>>>(p);
                return launched(me);
            });
        });
    });
}

