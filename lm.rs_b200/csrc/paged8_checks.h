// paged8_checks.h -- what the entry points over 8-bit pages share on the host (paged8.cu, paged8_rows.cu)
#pragma once
#include "paged8.h"
#include "paged_checks.h"

namespace lmrs {
namespace paged {

inline std::string bad_pages8(const lmrs_b200_pages8_t* p) {
    if (!p || !p->k || !p->v || !p->k_scale || !p->v_scale) return "null pages";
    if (p->form != FORM_INT8 && p->form != FORM_E4M3) return "form must be 0 (int8) or 1 (e4m3)";
    if (p->pages < 1 || p->page_size < 1 || p->kv_heads < 1 || p->kv_heads > MAX_HEADS) return "pages, page_size and kv_heads must be positive, kv_heads at most 65535";
    if (p->head_size < 1 || p->head_size > 256) return "head_size must be 1 .. 256";
    if (p->block < 1 || p->page_size % p->block) return "block must divide page_size";
    if (p->k_page < 0 || p->k_slot < 0 || p->k_head < 0 || p->v_page < 0 || p->v_slot < 0 || p->v_head < 0 || p->ks_page < 0 || p->ks_block < 0 || p->ks_head < 0 || p->vs_page < 0 || p->vs_block < 0 ||
        p->vs_head < 0)
        return "negative stride of pages";
    if (!aligned(p->k_scale, 4) || !aligned(p->v_scale, 4)) return "the scales do not lie on a boundary of their elements";
    return "";
}
inline std::string bad_pages8_memory(const lmrs_b200_pages8_t* p, int device) {
    if (!on_device(p->k, device) || !on_device(p->v, device)) return "the pages are not memory of the current device";
    return on_device(p->k_scale, device) && on_device(p->v_scale, device) ? "" : "the scales are not memory of the current device";
}
inline Pages8 pages8_as(const lmrs_b200_pages8_t* p) {
    return Pages8{(uint8_t*)p->k, (uint8_t*)p->v, p->k_scale, p->v_scale, p->k_page, p->k_slot, p->k_head, p->v_page, p->v_slot, p->v_head,
                  p->ks_page, p->ks_block, p->ks_head, p->vs_page, p->vs_block, p->vs_head, p->kv_heads, p->head_size, p->block};
}
inline Batch batch8_as(const lmrs_b200_batch_t* b, const lmrs_b200_pages8_t* p, int64_t n_rows) {
    return Batch{b->lens, b->rows, b->tables, b->prefix, b->table_stride, b->seqs, b->table_len, b->prefix_len, p->pages, p->page_size, n_rows};
}
template <typename F> int by_form(int form, F f) { return form == FORM_INT8 ? f(std::integral_constant<int, FORM_INT8>()) : f(std::integral_constant<int, FORM_E4M3>()); }
// do all codes that a head's begin with lie on 16-byte boundaries, and heads have whole pieces of 16?
inline bool wide_codes(const lmrs_b200_pages8_t* p) {
    return p->head_size % 16 == 0 && aligned(p->k, 16) && aligned(p->v, 16) && p->k_page % 16 == 0 && p->k_slot % 16 == 0 && p->k_head % 16 == 0 && p->v_page % 16 == 0 && p->v_slot % 16 == 0 &&
           p->v_head % 16 == 0;
}

}  // namespace paged
}  // namespace lmrs
