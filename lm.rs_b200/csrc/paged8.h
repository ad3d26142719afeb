// paged8.h -- pages that hold keys and values in 8 bits (paged8_rows.cuh writes them and reads them back, paged8_attn.cuh and paged8_tensor.cuh attend over them): the two formats of a code, how
// codes become numbers and numbers codes, and the pool as the kernels see it.
//
// A code c stands for c * scale.  int8: c is the whole number -127 .. 127 itself.  e4m3: a sign, four bits of exponent (biased by 7) and three of mantissa, up to 448; 0x7f and 0xff are NaN
// and are never written here.  Both formats' numbers are whole in float16 (11 bits of mantissa, exponents from 2^-24 to 2^15), where the tensor cores take them.
#pragma once
#include "paged.h"

namespace lmrs {
namespace paged {

enum { FORM_INT8 = 0, FORM_E4M3 = 1 };
template <int FORM> constexpr float FORM_MOST = FORM == FORM_INT8 ? 127.0f : 448.0f;
// Scales that are written stay within these, and scales of values that are read count as the nearest of them: weights times scales then stay within float32 (paged8_attn.cuh)
constexpr float SCALE_LEAST = 0x1p-60f, SCALE_MOST = 0x1p60f;

struct Pages8 {
    uint8_t *k, *v;
    float *ks, *vs;
    int64_t k_page, k_slot, k_head, v_page, v_slot, v_head, ks_page, ks_block, ks_head, vs_page, vs_block, vs_head;
    int kv_heads, head_size, block;   // block: tokens of a page that share a scale
};

// two codes (the lower 16 bits of w) as float16
PG_DEVINL uint32_t e4m3_pair(uint32_t w) {
    uint32_t r;
    asm("{.reg .b16 h; cvt.u16.u32 h, %1; cvt.rn.f16x2.e4m3x2 %0, h;}" : "=r"(r) : "r"(w));
    return r;
}
PG_DEVINL float2 half_pair(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
// four codes as floats
template <int FORM> PG_DEVINL float4 open_codes(uint32_t w) {
    if (FORM == FORM_INT8) return make_float4((float)(int8_t)w, (float)(int8_t)(w >> 8), (float)(int8_t)(w >> 16), (float)(int8_t)(w >> 24));
    const float2 a = half_pair(e4m3_pair(w)), b = half_pair(e4m3_pair(w >> 16));
    return make_float4(a.x, a.y, b.x, b.y);
}
template <int FORM> PG_DEVINL float open_code(uint8_t c) { return FORM == FORM_INT8 ? (float)(int8_t)c : half_pair(e4m3_pair(c)).x; }

// y / s to the format's nearest number, ties to even.  by: 1 / s to the nearest; y by is off by 2^-51 of itself at most, so whoever lies further from the middle of two numbers than that is on the right
// side of it, and the others (ties, most of them: y and s have few bits where y is a 16-bit input) take the division, which rounds a tie to itself
template <int FORM> PG_DEVINL uint8_t close_code(double y, double s, double by) {
    double r = y * by;
    int e = 0;   // numbers around r are whole multiples of 2^e
    if (FORM == FORM_E4M3) e = max((__double2hiint(r) >> 20 & 0x7ff) - 1023, -6) - 3;
    const double up = __hiloint2double((1023 - e) << 20, 0);   // (e is -9 at least; what lies above 448 is cut off below, so a large e need only be finite here)
    double t = r * up, n = rint(t);
    if (fabs(fabs(t - n) - 0.5) < 1e-9) n = rint(y / s * up);
    if (FORM == FORM_INT8) return (uint8_t)(int8_t)(int)fmin(fmax(n, -127.0), 127.0);   // (NaN: -127, of a block whose scale is NaN)
    const float v = (float)(n * __hiloint2double((1023 + e) << 20, 0));
    uint16_t c;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %1;" : "=h"(c) : "f"(v == v ? v : 0.0f));
    return (uint8_t)c;
}
// the scale of a block whose largest size is a (64 bits); NaN and infinity: NaN, so that all of the block reads as NaN
template <int FORM> PG_DEVINL float scale_for(double a) {
    if (!(a <= 1.7976931348623157e308)) return __int_as_float(0x7fffffff);
    return (float)fmin(fmax(a / (double)FORM_MOST<FORM>, (double)SCALE_LEAST), (double)SCALE_MOST);
}

}  // namespace paged
}  // namespace lmrs
