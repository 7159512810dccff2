// Rows to integers with a scale each:  s = max|x| / 127 (fp32),  q = round(x / s), ties to even.
//
// The quotient's rounding is the exact one: a product with 1 / s decides all but the values next to a half (it is off by
// 127 * 2^-23 at most), and there the remainder decides.  A row of zeros has the scale 0.  A row that holds an infinity or
// a NaN has the scale NaN: whatever is made of it is NaN.
#pragma once

#include "common.cuh"

namespace fwb {
namespace int8 {

constexpr int CHUNK = 8;                 // elements a thread takes at once
// A row of smaller values alone is taken as zeros: 127 * 2^-125, from where on half of the scale is a normal number and so every
// remainder beside it exact.
constexpr float TINY_ROW = 0x1.fcp-119f;

struct RowScale {
    float stored;                // what goes with the row
    float s, inv;                // what its values are divided and multiplied by; inv 0: integers 0
    bool checked;                // see quantize
};
// `top`: the largest magnitude's bits (in their order infinity lies above every number and NaN above infinity); `short_values`: the
// row's values have eight bits (bfloat16).
__device__ __forceinline__ RowScale row_scale(unsigned top, bool short_values) {
    const float most = __uint_as_float(top);
    const bool finite = top < 0x7f800000u, zero = most < TINY_ROW;
    RowScale r;
    r.s = most / 127.0f;
    r.inv = !finite || zero ? 0.0f : 1.0f / r.s;
    r.stored = !finite ? __int_as_float(0x7fffffff) : zero ? 0.0f : r.s;
    // which side of its half a tie of a bfloat16 row lies on: s above m / 127, towards zero; s below, away from it
    const float above = fmaf(r.s, 127.0f, -most);
    r.checked = !short_values || above == 0.0f;
    if (!r.checked) r.inv = fmaf(r.inv, above > 0.0f ? -0x1p-22f : 0x1p-22f, r.inv);
    return r;
}

// Eight values' integers.
//
// Checked: n = x (1 / s) rounded is the integer or its neighbour; e = x - n s has no rounding error (a multiple of the smaller
// of x's and s's last places, and at most about s / 2), so |e| against s / 2 tells.
//
// Not checked, for values of eight bits under a maximum m of eight bits (bfloat16 rows): with x = a 2^i, m = b 2^j and whole a, b below 256,
// i <= j, the quotient x / (m / 127) is a tie where 254 a = (2 n + 1) b 2^(j - i), and else the two sides, whole numbers, differ by 1 or
// more: the quotient is 1 / (254 a) of itself, more than 2^-16, away from a tie.  s is m / 127 rounded, so the ties all lie on one side of
// their halves, by 2^-24 of themselves at most; `inv` is 1 / s moved by 2^-22 of itself towards that side (with the roundings of s, of
// 1 / s and of the move less than 2^-21 in all), which decides every tie and nothing else.
template <bool CHECKED>
__device__ __forceinline__ uint2 quantize_by(const float (&v)[CHUNK], float s, float inv) {
    constexpr float ROUND = 12582912.0f;               // 1.5 * 2^23
    uint32_t word[CHUNK];
    float off = 0.0f;
#pragma unroll
    for (int i = 0; i < CHUNK; ++i) {
        const float n = fmaf(v[i], inv, ROUND);
        word[i] = __float_as_uint(n);
        if (CHECKED) off = fmaxf(off, fabsf(fmaf(-__fsub_rn(n, ROUND), s, v[i])));
    }
    const float half = 0.5f * s;
    if (CHECKED && off >= half) {
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) {
            const float n = __uint_as_float(word[i]), e = fmaf(-__fsub_rn(n, ROUND), s, v[i]);
            if (fabsf(e) > half || (fabsf(e) == half && (word[i] & 1))) word[i] += e > 0.0f ? 1 : -1;
        }
    }
    uint2 packed;
    packed.x = __byte_perm(__byte_perm(word[0], word[1], 0x0040), __byte_perm(word[2], word[3], 0x0040), 0x5410);
    packed.y = __byte_perm(__byte_perm(word[4], word[5], 0x0040), __byte_perm(word[6], word[7], 0x0040), 0x5410);
    return packed;
}

__device__ __forceinline__ uint2 quantize(const float (&v)[CHUNK], const RowScale& r) {
    const uint2 packed = r.checked ? quantize_by<true>(v, r.s, r.inv) : quantize_by<false>(v, r.s, r.inv);
    return r.inv == 0.0f ? make_uint2(0, 0) : packed;
}

}  // namespace int8
}  // namespace fwb
