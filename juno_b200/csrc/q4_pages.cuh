// 4-bit cache pages: layout and arithmetic.
//
// A group is kQ4Group neighbouring dimensions of one position and key/value head.  Its values are held as m + d q:
//   lo, hi   least and largest value (clamped to the range of FP16)
//   m        lo in FP16, d  (hi - lo) / 15 in BF16; 0 where hi - lo is below 2^-80
//   q        the whole number in [0, 15] nearest to (x - m) / d, ties to the even one, decided exactly
// d in BF16 has the whole FP32 range and widens with one AND; its 8 bits cost nothing, as q is found for the rounded d (the largest value of
// a group lies at most 15 d 2^-8 beyond the last number).  m needs the digits more: in FP16 a group far from zero loses what FP16 pages lose.
// A NaN makes its group NaN (m is NaN, d 0).
//
// The pages of a head (16 positions) are one block of 20 * hd bytes, [layer][page][kv_head] in the pool:
//   keys    codes  word [position][t][group], t = 0..3: the numbers of dimensions 8t .. 8t + 7 of the group, a unit of four to a half word
//           d      half word [position][group]
//           m      half word [position][group]
//   values  codes  half word [position][group][u], u = 0..7: the unit of dimensions 4u .. 4u + 3 of the group, in positions 8..15 of 15 - q: decode attention adds
//                  up (m + 15 d) - d (15 - q) there, so that its sums of numbers do not grow all one way; the 16-byte pieces of a position, one per group, are
//                  permuted so that eight positions' pieces of one group lie on different banks
//           d      half word [position][group]
//           m      half word [position][group]
// Every piece lies as the MMAs of decode attention want it: lane (g, t) of a warp finds the numbers of all groups of position g of the keys at 16 * lane
// (8 * lane for heads of 64), those of the values come by ldmatrix, and the keys' offsets are operands of an MMA as they are.
#pragma once
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "layout.cuh"

namespace juno {

constexpr int kQ4Group = 32;

JHD int q4_block_bytes(int hd) { return 20 * hd; }
JHD int q4_k_code(int hd, int p, int t, int g) { return ((p * 4 + t) * (hd / kQ4Group) + g) * 4; }
JHD int q4_k_step(int hd, int p, int g) { return 8 * hd + (p * (hd / kQ4Group) + g) * 2; }
JHD int q4_k_offset(int hd, int p, int g) { return 9 * hd + (p * (hd / kQ4Group) + g) * 2; }
JHD int q4_v_piece(int hd, int p, int g) { return g ^ (hd == 128 ? p >> 1 & 3 : p >> 2 & 1); }
JHD int q4_v_code(int hd, int p, int u, int g) { return 10 * hd + p * (hd / 2) + q4_v_piece(hd, p, g) * 16 + u * 2; }
JHD int q4_v_step(int hd, int p, int g) { return 18 * hd + (p * (hd / kQ4Group) + g) * 2; }
JHD int q4_v_offset(int hd, int p, int g) { return 19 * hd + (p * (hd / kQ4Group) + g) * 2; }
// A unit: the first number in bits 6..9, the second and third four bits higher and lower, the fourth's lower half in bits 14 and 15, its upper half in bits 0
// and 1.  Shifted by 4 either way, or with its bytes changed round, the half word has each of them in bits 6..9, the upper bits of an FP16 number's
// fraction: with an AND it is the FP16 number q 2^-18.
JHD uint32_t q4_unit(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return a << 6 | b << 10 | c << 2 | (d & 3u) << 14 | d >> 2; }
// 15 - q for q, all numbers of a word: what an XOR with this does.
JHD uint32_t q4_v_flip(int p) { return p & 8 ? 0xffffffffu : 0u; }

// The number of x in a group with offset m and step d, decided exactly (inv is about 1 / d).  s + r is x - m exactly; half-way points (q + 1/2) d have 13
// bits and are exact, so that the comparisons decide what the estimate may have missed by one.
JHD int q4_number_exact(float x, float m, float d, float inv) {
    if (!(d > 0.f)) return 0;
    const float s = x - m, a = s - x, r = (x - (s - a)) + (-m - a);
    const float guess = s * inv + 0.5f;
    int q = guess >= 15.f ? 15 : guess > 0.f ? (int)guess : 0;
    const float above = ((float)q + 0.5f) * d, below = ((float)q - 0.5f) * d;
    if (s > above || (s == above && (r > 0.f || (r == 0.f && (q & 1))))) q++;
    else if (s < below || (s == below && (r < 0.f || (r == 0.f && (q & 1))))) q--;
    return q < 0 ? 0 : q > 15 ? 15 : q;
}
// The same from an estimate (inv is about 1 / (15 d), 0 for d = 0), and how far that lies from its whole number.  t = (x - m) inv 15 is off by less than 2^-17
// (x - m and the product are rounded once, inv is off by two of its last digits, t <= 15.1), so a t farther than 2^-16 from half-way between two numbers has the
// right one next to it; where *off is above kQ4Near q4_number_exact decides.
JHD uint32_t q4_number_near(float x, float m, float inv, float *off) {
#if defined(__CUDA_ARCH__)
    const float part = __saturatef((x - m) * inv);
#else
    const float t = (x - m) * inv, part = t > 1.f ? 1.f : t > 0.f ? t : 0.f;
#endif
    const float near = fmaf(part, 15.f, 12582912.f);  // 1.5 * 2^23: the sum's last digit is 1
    *off = fabsf(fmaf(part, 15.f, 12582912.f - near));
    uint32_t bits;
    memcpy(&bits, &near, 4);
    return bits - 0x4b400000u;
}
constexpr float kQ4Near = 0.49998474f;
constexpr float kQ4Most = 65504.f, kQ4Nothing = 8.271806125530277e-25f;  // 2^-80

}  // namespace juno
