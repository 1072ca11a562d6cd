// Test-only host build of the layout and arithmetic of 4-bit cache pages (csrc/q4_pages.cuh): the functions that the device kernels call.
#include "../../juno_b200/csrc/q4_pages.cuh"

using namespace juno;

extern "C" int q4_host_number(float x, float m, float d) {
    float off;
    const int q = (int)q4_number_near(x, m, d > 0.f ? 1.f / (15.f * d) : 0.f, &off);
    return off > kQ4Near ? q4_number_exact(x, m, d, d > 0.f ? 1.f / d : 0.f) : q;
}
extern "C" int q4_host_number_exact(float x, float m, float d) { return q4_number_exact(x, m, d, d > 0.f ? 1.f / d : 0.f); }
extern "C" int q4_host_block_bytes(int hd) { return q4_block_bytes(hd); }

// Marks every half byte of a block that a number takes and every byte of its factors; returns how many were marked twice, or lie outside.
extern "C" int q4_host_cover(int hd, unsigned char *nibbles) {
    int twice = 0;
    const int size = 2 * q4_block_bytes(hd);
    auto mark = [&](int nibble) {
        if (nibble < 0 || nibble >= size || nibbles[nibble]++) twice++;
    };
    for (int p = 0; p < 16; p++)
        for (int g = 0; g < hd / kQ4Group; g++) {
            for (int t = 0; t < 4; t++)
                for (int e = 0; e < 8; e++) mark(2 * q4_k_code(hd, p, t, g) + e);
            for (int u = 0; u < 8; u++)
                for (int i = 0; i < 4; i++) mark(2 * q4_v_code(hd, p, u, g) + i);
            for (int b = 0; b < 4; b++) {
                mark(2 * q4_k_step(hd, p, g) + b);
                mark(2 * q4_k_offset(hd, p, g) + b);
                mark(2 * q4_v_step(hd, p, g) + b);
                mark(2 * q4_v_offset(hd, p, g) + b);
            }
        }
    return twice;
}

// The four numbers of a packed unit, each from bits 6..9 of the half word as it is shifted or turned for it.
extern "C" void q4_host_unit(int a, int b, int c, int d, int *out) {
    const uint32_t u = q4_unit((uint32_t)a, (uint32_t)b, (uint32_t)c, (uint32_t)d), turned = (u >> 8 | u << 8) & 0xffffu;
    out[0] = (int)(u >> 6 & 15u);
    out[1] = (int)(u >> 4 >> 6 & 15u);
    out[2] = (int)(u << 4 >> 6 & 15u);
    out[3] = (int)(turned >> 6 & 15u);
}
