// 4-bit codes as operands of m16n8k16 tensor-core products (scan_q4.cu, attend_q4.cu).
#pragma once

#include "q4.cuh"

namespace dc {

// Lane (g, t) = (lane / 4, lane % 4).  A: a0 = (row g, k = 2t, 2t + 1), a1 = row g + 8, a2 / a3 = the same rows at k + 8;
// B: b0 = (k = 2t, 2t + 1; column g), b1 at k + 8; D: d0, d1 = (row g; columns 2t, 2t + 1), d2, d3 = row g + 8.
template <bool BF16>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The first product of a sum: nothing to add to.
template <bool BF16>
__device__ __forceinline__ void mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// N 32-bit words from a naturally aligned address that is read once.
template <int N>
__device__ __forceinline__ void ldg_words(uint32_t (&r)[N], const void* p) {
    if (N == 2) {
        asm volatile("ld.global.nc.L1::no_allocate.v2.b32 {%0,%1}, [%2];\n" : "=r"(r[0]), "=r"(r[1]) : "l"(p));
    } else {
#pragma unroll
        for (int i = 0; i + 3 < N; i += 4)
            asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];\n"
                         : "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]) : "l"(static_cast<const char*>(p) + 4 * i));
    }
}

// Constants of the code conversion, kept in registers: with an immediate operand the packed 16-bit subtraction issues to
// the integer pipe, which the masks already fill, instead of the FMA pipe.
struct CodeConst {
    uint32_t bf16_one, bf16_off;
    __device__ __forceinline__ explicit CodeConst(uint32_t zero) {   // 0, in a form the compiler cannot fold
        bf16_one = 0x43004300u | zero;   // 128, 128
        bf16_off = 0xC308C308u | zero;   // -136
    }
};

// Four pairs of codes of a word as bf16: pair j = (nibble j, nibble j + 4).  Inserting a nibble into the mantissa of 128 makes
// it 128 plus the nibble, exactly; the offset and the 8 of the encoding go with one addition.
__device__ __forceinline__ void codes_bf16(const CodeConst& k, uint32_t w, uint32_t (&p)[4]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t t = ((w >> (4 * i)) & 0x000F000Fu) | k.bf16_one;
        asm("add.bf16x2 %0, %1, %2;\n" : "=r"(p[i]) : "r"(t), "r"(k.bf16_off));
    }
}

// (x, y) rounded to a pair of 16-bit values, x in the low half; what is lost goes to a second pair.
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    uint32_t r;
    if (BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(y), "f"(x));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(r) : "f"(y), "f"(x));
    return r;
}
template <int DT>
__device__ __forceinline__ float low_elem(uint32_t w) { return elem_to_float<DT>(static_cast<uint16_t>(w & 0xFFFFu)); }
template <int DT>
__device__ __forceinline__ float high_elem(uint32_t w) {
    return DT == DC_BF16 ? __uint_as_float(w & 0xFFFF0000u) : elem_to_float<DT>(static_cast<uint16_t>(w >> 16));
}

// The same pairs as fp16 subnormals: nibble u is u * 2^-24 as it stands in the low bits, and u * 2^-20 four bits up, so one mask
// is all a pair takes.  What is left of the encoding, 2^-24 or 2^-20 and the 8, goes into the other operand (odd pairs: a
// sixteenth of it) and the sum the products start from (- 8 * 2^-24 of the other operand's sum).  A sum then passes through values
// of up to (|c| + 16) |q| per element instead of |c| |q|: its fp32 rounding is relative to those, about 2^-18 of what half a step of
// the codes may change it by even where the codes themselves are small.
__device__ __forceinline__ void codes_subnormal(uint32_t w, uint32_t (&p)[4]) {
    const uint32_t hi = w >> 8;
    p[0] = w & 0x000F000Fu;
    p[1] = w & 0x00F000F0u;
    p[2] = hi & 0x000F000Fu;
    p[3] = hi & 0x00F000F0u;
}
// d = a b + c with c left as it is
__device__ __forceinline__ void mma_from(float (&d)[4], const float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// Powers of two that bring a vector whose largest magnitude is `top` to [2^14, 2^15) and back: a bf16 element, and a sixteenth
// of it, is then exact in fp16 unless it is more than 2^27 times smaller than the largest.
__device__ __forceinline__ void q4_normalise(float top, float& down, float& up) {
    int ex = static_cast<int>((__float_as_uint(top) >> 23) & 255u);   // 0: zero or subnormal, 255: infinite
    ex = ex == 255 ? 127 + 14 : max(ex, 15);   // the smallest for which both are normal numbers
    down = __uint_as_float(static_cast<uint32_t>(127 + 14 - ex + 127) << 23);   // 2^(14 - e)
    up = __uint_as_float(static_cast<uint32_t>(ex - 14) << 23);                 // 2^(e - 14)
}

}  // namespace dc
