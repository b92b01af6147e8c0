// Matrices held in four bits: the layout, and codes to the bfloat16 values that they stand for.
//
// A row's K is cut into groups of 32, 64 or 128 neighbours.  A group keeps a bfloat16 scale s and offset b, its elements a code q from 0
// to 15, and an element is W = bfloat16(q s + b): q s + b is rounded once, so every kernel multiplies with the same matrix, whatever the
// number of rows.  (A scale has 8 significant bits and a code 4, so W would need 12 and more to be exact.  The rounding moves W by at most
// half a step, 2^-8 of it; the code has moved it by up to half a scale, a thirtieth of the group's range.)
//
// Codes: blocks of 16 rows by 64 k, 512 bytes, along K first: [N / 16][K / 64][t 4][r 8][half 2][word 2] of 32 bits; row 16 i + 8 half + r,
// k = 64 c + 16 t + 8 word + 2 p + e in bits 4 (4 e + p).
//   - A lane 4 r + t of mma.sync.m16n8k16 has rows r and r + 8 on its side: its 32 codes of a block are 16 neighbouring bytes.
//   - A thread that owns a row (a lane of tensor memory) takes four times 8 bytes, and the threads of 16 rows 128 neighbouring ones.
//   - `(word >> 4 p) & 0x000f000f` is a pair of neighbouring k, the lower one in the lower half.
// Scales and offsets: [N / 16][groups][r 8][half 2] pairs (s in the lower half of 32 bits, b in the upper), groups = K / group with K rounded
// up to 64.  Rows and k beyond the matrix have codes, scales and offsets of 0, so they stand for 0.
#pragma once
#include "common.cuh"

#define Q4_BLOCK_WORDS 128   // 32-bit words of a block of 16 rows by 64 k

// Sizes up to here can be rounded up to a tile's and stay within 31 bits.
#define Q4_MOST 0x7fffff00

// Both halves of a register: the scale, the offset.
__device__ __forceinline__ unsigned q4_scale(unsigned affine) { return __byte_perm(affine, 0, 0x1010); }
__device__ __forceinline__ unsigned q4_offset(unsigned affine) { return __byte_perm(affine, 0, 0x3232); }
// Eight codes to four pairs of bfloat16, W = q s + b rounded once.
//
// SMALL (a scale from 2^-126 up to 2^-5, as trained matrices have): a code in the lower bits of an otherwise empty bfloat16 is q 2^-133, a
// subnormal number, exactly; with `scale` 2^133 as large their product is q s, and the multiply-add rounds q s + b once.
// Else: a code in the lower bits of 128.0 (0x4300) is 128 + q exactly; less 128 exactly q.  That takes four more instructions for eight codes,
// 15 instead of 11, on a pipe that is as busy as the one for shifts and logic.  (2048 rows, gated 12288 x 4096: 339 us this way, 322 with the shorter
// one, on one box.  The kernel for a few rows takes the longer way alone: both of them in its loop cost more than the shorter one gains, 4 rows
// 151936 x 2560 58.9 us instead of 48.7.)
template <bool SMALL>
__device__ __forceinline__ void q4_values(unsigned word, unsigned scale, unsigned offset, unsigned (&w)[4]) {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        unsigned v;
        if (SMALL) {
            v = (word >> (4 * p)) & 0x000f000fu;
        } else {   // (one three-input operation: written in C it became two)
            asm("lop3.b32 %0, %1, %2, %3, 0xea;\n" : "=r"(v) : "r"(word >> (4 * p)), "n"(0x000f000f), "r"(0x43004300u));
            asm("sub.rn.bf16x2 %0, %1, %2;\n" : "=r"(v) : "r"(v), "r"(0x43004300u));
        }
        asm("fma.rn.bf16x2 %0, %1, %2, %3;\n" : "=r"(w[p]) : "r"(v), "r"(scale), "r"(offset));
    }
}
// Whether a scale (the lower half) is one for SMALL, and that scale times 2^133 in both halves of a register (133 more in the exponents).
__device__ __forceinline__ bool q4_small(unsigned affine) { return (affine & 0xffffu) - 0x80u < 0x3d00u - 0x80u; }
__device__ __forceinline__ unsigned q4_raised(unsigned scale) { return scale + 0x42804280u; }
