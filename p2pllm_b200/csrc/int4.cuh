// The 4-bit weight layout (p2p_int4_layout), shared by the kernels that read it.
//
// A module is cut into units of 128 rows by 128 columns, each a record of consecutive bytes, the units of a row tile one
// after the other: a run of units is one linear stream.
//   record   codes [8 row blocks of 16][2 column blocks of 64][512 bytes]
//            zero points [groups of the unit][8 row blocks][8][2], a byte each: rows n and n + 8 (only if there are any)
//            scales [groups of the unit][8 row blocks][8][2], 16 bits each, the same order
//   layout   [experts][row tiles][units of 128 columns][record]
// Of a (row block, column block)'s 512 bytes lane t = 4 n + j of a warp owns the 16 at 16 t, word r of them (r = 0..3)
// holding the codes of rows n and n + 8 at columns 16 r + 4 j .. + 3, as four pairs of neighbouring columns whose low
// column is nibble i and high column nibble i + 4:
//   i = 0: row n, columns 0 and 1    i = 1: row n, columns 2 and 3    i = 2, 3: the same of row n + 8
// so that one mask leaves a pair in the low bits of both halves of the word, ready to become two 16-bit floats. That is
// a lane's A fragment of four m16n8k16 products whose k runs 4 j .. 4 j + 3 instead of {2 j, 2 j + 1, 2 j + 8, 2 j + 9}
// (the sum over k does not mind, B's fragment takes the same columns: one 8-byte load of x), and also a lane's part of
// a tcgen05.st.16x256b.x4 of 16 rows by 64 columns into tensor memory.
// Of a gated module the even row blocks are gate rows, the odd ones the same units' up rows.
#pragma once
#include "sm100.cuh"

namespace p2p {
namespace q4 {

constexpr int kRows = 16;
constexpr int kCols = 64;
constexpr int kBlockBytes = 512;
constexpr int kUnitCols = 128;
constexpr int kTileBlocks = 8;                         // row blocks of a unit
constexpr int kCodeBytes = kTileBlocks * 2 * kBlockBytes;

__host__ __device__ inline int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }
// Row blocks of one expert; a gated module's halves are padded to whole blocks each.
__host__ __device__ inline int64_t row_blocks(int64_t rows, int gated) {
    return gated ? 2 * div_up(rows / 2, kRows) : div_up(rows, kRows);
}

__host__ __device__ inline int64_t row_tiles(int64_t rows, int gated) { return div_up(row_blocks(rows, gated), kTileBlocks); }
__host__ __device__ inline int unit_zero_bytes(int group, bool zeros) { return zeros ? kUnitCols / group * 128 : 0; }
__host__ __device__ inline int unit_scale_bytes(int group) { return kUnitCols / group * 256; }
__host__ __device__ inline int unit_bytes(int group, bool zeros) {
    return kCodeBytes + unit_zero_bytes(group, zeros) + unit_scale_bytes(group);
}
inline int64_t layout_bytes(int64_t experts, int64_t rows, int64_t cols, int group, bool zeros, int gated) {
    return experts * row_tiles(rows, gated) * div_up(cols, kUnitCols) * unit_bytes(group, zeros);
}

// (v & mask) | magic in one instruction: with both constants in registers (opaque: as immediates they take two).
// Logic and shifts bind these kernels -- their pipe takes two cycles an instruction, 20 cycles a word of eight codes and
// one m16n8k16 product against 27 with two instructions here (148 CTAs of 16 warps, one word a lane).
__device__ __forceinline__ uint32_t opaque(uint32_t v) {
    asm volatile("" : "+r"(v));
    return v;
}
__device__ __forceinline__ uint32_t and_or(uint32_t v, uint32_t mask, uint32_t magic) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(v), "r"(mask), "r"(magic));
    return r;
}

template <typename T> struct Codes;

// bf16 holds 128 + q exactly (8 significant bits): q lands in the last mantissa bits of 0x4300 = 128.
template <> struct Codes<__nv_bfloat16> {
    uint32_t sub[2];                                   // 128 + zero of rows n and n + 8, twice
    uint32_t mask, magic;
    __device__ __forceinline__ Codes() : mask(opaque(0x000f000fu)), magic(opaque(0x43004300u)) {}
    __device__ __forceinline__ void zeros(uint32_t z0, uint32_t z1) {
        sub[0] = (0x4300u | z0) * 0x10001u;
        sub[1] = (0x4300u | z1) * 0x10001u;
    }
    // The four A registers of one word: (row n, k 0 1), (row n + 8, k 0 1), (row n, k 2 3), (row n + 8, k 2 3), each
    // the exact difference code - zero.
    __device__ __forceinline__ void expand(uint32_t w, uint32_t (&a)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t q = and_or(w >> (4 * i), mask, magic);
            const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&q),
                                             *reinterpret_cast<const __nv_bfloat162*>(&sub[i >> 1]));
            a[(i >> 1) + 2 * (i & 1)] = *reinterpret_cast<const uint32_t*>(&d);
        }
    }
};

// f16 holds 1024 + 16 q exactly (11 significant bits): two of the four pairs need no shift, (1024 + 16 q) / 16 - (64 +
// zero) being exact too.
template <> struct Codes<__half> {
    uint32_t sub[2], sub16[2], mask, mask16, magic;
    __device__ __forceinline__ Codes() : mask(opaque(0x000f000fu)), mask16(opaque(0x00f000f0u)), magic(opaque(0x64006400u)) {}
    __device__ __forceinline__ void zeros(uint32_t z0, uint32_t z1) {
        sub[0] = (0x6400u | z0) * 0x10001u;
        sub[1] = (0x6400u | z1) * 0x10001u;
        sub16[0] = (0xd400u | (z0 << 4)) * 0x10001u;   // -(64 + zero): 64's mantissa steps are 1 / 16
        sub16[1] = (0xd400u | (z1 << 4)) * 0x10001u;
    }
    __device__ __forceinline__ void expand(uint32_t w, uint32_t (&a)[4]) const {
        const __half2 sixteenth = __half2half2(__ushort_as_half((unsigned short)0x2c00));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t v = h ? w >> 8 : w;
            const uint32_t q0 = and_or(v, mask, magic), q1 = and_or(v, mask16, magic);
            const __half2 d0 = __hsub2(*reinterpret_cast<const __half2*>(&q0), *reinterpret_cast<const __half2*>(&sub[h]));
            const __half2 d1 = __hfma2(*reinterpret_cast<const __half2*>(&q1), sixteenth,
                                       *reinterpret_cast<const __half2*>(&sub16[h]));
            a[h] = *reinterpret_cast<const uint32_t*>(&d0);
            a[h + 2] = *reinterpret_cast<const uint32_t*>(&d1);
        }
    }
};

template <typename T> struct alignas(8) Quad { T v[4]; };

// `things` (units, or row tiles of `each` units) dealt to n runs, the first `rest` of which take one more. Below 2^31
// units in all, and arithmetic in 32 bits: a 64-bit division takes the time of a unit.
struct Runs {
    uint32_t whole, rest, each;
    __device__ __forceinline__ Runs(uint32_t things, uint32_t n, uint32_t each_) {
        each = each_;
        whole = things / n;
        rest = things - whole * n;
    }
    __device__ __forceinline__ uint32_t begin(uint32_t b) const { return (b * whole + min(b, rest)) * each; }
    // The run that holds unit u, of units dealt one by one, at least one a run.
    __device__ __forceinline__ uint32_t of(uint32_t u) const {
        const uint32_t longer = rest * (whole + 1);
        return u < longer ? u / (whole + 1) : rest + (u - longer) / whole;
    }
};

}  // namespace q4
namespace sm100 {

// mbar_wait, with many tests of the phase before it looks at the clock and the failure flag: each such look takes about a
// microsecond, which a hand-over between two roles cannot wait for. A test sleeps for at most two microseconds, so all of
// them last a millisecond: the limit starts, and another wait's failure is seen, that much later at most.
__device__ __forceinline__ bool wait_one(uint32_t bar, uint32_t parity, int site, const WaitCtl& wc) {
#pragma unroll 1
    for (int i = 0; i < 512; ++i)
        if (mbar_try<2000u>(bar, parity)) return true;
    return mbar_wait(bar, parity, site, wc);
}

// One thread of the warp, the same one every time. A branch on elect.sync, unlike one on the lane number, tells the
// compiler that a single thread runs it: tensor-core and copy instructions then take their operands straight from
// uniform registers.
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

}  // namespace sm100

}  // namespace p2p
