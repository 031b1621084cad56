// The 4-bit key/value cache: what a page holds, and how its codes become numbers.
//
// Sixteen tokens of one kv head are a record, laid out as the lanes of an mma.sync A operand read it, so that a warp takes a record with
// whole 16-byte reads and no shuffles, and one contiguous copy brings it.  The pool is [pages][kv heads][page size / 16][record]:
//   K codes   [16 tokens][HD / 2] bytes, a u32 = 8 adjacent dims, lowest nibble first
//   V codes   u32 [2 halves h][8 blocks g][4 pairs c][HD / 32]: low half word d: token 8h + 2c, high half word: token 8h + 2c + 1, each the
//             4 dims g HD/8 + 4d ..., lowest nibble first (a byte never holds two tokens, so tokens are written independently)
//   K, then V scale | bias << 16 (bf16 both), u32 [HD / 64][16 tokens]
// 2304 bytes at head size 128 and 1152 at 64: 144 and 72 bytes per token and kv head, against 512 and 256 in bf16.
//
// A code c stands for bf16(c scale + bias), one rounding.
#pragma once
#include "common.cuh"
#include "dequant.cuh"

namespace q4 {

template <int HD>
struct Record {
    static constexpr int kGroups = HD / 64;
    static constexpr int kV = 8 * HD, kKsb = 16 * HD, kVsb = kKsb + 64 * kGroups, kBytes = kVsb + 64 * kGroups;
};
inline int record_bytes(int hd) { return hd == 128 ? Record<128>::kBytes : Record<64>::kBytes; }

// Codes become numbers as the weights' codes do (dequant.cuh): a nibble in the low bits of a bf16 is the number c 2^-133, so one fma with
// scale 2^69 and bias 2^-64 gives the value times 2^-64 with one rounding: bf16(c scale + bias) 2^-64, wherever that is no subnormal
// (values from 2^-62 on; smaller ones lose bits beside what the 4 bits lose).  A scale times 2^69 is finite below 2^59; the append writes
// none from there on.
constexpr float kScaleEnd = 576460752303423488.f;  // 2^59
constexpr float kUnscale = 18446744073709551616.f;  // 2^64
struct Scales {
    uint32_t lo, hi, bias;  // for nibbles 0, 2 (bits 0-3 of a half word), for nibbles 1, 3 (bits 4-7), and the biases
};
__device__ __forceinline__ Scales scales_of(uint32_t s2, uint32_t b2) {
    return {mul_bf2(s2, 0x62006200u), mul_bf2(s2, 0x60006000u), mul_bf2(b2, 0x1f801f80u)};
}
// one token's, for both halves of a word, and two tokens', one for each half
__device__ __forceinline__ Scales scales_twice(uint32_t sb) { return scales_of(prmt(sb, 0u, 0x1010u), prmt(sb, 0u, 0x3232u)); }
__device__ __forceinline__ Scales scales_pair(uint32_t sb0, uint32_t sb1) { return scales_of(prmt(sb0, sb1, 0x5410u), prmt(sb0, sb1, 0x7632u)); }
// whether values of this scale and bias may be infinite or NaN: a scale from 2^59 (0x5d00) on, a bias that is one
__device__ __forceinline__ bool poisoned(uint32_t sb) { return (sb & 0x7fffu) >= 0x5d00u || (sb & 0x7f800000u) == 0x7f800000u; }
// nibble i of the low half word beside nibble i of the high one
__device__ __forceinline__ void values(uint32_t w, const Scales& s, uint32_t (&out)[4]) { scaled_q4_paired(w, s.lo, s.hi, s.bias, out); }

}  // namespace q4
