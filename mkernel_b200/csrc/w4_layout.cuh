// Layout of 4-bit weights, shared by the kernels that write it (pack, quantise) and read it.
//
// The matrix [N, K] is cut into strips of 64 rows and blocks of 128 columns.  A (strip, block)
// chunk is contiguous, and the chunks of a strip follow one another along K, so that a warp that
// walks a strip reads one stream:
//   4096 bytes of codes | per group of the block: 64 scales | per group: 64 offsets (zero points)
// Codes are stored in the order in which the lanes of a warp need them as the A operand of the
// 16x8x16 matrix instruction: [half of 64 columns][tile of 16 rows][lane][16 bytes], so a lane
// loads its operands of four such instructions with one 16-byte access.  Lane (g = lane / 4,
// t = lane % 4) holds rows g and g + 8 of the tile; word j of its 16 bytes holds columns
// 32 (j / 2) + 8 t + 4 (j % 2) + {0, 1, 2, 3} of the half.  Which column of the instruction a
// matrix column lands on does not matter to a dot product as long as both operands agree; this
// order gives a lane 8 consecutive columns (16 bytes of the other operand) and keeps every
// instruction inside a group of 32.  Nibble i + 4 e of the word is operand register i (row
// g + 8 (i % 2), column pair i / 2), element e: (word >> 4 i) & 0x000f000f is the register's two
// codes in the low bits of its two halves.
// Scales and offsets of a group: [g][tile][2], 16 bits each, so that a lane takes the eight that
// belong to its rows with one 16-byte access.  An offset is the 16-bit float of base + zero point
// (see W4Traits).
//
// A strip's rows are chosen so that rows g and g + 8 of a tile, which end in one thread, are the
// two rows that an epilogue combines: neighbours 8 apart (plain), gate and up of one output, or
// the two features that a rotary position turns together.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include "../../include/mkernel_b200.h"

namespace mkb {

constexpr int kW4Strip = 64;
constexpr int kW4Block = 128;
constexpr int kW4CodeBytes = kW4Strip * kW4Block / 2;

struct W4Form {
  int N, K, group, zeros, form;
  int head_dim, rotary_dim, rotated_heads, interleaved;
  int strips, blocks, chunk_bytes;
};

__host__ __device__ inline W4Form w4_form(const mk_w4& w) {
  W4Form f;
  f.N = w.N; f.K = w.K; f.group = w.group; f.zeros = w.zeros != 0; f.form = w.form;
  f.head_dim = w.head_dim; f.rotary_dim = w.rotary_dim;
  f.rotated_heads = w.rotated_heads; f.interleaved = w.interleaved;
  f.strips = (int)(((long long)w.N + kW4Strip - 1) / kW4Strip);
  f.blocks = (int)(((long long)w.K + kW4Block - 1) / kW4Block);
  f.chunk_bytes = kW4CodeBytes + (kW4Block / w.group) * kW4Strip * 2 * (w.zeros ? 2 : 1);
  return f;
}

// Row of the matrix held at pair `p` (tile p / 8, g = p % 8) of a strip, first (j = 0) or second
// (j = 1) of the pair; -1 behind the last row.
__host__ __device__ inline int w4_row(const W4Form& f, int strip, int p, int j) {
  if (f.form == MK_W4_PLAIN) {
    const long long n = (long long)strip * kW4Strip + (p / 8) * 16 + j * 8 + p % 8;
    return n < f.N ? (int)n : -1;
  }
  const long long pair = (long long)strip * (kW4Strip / 2) + p;
  if (pair >= f.N / 2) return -1;
  if (f.form == MK_W4_GATE_UP) return (int)pair + j * (f.N / 2);
  const int half = f.head_dim / 2, head = (int)(pair / half), i = (int)(pair % half);
  const bool apart = !f.interleaved && head < f.rotated_heads && i < f.rotary_dim / 2;
  return head * f.head_dim + (apart ? i + j * (f.rotary_dim / 2) : 2 * i + j);
}

// Per type of the scales and activations.  A code 0..15 put into the low mantissa bits of `magic`
// is magic's value plus the code, exactly; taking away the offset (that value plus the zero
// point, also exact) leaves code - zero exactly.
template <typename T> struct W4Traits;
template <> struct W4Traits<__nv_bfloat16> {
  using T2 = __nv_bfloat162;
  static constexpr uint32_t kMagic = 0x43004300u;   // 128, one unit in the last place is 1
  static constexpr uint32_t kEight = 0x43084308u;   // 136: the offset without zero points
  static __device__ __forceinline__ float to_float(uint32_t bits) {
    return __uint_as_float(bits << 16);
  }
  static __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
};
template <> struct W4Traits<__half> {
  using T2 = __half2;
  static constexpr uint32_t kMagic = 0x64006400u;   // 1024
  static constexpr uint32_t kEight = 0x64086408u;   // 1032
  static __device__ __forceinline__ float to_float(uint32_t bits) {
    return __half2float(__ushort_as_half((unsigned short)bits));
  }
  static __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
};

// The two codes of operand register i of a word as (code - zero) in T, given the offset twice.
template <typename T>
__device__ __forceinline__ uint32_t w4_decode(uint32_t word, int i, uint32_t offset2) {
  using T2 = typename W4Traits<T>::T2;
  uint32_t v;
  // (word >> 4 i) & 0x000f000f | magic as one three-input operation after the shift
  asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xea;" : "=r"(v) : "r"(word >> (4 * i)), "r"(W4Traits<T>::kMagic));
  T2 r = __hsub2(*reinterpret_cast<T2*>(&v), *reinterpret_cast<T2*>(&offset2));
  return *reinterpret_cast<uint32_t*>(&r);
}

}  // namespace mkb
