// Layout of 4-bit weights, shared by the kernels that write it (pack, quantise) and read it.
//
// The matrix [N, K] is cut into strips of 64 rows and blocks of 128 columns.  A (strip, block)
// chunk is contiguous, and the chunks of a strip follow one another along K, so that a warp that
// walks a strip reads one stream:
//   4096 bytes of codes | per group of the block: 64 scales | per group: 64 offsets (zero points)
// Codes are stored in the order in which the lanes of a warp need them as the A operand of the
// 16x8x16 matrix instruction: [half of 64 columns][tile of 16 rows][lane][16 bytes], so a lane
// loads its operands of four such instructions with one 16-byte access.  Lane (g = lane / 4,
// t = lane % 4) holds rows g and g + 8 of the tile; word v of its 16 bytes holds columns
// 16 v + 4 t + {0, 1, 2, 3} of the half.  Which column of the instruction a matrix column lands on
// does not matter to a dot product as long as both operands agree; with this order a lane needs four
// consecutive columns (8 bytes) of the other operand for an instruction, an instruction stays inside 16
// consecutive columns, and the same words written to tensor memory as 16x256b (whose lanes are the
// same lanes) put the columns there in their natural order.  Nibble i + 4 e of the word is operand
// register i (row g + 8 (i % 2), column pair i / 2), element e: (word >> 4 i) & 0x000f000f is the
// register's two codes in the low bits of its two halves.
// Scales and offsets of a group: [g][tile][2], 16 bits each, so that a lane takes the eight that
// belong to its rows with one 16-byte access.  An offset is -zero point * kUnit (see W4Traits); both types
// hold it exactly for any byte, and code - zero, at most 8 bits, as well.
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

// Per type of the scales and activations.  Up to 8 low bits of a 16-bit float, its exponent otherwise
// 0, are a subnormal: that whole number of the smallest steps (2^-133 in bf16, 2^-24 in fp16; bf16's eighth
// bit is the lowest of the exponent, where the steps are still the same).  So a code needs no
// conversion: masked in place it is a float, and one fused multiply-add scales it up by a power of
// two and takes the zero point away, exactly.  What comes out is (code - zero) * kUnit, the largest unit
// that the largest power of two allows; its inverse is multiplied in at the end, also exactly.
template <typename T> struct W4Traits;
template <> struct W4Traits<__nv_bfloat16> {
  static constexpr uint32_t kLow = 0x7f007f00u;       // 2^127: a code in bits 0..3
  static constexpr uint32_t kHigh = 0x7d007d00u;      // 2^123: in bits 4..7, where it is 16 times as much
  static constexpr uint32_t kMinusEight = 0xbe00be00u;   // -8 kUnit
  static constexpr float kUnit = 0x1p-6f;
  static constexpr uint32_t kBack = 0x42804280u;      // 1 / kUnit, twice
  static __device__ __forceinline__ float to_float(uint32_t bits) { return __uint_as_float(bits << 16); }
  static __device__ __forceinline__ float2 to_float2(uint32_t two) {
    return make_float2(__uint_as_float(two << 16), __uint_as_float(two & 0xffff0000u));
  }
  static __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
  }
};
template <> struct W4Traits<__half> {
  static constexpr uint32_t kLow = 0x78007800u;       // 2^15
  static constexpr uint32_t kHigh = 0x68006800u;      // 2^11
  static constexpr uint32_t kMinusEight = 0xa400a400u;
  static constexpr float kUnit = 0x1p-9f;
  static constexpr uint32_t kBack = 0x60006000u;
  static __device__ __forceinline__ float to_float(uint32_t bits) {
    return __half2float(__ushort_as_half((unsigned short)bits));
  }
  static __device__ __forceinline__ float2 to_float2(uint32_t two) {
    return __half22float2(*reinterpret_cast<const __half2*>(&two));
  }
  static __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ uint32_t min2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
  }
};

// The four operand registers of a word, each two codes as (code - zero) kUnit; off0 and off1: -zero kUnit
// of rows g and g + 8, each twice.  Nibble 0 is row g, nibble 1 row g + 8, nibbles 2 and 3 the next pair
// of columns.
template <typename T>
__device__ __forceinline__ void w4_decode(uint32_t word, uint32_t off0, uint32_t off1, uint32_t (&a)[4]) {
  using W = W4Traits<T>;
  const uint32_t next = word >> 8;
  a[0] = W::fma2(word & 0x000f000fu, W::kLow, off0);
  a[1] = W::fma2(word & 0x00f000f0u, W::kHigh, off1);
  a[2] = W::fma2(next & 0x000f000fu, W::kLow, off0);
  a[3] = W::fma2(next & 0x00f000f0u, W::kHigh, off1);
}

// The same as the weights themselves, rounded to T: (code - zero) * scale.  sc0, sc1: the scales of rows g and
// g + 8, each twice; off0, off1: their zero points as the layout holds them.  With `rest`, what the rounding
// left: the two together are the weight exactly (8 bits times 8 in bf16, 8 times 11 in fp16, and the two
// parts have 16 and 22), down to fp16's smallest subnormal.  At the other end a weight beyond the type's
// largest number is an infinity here, its rest the other one and their products NaN; in bf16 so is any weight with a
// scale of 2^122 or more, which is held 64 times as large.
template <typename T>
struct W4Round;
template <>
struct W4Round<__nv_bfloat16> {
  uint32_t off0, off1, sc0, sc1;
  __device__ __forceinline__ W4Round(uint32_t o0, uint32_t o1, uint32_t s0, uint32_t s1) : off0(o0), off1(o1) {
    // a power of two: bf16 has room for it in the exponent
    sc0 = mul2(s0, W4Traits<__nv_bfloat16>::kBack);
    sc1 = mul2(s1, W4Traits<__nv_bfloat16>::kBack);
  }
  static __device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  template <bool REST>
  __device__ __forceinline__ void get(uint32_t word, uint32_t (&a)[4], uint32_t (&rest)[4]) const {
    uint32_t v[4];
    w4_decode<__nv_bfloat16>(word, off0, off1, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t sc = i & 1 ? sc1 : sc0;
      a[i] = mul2(v[i], sc);
      if (REST) rest[i] = W4Traits<__nv_bfloat16>::fma2(v[i], sc, a[i] ^ 0x80008000u);
    }
  }
};
template <>
struct W4Round<__half> {
  // fp16 has not, so the code is made whole another way: in the low bits of 1024 (or, 16 times as much, four
  // bits up), less 1024 (64) and the zero point; a known way to turn whole numbers into fp16 (Kim, Henry, Fahim,
  // Awadalla: Who Says Elephants Can't Run, 2022).
  uint32_t less0, less1, sc0, sc1;
  __device__ __forceinline__ W4Round(uint32_t o0, uint32_t o1, uint32_t s0, uint32_t s1) : sc0(s0), sc1(s1) {
    less0 = W4Traits<__half>::fma2(o0, W4Traits<__half>::kBack, 0xe400e400u);   // -zero - 1024
    less1 = W4Traits<__half>::fma2(o1, W4Traits<__half>::kBack, 0xd400d400u);   // -zero - 64
  }
  static __device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ uint32_t low(uint32_t word, uint32_t less) {
    uint32_t v, r;
    asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xea;" : "=r"(v) : "r"(word), "n"(0x64006400));
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(less));
    return r;
  }
  static __device__ __forceinline__ uint32_t high(uint32_t word, uint32_t less) {
    uint32_t v;
    asm("lop3.b32 %0, %1, 0x00f000f0, %2, 0xea;" : "=r"(v) : "r"(word), "n"(0x64006400));
    return W4Traits<__half>::fma2(v, 0x2c002c00u, less);   // times 1/16
  }
  template <bool REST>
  __device__ __forceinline__ void get(uint32_t word, uint32_t (&a)[4], uint32_t (&rest)[4]) const {
    const uint32_t next = word >> 8;
    const uint32_t v[4] = {low(word, less0), high(word, less1), low(next, less0), high(next, less1)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t sc = i & 1 ? sc1 : sc0;
      a[i] = mul2(v[i], sc);
      if (REST) rest[i] = W4Traits<__half>::fma2(v[i], sc, a[i] ^ 0x80008000u);
    }
  }
};

}  // namespace mkb
