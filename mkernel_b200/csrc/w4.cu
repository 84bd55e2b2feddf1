// Products with 4-bit weights (group scales, optional zero points), their SwiGLU and rotary forms,
// and the kernels that lay the weights out.  The layout is described in w4_layout.cuh.
#include <cuda_runtime.h>

#include <cstring>
#include <type_traits>

#include "../../include/mkernel_b200.h"
#include "host_util.h"
#include "ptx.cuh"
#include "w4_product.cuh"

namespace mkb {

// ------------------------------------------------------------------------------------------
// laying the weights out
// ------------------------------------------------------------------------------------------
// A thread of all three kernels has a pair of rows and, of a half of a block, 8 consecutive columns and the 8
// that lie 32 further: 16-byte accesses, four neighbouring threads covering 64 bytes in order.  That is
// two words of the layout for each of two lanes; after exchanging one of each piece with its neighbour
// (w4_exchange) it has the 16 bytes of one lane.  A group is reduced by shuffles, and nothing passes
// through shared memory.
constexpr int kW4PackThreads = 256;

struct W4PackParams {
  W4Form form;
  uint8_t* data;
  // pack
  const uint8_t* codes;
  const uint16_t* scales;
  const uint8_t* zero_points;
  // quantise
  const void* src;
  long long ld;
  int vec;   // 16-byte accesses to eight columns are aligned
};

struct W4Unit { int pair, col; };   // columns col .. col + 7 and col + 32 .. col + 39 of the block
__device__ __forceinline__ W4Unit w4_unit() {
  const int t = (int)threadIdx.x & 3;
  return {(int)threadIdx.x >> 3, ((int)threadIdx.x >> 2 & 1) * 64 + (t & 1) * 16 + (t >> 1) * 8};
}
// Place of the lane that the unit's thread has after the exchange: t = thread % 4.
__device__ __forceinline__ int w4_unit_offset(const W4Unit& u) {
  return (((u.col >> 6) * 4 + (u.pair >> 3)) * 32 + (u.pair & 7) * 4 + (threadIdx.x & 3)) * 16;
}

// Between the words of a thread's columns, {first four, last four} of both pieces, and the words of its lane.
__device__ __forceinline__ void w4_exchange(uint32_t (&w)[4]) {
  const bool odd = threadIdx.x & 1;
#pragma unroll
  for (int p = 0; p < 4; p += 2) {
    const uint32_t other = __shfl_xor_sync(~0u, odd ? w[p] : w[p + 1], 1);
    if (odd) w[p] = other;
    else w[p + 1] = other;
  }
}

// A word of the layout from four codes each of the pair's rows, a byte each, first column lowest: columns
// 0, 1, 2, 3 go to bits 0, 16, 8, 24.
__device__ __forceinline__ uint32_t w4_word(uint32_t first, uint32_t second) {
  return __byte_perm(first, 0, 0x3120) | __byte_perm(second, 0, 0x3120) << 4;
}

// Place of the scales of a pair (two 16-bit values) in a group of the block, in bytes.
__device__ __forceinline__ int w4_scale_offset(int pair, int group) {
  return kW4CodeBytes + group * 128 + (pair & 7) * 16 + (pair >> 3) * 4;
}

template <typename T>
__device__ __forceinline__ uint16_t w4_offset_bits(int zero) {
  const T v = W4Traits<T>::from_float(-zero * W4Traits<T>::kUnit);
  return *reinterpret_cast<const uint16_t*>(&v);
}

template <typename T>
__device__ __forceinline__ void w4_store_scales(const W4Form& f, uint8_t* chunk, int pair, int col, const uint16_t (&s)[2],
                                                const int (&zero)[2]) {
  uint8_t* p = chunk + w4_scale_offset(pair, col / f.group);
  *reinterpret_cast<uint32_t*>(p) = s[0] | (uint32_t)s[1] << 16;
  if (f.zeros)
    *reinterpret_cast<uint32_t*>(p + kW4Block / f.group * 128) =
        w4_offset_bits<T>(zero[0]) | (uint32_t)w4_offset_bits<T>(zero[1]) << 16;
}

// Codes behind the matrix are 8, their scales 0 and zero points 8, whoever lays them out.
template <typename T>
__global__ void __launch_bounds__(kW4PackThreads) w4_pack_kernel(W4PackParams p) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const W4Form& f = p.form;
  const int strip = blockIdx.y, block = blockIdx.x;
  uint8_t* chunk = p.data + ((size_t)strip * f.blocks + block) * f.chunk_bytes;
  const long long row_bytes = ((long long)f.K + 1) / 2, groups = ((long long)f.K + f.group - 1) / f.group;
  const W4Unit u = w4_unit();
  uint32_t words[4];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int col = u.col + 32 * q;
    const long long k = (long long)block * kW4Block + col;
    uint32_t low[2], high[2];
    uint16_t scale[2] = {0, 0};
    int zero[2] = {8, 8};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = w4_row(f, strip, u.pair, j);
      uint32_t v = 0x88888888u;   // nibbles of 8 columns
      if (n >= 0 && k < f.K) {
        const uint8_t* c = p.codes + n * row_bytes + k / 2;
        v = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) v |= (k + 2 * e < f.K ? (uint32_t)c[e] : 0x88u) << (8 * e);
        if (k + 8 > f.K) {
          const uint32_t mask = (1u << (4 * (int)(f.K - k))) - 1;
          v = (v & mask) | (0x88888888u & ~mask);
        }
        if (col % f.group == 0) {
          scale[j] = p.scales[n * groups + k / f.group];
          if (f.zeros) zero[j] = p.zero_points[n * groups + k / f.group];
        }
      }
      low[j] = __byte_perm(v & 0x0f0f, (v >> 4) & 0x0f0f, 0x5140);
      high[j] = __byte_perm((v >> 16) & 0x0f0f, (v >> 20) & 0x0f0f, 0x5140);
    }
    words[2 * q] = w4_word(low[0], low[1]);
    words[2 * q + 1] = w4_word(high[0], high[1]);
    if (col % f.group == 0) w4_store_scales<T>(f, chunk, u.pair, col, scale, zero);
  }
  w4_exchange(words);
  *reinterpret_cast<uint4*>(chunk + w4_unit_offset(u)) = make_uint4(words[0], words[1], words[2], words[3]);
}

// Eight columns of a source row, and the smallest and largest of them and 0 (symmetric: the largest
// magnitude alone); NaN where there is one.  16-bit types two at a time.
__device__ __forceinline__ float w4_max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float w4_min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
template <typename S> struct W4Source;
template <> struct W4Source<float> {
  float v[8];
  __device__ __forceinline__ float operator[](int i) const { return v[i]; }
  __device__ __forceinline__ void load(const float* p) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  }
  __device__ __forceinline__ void load(const float* p, int n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.0f;
  }
  template <bool ZEROS> __device__ __forceinline__ void range(float& lo, float& hi) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (ZEROS) lo = w4_min_nan(lo, v[i]);
      hi = w4_max_nan(hi, ZEROS ? v[i] : fabsf(v[i]));
    }
  }
};
template <typename S> struct W4Source16 {
  uint32_t v[4];
  __device__ __forceinline__ float operator[](int i) const {
    const float2 two = W4Traits<S>::to_float2(v[i / 2]);
    return i & 1 ? two.y : two.x;
  }
  __device__ __forceinline__ void load(const S* p) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  }
  __device__ __forceinline__ void load(const S* p, int n) {
    const uint16_t* e = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      v[i] = (2 * i < n ? (uint32_t)e[2 * i] : 0u) | (2 * i + 1 < n ? (uint32_t)e[2 * i + 1] << 16 : 0u);
  }
  template <bool ZEROS> __device__ __forceinline__ void range(float& lo, float& hi) const {
    uint32_t least = 0, most = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (ZEROS) least = W4Traits<S>::min2(least, v[i]);
      most = W4Traits<S>::max2(most, ZEROS ? v[i] : v[i] & 0x7fff7fffu);
    }
    const float2 a = W4Traits<S>::to_float2(least), b = W4Traits<S>::to_float2(most);
    if (ZEROS) lo = w4_min_nan(lo, w4_min_nan(a.x, a.y));
    hi = w4_max_nan(hi, w4_max_nan(b.x, b.y));
  }
};
template <> struct W4Source<__nv_bfloat16> : W4Source16<__nv_bfloat16> {};
template <> struct W4Source<__half> : W4Source16<__half> {};

// w / d rounded to fp32, given r within a few units of 1 / d: a correction by the remainder, which the
// fused multiply-add gives exactly (Markstein).
__device__ __forceinline__ float w4_quotient(float w, float d, float r) {
  const float q = w * r;
  return __fmaf_rn(__fmaf_rn(-q, d, w), r, q);
}

// Quantiser: reads the matrix once and writes the chunk.  Memory bounds it (2 or 4 bytes in, 0.53 out a
// weight), instructions closely behind.  Hence no division in the common case: the rounded quotient
// of two 16-bit values is far from half way between whole numbers (2^-12 of it) unless it is exactly
// there, and then w4_quotient is exact too, so both go the same way.  Nor a clamp below: the
// quotient of the largest magnitude is within 2^-8 of 7, that of hi - lo of 15.  Both need a scale that
// is no subnormal (or 0, when all quotients round to 0); for others, and for fp32 weights, it is divided and
// clamped as the definition says.  8192 x 8192 in bf16: 37.8 us, 4.5 TB/s; 16 instructions a weight keep the issue slots
// 79 % busy.
template <typename T, typename S, int GROUP, bool ZEROS>
__global__ void __launch_bounds__(kW4PackThreads) w4_quantize_kernel(W4PackParams p) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const W4Form& f = p.form;
  const int strip = blockIdx.y, block = blockIdx.x;
  uint8_t* chunk = p.data + ((size_t)strip * f.blocks + block) * f.chunk_bytes;
  const W4Unit u = w4_unit();
  const int k0 = block * kW4Block + u.col;
  W4Source<S> w[2][2];   // row, piece
  bool row[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int n = w4_row(f, strip, u.pair, j);
    row[j] = n >= 0;
    const S* src = static_cast<const S*>(p.src) + (long long)(n < 0 ? 0 : n) * p.ld + k0;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int k = k0 + 32 * q;
      if (row[j] && p.vec && k + 8 <= f.K) w[j][q].load(src + 32 * q);
      else w[j][q].load(src + 32 * q, row[j] ? f.K - k : 0);
    }
  }
  uint32_t words[4];
  uint32_t codes[2][2][2];                       // row, piece, first or last four columns; a byte each
  constexpr int kPasses = GROUP == 32 ? 2 : 1;   // groups that a thread meets
#pragma unroll
  for (int pass = 0; pass < kPasses; ++pass) {
    const int col = u.col + 32 * pass;
    uint16_t scale_bits[2];
    int zeros[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float lo = 0.0f, hi = 0.0f;
#pragma unroll
      for (int q = 0; q < 2; ++q)
        if (kPasses == 1 || q == pass) w[j][q].template range<ZEROS>(lo, hi);
#pragma unroll
      for (int d = 1; d < (GROUP == 128 ? 8 : 4); d *= 2) {
        if (ZEROS) lo = w4_min_nan(lo, __shfl_xor_sync(~0u, lo, d));
        hi = w4_max_nan(hi, __shfl_xor_sync(~0u, hi, d));
      }
      const float span = ZEROS ? hi - lo : hi;
      // Markstein's division by a constant is the division, but for subnormal results
      const float n = ZEROS ? 15.0f : 7.0f;
      float range = span < 0x1p-100f ? __fdiv_rn(span, n) : w4_quotient(span, n, 1.0f / n);
      if (!(span <= 3.402823466e38f)) range = __int_as_float(0x7fc00000);   // an infinity or NaN in the group
      const T scale_t = W4Traits<T>::from_float(range);
      scale_bits[j] = *reinterpret_cast<const uint16_t*>(&scale_t);
      const float scale = W4Traits<T>::to_float(scale_bits[j]);
      const float divisor = scale == 0.0f ? 1.0f : scale;
      const float least = std::is_same<T, __half>::value ? 0x1p-14f : 0x1p-90f;
      const bool plain = sizeof(S) == 2 && (scale == 0.0f || (scale >= least && scale <= 0x1p90f));
      // quotient + 1.5 2^23 is the rounded quotient in the low bits (ties to even)
      constexpr float kRound = 12582912.0f;
      float inverse;
      asm("rcp.approx.f32 %0, %1;" : "=f"(inverse) : "f"(divisor));
      zeros[j] = 8;
      if (ZEROS)
        zeros[j] = plain ? (int)(__float_as_uint(w4_quotient(-lo, divisor, inverse) + kRound) & 15)
                         : (int)fminf(fmaxf(rintf(__fdiv_rn(-lo, divisor)), 0.0f), 15.0f);
      const float most = kRound + (15 - zeros[j]);
      const uint32_t add = zeros[j] * 0x01010101u;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (kPasses == 2 && q != pass) continue;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (plain) {
            uint32_t b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float x = w4_quotient(w[j][q][4 * e + i], divisor, inverse) + kRound;
              b[i] = __float_as_uint(ZEROS ? fminf(x, most) : x);
            }
            // the low bytes are -15..15: their low nibbles plus the zero point, modulo 16
            const uint32_t v = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
            codes[j][q][e] = ZEROS ? ((v & 0x0f0f0f0fu) + add) & 0x0f0f0f0fu : (v & 0x0f0f0f0fu) ^ 0x08080808u;
          } else {
            codes[j][q][e] = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float c = fminf(fmaxf(rintf(__fdiv_rn(w[j][q][4 * e + i], divisor)) + zeros[j], 0.0f), 15.0f);
              codes[j][q][e] |= (uint32_t)(int)c << (8 * i);
            }
          }
        }
        const int have = row[j] ? f.K - k0 - 32 * q : 0;
        if (have < 8) {   // behind the matrix: as pack leaves it
          const uint32_t keep0 = have >= 4 ? ~0u : have <= 0 ? 0u : (1u << (8 * have)) - 1;
          const uint32_t keep1 = have <= 4 ? 0u : (1u << (8 * (have - 4))) - 1;
          codes[j][q][0] = (codes[j][q][0] & keep0) | (0x08080808u & ~keep0);
          codes[j][q][1] = (codes[j][q][1] & keep1) | (0x08080808u & ~keep1);
        }
      }
      if (!row[j] || block * kW4Block + col - col % GROUP >= f.K) zeros[j] = 8;
    }
    if (col % GROUP == 0) w4_store_scales<T>(f, chunk, u.pair, col, scale_bits, zeros);
  }
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int e = 0; e < 2; ++e) words[2 * q + e] = w4_word(codes[0][q][e], codes[1][q][e]);
  w4_exchange(words);
  *reinterpret_cast<uint4*>(chunk + w4_unit_offset(u)) = make_uint4(words[0], words[1], words[2], words[3]);
}

// The matrix back from its layout, 8 consecutive columns of a row as one 16-byte store (two for fp32).
// code - zero times scale is exact in fp32 (8 bits times at most 11), so it is rounded once.  8192 x 8192 to
// bf16: 27.3 us, 6.2 TB/s.
template <typename T, typename O>
__global__ void __launch_bounds__(kW4PackThreads) w4_dequantize_kernel(W4Form f, const uint8_t* data, O* out,
                                                                       long long ld, int vec) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int strip = blockIdx.y, block = blockIdx.x;
  const uint8_t* chunk = data + ((size_t)strip * f.blocks + block) * f.chunk_bytes;
  const W4Unit u = w4_unit();
  const uint4 code = *reinterpret_cast<const uint4*>(chunk + w4_unit_offset(u));
  uint32_t words[4] = {code.x, code.y, code.z, code.w};
  w4_exchange(words);
  const int n[2] = {w4_row(f, strip, u.pair, 0), w4_row(f, strip, u.pair, 1)};
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int col = u.col + 32 * q, k = block * kW4Block + col;
    if (k >= f.K) break;
    const uint8_t* sp = chunk + w4_scale_offset(u.pair, col / f.group);
    const float2 scale = W4Traits<T>::to_float2(*reinterpret_cast<const uint32_t*>(sp));
    uint32_t off0 = W4Traits<T>::kMinusEight, off1 = off0;
    if (f.zeros) {
      const uint32_t both = *reinterpret_cast<const uint32_t*>(sp + kW4Block / f.group * 128);
      off0 = __byte_perm(both, 0, 0x1010);
      off1 = __byte_perm(both, 0, 0x3232);
    }
    float v[2][8];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      uint32_t a[4];   // row of the pair: i % 2; columns 2 (i / 2) and the next
      w4_decode<T>(words[2 * q + e], off0, off1, a);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 two = W4Traits<T>::to_float2(W4Traits<T>::fma2(a[i], W4Traits<T>::kBack, 0x80008000u));
        const float by = i & 1 ? scale.y : scale.x;
        v[i & 1][4 * e + 2 * (i >> 1)] = two.x * by;
        v[i & 1][4 * e + 2 * (i >> 1) + 1] = two.y * by;
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (n[j] < 0) continue;
      O* dst = out + (long long)n[j] * ld + k;
      if (vec && k + 8 <= f.K) {
        if constexpr (sizeof(O) == 4) {
          reinterpret_cast<float4*>(dst)[0] = make_float4(v[j][0], v[j][1], v[j][2], v[j][3]);
          reinterpret_cast<float4*>(dst)[1] = make_float4(v[j][4], v[j][5], v[j][6], v[j][7]);
        } else {
          *reinterpret_cast<uint4*>(dst) =
              make_uint4(w4_round2(v[j][0], v[j][1], O()), w4_round2(v[j][2], v[j][3], O()),
                         w4_round2(v[j][4], v[j][5], O()), w4_round2(v[j][6], v[j][7], O()));
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (k + e < f.K) dst[e] = (O)v[j][e];
      }
    }
  }
}

// ------------------------------------------------------------------------------------------
// the product for few tokens
// ------------------------------------------------------------------------------------------
// d = a b (fresh) or d += a b.
template <typename T>
__device__ __forceinline__ void w4_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, bool fresh) {
  const float c0 = fresh ? 0.0f : d[0], c1 = fresh ? 0.0f : d[1], c2 = fresh ? 0.0f : d[2], c3 = fresh ? 0.0f : d[3];
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  }
}

// C^T = W A^T with the weights as the 16-row operand and the tokens, at most 8 NT, as columns.  A warp takes
// every so many-th chunk of one strip; codes go to the matrix instruction as whole numbers
// (code - zero, times a power of two), which the 16-bit types hold exactly.  The sums of a group are exact products
// added in fp32, then times the group's scale in fp32: no weight is rounded on the way.  The warps
// of a CTA and the CTAs of a cluster share a strip along K and add up in a fixed order through
// (distributed) shared memory.
//
// What bounds it is bytes in flight, so a warp keeps kW4Stages chunks, each with the activations that
// meet it, in a shared-memory ring of its own that asynchronous 16-byte copies fill.  A lane copies
// just the pieces that it will itself use, so the ring needs no barrier between warps and no
// registers while the copies fly; lanes meet only over the scales, which four of them share.  One token
// of 8192 x 8192 takes 8.7 us (2 of them a launch and the last CTA's end) with the weights in L2 and 9.3 from memory, so
// neither's bandwidth is the bound; the 128 strips leave 20 SMs without one, and issue slots are half busy.
constexpr int kW4Stages = 2;      // the kernel switches between two offsets
constexpr int kW4SmemMax = 227 * 1024;
constexpr int kW4Pitch = 34;   // float2 per token: the four tokens a warp writes at once hit different banks

// Bytes of a stage: codes of `tiles` of a chunk's four tiles, all its scales, then 256 bytes of
// activations for each of `tokens`.
__host__ __device__ constexpr int w4_stage_bytes(int chunk, int tiles, int tokens) {
  return chunk - (4 - tiles) * 1024 + tokens * 256;
}

// Place of 16 columns (slot of the block) of a token behind the chunk.  Neighbouring tokens swap slots, so
// that the four tokens whose columns a half-warp reads at once lie in different banks.
__device__ __forceinline__ int w4_x_slot(int token, int slot) { return token * 256 + (slot ^ (token & 3)) * 32; }

// Starts the copies of TILES tiles of a chunk (`chunk`: the address of the first, plus this lane's
// 16 bytes; `tail`: that of the chunk's scales) and of the activations of block `block` into a stage.
// x: column 8 t of this lane's token (g of each eight); x_to: where its columns 8 t and 32 + 8 t go.
template <int NT, int TILES, int TAIL>
__device__ __forceinline__ void w4_fill(const W4Params& p, const uint8_t* chunk, const uint8_t* tail,
                                        int block, const uint16_t* const (&x)[NT], const bool (&have)[NT],
                                        const int (&x_to)[2], uint32_t stage, uint8_t* stage_ptr, int lane) {
  const uint32_t dst = stage + lane * 16;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int r = 0; r < TILES; ++r) ptx::cp_async_16(dst + (h * TILES + r) * 512, chunk + (h * 4 + r) * 512);
#pragma unroll
  for (int i = 0; i < TAIL; i += 512)
    if (i + 512 <= TAIL || lane * 16 < TAIL - i) ptx::cp_async_16(dst + TILES * 1024 + i, tail + i);
  const int k0 = block * kW4Block;
  if (p.vec && k0 + kW4Block <= p.form.K) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
      if (have[n]) {
        const uint16_t* from = x[n] + k0;
#pragma unroll
        for (int hq = 0; hq < 4; ++hq)
          ptx::cp_async_16(stage + x_to[hq & 1] + n * 2048 + (hq >> 1) * 128, from + hq * 32);
      }
  } else {
    // The last block of K, and rows that no 16-byte access can start on: lanes take consecutive
    // elements.  Columns behind K are zeroed, so that no product there is a NaN.
    const uint16_t* A = static_cast<const uint16_t*>(p.A) + k0 + lane;
    const int tokens = p.M;
    for (int m0 = 0; m0 < tokens; m0 += 8) {
      uint16_t v[8][4];
#pragma unroll
      for (int m = 0; m < 8; ++m) {
        const uint16_t* row = A + (long long)(m0 + m) * p.lda;
#pragma unroll
        for (int hq = 0; hq < 4; ++hq)
          v[m][hq] = m0 + m < tokens && k0 + hq * 32 + lane < p.form.K ? row[hq * 32] : (uint16_t)0;
      }
#pragma unroll
      for (int m = 0; m < 8; ++m)
        if (m0 + m < tokens)
#pragma unroll
          for (int hq = 0; hq < 4; ++hq)
            *reinterpret_cast<uint16_t*>(stage_ptr + TILES * 1024 + TAIL + w4_x_slot(m0 + m, hq * 2 + (lane >> 4)) + (lane & 15) * 2) = v[m][hq];
    }
  }
}

// The scales (or offsets) of a lane's rows in TILES tiles.
__device__ __forceinline__ void w4_ld_tiles(const uint8_t* p, uint32_t (&v)[4]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
}
__device__ __forceinline__ void w4_ld_tiles(const uint8_t* p, uint32_t (&v)[2]) {
  const uint2 a = *reinterpret_cast<const uint2*>(p);
  v[0] = a.x; v[1] = a.y;
}
__device__ __forceinline__ void w4_ld_tiles(const uint8_t* p, uint32_t (&v)[1]) {
  v[0] = *reinterpret_cast<const uint32_t*>(p);
}

// One CTA to an SM is asked for by name where a warp has one or two tiles: left to itself the compiler makes room for two
// by spilling (12 tokens of 3584 x 8192: 8.6 us so, 7.5 by name; 1 token 5.65 and 5.45; 4 tokens of 1280 x 8192, rotary,
// 4.95 and 4.83).  With four tiles it finds 168 registers at most by itself, and asked by name it spills.
template <typename T, int NT, int TILES, int GROUP, bool ZEROS>
__global__ void __launch_bounds__(NT == 1 ? 512 : 384, TILES <= 2 ? 1 : 0) w4_stream_kernel(const __grid_constant__ W4Params p) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int kGroups = kW4Block / GROUP;
  constexpr int kTail = kGroups * 128 * (ZEROS ? 2 : 1);
  constexpr int kChunk = kW4CodeBytes + kTail;
  constexpr int kCodes = TILES * 1024;   // of a stage
  const W4Form& f = p.form;
  const int warps = blockDim.x >> 5;
  const int strip = blockIdx.x / p.split / (4 / TILES);
  const int tile0 = blockIdx.x / p.split % (4 / TILES) * TILES;
  const int rank = blockIdx.x % p.split;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint8_t* const ring_ptr = smem + warp * p.stage_bytes * kW4Stages;
  const uint32_t ring = ptx::smem_u32(ring_ptr);

  const int step = p.split * warps;
  const int first = rank * warps + warp;
  const size_t chunk_step = (size_t)step * kChunk;
  const uint8_t* tail = p.data + ((size_t)strip * f.blocks + first) * kChunk + kW4CodeBytes + lane * 16;
  const uint8_t* chunk = tail - kW4CodeBytes + tile0 * 512;
  // Before the kernel ahead in the stream has finished nothing is read, but what will be may
  // already be asked into L2.
#pragma unroll
  for (int i = 0; i < kW4Stages; ++i)
    if (first + i * step < f.blocks)
      for (int o = lane * 128; o < kChunk; o += 32 * 128)
        if (TILES == 4 || o >= kW4CodeBytes || (o / 512 % 4 >= tile0 && o / 512 % 4 < tile0 + TILES))
          asm volatile("prefetch.global.L2 [%0];" ::"l"(tail - kW4CodeBytes - lane * 16 + i * chunk_step + o));
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();

  // Columns of the matrix instruction behind the last token compute something that is never stored;
  // their lanes read another token's activations.
  const uint16_t* x[NT];
  bool have[NT];
  const int last = p.M - 1;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    have[n] = n * 8 + g <= last;
    x[n] = static_cast<const uint16_t*>(p.A) + (long long)(have[n] ? n * 8 + g : 0) * p.lda + 8 * t;
  }
  const int gx = min(g, last);
  const int x_to[2] = {kCodes + kTail + w4_x_slot(gx, t >> 1) + (t & 1) * 16,
                       kCodes + kTail + w4_x_slot(gx, 2 + (t >> 1)) + (t & 1) * 16};
#pragma unroll
  for (int i = 0; i < kW4Stages; ++i) {
    if (first + i * step < f.blocks)
      w4_fill<NT, TILES, kTail>(p, chunk, tail, first + i * step, x, have, x_to,
                                ring + i * p.stage_bytes, ring_ptr + i * p.stage_bytes, lane);
    chunk += chunk_step;
    tail += chunk_step;
    ptx::cp_async_commit();
  }

  float acc[TILES][NT][4];
#pragma unroll
  for (int r = 0; r < TILES; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[r][n][i] = 0.0f;

  int at = 0;   // byte offset of the stage
  for (int block = first; block < f.blocks; block += step) {
    ptx::cp_async_wait<kW4Stages - 1>();
    __syncwarp();
    const uint8_t* base = ring_ptr + at;
    const uint8_t* base_codes = base + lane * 16;
    const uint8_t* base_scales = base + kCodes + g * 16 + tile0 * 4;
    const uint8_t* base_x[4];   // this lane's 4 columns of the first four 16
#pragma unroll
    for (int i = 0; i < 4; ++i) base_x[i] = base + kCodes + kTail + w4_x_slot(gx, i) + t * 8;
    float part[TILES][NT][4];
    uint32_t off[TILES][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint4 codes[TILES];
#pragma unroll
      for (int r = 0; r < TILES; ++r) codes[r] = *reinterpret_cast<const uint4*>(base_codes + (h * TILES + r) * 512);
#pragma unroll
      for (int q = 0; q < 2; ++q) {          // 32 columns at a time
        const int hq = h * 2 + q, gi = hq * 32 / GROUP;
        uint2 xv[2][NT];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int n = 0; n < NT; ++n)
            // past the last token of a second eight: another token of the stage (see above)
            xv[s][n] = *reinterpret_cast<const uint2*>(base_x[q * 2 + s] + (n * 8 + g <= last ? n * 2048 : 0) + h * 128);
        const bool fresh = hq * 32 % GROUP == 0;
        if (ZEROS && fresh) {
          uint32_t both[TILES];
          w4_ld_tiles(base_scales + (kGroups + gi) * 128, both);
#pragma unroll
          for (int r = 0; r < TILES; ++r) {
            off[r][0] = __byte_perm(both[r], 0, 0x1010);
            off[r][1] = __byte_perm(both[r], 0, 0x3232);
          }
        }
        // the two instructions of a tile add to one accumulator: other tiles go between them
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
          for (int r = 0; r < TILES; ++r) {
            const uint32_t word = q ? (s ? codes[r].w : codes[r].z) : (s ? codes[r].y : codes[r].x);
            uint32_t a[4];
            w4_decode<T>(word, ZEROS ? off[r][0] : W4Traits<T>::kMinusEight,
                         ZEROS ? off[r][1] : W4Traits<T>::kMinusEight, a);
#pragma unroll
            for (int n = 0; n < NT; ++n)
              w4_mma<T>(part[r][n], a, xv[s][n].x, xv[s][n].y, fresh && s == 0);
          }
        }
        if ((hq + 1) * 32 % GROUP == 0) {
          uint32_t sc[TILES];
          w4_ld_tiles(base_scales + gi * 128, sc);
#pragma unroll
          for (int r = 0; r < TILES; ++r) {
            const float2 sv = W4Traits<T>::to_float2(sc[r]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              acc[r][n][0] += sv.x * part[r][n][0];
              acc[r][n][1] += sv.x * part[r][n][1];
              acc[r][n][2] += sv.y * part[r][n][2];
              acc[r][n][3] += sv.y * part[r][n][3];
            }
          }
        }
      }
    }
    __syncwarp();
    const int ahead = block + kW4Stages * step;
    if (ahead < f.blocks)
      w4_fill<NT, TILES, kTail>(p, chunk, tail, ahead, x, have, x_to, ring + at, ring_ptr + at,
                                lane);
    chunk += chunk_step;
    tail += chunk_step;
    ptx::cp_async_commit();
    at = at == 0 ? p.stage_bytes : 0;
  }

  // The first result's angle is worked out while other warps still multiply.
  const int entry = rank * (warps * 32) + threadIdx.x;
  W4Turn turn = {};
  if (p.epilogue == W4_EPI_ROTARY && entry < p.M * 8 * TILES)
    turn = w4_turn(p, strip, tile0 * 8 + entry % (8 * TILES), entry / (8 * TILES));
  // The warp's sums over its own ring, which nothing is copied into any more and which has room for them: at least
  // 2816 bytes for 8 tokens' 2176, and from 9 tokens on 6912 for 4352.
  static_assert(2 * w4_stage_bytes(kW4CodeBytes + 128, 1, NT == 1 ? 1 : 9) >= NT * 8 * kW4Pitch * 8, "room for the sums");
  float2* red = reinterpret_cast<float2*>(ring_ptr);
  __syncwarp();
#pragma unroll
  for (int r = 0; r < TILES; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      constexpr float kBack = 1.0f / W4Traits<T>::kUnit;
      red[(n * 8 + 2 * t) * kW4Pitch + r * 8 + g] = make_float2(acc[r][n][0] * kBack, acc[r][n][2] * kBack);
      red[(n * 8 + 2 * t + 1) * kW4Pitch + r * 8 + g] = make_float2(acc[r][n][1] * kBack, acc[r][n][3] * kBack);
    }
  if (p.split > 1) ptx::cluster_sync_all();
  else __syncthreads();
  // the CTAs of a cluster share the entries of the result among themselves
  const uint32_t red0 = ptx::smem_u32(smem);
  for (int e = entry; e < p.M * 8 * TILES; e += step * 32) {
    const int token = e / (8 * TILES), pair = e % (8 * TILES);
    float2 v = make_float2(0.0f, 0.0f);
    for (int c = 0; c < p.split; ++c) {
      const uint32_t base = p.split > 1 ? ptx::map_to_cta(red0, c) : red0;
#pragma unroll 4
      for (int w = 0; w < warps; ++w) {
        const float2 a = ptx::ld_cluster_f2(base + w * p.stage_bytes * kW4Stages + (token * kW4Pitch + pair) * 8);
        v.x += a.x;
        v.y += a.y;
      }
    }
    if (p.epilogue == W4_EPI_ROTARY && e != entry) turn = w4_turn(p, strip, tile0 * 8 + pair, token);
    w4_epilogue<T>(p, strip, tile0 * 8 + pair, token, v, turn);
  }
  if (p.split > 1) ptx::cluster_sync_all();   // nobody leaves while its shared memory is read
}

// Rows of 16-bit elements copied to where 16-byte accesses can read them: eight elements a thread.
__global__ void __launch_bounds__(128) align_rows_kernel(const uint16_t* src, long long ld, int rows, int cols,
                                                         uint16_t* dst, long long ld_dst) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const long long pieces = ld_dst / 8, total = rows * pieces;
  for (long long e = (long long)blockIdx.x * 128 + threadIdx.x; e < total; e += (long long)gridDim.x * 128) {
    const long long row = e / pieces;
    const int col = (int)(e - row * pieces) * 8;
    const uint16_t* from = src + row * ld + col;
    uint32_t v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < cols ? from[i] : 0u;
    *reinterpret_cast<uint4*>(dst + row * ld_dst + col) =
        make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
  }
}

// ------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------
static int w4_check(const mk_w4* w, const char* what, bool need_data) {
  if (!w) return set_error(MK_ERR_INVALID, "%s: null weights", what);
  if (w->N < 1 || w->K < 1) return set_error(MK_ERR_INVALID, "%s: N=%d and K=%d must be positive", what, w->N, w->K);
  if (w->group != 32 && w->group != 64 && w->group != 128)
    return set_error(MK_ERR_INVALID, "%s: group=%d must be 32, 64 or 128", what, w->group);
  if (w->dtype != MK_BF16 && w->dtype != MK_FP16)
    return set_error(MK_ERR_INVALID, "%s: dtype=%d must be MK_BF16 or MK_FP16", what, w->dtype);
  if (w->form < MK_W4_PLAIN || w->form > MK_W4_ROTARY)
    return set_error(MK_ERR_INVALID, "%s: unknown form %d", what, w->form);
  if (w->form == MK_W4_GATE_UP && w->N % 2 != 0)
    return set_error(MK_ERR_INVALID, "%s: N=%d must be even (gate rows, then as many up rows)", what, w->N);
  if (w->form == MK_W4_ROTARY) {
    if (w->head_dim < 2 || w->head_dim % 2 != 0 || w->N % w->head_dim != 0)
      return set_error(MK_ERR_INVALID, "%s: head_dim=%d must be even and divide N=%d", what, w->head_dim, w->N);
    if (w->rotary_dim < 2 || w->rotary_dim % 2 != 0 || w->rotary_dim > w->head_dim)
      return set_error(MK_ERR_INVALID, "%s: rotary_dim=%d must be even and within head_dim=%d", what,
                       w->rotary_dim, w->head_dim);
    if (w->rotated_heads < 0 || w->rotated_heads > w->N / w->head_dim)
      return set_error(MK_ERR_INVALID, "%s: rotated_heads=%d of %d heads", what, w->rotated_heads,
                       w->N / w->head_dim);
  }
  const W4Form f = w4_form(*w);
  if (f.strips > 65535)
    return set_error(MK_ERR_INVALID, "%s: N=%d is above %d", what, w->N, 65535 * kW4Strip);
  if (w->K > 1 << 30) return set_error(MK_ERR_INVALID, "%s: K=%d is above %d", what, w->K, 1 << 30);
  if (need_data && (!w->data || (reinterpret_cast<uintptr_t>(w->data) & 15) != 0))
    return set_error(MK_ERR_INVALID, "%s: packed weights must be a 16-byte aligned device buffer", what);
  return MK_OK;
}

// How the few-token product is cut.  All choices follow from how many CTAs there are to fill the SMs;
// figures are microseconds, bf16, group 128, 1 token where none are given, medians of graph replays.
struct W4StreamPlan { int nt, tiles, warps, split, ctas, stage_bytes; };

static W4StreamPlan w4_stream_plan(const W4Form& f, int M, int sms) {
  W4StreamPlan pl;
  pl.nt = M <= 8 ? 1 : 2;
  // Four tiles of rows to a warp share each load of activations, but a narrow matrix gives too few
  // CTAs then: 1280 x 8192 takes 8.5 with 4 tiles, 5.3 with 2, 4.2 with 1; 3584 x 8192: 8.5, 5.4, 8.1;
  // 8192 x 8192: 8.6, 10.6, 15.7.
  pl.tiles = f.strips * 2 > sms ? 4 : f.strips * 4 > sms ? 2 : 1;
  pl.ctas = f.strips * (4 / pl.tiles);
  // One CTA to an SM brings as many warps as fit; more CTAs than SMs share them with fewer (28672 x
  // 8192: 28 with 8 warps, 33 with 16; 13 tokens, whose CTAs are larger: 41 with 4, 47 with 8, 48 with 12).  A
  // warp without a chunk is of no use.
  pl.warps = pl.ctas > sms ? (pl.nt == 1 ? 8 : 4) : pl.nt == 1 ? 16 : 12;
  if (pl.warps > f.blocks) pl.warps = f.blocks < 4 ? 4 : f.blocks;
  // Clusters along K only where most SMs would be idle and a CTA keeps 8 blocks or more: 256 x 8192 takes 3.9
  // in clusters of 4 and 4.1 without, 1024 x 1024 3.5 in clusters of 2 and 2.1 without.
  pl.split = 1;
  while (pl.split < 8 && pl.ctas * pl.split * 4 <= sms && pl.split * 16 <= f.blocks) pl.split *= 2;
  if (pl.split > 1) pl.warps = 8;
  pl.ctas *= pl.split;
  pl.stage_bytes = w4_stage_bytes(f.chunk_bytes, pl.tiles, M);
  return pl;
}

template <typename T, int NT, int TILES, int GROUP, bool ZEROS>
static int w4_stream_launch(const W4Params& p, dim3 grid, int warps, cudaStream_t stream) {
  auto kern = w4_stream_kernel<T, NT, TILES, GROUP, ZEROS>;
  static bool attr_set[64];
  int dev = 0;
  MKB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    MKB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kW4SmemMax));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  return w4_launch(kern, grid, warps * 32, warps * kW4Stages * p.stage_bytes, p.split, stream, p);
}
template <typename T, int NT, int TILES>
static int w4_stream_group(const W4Params& p, dim3 grid, int warps, cudaStream_t stream) {
  const bool z = p.form.zeros;
  switch (p.form.group) {
    case 32: return z ? w4_stream_launch<T, NT, TILES, 32, true>(p, grid, warps, stream)
                      : w4_stream_launch<T, NT, TILES, 32, false>(p, grid, warps, stream);
    case 64: return z ? w4_stream_launch<T, NT, TILES, 64, true>(p, grid, warps, stream)
                      : w4_stream_launch<T, NT, TILES, 64, false>(p, grid, warps, stream);
    default: return z ? w4_stream_launch<T, NT, TILES, 128, true>(p, grid, warps, stream)
                      : w4_stream_launch<T, NT, TILES, 128, false>(p, grid, warps, stream);
  }
}
template <typename T>
static int w4_stream_type(const W4Params& p, const W4StreamPlan& pl, dim3 grid, cudaStream_t s) {
  if (pl.nt == 1)
    return pl.tiles == 4   ? w4_stream_group<T, 1, 4>(p, grid, pl.warps, s)
           : pl.tiles == 2 ? w4_stream_group<T, 1, 2>(p, grid, pl.warps, s)
                           : w4_stream_group<T, 1, 1>(p, grid, pl.warps, s);
  return pl.tiles == 4   ? w4_stream_group<T, 2, 4>(p, grid, pl.warps, s)
         : pl.tiles == 2 ? w4_stream_group<T, 2, 2>(p, grid, pl.warps, s)
                         : w4_stream_group<T, 2, 1>(p, grid, pl.warps, s);
}

// Whether the tile kernel multiplies what rounding the weights leaves.
static bool w4_rest(int form, int flags) { return form == MK_W4_GATE_UP || (flags & MK_W4_EXACT) != 0; }

static int w4_product(const char* what, const void* A, long long lda, const mk_w4* w, void* C, long long ldc,
                      int M, int form, int epilogue, const RotaryArgs& rotary, int flags, void* stream) {
  int rc = w4_check(w, what, true);
  if (rc != MK_OK) return rc;
  if (w->form != form)
    return set_error(MK_ERR_INVALID, "%s: the weights were laid out in form %d, this product takes form %d", what,
                     w->form, form);
  const int n_out = epilogue == W4_EPI_SWIGLU ? w->N / 2 : w->N;
  if (M < 0) return set_error(MK_ERR_INVALID, "%s: M=%d is negative", what, M);
  if ((flags & ~MK_W4_EXACT) != 0) return set_error(MK_ERR_INVALID, "%s: unknown flags %d", what, flags);
  if (M == 0) return MK_OK;
  if (!A || !C) return set_error(MK_ERR_INVALID, "%s: null operand", what);
  if (lda < w->K || ldc < n_out)
    return set_error(MK_ERR_INVALID, "%s: row strides %lld and %lld must be at least K=%d and %d", what, lda, ldc,
                     w->K, n_out);
  if (((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(C)) & 1) != 0)
    return set_error(MK_ERR_INVALID, "%s: operands must be 2-byte aligned", what);
  const bool vec = (reinterpret_cast<uintptr_t>(A) & 15) == 0 && (lda % 8 == 0 || M == 1);
  if (M > kW4StreamTokens && !vec)
    return set_error(MK_ERR_INVALID, "%s: for more than 16 rows A's must start on 16 bytes (mk_align_rows copies them so)",
                     what);
  int sms = 0;
  rc = device_sm_count(&sms);
  if (rc != MK_OK) return rc;
  W4Params p;
  memset(&p, 0, sizeof(p));
  p.form = w4_form(*w);
  p.data = static_cast<const uint8_t*>(w->data);
  p.A = A; p.lda = lda; p.C = C; p.ldc = ldc; p.M = M;
  p.vec = vec;
  p.epilogue = epilogue;
  p.rotary = rotary;
  p.wide = (reinterpret_cast<uintptr_t>(C) & 7) == 0 && ldc % 4 == 0;
  p.wait_limit_ns = option_wait_limit_ns();
  p.debug_flags = option_debug_flags();
  // Up to 16 tokens one pass of the stream kernel over the weights does, and the next 16 would take another: 8192 x
  // 8192 takes it 12.7 us for 16 tokens and the tile kernel 14.5 for 17 (1024 x 8192: 7.1 and 10.5; 28672 x 8192: 43
  // and 47).
  if (M > kW4StreamTokens) return w4_tile_launch(p, w->dtype, w4_rest(form, flags), sms, static_cast<cudaStream_t>(stream));
  const W4StreamPlan pl = w4_stream_plan(p.form, M, sms);
  p.stage_bytes = pl.stage_bytes;
  p.split = pl.split;
  const dim3 grid(pl.ctas, 1, 1);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return w->dtype == MK_BF16 ? w4_stream_type<__nv_bfloat16>(p, pl, grid, s)
                             : w4_stream_type<__half>(p, pl, grid, s);
}

template <typename T, typename S>
static int w4_quantize_group(const W4PackParams& p, dim3 grid, cudaStream_t s) {
  const bool z = p.form.zeros;
  auto kern = p.form.group == 32   ? (z ? w4_quantize_kernel<T, S, 32, true> : w4_quantize_kernel<T, S, 32, false>)
              : p.form.group == 64 ? (z ? w4_quantize_kernel<T, S, 64, true> : w4_quantize_kernel<T, S, 64, false>)
                                   : (z ? w4_quantize_kernel<T, S, 128, true> : w4_quantize_kernel<T, S, 128, false>);
  return w4_launch(kern, grid, kW4PackThreads, 0, 1, s, p);
}

template <typename T>
static int w4_quantize_launch(const W4PackParams& p, int src_dtype, dim3 grid, cudaStream_t s) {
  if (src_dtype == MK_BF16) return w4_quantize_group<T, __nv_bfloat16>(p, grid, s);
  if (src_dtype == MK_FP16) return w4_quantize_group<T, __half>(p, grid, s);
  return w4_quantize_group<T, float>(p, grid, s);
}

template <typename T>
static int w4_dequantize_launch(const W4Form& f, const uint8_t* data, void* out, long long ld, int dtype, int vec,
                                dim3 grid, cudaStream_t s) {
  if (dtype == MK_BF16)
    return w4_launch(w4_dequantize_kernel<T, __nv_bfloat16>, grid, kW4PackThreads, 0, 1, s, f, data,
                     static_cast<__nv_bfloat16*>(out), ld, vec);
  if (dtype == MK_FP16)
    return w4_launch(w4_dequantize_kernel<T, __half>, grid, kW4PackThreads, 0, 1, s, f, data, static_cast<__half*>(out),
                     ld, vec);
  return w4_launch(w4_dequantize_kernel<T, float>, grid, kW4PackThreads, 0, 1, s, f, data, static_cast<float*>(out), ld,
                   vec);
}

static int w4_dtype_size(int dtype) { return dtype == MK_FP32 ? 4 : 2; }

}  // namespace mkb

using namespace mkb;

extern "C" {

long long mk_w4_bytes(const mk_w4* w) {
  const int rc = w4_check(w, "mk_w4_bytes", false);
  if (rc != MK_OK) return rc;
  const W4Form f = w4_form(*w);
  return (long long)f.strips * f.blocks * f.chunk_bytes;
}

int mk_w4_pack(const mk_w4* w, const uint8_t* codes, const void* scales, const uint8_t* zero_points, void* stream) {
  int rc = w4_check(w, "mk_w4_pack", true);
  if (rc != MK_OK) return rc;
  if (!codes || !scales || (w->zeros != 0) != (zero_points != nullptr))
    return set_error(MK_ERR_INVALID, "mk_w4_pack: codes and scales are needed, zero points exactly when zeros is 1");
  if ((reinterpret_cast<uintptr_t>(scales) & 1) != 0)
    return set_error(MK_ERR_INVALID, "mk_w4_pack: scales must be 2-byte aligned");
  int sms = 0;
  rc = device_sm_count(&sms);
  if (rc != MK_OK) return rc;
  W4PackParams p;
  memset(&p, 0, sizeof(p));
  p.form = w4_form(*w);
  p.data = static_cast<uint8_t*>(w->data);
  p.codes = codes;
  p.scales = static_cast<const uint16_t*>(scales);
  p.zero_points = zero_points;
  const dim3 grid(p.form.blocks, p.form.strips, 1);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return w->dtype == MK_BF16 ? w4_launch(w4_pack_kernel<__nv_bfloat16>, grid, kW4PackThreads, 0, 1, s, p)
                             : w4_launch(w4_pack_kernel<__half>, grid, kW4PackThreads, 0, 1, s, p);
}

int mk_w4_quantize(const mk_w4* w, const void* src, long long ld, int src_dtype, void* stream) {
  int rc = w4_check(w, "mk_w4_quantize", true);
  if (rc != MK_OK) return rc;
  if (!src || ld < w->K) return set_error(MK_ERR_INVALID, "mk_w4_quantize: null source, or row stride below K=%d", w->K);
  if (src_dtype < MK_BF16 || src_dtype > MK_FP32)
    return set_error(MK_ERR_INVALID, "mk_w4_quantize: unknown source dtype %d", src_dtype);
  const int size = w4_dtype_size(src_dtype);
  if (reinterpret_cast<uintptr_t>(src) % size != 0)
    return set_error(MK_ERR_INVALID, "mk_w4_quantize: misaligned source");
  int sms = 0;
  rc = device_sm_count(&sms);
  if (rc != MK_OK) return rc;
  W4PackParams p;
  memset(&p, 0, sizeof(p));
  p.form = w4_form(*w);
  p.data = static_cast<uint8_t*>(w->data);
  p.src = src;
  p.ld = ld;
  p.vec = (reinterpret_cast<uintptr_t>(src) & 15) == 0 && ld * size % 16 == 0;
  const dim3 grid(p.form.blocks, p.form.strips, 1);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  return w->dtype == MK_BF16 ? w4_quantize_launch<__nv_bfloat16>(p, src_dtype, grid, s)
                             : w4_quantize_launch<__half>(p, src_dtype, grid, s);
}

int mk_w4_dequantize(const mk_w4* w, void* out, long long ld, int out_dtype, void* stream) {
  int rc = w4_check(w, "mk_w4_dequantize", true);
  if (rc != MK_OK) return rc;
  if (!out || ld < w->K) return set_error(MK_ERR_INVALID, "mk_w4_dequantize: null output, or row stride below K=%d", w->K);
  if (out_dtype < MK_BF16 || out_dtype > MK_FP32)
    return set_error(MK_ERR_INVALID, "mk_w4_dequantize: unknown output dtype %d", out_dtype);
  const int size = w4_dtype_size(out_dtype);
  if (reinterpret_cast<uintptr_t>(out) % size != 0)
    return set_error(MK_ERR_INVALID, "mk_w4_dequantize: misaligned output");
  int sms = 0;
  rc = device_sm_count(&sms);
  if (rc != MK_OK) return rc;
  const W4Form f = w4_form(*w);
  const int vec = (reinterpret_cast<uintptr_t>(out) & 15) == 0 && ld * size % 16 == 0;
  const dim3 grid(f.blocks, f.strips, 1);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uint8_t* data = static_cast<const uint8_t*>(w->data);
  return w->dtype == MK_BF16 ? w4_dequantize_launch<__nv_bfloat16>(f, data, out, ld, out_dtype, vec, grid, s)
                             : w4_dequantize_launch<__half>(f, data, out, ld, out_dtype, vec, grid, s);
}

int mk_align_rows(const void* src, long long ld, int rows, int cols, void* dst, long long ld_dst, void* stream) {
  if (rows < 0 || cols < 1) return set_error(MK_ERR_INVALID, "mk_align_rows: bad shape %d x %d", rows, cols);
  if (rows == 0) return MK_OK;
  if (!src || !dst || ld < cols || ld_dst < cols || ld_dst % 8 != 0 || (reinterpret_cast<uintptr_t>(dst) & 15) != 0 ||
      (reinterpret_cast<uintptr_t>(src) & 1) != 0)
    return set_error(MK_ERR_INVALID, "mk_align_rows: needs whole rows, a 16-byte aligned copy and its stride a multiple of 8");
  int sms = 0;
  const int rc = device_sm_count(&sms);
  if (rc != MK_OK) return rc;
  long long blocks = ((long long)rows * (ld_dst / 8) + 127) / 128;
  if (blocks > 16LL * sms) blocks = 16LL * sms;
  return w4_launch(align_rows_kernel, dim3((unsigned)blocks), 128, 0, 1, static_cast<cudaStream_t>(stream),
                   static_cast<const uint16_t*>(src), ld, rows, cols, static_cast<uint16_t*>(dst), ld_dst);
}

int mk_w4_plan_product(const mk_w4* w, int M, int flags, mk_w4_plan* out) {
  int rc = w4_check(w, "mk_w4_plan_product", false);
  if (rc != MK_OK) return rc;
  if (!out || M < 1 || (flags & ~MK_W4_EXACT) != 0)
    return set_error(MK_ERR_INVALID, "mk_w4_plan_product: null plan, M=%d below 1 or unknown flags %d", M, flags);
  int sms = 0;
  rc = device_sm_count(&sms);
  if (rc != MK_OK) return rc;
  const W4Form f = w4_form(*w);
  memset(out, 0, sizeof(*out));
  if (M > kW4StreamTokens) {
    W4TilePlan pl;
    const bool rest = w4_rest(w->form, flags);
    rc = w4_tile_plan(f, M, rest, sms, &pl);
    if (rc != MK_OK) return rc;
    out->tile = 1; out->tokens = pl.tokens; out->split = pl.split; out->ctas = (int)pl.ctas; out->rest = rest;
    return MK_OK;
  }
  const W4StreamPlan pl = w4_stream_plan(f, M, sms);
  out->tokens = 8 * pl.nt; out->split = pl.split; out->ctas = pl.ctas; out->tiles = pl.tiles; out->warps = pl.warps;
  return MK_OK;
}

int mk_w4_gemm_ex(const void* A, long long lda, const mk_w4* w, void* C, long long ldc, int M, int flags, void* stream) {
  return w4_product("mk_w4_gemm", A, lda, w, C, ldc, M, MK_W4_PLAIN, W4_EPI_NONE, RotaryArgs{}, flags, stream);
}

int mk_w4_gemm(const void* A, long long lda, const mk_w4* w, void* C, long long ldc, int M, void* stream) {
  return mk_w4_gemm_ex(A, lda, w, C, ldc, M, 0, stream);
}

int mk_w4_gemm_swiglu(const void* A, long long lda, const mk_w4* w, void* H, long long ldh, int M, void* stream) {
  return w4_product("mk_w4_gemm_swiglu", A, lda, w, H, ldh, M, MK_W4_GATE_UP, W4_EPI_SWIGLU, RotaryArgs{}, 0, stream);
}

int mk_w4_gemm_rotary_ex(const void* A, long long lda, const mk_w4* w, void* C, long long ldc, int M,
                         const void* positions, int pos64, const float* inv_freq, float scale, int flags, void* stream) {
  if (M > 0 && (!positions || !inv_freq)) return set_error(MK_ERR_INVALID, "mk_w4_gemm_rotary: null positions or frequencies");
  if (reinterpret_cast<uintptr_t>(positions) % (pos64 ? 8 : 4) != 0 || reinterpret_cast<uintptr_t>(inv_freq) % 4 != 0)
    return set_error(MK_ERR_INVALID, "mk_w4_gemm_rotary: misaligned positions or frequencies");
  RotaryArgs r;
  r.positions = positions; r.pos64 = pos64 != 0; r.inv_freq = inv_freq; r.scale = scale;
  return w4_product("mk_w4_gemm_rotary", A, lda, w, C, ldc, M, MK_W4_ROTARY, W4_EPI_ROTARY, r, flags, stream);
}

int mk_w4_gemm_rotary(const void* A, long long lda, const mk_w4* w, void* C, long long ldc, int M,
                      const void* positions, int pos64, const float* inv_freq, float scale, void* stream) {
  return mk_w4_gemm_rotary_ex(A, lda, w, C, ldc, M, positions, pos64, inv_freq, scale, 0, stream);
}

}  // extern "C"
