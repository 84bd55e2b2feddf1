// Products with 4-bit weights (group scales, optional zero points), their SwiGLU and rotary forms,
// and the kernels that lay the weights out.  The layout is described in w4_layout.cuh.
#include <cuda_runtime.h>

#include <cstring>

#include "../../include/mkernel_b200.h"
#include "host_util.h"
#include "ptx.cuh"
#include "rotary.cuh"
#include "w4_layout.cuh"

namespace mkb {

// ------------------------------------------------------------------------------------------
// laying the weights out
// ------------------------------------------------------------------------------------------
// One CTA of 256 threads per chunk.  Thread = (row of the strip, segment of 32 columns); the four
// segments of a row are neighbouring lanes, so a group of 64 or 128 columns is reduced by shuffles.
// Codes pass through shared memory once to change from row order to the layout's order.
constexpr int kW4PackThreads = 256;
constexpr int kW4CodePitch = kW4Block + 4;   // bytes; 33 words: rows start in different banks

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
  int vec;   // source rows are 16-byte aligned
};

// Row (within a strip) of pair p, member j, in the order of the layout's tiles.
__device__ __forceinline__ int w4_tile_row(int p, int j) { return (p / 8) * 16 + j * 8 + p % 8; }

// Writes a chunk from codes [64 tile rows][128 columns] in shared memory.
__device__ __forceinline__ void w4_store_codes(const uint8_t* sh, uint8_t* chunk) {
  const int tid = threadIdx.x;
  const int lane = tid & 31, ht = tid >> 5;          // ht: half (bit 2) and tile (bits 0, 1)
  const int g = lane >> 2, t = lane & 3;
  const uint8_t* base = sh + ((ht & 3) * 16 + g) * kW4CodePitch + (ht >> 2) * 64;
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int col = 32 * (j >> 1) + 8 * t + 4 * (j & 1);
    uint32_t v = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        v |= (uint32_t)base[(i & 1) * 8 * kW4CodePitch + col + 2 * (i >> 1) + e] << (4 * i + 16 * e);
    w[j] = v;
  }
  reinterpret_cast<uint4*>(chunk)[tid] = make_uint4(w[0], w[1], w[2], w[3]);
}

// Place of (tile row, group of the block) among a chunk's scales, in 16-bit units.
__device__ __forceinline__ int w4_scale_slot(int row, int group) {
  return group * kW4Strip + (row & 7) * 8 + (row >> 4) * 2 + ((row >> 3) & 1);
}

template <typename T>
__device__ __forceinline__ void w4_store_scale(const W4Form& f, uint8_t* chunk, int row, int group,
                                               uint16_t scale, int zero) {
  uint16_t* s = reinterpret_cast<uint16_t*>(chunk + kW4CodeBytes);
  const int slot = w4_scale_slot(row, group);
  s[slot] = scale;
  if (f.zeros)
    s[(kW4Block / f.group) * kW4Strip + slot] = (uint16_t)((W4Traits<T>::kMagic & 0xffff) + zero);
}

template <typename T>
__global__ void __launch_bounds__(kW4PackThreads) w4_pack_kernel(W4PackParams p) {
  __shared__ uint8_t sh[kW4Strip * kW4CodePitch];
  const W4Form& f = p.form;
  const int strip = blockIdx.x / f.blocks, block = blockIdx.x % f.blocks;
  uint8_t* chunk = p.data + (size_t)blockIdx.x * f.chunk_bytes;
  const int row = threadIdx.x >> 2, seg = threadIdx.x & 3;
  const int pair = (row >> 4) * 8 + (row & 7);
  const int n = w4_row(f, strip, pair, (row >> 3) & 1);
  const long long k0 = (long long)block * kW4Block + seg * 32;
  const long long row_bytes = ((long long)f.K + 1) / 2;
  for (int c = 0; c < 32; c += 2) {
    const bool in = n >= 0 && k0 + c < f.K;
    const uint8_t b = in ? __ldg(p.codes + n * row_bytes + (k0 + c) / 2) : 0x88;
    sh[row * kW4CodePitch + seg * 32 + c] = b & 15;
    sh[row * kW4CodePitch + seg * 32 + c + 1] = k0 + c + 1 < f.K ? b >> 4 : 8;
  }
  const int segs = f.group / 32;
  if (seg % segs == 0) {
    const long long groups = ((long long)f.K + f.group - 1) / f.group;
    const long long gi = k0 / f.group;
    const bool in = n >= 0 && k0 < f.K;
    const uint16_t s = in ? __ldg(p.scales + n * groups + gi) : 0;
    const int z = in && f.zeros ? __ldg(p.zero_points + n * groups + gi) & 15 : 8;
    w4_store_scale<T>(f, chunk, row, seg / segs, s, z);
  }
  __syncthreads();
  w4_store_codes(sh, chunk);
}

// Quantiser: reads the matrix once, writes the chunk.  Bound by memory: 2 (or 4) bytes in, 0.53
// out per weight.
template <typename S>
__device__ __forceinline__ float w4_src(const S* p) { return (float)__ldg(p); }

template <typename T, typename S>
__global__ void __launch_bounds__(kW4PackThreads) w4_quantize_kernel(W4PackParams p) {
  __shared__ uint8_t sh[kW4Strip * kW4CodePitch];
  const W4Form& f = p.form;
  const int strip = blockIdx.x / f.blocks, block = blockIdx.x % f.blocks;
  uint8_t* chunk = p.data + (size_t)blockIdx.x * f.chunk_bytes;
  const int row = threadIdx.x >> 2, seg = threadIdx.x & 3;
  const int pair = (row >> 4) * 8 + (row & 7);
  const int n = w4_row(f, strip, pair, (row >> 3) & 1);
  const long long k0 = (long long)block * kW4Block + seg * 32;
  const S* src = static_cast<const S*>(p.src) + (long long)(n < 0 ? 0 : n) * p.ld + k0;
  float w[32];
  if (n >= 0 && p.vec && k0 + 32 <= f.K) {
    constexpr int kPer = 16 / sizeof(S);
#pragma unroll
    for (int c = 0; c < 32; c += kPer) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(src + c));
      const S* e = reinterpret_cast<const S*>(&v);
#pragma unroll
      for (int i = 0; i < kPer; ++i) w[c + i] = (float)e[i];
    }
  } else {
#pragma unroll
    for (int c = 0; c < 32; ++c) w[c] = n >= 0 && k0 + c < f.K ? w4_src(src + c) : 0.0f;
  }
  float lo = 0.0f, hi = 0.0f;
  bool finite = true;
#pragma unroll
  for (int c = 0; c < 32; ++c) {
    lo = fminf(lo, w[c]);
    hi = fmaxf(hi, w[c]);
    finite = finite && isfinite(w[c]);
  }
  for (int d = 1; d < f.group / 32; d *= 2) {
    lo = fminf(lo, __shfl_xor_sync(~0u, lo, d));
    hi = fmaxf(hi, __shfl_xor_sync(~0u, hi, d));
    finite = __shfl_xor_sync(~0u, (int)finite, d) && finite;
  }
  const float range = f.zeros ? __fdiv_rn(hi - lo, 15.0f) : __fdiv_rn(fmaxf(fabsf(lo), hi), 7.0f);
  T scale_t = W4Traits<T>::from_float(finite ? range : __int_as_float(0x7fc00000));
  const uint16_t scale_bits = *reinterpret_cast<uint16_t*>(&scale_t);
  const float scale = W4Traits<T>::to_float(scale_bits);
  const float divisor = scale == 0.0f ? 1.0f : scale;
  const float zero = f.zeros ? fminf(fmaxf(rintf(__fdiv_rn(-lo, divisor)), 0.0f), 15.0f) : 8.0f;
#pragma unroll
  for (int c = 0; c < 32; c += 4) {
    uint32_t v = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float q = fminf(fmaxf(rintf(__fdiv_rn(w[c + i], divisor)) + zero, 0.0f), 15.0f);
      if (n < 0 || k0 + c + i >= f.K) q = 8.0f;   // behind the matrix: as pack leaves it
      v |= (uint32_t)(int)q << (8 * i);
    }
    *reinterpret_cast<uint32_t*>(sh + row * kW4CodePitch + seg * 32 + c) = v;
  }
  const int segs = f.group / 32;
  if (seg % segs == 0)
    w4_store_scale<T>(f, chunk, row, seg / segs, scale_bits, n >= 0 && k0 < f.K ? (int)zero : 8);
  __syncthreads();
  w4_store_codes(sh, chunk);
}

// The matrix back from its layout: one CTA per chunk, one 16-byte access of codes per thread, whose
// 8 consecutive columns of a row leave as one 16-byte store (two for fp32 output).
template <typename T, typename O>
__global__ void __launch_bounds__(256) w4_dequantize_kernel(W4Form f, const uint8_t* data, O* out,
                                                            long long ld, int vec) {
  const int strip = blockIdx.x / f.blocks, block = blockIdx.x % f.blocks;
  const uint8_t* chunk = data + (size_t)blockIdx.x * f.chunk_bytes;
  const int lane = threadIdx.x & 31, ht = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3, tile = ht & 3;
  const uint4 c = __ldg(reinterpret_cast<const uint4*>(chunk) + threadIdx.x);
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
  const uint16_t* s = reinterpret_cast<const uint16_t*>(chunk + kW4CodeBytes);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int row = tile * 16 + j * 8 + g;
    const int n = w4_row(f, strip, tile * 8 + g, j);
    if (n < 0) continue;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int col = (ht >> 2) * 64 + q * 32 + 8 * t;
      const long long k = (long long)block * kW4Block + col;
      if (k >= f.K) continue;
      const int slot = w4_scale_slot(row, col / f.group);
      const float scale = W4Traits<T>::to_float(__ldg(s + slot));
      const int zero = f.zeros ? (int)__ldg(s + (kW4Block / f.group) * kW4Strip + slot) -
                                     (int)(W4Traits<T>::kMagic & 0xffff)
                               : 8;
      O v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int code = (w[2 * q + (e >> 2)] >> (4 * (j + 2 * ((e >> 1) & 1)) + 16 * (e & 1))) & 15;
        const float x = (float)(code - zero) * scale;
        v[e] = (O)x;   // to the nearest, ties to even
      }
      O* dst = out + (long long)n * ld + k;
      if (vec && k + 8 <= f.K) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(O) / 2; ++i)
          reinterpret_cast<uint4*>(dst)[i] = reinterpret_cast<const uint4*>(v)[i];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (k + e < f.K) dst[e] = v[e];
      }
    }
  }
}

// ------------------------------------------------------------------------------------------
// the product for few tokens
// ------------------------------------------------------------------------------------------
enum W4Epilogue : int { W4_EPI_NONE = 0, W4_EPI_SWIGLU = 1, W4_EPI_ROTARY = 2 };

struct W4Params {
  W4Form form;
  const uint8_t* data;
  const void* A;
  long long lda;
  void* C;
  long long ldc;
  int M;
  int vec;        // rows of A are 16-byte aligned and K is a multiple of 8
  int split;      // CTAs of a cluster, which share a strip along K
  int epilogue;
  RotaryArgs rotary;
};

// C's entries of one pair of rows and one token.
template <typename T>
__device__ __forceinline__ void w4_epilogue(const W4Params& p, int strip, int pair, int token, float2 v) {
  const W4Form& f = p.form;
  const int n0 = w4_row(f, strip, pair, 0);
  if (n0 < 0) return;
  T* row = static_cast<T*>(p.C) + (long long)token * p.ldc;
  if (p.epilogue == W4_EPI_SWIGLU) {
    // silu in fp32; for a gate below -88 the exponential is inf and the quotient -0, as it should be
    row[n0] = W4Traits<T>::from_float(v.x / (1.0f + __expf(-v.x)) * v.y);
    return;
  }
  const int n1 = w4_row(f, strip, pair, 1);
  if (p.epilogue == W4_EPI_ROTARY) {
    const int half = f.head_dim / 2;
    const int index = strip * (kW4Strip / 2) + pair, head = index / half, i = index % half;
    if (head < f.rotated_heads && i < f.rotary_dim / 2)
      v = rotary_turn(v.x, v.y, rotary_cos_sin(rotary_position(p.rotary, token),
                                               __ldg(p.rotary.inv_freq + i), p.rotary.scale));
  }
  row[n0] = W4Traits<T>::from_float(v.x);
  if (n1 >= 0) row[n1] = W4Traits<T>::from_float(v.y);
}

__device__ __forceinline__ uint4 w4_ld_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

template <typename T>
__device__ __forceinline__ void w4_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (sizeof(T) == 2 && W4Traits<T>::kMagic == 0x43004300u) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

// Eight consecutive activations of a token, zeros outside of [M, K].
template <typename T>
__device__ __forceinline__ uint4 w4_ld_x(const W4Params& p, int token, long long k) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (token < p.M && k < p.form.K) {
    const uint16_t* x = static_cast<const uint16_t*>(p.A) + (long long)token * p.lda + k;
    if (p.vec) {
      v = __ldg(reinterpret_cast<const uint4*>(x));
    } else {
      uint16_t e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = k + i < p.form.K ? __ldg(x + i) : (uint16_t)0;
      v.x = e[0] | (uint32_t)e[1] << 16;
      v.y = e[2] | (uint32_t)e[3] << 16;
      v.z = e[4] | (uint32_t)e[5] << 16;
      v.w = e[6] | (uint32_t)e[7] << 16;
    }
  }
  return v;
}

// C^T = W A^T with the weights as the 16-row operand and up to 8 NT tokens as columns.  A warp walks
// the chunks of one strip, its share of K; codes go from memory straight into the registers that
// the matrix instruction takes them from, as whole numbers (code - zero), which the 16-bit types
// hold exactly.  The sums of a group are exact products added in fp32, then times the group's
// scale in fp32: no weight is rounded on the way.  The warps of a CTA and the CTAs of a cluster share a strip
// along K and add up in a fixed order through (distributed) shared memory.
constexpr int kW4Warps = 4;
constexpr int kW4Pitch = 34;   // float2 per token: the four tokens a warp writes at once hit different banks

template <typename T, int NT, int GROUP, bool ZEROS>
__global__ void __launch_bounds__(kW4Warps * 32) w4_stream_kernel(const __grid_constant__ W4Params p) {
  __shared__ float2 red[kW4Warps][NT * 8][kW4Pitch];
  constexpr int kGroups = kW4Block / GROUP;
  const W4Form& f = p.form;
  const int strip = blockIdx.x / p.split;
  const int rank = blockIdx.x % p.split;
  const int token0 = blockIdx.y * 8 * NT;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();

  float acc[4][NT][4];
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[r][n][i] = 0.0f;

  const uint8_t* data = p.data + (size_t)strip * f.blocks * f.chunk_bytes;
  for (int block = rank * kW4Warps + warp; block < f.blocks; block += p.split * kW4Warps) {
    const uint8_t* chunk = data + (size_t)block * f.chunk_bytes;
    uint4 codes[8], scales[kGroups], offsets[kGroups];
#pragma unroll
    for (int i = 0; i < 8; ++i) codes[i] = w4_ld_stream(chunk + (i * 32 + lane) * 16);
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      scales[i] = w4_ld_stream(chunk + kW4CodeBytes + i * 128 + g * 16);
      if (ZEROS) offsets[i] = w4_ld_stream(chunk + kW4CodeBytes + (kGroups + i) * 128 + g * 16);
    }
    float part[4][NT][4];
#pragma unroll
    for (int hq = 0; hq < 4; ++hq) {          // 32 columns at a time
      const int gi = hq * 32 / GROUP;
      uint4 x[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n)
        x[n] = w4_ld_x<T>(p, token0 + n * 8 + g, (long long)block * kW4Block + hq * 32 + 8 * t);
      if (hq * 32 % GROUP == 0) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) part[r][n][i] = 0.0f;
      }
      const uint32_t off[4] = {offsets[gi].x, offsets[gi].y, offsets[gi].z, offsets[gi].w};
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint4 c = codes[(hq >> 1) * 4 + r];
          const uint32_t word = (hq & 1) ? (s ? c.w : c.z) : (s ? c.y : c.x);
          uint32_t off0 = W4Traits<T>::kEight, off1 = W4Traits<T>::kEight;
          if (ZEROS) {
            off0 = __byte_perm(off[r], 0, 0x1010);
            off1 = __byte_perm(off[r], 0, 0x3232);
          }
          const uint32_t a[4] = {w4_decode<T>(word, 0, off0), w4_decode<T>(word, 1, off1),
                                 w4_decode<T>(word, 2, off0), w4_decode<T>(word, 3, off1)};
#pragma unroll
          for (int n = 0; n < NT; ++n)
            w4_mma<T>(part[r][n], a, s ? x[n].z : x[n].x, s ? x[n].w : x[n].y);
        }
      }
      if ((hq + 1) * 32 % GROUP == 0) {
        const uint32_t sc[4] = {scales[gi].x, scales[gi].y, scales[gi].z, scales[gi].w};
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float s0 = W4Traits<T>::to_float(sc[r] & 0xffff), s1 = W4Traits<T>::to_float(sc[r] >> 16);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            acc[r][n][0] += s0 * part[r][n][0];
            acc[r][n][1] += s0 * part[r][n][1];
            acc[r][n][2] += s1 * part[r][n][2];
            acc[r][n][3] += s1 * part[r][n][3];
          }
        }
      }
    }
  }

#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      red[warp][n * 8 + 2 * t][r * 8 + g] = make_float2(acc[r][n][0], acc[r][n][2]);
      red[warp][n * 8 + 2 * t + 1][r * 8 + g] = make_float2(acc[r][n][1], acc[r][n][3]);
    }
  if (p.split > 1) ptx::cluster_sync_all();
  else __syncthreads();
  // the CTAs of a cluster share the entries of the result among themselves
  const uint32_t red0 = ptx::smem_u32(&red[0][0][0]);
  for (int e = rank * (kW4Warps * 32) + threadIdx.x; e < NT * 8 * 32; e += p.split * kW4Warps * 32) {
    const int token = e >> 5, pair = e & 31;
    if (token0 + token >= p.M) break;
    float2 v = make_float2(0.0f, 0.0f);
    for (int c = 0; c < p.split; ++c) {
      const uint32_t base = p.split > 1 ? ptx::map_to_cta(red0, c) : red0;
#pragma unroll
      for (int w = 0; w < kW4Warps; ++w) {
        const float2 a = ptx::ld_cluster_f2(base + ((w * NT * 8 + token) * kW4Pitch + pair) * 8);
        v.x += a.x;
        v.y += a.y;
      }
    }
    w4_epilogue<T>(p, strip, pair, token0 + token, v);
  }
  if (p.split > 1) ptx::cluster_sync_all();   // nobody leaves while its shared memory is read
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
  if ((long long)f.strips * f.blocks > 0x7fffffffLL)
    return set_error(MK_ERR_INVALID, "%s: %d x %d is too large", what, w->N, w->K);
  if (need_data && (!w->data || (reinterpret_cast<uintptr_t>(w->data) & 15) != 0))
    return set_error(MK_ERR_INVALID, "%s: packed weights must be a 16-byte aligned device buffer", what);
  return MK_OK;
}

template <typename K>
static int w4_launch(K kern, dim3 grid, int threads, int smem, int cluster, cudaStream_t stream,
                     const W4Params& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (option_pdl()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  MKB_CUDA(cudaLaunchKernelEx(&cfg, kern, p));
  return MK_OK;
}

template <typename T, int NT, int GROUP>
static int w4_stream_launch(const W4Params& p, dim3 grid, cudaStream_t stream) {
  return p.form.zeros
             ? w4_launch(w4_stream_kernel<T, NT, GROUP, true>, grid, kW4Warps * 32, 0, p.split, stream, p)
             : w4_launch(w4_stream_kernel<T, NT, GROUP, false>, grid, kW4Warps * 32, 0, p.split, stream, p);
}
template <typename T, int NT>
static int w4_stream_group(const W4Params& p, dim3 grid, cudaStream_t stream) {
  if (p.form.group == 32) return w4_stream_launch<T, NT, 32>(p, grid, stream);
  if (p.form.group == 64) return w4_stream_launch<T, NT, 64>(p, grid, stream);
  return w4_stream_launch<T, NT, 128>(p, grid, stream);
}

static int w4_product(const char* what, const void* A, long long lda, const mk_w4* w, void* C, long long ldc,
                      int M, int form, int epilogue, const RotaryArgs& rotary, void* stream) {
  int rc = w4_check(w, what, true);
  if (rc != MK_OK) return rc;
  if (w->form != form)
    return set_error(MK_ERR_INVALID, "%s: the weights were laid out in form %d, this product takes form %d", what,
                     w->form, form);
  const int n_out = epilogue == W4_EPI_SWIGLU ? w->N / 2 : w->N;
  if (M < 0) return set_error(MK_ERR_INVALID, "%s: M=%d is negative", what, M);
  if (M == 0) return MK_OK;
  if (!A || !C) return set_error(MK_ERR_INVALID, "%s: null operand", what);
  if (lda < w->K || ldc < n_out)
    return set_error(MK_ERR_INVALID, "%s: row strides %lld and %lld must be at least K=%d and %d", what, lda, ldc,
                     w->K, n_out);
  if (((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(C)) & 1) != 0)
    return set_error(MK_ERR_INVALID, "%s: operands must be 2-byte aligned", what);
  int sms = 0;
  rc = device_sm_count(&sms);
  if (rc != MK_OK) return rc;
  W4Params p;
  memset(&p, 0, sizeof(p));
  p.form = w4_form(*w);
  p.data = static_cast<const uint8_t*>(w->data);
  p.A = A; p.lda = lda; p.C = C; p.ldc = ldc; p.M = M;
  p.vec = (reinterpret_cast<uintptr_t>(A) & 15) == 0 && lda % 8 == 0 && w->K % 8 == 0;
  p.epilogue = epilogue;
  p.rotary = rotary;
  const int nt = M <= 8 ? 1 : 2;
  const long long tiles = ((long long)M + 8 * nt - 1) / (8 * nt);
  if (tiles > 65535) return set_error(MK_ERR_INVALID, "%s: M=%d is too large", what, M);
  p.split = 1;
  while (p.split < 8 && p.form.strips * tiles * p.split < 4LL * sms && p.split * kW4Warps < p.form.blocks)
    p.split *= 2;
  const dim3 grid((unsigned)(p.form.strips * p.split), (unsigned)tiles, 1);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (w->dtype == MK_BF16)
    return nt == 1 ? w4_stream_group<__nv_bfloat16, 1>(p, grid, s) : w4_stream_group<__nv_bfloat16, 2>(p, grid, s);
  return nt == 1 ? w4_stream_group<__half, 1>(p, grid, s) : w4_stream_group<__half, 2>(p, grid, s);
}

template <typename T>
static int w4_quantize_launch(const W4PackParams& p, int src_dtype, unsigned grid, cudaStream_t s) {
  if (src_dtype == MK_BF16) w4_quantize_kernel<T, __nv_bfloat16><<<grid, kW4PackThreads, 0, s>>>(p);
  else if (src_dtype == MK_FP16) w4_quantize_kernel<T, __half><<<grid, kW4PackThreads, 0, s>>>(p);
  else w4_quantize_kernel<T, float><<<grid, kW4PackThreads, 0, s>>>(p);
  MKB_CUDA(cudaGetLastError());
  return MK_OK;
}

template <typename T>
static int w4_dequantize_launch(const W4Form& f, const uint8_t* data, void* out, long long ld, int dtype, int vec,
                                unsigned grid, cudaStream_t s) {
  if (dtype == MK_BF16)
    w4_dequantize_kernel<T><<<grid, 256, 0, s>>>(f, data, static_cast<__nv_bfloat16*>(out), ld, vec);
  else if (dtype == MK_FP16)
    w4_dequantize_kernel<T><<<grid, 256, 0, s>>>(f, data, static_cast<__half*>(out), ld, vec);
  else
    w4_dequantize_kernel<T><<<grid, 256, 0, s>>>(f, data, static_cast<float*>(out), ld, vec);
  MKB_CUDA(cudaGetLastError());
  return MK_OK;
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
  const unsigned grid = (unsigned)(p.form.strips * p.form.blocks);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (w->dtype == MK_BF16) w4_pack_kernel<__nv_bfloat16><<<grid, kW4PackThreads, 0, s>>>(p);
  else w4_pack_kernel<__half><<<grid, kW4PackThreads, 0, s>>>(p);
  MKB_CUDA(cudaGetLastError());
  return MK_OK;
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
  const unsigned grid = (unsigned)(p.form.strips * p.form.blocks);
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
  const unsigned grid = (unsigned)(f.strips * f.blocks);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uint8_t* data = static_cast<const uint8_t*>(w->data);
  return w->dtype == MK_BF16 ? w4_dequantize_launch<__nv_bfloat16>(f, data, out, ld, out_dtype, vec, grid, s)
                             : w4_dequantize_launch<__half>(f, data, out, ld, out_dtype, vec, grid, s);
}

int mk_w4_gemm(const void* A, long long lda, const mk_w4* w, void* C, long long ldc, int M, void* stream) {
  return w4_product("mk_w4_gemm", A, lda, w, C, ldc, M, MK_W4_PLAIN, W4_EPI_NONE, RotaryArgs{}, stream);
}

int mk_w4_gemm_swiglu(const void* A, long long lda, const mk_w4* w, void* H, long long ldh, int M, void* stream) {
  return w4_product("mk_w4_gemm_swiglu", A, lda, w, H, ldh, M, MK_W4_GATE_UP, W4_EPI_SWIGLU, RotaryArgs{}, stream);
}

int mk_w4_gemm_rotary(const void* A, long long lda, const mk_w4* w, void* C, long long ldc, int M,
                      const void* positions, int pos64, const float* inv_freq, float scale, void* stream) {
  if (M > 0 && (!positions || !inv_freq)) return set_error(MK_ERR_INVALID, "mk_w4_gemm_rotary: null positions or frequencies");
  if (reinterpret_cast<uintptr_t>(positions) % (pos64 ? 8 : 4) != 0 || reinterpret_cast<uintptr_t>(inv_freq) % 4 != 0)
    return set_error(MK_ERR_INVALID, "mk_w4_gemm_rotary: misaligned positions or frequencies");
  RotaryArgs r;
  r.positions = positions; r.pos64 = pos64 != 0; r.inv_freq = inv_freq; r.scale = scale;
  return w4_product("mk_w4_gemm_rotary", A, lda, w, C, ldc, M, MK_W4_ROTARY, W4_EPI_ROTARY, r, stream);
}

}  // extern "C"
