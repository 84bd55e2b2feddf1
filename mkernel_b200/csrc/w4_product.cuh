// What the two kernels of the 4-bit products share: their parameters, what is done with a finished
// pair of sums, and the launch.
#pragma once
#include <cuda_runtime.h>

#include "host_util.h"
#include "ptx.cuh"
#include "rotary.cuh"
#include "w4_layout.cuh"

namespace mkb {

enum W4Epilogue : int { W4_EPI_NONE = 0, W4_EPI_SWIGLU = 1, W4_EPI_ROTARY = 2 };

struct W4Params {
  W4Form form;
  const uint8_t* data;
  const void* A;
  long long lda;
  void* C;
  long long ldc;
  int M;
  int vec;             // rows of A start on 16 bytes
  int stage_bytes;     // of a shared-memory ring
  int split;           // CTAs of a cluster, which share a strip along K
  int token_tiles;     // tile kernel
  int wide;            // C takes 8-byte stores at every fourth column
  uint64_t wait_limit_ns;
  int debug_flags;     // diagnostics build only
  int epilogue;
  RotaryArgs rotary;
};
// A launch with 8 bytes more costs the host 0.4 us more (3.2 for a token of 1024 x 1024, 3.6 with 168 bytes).
static_assert(sizeof(W4Params) <= 160, "parameters of the products");

// silu(gate) up in fp32; for a gate below -88 the exponential is inf and the quotient -0, as it should be.
__device__ __forceinline__ float w4_silu_mul(float gate, float up) { return gate / (1.0f + __expf(-gate)) * up; }

__device__ __forceinline__ uint32_t w4_round2(float a, float b, __nv_bfloat16) { return ptx::pack_bf16x2(a, b); }
__device__ __forceinline__ uint32_t w4_round2(float a, float b, __half) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Whether a pair of rows is turned for a token, and by which cosine and sine.
struct W4Turn { bool on; float2 angle; };
__device__ __forceinline__ W4Turn w4_turn(const W4Params& p, int strip, int pair, int token) {
  const W4Form& f = p.form;
  const int half = f.head_dim / 2, index = strip * (kW4Strip / 2) + pair, head = index / half, i = index - head * half;
  if (head >= f.rotated_heads || i >= f.rotary_dim / 2) return {false, make_float2(1.0f, 0.0f)};
  return {true, rotary_cos_sin(rotary_position(p.rotary, token), p.rotary.inv_freq[i], p.rotary.scale)};
}

// C's entries of one pair of rows and one token.  turn: w4_turn, in the rotary form.
template <typename T>
__device__ __forceinline__ void w4_epilogue(const W4Params& p, int strip, int pair, int token, float2 v, const W4Turn& turn) {
  const W4Form& f = p.form;
  const int n0 = w4_row(f, strip, pair, 0);
  if (n0 < 0) return;
  T* row = static_cast<T*>(p.C) + (long long)token * p.ldc;
  if (p.epilogue == W4_EPI_SWIGLU) {
    row[n0] = W4Traits<T>::from_float(w4_silu_mul(v.x, v.y));
    return;
  }
  const int n1 = w4_row(f, strip, pair, 1);
  if (turn.on) v = rotary_turn(v.x, v.y, turn.angle);
  row[n0] = W4Traits<T>::from_float(v.x);
  if (n1 >= 0) row[n1] = W4Traits<T>::from_float(v.y);
}

// The same of four consecutive pairs (pair a multiple of 4).  first[i], second[i]: their two sums.
template <typename T>
__device__ __forceinline__ void w4_epilogue4(const W4Params& p, int strip, int pair, int token, float4 first, float4 second) {
  const W4Form& f = p.form;
  const float a[4] = {first.x, first.y, first.z, first.w}, b[4] = {second.x, second.y, second.z, second.w};
  // the two forms whose outputs of four pairs are neighbours
  if (p.wide && p.epilogue != W4_EPI_ROTARY) {
    T* row = static_cast<T*>(p.C) + (long long)token * p.ldc;
    float v[4];
    const bool glu = p.epilogue == W4_EPI_SWIGLU;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = glu ? w4_silu_mul(a[i], b[i]) : a[i];
    const int n0 = w4_row(f, strip, pair, 0), n1 = glu ? -1 : w4_row(f, strip, pair, 1);
    const int n_out = glu ? f.N / 2 : f.N;
    if (n0 >= 0 && n0 + 4 <= n_out && (n1 >= 0 || glu) && n1 + 4 <= n_out) {
      *reinterpret_cast<uint2*>(row + n0) = make_uint2(w4_round2(v[0], v[1], T()), w4_round2(v[2], v[3], T()));
      if (!glu) *reinterpret_cast<uint2*>(row + n1) = make_uint2(w4_round2(b[0], b[1], T()), w4_round2(b[2], b[3], T()));
      return;
    }
  }
  if (p.epilogue == W4_EPI_ROTARY) {
    T* row = static_cast<T*>(p.C) + (long long)token * p.ldc;
    const int half = f.head_dim / 2, n_pairs = f.N / 2;
    int index = strip * (kW4Strip / 2) + pair, head = index / half, at = index - head * half;
    const long long position = rotary_position(p.rotary, token);
    float2 v[4];
    // Heads of whole fours of pairs, the usual ones: the four turn or do not turn together, and their outputs are
    // neighbours, in two rows of four or one of eight.
    if (p.wide && half % 4 == 0 && f.rotary_dim / 2 % 4 == 0) {
      if (index >= n_pairs) return;
      const bool rotated = head < f.rotated_heads && at < f.rotary_dim / 2;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = make_float2(a[i], b[i]);
        if (rotated)
          v[i] = rotary_turn(a[i], b[i], rotary_cos_sin(position, p.rotary.inv_freq[at + i], p.rotary.scale));
      }
      const bool apart = rotated && !f.interleaved;
      T* to = row + head * f.head_dim + (apart ? at : 2 * at);
      const float2 e[4] = {{v[0].x, apart ? v[1].x : v[0].y}, {apart ? v[2].x : v[1].x, apart ? v[3].x : v[1].y},
                           {apart ? v[0].y : v[2].x, apart ? v[1].y : v[2].y}, {apart ? v[2].y : v[3].x, v[3].y}};
      *reinterpret_cast<uint2*>(to) = make_uint2(w4_round2(e[0].x, e[0].y, T()), w4_round2(e[1].x, e[1].y, T()));
      to += apart ? f.rotary_dim / 2 : 4;
      *reinterpret_cast<uint2*>(to) = make_uint2(w4_round2(e[2].x, e[2].y, T()), w4_round2(e[3].x, e[3].y, T()));
      return;
    }
    int n[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool rotated = head < f.rotated_heads && at < f.rotary_dim / 2;
      const bool apart = rotated && !f.interleaved;
      n[i][0] = index + i < n_pairs ? head * f.head_dim + (apart ? at : 2 * at) : -1;
      n[i][1] = n[i][0] + (apart ? f.rotary_dim / 2 : 1);
      v[i] = make_float2(a[i], b[i]);
      if (rotated && n[i][0] >= 0)
        v[i] = rotary_turn(a[i], b[i], rotary_cos_sin(position, p.rotary.inv_freq[at], p.rotary.scale));
      if (++at == half) { at = 0; ++head; }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n[i][0] >= 0) {
        row[n[i][0]] = W4Traits<T>::from_float(v[i].x);
        row[n[i][1]] = W4Traits<T>::from_float(v[i].y);
      }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) w4_epilogue<T>(p, strip, pair + i, token, make_float2(a[i], b[i]), {});
}

template <typename K, typename... Args>
inline int w4_launch(K kern, dim3 grid, int threads, int smem, int cluster, cudaStream_t stream, const Args&... args) {
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
  MKB_CUDA(cudaLaunchKernelEx(&cfg, kern, args...));
  return MK_OK;
}

// The product for more tokens than the stream kernel takes (w4_tile.cu), and how it is cut: tokens to a CTA, CTAs to a
// cluster along K.  rest: what rounding the weights leaves is multiplied as well.
constexpr int kW4StreamTokens = 16;
struct W4TilePlan { int tokens, split, token_tiles; long long ctas; };
int w4_tile_plan(const W4Form& f, int M, bool rest, int sms, W4TilePlan* out);
int w4_tile_launch(W4Params& p, int dtype, bool rest, int sms, cudaStream_t stream);

}  // namespace mkb
