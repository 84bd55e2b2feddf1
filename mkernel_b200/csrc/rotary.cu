// Rotary positions on rows of heads: y = x with the first rotary_dim features of every head turned by
// position * inv_freq.  Nothing but one read and one write of every element, so bound by memory.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/mkernel_b200.h"
#include "host_util.h"
#include "ptx.cuh"
#include "rotary.cuh"

namespace mkb {

struct RotaryParams {
  const void* x;
  void* y;
  long long x_row, x_head, y_row, y_head;   // strides in elements
  long long rows;
  int heads, head_dim, rotary_dim, interleaved;
  float sign;
  RotaryArgs rotary;
};

__device__ __forceinline__ float rotary_to_float(float v) { return v; }
__device__ __forceinline__ float rotary_to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float rotary_to_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T rotary_from_float(float v) { return (T)v; }

// One thread per pair of features of a row; it takes the angle once and walks the heads.
template <typename T>
__global__ void __launch_bounds__(128) rotary_kernel(const __grid_constant__ RotaryParams p) {
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int pairs = p.head_dim / 2 + (p.head_dim & 1);
  const long long total = p.rows * pairs;
  for (long long e = (long long)blockIdx.x * blockDim.x + threadIdx.x; e < total;
       e += (long long)gridDim.x * blockDim.x) {
    const long long row = e / pairs;
    const int i = (int)(e % pairs);
    const bool turned = i < p.rotary_dim / 2;
    const int a = turned && !p.interleaved ? i : 2 * i;
    const int b = turned && !p.interleaved ? i + p.rotary_dim / 2 : 2 * i + 1;
    float2 cs = make_float2(1.0f, 0.0f);
    if (turned) {
      cs = rotary_cos_sin(rotary_position(p.rotary, row), __ldg(p.rotary.inv_freq + i), p.rotary.scale);
      cs.y *= p.sign;
    } else if (p.x == p.y) {
      continue;
    }
    const T* x = static_cast<const T*>(p.x) + row * p.x_row;
    T* y = static_cast<T*>(p.y) + row * p.y_row;
    for (int h = 0; h < p.heads; ++h, x += p.x_head, y += p.y_head) {
      if (turned) {
        const float2 v = rotary_turn(rotary_to_float(x[a]), rotary_to_float(x[b]), cs);
        y[a] = rotary_from_float<T>(v.x);
        y[b] = rotary_from_float<T>(v.y);
      } else {
        y[a] = x[a];
        if (b < p.head_dim) y[b] = x[b];
      }
    }
  }
}

template <typename T>
static int rotary_launch(const RotaryParams& p, cudaStream_t stream, int sms) {
  const long long threads = p.rows * ((p.head_dim + 1) / 2);
  long long grid = (threads + 127) / 128;
  if (grid > 32LL * sms) grid = 32LL * sms;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid, 1, 1);
  cfg.blockDim = dim3(128, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = option_pdl() ? 1 : 0;
  MKB_CUDA(cudaLaunchKernelEx(&cfg, rotary_kernel<T>, p));
  return MK_OK;
}

}  // namespace mkb

using namespace mkb;

extern "C" int mk_rotary(const void* x, long long x_row, long long x_head, void* y, long long y_row,
                         long long y_head, long long rows, int heads, int head_dim, int rotary_dim, int dtype,
                         const void* positions, int pos64, const float* inv_freq, float scale, int interleaved,
                         int inverse, void* stream) {
  if (rows < 0 || heads < 0 || head_dim < 1)
    return set_error(MK_ERR_INVALID, "mk_rotary: bad shape [%lld, %d, %d]", rows, heads, head_dim);
  if (rotary_dim < 2 || rotary_dim % 2 != 0 || rotary_dim > head_dim)
    return set_error(MK_ERR_INVALID, "mk_rotary: rotary_dim=%d must be even and within head_dim=%d", rotary_dim,
                     head_dim);
  if (dtype < MK_BF16 || dtype > MK_FP32) return set_error(MK_ERR_INVALID, "mk_rotary: unknown dtype %d", dtype);
  if (rows == 0 || heads == 0) return MK_OK;
  if (!x || !y || !positions || !inv_freq) return set_error(MK_ERR_INVALID, "mk_rotary: null operand");
  const int size = dtype == MK_FP32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) % size != 0 ||
      reinterpret_cast<uintptr_t>(positions) % (pos64 ? 8 : 4) != 0 || reinterpret_cast<uintptr_t>(inv_freq) % 4 != 0)
    return set_error(MK_ERR_INVALID, "mk_rotary: misaligned operand");
  if (x == y && (x_row != y_row || x_head != y_head))
    return set_error(MK_ERR_INVALID, "mk_rotary: in place needs equal strides");
  int sms = 0;
  const int rc = device_sm_count(&sms);
  if (rc != MK_OK) return rc;
  RotaryParams p;
  p.x = x; p.y = y; p.x_row = x_row; p.x_head = x_head; p.y_row = y_row; p.y_head = y_head;
  p.rows = rows; p.heads = heads; p.head_dim = head_dim; p.rotary_dim = rotary_dim;
  p.interleaved = interleaved != 0;
  p.sign = inverse ? -1.0f : 1.0f;
  p.rotary.positions = positions; p.rotary.pos64 = pos64 != 0; p.rotary.inv_freq = inv_freq; p.rotary.scale = scale;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == MK_BF16) return rotary_launch<__nv_bfloat16>(p, s, sms);
  if (dtype == MK_FP16) return rotary_launch<__half>(p, s, sms);
  return rotary_launch<float>(p, s, sms);
}
