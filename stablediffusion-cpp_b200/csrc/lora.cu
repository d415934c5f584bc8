// lora.cu - a projection shared by every row plus each row's own low-rank adapter:
//   y[t, n] = sum_k x[t, k] W[n, k] + bias[n] + s_a sum_j h[t, j] B_a[n, j],
//   h[t, j] = sum_k x[t, k] A_a[j, k],   a = row_adapter[t] (no second term for a < 0).
#include <algorithm>

#include "elem.cuh"
#include "internal.h"
#include "ptx.cuh"
#include "serving.h"

namespace sdb {
namespace {

__device__ __forceinline__ float load_x(const LoraLinear& p, int64_t t, int64_t k) {
  return p.x_bf16 ? bf16_to_f32(((const uint16_t*)p.X)[t * p.ldx + k])
                  : bf16_to_f32(f32_to_bf16_rne(((const float*)p.X)[t * p.ldx + k]));
}

// h[t, j], one warp per value.
__global__ void __launch_bounds__(256) k_lora_down(const LoraLinear p, float* __restrict__ h) {
  const int lane = threadIdx.x & 31;
  for (int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); w < p.T * p.r; w += (int64_t)gridDim.x * 8) {
    const int64_t t = w / p.r, j = w - t * p.r;
    const int a = p.row_adapter[t];
    float s = 0.0f;
    if (a >= p.n_adapters) {
      if (lane == 0) atomicOr(p.err, kErrBadIndex);
    } else if (a >= 0) {
      const uint16_t* A = p.A + (a * p.r + j) * p.lda;
      for (int64_t k = lane; k < p.K; k += 32) s = fmaf(load_x(p, t, k), bf16_to_f32(A[k]), s);
      s = warp_add(s) * (p.scale ? p.scale[a] : 1.0f);
    }
    if (lane == 0) h[w] = s;
  }
}

constexpr int kTM = 64, kTN = 64, kTK = 16;

// 64 x 64 outputs a block, 4 x 4 a thread.
__global__ void __launch_bounds__(256) k_lora_gemm(const LoraLinear p, const float* __restrict__ h) {
  __shared__ float xs[kTK][kTM + 1], wsh[kTK][kTN + 1];
  const int64_t t0 = (int64_t)blockIdx.x * kTM, n0 = (int64_t)blockIdx.y * kTN;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < p.K; k0 += kTK) {
    for (int i = threadIdx.x; i < kTM * kTK; i += 256) {
      const int r = i / kTK, c = i % kTK;
      xs[c][r] = (t0 + r < p.T && k0 + c < p.K) ? load_x(p, t0 + r, k0 + c) : 0.0f;
      wsh[c][r] = (n0 + r < p.N && k0 + c < p.K) ? bf16_to_f32(p.W[(n0 + r) * p.ldw + k0 + c]) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < kTK; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xs[c][ty * 4 + i], wsh[c][tx * 4 + j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i) {
    const int64_t t = t0 + ty * 4 + i;
    if (t >= p.T) break;
    const int a = p.row_adapter[t];
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + tx * 4 + j;
      if (n >= p.N) break;
      float y = acc[i][j] + (p.bias ? p.bias[n] : 0.0f);
      if (a >= 0 && a < p.n_adapters) {
        const uint16_t* B = p.B + (a * p.N + n) * p.ldb;
        for (int64_t c = 0; c < p.r; ++c) y = fmaf(h[t * p.r + c], bf16_to_f32(B[c]), y);
      }
      if (p.y_bf16)
        ((uint16_t*)p.Y)[t * p.ldy + n] = f32_to_bf16_rne(y);
      else
        ((float*)p.Y)[t * p.ldy + n] = y;
    }
  }
}

}  // namespace

size_t lora_linear_workspace(const LoraLinear& p) { return (size_t)(p.T * p.r) * 4; }

void launch_lora_linear(LoraLinear p, void* ws) {
  DeviceContext& c = ctx();
  p.err = c.err_word;
  float* h = static_cast<float*>(ws);
  const int64_t w = p.T * p.r;
  k_lora_down<<<(unsigned)std::min<int64_t>((w + 7) / 8, (int64_t)c.num_sms * 16), 256, 0, c.stream>>>(p, h);
  check_launch("lora_down");
  k_lora_gemm<<<dim3((unsigned)((p.T + kTM - 1) / kTM), (unsigned)((p.N + kTN - 1) / kTN)), 256, 0, c.stream>>>(p, h);
  check_launch("lora_gemm");
}

}  // namespace sdb
