// qk_norm_rope.cu - RMS norm of every query and key head and the rotary embedding in one
// pass (the reference runs rms_norm_heads and rope as separate passes over q and over k,
// zimage.cpp:117-120, qwen3.cpp): per head x[d],
//   u = x / sqrt(mean(x^2) + eps) * gamma
//   (u_i, u_j) -> (u_i cos_i - u_j sin_i, u_j cos_j + u_i sin_j)   for the pairs of the
//   first `rot` channels (i, j) = (2m, 2m + 1) or (m, m + rot / 2); the rest stays u.
#include <algorithm>

#include "elem.cuh"
#include "internal.h"
#include "ptx.cuh"
#include "serving.h"

namespace sdb {
namespace {

constexpr int kWarps = 8;

// One warp per (token, head); the head is staged in shared memory in fp32, so it may be
// written in place.
template <class TI, class TO>
__global__ void __launch_bounds__(kWarps * 32) k_qk_norm_rope_any(const QkNormRope p) {
  extern __shared__ float sh[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* u = sh + (size_t)warp * p.d;
  const int nh = p.heads + p.kv_heads;
  const int64_t units = p.T * nh;
  for (int64_t w = (int64_t)blockIdx.x * kWarps + warp; w < units; w += (int64_t)gridDim.x * kWarps) {
    const int64_t t = w / nh;
    const int h = (int)(w - t * nh);
    const int64_t row = p.pos ? p.pos[t] : t % p.n_pos;
    if (row < 0 || row >= p.n_pos) {
      if (lane == 0) atomicOr(p.err, kErrBadIndex);
      continue;
    }
    const bool is_k = h >= p.heads;
    const TI* x = is_k ? (const TI*)p.k + t * p.ldk + (int64_t)(h - p.heads) * p.d : (const TI*)p.q + t * p.ldq + (int64_t)h * p.d;
    TO* y = is_k ? (TO*)p.k_out + t * p.ldko + (int64_t)(h - p.heads) * p.d : (TO*)p.q_out + t * p.ldqo + (int64_t)h * p.d;
    const float* g = is_k ? p.gk : p.gq;
    float s = 0.0f;
    for (int c = lane; c < p.d; c += 32) {
      const float v = to_f32(x[c]);
      u[c] = v;
      s = fmaf(v, v, s);
    }
    const float rstd = rsqrtf(warp_add(s) / (float)p.d + p.eps);
    __syncwarp();
    const float* cs = p.cos + row * p.rot;
    const float* sn = p.sin + row * p.rot;
    for (int c = lane; c < p.d; c += 32) {
      float v = u[c] * rstd * (g ? g[c] : 1.0f);
      if (c < p.rot) {
        const bool second = p.interleaved ? (c & 1) : c >= p.rot / 2;
        const int o = p.interleaved ? (c ^ 1) : second ? c - p.rot / 2 : c + p.rot / 2;
        const float w2 = u[o] * rstd * (g ? g[o] : 1.0f);
        v = second ? v * cs[c] + w2 * sn[c] : v * cs[c] - w2 * sn[c];
      }
      y[c] = from_f32<TO>(v);
    }
    __syncwarp();
  }
}

template <class TI, class TO>
void launch(const QkNormRope& p) {
  const int64_t units = p.T * (p.heads + p.kv_heads);
  const unsigned grid = (unsigned)std::min<int64_t>((units + kWarps - 1) / kWarps, (int64_t)ctx().num_sms * 8);
  k_qk_norm_rope_any<TI, TO><<<grid, kWarps * 32, (size_t)kWarps * p.d * 4, ctx().stream>>>(p);
  check_launch("qk_norm_rope");
}

template <class TI>
void launch_in(const QkNormRope& p, int out_type) {
  if (out_type == kF32) return launch<TI, float>(p);
  if (out_type == kBF16) return launch<TI, __nv_bfloat16>(p);
  launch<TI, __half>(p);
}

}  // namespace

void launch_qk_norm_rope(QkNormRope p, int in_type, int out_type) {
  p.err = ctx().err_word;
  if (in_type == kF32) return launch_in<float>(p, out_type);
  if (in_type == kBF16) return launch_in<__nv_bfloat16>(p, out_type);
  launch_in<__half>(p, out_type);
}

}  // namespace sdb
