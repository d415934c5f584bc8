// attention_ragged.cu - attention of sequences with their own lengths. Sequence s owns the
// query rows [q_begin, q_begin + q_len) and the key rows [kv_begin, kv_begin + kv_len);
// its query i stands at position p = i + kv_len - q_len among its keys, and per head
//   z_j = scale q.k_j,  z_j = cap tanh(z_j / cap) if cap > 0,  z_j -= slope |p - j|,
// over all keys, the keys j <= p (causal), or those and j < prefix; out = softmax(z) v, and
// 0 where no key is left. Masked keys and values are not used, whatever they hold.
#include <algorithm>
#include <cmath>

#include "elem.cuh"
#include "internal.h"
#include "ptx.cuh"
#include "serving.h"

namespace sdb {
namespace {

constexpr int kWarps = 8;
constexpr int kMaxPer = 8;  // channels a lane holds: d <= 256

// Bounds of sequence s; false (and the error bit) when they leave the tensors or exceed
// the maxima that the launch was sized for.
__device__ __forceinline__ bool sequence(const RaggedAttention& p, int s, int64_t& q0, int64_t& ql, int64_t& k0,
                                         int64_t& kl) {
  q0 = p.q_begin[s];
  ql = p.q_len[s];
  k0 = p.kv_begin[s];
  kl = p.kv_len[s];
  const bool ok = q0 >= 0 && ql >= 0 && k0 >= 0 && kl >= 0 && q0 + ql <= p.Tq && k0 + kl <= p.Tkv && ql <= p.max_q &&
                  kl <= p.max_kv;
  if (!ok && threadIdx.x == 0) atomicOr(p.err, kErrBadIndex);
  return ok;
}

// One warp per (query row, head), lanes over channels, keys one after another.
template <class TI, class TO>
__global__ void __launch_bounds__(kWarps * 32) k_attention_ragged_any(const RaggedAttention p) {
  const int lane = threadIdx.x & 31;
  int64_t q0, ql, k0, kl;
  if (!sequence(p, blockIdx.z, q0, ql, k0, kl)) return;
  const int64_t i = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (i >= ql) return;
  const int h = blockIdx.y, kh = h / (p.heads / p.kv_heads);
  const int64_t pos = i + kl - ql;
  const int64_t pre = p.causal && p.prefix ? p.prefix[blockIdx.z] : 0;
  const float slope = p.slopes ? p.slopes[h] : 0.0f;
  const TI* qr = (const TI*)p.q + (q0 + i) * p.ldq + (int64_t)h * p.d;
  float q[kMaxPer], o[kMaxPer];
#pragma unroll
  for (int c = 0; c < kMaxPer; ++c) {
    q[c] = lane + 32 * c < p.d ? to_f32(qr[lane + 32 * c]) : 0.0f;
    o[c] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  const int64_t end = p.causal ? min(kl, max(pos + 1, pre)) : kl;
  for (int64_t j = 0; j < end; ++j) {
    const TI* kr = (const TI*)p.k + (k0 + j) * p.ldk + (int64_t)kh * p.d;
    float z = 0.0f;
#pragma unroll
    for (int c = 0; c < kMaxPer; ++c)
      if (lane + 32 * c < p.d) z = fmaf(q[c], to_f32(kr[lane + 32 * c]), z);
    z = warp_add(z) * p.scale;
    if (p.cap > 0.0f) z = p.cap * tanhf(z / p.cap);
    if (p.slopes) z -= slope * (float)(pos > j ? pos - j : j - pos);
    if (z == -INFINITY) continue;
    const float mn = fmaxf(m, z), f = expf(m - mn), w = expf(z - mn);
    m = mn;
    l = l * f + w;
    const TI* vr = (const TI*)p.v + (k0 + j) * p.ldv + (int64_t)kh * p.d;
#pragma unroll
    for (int c = 0; c < kMaxPer; ++c)
      if (lane + 32 * c < p.d) o[c] = fmaf(w, to_f32(vr[lane + 32 * c]), o[c] * f);
  }
  TO* y = (TO*)p.out + (q0 + i) * p.ldo + (int64_t)h * p.d;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // a NaN score leaves l NaN
#pragma unroll
  for (int c = 0; c < kMaxPer; ++c)
    if (lane + 32 * c < p.d) y[lane + 32 * c] = from_f32<TO>(o[c] * inv);
}

template <class TI, class TO>
void launch_any(const RaggedAttention& p) {
  const dim3 grid((unsigned)((p.max_q + kWarps - 1) / kWarps), (unsigned)p.heads, (unsigned)p.n_seq);
  k_attention_ragged_any<TI, TO><<<grid, kWarps * 32, 0, ctx().stream>>>(p);
  check_launch("attention_ragged");
}

}  // namespace

size_t ragged_attention_workspace(const RaggedAttention&) { return 0; }

void launch_ragged_attention(RaggedAttention p, void*) {
  p.err = ctx().err_word;
  if (p.in_type == kBF16) return p.out_type == kBF16 ? launch_any<__nv_bfloat16, __nv_bfloat16>(p) : launch_any<__nv_bfloat16, __half>(p);
  p.out_type == kBF16 ? launch_any<__half, __nv_bfloat16>(p) : launch_any<__half, __half>(p);
}

}  // namespace sdb
