// attention_ragged.cu - attention of sequences with their own lengths. Sequence s owns the
// query rows [q_begin, q_begin + q_len) and the key rows [kv_begin, kv_begin + kv_len);
// its query i stands at position p = i + kv_len - q_len among its keys, and per head
//   z_j = scale q.k_j,  z_j = cap tanh(z_j / cap) if cap > 0,  z_j -= slope |p - j|,
// over all keys, the keys j <= p (causal), or those and j < prefix; out = softmax(z) v, and
// 0 where no key is left. Masked keys and values are not used, whatever they hold.
#include <algorithm>
#include <cmath>

#include "attention_ragged_tc.cuh"

namespace sdb {
namespace ragged {
#define SDB_RAGGED_TC(DP, T) \
  extern template void launch_tc<DP, T>(TcParams, const CUtensorMap&, const CUtensorMap&, const CUtensorMap&, bool);
SDB_RAGGED_TC(64, __half)
SDB_RAGGED_TC(128, __half)
SDB_RAGGED_TC(64, __nv_bfloat16)
SDB_RAGGED_TC(128, __nv_bfloat16)
#undef SDB_RAGGED_TC
}  // namespace ragged
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
  const dim3 grid((unsigned)((std::min(p.max_q, p.Tq) + kWarps - 1) / kWarps), (unsigned)p.heads, (unsigned)p.n_seq);
  k_attention_ragged_any<TI, TO><<<grid, kWarps * 32, 0, ctx().stream>>>(p);
  check_launch("attention_ragged");
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// TMA reads rows and heads that start on 16-byte boundaries; wider heads than two swizzle
// atoms do not fit the tensor-core kernels' shared memory.
bool tensor_core_shape(const RaggedAttention& p) {
  return p.d <= 128 && p.d % 8 == 0 && p.ldq % 8 == 0 && p.ldk % 8 == 0 && p.ldv % 8 == 0 && p.max_kv > 0 && p.Tkv > 0 &&
         aligned16(p.q) && aligned16(p.k) && aligned16(p.v);
}

// Whether every sequence's queries fit one tile of 128 rows.
bool one_tile(const RaggedAttention& p) { return p.max_q <= ragged::kBQ / (p.heads / p.kv_heads); }

void launch_tensor_core(const RaggedAttention& a, void* ws) {
  using namespace ragged;
  TcParams p{};
  p.a = a;
  p.G = a.heads / a.kv_heads;
  p.scale_log2 = a.scale * kLog2e;
  if (a.cap > 0.0f) {
    p.cap_in = 2.0f * kLog2e * a.scale / a.cap;
    p.cap_log2 = a.cap * kLog2e;
    p.cap_x = a.scale / a.cap;
    p.cap_small = a.cap / a.scale;
    const float c[6] = {0.9999968409538269f, -0.3332400321960449f, 0.13253524899482727f, -0.05097286403179169f, 0.016114182770252228f, -0.002839465858414769f};
    for (int i = 0; i < 6; ++i) p.tanh_c[i] = c[i] * p.cap_log2;
  }
  p.out_vec = aligned16(a.out) && a.ldo % 8 == 0;
  const bool streams = one_tile(a);
  // One tile holds all tokens, however few: the Q box and its shared memory shrink with them.
  p.tpt = streams ? (int)a.max_q : kBQ / p.G;
  p.part = static_cast<float*>(ws);
  p.part_rows = p.G * (int)std::min<int64_t>(a.max_q, kBQ);
  p.q_atom = (p.G * p.tpt + 7) / 8 * 8 * 128;
  const CUtensorMapDataType dt = a.in_type == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUtensorMap tq, tk, tv;
  auto map = [&](CUtensorMap* m, const void* x, int heads, int64_t rows, int64_t ld, int box_heads, int box_rows) {
    const uint64_t dims[3] = {(uint64_t)a.d, (uint64_t)heads, (uint64_t)rows};
    const uint64_t str[2] = {(uint64_t)a.d * 2, (uint64_t)ld * 2};
    const uint32_t box[3] = {64, (uint32_t)box_heads, (uint32_t)box_rows};
    encode_tmap(m, dt, 3, x, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  map(&tq, a.q, a.heads, a.Tq, a.ldq, p.G, p.tpt);
  map(&tk, a.k, a.kv_heads, a.Tkv, a.ldk, 1, kBK);
  map(&tv, a.v, a.kv_heads, a.Tkv, a.ldv, 1, kBK);
  if (a.in_type == kBF16)
    a.d <= 64 ? launch_tc<64, __nv_bfloat16>(p, tq, tk, tv, streams) : launch_tc<128, __nv_bfloat16>(p, tq, tk, tv, streams);
  else
    a.d <= 64 ? launch_tc<64, __half>(p, tq, tk, tv, streams) : launch_tc<128, __half>(p, tq, tk, tv, streams);
}

}  // namespace

// The cut rows of k_ragged_streams: two pieces per worker.
size_t ragged_attention_workspace(const RaggedAttention& p) {
  if (!one_tile(p) || p.max_kv <= ragged::kBK || p.d > 128) return 0;
  return (size_t)(4 * ctx().num_sms) * (size_t)(p.heads / p.kv_heads * p.max_q) * (size_t)(p.d + 2) * 4;
}

void launch_ragged_attention(RaggedAttention p, void* ws) {
  p.err = ctx().err_word;
  if (tensor_core_shape(p)) return launch_tensor_core(p, ws);
  if (p.in_type == kBF16) return p.out_type == kBF16 ? launch_any<__nv_bfloat16, __nv_bfloat16>(p) : launch_any<__nv_bfloat16, __half>(p);
  p.out_type == kBF16 ? launch_any<__half, __nv_bfloat16>(p) : launch_any<__half, __half>(p);
}

}  // namespace sdb
