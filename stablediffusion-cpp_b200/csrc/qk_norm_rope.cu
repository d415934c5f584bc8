// qk_norm_rope.cu - RMS norm of every query and key head and the rotary embedding in one
// pass (the reference runs rms_norm_heads and rope as separate passes over q and over k,
// zimage.cpp:117-120, qwen3.cpp): per head x[d],
//   u = x / sqrt(mean(x^2) + eps) * gamma
//   (u_i, u_j) -> (u_i cos_i - u_j sin_i, u_j cos_j + u_i sin_j)   for the pairs of the
//   first `rot` channels (i, j) = (2m, 2m + 1) or (m, m + rot / 2); the rest stays u.
#include <algorithm>
#include <type_traits>

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

// VE consecutive channels as they lie in memory (4, 8, 16 or 32 aligned bytes).
template <class T, int VE>
struct Chunk {
  using Raw = typename std::conditional<sizeof(T) * VE >= 16, uint4,
                                        typename std::conditional<sizeof(T) * VE == 8, uint2, uint32_t>::type>::type;
  static constexpr int kRaw = sizeof(T) * VE / sizeof(Raw);
  Raw raw[kRaw];
  __device__ __forceinline__ void load(const T* x) {
#pragma unroll
    for (int i = 0; i < kRaw; ++i) raw[i] = reinterpret_cast<const Raw*>(x)[i];
  }
  __device__ __forceinline__ void store(T* y) const {
#pragma unroll
    for (int i = 0; i < kRaw; ++i) reinterpret_cast<Raw*>(y)[i] = raw[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kRaw; ++i) raw[i] = Raw{};
  }
  __device__ __forceinline__ void get(float (&v)[VE]) const {
#pragma unroll
    for (int i = 0; i < VE; ++i) v[i] = to_f32(reinterpret_cast<const T*>(raw)[i]);
  }
  __device__ __forceinline__ void set(const float (&v)[VE]) {
#pragma unroll
    for (int i = 0; i < VE; ++i) reinterpret_cast<T*>(raw)[i] = from_f32<T>(v[i]);
  }
};

constexpr int kThreads = 64;

// `n` heads of one token starting at x, a group of 2^lg lanes per head. A lane holds two
// chunks of VE channels, at c0 and c1, that form whole pairs: the two halves of a rotation
// halves apart, or neighbours. With gamma folded into the tables (A = gamma cos, B = -+ the
// partner's gamma sin) a channel is x A + (partner) B, times the head's rstd: no exchange
// between lanes but the sum of squares. With one chunk per lane and the partner's fetched by
// shuffles the arithmetic alone (200 instructions a chunk) kept bf16 rows at a third of the
// memory rate. Two heads are loaded ahead of the arithmetic.
template <class TI, class TO, int VE, bool INTER>
__device__ __forceinline__ void heads_of(const QkNormRope& p, const TI* x, TO* y, int n, const float* gamma, int lg, bool on,
                                         int c0, int c1, const float* cos, const float* sin) {
  if (n <= 0) return;  // uniform over the warp
  constexpr int U = 2;
  Chunk<TI, VE> raw[U][2];
  auto fetch = [&](int u, int h) {
    if (on && h < n) {
      raw[u][0].load(x + (int64_t)h * p.d + c0);
      raw[u][1].load(x + (int64_t)h * p.d + c1);
    }
  };
#pragma unroll
  for (int u = 0; u < U; ++u) {
    raw[u][0].zero();
    raw[u][1].zero();
    fetch(u, u);
  }
  float2 A[VE], B[VE];  // chunk 0: [0, VE / 2), chunk 1: the rest
  {
    float a[2 * VE], b[2 * VE], g[2 * VE];
    Chunk<float, VE> t;
    float c[2 * VE], w[2 * VE];
#pragma unroll
    for (int i = 0; i < 2 * VE; ++i) {
      g[i] = gamma && on ? __ldg(gamma + (i < VE ? c0 + i : c1 + i - VE)) : 1.0f;
      c[i] = 1.0f;
      w[i] = 0.0f;
    }
    if (cos) {
      float v[VE];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        t.load(cos + (k ? c1 : c0));
        t.get(v);
#pragma unroll
        for (int i = 0; i < VE; ++i) c[k * VE + i] = v[i];
        t.load(sin + (k ? c1 : c0));
        t.get(v);
#pragma unroll
        for (int i = 0; i < VE; ++i) w[k * VE + i] = v[i];
      }
    }
#pragma unroll
    for (int i = 0; i < 2 * VE; ++i) {
      const int o = INTER ? (i ^ 1) : (i + VE) % (2 * VE);
      const bool first = INTER ? (i & 1) == 0 : i < VE;
      a[i] = g[i] * c[i];
      b[i] = (first ? -g[o] : g[o]) * w[i];
    }
#pragma unroll
    for (int i = 0; i < VE; ++i) {
      A[i] = make_float2(a[2 * i], a[2 * i + 1]);
      B[i] = make_float2(b[2 * i], b[2 * i + 1]);
    }
  }
  const float inv_d = 1.0f / (float)p.d;
  for (int h0 = 0; h0 < n; h0 += U) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u;
      float2 v[VE];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float f[VE];
        raw[u][k].get(f);
#pragma unroll
        for (int i = 0; i < VE / 2; ++i) v[k * VE / 2 + i] = make_float2(f[2 * i], f[2 * i + 1]);
      }
      fetch(u, h + U);
      float2 s2 = fmul2(v[0], v[0]);
#pragma unroll
      for (int i = 1; i < VE; ++i) s2 = ffma2(v[i], v[i], s2);
      float s = s2.x + s2.y;
      for (int o = 1 << lg >> 1; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      const float rstd = rsqrtf(fmaf(s, inv_d, p.eps));
      const float2 r2 = make_float2(rstd, rstd);
      // A channel that is not rotated has B = 0, but 0 times an infinity in its partner is NaN: it leaves
      // the partner out, by a choice between values. (Branches took 12.75 instead of 12.4 us a call for
      // 2397 tokens of 40 heads, 6.1 instead of 5.2 us for 976 of 60 heads of 40.)
      float2 r[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float2 o = INTER ? make_float2(v[e].y, v[e].x) : v[(e + VE / 2) % VE];
        r[e] = fmul2(v[e], A[e]);
        if (cos) r[e] = ffma2(o, B[e], r[e]);
        r[e] = fmul2(r2, r[e]);
      }
      if (on && h < n) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float f[VE];
#pragma unroll
          for (int i = 0; i < VE / 2; ++i) {
            f[2 * i] = r[k * VE / 2 + i].x;
            f[2 * i + 1] = r[k * VE / 2 + i].y;
          }
          Chunk<TO, VE> out;
          out.set(f);
          out.store(y + (int64_t)h * p.d + (k ? c1 : c0));
        }
      }
    }
  }
}

// Bound by memory: 33792 tokens of 60 heads of 128, fp32 in, fp16 out, 242 us, 98% of the copy
// rate; 2397 tokens of 40 heads, bf16, 11.1 us, a single wave of blocks. The kernel for any shape
// takes 1038 and 51 us.
template <class TI, class TO, int VE, bool INTER>
__global__ void __launch_bounds__(kThreads, 10) k_qk_norm_rope(const QkNormRope p, int lg, int parts, int part_heads) {
  const int lane = threadIdx.x & 31, in = lane & ((1 << lg) - 1);
  // Groups of one warp take consecutive tokens of the same part of the heads.
  const int64_t warp = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  const int64_t t = warp / parts * (32 >> lg) + (lane >> lg);
  const int part = (int)(warp % parts);
  // Units of 2 VE channels: first the pairs of the rotated part, then the rest in order.
  int c0 = in * 2 * VE, c1 = c0 + VE;
  if (!INTER && c0 < p.rot) {
    c0 = in * VE;
    c1 = c0 + p.rot / 2;
  }
  bool on = t < p.T && in * 2 * VE < p.d;
  int64_t row = 0;
  if (t < p.T) {
    row = p.pos ? p.pos[t] : t % p.n_pos;
    if (row < 0 || row >= p.n_pos) {
      if (in == 0) atomicOr(p.err, kErrBadIndex);
      on = false;
      row = 0;
    }
  }
  const bool turned = on && in * 2 * VE < p.rot;
  const float* cos = turned ? p.cos + row * p.rot : nullptr;
  const float* sin = turned ? p.sin + row * p.rot : nullptr;
  const int h0 = part * part_heads, h1 = min(p.heads + p.kv_heads, h0 + part_heads);
  const int64_t tt = on ? t : 0;
  const int qn = min(h1, p.heads) - h0;
  heads_of<TI, TO, VE, INTER>(p, (const TI*)p.q + tt * p.ldq + (int64_t)h0 * p.d,
                              (TO*)p.q_out + tt * p.ldqo + (int64_t)h0 * p.d, qn, p.gq, lg, on, c0, c1, cos, sin);
  const int k0 = max(h0 - p.heads, 0);
  heads_of<TI, TO, VE, INTER>(p, (const TI*)p.k + tt * p.ldk + (int64_t)k0 * p.d,
                              (TO*)p.k_out + tt * p.ldko + (int64_t)k0 * p.d, h1 - p.heads - k0, p.gk, lg, on, c0, c1, cos,
                              sin);
}

// Channels of a chunk: base, pitch and head width, the pairs' distance and the tables must
// fall on whole chunks, and a head must fit a warp. 0: none. Chunks of two are slow in bytes
// (33000 tokens of 60 heads of 40 channels, bf16: 114 us, 43% of the copy rate), but the
// kernel for any shape takes 787 us.
template <class TI, class TO>
int chunk(const QkNormRope& p) {
  auto fits = [&](int ve) {
    auto ok = [&](const void* x, int64_t ld, int heads, int es) {
      const int bytes = std::min(16, ve * es);
      return !heads || (reinterpret_cast<uintptr_t>(x) % bytes == 0 && ld * es % bytes == 0);
    };
    return p.d % (2 * ve) == 0 && p.d / (2 * ve) <= 32 && p.rot % (2 * ve) == 0 &&
           reinterpret_cast<uintptr_t>(p.cos) % 16 == 0 && reinterpret_cast<uintptr_t>(p.sin) % 16 == 0 &&
           ok(p.q, p.ldq, p.heads, sizeof(TI)) && ok(p.q_out, p.ldqo, p.heads, sizeof(TO)) &&
           ok(p.k, p.ldk, p.kv_heads, sizeof(TI)) && ok(p.k_out, p.ldko, p.kv_heads, sizeof(TO));
  };
  if (sizeof(TI) == 2 && fits(8)) return 8;
  return fits(4) ? 4 : fits(2) ? 2 : 0;
}

template <class TI, class TO, int VE>
void launch_chunks(const QkNormRope& p) {
  const int nh = p.heads + p.kv_heads;
  int lg = 0;
  while ((2 << lg) * VE < p.d) ++lg;
  const int64_t warps = (p.T + (32 >> lg) - 1) / (32 >> lg);
  // A warp runs through all heads of its tokens with one set of table values; where that leaves
  // fewer than ten warps a processor, half of what fit, through fewer. 2397 tokens of 40 heads,
  // bf16: 11.1 us; 12.7 if filled up to twenty, which makes every set serve half as many heads,
  // 14.6 with seven.
  const int64_t want = (int64_t)ctx().num_sms * 10;
  int part_heads = nh;
  while (part_heads > 1 && warps * ((nh + part_heads - 1) / part_heads) < want) part_heads = (part_heads + 1) / 2;
  const int parts = (nh + part_heads - 1) / part_heads;
  const int64_t grid = (warps * parts + kThreads / 32 - 1) / (kThreads / 32);
  if (grid >= ((int64_t)1 << 31)) fail(kErrInvalidArg, "qk_norm_rope: too many rows");
  if (p.interleaved)
    k_qk_norm_rope<TI, TO, VE, true><<<(unsigned)grid, kThreads, 0, ctx().stream>>>(p, lg, parts, part_heads);
  else
    k_qk_norm_rope<TI, TO, VE, false><<<(unsigned)grid, kThreads, 0, ctx().stream>>>(p, lg, parts, part_heads);
  check_launch("qk_norm_rope");
}

template <class TI, class TO>
void launch(const QkNormRope& p) {
  const int ve = chunk<TI, TO>(p);
  if constexpr (sizeof(TI) == 2)
    if (ve == 8) return launch_chunks<TI, TO, 8>(p);
  if (ve == 4) return launch_chunks<TI, TO, 4>(p);
  if (ve == 2) return launch_chunks<TI, TO, 2>(p);
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
