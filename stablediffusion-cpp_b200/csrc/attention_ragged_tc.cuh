// attention_ragged_tc.cuh - tensor-core kernels of attention_ragged (sm_100a), for head
// widths up to 128. Flash attention: the running maximum m and sum l of a softmax, so
// scores never leave the SM:
//   S = Q K^T (tcgen05, fp32 in TMEM);  P = 2^(S' - m) in the operand type, back in TMEM over
//   S;  O += P V (tcgen05);  O is rescaled when m grows by more than 2^8 (2^4 for fp16); out = O / l.
// P is rounded to the operand type because the tensor core multiplies it so: 2^-8 (bf16) or
// 2^-11 (fp16) of each probability, averaged over the keys; l, m, S and O stay fp32. fp16 ends
// at 2^-24, and a long cache has many keys of little weight each, so its P (and l and O with it)
// is 2^11 times as large: up to 2^15, and what rounds away is 2^-36 of the largest or less. With
// the largest at 1, 60000 keys of 2^-26 each left the sum without a trace.
//
// The G = heads / kv_heads query heads of a key head share its keys, so a 128-row tile
// holds floor(128 / G) tokens x G heads (row r is token r / G, head r % G): K and V are read
// once per key head, and one token of 4 heads fills 4 rows of a tile.
//
// Two kernels:
//   k_ragged_tiles    sequences of several tiles: a CTA owns two neighbouring tiles of one
//                     key head, which share one ring of K / V slots and take turns at the
//                     exp pass (as attention_tc.cu). Bound by the exponentials in the
//                     chain of a tile step: 4 x 4200 tokens, 30 heads of 128, 1040 to
//                     1160 us (0.92 to 1.02 PFLOP/s).
//   k_ragged_streams  sequences of one tile (single tokens, short prompts): the CTAs are
//                     persistent, each with two workers that own a tile and a ring of
//                     their own. The key tiles of all sequences and heads form one list,
//                     cut into equal parts, one per worker, whatever the lengths are;
//                     a worker's first and last piece may be part of a row, kept as
//                     (m, l, O) in fp32 and joined by k_ragged_join. Bound by memory
//                     with long caches (16 tokens over 152525 keys, 8 key heads of 128:
//                     110 us, 86% of the copy rate), by the latency of a tile with short
//                     prompts (64 of 5 to 77 tokens, 12 heads of 64: 17.7 us).
// A score's modifications (MOD bit 0: cap tanh(z / cap), bit 1: minus slope x distance) are
// applied between the TMEM load and the maximum. Masks are row limits: row r sees keys
// j < lim = min(kv_len, max(p + 1, prefix)).
#pragma once

#include <algorithm>
#include <string>

#include "elem.cuh"
#include "internal.h"
#include "ptx.cuh"
#include "serving.h"

namespace sdb {
namespace ragged {

constexpr int kBQ = 128;       // rows of a query tile (TMEM lanes)
constexpr int kBK = 128;       // keys of a K / V tile
constexpr int kThreads = 384;  // control warpgroup + two softmax warpgroups
// setmaxnreg split as in attention_tc.cu: 128 x 56 + 256 x 224 = 384 x 168.
constexpr int kRegsLaunch = 168, kRegsControl = 56, kRegsSoftmax = 224;
static_assert(128 * kRegsControl + 256 * kRegsSoftmax <= kThreads * kRegsLaunch, "register split");
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxSeqs = 512;  // sequences of one k_ragged_streams launch
constexpr int kMaxSmem = 232448;
constexpr int kFewRows = 16, kFewPad = 32 * 128;

struct TcParams {
  RaggedAttention a;
  int G, tpt;          // heads per key head, tokens per tile
  float scale_log2;    // scale log2(e)
  float cap_in;        // 2 log2(e) scale / cap
  float cap_log2;      // cap log2(e)
  float cap_x;         // scale / cap
  float cap_small;     // |q.k| up to which tanh is a polynomial: cap / scale
  float tanh_c[6];     // its coefficients, times cap log2(e)
  int out_vec;         // 16-byte stores allowed
  // k_ragged_streams
  int slots, q_atom;   // K / V slots per worker, bytes of one 64-channel Q atom
  float* part;         // [2 workers' pieces][rows][d + 2]: O, m, l
  int part_rows;       // rows of a piece: G * max_q
  int seq0, seqs;      // first sequence of this launch, most sequences of one
};

template <class T>
struct Op;
// kLift: log2 of what P is multiplied by; kSlack: how far m may stay behind, so P <= 2^(kLift + kSlack).
template <>
struct Op<__half> {
  static constexpr uint32_t kFmt = 0;
  static constexpr float kLift = 11.0f, kSlack = 4.0f;
  __device__ static uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Op<__nv_bfloat16> {
  static constexpr uint32_t kFmt = 1;
  static constexpr float kLift = 0.0f, kSlack = 8.0f;
  __device__ static uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// One sequence's rows, and whether its numbers fit the tensors and the launch.
struct Seq {
  int q0, ql, k0, kl;
};
__device__ __forceinline__ bool load_seq(const RaggedAttention& p, int s, Seq& q) {
  q.q0 = p.q_begin[s];
  q.ql = p.q_len[s];
  q.k0 = p.kv_begin[s];
  q.kl = p.kv_len[s];
  return q.q0 >= 0 && q.ql >= 0 && q.k0 >= 0 && q.kl >= 0 && (int64_t)q.q0 + q.ql <= p.Tq &&
         (int64_t)q.k0 + q.kl <= p.Tkv && q.ql <= p.max_q && q.kl <= p.max_kv;
}

// What one thread of a softmax warpgroup knows of its row.
struct Row {
  int tok, head;  // token of the sequence, query head
  bool valid;
  int lim;        // keys [0, lim) are seen
  int pos;        // position among the keys (beyond 2^24 not every one is an fp32 number; distances are taken first)
  float nslope;   // -slope log2(e)
};
__device__ __forceinline__ Row make_row(const TcParams& p, const Seq& q, int s, int kvh, int tok0, int r) {
  Row w;
  const int t = r / p.G;
  w.tok = tok0 + t;
  w.head = kvh * p.G + (r - t * p.G);
  w.valid = t < p.tpt && w.tok < q.ql;
  const int pos = w.tok + q.kl - q.ql;
  w.lim = q.kl;
  if (p.a.causal) w.lim = min(q.kl, max(pos + 1, p.a.prefix ? p.a.prefix[s] : 0));
  w.pos = pos;
  w.nslope = p.a.slopes && w.valid ? -p.a.slopes[w.head] * kLog2e : 0.0f;
  return w;
}

__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// Two scores q.k to log2 units, MOD bit 0: capped. tanh(x) is x p(x^2) for |x| <= 1, p of
// degree 5, fitted so that x p(x^2) has the least maximal error: within 3.2e-7 of tanh(x) in
// fp32 (p itself is 3.2e-6 below 1 at 0). Eight packed multiply-adds a pair. A row with a larger
// score among those it sees of the tile (small = false) takes 1 - 2 / (1 + e^2x), as exact
// (e^2x = inf gives 1), but two more MUFU operations a score beside the exponential: that
// bounded the kernel (286 instead of 230 us on six documents of 333 to 2500 tokens, 32 heads).
// The two differ in the last bits, so each row chooses by what it sees alone: hidden keys and
// other rows, which may hold anything, do not reach its result. A warp with rows of both kinds
// runs both: the same documents with scores ten times as large took 348 us, and 288 when the warp
// chose for all of its rows. tanh.approx is exact to 2^-11
// only, which times a cap of 50 would be 2% of a probability.
template <int MOD>
__device__ __forceinline__ float2 to_log2(const TcParams& p, float2 z, bool small) {
  if constexpr (!(MOD & 1)) {
    return fmul2(z, both(p.scale_log2));
  } else if (small) {
    const float2 x = fmul2(z, both(p.cap_x)), y = fmul2(x, x);
    float2 r = ffma2(y, both(p.tanh_c[5]), both(p.tanh_c[4]));
#pragma unroll
    for (int i = 3; i >= 0; --i) r = ffma2(y, r, both(p.tanh_c[i]));
    return fmul2(x, r);
  } else {
    z = fmul2(z, both(p.cap_in));
    const float2 e = fadd2(make_float2(ex2_approx(z.x), ex2_approx(z.y)), both(1.0f));
    return ffma2(make_float2(rcp_approx(e.x), rcp_approx(e.y)), both(-2.0f * p.cap_log2), both(p.cap_log2));
  }
}

// One softmax step of a warp's 32 rows: S (128 keys, TMEM) -> P over its first 64 columns.
// `turn` runs before the exp pass and returns false to abandon; `half` runs when keys 0..63
// of P are stored. masked: some row of the tile sees only the first n_ok < 128 keys.
template <int DP, class T, int MOD, class Turn, class Half>
__device__ __forceinline__ bool softmax_step(const TcParams& p, uint32_t s_addr, uint32_t o_addr, bool have_o, bool masked,
                                             int n_ok, float dist0, float nslope, float& m_used, float& l, Turn turn,
                                             Half half) {
  uint32_t u[4][32];
  __syncwarp();
#pragma unroll
  for (int g = 0; g < 4; ++g) tmem_ld_32x32b_x32(s_addr + (uint32_t)(g * 32), u[g]);
  tmem_wait_ld();
  if constexpr (MOD != 0) {
    bool small = true;
    if constexpr (MOD & 1) {
      float top[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < kBK; c += 8)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          top[i] = fmax3(top[i], fabsf(__uint_as_float(u[c >> 5][(c & 31) + 2 * i])),
                         fabsf(__uint_as_float(u[c >> 5][(c & 31) + 2 * i + 1])));
      small = n_ok <= 0 || !(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) > p.cap_small);
      if (masked && !small) {  // rarely: again over the keys that the row sees
        small = true;
#pragma unroll
        for (int c = 0; c < kBK; ++c) small &= c >= n_ok || !(fabsf(__uint_as_float(u[c >> 5][c & 31])) > p.cap_small);
      }
    }
    auto modify = [&](bool sm) {
#pragma unroll
      for (int c = 0; c < kBK; c += 2) {
        float2 z = to_log2<MOD>(p, make_float2(__uint_as_float(u[c >> 5][c & 31]), __uint_as_float(u[c >> 5][(c & 31) + 1])), sm);
        if constexpr (MOD & 2) {
          z.x = fmaf(nslope, fabsf(dist0 - (float)c), z.x);
          z.y = fmaf(nslope, fabsf(dist0 - (float)(c + 1)), z.y);
        }
        u[c >> 5][c & 31] = __float_as_uint(z.x);
        u[c >> 5][(c & 31) + 1] = __float_as_uint(z.y);
      }
    };
    if (small)
      modify(true);
    else
      modify(false);
    __syncwarp();
  }
  if (masked) {
#pragma unroll
    for (int c = 0; c < kBK; ++c)
      if (c >= n_ok) u[c >> 5][c & 31] = 0xff800000u;
  }
  float pm[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int c = 0; c < kBK; c += 8)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      pm[i] = fmax3(pm[i], __uint_as_float(u[c >> 5][(c & 31) + 2 * i]), __uint_as_float(u[c >> 5][(c & 31) + 2 * i + 1]));
  const float sc = MOD ? 1.0f : p.scale_log2;  // positive, so max(s) sc = max(s sc)
  const float m_new = fmaxf(m_used, fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3])) * sc);
  const bool need = m_new > m_used + Op<T>::kSlack;
  if (__any_sync(0xffffffffu, need)) {
    // The PV of the step before completed before S was posted, so O is at rest here.
    if (have_o) {
      const float f = need ? ex2_approx(m_used - m_new) : 1.0f;
#pragma unroll 1
      for (int c = 0; c < DP; c += 32) {
        uint32_t o[32];
        __syncwarp();
        tmem_ld_32x32b_x32(o_addr + (uint32_t)c, o);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
        tmem_st_32x32b_x32(o_addr + (uint32_t)c, o);
      }
    }
    if (need) {
      l *= ex2_approx(m_used - m_new);
      m_used = m_new;
    }
  }
  if (!turn()) return false;
  const float neg_m = (m_used == -INFINITY) ? 0.0f : Op<T>::kLift - m_used;
  const float2 sc2 = make_float2(sc, sc), nm2 = make_float2(neg_m, neg_m);
  float2 psa = make_float2(0.0f, 0.0f), psb = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    uint32_t w[16];
#pragma unroll
    for (int c = 0; c < 16; ++c) {
      const float2 z = make_float2(__uint_as_float(u[g][2 * c]), __uint_as_float(u[g][2 * c + 1]));
      const float2 x = MOD ? fadd2(z, nm2) : ffma2(z, sc2, nm2);
      const float e0 = ex2_approx(x.x), e1 = ex2_approx(x.y);
      if (c & 1)
        psb = fadd2(psb, make_float2(e0, e1));
      else
        psa = fadd2(psa, make_float2(e0, e1));
      w[c] = Op<T>::pack(e0, e1);
    }
    tmem_st_32x32b_x16(s_addr + (uint32_t)(g * 16), w);
    if (g == 1) {
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      half();
    }
  }
  l += (psa.x + psb.x) + (psa.y + psb.y);
  tmem_wait_st();
  tc_fence_before();
  __syncwarp();
  return true;
}

// The state of one row of softmax_step_few: the four lanes of a quad hold it alike, but for
// l, of which each has its own keys' part.
struct FewRow {
  float m = -INFINITY, l = 0.0f;
  int lim = 0, pos = 0;
  float nslope = 0.0f;
};

// softmax_step for a tile of at most 16 rows, TMEM lanes 0 to 15 of the warp: a quad of lanes
// shares a row (and, two = true, the one eight further), 32 scores a lane and row instead of
// 128 on as many lanes as there are rows. A step of one token of four heads takes a third of the time;
// for heads of 64 channels it is longer than the loads of its keys otherwise.
template <int DP, class T, int MOD>
__device__ __forceinline__ void softmax_step_few(const TcParams& p, uint32_t s_addr, uint32_t o_addr, bool have_o, bool two,
                                                 int kbase, FewRow (&row)[2]) {
  const int lane = threadIdx.x & 31, j2 = 2 * (lane & 3);
  uint32_t u[64], w[32];
  __syncwarp();
  tmem_ld_16x256b_x16(s_addr, u);
  tmem_wait_ld();
  float f[2] = {1.0f, 1.0f};
  bool need_any = false;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (h && !two) break;
    FewRow& r = row[h];
    auto at = [&](int i, int e) -> uint32_t& { return u[4 * i + 2 * h + e]; };
    const int n_ok = r.lim - kbase - j2;
    bool small = true;
    if constexpr (MOD & 1) {
      float top = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmax3(top, fabsf(__uint_as_float(at(i, 0))), fabsf(__uint_as_float(at(i, 1))));
      small = !(top > p.cap_small) || n_ok <= 0;
      if (!small) {  // rarely: again over the keys that the row sees
        small = true;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          small &= 8 * i >= n_ok || !(fabsf(__uint_as_float(at(i, 0))) > p.cap_small);
          small &= 8 * i + 1 >= n_ok || !(fabsf(__uint_as_float(at(i, 1))) > p.cap_small);
        }
      }
    }
    const float dist0 = (float)(r.pos - (kbase + j2));
    float top = -INFINITY;
    auto modify = [&](bool sm) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float2 z = to_log2<MOD>(p, make_float2(__uint_as_float(at(i, 0)), __uint_as_float(at(i, 1))), sm);
        if constexpr (MOD & 2) {
          z.x = fmaf(r.nslope, fabsf(dist0 - (float)(8 * i)), z.x);
          z.y = fmaf(r.nslope, fabsf(dist0 - (float)(8 * i + 1)), z.y);
        }
        z.x = 8 * i < n_ok ? z.x : -INFINITY;
        z.y = 8 * i + 1 < n_ok ? z.y : -INFINITY;
        top = fmax3(top, z.x, z.y);
        at(i, 0) = __float_as_uint(z.x);
        at(i, 1) = __float_as_uint(z.y);
      }
    };
    if (small)
      modify(true);
    else
      modify(false);
    __syncwarp();
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float m_new = fmaxf(r.m, top);
    if (m_new > r.m + Op<T>::kSlack) {
      f[h] = ex2_approx(r.m - m_new);
      r.l *= f[h];
      r.m = m_new;
      need_any = true;
    }
    const float neg_m = r.m == -INFINITY ? 0.0f : Op<T>::kLift - r.m;
    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float e0 = ex2_approx(__uint_as_float(at(i, 0)) + neg_m), e1 = ex2_approx(__uint_as_float(at(i, 1)) + neg_m);
      sum = fadd2(sum, make_float2(e0, e1));
      w[2 * i + h] = Op<T>::pack(e0, e1);
    }
    r.l += sum.x + sum.y;
  }
  if (!two) {
#pragma unroll
    for (int i = 0; i < 16; ++i) w[2 * i + 1] = 0;  // rows 8 to 15 are nobody's
  }
  if (__any_sync(0xffffffffu, need_any) && have_o) {
    // TMEM lane = row here: the factor of row `lane` is with quad lane % 8.
    const float f0 = __shfl_sync(0xffffffffu, f[0], 4 * (lane & 7)), f1 = __shfl_sync(0xffffffffu, f[1], 4 * (lane & 7));
    const float mine = lane < 8 ? f0 : lane < 16 ? f1 : 1.0f;
#pragma unroll 1
    for (int c = 0; c < DP; c += 32) {
      uint32_t o[32];
      __syncwarp();
      tmem_ld_32x32b_x32(o_addr + (uint32_t)c, o);
      tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * mine);
      tmem_st_32x32b_x32(o_addr + (uint32_t)c, o);
    }
  }
  __syncwarp();
  tmem_st_16x128b_x16(s_addr, w);
  tmem_wait_st();
  tc_fence_before();
  __syncwarp();
}

// Stores n <= 32 fp32 values times inv as bf16 / fp16.
__device__ __forceinline__ void store_out(const TcParams& p, int64_t at, const uint32_t (&o)[32], float inv, int n) {
  uint16_t* dst = reinterpret_cast<uint16_t*>(p.a.out) + at;
  const bool bf = p.a.out_type == kBF16;
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float a = __uint_as_float(o[i + 2 * e]) * inv, b = __uint_as_float(o[i + 2 * e + 1]) * inv;
      w[e] = bf ? Op<__nv_bfloat16>::pack(a, b) : Op<__half>::pack(a, b);
    }
    if (p.out_vec) {  // d % 8 == 0: whole 16-byte pieces
      if (i < n) *reinterpret_cast<uint4*>(dst + i) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (i + e < n) dst[i + e] = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
    }
  }
}

// A row computed again by one warp without the tensor core, lanes over channels, keys
// [j0, j1) of the sequence one after another: for a row whose accumulator holds an
// infinity or NaN. A masked key's probability is 0, but 0 times a value that is not finite
// is NaN in a matrix product; here such keys are left out.
template <class T>
__device__ __noinline__ void slow_row(const TcParams& p, int64_t qrow, int head, int k0, int j0, int j1, int pos, float nslope,
                                      float (&o)[4], float& m, float& l) {
  const RaggedAttention& a = p.a;
  const int lane = threadIdx.x & 31, kvh = head / p.G;
  const T* q = reinterpret_cast<const T*>(a.q) + qrow * a.ldq + (int64_t)head * a.d;
  float qv[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    qv[c] = lane + 32 * c < a.d ? to_f32(q[lane + 32 * c]) : 0.0f;
    o[c] = 0.0f;
  }
  m = -INFINITY;
  l = 0.0f;
  for (int j = j0; j < j1; ++j) {
    const T* k = reinterpret_cast<const T*>(a.k) + (int64_t)(k0 + j) * a.ldk + (int64_t)kvh * a.d;
    const T* v = reinterpret_cast<const T*>(a.v) + (int64_t)(k0 + j) * a.ldv + (int64_t)kvh * a.d;
    float z = 0.0f;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (lane + 32 * c < a.d) z = fmaf(qv[c], to_f32(k[lane + 32 * c]), z);
    z = warp_add(z);
    z = a.cap > 0.0f ? p.cap_log2 - 2.0f * p.cap_log2 * rcp_approx(1.0f + ex2_approx(z * p.cap_in)) : z * p.scale_log2;
    z = fmaf(nslope, fabsf((float)(pos - j)), z);
    if (z == -INFINITY) continue;
    const float mn = fmaxf(m, z), f = ex2_approx(m - mn), w = ex2_approx(z - mn);
    m = mn;
    l = l * f + w;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (lane + 32 * c < a.d) o[c] = fmaf(w, to_f32(v[lane + 32 * c]), o[c] * f);
  }
}

// The rows of a warp whose accumulators are not finite, again by slow_row: normalised into
// out, or (m, l, O) into a piece.
template <class T>
__device__ __noinline__ void redo_rows(const TcParams& p, const Seq& q, const Row& w, bool bad, int j0, int j1, float* piece,
                                       int r) {
  const int lane = threadIdx.x & 31;
  for (unsigned todo = __ballot_sync(0xffffffffu, bad); todo; todo &= todo - 1) {
    const int src = __ffs(todo) - 1;
    const int tok = __shfl_sync(0xffffffffu, w.tok, src), head = __shfl_sync(0xffffffffu, w.head, src);
    const int lim = __shfl_sync(0xffffffffu, w.lim, src), row = __shfl_sync(0xffffffffu, r, src);
    const int pos = __shfl_sync(0xffffffffu, w.pos, src);
    const float ns = __shfl_sync(0xffffffffu, w.nslope, src);
    float o[4], m, l;
    slow_row<T>(p, (int64_t)q.q0 + tok, head, q.k0, j0, min(j1, lim), pos, ns, o, m, l);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const float lift = ex2_approx(Op<T>::kLift);  // as the other pieces of the row
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int ch = lane + 32 * c;
      if (ch >= p.a.d) continue;
      if (piece) {
        piece[(int64_t)row * (p.a.d + 2) + ch] = o[c] * lift;
      } else {
        const int64_t at = ((int64_t)q.q0 + tok) * p.a.ldo + (int64_t)head * p.a.d + ch;
        if (p.a.out_type == kBF16)
          reinterpret_cast<__nv_bfloat16*>(p.a.out)[at] = from_f32<__nv_bfloat16>(o[c] * inv);
        else
          reinterpret_cast<__half*>(p.a.out)[at] = from_f32<__half>(o[c] * inv);
      }
    }
    if (piece && lane == 0) {
      piece[(int64_t)row * (p.a.d + 2) + p.a.d] = m;
      piece[(int64_t)row * (p.a.d + 2) + p.a.d + 1] = l * lift;
    }
  }
}

// O of one row from TMEM to out (normalised), or to a piece with m and l.
template <int DP, class T>
__device__ __forceinline__ void finish_rows(const TcParams& p, const Seq& q, const Row& w, uint32_t o_addr, bool have_o,
                                            float m, float l, int j0, int j1, float* piece, int r) {
  const bool none = !have_o || l == 0.0f;
  const float inv = none ? 0.0f : 1.0f / l;
  uint32_t big = 0;
#pragma unroll 1
  for (int c = 0; c < DP; c += 32) {
    uint32_t o[32];
    __syncwarp();
    if (have_o) {
      tmem_ld_32x32b_x32(o_addr + (uint32_t)c, o);
      tmem_wait_ld();
    }
    if (!w.valid || c >= p.a.d) continue;
    if (none) {  // no key: zero, whatever TMEM holds
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        if (have_o) big = max(big, o[i] & 0x7fffffffu);
        o[i] = 0;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) big = max(big, o[i] & 0x7fffffffu);
    }
    const int n = min(32, p.a.d - c);
    if (piece) {
      float* dst = piece + (int64_t)r * (p.a.d + 2) + c;
#pragma unroll
      for (int i = 0; i < 32; i += 2)  // d is a multiple of 8, so pairs are 8-byte aligned
        if (i < n) *reinterpret_cast<float2*>(dst + i) = make_float2(__uint_as_float(o[i]), __uint_as_float(o[i + 1]));
    } else {
      store_out(p, ((int64_t)q.q0 + w.tok) * p.a.ldo + (int64_t)w.head * p.a.d + c, o, inv, n);
    }
  }
  if (piece && w.valid)
    *reinterpret_cast<float2*>(piece + (int64_t)r * (p.a.d + 2) + p.a.d) = make_float2(none ? -INFINITY : m, none ? 0.0f : l);
  const bool bad = p.a.causal && w.valid && !none && big >= 0x7f800000u;
  __syncwarp();
  if (__any_sync(0xffffffffu, bad)) redo_rows<T>(p, q, w, bad, j0, j1, piece, r);
}

// Rows [valid, 128) of a V tile in shared memory to zero (the whole warp): keys past the
// sequence belong to others, and 0 times what they hold need not be 0. The 128-byte
// swizzle moves 16-byte pieces within a row only.
template <int DP>
__device__ __forceinline__ void zero_v_tail(uint8_t* v, int valid) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int a = 0; a < DP / 64; ++a)
    for (int i = valid * 8 + lane; i < kBK * 8; i += 32)
      *reinterpret_cast<uint4*>(v + a * (kBK * 128) + i * 16) = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  __syncwarp();
}

// ------------------------------------------------------------------------------------
// Two neighbouring tiles of one key head of one sequence.
// ------------------------------------------------------------------------------------
template <int DP>
struct TilesCfg {
  static constexpr int ATOM = kBQ * 128;
  static constexpr int ATOMS = DP / 64;
  static constexpr int Q_BYTES = ATOMS * ATOM;
  static constexpr int KV_BYTES = ATOMS * ATOM;
  static constexpr int SLOTS = DP == 128 ? 5 : 10;
  static constexpr int SMEM = 2 * Q_BYTES + SLOTS * KV_BYTES + 1024 + 512;  // 512: barriers, TMEM address, abort words, scan
  static_assert((13 + 2 * SLOTS) * 8 + 4 + kAbortWords(kThreads / 32) * 4 + 64 <= 512, "room behind the slots");
};
constexpr uint32_t kOCol = 256;  // TMEM: S_A | S_B | O_A | O_B

// The pair of tiles `want` (counted over all sequences) belongs to: sequence and first
// pair, or -1. All threads; two barriers per 384 sequences.
__device__ __forceinline__ int find_pair(const TcParams& p, int want, int* sh, int& pair) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int base = 0;
  if (threadIdx.x == 0) sh[13] = -1;
  for (int s0 = 0; s0 < p.a.n_seq; s0 += kThreads) {
    const int s = s0 + threadIdx.x;
    Seq q;
    int n = 0;
    if (s < p.a.n_seq) {
      if (load_seq(p.a, s, q))
        n = (q.ql + 2 * p.tpt - 1) / (2 * p.tpt);
      else
        atomicOr(p.a.err, kErrBadIndex);
    }
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) sh[warp] = x;
    __syncthreads();
    int before = base, all = base;
    for (int i = 0; i < kThreads / 32; ++i) {
      if (i < warp) before += sh[i];
      all += sh[i];
    }
    const int first = before + x - n;
    if (want >= first && want < first + n) {
      sh[13] = s;
      sh[14] = want - first;
    }
    __syncthreads();
    base = all;
    if (sh[13] >= 0 && blockIdx.x < gridDim.x - 1) break;
  }
  // The launch has room for the pairs of sequences that share no query row.
  if (threadIdx.x == 0 && blockIdx.x == gridDim.x - 1 && base > (int)(gridDim.x / p.a.kv_heads)) atomicOr(p.a.err, kErrBadIndex);
  pair = sh[14];
  return sh[13];
}

template <int DP, class T, int MOD>
__global__ void __launch_bounds__(kThreads, 1)
    k_ragged_tiles(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                   const __grid_constant__ CUtensorMap tmV, const __grid_constant__ TcParams p) {
  using C_ = TilesCfg<DP>;
  constexpr uint32_t IDESC_S = make_idesc(Op<T>::kFmt, 0, 0, kBQ, kBK);
  constexpr uint32_t IDESC_O = make_idesc(Op<T>::kFmt, 0, 1 /*V is MN-major*/, kBQ, DP);
  constexpr int SLOTS = C_::SLOTS;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sR = sQ + 2 * C_::Q_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sR + SLOTS * C_::KV_BYTES);
  uint64_t* q_full = bars;
  uint64_t* s_full = bars + 1;   // [2] S_t(j) ready (and PV_t(j-1) done)
  uint64_t* p_half = bars + 3;   // [2] keys 0..63 of P_t(j) stored, O_t rescaled
  uint64_t* p_full = bars + 5;   // [2]
  uint64_t* turn = bars + 7;     // [2] the tile finished its exp pass
  uint64_t* o_final = bars + 9;  // [2]
  uint64_t* drain = bars + 11;   // [2]
  uint64_t* r_full = bars + 13;  // [SLOTS]
  uint64_t* r_empty = r_full + SLOTS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(r_empty + SLOTS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* scan = reinterpret_cast<int*>(tmem_slot + 1 + kAbortWords(kThreads / 32));  // [16]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvh = blockIdx.x % p.a.kv_heads;
  int pair;
  const int s = find_pair(p, blockIdx.x / p.a.kv_heads, scan, pair);
  if (s < 0) return;  // uniform: fewer pairs than the launch allowed for
  Seq q;
  load_seq(p.a, s, q);
  // Late tiles first: with a causal mask they have the most keys.
  const int pairs = (q.ql + 2 * p.tpt - 1) / (2 * p.tpt);
  const int tok0 = (pairs - 1 - pair) * 2 * p.tpt;
  const int pre = p.a.causal && p.a.prefix ? p.a.prefix[s] : 0;
  // Key tiles of each of the two tiles (0: the tile has no token or no key).
  auto tiles_of = [&](int t) {
    const int first = tok0 + t * p.tpt;
    if (first >= q.ql) return 0;
    const int last = min(q.ql, first + p.tpt) - 1;
    const int lim = p.a.causal ? min(q.kl, max(last + q.kl - q.ql + 1, pre)) : q.kl;
    return (max(lim, 0) + kBK - 1) / kBK;
  };
  const int nA = tiles_of(0), nB = tiles_of(1);
  const int nkv = max(nA, nB);
  const bool two = nB > 0;  // nA <= nB then, tile limits grow with the tokens

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < SLOTS; ++i) {
      mbar_init(&r_full[i], 1);
      mbar_init(&r_empty[i], two ? 2 : 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_half[i], 4);
      mbar_init(&p_full[i], 4);
      mbar_init(&turn[i], 4);
      mbar_init(&o_final[i], 1);
      mbar_init(&drain[i], 1);
    }
    for (int i = 0; i < kAbortWords(kThreads / 32); ++i) abort_flag[i] = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  int* err = p.a.err;
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsControl));
    if (warp == 0) {
      // ------------------------------ TMA producer ------------------------------
      if (nkv > 0) {  // the whole warp: an elected lane issues
        const int nq = two ? 2 : 1;
        const uint32_t qbar = smem_u32(q_full), ring = smem_u32(sR), full0 = smem_u32(r_full);
        mbar_expect_tx_elect(qbar, nq * C_::ATOMS * p.G * p.tpt * 128);
        for (int t = 0; t < nq; ++t)
          for (int a = 0; a < C_::ATOMS; ++a)
            tma_load_3d_elect(smem_u32(sQ) + t * C_::Q_BYTES + a * C_::ATOM, &tmQ, qbar, a * 64, kvh * p.G,
                              q.q0 + tok0 + t * p.tpt);
        int issued = -1;
        RingPos at;
        for (int i = 0; i < 2 * nkv; ++i, at.next(SLOTS)) {
          if (!mbar_wait_warp(&r_empty[at.slot], at.phase ^ 1u, abort_flag, err, kErrAttnWait)) break;
          const uint32_t bar = full0 + (uint32_t)(at.slot * 8), dst = ring + (uint32_t)(at.slot * C_::KV_BYTES);
          mbar_expect_tx_elect(bar, C_::KV_BYTES);
          const CUtensorMap* tm = (i & 1) ? &tmV : &tmK;
          for (int a = 0; a < C_::ATOMS; ++a)
            tma_load_3d_elect(dst + a * C_::ATOM, tm, bar, a * 64, kvh, q.k0 + (i >> 1) * kBK);
          issued = i;
        }
        if (issued < 2 * nkv - 1) {
          // Aborted: wait (bounded) for the loads this CTA still has in flight.
          const uint64_t t0 = globaltimer_ns();
          while (!mbar_try_wait(q_full, 0) && globaltimer_ns() - t0 < kWaitLimitNs) {
          }
          for (int i = max(0, issued - SLOTS + 1); i <= issued; ++i)
            while (!mbar_try_wait(&r_full[i % SLOTS], (i / SLOTS) & 1) && globaltimer_ns() - t0 < kWaitLimitNs) {
            }
          __syncwarp();
        }
      }
    } else if (warp == 1 || warp == 2) {
      // ------------------------------ MMA issuers -------------------------------
      // The whole warp runs the loop (it zeroes the last V tile's tail); an elected lane issues.
      const int t = warp - 1, nt = t ? nB : nA;
      if (nt > 0 || (t == 0 && two)) {
        bool ok = mbar_wait_warp(q_full, 0, abort_flag, err, kErrAttnWait);
        tc_fence_after();
        const uint64_t qd = sdesc_k_sw128(smem_u32(sQ + t * C_::Q_BYTES)), kd0 = sdesc_k_sw128(smem_u32(sR));
        const uint64_t vd0 = sdesc_mn_sw128(smem_u32(sR), C_::ATOM, 1024);
        const uint32_t d_s = tmem + (uint32_t)(t * kBK);
        const uint32_t d_o = tmem + kOCol + (uint32_t)(t * DP);
        RingPos k, v;  // K_j is load 2j of the ring, V_j load 2j + 1
        v.next(SLOTS);
        for (int j = 0; ok && j <= nkv; ++j) {
          // K_j and V_(j-1) normally landed long ago; waiting for them before P_t(j-1) lets the
          // PV and the QK^T go out back to back once P is there.
          if (j > 0 && !mbar_wait_warp(&r_full[v.slot], v.phase, abort_flag, err, kErrAttnWait)) break;
          if (j < nkv && !mbar_wait_warp(&r_full[k.slot], k.phase, abort_flag, err, kErrAttnWait)) break;
          if (j > 0) {
            if (j <= nt) {
              if (j * kBK > q.kl) zero_v_tail<DP>(sR + v.slot * C_::KV_BYTES, q.kl - (j - 1) * kBK);
              const uint64_t vd = vd0 + (uint64_t)(v.slot * (C_::KV_BYTES >> 4));
              if (!mbar_wait_warp(&p_half[t], (j - 1) & 1, abort_flag, err, kErrAttnWait)) break;
              tc_fence_after();
              umma4_f16_ts_elect(d_o, d_s, vd, IDESC_O, j > 1 ? 1u : 0u);
              if (!mbar_wait_warp(&p_full[t], (j - 1) & 1, abort_flag, err, kErrAttnWait)) break;
              tc_fence_after();
              umma4_f16_ts_elect(d_o, d_s + 32, vd + 512, IDESC_O, 1u);
              umma_commit_elect(&r_empty[v.slot]);
              if (j == nt) umma_commit_elect(&o_final[t]);
            } else if (lane == 0) {
              mbar_arrive(&r_empty[v.slot]);  // the other tile's keys
            }
            v.next(SLOTS);
            v.next(SLOTS);
          }
          if (j < nkv) {
            if (j < nt) {
              const uint64_t kd = kd0 + (uint64_t)(k.slot * (C_::KV_BYTES >> 4));
              tc_fence_after();
              if constexpr (DP == 128)
                umma8_f16_ss_elect(d_s, qd, kd, IDESC_S);
              else
                umma4_f16_ss_elect(d_s, qd, kd, IDESC_S);
              umma_commit_elect(&s_full[t]);
              umma_commit_elect(&r_empty[k.slot]);
            } else if (lane == 0) {
              mbar_arrive(&r_empty[k.slot]);
            }
            k.next(SLOTS);
            k.next(SLOTS);
          }
          __syncwarp();
        }
        umma_commit_elect(&drain[t]);
        {
          const uint64_t t0 = globaltimer_ns();
          while (!mbar_try_wait(&drain[t], 0))
            if (globaltimer_ns() - t0 > kWaitLimitNs) {
              if (lane == 0) atomicOr(err, kErrWaitDrain);
              break;
            }
        }
        __syncwarp();
      }
    }
  } else {
    // ------------------------------ softmax / epilogue ------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const int t = (warp - 4) >> 2, qq = warp & 3;
    const int r = qq * 32 + lane, nt = t ? nB : nA;
    Row w = make_row(p, q, s, kvh, tok0 + t * p.tpt, r);
    if ((MOD & 1) && !w.valid) w.lim = 0;  // what nobody's row holds must not cost the warp the longer tanh
    const uint32_t lane_base = tmem + ((uint32_t)(qq * 32) << 16);
    const uint32_t s_addr = lane_base + (uint32_t)(t * kBK);
    const uint32_t o_addr = lane_base + kOCol + (uint32_t)(t * DP);
    // The tile's first token has the smallest limit.
    const int lim0 = p.a.causal ? min(q.kl, max(tok0 + t * p.tpt + q.kl - q.ql + 1, pre)) : q.kl;
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    for (int j = 0; j < nt; ++j) {
      if (!mbar_wait_warp(&s_full[t], j & 1, abort_flag, err, kErrAttnWait)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int kbase = j * kBK;
      ok = softmax_step<DP, T, MOD>(
          p, s_addr, o_addr, j > 0, kbase + kBK > lim0, w.lim - kbase, (float)(w.pos - kbase), w.nslope, m, l,
          [&]() {
            // The tiles take turns (A(0), B(0), A(1), ...) while both have keys.
            if (!two || (t == 0 ? j == 0 : j >= nA)) return true;
            return mbar_wait_warp(&turn[t ^ 1], (t == 0 ? j - 1 : j) & 1, abort_flag, err, kErrAttnWait);
          },
          [&]() {
            if (lane == 0) mbar_arrive(&p_half[t]);
          });
      if (!ok) break;
      if (lane == 0) {
        mbar_arrive(&p_full[t]);
        mbar_arrive(&turn[t]);
      }
    }
    if (ok && (nt == 0 || mbar_wait_warp(&o_final[t], 0, abort_flag, err, kErrAttnWait))) {
      tc_fence_after();
      finish_rows<DP, T>(p, q, w, o_addr, nt > 0, m, l, 0, q.kl, nullptr, r);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------------------------
// Sequences of one tile each.
// ------------------------------------------------------------------------------------
// Shared list of the launch's sequences: first[s] is the number of key tiles (steps) of
// the sequences before s over all key heads, first[n] the total. A sequence with queries has at
// least one step per key head, so that rows without a key are written.
struct StepList {
  int first[kMaxSeqs + 1];
  int per, extra;  // steps of a worker, one more for the first `extra`
  Seq seq[kMaxSeqs];
  int warp_sum[32];

  __device__ __forceinline__ int begin(int worker) const { return worker * per + min(worker, extra); }
  __device__ __forceinline__ int worker_of(int step) const {
    const int longer = extra * (per + 1);
    return step < longer ? step / (per + 1) : extra + (step - longer) / per;
  }
};
__device__ __forceinline__ int steps_of(const Seq& q) { return max(1, (q.kl + kBK - 1) / kBK); }

// All threads of the block (a multiple of 32, at most 1024); ends with a barrier. The launcher
// keeps the total below 2^31.
__device__ __forceinline__ void build_steps(const TcParams& p, StepList& L, int n, int workers) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  int base = 0;
  for (int s0 = 0; s0 < n; s0 += blockDim.x) {
    const int s = s0 + threadIdx.x;
    Seq q = {0, 0, 0, 0};
    if (s < n && !load_seq(p.a, p.seq0 + s, q)) {
      atomicOr(p.a.err, kErrBadIndex);
      q = {0, 0, 0, 0};
    }
    int x = q.ql > 0 ? steps_of(q) * p.a.kv_heads : 0;
    const int own = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) L.warp_sum[warp] = x;
    __syncthreads();
    int all = base;
    for (int i = 0; i < nw; ++i) {
      if (i < warp) x += L.warp_sum[i];
      all += L.warp_sum[i];
    }
    if (s < n) {
      L.first[s] = base + x - own;
      L.seq[s] = q;
    }
    base = all;
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    L.first[n] = base;
    L.per = base / workers;
    L.extra = base % workers;
  }
  __syncthreads();
}
// The sequence that step belongs to: the last one with first[s] <= step.
__device__ __forceinline__ int find_step(const StepList& L, int n, int step) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (L.first[mid] <= step)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// A worker's pieces in order: key tiles [kt0, kt1) of key head kvh of sequence s.
struct Pieces {
  const StepList& L;
  int n, at, end;
  int s, kvh, kt0, kt1;
  bool whole;
  __device__ Pieces(const StepList& L_, int n_, int w) : L(L_), n(n_), at(L_.begin(w)), end(L_.begin(w + 1)) {}
  __device__ bool next() {
    if (at >= end) return false;
    s = find_step(L, n, at);
    const int e = steps_of(L.seq[s]), rem = at - L.first[s];
    kvh = rem / e;
    kt0 = rem - kvh * e;
    kt1 = min(e, kt0 + (end - at));
    whole = kt0 == 0 && kt1 == e;
    at += kt1 - kt0;
    return true;
  }
  __device__ int tiles() const { return L.seq[s].kl > 0 ? kt1 - kt0 : 0; }  // to load
};

template <int DP, class T, int MOD, bool FEW>
__global__ void __launch_bounds__(kThreads, 1)
    k_ragged_streams(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                     const __grid_constant__ CUtensorMap tmV, const __grid_constant__ TcParams p) {
  constexpr int ATOM = kBK * 128, ATOMS = DP / 64, KV_BYTES = ATOMS * ATOM;
  constexpr uint32_t IDESC_S = make_idesc(Op<T>::kFmt, 0, 0, kBQ, kBK);
  constexpr uint32_t IDESC_O = make_idesc(Op<T>::kFmt, 0, 1, kBQ, DP);
  constexpr int kMaxSlots = 8;

  extern __shared__ uint8_t smem_raw[];
  __shared__ StepList steps;
  __shared__ uint64_t bars[2][8 + 2 * kMaxSlots];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_words[kAbortWords(kThreads / 32)];
  volatile int* abort_flag = abort_words;
  // Q of worker 0 | Q of worker 1 | slots of worker 0 | of worker 1. A Q atom may be shorter
  // than 128 rows: the MMA then reads rows of what follows, into rows that nobody uses.
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int SL = p.slots;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // Worker of this warp: producers are warps 0 and 3, issuers 1 and 2, softmax 4-7 and 8-11.
  const int t = warp < 4 ? (warp >= 2 ? 1 : 0) : (warp - 4) >> 2;
  // With few rows worker 1 has them in TMEM lanes 32 on (its MMA reads 32 rows of what lies
  // before them), so that the two workers' softmax warps run on different schedulers.
  const int lane0 = FEW ? 32 * t : 0;
  smem += FEW ? kFewPad : 0;
  uint8_t* sQ = smem + t * ATOMS * p.q_atom;
  uint8_t* sR = smem + 2 * ATOMS * p.q_atom + t * SL * KV_BYTES;
  uint64_t* b = bars[t];
  uint64_t *q_full = b, *q_empty = b + 1, *s_full = b + 2, *p_half = b + 3, *p_full = b + 4, *o_full = b + 5,
           *drain = b + 6, *r_full = b + 8, *r_empty = b + 8 + kMaxSlots;
  const int worker = t * gridDim.x + blockIdx.x, workers = 2 * gridDim.x;
  const int n = min(p.a.n_seq - p.seq0, p.seqs);

  if (threadIdx.x < 2) {
    uint64_t* z = bars[threadIdx.x];
    mbar_init(z + 0, 1);
    mbar_init(z + 1, 1);
    mbar_init(z + 2, 1);
    mbar_init(z + 3, 4);
    mbar_init(z + 4, 4);
    mbar_init(z + 5, 1);
    mbar_init(z + 6, 1);
    for (int i = 0; i < SL; ++i) {
      mbar_init(z + 8 + i, 1);
      mbar_init(z + 8 + kMaxSlots + i, 1);
    }
    for (int& w : abort_words) w = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  if (warp == 2 && lane == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  tc_fence_before();
  build_steps(p, steps, n, workers);
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  int* err = p.a.err;
  Pieces it(steps, n, worker);
  // The next launch (k_ragged_join) may be set up now; it waits for this grid's end.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsControl));
    if (warp == 0 || warp == 3) {
      // ------------------------------ TMA producer ------------------------------
      {  // the whole warp: an elected lane issues
        const uint32_t qbar = smem_u32(q_full), ring = smem_u32(sR), full0 = smem_u32(r_full);
        int ld = 0, nq = 0;  // loads and Q tiles so far
        RingPos at;
        bool ok = true;
        while (ok && it.next()) {
          const int nt = it.tiles();
          if (nt == 0) continue;
          const Seq& q = steps.seq[it.s];
          ok = mbar_wait_warp(q_empty, (nq & 1) ^ 1u, abort_flag, err, kErrAttnWait);
          if (!ok) break;
          mbar_expect_tx_elect(qbar, ATOMS * p.G * p.tpt * 128);
          for (int a = 0; a < ATOMS; ++a)
            tma_load_3d_elect(smem_u32(sQ) + a * p.q_atom, &tmQ, qbar, a * 64, it.kvh * p.G, q.q0);
          ++nq;
          for (int i = 0; i < 2 * nt && ok; ++i, at.next(SL)) {
            ok = mbar_wait_warp(&r_empty[at.slot], at.phase ^ 1u, abort_flag, err, kErrAttnWait);
            if (!ok) break;
            const uint32_t bar = full0 + (uint32_t)(at.slot * 8), dst = ring + (uint32_t)(at.slot * KV_BYTES);
            mbar_expect_tx_elect(bar, KV_BYTES);
            const CUtensorMap* tm = (i & 1) ? &tmV : &tmK;
            for (int a = 0; a < ATOMS; ++a)
              tma_load_3d_elect(dst + a * ATOM, tm, bar, a * 64, it.kvh, q.k0 + (it.kt0 + (i >> 1)) * kBK);
            ++ld;
          }
        }
        if (!ok) {
          // Aborted: wait (bounded) for the loads this worker still has in flight.
          const uint64_t t0 = globaltimer_ns();
          if (nq > 0)
            while (!mbar_try_wait(q_full, (nq - 1) & 1) && globaltimer_ns() - t0 < kWaitLimitNs) {
            }
          for (int i = max(0, ld - SL); i < ld; ++i)
            while (!mbar_try_wait(&r_full[i % SL], (i / SL) & 1) && globaltimer_ns() - t0 < kWaitLimitNs) {
            }
          __syncwarp();
        }
      }
    } else {
      // ------------------------------ MMA issuer --------------------------------
      const uint64_t qd = sdesc_k_sw128(smem_u32(sQ) - (uint32_t)(lane0 * 128)), kd0 = sdesc_k_sw128(smem_u32(sR));
      const uint64_t vd0 = sdesc_mn_sw128(smem_u32(sR), ATOM, 1024);
      const uint64_t q_jump = (uint64_t)(p.q_atom >> 4);  // a Q atom may be shorter than 128 rows
      const uint32_t d_s = tmem + (uint32_t)(t * kBK), d_o = tmem + kOCol + (uint32_t)(t * DP);
      int nq = 0, step = 0;
      RingPos at;  // loads in order: K_0, V_0, K_1, V_1, ... of every piece
      bool ok = true;
      while (ok && it.next()) {
        const int nt = it.tiles();
        if (nt == 0) continue;
        const int kl = steps.seq[it.s].kl;
        ok = mbar_wait_warp(q_full, nq & 1, abort_flag, err, kErrAttnWait);
        ++nq;
        tc_fence_after();
        RingPos v = at;
        v.next(SL);
        for (int j = 0; ok && j <= nt; ++j) {
          if (j > 0) {
            uint8_t* vp = sR + v.slot * KV_BYTES;
            ok = mbar_wait_warp(&r_full[v.slot], v.phase, abort_flag, err, kErrAttnWait);
            if (!ok) break;
            const int left = kl - (it.kt0 + j - 1) * kBK;
            if (left < kBK) zero_v_tail<DP>(vp, left);
            const uint64_t vd = vd0 + (uint64_t)(v.slot * (KV_BYTES >> 4));
            ok = mbar_wait_warp(p_half, (step - 1) & 1, abort_flag, err, kErrAttnWait);
            if (!ok) break;
            tc_fence_after();
            umma4_f16_ts_elect(d_o, d_s, vd, IDESC_O, j > 1 ? 1u : 0u);
            ok = mbar_wait_warp(p_full, (step - 1) & 1, abort_flag, err, kErrAttnWait);
            if (!ok) break;
            tc_fence_after();
            umma4_f16_ts_elect(d_o, d_s + 32, vd + 512, IDESC_O, 1u);
            umma_commit_elect(&r_empty[v.slot]);
            if (j == nt) umma_commit_elect(o_full);
            v.next(SL);
            v.next(SL);
          }
          if (j < nt) {
            ok = mbar_wait_warp(&r_full[at.slot], at.phase, abort_flag, err, kErrAttnWait);
            if (!ok) break;
            tc_fence_after();
            const uint64_t kd = kd0 + (uint64_t)(at.slot * (KV_BYTES >> 4));
            umma4_f16_ss_elect(d_s, qd, kd, IDESC_S);
            if constexpr (DP == 128) umma4_f16_ss_elect(d_s, qd + q_jump, kd + (ATOM >> 4), IDESC_S, 1u);
            umma_commit_elect(s_full);
            umma_commit_elect(&r_empty[at.slot]);
            if (j == nt - 1) umma_commit_elect(q_empty);
            at.next(SL);
            at.next(SL);
            ++step;
          }
          __syncwarp();
        }
      }
      umma_commit_elect(drain);
      {
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(drain, 0))
          if (globaltimer_ns() - t0 > kWaitLimitNs) {
            if (lane == 0) atomicOr(err, kErrWaitDrain);
            break;
          }
      }
      __syncwarp();
    }
  } else {
    // ------------------------------ softmax / epilogue ------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const int qq = warp & 3, r = qq * 32 + lane - lane0;
    const uint32_t lane_base = tmem + ((uint32_t)(qq * 32) << 16);
    const uint32_t s_addr = lane_base + (uint32_t)(t * kBK);
    const uint32_t o_addr = lane_base + kOCol + (uint32_t)(t * DP);
    int step = 0, pieces = 0;
    bool ok = true;
    while (ok && it.next()) {
      const Seq q = steps.seq[it.s];
      const int nt = it.tiles(), rows = p.G * q.ql;
      const bool busy = qq * 32 >= lane0 && qq * 32 - lane0 < rows;  // the warp has rows (uniform)
      Row w = make_row(p, q, p.seq0 + it.s, it.kvh, 0, max(r, 0));
      if ((MOD & 1) && !w.valid) w.lim = 0;
      const int lim0 = p.a.causal ? min(q.kl, max(q.kl - q.ql + 1, p.a.prefix ? p.a.prefix[p.seq0 + it.s] : 0)) : q.kl;
      float m = -INFINITY, l = 0.0f;
      FewRow few[2];
      if (FEW && busy) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const Row x = make_row(p, q, p.seq0 + it.s, it.kvh, 0, (lane >> 2) + 8 * h);
          few[h].lim = !(MOD & 1) || x.valid ? x.lim : 0;
          few[h].pos = x.pos;
          few[h].nslope = x.nslope;
        }
      }
      for (int j = 0; j < nt; ++j, ++step) {
        if (!mbar_wait_warp(s_full, step & 1, abort_flag, err, kErrAttnWait)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const int kbase = (it.kt0 + j) * kBK;
        if (!busy) {
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(p_half);
            mbar_arrive(p_full);
          }
        } else if constexpr (FEW) {
          softmax_step_few<DP, T, MOD>(p, s_addr, o_addr, j > 0, rows > 8, kbase, few);
          if (lane == 0) {
            mbar_arrive(p_half);
            mbar_arrive(p_full);
          }
        } else {
          softmax_step<DP, T, MOD>(
              p, s_addr, o_addr, j > 0, kbase + kBK > lim0, w.lim - kbase, (float)(w.pos - kbase), w.nslope, m, l,
              []() { return true; },
              [&]() {
                if (lane == 0) mbar_arrive(p_half);
              });
          if (lane == 0) mbar_arrive(p_full);
        }
      }
      if (FEW) {
        // To one row per lane.
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          few[h].l += __shfl_xor_sync(0xffffffffu, few[h].l, 1);
          few[h].l += __shfl_xor_sync(0xffffffffu, few[h].l, 2);
          const float mh = __shfl_sync(0xffffffffu, few[h].m, 4 * (lane & 7));
          const float lh = __shfl_sync(0xffffffffu, few[h].l, 4 * (lane & 7));
          if (lane >> 3 == h) {
            m = mh;
            l = lh;
          }
        }
      }
      if (!ok) break;
      if (nt > 0) {
        if (!mbar_wait_warp(o_full, pieces & 1, abort_flag, err, kErrAttnWait)) break;
        ++pieces;
        tc_fence_after();
      }
      if (busy) {
        float* piece = nullptr;
        if (!it.whole) piece = p.part + (int64_t)(2 * worker + (it.kt0 > 0 ? 0 : 1)) * p.part_rows * (p.a.d + 2);
        finish_rows<DP, T>(p, q, w, o_addr, nt > 0, m, l, it.kt0 * kBK, it.kt1 * kBK, piece, r);
      }
      tc_fence_before();  // O is read before the next piece's P lets a PV write it
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// The pieces of the rows that k_ragged_streams cut, joined: W warps per row (sequence, token,
// head), each for every W-th piece. Which workers hold them follows from the step list alone;
// rows that one worker finished are already in out. With one warp a row of many pieces is a
// chain of loads: a query over 12828 keys (101 pieces) took 39 us in all, 15 with eight warps to
// a row; for many rows of few pieces eight would mostly idle.
template <class T, int W>
__global__ void __launch_bounds__(256) k_ragged_join(const __grid_constant__ TcParams p, int workers) {
  __shared__ StepList steps;
  __shared__ float4 sum[W > 1 ? W : 1][32];
  __shared__ float sum_l[W];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = min(p.a.n_seq - p.seq0, p.seqs);
  build_steps(p, steps, n, workers);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long rows = (long long)n * p.a.max_q * p.a.heads;
  const int pitch = p.a.d + 2, part = warp % W;
  for (long long x = (long long)blockIdx.x * (8 / W) + warp / W; x < rows; x += (long long)gridDim.x * (8 / W)) {
    const int h = (int)(x % p.a.heads);
    const int y = (int)(x / p.a.heads);
    const int tok = (int)(y % p.a.max_q), s = (int)(y / p.a.max_q);
    const Seq q = steps.seq[s];
    if (tok >= q.ql) continue;
    const int kvh = h / p.G, r = tok * p.G + (h - kvh * p.G), e = steps_of(q);
    const int a = steps.first[s] + kvh * e, w0 = steps.worker_of(a), w1 = steps.worker_of(a + e - 1);
    if (w0 == w1) continue;  // whole
    // The first worker's piece is its last one (slot 1), the others' their first (slot 0).
    auto piece = [&](int w) { return p.part + ((int64_t)(2 * w + (w == w0 ? 1 : 0)) * p.part_rows + r) * pitch; };
    float top = -INFINITY;
    for (int w = w0 + lane; w <= w1; w += 32) top = fmaxf(top, piece(w)[p.a.d]);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (top == -INFINITY) top = 0.0f;
    float l = 0.0f;
    float2 o[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
    for (int b = w0 + part; b <= w1; b += 32 * W) {
      float f = 0.0f;
      if (b + W * lane <= w1) {
        const float2 ml = *reinterpret_cast<const float2*>(piece(b + W * lane) + p.a.d);
        f = ex2_approx(ml.x - top);
        l = fmaf(f, ml.y, l);
      }
      const int cnt = min(32, (w1 - b) / W + 1);
#pragma unroll 4
      for (int i = 0; i < cnt; ++i) {
        const float fi = __shfl_sync(0xffffffffu, f, i);
        const float* src = piece(b + W * i) + 2 * lane;
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if (2 * lane + 64 * c < p.a.d) o[c] = ffma2(both(fi), *reinterpret_cast<const float2*>(src + 64 * c), o[c]);
      }
    }
    l = warp_add(l);
    if constexpr (W > 1) {  // x is the same for the whole block then
      static_assert(W == 8, "a block is one row or eight");
      sum[part][lane] = make_float4(o[0].x, o[0].y, o[1].x, o[1].y);
      if (lane == 0) sum_l[part] = l;
      __syncthreads();
      if (warp == 0) {
#pragma unroll
        for (int i = 1; i < W; ++i) {
          const float4 v = sum[i][lane];
          o[0].x += v.x;
          o[0].y += v.y;
          o[1].x += v.z;
          o[1].y += v.w;
          l += sum_l[i];
        }
      }
      __syncthreads();
      if (warp > 0) continue;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T* out = reinterpret_cast<T*>(p.a.out) + ((int64_t)q.q0 + tok) * p.a.ldo + (int64_t)h * p.a.d;
#pragma unroll
    for (int c = 0; c < 2; ++c)
      if (2 * lane + 64 * c < p.a.d) {
        out[2 * lane + 64 * c] = from_f32<T>(o[c].x * inv);
        out[2 * lane + 64 * c + 1] = from_f32<T>(o[c].y * inv);
      }
  }
}

template <class T>
void launch_join(const TcParams& p) {
  DeviceContext& c = ctx();
  const int64_t rows = (int64_t)std::min(p.a.n_seq - p.seq0, p.seqs) * p.a.max_q * p.a.heads;
  const int64_t most = (int64_t)c.num_sms * 4;
  const bool wide = rows <= most;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)std::min<int64_t>(wide ? rows : (rows + 7) / 8, most));
  cfg.blockDim = dim3(256);
  cfg.stream = c.stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  check_cuda(cudaLaunchKernelEx(&cfg, wide ? k_ragged_join<T, 8> : k_ragged_join<T, 1>, p, 2 * c.num_sms),
             "attention_ragged_join");
  check_launch("attention_ragged_join");
}

template <class K>
void prepare_kernel(K kern, int smem, bool (&done)[64]) {
  const int dev = ctx().device;
  if (done[dev]) return;
  // setmaxnreg.inc waits until the registers it asks for are free; the split only adds up if
  // the kernel was compiled to exactly kRegsLaunch registers per thread.
  cudaFuncAttributes fa{};
  check_cuda(cudaFuncGetAttributes(&fa, kern), "cudaFuncGetAttributes(attention_ragged)");
  if (fa.numRegs != kRegsLaunch)
    fail(kErrUnsupported, "attention_ragged: compiled with " + std::to_string(fa.numRegs) + " registers per thread, the " +
                              "register split needs " + std::to_string(kRegsLaunch));
  check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem),
             "cudaFuncSetAttribute(attention_ragged)");
  done[dev] = true;
}

template <int DP, class T, int MOD, bool FEW>
void launch_streams(TcParams& p, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv) {
  DeviceContext& c = ctx();
  constexpr int kKv = DP / 64 * kBK * 128;
  const int fixed = 1024 + (FEW ? kFewPad : 0) + 2 * (DP / 64) * p.q_atom;
  p.slots = std::min(8, (kMaxSmem - (int)sizeof(StepList) - 1024 - fixed) / (2 * kKv));
  const int smem = fixed + 2 * p.slots * kKv;
  static bool done[64] = {};
  prepare_kernel(k_ragged_streams<DP, T, MOD, FEW>, kMaxSmem - (int)sizeof(StepList) - 1024, done);
  // Sequences of one launch: as many as its step list holds, below 2^31 steps.
  const int64_t most = ((std::min(p.a.max_kv, p.a.Tkv) + kBK - 1) / kBK) * p.a.kv_heads + p.a.kv_heads;
  if (most >= ((int64_t)1 << 31)) fail(kErrInvalidArg, "attention_ragged: too many keys");
  p.seqs = (int)std::min<int64_t>(kMaxSeqs, (((int64_t)1 << 31) - 1) / most);
  for (p.seq0 = 0; p.seq0 < p.a.n_seq; p.seq0 += p.seqs) {
    k_ragged_streams<DP, T, MOD, FEW><<<(unsigned)c.num_sms, kThreads, smem, c.stream>>>(tq, tk, tv, p);
    check_launch("attention_ragged_streams");
    if (p.a.max_kv <= kBK) continue;  // every piece is a whole row
    p.a.out_type == kBF16 ? launch_join<__nv_bfloat16>(p) : launch_join<__half>(p);
  }
}

template <int DP, class T, int MOD>
void launch_mod(TcParams& p, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, bool streams) {
  DeviceContext& c = ctx();
  if (!streams) {
    static bool done[64] = {};
    prepare_kernel(k_ragged_tiles<DP, T, MOD>, TilesCfg<DP>::SMEM, done);
    // Pairs of tiles: at most one per sequence more than the rows make.
    const int64_t pairs = std::min<int64_t>((int64_t)p.a.n_seq * ((p.a.max_q + 2 * p.tpt - 1) / (2 * p.tpt)),
                                            p.a.Tq / (2 * p.tpt) + p.a.n_seq);
    const int64_t grid = pairs * p.a.kv_heads;
    if (grid >= ((int64_t)1 << 31)) fail(kErrInvalidArg, "attention_ragged: too many query tiles");
    k_ragged_tiles<DP, T, MOD><<<(unsigned)grid, kThreads, TilesCfg<DP>::SMEM, c.stream>>>(tq, tk, tv, p);
    check_launch("attention_ragged_tiles");
    return;
  }
  if (p.G * p.tpt <= kFewRows) return launch_streams<DP, T, MOD, true>(p, tq, tk, tv);
  launch_streams<DP, T, MOD, false>(p, tq, tk, tv);
}

template <int DP, class T>
void launch_tc(TcParams p, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, bool streams) {
  const int mod = (p.a.cap > 0.0f ? 1 : 0) | (p.a.slopes ? 2 : 0);
  if (mod == 0) return launch_mod<DP, T, 0>(p, tq, tk, tv, streams);
  if (mod == 1) return launch_mod<DP, T, 1>(p, tq, tk, tv, streams);
  if (mod == 2) return launch_mod<DP, T, 2>(p, tq, tk, tv, streams);
  launch_mod<DP, T, 3>(p, tq, tk, tv, streams);
}

}  // namespace ragged
}  // namespace sdb
