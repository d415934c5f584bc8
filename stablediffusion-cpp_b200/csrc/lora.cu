// lora.cu - a projection shared by every row plus each row's own low-rank adapter:
//   y[t, n] = sum_k x[t, k] W[n, k] + bias[n] + sum_j h[t, j] B_a[n, j],
//   h[t, j] = s_a sum_k x[t, k] A_a[j, k],   a = row_adapter[t] (no second term for a < 0).
//
// With few rows the work is reading W and the adapters once (k_lora_down_rows, k_lora_rows);
// with many it is a GEMM (k_lora_lists, k_lora_gemm).
#include <algorithm>
#include <cmath>

#include "elem.cuh"
#include "internal.h"
#include "ptx.cuh"
#include "serving.h"

namespace sdb {
namespace {

inline int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }
inline size_t align256(size_t b) { return (b + 255) & ~size_t(255); }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

constexpr int kMaxSmem = 232448;
constexpr int kMaxRowsSmall = 128;  // rows of a block of k_lora_rows

// The adapter term rides on the same tensor-core product as W: next to the K blocks of X and
// W, an accumulator runs through the chunks of H and B, where H holds h in the columns of the
// row's own adapter and zeros in those of the other adapters among the rows it is multiplied with.
// A chunk is cw = 16, 32 or 64 ranks of one adapter. For a bf16 output h is rounded to bf16, as a
// bf16 tensor between two products would be: y is off by up to 2^-8 sum_j |h_j B_j| besides its own
// rounding, which is more than that where the terms cancel one another or the shared product.
// For an fp32 output h is kept in two bf16 parts, high and low, and each chunk has one of either:
// 2^-16 sum_j |h_j B_j|. Two parts for bf16 outputs as well took 48 rows with 32 adapters of rank 32,
// 9728 x 2560, 30.8 instead of 28 us a call, and 129 rows of 64 requests of rank 128, 3840 x 3840, 73
// instead of 52.
// K-major operand rows of `pitch` = 32, 64 or 128 bytes in the swizzle of that width.
__device__ __forceinline__ uint64_t sdesc_k(uint32_t saddr, int pitch) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3FFFu);
  d |= (uint64_t)1u << 16;
  d |= (uint64_t)((uint32_t)(8 * pitch) >> 4) << 32;  // 8 rows
  d |= (uint64_t)1u << 46;
  d |= (uint64_t)(pitch == 128 ? 2u : pitch == 64 ? 4u : 6u) << 61;
  return d;
}
// Conversions by the processor's own instructions: eight integer ones and a branch per value
// (f32_to_bf16_rne) were two thirds of the time of products of short rows.
__device__ __forceinline__ uint16_t bf16_bits(float x) { return __bfloat16_as_ushort(__float2bfloat16_rn(x)); }
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// Two bf16 of a word, the low half first.
__device__ __forceinline__ float2 bf16x2_to_f32(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
// h in bf16 (part 0), and what that lost (part 1): together h to 2^-16.
__device__ __forceinline__ uint32_t h_part(float h, int part) {
  const uint32_t hi = bf16_bits(h);
  if (!part) return hi;
  const float v = bf16_to_f32((uint16_t)hi);
  return bf16_bits(fabsf(v) < INFINITY ? h - v : 0.0f);
}
inline int chunk_width(int64_t r) { return r <= 16 ? 16 : r <= 32 ? 32 : 64; }
inline CUtensorMapSwizzle swizzle_of(int cw) {
  return cw == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : cw == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;
}


// ------------------------------------------------------------------------------------
// Few rows
// ------------------------------------------------------------------------------------
// Rows go in blocks of 128. H: [f][part][rc][TN][cw] bf16 for every row f that is the first
// of its adapter in its block.
struct RowsK {
  uint16_t* H;
  int cw, rc, parts;
  __host__ __device__ int per() const { return parts * rc; }  // chunks of an adapter
};

// Whether row i is the first of its adapter (ids of the T rows in shared memory).
__device__ __forceinline__ bool is_first(const int* ids, int i) {
  const int a = ids[i];
  bool first = a >= 0;
  for (int j = 0; j < i; ++j) first &= ids[j] != a;
  return first;
}

// h[t, 8 jb .. + 8] with one warp per value and 16-byte loads of both rows (pitches are
// multiples of 8, elements past K masked), then row t of every adapter's chunks: its own
// values, or zeros. Bound by the adapters' bytes.
__global__ void __launch_bounds__(256) k_lora_down_rows(const LoraLinear p, const uint16_t* __restrict__ X, int64_t ldx,
                                                        const uint16_t* __restrict__ A, int64_t lda, RowsK rk, int TN) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ int ids[kMaxRowsSmall];
  __shared__ float sh[8];
  const int64_t row0 = blockIdx.x / kMaxRowsSmall * kMaxRowsSmall;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = blockIdx.x % kMaxRowsSmall;
  const int T = (int)min(p.T - row0, (int64_t)kMaxRowsSmall), j = blockIdx.y * 8 + warp;
  if (threadIdx.x < T) {
    const int a = p.row_adapter[row0 + threadIdx.x];
    if (a >= p.n_adapters && threadIdx.x == t && blockIdx.y == 0) atomicOr(p.err, kErrBadIndex);
    ids[threadIdx.x] = a < p.n_adapters ? a : -1;
  }
  __syncthreads();
  const int a = ids[t];
  float s = 0.0f;
  if (a >= 0 && j < p.r) {
    const float scale = p.scale ? p.scale[a] : 1.0f;
    const uint16_t* x = X + (row0 + t) * ldx;
    const uint16_t* w = A + ((int64_t)a * p.r + j) * lda;
    float2 s2 = make_float2(0.0f, 0.0f);
    const int whole = (int)(p.K / 8);
#pragma unroll 8
    for (int c = lane; c < whole; c += 32) {
      const uint4 u = *reinterpret_cast<const uint4*>(x + 8 * c), v = __ldg(reinterpret_cast<const uint4*>(w + 8 * c));
      s2 = ffma2(bf16x2_to_f32(u.x), bf16x2_to_f32(v.x), s2);
      s2 = ffma2(bf16x2_to_f32(u.y), bf16x2_to_f32(v.y), s2);
      s2 = ffma2(bf16x2_to_f32(u.z), bf16x2_to_f32(v.z), s2);
      s2 = ffma2(bf16x2_to_f32(u.w), bf16x2_to_f32(v.w), s2);
    }
    s = s2.x + s2.y;
    for (int k = whole * 8 + lane; k < p.K; k += 32) s = fmaf(bf16_to_f32(x[k]), bf16_to_f32(w[k]), s);
    s = warp_add(s) * scale;
  }
  if (lane == 0) sh[warp] = s;
  __syncthreads();
  if (threadIdx.x < T && is_first(ids, threadIdx.x)) {
    const bool own = ids[threadIdx.x] == a;
    const int j0 = blockIdx.y * 8, c = j0 / rk.cw;
    for (int part = 0; part < rk.parts; ++part) {
      uint32_t w[4] = {0, 0, 0, 0};
      if (own)
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e >> 1] |= h_part(sh[e], part) << (16 * (e & 1));
      uint16_t* dst = rk.H + ((((row0 + threadIdx.x) * rk.parts + part) * rk.rc + c) * TN + t) * rk.cw + j0 % rk.cw;
      *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// The same for four rows a CTA: rows of requests come in runs of one adapter, whose A is then
// read once for up to four of them. (A template of both is slower for one row: the loop below
// takes the registers that keep eight loads of the one above in flight.)
constexpr int kRunRows = 4;
__global__ void __launch_bounds__(256) k_lora_down_runs(const LoraLinear p, const uint16_t* __restrict__ X, int64_t ldx,
                                                        const uint16_t* __restrict__ A, int64_t lda, RowsK rk) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  constexpr int R = kRunRows, TN = kMaxRowsSmall;
  static_assert(kMaxRowsSmall % R == 0, "a CTA's rows are of one block");
  __shared__ int ids[kMaxRowsSmall];
  __shared__ float sh[R][8];
  const int64_t row0 = (int64_t)blockIdx.x * R / kMaxRowsSmall * kMaxRowsSmall;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t0 = (int)((int64_t)blockIdx.x * R - row0);
  const int T = (int)min(p.T - row0, (int64_t)kMaxRowsSmall), j = blockIdx.y * 8 + warp, n = min(R, T - t0);
  if (threadIdx.x < T) {
    const int a = p.row_adapter[row0 + threadIdx.x];
    if (a >= p.n_adapters && threadIdx.x >= t0 && threadIdx.x < t0 + n && blockIdx.y == 0) atomicOr(p.err, kErrBadIndex);
    ids[threadIdx.x] = a < p.n_adapters ? a : -1;
  }
  __syncthreads();
  const int whole = (int)(p.K / 8);
  for (int i0 = 0; i0 < n;) {
    const int a = ids[t0 + i0];
    int m = 1;
    while (i0 + m < n && ids[t0 + i0 + m] == a) ++m;
    if (a < 0 || j >= p.r) {
      if (lane < m) sh[i0 + lane][warp] = 0.0f;
    } else {
      float2 s2[R];
      const uint16_t* x[R];
#pragma unroll
      for (int i = 0; i < R; ++i) {
        s2[i] = make_float2(0.0f, 0.0f);
        x[i] = X + (row0 + t0 + i0 + min(i, m - 1)) * ldx;
      }
      const float scale = p.scale ? p.scale[a] : 1.0f;
      const uint16_t* w = A + ((int64_t)a * p.r + j) * lda;
#pragma unroll 4
      for (int c = lane; c < whole; c += 32) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(w + 8 * c));
#pragma unroll
        for (int i = 0; i < R; ++i) {  // rows past m are the last one again: a test here would hold up the loads
          const uint4 u = *reinterpret_cast<const uint4*>(x[i] + 8 * c);
          s2[i] = ffma2(bf16x2_to_f32(u.x), bf16x2_to_f32(v.x), s2[i]);
          s2[i] = ffma2(bf16x2_to_f32(u.y), bf16x2_to_f32(v.y), s2[i]);
          s2[i] = ffma2(bf16x2_to_f32(u.z), bf16x2_to_f32(v.z), s2[i]);
          s2[i] = ffma2(bf16x2_to_f32(u.w), bf16x2_to_f32(v.w), s2[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (i >= m) break;
        float s = s2[i].x + s2[i].y;
        for (int k = whole * 8 + lane; k < p.K; k += 32) s = fmaf(bf16_to_f32(x[i][k]), bf16_to_f32(w[k]), s);
        s = warp_add(s) * scale;
        if (lane == 0) sh[i0 + i][warp] = s;
      }
    }
    i0 += m;
  }
  __syncthreads();
  if (threadIdx.x < T && is_first(ids, threadIdx.x)) {
    const int j0 = blockIdx.y * 8, c = j0 / rk.cw;
    for (int i = 0; i < n; ++i) {
      const bool own = ids[threadIdx.x] == ids[t0 + i];
      for (int part = 0; part < rk.parts; ++part) {
        uint32_t w[4] = {0, 0, 0, 0};
        if (own)
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e >> 1] |= h_part(sh[i][e], part) << (16 * (e & 1));
        uint16_t* dst = rk.H + ((((row0 + threadIdx.x) * rk.parts + part) * rk.rc + c) * TN + t0 + i) * rk.cw + j0 % rk.cw;
        *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
}

struct LoraRows {
  LoraLinear p;
  RowsK rk;
  const uint16_t *X, *W, *B;
  int64_t ldx, ldw, ldb;
  int splits;
};
__device__ __noinline__ int spoilt_feature(const LoraRows& g, const int* ids, const int* list, int count, int64_t n) {
  for (int i = 0; i < count; ++i) {
    const uint16_t* b = g.B + ((int64_t)ids[list[i]] * g.p.N + n) * g.ldb;
    for (int c = 0; c < g.p.r; ++c)
      if ((b[c] & 0x7f80u) == 0x7f80u) return 1;
  }
  return 0;
}
__device__ __noinline__ float redo_value(const LoraRows& g, const int* ids, int64_t row0, int t, int64_t n, int TN) {
  const uint16_t *x = g.X + (row0 + t) * g.ldx, *w = g.W + n * g.ldw;
  float s = g.p.bias ? g.p.bias[n] : 0.0f;
  for (int64_t k = 0; k < g.p.K; ++k) s = fmaf(bf16_to_f32(x[k]), bf16_to_f32(w[k]), s);
  const int a = ids[t];
  if (a < 0) return s;
  int f = 0;
  while (ids[f] != a) ++f;
  const uint16_t* b = g.B + ((int64_t)a * g.p.N + n) * g.ldb;
  for (int c = 0; c < g.p.r; ++c)
    for (int part = 0; part < g.rk.parts; ++part) {
      const uint16_t hv =
          g.rk.H[((((row0 + f) * g.rk.parts + part) * g.rk.rc + c / g.rk.cw) * TN + t) * g.rk.cw + c % g.rk.cw];
      s = fmaf(bf16_to_f32(hv), bf16_to_f32(b[c]), s);
    }
  return s;
}

// The rows are the N of one MMA tile: D[n, t] = sum_k W[n, k] x[t, k] (+ the chunks of B and
// H) on tcgen05, 128 rows of W (the M of the MMA) per cluster. K blocks and chunks are split
// over the cluster's CTAs, so that every processor streams W; the CTAs' partial sums are read
// from their shared memory in rank order (the result does not depend on timing). Bound by the
// reads of W and the latency of the K loops: 48 rows, 9728 x 2560, 32 adapters of rank 32, 25.7 us
// with k_lora_down_rows (2.9 TB/s); one row, 2560 x 2560, 8.4 us.
template <int TN>
struct RowsCfg {
  static constexpr int W_BYTES = 128 * 128, X_BYTES = TN * 128, STAGE = W_BYTES + X_BYTES;
  static constexpr int STAGES = TN >= 64 ? 3 : 4;  // two CTAs fit a processor
  static_assert(STAGES * STAGE >= 128 * TN * 4, "partial sums reuse the stages");
  static constexpr int SMEM = 1024 + STAGES * STAGE;
};
constexpr int kRowThreads = 192;  // TMA warp, MMA warp, four epilogue warps
constexpr int kSumThreads = 256;  // k_lora_rows: eight

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t peer_addr(uint32_t addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}

template <int TN>
__global__ void __launch_bounds__(64 + kSumThreads, 2)
    k_lora_rows(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmH,
                const __grid_constant__ LoraRows g) {
  using C_ = RowsCfg<TN>;
  constexpr uint32_t IDESC = make_idesc(1u, 0, 0, 128, TN);
  constexpr uint32_t COLS = TN < 32 ? 32 : TN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* sums = reinterpret_cast<float*>(smem);  // [TN][128] after the MMAs: features side by side, for reads of whole lines
  __shared__ uint64_t full[C_::STAGES], empty[C_::STAGES], acc_full, list_full;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_words[kAbortWords(2 + kSumThreads / 32)], ids[kMaxRowsSmall], list[kMaxRowsSmall], in_warp[4], mixed;
  volatile int* abort_flag = abort_words;
  const LoraLinear& p = g.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, splits = g.splits;
  const int rank = blockIdx.x % splits, blocks = (int)((p.T + kMaxRowsSmall - 1) / kMaxRowsSmall);
  const int tile = blockIdx.x / splits / blocks;  // the blocks of rows side by side: W comes from L2 for all but one
  const int row0 = (int)(blockIdx.x / splits % blocks) * kMaxRowsSmall;
  const int T = min((int)p.T - row0, kMaxRowsSmall), per_stage = 64 / g.rk.cw, cwb = 2 * g.rk.cw;
  const int64_t n0 = (int64_t)tile * 128;
  const int kblocks = (int)((p.K + 63) / 64);
  const int kb0 = (int)((int64_t)kblocks * rank / splits), kb1 = (int)((int64_t)kblocks * (rank + 1) / splits);

  if (threadIdx.x == 0) {
    for (int s = 0; s < C_::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&acc_full, 1);
    mbar_init(&list_full, 1);
    for (int& w : abort_words) w = 0;
    mixed = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  // This CTA's chunks: those of the listed adapters whose number is rank modulo splits.
  auto my_chunks = [&]() { return (in_warp[0] * g.rk.per() - rank + splits - 1) / splits; };
  if (warp == 0) {
    {  // the whole warp: an elected lane issues
      RingPos at;
      int done = 0;
      bool ok = true;
      const uint32_t smem0 = smem_u32(smem), full0 = smem_u32(&full[0]);
      auto stage = [&](int bytes) {
        ok = mbar_wait_warp(&empty[at.slot], at.phase ^ 1u, abort_flag, p.err, kErrWaitEmpty);
        if (ok) {
          mbar_expect_tx_elect(full0 + (uint32_t)(at.slot * 8), (uint32_t)bytes);
          ++done;
        }
        return smem0 + (uint32_t)(at.slot * C_::STAGE);
      };
      for (int kb = kb0; kb < kb1; ++kb, at.next(C_::STAGES)) {
        const uint32_t st = stage(C_::STAGE);
        if (!ok) break;
        tma_load_2d_elect(st, &tmW, full0 + (uint32_t)(at.slot * 8), kb * 64, (int)n0);
        tma_load_2d_elect(st + C_::W_BYTES, &tmX, full0 + (uint32_t)(at.slot * 8), kb * 64, row0);
      }
      if (ok && g.rk.rc > 0) {
        ok = mbar_wait_warp(&list_full, 0, abort_flag, p.err, kErrWaitFull);
        asm volatile("griddepcontrol.wait;" ::: "memory");
        const int nq = ok ? my_chunks() : 0;
        for (int q0 = 0; q0 < nq; q0 += per_stage, at.next(C_::STAGES)) {
          const int n = min(per_stage, nq - q0);
          const uint32_t st = stage(n * (128 + TN) * cwb), bar = full0 + (uint32_t)(at.slot * 8);
          if (!ok) break;
          for (int i = 0; i < n; ++i) {
            const int q = (q0 + i) * splits + rank, f = list[q / g.rk.per()], sub = q % g.rk.per();
            tma_load_3d_elect(st + i * 128 * cwb, &tmB, bar, sub % g.rk.rc * g.rk.cw, (int)n0, ids[f]);
            tma_load_2d_elect(st + C_::W_BYTES + i * TN * cwb, &tmH, bar, 0, ((row0 + f) * g.rk.per() + sub) * TN);
          }
        }
      }
      if (!ok) {
        // Aborted: wait (bounded) for the loads in flight.
        const uint64_t t0 = globaltimer_ns();
        for (int i = max(0, done - C_::STAGES); i < done; ++i)
          while (!mbar_try_wait(&full[i % C_::STAGES], (i / C_::STAGES) & 1) && globaltimer_ns() - t0 < kWaitLimitNs) {
          }
      }
    }
  } else if (warp == 1) {
    {  // the whole warp: an elected lane issues
      RingPos at;
      bool ok = true;
      const uint64_t ad0 = sdesc_k_sw128(smem_u32(smem)), bd0 = sdesc_k_sw128(smem_u32(smem) + C_::W_BYTES);
      const uint32_t empty0 = smem_u32(&empty[0]);
      for (int kb = kb0; kb < kb1; ++kb, at.next(C_::STAGES)) {
        ok = mbar_wait_warp(&full[at.slot], at.phase, abort_flag, p.err, kErrWaitFull);
        if (!ok) break;
        tc_fence_after();
        const uint64_t off = (uint64_t)(at.slot * (C_::STAGE >> 4));
        umma4_elect(tmem, ad0 + off, bd0 + off, IDESC, kb > kb0, empty0 + 8 * at.slot);
      }
      if (ok && g.rk.rc > 0 && mbar_wait_warp(&list_full, 0, abort_flag, p.err, kErrWaitFull)) {
        const int nq = my_chunks();
        for (int q0 = 0; q0 < nq; q0 += per_stage, at.next(C_::STAGES)) {
          const int s = at.slot;
          if (!mbar_wait_warp(&full[s], at.phase, abort_flag, p.err, kErrWaitFull)) break;
          tc_fence_after();
          const uint32_t a0 = smem_u32(smem + s * C_::STAGE), b0 = a0 + C_::W_BYTES;
          for (int i = 0; i < min(per_stage, nq - q0); ++i)
            for (int k = 0; k < g.rk.cw / 16; ++k)
              umma_elect(tmem, sdesc_k(a0 + i * 128 * cwb + k * 32, cwb), sdesc_k(b0 + i * TN * cwb + k * 32, cwb), IDESC,
                          kb1 > kb0 || q0 + i + k > 0);
          umma_commit_elect(&empty[s]);
        }
      }
      umma_commit_elect(&acc_full);
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(&acc_full, 0))
        if (globaltimer_ns() - t0 > kWaitLimitNs) {
          if (lane == 0) atomicOr(p.err, kErrWaitDrain);
          break;
        }
    }
  } else {
    const int tid = threadIdx.x - 64;
    if (g.rk.rc > 0) {
      // The adapters among the rows, in the order of their first rows.
      if (tid < T) {
        const int a = p.row_adapter[row0 + tid];
        ids[tid] = a < p.n_adapters ? a : -1;
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
      const bool first = tid < T && is_first(ids, tid);
      if (tid < T && max(ids[tid], -1) != max(ids[0], -1)) mixed = 1;
      const uint32_t firsts = __ballot_sync(0xffffffffu, first);
      if (tid < 128 && lane == 0) in_warp[tid >> 5] = __popc(firsts);
      asm volatile("bar.sync 1, 256;" ::: "memory");
      int at = __popc(firsts & ((1u << lane) - 1)), all = 0;
      for (int w = 0; w < 4; ++w) {
        if (w < tid >> 5) at += in_warp[w];
        all += in_warp[w];
      }
      if (first) list[at] = tid;
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (tid == 0) {
        in_warp[0] = all;
        mbar_arrive(&list_full);
      }
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int q = warp & 3;  // TMEM lane quarter
    if (warp < 6 && mbar_wait_warp(&acc_full, 0, abort_flag, p.err, kErrWaitAccFull)) {
      __syncwarp();
      tc_fence_after();
      const bool any = kb1 > kb0 || (g.rk.rc > 0 && my_chunks() > 0);
      float* mine = sums + q * 32 + lane;
#pragma unroll
      for (int c = 0; c < TN; c += 16) {
        uint32_t v[16];
        tmem_ld_32x32b_x16(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)c, v);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) mine[(c + i) * 128] = any ? __uint_as_float(v[i]) : 0.0f;
      }
    }
  }
  tc_fence_before();
  __syncwarp();
  cluster_sync();  // every CTA's partial sums are in its shared memory
  if (warp >= 2) {
    // Rows [rank R, + R) of the tile, neighbouring threads neighbouring features: a warp reads
    // 128 contiguous bytes of a peer (16-byte reads of 32 different rows took ten times as
    // long). Four tokens of up to eight parts are in flight.
    const int tid = threadIdx.x - 64, R = 128 / splits, row = tid % R, step = kSumThreads / R;
    const int64_t n = n0 + rank * R + row;
    if (n < p.N) {
      const float bias = p.bias ? p.bias[n] : 0.0f;
      const uint32_t base = smem_u32(sums + rank * R + row);
      int spoilt = -1;  // whether an adapter's B is not finite in this feature
      for (int t0 = tid / R; t0 < T; t0 += 4 * step) {
        float y[4] = {bias, bias, bias, bias};
#pragma unroll
        for (int s0 = 0; s0 < 8; s0 += 4) {
          if (s0 >= splits) break;
          float part[4][4];
#pragma unroll
          for (int s = 0; s < 4; ++s)
            if (s0 + s < splits) {
              const uint32_t peer = peer_addr(base, s0 + s);
#pragma unroll
              for (int u = 0; u < 4; ++u) part[s][u] = ld_cluster_f32(peer + 512 * min(t0 + u * step, TN - 1));
            }
#pragma unroll
          for (int s = 0; s < 4; ++s)
            if (s0 + s < splits)
#pragma unroll
              for (int u = 0; u < 4; ++u) y[u] += part[s][u];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int t = t0 + u * step;
          if (t >= T) break;
          if (mixed && !(fabsf(y[u]) < INFINITY)) {
            // Zero times what is not finite in another row's adapter is NaN: such a value is
            // computed again without the tensor core.
            if (spoilt < 0) spoilt = spoilt_feature(g, ids, list, in_warp[0], n);
            if (spoilt) y[u] = redo_value(g, ids, row0, t, n, TN);
          }
          if (p.y_bf16)
            ((uint16_t*)p.Y)[(row0 + t) * p.ldy + n] = bf16_bits(y[u]);
          else
            ((float*)p.Y)[(row0 + t) * p.ldy + n] = y[u];
        }
      }
    }
  }
  __syncwarp();
  cluster_sync();  // peers have read this CTA's sums
  if (warp == 1) tmem_dealloc(tmem, COLS);
}

// ------------------------------------------------------------------------------------
// Operands as TMA reads them: 16-byte rows of bf16, copied into the workspace where the
// caller's are not.
// ------------------------------------------------------------------------------------
struct Operands {
  bool pack_x, pack_w, pack_a, pack_b;
  int64_t Kp, rb;  // pitches of packed rows
  size_t x_at, w_at, a_at, b_at, h_at;
};
Operands lay_out(const LoraLinear& p) {
  Operands o{};
  o.Kp = round_up(p.K, 8);
  o.rb = round_up(std::max<int64_t>(p.r, 1), 8);
  const bool adapters = p.n_adapters > 0 && p.r > 0;
  o.pack_x = !p.x_bf16 || !aligned16(p.X) || p.ldx % 8 != 0;
  o.pack_w = !aligned16(p.W) || p.ldw % 8 != 0;
  o.pack_a = adapters && (!aligned16(p.A) || p.lda % 8 != 0);
  o.pack_b = adapters && (!aligned16(p.B) || p.ldb % 8 != 0);
  size_t at = 0;
  auto take = [&](bool need, int64_t rows, int64_t pitch) {
    const size_t here = at;
    if (need) at += align256((size_t)(rows * pitch) * 2);
    return here;
  };
  o.x_at = take(o.pack_x, p.T, o.Kp);
  o.w_at = take(o.pack_w, p.N, o.Kp);
  o.a_at = take(o.pack_a, p.n_adapters * p.r, o.Kp);
  o.b_at = take(o.pack_b, p.n_adapters * p.N, o.rb);
  o.h_at = at;
  return o;
}

// Up to four matrices in one launch: rows of `cols` values, bf16 or fp32 (rounded to bf16),
// to rows of `pitch` bf16, zero past cols. Eight values a thread: a 16-byte store of what lies
// in two aligned 16-byte words (bf16), or eight loads where those would leave the matrix.
struct PackOne {
  const void* src;
  uint16_t* dst;
  int64_t ld, rows;
  int cols, pitch, f32;
};
struct PackAll {
  PackOne m[4];
  int64_t end[4];  // chunks up to and with matrix i
  int n;
};
__global__ void __launch_bounds__(256) k_lora_pack(const __grid_constant__ PackAll all) {
  for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < all.end[all.n - 1]; u += (int64_t)gridDim.x * 256) {
    int i = 0;
    while (u >= all.end[i]) ++i;
    const PackOne& m = all.m[i];
    const int64_t x = i ? u - all.end[i - 1] : u;
    const int per = m.pitch / 8;
    const int64_t r = x / per;
    const int c = (int)(x - r * per) * 8;
    uint32_t w[4] = {0, 0, 0, 0};
    const uintptr_t from = reinterpret_cast<uintptr_t>(m.src) + (uintptr_t)(r * m.ld + c) * 2, word = from & ~uintptr_t(15);
    if (!m.f32 && c + 8 <= m.cols && word >= reinterpret_cast<uintptr_t>(m.src) &&
        word + 32 <= reinterpret_cast<uintptr_t>(m.src) + (uintptr_t)((m.rows - 1) * m.ld + m.cols) * 2) {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(word)), b = __ldg(reinterpret_cast<const uint4*>(word) + 1);
      const uint32_t v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
      const int skip = (int)(from & 15) >> 2, half = (int)(from & 2) * 8;  // whole words, and 16 bits of one
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t lo = v[i], hi = v[i + 1];
#pragma unroll
        for (int k = 1; k < 4; ++k)
          if (skip == k) {
            lo = v[i + k];
            hi = i + k + 1 < 8 ? v[i + k + 1] : 0u;
          }
        w[i] = __funnelshift_r(lo, hi, half);
      }
      *reinterpret_cast<uint4*>(m.dst + r * m.pitch + c) = make_uint4(w[0], w[1], w[2], w[3]);
      continue;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < m.cols) {
        const int64_t at = r * m.ld + c + e;
        const uint32_t v = m.f32 ? bf16_bits(((const float*)m.src)[at]) : ((const uint16_t*)m.src)[at];
        w[e >> 1] |= v << (16 * (e & 1));
      }
    *reinterpret_cast<uint4*>(m.dst + r * m.pitch + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// CTAs of k_lora_rows that run at a time in clusters of `splits`: two a processor, but clusters of
// four and eight leave some processors of a group out (132 and 120 of 148 have one). 296 CTAs in
// clusters of four ran in two waves: 48 rows, 9472 x 2560, 33 us instead of 25.6.
template <int TN>
int64_t row_units(int splits) {
  static int64_t units[64][9] = {};
  DeviceContext& c = ctx();
  if (!units[c.device][splits]) {
    using C_ = RowsCfg<TN>;
    constexpr int kOne = 120 * 1024;  // shared memory that one CTA a processor has, for the query
    static_assert(C_::SMEM <= kOne && 2 * (C_::SMEM + 8192) <= kMaxSmem, "two CTAs a processor");
    check_cuda(cudaFuncSetAttribute(k_lora_rows<TN>, cudaFuncAttributeMaxDynamicSharedMemorySize, kOne),
               "cudaFuncSetAttribute(linear_lora)");
    // The default carve-out would hold one CTA a processor, and the rest would run after it.
    check_cuda(cudaFuncSetAttribute(k_lora_rows<TN>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                    cudaSharedmemCarveoutMaxShared),
               "cudaFuncSetAttribute(linear_lora)");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)splits);
    cfg.blockDim = dim3(64 + kSumThreads);
    cfg.dynamicSmemBytes = kOne;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)splits;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int fit = 0;
    check_cuda(cudaOccupancyMaxActiveClusters(&fit, k_lora_rows<TN>, &cfg), "cudaOccupancyMaxActiveClusters(linear_lora)");
    units[c.device][splits] = std::max<int64_t>(1, 2 * (int64_t)fit * splits);
  }
  return units[c.device][splits];
}
// Four rows to a CTA of the down product where that leaves every processor six: 384 rows of rank
// 128, 3840 x 3840, 59 us instead of 71 with two requests, 77 instead of 81 with 64. With fewer
// CTAs a chain of four rows is slower (160 rows of rank 16: 29 instead of 26).
bool by_runs(const LoraLinear& p) {
  return (p.T + kRunRows - 1) / kRunRows * (round_up(p.r, chunk_width(p.r)) / 8) >= 6 * (int64_t)ctx().num_sms;
}
// K splits of k_lora_rows, while all CTAs run at a time, of two K blocks at least.
template <int TN>
int row_splits(const LoraLinear& p) {
  const int64_t tiles = (p.N + 127) / 128 * ((p.T + kMaxRowsSmall - 1) / kMaxRowsSmall), kblocks = (p.K + 63) / 64;
  int splits = 1;
  while (splits < 8 && kblocks >= 4 * splits && tiles * splits * 2 <= row_units<TN>(splits * 2)) splits *= 2;
  row_units<TN>(splits);  // the kernel's attributes are set
  return splits;
}
int rows_tile(int64_t T) { return T <= 16 ? 16 : T <= 32 ? 32 : T <= 64 ? 64 : 128; }
RowsK lay_out_rows(const LoraLinear& p, uint8_t* at, size_t* bytes) {
  RowsK k{};
  k.cw = 64;
  *bytes = 0;
  if (p.n_adapters <= 0 || p.r <= 0) return k;
  k.H = reinterpret_cast<uint16_t*>(at);
  k.cw = chunk_width(p.r);
  k.rc = (int)((p.r + k.cw - 1) / k.cw);
  k.parts = p.y_bf16 ? 1 : 2;
  *bytes = align256((size_t)(p.T * k.per() * rows_tile(p.T) * k.cw) * 2);
  return k;
}

void map_2d(CUtensorMap* m, const void* x, int64_t k, int64_t rows, int64_t ld, int box_k, int box_rows,
            CUtensorMapSwizzle sw) {
  const uint64_t dims[2] = {(uint64_t)k, (uint64_t)rows};
  const uint64_t str[1] = {(uint64_t)ld * 2};
  const uint32_t box[2] = {(uint32_t)box_k, (uint32_t)box_rows};
  encode_tmap(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, x, dims, str, box, sw);
}
// `rows` x `cols` of every adapter, one adapter at a time.
void map_adapters(CUtensorMap* m, const void* x, int64_t cols, int64_t rows, int64_t n, int64_t ld, int box_cols, int box_rows,
                  CUtensorMapSwizzle sw) {
  const uint64_t dims[3] = {(uint64_t)cols, (uint64_t)rows, (uint64_t)n};
  const uint64_t str[2] = {(uint64_t)ld * 2, (uint64_t)(rows * ld) * 2};
  const uint32_t box[3] = {(uint32_t)box_cols, (uint32_t)box_rows, 1};
  encode_tmap(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, x, dims, str, box, sw);
}

template <int TN>
void launch_rows(LoraRows g) {
  using C_ = RowsCfg<TN>;
  DeviceContext& c = ctx();
  const LoraLinear& p = g.p;
  const bool adapters = g.rk.rc > 0;
  CUtensorMap tw, tx, tb, th;
  map_2d(&tw, g.W, p.K, p.N, g.ldw, 64, 128, CU_TENSOR_MAP_SWIZZLE_128B);
  map_2d(&tx, g.X, p.K, p.T, g.ldx, 64, TN, CU_TENSOR_MAP_SWIZZLE_128B);
  if (adapters) {
    map_adapters(&tb, g.B, p.r, p.N, p.n_adapters, g.ldb, g.rk.cw, 128, swizzle_of(g.rk.cw));
    map_2d(&th, g.rk.H, g.rk.cw, p.T * g.rk.per() * TN, g.rk.cw, g.rk.cw, TN, swizzle_of(g.rk.cw));
  } else {
    tb = th = tx;  // no chunk is read
  }
  const int64_t tiles = (p.N + 127) / 128 * ((p.T + kMaxRowsSmall - 1) / kMaxRowsSmall);
  g.splits = row_splits<TN>(p);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(tiles * g.splits));
  cfg.blockDim = dim3(64 + kSumThreads);
  cfg.dynamicSmemBytes = C_::SMEM;
  cfg.stream = c.stream;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)g.splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = adapters ? 2 : 1;  // only k_lora_down_rows or k_lora_down_runs may be overtaken
  check_cuda(cudaLaunchKernelEx(&cfg, k_lora_rows<TN>, tw, tx, tb, th, (const LoraRows)g), "linear_lora");
  check_launch("linear_lora");
}

// ------------------------------------------------------------------------------------
// Many rows: Y = [X | H] [W | B]^T as one GEMM.
// ------------------------------------------------------------------------------------
constexpr int kGroup = 256;  // rows that share a list of adapters and a block of H
constexpr int kHash = 512;

struct GroupList {
  int count;             // distinct adapters of the rows
  int mixed;             // rows of different adapters, or some of none
  int adapter[kGroup];   // in the order of their first rows
  int16_t slot[kGroup];  // each row's place in that order, -1: no adapter
};
// H: [groups][q_max][kGroup][cw] bf16, chunk q = (slot * parts + part) * rc + c of a group.
struct LoraK {
  GroupList* lists;
  int* done;     // warps of k_lora_gemm that have stored their part of H
  int* arrived;  // [groups][8]: K splits that have stored their part, for 32 rows each
  float4* part;  // [32-row blocks][ksplit][rc cw / 4][32]: the splits' parts of the rows' own h, for whole lines
  int ksplit;
  uint16_t* H;
  int cw, rc, parts, q_max;
  __host__ __device__ int chunks(int count) const { return count * parts * rc; }
};

// The distinct adapters of a group's rows, through a hash table.
__global__ void __launch_bounds__(kGroup) k_lora_lists(const LoraLinear p, const LoraK lk, int64_t row0, int64_t rows) {
  __shared__ int hash_key[kHash], hash_row[kHash], first_at[kGroup], in_warp[kGroup / 32], mixed;
  const int i = threadIdx.x, lane = i & 31, warp = i >> 5;
  const int64_t t = (int64_t)blockIdx.x * kGroup + i;
  GroupList& L = lk.lists[blockIdx.x];
  for (int h = i; h < kHash; h += kGroup) {
    hash_key[h] = -1;
    hash_row[h] = kGroup;
  }
  if (i == 0) mixed = 0;
  if (i == 0 && blockIdx.x == 0) *lk.done = 0;
  if (i < 8) lk.arrived[blockIdx.x * 8 + i] = 0;
  int a = t < rows ? p.row_adapter[row0 + t] : -1;
  if (a >= p.n_adapters) {
    atomicOr(p.err, kErrBadIndex);
    a = -1;
  }
  a = max(a, -1);
  __syncthreads();
  uint32_t at = ((uint32_t)a * 2654435761u) >> 23;
  if (a >= 0) {
    for (;; at = (at + 1) % kHash) {
      const int k = atomicCAS(&hash_key[at], -1, a);
      if (k == -1 || k == a) break;  // at most kGroup of kHash places are taken
    }
    atomicMin(&hash_row[at], i);
  }
  first_at[i] = a;
  __syncthreads();
  if (t < rows && a != first_at[0]) mixed = 1;
  const int f = a >= 0 ? hash_row[at] : -1;  // the first row of this adapter
  const bool first = f == i;
  const uint32_t firsts = __ballot_sync(0xffffffffu, first);
  if (lane == 0) in_warp[warp] = __popc(firsts);
  __syncthreads();
  int place = __popc(firsts & ((1u << lane) - 1)), all = 0;
  for (int w = 0; w < kGroup / 32; ++w) {
    if (w < warp) place += in_warp[w];
    all += in_warp[w];
  }
  if (first) {
    first_at[i] = place;
    L.adapter[place] = a;
  }
  __syncthreads();
  L.slot[i] = (int16_t)(a >= 0 ? first_at[f] : -1);
  if (i == 0) {
    L.count = all;
    L.mixed = mixed;
  }
}

__device__ __forceinline__ int ld_acquire(const int* p) {
  int v;
  asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
// Waits (bounded, a whole warp) until *flag, counted up by other CTAs of this launch, reaches want.
__device__ __forceinline__ bool wait_count(const int* flag, int want, volatile int* abort_flag, int* err) {
  return wait_warp([&]() { return ld_acquire(flag) >= want; }, abort_flag, err, kErrWaitFull);
}

// The elements of one 32-column chunk of a warp's rows whose sums are not finite, again
// without the tensor core where an adapter of another row may have caused it: in a group of
// several adapters, zero times an infinity or NaN of another adapter's B is NaN.
__device__ __noinline__ void redo_chunk(const LoraLinear& p, const LoraK& lk, const uint16_t* X, int64_t ldx,
                                        const uint16_t* W, int64_t ldw, const uint16_t* B, int64_t ldb, int64_t row0,
                                        int local, int64_t col0, uint32_t bad) {
  const int lane = threadIdx.x & 31;
  const GroupList& L = lk.lists[local / kGroup];
  ld_acquire(lk.done);  // H is complete: the tile's MMAs have read it
  for (uint32_t cols = __reduce_or_sync(0xffffffffu, bad); cols; cols &= cols - 1) {
    const int j = __ffs(cols) - 1;
    const int64_t n = col0 + j;
    bool hit = false;
    for (int i = lane; i < L.count * (int)p.r; i += 32) {
      const uint16_t b = B[((int64_t)L.adapter[i / p.r] * p.N + n) * ldb + i % p.r];
      hit |= (b & 0x7f80u) == 0x7f80u;
    }
    if (!__any_sync(0xffffffffu, hit)) continue;
    for (uint32_t todo = __ballot_sync(0xffffffffu, bad >> j & 1); todo; todo &= todo - 1) {
      const int t = __shfl_sync(0xffffffffu, local, __ffs(todo) - 1);
      const uint16_t* x = X + (row0 + t) * ldx;
      const uint16_t* w = W + n * ldw;
      float s = 0.0f;
      for (int64_t k = lane; k < p.K; k += 32) s = fmaf(bf16_to_f32(x[k]), bf16_to_f32(w[k]), s);
      const int sl = L.slot[t % kGroup];
      if (sl >= 0) {
        const int a = L.adapter[sl];
        const uint16_t* b = B + ((int64_t)a * p.N + n) * ldb;
        for (int c = lane; c < p.r; c += 32)
          for (int part = 0; part < lk.parts; ++part) {
            const int q = (sl * lk.parts + part) * lk.rc + c / lk.cw;
            const uint16_t hv = lk.H[(((int64_t)(t / kGroup) * lk.q_max + q) * kGroup + t % kGroup) * lk.cw + c % lk.cw];
            s = fmaf(bf16_to_f32(hv), bf16_to_f32(b[c]), s);
          }
      }
      s = warp_add(s) + (p.bias ? p.bias[n] : 0.0f);
      if (lane == 0) {
        if (p.y_bf16)
          ((uint16_t*)p.Y)[(row0 + t) * p.ldy + n] = bf16_bits(s);
        else
          ((float*)p.Y)[(row0 + t) * p.ldy + n] = s;
      }
      __syncwarp();
    }
  }
}

// The GEMM: persistent, TMA warp / MMA warp / four epilogue warps, accumulators double
// buffered in TMEM, as gemm_tc.cu. PAIR: clusters of two CTAs share 256 x BN tiles
// (cta_group::2 MMAs, each CTA loads its 128 rows of X and its half of W's rows); else
// 128 x BN tiles.
//
// The first items of the launch, one per row of tiles, make H: X A_a^T for the adapters of
// the group's list, their ranks side by side as the columns of an accumulator (BN at a
// time), K split over several items where there are more units than rows of tiles; the
// epilogue keeps each row's own, scaled, and counts up `done`. The other items are
// the tiles of Y: the K blocks of X and W first, then, once `done` says that H is complete,
// the chunks of H and B, 64 / cw of them a stage. Every unit runs its items of the first kind
// before those of the second, only the second kind waits, and a cooperative launch has all units
// resident, so the wait ends. In a kernel of its
// own the adapter product cost a pass over X that nothing overlapped: 827 us at 33792 x 3840 x
// 3840 with one adapter of rank 16, now 692 (634 without adapters; 1440 TFLOP/s, torch.matmul 650).
// Bound by the tensor core under the power limit there, by the epilogue where K <= 400.
template <int BN, bool PAIR>
struct LoraGemmCfg {
  static constexpr int B_ROWS = PAIR ? BN / 2 : BN;
  static constexpr int A_BYTES = 128 * 128, B_BYTES = B_ROWS * 128, STAGE = A_BYTES + B_BYTES;
  static constexpr int STG_BYTES = 4 * 2 * 32 * 128;  // two 32 x 32 blocks of Y per epilogue warp
  static constexpr int FIT = (kMaxSmem - 1024 - STG_BYTES - 512 - 16 * BN) / STAGE;  // barriers, bias
  static constexpr int STAGES = FIT > 8 ? 8 : FIT;
  static constexpr int SMEM = 1024 + STAGES * STAGE + STG_BYTES;
  static constexpr uint32_t COLS = 2 * BN <= 128 ? 128 : 2 * BN <= 256 ? 256 : 512;
};
struct LoraGemm {
  LoraLinear p;
  LoraK lk;
  const uint16_t *X, *W, *B;
  int64_t ldx, ldw, ldb;
  int64_t row0, rows;
  int m_tiles, n_tiles, k_blocks;
  int y_tma;
  __device__ int down_items() const { return lk.q_max ? m_tiles * lk.ksplit : 0; }
};
// Columns of the accumulator that `n` ranks take: a pair's MMA has a multiple of 32.
template <int CTAS>
__device__ __forceinline__ int down_columns(int n) {
  return CTAS == 2 ? (n + 31) / 32 * 32 : n;
}
__device__ __forceinline__ int split_begin(int k_blocks, int splits, int s) { return (int)((int64_t)k_blocks * s / splits); }
constexpr int kGroupM = 16;  // M tiles walked together, for reuse in L2
__device__ __forceinline__ void tile_at(int t, int m_tiles, int n_tiles, int& mb, int& nb) {
  const int per = kGroupM * n_tiles, g = t / per, first = g * kGroupM;
  const int gs = min(m_tiles - first, kGroupM), r = t - g * per;
  mb = first + r % gs;
  nb = r / gs;
}

template <int BN, bool PAIR>
__global__ void __launch_bounds__(kRowThreads, 1)
    k_lora_gemm(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                const __grid_constant__ CUtensorMap tmH, const __grid_constant__ CUtensorMap tmB,
                const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmY,
                const __grid_constant__ LoraGemm g) {
  using C_ = LoraGemmCfg<BN, PAIR>;
  constexpr int STAGES = C_::STAGES, CTAS = PAIR ? 2 : 1;
  constexpr uint32_t IDESC = make_idesc(1u, 0, 0, PAIR ? 256 : 128, BN);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[STAGES], empty[STAGES], acc_full[2], acc_empty[2], drain;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_words[kAbortWords(kRowThreads / 32)], pass_ids[BN / 16];  // adapters of the chunks of a pass
  __shared__ float4 sbias[4][BN / 4];            // bias of the tile's columns, one copy an epilogue warp
  volatile int* abort_flag = abort_words;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0;
  const int unit = (int)blockIdx.x / CTAS, units = (int)gridDim.x / CTAS;
  const int downs = g.down_items(), items = downs + g.m_tiles * g.n_tiles;
  int* err = g.p.err;
  const int cw = g.lk.cw, cwb = 2 * cw, per_stage = 64 / cw, per_pass = BN / cw;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 4 * CTAS);
    }
    mbar_init(&drain, 1);
    for (int& w : abort_words) w = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmH);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(&tmem_slot, C_::COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(&tmem_slot, C_::COLS);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // both CTAs' barriers exist before any signal crosses
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  // The list of tile row mb's group (without adapters there is none), its adapters and the
  // passes over them that make H.
  auto list_of = [&](int mb) { return g.lk.lists + (PAIR ? mb : mb >> 1); };
  auto count_of = [&](int mb) { return g.lk.q_max ? __ldcg(&list_of(mb)->count) : 0; };
  auto passes_of = [&](int mb) { return (count_of(mb) * g.lk.rc + per_pass - 1) / per_pass; };

  if (warp == 0) {
    {  // the whole warp: an elected lane issues
      const uint32_t smem0 = smem_u32(smem), full_own = smem_u32(&full[0]);
      const uint32_t full0 = PAIR ? mapa_shared(&full[0], 0) : full_own;  // the leader's
      RingPos at;
      int done = 0;  // stages filled
      bool ok = true, have_h = false;
      auto stage = [&](int bytes, uint32_t& st) {
        ok = mbar_wait_warp(&empty[at.slot], at.phase ^ 1u, abort_flag, err, kErrWaitEmpty);
        if (!ok) return false;
        st = smem0 + (uint32_t)(at.slot * C_::STAGE);
        if (rank == 0) mbar_expect_tx_elect(full_own + (uint32_t)(at.slot * 8), (uint32_t)(CTAS * bytes));
        ++done;
        return true;
      };
      auto load2 = [&](uint32_t dst, const CUtensorMap* m, int x, int y) {
        if constexpr (PAIR)
          tma_load_2d_pair_elect(dst, m, full0 + (uint32_t)(at.slot * 8), x, y);
        else
          tma_load_2d_elect(dst, m, full0 + (uint32_t)(at.slot * 8), x, y);
      };
      auto load3 = [&](uint32_t dst, const CUtensorMap* m, int x, int y, int z) {
        if constexpr (PAIR)
          tma_load_3d_pair_elect(dst, m, full0 + (uint32_t)(at.slot * 8), x, y, z);
        else
          tma_load_3d_elect(dst, m, full0 + (uint32_t)(at.slot * 8), x, y, z);
      };
      for (int it = unit; it < items && ok; it += units) {
        uint32_t st;
        if (it < downs) {
          const int mb = it % g.m_tiles, sp = it / g.m_tiles;
          const int y0 = (mb * CTAS + (int)rank) * 128, nch = count_of(mb) * g.lk.rc;
          const int kb0 = split_begin(g.k_blocks, g.lk.ksplit, sp), kb1 = split_begin(g.k_blocks, g.lk.ksplit, sp + 1);
          for (int c0 = 0; c0 < nch && ok; c0 += per_pass) {
            const int n = min(per_pass, nch - c0);
            __syncwarp();
            if (lane < n) pass_ids[lane] = __ldcg(&list_of(mb)->adapter[(c0 + lane) / g.lk.rc]);
            __syncwarp();
            const int c_first = c0 % g.lk.rc;
            for (int kb = kb0; kb < kb1; ++kb, at.next(STAGES)) {
              if (!stage(C_::A_BYTES + n * (cw / CTAS) * 128, st)) break;
              load2(st, &tmX, kb * 64, (int)g.row0 + y0);
              for (int i = 0, c = c_first; i < n; ++i, c = c + 1 == g.lk.rc ? 0 : c + 1)
                load3(st + C_::A_BYTES + i * (cw / CTAS) * 128, &tmA, kb * 64, c * cw + (int)rank * (cw / CTAS), pass_ids[i]);
            }
          }
          continue;
        }
        int mb, nb;
        tile_at(it - downs, g.m_tiles, g.n_tiles, mb, nb);
        const int y0 = (mb * CTAS + (int)rank) * 128, n0 = nb * BN + (int)rank * C_::B_ROWS;
        // Read ahead: the loads arrive while the K blocks are on their way.
        const int count = count_of(mb), adapter0 = downs ? __ldcg(&list_of(mb)->adapter[0]) : 0;
        const int adapter1 = downs ? __ldcg(&list_of(mb)->adapter[1]) : 0;
        for (int kb = 0; kb < g.k_blocks; ++kb, at.next(STAGES)) {
          if (!stage(C_::STAGE, st)) break;
          load2(st, &tmX, kb * 64, (int)g.row0 + y0);
          load2(st + C_::A_BYTES, &tmW, kb * 64, n0);
        }
        if (!ok) break;
        if (!downs) continue;
        const int nq = g.lk.chunks(count), group = y0 / kGroup;
        if (!have_h) {
          ok = wait_count(g.lk.done, 4 * CTAS * g.m_tiles, abort_flag, err);
          if (!ok) break;
          asm volatile("fence.proxy.async;" ::: "memory");  // H was stored by other CTAs, TMA reads it
          have_h = true;
        }
        for (int q0 = 0; q0 < nq; q0 += per_stage, at.next(STAGES)) {
          const int n = min(per_stage, nq - q0);
          if (!stage(n * (128 + C_::B_ROWS) * cwb, st)) break;
          for (int i = 0; i < n; ++i) {
            const int q = q0 + i, c = q % g.lk.rc, sl = q / (g.lk.rc * g.lk.parts);
            load2(st + i * 128 * cwb, &tmH, 0, (group * g.lk.q_max + q) * kGroup + y0 % kGroup);
            load3(st + C_::A_BYTES + i * C_::B_ROWS * cwb, &tmB, c * cw, n0,
                  sl == 0 ? adapter0 : sl == 1 ? adapter1 : __ldcg(&list_of(mb)->adapter[sl]));
          }
        }
      }
      if (!ok && rank == 0) {
        // Aborted: wait (bounded) for the loads in flight (a pair's all complete here).
        const uint64_t t0 = globaltimer_ns();
        for (int i = max(0, done - STAGES); i < done; ++i)
          while (!mbar_try_wait(&full[i % STAGES], (i / STAGES) & 1) && globaltimer_ns() - t0 < kWaitLimitNs) {
          }
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {  // the whole warp: an elected lane issues
      RingPos at;
      int n = 0;
      const uint64_t ad0 = sdesc_k_sw128(smem_u32(smem)), bd0 = sdesc_k_sw128(smem_u32(smem) + C_::A_BYTES);
      const uint32_t empty0 = smem_u32(&empty[0]);
      bool ok = true;
      auto commit = [&](uint64_t* bar) {
        if constexpr (PAIR)
          umma_commit_pair_elect(bar, 0x3);
        else
          umma_commit_elect(bar);
      };
      for (int it = unit; it < items && ok; it += units) {
        const bool down = it < downs;
        int mb = it % g.m_tiles, nb = 0, nch = 0, passes = 1, kb0 = 0, kb1 = g.k_blocks;
        if (down) {
          nch = count_of(mb) * g.lk.rc;
          passes = passes_of(mb);
          kb0 = split_begin(g.k_blocks, g.lk.ksplit, it / g.m_tiles);
          kb1 = split_begin(g.k_blocks, g.lk.ksplit, it / g.m_tiles + 1);
        } else {
          tile_at(it - downs, g.m_tiles, g.n_tiles, mb, nb);
        }
        const int count = count_of(mb);
        for (int ps = 0; ps < passes; ++ps, ++n) {
          const int acc = n & 1;
          ok = mbar_wait_warp(&acc_empty[acc], ((n >> 1) & 1) ^ 1u, abort_flag, err, kErrWaitAccEmpty);
          if (!ok) break;
          tc_fence_after();
          const uint32_t d = tmem + (uint32_t)(acc * BN);
          // A pair's MMA takes a multiple of 32 columns; what the last ones hold is not read.
          const int N = down ? down_columns<CTAS>(min(per_pass, nch - ps * per_pass) * cw) : BN;
          const uint32_t idesc = down ? make_idesc(1u, 0, 0, 128 * CTAS, (uint32_t)N) : IDESC;
          const uint32_t d_step = 4 * N <= BN ? (uint32_t)N : 0;  // four accumulators where they fit
          for (int kb = kb0; kb < kb1; ++kb, at.next(STAGES)) {
            ok = mbar_wait_warp(&full[at.slot], at.phase, abort_flag, err, kErrWaitFull);
            if (!ok) break;
            tc_fence_after();
            const uint64_t off = (uint64_t)(at.slot * (C_::STAGE >> 4));
            if constexpr (PAIR)
              umma4_pair_elect(d, ad0 + off, bd0 + off, idesc, kb != kb0, empty0 + 8 * at.slot, d_step);
            else
              umma4_elect(d, ad0 + off, bd0 + off, idesc, kb != kb0, empty0 + 8 * at.slot, d_step);
          }
          if (!ok) break;
          if (!down && downs) {
            const int nq = g.lk.chunks(count);
            for (int q0 = 0; q0 < nq; q0 += per_stage, at.next(STAGES)) {
              const int s = at.slot;
              ok = mbar_wait_warp(&full[s], at.phase, abort_flag, err, kErrWaitFull);
              if (!ok) break;
              tc_fence_after();
              const uint32_t a0 = smem_u32(smem + s * C_::STAGE), b0 = a0 + C_::A_BYTES;
              for (int i = 0; i < min(per_stage, nq - q0); ++i)
                for (int k = 0; k < cw / 16; ++k) {
                  const uint64_t ad = sdesc_k(a0 + i * 128 * cwb + k * 32, cwb);
                  const uint64_t bd = sdesc_k(b0 + i * C_::B_ROWS * cwb + k * 32, cwb);
                  if constexpr (PAIR)
                    umma_pair_elect(d, ad, bd, IDESC, 1u);
                  else
                    umma_elect(d, ad, bd, IDESC, 1u);
                }
              commit(&empty[s]);
            }
            if (!ok) break;
          }
          commit(&acc_full[acc]);
        }
      }
      commit(&drain);
    }
    if (lane == 0) {
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(&drain, 0))
        if (globaltimer_ns() - t0 > kWaitLimitNs) {
          atomicOr(err, kErrWaitDrain);
          break;
        }
    }
  } else {
    const int q = warp & 3;
    const uint32_t acc_empty0 = PAIR ? mapa_shared(&acc_empty[0], 0) : 0;
    uint8_t* const stg = smem + STAGES * C_::STAGE + q * 8192;
    uint8_t* buf = stg;
    int n = 0;
    bool ok = true;
    auto release = [&](int acc) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR)
          mbar_arrive_cluster(acc_empty0 + (uint32_t)(acc * 8));
        else
          mbar_arrive(&acc_empty[acc]);
      }
    };
    for (int it = unit; it < items && ok; it += units) {
      if (it < downs) {
        // H of this warp's rows: their own adapter's columns, zeros in the others' chunks.
        const int mb = it % g.m_tiles, sp = it / g.m_tiles, nch = count_of(mb) * g.lk.rc;
        const int me = (mb * CTAS + (int)rank) * 128 % kGroup + q * 32 + lane;
        const GroupList* L = list_of(mb);
        const int mine = L->slot[me];
        const float scale = mine >= 0 && g.p.scale ? g.p.scale[L->adapter[mine]] : 1.0f;
        uint16_t* rowH = g.lk.H + ((int64_t)(L - g.lk.lists) * g.lk.q_max * kGroup + me) * cw;
        const int rp = g.lk.rc * cw;
        float4* part = g.lk.part + ((int64_t)(mb * CTAS + (int)rank) * 4 + q) * g.lk.ksplit * (rp / 4) * 32 + lane;
        auto store_h = [&](int sl, int c, int e0, const float (&v)[8]) {
          for (int pt = 0; pt < g.lk.parts; ++pt) {
            uint32_t w[4] = {0, 0, 0, 0};
            if (sl == mine) {
#pragma unroll
              for (int e = 0; e < 8; ++e) w[e >> 1] |= h_part(v[e] * scale, pt) << (16 * (e & 1));
            }
            const int64_t qi = (int64_t)(sl * g.lk.parts + pt) * g.lk.rc + c;
            *reinterpret_cast<uint4*>(rowH + qi * kGroup * cw + e0) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        };
        for (int c0 = 0; c0 < nch; c0 += per_pass, ++n) {
          const int acc = n & 1, used = min(per_pass, nch - c0), N = down_columns<CTAS>(used * cw);
          ok = mbar_wait_warp(&acc_full[acc], (n >> 1) & 1, abort_flag, err, kErrWaitAccFull);
          if (!ok) break;
          tc_fence_after();
          const uint32_t base = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * BN);
          for (int i = 0; i < used; ++i) {
            const int sl = (c0 + i) / g.lk.rc, c = (c0 + i) % g.lk.rc;
            if (g.lk.ksplit > 1 && !__any_sync(0xffffffffu, sl == mine)) continue;
            for (int e0 = 0; e0 < cw; e0 += 8) {
              // A pair's two CTAs hold the two halves of each chunk's ranks.
              const int half = e0 >= cw / CTAS;
              const int col = half * (N / CTAS) + i * (cw / CTAS) + e0 - half * (cw / CTAS);
              uint32_t r[4][8];
              float v[8];
              __syncwarp();
              tmem_ld_32x32b_x8(base + (uint32_t)col, r[0]);
              if (4 * N <= BN) {  // four accumulators
#pragma unroll
                for (int a = 1; a < 4; ++a) tmem_ld_32x32b_x8(base + (uint32_t)(col + a * N), r[a]);
              }
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                v[e] = __uint_as_float(r[0][e]);
                if (4 * N <= BN)
                  v[e] = (v[e] + __uint_as_float(r[1][e])) + (__uint_as_float(r[2][e]) + __uint_as_float(r[3][e]));
              }
              if (g.lk.ksplit == 1) {
                store_h(sl, c, e0, v);
              } else if (sl == mine) {
                float4* dst = part + (sp * rp + c * cw + e0) / 4 * 32;
                dst[0] = make_float4(v[0], v[1], v[2], v[3]);
                dst[32] = make_float4(v[4], v[5], v[6], v[7]);
              }
            }
          }
          release(acc);
        }
        bool last = true;
        if (g.lk.ksplit > 1) {
          // The last split to arrive adds the parts in their order.
          __threadfence();
          __syncwarp();
          int before = 0;
          if (lane == 0) before = atomicAdd(&g.lk.arrived[(mb * CTAS + (int)rank) * 4 + q], 1);
          last = __shfl_sync(0xffffffffu, before, 0) == g.lk.ksplit - 1;
          __threadfence();
          if (last)
            for (int x = 0; x < rp; x += 8) {
              float4 a[8], b[8];  // this row's own eight ranks of every split, all loads in flight
#pragma unroll
              for (int s = 0; s < 8; ++s) {
                const bool there = mine >= 0 && s < g.lk.ksplit;
                const float4* src = part + ((there ? s : 0) * rp + x) / 4 * 32;
                a[s] = there ? __ldcg(src) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                b[s] = there ? __ldcg(src + 32) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
              }
              float v[8] = {};
#pragma unroll
              for (int s = 0; s < 8; ++s) {
                v[0] += a[s].x;
                v[1] += a[s].y;
                v[2] += a[s].z;
                v[3] += a[s].w;
                v[4] += b[s].x;
                v[5] += b[s].y;
                v[6] += b[s].z;
                v[7] += b[s].w;
              }
              for (int sl = 0; sl * g.lk.rc < nch; ++sl) store_h(sl, x / cw, x % cw, v);
            }
        }
        if (last) {
          asm volatile("fence.proxy.async;" ::: "memory");  // for the TMA loads of other CTAs
          __threadfence();
          __syncwarp();
          if (lane == 0) {
            __threadfence();
            atomicAdd(g.lk.done, 1);
          }
        }
        continue;
      }
      const int acc = n & 1;
      int mb, nb;
      tile_at(it - downs, g.m_tiles, g.n_tiles, mb, nb);
      // What the tile needs beside its sums is read before they are complete.
      const int local = (mb * CTAS + (int)rank) * 128 + q * 32 + lane;
      const bool row_ok = local < g.rows, mixed = g.lk.q_max && __ldcg(&list_of(mb)->mixed);
      // Each warp has a copy of the bias: a warp whose wait expires leaves this loop alone, so none
      // may wait for another in it.
      if (g.p.bias) {
        __syncwarp();
        for (int c = lane; c < BN; c += 32) {
          const int64_t col = (int64_t)nb * BN + c;
          reinterpret_cast<float*>(sbias[q])[c] = col < g.p.N ? __ldg(g.p.bias + col) : 0.0f;
        }
        __syncwarp();
      }
      ok = mbar_wait_warp(&acc_full[acc], (n >> 1) & 1, abort_flag, err, kErrWaitAccFull);
      if (!ok) break;
      ++n;
      tc_fence_after();
      const int64_t row = g.row0 + local;
#pragma unroll 1
      for (int c = 0; c < BN / 32; ++c) {
        uint32_t r[32];
        __syncwarp();
        tmem_ld_32x32b_x32(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * BN + c * 32), r);
        tmem_wait_ld();
        const int64_t col0 = (int64_t)nb * BN + c * 32;
        if (col0 >= g.p.N) continue;
        const int cols = (int)min((int64_t)32, g.p.N - col0);
        if (g.y_tma) {
          // The block that used this buffer has left it (of 2 fp32 or 4 bf16 buffers).
          if (lane == 0) {
            if (g.p.y_bf16)
              tma_store_wait_read<3>();
            else
              tma_store_wait_read<1>();
          }
          __syncwarp();
        }
        if (row_ok) {
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
          if (g.p.bias) {
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              const float4 b = sbias[q][(c * 32 + j) / 4];
              v[j] += b.x;
              v[j + 1] += b.y;
              v[j + 2] += b.z;
              v[j + 3] += b.w;
            }
          }
          if (g.y_tma) {
            // 16-byte pieces in the swizzle of the box's row: 64 bytes of bf16 or 128 of fp32.
            if (g.p.y_bf16) {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                *reinterpret_cast<uint4*>(buf + lane * 64 + (j ^ (lane >> 1 & 3)) * 16) =
                    make_uint4(bf16_pair(v[8 * j], v[8 * j + 1]), bf16_pair(v[8 * j + 2], v[8 * j + 3]),
                               bf16_pair(v[8 * j + 4], v[8 * j + 5]), bf16_pair(v[8 * j + 6], v[8 * j + 7]));
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                *reinterpret_cast<float4*>(buf + lane * 128 + (j ^ (lane & 7)) * 16) =
                    make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) reinterpret_cast<float*>(buf)[lane * 32 + (j ^ lane)] = v[j];
          }
        }
        if (!g.y_tma) {
          // Rows that TMA cannot write, one after another, a lane per column: with a lane per
          // row the 32 stores of a warp met 32 lines (154 us for 9955 x 1197 bf16, K 366).
          __syncwarp();
          const int64_t first = row - lane;
          if (lane < cols)
            for (int i = 0; i < (int)min((int64_t)32, g.row0 + g.rows - first); ++i) {
              const float x = reinterpret_cast<const float*>(buf)[i * 32 + (lane ^ i)];
              if (g.p.y_bf16)
                ((uint16_t*)g.p.Y)[(first + i) * g.p.ldy + col0 + lane] = bf16_bits(x);
              else
                ((float*)g.p.Y)[(first + i) * g.p.ldy + col0 + lane] = x;
            }
          __syncwarp();
        } else {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) tma_store_2d(&tmY, buf, (int)col0, (int)(row - lane));
          buf = stg + (buf - stg + (g.p.y_bf16 ? 2048 : 4096)) % 8192;
        }
        if (mixed) {
          uint32_t bad = 0, top = 0;
#pragma unroll
          for (int j = 0; j < 32; ++j) top = max(top, r[j] & 0x7fffffffu);
          if (row_ok && top >= 0x7f800000u) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j < cols && (r[j] & 0x7fffffffu) >= 0x7f800000u) bad |= 1u << j;
          }
          __syncwarp();
          if (__any_sync(0xffffffffu, bad != 0)) {
            if (lane == 0) tma_store_wait_all();  // what was stored above is replaced
            __syncwarp();
            redo_chunk(g.p, g.lk, g.X, g.ldx, g.W, g.ldw, g.B, g.ldb, g.row0, local, col0, bad);
          }
        }
      }
      release(acc);
    }
    if (lane == 0) tma_store_wait_all();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    if constexpr (PAIR)
      tmem_dealloc_pair(tmem, C_::COLS);
    else
      tmem_dealloc(tmem, C_::COLS);
  }
}

template <int BN, bool PAIR>
void launch_lora_gemm(LoraGemm g, const uint16_t* A, int64_t lda, bool adapters) {
  const int64_t r = g.p.r;
  using C_ = LoraGemmCfg<BN, PAIR>;
  DeviceContext& c = ctx();
  CUtensorMap tx, tw, th, tb, ta;
  map_2d(&tx, g.X, g.p.K, g.p.T, g.ldx, 64, 128, CU_TENSOR_MAP_SWIZZLE_128B);
  map_2d(&tw, g.W, g.p.K, g.p.N, g.ldw, 64, C_::B_ROWS, CU_TENSOR_MAP_SWIZZLE_128B);
  g.m_tiles = (int)((g.rows + (PAIR ? 255 : 127)) / (PAIR ? 256 : 128));
  g.n_tiles = (int)((g.p.N + BN - 1) / BN);
  g.k_blocks = (int)((g.p.K + 63) / 64);
  // Units that would wait for H take part in making it: up to 8 K splits of 2 blocks at least.
  const int units = c.num_sms / (PAIR ? 2 : 1);
  g.lk.ksplit = std::max(1, std::min({8, units / g.m_tiles, g.k_blocks / 2}));
  if (adapters) {
    const int64_t groups = (g.rows + kGroup - 1) / kGroup;
    map_2d(&th, g.lk.H, g.lk.cw, groups * g.lk.q_max * kGroup, g.lk.cw, g.lk.cw, 128, swizzle_of(g.lk.cw));
    map_adapters(&tb, g.B, r, g.p.N, g.p.n_adapters, g.ldb, g.lk.cw, C_::B_ROWS, swizzle_of(g.lk.cw));
    map_adapters(&ta, A, g.p.K, r, g.p.n_adapters, lda, 64, PAIR ? g.lk.cw / 2 : g.lk.cw, CU_TENSOR_MAP_SWIZZLE_128B);
  } else {
    th = tb = ta = tx;  // not read
  }
  CUtensorMap ty = tx;
  if (g.y_tma) {
    const uint64_t dims[2] = {(uint64_t)g.p.N, (uint64_t)g.p.T};
    const uint64_t str[1] = {(uint64_t)g.p.ldy * (g.p.y_bf16 ? 2 : 4)};
    const uint32_t box[2] = {32, 32};
    encode_tmap(&ty, g.p.y_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, g.p.Y, dims, str, box,
                g.p.y_bf16 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
  }
  static int clusters[64] = {};
  auto kern = k_lora_gemm<BN, PAIR>;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2] = {};
  int n = 0;
  if (PAIR) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = 2;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.gridDim = dim3(2);
  cfg.blockDim = dim3(kRowThreads);
  cfg.dynamicSmemBytes = C_::SMEM;
  cfg.stream = c.stream;
  cfg.attrs = attr;
  cfg.numAttrs = n;
  if (!clusters[c.device]) {
    check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C_::SMEM),
               "cudaFuncSetAttribute(linear_lora)");
    int fit = c.num_sms;
    if (PAIR) check_cuda(cudaOccupancyMaxActiveClusters(&fit, kern, &cfg), "cudaOccupancyMaxActiveClusters(linear_lora)");
    if (fit <= 0) fail(kErrUnsupported, "linear_lora: no cluster of 2 fits");
    clusters[c.device] = fit;
  }
  if (adapters) {
    // Units wait for H that others make, so all must be resident: two such launches at once,
    // each with a part of the processors, would wait for each other's. (Starting beside
    // k_lora_lists as well would save under 1 us, but the profiler fails on such a launch.)
    attr[n].id = cudaLaunchAttributeCooperative;
    attr[n].val.cooperative = 1;
    ++n;
  }
  cfg.numAttrs = n;
  const int64_t items = (int64_t)g.m_tiles * (g.n_tiles + (adapters ? g.lk.ksplit : 0));
  cfg.gridDim = dim3((unsigned)(std::min<int64_t>(clusters[c.device], items) * (PAIR ? 2 : 1)));
  check_cuda(cudaLaunchKernelEx(&cfg, kern, tx, tw, th, tb, ta, ty, g), "linear_lora");
  check_launch("linear_lora");
}

// Tile shape by waves, as gemm_tc.cu prices them: a tile costs its width and 48 columns of
// fixed cost, a pair tile (256 rows over two processors) 8% less. Several pair widths, because
// a few rows of tiles leave the last wave nearly empty: 2397 x 4096 outputs are 2.2 waves of
// 256 columns (3 x 280) but 3.0 waves of 192 (3 x 221).
struct Tile {
  int bm, bn;
  double cost;
};
Tile choose_tile(int64_t rows, int64_t N, bool adapters) {
  const int sms = ctx().num_sms;
  Tile best{128, 64, 1e30};
  for (int bn : {256, 224, 192, 160, 128, 64})
    for (int bm : {256, 128}) {
      if (bm == 256 ? bn == 64 || rows <= 128 : bn != 256 && bn != 128 && bn != 64) continue;
      const int64_t m = (rows + bm - 1) / bm;
      const double down = adapters ? 0.3 * (double)m : 0.0;  // the items that make H
      const double x = std::ceil(((double)(m * ((N + bn - 1) / bn)) + down) / (bm == 256 ? sms / 2 : sms)) * (bn + 48) *
                       (bm == 256 ? 0.92 : 1.0);
      if (x < best.cost - 1e-9) best = Tile{bm, bn, x};
    }
  return best;
}

// Whether k_lora_rows, in blocks of 128 rows, takes fewer microseconds than the GEMM. The
// GEMM's groups of 256 rows multiply every row with all adapters of the group, so requests of few
// rows each cost it dearly: 129 rows, 3840 x 3840, rank 128, take 40 us with 2 requests, 144
// with 16 and 506 with 64; k_lora_rows takes 38, 40 and 52. With 512 rows the GEMM takes 38, 71
// and 202 and k_lora_rows 70, 69 and 76, with 1024 the GEMM 40, 54 and 112 and k_lora_rows over
// 100, because it reads an adapter for every row or every four. How many adapters the rows
// use is known on the device only; a mixture of 16 is assumed, or all there are. The constants
// are fitted to N, K from 224 to 10240, ranks 16 and 128, T from 129 to 1024.
bool few_rows(const LoraLinear& p) {
  if (p.T <= kMaxRowsSmall) return true;
  if (p.T > 1024 || p.n_adapters <= 0 || p.r <= 0) return false;
  const int sms = ctx().num_sms, splits = row_splits<kMaxRowsSmall>(p);
  const double kb = (double)((p.K + 63) / 64), t = (double)p.T;
  const int64_t tiles = (p.N + 127) / 128 * ((p.T + kMaxRowsSmall - 1) / kMaxRowsSmall);
  const double rows = 12.0 + std::ceil((double)(tiles * splits) / (double)row_units<kMaxRowsSmall>(splits)) * (kb / splits) * 0.6 +
                      t * (double)p.r * ((by_runs(p) ? 0.7e-4 : 2.7e-4) + 1.5e-7 * (double)p.K);
  const Tile tile = choose_tile(p.T, p.N, true);
  const int64_t m = (p.T + tile.bm - 1) / tile.bm;
  const double ksplit = std::max(1.0, std::min({8.0, (double)sms / (tile.bm / 128) / (double)m, kb / 2}));
  const double chunks = (double)std::min<int64_t>(p.n_adapters, 16) / (double)((p.T + kGroup - 1) / kGroup) *
                        (double)round_up(p.r, chunk_width(p.r)) / 64.0;
  return rows < 12.0 + tile.cost * kb * 1.1e-3 + chunks * (1.8 + 0.25 * kb / ksplit);
}

// What the large path keeps in the workspace: one block of rows' lists and H.
struct Big {
  LoraK lk;
  int64_t rows;  // rows of a block, a multiple of kGroup
  size_t lists_at, arrived_at, part_at, h_at, bytes;
};
Big lay_out_big(const LoraLinear& p, size_t at) {
  Big b{};
  b.lists_at = b.h_at = b.bytes = at;
  b.rows = round_up(p.T, kGroup);
  b.lk.cw = 64;
  if (p.n_adapters <= 0 || p.r <= 0) return b;
  b.lk.parts = p.y_bf16 ? 1 : 2;
  b.lk.cw = chunk_width(p.r);
  b.lk.rc = (int)((p.r + b.lk.cw - 1) / b.lk.cw);
  b.lk.q_max = b.lk.chunks((int)std::min<int64_t>(p.n_adapters, kGroup));
  // H holds every chunk a group could need; blocks of rows keep it within 128 MB.
  const int64_t group = (int64_t)b.lk.q_max * kGroup * b.lk.cw * 2;
  b.rows = std::min(b.rows, std::max<int64_t>(1, ((int64_t)128 << 20) / group) * kGroup);
  // `done`, the lists, `arrived`, the K splits' parts (splits x rows of tiles <= units), H.
  const int64_t groups = b.rows / kGroup;
  b.arrived_at = at + 256 + align256((size_t)groups * sizeof(GroupList));
  b.part_at = b.arrived_at + align256((size_t)groups * 32);
  const int64_t part_rows = std::min<int64_t>(8 * b.rows, std::max<int64_t>(b.rows, (int64_t)ctx().num_sms * 128 + kGroup));
  b.h_at = b.part_at + align256((size_t)(part_rows * b.lk.rc * b.lk.cw) * 4);
  b.bytes = b.h_at + align256((size_t)groups * group);
  return b;
}

void launch_big(const LoraLinear& p, const uint16_t* X, int64_t ldx, const uint16_t* W, int64_t ldw, const uint16_t* A,
                int64_t lda, const uint16_t* B, int64_t ldb, uint8_t* ws, const Big& big) {
  DeviceContext& c = ctx();
  const bool adapters = p.n_adapters > 0 && p.r > 0;
  LoraGemm g{};
  g.p = p;
  g.lk = big.lk;
  g.lk.done = reinterpret_cast<int*>(ws + big.lists_at);
  g.lk.lists = reinterpret_cast<GroupList*>(ws + big.lists_at + 256);
  g.lk.arrived = reinterpret_cast<int*>(ws + big.arrived_at);
  g.lk.part = reinterpret_cast<float4*>(ws + big.part_at);
  g.lk.H = reinterpret_cast<uint16_t*>(ws + big.h_at);
  g.X = X;
  g.W = W;
  g.B = B;
  g.ldx = ldx;
  g.ldw = ldw;
  g.ldb = ldb;
  g.y_tma = aligned16(p.Y) && p.ldy % (p.y_bf16 ? 8 : 4) == 0;
  for (g.row0 = 0; g.row0 < p.T; g.row0 += big.rows) {
    g.rows = std::min(big.rows, p.T - g.row0);
    const Tile tile = choose_tile(g.rows, p.N, adapters);
    if (adapters) {
      k_lora_lists<<<(unsigned)((g.rows + kGroup - 1) / kGroup), kGroup, 0, c.stream>>>(p, g.lk, g.row0, g.rows);
      check_launch("lora_lists");
    }
    const int bm = tile.bm, bn = tile.bn;
    if (bm == 256) {
      if (bn == 256) launch_lora_gemm<256, true>(g, A, lda, adapters);
      if (bn == 224) launch_lora_gemm<224, true>(g, A, lda, adapters);
      if (bn == 192) launch_lora_gemm<192, true>(g, A, lda, adapters);
      if (bn == 160) launch_lora_gemm<160, true>(g, A, lda, adapters);
      if (bn == 128) launch_lora_gemm<128, true>(g, A, lda, adapters);
    } else {
      if (bn == 256) launch_lora_gemm<256, false>(g, A, lda, adapters);
      if (bn == 128) launch_lora_gemm<128, false>(g, A, lda, adapters);
      if (bn == 64) launch_lora_gemm<64, false>(g, A, lda, adapters);
    }
  }
}

}  // namespace

size_t lora_linear_workspace(const LoraLinear& p) {
  const Operands o = lay_out(p);
  if (!few_rows(p)) return lay_out_big(p, o.h_at).bytes;
  size_t h;
  lay_out_rows(p, nullptr, &h);
  return o.h_at + h;
}

void launch_lora_linear(LoraLinear p, void* ws_) {
  DeviceContext& c = ctx();
  p.err = c.err_word;
  const Operands o = lay_out(p);
  uint8_t* ws = static_cast<uint8_t*>(ws_);
  const uint16_t *X = (const uint16_t*)p.X, *W = p.W, *A = p.A, *B = p.B;
  int64_t ldx = p.ldx, ldw = p.ldw, lda = p.lda, ldb = p.ldb;
  PackAll all{};
  auto pack = [&](bool need, const uint16_t*& x, int64_t& ld, int64_t rows, int64_t cols, int64_t pitch, size_t at, bool f32) {
    if (!need) return;
    uint16_t* dst = reinterpret_cast<uint16_t*>(ws + at);
    all.m[all.n] = PackOne{x, dst, ld, rows, (int)cols, (int)pitch, f32 ? 1 : 0};
    all.end[all.n] = (all.n ? all.end[all.n - 1] : 0) + rows * (pitch / 8);
    ++all.n;
    x = dst;
    ld = pitch;
  };
  pack(o.pack_x, X, ldx, p.T, p.K, o.Kp, o.x_at, !p.x_bf16);
  pack(o.pack_w, W, ldw, p.N, p.K, o.Kp, o.w_at, false);
  pack(o.pack_a, A, lda, p.n_adapters * p.r, p.K, o.Kp, o.a_at, false);
  pack(o.pack_b, B, ldb, p.n_adapters * p.N, p.r, o.rb, o.b_at, false);
  if (all.n) {
    const int64_t grid = std::min<int64_t>((all.end[all.n - 1] + 255) / 256, (int64_t)c.num_sms * 16);
    k_lora_pack<<<(unsigned)grid, 256, 0, c.stream>>>(all);
    check_launch("lora_pack");
  }
  if (!few_rows(p)) return launch_big(p, X, ldx, W, ldw, A, lda, B, ldb, ws, lay_out_big(p, o.h_at));
  size_t h;
  LoraRows g{p, lay_out_rows(p, ws + o.h_at, &h), X, W, B, ldx, ldw, ldb, 1};
  const int tn = rows_tile(p.T);
  if (g.rk.rc > 0) {
    const unsigned eights = (unsigned)(g.rk.rc * g.rk.cw / 8);
    if (by_runs(p))
      k_lora_down_runs<<<dim3((unsigned)((p.T + kRunRows - 1) / kRunRows), eights), 256, 0, c.stream>>>(p, X, ldx, A, lda, g.rk);
    else
      k_lora_down_rows<<<dim3((unsigned)p.T, eights), 256, 0, c.stream>>>(p, X, ldx, A, lda, g.rk, tn);
    check_launch("lora_down_rows");
  }
  if (tn == 16) return launch_rows<16>(g);
  if (tn == 32) return launch_rows<32>(g);
  if (tn == 64) return launch_rows<64>(g);
  launch_rows<128>(g);
}

}  // namespace sdb
