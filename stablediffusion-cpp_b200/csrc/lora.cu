// lora.cu - a projection shared by every row plus each row's own low-rank adapter:
//   y[t, n] = sum_k x[t, k] W[n, k] + bias[n] + sum_j h[t, j] B_a[n, j],
//   h[t, j] = s_a sum_k x[t, k] A_a[j, k],   a = row_adapter[t] (no second term for a < 0).
//
// Up to 64 rows the work is reading W and the adapters once (k_lora_down_rows, k_lora_rows);
// above, it is a GEMM (k_lora_down and the adapter form of gemm_tc.cu).
#include <algorithm>

#include "elem.cuh"
#include "internal.h"
#include "ptx.cuh"
#include "serving.h"

namespace sdb {
namespace {

inline int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }
inline size_t align256(size_t b) { return (b + 255) & ~size_t(255); }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

constexpr int kMaxRowsSmall = 64;

// ------------------------------------------------------------------------------------
// Few rows
// ------------------------------------------------------------------------------------
// h[t, j], one warp per value, 16-byte loads of both rows (pitches multiples of 8, packed
// where they were not; elements past K are masked). Bound by the adapters' bytes.
__global__ void __launch_bounds__(256) k_lora_down_rows(const LoraLinear p, const uint16_t* __restrict__ X, int64_t ldx,
                                                        const uint16_t* __restrict__ A, int64_t lda, float* __restrict__ h) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int lane = threadIdx.x & 31, t = blockIdx.x;
  const int64_t j = (int64_t)blockIdx.y * 8 + (threadIdx.x >> 5);
  if (j >= p.r) return;
  const int a = p.row_adapter[t];
  if (a >= p.n_adapters && lane == 0 && j == 0) atomicOr(p.err, kErrBadIndex);
  float s = 0.0f;
  if (a >= 0 && a < p.n_adapters) {
    const uint16_t* x = X + (int64_t)t * ldx;
    const uint16_t* w = A + ((int64_t)a * p.r + j) * lda;
    float2 s2 = make_float2(0.0f, 0.0f);
    const int64_t whole = p.K / 8;
#pragma unroll 4
    for (int64_t c = lane; c < whole; c += 32) {
      const uint4 u = *reinterpret_cast<const uint4*>(x + 8 * c), v = __ldg(reinterpret_cast<const uint4*>(w + 8 * c));
      const uint32_t ux[4] = {u.x, u.y, u.z, u.w}, vx[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        s2 = ffma2(make_float2(__uint_as_float(ux[i] << 16), __uint_as_float(ux[i] & 0xffff0000u)),
                   make_float2(__uint_as_float(vx[i] << 16), __uint_as_float(vx[i] & 0xffff0000u)), s2);
    }
    s = s2.x + s2.y;
    for (int64_t k = whole * 8 + lane; k < p.K; k += 32) s = fmaf(bf16_to_f32(x[k]), bf16_to_f32(w[k]), s);
    s = warp_add(s) * (p.scale ? p.scale[a] : 1.0f);
  }
  if (lane == 0) h[t * p.r + j] = s;
}

// All rows in one tile of N_mma columns: D[n, t] = sum_k W[n, k] x[t, k] on tcgen05, 128
// rows of W (the M of the MMA) per cluster, K split over the cluster's CTAs, so that every
// processor streams W. While the copies run, the epilogue warps add up the adapter term in
// fp32 for the CTA's share of the rows n; then the CTAs' partial sums are read from their
// shared memory in rank order (the result does not depend on timing).
template <int TN>
struct RowsCfg {
  static constexpr int W_BYTES = 128 * 128, X_BYTES = TN * 128, STAGE = W_BYTES + X_BYTES;
  static constexpr int STAGES = 4;
  static constexpr int PITCH = TN + 1;  // floats of a row of partial sums: spreads banks
  static constexpr int SUM_BYTES = 128 * PITCH * 4;
  static_assert(STAGES * STAGE >= SUM_BYTES, "partial sums reuse the stages");
};
constexpr int kRowThreads = 192;  // TMA warp, MMA warp, four epilogue warps

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

template <int TN>
__global__ void __launch_bounds__(kRowThreads)
    k_lora_rows(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                const __grid_constant__ LoraLinear p, const float* __restrict__ h, const uint16_t* __restrict__ B,
                int64_t ldb, int splits, int b_vec) {
  using C_ = RowsCfg<TN>;
  constexpr uint32_t IDESC = make_idesc(1u, 0, 0, 128, TN);
  constexpr uint32_t COLS = TN < 32 ? 32 : TN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* sums = reinterpret_cast<float*>(smem);                               // [128][PITCH], after the MMAs
  float* delta = reinterpret_cast<float*>(smem + C_::STAGES * C_::STAGE);    // [128 / splits][PITCH]
  float* sh = delta + (128 / splits) * C_::PITCH;                            // [T][r]
  __shared__ uint64_t full[C_::STAGES], empty[C_::STAGES], acc_full;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % splits, tile = blockIdx.x / splits;
  const int T = (int)p.T, r = (int)p.r;
  const int64_t n0 = (int64_t)tile * 128;
  const int kblocks = (int)((p.K + 63) / 64);
  const int kb0 = (int)((int64_t)kblocks * rank / splits), kb1 = (int)((int64_t)kblocks * (rank + 1) / splits);

  if (threadIdx.x == 0) {
    for (int s = 0; s < C_::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(&acc_full, 1);
    abort_word = 0;
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
  if (warp == 0) {
    if (lane == 0) {
      int done = 0;
      for (int kb = kb0; kb < kb1; ++kb, ++done) {
        const int s = done % C_::STAGES;
        if (!mbar_wait(&empty[s], ((done / C_::STAGES) & 1) ^ 1u, abort_flag, p.err, kErrWaitEmpty)) break;
        mbar_arrive_expect_tx(&full[s], C_::STAGE);
        tma_load_2d(smem + s * C_::STAGE, &tmW, &full[s], kb * 64, (int)n0);
        tma_load_2d(smem + s * C_::STAGE + C_::W_BYTES, &tmX, &full[s], kb * 64, 0);
      }
      if (done < kb1 - kb0) {
        // Aborted: wait (bounded) for the loads in flight.
        const uint64_t t0 = globaltimer_ns();
        for (int i = max(0, done - C_::STAGES); i < done; ++i)
          while (!mbar_try_wait(&full[i % C_::STAGES], (i / C_::STAGES) & 1) && globaltimer_ns() - t0 < kWaitLimitNs) {
          }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      for (int i = 0; i < kb1 - kb0; ++i) {
        const int s = i % C_::STAGES;
        if (!mbar_wait(&full[s], (i / C_::STAGES) & 1, abort_flag, p.err, kErrWaitFull)) break;
        tc_fence_after();
        const uint32_t a0 = smem_u32(smem + s * C_::STAGE), b0 = a0 + C_::W_BYTES;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_f16_ss(tmem, sdesc_k_sw128(a0 + k * 32), sdesc_k_sw128(b0 + k * 32), IDESC, (i | k) != 0);
        umma_commit(&empty[s]);
      }
      umma_commit(&acc_full);
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(&acc_full, 0))
        if (globaltimer_ns() - t0 > kWaitLimitNs) {
          atomicOr(p.err, kErrWaitDrain);
          break;
        }
    }
  } else {
    // The adapter term of rows [rank R, + R) of the tile, one output feature n and every
    // `splits`-th token per thread.
    const int tid = threadIdx.x - 64, R = 128 / splits;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int i = tid; i < T * r; i += 128) sh[i] = h[i];
    asm volatile("bar.sync 1, 128;" ::: "memory");
    const int row = tid % R;
    const int64_t n = n0 + rank * R + row;
    for (int t = tid / R; t < T; t += splits) {
      const int a = p.row_adapter ? p.row_adapter[t] : -1;
      float d = 0.0f;
      if (r > 0 && a >= 0 && a < p.n_adapters && n < p.N) {
        const uint16_t* b = B + ((int64_t)a * p.N + n) * ldb;
        const float* ht = sh + t * r;
        if (b_vec) {  // 16-byte rows of B, r a multiple of 8
          float2 d2 = make_float2(0.0f, 0.0f);
#pragma unroll 4
          for (int c = 0; c < r; c += 8) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(b + c));
            const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
              d2 = ffma2(make_float2(ht[c + 2 * i], ht[c + 2 * i + 1]),
                         make_float2(__uint_as_float(x[i] << 16), __uint_as_float(x[i] & 0xffff0000u)), d2);
          }
          d = d2.x + d2.y;
        } else {
          for (int c = 0; c < r; ++c) d = fmaf(ht[c], bf16_to_f32(b[c]), d);
        }
      }
      delta[row * C_::PITCH + t] = d;
    }
    const int q = warp & 3;  // TMEM lane quarter
    if (mbar_wait(&acc_full, 0, abort_flag, p.err, kErrWaitAccFull)) {
      tc_fence_after();
      float* mine = sums + (q * 32 + lane) * C_::PITCH;
#pragma unroll
      for (int c = 0; c < TN; c += 16) {
        uint32_t v[16];
        tmem_ld_32x32b_x16(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)c, v);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) mine[c + i] = kb1 > kb0 ? __uint_as_float(v[i]) : 0.0f;
      }
    }
  }
  tc_fence_before();
  __syncwarp();
  cluster_sync();  // every CTA's partial sums are in its shared memory
  tc_fence_after();
  if (warp >= 2) {
    const int tid = threadIdx.x - 64, R = 128 / splits;
    const int row = tid % R;
    const int64_t n = n0 + rank * R + row;
    if (n < p.N) {
      const float bias = p.bias ? p.bias[n] : 0.0f;
      for (int t = tid / R; t < T; t += splits) {
        const uint32_t at = smem_u32(sums + (rank * R + row) * C_::PITCH + t);
        float y = 0.0f;
        for (int s = 0; s < splits; ++s) {
          uint32_t peer;
          asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(at), "r"(s));
          y += ld_cluster_f32(peer);
        }
        y += bias + delta[row * C_::PITCH + t];
        if (p.y_bf16)
          ((uint16_t*)p.Y)[t * p.ldy + n] = f32_to_bf16_rne(y);
        else
          ((float*)p.Y)[t * p.ldy + n] = y;
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
  size_t x_at, w_at, a_at, b_at, h_at, bytes;
};
Operands lay_out(const LoraLinear& p) {
  Operands o{};
  o.Kp = round_up(p.K, 8);
  o.rb = round_up(std::max<int64_t>(p.r, 1), 8);
  const bool adapters = p.n_adapters > 0 && p.r > 0;
  o.pack_x = !p.x_bf16 || !aligned16(p.X) || p.ldx % 8 != 0;
  o.pack_w = !aligned16(p.W) || p.ldw % 8 != 0;
  o.pack_a = adapters && (!aligned16(p.A) || p.lda % 8 != 0);
  o.pack_b = adapters && p.T > kMaxRowsSmall && (!aligned16(p.B) || p.ldb % 8 != 0);
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
  o.bytes = at + align256((size_t)(p.T * p.r) * 4);
  return o;
}

template <int TN>
void launch_rows(const LoraLinear& p, const uint16_t* X, int64_t ldx, const uint16_t* W, int64_t ldw, const float* h) {
  using C_ = RowsCfg<TN>;
  DeviceContext& c = ctx();
  CUtensorMap tw, tx;
  {
    const uint64_t dims[2] = {(uint64_t)p.K, (uint64_t)p.N};
    const uint64_t str[1] = {(uint64_t)ldw * 2};
    const uint32_t box[2] = {64, 128};
    encode_tmap(&tw, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, W, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
  }
  {
    const uint64_t dims[2] = {(uint64_t)p.K, (uint64_t)p.T};
    const uint64_t str[1] = {(uint64_t)ldx * 2};
    const uint32_t box[2] = {64, (uint32_t)TN};
    encode_tmap(&tx, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, X, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
  }
  const int64_t tiles = (p.N + 127) / 128;
  const int kblocks = (int)((p.K + 63) / 64);
  auto smem_of = [&](int s) {
    return 1024 + C_::STAGES * C_::STAGE + 128 / s * C_::PITCH * 4 + (int)(p.T * p.r) * 4;
  };
  // K splits until two CTAs a processor (where they fit) have a part, of two K blocks at least.
  int splits = 1;
  while (splits < 8 && kblocks >= 4 * splits &&
         tiles * splits * 2 <= (int64_t)c.num_sms * (smem_of(2 * splits) <= 113 * 1024 ? 2 : 1))
    splits *= 2;
  const int smem = smem_of(splits);
  static bool done[64] = {};
  if (!done[c.device]) {
    check_cuda(cudaFuncSetAttribute(k_lora_rows<TN>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024),
               "cudaFuncSetAttribute(linear_lora)");
    done[c.device] = true;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(tiles * splits));
  cfg.blockDim = dim3(kRowThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = c.stream;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.r > 0 ? 2 : 1;  // only k_lora_down_rows may be overtaken
  const int b_vec = p.r % 8 == 0 && p.ldb % 8 == 0 && aligned16(p.B);
  check_cuda(cudaLaunchKernelEx(&cfg, k_lora_rows<TN>, tw, tx, p, h, p.B, p.ldb, splits, b_vec), "linear_lora");
  check_launch("linear_lora");
}

// ------------------------------------------------------------------------------------
// Many rows: Y = [X | H] [W | B]^T as one GEMM, where H holds h in the columns of the row's
// own adapter and zeros in those of the other adapters of its tile.
// ------------------------------------------------------------------------------------
constexpr int kGroup = 256;     // rows that share a list of adapters and a block of H
constexpr int kMaxPass = 256;   // accumulator columns of k_lora_down

struct GroupList {
  int count;            // distinct adapters of the rows
  int mixed;            // rows of different adapters, or some of none
  int adapter[kGroup];  // in the order of their first rows
};
// H: [groups][q_max][kGroup][cw] bf16. A chunk q of a group is cw ranks of one adapter (and,
// with two parts, of the high or low half of h): q = (slot * parts + part) * rc + c.
struct LoraK {
  const GroupList* lists;
  uint16_t* H;
  int cw, rc, parts, q_max;
  __host__ __device__ int chunks(int count) const { return count * parts * rc; }
};

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
inline CUtensorMapSwizzle swizzle_of(int cw) {
  return cw == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : cw == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;
}

// H of one tile of 128 rows: x A_a^T on tcgen05 for every adapter a of the group (an N of
// rpr = round_up(r, 16) columns each, at most 256 a pass), K split over the cluster's CTAs.
// Each row keeps the columns of its own adapter; the CTAs' parts are added in rank order.
// Reading X bounds it: 128 x K bf16 per tile, once per 256 columns of adapters.
struct DownCfg {
  static constexpr int X_BYTES = 128 * 128, A_BYTES = kMaxPass * 128, STAGE = X_BYTES + A_BYTES;
  static constexpr int MAX_STAGES = 4;
  static int stages(int rpr) { return std::min(MAX_STAGES, (222 * 1024 - 128 * (rpr + 1) * 4) / STAGE); }
  static int smem(int rpr) { return 1024 + stages(rpr) * STAGE + 128 * (rpr + 1) * 4; }
};

__global__ void __launch_bounds__(kRowThreads)
    k_lora_down(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmA,
                const __grid_constant__ LoraLinear p, const LoraK lk, GroupList* __restrict__ lists, int rpr, int stages,
                int splits, int64_t row0, int64_t rows) {
  using C_ = DownCfg;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* sums = reinterpret_cast<float*>(smem + stages * C_::STAGE);  // [128][pitch]
  const int pitch = rpr + 1;
  __shared__ uint64_t full[C_::MAX_STAGES], empty[C_::MAX_STAGES], acc_full[2], acc_empty[2], drain;
  __shared__ int ids[kGroup], slot[kGroup], rank_of[kGroup], list[kGroup], wsum[8], count, mixed;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % splits, tile = blockIdx.x / splits, group = tile >> 1, half = tile & 1;
  const int kblocks = (int)((p.K + 63) / 64);
  const int kb0 = (int)((int64_t)kblocks * rank / splits), kb1 = (int)((int64_t)kblocks * (rank + 1) / splits);

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 4);
    }
    mbar_init(&drain, 1);
    abort_word = 0;
    mixed = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  // The group's distinct adapters, in the order of their first rows.
  for (int i = threadIdx.x; i < kGroup; i += kRowThreads) {
    const int64_t t = (int64_t)group * kGroup + i;
    int a = t < rows ? p.row_adapter[row0 + t] : -2;  // -2: no row
    if (a >= p.n_adapters) {
      if (rank == 0 && half == 0) atomicOr(p.err, kErrBadIndex);
      a = -1;
    }
    if (a < 0 && a != -2) a = -1;
    if (t >= rows) a = -2;
    ids[i] = a;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kGroup; i += kRowThreads) {
    const int a = ids[i];
    int f = 0;
    while (ids[f] != a) ++f;  // ends at i at the latest
    slot[i] = f;
    if (a != -2 && a != ids[0]) mixed = 1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kGroup; i += kRowThreads) rank_of[i] = slot[i] == i && ids[i] >= 0;
  __syncthreads();
  if (warp < 1) {  // exclusive prefix over the 256 flags, 8 per lane
    int n = 0, f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f[i] = rank_of[lane * 8 + i];
      n += f[i];
    }
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    int at = x - n;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (f[i]) list[at] = ids[lane * 8 + i];
      rank_of[lane * 8 + i] = at;
      at += f[i];
    }
    if (lane == 31) count = x;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const int m = count, per_pass = kMaxPass / rpr, passes = (m + per_pass - 1) / per_pass;
  if (rank == 0 && half == 0) {
    for (int i = threadIdx.x; i < m; i += kRowThreads) lists[group].adapter[i] = list[i];
    if (threadIdx.x == 0) {
      lists[group].count = m;
      lists[group].mixed = mixed;
    }
  }
  if (warp == 0) {
    if (lane == 0) {
      int done = 0;
      bool ok = true;
      for (int ps = 0; ps < passes && ok; ++ps) {
        const int s0 = ps * per_pass, used = min(per_pass, m - s0);
        for (int kb = kb0; kb < kb1; ++kb, ++done) {
          const int s = done % stages;
          ok = mbar_wait(&empty[s], ((done / stages) & 1) ^ 1u, abort_flag, p.err, kErrWaitEmpty);
          if (!ok) break;
          uint8_t* st = smem + s * C_::STAGE;
          mbar_arrive_expect_tx(&full[s], C_::X_BYTES + used * rpr * 128);
          tma_load_2d(st, &tmX, &full[s], kb * 64, (int)(row0 + (int64_t)tile * 128));
          for (int i = 0; i < used; ++i)
            tma_load_3d(st + C_::X_BYTES + i * rpr * 128, &tmA, &full[s], kb * 64, 0, list[s0 + i]);
        }
      }
      if (!ok) {
        const uint64_t t0 = globaltimer_ns();
        for (int i = max(0, done - stages); i < done; ++i)
          while (!mbar_try_wait(&full[i % stages], (i / stages) & 1) && globaltimer_ns() - t0 < kWaitLimitNs) {
          }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int done = 0;
      bool ok = true;
      for (int ps = 0; ps < passes && ok; ++ps) {
        const int acc = ps & 1, used = min(per_pass, m - ps * per_pass);
        const uint32_t idesc = make_idesc(1u, 0, 0, 128, (uint32_t)(used * rpr)), d = tmem + (uint32_t)(acc * kMaxPass);
        ok = mbar_wait(&acc_empty[acc], ((ps >> 1) & 1) ^ 1u, abort_flag, p.err, kErrWaitAccEmpty);
        if (!ok) break;
        tc_fence_after();
        for (int kb = kb0; kb < kb1; ++kb, ++done) {
          const int s = done % stages;
          ok = mbar_wait(&full[s], (done / stages) & 1, abort_flag, p.err, kErrWaitFull);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a0 = smem_u32(smem + s * C_::STAGE), b0 = a0 + C_::X_BYTES;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16_ss(d, sdesc_k_sw128(a0 + k * 32), sdesc_k_sw128(b0 + k * 32), idesc, kb > kb0 || k > 0);
          umma_commit(&empty[s]);
        }
        if (!ok) break;
        umma_commit(&acc_full[acc]);
      }
      umma_commit(&drain);
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(&drain, 0))
        if (globaltimer_ns() - t0 > kWaitLimitNs) {
          atomicOr(p.err, kErrWaitDrain);
          break;
        }
    }
  } else {
    const int q = warp & 3, rr = q * 32 + lane, me = half * 128 + rr;
    const int mine = ids[me] >= 0 ? rank_of[slot[me]] : -1;
    float* row = sums + rr * pitch;
    for (int ps = 0; ps < passes; ++ps) {
      const int acc = ps & 1, s0 = ps * per_pass, used = min(per_pass, m - s0);
      if (!mbar_wait(&acc_full[acc], (ps >> 1) & 1, abort_flag, p.err, kErrWaitAccFull)) break;
      tc_fence_after();
      for (int i = 0; i < used; ++i) {
        if (!__any_sync(0xffffffffu, mine == s0 + i)) continue;
        for (int c = 0; c < rpr; c += 16) {
          uint32_t v[16];
          __syncwarp();
          tmem_ld_32x32b_x16(tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * kMaxPass + i * rpr + c), v);
          tmem_wait_ld();
          if (mine == s0 + i) {
#pragma unroll
            for (int e = 0; e < 16; ++e) row[c + e] = kb1 > kb0 ? __uint_as_float(v[e]) : 0.0f;
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[acc]);
    }
  }
  tc_fence_before();
  __syncwarp();
  cluster_sync();
  if (warp >= 2) {
    // This CTA's share of the rows: 8 ranks of one chunk per step and thread.
    const int share = 128 / splits, pieces = lk.cw / 8, nq = lk.chunks(m);
    for (int i = threadIdx.x - 64; i < share * pieces * nq; i += 128) {
      const int pc = i % pieces, rr = rank * share + i / pieces % share, qi = i / (pieces * share);
      const int c = qi % lk.rc, part = qi / lk.rc % lk.parts, sl = qi / (lk.rc * lk.parts);
      const int me = half * 128 + rr, a = ids[me];
      uint32_t w[4] = {0, 0, 0, 0};
      if (a >= 0 && rank_of[slot[me]] == sl) {
        const float scale = p.scale ? p.scale[a] : 1.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int j = c * lk.cw + pc * 8 + e;
          float v = 0.0f;
          if (j < p.r) {
            const uint32_t at = smem_u32(sums + rr * pitch + j);
            for (int s = 0; s < splits; ++s) {
              uint32_t peer;
              asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(at), "r"(s));
              v += ld_cluster_f32(peer);
            }
            v *= scale;
          }
          uint32_t b = f32_to_bf16_rne(v);
          if (part) {  // what bf16 lost: h = high + low to 2^-16
            const float hi = bf16_to_f32((uint16_t)b);
            b = f32_to_bf16_rne(fabsf(hi) < INFINITY ? v - hi : 0.0f);
          }
          w[e >> 1] |= b << (16 * (e & 1));
        }
      }
      uint16_t* dst = lk.H + (((int64_t)group * lk.q_max + qi) * kGroup + me) * lk.cw + pc * 8;
      *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  __syncwarp();
  cluster_sync();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// The elements of one 32-column chunk of a warp's rows whose sums are not finite, again
// without the tensor core where an adapter of another row may have caused it: in a group of
// several adapters, zero times an infinity or NaN of another adapter's B is NaN.
__device__ __noinline__ void redo_chunk(const LoraLinear& p, const LoraK& lk, const uint16_t* X, int64_t ldx,
                                        const uint16_t* W, int64_t ldw, const uint16_t* B, int64_t ldb, int64_t row0,
                                        int local, int64_t col0, uint32_t bad) {
  const int lane = threadIdx.x & 31;
  const GroupList& L = lk.lists[local / kGroup];
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
      int a = p.row_adapter[row0 + t], sl = 0;
      if (a >= 0 && a < p.n_adapters) {
        while (L.adapter[sl] != a) ++sl;
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
          ((uint16_t*)p.Y)[(row0 + t) * p.ldy + n] = f32_to_bf16_rne(s);
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
// 128 x BN tiles. After the K blocks of X and W a tile runs through the chunks of H and B
// of its group's list, 64 / cw of them a stage; they are read only once k_lora_down has
// ended (griddepcontrol.wait), so the base product of the first tiles overlaps it.
template <int BN, bool PAIR>
struct LoraGemmCfg {
  static constexpr int B_ROWS = PAIR ? BN / 2 : BN;
  static constexpr int A_BYTES = 128 * 128, B_BYTES = B_ROWS * 128, STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = 208 * 1024 / STAGE > 8 ? 8 : 208 * 1024 / STAGE;
  static constexpr int SMEM = 1024 + STAGES * STAGE;
  static constexpr uint32_t COLS = 2 * BN <= 128 ? 128 : 2 * BN <= 256 ? 256 : 512;
};
struct LoraGemm {
  LoraLinear p;
  LoraK lk;
  const uint16_t *X, *W, *B;
  int64_t ldx, ldw, ldb;
  int64_t row0, rows;
  int m_tiles, n_tiles, k_blocks;
  int y_vec, bias_vec;
};
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
                const __grid_constant__ LoraGemm g) {
  using C_ = LoraGemmCfg<BN, PAIR>;
  constexpr int STAGES = C_::STAGES, CTAS = PAIR ? 2 : 1;
  constexpr uint32_t IDESC = make_idesc(1u, 0, 0, PAIR ? 256 : 128, BN);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[STAGES], empty[STAGES], acc_full[2], acc_empty[2], drain;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0;
  const int unit = (int)blockIdx.x / CTAS, units = (int)gridDim.x / CTAS, tiles = g.m_tiles * g.n_tiles;
  int* err = g.p.err;
  const int cw = g.lk.cw, cwb = 2 * cw, per_stage = 64 / cw;

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
    abort_word = 0;
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
  // The list of tile row mb's group, complete once k_lora_down has ended (without adapters
  // there is none).
  auto list_of = [&](int mb) { return g.lk.lists + (PAIR ? mb : mb >> 1); };
  auto chunks_of = [&](int mb) { return g.lk.q_max ? g.lk.chunks(__ldcg(&list_of(mb)->count)) : 0; };

  if (warp == 0) {
    if (lane == 0) {
      const uint32_t full0 = PAIR ? mapa_shared(&full[0], 0) : 0;
      int done = 0;
      bool ok = true;
      auto stage = [&](int bytes, uint8_t*& st) {
        const int s = done % STAGES;
        ok = mbar_wait(&empty[s], ((done / STAGES) & 1) ^ 1u, abort_flag, err, kErrWaitEmpty);
        if (!ok) return false;
        st = smem + s * C_::STAGE;
        if (rank == 0) mbar_arrive_expect_tx(&full[s], CTAS * bytes);
        return true;
      };
      auto load2 = [&](uint8_t* dst, const CUtensorMap* m, int x, int y) {
        const int s = done % STAGES;
        if constexpr (PAIR)
          tma_load_2d_pair(dst, m, full0 + (uint32_t)(s * 8), x, y);
        else
          tma_load_2d(dst, m, &full[s], x, y);
      };
      auto load3 = [&](uint8_t* dst, const CUtensorMap* m, int x, int y, int z) {
        const int s = done % STAGES;
        if constexpr (PAIR)
          tma_load_3d_pair(dst, m, full0 + (uint32_t)(s * 8), x, y, z);
        else
          tma_load_3d(dst, m, &full[s], x, y, z);
      };
      for (int t = unit; t < tiles && ok; t += units) {
        int mb, nb;
        tile_at(t, g.m_tiles, g.n_tiles, mb, nb);
        const int y0 = (mb * CTAS + (int)rank) * 128, n0 = nb * BN + (int)rank * C_::B_ROWS;
        uint8_t* st;
        for (int kb = 0; kb < g.k_blocks; ++kb, ++done) {
          if (!stage(C_::STAGE, st)) break;
          load2(st, &tmX, kb * 64, (int)g.row0 + y0);
          load2(st + C_::A_BYTES, &tmW, kb * 64, n0);
        }
        if (!ok) break;
        asm volatile("griddepcontrol.wait;" ::: "memory");
        const int nq = chunks_of(mb), group = y0 / kGroup;
        for (int q0 = 0; q0 < nq; q0 += per_stage, ++done) {
          const int n = min(per_stage, nq - q0);
          if (!stage(n * (128 + C_::B_ROWS) * cwb, st)) break;
          for (int i = 0; i < n; ++i) {
            const int q = q0 + i, c = q % g.lk.rc, sl = q / (g.lk.rc * g.lk.parts);
            load2(st + i * 128 * cwb, &tmH, 0, (group * g.lk.q_max + q) * kGroup + y0 % kGroup);
            load3(st + C_::A_BYTES + i * C_::B_ROWS * cwb, &tmB, c * cw, n0, __ldcg(&list_of(mb)->adapter[sl]));
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
    if (lane == 0 && rank == 0) {
      int done = 0, n = 0;
      bool ok = true;
      auto mma = [&](uint32_t d, uint64_t a, uint64_t b, bool acc) {
        if constexpr (PAIR)
          umma_f16_ss_pair(d, a, b, IDESC, acc);
        else
          umma_f16_ss(d, a, b, IDESC, acc);
      };
      auto commit = [&](uint64_t* bar) {
        if constexpr (PAIR)
          umma_commit_pair(bar, 0x3);
        else
          umma_commit(bar);
      };
      for (int t = unit; t < tiles && ok; t += units, ++n) {
        const int acc = n & 1;
        ok = mbar_wait(&acc_empty[acc], ((n >> 1) & 1) ^ 1u, abort_flag, err, kErrWaitAccEmpty);
        if (!ok) break;
        tc_fence_after();
        int mb, nb;
        tile_at(t, g.m_tiles, g.n_tiles, mb, nb);
        const uint32_t d = tmem + (uint32_t)(acc * BN);
        for (int kb = 0; kb < g.k_blocks; ++kb, ++done) {
          const int s = done % STAGES;
          ok = mbar_wait(&full[s], (done / STAGES) & 1, abort_flag, err, kErrWaitFull);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a0 = smem_u32(smem + s * C_::STAGE), b0 = a0 + C_::A_BYTES;
#pragma unroll
          for (int k = 0; k < 4; ++k) mma(d, sdesc_k_sw128(a0 + k * 32), sdesc_k_sw128(b0 + k * 32), (kb | k) != 0);
          commit(&empty[s]);
        }
        if (!ok) break;
        asm volatile("griddepcontrol.wait;" ::: "memory");
        const int nq = chunks_of(mb);
        for (int q0 = 0; q0 < nq; q0 += per_stage, ++done) {
          const int s = done % STAGES;
          ok = mbar_wait(&full[s], (done / STAGES) & 1, abort_flag, err, kErrWaitFull);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a0 = smem_u32(smem + s * C_::STAGE), b0 = a0 + C_::A_BYTES;
          for (int i = 0; i < min(per_stage, nq - q0); ++i)
            for (int k = 0; k < cw / 16; ++k)
              mma(d, sdesc_k(a0 + i * 128 * cwb + k * 32, cwb), sdesc_k(b0 + i * C_::B_ROWS * cwb + k * 32, cwb), true);
          commit(&empty[s]);
        }
        if (!ok) break;
        commit(&acc_full[acc]);
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
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int n = 0;
    for (int t = unit; t < tiles; t += units, ++n) {
      const int acc = n & 1;
      int mb, nb;
      tile_at(t, g.m_tiles, g.n_tiles, mb, nb);
      if (!mbar_wait(&acc_full[acc], (n >> 1) & 1, abort_flag, err, kErrWaitAccFull)) break;
      tc_fence_after();
      const int local = (mb * CTAS + (int)rank) * 128 + q * 32 + lane;
      const bool row_ok = local < g.rows, mixed = g.lk.q_max && __ldcg(&list_of(mb)->mixed);
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
        if (row_ok) {
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
          if (g.p.bias) {
            if (g.bias_vec && cols == 32) {
#pragma unroll
              for (int j = 0; j < 32; j += 4) {
                const float4 b = __ldg(reinterpret_cast<const float4*>(g.p.bias + col0 + j));
                v[j] += b.x;
                v[j + 1] += b.y;
                v[j + 2] += b.z;
                v[j + 3] += b.w;
              }
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (j < cols) v[j] += __ldg(g.p.bias + col0 + j);
            }
          }
          if (g.p.y_bf16) {
            uint16_t* y = (uint16_t*)g.p.Y + row * g.p.ldy + col0;
            if (g.y_vec && cols == 32) {
#pragma unroll
              for (int j = 0; j < 32; j += 8)
                *reinterpret_cast<uint4*>(y + j) = make_uint4(pack_bf16x2(v[j], v[j + 1]), pack_bf16x2(v[j + 2], v[j + 3]),
                                                              pack_bf16x2(v[j + 4], v[j + 5]), pack_bf16x2(v[j + 6], v[j + 7]));
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (j < cols) y[j] = f32_to_bf16_rne(v[j]);
            }
          } else {
            float* y = (float*)g.p.Y + row * g.p.ldy + col0;
            if (g.y_vec && cols == 32) {
#pragma unroll
              for (int j = 0; j < 32; j += 4) *reinterpret_cast<float4*>(y + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (j < cols) y[j] = v[j];
            }
          }
        }
        if (mixed) {
          uint32_t bad = 0;
          if (row_ok) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j < cols && (r[j] & 0x7fffffffu) >= 0x7f800000u) bad |= 1u << j;
          }
          __syncwarp();
          if (__any_sync(0xffffffffu, bad != 0))
            redo_chunk(g.p, g.lk, g.X, g.ldx, g.W, g.ldw, g.B, g.ldb, g.row0, local, col0, bad);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR)
          mbar_arrive_cluster(acc_empty0 + (uint32_t)(acc * 8));
        else
          mbar_arrive(&acc_empty[acc]);
      }
    }
  }
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
void launch_lora_gemm(LoraGemm g, int64_t r, bool overlap) {
  using C_ = LoraGemmCfg<BN, PAIR>;
  DeviceContext& c = ctx();
  const CUtensorMapDataType bf = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  CUtensorMap tx, tw, th, tb;
  auto map2 = [&](CUtensorMap* m, const void* x, int64_t k, int64_t rows, int64_t ld, int box_k, int box_rows,
                  CUtensorMapSwizzle sw) {
    const uint64_t dims[2] = {(uint64_t)k, (uint64_t)rows};
    const uint64_t str[1] = {(uint64_t)ld * 2};
    const uint32_t box[2] = {(uint32_t)box_k, (uint32_t)box_rows};
    encode_tmap(m, bf, 2, x, dims, str, box, sw);
  };
  map2(&tx, g.X, g.p.K, g.p.T, g.ldx, 64, 128, CU_TENSOR_MAP_SWIZZLE_128B);
  map2(&tw, g.W, g.p.K, g.p.N, g.ldw, 64, C_::B_ROWS, CU_TENSOR_MAP_SWIZZLE_128B);
  g.m_tiles = (int)((g.rows + (PAIR ? 255 : 127)) / (PAIR ? 256 : 128));
  g.n_tiles = (int)((g.p.N + BN - 1) / BN);
  g.k_blocks = (int)((g.p.K + 63) / 64);
  if (overlap) {
    const int64_t groups = (g.rows + kGroup - 1) / kGroup;
    map2(&th, g.lk.H, g.lk.cw, groups * g.lk.q_max * kGroup, g.lk.cw, g.lk.cw, 128, swizzle_of(g.lk.cw));
    const uint64_t dims[3] = {(uint64_t)r, (uint64_t)g.p.N, (uint64_t)g.p.n_adapters};
    const uint64_t str[2] = {(uint64_t)g.ldb * 2, (uint64_t)g.p.N * g.ldb * 2};
    const uint32_t box[3] = {(uint32_t)g.lk.cw, (uint32_t)C_::B_ROWS, 1};
    encode_tmap(&tb, bf, 3, g.B, dims, str, box, swizzle_of(g.lk.cw));
  } else {
    th = tb = tx;  // no chunk is read
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
  if (overlap) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.numAttrs = n;
  cfg.gridDim = dim3((unsigned)(std::min<int64_t>(clusters[c.device], (int64_t)g.m_tiles * g.n_tiles) * (PAIR ? 2 : 1)));
  check_cuda(cudaLaunchKernelEx(&cfg, kern, tx, tw, th, tb, g), "linear_lora");
  check_launch("linear_lora");
}

// What the large path keeps in the workspace: one block of rows' lists and H.
struct Big {
  LoraK lk;
  int64_t rows;  // rows of a block, a multiple of kGroup
  size_t lists_at, h_at, bytes;
};
Big lay_out_big(const LoraLinear& p, size_t at) {
  Big b{};
  b.lists_at = b.h_at = b.bytes = at;
  b.rows = round_up(p.T, kGroup);
  b.lk.cw = 64;
  if (p.n_adapters <= 0 || p.r <= 0) return b;
  b.lk.parts = p.y_bf16 ? 1 : 2;
  b.lk.cw = p.r <= 16 ? 16 : p.r <= 32 ? 32 : 64;
  b.lk.rc = (int)((p.r + b.lk.cw - 1) / b.lk.cw);
  b.lk.q_max = b.lk.chunks((int)std::min<int64_t>(p.n_adapters, kGroup));
  // H holds every chunk a group could need; blocks of rows keep it within 128 MB.
  const int64_t group = (int64_t)b.lk.q_max * kGroup * b.lk.cw * 2;
  b.rows = std::min(b.rows, std::max<int64_t>(1, ((int64_t)128 << 20) / group) * kGroup);
  b.h_at = at + align256((size_t)(b.rows / kGroup) * sizeof(GroupList));
  b.bytes = b.h_at + align256((size_t)(b.rows / kGroup) * group);
  return b;
}

void launch_big(const LoraLinear& p, const uint16_t* X, int64_t ldx, const uint16_t* W, int64_t ldw, const uint16_t* A,
                int64_t lda, const uint16_t* B, int64_t ldb, uint8_t* ws, const Big& big) {
  DeviceContext& c = ctx();
  const bool adapters = p.n_adapters > 0 && p.r > 0;
  LoraGemm g{};
  g.p = p;
  g.lk = big.lk;
  g.lk.lists = reinterpret_cast<const GroupList*>(ws + big.lists_at);
  g.lk.H = reinterpret_cast<uint16_t*>(ws + big.h_at);
  g.X = X;
  g.W = W;
  g.B = B;
  g.ldx = ldx;
  g.ldw = ldw;
  g.ldb = ldb;
  g.y_vec = aligned16(p.Y) && p.ldy % (p.y_bf16 ? 8 : 4) == 0;
  g.bias_vec = p.bias && aligned16(p.bias);
  for (g.row0 = 0; g.row0 < p.T; g.row0 += big.rows) {
    g.rows = std::min(big.rows, p.T - g.row0);
    if (adapters) {
      const int rpr = (int)round_up(p.r, 16), stages = DownCfg::stages(rpr);
      CUtensorMap tx, ta;
      {
        const uint64_t dims[2] = {(uint64_t)p.K, (uint64_t)p.T};
        const uint64_t str[1] = {(uint64_t)ldx * 2};
        const uint32_t box[2] = {64, 128};
        encode_tmap(&tx, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, X, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
      }
      {
        const uint64_t dims[3] = {(uint64_t)p.K, (uint64_t)p.r, (uint64_t)p.n_adapters};
        const uint64_t str[2] = {(uint64_t)lda * 2, (uint64_t)p.r * lda * 2};
        const uint32_t box[3] = {64, (uint32_t)rpr, 1};
        encode_tmap(&ta, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, A, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
      }
      const int64_t tiles = 2 * ((g.rows + kGroup - 1) / kGroup);
      const int kblocks = (int)((p.K + 63) / 64);
      int splits = 1;
      while (splits < 8 && tiles * splits * 2 <= c.num_sms && kblocks >= 4 * splits) splits *= 2;
      static bool done[64] = {};
      if (!done[c.device]) {
        check_cuda(cudaFuncSetAttribute(k_lora_down, cudaFuncAttributeMaxDynamicSharedMemorySize, 222 * 1024),
                   "cudaFuncSetAttribute(lora_down)");
        done[c.device] = true;
      }
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3((unsigned)(tiles * splits));
      cfg.blockDim = dim3(kRowThreads);
      cfg.dynamicSmemBytes = DownCfg::smem(rpr);
      cfg.stream = c.stream;
      cudaLaunchAttribute attr{};
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = (unsigned)splits;
      attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      check_cuda(cudaLaunchKernelEx(&cfg, k_lora_down, tx, ta, p, (const LoraK)g.lk, const_cast<GroupList*>(g.lk.lists), rpr,
                                    stages, splits, g.row0, g.rows),
                 "lora_down");
      check_launch("lora_down");
    }
    // Tile shape by waves, as gemm_tc.cu prices them: a tile costs its width and 48 columns
    // of fixed cost, a 256 x 256 pair tile 8% less.
    auto waves = [&](int bm, int bn, int64_t units) {
      const int64_t t = ((g.rows + bm - 1) / bm) * ((p.N + bn - 1) / bn);
      return (double)((t + units - 1) / units);
    };
    double best = g.rows > 128 ? waves(256, 256, c.num_sms / 2) * (256 + 48) * 0.92 : 1e30;
    int bn = 0;
    for (int cand : {256, 128, 64}) {
      const double cost = waves(128, cand, c.num_sms) * (cand + 48);
      if (cost < best) {
        best = cost;
        bn = cand;
      }
    }
    if (bn == 0) launch_lora_gemm<256, true>(g, p.r, adapters);
    if (bn == 256) launch_lora_gemm<256, false>(g, p.r, adapters);
    if (bn == 128) launch_lora_gemm<128, false>(g, p.r, adapters);
    if (bn == 64) launch_lora_gemm<64, false>(g, p.r, adapters);
  }
}

}  // namespace

size_t lora_linear_workspace(const LoraLinear& p) {
  const Operands o = lay_out(p);
  return p.T <= kMaxRowsSmall ? o.bytes : lay_out_big(p, o.h_at).bytes;
}

void launch_lora_linear(LoraLinear p, void* ws_) {
  DeviceContext& c = ctx();
  p.err = c.err_word;
  const Operands o = lay_out(p);
  uint8_t* ws = static_cast<uint8_t*>(ws_);
  const uint16_t *X = (const uint16_t*)p.X, *W = p.W, *A = p.A, *B = p.B;
  int64_t ldx = p.ldx, ldw = p.ldw, lda = p.lda, ldb = p.ldb;
  auto take = [&](size_t at) { return reinterpret_cast<uint16_t*>(ws + at); };
  if (o.pack_x) {
    if (p.x_bf16)
      launch_copy2d(p.X, p.ldx, take(o.x_at), o.Kp, p.T, p.K, 2);
    else
      launch_pack_bf16((const float*)p.X, p.ldx, take(o.x_at), o.Kp, p.T, p.K);
    X = take(o.x_at);
    ldx = o.Kp;
  }
  if (o.pack_w) {
    launch_copy2d(W, ldw, take(o.w_at), o.Kp, p.N, p.K, 2);
    W = take(o.w_at);
    ldw = o.Kp;
  }
  if (o.pack_a) {
    launch_copy2d(A, lda, take(o.a_at), o.Kp, p.n_adapters * p.r, p.K, 2);
    A = take(o.a_at);
    lda = o.Kp;
  }
  if (o.pack_b) {
    launch_copy2d(B, ldb, take(o.b_at), o.rb, p.n_adapters * p.N, p.r, 2);
    B = take(o.b_at);
    ldb = o.rb;
  }
  if (p.T > kMaxRowsSmall) return launch_big(p, X, ldx, W, ldw, A, lda, B, ldb, ws, lay_out_big(p, o.h_at));
  float* h = reinterpret_cast<float*>(ws + o.h_at);
  if (p.n_adapters <= 0 || p.r <= 0) {
    p.n_adapters = p.r = 0;
    p.row_adapter = nullptr;
  } else {
    k_lora_down_rows<<<dim3((unsigned)p.T, (unsigned)((p.r + 7) / 8)), 256, 0, c.stream>>>(p, X, ldx, A, lda, h);
    check_launch("lora_down_rows");
  }
  if (p.T <= 16) return launch_rows<16>(p, X, ldx, W, ldw, h);
  if (p.T <= 32) return launch_rows<32>(p, X, ldx, W, ldw, h);
  launch_rows<64>(p, X, ldx, W, ldw, h);
}

}  // namespace sdb
