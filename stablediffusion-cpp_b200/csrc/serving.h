// serving.h - launchers of the operators for several requests at once (serving_api.cu
// checks their arguments): per-head norms with the rotation, low-rank adapters beside a
// shared projection, attention of sequences with their own lengths.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace sdb {

enum : int { kF32 = 0, kBF16 = 1, kF16 = 2 };  // SDB200_F32, SDB200_BF16, SDB200_F16

struct QkNormRope {
  int64_t T;
  const void* q;
  const void* k;
  int64_t ldq, ldk;
  int heads, kv_heads;
  int d, rot;
  const float* gq;  // [d] or null (1)
  const float* gk;
  float eps;
  const float* cos;  // [n_pos, rot]
  const float* sin;
  int64_t n_pos;
  const int32_t* pos;  // [T] or null: row t uses table row t % n_pos
  int interleaved;
  void* q_out;
  void* k_out;
  int64_t ldqo, ldko;
  int* err;
};
void launch_qk_norm_rope(QkNormRope p, int in_type, int out_type);

struct LoraLinear {
  int64_t T, N, K;
  const void* X;
  int64_t ldx;
  bool x_bf16;
  const uint16_t* W;
  int64_t ldw;
  const float* bias;            // [N] or null
  const int32_t* row_adapter;   // [T], < 0: none
  int64_t n_adapters, r;
  const uint16_t* A;            // [n_adapters, r, lda]
  int64_t lda;
  const uint16_t* B;            // [n_adapters, N, ldb]
  int64_t ldb;
  const float* scale;           // [n_adapters] or null (1)
  void* Y;
  int64_t ldy;
  bool y_bf16;
  int* err;
};
size_t lora_linear_workspace(const LoraLinear& p);
void launch_lora_linear(LoraLinear p, void* ws);

struct RaggedAttention {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  int64_t ldq, ldk, ldv, ldo;
  int in_type, out_type;
  int64_t Tq, Tkv;
  int n_seq;
  const int32_t* q_begin;
  const int32_t* q_len;
  const int32_t* kv_begin;
  const int32_t* kv_len;
  int64_t max_q, max_kv;
  int heads, kv_heads, d;
  float scale, cap;
  const float* slopes;     // [heads] or null
  int causal;
  const int32_t* prefix;   // [n_seq] or null
  int* err;
};
size_t ragged_attention_workspace(const RaggedAttention& p);
void launch_ragged_attention(RaggedAttention p, void* ws);

}  // namespace sdb
