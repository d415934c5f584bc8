// serving_api.cu - C ABI of the operators for several requests at once: argument checks
// and dispatch (serving.h). Index and length arrays live on the device and are checked
// there: a value outside its range sets the device error word, its row or sequence is
// skipped, and the next sdb200_synchronize reports it.
#include <algorithm>
#include <cmath>
#include <string>

#include "internal.h"
#include "sdb200.h"
#include "serving.h"

namespace sdb {
namespace {

constexpr int64_t kMaxRows = (int64_t)1 << 31;

// Messages are put together where a check fails only: a call makes dozens.
void require(bool ok, const char* op, const char* what) {
  if (!ok) fail(kErrInvalidArg, std::string(op) + ": " + what);
}
void require_workspace(int64_t got, int64_t need, const char* op) {
  if (got < need) fail(kErrInvalidArg, std::string(op) + ": workspace of " + std::to_string(need) + " bytes needed");
}
void require_ptr(const void* p, int64_t align, const char* op, const char* name) {
  if (!p) fail(kErrInvalidArg, std::string(op) + ": null pointer " + name);
  if (reinterpret_cast<uintptr_t>(p) % align) fail(kErrInvalidArg, std::string(op) + ": misaligned pointer " + name);
}
int64_t esize(int type) { return type == kF32 ? 4 : 2; }

// Memory that a call reads or writes: `rows` rows of `bytes` bytes, `pitch` bytes apart.
struct Rows {
  const void* p;
  int64_t rows, pitch, bytes;
};
Rows vec(const void* p, int64_t bytes) { return Rows{p, 1, bytes, bytes}; }
// Whether two share bytes; rows of one pitch may lie side by side.
bool share(const Rows& x, const Rows& y) {
  if (!x.p || !y.p || x.rows <= 0 || y.rows <= 0 || x.bytes <= 0 || y.bytes <= 0) return false;
  const char *x0 = (const char*)x.p, *y0 = (const char*)y.p;
  if (y0 + (y.rows - 1) * y.pitch + y.bytes <= x0 || x0 + (x.rows - 1) * x.pitch + x.bytes <= y0) return false;
  if (x.pitch != y.pitch) return true;
  const int64_t off = (((y0 - x0) % x.pitch) + x.pitch) % x.pitch;
  return off < x.bytes || off + y.bytes > x.pitch;
}
void require_apart(const char* op, const char* out_name, const Rows& out, const char* name, const Rows& x) {
  if (share(out, x)) fail(kErrInvalidArg, std::string(op) + ": " + out_name + " overlaps " + name);
}
bool same(const Rows& x, const Rows& y) { return x.p == y.p && x.pitch == y.pitch && x.bytes == y.bytes; }

void check_lora(const LoraLinear& p) {
  const char* op = "linear_lora";
  require(p.T >= 0 && p.N >= 0 && p.K > 0 && p.n_adapters >= 0 && p.r >= 0, op, "bad shape");
  // A tile may end up to 512 rows or columns past the last one; that is still an int.
  require(std::max({p.T, p.N, p.K, p.n_adapters}) < kMaxRows - 512, op, "dimension >= 2^31 - 512");
  require(p.r <= 256, op, "rank > 256");
  if (p.T == 0 || p.N == 0) return;
  require(p.ldx >= p.K && p.ldw >= p.K && p.ldy >= p.N, op, "leading dimension too small");
  require_ptr(p.X, p.x_bf16 ? 2 : 4, op, "X");
  require_ptr(p.W, 2, op, "W");
  if (p.bias) require_ptr(p.bias, 4, op, "bias");
  if (p.n_adapters > 0 && p.r > 0) {
    require(p.lda >= p.K && p.ldb >= p.r, op, "adapter leading dimension too small");
    require_ptr(p.row_adapter, 4, op, "row_adapter");
    require_ptr(p.A, 2, op, "A");
    require_ptr(p.B, 2, op, "B");
    if (p.scale) require_ptr(p.scale, 4, op, "scale");
  }
}

LoraLinear lora_args(int64_t T, int64_t N, int64_t K, const void* X, int64_t ldx, int x_bf16, const uint16_t* W,
                     int64_t ldw, const float* bias, const int32_t* row_adapter, int64_t n_adapters, int64_t r,
                     const uint16_t* A, int64_t lda, const uint16_t* B, int64_t ldb, const float* scale, void* Y,
                     int64_t ldy, int y_bf16) {
  return LoraLinear{T, N, K, X, ldx, x_bf16 != 0, W, ldw, bias, row_adapter, n_adapters, r, A, lda, B, ldb, scale, Y,
                    ldy, y_bf16 != 0, nullptr};
}

void check_attention(const RaggedAttention& p) {
  const char* op = "attention_ragged";
  require(p.in_type == kBF16 || p.in_type == kF16, op, "operands must be bf16 or fp16");
  require(p.out_type == kBF16 || p.out_type == kF16, op, "output must be bf16 or fp16");
  require(p.n_seq >= 0 && p.n_seq <= 65535, op, "n_seq must be 0..65535");
  require(p.Tq >= 0 && p.Tkv >= 0 && p.max_q >= 0 && p.max_kv >= 0, op, "bad shape");
  // A tile may end up to 256 rows past the last one; that is still an int.
  require(p.Tq < kMaxRows - 256 && p.Tkv < kMaxRows - 256, op, "row count >= 2^31 - 256");
  require(p.heads > 0 && p.kv_heads > 0 && p.heads % p.kv_heads == 0, op, "heads must be a multiple of kv_heads");
  require(p.heads <= 65535 && p.heads / p.kv_heads <= 128, op, "too many heads");
  require(p.d > 0 && p.d <= 256, op, "head width must be 1..256");
  require(std::isfinite(p.scale) && p.scale > 0.0f, op, "scale must be positive and finite");
  require(std::isfinite(p.cap) && p.cap >= 0.0f, op, "cap must be 0 (off) or positive and finite");
  // The kernels multiply scores with these; an infinite one makes NaN of 0, a subnormal one has lost its digits.
  const float log2e = 1.4426950f;
  bool usable = std::isnormal(p.scale) && std::isnormal(p.scale * log2e);
  if (p.cap > 0.0f)
    for (const float x : {p.scale / p.cap, p.cap / p.scale, 2.0f * log2e * p.scale / p.cap, p.cap * log2e, p.cap * 1e-3f})
      usable = usable && std::isnormal(x);
  require(usable, op, "scale and cap leave fp32's range");
  require(!p.prefix || p.causal, op, "a prefix needs the causal mask");
}

}  // namespace
}  // namespace sdb

using namespace sdb;

#define SDB_GUARD(...)                  \
  try {                                 \
    __VA_ARGS__;                        \
    return kOk;                         \
  } catch (const sdb::Error& e) {       \
    sdb::set_last_error(e.msg);         \
    return e.code;                      \
  } catch (const std::exception& e) {   \
    sdb::set_last_error(e.what());      \
    return kErrCuda;                    \
  }

extern "C" {

int sdb200_qk_norm_rope(int64_t T, const void* q, int64_t ldq, int heads, const void* k, int64_t ldk, int kv_heads,
                        int in_type, int64_t d, int64_t rot, const float* gq, const float* gk, float eps,
                        const float* cos, const float* sin, int64_t n_pos, const int32_t* pos, int interleaved,
                        void* q_out, int64_t ldqo, void* k_out, int64_t ldko, int out_type) {
  SDB_GUARD({
    const char* op = "qk_norm_rope";
    require(in_type >= kF32 && in_type <= kF16 && out_type >= kF32 && out_type <= kF16, op, "unknown element type");
    require(T >= 0 && T < kMaxRows && heads >= 0 && kv_heads >= 0 && heads + kv_heads > 0, op, "bad shape");
    require(d > 0 && d <= 1024, op, "head width must be 1..1024");
    require(rot >= 0 && rot <= d && rot % 2 == 0, op, "rot must be even and at most d");
    require((int64_t)heads + kv_heads <= 65535, op, "too many heads");
    if (T == 0) return kOk;
    const int64_t ei = esize(in_type);
    const int64_t eo = esize(out_type);
    const Rows rq{heads ? q : nullptr, T, ldq * ei, heads * d * ei};
    const Rows rk{kv_heads ? k : nullptr, T, ldk * ei, kv_heads * d * ei};
    const Rows rqo{heads ? q_out : nullptr, T, ldqo * eo, heads * d * eo};
    const Rows rko{kv_heads ? k_out : nullptr, T, ldko * eo, kv_heads * d * eo};
    if (heads) {
      require(ldq >= heads * d && ldqo >= heads * d, op, "row pitch of q smaller than heads * d");
      require_ptr(q, ei, op, "q");
      require_ptr(q_out, eo, op, "q_out");
      if (!same(rq, rqo)) require_apart(op, "q_out", rqo, "q (and is not q itself)", rq);
      require(q != q_out || in_type == out_type, op, "in place needs one type");
    }
    if (kv_heads) {
      require(ldk >= kv_heads * d && ldko >= kv_heads * d, op, "row pitch of k smaller than kv_heads * d");
      require_ptr(k, ei, op, "k");
      require_ptr(k_out, eo, op, "k_out");
      if (!same(rk, rko)) require_apart(op, "k_out", rko, "k (and is not k itself)", rk);
      require(k != k_out || in_type == out_type, op, "in place needs one type");
    }
    if (gq) require_ptr(gq, 4, op, "gq");
    if (gk) require_ptr(gk, 4, op, "gk");
    if (rot) {
      require_ptr(cos, 4, op, "cos");
      require_ptr(sin, 4, op, "sin");
      require(n_pos > 0 && n_pos < kMaxRows, op, "n_pos must be positive");
    }
    if (pos) require_ptr(pos, 4, op, "pos");
    // Warps write q_out and k_out while others still read the rest.
    require_apart(op, "q_out", rqo, "k", rk);
    require_apart(op, "k_out", rko, "q", rq);
    require_apart(op, "k_out", rko, "q_out", rqo);
    const int64_t table = rot ? n_pos * rot * 4 : 0;
    auto apart = [&](const char* name, const void* x, int64_t bytes) {
      require_apart(op, "q_out", rqo, name, vec(x, bytes));
      require_apart(op, "k_out", rko, name, vec(x, bytes));
    };
    apart("cos", cos, table);
    apart("sin", sin, table);
    apart("gq", gq, d * 4);
    apart("gk", gk, d * 4);
    apart("pos", pos, T * 4);
    QkNormRope p{T, q, k, ldq, ldk, heads, kv_heads, (int)d, (int)rot, gq, gk, eps, cos, sin, rot ? n_pos : T,
                 rot ? pos : nullptr, interleaved != 0, q_out, k_out, ldqo, ldko, nullptr};
    launch_qk_norm_rope(p, in_type, out_type);
  })
}

int64_t sdb200_linear_lora_workspace(int64_t T, int64_t N, int64_t K, const void* X, int64_t ldx, int x_bf16,
                                     const uint16_t* W, int64_t ldw, int64_t n_adapters, int64_t r, const uint16_t* A,
                                     int64_t lda, const uint16_t* B, int64_t ldb) {
  try {
    require(K > 0 && n_adapters >= 0 && r >= 0 && r <= 256 && std::max({T, N, K, n_adapters}) < kMaxRows - 512, "linear_lora",
            "bad shape");
    if (T <= 0 || N <= 0) return 0;
    // For either type of Y: an fp32 one has more chunks to a group of rows and so fewer groups at a
    // time, a bf16 one longer lists.
    size_t need = 0;
    for (int y_bf16 = 0; y_bf16 < 2; ++y_bf16)
      need = std::max(need, lora_linear_workspace(lora_args(T, N, K, X, ldx, x_bf16, W, ldw, nullptr, nullptr, n_adapters, r,
                                                            A, lda, B, ldb, nullptr, nullptr, N, y_bf16)));
    return (int64_t)need;
  } catch (const sdb::Error& e) {
    sdb::set_last_error(e.msg);
    return -1;
  } catch (const std::exception& e) {
    sdb::set_last_error(e.what());
    return -1;
  }
}

int sdb200_linear_lora(int64_t T, int64_t N, int64_t K, const void* X, int64_t ldx, int x_bf16, const uint16_t* W,
                       int64_t ldw, const float* bias, const int32_t* row_adapter, int64_t n_adapters, int64_t r,
                       const uint16_t* A, int64_t lda, const uint16_t* B, int64_t ldb, const float* scale, void* Y,
                       int64_t ldy, int y_bf16, void* ws, int64_t ws_bytes) {
  SDB_GUARD({
    const char* op = "linear_lora";
    LoraLinear p = lora_args(T, N, K, X, ldx, x_bf16, W, ldw, bias, row_adapter, n_adapters, r, A, lda, B, ldb, scale,
                             Y, ldy, y_bf16);
    check_lora(p);
    if (T == 0 || N == 0) return kOk;
    require_ptr(Y, p.y_bf16 ? 2 : 4, op, "Y");
    const int64_t ey = p.y_bf16 ? 2 : 4;
    const int64_t ex = p.x_bf16 ? 2 : 4;
    const bool adapters = n_adapters > 0 && r > 0;
    const Rows y{Y, T, ldy * ey, N * ey};
    const struct {
      const char* name;
      Rows at;
    } inputs[] = {{"X", {X, T, ldx * ex, K * ex}},
                  {"W", {W, N, ldw * 2, K * 2}},
                  {"A", {adapters ? A : nullptr, n_adapters * r, lda * 2, K * 2}},
                  {"B", {adapters ? B : nullptr, n_adapters * N, ldb * 2, r * 2}},
                  {"bias", vec(bias, N * 4)},
                  {"row_adapter", vec(adapters ? row_adapter : nullptr, T * 4)},
                  {"scale", vec(adapters ? scale : nullptr, n_adapters * 4)}};
    for (const auto& x : inputs) require_apart(op, "Y", y, x.name, x.at);
    const int64_t need = (int64_t)lora_linear_workspace(p);
    require_workspace(ws_bytes, need, op);
    if (need) {
      require_ptr(ws, 256, op, "ws");
      require_apart(op, "Y", y, "ws", vec(ws, need));
      for (const auto& x : inputs) require_apart(op, "ws", vec(ws, need), x.name, x.at);
    }
    launch_lora_linear(p, ws);
  })
}

static RaggedAttention attention_args(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v,
                                      int64_t ldv, int in_type, void* out, int64_t ldo, int out_type, int64_t Tq,
                                      int64_t Tkv, int n_seq, const int32_t* q_begin, const int32_t* q_len,
                                      const int32_t* kv_begin, const int32_t* kv_len, int64_t max_q, int64_t max_kv,
                                      int heads, int kv_heads, int64_t d, float scale, float cap, const float* slopes,
                                      int causal, const int32_t* prefix) {
  return RaggedAttention{q, k, v, out, ldq, ldk, ldv, ldo, in_type, out_type, Tq, Tkv, n_seq, q_begin, q_len, kv_begin,
                         kv_len, std::min(max_q, kMaxRows), std::min(max_kv, kMaxRows), heads, kv_heads,
                         (int)std::min<int64_t>(d, 1 << 30), scale, cap, slopes, causal != 0, prefix, nullptr};
}

int64_t sdb200_attention_ragged_workspace(int n_seq, int64_t max_q, int64_t max_kv, int heads, int kv_heads,
                                          int64_t d) {
  try {
    RaggedAttention p = attention_args(nullptr, 0, nullptr, 0, nullptr, 0, kBF16, nullptr, 0, kBF16, 0, 0, n_seq,
                                       nullptr, nullptr, nullptr, nullptr, max_q, max_kv, heads, kv_heads, d, 1.0f,
                                       0.0f, nullptr, 0, nullptr);
    check_attention(p);
    if (n_seq == 0 || max_q == 0) return 0;
    return (int64_t)ragged_attention_workspace(p);
  } catch (const sdb::Error& e) {
    sdb::set_last_error(e.msg);
    return -1;
  } catch (const std::exception& e) {
    sdb::set_last_error(e.what());
    return -1;
  }
}

int sdb200_attention_ragged(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv,
                            int in_type, void* out, int64_t ldo, int out_type, int64_t Tq, int64_t Tkv, int n_seq,
                            const int32_t* q_begin, const int32_t* q_len, const int32_t* kv_begin,
                            const int32_t* kv_len, int64_t max_q, int64_t max_kv, int heads, int kv_heads, int64_t d,
                            float scale, float cap, const float* slopes, int causal, const int32_t* prefix, void* ws,
                            int64_t ws_bytes) {
  SDB_GUARD({
    const char* op = "attention_ragged";
    RaggedAttention p = attention_args(q, ldq, k, ldk, v, ldv, in_type, out, ldo, out_type, Tq, Tkv, n_seq, q_begin,
                                       q_len, kv_begin, kv_len, max_q, max_kv, heads, kv_heads, d, scale, cap, slopes,
                                       causal, prefix);
    check_attention(p);
    if (n_seq == 0 || max_q == 0 || Tq == 0) return kOk;
    require_ptr(q_begin, 4, op, "q_begin");
    require_ptr(q_len, 4, op, "q_len");
    require_ptr(kv_begin, 4, op, "kv_begin");
    require_ptr(kv_len, 4, op, "kv_len");
    require(ldq >= heads * d && ldo >= heads * d, op, "row pitch smaller than heads * d");
    require_ptr(q, 2, op, "q");
    require_ptr(out, 2, op, "out");
    if (p.max_kv > 0 && Tkv > 0) {
      require(ldk >= kv_heads * d && ldv >= kv_heads * d, op, "row pitch smaller than kv_heads * d");
      require_ptr(k, 2, op, "k");
      require_ptr(v, 2, op, "v");
    }
    const Rows o{out, Tq, ldo * 2, heads * d * 2};
    const bool keys = p.max_kv > 0 && Tkv > 0;
    const int64_t per_seq = (int64_t)n_seq * 4;
    const struct {
      const char* name;
      Rows at;
    } inputs[] = {{"q", {q, Tq, ldq * 2, heads * d * 2}},
                  {"k", {keys ? k : nullptr, Tkv, ldk * 2, kv_heads * d * 2}},
                  {"v", {keys ? v : nullptr, Tkv, ldv * 2, kv_heads * d * 2}},
                  {"q_begin", vec(q_begin, per_seq)},
                  {"q_len", vec(q_len, per_seq)},
                  {"kv_begin", vec(kv_begin, per_seq)},
                  {"kv_len", vec(kv_len, per_seq)},
                  {"slopes", vec(slopes, (int64_t)heads * 4)},
                  {"prefix", vec(prefix, per_seq)}};
    if (slopes) require_ptr(slopes, 4, op, "slopes");
    if (prefix) require_ptr(prefix, 4, op, "prefix");
    for (const auto& x : inputs) require_apart(op, "out", o, x.name, x.at);
    const int64_t need = (int64_t)ragged_attention_workspace(p);
    require_workspace(ws_bytes, need, op);
    if (need) {
      require_ptr(ws, 256, op, "ws");
      require_apart(op, "out", o, "ws", vec(ws, need));
      for (const auto& x : inputs) require_apart(op, "ws", vec(ws, need), x.name, x.at);
    }
    launch_ragged_attention(p, ws);
  })
}

}  // extern "C"
