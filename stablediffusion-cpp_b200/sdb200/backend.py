"""Torch-facing wrappers of the C ABI, named after the reference backend API
(src/backend_cuda.h, namespace sd::cuda) and the tensor ops that call it
(src/tensor.h: linear, attention, rms_norm, ...).

Tensors are CUDA torch tensors used as plain device buffers: fp32 activations
(torch.float32) and bf16 weights (torch.bfloat16, whose bit pattern is the
reference's uint16 bf16). Every call goes through libsdb200.so on the thread's stream
for the current device; the wrappers bind it to torch's current stream first so
CUDA events recorded by torch order correctly with the library's kernels.
"""
from __future__ import annotations

import torch

from . import check, lib


def _p(t):
    return None if t is None else t.data_ptr()


def bind_stream(device=None) -> None:
    """Issues the library's ops for `device` on torch's current stream."""
    if device is not None:
        check(lib().sdb200_set_device(torch.device(device).index or 0))
    s = torch.cuda.current_stream()
    check(lib().sdb200_set_stream(s.cuda_stream))


def _need(t, dtype, name):
    if not t.is_cuda or t.dtype != dtype:
        raise TypeError(f"{name}: expected a CUDA {dtype} tensor, got {t.dtype} on {t.device}")


# ---------------------------------------------------------------------------------
# GEMM (backend_cuda.h:39-43)
# ---------------------------------------------------------------------------------
def gemm_nt_bf16(A, B, bias=None, C=None, accumulate=False, M=None, N=None, K=None, lda=None, ldb=None, ldc=None):
    """C[M,N] = A[M,K] B[N,K]^T (+bias) (+C): A fp32, B bf16. Returns C."""
    _need(A, torch.float32, "A")
    _need(B, torch.bfloat16, "B")
    M = A.shape[0] if M is None else M
    N = B.shape[0] if N is None else N
    K = A.shape[1] if K is None else K
    lda = A.stride(0) if lda is None else lda
    ldb = B.stride(0) if ldb is None else ldb
    if C is None:
        C = torch.empty((M, N), device=A.device, dtype=torch.float32)
    ldc = C.stride(0) if ldc is None else ldc
    bind_stream()
    check(lib().sdb200_gemm_nt_bf16(M, N, K, _p(A), lda, _p(B), ldb, _p(C), ldc, _p(bias), int(accumulate)))
    return C


def gemm_nt_bf16a(A, B, bias=None, C=None, accumulate=False):
    """Same with A already bf16."""
    _need(A, torch.bfloat16, "A")
    _need(B, torch.bfloat16, "B")
    M, K = A.shape
    N = B.shape[0]
    if C is None:
        C = torch.empty((M, N), device=A.device, dtype=torch.float32)
    bind_stream()
    check(lib().sdb200_gemm_nt_bf16a(M, N, K, _p(A), A.stride(0), _p(B), B.stride(0), _p(C), C.stride(0), _p(bias),
                                     int(accumulate)))
    return C


def gemm_nt_f32(A, B, bias=None, C=None, accumulate=False, M=None, N=None, K=None, lda=None, ldb=None, ldc=None):
    """C[M,N] = A[M,K] B[N,K]^T (+bias) (+C), fp32 weights (tf32 tensor cores)."""
    _need(A, torch.float32, "A")
    _need(B, torch.float32, "B")
    M = A.shape[0] if M is None else M
    N = B.shape[0] if N is None else N
    K = A.shape[1] if K is None else K
    lda = A.stride(0) if lda is None else lda
    ldb = B.stride(0) if ldb is None else ldb
    if C is None:
        C = torch.empty((M, N), device=A.device, dtype=torch.float32)
    ldc = C.stride(0) if ldc is None else ldc
    bind_stream()
    check(lib().sdb200_gemm_nt_f32(M, N, K, _p(A), lda, _p(B), ldb, _p(C), ldc, _p(bias), int(accumulate)))
    return C


def gemm_bf16_epilogue(A, B, bias=None, epi=0, y_bf16=False, Y=None):
    """Fused-epilogue GEMM: epi 0 plain, 1 SwiGLU, 2 GEGLU (B rows interleaved in
    blocks of 16, see interleave_gated). A fp32 or bf16."""
    a_bf16 = A.dtype == torch.bfloat16
    _need(B, torch.bfloat16, "B")
    M, K = A.shape
    N = B.shape[0]
    ncols = N if epi == 0 else N // 2
    if Y is None:
        Y = torch.empty((M, ncols), device=A.device, dtype=torch.bfloat16 if y_bf16 else torch.float32)
    bind_stream()
    check(lib().sdb200_gemm_bf16_epilogue(M, N, K, _p(A), A.stride(0), int(a_bf16), _p(B), B.stride(0), _p(Y),
                                          Y.stride(0), int(y_bf16), _p(bias), epi))
    return Y


def gemm_bf16_qkv_rope(X, Wqkv, cos, sin, gq=None, gk=None, bias=None, eps=1e-5):
    """Fused-QKV projection: X [M, K] (fp32 or bf16) times Wqkv [3 Dq, K] (bf16, rows
    q | k | v) (+bias), then the per-head RMS norm (gq / gk) and the interleaved rotary
    embedding (cos / sin [S, 128], row m uses m % S) of q and k. Returns fp16 (q, k, v),
    each [M, Dq]."""
    x_bf16 = X.dtype == torch.bfloat16
    _need(Wqkv, torch.bfloat16, "Wqkv")
    _need(cos, torch.float32, "cos")
    _need(sin, torch.float32, "sin")
    M, K = X.shape
    Dq = Wqkv.shape[0] // 3
    S = cos.shape[0]
    q, k, v = (torch.empty((M, Dq), device=X.device, dtype=torch.float16) for _ in range(3))
    bind_stream()
    check(lib().sdb200_gemm_bf16_qkv_rope(M, K, _p(X), X.stride(0), int(x_bf16), _p(Wqkv), Wqkv.stride(0), _p(bias),
                                          Dq, S, _p(cos), _p(sin), _p(gq), _p(gk), eps, _p(q), _p(k), _p(v)))
    return q, k, v


def interleave_gated(first, second, block=16):
    """Interleaves the rows of two [D, K] weights in blocks of `block`:
    rows [2jb, 2jb+b) from `first`, [2jb+b, 2jb+2b) from `second`. For SwiGLU
    first = gate (w1), second = up (w3); for GEGLU first = value, second = gate.
    Works on 1-D biases too."""
    D = first.shape[0]
    assert second.shape == first.shape and D % block == 0
    rest = first.shape[1:]
    f = first.reshape(D // block, block, *rest)
    s = second.reshape(D // block, block, *rest)
    return torch.stack([f, s], dim=1).reshape(2 * D, *rest).contiguous()


def linear(x, W, b=None):
    """tensor.cpp:481-501 linear(): flattens leading dims, bf16 or fp32 weights."""
    rows = x.numel() // x.shape[-1]
    x2 = x.reshape(rows, x.shape[-1])
    if W.dtype == torch.bfloat16:
        y = gemm_nt_bf16(x2, W, b)
    else:
        y = gemm_nt_f32(x2, W, b)
    return y.reshape(*x.shape[:-1], W.shape[0])


# ---------------------------------------------------------------------------------
# Attention and layers (backend_cuda.h:45-61)
# ---------------------------------------------------------------------------------
def attention(q, k, v, heads, causal=False, kv_heads=0):
    """tensor.cpp:776-810 attention(): q [N,Sq,heads*d], k/v [N,Skv,kv_heads*d]."""
    kv_heads = kv_heads or heads
    N, Sq, inner = q.shape
    Skv = k.shape[1]
    d = inner // heads
    out = torch.empty_like(q)
    bind_stream()
    check(lib().sdb200_attention(_p(q), _p(k), _p(v), _p(out), N, Sq, Skv, heads, kv_heads, d, int(causal)))
    return out


def rms_norm(x, gamma=None, eps=1e-5):
    y = torch.empty_like(x)
    C = x.shape[-1]
    bind_stream()
    check(lib().sdb200_rms_norm(_p(x), _p(y), x.numel() // C, C, _p(gamma), eps))
    return y


def layer_norm(x, gamma=None, beta=None, eps=1e-5):
    y = torch.empty_like(x)
    C = x.shape[-1]
    bind_stream()
    check(lib().sdb200_layer_norm(_p(x), _p(y), x.numel() // C, C, _p(gamma), _p(beta), eps))
    return y


def rms_norm_heads_(x, dim, gamma=None, eps=1e-5):
    bind_stream()
    check(lib().sdb200_rms_norm_heads(_p(x), x.numel() // dim, dim, _p(gamma), eps))
    return x


def rope_(x, dim, cos, sin, interleaved):
    N, S, inner = x.shape
    bind_stream()
    check(lib().sdb200_rope(_p(x), N, S, inner, dim, _p(cos), _p(sin), int(interleaved)))
    return x


def softmax_rows_(x, scale, causal=False):
    bind_stream()
    check(lib().sdb200_softmax_rows(_p(x), x.shape[0], x.shape[1], scale, int(causal)))
    return x


def swiglu(g, u):
    y = torch.empty_like(g)
    bind_stream()
    check(lib().sdb200_swiglu(_p(g), _p(u), _p(y), g.numel()))
    return y


def geglu(x):
    D2 = x.shape[-1]
    y = torch.empty(*x.shape[:-1], D2 // 2, device=x.device, dtype=torch.float32)
    bind_stream()
    check(lib().sdb200_geglu(_p(x), _p(y), x.numel() // D2, D2 // 2))
    return y


def group_norm(x, groups, gamma, beta, eps):
    N, C = x.shape[:2]
    y = torch.empty_like(x)
    bind_stream()
    check(lib().sdb200_group_norm(_p(x), _p(y), N, C, x.numel() // (N * C), groups, _p(gamma), _p(beta), eps))
    return y


def conv2d(x, w, bias, stride, pad):
    N, Cin, H, W = x.shape
    Cout, _, kh, kw = w.shape
    Ho = (H + 2 * pad - kh) // stride + 1
    Wo = (W + 2 * pad - kw) // stride + 1
    out = torch.empty((N, Cout, Ho, Wo), device=x.device, dtype=torch.float32)
    bind_stream()
    check(lib().sdb200_conv2d(_p(x), N, Cin, H, W, _p(w), Cout, kh, kw, _p(bias), stride, pad, _p(out), Ho, Wo))
    return out


# ---------------------------------------------------------------------------------
# Several requests at once: adapters, per-head norms with the rotation, ragged attention
# ---------------------------------------------------------------------------------
_TYPES = (torch.float32, torch.bfloat16, torch.float16)
_F32, _BF16, _I32 = torch.float32, torch.bfloat16, torch.int32
_calls = None


def _serving():
    """The compiled calls (binding/serving_py.cpp), bound to the library's functions."""
    global _calls
    if _calls is None:
        import ctypes
        import os

        path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_serving.so")
        if not os.path.exists(path):
            raise RuntimeError(f"_serving.so not built at {path}; run `make -C stablediffusion-cpp_b200`")
        from . import _serving as module

        L = lib()
        module.bind(*(ctypes.cast(f, ctypes.c_void_p).value for f in (
            L.sdb200_set_stream, L.sdb200_qk_norm_rope, L.sdb200_linear_lora_workspace, L.sdb200_linear_lora,
            L.sdb200_attention_ragged_workspace, L.sdb200_attention_ragged)))
        _calls = module
    return _calls


def _refuse_args(op, like, **tensors):
    """Names what is wrong with the tensors, (tensor, dtype, shape or None) by name: all on
    like's device, which must be the current one, and contiguous where a shape is given."""
    if not like.is_cuda or like.device.index != torch.cuda.current_device():
        raise ValueError(f"{op}: tensors must be on the current CUDA device, got {like.device}")
    for name, (t, dtype, shape) in tensors.items():
        if t is None:
            continue
        if t.dtype != dtype:
            raise TypeError(f"{op}: {name} must be {dtype}, got {t.dtype}")
        if t.device != like.device:
            raise ValueError(f"{op}: {name} is on {t.device}, expected {like.device}")
        if shape is not None and (tuple(t.shape) != tuple(shape) or not t.is_contiguous()):
            raise ValueError(f"{op}: {name} must be contiguous {tuple(shape)}, got {tuple(t.shape)}")


def _refuse_heads(op, **tensors):
    for name, t in tensors.items():
        if t is not None:
            _, h, d = t.shape
            _, head, one = t.stride()
            if (one != 1 and d > 1) or (head != d and h > 1):
                raise ValueError(f"{op}: the heads of {name} must be dense within a row")


def _refuse_rows(op, **tensors):
    for name, t in tensors.items():
        if t is not None and t.stride(1) != 1 and t.shape[1] > 1:
            raise ValueError(f"{op}: the rows of {name} must be dense")


def _refuse_stacks(op, **tensors):
    for name, t in tensors.items():
        n, rows, cols = t.shape
        s0, s1, s2 = t.stride()
        ld = s1 if rows > 1 else s0 if n > 1 else cols
        if t.numel() and ((s2 != 1 and cols > 1) or (n > 1 and s0 != rows * ld)):
            raise ValueError(f"{op}: the adapters of {name} must follow one another in rows of one pitch")


def qk_norm_rope(q, k, cos, sin, gq=None, gk=None, eps=1e-6, pos=None, interleaved=False, out_dtype=None, q_out=None,
                 k_out=None):
    """rms_norm_heads and rope of q [T, heads, d] and k [T, kv_heads, d] in one pass (rows may
    be strided, as views of a fused projection); cos / sin [n_pos, rot] fp32 with rot <= d,
    row pos[t] (int32), or t % n_pos without pos. Returns (q, k) in out_dtype (default: as
    given), or in q_out / k_out, which may be q / k themselves. k may be None."""
    r = (_calls or _serving()).qk_norm_rope(q, k, cos, sin, gq, gk, eps, pos, interleaved, out_dtype, q_out, k_out)
    if r.__class__ is tuple:
        return r
    if r is not None:
        check(r)
    op, dtype = "qk_norm_rope", q.dtype
    if dtype not in _TYPES or q.dim() != 3:
        raise TypeError(f"{op}: q must be [T, heads, d] fp32, bf16 or fp16, got {dtype} {tuple(q.shape)}")
    T, _, d = q.shape
    out_dtype = out_dtype or (q_out.dtype if q_out is not None else dtype)
    if out_dtype not in _TYPES:
        raise TypeError(f"{op}: output type {out_dtype}")
    if cos.dim() != 2:
        raise ValueError(f"{op}: cos must be [n_pos, rot]")
    _refuse_args(op, q, k=(k, dtype, None), cos=(cos, _F32, cos.shape), sin=(sin, _F32, cos.shape), gq=(gq, _F32, (d,)),
                 gk=(gk, _F32, (d,)), pos=(pos, _I32, (T,)), q_out=(q_out, out_dtype, None), k_out=(k_out, out_dtype, None))
    if k is not None and (k.dim() != 3 or k.shape[0] != T or k.shape[2] != d):
        raise ValueError(f"{op}: k must be [{T}, kv_heads, {d}], got {tuple(k.shape)}")
    if q_out is not None and q_out.shape != q.shape:
        raise ValueError(f"{op}: q_out must have the shape of q")
    if k is not None and k_out is not None and k_out.shape != k.shape:
        raise ValueError(f"{op}: k_out must have the shape of k")
    _refuse_heads(op, q=q, k=k, q_out=q_out, k_out=k_out)
    raise TypeError(f"{op}: an argument is not of its kind")


def linear_lora(x, W, A, B, rows, scale=None, bias=None, out_dtype=torch.float32, out=None):
    """x W^T (+ bias) + scale[a] (x A[a]^T) B[a]^T with a = rows[t] for row t (int32, < 0: no
    adapter). x [T, K] bf16 or fp32 (rounded to bf16), W [N, K], A [n, r, K], B [n, N, r] bf16,
    scale [n] and bias [N] fp32. Returns [T, N] in out_dtype (fp32 or bf16), or out. For a bf16 result
    scale[a] (x A[a]^T) is rounded to bf16 before it meets B; for an fp32 one to 2^-16."""
    r = (_calls or _serving()).linear_lora(x, W, A, B, rows, scale, bias, out_dtype, out)
    if r is not None and r.__class__ is not int:
        return r
    if r is not None:
        check(r)
    op = "linear_lora"
    if x.dtype not in (_F32, _BF16) or x.dim() != 2 or W.dim() != 2 or A.dim() != 3 or B.dim() != 3:
        raise TypeError(f"{op}: x [T, K] fp32 or bf16, W [N, K], A [n, r, K], B [n, N, r]")
    T, K = x.shape
    N, (n, r, Ka) = W.shape[0], A.shape
    if W.shape[1] != K or Ka != K or B.shape != (n, N, r):
        raise ValueError(f"{op}: shapes {tuple(x.shape)}, {tuple(W.shape)}, {tuple(A.shape)}, {tuple(B.shape)}")
    if out is not None:
        out_dtype = out.dtype
    if out_dtype not in (_F32, _BF16):
        raise TypeError(f"{op}: output type {out_dtype}")
    _refuse_args(op, x, W=(W, _BF16, None), A=(A, _BF16, None), B=(B, _BF16, None), rows=(rows, _I32, (T,)),
                 scale=(scale, _F32, (n,)), bias=(bias, _F32, (N,)), out=(out, out_dtype, None))
    if out is not None and out.shape != (T, N):
        raise ValueError(f"{op}: out must be [{T}, {N}]")
    _refuse_rows(op, x=x, W=W, out=out)
    _refuse_stacks(op, A=A, B=B)
    raise TypeError(f"{op}: an argument is not of its kind")


def attention_ragged(q, k, v, q_begin, q_len, kv_begin, kv_len, max_q, max_kv, scale=None, causal=False, prefix=None,
                     cap=0.0, slopes=None, out_dtype=None, out=None):
    """Attention of sequences of their own lengths: sequence s reads query rows
    q_begin[s] .. + q_len[s] of q [Tq, heads, d] and key rows kv_begin[s] .. + kv_len[s] of
    k, v [Tkv, kv_heads, d] (bf16 or fp16; rows may be strided), at most max_q and max_kv long.
    Query i stands at position i + kv_len - q_len; causal hides later keys except the first
    prefix[s]; cap > 0 turns a score z into cap tanh(z / cap); slopes [heads] subtract
    slope * distance. scale defaults to 1 / sqrt(d). Returns out [Tq, heads, d] in out_dtype
    (bf16 or fp16, default as q); rows of no sequence keep what out held (zeros without out).
    Fast for d <= 128, a multiple of 8, in aligned rows; single tokens over long caches want the
    least max_q that holds."""
    r = (_calls or _serving()).attention_ragged(q, k, v, q_begin, q_len, kv_begin, kv_len, max_q, max_kv, scale, causal,
                                                prefix, cap, slopes, out_dtype, out)
    if r is not None and r.__class__ is not int:
        return r
    if r is not None:
        check(r)
    op, dtype = "attention_ragged", q.dtype
    if dtype not in (_BF16, torch.float16) or q.dim() != 3 or k.dim() != 3:
        raise TypeError(f"{op}: q, k, v must be [T, heads, d] bf16 or fp16, got {dtype}")
    if k.shape[2] != q.shape[2] or v.shape != k.shape:
        raise ValueError(f"{op}: shapes {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    out_dtype = out.dtype if out is not None else (out_dtype or dtype)
    if out_dtype not in (_BF16, torch.float16):
        raise TypeError(f"{op}: output type {out_dtype}")
    one = (q_begin.numel(),)
    _refuse_args(op, q, k=(k, dtype, None), v=(v, dtype, None), q_begin=(q_begin, _I32, one), q_len=(q_len, _I32, one),
                 kv_begin=(kv_begin, _I32, one), kv_len=(kv_len, _I32, one), prefix=(prefix, _I32, one),
                 slopes=(slopes, _F32, (q.shape[1],)), out=(out, out_dtype, None))
    if out is not None and out.shape != q.shape:
        raise ValueError(f"{op}: out must have the shape of q")
    _refuse_heads(op, q=q, k=k, v=v, out=out)
    raise TypeError(f"{op}: an argument is not of its kind")


def mul_rows_(x, v):
    bind_stream()
    check(lib().sdb200_mul_rows(_p(x), _p(v), x.numel() // v.numel(), v.numel()))
    return x


def add_rows_scaled_(x, y, g):
    bind_stream()
    check(lib().sdb200_add_rows_scaled(_p(x), _p(y), _p(g), x.numel() // g.numel(), g.numel()))
    return x


def unary_(name, x):
    bind_stream()
    check(getattr(lib(), "sdb200_" + name)(_p(x), x.numel()))
    return x


def synchronize():
    check(lib().sdb200_synchronize())


def device_error_word() -> int:
    import ctypes

    w = ctypes.c_int(0)
    check(lib().sdb200_device_error_word(ctypes.byref(w)))
    return w.value
