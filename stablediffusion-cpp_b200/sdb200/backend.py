"""Torch-facing wrappers of the C ABI, named after the reference backend API
(src/backend_cuda.h, namespace sd::cuda) and the tensor ops that call it
(src/tensor.h: linear, attention, rms_norm, ...).

Tensors are CUDA torch tensors used as plain device buffers: fp32 activations
(torch.float32) and bf16 weights (torch.bfloat16, whose bit pattern is the
reference's uint16 bf16). Every call goes through libsdb200.so on the current
device's stream; the wrappers bind that stream to torch's current stream first so
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
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _check_args(op, like, **tensors):
    """Every tensor on `like`'s device, which must be the current one. (name, dtype, shape)
    triples; None tensors are skipped, a shape of None is not checked."""
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


def _head_pitch(op, name, t):
    """Row pitch (elements) of [T, heads, d] whose heads lie next to each other."""
    T, h, d = t.shape
    if (d > 1 and t.stride(2) != 1) or (h > 1 and t.stride(1) != d):
        raise ValueError(f"{op}: the heads of {name} must be dense within a row")
    return t.stride(0) if T > 1 else max(t.stride(0), h * d)


def qk_norm_rope(q, k, cos, sin, gq=None, gk=None, eps=1e-6, pos=None, interleaved=False, out_dtype=None, q_out=None,
                 k_out=None):
    """rms_norm_heads and rope of q [T, heads, d] and k [T, kv_heads, d] in one pass (rows may
    be strided, as views of a fused projection); cos / sin [n_pos, rot] fp32 with rot <= d,
    row pos[t] (int32), or t % n_pos without pos. Returns (q, k) in out_dtype (default: as
    given), or in q_out / k_out, which may be q / k themselves. k may be None."""
    op = "qk_norm_rope"
    if q.dtype not in _TYPES or q.dim() != 3:
        raise TypeError(f"{op}: q must be [T, heads, d] fp32, bf16 or fp16, got {q.dtype} {tuple(q.shape)}")
    T, heads, d = q.shape
    out_dtype = out_dtype or (q_out.dtype if q_out is not None else q.dtype)
    if out_dtype not in _TYPES:
        raise TypeError(f"{op}: output type {out_dtype}")
    if cos.dim() != 2:
        raise ValueError(f"{op}: cos must be [n_pos, rot]")
    _check_args(op, q, k=(k, q.dtype, None), cos=(cos, torch.float32, cos.shape), sin=(sin, torch.float32, cos.shape),
                gq=(gq, torch.float32, (d,)), gk=(gk, torch.float32, (d,)), pos=(pos, torch.int32, (T,)),
                q_out=(q_out, out_dtype, None), k_out=(k_out, out_dtype, None))
    if q_out is None:
        q_out = torch.empty((T, heads, d), device=q.device, dtype=out_dtype)
    kv, ldk, ldko = 0, 0, 0
    if k is not None:
        if k.dim() != 3 or k.shape[0] != T or k.shape[2] != d:
            raise ValueError(f"{op}: k must be [{T}, kv_heads, {d}], got {tuple(k.shape)}")
        if k_out is None:
            k_out = torch.empty(k.shape, device=q.device, dtype=out_dtype)
        if k_out.shape != k.shape:
            raise ValueError(f"{op}: k_out must have the shape of k")
        kv, ldk, ldko = k.shape[1], _head_pitch(op, "k", k), _head_pitch(op, "k_out", k_out)
    if q_out.shape != q.shape:
        raise ValueError(f"{op}: q_out must have the shape of q")
    bind_stream()
    check(lib().sdb200_qk_norm_rope(T, q.data_ptr(), _head_pitch(op, "q", q), heads, _p(k), ldk, kv, _TYPES[q.dtype],
                                    d, cos.shape[1], _p(gq), _p(gk), eps, cos.data_ptr(), sin.data_ptr(), cos.shape[0],
                                    _p(pos), int(interleaved), q_out.data_ptr(), _head_pitch(op, "q_out", q_out),
                                    _p(k_out) if k is not None else None, ldko, _TYPES[out_dtype]))
    return q_out, (k_out if k is not None else None)


def linear_lora(x, W, A, B, rows, scale=None, bias=None, out_dtype=torch.float32, out=None):
    """x W^T (+ bias) + scale[a] (x A[a]^T) B[a]^T with a = rows[t] for row t (int32, < 0: no
    adapter). x [T, K] bf16 or fp32 (rounded to bf16), W [N, K], A [n, r, K], B [n, N, r] bf16,
    scale [n] and bias [N] fp32. Returns [T, N] in out_dtype (fp32 or bf16), or out."""
    op = "linear_lora"
    if x.dtype not in (torch.float32, torch.bfloat16) or x.dim() != 2 or W.dim() != 2 or A.dim() != 3 or B.dim() != 3:
        raise TypeError(f"{op}: x [T, K] fp32 or bf16, W [N, K], A [n, r, K], B [n, N, r]")
    T, K = x.shape
    N, (n, r) = W.shape[0], A.shape[:2]
    if W.shape[1] != K or A.shape[2] != K or B.shape != (n, N, r):
        raise ValueError(f"{op}: shapes {tuple(x.shape)}, {tuple(W.shape)}, {tuple(A.shape)}, {tuple(B.shape)}")
    if out is not None:
        out_dtype = out.dtype
    if out_dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"{op}: output type {out_dtype}")
    bf = torch.bfloat16
    _check_args(op, x, W=(W, bf, None), A=(A, bf, None), B=(B, bf, None), rows=(rows, torch.int32, (T,)),
                scale=(scale, torch.float32, (n,)), bias=(bias, torch.float32, (N,)), out=(out, out_dtype, None))
    for name, t in (("x", x), ("W", W)):
        if t.shape[1] > 1 and t.stride(1) != 1:
            raise ValueError(f"{op}: the rows of {name} must be dense")
    pitch = []
    for name, t in (("A", A), ("B", B)):
        ld = t.stride(1) if t.shape[1] > 1 else max(t.stride(1), t.shape[2])
        if (t.shape[2] > 1 and t.stride(2) != 1) or (n > 1 and t.stride(0) != t.shape[1] * ld):
            raise ValueError(f"{op}: the adapters of {name} must follow one another in rows of one pitch")
        pitch.append(ld)
    if out is None:
        out = torch.empty((T, N), device=x.device, dtype=out_dtype)
    if out.shape != (T, N) or (N > 1 and out.stride(1) != 1):
        raise ValueError(f"{op}: out must be [{T}, {N}] with dense rows")
    ldx, ldw, ldy = (t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1]) for t in (x, W, out))
    L = lib()
    need = L.sdb200_linear_lora_workspace(T, N, K, x.data_ptr(), ldx, int(x.dtype == bf), W.data_ptr(), ldw, n, r,
                                          A.data_ptr(), pitch[0], B.data_ptr(), pitch[1])
    ws = torch.empty(max(need, 1), device=x.device, dtype=torch.uint8)
    bind_stream()
    check(L.sdb200_linear_lora(T, N, K, x.data_ptr(), ldx, int(x.dtype == bf), W.data_ptr(), ldw, _p(bias),
                               rows.data_ptr(), n, r, A.data_ptr(), pitch[0], B.data_ptr(), pitch[1], _p(scale),
                               out.data_ptr(), ldy, int(out_dtype == bf), ws.data_ptr(), need))
    return out


def attention_ragged(q, k, v, q_begin, q_len, kv_begin, kv_len, max_q, max_kv, scale=None, causal=False, prefix=None,
                     cap=0.0, slopes=None, out_dtype=None, out=None):
    """Attention of sequences of their own lengths: sequence s reads query rows
    q_begin[s] .. + q_len[s] of q [Tq, heads, d] and key rows kv_begin[s] .. + kv_len[s] of
    k, v [Tkv, kv_heads, d] (bf16 or fp16; rows may be strided), at most max_q and max_kv long.
    Query i stands at position i + kv_len - q_len; causal hides later keys except the first
    prefix[s]; cap > 0 turns a score z into cap tanh(z / cap); slopes [heads] subtract
    slope * distance. scale defaults to 1 / sqrt(d). Returns out [Tq, heads, d] in out_dtype
    (bf16 or fp16, default as q); rows of no sequence keep what out held (zeros without out)."""
    op = "attention_ragged"
    if q.dtype not in (torch.bfloat16, torch.float16) or q.dim() != 3 or k.dim() != 3:
        raise TypeError(f"{op}: q, k, v must be [T, heads, d] bf16 or fp16, got {q.dtype}")
    (Tq, heads, d), (Tkv, kv_heads, dk) = q.shape, k.shape
    if dk != d or v.shape != k.shape:
        raise ValueError(f"{op}: shapes {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    out_dtype = out.dtype if out is not None else (out_dtype or q.dtype)
    if out_dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"{op}: output type {out_dtype}")
    n = q_begin.numel()
    i32 = torch.int32
    _check_args(op, q, k=(k, q.dtype, None), v=(v, q.dtype, None), q_begin=(q_begin, i32, (n,)),
                q_len=(q_len, i32, (n,)), kv_begin=(kv_begin, i32, (n,)), kv_len=(kv_len, i32, (n,)),
                prefix=(prefix, i32, (n,)), slopes=(slopes, torch.float32, (heads,)), out=(out, out_dtype, None))
    if out is None:
        out = torch.zeros((Tq, heads, d), device=q.device, dtype=out_dtype)
    if out.shape != q.shape:
        raise ValueError(f"{op}: out must have the shape of q")
    L = lib()
    max_q, max_kv = min(max_q, Tq), min(max_kv, Tkv)
    need = L.sdb200_attention_ragged_workspace(n, max_q, max_kv, heads, kv_heads, d)
    ws = torch.empty(max(need, 1), device=q.device, dtype=torch.uint8)
    bind_stream()
    check(L.sdb200_attention_ragged(q.data_ptr(), _head_pitch(op, "q", q), k.data_ptr(), _head_pitch(op, "k", k),
                                    v.data_ptr(), _head_pitch(op, "v", v), _TYPES[q.dtype], out.data_ptr(),
                                    _head_pitch(op, "out", out), _TYPES[out_dtype], Tq, Tkv, n, q_begin.data_ptr(),
                                    q_len.data_ptr(), kv_begin.data_ptr(), kv_len.data_ptr(), max_q, max_kv, heads,
                                    kv_heads, d, d ** -0.5 if scale is None else scale, cap, _p(slopes), int(causal),
                                    _p(prefix), ws.data_ptr(), need))
    return out


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
