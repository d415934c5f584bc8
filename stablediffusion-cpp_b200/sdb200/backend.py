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
_F32, _BF16, _I32 = torch.float32, torch.bfloat16, torch.int32
_raw_stream, _current = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _refuse_args(op, like, **tensors):
    """Names what is wrong with the tensors, (tensor, dtype, shape or None) by name: all on
    like's device, which must be the current one, and contiguous where a shape is given. The
    operators below test all of it in one expression and come here only when it fails: at one
    token a call's GPU time is that of a few tensor checks."""
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


_lora_bytes, _attention_bytes = {}, {}  # workspace sizes by argument sizes


def _remember(sizes, key, need):
    if need >= 0:  # -1: the operator itself says what is wrong
        if len(sizes) >= 4096:
            sizes.clear()
        sizes[key] = need


def _head_pitch(op, name, t):
    """Row pitch (elements) of [T, heads, d] whose heads lie next to each other."""
    T, h, d = t.shape
    row, head, one = t.stride()
    if (one != 1 and d > 1) or (head != d and h > 1):
        raise ValueError(f"{op}: the heads of {name} must be dense within a row")
    return row if T > 1 else h * d


def _row_pitch(op, name, t):
    rows, cols = t.shape
    row, one = t.stride()
    if one != 1 and cols > 1:
        raise ValueError(f"{op}: the rows of {name} must be dense")
    return row if rows > 1 else cols


def _stack_pitch(op, name, t):
    n, rows, cols = t.shape
    s0, s1, s2 = t.stride()
    ld = s1 if rows > 1 else s0 if n > 1 else cols
    if (s2 != 1 and cols > 1) or (n > 1 and s0 != rows * ld):
        raise ValueError(f"{op}: the adapters of {name} must follow one another in rows of one pitch")
    return ld


def qk_norm_rope(q, k, cos, sin, gq=None, gk=None, eps=1e-6, pos=None, interleaved=False, out_dtype=None, q_out=None,
                 k_out=None):
    """rms_norm_heads and rope of q [T, heads, d] and k [T, kv_heads, d] in one pass (rows may
    be strided, as views of a fused projection); cos / sin [n_pos, rot] fp32 with rot <= d,
    row pos[t] (int32), or t % n_pos without pos. Returns (q, k) in out_dtype (default: as
    given), or in q_out / k_out, which may be q / k themselves. k may be None."""
    op = "qk_norm_rope"
    dtype, dev = q.dtype, q.get_device()
    if dtype not in _TYPES or q.dim() != 3:
        raise TypeError(f"{op}: q must be [T, heads, d] fp32, bf16 or fp16, got {dtype} {tuple(q.shape)}")
    T, heads, d = q.shape
    out_dtype = out_dtype or (q_out.dtype if q_out is not None else dtype)
    if out_dtype not in _TYPES:
        raise TypeError(f"{op}: output type {out_dtype}")
    table = cos.shape
    if len(table) != 2:
        raise ValueError(f"{op}: cos must be [n_pos, rot]")
    if not (0 <= dev == _current() and cos.dtype is _F32 and cos.get_device() == dev and cos.is_contiguous()
            and sin.dtype is _F32 and sin.get_device() == dev and sin.shape == table and sin.is_contiguous()
            and (gq is None or (gq.dtype is _F32 and gq.get_device() == dev and gq.shape == (d,) and gq.is_contiguous()))
            and (gk is None or (gk.dtype is _F32 and gk.get_device() == dev and gk.shape == (d,) and gk.is_contiguous()))
            and (pos is None or (pos.dtype is _I32 and pos.get_device() == dev and pos.shape == (T,)
                                 and pos.is_contiguous()))
            and (k is None or (k.dtype is dtype and k.get_device() == dev))
            and (q_out is None or (q_out.dtype is out_dtype and q_out.get_device() == dev))
            and (k_out is None or (k_out.dtype is out_dtype and k_out.get_device() == dev))):
        _refuse_args(op, q, k=(k, dtype, None), cos=(cos, _F32, table), sin=(sin, _F32, table), gq=(gq, _F32, (d,)),
                     gk=(gk, _F32, (d,)), pos=(pos, _I32, (T,)), q_out=(q_out, out_dtype, None),
                     k_out=(k_out, out_dtype, None))
    ldqo, kv, ldk, ldko, kp, kop = heads * d, 0, 0, 0, None, None
    if q_out is None:
        q_out = q.new_empty((T, heads, d), dtype=out_dtype)
    else:
        if q_out.shape != q.shape:
            raise ValueError(f"{op}: q_out must have the shape of q")
        ldqo = _head_pitch(op, "q_out", q_out)
    if k is None:
        k_out = None
    else:
        if k.dim() != 3 or k.shape[0] != T or k.shape[2] != d:
            raise ValueError(f"{op}: k must be [{T}, kv_heads, {d}], got {tuple(k.shape)}")
        kv = k.shape[1]
        ldk, ldko = _head_pitch(op, "k", k), kv * d
        if k_out is None:
            k_out = q.new_empty((T, kv, d), dtype=out_dtype)
        else:
            if k_out.shape != k.shape:
                raise ValueError(f"{op}: k_out must have the shape of k")
            ldko = _head_pitch(op, "k_out", k_out)
        kp, kop = k.data_ptr(), k_out.data_ptr()
    L = lib()
    rc = L.sdb200_set_stream(_raw_stream(dev)) or L.sdb200_qk_norm_rope(
        T, q.data_ptr(), _head_pitch(op, "q", q), heads, kp, ldk, kv, _TYPES[dtype], d, table[1],
        None if gq is None else gq.data_ptr(), None if gk is None else gk.data_ptr(), eps, cos.data_ptr(), sin.data_ptr(),
        table[0], None if pos is None else pos.data_ptr(), 1 if interleaved else 0, q_out.data_ptr(), ldqo, kop, ldko,
        _TYPES[out_dtype])
    if rc:
        check(rc)
    return q_out, k_out


def linear_lora(x, W, A, B, rows, scale=None, bias=None, out_dtype=torch.float32, out=None):
    """x W^T (+ bias) + scale[a] (x A[a]^T) B[a]^T with a = rows[t] for row t (int32, < 0: no
    adapter). x [T, K] bf16 or fp32 (rounded to bf16), W [N, K], A [n, r, K], B [n, N, r] bf16,
    scale [n] and bias [N] fp32. Returns [T, N] in out_dtype (fp32 or bf16), or out."""
    op = "linear_lora"
    dtype, dev = x.dtype, x.get_device()
    if dtype not in (_F32, _BF16) or x.dim() != 2 or W.dim() != 2 or A.dim() != 3 or B.dim() != 3:
        raise TypeError(f"{op}: x [T, K] fp32 or bf16, W [N, K], A [n, r, K], B [n, N, r]")
    T, K = x.shape
    N, (n, r, Ka) = W.shape[0], A.shape
    if W.shape[1] != K or Ka != K or B.shape != (n, N, r):
        raise ValueError(f"{op}: shapes {tuple(x.shape)}, {tuple(W.shape)}, {tuple(A.shape)}, {tuple(B.shape)}")
    if out is not None:
        out_dtype = out.dtype
    if out_dtype not in (_F32, _BF16):
        raise TypeError(f"{op}: output type {out_dtype}")
    if not (0 <= dev == _current() and W.dtype is _BF16 and A.dtype is _BF16 and B.dtype is _BF16 and W.get_device() == dev
            and A.get_device() == dev and B.get_device() == dev and rows.dtype is _I32 and rows.get_device() == dev
            and rows.shape == (T,) and rows.is_contiguous()
            and (scale is None or (scale.dtype is _F32 and scale.get_device() == dev and scale.shape == (n,)
                                   and scale.is_contiguous()))
            and (bias is None or (bias.dtype is _F32 and bias.get_device() == dev and bias.shape == (N,)
                                  and bias.is_contiguous()))
            and (out is None or out.get_device() == dev)):
        _refuse_args(op, x, W=(W, _BF16, None), A=(A, _BF16, None), B=(B, _BF16, None), rows=(rows, _I32, (T,)),
                     scale=(scale, _F32, (n,)), bias=(bias, _F32, (N,)), out=(out, out_dtype, None))
    if out is None:
        out, ldy = x.new_empty((T, N), dtype=out_dtype), N
    else:
        if out.shape != (T, N):
            raise ValueError(f"{op}: out must be [{T}, {N}]")
        ldy = _row_pitch(op, "out", out)
    px, pw, pa, pb = x.data_ptr(), W.data_ptr(), A.data_ptr(), B.data_ptr()
    ldx, ldw, lda, ldb = _row_pitch(op, "x", x), _row_pitch(op, "W", W), _stack_pitch(op, "A", A), _stack_pitch(op, "B", B)
    bf = 1 if dtype is _BF16 else 0
    L = lib()
    # The workspace follows from sizes, pitches and alignment alone.
    key = (T, N, K, n, r, ldx, ldw, lda, ldb, bf, px & 15, pw & 15, pa & 15, pb & 15, dev)
    need = _lora_bytes.get(key)
    if need is None:
        need = L.sdb200_linear_lora_workspace(T, N, K, px, ldx, bf, pw, ldw, n, r, pa, lda, pb, ldb)
        _remember(_lora_bytes, key, need)
    ws = x.new_empty(need, dtype=torch.uint8) if need > 0 else None
    rc = L.sdb200_set_stream(_raw_stream(dev)) or L.sdb200_linear_lora(
        T, N, K, px, ldx, bf, pw, ldw, None if bias is None else bias.data_ptr(), rows.data_ptr(), n, r, pa, lda, pb, ldb,
        None if scale is None else scale.data_ptr(), out.data_ptr(), ldy, 1 if out_dtype is _BF16 else 0,
        None if ws is None else ws.data_ptr(), need)
    if rc:
        check(rc)
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
    dtype, dev = q.dtype, q.get_device()
    if dtype not in (_BF16, torch.float16) or q.dim() != 3 or k.dim() != 3:
        raise TypeError(f"{op}: q, k, v must be [T, heads, d] bf16 or fp16, got {dtype}")
    (Tq, heads, d), (Tkv, kv_heads, dk) = q.shape, k.shape
    if dk != d or v.shape != k.shape:
        raise ValueError(f"{op}: shapes {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    out_dtype = out.dtype if out is not None else (out_dtype or dtype)
    if out_dtype not in (_BF16, torch.float16):
        raise TypeError(f"{op}: output type {out_dtype}")
    n = q_begin.numel()
    one = (n,)
    if not (0 <= dev == _current() and k.dtype is dtype and v.dtype is dtype and k.get_device() == dev
            and v.get_device() == dev
            and q_begin.dtype is _I32 and q_begin.get_device() == dev and q_begin.shape == one and q_begin.is_contiguous()
            and q_len.dtype is _I32 and q_len.get_device() == dev and q_len.shape == one and q_len.is_contiguous()
            and kv_begin.dtype is _I32 and kv_begin.get_device() == dev and kv_begin.shape == one
            and kv_begin.is_contiguous()
            and kv_len.dtype is _I32 and kv_len.get_device() == dev and kv_len.shape == one and kv_len.is_contiguous()
            and (prefix is None or (prefix.dtype is _I32 and prefix.get_device() == dev and prefix.shape == one
                                    and prefix.is_contiguous()))
            and (slopes is None or (slopes.dtype is _F32 and slopes.get_device() == dev and slopes.shape == (heads,)
                                    and slopes.is_contiguous())) and (out is None or out.get_device() == dev)):
        _refuse_args(op, q, k=(k, dtype, None), v=(v, dtype, None), q_begin=(q_begin, _I32, one), q_len=(q_len, _I32, one),
                     kv_begin=(kv_begin, _I32, one), kv_len=(kv_len, _I32, one), prefix=(prefix, _I32, one),
                     slopes=(slopes, _F32, (heads,)), out=(out, out_dtype, None))
    if out is None:
        out, ldo = q.new_zeros((Tq, heads, d), dtype=out_dtype), heads * d
    else:
        if out.shape != q.shape:
            raise ValueError(f"{op}: out must have the shape of q")
        ldo = _head_pitch(op, "out", out)
    L = lib()
    max_q, max_kv = min(max_q, Tq), min(max_kv, Tkv)
    key = (n, max_q, max_kv, heads, kv_heads, d, dev)
    need = _attention_bytes.get(key)
    if need is None:
        need = L.sdb200_attention_ragged_workspace(n, max_q, max_kv, heads, kv_heads, d)
        _remember(_attention_bytes, key, need)
    ws = q.new_empty(need, dtype=torch.uint8) if need > 0 else None
    rc = L.sdb200_set_stream(_raw_stream(dev)) or L.sdb200_attention_ragged(
        q.data_ptr(), _head_pitch(op, "q", q), k.data_ptr(), _head_pitch(op, "k", k), v.data_ptr(),
        _head_pitch(op, "v", v), _TYPES[dtype], out.data_ptr(), ldo, _TYPES[out_dtype], Tq, Tkv, n, q_begin.data_ptr(),
        q_len.data_ptr(), kv_begin.data_ptr(), kv_len.data_ptr(), max_q, max_kv, heads, kv_heads, d,
        d ** -0.5 if scale is None else scale, cap, None if slopes is None else slopes.data_ptr(), 1 if causal else 0,
        None if prefix is None else prefix.data_ptr(), None if ws is None else ws.data_ptr(), need)
    if rc:
        check(rc)
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
