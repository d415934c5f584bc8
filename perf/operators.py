"""The operators a server of several text-to-image requests needs around one transformer layer, as cases to be timed:

  qk    norms of q and k for each head with the rotary embedding (``qk_norm_rope``)
  lora  a projection shared by all requests plus each request's own low-rank adapter (``linear_lora``)
  attn  attention of sequences with their own lengths: causal and prefix masks, capped scores, distance bias
        (``attention_ragged``)

``run`` computes the plain form in 32 bits, or, with ``own``, calls the framework.
"""
import math
import random
import sys

import torch

own = False

_F = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_be = None


def _backend():
    global _be
    if _be is None:
        sys.path.insert(0, "stablediffusion-cpp_b200")
        import sdb200

        _be = sdb200.backend
    return _be


def _ints(text):
    return [int(v) for v in text.split(",")]


def _text(values):
    return ",".join(str(v) for v in values)


# ------------------------------------------------------------------------------- cases
def listed():
    cases = []
    # Eight requests of the Qwen3 encoder shape (32 query and 8 key heads of 128), one token each.
    cases.append(dict(name="qk-tokens", op="qk", T=8, heads=32, kv=8, d=128, rot=128, inter=False, fused=True,
                      x="bf16", y="bf16", n_pos=4096, by_pos=True))
    # Prompts of several requests, packed, read out of the fused QKV projection.
    cases.append(dict(name="qk-prompts", op="qk", T=2397, heads=32, kv=8, d=128, rot=128, inter=False, fused=True,
                      x="bf16", y="bf16", n_pos=1024, by_pos=True))
    # A head width that is no power of two, half of it rotated, in 32 bits.
    cases.append(dict(name="qk-part", op="qk", T=4097, heads=12, kv=4, d=80, rot=40, inter=False, fused=False,
                      x="f32", y="f32", n_pos=5000, by_pos=True))
    # The DiT block at 1024 x 1024 pixels: eight images of 4224 tokens, 30 heads, fp32 in, fp16 attention operands out.
    cases.append(dict(name="qk-dit", op="qk", T=33792, heads=30, kv=30, d=128, rot=128, inter=True, fused=False,
                      x="f32", y="f16", n_pos=4224, by_pos=False))
    # One request with one token.
    cases.append(dict(name="lora-token", op="lora", T=1, N=2560, K=2560, r=16, n_req=1, n_ad=4, bias=False))
    # One token of each of 48 requests over 32 adapters, the encoder's widest projection.
    cases.append(dict(name="lora-tokens", op="lora", T=48, N=9728, K=2560, r=32, n_req=48, n_ad=32, bias=False))
    # Prompts of twelve requests.
    cases.append(dict(name="lora-prompts", op="lora", T=2397, N=4096, K=2560, r=16, n_req=12, n_ad=9, bias=True))
    # Eight images through a DiT projection, each with its own adapter.
    cases.append(dict(name="lora-dit", op="lora", T=33792, N=3840, K=3840, r=64, n_req=8, n_ad=8, bias=True))
    # One new token of 16 requests against caches of different lengths, with a distance bias.
    cases.append(dict(name="attn-tokens", op="attn", q=_text([1] * 16),
                      kv="9000,211,17000,1024,30001,4096,777,12345,64,20480,3333,8192,1,15000,6001,25000", heads=32,
                      kv_heads=8, d=128, t="bf16", y="bf16", mask="causal", cap=0.0, bias=True))
    # Short prompts of the CLIP shape (12 heads of 64, at most 77 tokens), packed one after another.
    lens = [5 + (i * 37) % 73 for i in range(64)]
    cases.append(dict(name="attn-prompts", op="attn", q=_text(lens), kv=_text(lens), heads=12, kv_heads=12, d=64,
                      t="f16", y="f16", mask="causal", cap=0.0, bias=False))
    # Documents whose first part is seen by all of their tokens, with capped scores.
    cases.append(dict(name="attn-prefix", op="attn", q="700,2500,1111,1900,333,1025", kv="700,2500,1111,1900,333,1025",
                      heads=32, kv_heads=8, d=128, t="bf16", y="bf16", mask="prefix", cap=30.0, bias=False))
    # Four images with their captions, packed: every token of a document sees the whole document.
    cases.append(dict(name="attn-dit", op="attn", q="4224,4130,4173,4101", kv="4224,4130,4173,4101", heads=30,
                      kv_heads=30, d=128, t="f16", y="bf16", mask="full", cap=0.0, bias=False))
    return cases


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["qk", "lora", "attn"])
    if op == "qk":
        kv = rng.choice([1, 2, 4, 8, 12, 30])
        heads = kv * rng.choice([1, 2, 4]) if kv < 12 else kv
        d = rng.choice([40, 64, 80, 96, 128, 128, 256])
        rot = d if rng.random() < 0.7 else d // 2
        x = rng.choice(["f32", "bf16", "f16"])
        T = _log(rng, 1, min(33792, 33792 * 60 * 128 // ((heads + kv) * d)))
        return dict(op=op, T=T, heads=heads, kv=kv, d=d, rot=rot, inter=rng.random() < 0.5,
                    fused=rng.random() < 0.5, x=x, y=rng.choice([x, "bf16", "f16"]), n_pos=rng.randint(1, 5000),
                    by_pos=rng.random() < 0.6)
    if op == "lora":
        N, K = _log(rng, 64, 10240), _log(rng, 64, 10240)
        if rng.random() < 0.8:
            N, K = (N + 7) // 8 * 8, (K + 7) // 8 * 8
        T = _log(rng, 1, min(33792, 33792 * 3840 * 3840 // (N * K)))
        n_req = T if T <= 128 and rng.random() < 0.5 else rng.randint(1, min(T, 64))
        return dict(op=op, T=T, N=N, K=K, r=rng.choice([4, 8, 16, 32, 64, 128]), n_req=n_req, n_ad=rng.randint(1, 64),
                    bias=rng.random() < 0.5)
    kv_heads = rng.choice([1, 2, 4, 8, 12, 30])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8]) if kv_heads < 12 else kv_heads
    n = _log(rng, 1, 64)
    tokens = rng.random() < 0.4
    if tokens:
        kv = [_log(rng, 1, 32768) for _ in range(n)]
        q = [min(k, rng.choice([1, 1, 1, 2, 4])) for k in kv]
    else:
        top = min(8192, int(math.sqrt(2.0e9 / (n * heads))))
        q = [_log(rng, 1, top) for _ in range(n)]
        kv = [min(8192, v + (rng.randint(0, v) if rng.random() < 0.3 else 0)) for v in q]
    while n * heads * max(q) * max(kv) > 2.1e9 or n * max(kv) * kv_heads > 5e6:  # the plain form's padded scores and keys
        kv = [max(1, v // 2) for v in kv]
        q = [min(a, b) for a, b in zip(q, kv)] if tokens else [max(1, v // 2) for v in q]
    t = rng.choice(["bf16", "f16"])
    return dict(op=op, q=_text(q), kv=_text(kv), heads=heads, kv_heads=kv_heads,
                d=rng.choice([40, 64, 64, 80, 128, 128, 128]), t=t, y=rng.choice([t, t, "bf16"]),
                mask=rng.choice(["full", "causal", "causal", "prefix"]), cap=rng.choice([0.0, 0.0, 20.0, 50.0]),
                bias=rng.random() < 0.35)


# ------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _rows(case):
    """The adapter of every row: requests of nearly equal lengths one after another, every sixth without an adapter
    where there is more than one."""
    T, n = case["T"], case["n_req"]
    ids = []
    for i in range(n):
        a = -1 if n > 1 and i % 6 == 5 else (i * 5 + 1) % case["n_ad"]
        ids += [a] * (T * (i + 1) // n - T * i // n)
    return ids


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "qk":
        T, H, Hk, d, dt = case["T"], case["heads"], case["kv"], case["d"], _F[case["x"]]
        if case["fused"]:  # q | k | v rows of one projection
            y = _normal(g, (T, (H + 2 * Hk) * d), dt, 1.5)
            q, k = y[:, : H * d].unflatten(1, (H, d)), y[:, H * d: (H + Hk) * d].unflatten(1, (Hk, d))
        else:
            q, k = _normal(g, (T, H, d), dt, 1.5), _normal(g, (T, Hk, d), dt, 1.5)
        P, rot = case["n_pos"], case["rot"]
        ang = torch.arange(P, device="cuda", dtype=torch.float64)[:, None] * (
            10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot))[None]
        full = ang.repeat_interleave(2, 1) if case["inter"] else torch.cat([ang, ang], 1)
        pos = torch.randint(0, P, (T,), generator=g, device="cuda", dtype=torch.int32) if case["by_pos"] else None
        return dict(case=case, q=q, k=k, cos=full.cos().float(), sin=full.sin().float(), pos=pos,
                    gq=1.0 + _normal(g, (d,), scale=0.2), gk=1.0 + _normal(g, (d,), scale=0.2))
    if case["op"] == "lora":
        T, N, K, r, n = case["T"], case["N"], case["K"], case["r"], case["n_ad"]
        b = torch.bfloat16
        return dict(case=case, x=_normal(g, (T, K), b), W=_normal(g, (N, K), b, K ** -0.5),
                    A=_normal(g, (n, r, K), b, K ** -0.5), B=_normal(g, (n, N, r), b, 0.3 * r ** -0.5),
                    scale=0.5 + torch.rand((n,), generator=g, device="cuda"),
                    bias=_normal(g, (N,)) if case["bias"] else None,
                    rows=torch.tensor(_rows(case), dtype=torch.int32, device="cuda"))
    q, kv = _ints(case["q"]), _ints(case["kv"])
    H, Hk, d, dt = case["heads"], case["kv_heads"], case["d"], _F[case["t"]]
    i32 = dict(dtype=torch.int32, device="cuda")
    starts = lambda v: [sum(v[:i]) for i in range(len(v))]  # noqa: E731
    s = dict(case=case, q=_normal(g, (sum(q), H, d), dt), k=_normal(g, (sum(kv), Hk, d), dt),
             v=_normal(g, (sum(kv), Hk, d), dt), q_begin=torch.tensor(starts(q), **i32), q_len=torch.tensor(q, **i32),
             kv_begin=torch.tensor(starts(kv), **i32), kv_len=torch.tensor(kv, **i32), max_q=max(q), max_kv=max(kv),
             slopes=None, prefix=None,
             out=torch.zeros((sum(q), H, d), dtype=_F[case["y"]], device="cuda"))
    if case["bias"]:
        s["slopes"] = 2.0 ** (-8.0 * torch.arange(1, H + 1, device="cuda", dtype=torch.float32) / H)
    if case["mask"] == "prefix":
        s["prefix"] = (torch.rand((len(kv),), generator=g, device="cuda") * s["kv_len"]).to(torch.int32)
    return s


# ----------------------------------------------------------------------------- plain forms
def _plain_qk(s):
    c = s["case"]
    d, rot = c["d"], c["rot"]
    at = s["pos"].long() if s["pos"] is not None else torch.arange(c["T"], device="cuda") % c["n_pos"]
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]

    def one(x, gamma):
        u = x.float()
        u = u * torch.rsqrt(u.square().mean(-1, keepdim=True) + 1e-6) * gamma
        a = u[..., :rot]
        if c["inter"]:
            turned = torch.stack([-a[..., 1::2], a[..., 0::2]], -1).flatten(-2)
        else:
            turned = torch.cat([-a[..., rot // 2:], a[..., : rot // 2]], -1)
        a = a * cos + turned * sin
        return (torch.cat([a, u[..., rot:]], -1) if rot < d else a).to(_F[c["y"]])

    return one(s["q"], s["gq"]), one(s["k"], s["gk"])


def _plain_lora(s):
    n, r, K = s["A"].shape
    N = s["W"].shape[0]
    x = s["x"].float()
    y = x @ s["W"].float().t()
    if s["bias"] is not None:
        y += s["bias"]
    pick = (s["rows"][:, None] == torch.arange(n, device="cuda")).float() * s["scale"]
    h = (x @ s["A"].float().view(n * r, K).t()).view(-1, n, r) * pick[..., None]
    y += h.reshape(-1, n * r) @ s["B"].float().permute(0, 2, 1).reshape(n * r, N)
    return y.to(torch.bfloat16)


def _plain_attn(s):
    c = s["case"]
    H, Hk, d = c["heads"], c["kv_heads"], c["d"]
    n, Mq, Mk = s["q_len"].numel(), s["max_q"], s["max_kv"]
    i, j = torch.arange(Mq, device="cuda"), torch.arange(Mk, device="cuda")
    live_q, live_k = i < s["q_len"][:, None], j < s["kv_len"][:, None]
    at_q = s["q_begin"][:, None].long() + torch.where(live_q, i, 0)
    at_k = s["kv_begin"][:, None].long() + torch.where(live_k, j, 0)
    q = s["q"][at_q].float().view(n, Mq, Hk, H // Hk, d).permute(0, 2, 3, 1, 4).reshape(n, Hk, -1, d)
    k, v = (x[at_k].float().permute(0, 2, 1, 3) for x in (s["k"], s["v"]))
    z = (q @ k.transpose(-1, -2)).view(n, Hk, H // Hk, Mq, Mk)
    z *= d ** -0.5
    if c["cap"]:
        z = z.div_(c["cap"]).tanh_().mul_(c["cap"])
    p = i + (s["kv_len"] - s["q_len"])[:, None]  # the position of each query among the keys
    if s["slopes"] is not None:
        far = (p[:, :, None] - j).abs().float()
        z -= s["slopes"].view(1, Hk, H // Hk, 1, 1) * far[:, None, None]
    allowed = live_k[:, None, :] & live_q[:, :, None]
    if c["mask"] == "causal":
        allowed = allowed & (j <= p[:, :, None])
    elif c["mask"] == "prefix":
        allowed = allowed & ((j <= p[:, :, None]) | (j < s["prefix"][:, None, None]))
    z.masked_fill_(~allowed[:, None, None], -math.inf)
    top = z.amax(-1, keepdim=True)
    z = z.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = z.sum(-1, keepdim=True)
    o = z.view(n, Hk, -1, Mk) @ v
    o = o.view(n, Hk, H // Hk, Mq, d) / torch.where(total == 0, 1.0, total)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, Mq, H, d).to(s["out"].dtype)
    s["out"][at_q[live_q]] = o[live_q]
    return s["out"]


def run(s):
    c = s["case"]
    if not own:
        return {"qk": _plain_qk, "lora": _plain_lora, "attn": _plain_attn}[c["op"]](s)
    be = _backend()
    if c["op"] == "qk":
        return be.qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], s["gq"], s["gk"], eps=1e-6, pos=s["pos"],
                               interleaved=c["inter"], out_dtype=_F[c["y"]])
    if c["op"] == "lora":
        return be.linear_lora(s["x"], s["W"], s["A"], s["B"], s["rows"], scale=s["scale"], bias=s["bias"],
                              out_dtype=torch.bfloat16)
    return be.attention_ragged(s["q"], s["k"], s["v"], s["q_begin"], s["q_len"], s["kv_begin"], s["kv_len"],
                               s["max_q"], s["max_kv"], causal=c["mask"] != "full", prefix=s["prefix"], cap=c["cap"],
                               slopes=s["slopes"], out=s["out"])


# -------------------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    f = torch.float64
    if case["op"] == "qk":
        T, d, rot, P = case["T"], case["d"], case["rot"], case["n_pos"]
        at = s["pos"].long() if s["pos"] is not None else torch.arange(T, device="cuda").remainder(P)
        first = torch.arange(0, rot, 2, device="cuda") if case["inter"] else torch.arange(rot // 2, device="cuda")
        second = first + (1 if case["inter"] else rot // 2)
        outs = []
        for x, gamma in ((s["q"], s["gq"]), (s["k"], s["gk"])):
            u = x.to(f)
            u = u / ((u * u).sum(-1, keepdim=True) / d + 1e-6).sqrt() * gamma.to(f)
            y = u.clone()
            c, w = s["cos"].to(f)[at].unsqueeze(1), s["sin"].to(f)[at].unsqueeze(1)
            y[..., first] = u[..., first] * c[..., first] - u[..., second] * w[..., first]
            y[..., second] = u[..., second] * c[..., second] + u[..., first] * w[..., second]
            outs.append(y)
        return tuple(outs)
    if case["op"] == "lora":
        x, W = s["x"].to(f), s["W"].to(f)
        y = torch.matmul(x, W.t())
        if s["bias"] is not None:
            y = y + s["bias"].to(f)
        for a in range(case["n_ad"]):
            t = (s["rows"] == a).nonzero().flatten()
            if t.numel():
                y[t] += float(s["scale"][a]) * ((x[t] @ s["A"][a].to(f).t()) @ s["B"][a].to(f).t())
        return y
    H, Hk, d = case["heads"], case["kv_heads"], case["d"]
    out = torch.zeros((s["q"].shape[0], H, d), dtype=f, device="cuda")
    for b, (nq, nk) in enumerate(zip(_ints(case["q"]), _ints(case["kv"]))):
        q0, k0 = int(s["q_begin"][b]), int(s["kv_begin"][b])
        pre = int(s["prefix"][b]) if s["prefix"] is not None else 0
        j = torch.arange(nk, device="cuda")
        for lo in range(0, nq, 1024):
            hi = min(nq, lo + 1024)
            p = torch.arange(lo, hi, device="cuda") + (nk - nq)
            hide = None
            if case["mask"] != "full":
                hide = (j[None] > p[:, None]) & (j[None] >= pre)
            for h in range(Hk):
                kk, vv = s["k"][k0: k0 + nk, h].to(f), s["v"][k0: k0 + nk, h].to(f)
                qq = s["q"][q0 + lo: q0 + hi, h * (H // Hk): (h + 1) * (H // Hk)].to(f).transpose(0, 1)
                z = torch.matmul(qq, kk.t()) / math.sqrt(d)
                if case["cap"]:
                    z = case["cap"] * torch.tanh(z / case["cap"])
                if s["slopes"] is not None:
                    m = s["slopes"][h * (H // Hk): (h + 1) * (H // Hk)].to(f)
                    z = z - m[:, None, None] * (p[:, None] - j[None]).abs()
                if hide is not None:
                    z = z.masked_fill(hide, -math.inf)
                w = torch.softmax(z, -1).nan_to_num(0.0)
                out[q0 + lo: q0 + hi, h * (H // Hk): (h + 1) * (H // Hk)] = torch.matmul(w, vv).transpose(0, 1)
    return out


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if case["op"] == "qk":
        n = case["T"] * (case["heads"] + case["kv"]) * case["d"]
        tables = min(case["T"], case["n_pos"]) * case["rot"] * 8
        return {"bytes": n * (size[case["x"]] + size[case["y"]]) + tables, "flops": 8 * n}
    if case["op"] == "lora":
        T, N, K, r = case["T"], case["N"], case["K"], case["r"]
        ids = _rows(case)
        used = len(set(a for a in ids if a >= 0))
        live = sum(1 for a in ids if a >= 0)
        return {"bytes": 2 * (T * K + N * K + T * N + used * r * (K + N)),
                "flops": 2 * T * N * K + 2 * live * r * (K + N)}
    q, kv, H, Hk, d = _ints(case["q"]), _ints(case["kv"]), case["heads"], case["kv_heads"], case["d"]
    pairs = 0
    for a, b in zip(q, kv):
        if case["mask"] == "full":
            pairs += a * b
        else:  # a prefix adds to the triangle what it covers above it: on average a third of that part
            tri = a * b - a * (a - 1) // 2
            pairs += tri if case["mask"] == "causal" else tri + (a * b - tri) // 3
    return {"bytes": 2 * (sum(q) * H + 2 * sum(kv) * Hk) * d + sum(q) * H * d * size[case["y"]],
            "flops": 4 * d * H * pairs}
