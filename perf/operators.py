"""Cases of the integer text-conditioning operators: the RMS norm with the residual's
addition and an 8-bit output, the int8 matrix product with per-token and per-channel
scales, and cross attention to an encoder's states.

``run`` makes one pass through an operator: the framework's own call where ``own`` is
set, else the operator in elementary torch operations in 32 bits. Where a case's sizes
come from the refiner they are its configuration's: width 3072, 24 heads of 128, ffn
14336, chunks of 3 frames of 36 x 64 tokens (6912), 512 text tokens of width 4096.
"""
import importlib
import math

import torch

own = False

EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
QMAX = {"int8": 127.0, "e4m3": 448.0}


def listed():
    return [
        # one token of a serving step: the text width, latency alone
        dict(name="norm token", op="norm", rows=1, width=4096, dtype="bf16", residual=True,
             out="e4m3"),
        # odd rows of an odd width in half precision, without a residual (a first norm)
        dict(name="norm ragged", op="norm", rows=1003, width=2570, dtype="fp16", residual=False,
             out="e4m3"),
        # one chunk of the refiner: 3 frames of 36 x 64 tokens
        dict(name="norm chunk", op="norm", rows=6912, width=3072, dtype="bf16", residual=True,
             out="e4m3"),
        # one token through the ffn's first product: the weights' bytes
        dict(name="gemm token", op="gemm", rows=1, width=3072, cols=14336, dtype="bf16",
             bias=True),
        # a few tokens of a batch being served, an odd count, half precision out
        dict(name="gemm few", op="gemm", rows=37, width=4096, cols=4096, dtype="fp16",
             bias=False),
        # one chunk through the ffn's first product: the tensor cores
        dict(name="gemm chunk", op="gemm", rows=6912, width=3072, cols=14336, dtype="bf16",
             bias=True),
        # norm, quantise and the fused q|k|v product of one frame
        dict(name="norm gemm frame", op="norm_gemm", rows=2304, width=3072, cols=9216,
             dtype="bf16", residual=True, bias=True),
        # one query token of each of 8 samples against its own prompt's length
        dict(name="attn token", op="attn", batch=8, q=1, kv=512, heads=24, kv_heads=24, dim=128,
             dtype="bf16", lens="ragged", mask=False),
        # one query token against a long context with grouped heads: the cache's bytes
        dict(name="attn token long", op="attn", batch=4, q=1, kv=32768, heads=32, kv_heads=8,
             dim=128, dtype="bf16", lens="full", mask=False),
        # odd lengths, an empty sample, holes in the keys' mask, grouped heads of 64
        dict(name="attn ragged", op="attn", batch=3, q=777, kv=1501, heads=16, kv_heads=4, dim=64,
             dtype="fp16", lens="ragged", mask=True),
        # one chunk's tokens against the 512 text tokens
        dict(name="attn chunk", op="attn", batch=1, q=6912, kv=512, heads=24, kv_heads=24,
             dim=128, dtype="bf16", lens="full", mask=False),
        # a long query against a longer context: the tensor cores and the exponentials
        dict(name="attn long", op="attn", batch=1, q=4096, kv=8192, heads=24, kv_heads=24,
             dim=128, dtype="bf16", lens="full", mask=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the listed ranges: one token to a chunk, odd sizes among them."""
    op = rng.choice(("norm", "norm", "gemm", "gemm", "norm_gemm", "attn", "attn", "attn"))
    if op == "attn":
        while True:
            hkv = rng.choice((1, 2, 4, 8, 12, 24))
            c = dict(op=op, batch=_log(rng, 1, 8), q=rng.choice((1, _log(rng, 1, 8192))),
                     kv=_log(rng, 1, 32768), heads=hkv * rng.choice((1, 1, 2, 4, 8)), kv_heads=hkv,
                     dim=rng.choice((64, 80, 96, 128, 128)), dtype=rng.choice(("bf16", "fp16")),
                     lens=rng.choice(("full", "ragged")), mask=rng.random() < 0.3)
            scores = c["batch"] * c["heads"] * c["q"] * c["kv"]
            cache = c["batch"] * c["kv_heads"] * c["kv"] * c["dim"]
            if scores <= 24 * 4096 * 8192 and cache <= 4 * 8 * 32768 * 128:
                return c
    # the chained case is held in 16 bits, as a model's rows are
    dtype = rng.choice(("bf16", "fp16") if op == "norm_gemm" else ("bf16", "fp16", "fp32"))
    while True:
        rows = _log(rng, 1, 6912)
        width = _log(rng, 64, 8192)
        if rng.random() < 0.75:
            width = max(16, width // 16 * 16)
        cols = _log(rng, 64, 16384)
        if op == "norm":
            return dict(op=op, rows=rows, width=width, dtype=dtype, residual=rng.random() < 0.7,
                        out="e4m3")
        if rng.random() < 0.75:
            cols = max(16, cols // 16 * 16)
        if rows * width * cols <= 6912 * 3072 * 14336 and (rows + cols) * width <= 1 << 27:
            c = dict(op=op, rows=rows, width=width, cols=cols, dtype=dtype,
                     bias=rng.random() < 0.5)
            if op == "norm_gemm":
                c["residual"] = rng.random() < 0.7
            return c


# ------------------------------------------------------------------ inputs
def _lens(case):
    """Visible keys of each sample: all, or lengths from none to all of them."""
    B, L = case["batch"], case["kv"]
    if case["lens"] == "full":
        return [L] * B
    if B == 1:
        return [(2 * L + 2) // 3]
    return [L * b // (B - 1) for b in range(B)]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _norm_inputs(case, g):
    dt = TYPES[case["dtype"]]
    M, K = case["rows"], case["width"]
    # a residual stream: rows of different size, a few wide columns
    size = torch.exp(0.5 * torch.randn(M, 1, generator=g, device="cuda"))
    col = 1 + 4 * (torch.rand(K, generator=g, device="cuda") < 0.02).float()
    s = {"x": (torch.randn(M, K, generator=g, device="cuda") * size * col).to(dt),
         "weight": (1 + 0.1 * torch.randn(K, generator=g, device="cuda")).to(dt),
         "sum": None, "residual": None}
    if case["residual"]:
        s["residual"] = torch.randn(M, K, generator=g, device="cuda").to(dt)
        s["sum"] = torch.empty(M, K, dtype=dt, device="cuda")
    return s


def _rows16(M, K, dtype):
    """[M, K] with rows 16 values apart at least (the product's operand alignment)."""
    return torch.empty(M, -(-K // 16) * 16, dtype=dtype, device="cuda")[:, :K]


def _codes(M, K, g):
    """int8 rows as a quantiser leaves them: a normal spread, the largest at 127."""
    t = _rows16(M, K, torch.int8)
    r = torch.randn(M, K, generator=g, device="cuda")
    t.copy_(torch.round(r * (127.0 / r.abs().amax(1, keepdim=True))))
    return t


def _gemm_inputs(case, g):
    N, K = case["cols"], case["width"]
    dt = TYPES[case["dtype"]]
    return {"w": _codes(N, K, g),
            "w_scale": (0.5 + torch.rand(N, generator=g, device="cuda")) / 127 / K ** 0.5,
            "bias": ((0.1 * torch.randn(N, generator=g, device="cuda")).to(dt)
                     if case["bias"] else None),
            "out": torch.empty(case["rows"], N, dtype=dt, device="cuda")}


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    s = {"case": case, "op": op}
    if op in ("norm", "norm_gemm"):
        s.update(_norm_inputs(case, g))
        M, K = case["rows"], case["width"]
        s["q"] = _rows16(M, K, torch.float8_e4m3fn if op == "norm" else torch.int8)
        s["scale"] = torch.empty(M, device="cuda")
    if op in ("gemm", "norm_gemm"):
        s.update(_gemm_inputs(case, g))
    if op == "gemm":
        M = case["rows"]
        s["a"] = _codes(M, case["width"], g)
        s["a_scale"] = (0.5 + torch.rand(M, generator=g, device="cuda")) * 4 / 127
    if op == "attn":
        B, Lq, Lk = case["batch"], case["q"], case["kv"]
        H, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
        dt = TYPES[case["dtype"]]
        s["q"] = torch.randn(B, Lq, H, D, generator=g, device="cuda").to(dt)
        # the keys and values of one projection of the encoder's states, side by side
        kv = torch.randn(B, Lk, 2, Hkv, D, generator=g, device="cuda").to(dt)
        s["k"], s["v"] = kv[:, :, 0], kv[:, :, 1]
        s["lens"] = s["mask"] = None
        keep = torch.ones(B, Lk, dtype=torch.bool, device="cuda")
        if case["lens"] != "full":
            s["lens"] = torch.tensor(_lens(case), dtype=torch.int32, device="cuda")
            keep &= torch.arange(Lk, device="cuda")[None] < s["lens"][:, None]
        if case["mask"]:
            s["mask"] = torch.rand(B, Lk, generator=g, device="cuda") < 0.9
            keep &= s["mask"]
        # rows past a sample's length hold whatever the buffer held before
        kv.masked_fill_(~keep[:, :, None, None, None], float("nan"))
        s["out"] = torch.empty(B, Lq, H, D, dtype=dt, device="cuda")
    return s


# ------------------------------------------------------------------ plain forms
def _plain_norm(s, qmax):
    """(codes before rounding, scale, the sum in x's type) in 32 bits."""
    x = s["x"].float()
    if s["residual"] is not None:
        x = x + s["residual"].float()
    y = x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * s["weight"].float()
    scale = (y.abs().amax(1) / qmax).clamp_min(1e-12)
    codes = (y / scale[:, None]).clamp(-qmax, qmax)
    return codes, scale, x.to(s["x"].dtype) if s["residual"] is not None else None


def _plain_gemm(s, a, a_scale):
    y = (a.float() @ s["w"].float().t()) * a_scale[:, None] * s["w_scale"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["out"].dtype)


def _plain_attn(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    B, Lq, H, D = q.shape
    Lk, Hkv = k.shape[1:3]
    keep = torch.ones(B, Lk, dtype=torch.bool, device=q.device)
    if s["lens"] is not None:
        keep = keep & (torch.arange(Lk, device=q.device)[None] < s["lens"][:, None])
    if s["mask"] is not None:
        keep = keep & s["mask"]
    # the query heads of one key head side by side: [B, Hkv, group * Lq, D]
    q = q.view(B, Lq, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    p = q @ k.permute(0, 2, 3, 1) * D ** -0.5
    p = p.masked_fill(~keep[:, None, None, :], float("-inf"))
    top = p.amax(-1, keepdim=True)
    p = torch.exp(p - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    v = torch.where(keep[:, :, None, None], v, 0.0).permute(0, 2, 1, 3)
    o = (p @ v) / torch.where(total == 0, 1.0, total)
    o = o.view(B, Hkv, H // Hkv, Lq, D).permute(0, 3, 1, 2, 4).reshape(B, Lq, H, D)
    return o.to(s["q"].dtype)


def _plain(s):
    op = s["op"]
    if op == "norm":
        codes, scale, total = _plain_norm(s, QMAX["e4m3"])
        return {"q": codes.to(torch.float8_e4m3fn), "scale": scale, "sum": total}
    if op == "gemm":
        return {"out": _plain_gemm(s, s["a"], s["a_scale"])}
    if op == "norm_gemm":
        codes, scale, total = _plain_norm(s, QMAX["int8"])
        return {"out": _plain_gemm(s, torch.round(codes), scale), "sum": total}
    return {"out": _plain_attn(s)}


# ------------------------------------------------------------------ the operators' calls
_ops = None


def run(state):
    global _ops
    s = state
    if not own:
        return _plain(s)
    if _ops is None:
        _ops = importlib.import_module("dreamx-creator_b200").ops
    op = s["op"]
    if op in ("norm", "norm_gemm"):
        q, scale, total = _ops.add_rms_quant(s["x"], s["weight"], EPS, residual=s["residual"],
                                             sum_out=s["sum"], q=s["q"], qscale=s["scale"])
        if op == "norm":
            return {"q": q, "scale": scale, "sum": total}
        out = _ops.int8_gemm(q, scale, s["w"], s["w_scale"], s["bias"], s["out"])
        return {"out": out, "sum": total}
    if op == "gemm":
        return {"out": _ops.int8_gemm(s["a"], s["a_scale"], s["w"], s["w_scale"], s["bias"],
                                      s["out"])}
    return {"out": _ops.cross_attn(s["q"], s["k"], s["v"], s["out"], kv_lens=s["lens"],
                                   key_mask=s["mask"])}


# ------------------------------------------------------------------ the work of a pass
def _norm_work(case, out_bytes):
    M, K = case["rows"], case["width"]
    e = TYPES[case["dtype"]].itemsize
    arrays = 3 if case["residual"] else 1
    return M * K * (arrays * e + out_bytes) + 4 * M * bool(out_bytes) + K * e, 8 * M * K


def _gemm_work(case, a_bytes):
    M, N, K = case["rows"], case["cols"], case["width"]
    e = TYPES[case["dtype"]].itemsize
    return (M * (K + 4) * a_bytes + N * (K + 4) + M * N * e + (N * e if case["bias"] else 0),
            2 * M * N * K)


def work(case):
    op = case["op"]
    if op == "norm":
        b, f = _norm_work(case, 1)
    elif op == "gemm":
        b, f = _gemm_work(case, 1)
    elif op == "norm_gemm":
        # the codes between the two need not leave the chip: they are not counted
        (b0, f0), (b1, f1) = _norm_work(case, 0), _gemm_work(case, 0)
        b, f = b0 + b1, f0 + f1
    else:
        e = TYPES[case["dtype"]].itemsize
        keys = sum(_lens(case))
        D, H = case["dim"], case["heads"]
        b = 2 * case["batch"] * case["q"] * H * D * e + 2 * keys * case["kv_heads"] * D * e
        b += case["batch"] * case["kv"] if case["mask"] else 0
        f = 4 * case["q"] * keys * H * D
    return {"bytes": b, "flops": f}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "attn":
        return {"out": _exact_attn(s)}
    if op == "gemm":
        return {"out": _exact_product(s, s["a"].double() * s["a_scale"].double()[:, None])}
    h = s["x"].double()
    if s["residual"] is not None:
        h += s["residual"].double()
    norm = h.pow(2).sum(1).div(h.shape[1]).add(EPS).sqrt()
    y = h / norm[:, None] * s["weight"].double()
    limit = QMAX["e4m3" if op == "norm" else "int8"]
    step = torch.clamp(y.abs().max(1).values / limit, min=1e-12)[:, None]
    total = h if s["residual"] is not None else None
    if op == "norm":
        # the values that the codes round
        return {"q": y / step, "scale": step[:, 0], "sum": total}
    return {"out": _exact_product(s, torch.round(y / step) * step), "sum": total}


def _exact_product(s, a):
    y = torch.einsum("mk,nk->mn", a, s["w"].double() * s["w_scale"].double()[:, None])
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_attn(s):
    B, Lq, H, D = s["q"].shape
    group = H // s["k"].shape[2]
    out = torch.zeros(B, Lq, H, D, dtype=torch.float64, device="cuda")
    for b in range(B):
        at = torch.arange(s["k"].shape[1], device="cuda")
        if s["lens"] is not None:
            at = at[: int(s["lens"][b])]
        if s["mask"] is not None:
            at = at[s["mask"][b, : at.numel()]]
        if not at.numel():
            continue
        for h in range(H):
            k, v = s["k"][b, at, h // group].double(), s["v"][b, at, h // group].double()
            w = torch.softmax(torch.einsum("id,jd->ij", s["q"][b, :, h].double(), k)
                              / math.sqrt(D), dim=1)
            out[b, :, h] = w @ v
    return out
