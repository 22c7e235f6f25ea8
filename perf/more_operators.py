"""Cases of the paged key/value cache: writing new tokens into pages (8-bit codes with a scale
per token and head), reading pages back, attention of new tokens over the cached ones, and
attention over whole packed prompts.

``run`` makes one pass through an operator: the framework's own call where ``own`` is set,
else the operator in elementary torch operations in 32 bits. Where a case's sizes come from
the refiner they are its configuration's: chunks of 3 frames of 36 x 64 tokens (6912), 24
heads of 128, a cache of whole frames (pages of 2304 tokens).
"""
import importlib
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
CODES = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}


def listed():
    return [
        # one new token of each of a batch of sequences: latency alone
        dict(name="write tokens", op="write", batch=32, new=1, kv=2048, kv_heads=8, dim=128,
             page=16, dtype="bf16", cache="e4m3", lens="ragged"),
        # chunks of different lengths, one empty, odd positions in their pages
        dict(name="write ragged", op="write", batch=5, new=777, kv=1501, kv_heads=4, dim=80,
             page=32, dtype="fp16", cache="int8", lens="ragged"),
        # one chunk of the refiner into pages of a frame
        dict(name="write chunk", op="write", batch=1, new=6912, kv=13824, kv_heads=24, dim=128,
             page=2304, dtype="bf16", cache="e4m3", lens="full"),
        # a few short sequences, one of them empty
        dict(name="read ragged", op="read", batch=7, new=1, kv=1003, kv_heads=4, dim=64, page=16,
             dtype="fp16", cache="int8", lens="ragged"),
        # long contexts back to 16 bits
        dict(name="read long", op="read", batch=4, new=1, kv=16384, kv_heads=8, dim=128, page=64,
             dtype="bf16", cache="e4m3", lens="full"),
        # a serving step: one token of each sequence, small pages, every length another
        dict(name="decode", op="paged", batch=32, new=1, kv=4096, heads=32, kv_heads=8, dim=128,
             page=16, dtype="bf16", cache="16", lens="ragged", causal=True),
        # long contexts held in 8 bits: the cache's bytes
        dict(name="decode long e4m3", op="paged", batch=8, new=1, kv=32768, heads=32, kv_heads=8,
             dim=128, page=64, dtype="bf16", cache="e4m3", lens="full", causal=True),
        # a few tokens of several sequences, one empty, heads of 64, integer codes
        dict(name="chunk ragged int8", op="paged", batch=6, new=201, kv=3001, heads=16, kv_heads=4,
             dim=64, page=32, dtype="fp16", cache="int8", lens="ragged", causal=True),
        # the next piece of a long prompt over what is cached of it
        dict(name="chunk long e4m3", op="paged", batch=2, new=512, kv=16384, heads=32, kv_heads=8,
             dim=128, page=16, dtype="bf16", cache="e4m3", lens="full", causal=True),
        # one chunk of the refiner over three cached frames and itself, every token seen
        dict(name="chunk frames", op="paged", batch=1, new=6912, kv=13824, heads=24, kv_heads=24,
             dim=128, page=2304, dtype="bf16", cache="16", lens="full", causal=False),
        # a batch of prompts of different lengths
        dict(name="prompts ragged", op="packed", batch=16, new=512, heads=24, kv_heads=24, dim=64,
             dtype="fp16", lens="ragged", causal=True),
        # one long prompt with grouped heads: the tensor cores and the exponentials
        dict(name="prompt long", op="packed", batch=1, new=8192, heads=32, kv_heads=8, dim=128,
             dtype="bf16", lens="full", causal=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the listed ranges: one token to a chunk, odd lengths among them."""
    op = rng.choice(("write", "read", "paged", "paged", "paged", "packed", "packed"))
    while True:
        hkv = rng.choice((1, 2, 4, 8, 12, 24))
        c = dict(op=op, batch=_log(rng, 1, 32), dtype=rng.choice(("bf16", "fp16")), kv_heads=hkv,
                 dim=rng.choice((64, 80, 96, 128, 128)), lens=rng.choice(("full", "ragged")))
        c["new"] = rng.choice((1, _log(rng, 1, 8192)))
        if op in ("paged", "packed"):
            c["heads"] = hkv * rng.choice((1, 1, 2, 4, 8))
            c["causal"] = rng.random() < 0.8
        if op == "packed":
            c["new"] = _log(rng, 1, 8192)
            kv = c["new"]
        else:
            kv = c["kv"] = c["new"] + rng.choice((0, _log(rng, 1, 32768)))
            c["page"] = rng.choice((16, 16, 32, 64, 128, 2304))
            c["cache"] = rng.choice(("int8", "e4m3", "16") if op == "paged" else ("int8", "e4m3"))
        if op == "read":
            c["new"] = 1
        pages = c["batch"] * (kv + c.get("page", 0)) * hkv * c["dim"]
        scores = c["batch"] * c.get("heads", 0) * c["new"] * kv
        if scores <= 24 * 6912 * 13824 // 2 and pages <= 8 * 32768 * 8 * 128:
            return c


# ------------------------------------------------------------------ inputs
def _frac(b):
    return (0.5 + 0.618034 * b) % 1.0


def _lens(case):
    """(new tokens, all tokens) of each sequence: the first has the most; of three or more
    ragged ones the second has none that are new (nothing at all, in a read or a prompt)."""
    B, new, kv = case["batch"], case["new"], case.get("kv", case["new"])
    if case["lens"] == "full":
        return [new] * B, [kv] * B
    n = [new if b == 0 or new == 1 else int(new * _frac(b + 3)) for b in range(B)]
    t = [kv if b == 0 else max(1, int(kv * _frac(b))) for b in range(B)]
    if B >= 3 and case["op"] in ("read", "packed"):
        n[1] = t[1] = 0
    elif B >= 3 and new > 1:
        n[1] = 0
    if case["op"] == "packed":
        return n, list(n)
    return n, [max(x, y) for x, y in zip(n, t)]


def _offsets(n):
    cu = [0]
    for x in n:
        cu.append(cu[-1] + x)
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


def _rows(g, *shape):
    """Keys or values as a projection leaves them: tokens and heads of different size."""
    x = torch.randn(*shape, generator=g, device="cuda")
    return x.mul_(torch.exp(0.3 * torch.randn(*shape[:-1], 1, generator=g, device="cuda")))


def _quantise(x, cache):
    """(codes, scales) of rows: scale = max(max|x| / Q, 1e-12), code = round(x / scale), by the
    reciprocals of Q and of the scale in 32 bits."""
    dt, q = CODES[cache]
    x = x.float()
    scale = (x.abs().amax(-1) * (1.0 / q)).clamp_min(1e-12)
    y = (x * (torch.ones_like(scale) / scale)[..., None]).clamp(-q, q)
    return (torch.round(y) if cache == "int8" else y).to(dt), scale


def _pools(case, g, filled):
    """Pages, their scales and the sequences' tables: every page somewhere in the pool."""
    B, P, H, D = case["batch"], case["page"], case["kv_heads"], case["dim"]
    _, total = _lens(case)
    count = [-(-t // P) for t in total]
    used = sum(count)
    n, width = used + 2, max(1, max(count))
    order = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
    at = torch.arange(width, device="cuda")[None]
    count = torch.tensor(count, device="cuda")[:, None]
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    table[at < count] = order[:used]
    pools = []
    for _ in range(2):
        if not filled:
            dt, _ = CODES[case["cache"]]
            pools.append((torch.zeros(n, P, H, D, dtype=dt, device="cuda"),
                          torch.zeros(n, P, H, device="cuda")))
            continue
        x = _rows(g, n, P, H, D)
        if case["cache"] == "16":
            x, scale = x.to(TYPES[case["dtype"]]), None
        else:
            x, scale = _quantise(x, case["cache"])
        pools.append((x, scale))
    lens = torch.tensor(total, dtype=torch.int32, device="cuda")
    if filled:  # rows past a sequence's length hold whatever the page held before
        last = (lens - 1).clamp_min(0)
        page = table.gather(1, (last // P).long()[:, None])[:, 0]
        behind = torch.arange(P, device="cuda")[None] > (last % P)[:, None]
        behind &= (lens > 0)[:, None]
        for x, scale in pools:
            t = x if scale is None else scale
            view = t[page.clamp_min(0).long()]
            view[behind] = float("nan")
            t.index_copy_(0, page[lens > 0].long(), view[lens > 0])
    (k, ks), (v, vs) = pools
    return dict(k_pages=k, v_pages=v, k_scale=ks, v_scale=vs, table=table, lens=lens)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op, dt = case["op"], TYPES[case["dtype"]]
    n, total = _lens(case)
    T, Hkv, D = sum(n), case["kv_heads"], case["dim"]
    s = {"case": case, "op": op, "cu_q": _offsets(n), "max_q": max(n), "max_kv": max(total)}
    if op != "packed":
        s.update(_pools(case, g, op != "write"))
    if op in ("write", "packed"):
        # keys and values of one projection, side by side
        kv = _rows(g, T, 2, Hkv, D).to(dt)
        s["k"], s["v"] = kv[:, 0], kv[:, 1]
    if op in ("paged", "packed"):
        s["q"] = torch.randn(T, case["heads"], D, generator=g, device="cuda").to(dt)
        s["out"] = torch.empty_like(s["q"])
    if op == "read":
        s["cu_k"] = _offsets(total)
        s["k"], s["v"] = (torch.empty(sum(total), Hkv, D, dtype=dt, device="cuda")
                          for _ in range(2))
    return s


# ------------------------------------------------------------------ plain forms
def _places(cu, first, rows):
    """(sequence, position) of every packed row: row cu[b] + i is at first[b] + i."""
    row = torch.arange(rows, device=cu.device)
    b = torch.searchsorted(cu[1:].long(), row, right=True)
    return b, row - cu[b] + first[b]


def _plain_write(s):
    cu, P = s["cu_q"], s["case"]["page"]
    b, pos = _places(cu, s["lens"] - (cu[1:] - cu[:-1]), s["k"].shape[0])
    page = s["table"][b, pos // P].long()
    out = {}
    for x in ("k", "v"):
        codes, scale = _quantise(s[x], s["case"]["cache"])
        s[x + "_pages"].view(torch.uint8)[page, pos % P] = codes.view(torch.uint8)
        s[x + "_scale"][page, pos % P] = scale
        out[x + "_pages"], out[x + "_scale"] = s[x + "_pages"], s[x + "_scale"]
    return out


def _taken(pages, *at):
    """Pages, or rows of them, in 32 bits."""
    return pages.view(torch.uint8)[at].view(pages.dtype).float()


def _plain_read(s):
    P = s["case"]["page"]
    b, pos = _places(s["cu_k"], torch.zeros_like(s["lens"]), s["k"].shape[0])
    page = s["table"][b, pos // P].long()
    return {x: (_taken(s[x + "_pages"], page, pos % P)
                * s[x + "_scale"][page, pos % P][..., None]).to(s[x].dtype)
            for x in ("k", "v")}


def _padded(x, cu, most):
    """Packed rows [T, ...] as [B, most, ...], zeros behind each sequence, and which are real."""
    at = torch.arange(most, device=x.device)[None]
    real = at < (cu[1:] - cu[:-1])[:, None]
    rows = (cu[:-1, None] + at).clamp_max(max(x.shape[0] - 1, 0)).long()
    return x[rows], real


def _plain_attn(s):
    c, q = s["case"], s["q"]
    T, H, D = q.shape
    qp, real = _padded(q.float(), s["cu_q"], s["max_q"])
    n = (s["cu_q"][1:] - s["cu_q"][:-1])[:, None, None]
    if s["op"] == "packed":
        k, v = (_padded(s[x].float(), s["cu_q"], s["max_q"])[0] for x in ("k", "v"))
        total = n
    else:
        pages = s["table"].clamp_min(0).long()
        k, v = (_taken(s[x + "_pages"], pages).flatten(1, 2) for x in ("k", "v"))
        if s["k_scale"] is not None:
            k, v = (x * y[pages].flatten(1, 2)[..., None]
                    for x, y in ((k, s["k_scale"]), (v, s["v_scale"])))
        total = s["lens"][:, None, None]
    B, Lk, Hkv = k.shape[:3]
    j = torch.arange(Lk, device=q.device)
    keep = j < total
    # the query heads of one key head side by side: [B, Hkv, group * tokens, D]
    qp = qp.view(B, -1, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    p = (qp @ k.permute(0, 2, 3, 1)).mul_(D ** -0.5).view(B, Hkv, H // Hkv, -1, Lk)
    seen = keep
    if c["causal"]:
        i = torch.arange(p.shape[3], device=q.device)[None, :, None]
        seen = keep & (j <= total - n + i)
    p.masked_fill_(~seen[:, None, None], float("-inf"))
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    sums = p.sum(-1, keepdim=True)
    v = torch.where(keep.transpose(1, 2)[..., None], v, 0.0).permute(0, 2, 1, 3)
    o = (p.flatten(2, 3) @ v).view(B, Hkv, H // Hkv, -1, D) / torch.where(sums == 0, 1.0, sums)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, -1, H, D)
    return {"out": o[real].to(q.dtype)}


# ------------------------------------------------------------------ the operators' calls
_ops = None


def run(state):
    global _ops
    s, op = state, state["op"]
    if not own:
        return {"write": _plain_write, "read": _plain_read}.get(op, _plain_attn)(s)
    if _ops is None:
        _ops = importlib.import_module("dreamx-creator_b200").ops
    if op == "write":
        _ops.kv_write(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"],
                      cu_q=s["cu_q"], k_scale=s["k_scale"], v_scale=s["v_scale"])
        return {x: s[x] for x in ("k_pages", "k_scale", "v_pages", "v_scale")}
    if op == "read":
        k, v = _ops.kv_read(s["k_pages"], s["v_pages"], s["table"], s["cu_k"], s["k"], s["v"],
                            k_scale=s["k_scale"], v_scale=s["v_scale"])
        return {"k": k, "v": v}
    if op == "paged":
        return {"out": _ops.paged_attn(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"],
                                       s["out"], cu_q=s["cu_q"], max_q=s["max_q"],
                                       max_kv=s["max_kv"], causal=s["case"]["causal"],
                                       k_scale=s["k_scale"], v_scale=s["v_scale"])}
    return {"out": _ops.packed_attn(s["q"], s["k"], s["v"], s["cu_q"], s["out"],
                                    causal=s["case"]["causal"])}


# ------------------------------------------------------------------ the work of a pass
def work(case):
    op, Hkv, D, P = case["op"], case["kv_heads"], case["dim"], case.get("page", 1)
    e = 2
    n, total = _lens(case)
    held = e if case.get("cache", "16") == "16" else 1
    scales = 0 if held == 2 else 4
    if op in ("write", "read"):
        rows = sum(n if op == "write" else total)
        pages = 4 * sum(-(-t // P) for t in (n if op == "write" else total))
        return {"bytes": 2 * rows * Hkv * (D * (e + 1) + 4) + pages, "flops": 4 * rows * Hkv * D}
    H = case["heads"]
    b = 2 * sum(n) * H * D * e + 2 * Hkv * (D * held + scales) * sum(
        t for x, t in zip(n, total) if x)
    pairs = sum(x * t - (x * (x - 1) // 2 if case["causal"] else 0) for x, t in zip(n, total))
    return {"bytes": b, "flops": 4 * pairs * H * D}


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "write":
        return _exact_write(s)
    if op == "read":
        return {x: torch.cat([_cached(s, x, b) for b in range(case["batch"])]) for x in "kv"}
    q = s["q"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    cu = s["cu_q"].tolist()
    group = case["heads"] // case["kv_heads"]
    for b in range(case["batch"]):
        lo, hi = cu[b], cu[b + 1]
        if lo == hi:
            continue
        if op == "packed":
            k, v = s["k"][lo:hi].double(), s["v"][lo:hi].double()
        else:
            k, v = _cached(s, "k", b), _cached(s, "v", b)
        hidden = None
        if case["causal"]:
            hidden = torch.ones(hi - lo, len(k), dtype=torch.bool, device="cuda")
            hidden = hidden.triu(len(k) - (hi - lo) + 1)
        for h in range(case["heads"]):
            w = torch.einsum("id,jd->ij", q[lo:hi, h].double(), k[:, h // group])
            w /= math.sqrt(case["dim"])
            if hidden is not None:
                w[hidden] = -math.inf
            out[lo:hi, h] = torch.softmax(w, dim=1) @ v[:, h // group]
    return {"out": out}


def _cached(s, x, b):
    """Sequence b's cached rows [length, heads, dim]."""
    length = int(s["lens"][b])
    pages = s["table"][b, : -(-length // s["case"]["page"])].long()
    rows = s[x + "_pages"].view(torch.uint8)[pages].view(s[x + "_pages"].dtype)
    rows = rows.double().flatten(0, 1)[:length]
    if s[x + "_scale"] is None:
        return rows
    return rows * s[x + "_scale"][pages].double().flatten(0, 1)[:length, :, None]


def _exact_write(s):
    """The values that the codes round, and the scales; integer codes have no such value."""
    case, out = s["case"], {}
    cu, lens = s["cu_q"].tolist(), s["lens"].tolist()
    for x in "kv":
        codes = torch.zeros(s[x + "_pages"].shape, dtype=torch.float64, device="cuda")
        scales = torch.zeros(s[x + "_scale"].shape, dtype=torch.float64, device="cuda")
        for b in range(case["batch"]):
            n = cu[b + 1] - cu[b]
            at = torch.arange(lens[b] - n, lens[b], device="cuda")
            page, row = s["table"][b][at // case["page"]].long(), at % case["page"]
            r = s[x][cu[b]: cu[b + 1]].double()
            step = torch.clamp(r.abs().max(2).values / CODES[case["cache"]][1], min=1e-12)
            codes[page, row], scales[page, row] = r / step[..., None], step
        out[x + "_pages"] = codes if case["cache"] == "e4m3" else None
        out[x + "_scale"] = scales
    return out
