"""Caches in pages and packed sequences for tests, and what the operators on them compute, in
64 bits.

Tolerances, with u the unit roundoff of a type (2^-8 bf16, 2^-11 fp16):

- codes and what they stand for: every step is one fp32 operation, rounded as IEEE says, so
  they are equal bit for bit to the same steps in torch.
- attention: a weight is rounded once before the second product, to the queries' type or, with
  a cache of codes, to fp16 (u_p); scores and exponentials are off by less than 2^-11 together
  (scores of these rows are below 16, summed in fp32; the exponential's approximation is
  2^-22), so the output is off by (u_p + 2^-11) sum_j p_j |v_j| / sum_j p_j, plus one rounding u
  of the output. Weights below the smallest fp16 step add 2^-25 |v_j| each; with codes they
  are held in units of at most twice the largest scale of a value, so 2^-24 of that scale times
  |code_j|.
- with bf16 queries many rows' codes are multiplied by their scales and rounded once to fp16 (2^-11
  of each key and value): the values add 2^-11 sum_j p_j |v_j| / sum_j p_j, and the keys move the
  score of key j by up to e_j = 2^-11 scale sum_d |q_d k_jd|, its weight by that part of itself,
  and so the answer by sum_j p_j e_j |v_j| + |o| sum_j p_j e_j over sum_j p_j. What rounds to less
  than fp16's smallest step is 2^-25 of a unit in which the largest scale is 2^6 or more: far
  below the 2^-24 of that scale that stands for the weights.
"""
import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
Q = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def offsets(counts, start=0):
    cu = [start]
    for n in counts:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


def take(t, *at):
    """Indexing of any element type."""
    return t.view(torch.uint8)[at].view(t.dtype)


def quantise(x, dtype):
    """(codes, scales) by the documented fp32 steps."""
    q = Q[dtype]
    x = x.float()
    one = torch.ones((), device=x.device)
    scale = (x.abs().amax(-1) * torch.tensor(1.0 / q, dtype=torch.float32)).clamp_min(1e-12)
    y = x * (one / scale)[..., None]
    if dtype == torch.int8:
        return torch.round(y).to(torch.int8), scale
    return y.clamp(-q, q).to(dtype), scale


class Cache:
    """Pages in random order, tables with junk behind their ends, NaN wherever nothing is."""

    def __init__(self, g, lens, Hkv, D, page, dtype, layout="tokens", spare=3, width=None):
        self.lens, self.page, self.Hkv, self.D, self.dtype = list(lens), page, Hkv, D, dtype
        count = [-(-n // page) for n in lens]
        n, width = sum(count) + spare, width or max([1] + count) + 1
        order = torch.randperm(n, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((len(lens), width), -7, dtype=torch.int32, device="cuda")
        self.table[:, 1::2] = 1 << 30
        at = 0
        for b, c in enumerate(count):
            self.table[b, :c] = order[at:at + c]
            at += c
        shape = (n, page, Hkv, D)
        if layout == "heads":
            shape = (n, Hkv, page, D)
        elif layout == "both":   # k and v of a token side by side
            shape = (n, page, Hkv, 2 * D)
        bufs = [torch.full(shape, 0x7F, dtype=torch.uint8, device="cuda").to(torch.uint8)
                if dtype in Q else torch.full(shape, float("nan"), dtype=dtype, device="cuda")
                for _ in range(1 if layout == "both" else 2)]
        bufs = [b.view(dtype) if dtype in Q else b for b in bufs]
        if layout == "heads":
            bufs = [b.transpose(1, 2) for b in bufs]
        elif layout == "both":
            bufs = [bufs[0][..., :D], bufs[0][..., D:]]
        self.k, self.v = bufs
        self.ks = self.vs = None
        if dtype in Q:
            s = [torch.full((n, Hkv, page), float("nan"), device="cuda") for _ in range(2)]
            self.ks, self.vs = (x.transpose(1, 2) for x in s)
            if layout == "tokens":
                self.ks = self.ks.contiguous()
        self.lens_dev = torch.tensor(self.lens, dtype=torch.int32, device="cuda")

    @property
    def scales(self):
        return dict(k_scale=self.ks, v_scale=self.vs)

    def places(self, b, first, last):
        """(pages, rows) of a sequence's tokens [first, last)."""
        p = torch.arange(first, last, device="cuda")
        return self.table[b][p // self.page].long(), p % self.page

    def put(self, b, first, k, v):
        """Tokens from `first` on as the operator writes them, by torch."""
        at = self.places(b, first, first + k.shape[0])
        for x, pool, scale in ((k, self.k, self.ks), (v, self.v, self.vs)):
            if scale is not None:
                x, s = quantise(x, self.dtype)
                scale[at] = s
                pool.view(torch.uint8)[at] = x.view(torch.uint8)
            else:
                pool[at] = x

    def fill(self, g, dtype, size=0.3):
        for b, n in enumerate(self.lens):
            k, v = (randn(g, n, self.Hkv, self.D) * torch.exp(size * randn(g, n, self.Hkv, 1))
                    for _ in range(2))
            self.put(b, 0, k.to(dtype), v.to(dtype))
        return self

    def rows(self, b, which, n=None):
        """(values [n, Hkv, D] in 64 bits, codes or None, scales or None)"""
        n = self.lens[b] if n is None else n
        pool, scale = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        at = self.places(b, 0, n)
        if scale is None:
            return pool[at].double(), None, None
        codes, s = pool.view(torch.uint8)[at].view(self.dtype), scale[at]
        codes = codes.float().double()
        return codes * s.double()[..., None], codes, s.double()


def attention(q, k, v, scale, causal, u_p, out_dtype, codes=None, vs=None, hide=None):
    """(output, tolerance) of one sequence: q [n, H, D], k, v [L, Hkv, D] in 64 bits.
    ``hide`` (bool [L]): keys that are not there."""
    n, H, D = q.shape
    L, Hkv = k.shape[:2]
    out = torch.zeros(n, H, D, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    seen = torch.ones(n, L, dtype=torch.bool, device=q.device)
    if causal:
        seen = seen.tril(L - n)
    if hide is not None:
        seen &= ~hide
    any_ = seen.any(1)
    for h in range(H):
        g = h // (H // Hkv)
        s = (q[:, h].double() @ k[:, g].t()) * scale
        s = s.masked_fill(~seen, float("-inf"))
        p = torch.softmax(s, 1)
        p = torch.where(any_[:, None], p, 0.0)
        o, a = p @ v[:, g], p @ v[:, g].abs()
        out[:, h] = o
        tol[:, h] = (u_p + 2.0 ** -11) * a + U[out_dtype] * o.abs() * (1 + 2.0 ** -6) + 1e-30
        if codes is not None and out_dtype == torch.bfloat16:
            e = 2.0 ** -11 * scale * (q[:, h].double().abs() @ k[:, g].abs().t())
            pe = p * torch.where(seen, e, 0.0)
            tol[:, h] += 2.0 ** -11 * a + pe @ v[:, g].abs() + o.abs() * pe.sum(1, keepdim=True)
        if codes is not None:
            tol[:, h] += 2.0 ** -24 * vs[:, g].max() * codes[:, g].abs().sum(0) if L else 0
        elif u_p == U[torch.float16]:
            tol[:, h] += 2.0 ** -25 * v[:, g].abs().sum(0)
        if out_dtype == torch.float16:
            tol[:, h] += 2.0 ** -25
    return out, tol


def check_paged(cache, q, cu, out, causal, scale, hide=None):
    for b in range(len(cache.lens)):
        lo, hi = int(cu[b]), int(cu[b + 1])
        if lo == hi:
            continue
        k, _, _ = cache.rows(b, "k")
        v, codes, vs = cache.rows(b, "v")
        if hide is not None:
            k, v = (x.masked_fill(hide[b][:, None, None], 0) for x in (k, v))
        u_p = U[q.dtype if codes is None else torch.float16]
        ref, tol = attention(q[lo:hi], k, v, scale, causal, u_p, q.dtype, codes, vs,
                             None if hide is None else hide[b])
        err = (out[lo:hi].double() - ref).abs()
        assert (err <= tol).all(), (b, float((err / tol).max()), (err > tol).nonzero()[:5].tolist())


def check_packed(q, k, v, cu_q, cu_k, out, causal, scale):
    for b in range(cu_q.numel() - 1):
        lo, hi = int(cu_q[b]), int(cu_q[b + 1])
        k0, k1 = int(cu_k[b]), int(cu_k[b + 1])
        if lo == hi:
            continue
        ref, tol = attention(q[lo:hi], k[k0:k1].double(), v[k0:k1].double(), scale, causal,
                             U[q.dtype], q.dtype)
        err = (out[lo:hi].double() - ref).abs()
        assert (err <= tol).all(), (b, float((err / tol).max()), (err > tol).nonzero()[:5].tolist())
