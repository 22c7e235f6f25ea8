"""Text-conditioning blocks in 8-bit integers: the integer operators as they are used together.

A stack of pre-norm blocks refines video tokens by attending to a prompt's encoder states,
every Linear an ``Int8Linear``. Per block:

  add_rms_quant(x, y)    x + y, RMS norm, int8 rows   (y: the block before's output; in a
                         stack the sum takes its place)
  int8_gemm              q = W_q n
  cross_attn             q over the prompt's k | v, each sample its own length
  quant_rows, int8_gemm  y = W_o a

The prompt's k | v of every block are computed once per prompt (``text_kv``: one
``quant_rows`` of the encoder's states and an ``int8_gemm`` per block, k and v side by side)
and read in place by every step, be it a chunk of tokens or a single one.

  stack = CrossStack.random_init(dim=3072, text_dim=4096, heads=24, layers=4)
  kv = stack.text_kv(states)                    # [B, text_len, text_dim], padded prompts
  out = stack(x, kv, kv_lens=lens)              # [B, tokens, dim], int32 [B]
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _lib, ops
from .int8_linear import Int8Linear


class CrossBlock(nn.Module):
    """One block: ``norm``, ``q``, ``kv`` (k | v over the encoder's states) and ``o``."""

    def __init__(self, norm_weight, q, kv, o, heads, kv_heads, eps=1e-6):
        super().__init__()
        self.heads, self.kv_heads, self.eps = int(heads), int(kv_heads), float(eps)
        self.head_dim = q.out_features // self.heads
        if (q.out_features != self.heads * self.head_dim or o.in_features != q.out_features
                or kv.out_features != 2 * self.kv_heads * self.head_dim
                or self.heads % self.kv_heads):
            raise _lib.SrditError(f"{self.heads} heads of {self.head_dim} and {self.kv_heads} key "
                                  f"heads do not fit q {q.out_features}, kv {kv.out_features}, "
                                  f"o {o.in_features}")
        self.register_buffer("norm", norm_weight.detach().clone(), persistent=False)
        self.q, self.kv, self.o = q, kv, o

    def forward(self, x, y, kv, kv_lens=None, key_mask=None, *, into_y=False):
        """x [B, L, dim] the residual stream, y [B, L, dim] what is still to be added to it
        (or None), kv [B, Lk, 2, kv_heads, head_dim]. Returns (x + y, this block's output);
        with ``into_y`` the sum takes the place of a contiguous y, else y is left as it is."""
        B, L, D = x.shape
        rows = ops.as_rows(x, D)
        add = None if y is None else ops.as_rows(y, D)
        n, scale, total = ops.add_rms_quant(rows, self.norm, self.eps, residual=add,
                                            sum_out=add if into_y else None)
        q = self.q.forward_codes(n, scale, x.dtype).view(B, L, self.heads, self.head_dim)
        a = ops.cross_attn(q, kv[:, :, 0], kv[:, :, 1], kv_lens=kv_lens, key_mask=key_mask)
        out = self.o.forward_codes(*ops.quant_rows(a.view(B * L, self.o.in_features)), x.dtype)
        return (x if total is None else total.view(B, L, D)), out.view(B, L, D)


class CrossStack(nn.Module):
    """Blocks in a row; each block's output is added to the stream by the next one's norm."""

    def __init__(self, blocks):
        super().__init__()
        self.blocks = nn.ModuleList(blocks)

    @classmethod
    def random_init(cls, *, dim, text_dim, heads, kv_heads=None, layers=1, device="cuda",
                    dtype=torch.bfloat16, seed=0):
        """Seeded random weights: Linears N(0, 1 / inputs), norms 1 + N(0, 0.1)."""
        if not torch.cuda.is_available():
            raise _lib.SrditError("CrossStack needs a CUDA device (there is no CPU path)")
        kv_heads = kv_heads or heads
        g = torch.Generator(device=device).manual_seed(seed)

        def lin(n_out, n_in):
            w = torch.randn(n_out, n_in, generator=g, device=device) / n_in ** 0.5
            b = 0.02 * torch.randn(n_out, generator=g, device=device)
            return Int8Linear(w.to(dtype), b.to(dtype))

        hd = dim // heads
        return cls([CrossBlock((1 + 0.1 * torch.randn(dim, generator=g, device=device)).to(dtype),
                               lin(dim, dim), lin(2 * kv_heads * hd, text_dim), lin(dim, dim),
                               heads, kv_heads) for _ in range(layers)])

    def text_kv(self, states):
        """Every block's k | v [B, Lk, 2, kv_heads, head_dim] of the encoder's states
        [B, Lk, text_dim], once per prompt."""
        B, Lk, D = states.shape
        q, scale = ops.quant_rows(ops.as_rows(states, D))
        return [b.kv.forward_codes(q, scale, states.dtype).view(B, Lk, 2, b.kv_heads, b.head_dim)
                for b in self.blocks]

    def forward(self, x, kv, kv_lens=None, key_mask=None):
        """x [B, L, dim] through every block: the residual stream with all outputs added.
        A row whose prompt has no visible key only gets the output Linears' biases."""
        y = None
        for block, bkv in zip(self.blocks, kv):
            x, y = block(x, y, bkv, kv_lens, key_mask, into_y=True)  # y is ours
        return x + y
