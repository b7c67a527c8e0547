"""Sliding-window attention with always-visible first tokens over long histories.

``windowed_attention(qkv, kstart, heads, lq, window, sinks)`` is the suffix attention of
``ops/attention.py`` with a bounded view: query token ``p`` of a sample whose first valid
token is ``kst = kstart[b]`` sees key ``j`` iff

``kst <= j <= p  and  (p - j < window  or  j - kst < sinks)``

so a query costs ``window + sinks`` keys whatever the length of the history. The first valid
tokens stay visible because a softmax trained with a window parks weight on them.

* ``qkv [B, Lk, (heads + 2 * kv_heads) * head_dim]``: per token the query heads, then the key
  heads, then the value heads; ``heads // kv_heads`` neighbouring query heads share one key
  head (``kv_heads`` defaults to ``heads``);
* the queries are the last ``lq`` tokens; padding is a per-sample prefix (``kstart``), is
  never read, and its queries give zero;
* returns ``[B, lq, heads * head_dim]``; the gradient of a shared key head sums over the
  query heads that share it;
* an infinity or a NaN in a valid token may reach every query of its sample, also those that
  do not see the token (a weight of zero times it is a NaN).

CUDA: the tcgen05 kernels of ``csrc/window_attn.cu`` (bf16, head widths 32 and 64), forward
and backward without atomics; a second derivative is refused. CPU: the same contract in fp32 PyTorch.
"""

from __future__ import annotations

import math

import torch

from ..utils.trace import trace_range
from ._ext import error_word, ext

HEAD_DIMS = (32, 64)


def windowed_attention_reference(qkv: torch.Tensor, kstart: torch.Tensor, heads: int, lq: int, window: int,
                                 sinks: int = 0, kv_heads: int | None = None, scale: float | None = None
                                 ) -> torch.Tensor:
    """fp32 PyTorch definition (differentiable)."""

    B, Lk, W = qkv.shape
    G = kv_heads or heads
    hd = W // (heads + 2 * G)
    scale = scale if scale else 1.0 / math.sqrt(hd)
    x = qkv.float().view(B, Lk, heads + 2 * G, hd)
    ks = kstart.to(qkv.device).long().clamp(0, Lk).view(B, 1, 1)
    kpos = torch.arange(Lk, device=qkv.device)
    # padding takes no part: neither its values nor their gradients
    x = torch.where((kpos.view(1, Lk) >= ks.view(B, 1)).view(B, Lk, 1, 1), x, torch.zeros_like(x)).transpose(1, 2)
    q = x[:, :heads, Lk - lq:]
    k = x[:, heads:heads + G].repeat_interleave(heads // G, 1)
    v = x[:, heads + G:].repeat_interleave(heads // G, 1)
    s = torch.matmul(q, k.transpose(-1, -2)) * scale                       # [B, H, lq, Lk]
    qpos = torch.arange(Lk - lq, Lk, device=qkv.device).view(lq, 1)
    allowed = (kpos >= ks) & (kpos <= qpos) & ((qpos - kpos < window) | (kpos - ks < sinks))
    allowed = allowed.unsqueeze(1)
    p = torch.softmax(s.masked_fill(~allowed, float("-inf")), dim=-1)
    p = torch.where(allowed, p, torch.zeros_like(p))                       # rows without a visible key
    return torch.matmul(p, v).transpose(1, 2).reshape(B, lq, heads * hd)


def window_attention_fwd(qkv, ks, heads: int, kv_heads: int, lq: int, window: int, sinks: int, scale: float = 0.0,
                         keep: bool = True):
    """Native forward: ``out [B, lq, heads * hd]`` bf16 and, for a backward (``keep``), what
    rounding took off it and the log-sum-exp ``[B, heads, lq]`` (else None and a workspace)."""

    return ext().window_attn_fwd(qkv, ks, heads, kv_heads, lq, window, sinks, scale, error_word(qkv.device), keep)


def window_attention_bwd(qkv, ks, out, out_lo, lse, dout, heads: int, kv_heads: int, lq: int, window: int, sinks: int,
                         scale: float = 0.0) -> torch.Tensor:
    """Native backward: the gradient of ``qkv`` (bf16, contiguous)."""

    return ext().window_attn_bwd(qkv, ks, out, out_lo, lse, dout, heads, kv_heads, lq, window, sinks, scale,
                                 error_word(qkv.device))


def windowed_attention(qkv: torch.Tensor, kstart: torch.Tensor, heads: int, lq: int, window: int, sinks: int = 0,
                       kv_heads: int | None = None, scale: float | None = None) -> torch.Tensor:
    """See the module's text; ``scale`` (positive) defaults to ``head_dim ** -0.5``."""

    with trace_range("mdl.attention.windowed"):
        G = heads if kv_heads is None else kv_heads
        if heads < 1 or G < 1 or heads % G:
            raise ValueError(f"windowed attention: {heads} query heads over {G} key heads")
        if qkv.dim() != 3 or qkv.shape[2] == 0 or qkv.shape[2] % (heads + 2 * G):
            raise ValueError(f"windowed attention: qkv {tuple(qkv.shape)} does not hold {heads} + 2 * {G} heads")
        B, Lk, W = qkv.shape
        if not 0 <= lq <= Lk:
            raise ValueError(f"windowed attention: {lq} queries of {Lk} tokens")
        if window < 1 or sinks < 0:
            raise ValueError(f"windowed attention: window {window} must be positive, sinks {sinks} not negative")
        if scale is not None and not 0.0 < scale < math.inf:
            raise ValueError(f"windowed attention: scale {scale} must be positive")
        if kstart.shape != (B,) or kstart.is_floating_point() or kstart.dtype == torch.bool:
            raise ValueError(f"windowed attention: kstart {tuple(kstart.shape)} {kstart.dtype}, expected whole numbers "
                             f"({B},)")
        if not qkv.is_cuda:
            return windowed_attention_reference(qkv, kstart, heads, lq, window, sinks, G, scale)
        hd = W // (heads + 2 * G)
        if hd not in HEAD_DIMS:
            raise NotImplementedError(f"windowed attention: head width {hd}, the native kernels take {HEAD_DIMS}")
        if qkv.dtype != torch.bfloat16:
            raise TypeError(f"windowed attention: qkv must be bf16, not {qkv.dtype}")
        if kstart.device != qkv.device:
            raise ValueError(f"windowed attention: kstart on {kstart.device}, qkv on {qkv.device}")
        if B == 0 or lq == 0:
            return qkv[:, :lq, :heads * hd] * 0
        s0, s1, s2 = qkv.stride()
        if s2 != 1 or s1 % 8 or s0 % 8 or s1 < W or s0 < s1 or qkv.data_ptr() % 16:
            qkv = qkv.contiguous()
            if qkv.data_ptr() % 16:
                qkv = qkv.clone()
        ks = kstart
        if ks.dtype is not torch.int32:
            ks = ks.to(torch.int64).clamp(0, Lk).to(torch.int32)  # what lies past 32 bits must not wrap
        ks = ks.contiguous()
        return ext().windowed_attention(qkv, ks, heads, G, lq, min(window, Lk), min(sinks, Lk),
                                        scale or 0.0, error_word(qkv.device))
