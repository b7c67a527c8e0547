"""Key/value cache held in 4 bits: written as tokens arrive, read back, attended to.

A request cache holds the keys and values of a history's tokens. In bf16 it costs
``4 * head_dim`` bytes a token and head; here a head's row of a token is one bf16
scale and ``head_dim`` 4-bit codes, ``head_dim + 4`` bytes for its key and value:

* ``s = bf16(max |x| / 7)``, ``c = clamp(round(x / s), -7, 7)`` (ties to even), value
  ``s * c``; a row of zeros (or one whose ``s`` underflows) has ``s = 0`` and ``c = 0``,
  a row that holds an infinity or a NaN reads back as NaN;
* tokens lie in pages of ``page`` positions, found through a table per cache row, so
  rows of very different lengths share one pool.

``kv_cache_write`` appends (or writes from a given position), ``kv_cache_read`` gives
the values of a run of positions, ``cached_attention`` attends to a row: a single new
token whose key is in the cache already, or candidates that bring fresh keys of their
own (OneTrans NS tokens over their request's history), with an optional sliding
window and always-visible first tokens. None of them has a gradient.

CUDA: the kernels of ``csrc/kv_cache.cu`` (bf16, head widths 32 and 64); rows, pages
and positions outside the cache are skipped (attention: hidden) and recorded in the device
error word (``check_error_word``). CPU: the same contract in fp32 PyTorch, which raises
instead.
"""

from __future__ import annotations

import math

import torch

from ..utils.trace import trace_range
from ._ext import error_word, ext

HEAD_DIMS = (32, 64)
MAX_CODE = 7


class QuantizedKVCache:
    """``rows`` histories of up to ``max_tokens`` tokens of ``kv_heads`` heads.

    ``table [rows, ceil(max_tokens / page)]`` (int32) names the page of each run of
    ``page`` positions; by default row ``r`` owns pages ``r * per_row ..``. A table with
    fewer pages than that (``num_pages``) is the caller's to fill before it writes. A page
    may be shared between rows that only read it. ``max_tokens`` 0: rows that hold nothing."""

    def __init__(self, rows: int, max_tokens: int, kv_heads: int, head_dim: int, page: int = 64,
                 table: torch.Tensor | None = None, num_pages: int | None = None, device=None) -> None:
        if rows < 1 or max_tokens < 0 or kv_heads < 1:
            raise ValueError(f"key/value cache: rows {rows} and kv_heads {kv_heads} must be positive, max_tokens "
                             f"{max_tokens} not negative")
        if head_dim not in HEAD_DIMS:
            raise NotImplementedError(f"key/value cache: head width {head_dim}, the cache takes {HEAD_DIMS}")
        if page < 16 or page & (page - 1):
            raise ValueError(f"key/value cache: page {page} must be a power of two of at least 16")
        per_row = -(-max_tokens // page)
        if per_row * page >= 2 ** 31:
            raise ValueError(f"key/value cache: {max_tokens} tokens a row")
        device = torch.device(device) if device is not None else torch.device("cpu")
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        if num_pages is None:
            num_pages = rows * per_row
        if num_pages < min(per_row, 1):
            raise ValueError(f"key/value cache: num_pages {num_pages}")
        if table is None:
            if num_pages < rows * per_row:
                raise ValueError(f"key/value cache: {rows} rows of {per_row} pages need a table to share {num_pages}")
            table = torch.arange(rows * per_row, dtype=torch.int32, device=device).view(rows, per_row)
        else:
            if table.shape != (rows, per_row):
                raise ValueError(f"key/value cache: table {tuple(table.shape)}, expected {(rows, per_row)}")
            if table.is_floating_point():
                raise TypeError("key/value cache: the page table holds whole numbers")
            if table.dtype is not torch.int32:  # past 32 bits: outside any cache, not wrapped into it
                table = table.to(torch.int64).clamp(-2 ** 31, 2 ** 31 - 1)
            table = table.to(device=device, dtype=torch.int32).contiguous()
        self.rows, self.kv_heads, self.head_dim, self.page = rows, kv_heads, head_dim, page
        self.num_pages, self.device = num_pages, device
        self.table = table
        self.lengths = torch.zeros(rows, dtype=torch.int32, device=device)
        self.codes = torch.empty(num_pages, kv_heads, 2, page, head_dim // 2, dtype=torch.uint8, device=device)
        self.err = error_word(device) if device.type == "cuda" else None
        self.scales = torch.empty(num_pages, kv_heads, page, 2, dtype=torch.bfloat16, device=device)

    @property
    def capacity(self) -> int:
        """Positions a row can hold."""

        return self.table.shape[1] * self.page

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + 2 * self.scales.numel()

    def reset(self, rows: torch.Tensor | None = None) -> None:
        """Empties the cache, or only ``rows`` (whole numbers)."""

        if rows is None:
            self.lengths.zero_()
            return
        rows = rows.reshape(-1).to(self.device)
        none = torch.empty(rows.shape[0], 0, self.kv_heads * self.head_dim, dtype=torch.bfloat16, device=self.device)
        # nothing written from position 0: rows outside the cache are met like those of any write
        kv_cache_write(self, none, none, start=torch.zeros_like(rows, dtype=torch.int32), rows=rows)

    # ------------------------------------------------------------------ definition in PyTorch
    def _slots(self, rows: torch.Tensor, pos: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        """Page and slot of positions ``pos`` of ``rows`` (broadcast together)."""

        pg = self.table[rows, pos // self.page].long()
        if bool(((pg < 0) | (pg >= self.num_pages)).any()):
            raise ValueError("key/value cache: page outside the cache")
        return pg, pos % self.page

    def values(self, rows: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
        """fp32 ``[..., kv_heads, 2, head_dim]`` at ``pos`` of ``rows``."""

        pg, slot = self._slots(rows, pos)
        n = self.codes[pg, :, :, slot]
        c = torch.stack([n & 15, n >> 4], -1).flatten(-2).float() - 8.0
        return c * self.scales[pg, :, slot].float().unsqueeze(-1)


# ----------------------------------------------------------------------------- checks
# (of the definitions on the CPU; the native entry points make the same ones)
def _index(t: torch.Tensor | None, n: int, cache: QuantizedKVCache, name: str) -> torch.Tensor | None:
    if t is None:
        return None
    if t.is_floating_point() or t.dtype == torch.bool:
        raise TypeError(f"{name} holds whole numbers, not {t.dtype}")
    if t.shape != (n,):
        raise ValueError(f"{name} {tuple(t.shape)}, expected ({n},)")
    if t.device != cache.device:
        raise ValueError(f"{name} on {t.device}, the cache on {cache.device}")
    return t


def _rows(t: torch.Tensor | None, n: int, cache: QuantizedKVCache) -> torch.Tensor | None:
    t = _index(t, n, cache, "rows")
    if t is not None and bool(((t < 0) | (t >= cache.rows)).any()):
        raise IndexError(f"key/value cache: rows outside the cache's {cache.rows}")
    return t


def _tokens(t: torch.Tensor, width: int, cache: QuantizedKVCache, name: str) -> None:
    if t.dim() != 3 or t.shape[2] != width:
        raise ValueError(f"{name} {tuple(t.shape)}, expected [rows, tokens, {width}]")
    if t.device != cache.device:
        raise ValueError(f"{name} on {t.device}, the cache on {cache.device}")
    if not t.is_floating_point():
        raise TypeError(f"{name} must be a floating type, not {t.dtype}")
    if torch.is_grad_enabled() and t.requires_grad:
        raise RuntimeError("the key/value cache has no gradient: call it under torch.no_grad() or on detached tensors")


# ----------------------------------------------------------------------------- write
def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes ``-7 .. 7`` (int8) and bf16 scales of the rows (last dimension) of ``x``."""

    x = x.float()
    top = x.abs().amax(-1)
    finite = torch.isfinite(top)
    s = torch.where(finite, top / float(MAX_CODE), torch.nan).to(torch.bfloat16)
    sf = s.float().unsqueeze(-1)
    ok = finite.unsqueeze(-1) & (sf > 0)
    c = torch.where(ok, torch.round(x / torch.where(ok, sf, torch.ones_like(sf))), torch.zeros_like(x))
    return c.clamp(-MAX_CODE, MAX_CODE).to(torch.int8), s


def kv_cache_write_reference(cache: QuantizedKVCache, k, v, start=None, kstart=None, rows=None) -> None:
    """PyTorch definition of ``kv_cache_write``."""

    n, T, _ = k.shape
    dev = cache.device
    r = (torch.arange(n, device=dev) if rows is None else rows.long())
    first = (torch.zeros(n, device=dev, dtype=torch.long) if kstart is None else kstart.long().clamp(0, T))
    begin = cache.lengths[r].long() if start is None else start.long()
    if bool(((begin < 0) | (begin > cache.capacity)).any()):
        raise ValueError("key/value cache: start outside the row")
    x = torch.stack([k, v], 2).view(n, T, 2, cache.kv_heads, cache.head_dim).to(torch.bfloat16)
    c, s = quantize_rows(x)
    u = (c + 8).to(torch.uint8)
    packed = (u[..., 0::2] | (u[..., 1::2] << 4)).transpose(2, 3)
    t = torch.arange(T, device=dev)
    pos = begin.view(-1, 1) + t - first.view(-1, 1)
    live = t >= first.view(-1, 1)
    if bool((live & (pos >= cache.capacity)).any()):
        raise ValueError("key/value cache: a row is full")
    i, ti = live.nonzero(as_tuple=True)
    pg, slot = cache._slots(r[i], pos[i, ti])
    cache.codes[pg, :, :, slot] = packed[i, ti]
    cache.scales[pg, :, slot] = s.transpose(2, 3)[i, ti]
    cache.lengths[r] = (begin + T - first).to(torch.int32)


def kv_cache_write(cache: QuantizedKVCache, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor | None = None,
                   kstart: torch.Tensor | None = None, rows: torch.Tensor | None = None) -> None:
    """Quantises ``k, v [n, T, kv_heads * head_dim]`` into cache rows ``rows [n]`` (distinct;
    default all rows in order). Source row ``i``'s tokens ``kstart[i] ..`` (default 0: none is
    padding) go to positions ``start[i] ..`` (default: append), and the row's length becomes
    the end of what was written. A start past the row's length leaves a gap whose values are
    not defined."""

    with trace_range("mdl.kv_cache.write"):
        if cache.err is not None:
            ext().kv_write(cache.codes, cache.scales, cache.table, cache.lengths, cache.err, k, v, rows, start, kstart)
            return
        width = cache.kv_heads * cache.head_dim
        _tokens(k, width, cache, "k")
        _tokens(v, width, cache, "v")
        n = k.shape[0]
        if v.shape != k.shape:
            raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} differ")
        if rows is None and n != cache.rows:
            raise ValueError(f"{n} source rows for {cache.rows} cache rows: give rows")
        kv_cache_write_reference(cache, k, v, _index(start, n, cache, "start"), _index(kstart, n, cache, "kstart"),
                                 _rows(rows, n, cache))


# ----------------------------------------------------------------------------- read
def kv_cache_read(cache: QuantizedKVCache, count: int, start: torch.Tensor | None = None,
                  rows: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16
                  ) -> tuple[torch.Tensor, torch.Tensor]:
    """``(k, v)``, each ``[n, count, kv_heads * head_dim]``: the values at positions ``start[i]
    .. start[i] + count`` (default from 0) of rows ``rows [n]`` (default all); zero past a row's
    length. fp32 holds them exactly; bf16 rounds once."""

    with trace_range("mdl.kv_cache.read"):
        if dtype is not torch.bfloat16 and dtype is not torch.float32:
            raise TypeError(f"the cache reads back bf16 or fp32, not {dtype}")
        if cache.err is not None:
            return ext().kv_read(cache.codes, cache.scales, cache.table, cache.lengths, cache.err, count, rows, start,
                                 dtype is torch.float32)
        if count < 0:
            raise ValueError(f"count {count}")
        n = cache.rows if rows is None else rows.shape[0]
        rows = _rows(rows, n, cache)
        start = _index(start, n, cache, "start")
        width = cache.kv_heads * cache.head_dim
        r = (torch.arange(n) if rows is None else rows.long()).view(-1, 1)
        pos = (0 if start is None else start.long().view(-1, 1)) + torch.arange(count)
        if bool((pos < 0).any()):
            raise ValueError("key/value cache: start outside the row")
        live = pos < cache.lengths[r].long()
        x = torch.zeros(n, count, cache.kv_heads, 2, cache.head_dim)
        i, ti = live.expand(n, count).nonzero(as_tuple=True)
        x[i, ti] = cache.values(r.expand(n, count)[i, ti], pos.expand(n, count)[i, ti])
        x = x.to(dtype)
        return x[..., 0, :].reshape(n, count, width), x[..., 1, :].reshape(n, count, width)


# ----------------------------------------------------------------------------- attend
def cached_attention_reference(q, cache: QuantizedKVCache, rows=None, k_new=None, v_new=None, window: int = 0,
                               sinks: int = 0, scale: float | None = None) -> torch.Tensor:
    """fp32 PyTorch definition of ``cached_attention``."""

    B, N, W = q.shape
    G, hd = cache.kv_heads, cache.head_dim
    H = W // hd
    scale = scale if scale else 1.0 / math.sqrt(hd)
    dev = q.device
    r = (torch.arange(B, device=dev) if rows is None else rows.long())
    ln = cache.lengths[r].long()
    T = int(ln.max()) if B else 0
    kpos = torch.arange(T, device=dev)
    pos = torch.minimum(kpos.view(1, -1), (ln.view(-1, 1) - 1).clamp(min=0))
    kv = cache.values(r.view(-1, 1).expand(B, T), pos) if T else torch.zeros(B, 0, G, 2, hd, device=dev)
    kv = kv.permute(3, 0, 2, 1, 4).repeat_interleave(H // G, 2)                   # [2, B, H, T, hd]
    n = torch.arange(N, device=dev)
    ln = ln.view(-1, 1, 1)
    qpos = (ln if k_new is not None else ln - N) + n.view(1, -1, 1)

    def visible(at):
        ok = at <= qpos
        return ok & ((qpos - at < window) | (at < sinks)) if window else ok

    allowed = (kpos < ln) & visible(kpos)
    k, v = kv[0], kv[1]
    if k_new is not None:
        kn = k_new.float().view(B, N, G, hd).transpose(1, 2).repeat_interleave(H // G, 1)
        vn = v_new.float().view(B, N, G, hd).transpose(1, 2).repeat_interleave(H // G, 1)
        k, v = torch.cat([k, kn], 2), torch.cat([v, vn], 2)
        allowed = torch.cat([allowed, visible(ln + n.view(1, 1, -1))], 2)
    qh = q.float().view(B, N, H, hd).transpose(1, 2)
    s = (qh @ k.transpose(-1, -2)) * scale
    allowed = allowed.unsqueeze(1)
    p = torch.softmax(s.masked_fill(~allowed, float("-inf")), -1)
    p = torch.where(allowed, p, torch.zeros_like(p))                              # rows that see nothing
    v = torch.where(allowed.any(2).unsqueeze(-1), v, torch.zeros_like(v))         # keys that nobody sees
    return (p @ v).transpose(1, 2).reshape(B, N, W)


def cached_attention(q: torch.Tensor, cache: QuantizedKVCache, rows: torch.Tensor | None = None,
                     k_new: torch.Tensor | None = None, v_new: torch.Tensor | None = None, window: int = 0,
                     sinks: int = 0, scale: float | None = None) -> torch.Tensor:
    """``q [B, N, heads * head_dim]`` over cache row ``rows[b]`` (default row ``b``) ->
    ``[B, N, heads * head_dim]``.

    Query ``n`` of batch row ``b`` sits at position ``length - N + n`` (its token is in the
    cache), or, with fresh keys ``k_new, v_new [B, N, kv_heads * head_dim]`` that are not in the
    cache, at ``length + n``. It sees the positions up to its own: all of them (``window`` 0),
    or the last ``window`` and the first ``sinks``; a query that sees none gives zero. Heads
    ``g * heads / kv_heads ..`` share key head ``g``. ``scale`` (positive) defaults to ``head_dim ** -0.5``.
    On the GPU an infinity or a NaN in a cached token reaches only the queries that see it; one in
    ``v_new`` may reach every query of its batch row."""

    with trace_range("mdl.attention.cached"):
        if scale is not None and not 0.0 < scale < math.inf:
            raise ValueError(f"cached attention: scale {scale} must be positive")
        if cache.err is not None:
            return ext().kv_attend(cache.codes, cache.scales, cache.table, cache.lengths, cache.err, q, rows, k_new,
                                   v_new, window, sinks, scale or 0.0)
        G, hd = cache.kv_heads, cache.head_dim
        if q.dim() != 3 or q.shape[2] % (G * hd) or q.shape[2] == 0:
            raise ValueError(f"q {tuple(q.shape)}: the width must be a multiple of {G} key heads of {hd}")
        if window < 0 or sinks < 0:
            raise ValueError(f"window {window} and sinks {sinks} must not be negative")
        if (k_new is None) != (v_new is None):
            raise ValueError("k_new and v_new come together")
        B, N, width = q.shape
        _tokens(q, width, cache, "q")
        if rows is None and B != cache.rows:
            raise ValueError(f"{B} batch rows for {cache.rows} cache rows: give rows")
        rows = _rows(rows, B, cache)
        if k_new is not None:
            _tokens(k_new, G * hd, cache, "k_new")
            _tokens(v_new, G * hd, cache, "v_new")
            if k_new.shape[:2] != (B, N) or v_new.shape[:2] != (B, N):
                raise ValueError(f"k_new {tuple(k_new.shape)} and v_new {tuple(v_new.shape)} for {B} x {N} queries")
        return cached_attention_reference(q, cache, rows, k_new, v_new, window, sinks, scale).to(q.dtype)
