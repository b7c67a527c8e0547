"""4-bit key/value cache: quantising writes, reads and the attention over it, against plain
64-bit computations, on the CPU definitions and on the CUDA kernels.

Tolerances. The codes and scales are exact: a quotient of two bf16 numbers is either a tie or
at least 1/1020 away from one, so every correctly rounded route gives the same code. The
attention rounds the weighted probabilities and the output to bf16 (8 significant bits: up to
2^-8 relative each) and carries scores with errors below about 2^-13, so an output element is
within (2^-8 + 2^-8 + 2^-12) * sum_j p_j |v_j| of the exact one, cross terms below 2^-15; the
tests allow 1.05 * 2^-7 of that sum. The fp32 definitions on the CPU are held to 2^-16 of it.
"""

import math

import pytest
import torch

from mdl_b200.ops.kv_cache import (QuantizedKVCache, cached_attention, cached_attention_reference, kv_cache_read,
                                   kv_cache_write, quantize_rows)

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
GPU = pytest.mark.gpu


def _round4(x):
    """Values that the codes of bf16 rows ``x`` stand for, in 64 bits."""

    x = x.double()
    s = (x.abs().amax(-1, keepdim=True) / 7).to(torch.bfloat16).double()
    safe = torch.where(s > 0, s, torch.ones_like(s))
    return torch.where(s > 0, torch.round(x / safe).clamp(-7, 7) * s, torch.zeros_like(x))


def _kv(n, T, G, hd, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    k = (torch.randn(n, T, G * hd, generator=g) * 1.5).bfloat16().to(device)
    v = torch.randn(n, T, G * hd, generator=g).bfloat16().to(device)
    return k, v


def _int(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def _check_errors(device):
    if device == "cuda":
        from mdl_b200.ops._ext import check_error_word

        torch.cuda.synchronize()
        check_error_word(torch.device("cuda", 0))


def _shuffled(rows, tokens, G, hd, page, device, seed=3, spare=2):
    per = -(-tokens // page)
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(rows * per + spare, generator=g)[:rows * per].int().view(rows, per).to(device)
    c = QuantizedKVCache(rows, tokens, G, hd, page=page, table=table, num_pages=rows * per + spare, device=device)
    c.codes.fill_(0xA5)
    c.scales.fill_(float("nan"))       # what was never written must not matter
    return c


# ----------------------------------------------------------------------------- write and read
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("hd", [32, 64])
@pytest.mark.parametrize("G,T,page", [(1, 1, 16), (3, 5, 16), (8, 64, 64), (2, 65, 32), (5, 203, 64), (4, 130, 256)])
def test_write_then_read(device, hd, G, T, page):
    n = 3
    k, v = _kv(n, T, G, hd, device)
    cache = _shuffled(n, T + 7, G, hd, page, device)
    kstart, start = [0, T // 2, T], [7, 0, 3]
    kv_cache_write(cache, k, v, start=_int(start, device), kstart=_int(kstart, device))
    assert cache.lengths.tolist() == [s + T - f for s, f in zip(start, kstart)]
    for dtype in (torch.float32, torch.bfloat16):
        rk, rv = kv_cache_read(cache, T + 2, start=_int(start, device), dtype=dtype)
        assert rk.shape == (n, T + 2, G * hd) and rk.dtype == dtype
        for got, x in ((rk, k), (rv, v)):
            want = torch.zeros(n, T + 2, G * hd, dtype=torch.float64, device=device)
            y = _round4(x.view(n, T, G, hd)).view(n, T, G * hd)
            for i, f in enumerate(kstart):
                want[i, :T - f] = y[i, f:]
            assert torch.equal(got.double(), want.to(dtype).double())
    _check_errors(device)


@pytest.mark.parametrize("device", DEVICES)
def test_every_bf16_pair_of_value_and_maximum_rounds_as_in_64_bits(device):
    """All quotients of two bf16 significands, ties among them, in one exponent range."""

    sig = torch.arange(128, 256, dtype=torch.float64)
    rows = []
    for top in sig.tolist():
        for e in (0, -1, -2, -3, -4):
            x = torch.cat([sig * 2.0 ** e, -sig * 2.0 ** e])
            x = torch.where(x.abs() <= top, x, torch.zeros_like(x))
            for part in x.view(-1, 32):
                p = part.clone()
                p[0] = top
                rows.append(p)
    x = torch.stack(rows).to(torch.bfloat16).to(device)
    T = x.shape[0]
    cache = QuantizedKVCache(1, T, 1, 32, device=device)
    kv_cache_write(cache, x.view(1, T, 32), -x.view(1, T, 32))
    k, v = kv_cache_read(cache, T, dtype=torch.float32)
    want = _round4(x)
    assert torch.equal(k[0].double(), want) and torch.equal(v[0].double(), -want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("hd", [32, 64])
def test_extreme_rows(device, hd):
    """Zeros, the smallest and largest bf16 numbers, infinities and NaN, each in its own row:
    none touches a neighbour."""

    tiny, huge = 2.0 ** -133, torch.finfo(torch.bfloat16).max
    base = torch.linspace(-1, 1, hd).bfloat16().float()
    rows = [torch.zeros(hd), base * 0 + tiny, base * huge, base, base.clone(), base.clone(), base.clone(), -base]
    rows[1][1:] = 0
    rows.append(torch.arange(hd).float() * tiny)
    rows.append(base * 2.0 ** -126)
    rows[4][3], rows[5][3], rows[6][hd - 1] = float("inf"), float("-inf"), float("nan")
    x = torch.stack(rows).bfloat16().to(device).view(1, len(rows), hd)
    cache = _shuffled(1, len(rows), 1, hd, 16, device)
    kv_cache_write(cache, x, x.flip(1))
    k, v = kv_cache_read(cache, len(rows), dtype=torch.float32)
    want = _round4(torch.nan_to_num(x[0].float(), nan=0.0, posinf=0.0, neginf=0.0).bfloat16())
    want[4:7] = float("nan")
    assert torch.equal(torch.isnan(k[0]), torch.isnan(want)) and torch.equal(torch.isnan(v[0]), torch.isnan(want.flip(0)))
    assert torch.equal(torch.nan_to_num(k[0].double()), torch.nan_to_num(want))
    assert torch.equal(torch.nan_to_num(v[0].double()), torch.nan_to_num(want.flip(0)))


@pytest.mark.parametrize("device", DEVICES)
def test_append_grows_rows_and_leaves_others(device):
    """Appends of one and of many tokens, to some rows, from strided views of a projection."""

    G, hd, n = 2, 32, 5
    W = G * hd
    cache = _shuffled(n, 300, G, hd, 32, device)
    held = [[torch.zeros(0, W, dtype=torch.float64)] for _ in range(n)]
    for step, (rows, T) in enumerate([([0, 1, 2, 3, 4], 1), ([3, 1], 90), ([4], 130), ([0, 1, 2, 3, 4], 1), ([2, 0], 3),
                                      ([1], 70), ([0, 1, 2, 3, 4], 0)]):
        g = torch.Generator().manual_seed(step)
        qkv = torch.randn(len(rows), T + 2, 4 * W, generator=g).bfloat16().to(device)
        k, v = qkv[:, 1:T + 1, W:2 * W], qkv[:, 1:T + 1, 3 * W:]
        kv_cache_write(cache, k, v, rows=_int(rows, device))
        for i, r in enumerate(rows):
            held[r].append(_round4(k[i].cpu().view(T, G, hd)).view(T, W))
    got = kv_cache_read(cache, 300, dtype=torch.float32)[0]
    for r in range(n):
        want = torch.cat(held[r])
        assert int(cache.lengths[r]) == want.shape[0]
        assert torch.equal(got[r, :want.shape[0]].cpu().double(), want)
        assert not got[r, want.shape[0]:].any()
    cache.reset(_int([1], device))
    assert cache.lengths.tolist()[1] == 0 and cache.lengths.tolist()[3] > 0
    cache.reset()
    assert not cache.lengths.any()
    _check_errors(device)


@pytest.mark.parametrize("device", DEVICES)
def test_start_may_be_the_lengths_themselves(device):
    k, v = _kv(3, 200, 1, 32, device)
    cache = QuantizedKVCache(3, 512, 1, 32, device=device)
    kv_cache_write(cache, k[:, :100], v[:, :100])
    kv_cache_write(cache, k[:, 100:], v[:, 100:], start=cache.lengths)
    assert cache.lengths.tolist() == [200] * 3
    got = kv_cache_read(cache, 200, dtype=torch.float32)[0]
    assert torch.equal(got.double(), _round4(k.view(3, 200, 1, 32)).view(3, 200, 32))


# ----------------------------------------------------------------------------- attention
def _exact(q, cache_k, cache_v, lengths, rows, kn, vn, window, sinks, G, hd, scale=None):
    """64-bit outputs and the sums ``sum_j p_j |v_j|``; ``cache_k [R, T, G*hd]`` are the values."""

    B, N, width = q.shape
    H = width // hd
    out = torch.zeros(B, N, H, hd, dtype=torch.float64)
    mag = torch.zeros_like(out)
    for b in range(B):
        r = b if rows is None else rows[b]
        ln = lengths[r]
        for h in range(H):
            g = h // (H // G)
            k = cache_k[r, :ln, g * hd:(g + 1) * hd].double()
            v = cache_v[r, :ln, g * hd:(g + 1) * hd].double()
            if kn is not None:
                k = torch.cat([k, kn[b, :, g * hd:(g + 1) * hd].double()])
                v = torch.cat([v, vn[b, :, g * hd:(g + 1) * hd].double()])
            for n in range(N):
                p = (ln if kn is not None else ln - N) + n
                js = [j for j in range(k.shape[0]) if j <= p and (window == 0 or p - j < window or j < sinks)]
                if not js:
                    continue
                s = (k[js] @ q[b, n, h * hd:(h + 1) * hd].double()) * (scale or hd ** -0.5)
                w = torch.softmax(s, 0)
                out[b, n, h] = w @ v[js]
                mag[b, n, h] = w @ v[js].abs()
    return out.view(B, N, width), mag.view(B, N, width)


def _attend_case(device, lengths, N, H, G, hd, window, sinks, fresh, rows=None, page=64, seed=0, scale=None, B=None):
    R, T = len(lengths), max(max(lengths), 1)
    B = B or (R if rows is None else len(rows))
    cache = _shuffled(R, T, G, hd, page, device)
    k, v = _kv(R, T, G, hd, device, seed)
    kv_cache_write(cache, k, v, start=_int([0] * R, device), kstart=_int([T - x for x in lengths], device))
    g = torch.Generator().manual_seed(seed + 9)
    qkv = torch.randn(B, N, (H + 2 * G) * hd, generator=g).bfloat16().to(device)
    q, kn, vn = qkv.split([H * hd, G * hd, G * hd], -1)
    if not fresh:
        kn = vn = None
    got = cached_attention(q, cache, rows=None if rows is None else _int(rows, device), k_new=kn, v_new=vn,
                           window=window, sinks=sinks, scale=scale)
    assert got.dtype == torch.bfloat16 and got.shape == q.shape
    vk = torch.zeros(R, T, G * hd, dtype=torch.float64)
    vv = torch.zeros_like(vk)
    for r, ln in enumerate(lengths):
        vk[r, :ln] = _round4(k[r, T - ln:].view(ln, G, hd)).view(ln, G * hd).cpu()
        vv[r, :ln] = _round4(v[r, T - ln:].view(ln, G, hd)).view(ln, G * hd).cpu()
    cpu = [None if x is None else x.cpu() for x in (q, kn, vn)]
    want, mag = _exact(cpu[0], vk, vv, lengths, rows, cpu[1], cpu[2], window, sinks, G, hd, scale)
    err = (got.cpu().double() - want).abs()
    assert torch.isfinite(got).all()
    assert (err <= 1.05 * 2.0 ** -7 * mag).all(), float((err / mag.clamp(min=1e-30)).max())
    ref = cached_attention_reference(q, cache, None if rows is None else _int(rows, device), kn, vn, window, sinks,
                                     scale)
    if device == "cpu":
        assert ((ref.double() - want).abs() <= 2.0 ** -16 * mag + 1e-12).all()
    _check_errors(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("hd", [32, 64])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (7, 2), (64, 4), (100, 70)])
def test_single_tokens(device, hd, window, sinks):
    """A token per row whose key is in the cache, over empty, one-token and page-crossing rows."""

    _attend_case(device, [0, 1, 2, 16, 63, 64, 65, 130, 201], 1, 4, 4, hd, window, sinks, False)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("hd", [32, 64])
@pytest.mark.parametrize("H,G,N", [(8, 2, 1), (6, 2, 3), (4, 1, 4), (3, 3, 9), (8, 1, 5), (2, 2, 40)])
def test_shared_heads_and_several_queries(device, hd, H, G, N):
    _attend_case(device, [3, 50, 0, 97], N, H, G, hd, 0, 0, False, page=16)
    _attend_case(device, [3, 50, 0, 97], N, H, G, hd, 20, 5, False, page=32)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("hd", [32, 64])
@pytest.mark.parametrize("N,window,sinks", [(1, 0, 0), (5, 3, 2), (16, 0, 0), (17, 24, 3), (32, 8, 1), (33, 100, 90)])
def test_candidates_with_fresh_keys(device, hd, N, window, sinks):
    """Candidates over their request's row, in any order, an empty request among them."""

    _attend_case(device, [70, 0, 5, 129], N, 4, 2, hd, window, sinks, True, rows=[3, 0, 0, 1, 2, 3, 1])


@pytest.mark.parametrize("device", DEVICES)
def test_scale_and_empty_batches(device):
    _attend_case(device, [40, 41], 2, 2, 2, 32, 0, 0, True, scale=0.5)
    cache = QuantizedKVCache(2, 16, 1, 32, device=device)
    k, v = _kv(2, 0, 1, 32, device)
    kv_cache_write(cache, k, v)
    assert cache.lengths.tolist() == [0, 0]
    assert kv_cache_read(cache, 0)[0].shape == (2, 0, 32)
    empty = torch.zeros(0, 3, 32, dtype=torch.bfloat16, device=device)
    assert cached_attention(empty, cache, rows=_int([], device)).shape == (0, 3, 32)
    one = torch.ones(2, 1, 32, dtype=torch.bfloat16, device=device)
    assert not cached_attention(one, cache).any()


@pytest.mark.parametrize("device", DEVICES)
def test_hidden_rows_that_hold_infinities_do_not_matter(device):
    """Non-finite rows out of the window, and stale pages past the length."""

    G, hd, T = 1, 64, 150
    k, v = _kv(1, T, G, hd, device)
    clean = _shuffled(1, T, G, hd, 16, device)
    dirty = _shuffled(1, T, G, hd, 16, device)
    kv_cache_write(clean, k, v)
    kd, vd = k.clone(), v.clone()
    kd[:, 2:90], vd[:, 2:90] = float("inf"), float("nan")
    kv_cache_write(dirty, kd, vd)
    q = torch.randn(1, 4, 2 * hd, generator=torch.Generator().manual_seed(5)).bfloat16().to(device)
    for c in (clean, dirty):
        c.lengths.fill_(T - 3)
    a = cached_attention(q, clean, window=50, sinks=2)
    b = cached_attention(q, dirty, window=50, sinks=2)
    assert torch.isfinite(a).all() and torch.equal(a, b)
    # a row that is seen does matter
    assert torch.isnan(cached_attention(q, dirty, window=70, sinks=2)).any()


@GPU
@pytest.mark.parametrize("hd,H,G,N,fresh,lengths,window", [
    (64, 8, 2, 1, False, [40000, 8191, 1], 0),        # split over blocks, joined afterwards
    (32, 2, 2, 1, False, [5000], 0),
    (32, 4, 4, 32, True, [3000, 100], 1000),
])
def test_long_rows(hd, H, G, N, fresh, lengths, window):
    """Rows that several blocks share, against the fp32 definition on the same cache (itself
    held to 2^-16 on the CPU); magnitudes from the same probabilities."""

    R, T = len(lengths), max(lengths)
    cache = _shuffled(R, T, G, hd, 64, "cuda")
    k, v = _kv(R, T, G, hd, "cuda", 4)
    kv_cache_write(cache, k, v, start=_int([0] * R, "cuda"), kstart=_int([T - x for x in lengths], "cuda"))
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(R, N, (H + 2 * G) * hd, generator=g).bfloat16().cuda()
    q, kn, vn = qkv.split([H * hd, G * hd, G * hd], -1)
    if not fresh:
        kn = vn = None
    got = cached_attention(q, cache, k_new=kn, v_new=vn, window=window, sinks=3)
    again = cached_attention(q, cache, k_new=kn, v_new=vn, window=window, sinks=3)
    assert torch.equal(got, again)
    ref = cached_attention_reference(q, cache, None, kn, vn, window, 3)
    pos = cache.codes.clone()
    # |v|: flip the negative codes of V
    c = torch.stack([pos[:, :, 1] & 15, pos[:, :, 1] >> 4], -1).int() - 8
    c = c.abs() + 8
    pos[:, :, 1] = (c[..., 0] | (c[..., 1] << 4)).to(torch.uint8)
    cache.codes.copy_(pos)
    mag = cached_attention_reference(q, cache, None, kn, None if vn is None else vn.abs(), window, 3)
    assert ((got.float() - ref).abs() <= 1.05 * 2.0 ** -7 * mag).all()
    _check_errors("cuda")


@GPU
def test_many_items_one_warp_each():
    """Enough candidates that each work item is one warp."""

    R, B, N, H, hd = 5, 700, 6, 4, 32
    lengths = [0, 17, 64, 200, 333]
    T = max(lengths)
    cache = _shuffled(R, T, H, hd, 64, "cuda")
    k, v = _kv(R, T, H, hd, "cuda", 2)
    kv_cache_write(cache, k, v, start=_int([0] * R, "cuda"), kstart=_int([T - x for x in lengths], "cuda"))
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(B, N, 3 * H * hd, generator=g).bfloat16().cuda()
    rows = torch.randint(0, R, (B,), generator=g).int().cuda()
    q, kn, vn = qkv.chunk(3, -1)
    got = cached_attention(q, cache, rows=rows, k_new=kn, v_new=vn, window=90, sinks=4)
    ref = cached_attention_reference(q, cache, rows, kn, vn, 90, 4)
    # |o| <= max |v| of what is seen: unit-normal values stay below 6
    assert (got.float() - ref).abs().max() <= 1.05 * 2.0 ** -7 * 6
    few = cached_attention(q[:9], cache, rows=rows[:9], k_new=kn[:9], v_new=vn[:9], window=90, sinks=4)
    assert (few.float() - ref[:9]).abs().max() <= 1.05 * 2.0 ** -7 * 6
    _check_errors("cuda")


@GPU
def test_on_another_stream():
    k, v = _kv(4, 500, 2, 64, "cuda")
    q = torch.randn(4, 1, 256, device="cuda").bfloat16()
    cache = QuantizedKVCache(4, 500, 2, 64, device="cuda")
    kv_cache_write(cache, k, v)
    want = cached_attention(q, cache)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = QuantizedKVCache(4, 500, 2, 64, device="cuda")
        kv_cache_write(other, k, v)
        got = cached_attention(q, other)
    side.synchronize()
    assert torch.equal(got, want)


# ----------------------------------------------------------------------------- refusals
@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    cache = QuantizedKVCache(2, 32, 2, 32, device=device)
    k, v = _kv(2, 4, 2, 32, device)
    q = torch.zeros(2, 1, 128, dtype=torch.bfloat16, device=device)
    for kw, exc in [(dict(rows=0), ValueError), (dict(head_dim=48), NotImplementedError), (dict(page=24), ValueError),
                    (dict(page=8), ValueError), (dict(num_pages=1), ValueError), (dict(num_pages=0), ValueError),
                    (dict(table=torch.zeros(2, 3, dtype=torch.int32)), ValueError),
                    (dict(table=torch.zeros(2, 1)), TypeError), (dict(max_tokens=2 ** 31), ValueError)]:
        args = dict(rows=2, max_tokens=32, kv_heads=2, head_dim=32)
        args.update(kw)
        with pytest.raises(exc):
            QuantizedKVCache(**args, device=device)
    bad = [lambda: kv_cache_write(cache, k[:1], v[:1]), lambda: kv_cache_write(cache, k, v[:, :3]),
           lambda: kv_cache_write(cache, k[..., :32], v[..., :32]),
           lambda: kv_cache_write(cache, k, v, start=_int([0], device)),
           lambda: kv_cache_read(cache, -1), lambda: cached_attention(q[..., :96], cache),
           lambda: cached_attention(q[:1], cache), lambda: cached_attention(q, cache, window=-1),
           lambda: cached_attention(q, cache, sinks=-1), lambda: cached_attention(q, cache, k_new=k[:, :1]),
           lambda: cached_attention(q, cache, k_new=k, v_new=v)]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        kv_cache_read(cache, 1, dtype=torch.float16)
    with pytest.raises(TypeError):
        kv_cache_write(cache, k, v, start=torch.zeros(2, device=device))
    with pytest.raises(RuntimeError):
        cached_attention(q.float().requires_grad_().bfloat16(), cache)
    if device == "cuda":
        with pytest.raises(TypeError):
            kv_cache_write(cache, k.float(), v.float())
        with pytest.raises(ValueError):
            kv_cache_write(cache, k.cpu(), v.cpu())
    assert not cache.lengths.any()


@pytest.mark.parametrize("device", DEVICES)
def test_writes_past_the_end_and_bad_rows(device):
    """On CUDA these are known only on the device: nothing outside the cache is touched, the
    error word says so; the CPU definition raises."""

    cache = QuantizedKVCache(3, 32, 1, 32, page=16, device=device)
    k, v = _kv(1, 20, 1, 32, device)
    kv_cache_write(cache, k, v, rows=_int([1], device))
    before = kv_cache_read(cache, 32, dtype=torch.float32)[0].clone()

    def full():
        kv_cache_write(cache, k, v, rows=_int([1], device))

    def outside():
        kv_cache_write(cache, k, v, rows=_int([7], device))

    def page():
        cache.table[2] = _int([99, -1], device)
        kv_cache_write(cache, k, v, rows=_int([2], device))

    for call, code in ((full, "overflow"), (outside, "outside"), (page, "outside")):
        if device == "cpu":
            with pytest.raises((ValueError, IndexError)):
                call()
            continue
        from mdl_b200.ops._ext import check_error_word

        call()
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match=code):
            check_error_word(torch.device("cuda", 0))
        if code == "overflow":
            assert cache.lengths.tolist() == [0, 32, 0]
    if device == "cuda":
        after = kv_cache_read(cache, 32, dtype=torch.float32)[0]
        torch.cuda.synchronize()
        from mdl_b200.ops._ext import error_word

        error_word(torch.device("cuda", 0)).zero_()
        assert torch.equal(after[1, :20], before[1, :20]) and not after[0].any()


def test_quantize_rows_definition():
    x = torch.tensor([[7.0, 0.5, -0.5, 1.5, 2.5, -7.0, 0.0, 3.49], [0.0] * 8])
    c, s = quantize_rows(x)
    assert s.tolist() == [1.0, 0.0]
    assert c.tolist() == [[7, 0, 0, 2, 2, -7, 0, 3], [0] * 8]
    assert math.isnan(float(quantize_rows(torch.tensor([[1.0, float("inf")]]))[1]))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("scale", [0.0, -0.25, math.inf, math.nan])
def test_scale_is_positive(device, scale):
    cache = QuantizedKVCache(2, 16, 2, 32, device=device)
    q = torch.zeros(2, 1, 64, dtype=torch.bfloat16, device=device)
    with pytest.raises(ValueError, match="scale"):
        cached_attention(q, cache, scale=scale)


@GPU
def test_split_calls_that_follow_one_another():
    """The join of a row's parts starts while they are computed: calls in a row on one stream, and
    captured ones, give what single calls give."""

    G, hd, T, H = 2, 64, 30000, 8
    cache = _shuffled(1, T, G, hd, 64, "cuda")
    k, v = _kv(1, T, G, hd, "cuda", 7)
    kv_cache_write(cache, k, v)
    g = torch.Generator().manual_seed(2)
    qs = [torch.randn(1, 1, H * hd, generator=g).bfloat16().cuda() for _ in range(8)]
    single = []
    for q in qs:
        single.append(cached_attention(q, cache))
        torch.cuda.synchronize()
    row = [cached_attention(q, cache) for q in qs]
    for a, b in zip(single, row):
        assert torch.equal(a, b)
    inputs = [torch.zeros_like(qs[0]) for _ in range(2)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [cached_attention(q, cache) for q in inputs]
    for i in range(0, 8, 2):
        for t, q in zip(inputs, qs[i:i + 2]):
            t.copy_(q)
        graph.replay()
        assert torch.equal(outs[0], single[i]) and torch.equal(outs[1], single[i + 1])
    _check_errors("cuda")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("hd", [32, 64])
@pytest.mark.parametrize("H,G", [(2, 2), (2, 1)])
@pytest.mark.parametrize("N,window,sinks", [(40, 1, 4), (64, 1, 4), (64, 8, 4), (96, 8, 4), (100, 32, 70), (128, 48, 4)])
def test_candidates_whose_window_has_left_the_cache(device, hd, H, G, N, window, sinks):
    """More fresh tokens than the window: the later queries see the sinks alone of the cache."""

    _attend_case(device, [31, 32, 64, 96, 100, 128, 3], N, H, G, hd, window, sinks, True, rows=[2, 0, 1, 3, 6, 5, 4])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("N,window,sinks", [(40, 1, 4), (100, 32, 4), (128, 48, 4)])
def test_candidates_far_past_long_rows(device, N, window, sinks):
    for hd in (32, 64):
        _attend_case(device, [1920, 1984, 2000], N, 1, 1, hd, window, sinks, True)


@GPU
def test_many_candidates_whose_window_has_left_the_cache():
    """The same with one warp an item: as many candidates as fill the device."""

    lengths, N, H, hd = [32, 64, 100, 333], 40, 4, 32
    R, B, T = len(lengths), 700, max(lengths)
    cache = _shuffled(R, T, H, hd, 64, "cuda")
    k, v = _kv(R, T, H, hd, "cuda", 2)
    kv_cache_write(cache, k, v, start=_int([0] * R, "cuda"), kstart=_int([T - x for x in lengths], "cuda"))
    g = torch.Generator().manual_seed(1)
    q, kn, vn = torch.randn(B, N, 3 * H * hd, generator=g).bfloat16().cuda().chunk(3, -1)
    rows = torch.randint(0, R, (B,), generator=g).int().cuda()
    got = cached_attention(q, cache, rows=rows, k_new=kn, v_new=vn, window=1, sinks=4)
    ref = cached_attention_reference(q, cache, rows, kn, vn, 1, 4)
    # |o| <= max |v| of what is seen: unit-normal values stay below 6
    assert (got.float() - ref).abs().max() <= 1.05 * 2.0 ** -7 * 6
    _check_errors("cuda")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("hd,G,page,N", [(32, 2, 64, 1), (64, 1, 64, 1), (32, 1, 16, 20), (64, 2, 32, 3), (32, 2, 256, 33)])
def test_keys_of_a_page_outside_the_cache_are_hidden(device, hd, G, page, N):
    """A table entry outside the pool hides its tokens, whatever page 0 holds: as if the row ended
    before the page (its last one), or with the tokens of that page out of the sum (one in the
    middle); the error word says so. The CPU definition raises."""

    T, R = 5 * page, 3
    k, v = _kv(R, T, G, hd, device, 6)
    q = torch.randn(R, N, 2 * G * hd, generator=torch.Generator().manual_seed(3)).bfloat16().to(device)
    kn, vn = _kv(R, N, G, hd, device, 8)
    for bad, at in ((-1, 4), (10 ** 6, 2)):
        table = torch.arange(R * 5, dtype=torch.int32).view(R, 5).flip(0).contiguous()
        cache = QuantizedKVCache(R, T, G, hd, page=page, table=table, num_pages=R * 5, device=device)
        kv_cache_write(cache, k, v)
        row, pg = 1, int(cache.table[1, at])
        want = cached_attention(q, cache, k_new=kn, v_new=vn)
        if device == "cpu":
            cache.table[row, at] = bad
            with pytest.raises(ValueError, match="page"):
                cached_attention(q, cache, k_new=kn, v_new=vn)
            continue
        # what the row gives without the page: the other tokens moved together, no window, so that
        # positions do not matter
        short = QuantizedKVCache(1, 4 * page, G, hd, page=page, device=device)
        keep = [i for i in range(T) if i // page != at]
        kv_cache_write(short, k[row:row + 1, keep], v[row:row + 1, keep])
        want[row] = cached_attention(q[row:row + 1], short, k_new=kn[row:row + 1], v_new=vn[row:row + 1])[0]
        cache.table[row, at] = bad
        # NaN in page 0 and in the page that is gone would show
        zero = int((cache.table == 0).nonzero()[0, 0])
        got = cached_attention(q, cache, k_new=kn, v_new=vn)
        torch.cuda.synchronize()
        from mdl_b200.ops._ext import check_error_word

        with pytest.raises(RuntimeError, match="outside"):
            check_error_word(torch.device("cuda", 0))
        # another order of the same sums: the roundings of P and of the result (2^-8 each) on both
        # sides; |o| <= max |v| < 6
        assert (got.float() - want.float()).abs().max() <= 2 * 1.05 * 2.0 ** -7 * 6
        cache.scales[0] = float("nan")
        again = cached_attention(q, cache, k_new=kn, v_new=vn)
        others = [r for r in range(R) if r != zero]
        assert torch.equal(again[others], got[others]) and torch.isnan(again[zero]).any()
        rk, _ = kv_cache_read(cache, T, dtype=torch.float32)
        assert not rk[row, at * page:(at + 1) * page].any()
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="outside"):
            check_error_word(torch.device("cuda", 0))


@GPU
@pytest.mark.parametrize("hd,H,N", [(32, 4, 1), (32, 2, 12), (64, 2, 1), (64, 4, 20)])
def test_hidden_pages_with_one_warp_an_item(hd, H, N):
    """The same where candidates fill the device: they give what a few of them give (another order
    of the same sums: the roundings of P and of the result, on both sides)."""

    R, T, B = 4, 333, 1200
    cache = QuantizedKVCache(R, T, H, hd, device="cuda")
    k, v = _kv(R, T, H, hd, "cuda", 2)
    kv_cache_write(cache, k, v)
    cache.table[1, 2], cache.table[3, 5] = -5, 10 ** 6
    cache.scales[0] = float("nan")       # page 0 belongs to row 0
    g = torch.Generator().manual_seed(1)
    q, kn, vn = torch.randn(B, N, 3 * H * hd, generator=g).bfloat16().cuda().chunk(3, -1)
    rows = (torch.arange(B, device="cuda") % 3 + 1).int()
    got = cached_attention(q, cache, rows=rows, k_new=kn, v_new=vn, window=300, sinks=4)
    few = cached_attention(q[:6], cache, rows=rows[:6], k_new=kn[:6], v_new=vn[:6], window=300, sinks=4)
    assert torch.isfinite(got).all() and torch.isfinite(few).all()
    assert (got[:6].float() - few.float()).abs().max() <= 2 * 1.05 * 2.0 ** -7 * 6
    torch.cuda.synchronize()
    from mdl_b200.ops._ext import check_error_word

    with pytest.raises(RuntimeError, match="outside"):
        check_error_word(torch.device("cuda", 0))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("T", [2, 2 ** 20 + 70])
def test_write_at_the_end_of_a_row_of_two_billion_positions(device, T):
    """Positions past the capacity that 32 bits cannot hold are past the capacity too."""

    page = 2 ** 20
    per = 2 ** 31 // page - 1
    table = torch.zeros(1, per, dtype=torch.int32)
    cache = QuantizedKVCache(1, per * page, 1, 32, page=page, table=table, num_pages=1, device=device)
    k, v = _kv(1, 1, 1, 32, device)
    k, v = k.expand(1, T, 32), v.expand(1, T, 32)
    start = _int([cache.capacity - 1], device)
    if device == "cpu":
        with pytest.raises(ValueError, match="full"):
            kv_cache_write(cache, k, v, start=start)
        return
    kv_cache_write(cache, k, v, start=start)
    torch.cuda.synchronize()
    from mdl_b200.ops._ext import check_error_word

    with pytest.raises(RuntimeError, match="overflow"):
        check_error_word(torch.device("cuda", 0))
    assert cache.lengths.tolist() == [cache.capacity]
    got, _ = kv_cache_read(cache, 1, start=start, dtype=torch.float32)
    assert torch.equal(got[0, 0].double(), _round4(k[0, :1])[0])
    _check_errors(device)


@pytest.mark.parametrize("device", DEVICES)
def test_negative_rows_are_outside(device):
    """Row -1 is no row, not the last one."""

    cache = QuantizedKVCache(2, 32, 1, 32, device=device)
    k, v = _kv(2, 4, 1, 32, device)
    kv_cache_write(cache, k, v)
    q = torch.ones(1, 1, 32, dtype=torch.bfloat16, device=device)
    for call in (lambda: kv_cache_write(cache, k[:1], v[:1], rows=_int([-1], device)),
                 lambda: kv_cache_read(cache, 4, rows=_int([-1], device)),
                 lambda: cached_attention(q, cache, rows=_int([-1], device))):
        if device == "cpu":
            with pytest.raises(IndexError):
                call()
        else:
            from mdl_b200.ops._ext import check_error_word

            out = call()
            torch.cuda.synchronize()
            with pytest.raises(RuntimeError, match="outside"):
                check_error_word(torch.device("cuda", 0))
            if out is not None:
                assert not any(x.any() for x in (out if isinstance(out, tuple) else (out,)))
        assert cache.lengths.tolist() == [4, 4]


@pytest.mark.parametrize("device", DEVICES)
def test_indexes_past_32_bits_do_not_wrap(device):
    """64-bit rows, starts and pages that 32 bits would turn into valid ones are outside."""

    big = 2 ** 32
    cache = QuantizedKVCache(2, 32, 1, 32, page=16, device=device)
    k, v = _kv(2, 4, 1, 32, device)
    kv_cache_write(cache, k, v)
    held = kv_cache_read(cache, 32, dtype=torch.float32)[0].clone()
    wide = lambda *x: torch.tensor(x, dtype=torch.int64, device=device)
    q = torch.ones(1, 1, 32, dtype=torch.bfloat16, device=device)
    calls = [lambda: kv_cache_write(cache, k[:1], v[:1], rows=wide(big + 1)),
             lambda: kv_cache_write(cache, k, v, start=wide(big, big + 2)),
             lambda: kv_cache_write(cache, k[:1], v[:1], rows=wide(-big)),
             lambda: kv_cache_read(cache, 4, rows=wide(big)),
             lambda: kv_cache_read(cache, 4, start=wide(-big, -big)),
             lambda: cached_attention(q, cache, rows=wide(big + 1))]
    for call in calls:
        if device == "cpu":
            with pytest.raises((ValueError, IndexError)):
                call()
        else:
            from mdl_b200.ops._ext import check_error_word

            out = call()
            torch.cuda.synchronize()
            with pytest.raises(RuntimeError, match="outside"):
                check_error_word(torch.device("cuda", 0))
            if out is not None:
                assert not any(x.any() for x in (out if isinstance(out, tuple) else (out,)))
        assert cache.lengths.tolist() == [4, 4]
        assert torch.equal(kv_cache_read(cache, 32, dtype=torch.float32)[0], held)
    # padding past the last token is all of it, before the first is none
    kv_cache_write(cache, k, v, start=wide(0, 0), kstart=wide(big, -big))
    assert cache.lengths.tolist() == [0, 4]
    paged = QuantizedKVCache(1, 32, 1, 32, page=16, table=torch.tensor([[big, big + 1]]), num_pages=2, device=device)
    if device == "cpu":
        with pytest.raises(ValueError, match="page"):
            kv_cache_write(paged, k[:1], v[:1])
    else:
        kv_cache_write(paged, k[:1], v[:1])
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="outside"):
            check_error_word(torch.device("cuda", 0))


@pytest.mark.parametrize("device", DEVICES)
def test_reset_of_rows_outside_the_cache(device):
    """On CUDA they are skipped and recorded, on the CPU refused; no valid row is emptied for them."""

    cache = QuantizedKVCache(4, 32, 1, 32, device=device)
    k, v = _kv(4, 3, 1, 32, device)
    kv_cache_write(cache, k, v)
    for rows in ([4], [-1], [1, 2 ** 40]):
        rows = torch.tensor(rows, device=device)
        if device == "cpu":
            with pytest.raises(IndexError):
                cache.reset(rows)
            assert cache.lengths.tolist() == [3, 3, 3, 3]
            continue
        from mdl_b200.ops._ext import check_error_word

        cache.reset(rows)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="outside"):
            check_error_word(torch.device("cuda", 0))
        assert cache.lengths.tolist() == [3, 3 if len(rows) == 1 else 0, 3, 3]
    cache.reset(torch.tensor([[3, 0], [3, 3]], dtype=torch.int16))     # any shape, from the host too
    assert cache.lengths.tolist()[0] == 0 and cache.lengths.tolist()[3] == 0
    cache.reset(torch.tensor([], dtype=torch.int64, device=device))
    assert cache.lengths.tolist()[2] == 3
    with pytest.raises(TypeError):
        cache.reset(torch.tensor([True, False, True, False], device=device))
    _check_errors(device)


@pytest.mark.parametrize("device", DEVICES)
def test_indexes_may_lie_in_the_lengths_memory(device):
    """kstart read from the lengths that the write replaces, rows in another order."""

    R, T = 4096, 6
    cache = QuantizedKVCache(R, 16, 1, 32, page=16, device=device)
    first = torch.arange(R, dtype=torch.int32) % 5
    cache.lengths.copy_(first)
    k, v = _kv(R, T, 1, 32, device)
    rows = torch.arange(R - 1, -1, -1, dtype=torch.int32, device=device)
    kv_cache_write(cache, k, v, start=torch.zeros(R, dtype=torch.int32, device=device), kstart=cache.lengths, rows=rows)
    assert torch.equal(cache.lengths.cpu(), (T - first).flip(0))
    _check_errors(device)


@pytest.mark.parametrize("device", DEVICES)
def test_an_empty_cache(device):
    """Rows of no positions: nothing is held, candidates see their own tokens alone."""

    cache = QuantizedKVCache(2, 0, 1, 32, device=device)
    assert cache.capacity == 0 and cache.nbytes == 0
    k, v = _kv(2, 3, 1, 32, device)
    kv_cache_write(cache, k[:, :0], v[:, :0])
    rk, rv = kv_cache_read(cache, 2)
    assert rk.shape == (2, 2, 32) and not rk.any() and not rv.any()
    assert not cached_attention(k, cache).any()
    other = QuantizedKVCache(2, 5, 1, 32, device=device)
    assert torch.equal(cached_attention(k, cache, k_new=k, v_new=v), cached_attention(k, other, k_new=k, v_new=v))
    _check_errors(device)
    if device == "cpu":
        with pytest.raises(ValueError, match="full"):
            kv_cache_write(cache, k, v)
    else:
        from mdl_b200.ops._ext import check_error_word

        kv_cache_write(cache, k, v)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="overflow"):
            check_error_word(torch.device("cuda", 0))
    with pytest.raises(ValueError):
        QuantizedKVCache(2, -1, 1, 32, device=device)


@GPU
@pytest.mark.parametrize("hd,H,G,B,N,lengths,fresh", [
    (64, 10, 5, 4, 142, [405, 0, 273, 405], False), (64, 1, 1, 600, 10, [47, 0, 47, 20], True),
    (64, 15, 5, 5, 133, [2645, 0, 472, 90], True), (64, 8, 8, 40, 16, [700, 1], True),
    (32, 4, 4, 30, 32, [900, 64], True), (32, 8, 2, 60, 4, [1500, 33], False),
])
def test_repeated_calls_of_more_blocks_than_the_device_holds(hd, H, G, B, N, lengths, fresh):
    """Blocks that follow one another on a multiprocessor join their warps in shared memory: every
    call gives the same, near the fp32 definition."""

    R, T = len(lengths), max(lengths)
    cache = _shuffled(R, T, G, hd, 256, "cuda")
    k, v = _kv(R, T, G, hd, "cuda", 11)
    kv_cache_write(cache, k, v, start=_int([0] * R, "cuda"), kstart=_int([T - x for x in lengths], "cuda"))
    g = torch.Generator().manual_seed(12)
    q, kn, vn = torch.randn(B, N, (H + 2 * G) * hd, generator=g).bfloat16().cuda().split([H * hd, G * hd, G * hd], -1)
    rows = torch.randint(0, R, (B,), generator=g).int().cuda()
    if not fresh:
        kn = vn = None
    outs = [cached_attention(q, cache, rows=rows, k_new=kn, v_new=vn) for _ in range(60)]
    ref = cached_attention_reference(q, cache, rows, kn, vn)
    # |o| <= max |v| of what is seen: unit-normal values stay below 6
    assert (outs[0].float() - ref).abs().max() <= 1.05 * 2.0 ** -7 * 6
    for o in outs[1:]:
        assert torch.equal(o, outs[0])
    _check_errors("cuda")


@GPU
@pytest.mark.parametrize("hd,G,page", [(32, 8, 64), (64, 1, 256)])
def test_offsets_past_32_bits(hd, G, page):
    """Rows whose pages lie at both ends of a pool of more than 2^32 bytes of codes, and an output of
    more than 2^31 elements."""

    per, T = 5, 5 * page - 3
    num = 2 ** 32 // (G * page * hd) + 2 * per
    table = torch.stack([torch.arange(per), torch.arange(num - per, num), torch.arange(num - 2 * per, num - per)]).int()
    big = QuantizedKVCache(3, T, G, hd, page=page, table=table, num_pages=num, device="cuda")
    assert big.codes.numel() > 2 ** 32
    small = QuantizedKVCache(3, T, G, hd, page=page, device="cuda")
    k, v = _kv(3, T, G, hd, "cuda", 3)
    q = torch.randn(3, 2, 2 * G * hd, generator=torch.Generator().manual_seed(4)).bfloat16().cuda()
    for c in (big, small):
        kv_cache_write(c, k, v)
    assert torch.equal(big.lengths, small.lengths)
    for a, b in zip(kv_cache_read(big, T), kv_cache_read(small, T)):
        assert torch.equal(a, b)
    for window, sinks in ((0, 0), (50, 3)):
        assert torch.equal(cached_attention(q, big, window=window, sinks=sinks),
                           cached_attention(q, small, window=window, sinks=sinks))
    del big
    n = 2 ** 31 // (T * G * hd) + 2
    rows = torch.zeros(n, dtype=torch.int32, device="cuda")
    rows[-1] = 2
    rk, rv = kv_cache_read(small, T, rows=rows)
    assert rk.numel() > 2 ** 31
    for got, want in ((rk, kv_cache_read(small, T)[0]), (rv, kv_cache_read(small, T)[1])):
        assert torch.equal(got[-1], want[2]) and torch.equal(got[-2], want[0])
    _check_errors("cuda")


@GPU
def test_sources_and_queries_past_32_bits():
    """Tokens, queries and outputs of more than 2^31 elements."""

    G, hd, R = 2, 32, 6
    T = 2 ** 31 // (R * G * hd) // 8 + 9
    wide = torch.zeros(R, T, 8, G * hd, dtype=torch.bfloat16, device="cuda")
    assert wide.numel() > 2 ** 31
    k, v = wide[:, :, 7], wide[:, :, 0]       # token strides of 8 rows
    g = torch.Generator(device="cuda").manual_seed(1)
    k[:, -300:].normal_(generator=g)
    v[:, -300:].normal_(generator=g)
    cache = QuantizedKVCache(R, 300, G, hd, device="cuda")
    kv_cache_write(cache, k, v, kstart=_int([T - 300] * R, "cuda"))
    got, _ = kv_cache_read(cache, 300, dtype=torch.float32)
    want = _round4(k[:, -300:].reshape(R, 300, G, hd)).view(R, 300, G * hd)
    assert torch.equal(got.double(), want)
    del wide, k, v
    B, N, H = 2 ** 31 // (64 * 16 * hd) + 3, 64, 16
    q = torch.zeros(B, N, H * hd, dtype=torch.bfloat16, device="cuda")
    assert q.numel() > 2 ** 31
    q[-2:].normal_(generator=g)
    rows = (torch.arange(B, device="cuda") % R).int()
    out = cached_attention(q, cache, rows=rows)
    few = cached_attention(q[-2:], cache, rows=rows[-2:])
    # another order of the same sums (see above); |v| < 6
    assert (out[-2:].float() - few.float()).abs().max() <= 2 * 1.05 * 2.0 ** -7 * 6
    _check_errors("cuda")
