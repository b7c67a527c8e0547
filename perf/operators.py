"""Cases of the windowed attention and of the 4-bit key/value cache, with plain forms.

Four operators of long event histories:

* ``windowed_attention`` (training and prompts): a query sees the last ``window`` tokens up
  to itself and the first ``sinks`` valid tokens of its sample;
* ``kv_cache_write`` / ``kv_cache_read``: keys and values quantised to 4 bits as they are
  written to a paged cache, and read back;
* ``cached_attention``: single tokens, or candidates with a few fresh tokens of their own,
  over that cache.

``run`` computes a case with elementary torch operations in 32 bits (``own`` false) or through
the framework's entry points (``own`` true); ``exact`` computes it in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

PAGE = 64


# ----------------------------------------------------------------------------- cases
def listed() -> list[dict]:
    return [
        # One sample just over a hundred events: the smallest training step, where launches count.
        _train("train_one_sample", B=1, L=130, lq=130, H=8, G=8, hd=32, window=48, sinks=2),
        # The OneTrans workload's first layer (512 events + 32 other tokens, 8 heads of 32, 1024 samples).
        _train("train_onetrans", B=1024, L=544, lq=544, H=8, G=8, hd=32, window=128, sinks=4),
        # A late layer of a pyramid: a query suffix, odd sizes, query heads that share keys and values.
        _train("train_suffix_shared", B=37, L=1237, lq=401, H=6, G=2, hd=64, window=101, sinks=5),
        # A few very long histories (256 wide over 4 heads), where single samples have to fill the device.
        _train("train_long", B=2, L=8191, lq=8191, H=4, G=4, hd=64, window=1024, sinks=16),
        # Histories of the LONGER workload's length, forward only, as before a cache is written.
        _prompt("prompt_histories", B=64, L=2000, lq=2000, H=8, G=8, hd=32, window=256, sinks=8),
        # One new event per user, quantised at the end of each user's history.
        _store("store_one_event", R=512, T=1, G=8, hd=32, used=1900),
        # Histories of a request batch written whole, left-padded as the model lays them out.
        _store("store_histories", R=256, T=2000, G=8, hd=32, used=0),
        # A few rows read back, odd length.
        _read("read_few", R=3, T=777, G=4, hd=64),
        # A whole cache read back (to rebuild another layer's state).
        _read("read_cache", R=384, T=2048, G=8, hd=32),
        # One user's next event: latency of the smallest call.
        _attend("event_one_user", B=1, N=1, R=1, T=501, H=8, G=8, hd=32, window=0, sinks=0, fresh=False),
        # A serving batch over very long histories with shared key heads: the cache is read once.
        _attend("event_long", B=24, N=1, R=24, T=131071, H=8, G=2, hd=64, window=0, sinks=0, fresh=False),
        # Candidates of a few requests, 32 own tokens each, over their request's history (window and sinks).
        _attend("candidates", B=1024, N=32, R=12, T=2000, H=8, G=8, hd=32, window=512, sinks=4, fresh=True),
    ]


def _train(name, **kw):
    return {"name": name, "kind": "train", **kw}


def _prompt(name, **kw):
    return {"name": name, "kind": "prompt", **kw}


def _store(name, **kw):
    return {"name": name, "kind": "store", **kw}


def _read(name, **kw):
    return {"name": name, "kind": "read", **kw}


def _attend(name, **kw):
    return {"name": name, "kind": "attend", **kw}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    G = rng.choice([1, 2, 3, 4, 6, 8])
    H = G * rng.choice([1, 1, 1, 2, 4])
    return (H, G) if H <= 16 else (G, G)


def draw(rng) -> dict:
    kind = rng.choice(["train", "train", "prompt", "store", "read", "attend", "attend", "attend"])
    while True:
        H, G = _heads(rng)
        hd = rng.choice([32, 64])
        window, sinks = _log(rng, 1, 2048), rng.choice([0, 1, 2, 4, 7, 16, 64])
        if kind in ("train", "prompt"):
            L = _log(rng, 20, 8191)
            c = {"kind": kind, "B": _log(rng, 1, 512), "L": L, "lq": L if rng.random() < 0.5 else _log(rng, 1, L),
                 "H": H, "G": G, "hd": hd, "window": window, "sinks": sinks}
            # scores of the plain form, and elements of the inputs
            if c["B"] * H * c["lq"] * L <= 5e8 and c["B"] * L * (H + 2 * G) * hd <= 2.5e8:
                return c
        elif kind in ("store", "read"):
            c = {"kind": kind, "R": _log(rng, 1, 1024), "T": _log(rng, 1, 4096), "G": G, "hd": hd}
            if kind == "store":
                c["used"] = rng.choice([0, _log(rng, 1, 2000)])
            if c["R"] * (c["T"] + c.get("used", 0)) * G * hd <= 1.3e8:
                return c
        else:
            fresh = rng.random() < 0.5
            R = _log(rng, 1, 256)
            N = _log(rng, 1, 40) if fresh else rng.choice([1, 1, 1, 2, 5])
            c = {"kind": kind, "R": R, "B": _log(rng, R, 4 * R + 64) if fresh else R, "N": N,
                 "T": _log(rng, 1, 131071), "H": H, "G": G, "hd": hd,
                 "window": rng.choice([0, window]), "sinks": sinks, "fresh": fresh}
            if R * c["T"] * G * hd <= 2.0e8 and c["B"] * N * c["T"] * H <= 4e8 and c["B"] * c["T"] * G * hd <= 4e8:
                return c


# ----------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ragged(n, lo, hi, g):
    """``n`` whole numbers of ``lo .. hi``."""

    u = torch.rand(n, device="cuda", generator=g)
    return (lo + (u * (hi - lo + 1)).floor().long()).clamp(lo, hi)


def _projected(shape, g, heads, hd):
    """Projections of normalised tokens: unit normal, a few strong channels a head."""

    x = torch.randn(*shape, heads, hd, device="cuda", generator=g)
    gain = 1.0 + 2.0 * (torch.rand(heads, hd, device="cuda", generator=g) > 0.94)
    return x * gain


def _tokens(case, seed):
    """``qkv [B, L, (H + 2 G) hd]`` bf16, first valid token of each sample, output gradient."""

    g = _gen(seed)
    B, L, lq, H, G, hd = (case[k] for k in ("B", "L", "lq", "H", "G", "hd"))
    q = _projected((B, L), g, H, hd).bfloat16()
    k = _projected((B, L), g, G, hd).bfloat16()
    v = torch.randn(B, L, G, hd, device="cuda", generator=g).bfloat16()
    qkv = torch.cat([q, k, v], dim=2).view(B, L, (H + 2 * G) * hd)
    kstart = _ragged(B, 0, L // 2, g).int()
    dout = torch.randn(B, lq, H * hd, device="cuda", generator=g).bfloat16()
    return qkv, kstart, dout


def _kv(R, T, G, hd, g):
    k = _projected((R, T), g, G, hd).bfloat16().view(R, T, G * hd)
    v = torch.randn(R, T, G * hd, device="cuda", generator=g).bfloat16()
    return k, v


def _store_inputs(case, seed):
    g = _gen(seed)
    R, T, G, hd, used = (case[k] for k in ("R", "T", "G", "hd", "used"))
    k, v = _kv(R, T, G, hd, g)
    start = _ragged(R, 0, used, g).int()
    # whole histories come left-padded; a single event is always valid
    kstart = _ragged(R, 0, T // 2, g).int()
    return k, v, start, kstart


def _read_inputs(case, seed):
    g = _gen(seed)
    R, T, G, hd = (case[k] for k in ("R", "T", "G", "hd"))
    k, v = _kv(R, T, G, hd, g)
    return k, v, _ragged(R, 0, T // 3, g).int()      # kstart: T - kstart tokens are cached


def _attend_inputs(case, seed):
    g = _gen(seed)
    B, N, R, T, H, G, hd = (case[k] for k in ("B", "N", "R", "T", "H", "G", "hd"))
    k, v = _kv(R, T, G, hd, g)
    kstart = _ragged(R, 0, T // 4, g).int()
    q = _projected((B, N), g, H, hd).bfloat16()
    kn = _projected((B, N), g, G, hd).bfloat16()
    vn = torch.randn(B, N, G, hd, device="cuda", generator=g).bfloat16()
    qkv = torch.cat([q, kn, vn], dim=2).view(B, N, (H + 2 * G) * hd)
    rows = None
    if case["fresh"]:      # candidates in the order of their requests, a varying number each
        rows = torch.sort(_ragged(B, 0, R - 1, g)).values.int()
    return k, v, kstart, qkv, rows


def _own_cache(R, T, G, hd, seed):
    """An empty framework cache whose pages lie in no particular order."""

    from mdl_b200.ops.kv_cache import QuantizedKVCache

    per = -(-T // PAGE)
    perm = torch.randperm(R * per, device="cuda", generator=_gen(seed + 1)).int().view(R, per)
    return QuantizedKVCache(R, T, G, hd, page=PAGE, table=perm, num_pages=R * per, device="cuda")


def _plain_cache(R, T, G, hd):
    return {"codes": torch.zeros(R, T, 2, G, hd // 2, dtype=torch.uint8, device="cuda"),
            "scales": torch.zeros(R, T, 2, G, dtype=torch.bfloat16, device="cuda"),
            "lengths": torch.zeros(R, dtype=torch.int32, device="cuda")}


def prepare(case: dict, seed: int) -> dict:
    kind = case["kind"]
    st = {"case": case}
    if kind in ("train", "prompt"):
        qkv, kstart, dout = _tokens(case, seed)
        st.update(qkv=qkv.requires_grad_(kind == "train"), kstart=kstart)
        if kind == "train":
            st["dout"] = dout
        return st
    R, T, G, hd = (case[k] for k in ("R", "T", "G", "hd"))
    if kind == "store":
        k, v, start, kstart = _store_inputs(case, seed)
        st.update(k=k, v=v, start=start, kstart=kstart)
        T = T + case["used"]
        st["cache"] = _own_cache(R, T, G, hd, seed) if own else _plain_cache(R, T, G, hd)
        return st
    if kind == "read":
        k, v, kstart = _read_inputs(case, seed)
    else:
        k, v, kstart, qkv, rows = _attend_inputs(case, seed)
        st.update(qkv=qkv, rows=rows)
    zero = torch.zeros(R, dtype=torch.int32, device="cuda")
    if own:
        from mdl_b200.ops.kv_cache import kv_cache_write

        st["cache"] = _own_cache(R, T, G, hd, seed)
        kv_cache_write(st["cache"], k, v, start=zero, kstart=kstart)
    else:
        st["cache"] = _plain_cache(R, T, G, hd)
        _plain_write(st["cache"], k, v, zero, kstart, G, hd)
    return st


# ----------------------------------------------------------------------------- plain forms
def _chunks(n, cost):
    """Ranges of ``n`` whose cost (elements of the score matrix) stays within about 2 GB."""

    step = max(1, int(5e8 // max(1, cost)))
    return [(i, min(n, i + step)) for i in range(0, n, step)]


def _split(qkv, H, G, hd):
    """``[B, L, (H + 2 G) hd]`` -> fp32 q ``[B, H, L, hd]`` and, repeated to H heads, k and v."""

    B, L, _ = qkv.shape
    x = qkv.detach().float().view(B, L, H + 2 * G, hd).transpose(1, 2)
    return x[:, :H], x[:, H:H + G].repeat_interleave(H // G, 1), x[:, H + G:].repeat_interleave(H // G, 1)


def _softmax(s, visible):
    """Softmax over the visible columns; a row without one is zero."""

    s = torch.where(visible, s, torch.full_like(s, -math.inf))
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = torch.exp(s - m)
    z = e.sum(-1, keepdim=True)
    return e / torch.where(z == 0, torch.ones_like(z), z)


def _plain_window(st):
    case = st["case"]
    qkv, kstart = st["qkv"], st["kstart"]
    L, lq, H, G, hd, W, S = (case[k] for k in ("L", "lq", "H", "G", "hd", "window", "sinks"))
    B = qkv.shape[0]
    scale = 1.0 / math.sqrt(hd)
    out = torch.empty(B, lq, H * hd, dtype=torch.bfloat16, device="cuda")
    grad = torch.empty(B, L, (H + 2 * G) * hd, dtype=torch.bfloat16, device="cuda") if case["kind"] == "train" else None
    kpos = torch.arange(L, device="cuda")
    qpos = torch.arange(L - lq, L, device="cuda").view(-1, 1)
    for a, b in _chunks(B, H * lq * L):
        q, k, v = _split(qkv[a:b], H, G, hd)
        ks = kstart[a:b].long().view(-1, 1, 1)
        vis = (kpos >= ks) & (kpos <= qpos) & ((qpos - kpos < W) | (kpos - ks < S))
        q = q[:, :, L - lq:]
        p = _softmax((q @ k.transpose(-1, -2)) * scale, vis.unsqueeze(1))
        o = p @ v
        out[a:b] = o.transpose(1, 2).reshape(b - a, lq, H * hd).bfloat16()
        if grad is None:
            continue
        do = st["dout"][a:b].float().view(b - a, lq, H, hd).transpose(1, 2)
        dv = p.transpose(-1, -2) @ do
        dp = do @ v.transpose(-1, -2)
        ds = p * (dp - (do * o).sum(-1, keepdim=True)) * scale
        dq = torch.zeros(b - a, H, L, hd, device="cuda")
        dq[:, :, L - lq:] = ds @ k
        dk = ds.transpose(-1, -2) @ q
        dk = dk.view(b - a, G, H // G, L, hd).sum(2)
        dv = dv.view(b - a, G, H // G, L, hd).sum(2)
        grad[a:b] = torch.cat([dq, dk, dv], 1).transpose(1, 2).reshape(b - a, L, -1).bfloat16()
    return out if grad is None else (out, grad)


def _quantise(x):
    """fp32 ``[..., hd]`` -> codes ``-7 .. 7`` and bf16 scales (one a row of ``hd``)."""

    top = x.abs().amax(-1)
    s = (top / 7.0).bfloat16()
    sf = s.float().unsqueeze(-1)
    c = torch.round(x / torch.where(sf == 0, torch.ones_like(sf), sf)).clamp(-7, 7)
    return torch.where(sf == 0, torch.zeros_like(c), c), s


def _plain_write(cache, k, v, start, kstart, G, hd):
    R, T, _ = k.shape
    x = torch.stack([k, v], 2).float().view(R, T, 2, G, hd)
    c, s = _quantise(x)
    n = (c + 8).to(torch.uint8)
    packed = n[..., 0::2] | (n[..., 1::2] << 4)
    t = torch.arange(T, device="cuda")
    live = t >= kstart.long().view(-1, 1)
    pos = start.long().view(-1, 1) + t - kstart.long().view(-1, 1)
    r, ti = live.nonzero(as_tuple=True)
    cache["codes"][r, pos[r, ti]] = packed[r, ti]
    cache["scales"][r, pos[r, ti]] = s[r, ti]
    cache["lengths"] = (start + T - kstart).int()


def _plain_values(cache, r):
    """fp32 keys and values ``[len(r), T, 2, G, hd]`` of cache rows ``r``."""

    n = cache["codes"][r]
    c = torch.stack([n & 15, n >> 4], -1).flatten(-2).float() - 8.0
    return c * cache["scales"][r].float().unsqueeze(-1)


def _plain_read(cache, start, count, G, hd):
    R, T = cache["codes"].shape[:2]
    pos = start.long().view(-1, 1) + torch.arange(count, device="cuda")
    live = (pos < cache["lengths"].long().view(-1, 1)).view(R, count, 1, 1, 1)
    r = torch.arange(R, device="cuda").view(-1, 1)
    p = pos.clamp(max=T - 1)
    n = cache["codes"][r, p]
    c = torch.stack([n & 15, n >> 4], -1).flatten(-2).float() - 8.0
    x = c * cache["scales"][r, p].float().unsqueeze(-1)
    x = torch.where(live, x, torch.zeros_like(x)).bfloat16()
    return x[:, :, 0].reshape(R, count, G * hd), x[:, :, 1].reshape(R, count, G * hd)


def _plain_attend(st):
    case, cache = st["case"], st["cache"]
    B, N, R, T, H, G, hd, W, S = (case[k] for k in ("B", "N", "R", "T", "H", "G", "hd", "window", "sinks"))
    rows = torch.arange(B, device="cuda") if st["rows"] is None else st["rows"].long()
    out = torch.empty(B, N, H * hd, dtype=torch.bfloat16, device="cuda")
    fresh = case["fresh"]
    kpos = torch.arange(T, device="cuda")
    n = torch.arange(N, device="cuda")
    for a, b in _chunks(B, T * (H * N + 2 * H * hd)):
        r = rows[a:b]
        x = _plain_values(cache, r).permute(2, 0, 3, 1, 4).repeat_interleave(H // G, 2)    # [2, b, H, T, hd]
        ln = cache["lengths"].long()[r].view(-1, 1, 1)
        qpos = (ln if fresh else ln - N) + n.view(1, -1, 1)
        vis = (kpos < ln) & (kpos <= qpos)
        if W:
            vis = vis & ((qpos - kpos < W) | (kpos < S))
        q, kn, vn = _split(st["qkv"][a:b], H, G, hd)
        k, v = x[0], x[1]
        if fresh:
            k, v = torch.cat([k, kn], 2), torch.cat([v, vn], 2)
            own_vis = n.view(1, 1, -1) <= n.view(1, -1, 1)
            if W:
                own_vis = own_vis & ((n.view(1, -1, 1) - n.view(1, 1, -1) < W) | (ln + n.view(1, 1, -1) < S))
            vis = torch.cat([vis, own_vis.expand(b - a, N, N)], 2)
        p = _softmax((q @ k.transpose(-1, -2)) / math.sqrt(hd), vis.unsqueeze(1))
        out[a:b] = (p @ v).transpose(1, 2).reshape(b - a, N, H * hd).bfloat16()
    return out


# ----------------------------------------------------------------------------- one pass
def run(state: dict):
    case = state["case"]
    kind = case["kind"]
    if own:
        return _run_own(state, case, kind)
    if kind in ("train", "prompt"):
        return _plain_window(state)
    G, hd, T = case["G"], case["hd"], case["T"]
    cache = state["cache"]
    if kind == "store":
        _plain_write(cache, state["k"], state["v"], state["start"], state["kstart"], G, hd)
        return (*_plain_read(cache, state["start"], T, G, hd), cache["lengths"])
    if kind == "read":
        return _plain_read(cache, torch.zeros_like(cache["lengths"]), T, G, hd)
    return _plain_attend(state)


def _run_own(state, case, kind):
    if kind in ("train", "prompt"):
        from mdl_b200.ops.window_attention import windowed_attention

        out = windowed_attention(state["qkv"], state["kstart"], case["H"], case["lq"], case["window"], case["sinks"],
                                 kv_heads=case["G"])
        if kind == "prompt":
            return out
        (grad,) = torch.autograd.grad(out, state["qkv"], state["dout"])
        return out.detach(), grad
    from mdl_b200.ops.kv_cache import cached_attention, kv_cache_read, kv_cache_write

    cache = state["cache"]
    if kind == "store":
        kv_cache_write(cache, state["k"], state["v"], start=state["start"], kstart=state["kstart"])
        return (*kv_cache_read(cache, case["T"], start=state["start"]), cache.lengths)
    if kind == "read":
        return kv_cache_read(cache, case["T"])
    H, G, hd = case["H"], case["G"], case["hd"]
    qkv = state["qkv"]
    kn = vn = None
    if case["fresh"]:
        kn, vn = qkv[..., H * hd:(H + G) * hd], qkv[..., (H + G) * hd:]
    return cached_attention(qkv[..., :H * hd], cache, rows=state["rows"], k_new=kn, v_new=vn, window=case["window"],
                            sinks=case["sinks"])


# ----------------------------------------------------------------------------- 64 bits
def exact(case: dict, seed: int):
    """What ``run`` returns, from the definitions in 64 bits, one sample and head at a time."""

    kind = case["kind"]
    if kind in ("train", "prompt"):
        return _exact_window(case, seed)
    G, hd, T, R = case["G"], case["hd"], case["T"], case["R"]
    if kind == "store":
        k, v, start, kstart = _store_inputs(case, seed)
        ends = (start + T - kstart).int()
    elif kind == "read":
        k, v, kstart = _read_inputs(case, seed)
    else:
        return _exact_attend(case, seed)
    outs = []
    for x in (k, v):
        y = _round4(x.double().view(R, T, G, hd)).view(R, T, G * hd)
        # token t of row r sits at row kstart[r] + t of the left-padded input
        t = torch.arange(T, device="cuda").view(1, -1) + kstart.long().view(-1, 1)
        z = torch.gather(y, 1, t.clamp(max=T - 1).unsqueeze(-1).expand(-1, -1, G * hd))
        outs.append(z * (t < T).unsqueeze(-1))
    return (*outs, ends) if kind == "store" else tuple(outs)


def _round4(x):
    """64-bit values that 4-bit codes with one bf16 scale a row stand for."""

    s = (x.abs().max(-1, keepdim=True).values / 7).to(torch.bfloat16).double()
    inv = torch.where(s > 0, s, torch.ones_like(s))
    return torch.round(x / inv).clamp(-7, 7) * s


def _exact_window(case, seed):
    qkv, kstart, dout = _tokens(case, seed)
    B, L, lq, H, G, hd, W, S = (case[k] for k in ("B", "L", "lq", "H", "G", "hd", "window", "sinks"))
    if B * H * lq * L > 3e9:
        return None
    train = case["kind"] == "train"
    out = torch.zeros(B, lq, H, hd, dtype=torch.float64, device="cuda")
    grad = torch.zeros(B, L, H + 2 * G, hd, dtype=torch.float64, device="cuda") if train else None
    x = qkv.view(B, L, H + 2 * G, hd)
    first = kstart.tolist()
    per = max(1, int(2e8 // (lq * L)))       # heads of a sample taken together
    for b in range(B):
        ks = min(first[b], L)
        q0 = max(ks, L - lq)
        if q0 >= L:
            continue
        i = torch.arange(q0, L, device="cuda").unsqueeze(1)
        j = torch.arange(ks, L, device="cuda").unsqueeze(0)
        hidden = (j > i) | ((i - j >= W) & (j - ks >= S))
        for h0 in range(0, H, per):
            hs = list(range(h0, min(H, h0 + per)))
            kvh = [h // (H // G) for h in hs]
            q = x[b, q0:, hs].double().transpose(0, 1)
            k = x[b, ks:, [H + c for c in kvh]].double().transpose(0, 1)
            v = x[b, ks:, [H + G + c for c in kvh]].double().transpose(0, 1)
            s = torch.einsum("hid,hjd->hij", q, k).div_(math.sqrt(hd)).masked_fill_(hidden, -math.inf)
            p = torch.softmax(s, -1)
            del s
            o = torch.einsum("hij,hjd->hid", p, v)
            out[b, lq - (L - q0):, hs] = o.transpose(0, 1)
            if not train:
                continue
            do = dout.view(B, lq, H, hd)[b, lq - (L - q0):, hs].double().transpose(0, 1)
            dv = torch.einsum("hij,hid->hjd", p, do)
            ds = torch.einsum("hid,hjd->hij", do, v).sub_((do * o).sum(-1, keepdim=True)).mul_(p).div_(math.sqrt(hd))
            grad[b, q0:, hs] = torch.einsum("hij,hjd->hid", ds, k).transpose(0, 1)
            dk = torch.einsum("hij,hid->hjd", ds, q)
            for n, c in enumerate(kvh):
                grad[b, ks:, H + c] += dk[n]
                grad[b, ks:, H + G + c] += dv[n]
    out = out.view(B, lq, H * hd)
    return (out, grad.view(B, L, -1)) if train else out


def _exact_attend(case, seed):
    k, v, kstart, qkv, rows = _attend_inputs(case, seed)
    B, N, R, T, H, G, hd, W, S = (case[n] for n in ("B", "N", "R", "T", "H", "G", "hd", "window", "sinks"))
    rl = list(range(B)) if rows is None else rows.tolist()
    first = kstart.tolist()
    out = torch.zeros(B, N, H, hd, dtype=torch.float64, device="cuda")
    x = qkv.view(B, N, H + 2 * G, hd)
    held, kk, vv = None, None, None
    for b in range(B):
        r = rl[b]
        n = T - first[r]
        if r != held:
            held = r
            kk = _round4(k[r, first[r]:].double().view(n, G, hd))
            vv = _round4(v[r, first[r]:].double().view(n, G, hd))
        kb, vb = kk, vv
        p0 = n - N
        if case["fresh"]:
            kb = torch.cat([kk, x[b, :, H:H + G].double()])
            vb = torch.cat([vv, x[b, :, H + G:].double()])
            p0 = n
        i = p0 + torch.arange(N, device="cuda").unsqueeze(1)
        j = torch.arange(kb.shape[0], device="cuda").unsqueeze(0)
        hidden = j > i
        if W:
            hidden = hidden | ((i - j >= W) & (j >= S))
        q = x[b, :, :H].double().view(N, G, H // G, hd)
        s = torch.einsum("ngad,jgd->ngaj", q, kb) / math.sqrt(hd)
        s = s.masked_fill(hidden.view(N, 1, 1, -1), -math.inf)
        p = torch.nan_to_num(torch.softmax(s, -1))       # a query before the first token sees nothing
        out[b] = torch.einsum("ngaj,jgd->ngad", p, vb).reshape(N, H, hd)
    return out.view(B, N, H * hd)


# ----------------------------------------------------------------------------- work
def _pairs(L, lq, ks, W, S):
    """Visible (query, key) pairs of one sample and head, averaged start ``ks``."""

    n = 0
    for i in range(max(0, L - lq - ks), L - ks):
        n += min(i + 1, W + min(S, max(0, i + 1 - W)))
    return n


def work(case: dict) -> dict:
    kind = case["kind"]
    G, hd = case["G"], case["hd"]
    if kind in ("train", "prompt"):
        B, L, lq, H = case["B"], case["L"], case["lq"], case["H"]
        ks = L // 4                        # kstart is uniform over 0 .. L // 2
        pairs = B * H * _pairs(L, lq, ks, case["window"], case["sinks"])
        seen = L - ks
        qk = B * hd * (min(lq, seen) * H + 2 * seen * G) * 2
        o = B * lq * H * hd * 2
        if kind == "prompt":
            return {"bytes": qk + o, "flops": 4 * pairs * hd}
        # the output gradient is read and the whole input gradient written besides; six products
        return {"bytes": qk + 2 * o + B * L * (H + 2 * G) * hd * 2, "flops": 12 * pairs * hd}
    R, T = case["R"], case["T"]
    if kind in ("store", "read"):
        live = T - T // 4 if kind == "store" else T - T // 6
        held = R * live * G * 2 * (hd // 2 + 2)
        full = R * T * G * 2 * hd * 2
        src = R * live * G * 2 * hd * 2
        # a value costs about a scaling and a rounding
        if kind == "read":
            return {"bytes": held + full, "flops": R * live * G * 2 * hd}
        return {"bytes": src + 2 * held + full, "flops": 4 * R * live * G * 2 * hd}
    B, N, H, W = case["B"], case["N"], case["H"], case["window"]
    ln = T - T // 8
    vis = min(ln, W + case["sinks"]) if W else ln
    used = R if not case["fresh"] else min(R, B)
    b = used * vis * G * 2 * (hd // 2 + 2) + 2 * B * N * H * hd * 2
    pairs = B * N * H * vis
    if case["fresh"]:
        b += B * N * 2 * G * hd * 2
        pairs += B * H * N * (N + 1) // 2
    return {"bytes": b, "flops": 4 * pairs * hd}
