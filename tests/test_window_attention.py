"""Sliding-window attention with first-token sinks, forward and gradients, against plain 64-bit
computations, on the CPU definition and on the CUDA kernels.

Tolerances. The kernels round P, dS (bf16, 8 significant bits: up to 2^-8 relative) and the
results (2^-8) and keep scores, sums and accumulators in fp32, so elementwise, with sums over
the visible pairs,
  |out error|  <= 2^-8 |out|  + 2^-8 sum_j p |v|
  |dV error|   <= 2^-8 |dV|   + 2^-8 sum_i p |do|
  |dQ error|   <= 2^-8 |dQ|   + sum_j (2^-8 |ds| + e p) |k|,  likewise dK with |q|,
where e bounds the error of dP - D: D is formed from the rounded output, which is within
2^-8 |out| + 2^-8 sum p |v| of the exact one, so e = scale * sum_d |do| (2^-8 |out| + 2^-8 sum p |v|).
The tests allow 1.05 times these bounds plus 1e-5 of the largest magnitude (fp32 sums in another
order, exp2 to 2^-22).
"""

import math

import pytest
import torch

from mdl_b200.ops.attention import suffix_attention_reference
from mdl_b200.ops.window_attention import windowed_attention, windowed_attention_reference

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
GPU = pytest.mark.gpu


def _inputs(B, Lk, lq, H, G, hd, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(B, Lk, (H + 2 * G) * hd, generator=g) * 1.2).bfloat16().to(device)
    dout = torch.randn(B, lq, H * hd, generator=g).bfloat16().to(device)
    return qkv, dout


def _exact(qkv, kstart, dout, H, G, lq, window, sinks, scale=None):
    """64-bit outputs and gradient, and the bounds of the module's text for each."""

    B, Lk, W = qkv.shape
    hd = W // (H + 2 * G)
    scale = scale or hd ** -0.5
    x = qkv.double().cpu().view(B, Lk, H + 2 * G, hd)
    do_all = dout.double().cpu().view(B, lq, H, hd)
    out, out_tol = torch.zeros(B, lq, H, hd, dtype=torch.float64), torch.zeros(B, lq, H, hd, dtype=torch.float64)
    grad, grad_tol = torch.zeros_like(x), torch.zeros_like(x)
    u = 2.0 ** -8
    for b in range(B):
        ks = min(max(int(kstart[b]), 0), Lk)
        q0 = max(ks, Lk - lq)
        if q0 >= Lk:
            continue
        i = torch.arange(q0, Lk).view(-1, 1)
        j = torch.arange(ks, Lk).view(1, -1)
        seen = (j <= i) & ((i - j < window) | (j - ks < sinks))
        off = q0 - (Lk - lq)
        for h in range(H):
            g = h // (H // G)
            q, k, v = x[b, q0:, h], x[b, ks:, H + g], x[b, ks:, H + G + g]
            p = torch.softmax((q @ k.T * scale).masked_fill(~seen, -math.inf), -1)
            o = p @ v
            do = do_all[b, off:, h]
            o_mag = p @ v.abs()
            out[b, off:, h] = o
            out_tol[b, off:, h] = u * o.abs() + u * o_mag
            ds = p * (do @ v.T - (do * o).sum(-1, keepdim=True)) * scale
            e = scale * (do.abs() * (u * o.abs() + u * o_mag)).sum(-1, keepdim=True)
            ds_tol = u * ds.abs() + e * p
            for idx, val, tol in ((h, ds @ k, ds_tol @ k.abs()),):
                grad[b, q0:, idx] += val
                grad_tol[b, q0:, idx] += tol
            grad[b, ks:, H + g] += ds.T @ q
            grad_tol[b, ks:, H + g] += ds_tol.T @ q.abs()
            grad[b, ks:, H + G + g] += p.T @ do
            grad_tol[b, ks:, H + G + g] += u * (p.T @ do.abs())
    grad_tol += u * grad.abs()
    return (out.view(B, lq, -1), out_tol.view(B, lq, -1)), (grad.view(B, Lk, W), grad_tol.view(B, Lk, W))


def _close(got, want, tol):
    err = (got.detach().double().cpu() - want).abs()
    slack = 1e-5 * float(want.abs().max()) if want.numel() else 0.0
    assert torch.isfinite(got).all()
    assert (err <= 1.05 * tol + slack).all(), float((err / (tol + slack + 1e-300)).max())


def _errors():
    from mdl_b200.ops._ext import check_error_word

    torch.cuda.synchronize()
    check_error_word(torch.device("cuda", 0))


def _run(device, B, Lk, lq, H, G, hd, window, sinks, kstart, seed=0, scale=None):
    qkv, dout = _inputs(B, Lk, lq, H, G, hd, device, seed)
    ks = torch.tensor(kstart, dtype=torch.int32, device=device)
    (out, otol), (grad, gtol) = _exact(qkv, kstart, dout, H, G, lq, window, sinks, scale)
    x = (qkv if device == "cuda" else qkv.float()).clone().requires_grad_()
    got = windowed_attention(x, ks, H, lq, window, sinks, kv_heads=G, scale=scale)
    (dx,) = torch.autograd.grad(got, x, dout.to(got.dtype))
    if device == "cpu":
        otol, gtol = otol * 2.0 ** -8, gtol * 2.0 ** -8
    else:
        assert got.dtype == torch.bfloat16
        _errors()
    _close(got, out, otol)
    _close(dx, grad, gtol)
    return got, dx


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("hd", [32, 64])
@pytest.mark.parametrize("Lk,lq,window,sinks", [
    (1, 1, 1, 0), (5, 5, 2, 1), (64, 64, 64, 0), (127, 127, 16, 3), (128, 128, 1, 0), (129, 129, 128, 1),
    (200, 1, 50, 4), (255, 130, 129, 7), (300, 300, 1000, 0), (300, 17, 65, 130), (385, 257, 63, 64),
    (513, 513, 100, 5), (640, 640, 1, 2),
])
def test_sizes_windows_and_sinks(device, hd, Lk, lq, window, sinks):
    _run(device, 2, Lk, lq, 2, 2, hd, window, sinks, [0, Lk // 3], seed=Lk)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("H,G", [(1, 1), (3, 3), (4, 2), (6, 2), (4, 1)])
@pytest.mark.parametrize("hd", [32, 64])
def test_shared_heads(device, hd, H, G):
    _run(device, 2, 210, 150, H, G, hd, 40, 3, [0, 77], seed=H)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("Lk,lq,window,sinks", [(200, 200, 30, 2), (333, 60, 100, 0), (150, 150, 500, 9)])
def test_padding_prefix(device, Lk, lq, window, sinks):
    """Samples from no padding to nothing but padding, starts past the end and before 0."""

    kstart = [0, 1, 63, 64, 127, 128, Lk - lq, Lk - 1, Lk, Lk + 5, -3]
    got, dx = _run(device, len(kstart), Lk, lq, 2, 1, 32, window, sinks, kstart)
    for b, ks in enumerate(kstart):
        pad = max(0, min(ks, Lk) - (Lk - lq))
        assert not got[b, :pad].any() and not dx[b, :max(0, min(ks, Lk))].any()


@pytest.mark.parametrize("device", DEVICES)
def test_window_of_the_whole_history_is_the_suffix_attention(device):
    B, Lk, lq, H, hd = 3, 290, 140, 2, 32
    qkv, _ = _inputs(B, Lk, lq, H, H, hd, device)
    ks = torch.tensor([0, 30, 200], dtype=torch.int32, device=device)
    want = suffix_attention_reference(qkv, ks, H, lq)
    x = qkv if device == "cuda" else qkv.float()
    for window, sinks in ((Lk, 0), (10 ** 9, 5), (1, Lk), (7, 10 ** 9)):
        got = windowed_attention(x, ks, H, lq, window, sinks)
        bound = 1.05 * 2.0 ** -7 * suffix_attention_reference(
            torch.cat([qkv[..., :2 * H * hd], qkv[..., 2 * H * hd:].abs()], -1), ks, H, lq)
        assert ((got.float() - want).abs() <= bound + 1e-5).all()


@pytest.mark.parametrize("device", DEVICES)
def test_gradient_against_differences(device):
    """Directional derivative of a smooth function of the output by central differences of the
    64-bit forward, against the gradient; 2^-6 covers the bf16 roundings of a sum of this size."""

    B, Lk, lq, H, G, hd, window, sinks = 2, 90, 70, 4, 2, 32, 20, 3
    qkv, dout = _inputs(B, Lk, lq, H, G, hd, device, 5)
    ks = [0, 25]
    x = (qkv if device == "cuda" else qkv.float()).clone().requires_grad_()
    out = windowed_attention(x, torch.tensor(ks, device=device), H, lq, window, sinks, kv_heads=G)
    (dx,) = torch.autograd.grad(out, x, dout.to(out.dtype))
    g = torch.Generator().manual_seed(1)
    for part in (slice(0, H * hd), slice(H * hd, (H + G) * hd), slice((H + G) * hd, None)):
        # along the gradient itself, so that the derivative is a sum of squares
        direction = torch.zeros(qkv.shape, dtype=torch.float64)
        direction[..., part] = dx.double().cpu()[..., part] + 0.1 * torch.randn(
            direction[..., part].shape, generator=g, dtype=torch.float64)
        eps = 1e-5
        vals = []
        for s in (1, -1):
            (o, _), _ = _exact(qkv.double().cpu() + s * eps * direction, ks, dout, H, G, lq, window, sinks)
            vals.append(float((o * dout.double().cpu()).sum()))
        want = (vals[0] - vals[1]) / (2 * eps)
        got = float((dx.double().cpu() * direction).sum())
        assert abs(got - want) <= 2.0 ** -6 * abs(want)


@pytest.mark.parametrize("device", DEVICES)
def test_strides_and_scale(device):
    """A view into a wider buffer with a batch stride of its own, and an odd view."""

    B, Lk, lq, H, hd = 3, 140, 100, 2, 32
    W = 3 * H * hd
    qkv, dout = _inputs(B, Lk, lq, H, H, hd, device)
    ks = torch.tensor([0, 11, 139], dtype=torch.int32, device=device)
    want = windowed_attention(qkv, ks, H, lq, 33, 2, scale=0.3)
    wide = torch.full((B, Lk + 3, W + 24), float("nan"), dtype=torch.bfloat16, device=device)
    for at in (8, 5):
        view = wide[:, 2:Lk + 2, at:at + W]
        view.copy_(qkv)
        leaf = view.detach().requires_grad_()
        got = windowed_attention(leaf, ks, H, lq, 33, 2, scale=0.3)
        assert torch.equal(got, want)
        (dx,) = torch.autograd.grad(got, leaf, dout.to(got.dtype))
        assert torch.isfinite(dx).all() and dx.shape == qkv.shape
        wide.fill_(float("nan"))
    _run(device, 2, 77, 77, 2, 2, 64, 20, 1, [3, 0], scale=0.3)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_padding_may_hold_anything(device, bad):
    B, Lk, lq, H, hd = 2, 200, 200, 2, 64
    qkv, dout = _inputs(B, Lk, lq, H, H, hd, device)
    ks = torch.tensor([40, 131], dtype=torch.int32, device=device)
    res = []
    for fill in (0.0, bad):
        x = (qkv if device == "cuda" else qkv.float()).clone()
        for b in range(B):
            x[b, :int(ks[b])] = fill
        x.requires_grad_()
        o = windowed_attention(x, ks, H, lq, 50, 3)
        res.append((o, torch.autograd.grad(o, x, dout.to(o.dtype))[0]))
    assert torch.isfinite(res[1][0]).all() and torch.isfinite(res[1][1]).all()
    assert torch.equal(res[0][0], res[1][0]) and torch.equal(res[0][1], res[1][1])


@pytest.mark.parametrize("device", DEVICES)
def test_large_scores(device):
    """Scores of thousands: the running reference has to move, weights are 0 or 1."""

    qkv, dout = _inputs(1, 300, 300, 1, 1, 32, device)
    qkv[..., :64] *= 30
    # fp32 scores of about 3e4 (base 2) carry 2^-9; with gaps that small the weights differ by 2^-9
    x = qkv if device == "cuda" else qkv.float()
    ks = torch.zeros(1, dtype=torch.int32, device=device)
    got = windowed_attention(x, ks, 1, 300, 100, 2)
    want = windowed_attention_reference(qkv, ks, 1, 300, 100, 2)
    assert torch.isfinite(got).all()
    # |out| <= max |v| < 8: roundings 2^-7 and weights 2 * 2^-8 of it
    assert (got.float() - want).abs().max() <= 8 * 2.0 ** -6


@GPU
@pytest.mark.parametrize("B,Lk,lq,H,G,hd,window,sinks", [(2, 3000, 3000, 4, 2, 64, 700, 10),
                                                          (40, 544, 544, 8, 8, 32, 128, 4)])
def test_long_and_many(B, Lk, lq, H, G, hd, window, sinks):
    """Several work items a block, long streams; repeated runs agree bit for bit."""

    kstart = [(37 * b) % (Lk // 2) for b in range(B)]
    qkv, dout = _inputs(B, Lk, lq, H, G, hd, "cuda", 3)
    ks = torch.tensor(kstart, dtype=torch.int32, device="cuda")
    x = qkv.clone().requires_grad_()
    first = None
    for _ in range(3):
        o = windowed_attention(x, ks, H, lq, window, sinks, kv_heads=G)
        (dx,) = torch.autograd.grad(o, x, dout)
        if first is None:
            first = (o, dx)
        assert torch.equal(o, first[0]) and torch.equal(dx, first[1])
    _errors()
    n = 1 if Lk > 1000 else 3
    (out, otol), (grad, gtol) = _exact(qkv[-n:], kstart[-n:], dout[-n:], H, G, lq, window, sinks)
    _close(o[-n:], out, otol)
    _close(dx[-n:], grad, gtol)


@GPU
def test_on_another_stream():
    qkv, dout = _inputs(4, 400, 400, 4, 4, 64, "cuda")
    ks = torch.tensor([0, 5, 100, 399], dtype=torch.int32, device="cuda")
    want = windowed_attention(qkv, ks, 4, 400, 90, 4)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        x = qkv.clone().requires_grad_()
        got = windowed_attention(x, ks, 4, 400, 90, 4)
        got.backward(dout)
    side.synchronize()
    assert torch.equal(got, want) and torch.isfinite(x.grad).all()


@pytest.mark.parametrize("device", DEVICES)
def test_empty(device):
    qkv = torch.zeros(0, 10, 96, dtype=torch.bfloat16, device=device)
    assert windowed_attention(qkv, torch.zeros(0, dtype=torch.int32, device=device), 1, 10, 3).shape == (0, 10, 32)
    qkv = torch.zeros(2, 10, 96, dtype=torch.bfloat16, device=device)
    assert windowed_attention(qkv, torch.zeros(2, dtype=torch.int32, device=device), 1, 0, 3).shape == (2, 0, 32)


@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    qkv = torch.zeros(2, 10, 96, dtype=torch.bfloat16, device=device)
    ks = torch.zeros(2, dtype=torch.int32, device=device)
    for args, kw in [((qkv, ks, 1, 11, 3), {}), ((qkv, ks, 1, 10, 0), {}), ((qkv, ks, 1, 10, 3, -1), {}),
                     ((qkv, ks, 3, 10, 3), dict(kv_heads=2)), ((qkv, ks, 7, 10, 3), {}), ((qkv[0], ks, 1, 10, 3), {}),
                     ((qkv, ks[:1], 1, 10, 3), {}), ((qkv, ks.float(), 1, 10, 3), {}), ((qkv, ks, 0, 10, 3), {})]:
        with pytest.raises(ValueError):
            windowed_attention(*args, **kw)
    if device == "cuda":
        with pytest.raises(TypeError):
            windowed_attention(qkv.half(), ks, 1, 10, 3)
        with pytest.raises(NotImplementedError):
            windowed_attention(qkv, ks, 2, 10, 3)
        with pytest.raises(ValueError):
            windowed_attention(qkv, ks.cpu(), 1, 10, 3)


@GPU
@pytest.mark.parametrize("B,Lk,lq,H,G,hd,window,sinks,kstart", [
    (1, 6000, 6000, 2, 1, 64, 40, 3, [0]), (2, 5000, 4500, 1, 1, 32, 100, 200, [0, 4400]),
    (2, 4096, 4096, 2, 2, 32, 64, 1, [4095, 1]), (1, 9000, 9000, 1, 1, 64, 1, 129, [17]),
])
def test_sinks_of_few_long_samples(B, Lk, lq, H, G, hd, window, sinks, kstart):
    """The sinks' key tiles, which every query sees, are summed in parts."""

    qkv, dout = _inputs(B, Lk, lq, H, G, hd, "cuda", 8)
    ks = torch.tensor(kstart, dtype=torch.int32, device="cuda")
    x = qkv.clone().requires_grad_()
    o = windowed_attention(x, ks, H, lq, window, sinks, kv_heads=G)
    (dx,) = torch.autograd.grad(o, x, dout)
    o2 = windowed_attention(x, ks, H, lq, window, sinks, kv_heads=G)
    assert torch.equal(dx, torch.autograd.grad(o2, x, dout)[0])
    _errors()
    (out, otol), (grad, gtol) = _exact(qkv, kstart, dout, H, G, lq, window, sinks)
    _close(o, out, otol)
    _close(dx, grad, gtol)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("scale", [0.0, -0.25, math.inf, math.nan])
def test_scale_is_positive(device, scale):
    qkv = torch.zeros(2, 16, 3 * 2 * 32, dtype=torch.bfloat16, device=device)
    with pytest.raises(ValueError, match="scale"):
        windowed_attention(qkv, torch.zeros(2, dtype=torch.int32, device=device), 2, 16, 4, scale=scale)


@pytest.mark.parametrize("device", DEVICES)
def test_starts_past_32_bits_do_not_wrap(device):
    """A 64-bit start past the sample's end is all padding, one far below 0 is none."""

    qkv, _ = _inputs(3, 50, 50, 2, 2, 32, device)
    x = qkv if device == "cuda" else qkv.float()
    got = windowed_attention(x, torch.tensor([2 ** 32, -2 ** 32 + 7, 5], device=device), 2, 50, 9, 1)
    want = windowed_attention(x, torch.tensor([50, 0, 5], device=device), 2, 50, 9, 1)
    assert torch.equal(got, want) and not got[0].any() and got[1, 0].any()


@GPU
def test_forward_without_a_gradient_keeps_nothing_for_one():
    """Under no_grad a forward takes its output and the log-sum-exp, and no more."""

    B, L, H, hd = 64, 512, 8, 32
    qkv, _ = _inputs(B, L, L, H, H, hd, "cuda")
    ks = torch.zeros(B, dtype=torch.int32, device="cuda")
    out_bytes, lse_bytes = 2 * B * L * H * hd, 4 * B * L * H
    for leaf in (qkv, qkv.clone().requires_grad_()):
        for mode in (torch.no_grad, torch.inference_mode):
            with mode():
                windowed_attention(leaf, ks, H, L, 50, 2)
                torch.cuda.synchronize()
                torch.cuda.reset_peak_memory_stats()
                before = torch.cuda.memory_allocated()
                out = windowed_attention(leaf, ks, H, L, 50, 2)
                assert torch.cuda.max_memory_allocated() - before <= out_bytes + lse_bytes + 4096
                assert not out.requires_grad
                del out


@pytest.mark.parametrize("device", DEVICES)
def test_a_second_derivative_is_right_or_refused(device):
    """The CPU definition has one; the kernels refuse it instead of leaving its terms out."""

    qkv, dout = _inputs(1, 20, 20, 1, 1, 32, device)
    ks = torch.zeros(1, dtype=torch.int32, device=device)
    x = (qkv if device == "cuda" else qkv.float()).clone().requires_grad_()
    out = windowed_attention(x, ks, 1, 20, 7, 1)
    (dx,) = torch.autograd.grad(out, x, dout.to(out.dtype), create_graph=True)
    assert dx.requires_grad
    total = out.float().sum() + dx.float().square().sum()
    if device == "cuda":
        with pytest.raises(RuntimeError, match="second derivative"):
            torch.autograd.grad(total, x)
    else:
        assert torch.isfinite(torch.autograd.grad(total, x)[0]).all()
    # a first derivative in which it has no part stays possible
    out = windowed_attention(x, ks, 1, 20, 7, 1)
    (dx,) = torch.autograd.grad(out, x, dout.to(out.dtype), create_graph=True)
    want = torch.autograd.grad(windowed_attention(x, ks, 1, 20, 7, 1), x, dout.to(out.dtype))[0]
    assert torch.equal(dx.detach(), want)


def _rounded_gradients(q, k, v, do, seen):
    """dQ and dK of one head in 64 bits: exact, with the kernels' roundings (P of the output and the
    keys' dS to bf16, D from the output in two bf16 terms, the queries' dS in two), with D from the
    rounded output, and with the queries' dS in one term."""

    def bf(x):
        return x.float().bfloat16().double()

    scale = q.shape[1] ** -0.5
    s = (q @ k.T * scale).masked_fill(~seen, -math.inf)
    p, dp = torch.softmax(s, -1), do @ v.T
    e = torch.exp(s - s.amax(-1, keepdim=True))
    o = (bf(e) @ v) / e.sum(-1, keepdim=True)
    high = bf(o)

    def grads(d, terms):
        ds = p * (dp - d)
        hi = bf(ds)
        return bf(scale * (hi + bf(ds - hi) if terms == 2 else hi) @ k), bf(scale * hi.T @ q)

    def row_sum(x):
        return (do * x).sum(-1, keepdim=True)

    exact = p * (dp - row_sum(p @ v))
    return {"exact": (scale * exact @ k, scale * exact.T @ q), "kernel": grads(row_sum(high + bf(o - high)), 2),
            "rounded output": grads(row_sum(high), 2), "one term": grads(row_sum(high + bf(o - high)), 1)}


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("hd", [32, 64])
@pytest.mark.parametrize("gain,lost", [(2.0, "rounded output"), (0.5, "one term")])
def test_gradient_keeps_its_second_terms(device, hd, gain, lost):
    """The norm of the error of dQ (for D: of dK too) is that of the kernels' roundings, computed in 64
    bits, and not that of a form which has lost the output's low part or the queries' second term of
    dS. The limit is the geometric mean of the two, which are at least 1.2 apart for these inputs."""

    L, H, window, sinks = 400, 2, 64, 2
    g = torch.Generator().manual_seed(0)
    qkv = torch.randn(1, L, 3 * H * hd, generator=g)
    qkv[..., :2 * H * hd] *= gain
    qkv = qkv.bfloat16()
    dout = torch.randn(1, L, H * hd, generator=g).bfloat16()
    i, j = torch.arange(L).view(-1, 1), torch.arange(L).view(1, -1)
    seen = (j <= i) & ((i - j < window) | (j < sinks))
    x = qkv[0].double().view(L, 3 * H, hd)
    heads = [_rounded_gradients(x[:, h], x[:, H + h], x[:, 2 * H + h], dout[0].double().view(L, H, hd)[:, h], seen)
             for h in range(H)]
    forms = {name: [torch.cat([f[name][n] for f in heads], -1) for n in (0, 1)] for name in heads[0]}

    def error(form, n):
        return float((form[n] - forms["exact"][n]).norm() / forms["exact"][n].norm())

    if device == "cuda":
        leaf = qkv.cuda().requires_grad_()
        out = windowed_attention(leaf, torch.zeros(1, dtype=torch.int32, device="cuda"), H, L, window, sinks)
        (dx,) = torch.autograd.grad(out, leaf, dout.cuda())
        dx = dx[0].double().cpu()
        got = [dx[:, :H * hd], dx[:, H * hd:2 * H * hd]]
    for n in ((0, 1) if lost == "rounded output" else (0,)):
        now, without = error(forms["kernel"], n), error(forms[lost], n)
        assert without > 1.2 * now
        limit = math.sqrt(now * without)
        if device == "cuda":
            assert error(got, n) <= limit, (error(got, n), now, without)
        else:
            assert now <= limit < without


@GPU
def test_more_elements_than_32_bits_count():
    """2,800 samples of 1,024 tokens: the last of them as by itself."""

    B, L, H, hd, window, sinks = 2800, 1024, 8, 32, 60, 3
    g = torch.Generator(device="cuda").manual_seed(1)
    qkv = torch.zeros(B, L, 3 * H * hd, dtype=torch.bfloat16, device="cuda")
    dout = torch.zeros(B, L, H * hd, dtype=torch.bfloat16, device="cuda")
    assert qkv.numel() > 2 ** 31
    qkv[-1:].normal_(generator=g)
    dout[-1:].normal_(generator=g)
    ks = torch.full((B,), 5, dtype=torch.int32, device="cuda")
    x = qkv.requires_grad_()
    o = windowed_attention(x, ks, H, L, window, sinks)
    (dx,) = torch.autograd.grad(o, x, dout)
    (out, otol), (grad, gtol) = _exact(qkv[-1:].detach(), [5], dout[-1:], H, H, L, window, sinks)
    _close(o[-1:], out, otol)
    _close(dx[-1:], grad, gtol)
    assert not o[:-1].any() and not dx[:-1].any()
    _errors()


@GPU
def test_error_word_first_used_in_inference_mode(monkeypatch):
    """The device's error word can be cleared afterwards, outside the mode."""

    from mdl_b200.ops import _ext

    monkeypatch.setattr(_ext, "_ERROR_WORDS", {})
    qkv = torch.zeros(1, 16, 96, dtype=torch.bfloat16, device="cuda")
    with torch.inference_mode():
        windowed_attention(qkv, torch.zeros(1, dtype=torch.int32, device="cuda"), 1, 16, 4)
    word = _ext.error_word(qkv.device)
    torch.cuda.synchronize()
    word.fill_(8)
    with pytest.raises(RuntimeError, match="outside"):
        _ext.check_error_word(qkv.device)
    assert int(word) == 0
