"""OneTrans with a bounded view (``attention_window`` / ``attention_sinks``) and a 4-bit request
cache: the training step against the CPU definition, and a cache written, read and scored from."""

import pytest
import torch

from mdl_b200.config.loader import app_config_from_mapping
from mdl_b200.config.schema import ConfigError
from mdl_b200.data.baseline_configs import scaled_config
from mdl_b200.data.batch import PackedBatch
from mdl_b200.data.synthetic import SyntheticGenerator
from mdl_b200.models.factory import build_model
from mdl_b200.ops._ext import check_error_word
from mdl_b200.ops.kv_cache import QuantizedKVCache, kv_cache_read
from mdl_b200.ops.preflight import attention_preflight
from mdl_b200.train.trainer import Trainer

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _config(seq_len=40, layers=3, min_len=5, token_dim=64, heads=2, **model):
    m, spec = scaled_config(4, 1e-4, num_fields=12, batch=64, seq_len=seq_len, num_layers=layers,
                            pyramid_schedule="halve")
    m["model"].update({"hidden_dim": 128, "token_dim": token_dim, "num_heads": heads, "num_ns_tokens": 4,
                       "task_head_hidden_dim": 64, "pyramid_round_to": 8, **model})
    m["training"].update({"lr_warmup_steps": 0, "dense_optimizer": "adam", "lr_dense": 1e-3})
    spec.sequences["behavior"].min_len = min_len
    return m, spec


def test_settings():
    for model, message in (({"attention_window": -1}, "negative"), ({"attention_sinks": 2}, "attention_window"),
                           ({"request_cache_format": "8bit"}, "request_cache_format")):
        with pytest.raises(ConfigError, match=message):
            app_config_from_mapping(_config(**model)[0])
    m, _ = scaled_config(2, 1e-4, num_fields=12, batch=64)
    m["model"]["attention_window"] = 8
    with pytest.raises(ConfigError, match="windowed"):
        app_config_from_mapping(m)
    cfg = app_config_from_mapping(_config(attention_window=8, request_cache_format="4bit")[0])
    assert attention_preflight(cfg)["paths"]["mixed_causal"].startswith("tcgen05 windowed")
    with pytest.raises(ValueError, match="attention_window"):
        attention_preflight(app_config_from_mapping(_config(token_dim=64, heads=8, attention_window=8)[0]))


def test_a_window_of_everything_changes_nothing():
    losses = []
    for model in ({}, {"attention_window": 1000, "attention_sinks": 3}):
        m, spec = _config(**model)
        cfg = app_config_from_mapping(m)
        torch.manual_seed(0)
        net = build_model(cfg, device="cpu", base_seed=1)
        batch = SyntheticGenerator(net.encoder.batch_plan, spec).batch(16)
        losses.append(Trainer(cfg, net, device=torch.device("cpu")).forward_backward(batch)["logits"].detach())
    torch.testing.assert_close(losses[0], losses[1], atol=1e-6, rtol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("model", [dict(attention_window=9, attention_sinks=2),
                                   dict(seq_len=300, layers=4, min_len=50, token_dim=128, heads=2, attention_window=64,
                                        attention_sinks=4)])
def test_training_step_matches_the_cpu_definition(model):
    m, spec = _config(**model)
    cfg = app_config_from_mapping(m)
    torch.manual_seed(0)
    cpu_model = build_model(cfg, device="cpu", base_seed=1)
    gpu_model = build_model(cfg, device="cuda", base_seed=1)
    gpu_model.load_state_dict({k: v.cuda() for k, v in cpu_model.state_dict().items()})
    gpu_model.store.slab.copy_(cpu_model.store.slab)
    cpu_tr = Trainer(cfg, cpu_model, device=torch.device("cpu"))
    gpu_tr = Trainer(cfg, gpu_model, device=torch.device("cuda"))
    batch = SyntheticGenerator(cpu_model.encoder.batch_plan, spec).batch(64)
    out_c = cpu_tr.forward_backward(batch)
    out_g = gpu_tr.forward_backward(batch.to("cuda"))
    torch.cuda.synchronize()
    check_error_word(0)
    # the tolerances of the step without a window
    torch.testing.assert_close(out_g["logits"].cpu(), out_c["logits"].detach(), atol=6e-2, rtol=6e-2)
    gc, gg = cpu_tr.dense.grad, gpu_tr.dense.grad.cpu()
    for name in cpu_tr.dense.names:
        o = cpu_tr.dense.offsets[name]
        n = cpu_tr.dense.params[name].numel()
        err = ((gc[o:o + n] - gg[o:o + n]).norm() / (gc[o:o + n].norm() + 1e-9)).item()
        assert err < 0.06, f"{name}: grad error {err:.3f}"
    assert ((cpu_model.store.grad - gpu_model.store.grad.cpu()).norm() / (cpu_model.store.grad.norm() + 1e-9)) < 0.06


def _requests(batch, cfg, rows, per):
    seq = batch.sequences["behavior"]
    L = cfg.sequences[0].max_length
    nf = seq["ids"].shape[0]
    req = {"ids": seq["ids"].view(nf, rows, L)[:, ::per].reshape(nf, -1), "lengths": seq["lengths"][::per].clone(),
           "row_indices": torch.arange(rows) // per}
    b = batch
    return PackedBatch.pack(b.ids, b.offsets, b.dense, b.labels, b.label_mask, b.scenario_id, b.rows,
                            {**b.sequences, "behavior": req})


@pytest.mark.parametrize("window,sinks", [(7, 2), (25, 0)])
def test_full_request_cache_matches_the_full_forward(window, sinks):
    m, spec = _config(min_len=3, attention_window=window, attention_sinks=sinks)
    cfg = app_config_from_mapping(m)
    torch.manual_seed(0)
    model = build_model(cfg, device="cpu", base_seed=1).eval()
    rb = _requests(SyntheticGenerator(model.encoder.batch_plan, spec).batch(24), cfg, 24, 6)
    with torch.no_grad():
        full = model(rb)["logits"].float()
        cached = model.forward_with_cache(rb, model.precompute_request_cache(rb))
    torch.testing.assert_close(cached, full, atol=1e-4, rtol=1e-4)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("window,sinks,heads", [(0, 0, 2), (11, 3, 1)])
def test_four_bit_request_cache(device, window, sinks, heads):
    """Scores from a 4-bit cache equal those of a full cache that holds what the 4-bit one stands
    for (fp32 on the CPU; bf16 operands on CUDA, with the tolerance of the native step), and
    the cache takes the bytes it says."""

    m, spec = _config(min_len=3, heads=heads, attention_window=window, attention_sinks=sinks, request_cache_format="4bit")
    cfg = app_config_from_mapping(m)
    torch.manual_seed(0)
    model = build_model(cfg, device=device, base_seed=1).eval()
    rb = _requests(SyntheticGenerator(model.encoder.batch_plan, spec).batch(24), cfg, 24, 6).to(device)
    with torch.no_grad():
        cache = model.precompute_request_cache(rb)
        scores = model.forward_with_cache(rb, cache)
        layers = []
        for kv, kst in cache["layers"]:
            assert isinstance(kv, QuantizedKVCache)
            assert kv.nbytes == kv.num_pages * kv.page * kv.kv_heads * (kv.head_dim + 4)
            s_in = int((kv.lengths + kst).max())
            k, v = kv_cache_read(kv, s_in, dtype=torch.float32)
            back = torch.zeros(*k.shape[:2], 2 * k.shape[2], device=k.device)
            for r in range(k.shape[0]):
                n, p = int(kv.lengths[r]), int(kst[r])
                assert n + p == s_in
                back[r, p:] = torch.cat([k[r, :n], v[r, :n]], -1)
            layers.append((back, kst))
        want = model.forward_with_cache(rb, {**cache, "layers": layers})
    tol = 1e-4 if device == "cpu" else 6e-2
    torch.testing.assert_close(scores, want, atol=tol, rtol=tol)
    if device == "cuda":
        torch.cuda.synchronize()
        check_error_word(0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (5, 2)])
def test_four_bit_request_cache_of_a_pyramid_that_halves_to_nothing(device, window, sinks):
    """Layers that keep no sequence token have an empty cache: candidates see their own tokens
    alone. Against a full cache of the values that the 4-bit one stands for, as above."""

    m, spec = _config(seq_len=16, layers=6, min_len=3, pyramid_round_to=1, pyramid_halve_every=1,
                      attention_window=window, attention_sinks=sinks, request_cache_format="4bit")
    cfg = app_config_from_mapping(m)
    torch.manual_seed(0)
    model = build_model(cfg, device=device, base_seed=1).eval()
    assert model.query_counts[-2:] == [0, 0]
    rb = _requests(SyntheticGenerator(model.encoder.batch_plan, spec).batch(12), cfg, 12, 4).to(device)
    with torch.no_grad():
        cache = model.precompute_request_cache(rb)
        scores = model.forward_with_cache(rb, cache)
        layers = []
        for s_in, (kv, kst) in zip([16, *model.query_counts], cache["layers"]):
            k, v = kv_cache_read(kv, s_in, dtype=torch.float32)
            back = torch.zeros(k.shape[0], s_in, 2 * k.shape[2], device=k.device)
            for r in range(k.shape[0]):
                n = int(kv.lengths[r])
                assert n == s_in - int(kst[r])
                back[r, s_in - n:] = torch.cat([k[r, :n], v[r, :n]], -1)
            layers.append((back, kst))
        assert cache["layers"][-1][0].nbytes == 0
        want = model.forward_with_cache(rb, {**cache, "layers": layers})
    tol = 1e-4 if device == "cpu" else 6e-2
    torch.testing.assert_close(scores, want, atol=tol, rtol=tol)
    if device == "cuda":
        torch.cuda.synchronize()
        check_error_word(0)


@pytest.mark.parametrize("fmt", ["full", "4bit"])
def test_request_cache_of_no_requests(fmt):
    m, spec = _config(min_len=3, request_cache_format=fmt)
    cfg = app_config_from_mapping(m)
    model = build_model(cfg, device="cpu", base_seed=1).eval()
    rb = _requests(SyntheticGenerator(model.encoder.batch_plan, spec).batch(4), cfg, 4, 2)
    seq = rb.sequences["behavior"]
    none = {"ids": seq["ids"][:, :0], "lengths": seq["lengths"][:0], "row_indices": seq["row_indices"][:0]}
    rb.sequences["behavior"] = none
    cache = model.precompute_request_cache(rb)
    assert len(cache["layers"]) == 3 and cache["kstart"].shape == (0,)
    if fmt == "4bit":
        assert not any(kv.lengths.any() for kv, _ in cache["layers"])


@pytest.mark.gpu
@pytest.mark.parametrize("model", [dict(heads=1, attention_window=9, attention_sinks=2), dict(heads=1), dict(heads=8)])
def test_mdl_onetrans_takes_the_head_widths_that_preflight_promises(model):
    """64-wide heads, with a window and without, and 8-wide ones: a step against the CPU definition,
    with the tolerances of the 32-wide one."""

    model = dict(model)
    heads = model.pop("heads")
    m, spec = scaled_config(4, 1e-4, num_fields=12, batch=64, seq_len=40, num_layers=3, mdl=True)
    m["model"].update({"hidden_dim": 128, "token_dim": 64, "num_heads": heads, "num_ns_tokens": 4,
                       "task_head_hidden_dim": 64, "pyramid_round_to": 8, **model})
    m["training"].update({"lr_warmup_steps": 0, "dense_optimizer": "adam", "lr_dense": 1e-3})
    spec.sequences["behavior"].min_len = 10
    cfg = app_config_from_mapping(m)
    attention_preflight(cfg, "cuda")
    torch.manual_seed(0)
    cpu_model = build_model(cfg, device="cpu", base_seed=1)
    gpu_model = build_model(cfg, device="cuda", base_seed=1)
    gpu_model.load_state_dict({k: v.cuda() for k, v in cpu_model.state_dict().items()})
    gpu_model.store.slab.copy_(cpu_model.store.slab)
    cpu_tr = Trainer(cfg, cpu_model, device=torch.device("cpu"))
    gpu_tr = Trainer(cfg, gpu_model, device=torch.device("cuda"))
    batch = SyntheticGenerator(cpu_model.encoder.batch_plan, spec).batch(64)
    out_c = cpu_tr.forward_backward(batch)
    out_g = gpu_tr.forward_backward(batch.to("cuda"))
    torch.cuda.synchronize()
    check_error_word(0)
    torch.testing.assert_close(out_g["logits"].cpu(), out_c["logits"].detach(), atol=6e-2, rtol=6e-2)
    gc, gg = cpu_tr.dense.grad, gpu_tr.dense.grad.cpu()
    scale = gc.norm().item()
    for name in cpu_tr.dense.names:
        o = cpu_tr.dense.offsets[name]
        n = cpu_tr.dense.params[name].numel()
        ref, got = gc[o:o + n], gg[o:o + n]
        err = (ref - got).norm().item()
        assert err <= 0.1 * ref.norm().item() + 2e-3 * scale, (name, err, ref.norm().item())


@pytest.mark.gpu
def test_evaluation_keeps_nothing_for_a_backward(monkeypatch):
    from mdl_b200.models import onetrans

    kept = []
    native = onetrans.window_attention_fwd

    def spy(*args, **kw):
        res = native(*args, **kw)
        kept.append(res[1] is not None)
        return res

    monkeypatch.setattr(onetrans, "window_attention_fwd", spy)
    m, spec = _config(attention_window=9, attention_sinks=2)
    cfg = app_config_from_mapping(m)
    torch.manual_seed(0)
    model = build_model(cfg, device="cuda", base_seed=1)
    trainer = Trainer(cfg, model, device=torch.device("cuda"))
    batch = SyntheticGenerator(model.encoder.batch_plan, spec).batch(16).to("cuda")
    with torch.no_grad():
        scores = model(batch)["logits"].float()
    assert kept == [False] * 3
    kept.clear()
    trained = trainer.forward_backward(batch)["logits"].float()
    assert kept == [True] * 3
    assert torch.equal(scores, trained.detach())
