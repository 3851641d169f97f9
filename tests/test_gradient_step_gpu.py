"""The gradient operators used together: a transformers model trained with the fused capture
attention, its gradients clipped by their norm, QK-Clip on the maxima the same forwards recorded,
and the zeroth-order optimizer beside it."""

from __future__ import annotations

import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


def _tiny_llama(dtype, device, kv_heads=2, attn="sdpa"):
    from transformers import LlamaConfig, LlamaForCausalLM

    torch.manual_seed(0)
    cfg = LlamaConfig(hidden_size=256, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=kv_heads,
                      intermediate_size=688, vocab_size=1024, attn_implementation=attn, initializer_range=0.02)
    return LlamaForCausalLM(cfg).to(dtype=dtype, device=device)


def _gradients(model, ids, mask):
    model.zero_grad(set_to_none=True)
    # a padding query has no loss, for its attention is not defined: position t predicts the token
    # at t + 1, so the first token behind left padding has none either
    asked = torch.cat([mask[:, :1], mask[:, :-1]], dim=1) * mask
    labels = ids.masked_fill(asked == 0, -100)
    model(input_ids=ids, attention_mask=mask, labels=labels).loss.backward()
    return {n: p.grad.double() for n, p in model.named_parameters()}


@pytest.mark.parametrize("padding", ["none", "left", "right"])
@pytest.mark.parametrize("kv_heads", [4, 1])
def test_fused_training_gradients(device, padding, kv_heads):
    """Gradients of a bf16 model with the fused attention against the same weights in fp32 with
    eager attention (in fp64 the eager softmax, which is taken in fp32, turns the mask's lowest value
    into -inf and left-padded rows into NaN): no further off than 1.5 times the same model with SDPA is (both round the
    same states to bf16; only the attention differs), plus a bf16 half step of the gradient."""
    from muzo_clip_b200 import use_qk_capture_attention

    model = _tiny_llama(torch.bfloat16, device, kv_heads)
    sdpa = copy.deepcopy(model)
    exact = _tiny_llama(torch.float32, device, kv_heads, attn="eager")
    exact.load_state_dict({k: v.float() for k, v in model.state_dict().items()})
    ids = torch.randint(0, 1024, (3, 150), generator=torch.Generator().manual_seed(2)).to(device)
    mask = torch.ones_like(ids)
    if padding == "left":
        mask[1, :40] = 0
    elif padding == "right":
        mask[1, 90:] = 0
    assert use_qk_capture_attention(model, fused=True) == "muzo_qk_fused"
    got = _gradients(model, ids, mask)
    want = _gradients(sdpa, ids, mask)
    ref = _gradients(exact, ids, mask)
    for name in ref:
        size = ref[name].norm()
        mine, theirs = float((got[name] - ref[name]).norm() / size), float((want[name] - ref[name]).norm() / size)
        assert mine <= 1.5 * theirs + 2.0 ** -8, (name, mine, theirs)


def test_the_fused_kernel_runs_and_falls_back(device, monkeypatch):
    """Which calls reach attention_max: bf16 without a mask, with padding; not fp32, nor dropout."""
    from muzo_clip_b200 import _qk, use_qk_capture_attention

    calls = []
    real = _qk.attention_max
    monkeypatch.setattr(_qk, "attention_max", lambda *a, **k: calls.append(k.get("record")) or real(*a, **k))
    ids = torch.randint(0, 1024, (2, 40), generator=torch.Generator().manual_seed(3)).to(device)
    model = _tiny_llama(torch.bfloat16, device)
    use_qk_capture_attention(model, fused=True)
    model.train()
    model(input_ids=ids, labels=ids).loss.backward()
    assert calls == [False, False]
    mask = torch.ones_like(ids)
    mask[0, :9] = 0
    model(input_ids=ids, attention_mask=mask, labels=ids).loss.backward()
    assert len(calls) == 4
    model.config.attention_dropout = 0.1
    for layer in model.model.layers:
        layer.self_attn.attention_dropout = 0.1
    model(input_ids=ids, labels=ids).loss.backward()
    assert len(calls) == 4
    single = _tiny_llama(torch.float32, device)
    use_qk_capture_attention(single, fused=True)
    single(input_ids=ids, labels=ids).loss.backward()
    assert len(calls) == 4


@pytest.mark.parametrize("scaling", [-0.5, 0.0])
def test_capture_with_a_scale_the_kernel_refuses(device, monkeypatch, scaling):
    """MUZO_FUSED_ATTENTION=1, a scale that is not positive: the capture runs on SDPA, as without it."""
    from muzo_clip_b200 import _qk, attention_max

    class Recorder:
        kept = []

        def module_name(self, module):
            return "layer"

        def record_qk(self, module, query, key, scale, causal, mask):
            self.kept.append((scale, causal))

        def record_max(self, name, smax, valid):
            raise AssertionError("the fused kernel took a scale that it refuses")

    monkeypatch.setenv("MUZO_FUSED_ATTENTION", "1")
    gen = torch.Generator().manual_seed(11)
    q, k, v = (torch.randn((2, 4, 33, 64), generator=gen).to(device, torch.bfloat16) for _ in range(3))
    module = torch.nn.Module()
    module.is_causal = True
    recorder = Recorder()
    token = _qk._ACTIVE.set(recorder)
    try:
        with torch.no_grad():
            out, _ = _qk._probe_attention(module, q, k, v, None, scaling=scaling)
    finally:
        _qk._ACTIVE.reset(token)
    ref = torch.nn.functional.scaled_dot_product_attention(q, k, v, is_causal=True, scale=scaling).transpose(1, 2)
    assert torch.equal(out, ref) and recorder.kept == [(scaling, True)]
    with pytest.raises(ValueError, match="scaling must be positive"):
        attention_max(q, k, v, scaling)


def test_step_with_clipping_and_qk_clip(device):
    """One gradient step as a user writes it: forward under capture, backward, clip, update; then
    QK-Clip on the captured maxima, which are the eager ones; the zeroth-order projection still runs
    on the same model."""
    from muzo_clip_b200 import MuZOClipOptimizer, clip_grad_norm_, use_qk_capture_attention

    model = _tiny_llama(torch.bfloat16, device)
    with torch.no_grad():
        model.model.layers[0].self_attn.q_proj.weight.mul_(40.0)
    twin = copy.deepcopy(model)
    use_qk_capture_attention(model, fused=True)
    opt = MuZOClipOptimizer(model, enable_qk_clip=True, qk_clip_tau=5.0, restore_exact=True, seed=3)
    ids = torch.randint(0, 1024, (3, 100), generator=torch.Generator().manual_seed(5)).to(device)
    captured = {}
    with opt.qk_clip.capture():
        loss = model(input_ids=ids, labels=ids).loss
    loss.backward()
    captured = {k: v.cpu() for k, v in opt.qk_clip._captured_smax.items()}
    assert len(captured) == 2
    before = torch.linalg.vector_norm(torch.stack([p.grad.double().norm() for p in model.parameters()]))
    norm = clip_grad_norm_(model.parameters(), 0.5 * float(before))
    after = torch.linalg.vector_norm(torch.stack([p.grad.double().norm() for p in model.parameters()]))
    assert abs(float(norm) / float(before) - 1) <= 1e-6 and abs(float(after) / float(before) - 0.5) <= 2.0 ** -8
    # the captured maxima: eager logits of the twin
    probe = MuZOClipOptimizer(twin, enable_qk_clip=True, qk_clip_tau=5.0, seed=3)
    with probe.qk_clip.force_eager_attention(True), probe.qk_clip.capture(), torch.no_grad():
        twin(input_ids=ids)
    for name, want in probe.qk_clip._captured_smax.items():
        want = want.cpu()
        # the second layer's states pass through the first one's attention, computed by another kernel
        ulps = 1 if "layers.0" in name else 4
        step = torch.pow(2.0, torch.floor(torch.log2(want.abs().clamp_min(2.0 ** -126))) - 7)
        assert bool(((captured[name] - want).abs() <= ulps * step).all()), name
    with torch.no_grad():
        for p in model.parameters():
            p.sub_(p.grad, alpha=1e-3)
    stats = opt.qk_clip.apply()
    assert stats.enabled and stats.exact_logits and stats.qk_clip_count > 0
    model.zero_grad(set_to_none=True)

    def closure():
        with torch.no_grad():
            return model(input_ids=ids, labels=ids).loss

    assert not opt.estimate_projection(closure)["skipped"]
