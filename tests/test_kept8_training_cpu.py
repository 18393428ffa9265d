"""A training step with activations kept in 8 bits (CPU): options, gradients, what is kept."""
import pytest
import torch

from tiny import TINY_ARCH, tiny_batch


def _engine(bits, stash=False, recompute=True):
    from pan2_b200.training.engine import OptimConfig, TrainEngine
    eng = TrainEngine(dict(TINY_ARCH), torch.device("cpu"), seed=11, optim=OptimConfig(lr=1e-2), offload="off")
    eng.set_activation_checkpointing(recompute, bits=bits)
    eng.stash_in_grads = stash
    return eng


def _grads(eng, batch):
    loss = eng.forward_backward(batch)
    return float(loss), {s.name: u.slot_full(u.full_grad, s).float().clone() for u in eng.sharded.units for s in u.slots}


def test_step_in_8_bits_follows_the_exact_step():
    eng = _engine(16)
    batch, _ = tiny_batch(eng.model, seed=7)
    loss, exact = _grads(eng, batch)
    loss8, kept = _grads(_engine(8), batch)
    # the CPU forward is the same up to where the fused norms round
    assert abs(loss8 - loss) <= 1e-3 * abs(loss)
    for name, g in exact.items():
        if float(g.norm()) == 0:
            continue
        cos = float(torch.nn.functional.cosine_similarity(g.flatten(), kept[name].flatten(), dim=0))
        assert cos > 0.98, (name, cos)


def test_checkpoints_in_gradient_buffers_stay_exact(monkeypatch):
    """Only checkpoints that take memory of their own go to 8 bits (idle gradient buffers hold bf16 ones,
    so a stand-in takes their place for the CPU's fp32)."""
    from pan2_b200.training import engine as E
    seen = []
    keep = E.keep8
    monkeypatch.setattr(E, "keep8", lambda x: seen.append(x.shape) or keep(x))
    eng = _engine(8)
    batch, _ = tiny_batch(eng.model, seed=7)
    eng.forward_backward(batch)
    assert len(seen) == TINY_ARCH["num_layers"]
    seen.clear()
    monkeypatch.setattr(eng, "stash_checkpoint", lambda idx, x, st: (x.clone(), st.clone()) if idx > 0 else None)
    eng.forward_backward(batch)
    assert len(seen) == 1


def test_without_recompute_and_back_to_16_bits(monkeypatch):
    from pan2_b200.models import caption_encoder as C
    from pan2_b200.models import transformer as T
    from pan2_b200.training import engine as E
    calls = []
    for module, name in ((E, "keep8"), (C, "kept8_linear"), (C, "kept8_swiglu_ffn"), (C, "fused_rms_norm"),
                         (T, "kept8_linear"), (T, "fused_rms_norm")):
        fn = getattr(module, name)
        monkeypatch.setattr(module, name, lambda *a, _fn=fn, _n=name, **k: calls.append(_n) or _fn(*a, **k))
    eng = _engine(8, recompute=False)
    batch, _ = tiny_batch(eng.model, seed=7)
    loss, _ = _grads(eng, batch)
    assert loss == loss and "kept8_swiglu_ffn" in calls and "keep8" not in calls
    calls.clear()
    eng.set_activation_checkpointing(True)
    _grads(eng, batch)
    assert eng.checkpoint_bits == 16 and not calls  # the path of before, untouched


def test_dense_caption_path_matches_the_eager_one():
    from tiny import tiny_model
    m = tiny_model().eval()
    text, mask = torch.randn(2, 12, m.text_embed_dim), torch.ones(2, 12)
    mask[1, 5:] = 0
    with torch.no_grad():
        eager = m.encode_text(text, mask)
        m.set_kept8(True)
        kept = m.encode_text(text, mask)
    assert torch.allclose(eager, kept, rtol=1e-4, atol=1e-5)


def test_options():
    from pan2_b200.config.training import parse_training_config
    assert parse_training_config([]).activation_checkpoint_bits == 16
    assert parse_training_config(["--activation_checkpoint_bits", "8"]).activation_checkpoint_bits == 8
    with pytest.raises(SystemExit):
        parse_training_config(["--activation_checkpoint_bits", "4"])
    cfg = parse_training_config([])
    cfg.activation_checkpoint_bits = 4
    with pytest.raises(ValueError, match="16 or 8"):
        cfg.check()
    with pytest.raises(ValueError, match="16 or 8"):
        _engine(4)


def test_kept_attention_leaves_the_checkpoints_exact(monkeypatch):
    """The kept attention output belongs to the exact input: a recompute from 8 bits would join it to other q, k, v."""
    from pan2_b200.training import engine as E
    calls = []
    monkeypatch.setattr(E, "keep8", lambda x, _keep=E.keep8: calls.append(x.shape) or _keep(x))
    eng = _engine(16)
    batch, _ = tiny_batch(eng.model, seed=7)
    _, exact = _grads(eng, batch)
    eng = _engine(8)
    eng.set_activation_checkpointing(True, keep_attention=True, bits=8)
    _, kept = _grads(eng, batch)
    assert not calls and eng.model.kept8
    for name, g in exact.items():
        if name.startswith("blocks.") and float(g.norm()) > 0:
            # the joint blocks see the fused norms' rounding in the captions, nothing else
            assert float((kept[name] - g).norm() / g.norm()) < 1e-3, name
