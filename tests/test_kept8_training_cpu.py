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


def test_without_recompute_and_back_to_16_bits():
    eng = _engine(8, recompute=False)
    batch, _ = tiny_batch(eng.model, seed=7)
    loss, _ = _grads(eng, batch)
    assert loss == loss
    eng.set_activation_checkpointing(True)
    assert eng.checkpoint_bits == 16 and not any(b.kept8 for b in eng.model.caption_encoder.blocks)
    base = _engine(16, stash=True)
    eng.stash_in_grads = True
    a, b = _grads(eng, batch), _grads(base, batch)
    assert a[0] == b[0] and all(torch.equal(a[1][n], b[1][n]) for n in a[1])


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
