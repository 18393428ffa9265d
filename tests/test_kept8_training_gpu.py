"""A training step with activations kept in 8 bits on a B200."""
import pytest
import torch

from tiny import TINY_ARCH, tiny_batch

pytestmark = pytest.mark.gpu

ARCH = dict(TINY_ARCH, hidden_size=512, num_attention_heads=4, rope_axes_dim=(32, 48, 48))


def _step(bits):
    from pan2_b200.data.synthetic import batch_to_device
    from pan2_b200.training.engine import OptimConfig, TrainEngine
    eng = TrainEngine(ARCH, torch.device("cuda"), seed=5, optim=OptimConfig(lr=1e-3), offload="off")
    eng.set_activation_checkpointing(True, bits=bits)
    eng.stash_in_grads = False
    batch, _ = tiny_batch(eng.model)
    b = batch_to_device(batch, "cuda")
    for k in ("hidden_states", "text_states", "target"):
        b[k] = b[k].to(torch.bfloat16)
    loss = float(eng.forward_backward(b))
    grads = {s.name: u.slot_full(u.full_grad, s).float().clone() for u in eng.sharded.units for s in u.slots}
    eng.grad_norm()
    eng.optimizer_step()
    again = float(eng.forward_backward(b))
    return loss, grads, again


def test_step_in_8_bits_follows_the_exact_step():
    from pan2_b200.ops._ext import ext
    loss, exact, _ = _step(16)
    loss8, kept, again = _step(8)
    torch.cuda.synchronize()
    assert ext().error_flag(True) == 0
    assert abs(loss8 - loss) <= 1e-2 * abs(loss) and again == again
    for name, g in exact.items():
        if float(g.norm()) == 0:
            continue
        cos = float(torch.nn.functional.cosine_similarity(g.flatten(), kept[name].flatten(), dim=0))
        assert cos > 0.97, (name, cos)


def test_caption_encoder_holds_less_memory():
    from pan2_b200.models.caption_encoder import CaptionEncoder
    torch.manual_seed(0)
    enc = CaptionEncoder(512, 4, num_layers=2).cuda().to(torch.bfloat16)
    lens = [700, 0, 1300, 48]
    cu = torch.tensor([0, 700, 700, 2000, 2048], dtype=torch.int32, device="cuda")
    held, out, grads = {}, {}, {}
    for on in (False, True):
        enc.set_kept8(on)
        x = torch.randn(2048, 512, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).bfloat16()
        x.requires_grad_(True)
        for p in enc.parameters():
            p.grad = None
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = enc(x, cu_seqlens=cu, lens=lens, max_seqlen=1300)
        held[on] = torch.cuda.memory_allocated() - before
        y.float().square().sum().backward()
        out[on], grads[on] = y.detach().float(), torch.cat([p.grad.float().flatten() for p in enc.parameters()])
    assert float((out[True] - out[False]).norm() / out[False].norm()) < 2e-2  # norms round once instead of twice
    assert float(torch.nn.functional.cosine_similarity(grads[True], grads[False], dim=0)) > 0.99
    assert held[True] < 0.5 * held[False], held


def test_kept_attention_with_8_bits_follows_the_exact_step(monkeypatch):
    """Attention outputs kept by the forward are those of the exact input, so the blocks' checkpoints stay exact."""
    from pan2_b200.data.synthetic import batch_to_device
    from pan2_b200.training import engine as E
    calls, grads = [], {}
    monkeypatch.setattr(E, "keep8", lambda x, _keep=E.keep8: calls.append(x.shape) or _keep(x))
    for bits in (16, 8):
        eng = E.TrainEngine(ARCH, torch.device("cuda"), seed=5, optim=E.OptimConfig(lr=1e-3), offload="off")
        eng.set_activation_checkpointing(True, keep_attention=True, bits=bits)
        eng.stash_in_grads = False
        batch, _ = tiny_batch(eng.model)
        b = batch_to_device(batch, "cuda")
        for k in ("hidden_states", "text_states", "target"):
            b[k] = b[k].to(torch.bfloat16)
        eng.forward_backward(b)
        grads[bits] = {s.name: u.slot_full(u.full_grad, s).float().clone() for u in eng.sharded.units for s in u.slots}
        del eng
    assert not calls
    for name, g in grads[16].items():
        if float(g.norm()) > 0:
            cos = float(torch.nn.functional.cosine_similarity(g.flatten(), grads[8][name].flatten(), dim=0))
            assert cos > 0.99, (name, cos)
