"""What a DraftSession does to the decoder that it runs (no GPU needed)."""

import torch

from adapterslotsplusplus_b200.draft import DraftDecoder, DraftSession


def test_a_running_session_leaves_the_models_head_alone():
    """Others use the same decoder meanwhile: its LM head stays where it is, and
    a plain forward in the middle of a step gives logits."""
    model = DraftDecoder(layers=2, hidden=32, heads=2, inter=32, vocab=7, device="cpu", dtype=torch.float32)
    head = model.lm_head
    session = DraftSession.__new__(DraftSession)
    session.model = model
    x, seen = torch.randn(3, 32), []

    def attention(layer, q, k, v):
        seen.append((model.lm_head, model.forward(x, 3).shape))
        return v

    h = session._hidden(x, attention, {})
    assert h.shape == (3, 32)
    assert len(seen) == 2 and all(at is head and tuple(shape) == (3, 7) for at, shape in seen)
    assert model.lm_head is head
    assert torch.equal(torch.nn.functional.linear(h, head), model.forward(x, 0, attention=lambda layer, q, k, v: v))
