"""That a model which is asked for it checkpoints its blocks in 8 bits: by what autograd saves of them."""

from __future__ import annotations

import pytest
import torch

from moss_offload import dit

from gpu_util import requires_gpu
from test_gpu_norm import _randn

pytestmark = requires_gpu

DEV = torch.device("cuda", 0)


def _run(keep8, packed):
    """(the blocks' inputs, what autograd saved in the forward pass, the loss, the gradients)."""

    torch.manual_seed(0)
    model = dit.MOSSImageTransformer(dim=64, ffn_dim=128, num_heads=4, num_layers=3, text_dim=32, freq_dim=16, latent_channels=8,
                                     gradient_checkpointing=True, checkpoint_keep8=keep8)
    dit.init_weights(model)
    dit.inject_lora(model, rank=4, alpha=4.0)
    model = model.to(DEV).to(torch.bfloat16).train()
    inputs, saved = [], []
    hooks = [layer.register_forward_pre_hook(lambda module, args: inputs.append(args[0])) for layer in model.layers]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (saved.append(t), t)[1], lambda t: t):
        if packed:
            outs = model.forward_packed([_randn(8, 4, 4).bfloat16(), _randn(8, 2, 6, seed=1).bfloat16()], torch.tensor([500.0, 100.0], device=DEV),
                                        [_randn(6, 32, seed=2).bfloat16(), _randn(9, 32, seed=3).bfloat16()])
        else:
            outs = [model(_randn(1, 8, 4, 4).bfloat16(), torch.tensor([500.0], device=DEV), _randn(1, 6, 32, seed=2).bfloat16())]
    first = inputs[:]
    for hook in hooks:
        hook.remove()
    loss = sum(o.float().square().mean() for o in outs)
    loss.backward()
    return first, saved, loss.detach(), [p.grad for p in model.parameters() if p.requires_grad]


@pytest.mark.parametrize("packed", [False, True])
def test_a_model_saves_its_blocks_inputs_in_8_bits(packed) -> None:
    inputs, saved, loss, grads = _run(True, packed)
    assert len(inputs) == 3 and [t.shape for t in saved if t.dtype == torch.int8] == [t.shape for t in inputs]
    assert sum(t.dtype == torch.uint8 for t in saved) == 3
    # none of them is saved as it is; the last block's output, which the head reads, is no block's input
    places = {t.data_ptr() for t in inputs}
    assert not any(t.dtype == torch.bfloat16 and t.data_ptr() in places and t.shape == inputs[0].shape for t in saved)
    _, saved, exact, plain = _run(False, packed)
    assert not any(t.dtype == torch.int8 for t in saved)
    assert torch.equal(loss, exact)  # the forward pass is the exact input's
    # the gradients are taken at what 8 bits keep, so not all of them are the same
    assert any(not torch.equal(g, p) for g, p in zip(grads, plain))
