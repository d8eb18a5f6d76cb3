"""Models inside ``fused_feed_forward()`` against their separate layers.

The fused block rounds once less a layer (z stays fp32), so hidden states and gradients differ by bf16 roundings:
z, and what follows from it, is off by 2^-9 in the 2-norm a layer, four roundings a layer at most.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

LAYER = 4 * 2.0 ** -8


def _dev():
    return torch.device("cuda", 0)


def _rel(got, want):
    return float((got.double() - want.double()).norm() / want.double().norm())


def _modernbert(width=200):
    from representax_b200.models.modernvbert.config import ModernVBERTTextConfig
    from representax_b200.models.modernvbert.model import ModernBertTextTower
    from representax_b200.ops import nn as N

    cfg = ModernVBERTTextConfig(vocab_size=64, hidden_size=128, intermediate_size=width, num_hidden_layers=2,
                                num_attention_heads=2, pad_token_id=0)
    tower = ModernBertTextTower(cfg, torch.Generator().manual_seed(0)).to(_dev())
    seg = N.Segments.from_lengths([33, 1, 300], _dev())
    return tower, seg, torch.cat([torch.arange(n) for n in seg.lengths()]).to(_dev())


def _omni_block(width):
    from representax_b200.models.qwen2_5_omni import OmniVisionConfig, OmniVisionTower

    cfg = OmniVisionConfig(depth=2, hidden_size=64, intermediate_size=width, num_heads=2, patch_size=4, out_hidden_size=64,
                           fullatt_block_indexes=(1,), window_size=16)
    tower = OmniVisionTower(cfg, torch.Generator().manual_seed(0)).to(_dev())
    with torch.no_grad():
        for block in tower.blocks:  # biases that matter
            block.gate_up_b.normal_(std=0.3)
            block.down_b.normal_(std=0.3)
    pixels = torch.randn(8 * 12, 3 * 2 * 4 * 4, generator=torch.Generator().manual_seed(1)).to(_dev())
    return lambda: tower(pixels, torch.tensor([[1, 8, 12]]), torch.bfloat16)


def test_modernbert_hidden_states():
    from representax_b200.ops import nn as N

    tower, seg, pos = _modernbert()
    emb = torch.randn(seg.total, 128, device=_dev(), generator=torch.Generator(device="cuda").manual_seed(2)).to(torch.bfloat16)
    with torch.no_grad():
        plain = tower(emb, seg, pos)
        with N.fused_feed_forward():
            fused = tower(emb, seg, pos)
        assert torch.equal(tower(emb, seg, pos), plain)  # and as before outside
    assert not torch.equal(plain, fused) and _rel(fused, plain) < 2 * LAYER


@pytest.mark.parametrize("width,same", [(88, False), (60, True), (3420, True)])
def test_omni_vision_tower(width, same):
    """Widths that are not multiples of 8 (3420 is the tower's own) keep the separate layers: the same bits."""

    from representax_b200.ops import nn as N

    run = _omni_block(width)
    with torch.no_grad():
        plain = run()
        with N.fused_feed_forward():
            fused = run()
    assert torch.equal(fused, plain) if same else (not torch.equal(fused, plain) and _rel(fused, plain) < 3 * LAYER)


def test_training_parameters():
    """Parameters as the training engine makes them: fp32 masters with a bf16 copy and an fp32 accumulator, into which the
    fused block adds like the separate layers."""

    from representax_b200.ops import nn as N
    from representax_b200.train.flat import FlatParameterStore

    g = torch.Generator(device="cuda").manual_seed(3)
    grads = {}
    for fused in (False, True):
        tower, seg, pos = _modernbert()
        store = FlatParameterStore(tower, device=_dev(), compute_dtype=torch.bfloat16)
        emb = torch.randn(seg.total, 128, device=_dev(), generator=g.manual_seed(3)).to(torch.bfloat16)
        dy = torch.randn(seg.total, 128, device=_dev(), generator=g).to(torch.bfloat16)
        with N.fused_feed_forward(fused):
            for _ in range(2):  # twice: the accumulators are added into
                tower(emb.clone().requires_grad_(), seg, pos).backward(dy)
        names = [n for n in store.params if n.rsplit(".", 1)[-1] in ("Wi", "mlp_Wo", "Wqkv")]
        assert len(names) == 6 and all(store.params[n].grad is None for n in names)
        grads[fused] = {n: store.params[n].main_grad.clone() for n in names}
    for n, want in grads[False].items():
        assert _rel(grads[True][n], want) < 2 * LAYER, n


def test_fp8_policy_keeps_the_separate_layers():
    from representax_b200.ops import nn as N
    from representax_b200.precision import FP8_MIXED_POLICY, precision_context

    tower, seg, pos = _modernbert()
    emb = torch.randn(seg.total, 128, device=_dev(), generator=torch.Generator(device="cuda").manual_seed(4)).to(torch.bfloat16)
    with torch.no_grad(), precision_context(FP8_MIXED_POLICY):
        plain = tower(emb, seg, pos)
        with N.fused_feed_forward():
            assert torch.equal(tower(emb, seg, pos), plain)
