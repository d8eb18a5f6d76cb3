"""4-bit weights in every model family: what can run in 4 bits does, what cannot is refused untouched."""

import pytest
import torch

from representax_b200.models import DenseEncoder, FP4Weight, quantize_linears_fp4
from representax_b200.models.text_batch import TokenBatch

VS = 252


def _tokens(high, rows=2, length=9):
    ids = torch.randint(3, high, (rows, length), generator=torch.Generator().manual_seed(7))
    return ids, torch.ones_like(ids)


def _text_config(**more):
    from representax_b200.models.qwen3 import Qwen3TextConfig

    return Qwen3TextConfig(vocab_size=256, hidden_size=64, intermediate_size=96, num_hidden_layers=2, num_attention_heads=4,
                           num_key_value_heads=2, head_dimension=16, pad_token_id=0, **more)


def _jina():
    from representax_b200.models import JinaV5TextEncoder

    ids, mask = _tokens(240)
    return JinaV5TextEncoder(_text_config()), TokenBatch(attention_mask=mask, input_ids=ids)


def _qwen3_vl():
    from representax_b200.models.qwen3_vl import Qwen3VLBatch, Qwen3VLConfig, Qwen3VLEncoder, Qwen3VLVisionConfig

    cfg = Qwen3VLConfig(text=_text_config(mrope_section=(2, 3, 3)),
                        vision=Qwen3VLVisionConfig(depth=2, hidden_size=32, intermediate_size=64, num_heads=2, patch_size=4,
                                                   out_hidden_size=64, num_position_embeddings=16,
                                                   deepstack_visual_indexes=(0,)), image_token_id=250)
    ids, mask = _tokens(240)
    ids[:, 2:6] = 250  # a 4 x 4 grid of patches, merged 2 x 2
    pixels = torch.randn(32, 3 * 2 * 4 * 4, generator=torch.Generator().manual_seed(1))
    return Qwen3VLEncoder(cfg, seed=0), Qwen3VLBatch(ids, mask, pixels, torch.tensor([[1, 4, 4]] * 2))


def _omni():
    from representax_b200.models.qwen2_5_omni import (OmniAudioConfig, OmniVisionConfig, Qwen2_5OmniBatch, Qwen2_5OmniConfig,
                                                      Qwen2_5OmniEncoder)

    cfg = Qwen2_5OmniConfig(text=_text_config(qkv_bias=True, qk_norm=False, mrope_section=(2, 3, 3)),
                            vision=OmniVisionConfig(depth=2, hidden_size=32, intermediate_size=60, num_heads=2, patch_size=4,
                                                    out_hidden_size=64, fullatt_block_indexes=(1,), window_size=16),
                            audio=OmniAudioConfig(num_mel_bins=16, encoder_layers=1, encoder_attention_heads=2,
                                                  encoder_ffn_dim=64, d_model=32, output_dim=64, max_source_positions=100,
                                                  n_window=5), image_token_id=250, audio_token_id=251)
    g = torch.Generator().manual_seed(2)
    seq = [5, 6, VS] + [250] * 24 + [VS, 7, 253] + [251] * 6 + [254, 8, 9]
    ids = torch.tensor([seq, seq])
    pixels = torch.randn(2 * 8 * 12, 3 * 2 * 4 * 4, generator=g)
    batch = Qwen2_5OmniBatch(ids, torch.ones_like(ids), pixels, torch.tensor([[1, 8, 12]] * 2),
                             torch.randn(16, 46, generator=g), torch.tensor([23, 23]))
    return Qwen2_5OmniEncoder(cfg, seed=0), batch


def _modernvbert():
    from representax_b200.models.modernvbert import ModernVBERTBatch, ModernVBERTEncoder
    from representax_b200.models.modernvbert.config import ModernVBERTConfig, ModernVBERTTextConfig, SigLIPVisionConfig

    cfg = ModernVBERTConfig(text=ModernVBERTTextConfig(vocab_size=128, hidden_size=64, intermediate_size=96, num_hidden_layers=2,
                                                       num_attention_heads=2, local_attention=4, pad_token_id=0),
                            vision=SigLIPVisionConfig(hidden_size=64, intermediate_size=128, num_hidden_layers=1,
                                                      num_attention_heads=2, image_size=32, patch_size=8),
                            image_token_id=100, pixel_shuffle_factor=2)
    ids, mask = _tokens(99, length=12)
    ids[:, 2:6] = 100
    pixels = torch.randn(2, 1, 3, 32, 32, generator=torch.Generator().manual_seed(3))
    return ModernVBERTEncoder(cfg, seed=0), ModernVBERTBatch(mask, ids, pixels)


def _clip():
    from representax_b200.models.clip import CLIPBatch, CLIPConfig, CLIPEncoder, CLIPTextConfig, CLIPVisionConfig

    cfg = CLIPConfig(text=CLIPTextConfig(vocab_size=100, hidden_size=64, intermediate_size=128, num_hidden_layers=1,
                                         num_attention_heads=2, max_position_embeddings=20),
                     vision=CLIPVisionConfig(hidden_size=64, intermediate_size=128, num_hidden_layers=1, num_attention_heads=2,
                                             image_size=32, patch_size=8), projection_dimension=32)
    ids, mask = _tokens(90, rows=3)
    both = torch.tensor([True, True, True])
    pixels = torch.randn(3, 3, 32, 32, generator=torch.Generator().manual_seed(4))
    return CLIPEncoder(cfg, seed=0), CLIPBatch(ids, mask, both, pixels, both)


FAMILIES = {"jina": (_jina, 8), "qwen3_vl": (_qwen3_vl, 8 + 2 * 4 + 2 * 2), "omni": (_omni, 8 + 2 * 4 + 2 + 4 + 1),
            "modernvbert": (_modernvbert, 8 + 4), "clip": (_clip, 4 + 4 + 2)}


@pytest.mark.parametrize("fmt", ["mxfp4", "nvfp4"])
@pytest.mark.parametrize("family", FAMILIES)
def test_family_embeds_with_4bit_weights(family, fmt, monkeypatch):
    """Every swapped weight is reached as a 4-bit operand, and nothing else of the model was swapped."""

    build, count = FAMILIES[family]
    model, batch = build()
    before = model.encode(batch).detach()
    quantize_linears_fp4(model, fmt=fmt)
    weights = [m for m in model.modules() if isinstance(m, FP4Weight)]
    assert len(weights) == count
    reached = set()
    operand = FP4Weight.operand.fget

    def spy(self):
        reached.add(id(self))
        return operand(self)

    monkeypatch.setattr(FP4Weight, "operand", property(spy))
    after = model.encode(batch)
    assert after.isfinite().all() and not torch.equal(after, before)
    assert reached == {id(w) for w in weights}
    assert not any(p.requires_grad for p in model.parameters())


def _bert():
    from representax_b200.models.bert import BertConfig, BertEncoder

    ids, mask = _tokens(90)
    return BertEncoder(BertConfig(vocab_size=100, hidden_size=64, intermediate_size=128, num_hidden_layers=1,
                                  num_attention_heads=2, max_position_embeddings=32)), TokenBatch(attention_mask=mask, input_ids=ids)


def _mpnet():
    from representax_b200.models.mpnet import MPNetConfig, MPNetEncoder

    ids, mask = _tokens(90)
    return MPNetEncoder(MPNetConfig(vocab_size=100, hidden_size=64, intermediate_size=128, num_hidden_layers=1,
                                    num_attention_heads=2, max_position_embeddings=32)), TokenBatch(attention_mask=mask, input_ids=ids)


def _dense():
    return DenseEncoder(16, 8), torch.randn(3, 16, generator=torch.Generator().manual_seed(5))


def _state(model):
    return ({n: (id(p), p.requires_grad, p.detach().clone()) for n, p in model.named_parameters()},
            [n for n, _ in model.named_modules()])


def _untouched(model, state):
    params, modules = state
    assert [n for n, _ in model.named_modules()] == modules
    assert {n: (id(p), p.requires_grad) for n, p in model.named_parameters()} == {n: v[:2] for n, v in params.items()}
    assert all(torch.equal(p, params[n][2]) for n, p in model.named_parameters())


@pytest.mark.parametrize("build", [_bert, _mpnet, _dense])
def test_models_without_packed_linears_are_refused_untouched(build):
    model, batch = build()
    state, want = _state(model), model.encode(batch)
    with pytest.raises(ValueError, match="packed rows"):
        quantize_linears_fp4(model)
    _untouched(model, state)
    assert torch.equal(model.encode(batch), want)


def test_other_modules_beside_a_tower_keep_their_weights():
    """A classifier's head around a tower, and the factors of a LoRA weight inside one."""

    from representax_b200.models import PairClassifier
    from representax_b200.models.adapters import QuantizedLoRAWeight, apply_quantized_lora

    model, batch = _jina()
    head = PairClassifier(model, 3)
    kept = head.classifier_weight.detach().clone()
    quantize_linears_fp4(head)
    assert isinstance(head.classifier_weight, torch.nn.Parameter) and torch.equal(head.classifier_weight, kept)
    assert head.encode(batch).isfinite().all()

    model, batch = _jina()
    apply_quantized_lora(model, rank=4, alpha=8.0, target_pattern=r"o_proj$")
    lora = [m for m in model.modules() if isinstance(m, QuantizedLoRAWeight)]
    factors = [(m.lora_a.detach().clone(), m.merged_weight().detach()) for m in lora]
    quantize_linears_fp4(model)
    assert len(lora) == 2 and sum(isinstance(m, FP4Weight) for m in model.modules()) == 6
    for m, (a, merged) in zip(lora, factors):
        assert torch.equal(m.lora_a, a) and torch.equal(m.merged_weight(), merged)
    assert model.encode(batch).isfinite().all()


def test_a_refused_weight_leaves_the_model_as_it_was():
    """The last weight cannot be quantised (64-bit): none is swapped and nothing is frozen."""

    model, _ = _jina()
    layer = model.text.layers[-1] if hasattr(model, "text") else model.tower.layers[-1]
    layer.down = torch.nn.Parameter(layer.down.detach().double())
    state = _state(model)
    with pytest.raises(TypeError, match="float32"):
        quantize_linears_fp4(model)
    _untouched(model, state)
    for kwargs in ({"fmt": "int4"}, {"target_pattern": "nothing"}):
        with pytest.raises(ValueError, match="fmt|target_pattern"):
            quantize_linears_fp4(model, **kwargs)
        _untouched(model, state)
