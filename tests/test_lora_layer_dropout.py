"""``ManualLoRALayer`` and the dropout that it finds when it is called, by parts on the CPU."""

import pytest
import torch
import torch.nn as nn

from grpo_mi355x.core import lora
from grpo_mi355x.kernels import lora_forward
from grpo_mi355x.kernels.dropout import CounterDropout


class Base(nn.Module):
    in_features, out_features = 16, 8

    def __init__(self):
        super().__init__()
        self.weight = nn.Parameter(torch.randn(8, 16), requires_grad=False)

    def forward(self, x):
        return x @ self.weight.t()


def layer_of(**kw):
    torch.manual_seed(1)
    layer = lora.ManualLoRALayer(Base(), rank=4, alpha=8, **kw)
    nn.init.normal_(layer.lora_B.weight)
    return layer


@pytest.mark.parametrize("use_triton", [True, False])
@pytest.mark.parametrize("other", [nn.Identity, lambda: nn.Dropout(0.5).eval()])
def test_dropout_replaced_after_construction(use_triton, other):
    layer = layer_of(dropout=0.5, counter_dropout=True, use_triton=use_triton)
    layer.lora_dropout = other()
    x = torch.randn(2, 3, 16)
    want = x @ layer.base_layer.weight.t() + 2.0 * (x @ layer.lora_A.weight.t()
                                                    ) @ layer.lora_B.weight.t()
    assert torch.allclose(layer(x), want, atol=1e-5)


@pytest.mark.parametrize("counter", [True, False])
def test_one_draw_for_a_call(monkeypatch, counter):
    """Fused and by parts get the same draw, also where the dropout was put in afterwards."""
    layer = layer_of(dropout=0.5, counter_dropout=counter)
    layer.lora_dropout = CounterDropout(0.25)
    fused, parts, draws = [], [], []

    def refuse(x, dropout_rng=None, **kw):
        fused.append(dropout_rng)
        raise ValueError("not here")

    def drop(x, p, rng):
        parts.append(rng)
        return x

    draw = CounterDropout.draw
    monkeypatch.setattr(CounterDropout, "draw",
                        staticmethod(lambda d: draws.append(draw(d)) or draws[-1]))
    monkeypatch.setattr(lora, "lora_fused_forward", refuse)
    monkeypatch.setattr("grpo_mi355x.kernels.dropout.counter_dropout", drop)
    layer(torch.randn(2, 3, 16))
    assert len(draws) == 1 and fused == draws and parts == draws
    layer.eval()
    layer(torch.randn(2, 3, 16))
    assert len(draws) == 1 and fused[1] is None and len(parts) == 1


@pytest.mark.parametrize("other", [nn.AlphaDropout, nn.Dropout1d, nn.Dropout2d, nn.Dropout3d,
                                   nn.FeatureAlphaDropout])
def test_dropout_of_another_rule_is_refused(other):
    """A draw makes nn.Dropout's rule, element by element; a module with another rule has to
    raise rather than run that one. In eval mode none drops anything."""
    rng, cpu = torch.tensor([1, 2]), torch.device("cpu")
    with pytest.raises(ValueError, match="nn.Dropout or CounterDropout"):
        lora_forward._dropout_of(other(0.25), rng, cpu)
    assert lora_forward._dropout_of(other(0.25).eval(), rng, cpu) is None
    assert lora_forward._dropout_of(other(0.0), rng, cpu) is None
    for fine in (nn.Dropout(0.25), CounterDropout(0.25)):
        assert lora_forward._dropout_of(fine, rng, cpu) == (0.25, rng)
