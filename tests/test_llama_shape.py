"""LlamaShape's fields, and the rotary tables that LlamaDecoder takes from them, on the host."""
import torch

from sparseforge_amd.llama import LlamaDecoder, LlamaShape


def test_fields_by_position():
    """The order that code which names no field relies on: later fields come last."""
    s = LlamaShape(100, 32, 64, 1, 2, 1e-6, 500.0, True)
    assert s.output_hidden_state is True and s.rope_theta == 500.0 and s.rope_scaling is None
    decoder = LlamaDecoder(s, None)
    cos, sin = decoder._tables(7, torch.device("cpu"))
    assert cos.shape == sin.shape == (7, 16)


def test_tables_follow_the_configuration():
    """A trained model whose context is stretched, or whose theta is changed, turns by the new angles at lengths that it
    has seen before too, and by the old ones again when they are set back."""
    from sparseforge_amd.rotary import RotaryScaling, rotary_cos_sin

    m = LlamaDecoder(LlamaShape(100, 32, 64, 1, 2), None)
    cpu = torch.device("cpu")
    plain = m._tables(9, cpu)
    m.config.rope_scaling = RotaryScaling("linear", 4.0)
    c, s = rotary_cos_sin(9, 16, 10000.0, m.config.rope_scaling, "cpu")
    assert torch.equal(m._tables(9, cpu)[0], torch.cat([c, c], -1))
    assert torch.equal(m._tables(9, cpu)[1], torch.cat([s, s], -1))
    m.config.rope_scaling = None
    assert all(torch.equal(a, b) for a, b in zip(m._tables(9, cpu), plain))
    m.config.rope_theta = 500.0
    assert not torch.equal(m._tables(9, cpu)[0], plain[0])
    assert torch.equal(m._tables(9, cpu)[0], LlamaDecoder(LlamaShape(100, 32, 64, 1, 2, 1e-5, 500.0), None)._tables(9, cpu)[0])
