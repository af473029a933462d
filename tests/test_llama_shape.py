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
