"""rotary.rotary_cos_sin and RotaryScaling on the host: the formulas, and the existing tables as their plain case."""
import math

import pytest
import torch

from sparseforge_amd.llama import rotary_tables
from sparseforge_amd.rotary import RotaryScaling, rotary_cos_sin


def _angles(f, positions):
    return torch.outer(torch.arange(positions, dtype=torch.float64), torch.tensor(f, dtype=torch.float64))


def test_plain_tables_are_the_models():
    """The model's tables take the angle in float32: its rounding is at most 2^-23 of the angle (the frequency's and
    the product's), below 64 here."""
    cos, sin = rotary_cos_sin(64, 32, device="cpu")
    c, s = rotary_tables(64, 32, 10000.0, "cpu")
    bar = 64 * 2.0 ** -22
    assert (cos - c[:, :16]).abs().max() <= bar and (sin - s[:, :16]).abs().max() <= bar


@pytest.mark.parametrize("kind", ["linear", "ntk", "yarn"])
def test_scalings(kind):
    r, theta, F, length = 40, 10000.0, 8.0, 100
    f = [theta ** (-2 * i / r) for i in range(r // 2)]
    m = 1.0
    if kind == "linear":
        f = [x / F for x in f]
    elif kind == "ntk":
        f = [(theta * F ** (r / (r - 2))) ** (-2 * i / r) for i in range(r // 2)]
        assert math.isclose(f[-1], theta ** (-(r - 2) / r) / F)  # the slowest pair interpolates
    else:
        g = [min(max((length * x / (2 * math.pi) - 1) / 31, 0), 1) for x in f]
        f = [x * (w + (1 - w) / F) for x, w in zip(f, g)]
        m = 0.1 * math.log(F) + 1
    cos, sin = rotary_cos_sin(1000, r, theta, RotaryScaling(kind, F, length), device="cpu")
    angle = _angles(f, 1000)
    # float32 storage: half an ulp of at most m; the angles agree to 2^-50 of themselves
    assert (cos.double() - m * angle.cos()).abs().max() <= m * 2.0 ** -24
    assert (sin.double() - m * angle.sin()).abs().max() <= m * 2.0 ** -24


def test_refusals():
    with pytest.raises(ValueError):
        RotaryScaling("cubic", 2.0)
    with pytest.raises(ValueError):
        RotaryScaling("linear", 0.5)
    with pytest.raises(ValueError):
        RotaryScaling("linear", math.inf)
    with pytest.raises(ValueError):
        RotaryScaling("yarn", 2.0)
    with pytest.raises(ValueError):
        RotaryScaling("yarn", 2.0, 100, beta_fast=1.0, beta_slow=1.0)
    with pytest.raises(ValueError):
        rotary_cos_sin(4, 7, device="cpu")
    with pytest.raises(ValueError):
        rotary_cos_sin(0, 8, device="cpu")
    with pytest.raises(ValueError):
        rotary_cos_sin(4, 2, scaling=RotaryScaling("ntk", 2.0), device="cpu")
