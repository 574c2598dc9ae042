"""CPU: the frequencies of rope_cos_sin, every dim, against the published YaRN rule in 64 bits.

At position 1 the table holds gain * cos(f) and gain * sin(f) in float32, f <= 1: their angle gives f
within 2^-23 of itself or of 1."""
import math

import pytest
import torch

from glm53_flash_dual_dgx_spark_b200 import glm53_nvfp4_runtime as rt


def frequencies(table):
    half = table.shape[1] // 2
    row = table[1].double()
    return torch.atan2(row[half:], row[:half]), torch.hypot(row[half:], row[:half])


def yarn(rotary, base, factor, trained, fast=32.0, slow=1.0):
    """Peng et al., "YaRN: Efficient Context Window Extension": the dim that makes r turns over the
    trained length is rotary ln(trained / (2 pi r)) / (2 ln base); the ramp runs from the floor of fast's
    to the ceiling of slow's, kept within the numbers 0 .. rotary - 1."""
    def dim(r):
        return rotary * math.log(trained / (r * 2 * math.pi)) / (2 * math.log(base))

    lo, hi = max(math.floor(dim(fast)), 0), min(math.ceil(dim(slow)), rotary - 1)
    out = []
    for i in range(rotary // 2):
        f = base ** (-2 * i / rotary)
        ramp = min(max((i - lo) / (hi - lo), 0.0), 1.0)
        out.append(f / factor * ramp + f * (1 - ramp))
    return torch.tensor(out, dtype=torch.float64)


@pytest.mark.parametrize("trained", [4096, 32768, 46000, 65536, 131072, 262144])
@pytest.mark.parametrize("base", [1e4, 5e4, 1e6])
@pytest.mark.parametrize("rotary,factor", [(64, 4.0), (64, 40.0), (128, 16.0), (32, 2.0)])
def test_every_dim_follows_the_yarn_rule(rotary, factor, base, trained):
    f, gain = frequencies(rt.rope_cos_sin(4, rotary, base, factor, trained))
    want = yarn(rotary, base, factor, trained)
    assert float((f / want - 1).abs().max()) <= 2.0 ** -22
    assert float((gain / (0.1 * math.log(factor) + 1) - 1).abs().max()) <= 2.0 ** -22


@pytest.mark.parametrize("trained", [4096, 131072])
def test_dims_between_the_turns_are_neither_kept_nor_fully_divided(trained):
    """A dim that turns more than beta_slow and less than beta_fast times lies between both."""
    f, _ = frequencies(rt.rope_cos_sin(4, 64, 1e4, 4.0, trained))
    plain = 1e4 ** (-torch.arange(32, dtype=torch.float64) / 32)
    turns = trained * plain / (2 * math.pi)
    between = (turns > 1.0) & (turns < 32.0)
    assert bool(between.any())
    assert bool((f < plain * (1 - 1e-6))[between].all()) and bool((f > plain / 4 * (1 + 1e-6))[between].all())
    assert torch.allclose(f[turns >= 64.0], plain[turns >= 64.0], rtol=1e-6)
    assert torch.allclose(f[turns < 0.5], plain[turns < 0.5] / 4, rtol=1e-6)


def test_plain_and_interpolated_tables():
    plain = 1e4 ** (-torch.arange(32, dtype=torch.float64) / 32)
    for factor in (1.0, 4.0):
        f, gain = frequencies(rt.rope_cos_sin(4, factor=factor))
        assert float((f * factor / plain - 1).abs().max()) <= 2.0 ** -22 and float((gain - 1).abs().max()) <= 2.0 ** -22
    cs = rt.rope_cos_sin(300001, 64)
    angle = 300000 * plain
    assert float((cs[300000].double() - torch.cat([angle.cos(), angle.sin()])).abs().max()) <= 2.0 ** -24
