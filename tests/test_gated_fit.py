"""The polynomial that gelu's normal distribution is computed with, its coefficients as the kernels' source has them, against erfcx in 64 bits."""

import re
from pathlib import Path

import torch

SOURCE = Path(__file__).resolve().parent.parent / "tileccl_amd" / "csrc" / "tccl_gated.h"


def test_the_fit_is_as_good_as_its_comment_says():
    text = SOURCE.read_text()
    coefficients = re.search(r"constexpr float q\[\] = \{(.*?)\};", text).group(1).replace("f", "").split(",")
    q = torch.tensor([float(c) for c in coefficients], dtype=torch.float32).double()
    y = torch.linspace(0, 12, 200001, dtype=torch.float64)
    t = 1 / (1 + y / 2)
    s = torch.zeros_like(y)
    for c in q.flip(0):
        s = s * t + c
    exact = torch.special.erfcx(y)
    off = float(((t * s - exact) / exact).abs().max())
    said = float(re.search(r"largest relative error (\S+) with these coefficients", text).group(1))
    assert 0.9 * said < off <= said
