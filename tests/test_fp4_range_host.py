"""The 4-bit format at the top of bf16's range: what finite rows are held as is finite in bf16."""

from __future__ import annotations

import torch

from oracle import fp4


def test_the_largest_rows_are_held_as_bf16_values():
    """Scales end at 2^125, whose largest code, 6, is the last that bf16 holds: at 2^126 a 4 is 2^128."""
    top = torch.arange(0x7e80, 0x7f80, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    rows = torch.zeros(top.numel(), 1, 128, dtype=torch.bfloat16)
    rows[:, 0, 0], rows[:, 0, 33], rows[:, 0, 64], rows[:, 0, 65] = top, -top, top, top / 2
    codes, scales = fp4.quantize(rows)
    v = fp4.values(codes, scales)
    assert torch.equal(v.to(torch.bfloat16).double(), v) and v.isfinite().all()
    assert scales.max() == 252 and v.max() == 6 * 2.0 ** 125
    assert ((v - rows.double()).abs() <= rows.double().abs() / 4).all()
    # up to 7 x 2^125 every scale is the least that leaves the largest value at most 7 times it
    small = top.double() <= 7 * 2.0 ** 125
    least = torch.ceil(torch.log2(top.double()[small] / 7)) + 127
    assert torch.equal(scales[small, 0, 0].double(), least) and (scales[~small, 0, 0] == 252).all() and (~small).any()
