"""The stretched rotary tables over all of their pairs, from the definition in floats."""
import math

import pytest
import torch

import tdc_sequence as S


@pytest.mark.parametrize("dim,base,length,factor", [
    (64, 1e4, 131072, 4.0),      # the slowest pair turns 2.8 times: still blended
    (128, 1e4, 32768, 4.0), (128, 5e5, 8192, 32.0), (32, 1e4, 2048, 4.0), (16, 100.0, 65536, 8.0)])
def test_blend_of_kept_and_divided_frequencies(dim, base, length, factor):
    cos, sin = S.rotary_table(dim, 2, base, "parts", factor, length)
    half, size = dim // 2, 0.1 * math.log(factor) + 1
    at = lambda turns: half * math.log(length / (2 * math.pi * turns)) / math.log(base)  # noqa: E731
    low, high = max(math.floor(at(32.0)), 0), math.ceil(at(1.0))
    for i in range(half):
        freq = base ** (-i / half)
        share = min(max((i - low) / max(high - low, 1e-3), 0.0), 1.0)   # of the divided one
        if length * freq / (2 * math.pi) >= 32.0 and i <= low:
            assert share == 0.0
        if i < half - 1 and length * freq / (2 * math.pi) <= 1.0 and i >= high:
            assert share == 1.0
        angle = freq * (1 - share) + freq / factor * share
        # fp32's rounding of a value up to `size`: half a step
        assert abs(cos[1, i].item() - size * math.cos(angle)) <= 2 ** -23
        assert abs(sin[1, i].item() - size * math.sin(angle)) <= 2 ** -23


def test_slowest_pair_that_turns_more_than_once_is_not_divided_whole():
    _, sin = S.rotary_table(64, 2, 1e4, "parts", 4.0, 131072)
    kept = math.asin(sin[1, -1].item() / (0.1 * math.log(4.0) + 1)) / 1e4 ** (-31 / 32)
    assert 0.4 < kept < 0.6          # 2.8 turns: between 1/4 (one turn) and 1 (32 turns)
