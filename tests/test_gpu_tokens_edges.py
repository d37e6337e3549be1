"""Token rows at their edges: single rows and none, widths at the border of what a launch may have, states that change between a forward pass
and its backward pass, sums that have to come out exactly.

Products of whole numbers whose sums of magnitudes stay below 2^23 are exact in 32 bits in any order, also where additions cut off what lies below 2^-23 of
the largest addend: such tests want equality."""
import os
import subprocess
import sys

import pytest
import torch

import datago_b200 as dg
from datago_b200 import tokens as tk

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
MEAN, STD = (0.48, 0.46, 0.41), (0.27, 0.26, 0.28)


@pytest.fixture(scope="module")
def ctx():
    return dg.Context(0)


def rand(shape, dtype, seed, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * spread).to(dtype)


def some_pixels(shape, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8)


def stem_of(ctx, p=0.25, width=96, dtype=F32):
    return tk.PatchStem(ctx, 14, MEAN, STD, rand((width, 588), F32, 1, 0.02), rand((width,), F32, 2), p=p, seed=5, dtype=dtype)


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


# ---- states --------------------------------------------------------------------------------------------------------------
def test_a_backward_pass_goes_by_its_forward_pass(ctx):
    stem, pixels, positions, dy = stem_of(ctx), some_pixels((2, 28, 42, 3), 3), rand((6, 96), F32, 4), rand((12, 96), F32, 5)
    saved = stem.forward(pixels, positions, offset=11)[1]
    want = stem.backward(saved, dy)
    kept = stem.p, stem.seed, stem.norm_weight
    for change in (dict(p=0.0), dict(p=0.75), dict(seed=6), dict(norm_weight=None), dict(norm_weight=rand((96,), F32, 7))):
        for name, value in change.items():
            setattr(stem, name, value)
        assert same(stem.backward(saved, dy), want), change
        stem.p, stem.seed, stem.norm_weight = kept
    stem.p = 0.0  # and one without dropout stays one
    saved = stem.forward(pixels, positions)[1]
    want = stem.backward(saved, dy)
    stem.p = 0.5
    assert same(stem.backward(saved, dy), want)


def test_a_captured_stem_reads_the_weight_that_was_set(ctx):
    stem, pixels, positions = stem_of(ctx), some_pixels((2, 28, 42, 3), 13), rand((6, 96), F32, 14)
    stem.forward(pixels, positions)
    places = stem.weight8.values.data_ptr(), stem.weight8.scales.data_ptr()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = stem.forward(pixels, positions)[0]
    new = rand((96, 588), F32, 15, 0.05)
    stem.set_weight(new)
    assert (stem.weight8.values.data_ptr(), stem.weight8.scales.data_ptr()) == places
    graph.replay()
    other = tk.PatchStem(ctx, 14, MEAN, STD, new, stem.norm_weight, p=0.25, seed=5, dtype=F32)
    want = other.forward(pixels, positions)[0]
    assert torch.equal(norm.sum, want.sum) and torch.equal(norm.y.values.float(), want.y.values.float())
    stem.set_weight(rand((100, 588), F32, 16))  # of another shape: elsewhere
    assert stem.weight8.shape == (100, 588)
