"""ExpertMLP.decode where a wave of the second launch takes several of the plan's items one
after the other: the next item's operands and scales are fetched while one ends, and the
sums and rows change over after whole steps or after a step that the rows end in.

Bounds are those of test_gpu_experts_decode.py, whose oracle this uses.
"""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_experts_decode import DEV, Layer

pytestmark = pytest.mark.gpu

# E, H, T, k. A column tile's items go to 4 waves for each of min(512 / tiles, entries / 8, 8)
# workgroups, at least one.
LISTS = {
    "four_waves": (14, 80, 5, 3),        # 10 or more items, parts of 16 rows
    "four_waves_few": (14, 80, 3, 5),    # the same with at most four rows a part
    "all_parts": (100, 96, 32, 8),       # 90 or so items on 32 waves
    "all_parts_few": (300, 40, 4, 16),   # 58 or so items on 32 waves
    "long_items": (5, 64, 64, 3),        # experts with 38 rows or so: three items each
}
# I in whole steps of 128 and with a last one of 32 or 96 values; 17 steps are more than the
# 16 whose scales LDS holds of groups of 128 (8 for groups of 64, 4 for groups of 32)
INNER = {32: [128, 160, 544, 672], 64: [128, 192, 1088], 128: [128, 640, 2176]}
FORMS = [("mxfp4", "bf16", 32, {}), ("mxfp8", "bf16", 32, {})] + [
    ("affine", dtype, group, dict(bits=bits, group=group, params=params))
    for bits, dtype, params, group in ((4, "bf16", "bf16", 32), (4, "bf16", "bf16", 64),
                                       (4, "f16", "f32", 128), (8, "bf16", "f32", 64),
                                       (8, "f16", "f16", 32), (2, "bf16", "bf16", 128))]
CASES = [(f, d, I, kw) for f, d, group, kw in FORMS for I in INNER[group]] + [
    ("dense", d, I, {}) for d, I in (("bf16", 128), ("f16", 129), ("bf16", 255), ("bf16", 384),
                                     ("f16", 515), ("bf16", 1057))]


@pytest.mark.parametrize("fmt,dtype,I,kw", CASES)
@pytest.mark.parametrize("name", sorted(LISTS))
def test_waves_with_several_items(name, fmt, dtype, I, kw):
    E, H, T, k = LISTS[name]
    group = kw.get("group", 32)
    H = (H + group - 1) // group * group if fmt != "dense" else H + 1
    layer = Layer(fmt, E, H, I, dtype, seed=I + E, **kw)
    layer.check(*layer.inputs(T, k))


@pytest.mark.parametrize("fmt", ["dense", "mxfp4", "affine"])
@pytest.mark.parametrize("T", [4, 24])
def test_an_items_numbers_stay_its_own(fmt, T):
    """An expert of NaN between others that one wave takes in turn reaches its rows alone."""
    layer = Layer(fmt, 20, 64, 160)
    x, index, weights = layer.inputs(T, 4)
    index[index == 9] = 8
    index[T // 2, 1] = 9
    clean = index.clone()
    clean[T // 2] = -1
    want = layer.check(x, clean, weights)
    bad = layer.mlp.down if fmt == "dense" else layer.mlp.down[1]
    if fmt == "mxfp4":
        bad[9] = 255  # (the scale that is no number)
    else:
        bad[9] = torch.nan
    y = layer.mlp.decode(x.to(DEV), index.to(DEV), weights.to(DEV))
    keep = [t for t in range(T) if t != T // 2]
    assert bool(y[T // 2].isnan().all()) and torch.equal(y[keep], want[keep])
