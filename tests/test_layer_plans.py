"""How the products of the projection and the feed-forward block would run (host only): the sizes that the GPU tests take
reach every engine, and refusals of the plan queries."""
from __future__ import annotations

import ctypes

import pytest
import torch

from orda_ce_kernel import _native
from tests._engine_cases import BLOCK16, BLOCK32, LINEAR16, LINEAR32, TILES16, TILES32, every, reached


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_the_engine_tests_reach_every_engine(dtype):
    single = dtype == torch.float32
    tiles = TILES32 if single else TILES16
    plans = [_native.linear_plan(*s, dtype) for s in (LINEAR32 if single else LINEAR16)]
    assert reached(plans) == every(_native.LINEAR_PRODUCTS, tiles)
    plans = [_native.feed_forward_plan(*s, dtype) for s in (BLOCK32 if single else BLOCK16)]
    assert reached(plans) == every(_native.FFN_PRODUCTS, tiles)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_few_rows_have_their_own_engine(dtype):
    for tokens in (1, 16):
        plan = _native.linear_plan(tokens, 300, 129, dtype)
        assert plan["forward"] == {"engine": "few_rows", "tile_rows": 16, "tile_cols": 16, "splits": 1, "items": 9}
        assert plan["grad_x"]["engine"] != "few_rows"
        assert _native.feed_forward_plan(tokens, 300, 129, 40, dtype)["gate"]["engine"] == "few_rows"
    assert _native.linear_plan(17, 300, 129, dtype)["forward"]["engine"] != "few_rows"


def test_items_are_tiles_times_splits():
    p = _native.linear_plan(8192, 4096, 2048, torch.bfloat16)["forward"]
    assert p["engine"] == "ring" and p["items"] == 32 * 8 * p["splits"]
    p = _native.feed_forward_plan(512, 1024, 2730, 1024, torch.bfloat16)
    assert p["gate"]["items"] == (512 // p["gate"]["tile_rows"]) * (-(-2752 // (p["gate"]["tile_cols"] // 2))) * p["gate"]["splits"]


def test_plan_queries_refuse():
    with pytest.raises(ValueError, match="tokens"):
        _native.linear_plan(0, 8, 8, torch.bfloat16)
    with pytest.raises(ValueError, match="inner"):
        _native.feed_forward_plan(4, 8, 0, 8, torch.bfloat16)
    lib, out = _native.library(), _native.ProductPlan()
    lin = _native.Linear(_native.ABI_VERSION, 0, 0, 0, 4, 16, 16, 16, 16, 16, 16, 16)
    ffn = _native.FeedForward(_native.ABI_VERSION, 0, 0, 0, 4, 16, 16, 16, 16, 16, 16, 16, 16, 16, 16, 16)
    for fn, p, n in ((lib.orda_linear_plan, lin, 3), (lib.orda_ffn_plan, ffn, 7)):
        assert fn(ctypes.byref(p), 0, ctypes.byref(out)) == 0
        for product in (-1, n):
            assert fn(ctypes.byref(p), product, ctypes.byref(out)) == -1
        assert fn(ctypes.byref(p), 0, None) == -1 and fn(None, 0, ctypes.byref(out)) == -1


@pytest.mark.parametrize("size", [(1 << 30, 8, 8), ((1 << 30) - 63, 8, 8), (1 << 30, 8, 64), (1 << 29, 8, 200), (1 << 30, 72, 129)], ids=str)
def test_launches_have_fewer_than_2_to_32_threads(size):
    """A tile is a workgroup of 256 threads; 64-row tiles of 2^30 tokens are 2^24 of them."""
    for p in _native.linear_plan(*size, torch.bfloat16).values():
        assert p["engine"] == "ring" or p["items"] * 256 < 1 << 32
    for p in _native.feed_forward_plan(size[0], 8, 64, 8, torch.bfloat16).values():
        assert p["items"] * 256 < 1 << 32


def test_more_tiles_than_a_launch_takes_are_refused():
    with pytest.raises(ValueError, match="more tiles"):
        _native.linear_plan(1 << 30, 64, 129, torch.bfloat16)
    with pytest.raises(ValueError, match="more tiles"):
        _native.feed_forward_plan(1 << 30, 8, 128, 8, torch.bfloat16)
    lin = _native.Linear(_native.ABI_VERSION, 0, 0, 0, 1 << 30, 64, 129, 64, 64, 129, 64, 64)
    assert _native.library().orda_linear_forward(ctypes.byref(lin), 256, 256, None, None, 256, None, 256, 1 << 50, None) == -1
    assert _native.library().orda_linear_workspace_bytes(ctypes.byref(lin), 0) == 0
