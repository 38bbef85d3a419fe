"""Calls of 4-bit modules and of the token shuffle that test_gpu_int4.py and test_gpu_shuffle.py leave out. The bounds are
those files'."""
import copy
import pickle

import pytest
import torch

from p2pllm_b200 import compact, moe
from test_gpu_int4 import _block, _gen

pytestmark = pytest.mark.gpu


def test_modules_copied_behind_a_busy_stream():
    """9 MB of weights a module, each copy used right after it was made, on a stream that has 50 products to do first."""
    g = _gen(1)
    tiles = compact.Tiles([_block((), 4096, 4096, 128, True, torch.bfloat16, g)])
    experts = moe.Int4Experts([_block((8,), 1024, 2048, 64, True, torch.bfloat16, g)])
    x = torch.randn(17, 4096, generator=g, device="cuda").bfloat16()
    order = moe.sort_tokens(torch.randint(0, 8, (17, 1), generator=g, device="cuda"), 8)
    want = tiles(x), experts(x[:, :2048], order)
    a = torch.randn(4096, 4096, generator=g, device="cuda").bfloat16()
    for again in (copy.deepcopy, lambda t: pickle.loads(pickle.dumps(t))):
        for _ in range(50):
            a @ a
        assert torch.equal(again(tiles)(x), want[0])
        assert torch.equal(again(experts)(x[:, :2048], order), want[1])


@pytest.mark.parametrize("layout", ["tc", "mask"])
def test_pruned_modules_copied_behind_a_busy_stream(layout):
    g = _gen(2)
    w = torch.randn(4096, 4096, generator=g, device="cuda").bfloat16()
    from p2pllm_b200 import kernels
    kept = kernels.wanda_select(w, torch.ones(4096, device="cuda"), 1024)
    tiles = compact.Tiles([("compact", kept["values"], kept["idx"], 4096)], layout=layout)
    x = torch.randn(17, 4096, generator=g, device="cuda").bfloat16()
    want = tiles(x)
    for again in (copy.deepcopy, lambda t: pickle.loads(pickle.dumps(t))):
        for _ in range(50):
            w @ w
        assert torch.equal(again(tiles)(x), want)
