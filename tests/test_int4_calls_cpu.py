"""How 4-bit modules and the token shuffle take calls that their main tests leave out, without a GPU."""
import pytest
import torch

from p2pllm_b200 import _lib, compact, int4, moe


@pytest.fixture(scope="module")
def lib():
    from p2pllm_b200 import build
    build.build()
    build.build_ops()
    return _lib.load()


class OnGpu(torch.Tensor):
    """A CPU tensor that says it lies on a GPU."""
    is_cuda = True
    device = torch.device("cuda", 0)


class Stream:
    def __init__(self, log, device):
        self.log, self.device = log, device

    def synchronize(self):
        self.log.append(self.device)


@pytest.fixture
def waits(monkeypatch):
    """The devices whose current streams were waited for."""
    log = []
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream(log, device))
    return log


def _layout():
    layout = int4.Layout.__new__(int4.Layout)
    layout.__dict__.update(experts=1, rows=1, cols=1, group=32, gated=False, has_zeros=False, dtype=torch.bfloat16,
                           device=torch.device("cuda", 0), data=torch.zeros(64, dtype=torch.uint8).as_subclass(OnGpu))
    return layout


def test_a_layout_that_comes_back_waits_for_its_weights(lib, waits):
    """Products read weights ahead of their stream, so a layout that was just copied or loaded is waited for."""
    again = int4.Layout.__new__(int4.Layout)
    again.__setstate__(_layout().__getstate__())
    assert waits == [torch.device("cuda", 0)]


@pytest.mark.parametrize("kind", [compact.Tiles, compact.GatedTiles, moe.ExpertTiles])
def test_pruned_layouts_that_come_back_wait_for_their_weights(waits, kind):
    state = {"layout": "tc", "words": torch.zeros(8, dtype=torch.int32).as_subclass(OnGpu), "blocks": None}
    again = kind.__new__(kind)
    again.__setstate__(dict(state))
    assert waits == [torch.device("cuda", 0)] and again.words is state["words"]
