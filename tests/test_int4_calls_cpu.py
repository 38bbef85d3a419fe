"""How 4-bit modules and the token shuffle take calls that their main tests leave out, without a GPU."""
from types import SimpleNamespace

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from p2pllm_b200 import P2PError, _lib, compact, int4, moe, shard


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


def test_modules_pickled_before_4_bit_blocks_still_run(monkeypatch):
    """Their state has no word of 4 bits."""
    ran = []
    for name in ("spmm_tc", "spmm_tc_gated"):
        monkeypatch.setattr(compact.kernels, name, lambda *a, name=name, **k: ran.append(name))
    monkeypatch.setattr(moe, "route", lambda *a: ran.append("route") or (_ for _ in ()).throw(StopIteration))
    state = {"layout": "tc", "words": torch.zeros(8, dtype=torch.int32), "seg": torch.zeros(2, dtype=torch.int64), "rows": 4,
             "layout_rows": 8, "cols": 8, "seg_cap": 1, "blocks": None, "dtype": torch.bfloat16}
    for kind in (compact.Tiles, compact.GatedTiles):
        module = kind.__new__(kind)
        module.__setstate__(dict(state))
        module(torch.zeros(1, 8, dtype=torch.bfloat16))
        assert module.nbytes() == 48
    layer = moe.GroupedMoE.__new__(moe.GroupedMoE)
    torch.nn.Module.__init__(layer)
    experts = compact.Tiles.__new__(compact.Tiles)
    experts.__setstate__(state | {"experts": 2})
    layer.method, layer.w13 = None, experts
    x, ids = torch.zeros(1, 8, dtype=torch.bfloat16), torch.zeros(1, 2, dtype=torch.int64)
    topk = SimpleNamespace(topk_ids=ids, topk_weights=torch.zeros(1, 2))
    with pytest.raises(StopIteration):
        layer.apply(None, SimpleNamespace(hidden_states=x, topk_output=topk))
    assert ran == ["spmm_tc", "spmm_tc_gated", "route"]


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, device="meta", dtype=dtype)


@pytest.fixture
def order(lib):
    return moe.TokenOrder(*_lib.ops().moe_sort(_meta(17, 8, dtype=torch.int64), 128), 17, 8)


@pytest.mark.parametrize("which", ["rows there", "sums back", "weighted sums back", "weights", "gradient"])
def test_tangents_are_not_lost_on_the_way_to_the_experts_and_back(lib, order, which):
    """Forward-mode derivatives are refused, as they are where an input needs a gradient, and not returned as none."""
    ops, x, y, w = _lib.ops(), _meta(17, 96), _meta(136, 96), _meta(17, 8)
    call, t = {"rows there": (lambda t: ops.moe_spread(t, order.where, order.offsets, 8), x),
               "sums back": (lambda t: ops.moe_sum(t, order.where, order.offsets, None, 8), y),
               "weighted sums back": (lambda t: ops.moe_sum(t, order.where, order.offsets, w, 8), y),
               "weights": (lambda t: ops.moe_sum(y, order.where, order.offsets, t, 8), w),
               "gradient": (lambda t: ops.moe_sum_back(t, y, order.where, order.offsets, w, 8)[0], x)}[which]
    with fwAD.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        call(fwAD.make_dual(t, torch.empty_like(t)))
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(call, (t,), (torch.empty_like(t),))
    with fwAD.dual_level():                          # no tangent: the call goes through
        assert call(t).device.type == "meta"


@pytest.mark.parametrize("which", ["mm", "mm_into", "grouped", "grouped_into"])
def test_products_refuse_to_be_differentiated_in_any_mode(lib, order, which):
    """4-bit products are for inference: forward mode and torch.func's transforms are refused as requires_grad is, and so
    is an output that takes part in a graph."""
    ops, w = _lib.ops(), _meta(100, dtype=torch.uint8)
    sizes = (False, 40, 64, 64, False)
    sorted_ = (order.order, order.where, order.offsets, order.items, order.n_items, 8, True)
    x, out = _meta(17, 64), _meta(17 if "mm" in which else 136, 40)
    run = {"mm": lambda t: ops.int4_mm(t, w, *sizes), "mm_into": lambda t, y=out: ops.int4_mm_into(t, w, *sizes, y),
           "grouped": lambda t: ops.int4_grouped(t, w, False, 128, *sizes[1:], *sorted_),
           "grouped_into": lambda t, y=out: ops.int4_grouped_into(t, w, False, 128, *sizes[1:], *sorted_, y)}[which]
    total = lambda t: (run(t) if "into" not in which else run(t) or t).float().sum()
    run(x)
    with torch.no_grad():
        run(x.clone().requires_grad_(True))
    with pytest.raises(RuntimeError, match="inference"):
        run(x.clone().requires_grad_(True))
    with fwAD.dual_level(), pytest.raises(RuntimeError, match="inference"):
        run(fwAD.make_dual(x, torch.empty_like(x)))
    for transform in (lambda: torch.func.grad(total)(x), lambda: torch.func.vjp(total, x),
                      lambda: torch.func.jvp(total, (x,), (torch.empty_like(x),))):
        with pytest.raises(RuntimeError, match="inference"):
            transform()
    if "into" in which:
        with pytest.raises(RuntimeError, match="out must not"):
            run(x, out.clone().requires_grad_(True))
        with torch.no_grad():
            run(x, out.clone().requires_grad_(True))


def test_a_dual_x_is_refused_with_the_packages_own_error(lib, monkeypatch):
    monkeypatch.setattr(int4, "require_cuda", lambda *ts: None)
    layout = _layout()
    layout.device, layout.cols = torch.device("cpu"), 4
    x = torch.zeros(2, 4, dtype=torch.bfloat16)
    layout.check_x(x)
    with fwAD.dual_level(), pytest.raises(P2PError, match="gradient"):
        layout.check_x(fwAD.make_dual(x, torch.ones_like(x)))


def test_layouts_pickled_as_plain_bytes_come_back_with_their_dtype(lib, waits):
    again = int4.Layout.__new__(int4.Layout)
    again.__setstate__(_layout().__getstate__())
    assert again.data.dtype == torch.bfloat16 and again.data.numel() == 32 and again.nbytes() == 64


def test_zero_points_are_codes():
    for good in (None, torch.zeros(0, dtype=torch.uint8), torch.full((3,), 15, dtype=torch.uint8)):
        int4.check_zeros(good)
    with pytest.raises(P2PError, match="0 to 15, not 16"):
        int4.check_zeros(torch.tensor([[3, 16], [0, 1]], dtype=torch.uint8))


@pytest.mark.parametrize("world", [1, 2, 3, 8])
def test_4_bit_blocks_are_cut_by_rows(world):
    """Every rank's blocks, put together again, are the module's."""
    g = torch.Generator().manual_seed(world)
    rand = lambda *s: torch.randint(0, 256, s, generator=g, dtype=torch.uint8)
    blocks = [("int4", rand(r, 65), rand(r, 5).bfloat16(), rand(r, 5) % 16 if z else None, 130, 32)
              for r, z in ((200, True), (57, False), (143, True))]
    whole = [[], [], []]
    for start, stop in shard.row_ranges(400, world):
        mine = shard.shard_blocks(blocks, start, stop)
        assert sum(b[1].shape[0] for b in mine) == stop - start and all(b[0] == "int4" and b[4:] == (130, 32) for b in mine)
        for k, into in enumerate(whole, 1):
            into += [torch.full_like(b[1][:, :5], 8) if b[k] is None else b[k] for b in mine]
    for k, parts in enumerate(whole, 1):
        want = [torch.full_like(b[1][:, :5], 8) if b[k] is None else b[k] for b in blocks]
        assert torch.equal(torch.cat(parts), torch.cat(want))


def test_a_sharded_4_bit_module_knows_its_columns(monkeypatch):
    monkeypatch.setattr(compact, "Tiles", lambda blocks, layout=None: SimpleNamespace(blocks=blocks))
    block = ("int4", torch.zeros(200, 65, dtype=torch.uint8), torch.ones(200, 5, dtype=torch.bfloat16), None, 130, 32)
    module = shard.ShardedCompact([block])
    assert (module.rows, module.cols, module.mine) == (200, 130, 200) and module.local.tiles.blocks[0][1].shape == (200, 65)


def test_withhold_test_entry_checks_its_limits(lib):
    fake = 65536
    for hold, limit, needle in ((0, 10, b"1 ms to 2 s"), (0, 3000000, b"1 ms to 2 s"), (-1, 5000, b"load"), (4096, 5000, b"load")):
        assert lib.p2p_int4_withhold(fake, 0, 4, 64, 64, fake, 0, 16, 64, 0, fake, 16, None, 0, hold, limit, None) == -1
        assert needle in lib.p2p_last_error()


@pytest.mark.parametrize("call", ["to_experts", "from_experts", "mm"])
def test_a_call_that_fails_is_not_made_again(monkeypatch, call):
    """Out of memory, say: raised once and as it is."""
    tried = []

    def fail(*a):
        tried.append(1)
        raise torch.OutOfMemoryError("no room")
    monkeypatch.setattr(_lib, "ops", lambda: SimpleNamespace(moe_spread=fail, moe_sum=fail))
    for module in (moe, int4):
        monkeypatch.setattr(module, "require_cuda", lambda *ts: None)
    where = torch.zeros(6, dtype=torch.int32)
    order = moe.TokenOrder(where, where, torch.zeros(5, dtype=torch.int32), where, where, 3, 2)
    layout = _layout()
    layout.device, layout.cols, layout._op = torch.device("cpu"), 4, fail
    run = {"to_experts": lambda: moe.to_experts(torch.zeros(3, 8), order),
           "from_experts": lambda: moe.from_experts(torch.zeros(6, 8), order, torch.zeros(3, 2)),
           "mm": lambda: layout.mm(torch.zeros(3, 4, dtype=torch.bfloat16))}[call]
    with pytest.raises(torch.OutOfMemoryError, match="no room"):
        run()
    assert len(tried) == 1


@pytest.mark.parametrize("call", [
    lambda l, f: l.p2p_moe_spread(f, 0, 1, 1, 2 ** 30 + 1, 2 ** 30 + 1, f, f, f, 2 ** 30 + 1, None),
    lambda l, f: l.p2p_moe_sum(f, 0, 1, 1, 2 ** 31 - 1, 2 ** 31 - 1, f, None, 2, f, 2 ** 31 - 1, None),
    lambda l, f: l.p2p_moe_sum_back(f, f, 0, 1, 1, 2 ** 31 - 1, 2 ** 31, 2 ** 31, f, f, f, 2, f, 2 ** 31, f, None),
    lambda l, f: l.p2p_moe_sort(f, 4, 64, 8, f, f, f, f, 64, 2 ** 31 - 1, f, None)])
def test_sizes_whose_counters_would_pass_32_bits_are_refused(lib, call):
    """A column's number steps by the grid, an item's pairs are rounded up: both in 32 bits."""
    assert call(lib, 65536) == -1
    assert b"columns" in lib.p2p_last_error() or b"items of" in lib.p2p_last_error()
