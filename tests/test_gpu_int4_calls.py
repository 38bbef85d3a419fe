"""Calls of 4-bit modules and of the token shuffle that test_gpu_int4.py and test_gpu_shuffle.py leave out. The bounds are
those files'."""
import copy
import pickle

import pytest
import torch

from p2pllm_b200 import P2PError, _lib, compact, int4, kernels, moe, prepare, shard
from test_gpu_int4 import DT, Dispatch, TopK, _block, _check_gated, _check_product, _dense64, _gen

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


def test_sorts_of_different_sizes_from_several_threads():
    """1024 experts take 139 KB of shared memory, 512 with many pairs 70 KB: requests of one thread must not take room
    from another's."""
    import threading
    g = _gen(3)
    cases = [(torch.randint(0, e, (t, 8), generator=g, device="cuda"), e) for t, e in ((2048, 1024), (2048, 512), (16, 600))]
    want = [moe.sort_tokens(ids, e) for ids, e in cases]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(300):
                    got = moe.sort_tokens(*cases[i % 3])
                torch.cuda.current_stream().synchronize()
                assert torch.equal(got.where, want[i % 3].where) and torch.equal(got.offsets, want[i % 3].offsets)
        except BaseException as e:
            failed.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


@pytest.mark.parametrize("tokens", [3, 40])
def test_the_operators_know_the_weights_dtype(tokens):
    """A layout's bytes read with the wrong 16-bit type would be other scales: f16 tokens on bf16 weights are refused,
    and so is a layout whose tensor does not say what it holds."""
    g = _gen(4)
    q = compact.Tiles([_block((), 40, 64, 64, True, torch.bfloat16, g)]).int4
    e = moe.Int4Experts([_block((4,), 40, 64, 64, True, torch.bfloat16, g)])
    order = moe.sort_tokens(torch.zeros(tokens, 1, dtype=torch.int32, device="cuda"), 4)
    x = torch.randn(tokens, 64, generator=g, device="cuda").bfloat16()
    ops = _lib.ops()
    mm = lambda x, data: ops.int4_mm(x, data, True, 40, 64, 64, False)
    grouped = lambda x, data: ops.int4_grouped(x, data, True, 4, 40, 64, 64, False, order.order, order.where, order.offsets,
                                               order.items, order.n_items, 1, True)
    assert torch.equal(mm(x, q.data), q.mm(x)) and torch.equal(grouped(x, e.int4.data), e(x, order, gather=True))
    for call, data in ((mm, q.data), (grouped, e.int4.data)):
        for bad_x, bad in ((x.half(), data), (x.float(), data), (x, data.view(torch.uint8)), (x, data.view(torch.float16))):
            with pytest.raises(RuntimeError, match="4-bit layout's weights"):
                call(bad_x, bad)
    with pytest.raises(RuntimeError, match="does not hold"):
        mm(x, q.data[:-1])


@pytest.mark.parametrize("zero", [16, 255])
def test_zero_points_that_are_no_codes_are_refused(zero):
    """16 would multiply as 0 and expand as 16."""
    g = _gen(5)
    lead = ((), (3,))
    for make, dims in ((lambda b: compact.Tiles([b]), lead[0]), (lambda b: compact.GatedTiles([b]), lead[0]),
                       (lambda b: int4.expand(b), lead[0]), (lambda b: moe.Int4Experts([b]), lead[1]),
                       (lambda b: compact.CompactMoE(None, {"w2_weight": [b]}), lead[1])):
        block = _block(dims, 32, 130, 32, True, torch.bfloat16, g)
        make(block)
        block[3][..., -1, -1] = zero
        with pytest.raises(P2PError, match=f"0 to 15, not {zero}"):
            make(block)


def test_whole_blocks_can_be_expanded_while_a_graph_is_captured():
    g = _gen(6)
    block = _block((), 32, 128, 32, True, torch.bfloat16, g)
    want = int4.expand(block)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        dense = int4.expand(block)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(dense, want)


@pytest.mark.parametrize("tokens", [1, 17, 40])
def test_a_sharded_4_bit_module(tokens):
    """One rank's module, and two ranks' rows by hand, each rank writing its columns of y."""
    g = _gen(7)
    blocks = [_block((), r, 130, 32, z, torch.bfloat16, g) for r, z in ((200, True), (57, False))]
    x = torch.randn(tokens, 130, generator=g, device="cuda").bfloat16()
    want = compact.Tiles(blocks)(x)
    assert torch.equal(shard.ShardedCompact(blocks).apply(None, x), want)
    y = torch.zeros(tokens, 257, dtype=torch.bfloat16, device="cuda")
    for start, stop in shard.row_ranges(257, 2):
        mine = shard.shard_blocks(blocks, start, stop)
        compact.Tiles(mine)(x, out=y[:, start:stop])
        _check_product(y[:, start:stop], x, torch.cat([_dense64(b) for b in mine]), torch.bfloat16)


@pytest.mark.parametrize("tokens,rows,cols,hold", [
    (1, 256, 4096, 0), (17, 256, 4096, 1), (17, 20000, 1024, 0), (32, 40000, 1024, 3), (40, 300, 4096, 0), (64, 20000, 2048, 3),
    (100, 20000, 2048, 0), (150, 20000, 1024, 5), (190, 20000, 1024, 0), (190, 20000, 1024, 4), (272, 20000, 1024, 0),
    (272, 20000, 1024, 6), (600, 300, 1024, 0)])
def test_a_withheld_load_ends_the_launch_with_an_error_status(tokens, rows, cols, hold):
    """Failure detection without a fault: every CTA withholds one load of x, so the waits for it run out after 20 ms. The
    launch must end by itself and soon (a wait that does not see another's failure, or starts its limit late, takes
    seconds), the status must name the wait that gave up, and the next launch is an ordinary one."""
    import time
    g = _gen(8)
    block = _block((), rows, cols, 64, True, torch.bfloat16, g)
    tiles = compact.Tiles([block])
    x = torch.randn(tokens, cols, generator=g, device="cuda").bfloat16()
    want = tiles(x)
    kernels.int4_status()
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    kernels.int4_withhold(tiles.int4, x, hold=hold, wait_us=20000)
    torch.cuda.synchronize()
    elapsed = time.perf_counter() - t0
    assert elapsed < 1.0, elapsed
    with pytest.raises(P2PError, match="timed out"):
        kernels.int4_status(reset=True)
    kernels.int4_status()                                           # reset: clean again
    assert torch.equal(tiles(x), want)
    kernels.int4_status()


# Every width of the tensor-core product: its accumulators' spacing is the tokens of a tile in steps of 16.
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("tokens,rows,cols", [
    (34, 260, 640), (49, 4098, 321), (113, 300, 640), (129, 260, 1030), (145, 20000, 257), (160, 300, 640), (161, 300, 640),
    (177, 260, 1030), (192, 20000, 257), (193, 300, 640), (225, 260, 321), (257, 300, 640), (340, 300, 640), (384, 20000, 257),
    (385, 260, 640), (545, 300, 321)])
def test_products_of_every_width(tokens, rows, cols, gated, group, zeros, dtype):
    g = _gen(tokens * 1009 + rows)
    block = _block((), rows, cols, group, zeros, DT[dtype], g)
    if gated:
        x = (torch.randn(tokens, cols, generator=g, device="cuda") / cols ** 0.5).to(DT[dtype])
        _check_gated(compact.GatedTiles([block])(x), x, _dense64(block), DT[dtype])
    else:
        x = torch.randn(tokens, cols, generator=g, device="cuda").to(DT[dtype])
        _check_product(compact.Tiles([block])(x), x, _dense64(block), DT[dtype])


def _skewed(tokens, topk, experts, g, power):
    """Ids of which the low ones come up often and the high ones hardly ever, a tenth of the pairs nowhere."""
    ids = (torch.rand(tokens, topk, generator=g, device="cuda") ** power * experts).long().clamp(max=experts - 1)
    return torch.where(torch.rand(tokens, topk, generator=g, device="cuda") < 0.1, -1, ids)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("tokens,topk,experts,rows,cols,group,zeros,power", [
    (40, 1, 8, 66, 130, 32, True, 3),                                # items of 16 places, some experts with one pair or none
    (300, 2, 40, 66, 130, 64, False, 3),                             # 32
    (280, 4, 32, 130, 257, 32, True, 6),                             # 64, one expert with most of the pairs
    (250, 8, 25, 66, 320, 128, True, 4),                             # 128
    (260, 3, 7, 130, 257, 32, True, 1), (440, 4, 16, 300, 640, 128, False, 5),          # 160
    (500, 3, 8, 130, 257, 32, True, 1), (700, 4, 12, 300, 640, 64, True, 6), (1100, 1, 4, 66, 96, 128, False, 2),   # 256
    (600, 2, 3, 260, 1030, 32, False, 1)])
def test_experts_items_of_every_size(tokens, topk, experts, rows, cols, group, zeros, power, gather, gated, dtype):
    g = _gen(tokens + rows)
    block = _block((experts,), rows, cols, group, zeros, DT[dtype], g)
    order = moe.sort_tokens(_skewed(tokens, topk, experts, g, power), experts)
    x = torch.randn(tokens if gather else tokens * topk, cols, generator=g, device="cuda")
    x = (x / cols ** 0.5 if gated else x).to(DT[dtype])
    tiles = moe.Int4Experts([block], gated=gated)
    y = tiles(x, order, gather=gather)
    w, offsets = _dense64(block), order.offsets.tolist()
    xs = x[(order.order.clamp(min=0) // topk).long()] if gather else x
    for e in range(experts):
        a, b = offsets[e], offsets[e + 1]
        if a < b:
            (_check_gated if gated else _check_product)(y[a:b], xs[a:b], w[e], DT[dtype])
    assert bool((y[offsets[-1]:] == 0).all())
    out = torch.full_like(y, 5.0)
    tiles(x, order, gather=gather, out=out)
    assert torch.equal(out[:offsets[-1]], y[:offsets[-1]]) and bool((out[offsets[-1]:] == 5.0).all())


class _Experts(torch.nn.Module):
    def __init__(self, E, R, H, g):
        super().__init__()
        rand = lambda *s: torch.nn.Parameter((torch.randn(*s, generator=g, device="cuda") * 0.1).bfloat16(), False)
        self.w13_weight, self.w2_weight = rand(E, 2 * R, H), rand(E, H, R)


def _expert_model(E, R, H, seed):
    """One layer of routed experts beside two plain projections, of a seed."""
    g, nn = _gen(seed), torch.nn
    layer = nn.Module()
    layer.mlp = nn.Module()
    layer.mlp.experts = _Experts(E, R, H, g)
    for name, shape in (("gate_proj", (R, H)), ("down_proj", (H, R))):
        linear = nn.Module()
        linear.weight = nn.Parameter(torch.randn(shape, generator=g, device="cuda").bfloat16(), False)
        setattr(layer.mlp, name, linear)
    model = nn.Module()
    model.layers = nn.ModuleList([layer])
    return model


class _DenseMethod:
    """A layer's own method on whatever expert weights it is given, in 32 bits."""

    def apply(self, layer, d):
        t, out = d.topk_output, 0
        for j in range(t.topk_ids.shape[1]):
            gate, up = torch.einsum("trh,th->tr", layer.w13_weight[t.topk_ids[:, j]].float(), d.hidden_states.float()).chunk(2, -1)
            h = torch.nn.functional.silu(gate) * up
            out = out + t.topk_weights[:, j:j + 1] * torch.einsum("thr,tr->th", layer.w2_weight[t.topk_ids[:, j]].float(), h)
        return out


@pytest.mark.parametrize("zero_points", [False, True])
def test_4_bit_files_of_routed_experts_install_in_every_form(tmp_path, zero_points):
    """Dense rows written back, experts expanded in every pass, and experts multiplied in 4 bits. Bounds: the two weights
    that are expanded are the same; the product in 4 bits rounds h, the experts' rows and the sums to bf16, at most half
    a step each of its norm, and its weights not at all, where expanded ones are rounded once each: below 5 half steps."""
    E, R, H, T, K = 6, 40, 64, 33, 2
    g = _gen(9)
    paths = prepare.write_int4(_expert_model(E, R, H, 5).layers, [0], str(tmp_path), group=32, zero_points=zero_points)
    models = {}
    for form in ("dense", "compact", "grouped"):
        models[form] = _expert_model(E, R, H, 5)
        models[form].layers[0].mlp.experts.quant_method = _DenseMethod()
        prepare.install_replica(models[form], paths[0], form=form)
    original = _expert_model(E, R, H, 5).layers[0].mlp.experts
    dense = models["dense"].layers[0].mlp.experts
    for name in ("w13_weight", "w2_weight"):
        w = getattr(original, name)
        halves = w.chunk(2, dim=1) if name == "w13_weight" else (w,)
        want = torch.cat([int4.expand(int4.quantize(h, 32, zero_points)) for h in halves], dim=1)
        assert torch.equal(getattr(dense, name), want)
    x = torch.randn(T, H, generator=g, device="cuda").bfloat16()
    ids = torch.randint(0, E - 1, (T, K), generator=g, device="cuda")               # one expert that no token reaches
    weights = torch.rand(T, K, generator=g, device="cuda")
    d = Dispatch(x, TopK(weights / weights.sum(-1, keepdim=True), ids))
    want = _DenseMethod().apply(dense, d)
    layers = {f: m.layers[0].mlp.experts for f, m in models.items()}
    assert isinstance(layers["compact"].quant_method, compact.CompactMoE) and isinstance(layers["grouped"].quant_method, moe.GroupedMoE)
    assert layers["grouped"].quant_method.is_int4 and layers["grouped"].w13_weight.numel() == 0
    assert torch.equal(layers["compact"].quant_method.apply(layers["compact"], d), want)
    got = layers["grouped"].quant_method.apply(layers["grouped"], d)
    assert float((got.float() - want).norm() / want.norm()) <= 5 * torch.finfo(torch.bfloat16).eps / 2


def test_calls_under_inference_mode():
    g = _gen(10)
    tiles = compact.Tiles([_block((), 40, 128, 64, True, torch.bfloat16, g)])
    experts = moe.Int4Experts([_block((4,), 128, 128, 64, True, torch.bfloat16, g)])
    x = torch.randn(9, 128, generator=g, device="cuda").bfloat16()
    ids, w = torch.randint(0, 4, (9, 2), generator=g, device="cuda"), torch.rand(9, 2, generator=g, device="cuda")

    def run(x):
        order = moe.sort_tokens(ids, 4)
        out = torch.empty(9, 40, dtype=x.dtype, device="cuda")
        return (tiles(x), tiles(x, out=out), experts(x, order, gather=True), moe.to_experts(x, order),
                moe.from_experts(experts(x, order, gather=True), order, w))
    want = run(x)
    with torch.inference_mode():
        for t in (x, x.clone(), x.requires_grad_(False)):
            got = run(t)
            assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(a.is_inference() for a in got)
