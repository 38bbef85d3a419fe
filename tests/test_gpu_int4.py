"""Products with 4-bit weights (compact.Tiles on "int4" blocks, moe.Int4Experts, the 4-bit moe.GroupedMoE, 4-bit
replica files) against plain 64-bit arithmetic on the codes.

Bound of one output: half a step of its type, plus the fp32 sums', in units of 2^-23 of the terms' absolute sum. Inside a
group: at most 8 steps of 16 columns, 3 additions a step, each off by one unit at most (tensor cores may cut off): 24.
Then a chain of one fused multiply-add a group, each rounded to nearest, half a unit: at most cols / 32 of them, cols / 64
units; and of one addition a run of units that a row tile is cut into, at most cols / 128 of them and a few of the column
halves: cols / 256 + 4 units. 24 + 4 is below the 64 kept here: 64 + cols / 64 + cols / 256. (64 + cols / 256 before left out
the chain over groups, which a kernel that adds every group of a row tile one after another has.)"""
from typing import NamedTuple

import numpy as np
import pytest
import torch

from p2pllm_b200 import P2PError, compact, int4, moe, prepare

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _block(lead, rows, cols, group, zeros, dtype, g):
    """A block of random codes: every code, scale and zero point is its own."""
    groups = -(-cols // group)
    codes = torch.randint(0, 256, (*lead, rows, -(-cols // 2)), generator=g, device="cuda", dtype=torch.uint8)
    scales = (torch.rand(*lead, rows, groups, generator=g, device="cuda") * 0.05 + 0.001).to(dtype)
    z = torch.randint(0, 16, (*lead, rows, groups), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    return ("int4", codes, scales, z, cols, group)


def _dense64(block):
    _, codes, scales, zeros, cols, group = block
    q = torch.stack((codes % 16, codes // 16), dim=-1).flatten(-2)[..., :cols].double()
    per = lambda t: t.double().repeat_interleave(group, -1)[..., :cols]
    return (q - (8 if zeros is None else per(zeros))) * per(scales)


def _sum_bound(x, w):
    return (64 + w.shape[-1] / 64 + w.shape[-1] / 256) * 2.0 ** -23 * (x.abs() @ w.abs().mT)


def _half_step(want, dtype):
    return torch.finfo(dtype).eps / 2 * want.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def _check_product(y, x, w, dtype):
    x, want = x.double(), x.double() @ w.mT
    bound = _sum_bound(x, w)
    bound = bound + _half_step(want.abs() + bound, dtype)
    assert y.dtype == dtype and y.shape == want.shape
    assert bool(((y.double() - want).abs() <= bound).all()), float(((y.double() - want).abs() / bound).max())


def _check_gated(y, x, w, dtype):
    """silu(g) u, |silu'| <= 1.1, silu in fp32 within 8 roundings."""
    x = x.double()
    half = w.shape[0] // 2
    g, u = x @ w[:half].mT, x @ w[half:].mT
    dg, du = _sum_bound(x, w[:half]), _sum_bound(x, w[half:])
    silu = g * torch.sigmoid(g)
    want = silu * u
    bound = 1.1 * dg * (u.abs() + du) + silu.abs() * du + 8 * 2.0 ** -23 * want.abs()
    bound = bound + _half_step(want.abs() + bound, dtype)
    assert bool(((y.double() - want).abs() <= bound).all()), float(((y.double() - want).abs() / bound).max())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("tokens,rows,cols", [
    (1, 1, 1), (1, 16, 64), (1, 33, 130), (2, 17, 31), (7, 15, 63), (8, 130, 257), (9, 64, 1000), (16, 48, 512),
    (17, 100, 1030), (24, 31, 96), (31, 129, 321), (33, 128, 2048), (65, 257, 4100), (272, 300, 640), (300, 130, 96)])
def test_products_at_odd_sizes(tokens, rows, cols, group, zeros, dtype):
    g = _gen(tokens * 1000003 + rows * 1009 + cols)
    block = _block((), rows, cols, group, zeros, DT[dtype], g)
    x = torch.randn(tokens, cols, generator=g, device="cuda").to(DT[dtype])
    _check_product(compact.Tiles([block])(x), x, _dense64(block), DT[dtype])


@pytest.mark.parametrize("tokens,rows,cols,group", [(1, 1024, 4096, 128), (17, 4096, 4096, 128), (1, 4096, 14336, 64),
                                                    (272, 6144, 4096, 128), (64, 5120, 27648, 32)])
def test_products_at_projection_sizes(tokens, rows, cols, group):
    g = _gen(rows + cols)
    block = _block((), rows, cols, group, True, torch.bfloat16, g)
    x = torch.randn(tokens, cols, generator=g, device="cuda").bfloat16()
    _check_product(compact.Tiles([block])(x), x, _dense64(block), torch.bfloat16)


def test_blocks_of_a_module_are_its_rows_in_order():
    """q, k and v rows in one module, one of them with zero points."""
    g = _gen(5)
    blocks = [_block((), r, 200, 64, z, torch.bfloat16, g) for r, z in ((70, False), (18, True), (5, False))]
    x = torch.randn(17, 200, generator=g, device="cuda").bfloat16()
    tiles = compact.Tiles(blocks)
    assert (tiles.layout, tiles.rows, tiles.cols) == ("int4", 93, 200) and tiles.nbytes() > 0
    _check_product(tiles(x), x, torch.cat([_dense64(b) for b in blocks]), torch.bfloat16)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
@pytest.mark.parametrize("tokens,half,cols", [(1, 1, 1), (1, 40, 130), (7, 64, 257), (9, 100, 1000), (17, 640, 96),
                                              (32, 33, 2048), (33, 100, 640), (100, 129, 321), (200, 70, 1030),
                                              (272, 4096, 256), (300, 33, 130)])
def test_gate_and_up_in_one_module(tokens, half, cols, group, zeros, dtype):
    g = _gen(tokens * 10007 + half)
    blocks = [_block((), half, cols, group, z, DT[dtype], g) for z in (zeros, False)]
    x = (torch.randn(tokens, cols, generator=g, device="cuda") / cols ** 0.5).to(DT[dtype])
    tiles = compact.GatedTiles(blocks)
    assert (tiles.layout, tiles.rows, tiles.cols) == ("int4", half, cols) and tiles.nbytes() > 0
    w = torch.cat([_dense64(b) for b in blocks])
    y = tiles(x)
    assert y.shape == (tokens, half) and y.dtype == DT[dtype]
    _check_gated(y, x, w, DT[dtype])
    out = torch.full((tokens, half + 3), 7.0, dtype=DT[dtype], device="cuda")
    assert torch.equal(tiles(x, out=out[:, 1:-2]), y) and bool((out[:, 0] == 7).all()) and bool((out[:, -2:] == 7).all())


@pytest.mark.parametrize("cols,pad,offset", [(128, 8, 0), (128, 3, 0), (128, 8, 1), (127, 1, 0), (96, 0, 4), (100, 4, 2)])
def test_strided_and_unaligned_inputs(cols, pad, offset):
    g = _gen(cols + pad)
    block = _block((), 40, cols, 32, True, torch.float16, g)
    base = torch.randn(19 * (cols + pad) + offset, generator=g, device="cuda").half()
    x = base[offset:].view(19, cols + pad)[:, :cols]
    tiles = compact.Tiles([block])
    _check_product(tiles(x), x, _dense64(block), torch.float16)
    _check_product(tiles(x.t().contiguous().t()), x, _dense64(block), torch.float16)          # columns strided
    row = x[:1].expand(5, cols)                                                                # rows that overlap
    _check_product(tiles(row), row, _dense64(block), torch.float16)


def test_given_output_and_its_surroundings():
    g = _gen(1)
    block = _block((), 50, 192, 64, False, torch.bfloat16, g)
    tiles, x = compact.Tiles([block]), torch.randn(17, 192, generator=g, device="cuda").bfloat16()
    base = torch.full((19, 61), 7.0, device="cuda", dtype=torch.bfloat16)
    out = base[1:18, 3:53]
    assert tiles(x, out=out) is out
    assert torch.equal(out, tiles(x))
    base[1:18, 3:53] = 7.0
    assert bool((base == 7.0).all())


@pytest.mark.parametrize("tokens", [3, 40])
def test_a_token_that_is_not_finite_stays_alone(tokens):
    g = _gen(2)
    block = _block((), 64, 320, 128, True, torch.bfloat16, g)
    tiles, x = compact.Tiles([block]), torch.randn(tokens, 320, generator=g, device="cuda").bfloat16()
    want = tiles(x)
    bad = x.clone()
    bad[1, 100], bad[2, 5] = float("nan"), float("inf")
    y = tiles(bad)
    assert bool(y[1].isnan().all()) and not bool(y[2].isfinite().any())
    keep = [t for t in range(tokens) if t not in (1, 2)]
    assert torch.equal(y[keep], want[keep])


def test_values_at_the_edge_of_the_type():
    """f16 scales up to its largest value and down to its smallest: sums that pass the type's range become infinite,
    as rounding the exact sum makes them."""
    codes = torch.full((16, 32), 0xFF, dtype=torch.uint8, device="cuda")       # every weight 7 * scale
    scales = torch.full((16, 1), 65504.0, dtype=torch.float16, device="cuda")
    scales[8:] = 2.0 ** -24
    tiles = compact.Tiles([("int4", codes, scales, None, 64, 64)])
    x = torch.zeros(2, 64, dtype=torch.float16, device="cuda")
    x[0, 0], x[1, 0] = 0.125, 1.0
    y = tiles(x)
    assert torch.equal(y[0, :8], torch.full((8,), 57316.0, device="cuda").half()) and bool(y[1, :8].isinf().all())
    assert torch.equal(y[1, 8:], torch.full((8,), 7 * 2.0 ** -24, device="cuda").half())


def test_results_do_not_depend_on_the_launch():
    g = _gen(3)
    tiles = compact.Tiles([_block((), 4096, 4096, 128, True, torch.bfloat16, g)])
    x = torch.randn(272, 4096, generator=g, device="cuda").bfloat16()
    want = tiles(x)
    assert all(torch.equal(tiles(x), want) for _ in range(5))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ys = [tiles(x) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    here = [tiles(x) for _ in range(3)]
    assert all(torch.equal(y, want) for y in ys + here)


@pytest.mark.parametrize("tokens", [1, 8, 17, 40, 150])
@pytest.mark.parametrize("sizes", [(128, 640, 128, 96), (640, 100, 2048, 130), (64, 4096, 4096, 64)])
def test_modules_in_a_chain_read_what_the_one_before_wrote(tokens, sizes):
    """Each launch may begin before the one before has ended, joins of row tiles that no two runs share among them: the
    results are those of launches that wait."""
    g = _gen(tokens + sizes[1])
    chain = [compact.Tiles([_block((), r, c, 64, False, torch.bfloat16, g)]) for c, r in zip(sizes, sizes[1:])]
    x = torch.randn(tokens, sizes[0], generator=g, device="cuda").bfloat16()
    norm = lambda y: (y.float() / y.float().abs().amax().clamp(min=1)).bfloat16()

    def run(wait):
        y = x
        for tiles in chain:
            y = tiles(y)
            y = tiles(y[:, :tiles.cols]) if y.shape[1] >= tiles.cols else y      # straight after each other
            if wait:
                torch.cuda.synchronize()
            y = norm(y)
        return y
    want = run(True)
    assert all(torch.equal(run(False), want) for _ in range(10))
    from p2pllm_b200 import kernels
    kernels.int4_status()


def test_modules_can_be_copied_and_pickled():
    import copy
    import pickle
    g = _gen(78)
    tiles = compact.Tiles([_block((), 40, 128, 64, True, torch.bfloat16, g)])
    experts = moe.Int4Experts([_block((3,), 40, 128, 64, True, torch.bfloat16, g)])
    x = torch.randn(9, 128, generator=g, device="cuda").bfloat16()
    order = moe.sort_tokens(torch.randint(0, 3, (9, 1), generator=g, device="cuda"), 3)
    for again in (copy.deepcopy, lambda t: pickle.loads(pickle.dumps(t))):
        assert torch.equal(again(tiles)(x), tiles(x))
        assert torch.equal(again(experts)(x, order), experts(x, order))


def test_calls_from_several_threads_at_once():
    """Threads on streams of their own, modules of both kernels and routed experts among them."""
    import threading
    g = _gen(77)
    tiles = [compact.Tiles([_block((), r, c, 64, True, torch.bfloat16, g)]) for r, c in ((640, 2048), (4096, 1024))]
    experts = moe.Int4Experts([_block((16,), 128, 512, 32, False, torch.bfloat16, g)], gated=True)
    xs = [torch.randn(t, q.cols, generator=g, device="cuda").bfloat16() for q in tiles for t in (1, 17, 150)]
    xe, ids = torch.randn(70, 512, generator=g, device="cuda").bfloat16(), torch.randint(-1, 16, (70, 3), generator=g, device="cuda")

    def run():
        ys = [q(x) for q, part in zip(tiles, (xs[:3], xs[3:])) for x in part]
        order = moe.sort_tokens(ids, 16)
        y = experts(xe, order, gather=True)
        return ys + [y, moe.from_experts(y, order)]
    want = run()
    torch.cuda.synchronize()
    got, failed = {}, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                got[i] = [run() for _ in range(10)]
                torch.cuda.current_stream().synchronize()
        except BaseException as e:
            failed.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    assert all(torch.equal(a, b) for rounds in got.values() for ys in rounds for a, b in zip(ys, want))


def test_two_captured_graphs_replay_side_by_side():
    g = _gen(4)
    tiles = compact.Tiles([_block((), 4096, 4096, 128, False, torch.bfloat16, g)])
    xs = [torch.randn(272, 4096, generator=g, device="cuda").bfloat16() for _ in range(2)]
    tiles(xs[0])
    torch.cuda.synchronize()
    graphs, ys = [], []
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ys.append(tiles(x))
        graphs.append(graph)
    for x in xs:
        x.copy_(torch.randn(272, 4096, generator=g, device="cuda"))
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for x, y in zip(xs, ys):
        assert torch.equal(y, tiles(x))


# --- quantising -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("shape", [(3, 1), (5, 31), (2, 64), (7, 129), (2, 3, 200), (300, 512)])
def test_quantised_codes_are_those_of_exact_arithmetic(shape, group, zeros, dtype):
    g = _gen(shape[-1] + group)
    w = (torch.randn(shape, generator=g, device="cuda") * 0.02).to(DT[dtype])
    w[0, ..., :2] = 0
    kind, codes, scales, z, cols, grp = int4.quantize(w, group, zeros)
    assert (kind, cols, grp) == ("int4", shape[-1], group) and codes.shape == (*shape[:-1], -(-cols // 2))
    groups = -(-cols // group)
    pad = torch.zeros(*shape[:-1], groups * group, dtype=torch.float64, device="cuda")
    pad[..., :cols] = w.double()
    pad = pad.view(*shape[:-1], groups, group)
    if zeros:
        lo, hi = pad.amin(-1).clamp(max=0), pad.amax(-1).clamp(min=0)
        s = ((hi - lo) / 15).to(DT[dtype])
        zp = torch.where(s > 0, torch.round(-lo / s.double()).clamp(0, 15), 0.0)
        assert torch.equal(z.double(), zp)
    else:
        s, zp = (pad.abs().amax(-1) / 7).to(DT[dtype]), torch.full(scales.shape, 8.0, dtype=torch.float64, device="cuda")
        assert z is None
    assert torch.equal(scales, s)
    q = torch.where(s.unsqueeze(-1) > 0, torch.round(pad / s.double().unsqueeze(-1)), 0.0) + zp.unsqueeze(-1)
    q = q.clamp(0, 15).flatten(-2)[..., :cols]
    got = torch.stack((codes % 16, codes // 16), dim=-1).flatten(-2)
    assert torch.equal(got[..., :cols].double(), q) and bool((got[..., cols:] == 0).all())


def test_quantised_rows_come_back_within_half_a_scale():
    g = _gen(9)
    w = (torch.randn(64, 1000, generator=g, device="cuda") * 0.02).bfloat16()
    for zeros in (False, True):
        block = int4.quantize(w, 64, zeros)
        back = int4.expand(block)
        assert back.dtype == w.dtype and torch.equal(back, _dense64(block).bfloat16()) and torch.equal(back, compact.expand(block))
        s = block[2].double().repeat_interleave(64, -1)[:, :1000]
        # half a step of the code, or a whole one where the scale's or the zero point's rounding cuts the range's end
        assert bool(((back.double() - w.double()).abs() <= 1.01 * s).all())


def test_a_group_of_zeros_and_a_group_with_nan():
    w = torch.ones(2, 96, dtype=torch.bfloat16, device="cuda")
    w[0, :32], w[1, 40] = 0, float("nan")
    for zeros in (False, True):
        back = int4.expand(int4.quantize(w, 32, zeros))
        assert bool((back[0, :32] == 0).all()) and bool(back[1, 32:64].isnan().all())
        assert bool(back[1, 64:].isfinite().all()) and bool(back[0].isfinite().all())


# --- routed experts ---------------------------------------------------------------------------------------------------

def _ids(tokens, topk, experts, g, nowhere=0.1, favourite=None):
    ids = torch.randint(0, experts, (tokens, topk), generator=g, device="cuda")
    if favourite is not None:
        ids[:, 0] = favourite
    gone = torch.rand(tokens, topk, generator=g, device="cuda") < nowhere
    return torch.where(gone, -1, ids)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("tokens,topk,experts,rows,cols,group,zeros,favourite", [
    (1, 1, 1, 2, 1, 32, False, None), (1, 8, 128, 96, 64, 64, False, None), (3, 2, 4, 34, 130, 32, True, None),
    (17, 8, 16, 64, 320, 128, False, 3), (70, 3, 5, 50, 96, 64, True, 2), (272, 2, 7, 130, 257, 128, True, 0)])
def test_experts_products(tokens, topk, experts, rows, cols, group, zeros, favourite, gather, gated, dtype):
    g = _gen(tokens + experts)
    block = _block((experts,), rows, cols, group, zeros, DT[dtype], g)
    ids = _ids(tokens, topk, experts, g, favourite=favourite)
    order = moe.sort_tokens(ids, experts)
    x = torch.randn(tokens if gather else tokens * topk, cols, generator=g, device="cuda").to(DT[dtype])
    tiles = moe.Int4Experts([block], gated=gated)
    y = tiles(x, order, gather=gather)
    assert y.shape == (tokens * topk, rows // 2 if gated else rows)
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


class TopK(NamedTuple):
    topk_weights: torch.Tensor
    topk_ids: torch.Tensor


class Dispatch(NamedTuple):
    hidden_states: torch.Tensor
    topk_output: TopK


def _moe64(x, ids, weights, w13, w2):
    out = torch.zeros(x.shape[0], w2.shape[1], dtype=torch.float64, device=x.device)
    half = w13.shape[1] // 2
    for e in range(w13.shape[0]):
        t, j = (ids == e).nonzero(as_tuple=True)
        gu = x[t].double() @ w13[e].T
        h = gu[:, :half] * torch.sigmoid(gu[:, :half]) * gu[:, half:]
        out.index_add_(0, t, weights[t, j].double()[:, None] * (h @ w2[e].T))
    return out


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tokens", [0, 1, 17, 272])
def test_a_whole_layer_of_4_bit_experts(tokens, dtype):
    """Sort, gate and up, down, weighted sum, through the layer's quant_method: three roundings to the type (h, the
    experts' rows, the sums), each at most half a step of its value, so below 3 half steps of the result's norm (the
    weights of a token sum to 1, and the products of random signs keep relative errors of their inputs' norm)."""
    g = _gen(tokens)
    E, K, H, R = 16, 4, 256, 192
    blocks = {"w13_weight": [_block((E,), R, H, 64, False, DT[dtype], g), _block((E,), R, H, 64, True, DT[dtype], g)],
              "w2_weight": [_block((E,), H, R, 32, True, DT[dtype], g)]}
    layer = moe.GroupedMoE(None, blocks)
    x = torch.randn(tokens, H, generator=g, device="cuda").to(DT[dtype])
    ids = _ids(tokens, K, E, g)
    weights = torch.rand(tokens, K, generator=g, device="cuda")
    weights /= weights.sum(-1, keepdim=True)
    y = layer.apply(None, Dispatch(x, TopK(weights, ids)))
    assert y.shape == (tokens, H) and y.dtype == DT[dtype]
    if tokens:
        w13 = torch.cat([_dense64(b) for b in blocks["w13_weight"]], dim=1)
        want = _moe64(x, ids, weights, w13, _dense64(blocks["w2_weight"][0]))
        assert float((y.double() - want).norm() / want.norm()) <= 3 * torch.finfo(DT[dtype]).eps / 2
    expanded = [("dense", compact.expand(b)) for b in blocks["w13_weight"]]
    assert torch.equal(compact.expand(blocks["w2_weight"][0], torch.tensor([3, 1], device="cuda")),
                       compact.expand(blocks["w2_weight"][0])[[3, 1]]) and expanded[0][1].shape == (E, R, H)


def test_a_layer_of_4_bit_experts_is_captured_and_replayed():
    g = _gen(11)
    E, K, H, R, T = 32, 8, 128, 64, 33
    layer = moe.GroupedMoE(None, {"w13_weight": [_block((E,), 2 * R, H, 128, False, torch.bfloat16, g)],
                                  "w2_weight": [_block((E,), H, R, 64, False, torch.bfloat16, g)]})
    x = torch.randn(T, H, generator=g, device="cuda").bfloat16()
    ids = _ids(T, K, E, g).int()
    weights = torch.rand(T, K, generator=g, device="cuda")
    layer.apply(None, Dispatch(x, TopK(weights, ids)))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer.apply(None, Dispatch(x, TopK(weights, ids)))
    for k in range(3):
        x.copy_(torch.randn(T, H, generator=g, device="cuda"))
        ids.copy_(_ids(T, K, E, g, nowhere=0.3 * k, favourite=k))
        graph.replay()
        assert torch.equal(y, layer.apply(None, Dispatch(x, TopK(weights, ids))))


# --- modules and files ------------------------------------------------------------------------------------------------

def test_compact_applies_a_4_bit_module():
    g = _gen(6)
    block = _block((), 48, 128, 64, True, torch.bfloat16, g)
    method = compact.Compact([block])
    x = torch.randn(2, 5, 128, generator=g, device="cuda").bfloat16()
    bias = torch.randn(48, generator=g, device="cuda").bfloat16()
    y = method.apply(None, x, bias)
    assert y.shape == (2, 5, 48) and torch.equal(y, method.apply(None, x) + bias)
    assert method.nbytes() == method.tiles.nbytes() == 8192 + 2 * (256 + 128)     # one unit of 128 x 128 weights


@pytest.mark.parametrize("zero_points", [False, True])
def test_4_bit_replica_files_install(replica_golden, tmp_path, zero_points):
    from conftest import REPLICA_SIZES, replica_model
    model = replica_model(replica_golden, "cuda")
    paths = prepare.write_int4(model.layers, [0], str(tmp_path), group=32, zero_points=zero_points)
    assert paths == [str(tmp_path / "layer0.safetensors")]
    dense = replica_model(replica_golden, "cuda")
    assert prepare.install_replica(dense, paths[0], form="dense")["int4"] == {"group": 32}
    prepare.install_replica(model, paths[0])
    g = _gen(8)
    for path, (sizes, cols) in REPLICA_SIZES.items():
        module = model.layers[0].get_submodule(path)
        want = dense.layers[0].get_submodule(path).weight
        original = replica_model(replica_golden, "cuda").layers[0].get_submodule(path).weight
        assert module.quant_method.tiles.layout == "int4" and module.weight.shape == (sum(sizes), 0)
        assert torch.equal(want, int4.expand(int4.quantize(original, 32, zero_points)))
        x = torch.randn(17, cols, generator=g, device="cuda").bfloat16()
        w = _dense64(int4.quantize(original, 32, zero_points))
        _check_product(module(x), x, w, torch.bfloat16)


# --- refusals ---------------------------------------------------------------------------------------------------------

def test_calls_that_do_not_fit_are_refused():
    g = _gen(7)
    block = _block((), 32, 128, 64, True, torch.bfloat16, g)
    tiles = compact.Tiles([block])
    x = torch.randn(4, 128, generator=g, device="cuda").bfloat16()
    for bad, needle in ((x.half(), "the weights"), (x[:, :64], "128 columns"), (x.cpu(), "CUDA"), (x[0], "128 columns")):
        with pytest.raises(P2PError, match=needle):
            tiles(bad)
    with pytest.raises(P2PError, match="gradient"):
        tiles(x.clone().requires_grad_(True))
    with torch.no_grad():
        assert torch.equal(tiles(x.clone().requires_grad_(True)), tiles(x))
    with pytest.raises(P2PError, match="out of"):
        tiles(x, out=torch.empty(4, 31, dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(P2PError, match="whole module"):
        compact.Tiles([block, ("dense", torch.zeros(4, 128, dtype=torch.bfloat16, device="cuda"))])
    with pytest.raises(P2PError, match="whole module"):
        compact.Tiles([block], layout="tc")
    with pytest.raises(P2PError, match="same columns"):
        compact.Tiles([block, _block((), 4, 64, 64, True, torch.bfloat16, g)])
    with pytest.raises(P2PError, match="whole module"):
        compact.GatedTiles([block, ("dense", torch.zeros(32, 128, dtype=torch.bfloat16, device="cuda"))])
    with pytest.raises(P2PError, match="gate rows"):
        compact.GatedTiles([_block((), 33, 128, 64, True, torch.bfloat16, g)])
    kind, codes, scales, zeros, cols, group = block
    for bad, needle in (((kind, codes[:, 1:], scales, zeros, cols, group), "do not hold"),
                        ((kind, codes, scales[:, 1:], zeros, cols, group), "wanted"),
                        ((kind, codes, scales, zeros.int(), cols, group), "wanted"),
                        ((kind, codes, scales.float(), zeros, cols, group), "bfloat16 or float16"),
                        ((kind, codes, scales, zeros, cols, 48), "32, 64 or 128"),
                        ((kind, codes, scales, zeros, cols), "not a 4-bit block")):
        with pytest.raises(P2PError, match=needle):
            int4.expand(bad)
    with pytest.raises(P2PError, match="bfloat16 or float16"):
        int4.quantize(torch.zeros(4, 64, device="cuda"))


def test_expert_calls_that_do_not_fit_are_refused():
    g = _gen(12)
    block = _block((4,), 32, 64, 64, False, torch.bfloat16, g)
    tiles = moe.Int4Experts([block])
    order = moe.sort_tokens(torch.zeros(3, 2, dtype=torch.int64, device="cuda"), 4)
    x = torch.zeros(6, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(P2PError, match="wanted"):
        tiles(x, order, gather=True)
    with pytest.raises(P2PError, match="wanted"):
        tiles(x[:3], order)
    with pytest.raises(P2PError, match="experts"):
        tiles(x, moe.sort_tokens(torch.zeros(3, 2, dtype=torch.int64, device="cuda"), 5))
    with pytest.raises(P2PError, match="expert dimension"):
        moe.Int4Experts([_block((), 32, 64, 64, False, torch.bfloat16, g)])
    with pytest.raises(P2PError, match="gate rows"):
        moe.Int4Experts([_block((4,), 31, 64, 64, False, torch.bfloat16, g)], gated=True)
    with pytest.raises(P2PError, match="all 4-bit or none"):
        moe.GroupedMoE(None, {"w13_weight": [block], "w2_weight": [("dense", torch.zeros(4, 64, 16, dtype=torch.bfloat16, device="cuda"))]})
    with pytest.raises(P2PError, match="do not match"):
        moe.GroupedMoE(None, {"w13_weight": [block], "w2_weight": [block]})


# --- nothing to do, and a lot -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("tokens", [0, 1, 5, 60, 700])
def test_no_pair_has_an_expert(tokens):
    """Rows behind the last pair, which are all of them: zero, or in a given output as they were."""
    g = _gen(21)
    up = moe.Int4Experts([_block((4,), 64, 96, 32, True, torch.bfloat16, g)], gated=True)
    x = torch.randn(tokens, 96, generator=g, device="cuda").bfloat16()
    order = moe.sort_tokens(torch.full((tokens, 2), 4, device="cuda"), 4)
    assert int(order.n_items) == 0 and bool((order.where == -1).all()) and bool((order.order == -1).all())
    y = up(x, order, gather=True)
    assert y.shape == (tokens * 2, 32) and bool((y == 0).all())
    out = torch.full((tokens * 2, 32), 7.0, dtype=torch.bfloat16, device="cuda")
    assert bool((up(x, order, gather=True, out=out) == 7).all())
    back = moe.from_experts(y, order, torch.ones(tokens, 2, device="cuda"))
    assert back.shape == (tokens, 32) and bool((back == 0).all())
    assert compact.Tiles([_block((), 10, 96, 32, True, torch.bfloat16, g)])(x[:0]).shape == (0, 10)


def test_some_rows_of_a_given_output_stay():
    g = _gen(22)
    for tokens in (6, 400):
        experts = moe.Int4Experts([_block((8,), 48, 128, 64, False, torch.float16, g)])
        ids = _ids(tokens, 3, 8, g, nowhere=0.5)
        order = moe.sort_tokens(ids, 8)
        routed = int(order.offsets[-1])
        x = torch.randn(tokens, 128, generator=g, device="cuda").half()
        out = torch.full((tokens * 3, 48), 7.0, dtype=torch.float16, device="cuda")
        y = experts(x, order, gather=True)
        experts(x, order, gather=True, out=out)
        assert torch.equal(out[:routed], y[:routed]) and bool((out[routed:] == 7).all()) and bool((y[routed:] == 0).all())


def test_outputs_past_32_bits():
    """y of 2.3e9 elements: its last rows are those of a call of their own."""
    g = _gen(23)
    block = _block((), 28672, 128, 128, False, torch.bfloat16, g)
    x = torch.randn(80000, 128, generator=g, device="cuda").bfloat16()
    tiles = compact.Tiles([block])
    y = tiles(x)
    _check_product(y[-40:], x[-40:], _dense64(block), torch.bfloat16)
    _check_product(y[74880:74910], x[74880:74910], _dense64(block), torch.bfloat16)      # around element 2^31


@pytest.mark.parametrize("tokens", [1, 300])
def test_experts_past_32_bits_of_weights(tokens):
    """4.4 GB of layout: the last expert and the first one."""
    g = _gen(24)
    E, R, C = 520, 4096, 4096
    block = _block((E,), R, C, 128, False, torch.bfloat16, g)
    experts = moe.Int4Experts([block])
    assert experts.nbytes() > 2 ** 32
    ids = torch.tensor([[E - 1, 0]], device="cuda").expand(tokens, 2)
    x = torch.randn(tokens, C, generator=g, device="cuda").bfloat16()
    order = moe.sort_tokens(ids, E)
    y = moe.from_experts(experts(x, order, gather=True), order, torch.tensor([[1.0, 0.0]], device="cuda").expand(tokens, 2))
    for e, got in ((E - 1, y), (0, experts(x, order, gather=True)[:tokens])):
        one = tuple(t[e] if torch.is_tensor(t) else t for t in block)
        _check_product(got, x, _dense64(one), torch.bfloat16)
