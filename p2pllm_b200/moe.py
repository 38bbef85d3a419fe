"""Routed experts run compact: a FusedMoE quant_method that multiplies the experts' pruned weights where they lie,
instead of expanding every used expert to dense on every pass (p2p/compact.py:227-262, CompactMoE).

    ExpertTiles   one routed-expert tensor (row blocks with a leading expert dimension) in one tensor-core layout,
                  each expert starting on a 128-row tile
    Int4Experts   the same for 4-bit blocks (int4.py)
    GroupedMoE    quant_method.apply(layer, dispatch_output): gated-SiLU experts (w13 = gate then up, w2 = down)

and the tokens' way to the experts and back without a word to the host, so that a pass can be captured into a CUDA
graph, and with gradients, so that experts of any kind can be trained between the two:

    sort_tokens   ids [T, K] -> TokenOrder: the (token, slot) pairs sorted by expert
    to_experts    x [T, H] -> [T K, H]: the tokens' rows in that order
    from_experts  y [T K, H] -> [T, H]: each token's rows, weighted and added in slot order

A pass: one kernel (p2p_moe_route) sorts the routed (token, slot) pairs by expert (stable) and writes the grouped
GEMM's items; x's rows are gathered in that order; one grouped launch of the compact GEMM (p2p_spmm_tc_grouped_gated:
a CTA takes one row tile of one expert's run of up to 256 tokens, the expert's gate and up rows interleaved 64 and 64
so that its epilogue writes SiLU(gate) * up, in fp32 from the rounded outputs, rounded to x's dtype); a second grouped
launch gives down; p2p_moe_combine weights each token's outputs by its routing
weights and adds them in slot order in fp32 (deterministic). Three numbers (pairs, items, the largest item) are read
back once a pass to size the launches (the reference's CompactMoE also syncs, on torch.unique).
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib, int4, kernels
from ._lib import P2PError, call, dtype_code, ptr, require_cuda, stream_of
from .compact import _cols, gate_up_rows, to_compact

ITEM_TOKENS = 256                       # tokens one grouped CTA takes (an accumulator of at most 256 columns)


class ExpertTiles(kernels.Settled):
    """A routed-expert tensor [E, rows, cols] from its row blocks (each ("dense", W [E, r, C]) or ("sparse" |
    "compact", values [E, r, k], words | idx [E, r, ...], C), in row order), laid out for the grouped GEMM: expert
    e's rows start at row tile e * item_row_tiles. Built once at load (one layout build an expert)."""

    def __init__(self, blocks: list, gated: bool = False):
        self.gated = gated
        if gated:                               # gate rows then up rows, interleaved: one compact (or dense) block
            values, idx = gate_up_rows(blocks)
            blocks = [("compact", values, idx, _cols(blocks[0])) if idx is not None else ("dense", values)]
        blocks = [to_compact(b) for b in blocks]
        self.cols = _cols(blocks[0])
        self.experts = blocks[0][1].shape[0]
        self.rows = sum(b[1].shape[-2] for b in blocks)
        self.dtype, self.device = blocks[0][1].dtype, blocks[0][1].device
        if self.dtype not in (torch.bfloat16, torch.float16) or self.cols % 8:
            raise P2PError("grouped experts need bf16 / f16 weights with columns in multiples of 8")
        self.item_row_tiles = -(-self.rows // 128)
        words, segs, base = [], [], 0
        for e in range(self.experts):
            row_blocks, row0 = [], 0
            for b in blocks:
                v = b[1][e].contiguous()
                idx = b[2][e].contiguous() if b[0] == "compact" else None
                row_blocks.append((row0, v, idx))
                row0 += v.shape[0]
            w, seg, _ = kernels.tiles_build(row_blocks, self.cols)
            total = int(seg[-1].item())
            words.append(w[:total])
            segs.append(seg[:-1] + base)
            base += total
        self.words = torch.cat(words) if base else torch.zeros(4, dtype=torch.int32, device=self.device)
        self.seg = torch.cat(segs + [torch.tensor([base], dtype=torch.int64, device=self.device)])
        self.seg_cap = int((self.seg[1:] - self.seg[:-1]).max().item())
        self.layout_row_tiles = self.experts * self.item_row_tiles

    def __call__(self, x: torch.Tensor, items: torch.Tensor, max_tokens: int, out: torch.Tensor) -> torch.Tensor:
        """out [P, rows] rows s.. of an item = x rows s.. times the item's expert (items: int32 [n, 4] on the GPU);
        gated: out [P, rows / 2] = dtype(silu(gate) * up) of them, applied in the GEMM's epilogue."""
        call("p2p_spmm_tc_grouped_gated" if self.gated else "p2p_spmm_tc_grouped", ptr(x), dtype_code(x), x.shape[0], self.cols, x.stride(0), ptr(self.words),
             ptr(self.seg), self.layout_row_tiles, self.rows, self.item_row_tiles, self.seg_cap, ptr(items),
             items.shape[0], max_tokens, ptr(out), out.stride(0), stream_of(x))
        if kernels.CHECK_WAITS:
            kernels.spmm_tc_status(x.device)
        return out

    def gated_sums(self, x: torch.Tensor, items: torch.Tensor, max_tokens: int, out: torch.Tensor) -> torch.Tensor:
        """out [n_items, rows / 2] fp32: per item, the column sums over its tokens of (silu(g) * u)^2, g and u this
        gated layout's unrounded products (p2p_spmm_tc_grouped_gated_sums)."""
        if not self.gated:
            raise P2PError("gated sums need the interleaved gate / up layout")
        call("p2p_spmm_tc_grouped_gated_sums", ptr(x), dtype_code(x), x.shape[0], self.cols, x.stride(0),
             ptr(self.words), ptr(self.seg), self.layout_row_tiles, self.rows, self.item_row_tiles, self.seg_cap,
             ptr(items), items.shape[0], max_tokens, ptr(out), out.stride(0), stream_of(x))
        return out

    def nbytes(self) -> int:
        return self.words.numel() * 4 + self.seg.numel() * 8


def route(ids: torch.Tensor, experts: int) -> dict:
    """The pass's routing on the GPU (p2p_moe_route): order [P] (pairs sorted by expert, stable), where [T K] (each
    pair's place, -1 if routed nowhere), counts [E], items [n, 4] ({expert, first place, places, 0}), and on the host
    P, the item count and the largest item."""
    require_cuda(ids)
    flat = ids.reshape(-1).to(torch.int64).contiguous()
    n = flat.numel()
    dev = flat.device
    max_items = -(-n // ITEM_TOKENS) + experts
    order = torch.empty(max(n, 1), dtype=torch.int64, device=dev)
    where = torch.empty(max(n, 1), dtype=torch.int64, device=dev)
    counts = torch.empty(experts, dtype=torch.int32, device=dev)
    items = torch.empty(max_items, 4, dtype=torch.int32, device=dev)
    meta = torch.empty(3, dtype=torch.int64, device=dev)
    call("p2p_moe_route", ptr(flat), n, experts, ptr(order), ptr(where), ptr(counts), ptr(items), max_items, ptr(meta),
         stream_of(flat))
    pairs, n_items, most = meta.tolist()
    return {"order": order[:pairs], "where": where[:n], "counts": counts, "items": items[:n_items], "most": most}


@dataclass
class TokenOrder:
    """A pass's routed (token, slot) pairs sorted by expert, those of one expert in their own order; all on the GPU.
    Of the T K places the first offsets[-1] hold a pair."""
    order: torch.Tensor           # int32 [T K]: the pair token * K + slot at each place, -1 behind the last
    where: torch.Tensor           # int32 [T K]: each pair's place, -1 if it is routed nowhere
    offsets: torch.Tensor         # int32 [experts + 1]: each expert's first place, then the number of routed pairs
    items: torch.Tensor           # int32 [4 n]: n of {expert, first place, places, 0}, runs of one expert's places
    n_items: torch.Tensor         # int32 [1]
    tokens: int
    topk: int

    @property
    def experts(self) -> int:
        return self.offsets.numel() - 1

    @property
    def device(self) -> torch.device:
        return self.order.device


def sort_tokens(ids: torch.Tensor, experts: int) -> TokenOrder:
    """The order of ids [T, K] (int32 or int64 expert ids; any id outside 0..experts - 1 is routed nowhere). One launch,
    nothing read back; at most 1024 experts. The same expert may come up twice in a row: two pairs."""
    require_cuda(ids)
    if ids.dim() != 2 or ids.shape[1] < 1 or ids.dtype not in (torch.int32, torch.int64):
        raise P2PError(f"ids of {tuple(ids.shape)} {ids.dtype}: int32 or int64 [tokens, slots]")
    if not 1 <= experts <= 1024:
        raise P2PError(f"{experts} experts: 1 to 1024")
    return TokenOrder(*_lib.ops().moe_sort(ids, experts), ids.shape[0], ids.shape[1])


def _check_rows(t: torch.Tensor, order: TokenOrder, rows: int) -> None:
    require_cuda(t)
    if t.dim() != 2 or t.shape[0] != rows or t.device != order.device:
        raise P2PError(f"rows of {tuple(t.shape)} on {t.device}, wanted [{rows}, ..] on {order.device}")
    dtype_code(t)


def to_experts(x: torch.Tensor, order: TokenOrder) -> torch.Tensor:
    """[T K, H]: x's rows in the order's places, zero behind the last pair. bfloat16, float16 or float32. The gradient
    of x is the sum over its slots, in slot order and fp32."""
    try:                                            # the operator makes the same checks, at less cost
        return _lib.ops().moe_spread(x, order.where, order.offsets, order.topk)
    except RuntimeError:
        _check_rows(x, order, order.tokens)
        raise


def from_experts(y: torch.Tensor, order: TokenOrder, weights: torch.Tensor | None = None) -> torch.Tensor:
    """[T, H]: per token the sum over its slots, in slot order and fp32, of weights[t, j] times the slot's row of
    y [T K, H] (no weights: 1); slots routed nowhere add nothing. Gradients for y (zero behind the last pair) and for
    weights [T, K] (bfloat16, float16 or float32)."""
    try:                                            # the operator makes the same checks, at less cost
        return _lib.ops().moe_sum(y, order.where, order.offsets, weights, order.topk)
    except RuntimeError:
        _check_rows(y, order, order.tokens * order.topk)
        if weights is not None:
            require_cuda(weights)
            if tuple(weights.shape) != (order.tokens, order.topk) or weights.device != order.device:
                raise P2PError(f"weights of {tuple(weights.shape)} on {weights.device}, wanted "
                               f"{(order.tokens, order.topk)} on {order.device}") from None
            dtype_code(weights)
        raise


class Int4Experts:
    """A routed-expert tensor [E, rows, cols] from 4-bit row blocks with a leading expert dimension, laid out once at
    load. Calling it multiplies a sorted pass: with gather the rows of x [T, cols] go to the order's places as they are
    read, without it x [T K, cols] lies in that order already. Returns [T K, rows], gated [T K, rows / 2] =
    dtype(silu(gate) * up). Rows behind the last pair are zero, or in a given `out` left as they were. Nothing is read
    back. Inference only."""

    def __init__(self, blocks: list, gated: bool = False):
        self.int4 = int4.Layout(blocks, gated)
        if blocks[0][1].dim() != 3:
            raise P2PError("routed experts' blocks have a leading expert dimension")
        if self.int4.experts > 1024:
            raise P2PError(f"{self.int4.experts} experts: 1 to 1024")
        self.gated, self.experts = gated, self.int4.experts
        self._op = _lib.ops().int4_grouped
        self.rows, self.cols, self.dtype, self.device = (self.int4.rows, self.int4.cols, self.int4.dtype,
                                                         self.int4.device)

    def __getstate__(self) -> dict:
        return {k: v for k, v in self.__dict__.items() if k != "_op"}          # an operator cannot be pickled

    def __setstate__(self, state: dict) -> None:
        self.__dict__.update(state)
        self._op = _lib.ops().int4_grouped

    def __call__(self, x: torch.Tensor, order: TokenOrder, gather: bool = False,
                 out: torch.Tensor | None = None) -> torch.Tensor:
        q = self.int4
        if out is None and x.dtype is q.dtype:
            try:                                    # the operator makes the same checks, at less cost
                out = self._op(x, q.data, q.has_zeros, q.experts, q.rows, q.cols, q.group, q.gated, order.order,
                               order.where, order.offsets, order.items, order.n_items, order.topk, gather)
            except RuntimeError:
                self._check(x, order, gather)
                raise
        else:
            self._check(x, order, gather)
            out = kernels._out(out, (order.tokens * order.topk, q.rows // 2 if q.gated else q.rows), x)
            _lib.ops().int4_grouped_into(x, q.data, q.has_zeros, q.experts, q.rows, q.cols, q.group, q.gated,
                                         order.order, order.where, order.offsets, order.items, order.n_items,
                                         order.topk, gather, out)
        if kernels.CHECK_WAITS:
            kernels.int4_status(x.device)
        return out

    def _check(self, x: torch.Tensor, order: TokenOrder, gather: bool) -> None:
        self.int4.check_x(x)
        _check_rows(x, order, order.tokens if gather else order.tokens * order.topk)
        if order.experts != self.experts:
            raise P2PError(f"an order of {order.experts} experts, weights of {self.experts}")

    def nbytes(self) -> int:
        return self.int4.nbytes()


class GroupedMoE(torch.nn.Module):
    """A FusedMoE's quant_method for compact routed experts, gated SiLU: weights {"w13_weight": blocks of [E, 2R, H]
    (gate rows, then up rows), "w2_weight": blocks of [E, H, R]}, all of them 4-bit blocks or none. apply(layer,
    dispatch_output) returns the layer's output [T, H] in x's dtype. Other attributes are the layer's own method's."""

    is_int4 = False                 # also of layers pickled before there were 4-bit blocks

    def __init__(self, method, weights: dict):
        super().__init__()
        self.method = method
        two_r = sum(b[1].shape[-2] for b in weights["w13_weight"])
        kinds = {b[0] == "int4" for blocks in weights.values() for b in blocks}
        if len(kinds) > 1:
            raise P2PError("routed experts are all 4-bit or none of them")
        self.is_int4 = kinds == {True}
        if self.is_int4:
            self.w13 = Int4Experts(weights["w13_weight"], gated=True)
            self.w2 = Int4Experts(weights["w2_weight"])
            self._check()
            return
        # SiLU(gate) * up inside the gate/up launch when the rows allow it (R a multiple of 64, one k)
        try:
            self.w13 = ExpertTiles(weights["w13_weight"], gated=two_r % 128 == 0)
        except P2PError:
            self.w13 = ExpertTiles(weights["w13_weight"])
        self.w2 = ExpertTiles(weights["w2_weight"])
        self._check()

    def _check(self) -> None:
        if self.w13.rows % 2 or self.w2.cols != self.w13.rows // 2 or self.w2.rows != self.w13.cols:
            raise P2PError("w13 [E, 2R, H] and w2 [E, H, R] do not match")

    def __getattr__(self, name):
        try:
            return super().__getattr__(name)
        except AttributeError:
            return getattr(super().__getattr__("method"), name)

    def apply(self, layer, dispatch_output):
        x = dispatch_output.hidden_states
        topk = dispatch_output.topk_output
        ids, weights = topk.topk_ids, topk.topk_weights
        T, K = ids.shape
        x2 = x.reshape(-1, x.shape[-1])
        if x2.dtype != self.w13.dtype:
            raise P2PError(f"x is {x2.dtype}, the experts {self.w13.dtype}")
        if self.is_int4:                            # four to seven launches, no read back: the pass can be captured
            order = sort_tokens(ids if ids.dtype in (torch.int32, torch.int64) else ids.long(), self.w13.experts)
            down = self.w2(self.w13(x2, order, gather=True), order)
            return from_experts(down, order, weights).reshape(*x.shape[:-1], self.w2.rows)
        r = route(ids, self.w13.experts)
        P = r["order"].numel()
        out = torch.empty(T, self.w2.rows, dtype=x2.dtype, device=x.device)
        if P == 0:
            return out.zero_().reshape(*x.shape[:-1], self.w2.rows)
        xs = x2.index_select(0, r["order"] // K).contiguous()
        R = self.w13.rows // 2
        if self.w13.gated:
            h = self.w13(xs, r["items"], r["most"], torch.empty(P, R, dtype=x2.dtype, device=x.device))
        else:
            gu = self.w13(xs, r["items"], r["most"], torch.empty(P, self.w13.rows, dtype=x2.dtype, device=x.device))
            h = (torch.nn.functional.silu(gu[:, :R].float()) * gu[:, R:].float()).to(x2.dtype).contiguous()
        down = self.w2(h, r["items"], r["most"], torch.empty(P, self.w2.rows, dtype=x2.dtype, device=x.device))
        w = weights.reshape(-1).float().contiguous()
        call("p2p_moe_combine", ptr(down), dtype_code(down), down.stride(0), ptr(r["where"]), ptr(w), T, K,
             self.w2.rows, ptr(out), out.stride(0), stream_of(down))
        return out.reshape(*x.shape[:-1], self.w2.rows)

    def process_weights_after_loading(self, layer) -> None:
        pass

    def nbytes(self) -> int:
        return self.w13.nbytes() + self.w2.nbytes()
