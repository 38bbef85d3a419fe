"""Replica weights in 4 bits with group scales, the other small storage of a replica beside pruning: 0.5 bytes a weight
and a scale for every `group` columns of a row, against 0.85 bytes for keep 36 with a bitmask. p2pLLM has no counterpart
(p2p/compact.py stores pruned rows, 16 bits a kept weight); blocks of this kind go wherever that module's blocks go.

    ("int4", codes, scales, zeros, cols, group)      a row block
        codes   [.., rows, ceil(cols / 2)] uint8, the even column in the low half of a byte
        scales  [.., rows, ceil(cols / group)] in the weights' dtype (bfloat16 or float16), group 32, 64 or 128
        zeros   the same shape, uint8 0..15, or None: 8 everywhere
    W[r, c] = (code[r, c] - zero[r, c // group]) * scale[r, c // group]

    quantize(w)   a block from dense rows            expand(block)   the dense rows it stands for
    Layout        blocks in the layout that the products read (csrc/int4.cuh); compact.Tiles and moe.Int4Experts hold one
"""
from __future__ import annotations

import torch
import torch.autograd.forward_ad as fwAD

from . import _lib, kernels
from ._lib import P2PError, call, dtype_code, ptr, require_cuda, stream_of

__all__ = ["GROUPS", "quantize", "expand", "Layout"]

GROUPS = (32, 64, 128)


def _check_group(group: int) -> None:
    if group not in GROUPS:
        raise P2PError(f"groups of {group} columns: 32, 64 or 128")


def quantize(w: torch.Tensor, group: int = 128, zero_points: bool = False) -> tuple:
    """The ("int4", codes, scales, zeros, cols, group) block of dense rows w [.., rows, cols] (bfloat16 or float16).
    Without zero points a group's scale is max|w| / 7 and its codes reach from -8 to 7 around 8; with them the scale is
    the group's range (which takes in 0) over 15 and the zero point is where 0 falls. Scales are rounded to w's dtype,
    codes to the nearest. Weights are finite; a NaN makes its group NaN."""
    require_cuda(w)
    _check_group(group)
    if w.dtype not in (torch.bfloat16, torch.float16) or w.dim() < 2 or w.shape[-1] < 1:
        raise P2PError(f"4 bits hold bfloat16 or float16 rows of at least one column, not {w.dtype} {tuple(w.shape)}")
    lead, cols = w.shape[:-1], w.shape[-1]
    rows = w.reshape(-1, cols)
    if rows.stride(-1) != 1 or (rows.shape[0] > 1 and rows.stride(0) < cols):
        rows = rows.contiguous()
    groups = -(-cols // group)
    codes = torch.empty(*lead, -(-cols // 2), dtype=torch.uint8, device=w.device)
    scales = torch.empty(*lead, groups, dtype=w.dtype, device=w.device)
    zeros = torch.empty(*lead, groups, dtype=torch.uint8, device=w.device) if zero_points else None
    with torch.cuda.device(w.device):
        call("p2p_int4_quantize", ptr(rows), dtype_code(rows), rows.shape[0], cols, max(rows.stride(0), cols), group,
             ptr(codes), ptr(scales), ptr(zeros), stream_of(w))
    return ("int4", codes, scales, zeros, cols, group)


def check_block(block: tuple) -> tuple:
    """(codes, scales, zeros, cols, group) of a block, its shapes and types checked."""
    if len(block) != 6 or block[0] != "int4":
        raise P2PError(f"not a 4-bit block: {block[0]!r} of {len(block)} entries")
    _, codes, scales, zeros, cols, group = block
    _check_group(group)
    require_cuda(codes, scales, zeros)
    if codes.dtype != torch.uint8 or scales.dtype not in (torch.bfloat16, torch.float16):
        raise P2PError(f"4-bit codes are uint8 and their scales bfloat16 or float16, not {codes.dtype}, {scales.dtype}")
    if codes.dim() not in (2, 3) or cols < 1 or codes.shape[-1] != -(-cols // 2):
        raise P2PError(f"codes of {tuple(codes.shape)} do not hold rows of {cols} columns")
    want = (*codes.shape[:-1], -(-cols // group))
    if tuple(scales.shape) != want or (zeros is not None and (tuple(zeros.shape) != want or zeros.dtype != torch.uint8)):
        raise P2PError(f"scales (and uint8 zero points) of {tuple(scales.shape)}, wanted {want}")
    if codes.device != scales.device or (zeros is not None and zeros.device != codes.device):
        raise P2PError("codes, scales and zero points lie on one device")
    return codes, scales, zeros, cols, group


def check_zeros(zeros: torch.Tensor | None) -> None:
    """Zero points are codes, 0..15: a larger one is refused. Reads one number back: for load time."""
    if zeros is not None and zeros.numel() and int(zeros.max()) > 15:
        raise P2PError(f"4-bit zero points are 0 to 15, not {int(zeros.max())}")


def expand(block: tuple, experts=None) -> torch.Tensor:
    """The dense rows [.., rows, cols] that a block stands for, in its scales' dtype; of routed experts only `experts`,
    which is done in every pass and leaves the check of the zero points to who keeps the block."""
    codes, scales, zeros, cols, group = check_block(block)
    if experts is None:
        if zeros is not None and not torch.cuda.is_current_stream_capturing():
            check_zeros(zeros)
    else:
        codes, scales, zeros = codes[experts], scales[experts], None if zeros is None else zeros[experts]
    codes, scales, zeros = codes.contiguous(), scales.contiguous(), None if zeros is None else zeros.contiguous()
    dense = torch.empty(*codes.shape[:-1], cols, dtype=scales.dtype, device=scales.device)
    rows = dense.numel() // cols
    with torch.cuda.device(codes.device):
        call("p2p_int4_expand", ptr(codes), ptr(scales), ptr(zeros), dtype_code(scales), rows, cols, group, ptr(dense),
             stream_of(codes))
    return dense


class Layout(kernels.Settled):
    """Row blocks of one module (or, with a leading expert dimension, of one routed-expert tensor) in the layout of
    csrc/int4.cuh, built once at load. gated: the first half of the rows is the gate, the second half the up
    projection, and the products return silu(gate) * up.

    The products add a group's codes times x in fp32 and scale that sum, so the sum itself (up to 15 times the group's
    absolute x) has to stay below fp32's largest value. They may read the weights before the stream's previous kernel
    has ended: who rewrites `data` on the GPU waits for that (as building it does) before the next product."""

    def __init__(self, blocks: list, gated: bool = False):
        if not blocks:
            raise P2PError("a module needs at least one row block")
        parts = [check_block(b) for b in blocks]
        for p in parts:
            check_zeros(p[2])
        codes, scales, zeros, cols, group = parts[0]
        for c, s, _, n, g in parts[1:]:
            if (n, g, s.dtype, c.dim(), c.device) != (cols, group, scales.dtype, codes.dim(), codes.device) or \
                    c.shape[:-2] != codes.shape[:-2]:
                raise P2PError("every 4-bit block of a module has the same columns, groups, dtype, experts and device")
        if len(parts) > 1:
            if any(p[2] is not None for p in parts):           # blocks without zero points have 8
                zeros = torch.cat([torch.full(p[1].shape, 8, dtype=torch.uint8, device=codes.device)
                                   if p[2] is None else p[2] for p in parts], dim=-2)
            codes, scales = torch.cat([p[0] for p in parts], dim=-2), torch.cat([p[1] for p in parts], dim=-2)
        self.experts = codes.shape[0] if codes.dim() == 3 else 1
        self.rows, self.cols, self.group, self.gated = codes.shape[-2], cols, group, gated
        self.dtype, self.device = scales.dtype, scales.device
        if self.rows == 0 or self.experts == 0:
            raise P2PError("a 4-bit module needs at least one row")
        self.has_zeros = zeros is not None
        nbytes = _lib.load().p2p_int4_layout_bytes(self.experts, self.rows, cols, group, self.has_zeros, gated)
        if nbytes < 0:
            raise P2PError(f"a gated module has as many gate rows as up rows, not {self.rows} in all")
        self._op = _lib.ops().int4_mm
        # bytes in a tensor of the weights' dtype (a whole number of them), by which the operators know what they multiply
        self.data = torch.empty(nbytes // 2, dtype=self.dtype, device=self.device)
        codes, scales, zeros = codes.contiguous(), scales.contiguous(), None if zeros is None else zeros.contiguous()
        with torch.cuda.device(self.device):
            call("p2p_int4_layout", ptr(codes), ptr(scales), ptr(zeros), self.experts, self.rows, cols, group,
                 int(gated), ptr(self.data), stream_of(codes))
        kernels.settle(self.data)

    def __getstate__(self) -> dict:
        return {k: v for k, v in self.__dict__.items() if k != "_op"}          # an operator cannot be pickled

    def __setstate__(self, state: dict) -> None:
        super().__setstate__(state)
        if self.data.dtype == torch.uint8:                     # pickled when data was plain bytes
            self.data = self.data.view(self.dtype)
        self._op = _lib.ops().int4_mm

    def check_x(self, x: torch.Tensor) -> None:
        require_cuda(x)
        if x.dtype != self.dtype:
            raise P2PError(f"x is {x.dtype}, the weights {self.dtype}")
        if x.device != self.device:
            raise P2PError(f"x lies on {x.device}, the weights on {self.device}")
        if x.dim() != 2 or x.shape[1] != self.cols:
            raise P2PError(f"x of {tuple(x.shape)} does not have {self.cols} columns")
        if (x.requires_grad and torch.is_grad_enabled()) or fwAD.unpack_dual(x).tangent is not None:
            raise P2PError("4-bit weights are for inference: x must not need a gradient")

    def mm(self, x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """x [T, cols] W^T: [T, rows], gated [T, rows / 2] (p2p_int4_mm through the torch operator)."""
        if out is None and x.dtype is self.dtype:
            try:                                               # the operator makes the same checks, at less cost
                out = self._op(x, self.data, self.has_zeros, self.rows, self.cols, self.group, self.gated)
            except RuntimeError:
                self.check_x(x)
                raise
        else:
            self.check_x(x)
            out = kernels._out(out, (x.shape[0], self.rows // 2 if self.gated else self.rows), x)
            _lib.ops().int4_mm_into(x, self.data, self.has_zeros, self.rows, self.cols, self.group, self.gated, out)
        if kernels.CHECK_WAITS:
            kernels.int4_status(x.device)
        return out

    def nbytes(self) -> int:
        return self.data.nbytes
