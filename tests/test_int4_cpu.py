"""The 4-bit products and the token shuffle without a GPU: argument checks before any launch, operators on meta tensors,
and the host-side checks of blocks."""
import ctypes

import pytest
import torch

from p2pllm_b200 import P2PError, _lib, compact, int4, moe

FAKE = 65536                                         # a 16-byte aligned address that nothing reads


@pytest.fixture(scope="module")
def lib():
    from p2pllm_b200 import build
    build.build()
    return _lib.load()


def test_layout_bytes(lib):
    """Units of 128 x 128 weights: 8 KB of codes, 256 bytes of scales a group, 128 of zero points."""
    size = lib.p2p_int4_layout_bytes
    assert size(1, 128, 128, 128, 0, 0) == 8192 + 256 and size(1, 129, 129, 128, 0, 0) == 4 * (8192 + 256)
    assert size(3, 1, 1, 32, 1, 0) == 3 * (8192 + 4 * (256 + 128)) and size(1, 256, 64, 64, 1, 0) == 2 * (8192 + 768)
    assert size(1, 128, 128, 128, 0, 1) == size(1, 2 * 49, 128, 128, 0, 1) == 8448      # 4 blocks of gates, 4 of ups
    assert size(1, 2 * 65, 128, 128, 0, 1) == 2 * 8448
    assert size(1, 3, 64, 64, 0, 1) == size(0, 1, 1, 32, 0, 0) == size(1, 0, 1, 32, 0, 0) == size(1, 1, 1, 16, 0, 0) == -1


@pytest.mark.parametrize("call,status,needle", [
    (lambda l: l.p2p_int4_quantize(FAKE, 0, 4, 64, 64, 48, FAKE, FAKE, None, None), -1, b"48"),
    (lambda l: l.p2p_int4_quantize(FAKE, 2, 4, 64, 64, 64, FAKE, FAKE, None, None), -2, b"bf16 or f16"),
    (lambda l: l.p2p_int4_quantize(FAKE, 0, 4, 64, 63, 64, FAKE, FAKE, None, None), -1, b"shape"),
    (lambda l: l.p2p_int4_expand(FAKE, None, None, 0, 4, 64, 64, FAKE, None), -1, b"null"),
    (lambda l: l.p2p_int4_layout(FAKE, FAKE, None, 1, 3, 64, 64, 1, FAKE, None), -1, b"shape"),
    (lambda l: l.p2p_int4_layout(FAKE, None, FAKE, 1, 4, 64, 64, 0, FAKE, None), -1, b"null"),
    (lambda l: l.p2p_int4_layout(FAKE, FAKE, None, 1, 4, 64, 64, 0, FAKE + 8, None), -1, b"16-byte"),
    (lambda l: l.p2p_int4_mm(FAKE, 2, 4, 64, 64, FAKE, 0, 16, 64, 0, FAKE, 16, None, 0, None), -2, b"bf16 or f16"),
    (lambda l: l.p2p_int4_mm(FAKE, 0, 4, 64, 63, FAKE, 0, 16, 64, 0, FAKE, 16, None, 0, None), -1, b"stride"),
    (lambda l: l.p2p_int4_mm(FAKE, 0, 4, 64, 64, FAKE, 0, 16, 64, 0, FAKE, 15, None, 0, None), -1, b"stride"),
    (lambda l: l.p2p_int4_mm(FAKE, 0, 4, 64, 64, FAKE, 0, 15, 64, 1, FAKE, 16, None, 0, None), -1, b"gated"),
    (lambda l: l.p2p_int4_mm(FAKE, 0, 4, 64, 64, FAKE + 4, 0, 16, 64, 0, FAKE, 16, None, 0, None), -1, b"16-byte"),
    (lambda l: l.p2p_int4_mm(None, 0, 4, 64, 64, FAKE, 0, 16, 64, 0, FAKE, 16, None, 0, None), -1, b"null"),
    (lambda l: l.p2p_int4_grouped(FAKE, 0, 64, 64, FAKE, 0, 16, 64, 0, FAKE, FAKE, 4, 273, None, 1, None, 4,
                                  FAKE, 16, None, 0, None), -1, b"at most 272"),
    (lambda l: l.p2p_int4_grouped(FAKE, 0, 64, 64, FAKE, 0, 16, 64, 0, FAKE + 4, FAKE, 4, 8, None, 1, None, 4,
                                  FAKE, 16, None, 0, None), -1, b"16-byte"),
    (lambda l: l.p2p_int4_grouped(FAKE, 0, 64, 64, FAKE, 0, 16, 64, 0, FAKE, FAKE, 4, 8, FAKE, 0, None, 4,
                                  FAKE, 16, None, 0, None), -1, b"topk"),
    (lambda l: l.p2p_int4_grouped(FAKE, 0, 64, 64, FAKE, 0, 16, 64, 0, FAKE, FAKE, 4, 9, FAKE, 1, None, 4,
                                  FAKE, 16, None, 0, None), -1, b"in the order's places"),
    (lambda l: l.p2p_int4_grouped(FAKE, 0, 64, 68, FAKE, 0, 16, 64, 0, FAKE, FAKE, 4, 9, None, 1, None, 4,
                                  FAKE, 16, None, 0, None), -1, b"16-byte"),
    (lambda l: l.p2p_int4_mm(FAKE, 0, 9, 64, 68, FAKE, 0, 16, 64, 0, FAKE, 16, None, 0, None), -1, b"16-byte"),
    (lambda l: l.p2p_int4_mm(FAKE, 0, 33, 64, 64, FAKE, 0, 16, 64, 0, FAKE, 16, None, 0, None), -1, b"workspace"),
    (lambda l: l.p2p_moe_sort(FAKE, 4, 64, 1025, FAKE, FAKE, FAKE, FAKE, 2000, 32, FAKE, None), -2, b"at most 1024"),
    (lambda l: l.p2p_moe_sort(FAKE, 2, 64, 8, FAKE, FAKE, FAKE, FAKE, 64, 32, FAKE, None), -1, b"4 or 8"),
    (lambda l: l.p2p_moe_sort(FAKE, 4, 64, 8, FAKE, FAKE, FAKE, FAKE, 9, 32, FAKE, None), -1, b"10 needed"),
    (lambda l: l.p2p_moe_sort(FAKE, 4, 64, 8, FAKE, FAKE, FAKE, None, 64, 32, FAKE, None), -1, b"null"),
    (lambda l: l.p2p_moe_spread(FAKE, 5, 4, 2, 8, 8, FAKE, FAKE, FAKE, 8, None), -2, b"f32"),
    (lambda l: l.p2p_moe_spread(FAKE, 0, 4, 0, 8, 8, FAKE, FAKE, FAKE, 8, None), -1, b"shape"),
    (lambda l: l.p2p_moe_spread(FAKE, 0, 1 << 30, 8, 8, 8, FAKE, FAKE, FAKE, 8, None), -1, b"shape"),
    (lambda l: l.p2p_moe_sum(FAKE, 0, 4, 2, 8, 7, FAKE, None, 2, FAKE, 8, None), -1, b"stride"),
    (lambda l: l.p2p_moe_sum(FAKE, 0, 4, 2, 8, 8, FAKE, FAKE, 9, FAKE, 8, None), -1, b"weights"),
    (lambda l: l.p2p_moe_sum_back(FAKE, FAKE, 0, 4, 2, 8, 8, 8, FAKE, FAKE, None, 2, FAKE, 8, FAKE, None), -1, b"null"),
    (lambda l: l.p2p_moe_sum_back(FAKE, FAKE, 0, 4, 2, 8, 7, 8, FAKE, FAKE, FAKE, 2, FAKE, 8, FAKE, None), -1, b"stride"),
])
def test_entries_refuse_bad_arguments(lib, call, status, needle):
    assert call(lib) == status
    assert needle in lib.p2p_last_error(), lib.p2p_last_error()


def test_empty_work_launches_nothing(lib):
    assert lib.p2p_int4_quantize(None, 0, 0, 64, 64, 64, None, None, None, None) == 0
    assert lib.p2p_int4_mm(None, 0, 0, 64, 64, None, 0, 16, 64, 0, None, 16, None, 0, None) == 0
    assert lib.p2p_int4_grouped(None, 0, 64, 64, None, 0, 16, 64, 0, None, None, 0, 0, None, 1, None, 0, None,
                                16, None, 0, None) == 0
    assert lib.p2p_moe_spread(None, 0, 0, 2, 8, 8, None, None, None, 8, None) == 0
    assert lib.p2p_moe_sum(None, 0, 0, 2, 8, 8, None, None, 2, None, 8, None) == 0


def test_operators_propagate_shapes_on_meta_tensors(lib):
    ops = _lib.ops()
    meta = lambda *s, dtype=torch.bfloat16: torch.empty(*s, device="meta", dtype=dtype)
    w = meta(100, dtype=torch.uint8)
    assert ops.int4_mm(meta(17, 64), w, False, 40, 64, 64, False).shape == (17, 40)
    assert ops.int4_mm(meta(17, 64), w, False, 40, 64, 64, True).shape == (17, 20)
    order, where, offsets, items, n = ops.moe_sort(meta(17, 8, dtype=torch.int64), 128)
    assert order.shape == where.shape == (136,) and offsets.shape == (129,) and items.shape == (4 * 136,) and n.shape == (1,)
    assert ops.int4_grouped(meta(17, 64), w, False, 128, 40, 64, 64, True, order, where, offsets, items, n, 8, True).shape == (136, 20)
    x = meta(17, 96).requires_grad_(True)
    xs = ops.moe_spread(x, where, offsets, 8)
    assert xs.shape == (136, 96) and xs.requires_grad
    out = ops.moe_sum(xs, where, offsets, meta(17, 8, dtype=torch.float32), 8)
    out.backward(torch.empty_like(out))
    assert x.grad.shape == x.shape


def test_cpu_tensors_are_refused():
    w = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(P2PError, match="CUDA"):
        int4.quantize(w)
    with pytest.raises(P2PError, match="CUDA"):
        moe.sort_tokens(torch.zeros(3, 2, dtype=torch.int64), 4)
    with pytest.raises(P2PError, match="CUDA"):
        compact.Tiles([("int4", torch.zeros(4, 32, dtype=torch.uint8), torch.ones(4, 1, dtype=torch.bfloat16), None, 64, 64)])
    with pytest.raises(P2PError, match="32, 64 or 128"):
        int4.check_block(("int4", w, w, None, 64, 16))
