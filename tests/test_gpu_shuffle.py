"""Tokens sorted by expert and back (moe.sort_tokens, to_experts, from_experts) against plain torch in 64 bits.

Bounds: a sum over K slots in fp32 is off by at most K roundings (2^-24 each, of the terms' absolute sum) plus half a
step of its own type; a product w * dout by one rounding and half a step; a dot over H columns by H / 8 + 16 additions
(a thread's own columns, then shuffles and warps) of 2^-24 of the terms' absolute sum."""
import pytest
import torch

from p2pllm_b200 import P2PError, moe

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
U = 2.0 ** -24


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ids(tokens, topk, experts, g, nowhere=0.1, dtype=torch.int64):
    ids = torch.randint(0, experts, (tokens, topk), generator=g, device="cuda")
    gone = torch.rand(tokens, topk, generator=g, device="cuda") < nowhere
    return torch.where(gone, -1, ids).to(dtype)


def _plain_order(ids, experts):
    flat = ids.reshape(-1).long()
    ok = (flat >= 0) & (flat < experts)
    key = torch.where(ok, flat, experts)
    order = torch.sort(key, stable=True).indices
    where = torch.empty_like(order)
    where[order] = torch.arange(order.numel(), device=order.device)
    counts = torch.bincount(key, minlength=experts + 1)[:experts]
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    order[int(offsets[-1]):] = -1
    return order, torch.where(ok, where, -1), offsets


def _check_order(order, ids, experts):
    want, where, offsets = _plain_order(ids, experts)
    assert torch.equal(order.order.long(), want) and torch.equal(order.where.long(), where)
    assert torch.equal(order.offsets.long(), offsets)
    items = order.items.view(-1, 4)[:int(order.n_items)].tolist()
    at, plain = offsets.tolist(), []
    most, mean = ids.numel(), ids.numel() / experts                 # what one pass over an expert's weights takes
    if most > 8:
        most = next(n for n, up_to in ((8, 4), (16, 10), (32, 24), (64, 48), (128, 100), (160, 130), (256, 1e9)) if mean <= up_to)
    else:
        most = 8
    for e in range(experts):
        plain += [[e, a, min(most, at[e + 1] - a), 0] for a in range(at[e], at[e + 1], most)]
    assert items == plain


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens,topk,experts", [
    (0, 2, 4), (1, 1, 1), (1, 8, 128), (5, 3, 7), (31, 1, 33), (17, 8, 128), (33, 4, 1024), (272, 8, 128), (1024, 8, 60),
    (1025, 8, 60), (2048, 8, 128), (9001, 7, 256), (16384, 8, 1024), (70000, 1, 3)])
def test_order(tokens, topk, experts, dtype):
    ids = _ids(tokens, topk, experts, _gen(tokens + experts), dtype=dtype)
    order = moe.sort_tokens(ids, experts)
    assert (order.tokens, order.topk, order.experts) == (tokens, topk, experts)
    _check_order(order, ids, experts)


def test_order_of_lopsided_and_foreign_ids():
    g = _gen(1)
    for tokens in (40, 9000):
        ids = torch.full((tokens, 4), 2, dtype=torch.int32, device="cuda")                # all to one expert
        _check_order(moe.sort_tokens(ids, 5), ids, 5)
        _check_order(moe.sort_tokens(torch.full_like(ids, -1), 5), torch.full_like(ids, -1), 5)
        far = torch.randint(-2 ** 62, 2 ** 62, (tokens, 4), generator=g, device="cuda")  # mostly out of range
        far[::3] = far[::3] % 5
        far[0, 0], far[1, 1] = 5, 2 ** 32 + 1                                             # 1 in the low 32 bits
        _check_order(moe.sort_tokens(far, 5), far, 5)
    strided = _ids(50, 8, 6, g)[:, ::2]
    _check_order(moe.sort_tokens(strided, 6), strided, 6)


CASES = [(1, 1, 1, 1), (1, 8, 128, 2048), (3, 2, 4, 7), (17, 8, 16, 64), (40, 3, 5, 129), (33, 9, 20, 96),
         (5, 20, 8, 1000), (6, 40, 64, 300), (9, 75, 16, 16), (272, 8, 128, 512), (1300, 8, 64, 136), (2, 2, 3, 9000), (0, 2, 3, 16)]


def _half(want, dtype):
    fi = torch.finfo(dtype)
    return fi.eps / 2 * want.abs() + fi.smallest_normal * fi.eps / 2


def _near(got, want, dtype, slack):
    bound = slack + _half(want.abs() + slack, dtype)
    assert got.shape == want.shape and got.dtype == dtype
    assert bool(((got.double() - want).abs() <= bound).all()), float(((got.double() - want).abs() / bound).max())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("wtype", ["f32", "bf16"])
@pytest.mark.parametrize("tokens,topk,experts,hidden", CASES)
def test_there_and_back_and_the_gradients(tokens, topk, experts, hidden, wtype, dtype):
    g = _gen(tokens * 31 + hidden)
    dt, P = DT[dtype], tokens * topk
    ids = _ids(tokens, topk, experts, g)
    order = moe.sort_tokens(ids, experts)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, y = rand(tokens, hidden).to(dt).requires_grad_(True), rand(P, hidden).to(dt)
    y[int(order.offsets[-1]):] = float("nan")                       # rows behind the last pair are nobody's
    y.requires_grad_(True)
    w = rand(tokens, topk).to(DT[wtype]).requires_grad_(True)
    xs, out = moe.to_experts(x, order), moe.from_experts(y, order, w)
    plain = moe.from_experts(y, order)
    gxs, gout, gplain = rand(P, hidden).to(dt), rand(tokens, hidden).to(dt), rand(tokens, hidden).to(dt)
    dx, dy, dw = torch.autograd.grad((xs, out), (x, y, w), (gxs, gout))
    dyp, = torch.autograd.grad(plain, y, gplain)

    ord_, where, offsets = _plain_order(ids, experts)
    last = int(offsets[-1])
    pair = ord_[:last]
    token = pair // topk
    x6, y6, w6 = x.detach().double(), y.detach().double()[:last], w.detach().double().reshape(-1)
    zeros = lambda *s: torch.zeros(*s, dtype=torch.float64, device="cuda")
    assert torch.equal(xs[:last], x[token]) and bool((xs[last:] == 0).all()) and xs.shape == (P, hidden)
    terms = w6[pair, None] * y6
    _near(out, zeros(tokens, hidden).index_add_(0, token, terms), dt,
          topk * U * zeros(tokens, hidden).index_add_(0, token, terms.abs()))
    _near(plain, zeros(tokens, hidden).index_add_(0, token, y6), dt,
          topk * U * zeros(tokens, hidden).index_add_(0, token, y6.abs()))
    g6 = gxs.double()[:last]
    _near(dx, zeros(tokens, hidden).index_add_(0, token, g6), dt,
          topk * U * zeros(tokens, hidden).index_add_(0, token, g6.abs()))
    back = w6[pair, None] * gout.double()[token]
    _near(dy[:last], back, dt, U * back.abs())
    assert bool((dy[last:] == 0).all()) and bool((dyp[last:] == 0).all()) and torch.equal(dyp[:last], gplain[token])
    dots = gout.double()[token] * y6
    want = zeros(P)
    want[pair] = dots.sum(-1)
    slack = zeros(P)
    slack[pair] = (hidden / 8 + 16) * U * dots.abs().sum(-1)
    _near(dw, want.view(tokens, topk), DT[wtype], slack.view(tokens, topk))


def test_gradients_against_differences():
    """The maps are linear in each argument, so a central difference has no error but its sums' roundings: the loss's
    terms sum to below 4096 in absolute value here, in 64 bits; the step 1/4 keeps every perturbed input exact."""
    g = _gen(3)
    T, K, E, H = 6, 3, 4, 40
    ids = _ids(T, K, E, g, nowhere=0.2)
    order = moe.sort_tokens(ids, E)
    quarter = lambda *s: torch.randint(-8, 9, s, generator=g, device="cuda").float() / 4
    x, y, w, cx, co = quarter(T, H), quarter(T * K, H), quarter(T, K), quarter(T * K, H), quarter(T, H)

    def loss(x, y, w):
        # every value is a small multiple of 1/16, so fp32 sums are exact
        return ((moe.to_experts(x, order).double() * cx).sum() + (moe.from_experts(y, order, w).double() * co).sum())
    leaves = [t.clone().requires_grad_(True) for t in (x, y, w)]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    for which, (t, grad) in enumerate(zip((x, y, w), grads)):
        for i in torch.randint(0, t.numel(), (12,), generator=g, device="cuda").tolist():
            args = [x, y, w]
            both = []
            for step in (0.25, -0.25):
                moved = t.clone()
                moved.view(-1)[i] += step
                args[which] = moved
                both.append(loss(*args))
            assert float(grad.reshape(-1)[i]) == float((both[0] - both[1]) / 0.5)


def test_expanded_and_strided_inputs():
    g = _gen(4)
    T, K, E, H = 20, 4, 6, 72
    order = moe.sort_tokens(_ids(T, K, E, g), E)
    row = torch.randn(1, H, generator=g, device="cuda").requires_grad_(True)
    xs = moe.to_experts(row.expand(T, H), order)                     # a broadcast input: its gradient sums over tokens
    assert torch.equal(xs, moe.to_experts(row.expand(T, H).contiguous(), order))
    xs.sum().backward()                                               # and an expanded gradient
    assert bool((row.grad == int(order.offsets[-1])).all())
    base = torch.randn(T * K, H + 5, generator=g, device="cuda")
    y = base[:, 3:3 + H]
    w = torch.rand(K, T, generator=g, device="cuda").t()
    assert torch.equal(moe.from_experts(y, order, w), moe.from_experts(y.contiguous(), order, w.contiguous()))
    assert torch.equal(moe.from_experts(y.t().contiguous().t(), order, w), moe.from_experts(y, order, w))


def test_only_what_is_asked_has_a_gradient():
    g = _gen(5)
    order = moe.sort_tokens(_ids(9, 2, 3, g), 3)
    y, w = torch.randn(18, 16, generator=g, device="cuda"), torch.rand(9, 2, generator=g, device="cuda")
    assert not moe.from_experts(y, order, w).requires_grad and not moe.to_experts(y[:9], order).requires_grad
    w1 = w.clone().requires_grad_(True)
    y1 = y.clone().requires_grad_(True)
    moe.from_experts(y, order, w1).sum().backward()
    moe.from_experts(y1, order, w).sum().backward()
    y2, w2 = y.clone().requires_grad_(True), w.clone().requires_grad_(True)
    moe.from_experts(y2, order, w2).sum().backward()
    assert torch.equal(w1.grad, w2.grad) and torch.equal(y1.grad, y2.grad)
    with torch.no_grad():
        assert not moe.from_experts(y2, order, w2).requires_grad
    grad, = torch.autograd.grad(moe.from_experts(y2, order, w2).sum(), y2, create_graph=False)
    assert torch.equal(grad, y2.grad)
    with pytest.raises(RuntimeError, match="second derivatives"):
        torch.autograd.grad(moe.from_experts(y2, order, w2).sum(), y2, create_graph=True)


def test_experts_are_trained_between_the_two():
    """A layer of dense experts in 32 bits between to_experts and from_experts against the same layer computed token by
    token in 64 bits: outputs and every gradient."""
    g = _gen(6)
    T, K, E, H, R = 30, 2, 4, 24, 16
    ids = _ids(T, K, E, g)
    rand = lambda *s: (torch.randn(*s, generator=g, device="cuda") / s[-1] ** 0.5).requires_grad_(True)
    x, w_in, w_out, gate = rand(T, H), rand(E, R, H), rand(E, H, R), rand(T, K)
    cot = torch.randn(T, H, generator=g, device="cuda")
    order = moe.sort_tokens(ids, E)
    xs, at = moe.to_experts(x, order), order.offsets.tolist()
    rows = [torch.tanh(xs[a:b] @ w_in[e].T) @ w_out[e].T for e, (a, b) in enumerate(zip(at, at[1:]))]
    rows.append(xs[at[-1]:] * 0)
    out = moe.from_experts(torch.cat(rows), order, gate)
    grads = torch.autograd.grad(out, (x, w_in, w_out, gate), cot)
    ref = [t.detach().double().requires_grad_(True) for t in (x, w_in, w_out, gate)]
    want = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    for t in range(T):
        for j in range(K):
            e = int(ids[t, j])
            if e >= 0:
                term = ref[3][t, j] * (torch.tanh(ref[0][t] @ ref[1][e].T) @ ref[2][e].T)
                want = want.index_add(0, torch.tensor([t], device="cuda"), term[None])
    plain = torch.autograd.grad(want, ref, cot.double())
    # sums of at most T K H terms in fp32 through three products: 64 roundings of the result's norm cover them
    for a, b in zip((out, *grads), (want, *plain)):
        assert float(((a.double() - b).norm() / b.norm()).detach()) <= 64 * U


@pytest.mark.parametrize("tokens", [33, 2000])
def test_a_training_step_is_captured_and_replayed(tokens):
    g = _gen(7)
    K, E, H = 8, 16, 64
    ids = _ids(tokens, K, E, g)
    x = torch.randn(tokens, H, generator=g, device="cuda").requires_grad_(True)
    w = torch.rand(tokens, K, generator=g, device="cuda").requires_grad_(True)
    cot = torch.randn(tokens, H, generator=g, device="cuda")

    def step():
        order = moe.sort_tokens(ids, E)
        out = moe.from_experts(moe.to_experts(x, order) * 2, order, w)
        return (out.detach(), *torch.autograd.grad(out, (x, w), cot))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(tokens, H, generator=g, device="cuda"))
            w.copy_(torch.rand(tokens, K, generator=g, device="cuda"))
        ids.copy_(_ids(tokens, K, E, g, nowhere=0.4 * k))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in got]
        for a, b in zip(kept, step()):
            assert torch.equal(a, b)


def test_results_do_not_depend_on_the_launch():
    g = _gen(8)
    T, K, E, H = 3000, 8, 64, 256
    ids = _ids(T, K, E, g)
    y = torch.randn(T * K, H, generator=g, device="cuda").bfloat16().requires_grad_(True)
    w = torch.rand(T, K, generator=g, device="cuda").requires_grad_(True)
    cot = torch.randn(T, H, generator=g, device="cuda").bfloat16()

    def once():
        order = moe.sort_tokens(ids, E)
        out = moe.from_experts(y, order, w)
        return (order.order, order.where, out.detach(), *torch.autograd.grad(out, (y, w), cot))
    want = once()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = [once() for _ in range(3)]
    here = [once() for _ in range(3)]
    torch.cuda.synchronize()
    for got in there + here:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_calls_that_do_not_fit_are_refused():
    ids = torch.zeros(3, 2, dtype=torch.int64, device="cuda")
    for bad, experts, needle in ((ids.float(), 4, "int32 or int64"), (ids[0], 4, "int32 or int64"), (ids, 0, "1 to 1024"),
                                 (ids, 1025, "1 to 1024"), (ids[:, :0], 4, "slots")):
        with pytest.raises(P2PError, match=needle):
            moe.sort_tokens(bad, experts)
    order = moe.sort_tokens(ids, 4)
    x = torch.zeros(3, 8, device="cuda")
    with pytest.raises(P2PError, match="wanted"):
        moe.to_experts(x[:2], order)
    with pytest.raises(P2PError, match="wanted"):
        moe.from_experts(x, order)
    with pytest.raises(P2PError, match="dtype"):
        moe.to_experts(x.double(), order)
    with pytest.raises(P2PError, match="wanted"):
        moe.from_experts(torch.zeros(6, 8, device="cuda"), order, torch.zeros(6, device="cuda"))
    with pytest.raises(P2PError, match="dtype"):
        moe.from_experts(torch.zeros(6, 8, device="cuda"), order, torch.zeros(3, 2, device="cuda").int())
    with pytest.raises(P2PError, match="CUDA"):
        moe.to_experts(x.cpu(), order)


def test_rows_past_32_bits():
    """2.6e9 elements of rows: the last places, and the sums and gradients of the last tokens."""
    T, K, H, E = 40000, 8, 8192, 16
    g = _gen(30)
    ids = _ids(T, K, E, g)
    order = moe.sort_tokens(ids, E)
    x = torch.randn(T, H, generator=g, device="cuda").bfloat16()
    rows = moe.to_experts(x, order)
    last = int(order.offsets[-1])
    at = torch.arange(last - 50, last, device="cuda")
    assert torch.equal(rows[at], x[order.order[at].long() // K])
    w = torch.rand(T, K, generator=g, device="cuda").requires_grad_(True)
    out = moe.from_experts(rows, order, w)
    cot = torch.randn(T, H, generator=g, device="cuda").bfloat16()
    (dw,) = torch.autograd.grad(out, w, cot)
    t = slice(T - 20, T)
    there = (order.where.view(T, K)[t] >= 0).double()
    dot = (x[t].double() * cot[t].double()).sum(1, keepdim=True)
    # sums of 8192 fp32 terms, each addition off by half a unit, by lanes and warps in a tree: below 64 roundings of the
    # absolute sum
    slack = 64 * 2.0 ** -24 * (x[t].double() * cot[t].double()).abs().sum(1, keepdim=True)
    assert bool(((dw[t].double() - dot * there).abs() <= slack).all())
    want = x[t].double() * (w[t].detach().double() * there).sum(1, keepdim=True)
    # a product and an addition a slot, each half a unit of the absolute sum; then half a step of bf16
    bound = 2 * K * 2.0 ** -24 * want.abs()
    assert bool(((out[t].detach().double() - want).abs() <= bound + 2.0 ** -8 * (want.abs() + bound)).all())
