"""Projection cross entropy against the formula in 64 bits (needs a B200).

Tolerances, with U = 2^-24 and h, w the operands as given:
* a logit is a sum of D products of 16-bit numbers in fp32: off by at most D U (|h| . |w|) = L;
* an exponential is ex2.approx (relative error 2^-22) of an argument rounded three times at the
  size of the logits in powers of two: relative error E = 2^-22 + 8 U (max|l| + |lse|) + L;
* a sum of exponentials adds (64/4 + strips + 16) U to that, so a loss is off by at most
  2 L + E + (32 + strips) U (1 + |lse|);
* dl is exp(l - lse) less one at the target, rounded once: r = finfo.eps / 2 of its size and 2 E of
  the probability (fp16 holds it times 4096: below 2^-14 the rounding is at most 2^-25 / 4096);
* dh and dW are products of dl with K terms accumulated in fp32 (and, in pieces, one addition per
  piece), rounded once: (r + K U) (|dl| |.|) + 2 E (p |.|) + r |result|.
"""

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    from systems_for_llms_b200.ops import lib
    from systems_for_llms_b200.ops.gemm import status_word
    if not lib.available():
        pytest.skip("kernels need a compute-capability 10.x device")
    lib.lib()
    device = torch.device("cuda", torch.cuda.current_device())
    status_word(device)
    return device


def check(dev):
    from systems_for_llms_b200.ops.gemm import check_status
    torch.cuda.synchronize()
    check_status()


def make(dev, N, D, V, dtype, seed=0, scale=1.0, ignored=0.25):
    gen = torch.Generator(device=dev).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=gen)
    h = rnd(N, D).to(dtype)
    w = (rnd(V, D) * scale / D ** 0.5).to(dtype)
    t = torch.randint(0, V, (N,), device=dev, generator=gen)
    drop = torch.rand(N, device=dev, generator=gen) < ignored
    drop[0] = False
    return h, w, t.masked_fill(drop, -100)


class Exact:
    """Loss, gradients and the bounds above in 64 bits."""

    def __init__(self, h, w, t, ignore=-100):
        self.h, self.w = h.double(), w.double()
        D, V = w.shape[1], w.shape[0]
        self.valid = t != ignore
        logits = self.h @ self.w.t()
        self.lse = torch.logsumexp(logits, -1)
        index = torch.where(self.valid, t, 0)[:, None]
        self.loss = torch.where(self.valid, self.lse - logits.gather(1, index)[:, 0], 0.0)
        L = D * U * (self.h.abs() @ self.w.abs().t()).amax(-1)
        strips = 2 * (-(-V // 256))
        self.E = 2.0 ** -22 + 8 * U * (logits.abs().amax(-1) + self.lse.abs()) + L
        self.loss_bound = 2 * L + self.E + (32 + strips) * U * (1 + self.lse.abs())
        self.p = torch.exp(logits - self.lse[:, None]) * self.valid[:, None]
        self.dl = self.p.clone()
        self.dl.scatter_add_(1, index, -self.valid.double()[:, None])
        self.half = torch.finfo(h.dtype).eps / 2

    def grads(self, scale, pieces=1):
        N, V = self.dl.shape
        tiny = 2.0 ** -25 / 4096 if self.half < 2.0 ** -9 else 0.0
        err = (self.half * self.dl.abs() + 2 * self.E[:, None] * self.p
               + tiny * self.valid[:, None])
        dh, dw = scale * (self.dl @ self.w), scale * (self.dl.t() @ self.h)
        bh = scale * ((err + (V + pieces) * U * self.dl.abs()) @ self.w.abs()) + self.half * dh.abs()
        bw = scale * ((err + N * U * self.dl.abs()).t() @ self.h.abs()) + self.half * dw.abs()
        smallest = 2.0 ** -25 if self.half < 2.0 ** -9 else 0.0     # of fp16 results
        return dh, dw, bh + smallest, bw + smallest


def within(got, want, bound):
    excess = ((got.double() - want).abs() - bound).max().item()
    assert excess <= 0, excess


SHAPES = [  # N, D, V
    (1, 8, 1), (1, 64, 2), (5, 72, 255), (128, 64, 256), (129, 136, 257), (300, 200, 1000),
    (256, 64, 513), (257, 520, 384), (1000, 64, 3001), (33, 1024, 5000),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_loss_and_gradients(dev, shape, dtype):
    from systems_for_llms_b200.ops.linear_loss import linear_cross_entropy
    h, w, t = make(dev, *shape, dtype)
    e = Exact(h, w, t)
    rows = linear_cross_entropy(h, w, t, reduction="none")
    check(dev)
    within(rows, e.loss, e.loss_bound)
    assert (rows[~e.valid] == 0).all()
    count = e.valid.sum().item()
    for reduction in ("mean", "sum"):
        scale = 0.5 / count if reduction == "mean" else 0.5
        leaves = [h.detach().requires_grad_(), w.detach().requires_grad_()]
        loss = linear_cross_entropy(*leaves, t, reduction=reduction)
        dh, dw = torch.autograd.grad(loss, leaves, torch.tensor(0.5, device=dev))
        check(dev)
        total = e.loss.sum() / (count if reduction == "mean" else 1)
        bound = e.loss_bound.sum() / (count if reduction == "mean" else 1) + 2 * U * total.abs()
        assert loss.dtype == torch.float32 and loss.shape == ()
        within(loss.detach(), total, bound)
        want_h, want_w, bh, bw = e.grads(scale)
        assert dh.dtype == h.dtype and dw.dtype == w.dtype
        within(dh, want_h, bh + 4 * U * want_h.abs())
        within(dw, want_w, bw + 4 * U * want_w.abs())
        assert (dh[~e.valid] == 0).all()


@pytest.mark.parametrize("shape, piece", [((129, 136, 257), None), ((300, 200, 1000), 512),
                                          ((64, 128, 6000), None)])   # the last splits dh's sum
def test_one_gradient_alone(dev, shape, piece):
    """What is not asked for is not computed; the sum of dh may be split differently, so each is
    held to the formula and not to the other."""
    from systems_for_llms_b200.ops import linear_loss as L
    h, w, t = make(dev, *shape, torch.bfloat16)
    e = Exact(h, w, t)
    scale = 1.0 / e.valid.sum().item()
    want_h, want_w, bh, bw = e.grads(scale, pieces=16)
    hidden, weight = h.detach().requires_grad_(), w.detach().requires_grad_()
    dh, = torch.autograd.grad(L.linear_cross_entropy(hidden, w, t), hidden)
    dw, = torch.autograd.grad(L.linear_cross_entropy(h, weight, t), weight)
    within(dh, want_h, bh + 4 * U * want_h.abs())
    within(dw, want_w, bw + 4 * U * want_w.abs())
    _, lse2, totals, _ = L.linear_ce_forward(h, w, t, -100, True)
    one = torch.ones((), device=dev)
    dh = L.linear_ce_backward(h, w, t, -100, lse2, one, totals, None, piece=piece)
    out = torch.full_like(w, float("nan"))
    assert L.linear_ce_backward(h, w, t, -100, lse2, one, totals, out, piece=piece,
                                need_dh=False) is None
    check(dev)
    within(dh, want_h, bh + 4 * U * want_h.abs())
    within(out, want_w, bw + 4 * U * want_w.abs())
    with pytest.raises(ValueError):
        L.linear_ce_backward(h, w, t, -100, lse2, one, totals, None, need_dh=False)


@pytest.mark.parametrize("piece", [256, 512, 1024])
def test_pieces_and_weight_gradient_kinds(dev, piece):
    from systems_for_llms_b200.ops.linear_loss import linear_ce_backward, linear_ce_forward
    N, D, V = 300, 136, 1300
    h, w, t = make(dev, N, D, V, torch.bfloat16)
    e = Exact(h, w, t)
    _, lse2, totals, _ = linear_ce_forward(h, w, t, -100, True)
    one = torch.ones((), device=dev)
    want_h, want_w, bh, bw = e.grads(1.0 / e.valid.sum().item(), pieces=6)
    dw16 = torch.empty_like(w)
    first = linear_ce_backward(h, w, t, -100, lse2, one, totals, dw16, piece=piece)
    dw32 = torch.full((V, D), 7.0, device=dev)
    second = linear_ce_backward(h, w, t, -100, lse2, one, totals, dw32, piece=piece)
    start = torch.randn(V, D, device=dev)
    added = start.clone()
    linear_ce_backward(h, w, t, -100, lse2, one, totals, added, accumulate=True, piece=piece)
    check(dev)
    assert torch.equal(first, second)                     # the order of sums is fixed
    within(first, want_h, bh + 4 * U * want_h.abs())
    within(dw16, want_w, bw + 4 * U * want_w.abs())
    within(dw32, want_w, bw + 4 * U * want_w.abs())
    assert torch.equal(dw32.bfloat16(), dw16)
    assert torch.equal(added, start + dw32)
    with pytest.raises(ValueError, match="dw"):
        linear_ce_backward(h, w, t, -100, lse2, one, totals, dw16, accumulate=True)


def test_several_row_bands_and_persistent_tiles(dev):
    """More tiles than pairs of SMs, and more row tiles than a band of wide rows holds."""
    from systems_for_llms_b200.ops.linear_loss import linear_cross_entropy
    h, w, t = make(dev, 2600, 8192, 2100, torch.bfloat16)
    e = Exact(h, w, t)
    leaves = [h.requires_grad_(), w.requires_grad_()]
    loss = linear_cross_entropy(*leaves, t)
    dh, dw = torch.autograd.grad(loss, leaves)
    rows = linear_cross_entropy(h.detach(), w.detach(), t, reduction="none")
    check(dev)
    within(rows, e.loss, e.loss_bound)
    want_h, want_w, bh, bw = e.grads(1.0 / e.valid.sum().item())
    within(dh, want_h, bh + 4 * U * want_h.abs())
    within(dw, want_w, bw + 4 * U * want_w.abs())


def test_gradient_agrees_with_differences(dev):
    from systems_for_llms_b200.ops.linear_loss import linear_cross_entropy
    h, w, t = make(dev, 64, 64, 300, torch.float16)
    leaves = [h.requires_grad_(), w.requires_grad_()]
    dh, dw = torch.autograd.grad(linear_cross_entropy(*leaves, t, reduction="sum"), leaves)
    gen = torch.Generator(device=dev).manual_seed(3)
    for leaf, grad in zip(leaves, (dh, dw)):
        way = torch.randn(leaf.shape, device=dev, generator=gen) * 2.0 ** -5
        moved = [(leaf.detach().float() + s * way).half() for s in (1, -1)]
        losses = []
        for m in moved:
            args = [m if leaf is leaves[0] else h.detach(), m if leaf is leaves[1] else w.detach()]
            losses.append(linear_cross_entropy(*args, t, reduction="sum").double().item())
        step = moved[0].double() - moved[1].double()          # what was really moved
        slope = (step * grad.double()).sum().item()
        # third differences of a log-sum-exp are below |direction . operand|^3; the loss is a sum of
        # 64 rows known to about 2^-18 each; the gradient is rounded to fp16 (2^-11 of its size)
        other = w if leaf is leaves[0] else h
        size = way.norm().item() * other.detach().float().norm(dim=1).max().item()
        room = size ** 3 / 24 + 64 * 2.0 ** -18 + 2.0 ** -10 * (step * grad.double()).norm().item() * 8
        assert abs(losses[0] - losses[1] - slope) < room


def test_masks_and_odd_targets(dev):
    from systems_for_llms_b200.ops.linear_loss import linear_cross_entropy
    h, w, t = make(dev, 200, 64, 500, torch.bfloat16, ignored=0.0)
    # an index of the vocabulary as the one to ignore
    t[::3] = 7
    e = Exact(h, w, t, ignore=7)
    leaves = [h.requires_grad_(), w.requires_grad_()]
    loss = linear_cross_entropy(*leaves, t, ignore_index=7)
    dh, dw = torch.autograd.grad(loss, leaves)
    within(loss.detach(), e.loss.sum() / e.valid.sum(), e.loss_bound.max() + 1e-9)
    want_h, want_w, bh, bw = e.grads(1.0 / e.valid.sum().item())
    within(dh, want_h, bh + 4 * U * want_h.abs())
    within(dw, want_w, bw + 4 * U * want_w.abs())
    # every row ignored: a mean of nothing is NaN, a sum zero, gradients zero
    none = torch.full_like(t, -100)
    for reduction in ("mean", "sum"):
        loss = linear_cross_entropy(*leaves, none, reduction=reduction)
        assert loss.isnan() if reduction == "mean" else loss == 0
        assert all((g == 0).all() for g in torch.autograd.grad(loss, leaves))
    # a target outside the vocabulary shows, and only in its row
    for bad in (500, -1, 2 ** 40, -2 ** 63):
        odd = t.clone()
        odd[5] = bad
        rows = linear_cross_entropy(h.detach(), w.detach(), odd, reduction="none")
        clean = linear_cross_entropy(h.detach(), w.detach(), t, reduction="none")
        assert rows[5].isnan()
        keep = torch.arange(200, device=dev) != 5
        assert torch.equal(rows[keep], clean[keep])
        assert linear_cross_entropy(h.detach(), w.detach(), odd).isnan()
    check(dev)


def test_rows_that_are_not_numbers_stay_alone(dev):
    from systems_for_llms_b200.ops.linear_loss import linear_cross_entropy
    h, w, t = make(dev, 300, 64, 700, torch.bfloat16, ignored=0.0)
    clean = linear_cross_entropy(h, w, t, reduction="none")
    for value in (float("nan"), float("inf")):
        bad = h.clone()
        bad[130, 3] = value
        rows = linear_cross_entropy(bad, w, t, reduction="none")
        keep = torch.arange(300, device=dev) != 130
        assert rows[130].isnan() and torch.equal(rows[keep], clean[keep])
    # logits far apart: the winner's loss is zero, others finite
    big = torch.zeros_like(h)
    big[:, 0] = 3e4
    wide = w.clone()
    wide[:, 0] = -1.0
    wide[11, 0] = 1.0
    rows = linear_cross_entropy(big, wide, t, reduction="none")
    assert rows.isfinite().all() and (rows[t != 11] > 5e4).all()
    assert (linear_cross_entropy(big, wide, torch.full_like(t, 11), reduction="none") == 0).all()
    check(dev)


def test_strides_and_shapes(dev):
    from systems_for_llms_b200.ops.linear_loss import linear_cross_entropy
    h, w, t = make(dev, 96, 64, 320, torch.bfloat16)
    want = linear_cross_entropy(h, w, t, reduction="none")
    pitched = torch.empty(96, 80, dtype=h.dtype, device=dev)[:, :64].copy_(h)
    odd = torch.empty(96 * 65 + 1, dtype=h.dtype, device=dev)[1:].view(96, 65)[:, :64].copy_(h)
    columns = h.t().contiguous().t()
    for other in (pitched, odd, columns):
        leaf = other.detach().requires_grad_()
        assert torch.equal(linear_cross_entropy(other, w, t, reduction="none"), want)
        (grad,) = torch.autograd.grad(linear_cross_entropy(leaf, w, t), leaf)
        assert grad.shape == leaf.shape
    cube = linear_cross_entropy(h.view(4, 24, 64), w, t.view(4, 24), reduction="none")
    assert torch.equal(cube.view(-1), want)
    narrow = torch.empty(320, 72, dtype=h.dtype, device=dev)[:, :64].copy_(w)
    assert torch.equal(linear_cross_entropy(h, narrow, t, reduction="none"), want)
    one = linear_cross_entropy(h[0], w, t[0], reduction="none")
    assert one.shape == () and torch.equal(one, want[0])
    shared = h[:1].expand(96, 64)                       # one row, ninety-six targets
    leaf = h[:1].detach().requires_grad_()
    (grad,) = torch.autograd.grad(linear_cross_entropy(leaf.expand(96, 64), w, t), leaf)
    assert grad.shape == (1, 64)
    assert linear_cross_entropy(shared, w, t, reduction="none").isfinite().all()
    check(dev)


def test_empty_batch(dev):
    from systems_for_llms_b200.ops.linear_loss import linear_cross_entropy
    h = torch.empty(0, 64, dtype=torch.bfloat16, device=dev, requires_grad=True)
    w = torch.randn(10, 64, device=dev).bfloat16().requires_grad_()
    t = torch.empty(0, dtype=torch.int64, device=dev)
    assert linear_cross_entropy(h.detach(), w.detach(), t, reduction="none").shape == (0,)
    for reduction in ("mean", "sum"):
        loss = linear_cross_entropy(h, w, t, reduction=reduction)
        assert loss.isnan() if reduction == "mean" else loss == 0
        dh, dw = torch.autograd.grad(loss, (h, w))
        assert dh.shape == (0, 64) and (dw == 0).all()


def test_refusals_on_the_gpu(dev):
    from systems_for_llms_b200.ops.linear_loss import linear_cross_entropy
    h, w, t = make(dev, 8, 64, 16, torch.bfloat16)
    with pytest.raises(ValueError, match="scoring"):
        linear_cross_entropy(h.requires_grad_(), w, t, reduction="none")
    h = h.detach()
    with pytest.raises(TypeError):
        linear_cross_entropy(h, w.half(), t)
    with pytest.raises(TypeError):
        linear_cross_entropy(h.float(), w.float(), t)
    with pytest.raises(ValueError, match="multiple of 8"):
        linear_cross_entropy(h[:, :12], w[:, :12], t)
    with pytest.raises(ValueError, match="targets"):
        linear_cross_entropy(h, w, t.int())
    with pytest.raises(ValueError, match="targets"):
        linear_cross_entropy(h, w, t[:4])
    with pytest.raises(ValueError, match="device"):
        linear_cross_entropy(h, w.cpu(), t)
    with pytest.raises(ValueError, match="empty"):
        linear_cross_entropy(h, w[:0], t)


def test_streams_and_graphs(dev):
    from systems_for_llms_b200.ops.linear_loss import linear_cross_entropy

    def call(h, w, t):
        leaves = [h.detach().requires_grad_(), w.detach().requires_grad_()]
        loss = linear_cross_entropy(*leaves, t)
        return (loss.detach(), *torch.autograd.grad(loss, leaves))

    sets = [make(dev, 300, 64, 900, torch.bfloat16, seed=s) for s in (1, 2)]
    want = [call(*s) for s in sets]
    static = [make(dev, 300, 64, 900, torch.bfloat16, seed=9) for _ in range(2)]
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, results = [], []
    with torch.cuda.stream(side):
        call(*static[0])
        for s in static:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                results.append(call(*s))
            graphs.append(graph)
        for mine, theirs in zip(static, sets):
            for a, b in zip(mine, theirs):
                a.copy_(b)
        other.wait_stream(side)
        graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
        side.wait_stream(other)
    check(dev)
    for got, expected in zip(results, want):
        assert all(torch.equal(a, b) for a, b in zip(got, expected))


@pytest.mark.parametrize("rows, dim, vocab, piece", [(300, 64, 700, 256), (300, 64, 700, 768),
                                                     (1024, 512, 10000, 10240)])
def test_kernels_are_counted(dev, rows, dim, vocab, piece):
    from systems_for_llms_b200.ops import lib
    from systems_for_llms_b200.ops.linear_loss import linear_ce_backward, linear_ce_forward
    h = torch.randn(rows, dim, device=dev).bfloat16()
    w = torch.randn(vocab, dim, device=dev).bfloat16()
    t = torch.randint(vocab, (rows,), device=dev)
    dw = torch.empty_like(w)

    def both():
        _, lse2, totals, _ = linear_ce_forward(h, w, t, -100, True)
        linear_ce_forward(h, w, t, -100, None)
        linear_ce_backward(h, w, t, -100, lse2, None, totals, dw, piece=piece)
    both()
    torch.cuda.synchronize()
    before = lib.launch_count()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        both()
    nodes = ctypes.c_size_t()          # of the captured graph: kernels alone
    assert ctypes.CDLL("libcudart.so.12").cudaGraphGetNodes(
        ctypes.c_void_p(graph.raw_cuda_graph()), None, ctypes.byref(nodes)) == 0
    assert lib.launch_count() - before == nodes.value > 0


def test_offsets_beyond_32_bits(dev):
    from systems_for_llms_b200.ops.linear_loss import linear_ce_backward, linear_ce_forward
    h, w, t = make(dev, 130, 64, 300, torch.bfloat16)
    pitch = 2 ** 23                                    # 300 rows of it pass 2**31 elements

    def both(h, w, dw):
        rows, lse2, totals, loss = linear_ce_forward(h, w, t, -100, True)
        return rows, loss, linear_ce_backward(h, w, t, -100, lse2, None, totals, dw)

    want_dw = torch.empty(300, 64, device=dev)
    want = both(h, w, want_dw)
    store = torch.empty(299 * pitch + 128, dtype=torch.bfloat16, device=dev)
    fw = store.as_strided((300, 64), (pitch, 1)).copy_(w)
    fh = store.as_strided((130, 64), (pitch, 1), 64).copy_(h)
    out = torch.empty(299 * pitch + 64, device=dev)
    dw = out.as_strided((300, 64), (pitch, 1))
    got = both(fh, fw, dw)
    check(dev)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(dw, want_dw)
