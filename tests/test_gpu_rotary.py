"""Rotary embedding and per-head norm against the formulas in 64 bits (needs a B200).

Tolerances.  A result is computed in fp32 and rounded once, so it is off by at most
``finfo(t).eps / 2`` of its value, plus the fp32 error of the steps before the rounding.  Those
are a sum of squares over at most 256 elements (in chains of 8 and a tree), a square root, a
division and a handful of products: below 32 units of 2^-24 of the operands' size, and below 64
for dx, which subtracts two such terms.  A weight gradient adds one product per row; chains are
at most (rows / warps + 24) long, each addition off by 2^-24 of the running sum of magnitudes.
"""

import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    from systems_for_llms_b200.ops import lib
    if not lib.available():
        pytest.skip("kernels need a compute-capability 10.x device")
    lib.lib()
    return torch.device("cuda", torch.cuda.current_device())


def tables(dev, rotated, rows, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)
    angles = torch.rand(rows, rotated // 2, device=dev, generator=gen, dtype=torch.float64) * 6.3
    return angles.cos().float(), angles.sin().float()


def split(x, rotated, layout):
    head = x[..., :rotated]
    if layout == "interleaved":
        return head[..., 0::2], head[..., 1::2]
    return head[..., :rotated // 2], head[..., rotated // 2:]


def turned(x, cos, sin, positions, layout):
    """The rotation in 64 bits; positions [B, T]."""
    rotated = 2 * cos.shape[1]
    c, s = (t.double()[positions][:, None] for t in (cos, sin))
    a, b = split(x, rotated, layout)
    ya, yb = a * c - b * s, a * s + b * c
    if layout == "interleaved":
        y = torch.stack((ya, yb), -1).flatten(-2)
    else:
        y = torch.cat((ya, yb), -1)
    return torch.cat((y, x[..., rotated:]), -1)


def normed(x, weight, eps):
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight


def close(got, want, scale, units=32):
    """``scale``: size of the operands, broadcastable to the result."""
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * half * 2
    bound = half * want.abs() + units * U * (1 + half) * scale + tiny
    excess = (got.double() - want).abs() - bound
    assert excess.max().item() <= 0, excess.max().item()


def inputs(dev, dtype, B, H, G, T, D, seed=1, wide=True):
    """Queries and keys as views of one packed projection, and its gradients token-major."""
    gen = torch.Generator(device=dev).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=gen)
    packed = rnd(B, T, H + 2 * G, D).to(dtype)
    q, k = packed[:, :, :H].permute(0, 2, 1, 3), packed[:, :, H:H + G].permute(0, 2, 1, 3)
    weights = [1 + 0.3 * rnd(D) for _ in range(2)]
    grads = [rnd(B, T, n, D).to(dtype).permute(0, 2, 1, 3) for n in (H, G)]
    return q, k, weights, grads


SHAPES = [  # B, H, G, T, D, R
    (1, 1, 1, 1, 64, 64), (2, 4, 2, 5, 64, 64), (3, 5, 1, 33, 128, 128), (2, 8, 8, 130, 64, 32),
    (1, 3, 3, 7, 80, 80), (2, 2, 1, 9, 96, 48), (1, 6, 2, 17, 256, 256), (1, 2, 2, 65, 192, 64),
    (2, 3, 1, 11, 72, 20), (1, 2, 1, 4, 50, 22), (1, 2, 1, 3, 6, 6), (1, 2, 2, 5, 7, 2),
    (1, 1, 1, 2, 1, 0), (1, 40, 8, 3, 128, 96),
]


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_norm_and_rotation_with_gradients(dev, shape, dtype, layout):
    from systems_for_llms_b200.ops.rotary import qk_norm_rotary, rotary
    B, H, G, T, D, R = shape
    eps = 1e-5
    q, k, weights, grads = inputs(dev, dtype, B, H, G, T, D)
    cos, sin = tables(dev, R, 37 + T)
    positions = torch.randint(0, 37, (B, 1), device=dev) + torch.arange(T, device=dev)
    leaves = [t.detach().requires_grad_() for t in (q, k, *weights)]
    outs = qk_norm_rotary(*leaves, cos, sin, positions, eps=eps, layout=layout)
    got = torch.autograd.grad(outs, leaves, grads)
    for i, (x, w, g, y, dx) in enumerate(zip((q, k), weights, grads, outs, got)):
        x64 = x.double().requires_grad_()
        w64 = w.double().requires_grad_()
        y64 = turned(normed(x64, w64, eps), cos, sin, positions, layout)
        dx64, dw64 = torch.autograd.grad(y64, (x64, w64), g.double())
        u = normed(x.double(), w.double(), eps)
        close(y.detach(), y64.detach(), 2 * u.abs().amax(-1, keepdim=True))
        rstd = (x.double().square().mean(-1, keepdim=True) + eps).rsqrt()
        unit = (x.double() * rstd).abs()
        v = 2 * g.double().abs().amax(-1, keepdim=True) * w.double().abs().max()
        close(dx, dx64, rstd * v * (1 + unit.amax(-1, keepdim=True)), units=64)
        rows = B * x.shape[1] * T
        size = (2 * g.double().abs().amax(-1, keepdim=True) * unit).sum(dim=(0, 1, 2))
        bound = (rows / 8 + 24 + 32) * U * size + 1e-30
        assert got[2 + i].dtype == torch.float32
        assert ((got[2 + i].double() - dw64).abs() <= bound).all()
        # rotation alone, forward and gradient
        leaf = x.detach().requires_grad_()
        y = rotary(leaf, cos, sin, positions, layout=layout)
        (dx,) = torch.autograd.grad(y, leaf, g)
        x64 = x.double().requires_grad_()
        y64 = turned(x64, cos, sin, positions, layout)
        (dx64,) = torch.autograd.grad(y64, x64, g.double())
        close(y.detach(), y64.detach(), 2 * x.double().abs().amax(-1, keepdim=True), units=4)
        close(dx, dx64, 2 * g.double().abs().amax(-1, keepdim=True), units=4)


def test_many_tokens_take_several_rows_per_warp(dev):
    """Enough work for the four-heads-per-warp form and for several items per warp backward."""
    from systems_for_llms_b200.ops.rotary import qk_norm_rotary
    B, H, G, T, D = 2, 16, 4, 1500, 64
    q, k, weights, grads = inputs(dev, torch.bfloat16, B, H, G, T, D)
    cos, sin = tables(dev, D, T)
    leaves = [t.detach().requires_grad_() for t in (q, k, *weights)]
    outs = qk_norm_rotary(*leaves, cos, sin)
    got = torch.autograd.grad(outs, leaves, grads)
    again = torch.autograd.grad(qk_norm_rotary(*leaves, cos, sin), leaves, grads)
    assert all(torch.equal(a, b) for a, b in zip(got, again))     # fixed summation order
    positions = torch.arange(T, device=dev).expand(B, T)
    for i, (x, w, g, y) in enumerate(zip((q, k), weights, grads, outs)):
        x64, w64 = x.double().requires_grad_(), w.double().requires_grad_()
        y64 = turned(normed(x64, w64, 1e-5), cos, sin, positions, "interleaved")
        _, dw64 = torch.autograd.grad(y64, (x64, w64), g.double())
        close(y.detach(), y64.detach(),
              2 * normed(x.double(), w.double(), 1e-5).abs().amax(-1, keepdim=True))
        rstd = (x.double().square().mean(-1, keepdim=True) + 1e-5).rsqrt()
        size = (2 * g.double().abs().amax(-1, keepdim=True) * (x.double() * rstd).abs()).sum((0, 1, 2))
        assert ((got[2 + i].double() - dw64).abs() <= (B * H * T / 64 + 56) * U * size).all()


def test_gradient_agrees_with_differences(dev):
    from systems_for_llms_b200.ops.rotary import qk_norm_rotary
    q, k, weights, grads = inputs(dev, torch.float32, 1, 2, 1, 3, 16)
    cos, sin = tables(dev, 8, 4)
    leaves = [t.detach().contiguous().requires_grad_() for t in (q, k, *weights)]
    loss = lambda args: sum((y.double() * g.double()).sum()
                            for y, g in zip(qk_norm_rotary(*args, cos, sin, layout="half"), grads))
    got = torch.autograd.grad(loss(leaves), leaves)
    step = 2.0 ** -8
    for i, leaf in enumerate(leaves):
        for at in itertools.islice(torch.randperm(leaf.numel()).tolist(), 6):
            shifted = []
            for sign in (1, -1):
                args = [t.detach().clone() for t in leaves]
                args[i].view(-1)[at] += sign * step
                shifted.append(loss(args).item())
            slope = (shifted[0] - shifted[1]) / (2 * step)
            # central differences: third derivative (order one here) times step^2, and the
            # rounding of about 50 outputs of size one over the step
            assert abs(slope - got[i].reshape(-1)[at].item()) < 40 * step ** 2 + 50 * 16 * U / step


def test_strides_positions_and_out(dev):
    from systems_for_llms_b200.ops.rotary import qk_norm_rotary, rotary
    B, H, G, T, D = 2, 4, 2, 6, 64
    q, k, weights, _ = inputs(dev, torch.bfloat16, B, H, G, T, D)
    cos, sin = tables(dev, D, 64)
    want = qk_norm_rotary(q, k, *weights, cos, sin, layout="half")
    # head-major storage, a misaligned base and an odd row pitch give the same values
    raw = torch.empty(B * H * T * (D + 3) + 5, dtype=q.dtype, device=dev)
    odd = raw[5:].view(B, H, T, D + 3)[..., :D]
    odd.copy_(q)
    for other in (q.contiguous(), odd):
        got = qk_norm_rotary(other, k.contiguous(), *weights, cos, sin, layout="half")
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # one position per token for every batch row, or one row of positions for all
    shared = torch.arange(T, device=dev)
    for positions in (shared, shared.expand(B, T), shared.repeat(B, 1)):
        got = qk_norm_rotary(q, k, *weights, cos, sin, positions, layout="half")
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # new keys straight into their rows of a cache; nothing else of it is written
    cache = torch.full((B, G, 32, D), 7.0, dtype=k.dtype, device=dev)
    out_q = torch.empty_like(q)
    qk_norm_rotary(q, k, *weights, cos, sin, layout="half", out=(out_q, cache[:, :, 10:10 + T]))
    assert torch.equal(cache[:, :, 10:10 + T], want[1]) and torch.equal(out_q, want[0])
    assert (cache[:, :, :10] == 7).all() and (cache[:, :, 10 + T:] == 7).all()
    # in place
    mine = q.contiguous()
    assert rotary(mine, cos, sin, out=mine) is mine
    assert torch.equal(mine, rotary(q, cos, sin))
    # gradients in place of the incoming ones
    from systems_for_llms_b200.ops.rotary import qk_norm_rotary_grad
    grads = [torch.randn(B, n, T, D, device=dev).to(q.dtype) for n in (H, G)]
    kw = dict(eps=1e-5, layout="half")
    want = qk_norm_rotary_grad(q, k, *weights, cos, sin, None, *grads, **kw)
    got = qk_norm_rotary_grad(q, k, *weights, cos, sin, None, *grads, out=tuple(grads), **kw)
    assert got[0] is grads[0] and all(torch.equal(a, b) for a, b in zip(got, want))
    # an expanded tensor: heads that share one key
    one = k[:, :1].expand(B, 3, T, D)
    assert torch.equal(rotary(one, cos, sin)[:, 2], rotary(k[:, :1], cos, sin)[:, 0])
    leaf = k[:, :1].detach().requires_grad_()
    (grad,) = torch.autograd.grad(rotary(leaf.expand(B, 3, T, D), cos, sin).float().sum(), leaf)
    (once,) = torch.autograd.grad(rotary(leaf, cos, sin).float().sum(), leaf)
    # three bf16 gradients added by autograd: two more roundings
    assert ((grad.float() - 3 * once.float()).abs() <= 3 * 2.0 ** -8 * once.float().abs() * 3 + 1e-6).all()


def test_rows_that_are_not_numbers_stay_alone(dev):
    from systems_for_llms_b200.ops.rotary import qk_norm_rotary, rotary
    q, k, weights, grads = inputs(dev, torch.float16, 1, 3, 1, 8, 64)
    cos, sin = tables(dev, 32, 8)
    clean = rotary(q, cos, sin, layout="half")
    bad = q.clone()
    bad[0, 1, 2, 5] = float("inf")
    bad[0, 1, 3, 40] = float("inf")      # beyond the rotated lanes
    got = rotary(bad, cos, sin, layout="half")
    keep = torch.ones(3, 8, dtype=torch.bool, device=dev)
    keep[1, 2] = keep[1, 3] = False
    assert torch.equal(got[0][keep], clean[0][keep])
    assert got[0, 1, 3, 40] == float("inf")
    assert torch.equal(got[0, 1, 3, :40], clean[0, 1, 3, :40])
    # a position outside the tables: NaN in its rotated lanes, the rest of the call unharmed
    for where in (-1, 8, 2 ** 40):
        positions = torch.arange(8, device=dev)
        positions[4] = where
        got = rotary(q, cos, sin, positions, layout="half")
        assert got[0, :, 4, :32].isnan().all() and torch.equal(got[0, :, 4, 32:], q[0, :, 4, 32:])
        others = [0, 1, 2, 3, 5, 6, 7]
        assert torch.equal(got[0][:, others], clean[0][:, others])
    # rows of zeros: the norm divides by sqrt(eps), the gradient is finite
    zero = torch.zeros_like(q).requires_grad_()
    outs = qk_norm_rotary(zero, k, *weights, cos, sin)
    assert (outs[0] == 0).all()
    (dz,) = torch.autograd.grad(outs[0], zero, grads[0])
    assert dz.float().isfinite().all() and (dz != 0).any()


def test_empty_calls(dev):
    from systems_for_llms_b200.ops.rotary import qk_norm_rotary
    cos, sin = tables(dev, 64, 8)
    w = torch.ones(64, device=dev, requires_grad=True)
    for B, T in ((0, 4), (2, 0)):
        q = torch.empty(B, 4, T, 64, device=dev, dtype=torch.bfloat16, requires_grad=True)
        k = torch.empty(B, 2, T, 64, device=dev, dtype=torch.bfloat16, requires_grad=True)
        outs = qk_norm_rotary(q, k, w, w, cos, sin)
        assert outs[0].shape == q.shape and outs[1].shape == k.shape
        grads = torch.autograd.grad(outs, (q, k, w), tuple(torch.ones_like(o) for o in outs))
        assert (grads[2] == 0).all()


def test_streams_and_graphs(dev):
    """Replayed graphs read new contents of their inputs; two graphs share no workspace."""
    from systems_for_llms_b200.ops.rotary import qk_norm_rotary, qk_norm_rotary_grad
    cos, sin = tables(dev, 64, 64)
    sets = [inputs(dev, torch.bfloat16, 2, 4, 2, 16, 64, seed=s) for s in (1, 2, 3)]
    kw = dict(eps=1e-5, layout="interleaved")

    def call(q, k, weights, grads):
        outs = qk_norm_rotary(q, k, *weights, cos, sin, **kw)
        return outs + qk_norm_rotary_grad(q, k, *weights, cos, sin, None, *grads, **kw)

    want = [call(*s) for s in sets]
    static = [inputs(dev, torch.bfloat16, 2, 4, 2, 16, 64, seed=9) for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, results = [], []
    with torch.cuda.stream(side):
        call(*static[0])
        for s in static:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                results.append(call(*s))
            graphs.append(graph)
        for s, source in zip(static, sets):
            for mine, theirs in zip((s[0], s[1], *s[2], *s[3]),
                                    (source[0], source[1], *source[2], *source[3])):
                mine.copy_(theirs)
        other = torch.cuda.Stream()
        other.wait_stream(side)
        graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
        side.wait_stream(other)
    torch.cuda.synchronize()
    for got, expected in zip(results, want):
        assert all(torch.equal(a, b) for a, b in zip(got, expected))
    direct = call(*sets[2])
    assert all(torch.equal(a, b) for a, b in zip(direct, want[2]))


def test_offsets_beyond_32_bits(dev):
    """Heads of one tensor 2**31 elements apart, as in a long cache, read and written in place."""
    from systems_for_llms_b200.ops.rotary import qk_norm_rotary, qk_norm_rotary_grad
    q, k, weights, grads = inputs(dev, torch.bfloat16, 1, 2, 2, 5, 64)
    cos, sin = tables(dev, 64, 64)
    kw = dict(eps=1e-5, layout="half")
    want = qk_norm_rotary(q, k, *weights, cos, sin, **kw)
    want_grads = qk_norm_rotary_grad(q, k, *weights, cos, sin, None, *grads, **kw)
    store = torch.empty(2 ** 31 + 8192, dtype=torch.bfloat16, device=dev)
    far = lambda at: store[at:].as_strided((1, 2, 5, 64), (64, 2 ** 31, 64, 1), store[at:].storage_offset())
    fq, fk, fg, fh = (far(1024 * i).copy_(t) for i, t in enumerate((q, k, *grads)))
    got = qk_norm_rotary_grad(fq, fk, *weights, cos, sin, None, fg, fh, out=(fg, fh), **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, want_grads))
    got = qk_norm_rotary(fq, fk, *weights, cos, sin, out=(fq, fk), **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
