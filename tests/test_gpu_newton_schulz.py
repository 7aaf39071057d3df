"""Newton-Schulz orthogonalisation against the formula in 64 bits (needs a B200).

Tolerance.  Let u = 2^-11 (half a step of fp16), s the shorter side, F the Frobenius norm.  A step
rounds hi (dX = u |X|F), the Gram matrix (dG = u |G|F, and X dX^T twice), P = b G + c G G, in the
last two steps with a I added and hi standing for X (dP = (|b| + 2 |c| |G|) dG + u |P|F) and multiplies: dP X and P dX.  hi + lo keep X to 2^-21 of each entry and,
since fp16 numbers are at least 2^-24 apart and X is held times 2^12, to 2^-37 absolutely (half of
2^-24 over 2^12; it matters where eps dwarfs the norm: X is then far below 1).  Sums of K products in fp32 add K 2^-24 of the product of the norms (rms: the root of K).  What a step leaves is carried by the
steps after it: in the singular basis of that step's X entry (i, j) of an error is multiplied by
(f(si) -+ f(sj)) / (si -+ sj), f being the remaining steps' map of a singular value (f(si) / si
beyond the square part), the derivative of a matrix function.
Small matrices are held to the sum of worst cases: spectral norms and the largest multiplier.
Matrices of 1000 entries or more are held to twice the root of the sum of squares with rms norms
(|A dX|F = |A|F |dX|F / sqrt(rows of dX), the rms of a rounding is u / sqrt(3), the rms multiplier),
since roundings are many and independent.  The result's rounding to bf16 adds 2^-8 (rms: over
sqrt(3)) of its norm.
"""

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu

QUINTIC = (3.4445, -4.7750, 2.0315)


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


def multipliers(x, f):
    """Of each entry of an error in x, under the matrix function of f (x has no more rows than
    columns): the two of the square part and those of the columns beyond it."""
    sv = torch.linalg.svdvals(x)
    fv = f(sv)
    one, two = sv[:, None], sv[None, :]
    apart = one - two
    h = 1e-6
    slope = (f(sv + h) - f((sv - h))) / (2 * h)
    close = apart.abs() < 1e-6
    minus = torch.where(close, slope[:, None].expand_as(apart),
                        (fv[:, None] - fv[None, :]) / torch.where(close, 1.0, apart))
    plus = (fv[:, None] + fv[None, :]) / (one + two).clamp_min(1e-12)
    beyond = fv / sv.clamp_min(1e-12)
    return minus, plus, beyond


def carried(x, f, typical):
    s, n = x.shape
    minus, plus, beyond = multipliers(x, f)
    if not typical:
        return max(t.abs().max().item() for t in (minus, plus, beyond))
    square = (minus.square().sum() + plus.square().sum()) / 2
    return ((square + (n - s) * beyond.square().sum()) / (s * n)).sqrt().item()


def exact(update, steps=5, coefficients=QUINTIC, eps=1e-7):
    """Result and error bound of one matrix."""
    a, b, c = coefficients
    x = update.double()
    x = x / (x.square().sum().sqrt() + eps)
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    s, n = x.shape
    if not x.any():
        return (x.t() if tall else x), 0.0
    typical = x.numel() >= 1000
    u = 2.0 ** -11 / (3 ** 0.5 if typical else 1.0)
    join = (lambda *e: sum(v * v for v in e) ** 0.5) if typical else (lambda *e: sum(e))
    adds = lambda count: 2.0 ** -24 * (count ** 0.5 if typical else count)
    size = lambda t: torch.linalg.matrix_norm(t, 2).item()
    errors = []
    # what the first hi + lo leave out, carried by every step; later ones are part of `local`
    held = lambda t: 2.0 ** -21 * t.norm().item() + 2.0 ** -37 * t.numel() ** 0.5
    start = held(x) + 2.0 ** -22 * x.norm().item()
    for step in range(-1, steps):
        def after(v, left=steps - step - 1):
            for _ in range(left):
                v = v * (a + v ** 2 * (b + c * v ** 2))
            return v

        if step < 0:
            errors.append(start * carried(x, after, typical))
            continue
        k = a if step + 2 >= steps else 0.0
        g = x @ x.t()
        p = b * g + c * g @ g + k * torch.eye(s, dtype=x.dtype, device=x.device)
        # |A d| = act(A) |d|
        act = (lambda t: t.norm().item() / min(t.shape) ** 0.5) if typical else size
        dx = u * x.norm().item()
        spread = x.norm().item() / n ** 0.5 if typical else size(x)
        dg = join(u * g.norm().item(), 2 * spread * dx) + adds(n) * x.norm().item() ** 2
        dp = (join((abs(b) + 2 * abs(c) * act(g)) * dg, u * p.norm().item())
              + adds(s) * abs(c) * g.norm().item() ** 2)
        new = (a - k) * x + p @ x
        local = (join(dp * act(x), act(p) * dx) + held(new)
                 + adds(s) * p.norm().item() * x.norm().item())
        errors.append(local * carried(new, after, typical))
        x = new
    bound = (2 if typical else 1) * join(*errors)
    bound += 2.0 ** -8 * x.norm().item() / (3 ** 0.5 if typical else 1)
    return (x.t() if tall else x), bound


def compare(got, update, **kw):
    want, bound = exact(update, **kw)
    off = (got.double() - want).norm().item()
    assert off <= bound + 1e-30, (off, bound)
    return off / max(want.norm().item(), 1e-30)


def gradient(dev, *shape, dtype=torch.float32, seed=0, scale=1e-3):
    gen = torch.Generator(device=dev).manual_seed(seed)
    *lead, m, n = shape
    rank = max(1, min(m, n) // 4)
    fall = torch.exp(-3.0 * torch.arange(rank, device=dev) / rank)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=gen)
    low = (rnd(*lead, m, rank) * fall) @ rnd(*lead, rank, n) / rank ** 0.5
    return ((low + 0.2 * rnd(*shape)) * scale).to(dtype)


SHAPES = [(1, 1), (1, 9), (7, 1), (3, 5), (16, 40), (64, 64), (65, 63), (128, 384), (255, 257),
          (256, 256), (300, 520), (520, 300), (513, 513), (1000, 337), (72, 2052), (700, 1344)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_one_matrix(dev, shape, dtype):
    from systems_for_llms_b200.ops.newton_schulz import newton_schulz
    u = gradient(dev, *shape, dtype=dtype, scale=1.0 if dtype == torch.float16 else 1e-3)
    for steps in (1, 2, 5):
        got = newton_schulz(u, steps=steps)
        check(dev)
        assert got.shape == u.shape and got.dtype == torch.bfloat16 and got.is_contiguous()
        compare(got, u, steps=steps)


def test_accuracy_does_not_fall_behind(dev):
    """The result's own rounding is 1.7e-3 of its norm (2^-8 / sqrt(3) / 1.35, the mean mantissa);
    the fp16 roundings that remain come to less than that again: together below 2.5e-3."""
    from systems_for_llms_b200.ops.newton_schulz import newton_schulz
    for shape in ((256, 256), (512, 1344), (1024, 1024)):
        u = gradient(dev, *shape)
        noise = torch.randn(*shape, device=dev)
        assert compare(newton_schulz(u), u) < 2.5e-3
        assert compare(newton_schulz(noise), noise) < 2.5e-3


def test_singular_values_end_near_one(dev):
    from systems_for_llms_b200.ops.newton_schulz import newton_schulz
    u = torch.randn(256, 640, device=dev)
    left, _, right = torch.linalg.svd(u.double(), full_matrices=False)
    got = newton_schulz(u).double()
    along = left.t() @ got @ right.t()
    values = along.diagonal()
    # the quintic's band on singular values that are at least 0.01 of the norm
    assert values.min() > 0.65 and values.max() < 1.25
    off = along - torch.diag(values)
    assert off.norm() < 0.01 * values.norm()              # same singular vectors


def test_stacks_and_strides(dev):
    from systems_for_llms_b200.ops.newton_schulz import newton_schulz
    u = gradient(dev, 2, 3, 200, 136)
    got = newton_schulz(u)
    check(dev)
    for i in range(2):
        for j in range(3):
            alone = newton_schulz(u[i, j])
            assert torch.equal(alone, got[i, j])          # neighbours do not matter
            compare(alone, u[i, j])
    # the same parameter of every layer inside a flat buffer
    flat = torch.zeros(2, 7, 300, 144, device=dev)
    view = flat[:, 1:4, 50:250, 3:139]
    view.copy_(u)
    assert torch.equal(newton_schulz(view), got)
    assert torch.equal(newton_schulz(u.expand(2, 2, 3, 200, 136))[1], got)
    assert torch.equal(newton_schulz(u[:1].expand(2, 3, 200, 136))[1], got[0])
    turned = u.mT.contiguous().mT                         # column-major matrices
    assert torch.equal(newton_schulz(turned), got)
    out = torch.full((2, 3, 200, 136), 7.0, device=dev, dtype=torch.bfloat16)
    assert newton_schulz(u, out=out) is out and torch.equal(out, got)
    check(dev)


def test_a_transposed_matrix_gives_the_transposed_result(dev):
    from systems_for_llms_b200.ops.newton_schulz import newton_schulz
    u = gradient(dev, 320, 200)
    a, b = newton_schulz(u), newton_schulz(u.t())
    # both within the bound of the same exact matrix
    _, bound = exact(u)
    assert (a.double() - b.t().double()).norm().item() <= 2 * bound


def test_many_matrices_keep_the_persistent_grid_busy(dev):
    from systems_for_llms_b200.ops.newton_schulz import newton_schulz
    u = gradient(dev, 30, 520, 264)
    got = newton_schulz(u)
    again = newton_schulz(u)
    check(dev)
    assert torch.equal(got, again)
    for z in (0, 13, 29):
        compare(got[z], u[z])


def test_scales_zeros_and_values_that_are_not_numbers(dev):
    from systems_for_llms_b200.ops.newton_schulz import newton_schulz
    u = gradient(dev, 5, 96, 160, scale=1.0)
    clean = newton_schulz(u, eps=0.0)
    for factor in (2.0 ** 80, 2.0 ** -80):                 # squares far outside fp32
        assert torch.equal(newton_schulz(u * factor, eps=0.0), clean)
    bad = u.clone()
    bad[1] = 0
    bad[2, 5, 7] = float("nan")
    bad[3, 0, 0] = float("inf")
    got = newton_schulz(bad)
    check(dev)
    reference = newton_schulz(u)
    assert torch.equal(got[0], reference[0]) and torch.equal(got[4], reference[4])
    assert (got[1] == 0).all() and got[2].isnan().all() and got[3].isnan().any()
    # eps against the norm: a tiny update stays small
    tiny = newton_schulz(u * 1e-12, steps=1, eps=1e-3)
    compare(tiny[0], u[0] * 1e-12, steps=1, eps=1e-3)


def test_other_coefficients(dev):
    from systems_for_llms_b200.ops.newton_schulz import newton_schulz
    u = gradient(dev, 128, 200)
    compare(newton_schulz(u, steps=8, coefficients=(1.875, -1.25, 0.375)), u, steps=8,
            coefficients=(1.875, -1.25, 0.375))
    compare(newton_schulz(u, steps=8, coefficients=(1.5, -0.5, 0.0)), u, steps=8,
            coefficients=(1.5, -0.5, 0.0))


def test_empty_and_refused_calls(dev):
    from systems_for_llms_b200.ops.newton_schulz import newton_schulz
    for shape in ((0, 4), (4, 0), (0, 4, 4), (2, 0, 3)):
        assert newton_schulz(torch.empty(*shape, device=dev)).shape == shape
    u = gradient(dev, 8, 8)
    for kw in (dict(steps=0), dict(steps=65), dict(steps=2.0), dict(eps=-1.0),
               dict(coefficients=(3.0, 0.0, 0.0)), dict(coefficients=(float("nan"), 0, 0)),
               dict(out=torch.empty(8, 8, device=dev)),
               dict(out=torch.empty(8, 16, device=dev, dtype=torch.bfloat16)[:, ::2])):
        with pytest.raises(ValueError):
            newton_schulz(u, **kw)
    with pytest.raises(TypeError):
        newton_schulz(u.double())
    with pytest.raises(ValueError):
        newton_schulz(u[0])
    with pytest.raises(ValueError, match="differentiable"):
        newton_schulz(u.clone().requires_grad_())


def test_streams_and_graphs(dev):
    from systems_for_llms_b200.ops.newton_schulz import newton_schulz
    sets = [gradient(dev, 2, 200, 136, seed=s) for s in (1, 2)]
    want = [newton_schulz(s) for s in sets]
    static = [torch.zeros(2, 200, 136, device=dev) for _ in range(2)]
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, results = [], []
    with torch.cuda.stream(side):
        newton_schulz(static[0])
        for s in static:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                results.append(newton_schulz(s))
            graphs.append(graph)
        for mine, theirs in zip(static, sets):
            mine.copy_(theirs)
        other.wait_stream(side)
        graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
        side.wait_stream(other)
    check(dev)
    assert all(torch.equal(a, b) for a, b in zip(results, want))


def test_out_in_place_or_apart(dev):
    from systems_for_llms_b200.ops.newton_schulz import newton_schulz
    torch.manual_seed(40)
    for m, n in [(96, 200), (200, 300), (300, 400)]:     # the three forms
        u = torch.randn(2, m, n, device=dev).bfloat16()
        want = newton_schulz(u)
        same = u.clone()
        assert newton_schulz(same, out=same) is same
        assert torch.equal(same, want)
        store = torch.empty(3, m, n, device=dev, dtype=torch.bfloat16)
        store[:2] = u
        with pytest.raises(ValueError):
            newton_schulz(store[:2], out=store[1:])      # a block would overwrite the next input
        store = torch.randn(2, m, n, device=dev)
        with pytest.raises(ValueError):
            newton_schulz(store, out=store.view(torch.bfloat16).view(-1)[:2 * m * n].view(2, m, n))
        assert torch.equal(newton_schulz(u, out=store.view(torch.bfloat16).view(-1)[:2 * m * n]
                                         .view(2, m, n)), want)
    check(dev)


@pytest.mark.parametrize("shape, steps", [((2, 96, 200), 5), ((200, 300), 3), ((300, 280), 2)])
def test_kernels_are_counted(dev, shape, steps):
    from systems_for_llms_b200.ops import lib
    from systems_for_llms_b200.ops.newton_schulz import newton_schulz
    u = torch.randn(shape, device=dev)
    newton_schulz(u, steps=steps)
    torch.cuda.synchronize()
    before = lib.launch_count()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        newton_schulz(u, steps=steps)
    nodes = ctypes.c_size_t()          # of the captured graph: kernels alone
    assert ctypes.CDLL("libcudart.so.12").cudaGraphGetNodes(
        ctypes.c_void_p(graph.raw_cuda_graph()), None, ctypes.byref(nodes)) == 0
    assert lib.launch_count() - before == nodes.value > 0


@pytest.mark.parametrize("m, n", [(96, 200), (200, 96), (200, 300), (300, 280)])
def test_offsets_beyond_32_bits(dev, m, n):
    from systems_for_llms_b200.ops.newton_schulz import newton_schulz
    u = gradient(dev, 2, m, n).bfloat16()
    want = newton_schulz(u)
    pitch = -(-2 ** 31 // (m - 1)) + 8                 # a matrix whose last row is past 2**31
    store = torch.empty((m - 1) * pitch + 2 * n + 8, dtype=torch.bfloat16, device=dev)
    far = store.as_strided((2, m, n), (n + 4, pitch, 1)).copy_(u)
    assert torch.equal(newton_schulz(far), want)
    apart = torch.empty(2 ** 31 + m * n, dtype=torch.bfloat16, device=dev)
    far = apart.as_strided((2, m, n), (2 ** 31, n, 1)).copy_(u)
    assert torch.equal(newton_schulz(far), want)
    check(dev)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(128, 385), (96, 1000), (1000, 96), (50, 2000), (2, 2500), (1, 700),
                                   (1601, 128), (65, 769), (2049, 33)])
def test_matrices_shared_by_several_blocks(dev, shape, dtype):
    from systems_for_llms_b200.ops.newton_schulz import newton_schulz
    u = gradient(dev, *shape, dtype=dtype, seed=5)
    compare(newton_schulz(u), u)
    check(dev)


def test_stacks_of_shared_matrices(dev):
    from systems_for_llms_b200.ops.newton_schulz import newton_schulz
    for m, n in ((70, 900), (900, 70)):
        u = gradient(dev, 3, 7, m, n, seed=6)
        u[1, 2] = 0
        u[2, 3, 4, 5] = float("nan")
        got = newton_schulz(u)
        check(dev)
        assert (got[1, 2] == 0).all() and got[2, 3].isnan().all()
        for i, j in ((0, 0), (1, 1), (1, 3), (2, 2), (2, 4), (2, 6)):
            assert torch.equal(newton_schulz(u[i, j]), got[i, j])
            compare(got[i, j], u[i, j])
        flat = torch.zeros(3, 9, m + 2, n + 4, device=dev)
        view = flat[:, 1:8, 1:m + 1, 3:n + 3].copy_(u)
        again = newton_schulz(view)
        assert torch.equal(again.nan_to_num(7.0), got.nan_to_num(7.0))
    many = gradient(dev, 200, 40, 500, seed=7)
    got = newton_schulz(many)
    assert torch.equal(got[173], newton_schulz(many[173]))
    check(dev)


@pytest.mark.parametrize("shape", [(40, 72), (64, 500), (200, 300), (300, 280)])
def test_norms_at_the_ends_of_the_range(dev, shape):
    """Entries that are subnormal, or so large that their norm is not an fp32 number.  Scaling by
    powers of two is exact, so the bound is the ordinary one."""
    from systems_for_llms_b200.ops.newton_schulz import newton_schulz
    u = torch.randn(shape, device=dev).clamp(-3, 3)
    for scale in (2.0 ** -140, 2.0 ** -120, 2.0 ** 126):
        scaled = (u.double() * scale).float()
        assert scaled.isfinite().all() and (scaled != 0).any()
        compare(newton_schulz(scaled, eps=0.0), scaled, eps=0.0)
    assert newton_schulz(torch.zeros(shape, device=dev), eps=0.0).isnan().all()
    check(dev)


@pytest.mark.parametrize("shape", [(40, 72), (64, 500), (200, 300), (300, 280)])
def test_the_largest_coefficients(dev, shape):
    """Twice Chebyshev's polynomial of degree five reaches 2 and has the largest coefficients that
    are accepted; with singular values spread over [0, 1] the operands come to their extremes."""
    from systems_for_llms_b200.ops.newton_schulz import newton_schulz
    u = gradient(dev, *shape)
    left, values, right = torch.linalg.svd(u.double(), full_matrices=False)
    spread = torch.linspace(0, 1, values.numel(), device=dev, dtype=torch.float64)
    for few in (spread[-1:], spread):      # one singular value of the whole norm, or all of them
        sv = torch.cat([few, few.new_zeros(values.numel() - few.numel())])
        x = (left * sv @ right).float()
        got = newton_schulz(x, steps=1, coefficients=(10.0, -40.0, 32.0), eps=0.0)
        check(dev)
        compare(got, x, steps=1, coefficients=(10.0, -40.0, 32.0), eps=0.0)
