"""Rotary, projection loss and Newton-Schulz calls on two streams at once (needs a B200)."""

import pytest
import torch

pytestmark = pytest.mark.gpu


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


def jobs(dev, seed):
    from systems_for_llms_b200.ops import linear_loss as L
    from systems_for_llms_b200.ops import rotary as R
    from systems_for_llms_b200.ops.newton_schulz import newton_schulz
    gen = torch.Generator(device=dev).manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device=dev, generator=gen)
    h, w = rnd(700, 256).bfloat16().requires_grad_(), rnd(3000, 256).bfloat16().requires_grad_()
    t = torch.randint(3000, (700,), device=dev, generator=gen)
    q, k = rnd(2, 8, 300, 128).bfloat16(), rnd(2, 4, 300, 128).bfloat16()
    weight = 1 + 0.1 * rnd(128)
    cos, sin = R.rotary_tables(128, 512, device=dev)

    def loss():
        value = L.linear_cross_entropy(h, w, t)
        return (value.detach(), *torch.autograd.grad(value, (h, w)))

    def turn():
        return (*R.qk_norm_rotary(q, k, weight, weight, cos, sin),
                *R.qk_norm_rotary_grad(q, k, weight, weight, cos, sin, None, q, k, eps=1e-5,
                                       layout="interleaved"))

    stacks = [rnd(*s) for s in ((5, 100, 900), (3, 300, 500), (2, 200, 400), (4, 64, 64))]
    return [loss, turn, *((lambda u=u: (newton_schulz(u),)) for u in stacks)]


def test_calls_on_two_streams_do_not_disturb_each_other(dev):
    from systems_for_llms_b200.ops.gemm import check_status
    lists = [jobs(dev, seed) for seed in (1, 2)]
    want = [[job() for job in each] for each in lists]
    streams = [torch.cuda.Stream() for _ in lists]
    for stream in streams:
        stream.wait_stream(torch.cuda.current_stream())
    got = []
    for turn in range(20):
        for j in range(len(lists[0])):
            for i, stream in enumerate(streams):       # unlike kinds side by side
                at = (j + 3 * i + turn) % len(lists[i])
                with torch.cuda.stream(stream):
                    got.append((i, at, lists[i][at]()))
    torch.cuda.synchronize()
    check_status()
    for i, at, result in got:
        assert all(torch.equal(a, b) for a, b in zip(result, want[i][at])), (i, at)
