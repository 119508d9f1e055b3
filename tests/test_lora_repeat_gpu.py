"""GPU: the rank-side products fed by TMA give the same bits in every call, and the right ones in each.

A slot of their rings that is filled again before its last reads are done shows in few rows of few calls, so every shape is called
many times over and compared with its own first result, which is compared with 64 bits.  Sums of M or C bf16 products in fp32: the
largest error is the terms' number times 2^-24 of the sum of magnitudes, of which the square root is the usual size; 2^-15 of that
sum bounds both, and bf16 rounds by 2^-8 at the end."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _right(got, want, size):
    off = (got.double() - want).abs()
    assert bool((off <= want.abs() * 2.0 ** -8 + size * 2.0 ** -15).all()), float((off / (want.abs() * 2.0 ** -8 + size * 2.0 ** -15)).max())


@pytest.mark.parametrize("m,c,r", [(8192, 4096, 8), (8192, 2048, 16), (32768, 2048, 16), (32768, 512, 16), (4099, 4096, 5), (20000, 1160, 16)])
def test_factor_gradient(cuda, m, c, r):
    from b2g import ops

    g = torch.Generator(device=cuda).manual_seed(m + c)
    s = torch.zeros(m, 16, device=cuda, dtype=torch.bfloat16)
    s[:, :r] = torch.randn(m, r, generator=g, device=cuda)
    t = torch.randn(m, c, generator=g, device=cuda).bfloat16()
    first = ops.lora_wgrad(s, t, 0.5, r, False)
    _right(first, 0.5 * (s[:, :r].double().t() @ t.double()), 0.5 * (s[:, :r].double().abs().t() @ t.double().abs()))
    other = torch.zeros((), dtype=torch.int64, device=cuda)
    for _ in range(400):
        other += (ops.lora_wgrad(s, t, 0.5, r, False) != first).any()
    assert int(other) == 0
    ops.check_status()


@pytest.mark.parametrize("m,c,r", [(8192, 4096, 8), (32768, 2048, 16), (50000, 512, 16), (777, 4096, 3)])
def test_projection(cuda, m, c, r):
    from b2g import ops

    g = torch.Generator(device=cuda).manual_seed(m + c)
    x = torch.randn(m, c, generator=g, device=cuda).bfloat16()
    w = (torch.randn(r, c, generator=g, device=cuda) / 16).bfloat16()
    first, _ = ops.lora_down(x, w, False, 2.0, r)
    _right(first[:, :r], x.double() @ w.double().t(), x.double().abs() @ w.double().abs().t())
    assert bool((first[:, r:] == 0).all())
    other = torch.zeros((), dtype=torch.int64, device=cuda)
    for _ in range(400):
        other += (ops.lora_down(x, w, False, 2.0, r)[0] != first).any()
    assert int(other) == 0
    ops.check_status()
