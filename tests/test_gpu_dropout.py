"""Counter-based dropout (csrc/dropout.hip): the mask against a numpy Philox4x32-10, bit for bit."""
import numpy as np
import pytest
import torch

from conftest import pkg

pytestmark = pytest.mark.gpu


def philox(n, seed, step):
    """Word of each of n elements: key = seed, counter = (element // 4, step), word element % 4."""
    m = np.uint64(0xFFFFFFFF)
    blk = np.arange((n + 3) // 4, dtype=np.uint64)
    seed, step = seed % (1 << 64), step % (1 << 64)
    c = [blk & m, blk >> np.uint64(32), np.full_like(blk, step & 0xFFFFFFFF), np.full_like(blk, step >> 32)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & m, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & m]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, 1).reshape(-1)[:n]


def expected(x, rate, seed, step):
    keep = torch.from_numpy(philox(x.numel(), seed, step) >= np.uint64(round(rate * 2.0 ** 32))).reshape(x.shape)
    f = torch.tensor(1.0 / (1.0 - rate), dtype=torch.float32)
    return torch.where(keep, (x.float().cpu() * f).to(x.dtype), torch.zeros((), dtype=x.dtype))


def test_philox_published_vectors():
    """The three known-answer vectors of the Random123 distribution (philox4x32, 10 rounds) that have
    counter = (element // 4, step) form with element // 4 = 0 or all ones are covered by counter 0."""
    assert [hex(v) for v in philox(4, 0, 0)] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1,), (3,), (8,), (7, 5), (257, 333), (64, 2048), (4099, 17)])
@pytest.mark.parametrize("rate", [0.0, 0.2, 0.5, 0.9])
def test_mask_and_gradient(cuda, dtype, shape, rate):
    F = pkg("functional")
    g = torch.Generator().manual_seed(3)
    x = torch.randn(shape, generator=g).to(dtype).cuda().requires_grad_(True)
    dy = torch.randn(shape, generator=g).to(dtype).cuda()
    seed, step = 0x1234567890ABCDEF, 41
    y = F.dropout(x, rate, torch.tensor([seed, step], device="cuda"))
    dx, = torch.autograd.grad(y, (x,), dy)
    assert torch.equal(y.detach().cpu(), expected(x.detach(), rate, seed, step))
    assert torch.equal(dx.cpu(), expected(dy, rate, seed, step))
