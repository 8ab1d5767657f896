"""Counter-based dropout (csrc/dropout.hip): the mask against a numpy Philox4x32-10, bit for bit."""
import numpy as np
import pytest
import torch

from conftest import pkg

pytestmark = pytest.mark.gpu
DTYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
M32 = np.uint64(0xFFFFFFFF)


def philox(n, seed, step, first=0):
    """Words of elements first .. first + n - 1 (first % 4 == 0): key = seed, counter = (element // 4, step)."""
    blk = np.arange(first // 4, first // 4 + (n + 3) // 4, dtype=np.uint64)
    seed, step = seed % (1 << 64), step % (1 << 64)
    c = [blk & M32, blk >> np.uint64(32), np.full_like(blk, step & 0xFFFFFFFF), np.full_like(blk, step >> 32)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & M32, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & M32]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, 1).reshape(-1)[:n]


def kept(shape, rate, seed, step, first=0):
    n = int(np.prod(shape))
    return torch.from_numpy(philox(n, seed, step, first) >= np.uint64(round(rate * 2.0 ** 32))).reshape(shape)


def expected(x, rate, seed, step, first=0):
    f = torch.tensor(1.0 / (1.0 - rate), dtype=torch.float32)
    return torch.where(kept(x.shape, rate, seed, step, first), (x.float().cpu() * f).to(x.dtype),
                       torch.zeros((), dtype=x.dtype))


def ticket(seed, step):
    return torch.tensor([seed, step], device="cuda")


def test_philox_known_answer():
    """The generator's published known answer for a zero key and counter."""
    assert [hex(v) for v in philox(4, 0, 0)] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]


@DTYPES
@pytest.mark.parametrize("shape", [(1,), (3,), (8,), (7, 5), (257, 333), (64, 2048), (4099, 17)])
@pytest.mark.parametrize("rate", [0.0, 0.2, 0.5, 0.9])
def test_mask_and_gradient(cuda, dtype, shape, rate):
    F = pkg("functional")
    g = torch.Generator().manual_seed(3)
    x = torch.randn(shape, generator=g).to(dtype).cuda().requires_grad_(True)
    dy = torch.randn(shape, generator=g).to(dtype).cuda()
    seed, step = 0x1234567890ABCDEF, 41
    y = F.dropout(x, rate, ticket(seed, step))
    dx, = torch.autograd.grad(y, (x,), dy)
    assert torch.equal(y.detach().cpu(), expected(x.detach(), rate, seed, step))
    assert torch.equal(dx.cpu(), expected(dy, rate, seed, step))


@DTYPES
@pytest.mark.parametrize("seed,step", [(0, 0), (-1, -1), (1 << 40, (1 << 33) + 5), (-(1 << 63), 1 << 62)])
def test_every_bit_of_the_ticket_counts(cuda, dtype, seed, step):
    F = pkg("functional")
    x = torch.ones((37, 41), dtype=dtype, device="cuda")
    assert torch.equal(F.dropout_apply(x, 0.3, ticket(seed, step)).cpu(), expected(x, 0.3, seed, step))


@DTYPES
def test_layouts_in_place_and_what_is_dropped(cuda, dtype):
    F = pkg("functional")
    base = torch.randn(1001, device="cuda").to(dtype)
    x = base[1:]                      # off every vector boundary
    want = expected(x, 0.5, 7, 1)
    assert torch.equal(F.dropout_apply(x, 0.5, ticket(7, 1)).cpu(), want)
    buf = torch.zeros(1001, dtype=dtype, device="cuda")
    F.dropout_apply(x, 0.5, ticket(7, 1), out=buf[1:])
    assert torch.equal(buf[1:].cpu(), want) and float(buf[0]) == 0
    y = x.clone()
    assert F.dropout_apply(y, 0.5, ticket(7, 1), out=y) is y and torch.equal(y.cpu(), want)
    t = torch.randn(40, 50, device="cuda").to(dtype)
    assert torch.equal(F.dropout(t.t(), 0.5, ticket(7, 1)).cpu(), expected(t.t().contiguous(), 0.5, 7, 1))
    # whatever a dropped element holds, it is zero; a kept one passes on
    bad = torch.full((64, 64), float("nan"), dtype=dtype, device="cuda")
    bad[::2] = float("inf")
    out = F.dropout_apply(bad, 0.5, ticket(7, 1)).cpu()
    keep = kept(bad.shape, 0.5, 7, 1)
    assert bool((out[~keep] == 0).all()) and not bool(out[keep].isfinite().any())
    e = F.dropout(torch.empty((0, 5), dtype=dtype, device="cuda", requires_grad=True), 0.5, ticket(7, 1))
    assert e.shape == (0, 5)


@pytest.mark.parametrize("rate", [2.0 ** -32, 0.1, 1 - 2.0 ** -20])
def test_kept_share(cuda, rate):
    """The kept count of 2^24 elements lies within six standard deviations of its mean."""
    F = pkg("functional")
    n = 1 << 24
    got = int((F.dropout_apply(torch.ones(n, device="cuda"), rate, ticket(99, 3)) != 0).sum())
    assert abs(got - n * (1 - rate)) <= 6 * (n * rate * (1 - rate)) ** 0.5 + 1


def test_more_than_32_bits_of_elements(cuda):
    if torch.cuda.get_device_properties(0).total_memory < 40 << 30:
        pytest.skip("needs 40 GB")
    F = pkg("functional")
    n = (1 << 32) + 44
    x = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    F.dropout_apply(x, 0.25, ticket(5, 6), out=x)
    first = (1 << 32) - 4096
    tail = x[first:].cpu()
    assert torch.equal(tail, expected(torch.ones_like(tail), 0.25, 5, 6, first))


def test_tickets_and_streams(cuda):
    F = pkg("functional")
    state = F.dropout_state(123, "cuda")
    a, b = F.dropout_ticket(state), F.dropout_ticket(state)
    assert a.tolist() == [123, 0] and b.tolist() == [123, 1] and state.tolist() == [123, 2]
    # two masks before a backward: each backward makes its own again
    x = torch.randn((64, 33), device="cuda", requires_grad=True)
    ya, yb = F.dropout(x, 0.5, a), F.dropout(x, 0.5, b)
    ga, = torch.autograd.grad(ya, (x,), torch.ones_like(ya), retain_graph=True)
    gb, = torch.autograd.grad(yb, (x,), torch.ones_like(yb))
    ga2, = torch.autograd.grad(ya, (x,), torch.ones_like(ya))
    assert torch.equal(ga.cpu(), 2.0 * kept(x.shape, 0.5, 123, 0)) and torch.equal(ga, ga2)
    assert torch.equal(gb.cpu(), 2.0 * kept(x.shape, 0.5, 123, 1))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        yc = F.dropout(x, 0.5, a)
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(yc, ya)


def test_module_modes_and_replays(cuda):
    models = pkg("models")
    drop = models.Dropout(0.4, seed=17, device="cuda")
    x = torch.randn((128, 96), device="cuda")
    assert torch.equal(drop(x).cpu(), expected(x, 0.4, 17, 0))
    assert drop.eval()(x) is x and drop(x, training=False) is x
    assert torch.equal(drop(x, training=True).cpu(), expected(x, 0.4, 17, 1))
    drop.train()
    # a captured step: every replay advances the step on the device
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        drop(x)
    torch.cuda.current_stream().wait_stream(st)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = drop(x)
    for step in (3, 4, 5):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.cpu(), expected(x, 0.4, 17, step))
    assert drop.state.tolist() == [17, 6]
    models.set_dropout_seed(drop, 5)
    assert drop.state.tolist() == [5, 0]


def test_refusals(cuda):
    F = pkg("functional")
    x, t = torch.ones(8, device="cuda"), ticket(1, 2)
    for rate in (-0.1, 1.0, 2.0, float("nan")):
        with pytest.raises(ValueError, match="rate"):
            F.dropout_apply(x, rate, t)
        with pytest.raises(ValueError, match="rate"):
            F.dropout(x, rate, t)
    with pytest.raises(pkg("_native").NativeError, match="keeps no element"):
        F.dropout_apply(x, 1 - 2.0 ** -40, t)
    with pytest.raises(TypeError):
        F.dropout_apply(x.half(), 0.5, t)
    with pytest.raises(TypeError):
        F.dropout_apply(x, 0.5, t.int())
    with pytest.raises(ValueError, match="seed, step"):
        F.dropout_apply(x, 0.5, t[:1])
    with pytest.raises(RuntimeError, match="ROCm device"):
        F.dropout_apply(x, 0.5, t.cpu())
    with pytest.raises(ValueError, match="contiguous"):
        F.dropout_apply(torch.ones((4, 4), device="cuda").t()[1:], 0.5, t)
    with pytest.raises(ValueError, match="out"):
        F.dropout_apply(x, 0.5, t, out=torch.ones(9, device="cuda"))
    with pytest.raises(RuntimeError):
        v = x.clone().requires_grad_(True)
        g, = torch.autograd.grad(F.dropout(v, 0.5, t).sum(), (v,), create_graph=True)
        g.sum().backward()


def test_what_a_kernel_writes_counts_as_written(cuda):
    """A generator used as its own ticket and then advanced, or an activation that dropout wrote over, is refused by the
    backward that needs what they held."""
    F = pkg("functional")
    state = F.dropout_state(3, "cuda")
    x = torch.randn((16, 8), device="cuda", requires_grad=True)
    y = F.dropout(x, 0.5, state)
    F.dropout_ticket(state)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    F.dropout(x, 0.5, state).sum().backward()   # not advanced in between: its own mask
    assert torch.equal(x.grad.cpu(), 2.0 * kept(x.shape, 0.5, 3, 1))
    e = torch.exp(x)
    F.dropout_apply(e.detach(), 0.5, ticket(1, 2), out=e.detach())
    with pytest.raises(RuntimeError, match="inplace"):
        e.sum().backward()
    # the module's tickets are copies: two calls before a backward
    drop = pkg("models").Dropout(0.5, seed=9, device="cuda")
    a, b = drop(x), drop(x)
    x.grad = None
    (a + 2 * b).sum().backward()
    assert torch.equal(x.grad.cpu(), 2.0 * kept(x.shape, 0.5, 9, 0) + 4.0 * kept(x.shape, 0.5, 9, 1))
    with torch.inference_mode():
        F.dropout_apply(torch.ones(8, device="cuda"), 0.5, F.dropout_ticket(F.dropout_state(3, "cuda")))
