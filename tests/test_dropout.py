"""Dropout with a computed mask: the generator, the plain form and the kernel."""
import math

import pytest
import torch

from pippy_b200.ops import _lib
from pippy_b200.ops import functional as pf

gpu = pytest.mark.gpu
U = 2.0 ** -8  # a bf16 rounding is off by at most this much of the value


def _numbers(seed, stream, count):
    """Philox4x32-10 in Python's integers, block by block."""
    out = []
    for block in range(-(-count // 8)):
        x = [block % 2 ** 32, block >> 32, stream % 2 ** 32, stream >> 32]
        k = [seed % 2 ** 32, seed >> 32]
        for _ in range(10):
            a, b = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57
            x = [(b >> 32) ^ x[1] ^ k[0], b % 2 ** 32, (a >> 32) ^ x[3] ^ k[1], a % 2 ** 32]
            k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
        for w in x:
            out += [w % 2 ** 16, w >> 16]
    return torch.tensor(out[:count])


def test_generator():
    # the authors' known answer for a counter and a key of zeros
    words = [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert _numbers(0, 0, 8).tolist() == [h for w in words for h in (w % 2 ** 16, w >> 16)]
    for seed, stream in ((0, 0), (2 ** 63 - 1, 5), (2 ** 64 - 3, 2 ** 63 - 1), (1234567890123, 2 ** 32)):
        value = seed - 2 ** 64 if seed >= 2 ** 63 else seed
        assert torch.equal(pf._philox_numbers(value, stream, 101, "cpu"), _numbers(seed, stream, 101))


@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.9999])
def test_plain_form(p):
    x = torch.randn(37, 11, dtype=torch.float64, requires_grad=True)
    res = torch.randn(37, 11, dtype=torch.float64, requires_grad=True)
    threshold = math.floor(p * 65536 + 0.5)
    mask = (_numbers(77, 3, x.numel()) >= threshold).double().view(x.shape) * 65536 / (65536 - threshold)
    y = pf.dropout(x, p, 77, residual=res, stream=3)
    assert torch.allclose(y, x * mask + res, rtol=1e-14, atol=0)
    assert torch.equal(y, pf.dropout(x, p, torch.tensor([77]), residual=res, stream=3))
    g = torch.randn_like(y)
    dx, dr = torch.autograd.grad(y, (x, res), g)
    assert torch.allclose(dx, g * mask, rtol=1e-14, atol=0) and torch.equal(dr, g)
    assert torch.autograd.gradcheck(lambda a, b: pf.dropout(a, p, 77, residual=b, stream=3), (x, res))


def test_rate_and_streams():
    x = torch.ones(1 << 20)
    masks = [pf.dropout(x, 0.3, seed, stream=stream) != 0 for seed, stream in ((1, 0), (1, 1), (2, 0))]
    for m in masks:  # 5 standard deviations of a binomial share
        assert abs(m.double().mean() - 0.7) < 5 * math.sqrt(0.21 / x.numel())
    for a, b in ((0, 1), (0, 2), (1, 2)):
        assert abs((masks[a] == masks[b]).double().mean() - 0.58) < 5 * math.sqrt(0.58 * 0.42 / x.numel())


def test_refusals():
    x = torch.zeros(4, 4)
    for kw in (dict(p=1.0), dict(p=-0.1), dict(p=math.nan), dict(p=0.999999), dict(stream=-1), dict(stream=2 ** 63),
               dict(residual=x[:2]), dict(residual=x.double()), dict(seed=torch.zeros(2, dtype=torch.int64)),
               dict(seed=torch.zeros(1, dtype=torch.int32))):
        with pytest.raises(ValueError):
            pf.dropout(x, **{**dict(p=0.1, seed=1), **kw})


# ------------------------------------------------------------------------------------------------ GPU
@gpu
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (3, 5, 11), (257, 64), (1000, 1003)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.75])
@pytest.mark.parametrize("with_residual", [True, False])
def test_kernel(shape, p, with_residual):
    gen = torch.Generator().manual_seed(3)
    x, res, g = (torch.randn(shape, generator=gen).bfloat16() for _ in range(3))
    x[x == 0] = 1.0
    seed = 2 ** 62 + 12345
    y_cpu = pf.dropout(x.double(), p, seed, residual=res.double() if with_residual else None, stream=9)
    dx_cpu = pf.dropout(g.double(), p, seed, stream=9)
    a, r = x.cuda().requires_grad_(True), res.cuda().requires_grad_(True)
    y = pf.dropout(a, p, torch.tensor([seed], device="cuda"), residual=r if with_residual else None, stream=9)
    grads = torch.autograd.grad(y, (a, r) if with_residual else (a,), g.cuda())
    # one rounding to bf16; before it a product and a sum in fp32, and the factor itself, 2^-24 each
    for got, want, size in ((y.detach(), y_cpu, x.double().abs() + res.double().abs()), (grads[0], dx_cpu, g.double().abs())):
        assert got.dtype == torch.bfloat16
        fine = 4 * 2.0 ** -24 * size / (1 - p)
        assert ((got.cpu().double() - want).abs() <= U * want.abs() + fine).all()
        if not with_residual:
            assert torch.equal(got.cpu() == 0, want == 0)
    if with_residual:
        assert torch.equal(grads[1], g.cuda())
    assert torch.equal(y, pf.dropout(a, p, seed, residual=r if with_residual else None, stream=9))


@gpu
def test_kernel_views_and_masked_values():
    x = torch.randn(64, 129, device="cuda").bfloat16()
    seed = torch.tensor([5], device="cuda")
    want = pf.dropout(x[:, 1:].contiguous(), 0.4, seed)
    assert torch.equal(pf.dropout(x[:, 1:], 0.4, seed), want)  # rows with a gap
    assert torch.equal(pf.dropout(x.t(), 0.4, seed), pf.dropout(x.t().contiguous(), 0.4, seed))
    flat = torch.randn(1025, device="cuda").bfloat16()
    assert torch.equal(pf.dropout(flat[1:], 0.4, seed), pf.dropout(flat[1:].clone(), 0.4, seed))  # starts on 2 bytes
    dropped = want == 0
    bad = torch.where(dropped, math.nan, x[:, 1:].float()).bfloat16()
    assert torch.equal(pf.dropout(bad, 0.4, seed), want)
    assert pf.dropout(x[:0], 0.4, seed).shape == (0, 129)
    with pytest.raises(ValueError):
        pf.dropout(x, 0.1, torch.tensor([1]))


@gpu
def test_kernel_seed_on_the_device():
    """A captured call draws the mask of the seed that its tensor holds at each replay, in the forward and in the backward; a
    seed that changes between the two is an error, not another mask."""
    x = torch.randn(100, 64, device="cuda").bfloat16().requires_grad_(True)
    seed = torch.tensor([1], device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = pf.dropout(x, 0.5, seed)
        (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    for value in (1, 2, -7):
        seed.fill_(value)
        graph.replay()
        assert torch.equal(y, pf.dropout(x, 0.5, value)) and torch.equal(dx != 0, y != 0)
    y = pf.dropout(x, 0.5, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


@gpu
def test_kernel_second_derivative():
    x = torch.randn(64, 40, device="cuda").bfloat16().requires_grad_(True)
    g = torch.randn(64, 40, device="cuda").bfloat16().requires_grad_(True)
    (dx,) = torch.autograd.grad(pf.dropout(x, 0.5, 3), x, g, create_graph=True)
    (dg,) = torch.autograd.grad(dx, g, torch.ones_like(dx))
    assert torch.equal(dg, pf.dropout(torch.ones_like(x), 0.5, 3))


@gpu
def test_kernel_beyond_32_bits():
    """Element numbers beyond 2^32 reach the counter's second word."""
    n = 2 ** 32 + 4099
    x = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    y = pf.dropout(x, 0.5, 11)
    first = 2 ** 32 - 8
    block = torch.arange(first // 8, first // 8 + 600)
    low = 0xFFFFFFFF
    v, k = [block & low, block >> 32, torch.zeros_like(block), torch.zeros_like(block)], [11, 0]
    for _ in range(10):
        a, b = v[0] * 0xD2511F53, v[2] * 0xCD9E8D57
        v = [((b >> 32) & low) ^ v[1] ^ k[0], b & low, ((a >> 32) & low) ^ v[3] ^ k[1], a & low]
        k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
    words = torch.stack(v, 1)
    keep = torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[: n - first] >= 32768
    assert torch.equal(y[first:].cpu() != 0, keep[: n - first]) and len(keep) == n - first
    del x, y
    torch.cuda.empty_cache()
    assert _lib.lib().pb_dropout(None, None, None, -1, None, 0, 0, 0, None) == -1


def _replica_masks(rank, world):
    import torch.distributed as dist

    from pippy_b200.models.gpt2 import GPT2Config
    from pippy_b200.parallel.mesh import init_mesh
    from pippy_b200.train import build_gpt2_pipeline

    mesh = init_mesh(dp_size=world)
    cfg = GPT2Config(vocab_size=60, n_positions=16, dim=32, n_layers=2, n_heads=2, vocab_multiple=8, dropout=0.5)
    pipe = build_gpt2_pipeline(cfg, 4, 16, 2, torch.device("cpu"), group=mesh.pp_group, dp_group=mesh.dp_group,
                               dtype=torch.float32, lr=0.0, weight_decay=0.0)
    drawn, original = [], pf.dropout

    def record(x, p, seed, residual=None, stream=0):
        drawn.append(original(torch.ones(64), p, seed, stream=stream).tolist())
        return original(x, p, seed, residual=residual, stream=stream)

    weights = torch.cat([p.detach().reshape(-1) for p in pipe.stages[0].submod.parameters()]).tolist()
    ids = torch.randint(0, 60, (4, 16), generator=torch.Generator().manual_seed(1))
    pf.dropout = record
    try:
        pipe.train_step(ids, ids)
    finally:
        pf.dropout = original
    replicas = [None] * world
    dist.all_gather_object(replicas, (weights, drawn))
    assert replicas[0][0] == replicas[1][0]  # the same model
    masks = [tuple(m) for _, ms in replicas for m in ms]
    assert len(masks) == 2 * 2 * 5 and len(set(masks)) == len(masks)  # 2 microbatches of embedding and 2 masks a block


def test_data_parallel_replicas_draw_masks_of_their_own():
    from _mp import run_ranks

    run_ranks(_replica_masks, 2)


def test_blocks_beyond_32_bits():
    """A block's number beyond 2^32 (from 2^35 elements on) reaches the counter's second word; Python's integers."""
    blocks = [0, 2 ** 32 - 1, 2 ** 32, 2 ** 32 + 1, 2 ** 45 + 7]
    got = pf._philox_blocks(9, 2 ** 33 + 1, torch.tensor(blocks))
    for block, numbers in zip(blocks, got.tolist()):
        x, k = [block % 2 ** 32, block >> 32, 1, 2], [9, 0]
        for _ in range(10):
            a, b = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57
            x = [(b >> 32) ^ x[1] ^ k[0], b % 2 ** 32, (a >> 32) ^ x[3] ^ k[1], a % 2 ** 32]
            k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
        assert numbers == [h for w in x for h in (w % 2 ** 16, w >> 16)]
    assert len(set(map(tuple, got.tolist()))) == len(blocks)


@pytest.mark.parametrize("p", [-0.1, 1.0 - 2.0 ** -17, 1.0, math.nan])
def test_the_layer_refuses_what_its_forward_would(p):
    from pippy_b200.models.layers import Dropout

    with pytest.raises(ValueError):
        Dropout(p)
    assert Dropout(1.0 - 2.0 ** -16)(torch.ones(8), seed=1).shape == (8,)
