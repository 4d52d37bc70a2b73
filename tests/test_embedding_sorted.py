"""Scaled embedding with given positions and its gradient by sorted tokens, against sums in 64 bits."""
import pytest
import torch

from pippy_b200.ops import _lib
from pippy_b200.ops import functional as pf

gpu = pytest.mark.gpu
U = 2.0 ** -8  # a bf16 rounding is off by at most this much of the value
F32 = 2.0 ** -24


@pytest.fixture
def errors():
    yield
    _lib.check_device_errors()


def _sums(keys, rows, size, scale=1.0):
    """Sums of the rows of each key in 64 bits, sums of their absolute values, and how many there are."""
    ok = (keys >= 0) & (keys < size)
    value = torch.zeros(size, rows.shape[1], dtype=torch.float64, device=rows.device)
    size_of = torch.zeros_like(value)
    count = torch.zeros(size, 1, dtype=torch.float64, device=rows.device)
    value.index_add_(0, keys[ok], rows[ok].double() * scale)
    size_of.index_add_(0, keys[ok], (rows[ok].double() * scale).abs())
    count.index_add_(0, keys[ok], torch.ones(int(ok.sum()), 1, dtype=torch.float64, device=rows.device))
    return value, size_of, count


def test_plain_form():
    ids = torch.tensor([[3, 1, 1], [0, 3, 3]])
    wte, wpe = (torch.randn(n, 8, dtype=torch.float64, requires_grad=True) for n in (4, 3))
    pos = torch.tensor([0, 1, -1, 2, -1, 0])
    out = pf.embedding(ids, wte, wpe, 3, scale=2.5, positions=pos)
    want = 2.5 * wte.detach()[ids.reshape(-1)]
    want[pos >= 0] += wpe.detach()[pos[pos >= 0]]
    assert torch.allclose(out, want, rtol=1e-14, atol=0)
    g = torch.randn_like(out)
    dw, dp = torch.autograd.grad(out, (wte, wpe), g)
    assert torch.allclose(dw, _sums(ids.reshape(-1), g, 4, 2.5)[0]) and torch.allclose(dp, _sums(pos, g, 3)[0])
    assert torch.equal(pf.embedding(ids, wte, wpe, 3, sorted_grad=True), pf.embedding(ids, wte, wpe, 3))
    assert torch.autograd.gradcheck(lambda a, b: pf.embedding(ids, a, b, 3, scale=2.5, positions=pos), (wte, wpe))


def test_refusals():
    wte = torch.zeros(4, 8)
    for kw in (dict(positions=torch.zeros(2, dtype=torch.int32)), dict(wpe=wte, positions=torch.zeros(3, dtype=torch.int32)),
               dict(wpe=wte, positions=torch.zeros(2))):
        with pytest.raises(ValueError):
            pf.embedding(torch.tensor([1, 2]), wte, **kw)


@pytest.mark.skipif(not _lib.available(), reason="the CUDA library is not built")
def test_entry_points_refuse_before_they_launch():
    lib, at = _lib.lib(), 1 << 20  # an address that is only looked at

    def forward(H=64, wpe=None, positions=None, seq=4, out=at):
        return lib.pb_embed_scaled_fwd(at, at, wpe, positions, out, 8, H, seq, 10, 5, 1.0, at, None)

    def backward(T=8, H=64, V=10, gw=at, gp=None, P=5, seq=4, scratch=at):
        return lib.pb_embed_sorted_bwd(at, None, at, gw, gp, T, H, seq, V, P, 1.0, 1, scratch, None)

    assert forward(H=12) == forward(H=0) == forward(wpe=at, seq=0) == -1 and forward(out=at + 8) == -2
    assert backward(H=4) == backward(V=0) == backward(gp=at, P=0) == backward(gp=at, seq=0) == -1
    assert backward(T=-1) == backward(T=2 ** 31) == backward(V=2 ** 31 - 1) == -2 and backward(scratch=at + 4) == -3
    assert backward(gw=None) == 0  # no gradient wanted: nothing to do


# ------------------------------------------------------------------------------------------------ GPU
CASES = {  # tokens, rows of the table, width, share of one id
    "one": (1, 5, 8, 0.0),
    "few": (33, 300, 64, 0.0),
    "one_row": (1000, 1, 72, 0.0),
    "odd": (3001, 257, 1000, 0.0),
    "hot": (20_000, 5000, 128, 0.5),
    "wide": (700, 70_000, 2056, 0.1),
    "all_one": (5000, 40, 256, 1.0),
    "long": (200_003, 1 << 17, 16, 0.2),
}


def _ids(T, V, hot, seed=0):
    gen = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, V, (T,), generator=gen)
    ids[torch.rand(T, generator=gen) < hot] = V // 2
    return ids.cuda(), gen


@gpu
@pytest.mark.parametrize("case", sorted(CASES))
@pytest.mark.parametrize("buffers", [True, False])
@pytest.mark.parametrize("given", [True, False])
def test_kernel(case, buffers, given, errors):
    T, V, H, hot = CASES[case]
    S, P, scale = max(1, T // 3), max(1, T // 3) + 2, 1.5
    ids, gen = _ids(T, V, hot)
    wte, wpe = (torch.nn.Parameter(torch.randn(n, H, generator=gen).bfloat16().cuda()) for n in (V, P))
    pos = torch.randint(-1, P, (T,), generator=gen).cuda() if given else torch.arange(T, device="cuda") % S
    dout = torch.randn(T, H, generator=gen).bfloat16().cuda()
    start = [torch.randn(p.shape, generator=gen).cuda() for p in (wte, wpe)]

    def call():
        for p, b in zip((wte, wpe), start):
            p.grad = None
            if buffers:
                p.main_grad = b.clone()
        out = pf.embedding(ids, wte, wpe, S, scale=scale, positions=pos if given else None, sorted_grad=True)
        out.backward(dout)
        return out.detach(), [p.main_grad if buffers else p.grad for p in (wte, wpe)]

    out, grads = call()
    want = scale * wte.detach().double()[ids]
    want[pos >= 0] += wpe.detach().double()[pos[pos >= 0]]
    size = scale * wte.detach().double()[ids].abs() + wpe.detach().double().abs().max()
    assert ((out.double() - want).abs() <= U * want.abs() + 4 * F32 * size).all()
    for g, b, keys, factor in zip(grads, start, (ids, pos), (scale, 1.0)):
        value, magnitude, count = _sums(keys, dout, g.shape[0], factor)
        # n additions of bf16 values in fp32, a product, one more addition or the rounding to bf16
        bound = (count + 3) * F32 * magnitude
        if buffers:
            value, bound = value + b.double(), bound + 2 * F32 * (value.abs() + b.double().abs())
            assert g.dtype == torch.float32 and torch.equal(g[count.view(-1) == 0], b[count.view(-1) == 0])
        else:
            bound = bound * (1 + U) + U * value.abs()
            assert g.dtype == torch.bfloat16 and not g[count.view(-1) == 0].any()
        assert ((g.double() - value).abs() <= bound).all()
    again = call()
    assert torch.equal(again[0], out) and all(torch.equal(a, b) for a, b in zip(again[1], grads))


@gpu
def test_kernel_accumulates_and_respects_frozen_tables(errors):
    ids, gen = _ids(500, 60, 0.1)
    wte, wpe = (torch.nn.Parameter(torch.randn(n, 32, generator=gen).bfloat16().cuda()) for n in (60, 100))
    dout = torch.randn(500, 32, generator=gen).bfloat16().cuda()
    value = _sums(ids, dout, 60)
    for _ in range(2):  # .grad is added to
        pf.embedding(ids, wte, seq_len=100, sorted_grad=True).backward(dout)
    assert ((wte.grad.double() - 2 * value[0]).abs() <= 4 * U * (2 * value[0].abs()) + 200 * F32 * value[1]).all()
    wte.grad = None
    wte.requires_grad_(False)
    pf.embedding(ids, wte, wpe, 100, sorted_grad=True).backward(dout)
    assert wte.grad is None and wpe.grad is not None
    pf.embedding(ids, wte, wpe, 100, scale=3.0).backward(dout)
    wte.requires_grad_(True)
    wte.main_grad = torch.zeros(60, 32, device="cuda")  # one table with a buffer, one without
    wpe.grad = None
    pf.embedding(ids, wte, wpe, 100, sorted_grad=True).backward(dout)
    assert ((wte.main_grad.double() - value[0]).abs() <= U * value[0].abs() + 500 * F32 * value[1]).all()
    assert wpe.grad is not None
    with torch.no_grad():
        assert pf.embedding(ids[:0], wte, wpe, 100, sorted_grad=True).shape == (0, 32)


@gpu
def test_kernel_reports_bad_ids():
    ids = torch.tensor([3, -1, 60, 5, 2 ** 40], device="cuda")
    wte = torch.nn.Parameter(torch.ones(60, 16, device="cuda").bfloat16())
    out = pf.embedding(ids, wte, scale=2.0)
    out.backward(torch.ones_like(out))
    assert torch.equal(out[:, 0].float().cpu(), torch.tensor([2.0, 0, 0, 2.0, 0]))
    assert wte.grad.sum() == 2 * 16 * 2.0
    with pytest.raises(_lib.KernelError, match="code 5"):
        _lib.check_device_errors()
    wpe = torch.ones(4, 16, device="cuda").bfloat16()
    out = pf.embedding(ids[:1].repeat(3), wte, wpe, positions=torch.tensor([-1, 3, 4], device="cuda"))
    assert torch.equal(out[:, 0].float().cpu(), torch.tensor([1.0, 2.0, 1.0]))
    with pytest.raises(_lib.KernelError, match="code 5"):
        _lib.check_device_errors()
    with pytest.raises(ValueError):
        pf.embedding(ids.cpu(), wte, scale=2.0)
    with pytest.raises(ValueError):
        pf.embedding(ids, torch.ones(60, 12, device="cuda").bfloat16(), scale=2.0)


@gpu
def test_kernel_streams_graph_and_deferral(errors):
    from pippy_b200.backward import DeferredWeightGrads, defer_weight_grads

    T, V, H = 4000, 900, 256
    cases = []
    for seed in (1, 2):
        ids, gen = _ids(T, V, 0.2, seed)
        cases.append((ids, torch.randn(T, H, generator=gen).bfloat16().cuda()))
    wte = torch.nn.Parameter(torch.randn(V, H).bfloat16().cuda())

    def call(ids, dout):
        table = torch.nn.Parameter(wte.detach())
        table.main_grad = torch.zeros(V, H, device="cuda")
        pf.embedding(ids, table, sorted_grad=True).backward(dout)
        return table.main_grad

    want = [call(*c) for c in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], []
    for _ in range(3):
        for i, c in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got.append((i, call(*c)))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i, g in got)
    ids, dout = cases[0][0].clone(), cases[0][1].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(ids, dout)
    for i in (1, 0):
        ids.copy_(cases[i][0]), dout.copy_(cases[i][1])
        graph.replay()
        assert torch.equal(out, want[i])
    wte.main_grad = torch.zeros(V, H, device="cuda")
    queue = DeferredWeightGrads()
    with defer_weight_grads(queue):
        pf.embedding(cases[0][0], wte, sorted_grad=True).backward(cases[0][1])
    assert not wte.main_grad.any()
    queue.run()
    assert torch.equal(wte.main_grad, want[0])


@gpu
def test_kernel_captured_while_an_eager_graph_of_the_tables_lives(errors):
    T, V, H = 300, 50, 64
    ids, gen = _ids(T, V, 0.2)
    wte, wpe = (torch.nn.Parameter(torch.randn(n, H, generator=gen).bfloat16().cuda()) for n in (V, 100))
    dout = torch.randn(T, H, generator=gen).bfloat16().cuda()
    for p in (wte, wpe):
        p.main_grad = torch.zeros(p.shape, device="cuda")
    eager = pf.embedding(ids, wte, wpe, 100, sorted_grad=True)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        pf.embedding(ids, wte, wpe, 100, sorted_grad=True).backward(dout)
    eager.backward(dout)
    want = [p.main_grad.clone() for p in (wte, wpe)]
    for p in (wte, wpe):
        p.main_grad.zero_()
    graph.replay()
    assert all(w.any() and torch.equal(p.main_grad, w) for p, w in zip((wte, wpe), want))


@gpu
def test_kernel_empty_batch_wide_positions_and_refusals(errors):
    wte, wpe = (torch.nn.Parameter(torch.ones(n, 16, device="cuda").bfloat16()) for n in (60, 7))
    out = pf.embedding(torch.zeros(2, 0, dtype=torch.long, device="cuda"), wte, wpe, sorted_grad=True)
    out.backward(torch.ones_like(out))
    assert out.shape == (0, 16) and not wte.grad.any() and not wpe.grad.any()
    ids = torch.tensor([1, 2, 3], device="cuda")
    positions = torch.tensor([2, -5, 2 ** 32 + 1], device="cuda")  # the last would be 1 in 32 bits
    with torch.no_grad():
        assert torch.equal(pf.embedding(ids, wte, wpe, positions=positions)[:, 0].float().cpu(), torch.tensor([2.0, 1.0, 1.0]))
    with pytest.raises(_lib.KernelError, match="code 5"):
        _lib.check_device_errors()
    with pytest.raises(ValueError, match="both tables"):
        pf.embedding(ids, wte, wte, sorted_grad=True)
    with pytest.raises(ValueError, match="leaves"):
        pf.embedding(ids, wte * 2, sorted_grad=True)


@gpu
@pytest.mark.parametrize("V,H,T", [(5000, 1024, 40), (5000, 1024, 900), (300, 4096, 64), (129, 2048, 7)])
def test_kernel_writes_the_rows_that_do_not_occur(V, H, T, errors):
    """Gradients written whole, with few tokens for the table: zeros in every other row, whatever the memory held."""
    ids, gen = _ids(T, V, 0.1)
    ids[0], ids[-1] = 0, V - 1
    wte, wpe = (torch.nn.Parameter(torch.randn(n, H, generator=gen).bfloat16().cuda()) for n in (V, V + 1))
    pos = torch.randint(-1, V + 1, (T,), generator=gen).cuda()
    dout = torch.randn(T, H, generator=gen).bfloat16().cuda()
    torch.full((2 * V + 1, H), float("nan"), device="cuda", dtype=torch.bfloat16)  # leaves NaN in the memory that comes next
    pf.embedding(ids, wte, wpe, positions=pos, sorted_grad=True).backward(dout)
    for p, keys in ((wte, ids), (wpe, pos)):
        value, magnitude, count = _sums(keys, dout, p.shape[0])
        assert not p.grad[count.view(-1) == 0].any()
        assert ((p.grad.double() - value).abs() <= (1 + U) * (count + 3) * F32 * magnitude + U * value.abs()).all()


# ------------------------------------------------------------------------------------------------ place in the graph
def test_whose_accumulation_nodes_are_held_elsewhere():
    leaf = torch.nn.Parameter(torch.ones(3))
    assert not pf._held_elsewhere(leaf, 1) and not pf._held_elsewhere(leaf, 1)
    graph = leaf * 2
    assert pf._held_elsewhere(leaf, 1) and pf._held_elsewhere(leaf, 1)
    del graph
    assert not pf._held_elsewhere(leaf, 1)
    graph = leaf * 2
    torch.autograd.graph.get_gradient_edge(leaf).node.metadata[pf._MADE_ON] = 1
    assert not pf._held_elsewhere(leaf, 1) and pf._held_elsewhere(leaf, 2)
    del graph


def _tables(V=50, P=100, H=64, T=300):
    ids, gen = _ids(T, V, 0.2)
    wte, wpe = (torch.nn.Parameter(torch.randn(n, H, generator=gen).bfloat16().cuda()) for n in (V, P))
    return ids, wte, wpe, torch.randn(T, H, generator=gen).bfloat16().cuda()


@gpu
@pytest.mark.parametrize("buffers", [False, True])
def test_kernel_gradients_of_chosen_inputs_and_hooks(buffers, errors):
    """What goes by the tables' accumulation nodes: ``inputs=`` of a backward, and hooks."""
    ids, wte, wpe, dout = _tables()
    want = [_sums(ids, dout, 50), _sums(torch.arange(300, device="cuda") % 100, dout, 100)]
    seen = []
    for p in (wte, wpe):
        p.register_post_accumulate_grad_hook(seen.append)

    def check(chosen):
        for p, (value, magnitude, count) in zip((wte, wpe), want):
            got = p.main_grad if buffers else p.grad
            if any(p is q for q in chosen):
                assert ((got.double() - value).abs() <= (1 + U) * (count + 3) * F32 * magnitude + U * value.abs()).all()
        assert len(seen) == len(chosen) and all(any(p is q for q in seen) for p in chosen)

    for chosen in ([wte, wpe], [wte], [wpe]):
        for p in (wte, wpe):
            p.grad = None
            if buffers:
                p.main_grad = torch.zeros(p.shape, device="cuda")
        seen.clear()
        pf.embedding(ids, wte, wpe, 100, sorted_grad=True).backward(dout, inputs=chosen)
        check(chosen)


@gpu
def test_kernel_captured_gradients_of_chosen_inputs(errors):
    """Without another graph of the tables, a captured one has them as inputs: two at a time, and one capture after another."""
    ids, wte, wpe, dout = _tables()
    for p in (wte, wpe):
        p.main_grad = torch.zeros(p.shape, device="cuda")
    pf.embedding(ids, wte, wpe, 100, sorted_grad=True).backward(dout)
    want = [2 * p.main_grad for p in (wte, wpe)]  # exactly: two equal sums
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            for p in (wte, wpe):
                p.main_grad.zero_()
            outs = [pf.embedding(ids, wte, wpe, 100, sorted_grad=True) for _ in range(2)]
            for out in outs:
                out.backward(dout, inputs=[wte, wpe])
        graphs.append((graph, outs))
    for graph, _ in graphs:
        for p in (wte, wpe):
            p.main_grad.fill_(3.0)
        graph.replay()
        assert all(torch.equal(p.main_grad, w) for p, w in zip((wte, wpe), want))


def _ddp(rank, world):
    from torch.nn.parallel import DistributedDataParallel

    from pippy_b200.models.gpt2 import GPT2Config, GPT2Stage

    torch.cuda.set_device(0)
    cfg = GPT2Config(vocab_size=300, n_positions=128, dim=128, n_layers=1, n_heads=2)
    torch.manual_seed(0)
    model = GPT2Stage(cfg, range(1), True, True, device="cuda", dtype=torch.bfloat16)
    ids, lengths = torch.randint(0, 300, (2, 128), device="cuda"), torch.tensor([[100, 28], [40, 60]], device="cuda")
    g = torch.randn(2, 128, cfg.padded_vocab, device="cuda").bfloat16()

    def grads(m):
        for p in model.parameters():
            p.grad = None
        m(ids, lengths=lengths).backward(g)
        torch.cuda.synchronize()
        return [p.grad.clone() for p in model.parameters()]

    want = grads(model)
    wrapped = DistributedDataParallel(model, device_ids=[0])
    for _ in range(2):  # a parameter that was never counted as ready shows in the second step
        for a, b in zip(grads(wrapped), want):
            assert (a - b).norm() <= 2 * U * b.norm()  # the same sums, each rounded once, whatever their order


@gpu
def test_packed_stage_in_a_data_parallel_wrapper():
    from _mp import run_ranks

    run_ranks(_ddp, 1, backend="nccl")


@gpu
@pytest.mark.parametrize("which", ["wte", "wpe", "unaligned", "strided"])
def test_kernel_keeps_fp32_for_the_table_that_has_a_buffer(which, errors):
    """One table with an fp32 buffer and one without; buffers that the kernel cannot add to: no rounding to bf16 on the way."""
    ids, wte, wpe, dout = _tables()
    want = [_sums(ids, dout, 50), _sums(torch.arange(300, device="cuda") % 100, dout, 100)]
    for p, name in ((wte, "wte"), (wpe, "wpe")):
        if which == "unaligned":
            p.main_grad = torch.zeros(p.numel() + 1, device="cuda")[1:].view(p.shape)
        elif which == "strided":
            p.main_grad = torch.zeros(p.shape[0], 2 * p.shape[1], device="cuda")[:, : p.shape[1]]
        elif which == name:
            p.main_grad = torch.zeros(p.shape, device="cuda")
    pf.embedding(ids, wte, wpe, 100, sorted_grad=True).backward(dout)
    for p, (value, magnitude, count) in zip((wte, wpe), want):
        bound = (count + 3) * F32 * magnitude
        if hasattr(p, "main_grad"):
            assert p.grad is None and ((p.main_grad.double() - value).abs() <= bound).all()
        else:
            assert ((p.grad.double() - value).abs() <= (1 + U) * bound + U * value.abs()).all()


@gpu
@pytest.mark.parametrize("which", ["aligned", "unaligned", "strided", "unaligned_gradient"])
def test_adding_bf16_gradients_to_fp32_buffers_of_any_layout(which, errors):
    p = torch.nn.Parameter(torch.zeros(24, 16, device="cuda").bfloat16())
    room = torch.zeros(2 * p.numel() + 1, device="cuda")
    p.main_grad = {"aligned": room[: p.numel()].view(p.shape), "unaligned": room[1 : p.numel() + 1].view(p.shape),
                   "strided": room[: 2 * p.numel()].view(24, 32)[:, :16],
                   "unaligned_gradient": room[: p.numel()].view(p.shape)}[which]
    p.main_grad.fill_(1.0)
    g = torch.randn(p.numel() + 1, device="cuda").bfloat16()
    g = (g[1:] if which == "unaligned_gradient" else g[:-1]).view(p.shape)
    outside = room.sum() - p.main_grad.sum()
    pf._accumulate_param_grad(p, g)
    assert torch.equal(p.main_grad, 1.0 + g.float()) and p.grad is None
    assert outside == 0 and (room != 0).sum() <= p.numel()
