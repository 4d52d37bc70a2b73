"""Models on packed documents: a packed batch gives what its documents give one by one."""
import pytest
import torch

from _mp import run_ranks

LENGTHS = [[5, 0, 7, 3], [16, 0, 0, 0], [1, 1, 9, 4]]
S = 16


def _documents(ids, lengths):
    for row, counts in zip(ids, lengths):
        at = 0
        for n in counts:
            if n:
                yield row[at : at + n].unsqueeze(0)
            at += n


def _inside(lengths):
    return torch.tensor([[t < sum(row) for t in range(S)] for row in lengths])


def _llama(dtype):
    from pippy_b200.models.llama import Llama, LlamaConfig

    torch.manual_seed(0)
    return Llama(LlamaConfig.tiny(vocab_size=64, dim=32, n_layers=2, n_heads=4, n_kv_heads=2, ffn_dim=48), dtype=dtype)


def _gpt2(dtype, **kw):
    from pippy_b200.models.gpt2 import GPT2Config, GPT2Stage

    torch.manual_seed(0)
    cfg = GPT2Config(vocab_size=60, n_positions=S, dim=32, n_layers=2, n_heads=2, vocab_multiple=8, **kw)
    return GPT2Stage(cfg, range(2), True, True, dtype=dtype)


def _mixtral(dtype):
    from pippy_b200.models.mixtral import MixtralConfig, MixtralStage

    torch.manual_seed(0)
    cfg = MixtralConfig(vocab_size=64, dim=32, n_layers=2, n_heads=4, n_kv_heads=2, ffn_dim=48, n_experts=4, aux_coef=0.0)
    return MixtralStage(cfg, range(2), True, True, dtype=dtype)


def _tp(dtype):
    from pippy_b200.models.llama import LlamaConfig
    from pippy_b200.models.llama_tp import TPLlamaStage

    torch.manual_seed(0)
    cfg = LlamaConfig.tiny(vocab_size=64, dim=32, n_layers=2, n_heads=4, n_kv_heads=2, ffn_dim=48)
    return TPLlamaStage(cfg, range(2), True, True, None, 1, 0, len(LENGTHS), S, dtype=dtype)


@pytest.mark.parametrize("build", [_llama, _gpt2, _mixtral, _tp])
def test_packed_batch_equals_its_documents(build):
    model = build(torch.float64)
    ids = torch.randint(0, 60, (3, S), generator=torch.Generator().manual_seed(1))
    lengths = torch.tensor(LENGTHS)
    inside = _inside(LENGTHS)
    g = torch.randn(int(inside.sum()), 64, dtype=torch.float64, generator=torch.Generator().manual_seed(2))
    out = model(ids, lengths=lengths)[inside]
    packed = torch.autograd.grad(out, list(model.parameters()), g)
    if build is _tp:  # a module of one shape: each document alone in its row
        alone = []
        for b, d in enumerate(_documents(ids, LENGTHS)):
            rows = torch.zeros(3, S, dtype=torch.int64)
            rows[0, : d.shape[1]] = d
            alone.append(model(rows)[0, : d.shape[1]])
        alone = torch.cat(alone)
    else:
        alone = torch.cat([model(d)[0] for d in _documents(ids, LENGTHS)])
    # fp32 inside the plain norms and attention of the dense path: 2^-24 of sums of some tens of terms, a few layers deep
    assert torch.allclose(out, alone, rtol=1e-4, atol=1e-6)
    for a, b in zip(packed, torch.autograd.grad(alone, list(model.parameters()), g)):
        assert torch.allclose(a, b, rtol=1e-3, atol=1e-5)
    with pytest.raises(ValueError):
        model(ids, lengths=lengths[:2])


def test_recomputation_keeps_the_layout():
    from pippy_b200.models.llama import LlamaConfig, LlamaStage

    cfg = LlamaConfig.tiny(vocab_size=64, dim=32, n_layers=2, n_heads=4, ffn_dim=48)
    ids, lengths = torch.randint(0, 64, (3, S), generator=torch.Generator().manual_seed(1)), torch.tensor(LENGTHS)
    grads = []
    for again in (False, True):
        torch.manual_seed(0)
        model = LlamaStage(cfg, range(2), True, True, dtype=torch.float64, activation_checkpointing=again)
        model(ids, lengths=lengths)[_inside(LENGTHS)].square().sum().backward()
        grads.append([p.grad for p in model.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_dropout_of_gpt2():
    """Reproducible under a seed, another mask otherwise, nothing in evaluation; the gradient is that of the same masks."""
    model = _gpt2(torch.float64, dropout=0.2)
    plain = _gpt2(torch.float64)
    ids = torch.randint(0, 60, (2, S), generator=torch.Generator().manual_seed(1))

    def run(seed):
        torch.manual_seed(seed)
        return model(ids)

    assert torch.equal(run(1), run(1)) and not torch.equal(run(1), run(2))
    w = model.h["1"].mlp_c_fc.weight
    direction = torch.randn(w.shape, dtype=w.dtype, generator=torch.Generator().manual_seed(3))
    (grad,) = torch.autograd.grad(run(1).square().sum(), w)
    step = 1e-3
    with torch.no_grad():
        w += step * direction
        up = run(1).square().sum()
        w -= 2 * step * direction
        down = run(1).square().sum()
        w += step * direction
    # the difference's error is step^2 of the third derivative; norms run in 32 bits: 2^-24 of the sum over 2 step
    assert abs((up - down) / (2 * step) - (grad * direction).sum()) < 1e-2 * abs((grad * direction).sum()) + 1e-3
    model.eval()
    plain.load_state_dict(model.state_dict())
    assert torch.equal(model(ids), plain(ids))


def _train(rank, world, schedule):
    import torch.distributed as dist

    from pippy_b200.models.llama import LlamaConfig, causal_lm_loss
    from pippy_b200.train import build_llama_pipeline

    cfg = LlamaConfig.tiny(vocab_size=64, dim=32, n_layers=4, n_heads=4, ffn_dim=48)
    lengths = torch.tensor(LENGTHS + [[2, 2, 0, 12]])
    ids = torch.randint(0, 64, (4, S), generator=torch.Generator().manual_seed(1))
    target = torch.where(torch.cat([_inside(LENGTHS), torch.ones(1, S, dtype=torch.bool)]), ids.roll(-1, 1), -100)
    stages = 1 if schedule == "1f1b" else 2
    pipe = build_llama_pipeline(cfg, 4, S, 2, torch.device("cpu"), schedule=schedule, virtual_stages=stages, dtype=torch.float64,
                                lr=0.0, weight_decay=0.0)
    loss = pipe.train_step(ids if pipe.holds_first else None, target if pipe.holds_last else None, lengths)
    if not pipe.holds_last:
        return
    from pippy_b200.models.llama import build_llama_stage

    n = stages * world
    parts = []
    for s in range(n):
        torch.manual_seed(s)
        parts.append(build_llama_stage(cfg, s, n, dtype=torch.float64, pp_size=world, seq_len=S))
    want = []
    for mb in range(2):
        rows = slice(2 * mb, 2 * mb + 2)
        h = (ids[rows],)
        for part in parts:
            h = part(*h, lengths=lengths[rows])
            h = h if isinstance(h, tuple) else (h,)
        want.append(causal_lm_loss(h[0], target[rows]))
    # the losses are fp32 sums of 64 exponentials and some 30 tokens, the same on both sides but for their place in a batch
    assert abs(loss - torch.stack(want).mean()) < 100 * 2.0 ** -24 * loss, (loss, want, pipe.losses)


@pytest.mark.parametrize("schedule", ["1f1b", "interleaved_1f1b", "zero_bubble"])
def test_lengths_through_a_pipeline(schedule):
    run_ranks(_train, 2, schedule)


def _padding_free(lengths, ids, seq):
    """The documents of ``ids``, whose rows end in padding, in one row without any: ids, lengths, and where its tokens are."""
    inside = torch.tensor([[t < sum(row) for t in range(seq)] for row in lengths])
    return ids[inside].unsqueeze(0), torch.tensor([[n for row in lengths for n in row]]), inside


def test_padding_is_not_routed_to_experts():
    """With a balance loss, a batch whose rows end in padding trains as the same documents without any."""
    from pippy_b200.models.mixtral import MixtralConfig, MixtralStage

    torch.manual_seed(0)
    cfg = MixtralConfig(vocab_size=64, dim=32, n_layers=2, n_heads=4, n_kv_heads=2, ffn_dim=48, n_experts=4, aux_coef=0.5)
    model = MixtralStage(cfg, range(2), True, True, dtype=torch.float64)
    ids = torch.randint(0, 60, (3, S), generator=torch.Generator().manual_seed(1))
    ids[~_inside(LENGTHS)] = 7
    tight, tight_lengths, inside = _padding_free(LENGTHS, ids, S)
    g = torch.randn(int(inside.sum()), 64, dtype=torch.float64, generator=torch.Generator().manual_seed(2))
    results = []
    for tokens, lengths, rows in ((ids, torch.tensor(LENGTHS), inside), (tight, tight_lengths, torch.ones_like(tight).bool())):
        model.zero_grad()
        out = model(tokens, lengths=lengths)[rows]
        out.backward(g)
        results.append([out.detach(), *model.aux_losses(), *(p.grad.clone() for p in model.parameters())])
    # fp32 inside the plain attention, router and norms: as in the test above
    for a, b in zip(*results):
        assert torch.allclose(a, b, rtol=1e-3, atol=1e-5)
    model.zero_grad()
    out = model(ids, lengths=torch.zeros(3, 1, dtype=torch.int64))  # nothing but padding
    out.sum().backward()
    assert out.isfinite().all() and not torch.stack(model.aux_losses()).any()
    assert all(p.grad is None or not p.grad.any() for p in model.expert_parameters())
    moe = model.layers["0"].block_sparse_moe
    with pytest.raises(ValueError, match="positions"):
        moe(torch.zeros(4, 32, dtype=torch.float64), torch.zeros(3, dtype=torch.int32))


# ------------------------------------------------------------------------------------------------ GPU
@pytest.mark.gpu
def test_operators_together_on_the_gpu():
    """A GPT-2 with scaled embeddings, packed documents, sorted table gradients and dropout: the same in bf16 on the GPU, in the
    kernels, as on the CPU in 64 bits, whose masks are the same; and the same bits again."""
    from pippy_b200.models.gpt2 import GPT2Config, GPT2Stage
    from pippy_b200.ops import _lib
    from pippy_b200.ops import functional as pf

    lengths = torch.tensor([[100, 0, 257, 3], [128, 129, 1, 0], [384, 0, 0, 0]], dtype=torch.int32)
    S2 = 400
    cfg = GPT2Config(vocab_size=500, n_positions=S2, dim=128, n_layers=2, n_heads=2, dropout=0.1, sorted_embedding_grad=True)
    torch.manual_seed(0)
    model = GPT2Stage(cfg, range(2), True, True, dtype=torch.bfloat16)
    ids = torch.randint(0, 500, (3, S2))
    exact = GPT2Stage(cfg, range(2), True, True, dtype=torch.float64)
    exact.load_state_dict(model.state_dict())
    model = model.cuda()
    layout = pf.packed_layout(lengths, S2)
    inside = (layout.positions >= 0).view(3, S2)
    g = torch.randn(3, S2, cfg.padded_vocab).bfloat16() * inside.unsqueeze(2)

    def run(m, device, seed):
        m.zero_grad()
        for p in m.parameters():
            p.grad = None
        draw = pf_draw(seed)
        old, layers.Dropout.draw = layers.Dropout.draw, staticmethod(lambda d: draw.to(d))
        try:
            out = m(ids.to(device), lengths=lengths.to(device))
            out.backward(g.to(device).to(out.dtype))
        finally:
            layers.Dropout.draw = old
        return out.detach(), {n: p.grad for n, p in m.named_parameters()}

    from pippy_b200.models import layers

    def pf_draw(seed):
        return torch.tensor([seed])

    out, grads = run(model, "cuda", 7)
    again, grads2 = run(model, "cuda", 7)
    assert torch.equal(out, again) and torch.equal(grads["wte.positions"], grads2["wte.positions"])
    other, _ = run(model, "cuda", 8)
    assert not torch.equal(out, other)
    want, wanted = run(exact, "cpu", 7)
    # about 12 roundings to bf16 a block and 4 around the blocks, each 2^-9 of the value in the mean square, in random directions:
    # sqrt(28) 2^-9 = 0.010 forward; a gradient passes as many again: sqrt(56) 2^-9 = 0.015.  Twice that.
    def off(a, b):
        return ((a.double().cpu() - b).norm() / b.norm()).item()

    assert off(out[inside.cuda()], want[inside]) < 0.02
    for name, b in wanted.items():
        assert off(grads[name], b) < 0.03, name
    _lib.check_device_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("checkpointing", [False, True])
def test_packed_llama_training_step_on_the_gpu(checkpointing):
    """A packed batch through a pipeline with fp32 gradient buffers: each gradient against the documents' own, one by one."""
    from pippy_b200.models.llama import LlamaConfig
    from pippy_b200.ops import _lib
    from pippy_b200.train import build_llama_pipeline

    cfg = LlamaConfig.tiny(vocab_size=512, dim=256, n_layers=2, n_heads=4, n_kv_heads=2, ffn_dim=512)
    lengths = torch.tensor([[100, 0, 257, 3], [128, 129, 1, 0]], dtype=torch.int32)
    S2 = 400
    ids = torch.randint(0, 512, (2, S2), generator=torch.Generator().manual_seed(1))
    inside = torch.tensor([[t < int(row.sum()) for t in range(S2)] for row in lengths])
    target = torch.where(inside, ids.roll(-1, 1), -100)

    def build(batch, seq):
        return build_llama_pipeline(cfg, batch, seq, 1, torch.device("cuda"), schedule="1f1b", lr=0.0, weight_decay=0.0,
                                    activation_checkpointing=checkpointing)

    pipe = build(2, S2)
    pipe.optimizer, kept = None, pipe.optimizer
    pipe.flat.zero_grad()
    loss = pipe.train_step(ids.cuda(), target.cuda(), lengths.cuda())
    got = pipe.flat.grad.clone()
    model = pipe.stages[0].submod
    pipe.flat.zero_grad()
    # the same documents, one at a time, each loss weighted as in the packed mean
    from pippy_b200.models.llama import causal_lm_loss

    total, count = 0.0, int((target != -100).sum())
    for row in range(2):
        at = 0
        for n in lengths[row].tolist():
            if n:
                part = causal_lm_loss(model(ids[row : row + 1, at : at + n].cuda()), target[row : row + 1, at : at + n].cuda())
                (part * (n / count)).backward()
                total += part.item() * n / count
            at += n
    want = pipe.flat.grad.clone()
    # both sides round the same values to bf16, in tiles of other shapes: sqrt(2) times the 0.015 of the test above, twice
    assert abs(loss.item() - total) < 0.01 * total
    assert ((got - want).norm() / want.norm()).item() < 0.04
    _lib.check_device_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("T,share", [(384, 0.3), (1500, 0.9), (700, 1.0), (1, 0.0), (513, 0.0)])
def test_experts_leave_padding_out_on_the_gpu(T, share):
    """The kernels of the expert layer with padding among the rows, whatever it holds, against the dense layer on the others."""
    from pippy_b200.ops import _lib
    from pippy_b200.parallel.ep import EPContext, MoEFeedForward

    H, Fd, E, k = 256, 512, 4, 2
    gen = torch.Generator().manual_seed(T)
    inside = (torch.rand(T, generator=gen) < share).cuda()
    n = int(inside.sum())
    positions = torch.where(inside, 5, -1).int()
    # room for the tokens alone
    ep = EPContext(None, max_tokens=max(n, 1), hidden=H, top_k=k, n_experts=E, capacity_factor=1.0)
    torch.manual_seed(5)
    dense = MoEFeedForward(H, Fd, E, k, None, 1, 0, aux_coef=0.5, device="cuda", dtype=torch.bfloat16)
    fused = MoEFeedForward(H, Fd, E, k, ep, 1, 0, aux_coef=0.5, device="cuda", dtype=torch.bfloat16)
    fused.load_state_dict(dense.state_dict())
    for p in fused.parameters():
        p.main_grad = torch.zeros(p.shape, device="cuda")
    x = torch.randn(T, H, generator=gen).bfloat16().cuda()
    x[~inside] *= 100
    dy = torch.randn(T, H, generator=gen).bfloat16().cuda()
    x.requires_grad_(True)
    out = fused(x, positions)
    out.backward(dy)
    assert not out[~inside].any() and not x.grad[~inside].any()
    if n:
        xd = x.detach()[inside].requires_grad_(True)
        ref = dense(xd)
        ref.backward(dy[inside])

        def off(a, b):
            return ((a.float() - b.float()).norm() / b.float().norm()).item()

        # the tolerances that the layer is held to without padding
        assert off(out[inside], ref) < 2e-2 and off(x.grad[inside], xd.grad) < 2e-2
        assert off(fused.router.main_grad[:E], dense.router.grad[:E]) < 3e-2
        assert off(fused.w_down.main_grad, dense.w_down.grad) < 2e-2
        assert off(fused.w_gate_up.main_grad, dense.w_gate_up.grad) < 2e-2
        assert abs(float(fused.last_aux_loss) - float(dense.last_aux_loss)) < 1e-3
    else:
        assert float(fused.last_aux_loss) == 0.0 and not any(p.main_grad.any() for p in fused.parameters())
    _lib.check_device_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["mixtral", "tp"])
def test_packed_mixtral_and_tensor_parallel_on_the_gpu(form):
    """The packed forms in bf16 on the kernels against themselves in 64 bits on the CPU: outputs and gradients."""
    from pippy_b200.ops import _lib

    lengths = torch.tensor([[100, 0, 57, 3], [128, 65, 1, 0]], dtype=torch.int32)
    S2 = 200
    ids = torch.randint(0, 500, (2, S2), generator=torch.Generator().manual_seed(1))
    inside = torch.tensor([[t < int(row.sum()) for t in range(S2)] for row in lengths])

    def build(device, dtype):
        torch.manual_seed(0)
        if form == "tp":
            from pippy_b200.models.llama import LlamaConfig
            from pippy_b200.models.llama_tp import TPLlamaStage

            cfg = LlamaConfig.tiny(vocab_size=512, dim=256, n_layers=2, n_heads=4, n_kv_heads=2, ffn_dim=512)
            return TPLlamaStage(cfg, range(2), True, True, None, 1, 0, 2, S2, dtype=dtype).to(device)
        from pippy_b200.models.mixtral import MixtralConfig, MixtralStage
        from pippy_b200.parallel.ep import EPContext

        cfg = MixtralConfig(vocab_size=512, dim=256, n_layers=2, n_heads=4, n_kv_heads=2, ffn_dim=512, n_experts=4, top_k=4)
        ep = EPContext(None, 2 * S2, 256, 4, 4) if device == "cuda" else None
        # all experts for each token: a top-k that a rounding tips to another expert would be no error of the kernels
        return MixtralStage(cfg, range(2), True, True, ep, dtype=dtype).to(device)

    model, exact = build("cuda", torch.bfloat16), build("cpu", torch.float64)
    exact.load_state_dict(model.state_dict())
    g = torch.randn(2, S2, 512, generator=torch.Generator().manual_seed(2)).bfloat16() * inside.unsqueeze(2)
    for m, device in ((model, "cuda"), (exact, "cpu")):
        for p in m.parameters():
            p.grad = None
        out = m(ids.to(device), lengths=lengths.to(device))
        out.backward(g.to(device).to(out.dtype))
        m.out = out.detach()

    def off(a, b):
        return ((a.double().cpu() - b).norm() / b.norm()).item()

    # as in test_operators_together_on_the_gpu; routing, gather and weighted sum of the experts add 6 roundings a block:
    # sqrt(28 + 12) 2^-9 = 0.012 forward, sqrt(80) 2^-9 = 0.0175 for a gradient.  Twice that and a little.
    assert off(model.out[inside.cuda()], exact.out[inside]) < 0.025
    for (name, a), b in zip(model.named_parameters(), exact.parameters()):
        assert off(a.grad, b.grad) < 0.04, (name, off(a.grad, b.grad))
    _lib.check_device_errors()


def _pipelined_gradients(pipe, stages, ids, target, lengths, loss_fn, device, n_mb):
    """Gradients of one packed step of ``pipe``, and of ``stages`` run one after the other: pairs by stage and name."""
    pipe.optimizer, pipe.tied = None, None
    pipe.flat.zero_grad()
    ids, target, lengths = ids.to(device), target.to(device), lengths.to(device)
    pipe.train_step(ids if pipe.holds_first else None, target if pipe.holds_last else None, lengths)
    pipe.flat.fold_autograd_grads()
    for rows, labels, counts in zip(ids.tensor_split(n_mb), target.tensor_split(n_mb), lengths.tensor_split(n_mb)):
        h = (rows,)
        for part in stages:
            h = part(*h, lengths=counts)
            h = h if isinstance(h, tuple) else (h,)
        loss_fn(h[0], labels).backward()
    for st in pipe.stages:
        for (name, p), q in zip(st.submod.named_parameters(), stages[st.stage_index].parameters()):
            yield f"{st.stage_index}.{name}", p.main_grad, q.grad


def _llama_pipeline(device, schedule, world, dtype, dim=32, seq=S):
    from pippy_b200.models.llama import LlamaConfig, build_llama_stage, causal_lm_loss
    from pippy_b200.train import build_llama_pipeline

    cfg = LlamaConfig.tiny(vocab_size=64, dim=dim, n_layers=4, n_heads=dim // 8 if dim < 128 else dim // 64, ffn_dim=48)
    v = 1 if schedule == "1f1b" else 2
    pipe = build_llama_pipeline(cfg, 4, seq, 2, device, schedule=schedule, virtual_stages=v, dtype=dtype, weight_decay=0.0)
    stages = []
    for s in range(v * world):
        torch.manual_seed(s)
        stages.append(build_llama_stage(cfg, s, v * world, device=device, dtype=dtype, pp_size=world, seq_len=seq))
    return pipe, stages, causal_lm_loss


def _gpt2_pipeline(device, schedule, world, dtype, dim=32, seq=S):
    from pippy_b200.models.gpt2 import GPT2Config, build_gpt2_stage, gpt2_loss
    from pippy_b200.train import build_gpt2_pipeline

    cfg = GPT2Config(vocab_size=60, n_positions=seq, dim=dim, n_layers=4, n_heads=dim // 16 if dim < 128 else dim // 64,
                     vocab_multiple=8)
    v = 1 if schedule == "1f1b" else 2
    pipe = build_gpt2_pipeline(cfg, 4, seq, 2, device, schedule=schedule, virtual_stages=v, dtype=dtype, weight_decay=0.0)
    stages = []
    for s in range(v * world):
        torch.manual_seed(s)
        stages.append(build_gpt2_stage(cfg, s, v * world, device=device, dtype=dtype))
    if len(stages) > 1 and not (pipe.holds_first and pipe.holds_last):
        with torch.no_grad():  # the embedding's values, as the pipeline's broadcast sets them; a gradient of its own
            stages[-1].lm_head.weight.copy_(stages[0].wte.weight)
    elif len(stages) > 1:
        stages[-1].lm_head.weight = stages[0].wte.weight
    return pipe, stages, gpt2_loss(cfg)


FAMILIES = {"llama": _llama_pipeline, "gpt2": _gpt2_pipeline}


def _gradients(rank, world, family, schedule):
    pipe, stages, loss_fn = FAMILIES[family](torch.device("cpu"), schedule, world, torch.float64)
    lengths = torch.tensor(LENGTHS + [[2, 2, 0, 12]])
    ids = torch.randint(0, 60, (4, S), generator=torch.Generator().manual_seed(1))
    target = torch.where(torch.cat([_inside(LENGTHS), torch.ones(1, S, dtype=torch.bool)]), ids.roll(-1, 1), -100)
    compared = 0
    for name, got, want in _pipelined_gradients(pipe, stages, ids, target, lengths, loss_fn, "cpu", 2):
        # fp32 inside the plain norms and the loss, and in the buffers: 2^-24 of sums of some tens of terms
        assert want.any() and torch.allclose(got.double(), want, rtol=1e-4, atol=1e-6), name
        compared += 1
    assert compared


@pytest.mark.parametrize("family", sorted(FAMILIES))
@pytest.mark.parametrize("schedule", ["1f1b", "interleaved_1f1b", "zero_bubble"])
def test_gradients_of_a_packed_step_through_a_pipeline(family, schedule):
    """Every stage of every rank: its parameters' gradients are those of the stages run one after the other."""
    run_ranks(_gradients, 2, family, schedule)


@pytest.mark.gpu
@pytest.mark.parametrize("family", sorted(FAMILIES))
@pytest.mark.parametrize("schedule", ["interleaved_1f1b", "zero_bubble"])
def test_gradients_of_a_packed_step_through_two_stages_on_the_gpu(family, schedule):
    """The kernels, two stages of one rank, weight gradients deferred (zero bubble) or not: against the stages run one after
    the other on the same kernels without buffers."""
    from pippy_b200.ops import _lib

    S2 = 300
    pipe, stages, loss_fn = FAMILIES[family](torch.device("cuda"), schedule, 1, torch.bfloat16, dim=128, seq=S2)
    lengths = torch.tensor([[100, 0, 150, 3], [128, 129, 1, 0], [300, 0, 0, 0], [64, 1, 1, 30]], dtype=torch.int32)
    ids = torch.randint(0, 60, (4, S2), generator=torch.Generator().manual_seed(1))
    inside = torch.tensor([[t < int(row.sum()) for t in range(S2)] for row in lengths])
    target = torch.where(inside, ids.roll(-1, 1), -100)
    for name, got, want in _pipelined_gradients(pipe, stages, ids, target, lengths, loss_fn, "cuda", 2):
        # the same bf16 activations on both sides; each of the two microbatches' gradients, and their sum, rounded to bf16 on
        # one side and added in fp32 on the other: 3 roundings of 2^-9 in the mean square, twice
        assert want.any() and (got - want.float()).norm() <= 2 * 3 ** 0.5 * 2.0 ** -9 * want.float().norm(), name
    _lib.check_device_errors()
