"""Cases of the operators that train on packed documents: attention over documents of different lengths in one batch, the
token embedding with its gradient by sorted tokens, and dropout whose mask is never stored.

  attention  ``packed_layout`` + ``packed_attention``: rotary positions that restart with every document, grouped heads,
             forward alone or forward and backward
  embedding  ``embedding`` with a scale and explicit positions; gradients of both tables by sorted tokens
  dropout    ``dropout``, with or without the residual add, forward and backward

Head counts, widths and vocabularies are those of the families' own configurations (GPT-2 small, Llama-2-7B, the
grouped-query MoE); documents are a log-normal mix of lengths, as text corpora are.
"""
import math
import random

import torch

own = False

BF16 = torch.bfloat16


def listed():
    return [
        # one short row of a small model's batch: latency of the launches; GPT-2's heads, learned positions
        dict(name="attention_small", kind="attention", rows=1, seq=333, docs=5, fill=1.0, sigma=1.0, heads=12, kv_heads=12,
             head_dim=64, rotary=False, causal=True, backward=True, mix=1),
        # GPT-2 small's microbatch filled with documents of some 170 tokens
        dict(name="attention_gpt2", kind="attention", rows=2, seq=1024, docs=6, fill=0.97, sigma=1.0, heads=12, kv_heads=12,
             head_dim=64, rotary=False, causal=True, backward=True, mix=2),
        # the 7B microbatch of 2 x 4096 tokens: a few long and many short documents
        dict(name="attention_7b", kind="attention", rows=2, seq=4096, docs=12, fill=1.0, sigma=1.3, heads=32, kv_heads=32,
             head_dim=128, rotary=True, causal=True, backward=True, mix=3),
        # instruction data: hundreds of short dialogues, rows that end in padding
        dict(name="attention_short_docs", kind="attention", rows=4, seq=2999, docs=48, fill=0.95, sigma=0.7, heads=32,
             kv_heads=8, head_dim=128, rotary=True, causal=True, backward=True, mix=4),
        # long context: one row of 16384 tokens, four documents, grouped heads (one tensor-parallel rank's share)
        dict(name="attention_long", kind="attention", rows=1, seq=16384, docs=4, fill=1.0, sigma=0.8, heads=8, kv_heads=2,
             head_dim=128, rotary=True, causal=True, backward=True, mix=5),
        # scoring a packed batch, forward only; documents end inside tiles
        dict(name="attention_score", kind="attention", rows=3, seq=1365, docs=7, fill=1.0, sigma=1.0, heads=32, kv_heads=8,
             head_dim=128, rotary=True, causal=True, backward=False, mix=6),
        # GPT-2's table on one microbatch, learned positions, gradient added to the fp32 accumulation buffer
        dict(name="embedding_gpt2", kind="embedding", rows=2, seq=1024, docs=6, fill=0.97, sigma=1.0, vocab=50304, dim=768,
             positions=1024, scale=1.0, main_grad=True, pad=0.0, mix=2),
        # the 7B table, scaled embeddings, the gradient in the parameter's own type
        dict(name="embedding_7b", kind="embedding", rows=2, seq=4096, docs=12, fill=1.0, sigma=1.3, vocab=32000, dim=4096,
             positions=0, scale=64.0, main_grad=False, pad=0.0, mix=3),
        # a padded batch: a third of all tokens is one id, which a gradient by tokens has to sum all the same
        dict(name="embedding_padded", kind="embedding", rows=16, seq=2047, docs=9, fill=0.66, sigma=1.0, vocab=32000,
             dim=1024, positions=2048, scale=1.0, main_grad=True, pad=0.34, mix=7),
        # the residual branch of a GPT-2 block on one microbatch
        dict(name="dropout_gpt2", kind="dropout", rows=2048, cols=768, p=0.1, residual=True, stream=3),
        # after an odd-sized classifier layer: a row length that no vector width divides, no residual
        dict(name="dropout_odd", kind="dropout", rows=777, cols=1003, p=0.25, residual=False, stream=0),
        # a wide residual stream
        dict(name="dropout_wide", kind="dropout", rows=8192, cols=4096, p=0.1, residual=True, stream=40),
    ]


def _between(rng, lo, hi):
    """An integer from lo to hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    kind = rng.choice(["attention", "attention", "embedding", "dropout"])
    if kind == "dropout":
        cols = _between(rng, 64, 5120)
        cols = cols if rng.random() < 0.4 else 8 * max(1, cols // 8)
        rows = min(_between(rng, 16, 16384), 33_000_000 // cols)
        return dict(kind=kind, rows=rows, cols=cols, p=round(rng.uniform(0.02, 0.6), 3), residual=rng.random() < 0.6,
                    stream=rng.randint(0, 100))
    rows, seq = rng.randint(1, 4), _between(rng, 64, 16384)
    docs = max(1, min(96, seq // _between(rng, 24, max(25, seq // 2))))
    case = dict(kind=kind, rows=rows, seq=seq, docs=docs, fill=round(rng.choice([1.0, rng.uniform(0.6, 1.0)]), 3),
                sigma=round(rng.uniform(0.2, 1.4), 2), mix=rng.randint(10, 10 ** 6))
    if kind == "embedding":
        vocab = _between(rng, 500, 50304)
        dim = 8 * _between(rng, 16, 640)
        while vocab * dim > 140_000_000:
            dim = 8 * (dim // 16)
        while rows * seq * dim > 34_000_000:
            case["seq"] = seq = seq // 2
        case.update(vocab=vocab, dim=dim, positions=seq if rng.random() < 0.5 else 0, scale=rng.choice([1.0, 1.0, math.sqrt(dim)]),
                    main_grad=rng.random() < 0.5, pad=round(rng.choice([0.0, rng.uniform(0.0, 0.5)]), 3))
        return case
    hd = rng.choice([64, 128, 128])
    heads = _between(rng, 2, 32)
    kv = heads // 4 if heads % 4 == 0 and rng.random() < 0.5 else heads
    causal = rng.random() < 0.85
    case.update(heads=heads, kv_heads=kv, head_dim=hd, rotary=rng.random() < 0.7, causal=causal,
                backward=rng.random() < 0.75)
    while case["rows"] * heads * case["seq"] ** 2 > 2 ** 30:  # the plain form holds every score
        case["seq"] = case["seq"] * 3 // 4
    case["docs"] = min(case["docs"], case["seq"])
    return case


def _lengths(c):
    """Document lengths of every row, shares of a log-normal; their sum is at most the row's length.  Some are one
    token long or empty."""
    rng = random.Random(c["mix"])
    table = [[math.exp(rng.gauss(0.0, c["sigma"])) for _ in range(c["docs"])] for _ in range(c["rows"])]
    return [[int(c["seq"] * c["fill"] * w / sum(row)) for w in row] for row in table]


def _places(lengths, seq, dev):
    """Document number of every token (-1 in none) and its position inside it, [rows, seq] each."""
    ends = lengths.long().cumsum(1)
    t = torch.arange(seq, device=dev).expand(lengths.shape[0], seq).contiguous()
    doc = torch.searchsorted(ends, t, right=True)
    inside = t < ends[:, -1:]
    start = torch.cat([torch.zeros_like(ends[:, :1]), ends], 1).gather(1, doc)
    return torch.where(inside, doc, -1), torch.where(inside, t - start, -1)


def prepare(case, seed):
    c, dev = case, "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    randn = lambda *shape, std=1.0: (torch.randn(*shape, device=dev, generator=gen) * std).to(BF16)  # noqa: E731
    state = dict(case=c)
    if c["kind"] == "dropout":
        state["x"] = randn(c["rows"], c["cols"])
        state["dy"] = randn(c["rows"], c["cols"])
        state["residual"] = randn(c["rows"], c["cols"]) if c["residual"] else None
        state["seed"] = torch.randint(0, 2 ** 62, (1,), device=dev, generator=gen)
        return state
    T = c["rows"] * c["seq"]
    state["lengths"] = torch.tensor(_lengths(c), dtype=torch.int32, device=dev)
    if c["kind"] == "attention":
        D = c["head_dim"]
        state["qkv"] = randn(T, (c["heads"] + 2 * c["kv_heads"]) * D)
        state["do"] = randn(T, c["heads"] * D)
        state["cos"] = state["sin"] = None
        if c["rotary"]:
            ang = _angles(torch.arange(c["seq"], device=dev), D)
            state["cos"], state["sin"] = ang.cos().float(), ang.sin().float()
        return state
    # token ids as text has them: a few very frequent, most rare
    u = torch.rand(T, device=dev, generator=gen)
    ids = ((c["vocab"] ** u.double()).long() - 1).clamp_(0, c["vocab"] - 1)
    ids = (ids * 7919) % c["vocab"]  # frequent ids all over the table
    if c["pad"]:
        ids = torch.where(torch.rand(T, device=dev, generator=gen) < c["pad"], 0, ids)
    state["ids"] = ids.view(c["rows"], c["seq"])
    state["wte"] = torch.nn.Parameter(randn(c["vocab"], c["dim"], std=0.02))
    state["wpe"] = torch.nn.Parameter(randn(c["positions"], c["dim"], std=0.02)) if c["positions"] else None
    state["tables"] = [t for t in (state["wte"], state["wpe"]) if t is not None]
    if c["main_grad"]:
        for t in state["tables"]:
            t.main_grad = torch.zeros(t.shape, device=dev)
    state["dout"] = randn(T, c["dim"])
    return state


def _angles(positions, D, theta=10000.0):
    inv = theta ** (-torch.arange(0, D, 2, dtype=torch.float64, device=positions.device) / D)
    return torch.outer(positions.double(), inv)


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"attention": _attention_own, "embedding": _embedding_own, "dropout": _dropout_own}[kind](state)
    return {"attention": _attention_plain, "embedding": _embedding_plain, "dropout": _dropout_plain}[kind](state)


# ------------------------------------------------------------------------------------------------
# the framework's calls
# ------------------------------------------------------------------------------------------------
def _attention_own(s):
    from pippy_b200.ops import functional as pf

    c = s["case"]
    layout = pf.packed_layout(s["lengths"], c["seq"])
    args = (s["cos"], s["sin"], layout, c["heads"], c["kv_heads"], c["head_dim"])
    if not c["backward"]:
        with torch.no_grad():
            return dict(o=pf.packed_attention(s["qkv"], *args, causal=c["causal"]), positions=layout.positions)
    qkv = s["qkv"].detach().requires_grad_(True)
    o = pf.packed_attention(qkv, *args, causal=c["causal"])
    (dqkv,) = torch.autograd.grad(o, qkv, s["do"])
    return dict(o=o.detach(), dqkv=dqkv, positions=layout.positions)


def _embedding_own(s):
    from pippy_b200.ops import functional as pf

    c = s["case"]
    positions = pf.packed_layout(s["lengths"], c["seq"]).positions if c["positions"] else None
    for t in s["tables"]:
        if c["main_grad"]:
            t.main_grad.zero_()
        else:
            t.grad = None
    out = pf.embedding(s["ids"], s["wte"], s["wpe"], c["seq"], scale=c["scale"], positions=positions, sorted_grad=True)
    out.backward(s["dout"])
    return dict(out=out.detach(), grads=[t.main_grad if c["main_grad"] else t.grad for t in s["tables"]])


def _dropout_own(s):
    from pippy_b200.ops import functional as pf

    c = s["case"]
    x = s["x"].detach().requires_grad_(True)
    y = pf.dropout(x, c["p"], s["seed"], residual=s["residual"], stream=c["stream"])
    (dx,) = torch.autograd.grad(y, x, s["dy"])
    return dict(y=y.detach(), dx=dx)


# ------------------------------------------------------------------------------------------------
# plain form
# ------------------------------------------------------------------------------------------------
def _heads(x, rows, seq, heads):  # [rows * seq, heads * D] -> [rows, heads, seq, D]
    return x.view(rows, seq, heads, -1).transpose(1, 2)


def _rotate(x, cos, sin, sign):  # [rows, heads, seq, D] by [rows, 1, seq, D / 2]
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * cos - sign * b * sin, b * cos + sign * a * sin], dim=-1)


def _attention_plain(s):
    c = s["case"]
    rows, seq, hq, hk, D = c["rows"], c["seq"], c["heads"], c["kv_heads"], c["head_dim"]
    scale, G = 1.0 / math.sqrt(D), hq // hk
    doc, pos = _places(s["lengths"], seq, "cuda")
    q, k, v = (_heads(t, rows, seq, t.shape[1] // D) for t in s["qkv"].float().split([hq * D, hk * D, hk * D], dim=1))
    if c["rotary"]:
        cos, sin = (s[n][pos.clamp(min=0)].unsqueeze(1) for n in ("cos", "sin"))
        q, k = _rotate(q, cos, sin, 1.0), _rotate(k, cos, sin, 1.0)
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    seen = (doc.unsqueeze(2) == doc.unsqueeze(1)) & (doc >= 0).unsqueeze(2)
    if c["causal"]:
        seen = seen & (pos.unsqueeze(2) >= pos.unsqueeze(1))
    hidden = ~seen.unsqueeze(1)
    p = (q @ k.transpose(2, 3)).mul_(scale).masked_fill_(hidden, float("-inf"))
    p = p.sub_(p.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny))
    o = p @ v
    back = lambda x: x.transpose(1, 2).reshape(rows * seq, -1)  # noqa: E731
    out = dict(o=back(o).to(BF16), positions=pos.reshape(-1).int())
    if not c["backward"]:
        return out
    do = _heads(s["do"].float(), rows, seq, hq)
    dv = p.transpose(2, 3) @ do
    ds = (do @ v.transpose(2, 3)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq, dk = ds @ k, ds.transpose(2, 3) @ q
    dk, dv = (t.view(rows, hk, G, seq, D).sum(2) for t in (dk, dv))
    if c["rotary"]:
        dq, dk = _rotate(dq, cos, sin, -1.0), _rotate(dk, cos, sin, -1.0)
    out["dqkv"] = torch.cat([back(t) for t in (dq, dk, dv)], dim=1).to(BF16)
    return out


def _embedding_plain(s):
    c = s["case"]
    ids = s["ids"].reshape(-1)
    out, dout = s["wte"].detach()[ids].float() * c["scale"], s["dout"].float()
    grads = [torch.zeros(s["wte"].shape, device=ids.device).index_add_(0, ids, dout * c["scale"])]
    if c["positions"]:
        pos = _places(s["lengths"], c["seq"], ids.device)[1].reshape(-1)
        inside = (pos >= 0).unsqueeze(1)
        out = out + torch.where(inside, s["wpe"].detach()[pos.clamp(min=0)].float(), 0.0)
        grads.append(torch.zeros(s["wpe"].shape, device=ids.device).index_add_(
            0, pos.clamp(min=0), torch.where(inside, dout, 0.0)))
    return dict(out=out.to(BF16), grads=grads if c["main_grad"] else [g.to(BF16) for g in grads])


def _keep(seed, stream, count, p):
    """Which of ``count`` elements stay: Philox4x32-10 (Salmon et al., SC 2011) with the 64-bit seed as key and the counter
    (element // 8, stream); eight 16-bit numbers a block, low halves first, an element stays if its number is at
    least round(65536 p)."""
    mask = 0xFFFFFFFF
    block = torch.arange((count + 7) // 8, device=seed.device)
    k0, k1 = seed & mask, (seed >> 32) & mask
    x0, x1 = block & mask, block >> 32
    x2, x3 = torch.full_like(block, stream & mask), torch.full_like(block, stream >> 32)
    for _ in range(10):
        # the product wraps modulo 2^64; its upper half is what the shift leaves in the low 32 bits
        a, b = x0 * 0xD2511F53, x2 * 0xCD9E8D57
        x0, x1, x2, x3 = ((b >> 32) & mask) ^ x1 ^ k0, b & mask, ((a >> 32) & mask) ^ x3 ^ k1, a & mask
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    words = torch.stack([x0, x1, x2, x3], dim=1)
    numbers = torch.stack([words & 0xFFFF, words >> 16], dim=2).reshape(-1)[:count]
    return numbers >= _threshold(p)


def _threshold(p):
    return int(math.floor(p * 65536 + 0.5))


def _dropout_plain(s):
    c = s["case"]
    keep = _keep(s["seed"], c["stream"], s["x"].numel(), c["p"]).view(s["x"].shape)
    factor = 65536.0 / (65536 - _threshold(c["p"]))
    y = torch.where(keep, s["x"].float() * factor, 0.0)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return dict(y=y.to(BF16), dx=torch.where(keep, s["dy"].float() * factor, 0.0).to(BF16))


# ------------------------------------------------------------------------------------------------
# the work that no implementation can do without
# ------------------------------------------------------------------------------------------------
def work(case):
    """Bytes: every input read once, every output written once.  Operations of attention: the products over the pairs of
    tokens that see each other, two forward and five backward.  Of the others, additions and products of elements."""
    c = case
    if c["kind"] == "dropout":
        n = c["rows"] * c["cols"]
        return dict(bytes=n * (10 if c["residual"] else 8), flops=n * (4 if c["residual"] else 3))
    T = c["rows"] * c["seq"]
    if c["kind"] == "attention":
        pairs = sum(n * (n + 1) // 2 if c["causal"] else n * n for row in _lengths(c) for n in row)
        q, qkv = c["heads"] * c["head_dim"], (c["heads"] + 2 * c["kv_heads"]) * c["head_dim"]
        if not c["backward"]:
            return dict(bytes=2 * T * (qkv + q) + 4 * T, flops=4 * pairs * q)
        return dict(bytes=2 * T * (2 * qkv + 2 * q) + 4 * T, flops=14 * pairs * q)
    tables = c["vocab"] + c["positions"]
    read = min(T, c["vocab"]) + min(c["seq"], c["positions"])
    return dict(bytes=T * (4 * c["dim"] + 8) + 2 * read * c["dim"] + tables * c["dim"] * (4 if c["main_grad"] else 2),
                flops=2 * T * c["dim"] * (2 if c["positions"] else 1))


# ------------------------------------------------------------------------------------------------
# the same results in 64 bits, from the definitions
# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["kind"] == "attention":
        return _attention_exact(c, s)
    if c["kind"] == "embedding":
        return _embedding_exact(c, s)
    keep = torch.tensor(_keep_exact(int(s["seed"].item()), c["stream"], c["rows"] * c["cols"], c["p"]), device="cuda")
    # the probability that the operator works with is a multiple of 2^-16
    factor = keep.view(c["rows"], c["cols"]).double() / (1.0 - math.floor(c["p"] * 65536 + 0.5) / 65536)
    y = s["x"].double() * factor
    return dict(y=y if s["residual"] is None else s["residual"].double() + y, dx=s["dy"].double() * factor)


def _attention_exact(c, s):
    """Document by document and head by head, each with its own tokens alone; the backward by automatic differentiation."""
    D, hq, hk, seq = c["head_dim"], c["heads"], c["kv_heads"], c["seq"]
    if work(case=c)["flops"] > 6e12:
        return None
    o = torch.zeros(c["rows"] * seq, hq * D, dtype=torch.float64, device="cuda")
    dqkv = torch.zeros(s["qkv"].shape, dtype=torch.float64, device="cuda")
    positions = torch.full((c["rows"] * seq,), -1, dtype=torch.int32, device="cuda")
    for row, lengths in enumerate(_lengths(c)):
        at = row * seq
        for n in lengths:
            here = slice(at, at + n)
            at += n
            if n == 0:
                continue
            positions[here] = torch.arange(n, device="cuda", dtype=torch.int32)
            future = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)
            turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), _angles(torch.arange(n, device="cuda"), D)) \
                if c["rotary"] else None
            for g in range(hk):
                per = hq // hk
                cols = [slice((g * per + j) * D, (g * per + j + 1) * D) for j in range(per)]
                kc, vc = slice((hq + g) * D, (hq + g + 1) * D), slice((hq + hk + g) * D, (hq + hk + g + 1) * D)
                k, v = (s["qkv"][here, x].double().requires_grad_(c["backward"]) for x in (kc, vc))
                for x in cols:
                    q = s["qkv"][here, x].double().requires_grad_(c["backward"])
                    scores = (_turned(q, turn) @ _turned(k, turn).T) / math.sqrt(D)
                    if c["causal"]:
                        scores = scores.masked_fill(future, float("-inf"))
                    y = torch.softmax(scores, dim=-1) @ v
                    o[here, x] = y.detach()
                    if c["backward"]:
                        dq, dk, dv = torch.autograd.grad(y, (q, k, v), s["do"][here, x].double())
                        dqkv[here, x] = dq
                        dqkv[here, kc] += dk
                        dqkv[here, vc] += dv
                    del scores, y
    return dict(o=o, positions=positions, dqkv=dqkv) if c["backward"] else dict(o=o, positions=positions)


def _turned(x, turn):
    """Pairs (i, i + D/2) as complex numbers, turned by the position's angle."""
    if turn is None:
        return x
    z = torch.complex(x[:, : x.shape[1] // 2], x[:, x.shape[1] // 2:]) * turn
    return torch.cat([z.real, z.imag], dim=1)


def _embedding_exact(c, s):
    """The gradients as sums over runs of equal keys: differences of a running sum over the sorted rows."""
    ids = s["ids"].reshape(-1)
    pos = torch.cat([torch.cat([torch.arange(n) for n in row] + [torch.full((c["seq"] - sum(row),), -1)])
                     for row in _lengths(c)]).to(ids.device)
    out, dout = c["scale"] * s["wte"].detach().double()[ids], s["dout"].double()
    if c["positions"]:
        table = torch.cat([s["wpe"].detach().double(), torch.zeros(1, c["dim"], dtype=torch.float64, device=ids.device)])
        out = out + table[pos]  # position -1 is the row of zeros at the end

    def by_key(keys, rows, size):
        order = keys.argsort(stable=True)
        running = torch.cat([torch.zeros_like(rows[:1]), rows[order].cumsum(0)])
        edges = torch.searchsorted(keys[order].contiguous(), torch.arange(size + 1, device=keys.device))
        return running[edges[1:]] - running[edges[:-1]]

    grads = [by_key(ids, c["scale"] * dout, c["vocab"])]
    if c["positions"]:
        grads.append(by_key(pos, dout, c["positions"]))
    return dict(out=out, grads=grads)


def _keep_exact(seed, stream, count, p):
    """The generator in numpy's unsigned 64-bit arithmetic."""
    import numpy as np

    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    block = np.arange((count + 7) // 8, dtype=np.uint64)
    x = [block & low, block >> half, np.full_like(block, stream % 2 ** 32), np.full_like(block, stream // 2 ** 32)]
    for r in range(10):
        key = [np.uint64((seed % 2 ** 32 + r * 0x9E3779B9) % 2 ** 32), np.uint64((seed // 2 ** 32 + r * 0xBB67AE85) % 2 ** 32)]
        a, b = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(b >> half) ^ x[1] ^ key[0], b & low, (a >> half) ^ x[3] ^ key[1], a & low]
    numbers = np.stack(x, axis=1).astype("<u4").view("<u2").reshape(-1)[:count]
    return numbers.astype(np.int64) >= math.floor(p * 65536 + 0.5)
