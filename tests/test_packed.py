"""Attention over packed documents: the layout, the plain form and the kernels against the definition in 64 bits."""
import math

import pytest
import torch

from pippy_b200.ops import _lib
from pippy_b200.ops import functional as pf

gpu = pytest.mark.gpu
U = 2.0 ** -8  # a bf16 rounding is off by at most this much of the value
SLACK = 2.0 ** -14  # fp32 sums, ex2 and log2 of the kernels, relative to sums of absolute values


@pytest.fixture
def errors():
    yield
    _lib.check_device_errors()


def _positions(lengths, S):
    out = []
    for row in lengths:
        line = [t for n in row for t in range(n)]
        out += line + [-1] * (S - len(line))
    return torch.tensor(out, dtype=torch.int32)


def _turn(x, c, s, sign=1.0):
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - sign * b * s, b * c + sign * a * s], -1)


def _definition(qkv, do, lengths, S, hq, hk, D, cos=None, sin=None, scale=None, causal=True):
    """(o, bound of its error), (dqkv, bound) in 64 bits, document by document.  The bounds follow the roundings to bf16, each
    at most U of the value: rotated q and k (scores off by e_s = 2 U scale sum |q||k|, probabilities by e_s of
    themselves), P, dS, the stored o (through delta) and the result; SLACK of the sums of absolute values for the rest."""
    scale = 1 / math.sqrt(D) if scale is None else scale
    dev = qkv.device
    x, g = qkv.double(), do.double()
    o, bo = torch.zeros(len(qkv), hq * D, dtype=torch.float64, device=dev), torch.zeros(len(qkv), hq * D, dtype=torch.float64, device=dev)
    d, bd = torch.zeros_like(x), torch.zeros_like(x)
    for r, row in enumerate(lengths):
        at = r * S
        for n in row:
            w = slice(at, at + n)
            at += n
            if n == 0:
                continue
            hidden = torch.ones(n, n, dtype=torch.bool, device=dev).triu(1) if causal else torch.zeros(n, n, dtype=torch.bool, device=dev)
            for h in range(hq):
                kv = h // (hq // hk)
                cq, ck, cv = (slice(i * D, (i + 1) * D) for i in (h, hq + kv, hq + hk + kv))
                q, k, v, gr = x[w, cq], x[w, ck], x[w, cv], g[w, cq]
                if cos is not None:
                    c, s = cos[:n].double(), sin[:n].double()
                    q, k = _turn(q, c, s), _turn(k, c, s)
                p = (q @ k.T * scale).masked_fill(hidden, -math.inf).softmax(-1)
                e_s = ((2 * U + U * U if cos is not None else 0.0) + SLACK) * scale * (q.abs() @ k.abs().T)
                e_s = torch.expm1(2 * e_s.masked_fill(hidden, 0.0).amax(1, keepdim=True))  # numerator and sum
                y = p @ v
                by = (U + e_s + SLACK) * (p @ v.abs())
                by = by + U * (y.abs() + by)
                o[w, cq], bo[w, cq] = y, by
                dp, delta = gr @ v.T, (gr * y).sum(1, keepdim=True)
                b_delta = (gr.abs() * by).sum(1, keepdim=True) + SLACK * (gr * y).abs().sum(1, keepdim=True)
                ds = p * (dp - delta)
                b_ds = p * ((1 + e_s) * (b_delta + SLACK * (gr.abs() @ v.abs().T)) + e_s * (dp - delta).abs())
                b_ds = b_ds + U * (ds.abs() + b_ds)
                b_p = (U + e_s + SLACK) * p
                parts = [(cq, scale * ds @ k, scale * (b_ds @ k.abs() * (1 + U) + (U + SLACK) * (ds.abs() @ k.abs())), True),
                         (ck, scale * ds.T @ q, scale * (b_ds.T @ q.abs() * (1 + U) + (U + SLACK) * (ds.abs().T @ q.abs())), True),
                         (cv, p.T @ gr, b_p.T @ gr.abs() + SLACK * (p.T @ gr.abs()), False)]
                for cols, value, bound, rotated in parts:
                    if rotated and cos is not None:
                        value = _turn(value, c, s, -1.0)
                        lo, hi = bound.chunk(2, -1)
                        bound = torch.cat([lo * c.abs() + hi * s.abs(), hi * c.abs() + lo * s.abs()], -1)
                    d[w, cols] += value
                    bd[w, cols] += bound
    return (o, bo), (d, bd + U * (d.abs() + bd))


def _inputs(lengths, S, hq, hk, D, rotary, device, seed=0, dtype=torch.bfloat16):
    gen = torch.Generator().manual_seed(seed)
    T = len(lengths) * S
    qkv = torch.randn(T, (hq + 2 * hk) * D, generator=gen).to(dtype).to(device)
    do = torch.randn(T, hq * D, generator=gen).to(dtype).to(device)
    cos = sin = None
    if rotary:
        cos, sin = (t.to(device) for t in pf.rope_tables(max(1, max(max(row, default=1) for row in lengths)), D, 10000.0, "cpu"))
    return qkv, do, cos, sin


def _layout(lengths, S, device):
    return pf.packed_layout(torch.tensor(lengths, dtype=torch.int32, device=device), S)


def _run(qkv, do, cos, sin, layout, hq, hk, D, **kw):
    leaf = qkv.detach().requires_grad_(True)
    o = pf.packed_attention(leaf, cos, sin, layout, hq, hk, D, **kw)
    (grad,) = torch.autograd.grad(o, leaf, do)
    return o.detach(), grad


# ------------------------------------------------------------------------------------------------ CPU
def test_layout_positions():
    lengths, S = [[3, 0, 2], [0, 7, 0], [0, 0, 0]], 7
    layout = _layout(lengths, S, "cpu")
    assert torch.equal(layout.positions, _positions(lengths, S)) and layout.total == 21
    one = pf.packed_layout(torch.tensor([2, 4]), 9)
    assert torch.equal(one.positions, _positions([[2, 4]], 9))
    assert torch.equal(pf.packed_layout(torch.zeros(2, 0, dtype=torch.int64), 3).positions, torch.full((6,), -1, dtype=torch.int32))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("rotary", [True, False])
def test_plain_form(causal, rotary):
    lengths, S, hq, hk, D = [[5, 0, 1, 9], [16, 0, 0, 0], [2, 3, 4, 0]], 16, 4, 2, 16
    qkv, do, cos, sin = _inputs(lengths, S, hq, hk, D, rotary, "cpu", dtype=torch.float64)
    inside = _positions(lengths, S) >= 0
    qkv[~inside], do[~inside] = math.nan, math.inf
    got = _run(qkv, do, cos, sin, _layout(lengths, S, "cpu"), hq, hk, D, causal=causal)
    want = _definition(qkv, do, lengths, S, hq, hk, D, cos, sin, causal=causal)
    for a, (b, _) in zip(got, want):
        assert (a - b).abs().max() < 1e-12 * S * D
        assert not a[~inside].any()


def test_plain_form_gradient_by_differences():
    lengths, S, hq, hk, D = [[3, 1]], 5, 2, 1, 8
    qkv, _, cos, sin = _inputs(lengths, S, hq, hk, D, True, "cpu", dtype=torch.float64)
    layout = _layout(lengths, S, "cpu")
    assert torch.autograd.gradcheck(lambda x: pf.packed_attention(x, cos, sin, layout, hq, hk, D), qkv.requires_grad_(True))


def test_refusals():
    layout = _layout([[3, 4]], 8, "cpu")
    qkv = torch.zeros(8, 4 * 16)
    cos, sin = pf.rope_tables(8, 16, 1e4, "cpu")
    pf.packed_attention(qkv, cos, sin, layout, 2, 1, 16)
    for bad in (dict(Hq=3), dict(D=32), dict(Hq=0), dict(scale=0.0), dict(scale=math.nan), dict(scale=-1.0), dict(sin=None),
                dict(cos=cos[:, :4]), dict(cos=cos.half()), dict(qkv=qkv[:7]), dict(cos=cos[:3], sin=sin[:3]),
                dict(cos=cos[:7])):
        kw = dict(qkv=qkv, cos=cos, sin=sin, layout=layout, Hq=2, Hkv=1, D=16)
        kw.update(bad)
        with pytest.raises(ValueError):
            pf.packed_attention(**kw)
    for lengths, S in (([[9]], 8), ([[-1, 2]], 8), ([[4, 5]], 8), ([[1.0]], 8), ([[True]], 8), ([[[1]]], 8), ([[1]], 0)):
        with pytest.raises(ValueError):
            pf.packed_layout(torch.tensor(lengths), S)
    with pytest.raises(ValueError):
        pf.packed_layout(torch.zeros(0, 3, dtype=torch.int32), 4)


@pytest.mark.skipif(not _lib.available(), reason="the CUDA library is not built")
def test_entry_points_refuse_before_they_launch():
    """Arguments that no launch could take come back as a negative code; nothing here has a GPU to launch on."""
    lib, at = _lib.lib(), 1 << 20  # an address that is only looked at

    def forward(T=256, Hq=4, Hkv=2, D=64, pitch=512, o=at, tiles=3):
        return lib.pb_packed_attention_fwd(at, at, at, o, at, at, 1, at, at, tiles, T, Hq, Hkv, D, pitch, pitch, pitch, 256, 0.1, 1, at, None)

    assert forward(D=32) == forward(D=96) == -1
    assert forward(Hkv=3) == forward(Hq=0) == forward(Hkv=0) == -2
    assert forward(pitch=513) == forward(o=at + 8) == -3
    assert forward(T=0) == forward(T=2 ** 31) == forward(tiles=0) == forward(tiles=2 ** 30) == -4

    def backward(T=256, Hq=4, Hkv=2, D=64, pitch=512, dq=at, tiles=3):
        return lib.pb_packed_attention_bwd(at, at, at, at, at, at, at, dq, at, at, None, None, 0, at, at, tiles, at, T, Hq, Hkv, D,
                                           pitch, pitch, pitch, 256, 256, 512, 0.1, 1, at, None)

    assert backward(D=256) == -1 and backward(Hkv=3) == -2 and backward(pitch=4) == backward(dq=at + 2) == -3
    assert backward(T=0) == backward(tiles=0) == -4
    assert lib.pb_packed_layout(at, 0, 1, 1, at, at, at, 1, at, 1, at, at, None) == -1
    assert lib.pb_packed_layout(at, 2 ** 16, 1, 2 ** 16, at, at, at, 1, at, 1, at, at, None) == -2
    assert lib.pb_packed_rope(at, 64, at, 64, at, at, at, 1, 1, 24, 1, None, at, None) == -1
    assert lib.pb_packed_rope(at, 64, at + 8, 64, at, at, at, 1, 1, 64, 1, None, at, None) == -2
    # the split of a key head's query heads: none where there are items enough, all of them where there are few
    plain, split = (lib.pb_packed_attention_bwd_scratch(4096, 32, 4, 128, tiles) for tiles in (2000, 4))
    assert plain == 16 + 4096 * 32 * 4 and split == plain + 8 * 2 * 4096 * 4 * 128 * 4


# ------------------------------------------------------------------------------------------------ GPU
def _read_tiles(layout, rows):
    tiles, counts = layout.tiles(rows)
    return tiles[: int(counts[0])].tolist()


@gpu
@pytest.mark.parametrize("case", ["mixed", "ones", "long", "empty", "many", "no_documents"])
def test_layout_kernel(case, errors):
    gen = torch.Generator().manual_seed(1)
    lengths, S = {
        "mixed": ([[3, 0, 2000, 129], [0, 0, 2500, 0], [128, 256, 255, 1]], 2500),
        "ones": ([[1] * 100], 100),
        "long": ([[300_001, 5]], 300_100),
        "empty": ([[0, 0], [0, 0]], 77),
        "many": (torch.randint(0, 9, (3, 3001), generator=gen).tolist(), 24_008),
        "no_documents": ([[], []], 5),
    }[case]
    layout = _layout(lengths, S, "cuda")
    assert torch.equal(layout.positions.cpu(), _positions(lengths, S))
    for rows in (128, 256):
        want = set()
        for r, row in enumerate(lengths):
            at = r * S
            for i, n in enumerate(row + [S - sum(row)]):
                want |= {(at, n, t, int(i == len(row))) for t in range(-(-n // rows))}
                at += n
        got = _read_tiles(layout, rows)
        assert len(got) == len(want) <= len(layout.tiles(rows)[0]) and {tuple(t) for t in got} == want
        ranks = [t[2] if not t[3] else -1 for t in got]  # longest first, as far as there are buckets; padding last
        assert all(a >= b or min(a, b) >= 2047 for a, b in zip(ranks, ranks[1:]) if b >= 0) and sorted(ranks, key=lambda t: t == -1) == ranks
        half = [t[1] <= 128 and not t[3] for t in got]  # the last ones before the padding
        n_first, n_docs = layout.tiles(rows)[1][1:3].tolist()
        assert n_docs == sum(1 for t in got if not t[3]) and half == [n_first <= i < n_docs for i in range(len(got))]


@gpu
@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int64])
def test_layout_kernel_takes_every_integer_type(dtype, errors):
    lengths = [[100, 0, 7], [120, 3, 1]]
    layout = pf.packed_layout(torch.tensor(lengths, dtype=dtype, device="cuda"), 130)
    assert torch.equal(layout.positions.cpu(), _positions(lengths, 130))


@gpu
@pytest.mark.parametrize("lengths", [[[5, -1, 4]], [[5, 9, 3]], [[2 ** 31 - 1, 2 ** 31 - 1, 3]], [[2 ** 40, 1, 1]]])
def test_layout_kernel_cuts_bad_lengths(lengths):
    """Nothing reaches beyond its row: the tiles and positions are those of the lengths cut to what fits, and the host hears of it."""
    S, cut, left = 12, [], 12
    for n in lengths[0]:
        cut.append(min(max(n, 0), left))
        left -= cut[-1]
    layout = pf.packed_layout(torch.tensor(lengths, device="cuda"), S)
    with pytest.raises(_lib.KernelError, match="code 6"):
        _lib.check_device_errors()
    assert torch.equal(layout.positions.cpu(), _positions([cut], S))
    assert sum(min(t[1], 128) for t in _read_tiles(layout, 128)) == S


SHAPES = [  # lengths, tokens per row
    ([[1]], 1),
    ([[1, 1, 1]], 5),
    ([[127, 1, 128]], 256),
    ([[129, 0, 256, 5], [64, 63, 250, 13]], 390),
    ([[257], [0], [300]], 300),
    ([[511, 640]], 1200),
]


@gpu
@pytest.mark.parametrize("lengths,S", SHAPES)
@pytest.mark.parametrize("heads", [(1, 1), (4, 2), (6, 1)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal,rotary", [(True, True), (True, False), (False, True)])
def test_attention_kernel(lengths, S, heads, D, causal, rotary, errors):
    hq, hk = heads
    qkv, do, cos, sin = _inputs(lengths, S, hq, hk, D, rotary, "cuda")
    layout = _layout(lengths, S, "cuda")
    got = _run(qkv, do, cos, sin, layout, hq, hk, D, causal=causal)
    want = _definition(qkv, do, lengths, S, hq, hk, D, cos, sin, causal=causal)
    for a, (b, bound) in zip(got, want):
        assert torch.isfinite(a).all() and ((a.double() - b).abs() <= bound).all()
    again = _run(qkv, do, cos, sin, layout, hq, hk, D, causal=causal)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@gpu
@pytest.mark.parametrize("heads", [(16, 16), (12, 4), (15, 5)])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_kernel_many_items(heads, D, errors):
    """Every resident block walks a dozen work items: documents of one block, of two and three, padding between them."""
    gen = torch.Generator().manual_seed(7)
    lengths = [torch.randint(0, 120, (30,), generator=gen).tolist() for _ in range(4)]
    lengths[1][3:6], lengths[2][0] = [128, 129, 400], 256
    S = max(sum(row) for row in lengths) + 17
    hq, hk = heads
    qkv, do, cos, sin = _inputs(lengths, S, hq, hk, D, True, "cuda")
    layout = _layout(lengths, S, "cuda")
    got = _run(qkv, do, cos, sin, layout, hq, hk, D)
    want = _definition(qkv, do, lengths, S, hq, hk, D, cos, sin)
    for a, (b, bound) in zip(got, want):
        assert torch.isfinite(a).all() and ((a.double() - b).abs() <= bound).all()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(got, _run(qkv, do, cos, sin, layout, hq, hk, D)))


@gpu
def test_attention_kernel_on_few_sms(errors):
    """The grid leaves the reserved SMs out; each of the few blocks walks hundreds of items, to the same bits."""
    from pippy_b200.ops.gemm import set_sm_reserve

    lengths, S, hq, hk, D = [[30, 200, 70, 300], [5, 0, 128, 129]], 640, 16, 4, 128
    qkv, do, cos, sin = _inputs(lengths, S, hq, hk, D, True, "cuda")
    layout = _layout(lengths, S, "cuda")
    want = _run(qkv, do, cos, sin, layout, hq, hk, D)
    try:
        for reserve in (145, 10_000):
            set_sm_reserve(reserve)
            assert all(torch.equal(a, b) for a, b in zip(want, _run(qkv, do, cos, sin, layout, hq, hk, D)))
    finally:
        set_sm_reserve(0)


@gpu
@pytest.mark.parametrize("causal", [True, False])
def test_attention_kernel_long_and_sharp(causal, errors):
    """Many blocks, growing maxima (the running maximum is moved), scores that saturate."""
    lengths, S, hq, hk, D = [[2500, 700], [3000, 1]], 3210, 2, 1, 128
    qkv, do, cos, sin = _inputs(lengths, S, hq, hk, D, False, "cuda")
    grow = torch.linspace(0.1, 6.0, S, device="cuda").repeat(2).unsqueeze(1)
    qkv[:, hq * D : (hq + hk) * D] = (qkv[:, hq * D : (hq + hk) * D].float() * grow).bfloat16()
    got = _run(qkv, do, cos, sin, _layout(lengths, S, "cuda"), hq, hk, D, causal=causal, scale=0.3)
    want = _definition(qkv, do, lengths, S, hq, hk, D, scale=0.3, causal=causal)
    for a, (b, bound) in zip(got, want):
        assert torch.isfinite(a).all() and ((a.double() - b).abs() <= bound).all()


@gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("value", [math.nan, math.inf, torch.finfo(torch.bfloat16).min])
def test_attention_kernel_keeps_documents_apart(D, value, errors):
    """What padding and other documents hold does not change a bit of a document's results."""
    lengths, S, hq, hk = [[100, 130, 3, 200], [1, 260, 0, 31]], 450, 2, 1
    qkv, do, cos, sin = _inputs(lengths, S, hq, hk, D, True, "cuda")
    layout = _layout(lengths, S, "cuda")
    clean = _run(qkv, do, cos, sin, layout, hq, hk, D)
    bad = (_positions(lengths, S) < 0).cuda()
    bad[100:230] = True  # a document between two others
    bad[451:711] = True  # and one right behind a document of one token
    dirty = qkv.clone(), do.clone()
    for t in dirty:
        t[bad] = value
    got = _run(*dirty, cos, sin, layout, hq, hk, D)
    for a, b in zip(got, clean):
        assert torch.equal(a[~bad], b[~bad])
    padding = (layout.positions < 0)
    assert padding.any() and not any(t[padding].any() for t in got)


@gpu
def test_attention_kernel_strides_and_inplace(errors):
    lengths, S, hq, hk, D = [[70, 200]], 300, 4, 2, 64
    qkv, do, cos, sin = _inputs(lengths, S, hq, hk, D, True, "cuda")
    layout = _layout(lengths, S, "cuda")
    want = _run(qkv, do, cos, sin, layout, hq, hk, D)
    wide = torch.randn(S, qkv.shape[1] + 24, device="cuda").bfloat16()
    for first in (8, 3):  # rows that start on a 16-byte boundary, and rows that do not
        wide[:, first : first + qkv.shape[1]] = qkv
        view = wide[:, first : first + qkv.shape[1]]
        o, grad = _run(view, do, cos, sin, layout, hq, hk, D)
        assert torch.equal(o, want[0]) and torch.equal(grad, want[1]) and torch.equal(view, qkv)
    back = torch.randn(S, hq * D + 4, device="cuda").bfloat16()[:, 4:]
    back.copy_(do)
    assert torch.equal(_run(qkv, back, cos, sin, layout, hq, hk, D)[1], want[1])
    mine = qkv.clone().requires_grad_(True)
    rotated = mine * 1.0
    version = rotated._version
    o = pf.packed_attention(rotated, cos, sin, layout, hq, hk, D, inplace=True)
    assert rotated._version > version and torch.equal(o, want[0])
    (grad,) = torch.autograd.grad(o, mine, do)
    assert torch.equal(grad, want[1])
    assert torch.equal(rotated[:, (hq + hk) * D :], qkv[:, (hq + hk) * D :]) and not torch.equal(rotated, qkv)
    with pytest.raises(ValueError):
        pf.packed_attention(wide[:, 3 : 3 + qkv.shape[1]], cos, sin, layout, hq, hk, D, inplace=True)
    with pytest.raises(ValueError):
        pf.packed_attention(torch.zeros(S, 8 * 32, device="cuda").bfloat16(), None, None, layout, 4, 2, 32)
    with pytest.raises(ValueError):
        pf.packed_attention(qkv, cos, sin, _layout(lengths, S, "cpu"), hq, hk, D)


@gpu
def test_attention_kernel_one_row_of_odd_pitch(errors):
    """A dimension of one row may have any stride."""
    hq, hk, D = 2, 1, 64
    qkv, do, cos, sin = _inputs([[1]], 1, hq, hk, D, True, "cuda")
    want = _run(qkv, do, cos, sin, _layout([[1]], 1, "cuda"), hq, hk, D)
    odd = qkv.clone().as_strided(qkv.shape, (5, 1))
    got = _run(odd, do, cos, sin, _layout([[1]], 1, "cuda"), hq, hk, D)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_attention_kernel_short_tables_are_reported():
    lengths, S, hq, hk, D = [[70, 20]], 100, 1, 1, 64
    qkv, do, cos, sin = _inputs(lengths, S, hq, hk, D, True, "cuda")
    _run(qkv, do, cos[:64].contiguous(), sin[:64].contiguous(), _layout(lengths, S, "cuda"), hq, hk, D)
    with pytest.raises(_lib.KernelError, match="code 5"):
        _lib.check_device_errors()


@gpu
def test_attention_kernel_streams_and_graph(errors):
    """Two calls at once on two streams, and a captured forward and backward replayed with other lengths and inputs."""
    S, hq, hk, D = 600, 4, 1, 128
    mixes = [[[600, 0, 0], [100, 200, 250]], [[1, 400, 199], [0, 300, 300]]]
    cases = []
    for i, lengths in enumerate(mixes):
        qkv, do, cos, sin = _inputs([[S]], S * 2, hq, hk, D, True, "cuda", seed=i)
        cases.append((torch.tensor(lengths, dtype=torch.int32, device="cuda"), qkv, do, cos, sin))
    want = [_run(q, g, c, s, pf.packed_layout(n, S), hq, hk, D) for n, q, g, c, s in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], [[], []]
    for _ in range(3):
        for i, (n, q, g, c, s) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].append(_run(q, g, c, s, pf.packed_layout(n, S), hq, hk, D))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in range(2) for run in got[i] for a, b in zip(run, want[i]))
    n, q, g, c, s = (t.clone() for t in cases[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _run(q, g, c, s, pf.packed_layout(n, S), hq, hk, D)
    for i in (1, 0, 1):
        n.copy_(cases[i][0]), q.copy_(cases[i][1]), g.copy_(cases[i][2])
        graph.replay()
        eager = _run(*cases[1 - i][1:], pf.packed_layout(cases[1 - i][0], S), hq, hk, D)
        assert all(torch.equal(a, b) for a, b in zip(out, want[i])) and all(torch.equal(a, b) for a, b in zip(eager, want[1 - i]))


@gpu
@pytest.mark.parametrize("rotary", [True, False])
def test_attention_kernel_many_items_at_once_and_captured(rotary, errors):
    """Launches whose blocks take their items from a counter: two calls at once, replays, a backward that runs twice."""
    lengths, S, hq, hk, D = [[30, 300, 128, 1000, 0, 71], [700, 5, 640, 100, 0, 0]], 1600, 48, 16, 64
    qkv, do, cos, sin = _inputs(lengths, S, hq, hk, D, rotary, "cuda")
    layout = _layout(lengths, S, "cuda")
    want = _run(qkv, do, cos, sin, layout, hq, hk, D)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(_run(qkv, do, cos, sin, layout, hq, hk, D))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for run in got for a, b in zip(run, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _run(qkv, do, cos, sin, layout, hq, hk, D)
    for _ in range(3):
        for t in out:
            t.zero_()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
    x = qkv.clone().requires_grad_(True)
    o = pf.packed_attention(x, cos, sin, layout, hq, hk, D)
    for _ in range(2):
        (grad,) = torch.autograd.grad(o, x, do, retain_graph=True)
        assert torch.equal(grad, want[1])
