"""theseus.vocab.embedding against float64: the rows, the table's gradient, what it refuses.

Tolerances.  A row is one float32 product (2^-24) rounded to the result's type: the same two roundings as
``(weight.float() * scale).to(dtype)``, so the same bits.  A gradient row of n tokens is a float32 sum of n values (in parts:
no more additions than n) times the scale: off by at most n 2^-24 sum|x| |scale| and the product's 2^-24,
and by the result's own half step, 2^-8 for bfloat16 and 2^-24 for float32.
"""
import math

import pytest
import torch

from theseus import vocab

gpu = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float32


def _inputs(M, D, V, seed, wt, ot, tokens="any"):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(V, D, generator=g).to(wt)
    up = torch.randn(M, D, generator=g).to(ot)
    if tokens == "any":
        ids = torch.randint(V, (M,), generator=g)
    elif tokens == "zipf":
        p = 1 / (torch.arange(V) + 2.7)
        ids = torch.randperm(V, generator=g)[torch.multinomial(p, M, replacement=True, generator=g)]
    elif tokens == "same":
        ids = torch.full((M,), V - 1)
    elif tokens == "falling":
        ids = (V - 1 - torch.arange(M)) % V
    else:  # stretches of a given length
        ids = (torch.arange(M) // int(tokens)) % V
    return w, up, ids


def _grad_close(got, ids, up, V, scale, skip=None):
    """Every row of the table's gradient against a float64 sum."""
    up, ids = up.double(), ids.clone()
    keep = (ids >= 0) & (ids < V)
    if skip is not None:
        keep &= ids != skip
    ids, up = ids[keep], up[keep]
    ref = torch.zeros(V, up.shape[1], dtype=torch.float64).index_add_(0, ids, up) * scale
    mass = torch.zeros(V, up.shape[1], dtype=torch.float64).index_add_(0, ids, up.abs()) * abs(scale)
    n = torch.zeros(V, dtype=torch.float64).index_add_(0, ids, torch.ones(len(ids), dtype=torch.float64))
    half = 2.0 ** -8 if got.dtype == BF else 2.0 ** -24
    tol = 1.01 * (((n + 1) * 2.0 ** -24)[:, None] * mass + half * ref.abs())
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    assert (got[n == 0] == 0).all()
    err = (got - ref).abs()
    assert (err <= tol).all(), f"worst {float((err / tol.clamp_min(1e-300)).max()):.2f} of the bound"


# M, D, V: one token, no vector of eight, around a vector, around the sorts' sizes and the runs' ends
SIZES = [(1, 1, 1), (1, 8, 5), (5, 7, 3), (17, 9, 40), (64, 64, 7), (33, 1001, 50), (2047, 12, 300), (2049, 20, 1000),
         (16384, 8, 70), (16385, 16, 5000), (40001, 9, 130000), (300, 2050, 20), (70, 4104, 33),
         (256, 3000, 12), (257, 3000, 12), (1023, 256, 2000), (1024, 64, 40), (1025, 64, 40), (512, 512, 700), (513, 512, 700), (900, 3, 70000), (4096, 24, 900), (4097, 24, 900),
         (6144, 8, 900), (6145, 8, 900)]


@gpu
@pytest.mark.parametrize("wt,ot", [(BF, BF), (BF, FP), (FP, BF), (FP, FP)], ids=["bf-bf", "bf-fp", "fp-bf", "fp-fp"])
@pytest.mark.parametrize("M,D,V", SIZES)
def test_rows_and_gradient_match_float64(M, D, V, wt, ot):
    print(f"  embed M={M} D={D} V={V} {wt} {ot}", flush=True)
    scale = 1.0 if M % 2 else math.sqrt(D) / 3
    w, up, ids = _inputs(M, D, V, M + D, wt, ot, "zipf" if M > 64 else "any")
    wc = w.cuda().requires_grad_()
    out = vocab.embedding(ids.cuda(), wc, scale=scale, dtype=ot)
    assert out.shape == (M, D) and out.dtype == ot
    s32 = torch.tensor(scale, dtype=FP)
    assert torch.equal(out.detach().cpu(), (w[ids].float() * s32).to(ot))
    dw, = torch.autograd.grad(out, (wc,), up.cuda())
    assert dw.dtype == wt and dw.shape == w.shape
    _grad_close(dw, ids, up, V, float(s32))


@gpu
@pytest.mark.parametrize("tokens", ["same", "falling", "1", "15", "16", "17", "31", "32", "48", "100"])
@pytest.mark.parametrize("M", [15, 16, 17, 32, 33, 500, 1024, 1025, 5000, 40000])
def test_stretches_of_one_token_inside_and_across_runs(M, tokens):
    print(f"  stretches M={M} {tokens}", flush=True)
    V, D = 997, 10
    w, up, ids = _inputs(M, D, V, M, FP, FP, tokens)
    wc = w.cuda().requires_grad_()
    dw, = torch.autograd.grad(vocab.embedding(ids.cuda(), wc), (wc,), up.cuda())
    _grad_close(dw, ids, up, V, 1.0)


@gpu
@pytest.mark.parametrize("tokens", ["same", "16", "17", "48"])
@pytest.mark.parametrize("M,D", [(256, 2500), (200, 2051), (512, 1000), (1024, 260), (100, 4)])
def test_stretches_of_few_tokens_in_rows_of_all_widths(M, D, tokens):
    """The one launch's rows that one group of threads adds, and those that all groups share."""
    print(f"  few tokens M={M} D={D} {tokens}", flush=True)
    V = 61
    w, up, ids = _inputs(M, D, V, M, BF, FP, tokens)
    wc = w.cuda().requires_grad_()
    dw, = torch.autograd.grad(vocab.embedding(ids.cuda(), wc, dtype=FP), (wc,), up.cuda())
    _grad_close(dw, ids, up, V, 1.0)


@gpu
def test_sorted_tokens_keep_their_order():
    """A sum whose value depends on the order: 2^24, ones that it swallows one by one, -2^24.  In the
    tokens' order nothing is left; sums of another order leave some ones."""
    for M in (16, 16384):
        up = torch.ones(M, 8)
        up[0], up[15] = 2.0 ** 25, -2.0 ** 25
        up[16:] = 0
        g = torch.Generator().manual_seed(M)
        ids = torch.zeros(M, dtype=torch.int64)
        ids[16:] = torch.randint(1, 50, (M - 16,), generator=g)
        w = torch.zeros(50, 8, device="cuda", requires_grad=True)
        dw, = torch.autograd.grad(vocab.embedding(ids.cuda(), w), (w,), up.cuda())
        assert (dw[0] == 0).all()


@gpu
@pytest.mark.parametrize("digits", [1, 2, 3])
@pytest.mark.parametrize("M", [250, 1000, 1500, 2048, 4000, 6000, 16000, 40000, 70000])
def test_every_sort_keeps_the_tokens_order(M, digits):
    """Sixteen tokens a row, dealt over all waves and blocks: 2^25, fourteen ones that it swallows (its neighbours are 4 apart),
    -2^25.  In the tokens' order nothing is left of any row; a last token ahead of another or a first one behind three leaves
    some.  A run has a multiple of 16 tokens, so that no row is added in parts."""
    print(f"  order M={M} digits={digits}", flush=True)
    rows = M // 16
    V = {1: rows, 2: 1 << 17, 3: (1 << 20) + 1}[digits]
    at = torch.arange(rows) * (V // rows)
    g = torch.Generator().manual_seed(M)
    ids = torch.cat([at.repeat(16), torch.full((M - 16 * rows,), -1)])[torch.randperm(M, generator=g)]
    order = ids.argsort(stable=True)
    order = order[ids[order] >= 0].reshape(rows, 16)
    up = torch.ones(M, 8)
    up[order[:, 0]], up[order[:, 15]] = 2.0 ** 25, -2.0 ** 25
    w = torch.zeros(V, 8, device="cuda", requires_grad=True)
    dw, = torch.autograd.grad(vocab.embedding(ids.cuda(), w), (w,), up.cuda())
    assert not dw.any()


@gpu
@pytest.mark.parametrize("M,D,V", [(4300001, 1, 3), (4300001, 1, 1 << 22), (200000, 8, 1 << 20)])
def test_many_tokens(M, D, V):
    """More blocks than one pass over their counts takes; one, two and three digits."""
    print(f"  many M={M} D={D} V={V}", flush=True)
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(V, (M,), generator=g)
    up = torch.randint(-8, 9, (M, D), generator=g).float()  # (sums below 2^24: exact)
    w = torch.zeros(V, D, device="cuda", requires_grad=True)
    dw, = torch.autograd.grad(vocab.embedding(ids.cuda(), w), (w,), up.cuda())
    ref = torch.zeros(V, D, dtype=torch.float64).index_add_(0, ids, up.double())
    assert ref.abs().max() < 2 ** 24 and torch.equal(dw.double().cpu(), ref)


@gpu
@pytest.mark.parametrize("M", [40, 20000])
def test_padding_and_indices_outside(M):
    """Padding gets its row and gives no gradient, an index outside a NaN row and none; what their rows of the
    upstream gradient hold (NaN, infinities) is not looked at."""
    V, D = 30, 24
    w, up, ids = _inputs(M, D, V, 3, FP, BF)
    ids[::7] = 4
    ids[1], ids[2], ids[3], ids[M - 1] = -1, V, 1 << 40, -(1 << 62)
    bad = (ids < 0) | (ids >= V)
    up[ids == 4] = math.inf
    up[bad] = math.nan
    for pad in (4, 4 - V):
        wc = w.cuda().requires_grad_()
        out = vocab.embedding(ids.cuda(), wc, padding_idx=pad, dtype=BF)
        o = out.detach().cpu()
        assert torch.isnan(o[bad]).all() and torch.equal(o[~bad], w[ids[~bad]].to(BF))
        dw, = torch.autograd.grad(out, (wc,), up.cuda())
        _grad_close(dw, ids, torch.where(torch.isfinite(up), up, 0), V, 1.0, skip=4)
    ids[:] = 4  # nothing counts
    wc = w.cuda().requires_grad_()
    dw, = torch.autograd.grad(vocab.embedding(ids.cuda(), wc, padding_idx=4), (wc,), torch.full((M, D), math.nan, device="cuda"))
    assert (dw == 0).all()


@gpu
def test_values_that_are_not_finite_pass_through():
    w = torch.tensor([[math.inf, -math.inf, math.nan, 1e38]] * 3, device="cuda")
    out = vocab.embedding(torch.tensor([2], device="cuda"), w, scale=8.0, dtype=BF).float().cpu()[0]
    assert out[0] == math.inf and out[1] == -math.inf and torch.isnan(out[2]) and out[3] == math.inf


@gpu
def test_no_tokens_and_shapes():
    w = torch.randn(9, 16, device="cuda", requires_grad=True)
    for shape in ((0,), (2, 0, 3)):
        out = vocab.embedding(torch.empty(shape, dtype=torch.int64, device="cuda"), w)
        assert out.shape == (*shape, 16)
        dw, = torch.autograd.grad(out.sum(), (w,))
        assert dw.shape == w.shape and (dw == 0).all()
    ids = torch.tensor(5, device="cuda")
    out = vocab.embedding(ids, w)
    assert out.shape == (16,) and torch.equal(out, w[5])
    ids = torch.randint(9, (2, 3, 5), device="cuda")
    assert torch.equal(vocab.embedding(ids, w), w[ids])


@gpu
def test_strides_and_alignment():
    """Rows apart, an offset base, a transposed table, strided ids, upstream gradients expanded and cut out of wider rows."""
    g = torch.Generator().manual_seed(0)
    big = torch.randn(40, 100, generator=g).bfloat16().cuda()
    ids = torch.randint(40, (70, 2), generator=g).cuda()
    for w in (big[:, 3:50], big[::2, 1:10], big[:, 7:8], big.t(), big[1:2].expand(5, 100)):
        for i in (ids[:, 0] % w.shape[0], (ids % w.shape[0]).t()):
            v = w.detach().requires_grad_()
            out = vocab.embedding(i, v)
            assert torch.equal(out.detach(), w[i])
            up = torch.randn(*i.shape, w.shape[1] + 3, generator=g).bfloat16().cuda()[..., 2:-1]
            dw, = torch.autograd.grad(out, (v,), up, retain_graph=True)
            _grad_close(dw, i.reshape(-1).cpu(), up.reshape(-1, w.shape[1]).cpu(), w.shape[0], 1.0)
            row = torch.randn(w.shape[1], generator=g).bfloat16().cuda()
            dw, = torch.autograd.grad(out, (v,), row.expand_as(out), retain_graph=True)
            _grad_close(dw, i.reshape(-1).cpu(), row.cpu().expand(i.numel(), -1), w.shape[0], 1.0)
            dw, = torch.autograd.grad(out.sum(), (v,))
            _grad_close(dw, i.reshape(-1).cpu(), torch.ones(i.numel(), w.shape[1]), w.shape[0], 1.0)


@gpu
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("table", ["transposed row", "column of a transposed table", "every third of it", "one number", "one number of all"])
def test_tables_of_one_column_of_any_stride(table, native, monkeypatch):
    """Of a dimension of one element torch keeps any stride, and calls the tensor contiguous all the same."""
    if not native:
        monkeypatch.setattr(vocab, "_native", lambda *a: None)
    g = torch.Generator().manual_seed(0)
    big = torch.randn(7, 60, generator=g).cuda()
    w = {"transposed row": torch.randn(1, 33, generator=g).cuda().t(), "column of a transposed table": big.t()[:, :1],
         "every third of it": big.t()[::3, 2:3], "one number": big.t()[5:6, 1:2], "one number of all": big.t()[5:6, 1:2].expand(9, 1)}[table]
    assert w.shape[1] == 1 and w.stride(1) != 1
    V = w.shape[0]
    for shape in ((40,), (3000,), (6, 5), (), (0,)):
        ids = torch.randint(V, shape, generator=g)
        for dtype in (FP, BF):
            v = w.detach().requires_grad_()
            out = vocab.embedding(ids.cuda(), v, scale=2.0, dtype=dtype)
            assert torch.equal(out.detach(), (2.0 * w[ids.cuda()]).to(dtype))
            up = torch.randn(*shape, 1, generator=g).to(dtype)
            dw, = torch.autograd.grad(out, (v,), up.cuda())
            assert dw.shape == w.shape
            _grad_close(dw, ids.reshape(-1), up.reshape(-1, 1), V, 2.0)


@gpu
def test_gradient_matches_differences():
    """The float32 gradient of a smooth function of the rows against central differences of it in float64."""
    g = torch.Generator().manual_seed(2)
    w = torch.randn(11, 5, generator=g)
    ids = torch.randint(11, (23,), generator=g)
    c = torch.randn(23, 5, generator=g)
    wc = w.cuda().requires_grad_()
    (torch.sin(vocab.embedding(ids.cuda(), wc, scale=1.5)) * c.cuda()).sum().backward()
    f = lambda t: float((torch.sin(1.5 * t[ids]) * c.double()).sum())  # noqa: E731
    for v, d in ((0, 0), (int(ids[0]), 3), (10, 4)):
        e = torch.zeros(11, 5, dtype=torch.float64)
        e[v, d] = 1e-5
        slope = (f(w.double() + e) - f(w.double() - e)) / 2e-5
        # (float32 sines and sums of at most 23 terms of size 1.5 |c| < 6, differences to 1e-9)
        assert abs(float(wc.grad[v, d]) - slope) < 23 * 6 * 2.0 ** -20


@gpu
def test_same_bits_every_time_and_from_python(monkeypatch):
    w, up, ids = _inputs(5000, 72, 300, 0, FP, BF, "zipf")
    def run():
        wc = w.cuda().requires_grad_()
        out = vocab.embedding(ids.cuda(), wc, scale=3.0, padding_idx=1, dtype=BF)
        return out.detach(), torch.autograd.grad(out, (wc,), up.cuda())[0]
    first = run()
    assert all(torch.equal(a, b) for a, b in zip(first, run()))
    monkeypatch.setattr(vocab, "_native", lambda *a: None)  # (where the binding was not built)
    assert all(torch.equal(a, b) for a, b in zip(first, run()))
    with torch.no_grad():
        assert torch.equal(first[0], vocab.embedding(ids.cuda(), w.cuda(), scale=3.0, padding_idx=1, dtype=BF))


@gpu
@pytest.mark.parametrize("native", [True, False])
def test_autograd_contract(native, monkeypatch):
    if not native:
        monkeypatch.setattr(vocab, "_native", lambda *a: None)
    ids = torch.randint(20, (6, 4), device="cuda")
    w = torch.randn(20, 8, device="cuda", requires_grad=True)
    out = vocab.embedding(ids, w)
    g, = torch.autograd.grad(out.square().sum(), (w,), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()
    flat = ids.reshape(-1)
    out = vocab.embedding(flat, w)
    flat[0] = 3
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    assert not vocab.embedding(ids, w.detach()).requires_grad
    # tied to a head: the two gradients add up
    w = torch.randn(20, 64, device="cuda", dtype=BF, requires_grad=True)
    h = vocab.embedding(ids, w)
    vocab.linear_cross_entropy(h, w, ids).backward()
    w2 = w.detach().clone().requires_grad_()
    h2 = h.detach().requires_grad_()
    vocab.linear_cross_entropy(h2, w2, ids).backward()
    dw, = torch.autograd.grad(vocab.embedding(ids, w2), (w2,), h2.grad)
    assert torch.equal(w.grad, dw + w2.grad)


@gpu
@pytest.mark.parametrize("native", [True, False])
def test_tokens_made_in_inference_mode(native, monkeypatch):
    """Sampled tokens, say: a copy is kept for the gradient, as of the losses' labels."""
    if not native:
        monkeypatch.setattr(vocab, "_native", lambda *a: None)
    with torch.inference_mode():
        ids = torch.randint(20, (6, 4), device="cuda")
    w = torch.randn(20, 8, device="cuda", requires_grad=True)
    kept = ids.clone()
    out = vocab.embedding(ids, w)
    assert torch.equal(out.detach(), w.detach()[kept])
    with torch.inference_mode():
        ids.zero_()
    dw, = torch.autograd.grad(out.sum(), (w,))
    _grad_close(dw, kept.reshape(-1).cpu(), torch.ones(24, 8), 20, 1.0)


@gpu
def test_a_trace_runs_again_and_forward_mode_is_refused():
    w = torch.randn(20, 8, device="cuda")
    f = lambda i, t: vocab.embedding(i, t, scale=2.0)  # noqa: E731
    i, j = torch.randint(20, (7,), device="cuda"), torch.randint(20, (7,), device="cuda")
    traced = torch.jit.trace(f, (i, w), check_trace=False)
    assert torch.equal(traced(j, 3 * w), 6 * w[j])
    with pytest.raises((RuntimeError, NotImplementedError)):
        with torch.autograd.forward_ad.dual_level():
            vocab.embedding(i, torch.autograd.forward_ad.make_dual(w, w))


@gpu
def test_on_another_stream_and_in_a_graph():
    """Captured with its gradient and replayed on new tokens, eager calls between, each replay against an eager call."""
    w, up, _ = _inputs(20000, 40, 500, 0, FP, BF)
    w, up = w.cuda(), up.cuda()
    ids = torch.zeros(20000, dtype=torch.int64, device="cuda")
    side = torch.cuda.Stream()

    def call():
        wc = w.detach().requires_grad_()
        out = vocab.embedding(ids, wc, padding_idx=0, dtype=BF)
        return out.detach(), torch.autograd.grad(out, (wc,), up)[0]

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for n in range(4):
        ids.copy_(torch.randint(500, (20000,), generator=torch.Generator().manual_seed(n)))
        graph.replay()
        torch.cuda.synchronize()
        want = call()
        assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1])
    del graph, held


@gpu
def test_a_capture_beside_a_living_graph_of_the_weight_is_refused():
    """Whose backward would draw the other graph's stream into the capture; once that graph is gone, the same capture works."""
    ids = torch.randint(500, (2000,), generator=torch.Generator().manual_seed(0)).cuda()
    w, up = torch.randn(500, 40, device="cuda", requires_grad=True), torch.randn(2000, 40, device="cuda")
    eager = vocab.embedding(ids, w)
    want = eager.detach(), torch.autograd.grad(eager, (w,), up, retain_graph=True)[0]
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="from another stream lives"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            vocab.embedding(ids, w)
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        with torch.no_grad():  # (nothing to go back through)
            vocab.embedding(ids, w)
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = vocab.embedding(ids, w)
        dw, = torch.autograd.grad(out, (w,), up)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.detach(), want[0]) and torch.equal(dw, want[1])
        again = vocab.embedding(ids, w.detach())
        assert torch.equal(again, want[0])
    del out, dw, graph


@gpu
def test_a_capture_of_a_computed_weight_beside_a_living_graph_is_refused():
    """A weight that is rounded inside the capture from a leaf of that graph, and one that was rounded before it."""
    ids = torch.randint(500, (2000,), generator=torch.Generator().manual_seed(0)).cuda()
    table, up = torch.randn(500, 40, device="cuda", requires_grad=True), torch.randn(2000, 40, device="cuda").bfloat16()
    eager = vocab.embedding(ids, table.to(BF))
    want = eager.detach(), torch.autograd.grad(eager, (table,), up, retain_graph=True)[0]
    early = table.detach().requires_grad_().to(BF)
    torch.cuda.synchronize()
    for weight in (lambda: table.to(BF), lambda: early):
        with pytest.raises(RuntimeError, match="from another stream lives"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                vocab.embedding(ids, weight())
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = vocab.embedding(ids, table.to(BF))
        dw, = torch.autograd.grad(out, (table,), up)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.detach(), want[0]) and torch.equal(dw, want[1])
        assert torch.equal(vocab.embedding(ids, table.detach().to(BF)), want[0])
    del out, dw, graph


@gpu
def test_offsets_past_32_bits():
    """A table of 4.6 GB (450001 x 5120): rows around 2^32 bytes, and rows behind."""
    V, D = 450001, 5120
    w = torch.zeros(V, D, dtype=BF, device="cuda")
    at = torch.tensor([0, 419429, 419430, 419431, V - 1], device="cuda")
    rows = torch.randn(5, D, device="cuda").bfloat16()
    w[at] = rows
    w.requires_grad_()
    out = vocab.embedding(at, w)
    assert torch.equal(out.detach(), rows)
    dw, = torch.autograd.grad(out, (w,), rows)
    assert torch.equal(dw[at], rows)
    dw[at] = 0
    assert not dw.any()


@gpu
def test_rows_past_32_bits():
    """Rows of 4.6 GB (450001 tokens of 5120): each against the table, and the gradient of small whole numbers, whose sums are exact."""
    M, V, D = 450001, 300, 5120
    g = torch.Generator(device="cuda").manual_seed(0)
    w = torch.randn(V, D, generator=g, device="cuda").bfloat16().requires_grad_()
    ids = torch.randint(V, (M,), generator=g, device="cuda")
    out = vocab.embedding(ids, w, dtype=BF)
    for at in range(0, M, 50000):
        assert torch.equal(out.detach()[at:at + 50000], w.detach()[ids[at:at + 50000]])
    up = torch.randint(-1, 2, (M, D), generator=g, device="cuda", dtype=torch.int8).bfloat16()
    dw, = torch.autograd.grad(out, (w,), up)
    ref = torch.zeros(V, D, device="cuda")
    for at in range(0, M, 50000):
        ref.index_add_(0, ids[at:at + 50000], up[at:at + 50000].float())
    assert torch.equal(dw, ref.bfloat16())


# ------------------------------------------------------------------------------ refusals
def test_refusals_of_the_c_abi_before_launching():
    lib = vocab._lib()
    p = 4096
    look = lambda M=4, V=9, D=8, wt=0, ot=0, ids=p, w=p, ld=8, out=p: lib.theseus_embed_lookup(  # noqa: E731
        M, V, D, wt, ot, ids, w, ld, 1.0, out, None)
    grad = lambda M=4, V=9, D=8, gt=0, wt=0, ids=p, g=p, ld=8, dw=p, ws=p, n=1 << 20: lib.theseus_embed_grad(  # noqa: E731
        M, V, D, gt, wt, ids, -1, g, ld, 1.0, dw, ws, n, None)
    # (status codes of theseus_wkv7.h: 1 shape, 2 type, 3 null pointer, 4 workspace)
    for kw in (dict(M=-1), dict(M=(1 << 30) + 1), dict(V=0), dict(V=(1 << 22) + 1), dict(D=0), dict(D=(1 << 17) + 1), dict(ld=7)):
        assert look(**kw) == 1 and grad(**kw) == 1
    for a in (2, -1):
        assert look(wt=a) == look(ot=a) == grad(gt=a) == grad(wt=a) == 2
    assert look(ids=None) == look(w=None) == look(out=None) == 3
    assert grad(ids=None) == grad(g=None) == grad(dw=None) == 3
    need = lib.theseus_embed_grad_workspace_size(4000, 9, 8)
    assert need > 0 and grad(M=4000, n=need - 1) == 4 and grad(M=4000, ws=None) == 4
    assert look(M=0, ids=None, w=None, out=None) == 0
    assert lib.theseus_embed_grad_workspace_size(-1, 9, 8) == 0
    assert lib.theseus_embed_grad_workspace_size(256, 65536, 5120) == 0  # (few tokens: one launch)
    sizes = [lib.theseus_embed_grad_workspace_size(M, 65536, 64) for M in (1, 100, 16384, 16385, 1 << 20)]
    assert sizes == sorted(sizes)


def test_refusals_of_the_call():
    ids, w = torch.zeros(3, dtype=torch.int64), torch.zeros(4, 8)
    with pytest.raises(ValueError, match="CUDA"):
        vocab.embedding(ids, w)


@gpu
def test_refusals_by_name():
    ids, w = torch.zeros(3, dtype=torch.int64, device="cuda"), torch.zeros(4, 8, device="cuda")
    for kw, error, match in [(dict(padding_idx=4), ValueError, "padding_idx"), (dict(padding_idx=-5), ValueError, "padding_idx"),
                             (dict(scale=math.inf), ValueError, "scale"), (dict(scale=math.nan), ValueError, "scale"),
                             (dict(scale=1e39), ValueError, "scale"), (dict(dtype=torch.float16), TypeError, "dtype")]:
        with pytest.raises(error, match=match):
            vocab.embedding(ids, w, **kw)
    for i, t, error, match in [(ids.int(), w, TypeError, "int64"), (ids.float(), w, TypeError, "int64"), (ids, w.half(), TypeError, "weight"),
                               (ids, w[0], ValueError, "V, D"), (ids, w[:0], ValueError, "V, D"), (ids, w[:, :0], ValueError, "V, D"),
                               (ids, w.cpu(), ValueError, "CUDA"), (ids.cpu(), w, ValueError, "CUDA"),
                               (ids, w[:1].expand((1 << 22) + 1, 8), ValueError, "at most"),
                               (ids[:1].expand((1 << 30) + 1), w, ValueError, "at most")]:
        with pytest.raises(error, match=match):
            vocab.embedding(i, t)
