"""The vocabulary operators (theseus.vocab) where calls are unusual: logits of any magnitude, rows far
apart, inputs changed between the call and its backward, traced and forward-mode calls, sizes
past a launch's, gradients of tokens that do not count.
"""
import pytest
import torch

from test_vocab import _dense, _grad_close, _oracle
from theseus import vocab

gpu = pytest.mark.gpu


def _lse_close(got, x, T):
    """The bound of a sum of V exponentials of 1 ulp each and one logarithm."""
    want = torch.logsumexp(x.double() / T, -1)
    assert ((got.double().cpu() - want).abs() <= 2.0 ** -20 * (want.abs() + 1)).all(), (got.tolist(), want.tolist())


# masks that are neither -inf nor the type's lowest value, and logits as large
LARGE = [s * v for v in (3e3, 2e5, 5e9, 1e10, 1e11, 1e15, 1e20) for s in (-1, 1)]


@gpu
@pytest.mark.parametrize("T", [1.0, 2.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_log_sum_exp_of_large_finite_rows(dtype, T):
    g = torch.Generator().manual_seed(0)
    c = torch.tensor(LARGE)[:, None]
    for V in (300, 5000):
        flat = c.expand(-1, V).to(dtype)
        near = (c * (1 + 1e-6 * torch.randn(len(LARGE), V, generator=g))).to(dtype)
        ends = flat.clone()
        ends[:, V // 3] = 4.0
        for x in (flat, near, ends):
            _lse_close(vocab.top_logits(x.cuda(), 5, temperature=T)[2], x, T)


@gpu
@pytest.mark.parametrize("T", [1.0, 2.0])
@pytest.mark.parametrize("dtype,V", [(torch.bfloat16, 140000), (torch.float32, 70001)])
def test_log_sum_exp_with_one_slab_of_large_values(dtype, V, T):
    """A row in three slabs, the first 60 % of it at one value: a whole slab, and a part of the next."""
    g = torch.Generator().manual_seed(1)
    x = 3 * torch.randn(len(LARGE), V, generator=g)
    x[:, :V * 6 // 10] = torch.tensor(LARGE)[:, None]
    x = x.to(dtype)
    values, _, lse = vocab.top_logits(x.cuda(), 5, temperature=T)
    _lse_close(lse, x, T)
    assert torch.equal(values.cpu(), x.topk(5, -1).values)


# ------------------------------------------------------------------------------ rows far apart
def _inputs(M, D, V, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(M, D, generator=g).bfloat16(), (torch.randn(V, D, generator=g) * (2 / D ** .5)).bfloat16(), g


def _python_path(monkeypatch, native):
    if not native:
        monkeypatch.setattr(vocab, "_native", lambda *xs: None)


@gpu
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("B,T,D", [(1, 410, 5120), (3, 410, 5120), (1, 33000, 64), (40, 33000, 64), (2, 30000, 72)])
def test_last_tokens_of_long_sequences(B, T, D, native, monkeypatch):
    """hidden[:, -1] of [B,T,D] with T D > 2^21: the loss and gradients of a contiguous copy."""
    _python_path(monkeypatch, native)
    print(f"  last of {B} x {T} x {D}", flush=True)
    x, w, g = _inputs(B, D, 700)
    labels = torch.randint(700, (B,), generator=g).cuda()
    full = torch.full((B, T, D), float("nan"), dtype=torch.bfloat16, device="cuda")
    full[:, -1] = x.cuda()
    for reduction in ("mean", "none"):
        got, want = [], []
        for out, h in ((got, full.clone().requires_grad_()), (want, x.cuda().requires_grad_())):
            wt = w.cuda().requires_grad_()
            loss = vocab.linear_cross_entropy(h[:, -1] if h.dim() == 3 else h, wt, labels, reduction=reduction)
            dh, dw = torch.autograd.grad(loss.sum(), (h, wt))
            out += [loss.detach(), dh[:, -1] if dh.dim() == 3 else dh, dw]
            assert dh.dim() == 2 or not dh[:, :-1].any()
        for p, q in zip(got, want):
            assert torch.equal(p, q)
        assert torch.equal(vocab.linear_cross_entropy(full[:, -1], w.cuda(), labels, reduction=reduction), want[0])


@gpu
@pytest.mark.parametrize("native", [True, False])
def test_weight_rows_far_apart(native, monkeypatch):
    _python_path(monkeypatch, native)
    x, w, g = _inputs(9, 64, 5)
    labels = torch.randint(5, (9,), generator=g).cuda()
    want = vocab.linear_cross_entropy(x.cuda(), w.cuda(), labels)
    wide = torch.full((5, (1 << 21) + 64), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, :64] = w.cuda()
    assert torch.equal(vocab.linear_cross_entropy(x.cuda(), wide[:, :64], labels), want)
    one = vocab.linear_cross_entropy(x.cuda(), wide[2:3, :64], torch.zeros(9, dtype=torch.int64).cuda(), reduction="none")
    assert one.abs().max() <= 1e-5  # (a vocabulary of one word)


def test_strides_are_sized_without_a_gpu():
    """Hidden rows at any distance; of one row no stride is used, of a weight's rows 2^21 is the limit;
    only what needs it is copied."""
    lib, p = vocab._lib(), 1 << 20
    ok = dict(rows=4, vocab=1000, width=64, targets=1, hidden=p, weight=p, hidden_stride=64, weight_stride=64, index=p,
              temperature=1.0, reduction=0, loss=p)
    size = lambda **kw: lib.theseus_vocab_loss_workspace_size(vocab.LossArgs(**{**ok, **kw}))  # noqa: E731
    far = 1 << 21
    assert size(hidden_stride=far) == size()
    copied = size(hidden_stride=far + 8)
    assert size() < copied <= size() + 4 * 64 * 2 + 256 and size(hidden_stride=1 << 40) == size(hidden=p + 2) == copied
    assert size(rows=1, hidden_stride=1 << 40) == size(rows=1) > 0
    assert size(weight_stride=far) == size() and size(weight_stride=far + 8) == 0
    assert size(vocab=1, weight_stride=far + 8) == size(vocab=1) > 0
    assert size(weight=p + 2) >= size() + 1000 * 64 * 2


# ------------------------------------------------------------------------------ targets changed before the backward
def _targets(g, M=300, V=700, K=6):
    return {"labels": torch.randint(V, (M,), generator=g).cuda(), "top_indices": torch.randint(V, (M, K), generator=g).cuda(),
            "top_values": torch.randn(M, K, generator=g).cuda(), "teacher_lse": torch.full((M,), 2.0).cuda(),
            "token_weight": torch.rand(M, generator=g).cuda()}


def _loss_of(name, h, w, t, **more):
    if name == "labels":
        return vocab.linear_cross_entropy(h, w, t["labels"], **more)
    return vocab.linear_top_distillation(h, w, t["top_values"], t["top_indices"], teacher_lse=t["teacher_lse"],
                                         token_weight=t["token_weight"], **more)


NAMES = ["labels", "top_indices", "top_values", "teacher_lse", "token_weight"]


@gpu
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("name", NAMES)
def test_changed_targets_never_give_other_gradients(name, native, monkeypatch):
    """A backward that reads the targets again raises once they were changed; the others give the call's."""
    _python_path(monkeypatch, native)
    x, w, g = _inputs(300, 64, 700)
    t = _targets(g)
    h, wt = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    for more, again in ((dict(reduction="none", piece_rows=256), True), (dict(reduction="none"), False), (dict(reduction="mean"), False)):
        want = torch.autograd.grad(_loss_of(name, h, wt, t, **more).sum(), (h, wt))
        old = t[name].clone()
        loss = _loss_of(name, h, wt, t, **more).sum()
        t[name].zero_()
        if not again:
            got = torch.autograd.grad(loss, (h, wt), retain_graph=True)
            assert all(torch.equal(p, q) for p, q in zip(got, want))
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(loss, (h, wt))
        t[name].copy_(old)
    loss = _loss_of(name, h, wt, t, reduction="none", piece_rows=256).sum()
    assert all(torch.isfinite(p).all() for p in torch.autograd.grad(loss, (h, wt)))


@gpu
@pytest.mark.parametrize("native", [True, False])
def test_targets_of_inference_mode(native, monkeypatch):
    """A teacher's tensors from torch.inference_mode, written again before a backward that reads the targets anew."""
    _python_path(monkeypatch, native)
    x, w, g = _inputs(300, 64, 700)
    t = _targets(g)
    h, wt = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    for name in ("labels", "top_values"):
        for more in (dict(reduction="none", piece_rows=256), dict(reduction="mean")):
            want = torch.autograd.grad(_loss_of(name, h, wt, t, **more).sum(), (h, wt))
            with torch.inference_mode():
                u = {k: v.clone() for k, v in t.items()}
            loss = _loss_of(name, h, wt, u, **more).sum()
            with torch.inference_mode():
                for v in u.values():
                    v.zero_()
            for _ in range(2):
                got = torch.autograd.grad(loss, (h, wt), retain_graph=True)
                assert all(torch.equal(p, q) for p, q in zip(got, want))


# ------------------------------------------------------------------------------ traces and forward mode
CALLS = {"cross_entropy": lambda h, w, y, tv, ti, lse, wt, **kw: vocab.linear_cross_entropy(h, w, y, **kw),
         "distillation": lambda h, w, y, tv, ti, lse, wt, **kw: vocab.linear_top_distillation(
             h, w, tv, ti, temperature=2.0, teacher_lse=lse, token_weight=wt, **kw)}


def _call_tensors(seed, M=40, V=300):
    x, w, g = _inputs(M, 64, V, seed)
    t = _targets(g, M, V)
    return x.cuda(), w.cuda(), t["labels"], t["top_values"], t["top_indices"], t["teacher_lse"], t["token_weight"]


@gpu
@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("name", list(CALLS))
def test_traced_losses_run_again(name, reduction):
    """torch.jit.trace, without gradients and with them: a replay computes the loss of its own inputs."""
    f = lambda *a: CALLS[name](*a, reduction=reduction)  # noqa: E731
    args, other = _call_tensors(1), _call_tensors(2)
    traced = torch.jit.trace(f, args, check_trace=False)
    for a in (args, other):
        assert torch.equal(traced(*a), f(*a))
    # (hidden states whose rows lie otherwise than the traced ones'; labels of other tokens)
    turned = (other[0].t().contiguous().t(), *other[1:])
    assert torch.equal(traced(*turned), f(*other))
    with pytest.raises(Exception, match="must have shape"):
        traced(*other[:2], *(t[:7] for t in other[2:]))
    args, other = ([x.requires_grad_() for x in a[:2]] + list(a[2:]) for a in (args, other))
    traced = torch.jit.trace(f, tuple(args), check_trace=False)
    got, want = traced(*other).sum(), f(*other).sum()
    assert torch.equal(got.detach(), want.detach())
    for p, q in zip(torch.autograd.grad(got, other[:2]), torch.autograd.grad(want, other[:2])):
        assert torch.equal(p, q)
    batch = [x.detach() if i == 1 else x.detach().reshape(2, 20, *x.shape[1:]) for i, x in enumerate(args)]
    traced = torch.jit.trace(f, tuple(batch), check_trace=False)
    assert torch.equal(traced(*batch), f(*batch))


@gpu
@pytest.mark.parametrize("at", [0, 1, 3, 5, 6])
def test_losses_refuse_a_tangent(at):
    """Forward mode is not supported: no derivative of 0 by leaving a tangent behind."""
    args = list(_call_tensors(3))
    with torch.autograd.forward_ad.dual_level():
        args[at] = torch.autograd.forward_ad.make_dual(args[at], torch.ones_like(args[at]))
        for name in CALLS if at < 2 else ["distillation"]:
            with pytest.raises(NotImplementedError, match="jvp"):
                CALLS[name](*args)


@gpu
def test_traced_top_logits_run_again():
    g = torch.Generator().manual_seed(4)
    f = lambda z: vocab.top_logits(z, 7, temperature=2.0)  # noqa: E731
    a, b = (torch.randn(6, 500, generator=g).cuda() for _ in range(2))
    traced = torch.jit.trace(f, (a,), check_trace=False)
    for z in (a, b, b.t().contiguous().t()):
        for p, q in zip(traced(z), f(b if z is not a else a)):
            assert torch.equal(p, q)
    with pytest.raises(Exception, match="k must be"):
        traced(b[:, :5])
    for shape in ((2, 3, 500), (500,)):
        z = torch.randn(shape, generator=g).cuda()
        traced = torch.jit.trace(f, (z,), check_trace=False)
        for p, q in zip(traced(2 * z), f(2 * z)):
            assert torch.equal(p, q)
    want = f(a)
    with torch.autograd.forward_ad.dual_level():  # (no tangent: the call itself)
        for p, q in zip(f(a), want):
            assert torch.equal(p, q)


# ------------------------------------------------------------------------------ sizes past one launch's
@gpu
@pytest.mark.parametrize("rows,V,k,dtype", [((1 << 22) + 5, 256, 129, torch.bfloat16), ((1 << 24) + 7, 16, 3, torch.float32)])
def test_top_logits_of_more_rows_than_one_launch_takes(rows, V, k, dtype):
    """Every row holds 0 .. V - 1 turned by its number: the answers are known."""
    print(f"  top of {rows} x {V}", flush=True)
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GB")
    col = torch.arange(V, device="cuda", dtype=torch.int32)
    x = torch.empty(rows, V, dtype=dtype, device="cuda")
    piece = 1 << 18
    for r in range(0, rows, piece):
        n = min(piece, rows - r)
        x[r:r + n] = (col[None] * 5 + torch.arange(r, r + n, device="cuda", dtype=torch.int32)[:, None]) % V
    values, indices, lse = vocab.top_logits(x, k)
    want = torch.arange(V - 1, V - 1 - k, -1, device="cuda", dtype=torch.int64)
    inverse = pow(5, -1, V)
    assert torch.equal(values[0].long(), want) and bool((values == values[0]).all()) and bool((lse == lse[0]).all())
    for r in range(0, rows, piece):
        n = min(piece, rows - r)
        row = torch.arange(r, r + n, device="cuda", dtype=torch.int64)[:, None]
        assert torch.equal(indices[r:r + n], (want[None] - row) * inverse % V), r
    _lse_close(lse[:1], x[:1].cpu(), 1.0)
    del x, values, indices, lse
    torch.cuda.empty_cache()


@gpu
@pytest.mark.parametrize("top", [torch.float32, torch.bfloat16])
def test_distillation_of_more_tokens_than_one_launch_takes(top):
    """2^26 + 9 tokens of width 1 and a vocabulary of 3, two targets each: every token's loss."""
    M, K = (1 << 26) + 9, 2
    print(f"  distillation of {M} tokens", flush=True)
    free, _ = torch.cuda.mem_get_info()
    if free < 40 << 30:
        pytest.skip("needs 40 GB")
    h = (torch.arange(M, device="cuda", dtype=torch.int32) % 97 - 48)[:, None].to(torch.bfloat16) / 16
    w = torch.tensor([[1.0], [-.5], [.25]], device="cuda").bfloat16()
    tv = torch.stack([(torch.arange(M, device="cuda", dtype=torch.int32) % p).to(top) / 8 for p in (31, 23)], 1)
    ti = torch.stack([torch.arange(M, device="cuda") % 3, (torch.arange(M, device="cuda") + 1) % 3], 1)
    weight = (torch.arange(M, device="cuda", dtype=torch.int32) % 5).float()
    loss = vocab.linear_top_distillation(h, w, tv, ti, token_weight=weight, reduction="none")
    piece = 1 << 23
    for i in range(0, M, piece):
        r = slice(i, i + piece)
        logp = torch.log_softmax(h[r].double() * w.double().t(), -1)
        q = torch.softmax(tv[r].double(), -1)
        want = weight[r] * (q * (q.log() - logp.gather(1, ti[r]))).sum(-1)
        # (losses of a few units of float32 exponentials and logarithms: 2^-20 of each of the terms, at most 10)
        assert ((loss[r] - want).abs() <= 2.0 ** -20 * 10 * (weight[r] + 1)).all(), i
    del h, tv, ti, weight, loss, logp, q, want
    torch.cuda.empty_cache()


# ------------------------------------------------------------------------------ tokens that do not count
@gpu
@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("M,piece", [(20, 0), (300, 0), (300, 256)])
def test_upstream_gradients_of_tokens_that_do_not_count_are_not_looked_at(M, piece, native, monkeypatch):
    """NaN and infinite upstream gradients (of a branch not taken) at ignored labels and weights of 0: 0, as
    torch.nn.functional.cross_entropy has it."""
    _python_path(monkeypatch, native)
    x, w, g = _inputs(M, 64, 700)
    t = _targets(g, M)
    out = torch.arange(M, device="cuda") % 3 == 0
    t["labels"][out] = -100
    t["token_weight"][out] = 0
    up = torch.rand(M, generator=g).cuda()
    bad = torch.where(out, torch.tensor([float("nan"), float("inf"), -float("inf")], device="cuda")[torch.arange(M, device="cuda") % 3], up)
    bad[::6] = float("inf")
    h, wt = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    for name in ("labels", "top_values"):
        loss = lambda: _loss_of(name, h, wt, t, reduction="none", piece_rows=piece)  # noqa: E731
        for p, q in zip(torch.autograd.grad(loss(), (h, wt), bad), torch.autograd.grad(loss(), (h, wt), torch.where(out, 0., up))):
            assert torch.isfinite(q).all() and torch.equal(p, q)


def test_any_number_of_piece_rows_is_taken():
    """"All of them" in one piece, however that is written."""
    lib, p = vocab._lib(), 1 << 20
    size = lambda piece: lib.theseus_vocab_loss_workspace_size(vocab.LossArgs(  # noqa: E731
        rows=100000, vocab=500, width=64, targets=1, hidden=p, weight=p, hidden_stride=64, weight_stride=64, index=p,
        temperature=1.0, reduction=2, loss=p, dhidden=p, piece_rows=piece))
    assert size(256) < size(32768) == size(100000) == size(2 ** 62) == size(2 ** 63 - 1)


@gpu
def test_sizes_out_of_range_are_named():
    y = torch.zeros(2, dtype=torch.int64, device="cuda")
    one = torch.zeros(1, 1, dtype=torch.bfloat16, device="cuda")
    for h, w in ((one.expand(2, 1), one.expand((1 << 22) + 1, 1)), (one.expand(2, (1 << 17) + 1), one.expand(3, (1 << 17) + 1)),
                 (one.expand((1 << 30) + 1, 1), one)):
        with pytest.raises(ValueError, match="at most"):
            vocab.linear_cross_entropy(h, w, y)
    with pytest.raises(ValueError, match="at most"):
        vocab.top_logits(one.expand(1, (1 << 30) + 1), 2)


# ------------------------------------------------------------------------------ distillation in pieces
@gpu
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("M,D,V,K,own_lse", [(700, 72, 900, 9, False), (513, 64, 500, 64, True), (1025, 128, 3001, 3, True)])
def test_distillation_in_pieces_matches_float64(M, D, V, K, own_lse, reduction):
    """Tokens in pieces of 256: targets, weights and their sum of every piece, the bounds of one piece."""
    print(f"  kd pieces M={M} D={D} V={V} K={K} lse={own_lse} {reduction}", flush=True)
    T = 2.0
    x, w, g = _inputs(M, D, V, M)
    tv = 2 * torch.randn(M, K, generator=g)
    tv[torch.rand(M, K, generator=g) < .1] = -float("inf")
    tv[:, 0] = 1.0
    ti = torch.randint(V, (M, K), generator=g)
    weight = torch.rand(M, generator=g)
    weight[::5] = 0
    up = torch.rand(M, generator=g) if reduction == "none" else torch.tensor(1.0)
    tz = tv.double() / T
    lse = torch.logsumexp(tz, -1).float() + (.25 if own_lse else 0.)
    q = torch.exp(tz - lse[:, None].double()) if own_lse else torch.softmax(tz, -1)
    logq = (tz - lse[:, None].double()) if own_lse else torch.log_softmax(tz, -1)
    H = torch.where(q > 0, q * logq, 0.).nan_to_num(0.).sum(-1)
    wd = weight.double()
    total = wd.sum() if reduction == "mean" else torch.tensor(1.0).double()
    o = _oracle(x, w, _dense(M, V, ti, q), H, wd, T, wd * up.double() / total)
    call = lambda a, b, **kw: vocab.linear_top_distillation(  # noqa: E731
        a, b, tv.cuda(), ti.cuda(), temperature=T, teacher_lse=lse.cuda() if own_lse else None, token_weight=weight.cuda(),
        reduction=reduction, **kw)
    # (q itself: float32 exponentials of |t / T - lse| < 20, 2^-20 of each term)
    qtol = T * T * wd * 2.0 ** -19 * (q * logq.abs().nan_to_num(0., 0., 0.)).sum(-1) + 1e-6 * o["loss"].abs()
    h, wt = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    loss = call(h, wt, piece_rows=256)
    assert torch.equal(loss.detach(), call(x.cuda(), w.cuda(), piece_rows=256))
    for got in (loss.detach().double().cpu(), call(x.cuda(), w.cuda()).double().cpu()):  # (whole: other tiles, other sums)
        if reduction == "none":
            assert ((got - o["loss"]).abs() <= o["ltol"] + qtol).all()
        else:
            assert abs(float(got) - float(o["loss"].sum() / total)) <= float((o["ltol"] + qtol).sum() / total)
    dx, dw = torch.autograd.grad(loss, (h, wt), up.cuda())
    _grad_close(dx, o["dx"], o["dx_tol"])
    _grad_close(dw, o["dw"], o["dw_tol"])
