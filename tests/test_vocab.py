"""The vocabulary operators (theseus.vocab) against float64: losses and gradients of
linear_cross_entropy and linear_top_distillation, top_logits' selection, what each refuses.

Tolerances.  z = sum of D products in float32: an error of at most zt = 2^-24 (sqrt(D) + 8)
sum|x w| (random rounding; the 8 covers the matrix instruction's own order) and, through exp2 and
log2 of about 1 ulp each and the sum over the vocabulary, 2^-20 (|lse| + 1) on top.  The gradients'
left factor G = c (Q p - q) is rounded to bfloat16 (half an ulp: at most 2^-8 of it; its float16
exponential and float32 factors less than 2^-4 of that), and p is off by 2 zt + 2^-22 of itself:
an element of G by at most E = 1.07 x 2^-8 |G| + (2 zt + 2^-22) c Q p, an element of G W by
(E |W|) and the result's own 2^-8.
"""
import ctypes
import math

import pytest
import torch

from theseus import vocab
from theseus.wkv7 import extension

gpu = pytest.mark.gpu


def _inputs(M, D, V, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, D, generator=g).bfloat16()
    w = (torch.randn(V, D, generator=g) * (spread / math.sqrt(D))).bfloat16()
    return x, w, g


def _oracle(x, w, q_dense, H, weight, T, c):
    """float64: per-token losses (weighted), G's two gradients and what G's error may make of them."""
    x, w, q = x.double(), w.double(), q_dense.double()
    z = x @ w.t() / T
    lse = torch.logsumexp(z, -1)
    Q = q.sum(-1)
    loss = T * T * weight * (H - (q * z).sum(-1) + Q * lse)
    P = T * c[:, None] * Q[:, None] * torch.exp(z - lse[:, None])
    G = P - T * c[:, None] * q
    ztol = 2.0 ** -24 * (math.sqrt(x.shape[1]) + 8) * (x.abs() @ w.abs().t()).amax(-1) / T
    ltol = T * T * weight.abs() * Q * (2 * ztol + 2.0 ** -20 * (lse.abs() + 1)) + 1e-6 * loss.abs()
    E = 1.07 * 2.0 ** -8 * G.abs() + (2 * ztol + 2.0 ** -22)[:, None] * P.abs()
    return dict(loss=loss, dx=G @ w, dw=G.t() @ x, dx_tol=E @ w.abs(), dw_tol=E.t() @ x.abs(), ltol=ltol)


def _grad_close(got, want, tol):
    err = (got.double().cpu() - want).abs()
    tol = tol + 1.01 * 2.0 ** -8 * want.abs() + 1e-30
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), f"worst {float((err / tol).max()):.2f} of the bound at {int((err / tol).argmax())}"


def _dense(M, V, idx, q):
    d = torch.zeros(M, V, dtype=torch.float64)
    return d.scatter_add_(1, idx.clamp(0, V - 1), q.double())


def _run(f, x, w, up, reduction, need=("x", "w")):
    x = x.cuda().requires_grad_("x" in need)
    w = w.cuda().requires_grad_("w" in need)
    loss = f(x, w)
    loss.backward(up.cuda() if reduction == "none" else torch.tensor(float(up), device="cuda"))
    return loss.detach(), x.grad, w.grad


SIZES = [(1, 64, 1), (1, 8, 5), (2, 1, 3), (3, 40, 300), (64, 64, 256), (65, 128, 257), (130, 7, 33), (257, 100, 513),
         (300, 192, 1000), (512, 64, 2049), (70, 320, 70)]


@gpu
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("M,D,V", SIZES)
def test_cross_entropy_matches_float64(M, D, V, reduction):
    print(f"  ce M={M} D={D} V={V} {reduction}", flush=True)
    x, w, g = _inputs(M, D, V, seed=M + V)
    labels = torch.randint(V, (M,), generator=g)
    labels[torch.rand(M, generator=g) < .2] = -100
    weight = (labels != -100).double()
    up = torch.randn(M, generator=g) if reduction == "none" else torch.tensor(.75)
    total = weight.sum().clamp_min(1) if reduction == "mean" else torch.tensor(1.0)
    o = _oracle(x, w, _dense(M, V, labels[:, None], torch.ones(M, 1)), 0.0, weight, 1.0, weight * up.double() / total)
    loss, dx, dw = _run(lambda a, b: vocab.linear_cross_entropy(a, b, labels.cuda(), reduction=reduction), x, w, up, reduction)
    assert loss.dtype == torch.float32 and dx.dtype == dw.dtype == torch.bfloat16
    if reduction == "none":
        assert loss.shape == (M,) and ((loss.double().cpu() - o["loss"]).abs() <= o["ltol"]).all()
    else:
        assert abs(float(loss) - float(o["loss"].sum() / total)) <= float(o["ltol"].sum() / total) + 1e-7
    # (the reduced losses' gradients are rounded before the upstream gradient too)
    extra = 0.0 if reduction == "none" else 1.01 * 2.0 ** -8
    _grad_close(dx, o["dx"], o["dx_tol"] + extra * o["dx"].abs())
    _grad_close(dw, o["dw"], o["dw_tol"] + extra * o["dw"].abs())


def _teacher(M, V, K, g, dtype=torch.float32):
    idx = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(M)]) if V >= K else torch.randint(V, (M, K), generator=g)
    return (2 * torch.randn(M, K, generator=g)).to(dtype), idx


@gpu
@pytest.mark.parametrize("own_lse", [False, True])
@pytest.mark.parametrize("T", [1.0, 2.5])
@pytest.mark.parametrize("M,D,V,K,dtype", [(1, 64, 40, 1, "f32"), (5, 24, 300, 7, "bf16"), (66, 128, 1000, 64, "f32"),
                                           (257, 96, 515, 200, "f32"), (40, 64, 256, 256, "bf16"), (33, 64, 10, 30, "f32")])
def test_top_distillation_matches_float64(M, D, V, K, dtype, T, own_lse):
    print(f"  kd M={M} D={D} V={V} K={K} {dtype} T={T} lse={own_lse}", flush=True)
    x, w, g = _inputs(M, D, V, seed=M + K)
    tv, ti = _teacher(M, V, K, g, torch.bfloat16 if dtype == "bf16" else torch.float32)
    tv[torch.rand(M, K, generator=g) < .1] = -math.inf
    tv[:, 0] = 1.0
    ti[torch.isinf(tv)] = V + 5  # (not looked at)
    weight = torch.rand(M, generator=g)
    weight[::3] = 0
    if M == 1:
        weight[:] = .5
    tz = tv.double() / T
    lse = torch.logsumexp(tz, -1) + (.3 if own_lse else 0.)
    q = torch.exp(tz - lse[:, None].float().double()) if own_lse else torch.softmax(tz, -1)
    H = torch.where(q > 0, q * (tz - (lse[:, None].float().double() if own_lse else lse[:, None])), 0.).nan_to_num(0.).sum(-1)
    total = weight.double().sum()
    o = _oracle(x, w, _dense(M, V, ti, q), H, weight.double(), T, weight.double() / total)
    call = lambda a, b: vocab.linear_top_distillation(  # noqa: E731
        a, b, tv.cuda(), ti.cuda(), temperature=T, teacher_lse=lse.float().cuda() if own_lse else None, token_weight=weight.cuda())
    loss, dx, dw = _run(call, x, w, torch.tensor(1.0), "mean")
    # (q itself: float32 exponentials of |t / T - lse| < 20, 2^-20 of each term)
    qtol = T * T * (weight.double() * 2.0 ** -19 * (q * (tz - lse[:, None]).abs().nan_to_num(0., 0., 0.)).sum(-1)).sum()
    assert abs(float(loss) - float(o["loss"].sum() / total)) <= float((o["ltol"].sum() + qtol) / total) + 1e-6 * abs(float(loss))
    _grad_close(dx, o["dx"], o["dx_tol"])
    _grad_close(dw, o["dw"], o["dw_tol"])


@gpu
def test_tokens_with_nothing_to_learn():
    """All labels ignored; a teacher of whom nothing is left; weights all 0: loss and gradients 0."""
    x, w, _ = _inputs(6, 64, 300)
    ign = torch.full((6,), -100).cuda()
    ninf = torch.full((6, 4), -math.inf).cuda()
    idx = torch.zeros(6, 4, dtype=torch.int64).cuda()
    for f in (lambda a, b: vocab.linear_cross_entropy(a, b, ign),
              lambda a, b: vocab.linear_top_distillation(a, b, ninf, idx),
              lambda a, b: vocab.linear_top_distillation(a, b, ninf + 1e9, idx, token_weight=torch.zeros(6).cuda()),
              lambda a, b: vocab.linear_top_distillation(a, b, torch.zeros(6, 4).cuda(), idx, token_weight=torch.zeros(6).cuda())):
        loss, dx, dw = _run(f, x, w, torch.tensor(1.0), "mean")
        assert float(loss) == 0 and not dx.any() and not dw.any()


@gpu
def test_equal_target_indices_add_up_and_bad_labels_are_nan():
    x, w, _ = _inputs(3, 64, 50)
    tv, ti = torch.zeros(3, 4), torch.tensor([[7, 7, 7, 9]] * 3)
    one = torch.tensor([[7, 9]] * 3)
    a = _run(lambda p, r: vocab.linear_top_distillation(p, r, tv.cuda(), ti.cuda(), reduction="sum"), x, w, torch.tensor(1.), "sum")
    q = torch.tensor([[.75, .25]] * 3)
    o = _oracle(x, w, _dense(3, 50, one, q), math.log(.25) * torch.ones(3).double(), torch.ones(3).double(), 1.0, torch.ones(3).double())
    assert abs(float(a[0]) - float(o["loss"].sum())) <= float(o["ltol"].sum())
    _grad_close(a[1], o["dx"], o["dx_tol"])
    _grad_close(a[2], o["dw"], o["dw_tol"])
    loss = vocab.linear_cross_entropy(x.cuda(), w.cuda(), torch.tensor([0, 50, -1]).cuda(), reduction="none")
    assert torch.isnan(loss).tolist() == [False, True, True]


@gpu
def test_a_confident_token_keeps_its_gradient():
    """p(label) = 1 - 1e-4: p - 1 has to come from float32, not from a rounded p (0 or 2^-8)."""
    D, V = 64, 400
    x, w = torch.zeros(1, D), torch.zeros(V, D)
    x[0, 0], w[3, 0] = 4.0, 4.0
    w[:, 1] = 1.0
    x, w = x.bfloat16(), w.bfloat16()
    one = torch.ones(1).double()
    o = _oracle(x, w, _dense(1, V, torch.tensor([[3]]), torch.ones(1, 1)), 0.0, one, 1.0, one)
    _, dx, dw = _run(lambda a, b: vocab.linear_cross_entropy(a, b, torch.tensor([3]).cuda()), x, w, torch.tensor(1.), "mean")
    _grad_close(dx, o["dx"], o["dx_tol"])
    _grad_close(dw, o["dw"], o["dw_tol"])
    assert float(o["dw"][3, 0]) != 0 and abs(float(dw[3, 0]) / float(o["dw"][3, 0]) - 1) < .01


@gpu
@pytest.mark.parametrize("need", [("x",), ("w",)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_one_gradient_alone_is_the_same(need, reduction):
    x, w, g = _inputs(100, 64, 600)
    labels = torch.randint(600, (100,), generator=g).cuda()
    up = torch.rand(100) if reduction == "none" else torch.tensor(1.)
    f = lambda a, b: vocab.linear_cross_entropy(a, b, labels, reduction=reduction)  # noqa: E731
    both, one = _run(f, x, w, up, reduction), _run(f, x, w, up, reduction, need)
    assert torch.equal(both[0], one[0])
    i = 1 if need == ("x",) else 2
    assert torch.equal(both[i], one[i]) and one[3 - i] is None


@gpu
def test_row_pieces_agree_with_one_piece():
    x, w, g = _inputs(1000, 96, 700)
    labels = torch.randint(700, (1000,), generator=g)
    o = _oracle(x, w, _dense(1000, 700, labels[:, None], torch.ones(1000, 1)), 0.0, torch.ones(1000).double(), 1.0,
                torch.full((1000,), 1e-3).double())
    whole = _run(lambda a, b: vocab.linear_cross_entropy(a, b, labels.cuda()), x, w, torch.tensor(1.), "mean")
    cut = _run(lambda a, b: vocab.linear_cross_entropy(a, b, labels.cuda(), piece_rows=256), x, w, torch.tensor(1.), "mean")
    assert torch.equal(whole[0], cut[0])
    for got in (whole, cut):
        _grad_close(got[1], o["dx"], o["dx_tol"])
        _grad_close(got[2], o["dw"], o["dw_tol"])


@gpu
def test_views_shapes_and_autocast():
    """Hidden states [B,T,D] cut from longer ones, a head that is a slice, float32 under autocast."""
    x, w, g = _inputs(2 * 9, 72, 100)
    labels = torch.randint(100, (2, 8), generator=g).cuda()
    xb = x.cuda().reshape(2, 9, 72)
    want = vocab.linear_cross_entropy(xb[:, :-1].contiguous(), w.cuda(), labels, reduction="none")
    assert want.shape == (2, 8)
    assert torch.equal(vocab.linear_cross_entropy(xb[:, :-1], w.cuda(), labels, reduction="none"), want)
    wide = torch.full((100, 80), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, 3:75] = w.cuda()
    assert torch.equal(vocab.linear_cross_entropy(xb[:, :-1], wide[:, 3:75], labels, reduction="none"), want)
    odd = torch.full((18 * 72 + 1,), float("nan"), dtype=torch.bfloat16, device="cuda")
    odd[1:] = x.cuda().reshape(-1)
    assert torch.equal(vocab.linear_cross_entropy(odd[1:].reshape(2, 9, 72)[:, :-1], w.cuda(), labels, reduction="none"), want)
    xf, wf = xb.float().requires_grad_(), w.cuda().float().requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = vocab.linear_cross_entropy(xf[:, :-1], wf, labels, reduction="none")
    assert torch.equal(got, want)
    got.sum().backward()
    assert xf.grad.dtype == wf.grad.dtype == torch.float32 and not xf.grad[:, -1].any() and xf.grad[:, 0].any()
    # one hidden state for every token: the gradient is summed over the tokens
    h = x[:1].cuda().requires_grad_()
    vocab.linear_cross_entropy(h.expand(16, 72), w.cuda(), labels.reshape(-1)).backward()
    r = x[:1].double().requires_grad_()
    torch.nn.functional.cross_entropy(r.expand(16, 72) @ w.double().t(), labels.reshape(-1).cpu()).backward()
    assert (h.grad.double().cpu() - r.grad).norm() <= 16 * 2.0 ** -8 * r.grad.norm()


@gpu
def test_gradients_against_differences():
    """Central differences of the operator's own loss in directions whose steps are exact in bfloat16."""
    M, D, V, eps = 16, 64, 200, 2.0 ** -5
    g = torch.Generator().manual_seed(4)
    x = (torch.randint(-32, 33, (M, D), generator=g) / 16).bfloat16()       # |x| <= 2 in 1/16: x +- eps exact (7 bits)
    w = (torch.randint(-16, 17, (V, D), generator=g) / 128).bfloat16()
    labels = torch.randint(V, (M,), generator=g).cuda()
    dx = torch.randint(-1, 2, (M, D), generator=g).bfloat16()
    f = lambda a, b: vocab.linear_cross_entropy(a.cuda(), b.cuda(), labels, reduction="sum").item()  # noqa: E731
    _, gx, gw = _run(lambda a, b: vocab.linear_cross_entropy(a, b, labels, reduction="sum"), x, w, torch.tensor(1.), "sum")
    up, down = (x.float() + eps * dx.float()).bfloat16(), (x.float() - eps * dx.float()).bfloat16()
    assert torch.equal(up.float() - x.float(), eps * dx.float())
    slope, want = (f(up, w) - f(down, w)) / (2 * eps), float((gx.double().cpu() * dx.double()).sum())
    # gradient's rounding 2^-8 of sum |g d|, loss' rounding 1e-5 / eps, third derivative eps^2 / 6 sum |d.w|^3
    tol = 2.0 ** -8 * float((gx.double().cpu() * dx.double()).abs().sum()) + 1e-4 / eps + eps ** 2 / 6 * M * float(((dx.double() @ w.double().t()).abs() ** 3).amax())
    assert abs(slope - want) <= tol
    dw = torch.randint(-1, 2, (V, D), generator=g).bfloat16()
    e2 = 2.0 ** -8
    up, down = (w.float() + e2 * dw.float()).bfloat16(), (w.float() - e2 * dw.float()).bfloat16()
    assert torch.equal(up.float() - w.float(), e2 * dw.float())
    slope, want = (f(x, up) - f(x, down)) / (2 * e2), float((gw.double().cpu() * dw.double()).sum())
    tol = 2.0 ** -8 * float((gw.double().cpu() * dw.double()).abs().sum()) + 1e-4 / e2 + e2 ** 2 / 6 * M * float(((x.double() @ dw.double().t()).abs() ** 3).amax())
    assert abs(slope - want) <= tol


@gpu
def test_backward_twice_streams_and_determinism():
    x, w, g = _inputs(300, 128, 1000)
    labels = torch.randint(1000, (300,), generator=g).cuda()
    a, b = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    loss = vocab.linear_cross_entropy(a, b, labels)
    g1 = torch.autograd.grad(loss, (a, b), retain_graph=True)
    g2 = torch.autograd.grad(2 * loss, (a, b))
    for p, q in zip(g1, g2):
        assert torch.equal(2 * p, q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = torch.autograd.grad(vocab.linear_cross_entropy(a, b, labels), (a, b))
    torch.cuda.synchronize()
    for p, q in zip(g1, other):
        assert torch.equal(p, q)


@gpu
def test_graph_replays_match_eager():
    x, w, g = _inputs(80, 64, 500)
    labels = torch.randint(500, (80,), generator=g).cuda()
    a, b = x.cuda().requires_grad_(), w.cuda().requires_grad_()

    def step():
        loss = vocab.linear_cross_entropy(a, b, labels)
        return (loss, *torch.autograd.grad(loss, (a, b)), *vocab.top_logits(b.detach().t(), 5))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(3):
        with torch.no_grad():
            a.copy_(_inputs(80, 64, 500, seed=seed + 10)[0])
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(outs, want):
            assert torch.equal(p, q)


@gpu
def test_no_tokens():
    x, w, _ = _inputs(0, 64, 40)
    labels = torch.zeros(0, dtype=torch.int64).cuda()
    loss, dx, dw = _run(lambda a, b: vocab.linear_cross_entropy(a, b, labels), x, w, torch.tensor(1.), "mean")
    assert float(loss) == 0 and dx.shape == (0, 64) and not dw.any()
    assert vocab.linear_cross_entropy(x.cuda(), w.cuda(), labels, reduction="none").shape == (0,)
    v, i, lse = vocab.top_logits(torch.zeros(0, 10).cuda(), 3)
    assert v.shape == i.shape == (0, 3) and lse.shape == (0,)


# ------------------------------------------------------------------------------ top_logits
def _top_oracle(x, k, T):
    f = x.float()
    key = torch.where(torch.isnan(f), torch.tensor(math.inf), f)
    nan = torch.isnan(f)
    # stable descending order, NaN first, equal values by index
    order = sorted(range(x.shape[0]), key=lambda i: (not bool(nan[i]), -float(key[i]), i))[:k]
    return order, torch.logsumexp(x.double() / T, -1)


def _check_top(x, k, T=1.0, rows=None):
    v, i, lse = vocab.top_logits(x, k, temperature=T)
    assert v.dtype == x.dtype and i.dtype == torch.int64 and lse.dtype == torch.float32
    xc, ic, lc = x.cpu(), i.cpu(), lse.double().cpu()
    for r in rows if rows is not None else range(x.shape[0]):
        want, want_lse = _top_oracle(xc[r], k, T)
        assert ic[r].tolist() == want, r
        if torch.isfinite(want_lse):  # (sum of V exponentials of 1 ulp each, one logarithm)
            assert abs(float(lc[r] - want_lse)) <= 2.0 ** -20 * (abs(float(want_lse)) + 1)
        else:
            assert str(float(lc[r])) == str(float(want_lse))
    got, ref = v.float().cpu(), xc.float().gather(1, ic)
    assert torch.equal(got.nan_to_num(7e30), ref.nan_to_num(7e30))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,V,k", [(1, 1, 1), (3, 7, 7), (2, 129, 128), (5, 1000, 50), (4, 8191, 256), (2, 32768, 129),
                                   (3, 50001, 100), (2, 65537, 64), (1, 140000, 256)])
def test_top_logits_matches_sorting(M, V, k, dtype):
    print(f"  top M={M} V={V} k={k} {dtype}", flush=True)
    g = torch.Generator().manual_seed(V + k)
    _check_top((3 * torch.randn(M, V, generator=g)).to(dtype).cuda(), k, 2.0 if V % 2 else 1.0)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [300, 5000, 70001])
def test_top_logits_ties_masks_and_specials(V, dtype):
    print(f"  top specials V={V} {dtype}", flush=True)
    g = torch.Generator().manual_seed(V)
    x = (3 * torch.randn(12, V, generator=g)).to(dtype)
    low = torch.finfo(dtype).min
    x[0] = 1.5                                    # all equal
    x[1] = -math.inf                              # all masked
    x[2] = -math.inf
    x[2, [V - 1, 17, 44]] = 2.0                   # three left
    x[3] = low
    x[3, V // 2] = 0.0
    x[4] = torch.round(x[4].float()).to(dtype)    # many ties
    x[5, [3, V - 2]] = math.nan
    x[6, [5, 9]] = math.inf
    x[7, :] = torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0).to(dtype)
    x[8, ::2] = -math.inf
    x[9] = torch.arange(V).float().to(dtype)      # ascending: every bound is passed
    x[10] = -torch.arange(V).float().to(dtype)
    x[11, : V // 3] = 40.0                        # more than the list at the top
    for k in (1, 40, 256):
        _check_top(x.cuda(), k)


@gpu
def test_top_logits_reads_strided_rows_in_place():
    g = torch.Generator().manual_seed(0)
    for dtype in (torch.bfloat16, torch.float32):
        wide = torch.full((6, 3011), math.nan, dtype=dtype)
        wide[:, 5:2006] = torch.randn(6, 2001, generator=g).to(dtype)
        _check_top(wide.cuda()[:, 5:2006], 30)
        _check_top(wide.cuda()[::2, 5:2006], 30)
        _check_top(wide[:, 5:1005].t().contiguous().cuda().t(), 10)
    x = torch.randn(2, 3, 400, generator=g).cuda()
    v, i, lse = vocab.top_logits(x, 4)
    assert v.shape == i.shape == (2, 3, 4) and lse.shape == (2, 3)


@gpu
def test_teacher_to_student():
    """top_logits feeds linear_top_distillation; at k = V (and the teacher's lse) it is the whole divergence."""
    g = torch.Generator().manual_seed(1)
    x, w, _ = _inputs(50, 64, 200)
    t = 2 * torch.randn(50, 200, generator=g)
    for T in (1.0, 3.0):
        v, i, lse = vocab.top_logits(t.cuda(), 200, temperature=T)
        p = torch.log_softmax(x.double() @ w.double().t() / T, -1)
        q = torch.log_softmax(t.double() / T, -1)
        want = T * T * (q.exp() * (q - p)).sum(-1)
        for more in ({}, {"teacher_lse": lse}):
            got = vocab.linear_top_distillation(x.cuda(), w.cuda(), v, i, temperature=T, reduction="none", **more)
            assert (got.double().cpu() - want).abs().max() <= 2.0 ** -18 * T * T * 20


# ------------------------------------------------------------------------------ refusals
def test_refusals_without_a_gpu():
    x, w, y = torch.zeros(2, 8).bfloat16(), torch.zeros(5, 8).bfloat16(), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        vocab.linear_cross_entropy(x, w, y)
    with pytest.raises(ValueError, match="unknown reduction"):
        vocab.linear_cross_entropy(x, w, y, reduction="avg")
    with pytest.raises(ValueError, match="CUDA"):
        vocab.top_logits(torch.zeros(2, 8), 1)


@gpu
def test_refusals():
    x, w, y = torch.zeros(2, 8).bfloat16().cuda(), torch.zeros(5, 8).bfloat16().cuda(), torch.zeros(2, dtype=torch.int64).cuda()
    tv, ti = torch.zeros(2, 3).cuda(), torch.zeros(2, 3, dtype=torch.int64).cuda()
    for call, kind, match in [
            (lambda: vocab.linear_cross_entropy(x.float(), w, y), TypeError, "bfloat16"),
            (lambda: vocab.linear_cross_entropy(x, w.float(), y), TypeError, "bfloat16"),
            (lambda: vocab.linear_cross_entropy(x, w[:, :4], y), ValueError, "expected hidden"),
            (lambda: vocab.linear_cross_entropy(x, w[:0], y), ValueError, "expected hidden"),
            (lambda: vocab.linear_cross_entropy(x, w, y[:1]), ValueError, "labels must have shape"),
            (lambda: vocab.linear_cross_entropy(x, w, y.int()), TypeError, "labels must be int64"),
            (lambda: vocab.linear_cross_entropy(x, w, y.cpu()), ValueError, "labels must be on"),
            (lambda: vocab.linear_cross_entropy(x, w, y, piece_rows=-1), ValueError, "piece_rows"),
            (lambda: vocab.linear_top_distillation(x, w, tv, ti[:, :2]), ValueError, "top_values must have shape"),
            (lambda: vocab.linear_top_distillation(x, w, tv.half(), ti), TypeError, "top_values"),
            (lambda: vocab.linear_top_distillation(x, w, tv, ti, temperature=0.0), ValueError, "temperature"),
            (lambda: vocab.linear_top_distillation(x, w, tv, ti, temperature=math.nan), ValueError, "temperature"),
            (lambda: vocab.linear_top_distillation(x, w, tv, ti, token_weight=y.float()[:1]), ValueError, "token_weight"),
            (lambda: vocab.linear_top_distillation(x, w, tv, ti, teacher_lse=y), TypeError, "teacher_lse"),
            (lambda: vocab.linear_top_distillation(x, w, torch.zeros(2, 300).cuda(), torch.zeros(2, 300).long().cuda()), ValueError, "top logits"),
            (lambda: vocab.top_logits(tv, 4), ValueError, "k must be"),
            (lambda: vocab.top_logits(tv, 0), ValueError, "k must be"),
            (lambda: vocab.top_logits(tv.half(), 1), TypeError, "logits"),
            (lambda: vocab.top_logits(tv, 1, temperature=-1.0), ValueError, "temperature")]:
        with pytest.raises(kind, match=match):
            call()


def test_c_abi_refuses_without_launching():
    lib = vocab._lib()
    p = 1 << 20  # (an address that is never read: the checks come first)
    ok = dict(rows=4, vocab=100, width=64, targets=1, hidden=p, weight=p, hidden_stride=64, weight_stride=64, index=p,
              temperature=1.0, reduction=0, loss=p)
    size = lambda **kw: lib.theseus_vocab_loss_workspace_size(ctypes.byref(vocab.LossArgs(**{**ok, **kw})))  # noqa: E731
    call = lambda ws=None, n=0, **kw: lib.theseus_vocab_loss(ctypes.byref(vocab.LossArgs(**{**ok, **kw})), ws, n, None)  # noqa: E731
    assert size() > 0
    for bad in (dict(rows=-1), dict(vocab=0), dict(width=0), dict(targets=0), dict(targets=2), dict(hidden_stride=63),
                dict(temperature=0.0), dict(temperature=math.nan), dict(piece_rows=-1), dict(weight_stride=(1 << 21) + 1),
                dict(targets=257, top_values=p)):
        assert size(**bad) == 0 and call(**bad) == 1, bad
    assert call(top_dtype=3) == 2 and call(reduction=4) == 7
    assert call(hidden=None) == 3 and call(index=None) == 3
    assert call(p, size() - 1) == 4 and call(None, size()) == 4
    assert lib.theseus_vocab_loss(None, None, 0, None) == 3
    assert lib.theseus_vocab_scale(None, 1, None, 0, p, None) == 3 and lib.theseus_vocab_scale(p, -1, None, 0, p, None) == 1
    assert lib.theseus_vocab_scale(None, 0, None, 0, p, None) == 0 and lib.theseus_vocab_scale(p, 1, p, 1, None, None) == 3
    top = lambda M=2, V=100, k=5, dt=1, T=1.0, x=p, ld=100, v=p, i=p, ws=None, n=0: lib.theseus_vocab_top(  # noqa: E731
        M, V, k, dt, T, x, ld, v, i, None, ws, n, None)
    for bad in (dict(M=-1), dict(V=0), dict(k=0), dict(k=101), dict(V=1000, ld=1000, k=257), dict(ld=99), dict(T=0.0), dict(x=p + 2)):
        assert top(**bad) == 1, bad
    assert top(dt=2) == 2 and top(x=None) == 3 and top(v=None) == 3
    assert lib.theseus_vocab_top_workspace_size(2, 100, 5, 1) == 0
    need = lib.theseus_vocab_top_workspace_size(2, 100000, 5, 1)
    assert need > 0 and top(V=100000, ld=100000, ws=p, n=need - 1) == 4
    assert extension().lib.theseus_wkv7_error_string(4) == b"workspace too small"


def test_sizes_are_planned_for_any_shape_without_a_gpu():
    """The host's planning divides by tile counts: no size may stop it, 0 tokens among them."""
    lib = vocab._lib()
    for M in (0, 1, 3, 255, 256, 257, 5000, 40000, 1 << 20):
        for V in (1, 2, 63, 65, 255, 257, 50001, 1 << 22):
            for D in (1, 8, 64, 5120):
                for grads in ({}, {"dhidden": 16}, {"dhidden": 16, "dweight": 16}):
                    a = vocab.LossArgs(rows=M, vocab=V, width=D, targets=1, hidden=1 << 20, weight=1 << 20, hidden_stride=D,
                                       weight_stride=D, index=16, temperature=1.0, reduction=2, loss=16, **grads)
                    assert lib.theseus_vocab_loss_workspace_size(ctypes.byref(a)) > 0, (M, V, D)


def test_workspace_holds_a_piece_not_the_logits():
    """65536 tokens of a vocabulary of 131072: 16 GB of 16-bit probabilities, 2 GiB at a time."""
    a = vocab.LossArgs(rows=65536, vocab=131072, width=4096, targets=1, hidden=1 << 20, weight=1 << 20, hidden_stride=4096,
                       weight_stride=4096, index=16, temperature=1.0, reduction=2, loss=16, dhidden=16)
    lib = vocab._lib()
    n = lib.theseus_vocab_loss_workspace_size(ctypes.byref(a))
    assert 2 << 30 <= n < 3.5 * (1 << 30)
    a.dhidden = None
    assert lib.theseus_vocab_loss_workspace_size(ctypes.byref(a)) < 1 << 29


@gpu
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_the_python_autograd_function_gives_the_native_ones_bits(reduction, monkeypatch):
    x, w, g = _inputs(70, 64, 300)
    tv, ti = _teacher(70, 300, 9, g)
    up = torch.rand(70, generator=g) if reduction == "none" else torch.tensor(.3)
    f = lambda a, b: vocab.linear_top_distillation(a, b, tv.cuda(), ti.cuda(), temperature=2.0, reduction=reduction)  # noqa: E731
    native = _run(f, x, w, up, reduction)
    top = vocab.top_logits(tv.cuda(), 4)
    quiet = f(x.cuda(), w.cuda())
    monkeypatch.setattr(vocab, "_native", lambda *xs: None)
    for p, q in zip(native, _run(f, x, w, up, reduction)):
        assert torch.equal(p, q)
    for p, q in zip(top, vocab.top_logits(tv.cuda(), 4)):
        assert torch.equal(p, q)
    assert torch.equal(quiet, f(x.cuda(), w.cuda())) and torch.equal(quiet, native[0])


@gpu
@pytest.mark.parametrize("native", [True, False])
def test_second_derivatives_are_refused(native, monkeypatch):
    if not native:
        monkeypatch.setattr(vocab, "_native", lambda *xs: None)
    x, w, _ = _inputs(5, 64, 30)
    x = x.cuda().requires_grad_()
    loss = vocab.linear_cross_entropy(x, w.cuda(), torch.zeros(5, dtype=torch.int64).cuda())
    dx, = torch.autograd.grad(loss, x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        dx.sum().backward()


@gpu
@pytest.mark.parametrize("M,D,V", [(1021, 64, 50001), (1500, 128, 20011), (130, 64, 33000), (40, 128, 16500)])
def test_every_tile_shape_matches_float64(M, D, V):
    """Sizes at which the plan takes other tiles, several shapes for one matrix, parts of the contraction."""
    print(f"  shapes M={M} D={D} V={V}", flush=True)
    x, w, g = _inputs(M, D, V, seed=M)
    labels = torch.randint(V, (M,), generator=g)
    labels[-1] = V - 1
    one = torch.ones(M).double()
    o = _oracle(x.cuda(), w.cuda(), _dense(M, V, labels[:, None], torch.ones(M, 1)).cuda(), 0.0, one.cuda(), 1.0, one.cuda())
    o = {k: v.cpu() for k, v in o.items()}
    loss, dx, dw = _run(lambda a, b: vocab.linear_cross_entropy(a, b, labels.cuda(), reduction="none"), x, w, torch.ones(M), "none")
    assert ((loss.double().cpu() - o["loss"]).abs() <= o["ltol"]).all()
    _grad_close(dx, o["dx"], o["dx_tol"])
    _grad_close(dw, o["dw"], o["dw_tol"])


@gpu
@pytest.mark.parametrize("M,D,V,piece", [(300, 128, 50000, 0), (1000, 768, 30000, 0), (70, 2560, 40000, 0), (600, 768, 30000, 256)])
def test_tiles_of_192_rows_and_split_weight_gradients_match_float64(M, D, V, piece):
    """Sizes planned with tiles of 192 rows, dhidden two tiles a CU, dweight in full rounds and a rest (one piece, several)."""
    print(f"  shapes M={M} D={D} V={V} piece={piece}", flush=True)
    x, w, g = _inputs(M, D, V, seed=M)
    labels = torch.randint(V, (M,), generator=g)
    labels[0], labels[-1] = 0, V - 1
    one = torch.ones(M).double()
    o = _oracle(x.cuda(), w.cuda(), _dense(M, V, labels[:, None], torch.ones(M, 1)).cuda(), 0.0, one.cuda(), 1.0, (one / M).cuda())
    o = {k: v.cpu() for k, v in o.items()}
    loss, dx, dw = _run(lambda a, b: vocab.linear_cross_entropy(a, b, labels.cuda(), piece_rows=piece), x, w, torch.tensor(1.), "mean")
    assert abs(float(loss) - float(o["loss"].mean())) <= float(o["ltol"].mean())
    _grad_close(dx, o["dx"], o["dx_tol"])
    _grad_close(dw, o["dw"], o["dw_tol"])


@gpu
@pytest.mark.parametrize("M,D,V,piece", [(1000, 192, 30000, 0), (1000, 128, 30000, 0), (130, 320, 120000, 0), (100, 320, 90001, 0),
                                         (64, 384, 80000, 0), (250, 384, 60001, 0), (8, 768, 30152, 0), (64, 1280, 20000, 0),
                                         (128, 1280, 20001, 0), (90, 1100, 30000, 0), (1025, 1280, 20003, 512), (4096, 4608, 3000, 0)])
def test_workgroups_that_make_several_tiles_match_float64(M, D, V, piece):
    """More tiles than run at once, of one step more than the stages hold and of many, of just as many (one tile a
    workgroup), in parts and pieces."""
    print(f"  several tiles M={M} D={D} V={V} piece={piece}", flush=True)
    x, w, g = _inputs(M, D, V, seed=D)
    labels = torch.randint(V, (M,), generator=g)
    one = torch.ones(M).double()
    o = _oracle(x.cuda(), w.cuda(), _dense(M, V, labels[:, None], torch.ones(M, 1)).cuda(), 0.0, one.cuda(), 1.0, (one / M).cuda())
    o = {k: v.cpu() for k, v in o.items()}
    loss, dx, dw = _run(lambda a, b: vocab.linear_cross_entropy(a, b, labels.cuda(), piece_rows=piece), x, w, torch.tensor(1.), "mean")
    assert abs(float(loss) - float(o["loss"].mean())) <= float(o["ltol"].mean())
    _grad_close(dx, o["dx"], o["dx_tol"])
    _grad_close(dw, o["dw"], o["dw_tol"])
    each = vocab.linear_cross_entropy(x.cuda(), w.cuda(), labels.cuda(), reduction="none")
    assert ((each.double().cpu() - o["loss"]).abs() <= o["ltol"]).all()


@gpu
def test_many_targets_of_several_tiles_match_float64():
    M, D, V, K = 300, 320, 80001, 100
    x, w, g = _inputs(M, D, V, seed=5)
    tv, ti = 2 * torch.randn(M, K, generator=g), torch.randint(V, (M, K), generator=g)
    q = torch.softmax(tv.double() / 2, -1)
    one = torch.ones(M).double()
    o = _oracle(x.cuda(), w.cuda(), _dense(M, V, ti, q).cuda(), (q * q.log()).sum(-1).cuda(), one.cuda(), 2.0, one.cuda())
    o = {k: v.cpu() for k, v in o.items()}
    loss, dx, dw = _run(lambda a, b: vocab.linear_top_distillation(a, b, tv.cuda(), ti.cuda(), temperature=2.0, reduction="none"),
                        x, w, torch.ones(M), "none")
    # (q itself: float32 exponentials of |t / T - lse| < 20, 2^-20 of each term)
    qtol = 4 * 2.0 ** -19 * (q * q.log().abs()).sum(-1)
    assert ((loss.double().cpu() - o["loss"]).abs() <= o["ltol"] + qtol + 1e-6 * o["loss"].abs()).all()
    _grad_close(dx, o["dx"], o["dx_tol"])
    _grad_close(dw, o["dw"], o["dw_tol"])


@gpu
@pytest.mark.parametrize("M,D,V", [(1, 128, 4000), (5, 100, 333), (31, 256, 9000), (32, 64, 50)])
def test_few_tokens_gradients_are_rounded_once(M, D, V):
    """Up to 32 tokens: G in two halves (2^-16), its softmax part from float16 exponentials (11 bits: 2^-11), so
    the gradients are within that of G W and their own rounding, 2^-8."""
    print(f"  few M={M} D={D} V={V}", flush=True)
    x, w, g = _inputs(M, D, V, seed=V)
    labels = torch.randint(V, (M,), generator=g)
    up = torch.rand(M, generator=g) + .5
    ones = torch.ones(M).double()
    o = _oracle(x, w, _dense(M, V, labels[:, None], torch.ones(M, 1)), 0.0, ones, 1.0, up.double())
    z = x.double() @ w.double().t()
    P = up.double()[:, None] * torch.softmax(z, -1)
    G = P - up.double()[:, None] * torch.nn.functional.one_hot(labels, V)
    ztol = 2.0 ** -24 * (math.sqrt(D) + 8) * (x.double().abs() @ w.double().abs().t()).amax(-1)
    E = 1.1 * 2.0 ** -11 * P + 2.0 ** -16 * G.abs() + (2 * ztol + 2.0 ** -20)[:, None] * P
    loss, dx, dw = _run(lambda a, b: vocab.linear_cross_entropy(a, b, labels.cuda(), reduction="none"), x, w, up, "none")
    _grad_close(dx, o["dx"], E @ w.double().abs())
    _grad_close(dw, o["dw"], E.t() @ x.double().abs())


@gpu
@pytest.mark.parametrize("M,K,V", [(300, 200, 260), (256, 64, 64), (70, 256, 1000)])
def test_many_targets_in_one_tile(M, K, V):
    """Every token has the same K targets side by side: all in one or two tiles' columns."""
    print(f"  crowded M={M} K={K} V={V}", flush=True)
    x, w, g = _inputs(M, 64, V, seed=K)
    tv = torch.randn(M, K, generator=g)
    ti = torch.arange(K).repeat(M, 1)
    q = torch.softmax(tv.double(), -1)
    one = torch.ones(M).double()
    o = _oracle(x, w, _dense(M, V, ti, q), (q * q.log()).sum(-1), one, 1.0, one)
    loss, dx, dw = _run(lambda a, b: vocab.linear_top_distillation(a, b, tv.cuda(), ti.cuda(), reduction="none"), x, w, torch.ones(M), "none")
    qtol = 2.0 ** -19 * (q * q.log().abs()).sum(-1)  # (float32 exponentials and logarithms of q)
    assert ((loss.double().cpu() - o["loss"]).abs() <= o["ltol"] + qtol).all()
    _grad_close(dx, o["dx"], o["dx_tol"] + 2.0 ** -19 * q.sum(-1, keepdim=True) * w.double().abs().amax(0))
    _grad_close(dw, o["dw"], o["dw_tol"] + 2.0 ** -19 * x.double().abs().sum(0))


@gpu
@pytest.mark.parametrize("native", [True, False])
def test_kept_exponentials_give_the_same_gradients(native, monkeypatch):
    """reduction="none": the first backward from what the forward kept, the second from the logits formed again;
    a piece of the tokens at a time nothing is kept."""
    if not native:
        monkeypatch.setattr(vocab, "_native", lambda *xs: None)
    x, w, g = _inputs(300, 72, 700)  # (72: padded copies in both)
    labels = torch.randint(700, (300,), generator=g).cuda()
    up = torch.rand(300, generator=g).cuda()
    a, b = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    loss = vocab.linear_cross_entropy(a, b, labels, reduction="none")
    g1 = torch.autograd.grad(loss, (a, b), up, retain_graph=True)
    g2 = torch.autograd.grad(loss, (a, b), up)
    for p, q in zip(g1, g2):
        assert torch.equal(p, q)
    cut = vocab.linear_cross_entropy(a, b, labels, reduction="none", piece_rows=256)
    assert torch.equal(cut, loss)
    o = _oracle(x, w, _dense(300, 700, labels.cpu()[:, None], torch.ones(300, 1)), 0.0, torch.ones(300).double(), 1.0, up.double().cpu())
    for got in (g1, torch.autograd.grad(cut, (a, b), up)):
        _grad_close(got[0], o["dx"], o["dx_tol"])
        _grad_close(got[1], o["dw"], o["dw_tol"])


def test_kept_sizes_and_phases_are_refused_without_launching():
    lib, p = vocab._lib(), 1 << 20
    base = dict(rows=1000, vocab=50000, width=64, targets=1, hidden=p, weight=p, hidden_stride=64, weight_stride=64, index=p,
                temperature=1.0, reduction=0, loss=p)
    kept = lambda **kw: lib.theseus_vocab_loss_kept_size(ctypes.byref(vocab.LossArgs(**{**base, **kw})))  # noqa: E731
    call = lambda **kw: lib.theseus_vocab_loss(ctypes.byref(vocab.LossArgs(**{**base, **kw})), p, 1 << 40, None)  # noqa: E731
    assert 1000 * 50000 * 2 <= kept() <= 256 << 20
    assert kept(rows=0) == kept(reduction=2) == kept(vocab=200000) == kept(piece_rows=256) == kept(vocab=0) == 0
    assert call(phase=3) == 7 and call(phase=1, reduction=1, kept=p) == 7
    assert call(phase=1) == 3 and call(phase=1, vocab=200000, kept=p) == 1
