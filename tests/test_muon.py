"""theseus.optim.orthogonalize and FusedMuon against float64, and what they refuse.

Tolerances.  Every rounding to float16 is off by at most 2^-11 of the value, r = 2^-11 / sqrt(3) in the mean square.
In a step X' = (a + b A + c A^2) X with singular values s <= 1.21, relative to |X|_F and to first order, the parts that
are rounded weigh at most: X in A = X X^T twice max |b + 2 c s^2| s^2 = 1.76 each, A 1.76, B = a + b A + c A^2 and X beside
it max |B| = 3.44 each: 6.2 r in the mean square.  These errors lie in X's row or column space and grow as X does, so five
steps add up to sqrt(5) 6.2 r = 3.9e-3 of |X|_F; the result's own rounding adds 2^-8 / sqrt(3) = 2.3e-3.  Together 4.5e-3 in
the mean square: TOL = 6e-3 of the whole matrix' norm, and no row or column off by more than 8 times its share.
A single number (one product of a kind, nothing averaged) may be off by sqrt(3) times as much.
"""
import copy
import ctypes
import math
import re
import subprocess
from pathlib import Path

import pytest
import torch

from theseus import optim
from theseus.optim import FusedMuon, orthogonalize

gpu = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "theseus_muon.h"
BF, FP = torch.bfloat16, torch.float32
TOL = 6e-3


def _exact(x, steps=5, coefficients=optim.COEFFICIENTS, eps=1e-7):
    """The polynomials in float64 on the given device."""
    a, b, c = coefficients
    x = x.double()
    x = x / max(float(x.norm()), eps)
    tall = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if tall else x
    for _ in range(steps):
        s = x @ x.t().contiguous()
        x = a * x + (b * s + c * (s @ s)) @ x
    return x.t() if tall else x


def _close(got, want, tol=TOL):
    assert got.shape == want.shape and torch.isfinite(got).all()
    err, norm = got.double() - want, float(want.norm())
    if min(want.shape) < 8:
        tol = tol * math.sqrt(3)
    assert float(err.norm()) <= tol * norm, f"{float(err.norm()) / norm:.2e} of the norm"
    for dim in (0, 1):
        share = norm / math.sqrt(want.shape[1 - dim])
        assert float(err.norm(dim=dim).max()) <= 8 * tol * share, f"a line of dimension {1 - dim}: {float(err.norm(dim=dim).max()) / share:.2e}"


def _gradient(m, n, seed=0, rank=None, noise=.05):
    """Directions of falling strength and noise, as a weight's gradient has them."""
    g = torch.Generator().manual_seed(seed)
    k = min(m, n, 512) if rank is None else rank
    s = torch.arange(1, k + 1).pow(-.5)
    return ((torch.randn(m, k, generator=g) * s) @ torch.randn(k, n, generator=g) + noise * torch.randn(m, n, generator=g)) * 1e-3


# one element, vectors, around a tile and the short path's limits, odd, long, each tile's range
SHAPES = [(1, 1), (1, 7), (7, 1), (3, 5000), (16, 300), (300, 16), (63, 65), (64, 64), (65, 64), (60, 260), (260, 60), (100, 100),
          (128, 128), (127, 2000), (2000, 127), (128, 129), (129, 129), (130, 1000), (1000, 130), (257, 1025), (640, 640),
          (1100, 700), (700, 1100), (1300, 1300), (2100, 512), (512, 2100), (2048, 2048), (150, 9000), (9001, 200), (900, 5000)]


@gpu
@pytest.mark.parametrize("dtype", [FP, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("m,n", SHAPES)
def test_orthogonalize_matches_float64(m, n, dtype):
    print(f"  orth {m}x{n} {dtype}", flush=True)
    x = _gradient(m, n, m + n).to(dtype).cuda()
    got = orthogonalize(x)
    assert got.dtype == BF
    _close(got, _exact(x))


@gpu
@pytest.mark.parametrize("m,n", [(100, 120), (300, 64), (400, 300), (700, 1000)])
@pytest.mark.parametrize("rank", [1, 8])
def test_few_strong_directions(m, n, rank):
    """Rounding noise outside of the directions is not raised with them (485 times in five steps)."""
    print(f"  rank {rank} {m}x{n}", flush=True)
    x = _gradient(m, n, rank, rank, 0.).cuda()
    want = _exact(x)
    got = orthogonalize(x)
    # (each number of the few directions' outer products: correlated errors, not averaged)
    assert float((got.double() - want).norm()) <= math.sqrt(3) * TOL * float(want.norm())


@gpu
@pytest.mark.parametrize("m,n", [(50, 70), (200, 300)])
@pytest.mark.parametrize("steps,coefficients", [(1, optim.COEFFICIENTS), (2, optim.COEFFICIENTS), (3, optim.COEFFICIENTS),
                                                (12, (2.0, -1.5, .5)), (8, (1.875, -1.25, .375))])
def test_steps_and_coefficients(m, n, steps, coefficients):
    """One, two and three steps (the last two differ in what they keep), and converging polynomials (errors of earlier steps die out)."""
    print(f"  {steps} steps of {coefficients} on {m}x{n}", flush=True)
    x = _gradient(m, n, steps).cuda()
    _close(orthogonalize(x, steps=steps, coefficients=coefficients), _exact(x, steps, coefficients))


@gpu
@pytest.mark.parametrize("m,n", [(40, 50), (129, 140)])
def test_scale_invariance_zeros_and_eps(m, n):
    x = _gradient(m, n).cuda()
    ref = orthogonalize(x)
    for k in (-60, -8, 20, 90):  # powers of two change no bit (nor leave the norm's range)
        assert torch.equal(ref, orthogonalize(x * 2.0 ** k, eps=0.0))
    assert (orthogonalize(torch.zeros_like(x)) == 0).all()
    small = x * (1e-9 / float(x.norm()))  # below eps: X_0 = x / eps
    _close(orthogonalize(small), _exact(small))
    _close(orthogonalize(small, eps=1e-12), _exact(small, eps=1e-12))


@gpu
@pytest.mark.parametrize("m,n", [(40, 50), (129, 140)])
def test_tiny_norms_without_eps(m, n):
    """Norms below 1e-30 count as 1e-30: no factor beyond float32, and zeros stay zeros."""
    x = _gradient(m, n).cuda()
    assert (orthogonalize(torch.zeros_like(x), eps=0.0) == 0).all()
    for norm in (1e-28, 1e-33):
        tiny = x * (norm / float(x.norm()))
        _close(orthogonalize(tiny, eps=0.0), _exact(tiny, eps=1e-30))


@gpu
@pytest.mark.parametrize("m,n", [(40, 50), (300, 200)])
def test_values_that_are_not_finite_make_their_matrix_nan(m, n):
    xs = [_gradient(m, n, i).cuda() for i in range(3)]
    want = orthogonalize(xs)
    for bad in (math.nan, math.inf, -math.inf):
        ys = [x.clone() for x in xs]
        ys[1][m - 1, n - 1] = bad
        got = orthogonalize(ys)
        assert torch.isnan(got[1]).all() and torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])


@gpu
def test_batches_lists_strides():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 3, 70, 90, generator=g).cuda()
    got = orthogonalize(x)
    assert got.shape == x.shape and got.is_contiguous()
    for i in range(2):
        for j in range(3):
            _close(got[i, j], _exact(x[i, j]))
    big = torch.randn(300, 401, generator=g).bfloat16().cuda()
    views = [big[:, 3:150], big[1::2, 5:396], big.t(), big[:, ::3], big[7:8], big[:, 9:10], big[:1].expand(30, 401), big[:90, 1:2].expand(90, 50)]
    for v, o, c in zip(views, orthogonalize(views), orthogonalize([v.contiguous() for v in views])):
        assert o.shape == v.shape
        _close(o, _exact(v), 4 * TOL if 0 in v.stride() else TOL)  # (expanded: rank one)
        assert torch.equal(o, c)
    mixed = [torch.randn(33, 20, generator=g).cuda(), torch.randn(200, 180, generator=g).bfloat16().cuda(), torch.empty(0, 5, device="cuda"),
             torch.randn(2, 40, 40, generator=g).cuda(), torch.empty(3, 0, 4, device="cuda")]
    out = orthogonalize(mixed)
    assert [o.shape for o in out] == [t.shape for t in mixed] and all(o.dtype == BF for o in out)
    _close(out[0], _exact(mixed[0])), _close(out[1], _exact(mixed[1])), _close(out[3][1], _exact(mixed[3][1]))
    assert orthogonalize([]) == [] and orthogonalize(torch.empty(4, 0, device="cuda")).shape == (4, 0)
    wide = torch.randn(5, (1 << 21) + 9, generator=g).bfloat16().cuda()[:, :100]  # rows too far apart: copied
    _close(orthogonalize(wide), _exact(wide))


@gpu
def test_many_matrices_share_launches():
    """More than a launch's list takes, every matrix alike: mirrored tiles of neighbours, two workgroups on a CU."""
    for shape, count in (((768, 768), 9), ((70, 64), 70), ((200, 130), 40), ((128, 700), 33)):
        print(f"  {count} of {shape}", flush=True)
        xs = torch.stack([_gradient(*shape, seed) for seed in range(4)]).cuda()
        got = orthogonalize([xs[i % 4] for i in range(count)])
        for i in range(4):
            _close(got[i], _exact(xs[i]))
        for i in range(4, count):
            assert torch.equal(got[i], got[i % 4]), i


@gpu
def test_a_layer_of_full_width():
    """The largest tiles, rounds of them and the last one in quarters, low-rank factors beside: 5120 wide."""
    shapes = [(5120, 5120)] * 2 + [(5120, 192), (192, 5120), (5120, 352), (352, 5120)]
    g = torch.Generator(device="cuda").manual_seed(0)
    xs = []
    for m, n in shapes:
        s = torch.arange(1, 193, device="cuda").pow(-.5)
        xs.append((torch.randn(m, 192, generator=g, device="cuda") * s) @ torch.randn(192, n, generator=g, device="cuda")
                  + .05 * torch.randn(m, n, generator=g, device="cuda"))
    print("  layer of 5120", flush=True)
    for x, o in zip(xs, orthogonalize(xs)):
        _close(o, _exact(x))


@gpu
def test_same_bits_every_time_other_streams_and_graphs():
    for shape in ((64, 100), (128, 3000), (300, 500)):
        print(f"  graph {shape}", flush=True)
        x = _gradient(*shape).cuda()
        want = orthogonalize(x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            again = orthogonalize(x)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert torch.equal(want, again)
        held = x.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = orthogonalize(held)
        for seed in range(3):
            held.copy_(_gradient(*shape, seed + 5))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, orthogonalize(held))
        del graph


@gpu
@pytest.mark.parametrize("wide", [False, True])
def test_offsets_past_32_bits(wide):
    """131072 x 17000 (4.5 GB): row i has its one in column i mod 17000, so the columns are orthogonal and
    each is scaled by itself.  And its transposed matrix."""
    m, n = 131072, 17000
    print(f"  orth {m}x{n}", flush=True)
    x = torch.zeros(m, n, dtype=BF, device="cuda")
    rows = torch.arange(m, device="cuda")
    x[rows, rows % n] = 1.0
    if wide:
        x = x.t().contiguous()
    out = orthogonalize(x)
    out = out.t() if wide else out
    got = out[rows, rows % n].double()
    ones = torch.bincount(rows % n).double()
    s = ones.sqrt() / math.sqrt(m)
    for _ in range(5):
        s = optim.COEFFICIENTS[0] * s + optim.COEFFICIENTS[1] * s ** 3 + optim.COEFFICIENTS[2] * s ** 5
    want = (s / ones.sqrt())[rows % n]
    # (equal numbers: nothing is averaged)
    assert float(((got - want) / want).abs().max()) <= math.sqrt(3) * 2 * TOL
    out[rows, rows % n] = 0
    assert float(out.abs().max()) <= 1e-6  # (products of zeros and ones: exact, but for second halves)


# ------------------------------------------------------------------------------ the optimizer
def _size(shape, scale):
    return math.sqrt(max(1.0, shape[0] / shape[1])) if scale == "shape" else .2 * math.sqrt(max(shape))


def _step64(p, g, buf, lr, wd, mu, nesterov, scale, factor=1.0):
    g = g.double() * factor
    buf = mu * buf + (1 - mu) * g
    u = mu * buf + (1 - mu) * g if nesterov else buf
    step = lr * _size(p.shape, scale) * _exact(u)
    return p * (1 - lr * wd) - step, buf, step


def _params_close(p, want, step, what):
    """The step's error, and float32 roundings of p keep and of the difference (2^-24 of p each, and of what is subtracted)."""
    tol = TOL * (math.sqrt(3) if min(want.shape) < 8 else 1) * float(step.norm()) + 3 * 2.0 ** -24 * float(want.norm())
    err = float((p.detach().double() - want).norm())
    assert err <= tol, f"{what}: {err / tol:.2f} of the bound"


MATRICES = [(96, 96), (40, 256), (256, 40), (1, 33), (33, 1), (300, 257)]


@gpu
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("scale", ["shape", "rms"])
@pytest.mark.parametrize("shapes", [MATRICES, [(64, 64), (20, 100), (128, 50)], [(64, 700), (901, 128), (33, 20), (300, 61)]],
                         ids=["any", "short", "long and short"])
def test_three_steps_match_float64(shapes, scale, nesterov):
    lr, wd, mu = .02, .1, .9
    g = torch.Generator().manual_seed(1)
    ps = [torch.randn(s, generator=g).cuda().requires_grad_() for s in shapes]
    idle = torch.randn(5, 5, device="cuda", requires_grad=True)  # no gradient: left alone
    kept = idle.detach().clone()
    opt = FusedMuon([{"params": ps[:2]}, {"params": ps[2:] + [idle], "lr": lr / 2, "weight_decay": 0.0}], lr=lr, weight_decay=wd, momentum=mu,
                    nesterov=nesterov, scale=scale)
    bufs = [torch.zeros(s, dtype=torch.float64, device="cuda") for s in shapes]
    for t in range(3):
        print(f"  step {t} {scale} {nesterov}", flush=True)
        old = [p.detach().double() for p in ps]
        for i, (p, s) in enumerate(zip(ps, shapes)):
            p.grad = _gradient(*s, seed=10 * t + i).cuda()
        opt.step()
        for i, p in enumerate(ps):
            l, w = (lr, wd) if i < 2 else (lr / 2, 0.0)
            want, bufs[i], step = _step64(old[i], p.grad, bufs[i], l, w, mu, nesterov, scale)
            _params_close(p, want, step, f"param {i} step {t}")
            got = opt.state[p]["momentum_buffer"]
            assert float((got.double() - bufs[i]).norm()) <= 3 * (t + 1) * 2.0 ** -24 * float(bufs[i].norm()) + 1e-30
    assert torch.equal(idle.detach(), kept) and not opt.state[idle]


@gpu
@pytest.mark.parametrize("shapes", [MATRICES, [(64, 64), (20, 100)], [(64, 700), (901, 128)]], ids=["any", "short", "long and short"])
def test_step_after_backward_scales_clips_and_raises(shapes):
    def fresh(seed=0):
        g = torch.Generator().manual_seed(seed)
        ps = [torch.randn(s, generator=g).cuda().requires_grad_() for s in shapes]
        for i, p in enumerate(ps):
            p.grad = _gradient(*p.shape, seed=i).cuda()
        opt = FusedMuon(ps, lr=.02, weight_decay=.1, momentum=.9)
        for i, p in enumerate(ps):
            opt.state[p]["momentum_buffer"] = _gradient(*p.shape, seed=20 + i).cuda()
        return ps, opt
    for scale, clip in ((3 / 7, None), (.5, 1e9), (2.0, .01), (1.0, math.inf)):
        ps, opt = fresh()
        old, bufs = [p.detach().double() for p in ps], [opt.state[p]["momentum_buffer"].double() for p in ps]
        norm = opt.step_after_backward(grad_scale=scale, max_norm=clip)
        want = math.sqrt(sum(float((p.grad.double() * scale).square().sum()) for p in ps))
        factor = scale
        if clip is None:
            assert norm is None
        else:
            assert abs(float(norm) - want) <= 1e-6 * want
            factor = scale * min(1.0, clip / (want + 1e-6))
        for i, p in enumerate(ps):
            new, buf, step = _step64(old[i], p.grad, bufs[i], .02, .1, .9, True, "shape", factor)
            _params_close(p, new, step, f"{scale} {clip} param {i}")
            assert float((opt.state[p]["momentum_buffer"].double() - buf).norm()) <= 1e-6 * float(buf.norm())
    # a norm that is not finite: raises and changes nothing, or goes through
    ps, opt = fresh()
    ps[0].grad[0, 0] = math.nan
    old, bufs = [p.detach().clone() for p in ps], [opt.state[p]["momentum_buffer"].clone() for p in ps]
    with pytest.raises(RuntimeError, match="non-finite"):
        opt.step_after_backward(max_norm=1.0)
    assert all(torch.equal(a, p.detach()) and torch.equal(b, opt.state[p]["momentum_buffer"]) for a, b, p in zip(old, bufs, ps))
    opt.step_after_backward(max_norm=1.0, error_if_nonfinite=False)
    assert all(torch.isnan(p).all() for p in ps)


@gpu
@pytest.mark.parametrize("limit", [-1.0, -math.inf, math.nan])
@pytest.mark.parametrize("shapes", [[(64, 64), (20, 100)], [(64, 700), (901, 128)], [(300, 257)]], ids=["whole", "short", "long"])
def test_limits_that_are_none(shapes, limit):
    """A negative max_norm or NaN: no norm and no clipping, as FusedAdamW, with NaN for the norm and no error."""
    def fresh(cls):
        ps = [_gradient(*s, seed=9).cuda().requires_grad_() for s in shapes]
        for i, p in enumerate(ps):
            p.grad = _gradient(*p.shape, seed=i).cuda()
        return ps, cls(ps, lr=.02)
    want, opt = fresh(FusedMuon)
    opt.step_after_backward(grad_scale=.5)
    for old in (0.0, 1.0):  # (what the memory of the result may hold)
        for cls in (FusedMuon, optim.FusedAdamW):
            ps, opt = fresh(cls)
            held = [torch.full((3,), old, device="cuda") for _ in range(8)]
            del held
            norm = opt.step_after_backward(grad_scale=.5, max_norm=limit)
            assert math.isnan(norm)
            assert cls is not FusedMuon or all(torch.equal(p, q) for p, q in zip(ps, want))


@gpu
def test_parameters_without_elements_have_a_norm():
    """FusedAdamW's result for them: 0."""
    for cls in (FusedMuon, optim.FusedAdamW):
        ps = [torch.nn.Parameter(torch.zeros(s, device="cuda")) for s in ((0, 5), (4, 0))]
        for p in ps:
            p.grad = torch.zeros_like(p)
        opt = cls(ps, lr=.02)
        assert float(opt.step_after_backward(max_norm=1.0)) == 0.0
        assert opt.step_after_backward() is None
        assert math.isnan(opt.step_after_backward(max_norm=-1.0))


@gpu
@pytest.mark.parametrize("shapes", [[(8 + 3 * i, 1 + 37 * i % 700) for i in range(40)], [(20 + 9 * i, 30 + 53 * i % 300) for i in range(40)]],
                         ids=["short", "long and short"])
def test_a_step_of_more_matrices_than_a_launch_takes(shapes):
    """One norm and clip factor over two sets of launches, which share the workspace; one that is not finite behind the first set."""
    assert len(shapes) > 32
    g = torch.Generator().manual_seed(0)
    ps = [torch.randn(s, generator=g).cuda().requires_grad_() for s in shapes]
    for i, p in enumerate(ps):
        p.grad = _gradient(*p.shape, seed=i).cuda()
    opt = FusedMuon(ps, lr=.02, weight_decay=.1, momentum=.9)
    for i, p in enumerate(ps):
        opt.state[p]["momentum_buffer"] = _gradient(*p.shape, seed=50 + i).cuda()
    held = lambda: [t.detach().clone() for p in ps for t in (p, opt.state[p]["momentum_buffer"])]  # noqa: E731
    old = [(p.detach().double(), opt.state[p]["momentum_buffer"].double()) for p in ps]
    want = math.sqrt(sum(float(p.grad.double().square().sum()) for p in ps))
    clip = .3 * want
    norm = opt.step_after_backward(max_norm=clip)
    assert abs(float(norm) - want) <= 1e-6 * want
    for i, (p, (w, b)) in enumerate(zip(ps, old)):
        new, buf, step = _step64(w, p.grad, b, .02, .1, .9, True, "shape", clip / (want + 1e-6))
        _params_close(p, new, step, f"param {i}")
        assert float((opt.state[p]["momentum_buffer"].double() - buf).norm()) <= 1e-6 * float(buf.norm())
    ps[35].grad[3, 0] = math.nan
    before = held()
    with pytest.raises(RuntimeError, match="non-finite"):
        opt.step_after_backward(max_norm=clip)
    assert all(torch.equal(a, b) for a, b in zip(before, held()))
    opt.step_after_backward(max_norm=clip, error_if_nonfinite=False)
    assert all(torch.isnan(p).all() for p in ps)


@gpu
@pytest.mark.parametrize("clip", [False, True])
@pytest.mark.parametrize("shapes", [[(64, 64), (20, 100)], [(64, 700), (901, 128)], [(300, 257), (40, 60)]], ids=["whole", "short", "long"])
def test_a_captured_step_runs_again(shapes, clip):
    """Every replay steps parameters and momentum on, from the gradients that are then in place: the eager steps' bits."""
    def fresh():
        ps = [_gradient(*s, seed=9).cuda().requires_grad_() for s in shapes]
        for p in ps:
            p.grad = torch.zeros_like(p)
        return ps, FusedMuon(ps, lr=.02, momentum=.9)

    def step(opt):
        if clip:
            return opt.step_after_backward(grad_scale=.5, max_norm=1e-3, error_if_nonfinite=False)
        opt.step()

    (ps, opt), (qs, other) = fresh(), fresh()
    for o in (opt, other):  # (the momentum's memory, outside of the capture)
        step(o)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = step(opt)
    for n in range(4):
        for i, (p, q) in enumerate(zip(ps, qs)):
            p.grad.copy_(_gradient(*p.shape, seed=10 * n + i))
            q.grad.copy_(p.grad)
        graph.replay()
        torch.cuda.synchronize()
        want = step(other)
        assert not clip or torch.equal(norm, want)
        for p, q in zip(ps, qs):
            assert torch.equal(p, q) and torch.equal(opt.state[p]["momentum_buffer"], other.state[q]["momentum_buffer"])
    del graph, norm


@gpu
def test_state_dict_and_scheduler():
    g = torch.Generator().manual_seed(0)
    make = lambda: [torch.randn(s, generator=torch.Generator().manual_seed(5)).cuda().requires_grad_() for s in ((50, 60), (200, 140))]  # noqa: E731
    a, b = make(), make()
    oa, ob = FusedMuon(a, lr=.01), FusedMuon(b, lr=.5)
    grads = [[torch.randn(p.shape, generator=g).cuda() for p in a] for _ in range(2)]
    for p, q in zip(a, grads[0]):
        p.grad = q.clone()
    sa = torch.optim.lr_scheduler.StepLR(oa, 1, .1)
    oa.step()
    ob.load_state_dict(copy.deepcopy(oa.state_dict()))  # (as a file holds it: its own tensors)
    with torch.no_grad():
        for p, q in zip(a, b):
            q.copy_(p)
    sa.step()
    ob.param_groups[0]["lr"] = oa.param_groups[0]["lr"]
    assert abs(oa.param_groups[0]["lr"] - .001) < 1e-12
    for ps in (a, b):
        for p, q in zip(ps, grads[1]):
            p.grad = q.clone()
    oa.step(), ob.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert oa.step(lambda: 7.0) == 7.0


@gpu
def test_traces_and_forward_mode_are_refused():
    """Where the bare kernels would leave nothing behind, or drop the tangent."""
    x = _gradient(30, 40).cuda()
    call = lambda t: orthogonalize(t)  # noqa: E731
    with pytest.raises(RuntimeError, match="theseus_muon: orthogonalize has no"):
        torch.jit.trace(call, (x,), check_trace=False)
    with pytest.raises(RuntimeError, match="theseus_muon: orthogonalize has no"):
        torch.func.vmap(call)(x[None])
    with pytest.raises(RuntimeError, match="theseus_muon: orthogonalize has no"):
        with torch.autograd.forward_ad.dual_level():
            orthogonalize([torch.autograd.forward_ad.make_dual(x, x)])
    assert orthogonalize(x.clone().requires_grad_()).requires_grad is False


@gpu
def test_refusals_on_the_gpu():
    w = torch.zeros(4, 4, device="cuda")
    for x, error, match in [(w.half(), TypeError, "bfloat16 or float32"), (w[0], ValueError, "m, n"), ([w, w.cpu()], ValueError, "CUDA"),
                            (w[:1, :1].expand((1 << 17) + 1, 4), ValueError, "2\\^17"), (w.long(), TypeError, "bfloat16")]:
        with pytest.raises(error, match=match):
            orthogonalize(x)
    for kw in (dict(steps=0), dict(steps=101), dict(eps=-1.0), dict(eps=math.nan), dict(coefficients=(1.0, 2.0)), dict(coefficients=(math.nan, 0., 0.))):
        with pytest.raises(ValueError):
            orthogonalize(w, **kw)

    def step(p, grad=None, **kw):
        opt = FusedMuon([p] if not isinstance(p, list) else p, **kw)
        for q in opt.param_groups[0]["params"]:
            q.grad = torch.ones_like(q) if grad is None else grad
        opt.step()
    P = torch.nn.Parameter
    with pytest.raises(RuntimeError, match="float32"):
        step(P(w.bfloat16()))
    with pytest.raises(RuntimeError, match="contiguous float32 CUDA"):
        step(P(torch.zeros(4, 6, device="cuda").t()))
    with pytest.raises(RuntimeError, match="gradients"):
        step(P(w.clone()), torch.zeros(4, 8, device="cuda")[:, ::2])
    opt = FusedMuon([{"params": [P(w.clone())]}, {"params": [P(w.clone())], "momentum": .5}])
    for gr in opt.param_groups:
        gr["params"][0].grad = torch.ones(4, 4, device="cuda")
    with pytest.raises(ValueError, match="share"):
        opt.step()


# ------------------------------------------------------------------------------ CPU
def test_muon_header_symbols_are_exported():
    lib = optim._lib()
    names = set(re.findall(r"\b(theseus_\w+)\s*\(", HEADER.read_text()))
    assert names == {"theseus_orthogonalize_workspace_size", "theseus_orthogonalize", "theseus_muon_workspace_size", "theseus_muon_step"}
    for n in names:
        assert hasattr(lib, n)


@pytest.mark.parametrize("cls,name", [(optim._Orth, "theseus_orthogonalize_matrix"), (optim._Matrix, "theseus_muon_matrix"),
                                      (optim._Schulz, "theseus_newton_schulz")])
def test_ctypes_structs_match_the_c_layout(tmp_path, cls, name):
    src, exe, fields = tmp_path / "layout.c", tmp_path / "layout", [f[0] for f in cls._fields_]
    src.write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"theseus_muon.h\"\nint main(void){\n"
                   + "".join(f'printf("%zu\\n", offsetof({name}, {f}));\n' for f in fields)
                   + f'printf("%zu\\n", sizeof({name}));\nreturn 0;}}\n')
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(cls, f).offset for f in fields] + [ctypes.sizeof(cls)]


def test_muon_abi_rejects_bad_arguments_before_launching():
    lib, p = optim._lib(), 4096
    ns = optim._Schulz(5, 3.4, -4.7, 2.0, 1e-7)
    orth = lambda x=p, out=p, ld=64, m=200, n=64, dt=1, count=1, ns=ns, ws=p, size=0: lib.theseus_orthogonalize(  # noqa: E731
        (optim._Orth * 1)(optim._Orth(x, out, ld, m, n, dt)), count, ctypes.byref(ns), ws, size, None)
    # (status codes of theseus_wkv7.h: 1 shape, 2 type, 3 null pointer, 4 workspace)
    for kw in (dict(m=-1), dict(n=-1), dict(m=(1 << 17) + 1), dict(n=(1 << 17) + 1), dict(ld=63), dict(ld=(1 << 21) + 1), dict(count=-1)):
        assert orth(**kw) == 1
    assert orth(dt=2) == orth(dt=-1) == 2 and orth(x=None) == orth(out=None) == 3
    assert orth() == 4 and orth(ws=None, size=1 << 40) == 4 and orth(m=0) == 0 and orth(count=0) == 0
    for bad in (optim._Schulz(0, 1, 1, 1, 0), optim._Schulz(101, 1, 1, 1, 0), optim._Schulz(5, math.nan, 1, 1, 0), optim._Schulz(5, 1, math.inf, 1, 0),
                optim._Schulz(5, 1, 1, 1, -1), optim._Schulz(5, 1, 1, 1, math.nan)):
        assert orth(ns=bad) == 1
    assert lib.theseus_orthogonalize(None, 1, ctypes.byref(ns), p, 0, None) == 3
    step = lambda param=p, grad=p, mom=p, m=64, n=64, norm=-1.0, res=p, ws=p, size=0: lib.theseus_muon_step(  # noqa: E731
        (optim._Matrix * 1)(optim._Matrix(param, grad, mom, m, n, 1.0, .1)), 1, ctypes.byref(ns), .9, 1, 1.0, norm, 0, res, ws, size, None)
    assert step(m=-1) == 1 and step(n=(1 << 17) + 1) == 1
    assert step(param=None) == step(grad=None) == step(mom=None) == step(norm=1.0, res=None) == 3
    assert step() == 4 and step(m=0) == 0
    sizes = [lib.theseus_muon_workspace_size((optim._Matrix * 1)(optim._Matrix(p, p, p, m, m, 1.0, .1)), 1) for m in (1, 64, 129, 512, 5120)]
    assert sizes == sorted(sizes) and sizes[0] > 0


@pytest.mark.parametrize("steps,coefficients,fine", [
    (100, optim.COEFFICIENTS, True), (100, (2.0, -1.5, .5), True), (100, (1.5, -.5, 0.0), True), (5, (1.0, 0.0, 0.0), True),
    (1, (30.0, 0.0, 0.0), True), (2, (30.0, 0.0, 0.0), False), (1, (40.0, 0.0, 0.0), False), (2, (2.9, 0.0, 0.0), True), (3, (2.0, 0.0, 0.0), False),
    (2, (.3, 0.0, 0.0), True), (3, (.3, 0.0, 0.0), False), (5, (8.28721, -23.5959, 17.3004), False), (5, (-3.4445, 4.7750, -2.0315), True)])
def test_coefficients_that_leave_the_range_are_refused(steps, coefficients, fine):
    """a s alone multiplies the largest singular value by a; the others' growth was followed on a fine grid."""
    for call in (lambda: orthogonalize([], steps=steps, coefficients=coefficients),
                 lambda: FusedMuon([torch.nn.Parameter(torch.zeros(3, 3))], steps=steps, coefficients=coefficients)):
        if fine:
            call()
        else:
            with pytest.raises(ValueError, match="float16's range"):
                call()


def test_constructor_validates():
    p = [torch.nn.Parameter(torch.zeros(3, 3))]
    for bad in (dict(lr=-1.0), dict(weight_decay=-.1), dict(momentum=1.0), dict(momentum=-.1), dict(steps=0), dict(eps=-1.0),
                dict(scale="other"), dict(coefficients=(1.0,))):
        with pytest.raises(ValueError):
            FusedMuon(p, **bad)
    for shape in ((3,), (2, 3, 4), ()):
        with pytest.raises(ValueError, match="matrices"):
            FusedMuon([torch.nn.Parameter(torch.zeros(shape))])
    with pytest.raises(ValueError, match="CUDA"):
        orthogonalize(torch.zeros(3, 3))
    opt = FusedMuon(p)
    p[0].grad = torch.zeros(3, 3)
    with pytest.raises(RuntimeError, match="CUDA"):
        opt.step()
