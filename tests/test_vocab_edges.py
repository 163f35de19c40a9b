"""The vocabulary operators (theseus.vocab) where calls are unusual: logits of any magnitude, rows far
apart, inputs changed between the call and its backward, traced and forward-mode calls, sizes
past a launch's, gradients of tokens that do not count.
"""
import pytest
import torch

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
