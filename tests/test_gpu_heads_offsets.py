"""Rows whose largest logit over the temperature lies far from zero, as masks of -1e10 or -1e20 throughout leave them: the
powers of a row count from its maximum, wherever that is.  Every operator that is made of logits, in every form of its kernels."""
import pytest
import torch

from lvd_pg_b200 import api
from tests import test_gpu_soft_evidence, test_gpu_token_logprobs
from tests.heads_reference import assert_within, make_logits
from tests.test_gpu_soft_evidence import _check as check_evidence
from tests.test_gpu_token_logprobs import _check as check_logprobs, _tokens

pytestmark = pytest.mark.gpu
WIDE = [torch.float32, torch.bfloat16]
FILLS = [2e9, -2e9, 5e9, -1e10, -1.0014e10, 1e12, -1e12, -1e20, 1e28, -1e28]


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("offset", [700.0, -9000.0, 60000.0, 4e5])
@pytest.mark.parametrize("rows,cats", [(55, 8), (400, 30), (60, 256), (55, 333), (51, 900), (50, 4100), (12, 70000), (700, 4099), (2400, 1501)])
def test_ordinary_rows_with_an_offset(dtype, offset, rows, cats):
    """Values some steps of the type apart, at temperatures of some steps: the parts of a row, which have maxima of their own,
    are joined as exactly as their powers are formed."""
    step = torch.finfo(dtype).eps * abs(offset)
    x = (offset + step * make_logits(rows, cats, torch.float32, cats, device="cpu").double()).to(dtype).cuda()
    for temperature in (max(1.0, step), 4 * max(1.0, step)):
        check_logprobs(x, _tokens(rows, cats), min(4, cats), temperature)
    check_evidence(x.view(rows // 2, 2, cats) if rows % 2 == 0 else x.view(rows, 1, cats), None, max(1.0, step))


def _rows(rows, cats, dtype, seed):
    """By turns: one value throughout, the same with an entry or two a few steps of the type above it, an ordinary row with that
    value (or its negative) in every third place, ordinary rows, and one large logit among zeros."""
    x = make_logits(rows, cats, torch.float32, seed, device="cpu")
    eps = torch.finfo(dtype).eps
    for r in range(rows):
        fill, kind = FILLS[r // 5 % len(FILLS)], r % 5
        if kind == 0:
            x[r] = fill
        elif kind == 1:
            x[r] = fill
            x[r, cats - 1] = fill + 2 * eps * abs(fill)
            x[r, cats // 2] = fill + 4 * eps * abs(fill)
        elif kind == 2:
            x[r, ::3] = -abs(fill)
        elif kind == 3:
            x[r] = 0.0
            x[r, cats // 3] = abs(fill)
    return x.to(dtype).cuda()


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("temperature", [1.0, 1e4, 1e-3, 1e-7, 3e8])
@pytest.mark.parametrize("rows,cats", [(55, 8), (400, 30), (60, 256), (55, 333), (51, 900), (50, 4100), (52, 70000), (700, 4099), (2400, 1501)])
def test_scores(dtype, temperature, rows, cats):
    check_logprobs(_rows(rows, cats, dtype, cats), _tokens(rows, cats), min(4, cats), temperature)


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("temperature", [1.0, 1e4, 1e-7])
@pytest.mark.parametrize("rows,variables,cats", [(26, 10, 2), (30, 11, 20), (33, 4, 100), (25, 4, 256), (40, 3, 333), (30, 4, 700), (52, 1, 3001)])
def test_evidence(dtype, temperature, rows, variables, cats):
    check_evidence(_rows(rows * variables, cats, dtype, cats).view(rows, variables, cats), None, temperature)


def within_up_to_the_last_step(got, want, tol, what=""):
    """`assert_within`, but for the end of the type's range: the largest number is (2 - eps) 2^e with steps of eps 2^e, so that
    values up to half a step above it round to it, not to infinity (fp16: 65504 up to 65520)."""
    f = torch.finfo(got.dtype)
    half_step = f.max / (2 - f.eps) * f.eps / 2
    want = torch.where((want.abs() > f.max) & (want.abs() < f.max + half_step), want.sign() * f.max, want)
    assert_within(got, want, tol, what)


@pytest.mark.parametrize("cats", [9, 300, 3000, 40000])
@pytest.mark.parametrize("temperature", [1e-5, 1e-7])
def test_half_precision_at_low_temperatures(cats, temperature, monkeypatch):
    for module in (test_gpu_soft_evidence, test_gpu_token_logprobs):   # gradients of 1 / T pass the range of fp16
        monkeypatch.setattr(module, "assert_within", within_up_to_the_last_step)
    x = make_logits(8, cats, torch.float32, cats, device="cpu")
    x[0], x[1], x[2], x[3] = 65504, -65504, 4000, -60000
    x[2, 1::2], x[2, 0], x[3, cats // 2] = 3999, 3998, -59968
    x[4] += 6000
    x[5, ::2] = -65504
    x = x.half().cuda()
    check_logprobs(x, _tokens(8, cats), 3, temperature)
    check_evidence(x.view(4, 2, cats), None, temperature)


@pytest.mark.parametrize("dtype", WIDE)
@pytest.mark.parametrize("cats", [7, 200, 4100, 70000])
def test_rows_of_no_weight_in_the_loss(dtype, cats):
    """A padded row has an upstream gradient of 0: its logits' gradient is 0, whatever fills it."""
    x = torch.stack([torch.full((cats,), fill) for fill in FILLS]).to(dtype).cuda().requires_grad_()
    out = api.token_logprobs(x, torch.zeros(len(FILLS), dtype=torch.int64, device="cuda"), 2)
    zero = torch.zeros_like(out.logp)
    dx, = torch.autograd.grad([out.logp, out.entropy, out.top_logp], x, [zero, zero, torch.zeros_like(out.top_logp)])
    assert (dx == 0).all()
    y = x.detach().view(5, 2, cats).requires_grad_()
    evidence = api.soft_evidence(y)
    assert (torch.autograd.grad(evidence, y, torch.zeros_like(evidence))[0] == 0).all()
