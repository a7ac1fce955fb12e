"""Limits of the categorical-head operators: large weights of the entropy, what the statistics hold, weights and derivatives
that are not numbers or not there."""
import math

import pytest
import torch

from lvd_pg_b200 import _lib, api
from tests.heads_reference import Logprobs, U, assert_within, make_logits
from tests.test_gpu_heads_offsets import within_up_to_the_last_step

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cats", [5, 100, 256, 333, 900, 5000])
@pytest.mark.parametrize("temperature,weight", [(1e-4, 50.0), (1e-3, 1e5), (0.5, 1e9)])
def test_impossible_categories_beside_a_large_weight_of_the_entropy(dtype, cats, temperature, weight):
    """p (log p + H) is 0 where p is, however large the entropy's weight over the temperature."""
    x = make_logits(40, cats, dtype, cats)
    x[:, 1::3] = -math.inf
    x[:, 2] = x[:, 0]
    x[3, 1:] = -math.inf
    leaf = x.requires_grad_()
    entropy = api.token_logprobs(leaf, None, 0, temperature).entropy
    dx, = torch.autograd.grad(entropy, leaf, torch.full_like(entropy, weight))
    want, tol = Logprobs(x, None, 0, temperature).grad(None, torch.full_like(entropy, weight), None, dtype)
    assert (dx[:, 1::3] == 0).all() and (dx[3, 1:] == 0).all()
    within_up_to_the_last_step(dx, want, tol, "gradient")   # fp16: some lie at the end of its range


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cats,rows", [(2, 40), (20, 9000), (256, 40), (333, 40), (900, 40), (5000, 40), (140000, 2)])
@pytest.mark.parametrize("temperature", [1.0, 0.01, 1e-4])
def test_statistics_are_of_the_softmax_itself(dtype, cats, rows, temperature):
    """The largest logit and the sum of exp((x - max) / T), as the header says, from the scores and from evidence: no more than
    the sum's bound, two roundings and a power of two (4 u) beside it, so that max / T + log(sum) is the logarithm of the sum
    of exponentials."""
    x = make_logits(rows, cats, torch.float32, cats, device="cpu")
    x += torch.linspace(-40, 40, rows)[:, None]
    x[0] = -math.inf
    x[rows - 1, 1:] = x[rows - 1, :1]
    x = x.to(dtype).cuda()
    ref = Logprobs(x, None, 0, temperature)
    shift = torch.where(ref.empty, 0.0, ref.x.amax(1))
    want = ((ref.x - shift[:, None]) / temperature).exp().sum(1)
    tol = want * (ref.tol_S + 8 * U)
    stream = torch.cuda.current_stream().cuda_stream
    entropy, stats = torch.empty(rows, device="cuda"), torch.empty(rows, 2, device="cuda")
    _lib.check(_lib.lib().pcb_token_logprobs(x.data_ptr(), DTYPES.index(dtype), rows, cats, cats, temperature, None, 0, 0, None,
                                             entropy.data_ptr(), stats.data_ptr(), None, None, stream))
    assert torch.equal(stats[:, 0], x.float().amax(1))
    assert_within(stats[:, 1], want, tol, "scores")
    for variables in (1, 2):   # [rows / variables, variables, cats]
        out, stats = torch.empty(rows * cats, device="cuda"), torch.empty(rows, 2, device="cuda")
        _lib.check(_lib.lib().pcb_soft_evidence(x.data_ptr(), DTYPES.index(dtype), rows // variables, variables, cats, variables * cats, cats,
                                                None, 0, 0, temperature, out.data_ptr(), stats.data_ptr(), stream))
        assert torch.equal(stats[:, 0], x.float().amax(1))
        assert_within(stats[:, 1], want, tol, "evidence")


def test_forward_mode_derivatives_are_refused():
    """A tangent would be lost without a word: these operators run backwards only."""
    import torch.autograd.forward_ad as forward_ad

    x = torch.randn(3, 4, 64, device="cuda")
    head = api.QuantHead(torch.randn(20, 64, device="cuda"))
    calls = (lambda t: api.token_logprobs(t), lambda t: api.token_logprobs(t[0], top_k=2), lambda t: api.soft_evidence(t), head.logits,
             head.logprobs, head.evidence)
    with forward_ad.dual_level():
        for requires_grad in (False, True):
            primal = x.clone().requires_grad_(requires_grad)
            dual = forward_ad.make_dual(primal, torch.randn_like(x))
            for call in calls:
                with pytest.raises((_lib.PcbError, RuntimeError), match="tangent|gradient"):
                    call(dual)
                with torch.no_grad(), pytest.raises(_lib.PcbError, match="tangent"):
                    call(dual)
        for call in calls:   # without a tangent: as ever
            call(x)


@pytest.mark.parametrize("dtype", DTYPES)
def test_weights_that_are_no_numbers_stay_so(dtype):
    """NaN or an infinite weight makes its group NaN, and nothing beside it."""
    cats, features, group = 20, 150, 32
    w = torch.randn(cats, features, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    clean = api.QuantHead(w, group).weight()
    bad = torch.zeros(cats, features, dtype=torch.bool, device="cuda")
    for n, k, value in ((0, 0, math.nan), (3, 40, math.inf), (4, 149, -math.inf), (19, 95, math.nan)):
        w[n, k] = value
        bad[n, k // group * group:(k // group + 1) * group] = True
    head = api.QuantHead(w, group)
    got = head.weight()
    assert torch.equal(torch.isnan(got), bad) and torch.equal(got[~bad], clean[~bad])
    y = head.logits(torch.ones(2, features, device="cuda"))
    assert torch.equal(torch.isnan(y), bad.any(1).expand(2, cats))


def test_scales_past_the_range_of_their_type():
    """fp32 weights with fp16 scales, which only the C call combines: from 7 * 65520 on the scale is infinite, the group NaN."""
    w = torch.ones(3, 64, device="cuda")
    w[1, 5], w[2, 5] = 7 * 65521.0, 7 * 65503.0
    codes, scales = torch.empty(3, 32, dtype=torch.uint8, device="cuda"), torch.empty(3, 1, dtype=torch.float16, device="cuda")
    _lib.check(_lib.lib().pcb_head_quantize(w.data_ptr(), 0, 3, 64, 64, 2, codes.data_ptr(), scales.data_ptr(),
                                            torch.cuda.current_stream().cuda_stream))
    head = api.QuantHead.from_codes(codes, scales, 64, 64)
    nan = torch.isnan(head.weight()).all(1)
    assert nan.tolist() == [False, True, False] and torch.equal(torch.isnan(head.logits(torch.ones(1, 64, device="cuda")))[0], nan)


@pytest.mark.parametrize("largest", [1e-3, 4e-4, 1e-4, 1e-5, 2e-6, 5e-7, 1.2e-7])
def test_small_weights_of_half_precision(largest):
    """Where max |w| / 7 is subnormal as an fp16 scale, a step of it is up to all of the scale: rounded up, so that no weight
    is cut off or lost.  A weight is off by half a scale at most; above that the scale was rounded down by half a step."""
    cats, features, group = 40, 200, 64
    gen = torch.Generator().manual_seed(7)
    w = ((2 * torch.rand(cats, features, generator=gen) - 1) * largest).half().cuda()
    w[1] = 0
    got = api.QuantHead(w, group).weight().double()
    step = 2.0 ** -24   # of subnormal numbers
    pad = torch.zeros(cats, 4 * group, dtype=torch.float64, device="cuda")
    pad[:, :features] = w.double()
    most = pad.view(cats, 4, group).abs().amax(2)
    scale = (most / 7).repeat_interleave(group, 1)[:, :features]
    small = scale < 2.0 ** -14
    each = torch.where(small, (scale / step).ceil() * step, scale * (1 + 2.0 ** -11))
    tol = torch.where(small, 0.5 * each, (0.5 + 7 * 2.0 ** -11) * each) * (1 + 1e-5)
    assert ((got - w.double()).abs() <= tol).all()
    assert (got[1] == 0).all() and (got[0] != 0).any()


def test_smallest_weights_under_bfloat16_scales():
    """fp32 weights around 1e-38: the scale is subnormal, the weights are kept to half of it."""
    w = ((2 * torch.rand(6, 64, generator=torch.Generator().manual_seed(3)) - 1) * torch.tensor([1e-37, 5e-38, 1e-38, 3e-39, 4e-40, 2e-41])[:, None]).cuda()
    got = api.QuantHead(w, 64).weight().double()
    step = 2.0 ** -133   # of subnormal bf16
    scale = w.double().abs().amax(1, keepdim=True) / 7
    small = scale < 2.0 ** -126
    each = torch.where(small, (scale / step).ceil() * step, scale * (1 + 2.0 ** -8))
    # quotient of fp32 and rounding of max / 7 to fp32: a step of its subnormal numbers each
    tol = torch.where(small, 0.5 * each, (0.5 + 7 * 2.0 ** -8) * each) * (1 + 1e-5) + 8 * 2.0 ** -149
    assert small.sum() >= 4 and ((got - w.double()).abs() <= tol).all()


@pytest.mark.parametrize("dtype", DTYPES[:2])
def test_features_up_to_where_a_groups_sum_ends(dtype):
    """Groups of 128 whose every product is -8 times 3.3e35, the documented end, or of alternating sign: finite sums in any
    order, exact up to the bound of 128 additions, scaled back into range."""
    codes = torch.zeros(20, 192, dtype=torch.uint8, device="cuda")   # code 0: -8
    scales = torch.full((20, 3), 2.0 ** -20, dtype=torch.bfloat16, device="cuda")
    head = api.QuantHead.from_codes(codes, scales, 384, 128)
    x = torch.full((3, 384), 3.3e35)
    x[1, ::2] *= -1
    x[2, 128:] = 0
    x = x.to(dtype).cuda()   # bf16: 3.2976e35
    got = head.logits(x, torch.float32)
    want = (-8.0 * x.double().sum(1) * 2.0 ** -20)[:, None].expand(3, 20)
    spread = 8.0 * x.double().abs().sum(1)[:, None] * 2.0 ** -20
    assert torch.isfinite(got).all() and ((got.double() - want).abs() <= 17 * 24 * 2.0 ** -23 * spread).all()
