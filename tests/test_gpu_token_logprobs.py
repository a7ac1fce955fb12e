"""Log-probabilities, entropy, alternatives and their gradient against the formulas in 64 bits."""
import math

import pytest
import torch

from lvd_pg_b200 import _lib, api
from tests.heads_reference import Logprobs, assert_within, make_logits

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
LOWEST = {t: torch.finfo(t).min for t in DTYPES}


def _tokens(rows, cats, seed=0):
    gen = torch.Generator().manual_seed(seed)
    t = torch.randint(0, cats, (rows,), generator=gen)
    t[::7] = -1
    return t.cuda()


def _check(x, tokens, top_k, temperature=1.0, grads=(1, 1, 1)):
    """Forward and gradient of a [rows, cats] view."""
    ref = Logprobs(x, tokens, top_k, temperature)
    leaf = x.detach().requires_grad_()
    out = api.token_logprobs(leaf, tokens, top_k, temperature)
    quiet = api.token_logprobs(x.detach(), tokens, top_k, temperature)
    for a, b in zip(out, quiet):
        assert (a is None) == (b is None) and (a is None or torch.equal(a.detach().nan_to_num(nan=7.0), b.nan_to_num(nan=7.0)))
    assert_within(out.entropy, ref.entropy, ref.tol_entropy, "entropy")
    if tokens is not None:
        assert_within(out.logp, ref.logp, ref.tol_logp, "logp")
    if top_k:
        assert torch.equal(out.top_ids, ref.top_ids)
        assert_within(out.top_logp, ref.top_logp, ref.tol_top, "top_logp")
    gen = torch.Generator().manual_seed(5)
    rows = x.shape[0]
    g_logp = torch.randn(rows, generator=gen).cuda() if grads[0] and tokens is not None else None
    g_entropy = torch.randn(rows, generator=gen).cuda() if grads[1] else None
    g_top = torch.randn(rows, top_k, generator=gen).cuda() if grads[2] and top_k else None
    pairs = [(o, g) for o, g in ((out.logp, g_logp), (out.entropy, g_entropy), (out.top_logp, g_top)) if g is not None]
    if not pairs:
        return out
    dx, = torch.autograd.grad([o for o, _ in pairs], leaf, [g for _, g in pairs])
    want, tol = ref.grad(g_logp, g_entropy, g_top, x.dtype)
    assert dx.dtype == x.dtype
    assert_within(dx, want, tol, "gradient")
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cats,top_k,temperature", [
    (1, 1, 1, 1.0), (5, 2, 0, 0.7), (33, 2, 2, 1.0), (7, 3, 3, 2.0), (64, 31, 5, 1.0), (9, 32, 32, 1.3), (17, 33, 1, 1.0),
    (40, 200, 4, 1.0), (513, 256, 1, 1.0), (3, 257, 20, 0.5), (12, 1000, 7, 1.0), (5, 1024, 32, 1.0), (4, 1025, 20, 1.0),
    (300, 1500, 8, 0.8), (2, 4099, 32, 1.0), (700, 4096, 3, 1.0), (1, 32000, 20, 1.0), (3, 50021, 5, 0.8), (2, 131072, 20, 1.0),
    (1, 262147, 32, 1.0), (1, 1000003, 4, 1.0), (2500, 1999, 5, 1.0), (700, 33001, 6, 0.9), (2400, 5000, 2, 1.0),
    (40000, 7, 3, 1.0), (9000, 63, 2, 1.0), (5000, 333, 12, 1.0), (30000, 128, 1, 1.0), (160, 9000, 32, 1.0)])
def test_shapes(dtype, rows, cats, top_k, temperature):
    _check(make_logits(rows, cats, dtype, rows + cats), _tokens(rows, cats), top_k, temperature)


@pytest.mark.parametrize("grads", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 0, 0)])
@pytest.mark.parametrize("rows,cats", [(6, 40), (3, 5000)])
def test_parts_of_the_gradient(rows, cats, grads):
    _check(make_logits(rows, cats, torch.float32, 3), _tokens(rows, cats), 5, 0.9, grads)
    _check(make_logits(rows, cats, torch.bfloat16, 4), None, 5, 0.9, grads)


def _masked(rows, cats, dtype, seed):
    """Rows: nothing masked, most masked, one left, two equal left, none left; by -inf, by the lowest value, by both."""
    x = make_logits(rows, cats, dtype, seed)
    gen = torch.Generator().manual_seed(seed)
    for r in range(rows):
        kind, fill = r % 5, [-math.inf, LOWEST[dtype]][r // 5 % 2]
        if kind:
            keep = {1: torch.randperm(cats, generator=gen)[:max(1, cats // 10)], 2: torch.tensor([cats - 1]),
                    3: torch.tensor([0, cats // 2]), 4: torch.tensor([], dtype=torch.long)}[kind]
            row = torch.full((cats,), fill, dtype=dtype, device=x.device)
            keep = keep.to(x.device)
            row[keep] = 1.5 if kind == 3 else x[r, keep]
            x[r] = row
    if rows > 10:   # the lowest value among impossible ones: all that is possible
        x[10] = -math.inf
        x[10, cats // 3] = LOWEST[dtype]
    return x


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("temperature", [1.0, 0.25])
@pytest.mark.parametrize("cats", [4, 37, 256, 1500, 40000])
def test_masks(dtype, cats, temperature):
    x = _masked(13, cats, dtype, cats)
    _check(x, _tokens(13, cats), min(cats, 20), temperature)
    empty = torch.full((2, cats), -math.inf, dtype=dtype, device="cuda", requires_grad=True)
    out = api.token_logprobs(empty, torch.zeros(2, dtype=torch.int64, device="cuda"), 3 if cats >= 3 else 1)
    assert (out.logp == -math.inf).all() and (out.entropy == 0).all() and (out.top_logp == -math.inf).all()
    assert torch.equal(out.top_ids[0], torch.arange(out.top_ids.shape[1], device="cuda"))
    assert (torch.autograd.grad([out.entropy, out.logp], empty, [torch.ones(2, device="cuda")] * 2)[0] == 0).all()


@pytest.mark.parametrize("cats", [30, 300, 3000, 40000])
@pytest.mark.parametrize("temperature", [1.0, 40.0, 150.0])
def test_logits_near_the_lowest_of_half_precision(cats, temperature):
    """Where what stands for impossible categories would still weigh beside the row's own: the sums change their form at a
    line that goes through the row."""
    gen = torch.Generator().manual_seed(cats)
    x = -65504 + 12000 * torch.rand(6, cats, generator=gen)
    x[1] = -65504 + 300 * torch.rand(cats, generator=gen)
    x[2, ::3] = -math.inf
    x[3, : cats // 2] = -65504
    _check(x.half().cuda(), _tokens(6, cats), 3, temperature)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("temperature", [1e-6, 1e-3, 1e4, 1e20])
def test_extreme_temperatures_and_offsets(dtype, temperature):
    for cats in (50, 2500):
        x = make_logits(5, cats, dtype, 3)
        x[1] += 1000.0
        x[2] *= 0.0
        x[3, 1:] = -math.inf
        x = x.to(dtype)
        _check(x, _tokens(5, cats), 2, temperature, (1, 0, 0) if temperature < 1e-2 else (1, 1, 1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cats", [5, 300, 3000, 40000])
def test_nan_and_inf_stay_in_their_rows(dtype, cats):
    x = make_logits(6, cats, dtype, 1)
    x[1, cats // 2] = math.nan
    x[2, cats - 1] = math.inf
    x[3] = -math.inf
    x[3, 1] = math.nan
    tokens = torch.zeros(6, dtype=torch.int64, device="cuda")
    leaf = x.clone().requires_grad_()
    out = api.token_logprobs(leaf, tokens, 2)
    bad = torch.tensor([False, True, True, True, False, False], device="cuda")
    for o in (out.logp, out.entropy, out.top_logp[:, 0]):
        assert torch.equal(torch.isnan(o), bad)
    assert out.top_ids[1, 0] == cats // 2 and out.top_ids[2, 0] == cats - 1 and out.top_ids[3, 0] == 1
    assert out.top_ids[3, 1] == 0
    dx, = torch.autograd.grad([out.logp, out.entropy], leaf, [torch.ones(6, device="cuda")] * 2)
    assert torch.equal(torch.isnan(dx).any(1), bad)
    good = ~bad
    ref = Logprobs(x[good], tokens[good], 2, 1.0)
    assert_within(out.logp[good], ref.logp, ref.tol_logp)
    assert torch.equal(out.top_ids[good], ref.top_ids)


@pytest.mark.parametrize("cats", [64, 1000, 5000, 70000, 300000])
@pytest.mark.parametrize("top_k", [1, 8, 32])
def test_alternatives_in_hard_orders(cats, top_k):
    """Rising and falling rows, rows of few different values, constant rows, +0 beside -0, the best ones side by side in
    the places of one thread, one value and a few below it, NaN in front."""
    j = torch.arange(cats, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(2)
    r = torch.randn(cats, generator=gen, device="cuda")
    rows = [j.float(), -j.float(), (j % 3).float(), torch.zeros(cats, device="cuda"), torch.where(j % 2 == 0, 0.0, -0.0),
            r.round(), torch.where(j % 256 == 7, r + 50, r), torch.where(j // 32 % 256 == 3, r + 50, r),
            torch.where(j >= cats - 40, r + 50, r), torch.where(j < 40, r + 50, r), torch.where(j % 1024 == 1023, 9.0, -math.inf),
            torch.where(j == cats - 1, 1.0, 0.0), torch.where(j % 8 == 5, r + 50, r), torch.where(j // 8 % 256 == 200, 50.0, r)]
    x = torch.stack(rows)
    for dtype in DTYPES:
        xt = x.clamp(-60000, 60000).to(dtype) if dtype == torch.float16 else x.to(dtype)
        _check(xt, None, top_k, 1.0, (0, 0, 0))
        _check(xt[:, 1:], None, top_k, 1.0, (0, 0, 0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cats", [30, 500, 6001])
def test_strides_and_alignment(dtype, cats):
    base = make_logits(24, cats + 9, dtype, 8)
    for first in (0, 1, 3, 8):
        _check(base[:, first:first + cats], _tokens(24, cats), 4)
    _check(base[::3, 2:2 + cats], _tokens(8, cats), 4)
    _check(base[3:4, :cats].expand(5, cats), _tokens(5, cats), 4, grads=(1, 1, 0))
    turned = make_logits(cats, 6, dtype, 9).t()   # categories far apart
    _check(turned, _tokens(6, cats), 4)
    three = make_logits(12, cats, dtype, 10).view(3, 4, cats)
    t3 = _tokens(12, cats).view(3, 4)
    out, flat = api.token_logprobs(three, t3, 2), api.token_logprobs(three.view(12, cats), t3.view(12).int(), 2)
    assert out.logp.shape == (3, 4) and out.top_ids.shape == (3, 4, 2)
    assert torch.equal(out.logp.view(-1), flat.logp) and torch.equal(out.top_ids.view(12, 2), flat.top_ids)
    out = api.token_logprobs(three.transpose(0, 1), t3.t(), 2)
    # rows that begin elsewhere between 16-byte boundaries are added up in another order: both sides within the bound of
    # heads_reference, which holds for any order
    ref = Logprobs(three.transpose(0, 1).reshape(12, cats), t3.t().reshape(12), 2, 1.0)
    assert_within(out.entropy.reshape(12), ref.entropy, ref.tol_entropy)
    assert_within(out.logp.reshape(12), ref.logp, ref.tol_logp)
    assert torch.equal(out.top_ids.reshape(12, 2), ref.top_ids)
    one = api.token_logprobs(three[1, 2], t3[1, 2], 2)
    assert one.logp.shape == () and torch.equal(one.logp, flat.logp[6]) and torch.equal(one.top_ids, flat.top_ids[6])


def test_tokens_that_are_not_given_or_not_there():
    x = make_logits(4, 50, torch.float32, 1).requires_grad_()
    t = torch.tensor([-1, 49, 50, -100], device="cuda")
    out = api.token_logprobs(x, t)
    assert out.logp[0] == 0 and out.logp[3] == 0 and torch.isnan(out.logp[2]) and out.logp[1] < 0
    dx, = torch.autograd.grad(out.logp.sum(), x)   # an expanded gradient
    assert (dx[0] == 0).all() and (dx[3] == 0).all() and torch.isnan(dx[2]).all() and torch.isfinite(dx[1]).all()
    out = api.token_logprobs(x)
    assert out.logp is None and out.top_ids is None and out.top_logp is None
    assert torch.autograd.grad(out.entropy.mean(), x)[0].abs().sum() > 0


def test_empty_batches():
    x = torch.zeros(0, 7, device="cuda", requires_grad=True)
    out = api.token_logprobs(x, torch.zeros(0, dtype=torch.int64, device="cuda"), 3)
    assert out.logp.shape == (0,) and out.top_ids.shape == (0, 3)
    assert torch.autograd.grad(out.entropy.sum(), x)[0].shape == (0, 7)
    assert api.token_logprobs(torch.zeros(2, 0, 7, device="cuda")).entropy.shape == (2, 0)


def test_refusals_on_the_device():
    x = torch.zeros(3, 10, device="cuda")
    for call in (lambda: api.token_logprobs(x, top_k=11), lambda: api.token_logprobs(x, top_k=-1), lambda: api.token_logprobs(x, temperature=0.0),
                 lambda: api.token_logprobs(x, temperature=math.inf), lambda: api.token_logprobs(x.double()), lambda: api.token_logprobs(x[0, 0]),
                 lambda: api.token_logprobs(x[:, :0]), lambda: api.token_logprobs(x, torch.zeros(3)), lambda: api.token_logprobs(x, torch.zeros(3).long()),
                 lambda: api.token_logprobs(x, torch.zeros(4, device="cuda").long()), lambda: api.token_logprobs(torch.zeros(2, 64, device="cuda"), top_k=33)):
        with pytest.raises(_lib.PcbError) as e:
            call()
        assert e.value.code == 1


@pytest.mark.parametrize("cats", [20, 3001])
def test_gradient_against_differences(cats):
    """Along a direction u with |u| <= 1 the third derivative of a log-probability is a third central moment of u / T, at
    most 8 / T^3; the difference over 2 h is off by h^2 / 6 of it and by the bound of the two values over 2 h."""
    T, h = 1.5, 2.0 ** -5
    x = make_logits(3, cats, torch.float32, 6).requires_grad_()
    t = torch.tensor([0, cats // 2, cats - 1], device="cuda")
    gen = torch.Generator().manual_seed(3)
    u = (2 * torch.rand(3, cats, generator=gen) - 1).cuda()
    out = api.token_logprobs(x, t, 1, T)
    dx, = torch.autograd.grad(out.logp.sum() + 2 * out.top_logp.sum(), x)
    tol = 0.0
    values = []
    for s in (h, -h):
        o = Logprobs((x + s * u), t, 1, T)
        got = api.token_logprobs((x + s * u).detach(), t, 1, T)
        ids = out.top_ids
        values.append(got.logp.double().sum() + 2 * o.logp_all.gather(1, ids).sum())
        tol += (o.tol_logp.sum().item()) / (2 * h)
    tol += 9 * 8 / T ** 3 * h * h / 6 + 9 * 2.0 ** -22 * 20 / h   # x + h u rounded to fp32: values of up to 20
    assert abs((values[0] - values[1]).item() / (2 * h) - (dx.double() * u.double()).sum().item()) <= tol
    # the entropy, by differences of its formula
    dh, = torch.autograd.grad(api.token_logprobs(x, None, 0, T).entropy.sum(), x)
    e = 1e-4
    xd = x.detach().double()
    num = (Logprobs(xd + e * u.double(), None, 0, T).entropy - Logprobs(xd - e * u.double(), None, 0, T).entropy) / (2 * e)
    # its third derivative along u stays below 8 (H + ln cats + 20) / T^3 < 400
    _, bound = Logprobs(x, None, 0, T).grad(None, torch.ones(3, device="cuda"), None, torch.float32)
    assert (((dh.double() * u.double()).sum(1) - num).abs() <= (bound * u.double().abs()).sum(1) + 400 * e * e / 6).all()


def test_another_stream_and_a_replayed_graph():
    cats = 9000
    x, t = make_logits(5, cats, torch.bfloat16, 1), _tokens(5, cats)
    want = api.token_logprobs(x, t, 6)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = api.token_logprobs(x, t, 6)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    static_x, static_t = x.clone(), t.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        leaf = static_x.detach().requires_grad_()
        out = api.token_logprobs(leaf, static_t, 6)
        dx, = torch.autograd.grad([out.logp, out.entropy], leaf, [torch.ones_like(out.logp), torch.ones_like(out.entropy)])
    for seed in (2, 3):
        x2 = make_logits(5, cats, torch.bfloat16, seed)
        static_x.copy_(x2)
        graph.replay()
        leaf2 = x2.requires_grad_()
        fresh = api.token_logprobs(leaf2, t, 6)
        assert all(torch.equal(a, b) for a, b in zip(out, fresh))
        assert torch.equal(dx, torch.autograd.grad([fresh.logp, fresh.entropy], leaf2, [torch.ones_like(out.logp)] * 2)[0])


def test_repeated_calls_agree_in_every_bit():
    for rows, cats in ((1, 131072), (400, 256), (50, 20001)):
        x, t = make_logits(rows, cats, torch.float32, 4).requires_grad_(), _tokens(rows, cats)
        runs = []
        for _ in range(3):
            out = api.token_logprobs(x, t, 8)
            runs.append([*out, torch.autograd.grad(out.logp.sum() + out.entropy.sum(), x)[0]])
        for again in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(runs[0], again))


def test_rows_further_apart_than_32_bits():
    cats, step = 5003, (1 << 30) + 7
    store = torch.empty(2 * step + cats + 64, dtype=torch.bfloat16, device="cuda")
    x = store.as_strided((3, cats), (step, 1), 11)
    fill = make_logits(3, cats, torch.bfloat16, 2)
    x.copy_(fill)
    t = _tokens(3, cats)
    # (another alignment, another order of the sums: the bound covers both)
    got, ref = api.token_logprobs(x, t, 5), Logprobs(fill, t, 5, 1.0)
    assert torch.equal(got.top_ids, ref.top_ids)
    assert_within(got.logp, ref.logp, ref.tol_logp)
    assert_within(got.entropy, ref.entropy, ref.tol_entropy)
    _check(x, t, 5)


def test_inputs_changed_after_the_call_are_noticed():
    x = make_logits(3, 40, torch.float32, 1).requires_grad_()
    out = api.token_logprobs(x, None, 2)
    with torch.no_grad():
        x.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out.entropy.sum(), x)


def test_no_gradient_of_the_gradient():
    x = make_logits(3, 40, torch.float32, 1).requires_grad_()
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(api.token_logprobs(x).entropy.sum(), x, create_graph=True)
    y = make_logits(6, 40, torch.float32, 1).view(2, 3, 40).requires_grad_()
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(api.soft_evidence(y).sum(), y, create_graph=True)
