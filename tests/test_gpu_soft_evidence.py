"""Soft evidence made of logits, its gradient, and the circuit's passes on it, against 64 bits and the oracle."""
import math

import numpy as np
import pytest
import torch

from lvd_pg_b200 import _lib, api
from tests.heads_reference import LOG2E, Logprobs, U, assert_within, chain_of, make_logits, rounding
from tests.helpers import random_hclt
from tests.test_gpu_em import TOL

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _logits(rows, variables, cats, dtype, seed=0):
    return make_logits(rows * variables, cats, dtype, seed).view(rows, variables, cats)


def _miss(rows, variables, seed=0):
    return (torch.rand(rows, variables, generator=torch.Generator().manual_seed(seed)) < 0.3).cuda()


def _check(x, miss, temperature=1.0, g=None):
    rows, variables, cats = x.shape
    leaf = x.detach().requires_grad_()
    out = api.soft_evidence(leaf, miss, temperature)
    assert out.shape == x.shape and out.dtype == torch.float32 and api._is_colmajor(out)
    assert torch.equal(out.detach(), api.soft_evidence(x.detach(), miss, temperature))
    ref = Logprobs(x.reshape(-1, cats), None, 0, temperature)
    want, tol = ref.logp_all.view(x.shape), ref.tol_logp_all.view(x.shape)
    gone = torch.zeros(rows, variables, dtype=torch.bool, device="cuda") if miss is None else miss.bool()
    want, tol = want.masked_fill(gone[:, :, None], 0.0), tol.masked_fill(gone[:, :, None], 0.0)
    assert_within(out, want, tol, "evidence")
    if g is None:
        g = torch.randn(cats, variables, rows, generator=torch.Generator().manual_seed(1)).cuda().permute(2, 1, 0)
    dx, = torch.autograd.grad(out, leaf, g)
    assert dx.dtype == x.dtype and dx.shape == x.shape
    g64, p, d = g.double(), ref.p.view(x.shape), ref.d.view(x.shape)
    total, spread = g64.sum(2, keepdim=True), g64.abs().sum(2, keepdim=True)
    nothing = (gone | ref.empty.view(rows, variables))[:, :, None]
    want = ((g64 - p * total) / temperature).masked_fill(nothing, 0.0)
    # the sum of g in a chain of cats / 32 + 40; p as in heads_reference; two products and a difference of their own
    tol_S = ref.tol_S.view(rows, variables, 1)
    tol = (3 * U * g64.abs() + p * (spread * U * (cats / 32 + 40) + total.abs() * (U * (12 + 8 * d) + 2 * tol_S)) + 2.0 ** -118 * spread) / temperature
    assert_within(dx, want, tol.masked_fill(nothing, 0.0) + rounding(want, x.dtype), "gradient")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,variables,cats,temperature", [
    (1, 1, 1, 1.0), (1, 3, 2, 1.0), (70, 5, 2, 0.7), (33, 2, 3, 1.0), (31, 4, 16, 1.0), (64, 3, 31, 1.3), (5, 9, 33, 1.0), (100, 3, 64, 1.0),
    (37, 3, 200, 1.0), (32, 2, 256, 1.0), (130, 2, 257, 0.5), (9, 2, 500, 1.0), (40, 2, 513, 1.0), (33, 2, 1000, 1.0), (20, 1, 1024, 1.0),
    (65, 1, 2049, 1.0), (3, 2, 5003, 1.0), (34, 1, 40000, 0.8), (300, 1, 7, 1.0), (40, 300, 3, 1.0), (35, 20, 30, 1.0), (70, 9, 41, 1.0),
    (33, 3, 130, 1.0), (32, 3, 767, 1.0), (40, 2, 1023, 1.0)])
def test_shapes(dtype, rows, variables, cats, temperature):
    x = _logits(rows, variables, cats, dtype, rows + cats)
    _check(x, None, temperature)
    _check(x, _miss(rows, variables), temperature)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cats", [2, 40, 700, 3000])
def test_masks(dtype, cats):
    x = _logits(6, 3, cats, dtype, 2)
    lowest = torch.finfo(dtype).min
    x[0, 0] = -math.inf
    x[1, 0] = lowest
    x[2, 1, 1:] = -math.inf
    x[3, 1, 1:] = lowest
    x[4, 2] = -math.inf
    x[4, 2, cats - 1] = lowest
    _check(x, None)
    _check(x, _miss(6, 3), 0.5)
    x[5, 0, 0] = math.nan
    x[5, 1, cats - 1] = math.inf
    out = api.soft_evidence(x)
    bad = torch.zeros(6, 3, dtype=torch.bool, device="cuda")
    bad[5, :2] = True
    assert torch.equal(torch.isnan(out).all(2), bad) and torch.equal(torch.isnan(out).any(2), bad)
    hide = bad.clone()
    assert (api.soft_evidence(x, hide)[5, :2] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(dtype):
    base = _logits(40, 7, 75, dtype, 3)
    for first in (0, 1, 4):
        _check(base[:, :, first:first + 66], None)
    _check(base[::3, 1:6:2, 5:69], _miss(14, 6)[:, ::2])
    _check(base.transpose(0, 1), _miss(40, 7).t())
    _check(base.permute(2, 1, 0), None)                       # categories far apart
    _check(base[:1].expand(33, 7, 75), _miss(1, 7).expand(33, 7))
    x = base.contiguous()
    _check(x, _miss(40, 7).to(torch.uint8) * 3)
    for g in (torch.ones((), device="cuda").expand(40, 7, 75), torch.randn(40, 7, 75, device="cuda"),
              torch.randn(7, 40, 75, device="cuda").transpose(0, 1)):
        _check(x, None, 1.0, g)


def test_refusals_and_empty_batches():
    x = torch.zeros(3, 4, 5, device="cuda")
    for call in (lambda: api.soft_evidence(x[0]), lambda: api.soft_evidence(x.double()), lambda: api.soft_evidence(x, temperature=-1.0),
                 lambda: api.soft_evidence(x, torch.zeros(3, 4)), lambda: api.soft_evidence(x, torch.zeros(4, 3, device="cuda", dtype=torch.bool)),
                 lambda: api.soft_evidence(x, torch.zeros(3, 4, device="cuda")), lambda: api.soft_evidence(x[:, :, :0])):
        with pytest.raises(_lib.PcbError) as e:
            call()
        assert e.value.code == 1
    assert api.soft_evidence(x[:0]).shape == (0, 4, 5) and api.soft_evidence(x[:, :0]).shape == (3, 0, 5)


def test_another_stream_and_a_replayed_graph():
    x, miss = _logits(50, 6, 90, torch.float16, 1), _miss(50, 6)
    want = api.soft_evidence(x, miss)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = api.soft_evidence(x, miss)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    static, g = x.clone(), torch.randn(90, 6, 50, device="cuda").permute(2, 1, 0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        leaf = static.detach().requires_grad_()
        out = api.soft_evidence(leaf, miss)
        dx, = torch.autograd.grad(out, leaf, g)
    for seed in (2, 3):
        x2 = _logits(50, 6, 90, torch.float16, seed)
        static.copy_(x2)
        graph.replay()
        leaf2 = x2.requires_grad_()
        fresh = api.soft_evidence(leaf2, miss)
        assert torch.equal(out, fresh) and torch.equal(dx, torch.autograd.grad(fresh, leaf2, g)[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,variables,cats", [(33, 300, 1), (40, 290, 2), (100, 70, 3), (5, 33, 8), (65, 13, 30), (40, 3, 300), (33, 2, 1500)])
def test_statistics_of_every_distribution(dtype, rows, variables, cats):
    """Many variables a tile, batches that end inside one; the largest logit exactly, the sum of powers within its bound, and
    nothing written behind them."""
    x, miss = _logits(rows, variables, cats, dtype, cats), _miss(rows, variables, 3)
    if cats > 1:
        x[1, 0] = -math.inf
    _check(x, miss)
    out = torch.full((cats * variables * rows + 64,), 7.0, device="cuda")
    stats = torch.full((rows * variables * 2 + 64,), 7.0, device="cuda")
    _lib.check(_lib.lib().pcb_soft_evidence(x.data_ptr(), DTYPES.index(dtype), rows, variables, cats, variables * cats, cats, miss.data_ptr(), variables,
                                            1, 1.0, out.data_ptr(), stats.data_ptr(), torch.cuda.current_stream().cuda_stream))
    assert torch.equal(out[:-64].view(cats, variables, rows).permute(2, 1, 0), api.soft_evidence(x, miss))
    assert (out[-64:] == 7).all() and (stats[-64:] == 7).all()
    got = stats[:-64].view(rows * variables, 2)
    ref = Logprobs(x.reshape(-1, cats), None, 0, 1.0)
    assert torch.equal(got[:, 0], x.reshape(-1, cats).float().amax(1))
    # S counts from the rounded product of the maximum and log2(e): half a step of it beside the bound of the sum itself
    shift = torch.where(ref.empty, 0.0, ref.x.amax(1))
    want = (ref.x - shift[:, None]).exp().sum(1)
    assert_within(got[:, 1], want, want * (ref.tol_S + 2 * U * (1 + shift.abs() * LOG2E)))


def test_more_elements_than_32_bits_count():
    rows, variables, cats = 70001, 64, 512
    x = torch.empty(rows, variables, cats, dtype=torch.bfloat16, device="cuda")
    part = _logits(1000, variables, cats, torch.bfloat16, 5)
    for at in range(0, rows, 1000):
        x[at:at + 1000] = part[:min(1000, rows - at)]
    out = api.soft_evidence(x)
    small = api.soft_evidence(part)
    assert torch.equal(out[69000:70000], small) and torch.equal(out[:1000], small) and torch.equal(out[70000:], small[:1])
    del x, out
    torch.cuda.empty_cache()


@pytest.mark.parametrize("c,rows,k", [(5, 20, 16), (33, 70, 17)])
def test_a_circuit_on_a_heads_evidence(oracle, c, rows, k):
    """Features -> head in 4 bits -> evidence -> likelihoods and an EM step: against the oracle on the same evidence in
    64 bits, rounded to the fp32 that the oracle takes."""
    fc = random_hclt(7, k, c, 4)
    rng = np.random.default_rng(c)
    weight = torch.from_numpy(rng.normal(0, 0.2, (c, 50)).astype(np.float32)).cuda()
    head = api.QuantHead(weight, 32, bias=torch.from_numpy(rng.normal(0, 1, c).astype(np.float32)).cuda())
    x = torch.from_numpy(rng.normal(0, 1, (rows, 7, 50)).astype(np.float32)).cuda()
    miss = torch.from_numpy(rng.random((rows, 7)) < 0.2).cuda()
    logits = x.double() @ head.weight().double().t() + head.bias.double()
    soft = torch.log_softmax(logits, -1).masked_fill(miss[:, :, None], 0.0).float().cpu().numpy()
    ref, m = fc.copy(), api.CuMetaBitsProbCircuit(fc)
    evidence = head.evidence(x, miss)
    mars_ref = oracle.forward_ex(ref, soft=soft)
    ll = torch.empty(rows, device="cuda")
    api.forward_ex(m, soft=evidence, ll_out=ll)
    assert np.abs(ll.cpu().numpy() - mars_ref[:, -1]).max() <= TOL * max(1.0, np.abs(mars_ref[:, -1]).max())
    lls = torch.zeros(1, device="cuda")
    ll_ref, _ = oracle.em_step_ex(ref, soft=soft, pseudocount=0.1, inertia=0.1)
    api.em_step_ex(m, soft=evidence, pseudocount=0.1, inertia=0.1, ll_sum=lls)
    assert abs(lls.item() - ll_ref) <= TOL * abs(ll_ref)
    assert np.abs(np.exp(api.vectorize_parameters(m)) - np.exp(oracle.vectorize(ref))).max() <= TOL
    # the network's own score of categories, beside the circuit's
    tokens = torch.from_numpy(rng.integers(0, c, (rows, 7))).cuda()
    scores = head.logprobs(x, tokens, min(c, 4))
    want = torch.log_softmax(logits, -1)
    assert (scores.logp.double() - want.gather(2, tokens[:, :, None])[:, :, 0]).abs().max() <= TOL
    assert torch.equal(scores.top_ids[:, :, 0], logits.argmax(-1))
