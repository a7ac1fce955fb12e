"""The head in 4 bits against products in 64 bits."""
import pytest
import torch

from lvd_pg_b200 import _lib, api
from tests.heads_reference import assert_within, rounding

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _codes(cats, features, group, scale_dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (cats, features + features % 2), generator=gen)
    packed = (codes[:, 0::2] | codes[:, 1::2] << 4).to(torch.uint8).cuda()
    scales = ((0.3 + torch.rand(cats, -(-features // group), generator=gen)) / 50).to(scale_dtype).cuda()
    values = codes[:, :features].double().cuda() - 8
    return packed, scales, values


def _weight(values, scales, group):
    return values * scales.double().repeat_interleave(group, 1)[:, :values.shape[1]]


def _tol(x, values, scales, group, y, bias, dtype):
    """A product of the tensor cores adds at most 17 terms, each cut off below 2^-23 of the largest: 17 * 2^-23 of the sum of
    magnitudes for each of a group's at most 8 * 3 products; then a scale, and one addition per group and the bias."""
    spread = x.double().abs() @ _weight(values.abs(), scales, group).t()
    groups = scales.shape[1]
    return (17 * 24 * 2.0 ** -23 + (groups + 4) * 2.0 ** -24) * spread + 2.0 ** -23 * (0 if bias is None else bias.double().abs()) + rounding(y, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cats,features,group", [
    (1, 1, 1, 32), (2, 15, 31, 32), (3, 16, 32, 32), (1, 17, 33, 64), (8, 100, 63, 64), (9, 33, 64, 64), (5, 40, 65, 128), (7, 1000, 777, 32),
    (1, 1000, 4096, 64), (16, 250, 1030, 128), (17, 48, 2048, 64), (64, 128, 200, 32), (133, 70, 129, 64), (1, 40000, 256, 64), (3, 5000, 8192, 128),
    (2, 64, 20000, 64), (12, 300, 9001, 32), (4, 90, 32768, 128), (40, 4800, 64, 64), (33, 9600, 100, 32),
    (2, 80001, 130, 64)])
def test_shapes(dtype, rows, cats, features, group):
    scale_dtype = torch.bfloat16 if dtype == torch.bfloat16 else torch.float16
    packed, scales, values = _codes(cats, features, group, scale_dtype, cats)
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(rows, features, generator=gen).to(dtype).cuda()
    bias = torch.randn(cats, generator=gen).cuda()
    weight = _weight(values, scales, group)
    for b in (None, bias):
        head = api.QuantHead.from_codes(packed, scales, features, group, bias=b)
        want = x.double() @ weight.t() + (0 if b is None else b.double())
        for out in (None, torch.float32):
            got = head.logits(x, out)
            assert got.dtype == (out or dtype)
            assert_within(got, want, _tol(x, values, scales, group, want, b, got.dtype))
    assert_within(head.weight(), weight, rounding(weight, torch.float32))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features,group", [(1, 64, 64), (3, 517, 32), (11, 4096, 128), (20, 1000, 64)])
def test_sums_that_are_exact(dtype, rows, features, group):
    """Small integers and scales that are powers of two: every partial sum is a number of fp32."""
    cats = 77
    packed, _, values = _codes(cats, features, group, torch.float16, 3)
    gen = torch.Generator().manual_seed(4)
    scales = (2.0 ** torch.randint(-2, 2, (cats, -(-features // group)), generator=gen)).to(torch.bfloat16).cuda()
    x = torch.randint(-8, 9, (rows, features), generator=gen).to(dtype).cuda()
    head = api.QuantHead.from_codes(packed, scales, features, group)
    assert torch.equal(head.logits(x, torch.float32).double(), x.double() @ _weight(values, scales, group).t())


@pytest.mark.parametrize("features", [64, 300, 2048])
def test_all_24_bits_of_fp32_features(features):
    """One feature of 24 bits per group, codes that are powers of two: the product is exact, and needs every bit."""
    cats, group = 40, 32
    groups = -(-features // group)
    gen = torch.Generator().manual_seed(6)
    codes = torch.tensor([7, 9, 10, 12, 4, 6, 0])[torch.randint(0, 7, (cats, features + features % 2), generator=gen)]   # -1 1 2 4 -4 -2 -8
    packed = (codes[:, 0::2] | codes[:, 1::2] << 4).to(torch.uint8).cuda()
    scales = torch.ones(cats, groups, dtype=torch.bfloat16, device="cuda")
    for group_at in (0, groups // 2, groups - 1):
        x = torch.zeros(5, features)
        for r in range(5):
            k = min(features - 1, group_at * group + int(torch.randint(0, group, (1,), generator=gen)))
            x[r, k] = float(torch.randint(2 ** 23, 2 ** 24, (1,), generator=gen)) * 2.0 ** (10 * r - 40)
        x = x.cuda()
        got = api.QuantHead.from_codes(packed, scales, features, group).logits(x)
        assert torch.equal(got.double(), x.double() @ (codes[:, :features].double().cuda() - 8).t())


@pytest.mark.parametrize("dtype", DTYPES)
def test_extreme_features(dtype):
    """The type's largest and smallest values; inf and NaN reach the logits of their own row only."""
    cats, features, group = 50, 200, 64
    packed, scales, values = _codes(cats, features, group, torch.bfloat16, 8)
    head = api.QuantHead.from_codes(packed, scales, features, group)
    f = torch.finfo(dtype)
    x = torch.zeros(6, features, dtype=dtype)
    x[0, 3], x[0, 100] = f.max, f.max
    x[1] = f.smallest_normal
    x[2, 5], x[3, 150] = float("inf"), float("nan")
    x[4] = torch.randn(features, generator=torch.Generator().manual_seed(1)).to(dtype)
    x = x.cuda()
    got = head.logits(x, torch.float32)
    weight = _weight(values, scales, group)
    fine = [0, 1, 4, 5]
    want = x[fine].double() @ weight.t()
    tol = _tol(x[fine], values, scales, group, want, None, torch.float32)
    ok = want.abs() < 3e38
    # an 8 * max of one group passes the range of fp32 before its scale brings it back
    inside = ok & ((x[fine].double().abs() @ values.abs().t()) < 3e38)
    assert ((got[fine].double() - want).abs() <= tol + 2.0 ** -126)[inside].all()
    assert torch.isnan(got[3]).all()
    w5 = values[:, 5]
    assert (got[2][w5 > 0] == float("inf")).all() and (got[2][w5 < 0] == -float("inf")).all()


@pytest.mark.parametrize("weight_dtype", DTYPES)
@pytest.mark.parametrize("cats,features,group", [(20, 64, 64), (33, 100, 32), (7, 129, 128), (3, 1, 32)])
def test_quantising(weight_dtype, cats, features, group):
    """scale = max |w| / 7 in 16 bits, codes the nearest: off by at most half a scale, and where the scale was rounded down the
    largest weights by 7 of its steps more."""
    gen = torch.Generator().manual_seed(2)
    w = torch.randn(cats, features, generator=gen).to(weight_dtype).cuda()
    w[0, : min(features, group)] = 0
    head = api.QuantHead(w, group)
    got = head.weight().double()
    groups = -(-features // group)
    pad = torch.zeros(cats, groups * group, dtype=torch.float64, device="cuda")
    pad[:, :features] = w.double()
    most = pad.view(cats, groups, group).abs().amax(2)
    scale_dtype = torch.float16 if weight_dtype == torch.float16 else torch.bfloat16
    scale = (most.float() / 7).to(scale_dtype).double()
    each = scale.repeat_interleave(group, 1)[:, :features]
    tol = each * (0.5 + 7 * torch.finfo(scale_dtype).eps / 2 * 1.01 + 1e-6)
    assert ((got - w.double()).abs() <= tol).all()
    codes = torch.where(each > 0, got / each, torch.zeros_like(got))
    assert (codes - codes.round()).abs().max() <= 1e-6 and codes.abs().max() <= 7.001
    assert (got[0, : min(features, group)] == 0).all()


def test_strides_shapes_and_streams():
    packed, scales, values = _codes(90, 130, 64, torch.bfloat16, 1)
    head = api.QuantHead.from_codes(packed, scales, 130, 64)
    x = torch.randn(12, 140, device="cuda").bfloat16()
    for v in (x[:, :130], x[:, 3:133], x[::2, 10:], x[:1, :130].expand(6, 130), torch.randn(130, 4, device="cuda").bfloat16().t()):
        assert torch.equal(head.logits(v), head.logits(v.contiguous()))
    three = x[:, :130].reshape(3, 4, 130)
    assert torch.equal(head.logits(three).view(12, 90), head.logits(x[:, :130]))
    assert head.logits(three[0, 0]).shape == (90,)
    assert head.logits(three[:0]).shape == (0, 4, 90)
    again = api.QuantHead.from_codes(torch.cat([packed, packed], 1)[:, :65], torch.cat([scales, scales], 1)[:, :3], 130, 64)
    assert torch.equal(again.packed, head.packed)
    side = torch.cuda.Stream()
    want = head.logits(x[:, :130])
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = head.logits(x[:, :130])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_two_replayed_graphs_of_a_head_and_its_scores():
    """A served step as a graph: head, log-probabilities, alternatives; two graphs of one head, replayed in turn."""
    packed, scales, values = _codes(5000, 512, 64, torch.bfloat16, 1)
    head = api.QuantHead.from_codes(packed, scales, 512, 64)
    graphs = []
    for rows in (1, 4):
        x, t = torch.zeros(rows, 512, device="cuda").bfloat16(), torch.zeros(rows, dtype=torch.int64, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = head.logprobs(x, t, 5, 0.9)
        graphs.append((graph, x, t, out))
    for seed in range(3):
        gen = torch.Generator().manual_seed(seed)
        wants = []
        for graph, x, t, out in graphs:
            x.copy_(torch.randn(x.shape, generator=gen).bfloat16())
            t.copy_(torch.randint(0, 5000, t.shape, generator=gen))
            graph.replay()
        for graph, x, t, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, head.logprobs(x, t, 5, 0.9)))


def test_more_weights_than_32_bits_count():
    cats, features, group = (1 << 20) + 5, 4160, 64
    gen = torch.Generator(device="cuda").manual_seed(1)
    packed = torch.randint(0, 256, (cats, features // 2), generator=gen, device="cuda", dtype=torch.uint8)
    scales = (0.5 + torch.rand(cats, features // group, generator=gen, device="cuda")).bfloat16()
    head = api.QuantHead.from_codes(packed, scales, features, group)
    x = torch.randn(2, features, generator=gen, device="cuda").bfloat16()
    got = head.logits(x, torch.float32)
    at = torch.cat([torch.arange(40), torch.randint(0, cats, (200,)), torch.arange(cats - 40, cats)]).cuda()
    part = packed[at].long()
    values = torch.stack([part & 15, part >> 4], -1).flatten(1).double() - 8
    want = x.double() @ _weight(values, scales[at], group).t()
    assert_within(got[:, at], want, _tol(x, values, scales[at], group, want, None, torch.float32))
    del head, packed, scales
    torch.cuda.empty_cache()


def test_refusals_on_the_device():
    packed, scales, _ = _codes(10, 40, 32, torch.bfloat16, 1)
    head = api.QuantHead.from_codes(packed, scales, 40, 32)
    x = torch.zeros(2, 40, device="cuda")
    for call in (lambda: head.logits(x.double()), lambda: head.logits(x[:, :39]), lambda: head.logits(x.cpu()), lambda: head.logits(x, torch.float64),
                 lambda: head.logits(x.clone().requires_grad_()), lambda: head.evidence(x), lambda: api.QuantHead(x, 48), lambda: api.QuantHead(x[0]),
                 lambda: api.QuantHead(x.double()), lambda: api.QuantHead(x, bias=torch.zeros(3, device="cuda")),
                 lambda: api.QuantHead.from_codes(packed, scales.float(), 40, 32), lambda: api.QuantHead.from_codes(packed, scales, 42, 32),
                 lambda: api.QuantHead.from_codes(packed, scales[:, :1], 40, 32), lambda: api.QuantHead.from_codes(packed.int(), scales, 40, 32),
                 lambda: api.QuantHead.from_codes(packed, scales.cpu(), 40, 32), lambda: api.QuantHead.from_codes(packed, scales, 40, 33)):
        with pytest.raises(_lib.PcbError) as e:
            call()
        assert e.value.code == 1
    with torch.no_grad():
        head.logits(x.clone().requires_grad_())


def test_more_vectors_than_one_launch_takes():
    packed, scales, values = _codes(20, 40, 32, torch.bfloat16, 1)
    bias = torch.randn(20, device="cuda")
    head = api.QuantHead.from_codes(packed, scales, 40, 32, bias=bias)
    x = torch.randn(70001, 40, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    want = x.double() @ _weight(values, scales, 32).t() + bias.double()
    assert_within(head.logits(x, torch.float32), want, _tol(x, values, scales, 32, want, bias, torch.float32))
    bias.zero_()   # the head has its own
    assert_within(head.logits(x[:9], torch.float32), want[:9], _tol(x[:9], values, scales, 32, want[:9], head.bias, torch.float32))


def test_a_head_used_and_dropped_on_another_stream():
    side = torch.cuda.Stream()
    packed, scales, values = _codes(3000, 512, 64, torch.bfloat16, 2)
    x = torch.randn(4, 512, device="cuda").bfloat16()
    want = api.QuantHead.from_codes(packed, scales, 512, 64).logits(x)
    torch.cuda.synchronize()
    for _ in range(20):
        head = api.QuantHead.from_codes(packed, scales, 512, 64)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = head.logits(x)
        size = head.packed.numel()
        del head
        junk = torch.full((size,), 255, dtype=torch.uint8, device="cuda")   # would take the weights' place
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        del junk


def test_calls_of_two_threads_at_once():
    """Two host threads on streams of their own, the same head and logits: head, scores, evidence and gradients as alone."""
    import threading

    packed, scales, values = _codes(3000, 256, 64, torch.bfloat16, 4)
    head = api.QuantHead.from_codes(packed, scales, 256, 64)
    x = torch.randn(6, 256, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    logits = torch.randn(40, 30, 60, generator=torch.Generator().manual_seed(2)).cuda()
    long = torch.randn(3, 200000, generator=torch.Generator().manual_seed(3)).cuda()
    tokens = torch.randint(0, 60, (40, 30), generator=torch.Generator().manual_seed(4)).cuda()

    def work():
        leaf = logits.detach().requires_grad_()
        scores = api.token_logprobs(leaf, tokens, 3)
        evidence = api.soft_evidence(leaf)
        grad, = torch.autograd.grad([scores.logp, evidence], leaf, [torch.ones_like(scores.logp), torch.ones_like(evidence)])
        return [*head.logprobs(x, None, 4)[1:], *scores, evidence, grad, *api.token_logprobs(long, None, 32)[1:]]

    want = [t.detach().clone() for t in work()]
    torch.cuda.synchronize()
    failures = []

    def run():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(15):
                    got = work()
                    torch.cuda.current_stream().synchronize()
                    assert all(torch.equal(a, b) for a, b in zip(got, want))
        except BaseException as e:   # for the main thread
            failures.append(e)

    threads = [threading.Thread(target=run) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures
