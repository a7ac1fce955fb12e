"""What the categorical-head operators refuse, before anything is launched: no GPU is needed."""
import ctypes as C

import pytest
import torch

from lvd_pg_b200 import _lib, api, build

INVALID, TOO_LARGE = 1, 4


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


def _buf(n=64):
    return C.create_string_buffer(n + 16)


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 3)
    for call in (lambda: api.token_logprobs(x), lambda: api.soft_evidence(x[None]), lambda: api.QuantHead(x),
                 lambda: api.QuantHead.from_codes(x.to(torch.uint8), x, 5)):
        with pytest.raises(_lib.PcbError) as e:
            call()
        assert e.value.code == INVALID


@pytest.mark.parametrize("change", [
    dict(x=None), dict(dtype=3), dict(dtype=-1), dict(cats=0), dict(cats=1 << 31), dict(temperature=0.0), dict(temperature=-1.0),
    dict(temperature=float("nan")), dict(temperature=float("inf")), dict(temperature=1e-39), dict(token_bytes=2), dict(logp=None),
    dict(top_k=33), dict(top_k=6), dict(top_k=2, ids=None), dict(top_k=2, top=None), dict(entropy=None), dict(stats=12)])
def test_token_logprobs_arguments(lib, change):
    b = _buf()
    a = dict(x=b, dtype=0, rows=1, cats=5, stride=5, temperature=1.0, tokens=b, token_bytes=8, top_k=0, logp=b, entropy=b, stats=b,
             ids=b, top=b)
    if change.get("top_k") == 33:
        a["cats"] = 100
    a.update(change)
    assert lib.pcb_token_logprobs(*a.values(), None) == INVALID
    assert lib.pcb_last_error()


@pytest.mark.parametrize("change", [
    dict(x=None), dict(dtype=9), dict(cats=0), dict(temperature=0.0), dict(stats=None), dict(entropy=None), dict(dx=None), dict(tokens=None),
    dict(token_bytes=1), dict(top_k=40), dict(top_k=0), dict(ids=None)])
def test_token_logprobs_backward_arguments(lib, change):
    b = _buf()
    a = dict(x=b, dtype=0, rows=1, cats=5, stride=5, temperature=1.0, tokens=b, token_bytes=8, top_k=2, ids=b, stats=b, entropy=b,
             g_logp=b, g_logp_stride=1, g_entropy=b, g_entropy_stride=1, g_top=b, dx=b)
    a.update(change)
    assert lib.pcb_token_logprobs_backward(*a.values(), None) == INVALID


@pytest.mark.parametrize("change", [dict(x=None), dict(dtype=3), dict(cats=0), dict(temperature=0.0), dict(out=None)])
def test_soft_evidence_arguments(lib, change):
    b = _buf()
    a = dict(x=b, dtype=0, rows=1, vars=1, cats=5, row_stride=5, var_stride=5, miss=None, mr=0, mv=0, temperature=1.0, out=b, stats=None)
    a.update(change)
    assert lib.pcb_soft_evidence(*a.values(), None) == INVALID


@pytest.mark.parametrize("change", [dict(x=None), dict(dtype=3), dict(cats=0), dict(temperature=0.0), dict(g=None), dict(stats=None), dict(dx=None)])
def test_soft_evidence_backward_arguments(lib, change):
    b = _buf()
    a = dict(x=b, dtype=0, rows=1, vars=1, cats=5, row_stride=5, var_stride=5, miss=None, mr=0, mv=0, temperature=1.0, stats=b, g=b, dx=b)
    a.update(change)
    assert lib.pcb_soft_evidence_backward(*a.values(), None) == INVALID


def test_head_arguments(lib):
    b = _buf(256)
    at = (C.addressof(b) + 15) // 16 * 16
    size = C.c_uint64()
    assert lib.pcb_head_packed_bytes(16, 64, 64, C.byref(size)) == 0
    assert size.value == 16 * 64 // 2 + 128     # codes, and one quad of groups' scales
    for cats, features, group in ((0, 64, 64), (16, 0, 64), (16, 64, 48), (16, 64, 0), (1 << 31, 64, 64)):
        assert lib.pcb_head_packed_bytes(cats, features, group, C.byref(size)) == INVALID
        assert lib.pcb_head_pack(at, at, cats, features, group, at, None) == INVALID
        assert lib.pcb_head_quantize(at, 0, cats, features, group, 1, at, at, None) == INVALID
        assert lib.pcb_head_weight(at, 1, cats, features, group, at, None) == INVALID
        assert lib.pcb_head_logits(at, 1, cats, features, group, at, 0, 1, 64, None, at, 0, None) == INVALID
    for features in (32769, 1 << 31):
        assert lib.pcb_head_packed_bytes(16, features, 64, C.byref(size)) == TOO_LARGE
        assert lib.pcb_head_logits(at, 1, 16, features, 64, at, 0, 1, features, None, at, 0, None) == TOO_LARGE
    assert lib.pcb_head_packed_bytes(16, 64, 64, None) == INVALID
    assert lib.pcb_head_pack(None, at, 16, 64, 64, at, None) == INVALID
    assert lib.pcb_head_pack(at, at, 16, 64, 64, at + 4, None) == INVALID          # not 16-byte aligned
    assert lib.pcb_head_quantize(at, 3, 16, 64, 64, 1, at, at, None) == INVALID
    assert lib.pcb_head_quantize(at, 0, 16, 64, 64, 0, at, at, None) == INVALID    # f32 scales
    assert lib.pcb_head_weight(at, 0, 16, 64, 64, at, None) == INVALID
    assert lib.pcb_head_weight(None, 1, 16, 64, 64, at, None) == INVALID
    good = dict(packed=at, scale_dtype=1, cats=16, features=64, group=64, x=at, dtype=0, rows=1, stride=64, bias=None, y=at, y_dtype=0)
    for change in (dict(packed=None), dict(packed=at + 8), dict(scale_dtype=0), dict(x=None), dict(dtype=3), dict(y=None), dict(y_dtype=-1)):
        assert lib.pcb_head_logits(*{**good, **change}.values(), None) == INVALID


def test_nothing_to_do_needs_no_device(lib):
    assert lib.pcb_token_logprobs(None, 0, 0, 5, 5, 1.0, None, 0, 0, None, None, None, None, None, None) == 0
    assert lib.pcb_soft_evidence(None, 0, 0, 3, 5, 15, 5, None, 0, 0, 1.0, None, None, None) == 0
