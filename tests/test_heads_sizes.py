"""Sizes, alignments and derivatives that the categorical-head operators refuse before anything is launched: no GPU is needed."""
import ctypes as C

import pytest
import torch

from lvd_pg_b200 import _lib, api, build

INVALID = 1


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.lib()


@pytest.mark.parametrize("variables", [1 << 31, (1 << 32) - 1])
def test_more_variables_than_tiles_are_counted(lib, variables):
    """A tile of one variable each: a block's count of them, 65535 at a time, would pass 2^32 and begin anew."""
    b = C.create_string_buffer(80)
    assert lib.pcb_soft_evidence(b, 0, 1, variables, 1, 0, 0, None, 0, 0, 1.0, b, None, None) == INVALID
    assert b"variables" in lib.pcb_last_error()
    assert lib.pcb_soft_evidence_backward(b, 0, 1, variables, 1, 0, 0, None, 0, 0, 1.0, b, b, b, None) == INVALID
    assert b"variables" in lib.pcb_last_error()


class _OnDevice(torch.Tensor):   # passes for a CUDA tensor where arguments are looked at
    is_cuda = property(lambda self: True)


def _wide(*shape, dtype=torch.float32):
    return torch.zeros((1,) * len(shape), dtype=dtype).expand(shape).as_subclass(_OnDevice)


def test_sizes_that_32_bits_do_not_hold():
    """The library is told of them in 32 bits, where 2^32 + 5 would be 5."""
    for wide in ((1 << 32) + 5, 1 << 31):
        for call in (lambda: api.token_logprobs(_wide(2, wide)), lambda: api.soft_evidence(_wide(1, 1, wide)),
                     lambda: api.soft_evidence(_wide(1, wide, 2)), lambda: api.QuantHead(_wide(wide, 32)), lambda: api.QuantHead(_wide(1, wide)),
                     lambda: api.QuantHead.from_codes(_wide(wide, 16, dtype=torch.uint8), _wide(wide, 1, dtype=torch.float16), 32),
                     lambda: api.QuantHead.from_codes(_wide(1, (wide + 1) // 2, dtype=torch.uint8), _wide(1, -(-wide // 64), dtype=torch.float16), wide)):
            with pytest.raises(_lib.PcbError) as e:
                call()
            assert e.value.code == INVALID


def test_tangents_of_forward_mode():
    import torch.autograd.forward_ad as forward_ad

    from lvd_pg_b200 import heads

    x = torch.zeros(2, 3, 4)
    heads._no_tangent(x)
    with forward_ad.dual_level():
        heads._no_tangent(x)
        with pytest.raises(_lib.PcbError, match="tangent") as e:
            heads._no_tangent(forward_ad.make_dual(x, x))
        assert e.value.code == INVALID


def test_pointers_off_their_types_alignment(lib):
    """Arguments that come without a type: tokens, scales, weights to quantise, a packed head."""
    b = C.create_string_buffer(512)
    at = (C.addressof(b) + 15) // 16 * 16
    for token_bytes, off in ((8, 4), (8, 1), (4, 2)):
        assert lib.pcb_token_logprobs(at, 0, 1, 5, 5, 1.0, at + off, token_bytes, 0, at, at, None, None, None, None) == INVALID
        assert lib.pcb_token_logprobs_backward(at, 0, 1, 5, 5, 1.0, at + off, token_bytes, 0, None, at, at, at, 1, None, 0, None, at, None) == INVALID
    for dtype, off in ((0, 2), (1, 1), (2, 1)):
        assert lib.pcb_head_quantize(at + off, dtype, 1, 32, 32, 1, at, at, None) == INVALID
    assert lib.pcb_head_quantize(at, 0, 1, 32, 32, 1, at, at + 1, None) == INVALID
    assert lib.pcb_head_pack(at, at + 1, 1, 32, 32, at, None) == INVALID
    assert lib.pcb_head_weight(at + 8, 1, 1, 32, 32, at, None) == INVALID
