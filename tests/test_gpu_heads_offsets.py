"""Rows whose largest logit over the temperature lies far from zero: the powers of a row count from its maximum, wherever that
is.  Every operator that is made of logits, in every form of its kernels."""
import pytest
import torch

from tests.heads_reference import make_logits
from tests.test_gpu_soft_evidence import _check as check_evidence
from tests.test_gpu_token_logprobs import _check as check_logprobs, _tokens

pytestmark = pytest.mark.gpu
WIDE = [torch.float32, torch.bfloat16]


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
