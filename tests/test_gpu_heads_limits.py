"""Limits of the categorical-head operators: large weights of the entropy, what the statistics hold, weights and derivatives
that are not numbers or not there."""
import math

import pytest
import torch

from lvd_pg_b200 import api
from tests.heads_reference import Logprobs, make_logits
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
