"""The paged cache's attention on the GPU, held to what its arithmetic gives.

Tolerances. fp32 work is off by less than 1e-4 for any element (normal
operands, scores below 32: products' sums 2^-18 a score, which moves a weight
by as much, and the mean's own sums 2^-18 of the largest value, 6).
"""

import math

import pytest
import torch

import kiln
import paged_reference as ref

TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float32)]
IDS = ["fp32", "bf16-cache", "fp16-cache"]


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def check(p, **more):
    got = kiln.tree_attention(**p, **more)
    torch.testing.assert_close(got.double().cpu(), ref.attention(**p, **more), equal_nan=True, rtol=0.0, atol=1e-4)
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("cache,act", TYPES, ids=IDS)
@pytest.mark.parametrize("draft,length", [(5, 100), (70, 100), (5, 3000), (70, 3000)])
def test_infinities_that_are_attended_to(cache, act, draft, length):
    """An infinite value makes its dimension infinite in the rows that attend to
    it, a key whose score is -inf has no weight: cached or drafted."""
    p = ref.problem(gen(7), draft=draft, heads=4, kv=2, lengths=(length, 41), cache=cache, act=act, device="cuda")
    page = p["table"][0, 2]
    p["v_pages"][page, 0, 3, 5] = math.inf
    p["v_pages"][page, 1, 7, 11] = -math.inf
    p["q"][0, :, :, 7] = p["q"][0, :, :, 7].abs() + 0.5
    p["k_pages"][page, 1, 9, 7] = -math.inf       # q[7] > 0: a score of -inf
    p["v"][1, 1, 0, 3] = math.inf
    p["q"][1, :, :, 2] = -p["q"][1, :, :, 2].abs() - 0.5
    p["k"][1, 2, 1, 2] = math.inf
    got = check(p)
    assert torch.isinf(got[0]).sum() == 4 * draft
