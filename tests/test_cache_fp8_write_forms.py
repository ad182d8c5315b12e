"""The rotary write over layouts and batches that take every number of warps of the kernel for many
tokens (eight to twelve, as many as fit), without query heads, and with values that are not finite."""

from __future__ import annotations

import math

import pytest
import torch

import fp8_reference as ref
from test_cache_fp8 import bits, call_write, check_write, write_case


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [True, False], ids=["norm", "plain"])
@pytest.mark.parametrize("tokens, heads, kv_heads, dim", [
    (148 * 9 + 1, 32, 4, 128),   # ten warps fit
    (148 * 10, 28, 4, 128),      # eleven
    (148 * 20 + 5, 8, 8, 128),   # twelve
    (148 * 16, 16, 8, 128),      # eight
    (148 * 65 + 3, 6, 2, 64),    # twelve, a long run
    (2000, 33, 3, 128),          # heads that end inside a pass
    (3001, 7, 5, 64),
    (1400, 0, 3, 128),           # no query heads
    (2000, 0, 1, 64),
    (1300, 64, 8, 128),          # five warps fit
])
def test_many_tokens(cuda, norm, tokens, heads, kv_heads, dim):
    c = write_case(tokens + heads, tokens, heads, kv_heads, dim, pad=2)
    check_write(c, call_write(c, cuda, heads, kv_heads, dim, norm), heads, kv_heads, dim, norm)


@pytest.mark.gpu
@pytest.mark.parametrize("heads, kv_heads, dim", [(16, 8, 128), (9, 3, 64)])
def test_values_that_are_not_finite_stay_in_their_rows(cuda, heads, kv_heads, dim):
    """V rows with infinities and NaN among many tokens: their codes to the bit, the others as without."""
    tokens = 1500
    c = write_case(3, tokens, heads, kv_heads, dim)
    clean = call_write(c, cuda, heads, kv_heads, dim, True)
    x = c["qkv"].view(tokens, heads + 2 * kv_heads, dim)
    at = torch.arange(0, tokens, 7)
    x[at, heads + kv_heads + kv_heads - 1, 3] = math.inf
    x[at[::2], heads + kv_heads, dim - 1] = math.nan
    q, caches, _ = call_write(c, cuda, heads, kv_heads, dim, True)
    assert torch.equal(q, clean[0])
    for i in (0, 2):  # K
        assert torch.equal(bits(caches[i]), bits(clean[1][i]))
    codes, scale, _ = ref.quantise(x[:, heads + kv_heads:].double())
    slots = c["slots"]
    assert torch.equal(bits(caches[1]).flatten(0, 1)[slots], bits(codes))
    assert torch.equal(bits(caches[3]).flatten(0, 1)[slots], bits(scale))
