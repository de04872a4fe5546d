"""The checks of norm_checks.py see what they are for: mistakes planted into the 64-bit form."""

import pytest
import torch

from attention_reference import assert_close, decode
from norm_checks import (assert_close_in_norm, assert_shares, one_hot_rows, relative_norm, shares)

BF16 = torch.bfloat16


def head(n, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(m, 128, generator=gen).to(BF16) for m in (1, n, n)]


@pytest.mark.parametrize("n", [20000, 30000])
@pytest.mark.parametrize("change", ["lost", "twice"])
def test_a_block_lost_or_taken_twice_is_seen(n, change):
    q, k, v = head(n)
    want, size = decode(lambda h: (k.double(), v.double()), q[0], 1, 1)
    at = torch.cat([torch.arange(6400), torch.arange(6464 if change == "lost" else 6336, n)])
    wrong, _ = decode(lambda h: (k[at].double(), v[at].double()), q[0], 1, 1)
    wrong = wrong.to(BF16)
    assert_close(wrong, want, size)                   # the bound for each element alone does not
    with pytest.raises(AssertionError, match="norm"):
        assert_close_in_norm(wrong, want, 2.0 ** -11)


@pytest.mark.parametrize("n", [1, 2, 64, 1000, 20000])
@pytest.mark.parametrize("bits", [8, 11])
def test_rounded_weights_pass(n, bits):
    """Weights and result rounded as the kernels round them."""
    q, k, v = head(n, n)
    s = (q.double() @ k.double().T)[0] * 128 ** -0.5
    p = torch.exp(s - s.max())
    want = (p @ v.double()) / p.sum()
    rounded = p.to(BF16 if bits == 8 else torch.float16).double()
    got = ((rounded @ v.double()) / p.sum()).to(BF16)
    assert_close_in_norm(got, want, 2.0 ** -bits)


def test_rows_without_output():
    zero = torch.zeros(2, 128)
    assert relative_norm(zero.to(BF16), zero).numel() == 0
    with pytest.raises(AssertionError):
        relative_norm(torch.ones(2, 128), zero)


@pytest.mark.parametrize("n", [300, 20000])
def test_one_key_lost_or_taken_twice_changes_a_share(n):
    values = one_hot_rows(torch.arange(n))
    lo, hi = torch.tensor([0]), torch.tensor([n])
    want = shares(values, lo, hi)
    assert_shares(want.to(BF16), want, 2.0 ** -20)
    for wrong in (torch.cat([values[:77], values[78:]]), torch.cat([values, values[77:78]])):
        got = shares(wrong, lo, torch.tensor([wrong.shape[0]]))
        with pytest.raises(AssertionError, match="shares"):
            assert_shares(got.to(BF16), want, 2.0 ** -20)
