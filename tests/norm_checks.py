"""Checks that do not weaken with the number of keys, beside attention_reference's element by
element: that bound grows with the sum of p |v|, which many keys leave as it is while the output
itself shrinks, so a lost block of 64 among 20000 keys stays below it."""

import torch

DIM = 128


def relative_norm(got, want):
    """|got - want| / |want| per row and head (2-norms over the head's 128 dims); a row without
    output must be without output in both."""
    got = got.double().reshape(-1, DIM)
    want = want.double().reshape(-1, DIM)
    size = want.norm(dim=-1)
    off = (got - want).norm(dim=-1)
    assert not bool(off[size == 0].any())
    return off[size > 0] / size[size > 0]


def assert_close_in_norm(got, want, weight_eps):
    """For values v_j of independent signs.  The result's rounding to BF16 is off by 2^-8 of it at
    most.  Let a weight be off by d_j p_j, |d_j| <= w = weight_eps + 2^-10 (its own rounding, and
    FP32 scores and exponentials).  Then the sum of d_j p_j v_j has the expected square
    sum d_j^2 p_j^2 |v_j|^2 <= w^2 sum p_j^2 |v_j|^2, w^2 times that of the result.  Over 128 dims
    either norm is within 6 % of its expectation (one deviation), so their ratio is above 1.6 w less
    than once in 10^9 rows (0.6 is six and a half deviations of 9 %)."""
    off = relative_norm(got, want)
    bound = 2.0 ** -8 + 1.6 * (weight_eps + 2.0 ** -10)
    assert off.numel() == 0 or float(off.max()) <= bound, \
        f"worst {float(off.max()):.5f} of a row's norm, bound {bound:.5f}"


def one_hot_rows(classes):
    """BF16 [n, 128]: row i is 1 at dim classes[i] (mod 128) and 0 elsewhere.  With equal scores an
    attention's output then counts, dim by dim, the keys of each class."""
    x = torch.zeros(classes.shape[0], DIM, dtype=torch.bfloat16, device=classes.device)
    return x.scatter_(1, (classes % DIM).long()[:, None], 1.0)


def shares(values, lo, hi):
    """float64 [rows, 128]: the mean of values[lo_i:hi_i] for each row i."""
    total = torch.cat([torch.zeros(1, DIM, dtype=torch.float64, device=values.device),
                       values.double().cumsum(0)])
    return (total[hi] - total[lo]) / (hi - lo).clamp(min=1)[:, None]


def assert_shares(got, want, eps):
    """A share is a quotient of exact whole numbers, rounded to BF16 (2^-8 of it at most) after FP32
    arithmetic that is off by `eps` of it; what has no key is exactly 0."""
    got = got.double()
    over = (got - want).abs() > (2.0 ** -8 + eps) * want
    assert not bool(over.any()), f"{int(over.sum())} of {over.numel()} shares are wrong"
