"""Every key counts, and counts once: attention and decode attention over values that show each key
by itself, and over random ones with a bound that long contexts do not loosen."""

import pytest
import torch

from attention_reference import DIM, attention, decode
from norm_checks import assert_close_in_norm, assert_shares, one_hot_rows, shares
from test_gpu_attention import contexts, make  # noqa: F401  (a fixture)
from test_gpu_kv_cache import filled, fresh, generator, ints, rows

pytestmark = pytest.mark.gpu


def seen(n, cu, prefix, causal):
    """[lo, hi) of every row that belongs to a document."""
    at = torch.arange(n, device="cuda")
    ends = torch.tensor([0, n] if cu is None else cu, device="cuda")
    doc = torch.searchsorted(ends, at, right=True) - 1
    lo, hi = ends[doc.clamp(max=len(ends) - 2)], ends[(doc + 1).clamp(max=len(ends) - 1)]
    if causal:
        hi = at + 1 if prefix is None else torch.maximum(
            at + 1, torch.minimum(lo + torch.tensor(prefix, device="cuda")[
                doc.clamp(max=len(ends) - 2)], hi))
    return lo, hi, int(ends[-1])


@pytest.mark.parametrize("mode", ["plain", "cap", "bias", "both"])
@pytest.mark.parametrize("n,cu,prefix,causal", [
    (5000, None, None, True),
    (5000, None, None, False),
    (2000, None, None, True),
    (2000, None, [700], True),
    (5000, [0, 1, 1, 130, 131, 1500, 4900], [0, 3, 1, 129, 200, 5000], True),
    (1800, [0, 300, 301, 1000, 1771], None, False),
    (1800, [0, 300, 301, 1000, 1771], None, True),
])
def test_attention_counts_every_key_once(contexts, mode, n, cu, prefix, causal):  # noqa: F811
    """Scores are all 0 (q is), so each weight is 1 over the row's keys; where values are 1 in one dim
    the output is a share of them.  K/V head 0 tells the rows apart modulo 128, head 1 blocks of 32.
    An exponential is good to 2^-13, rounds to 1 as a weight, and only its sum is not exact."""
    ctx = contexts(8, 2)
    q, k, _ = make(n, 8, 2)
    at = torch.arange(n, device="cuda")
    values = [one_hot_rows(at), one_hot_rows(at // 32)]
    options = {}
    if mode in ("cap", "both"):
        options["softcap"] = 20.0
    if mode in ("bias", "both"):
        options["alibi_slopes"] = torch.zeros(8, device="cuda")
    got = ctx.ulysses_attention_forward(
        torch.zeros_like(q), k, torch.cat(values, 1), causal=causal,
        cu_seqlens=None if cu is None else ints(cu),
        prefix_lens=None if prefix is None else ints(prefix), **options)
    ctx.check()
    lo, hi, end = seen(n, cu, prefix, causal)
    for h in range(8):
        want = shares(values[h // 4], lo[:end], hi[:end])
        assert_shares(got[:end, h * DIM:(h + 1) * DIM], want, 2.0 ** -13)


@pytest.mark.parametrize("n,causal,softcap", [(5000, True, 0.0), (5000, False, 0.0),
                                              (4000, True, 30.0), (1500, True, 0.0)])
def test_attention_in_norm(contexts, n, causal, softcap):  # noqa: F811
    ctx = contexts(8, 2)
    q, k, v = make(n, 8, 2, seed=n)
    got = ctx.ulysses_attention_forward(q, k, v, causal=causal, softcap=softcap)
    ctx.check()
    want, _ = attention(q, k, v, 8, 2, causal=causal, softcap=softcap)
    assert_close_in_norm(got, want, 2.0 ** -8)


LENS = [[20000], [64], [1], [100, 1, 63, 64, 65, 4096, 7777], [3] * 20 + [30000] + [70] * 20,
        [1 + 37 * i % 1500 for i in range(256)]]


@pytest.mark.parametrize("softcap", [0.0, 30.0, 1000.0])
@pytest.mark.parametrize("q_heads", [8, 24])
@pytest.mark.parametrize("lens", LENS, ids=len)
def test_decode_counts_every_key_once(contexts, lens, q_heads, softcap):  # noqa: F811
    """As above; head 0 tells the tokens apart modulo 128, head 1 the blocks.  Ones and zeros are
    exact in e4m3, equal weights are a power of two, and all sums are whole."""
    ctx = contexts(q_heads, 2)
    cache = fresh(ctx, max_seqs=len(lens), max_blocks=max(lens) // 64 + 1)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    at = torch.cat([torch.arange(n, device="cuda") for n in lens])
    values = [one_hot_rows(at), one_hot_rows(at // 64)]
    k = rows(generator(1), cu[-1], 2)
    slots = list(reversed(range(len(lens))))
    ctx.kv_cache_append(cache, k, torch.cat(values, 1), ints(slots), ints(lens),
                        cu_seqlens=ints(cu))
    q = torch.zeros(len(lens), q_heads * DIM, dtype=torch.bfloat16, device="cuda")
    got = ctx.kv_cache_attention(cache, q, ints(slots), ints(lens), softcap=softcap)
    ctx.check()
    lo, hi = (torch.tensor(x, device="cuda") for x in (cu[:-1], cu[1:]))
    for h in range(q_heads):
        want = shares(values[h // (q_heads // 2)], lo, hi)
        assert_shares(got[:, h * DIM:(h + 1) * DIM], want, 2.0 ** -18)


@pytest.mark.parametrize("q_heads", [8, 24])
@pytest.mark.parametrize("lens", LENS[:-1], ids=len)
def test_decode_in_norm(contexts, lens, q_heads):  # noqa: F811
    ctx = contexts(q_heads, 2)
    cache, reference, slots = filled(ctx, lens, 2, seed=len(lens))
    q = rows(generator(7), len(lens), q_heads)
    got = ctx.kv_cache_attention(cache, q, ints(slots), ints(lens))
    ctx.check()
    for i, s in enumerate(slots):
        want, _ = decode(lambda h: reference.values(s, h), q[i], q_heads, 2)
        assert_close_in_norm(got[i], want, 2.0 ** -11)
