"""Attention where its ring of K and V tiles fills in an unusual order: keys that come from memory
behind values that lie in L2, shared memory that holds NaN from the call before, and two calls at
once."""

import pytest
import torch

from test_gpu_attention import check, contexts, ints, make  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,end", [(384, 300), (640, 600), (2048, 1990)])
def test_values_that_arrive_before_the_keys(contexts, n, end):  # noqa: F811
    """The last key tile holds NaN in rows behind the documents, which no row sees."""
    ctx = contexts(32, 8)
    q, k, v = make(n, 32, 8)
    for x in (k, v):
        x[end:] = float("nan")
    nan = torch.full_like(k, float("nan"))
    cu = ints([0, end])
    want = check(ctx, q, k, v, 32, 8, cu=[0, end])[:end].clone()
    big = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    for _ in range(30):
        ctx.ulysses_attention_forward(q, nan, nan)        # what shared memory then holds
        big.zero_()                                       # everything out of L2 ..
        v.clone()                                         # .. and the values back
        got = ctx.ulysses_attention_forward(q, k, v, cu_seqlens=cu)
        assert torch.equal(got[:end], want)
    ctx.check()


def test_calls_on_two_streams(contexts):  # noqa: F811
    ctx = contexts(8, 2)
    work = []
    for n, options in ((3000, {}), (5000, dict(softcap=30.0)), (700, dict(causal=False)),
                       (2500, dict(alibi_slopes=torch.rand(8, device="cuda")))):
        q, k, v = make(n, 8, 2, seed=n)
        work.append((q, k, v, options, ctx.ulysses_attention_forward(q, k, v, **options)))
    ctx.check()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for turn in range(20):
        for s, pair in zip(streams, (work[:2], work[2:])):
            with torch.cuda.stream(s):
                for q, k, v, options, want in pair:
                    got.append((ctx.ulysses_attention_forward(q, k, v, **options), want))
    ctx.check()
    for a, b in got:
        assert torch.equal(a, b)
