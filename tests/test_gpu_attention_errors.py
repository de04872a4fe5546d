"""Attention calls whose document ends make no sense: reported whichever CTA does an item's work and
whether the first item has rows or not, and the context works on once the error is cleared."""

import pytest

from test_gpu_attention import check, ints, make, make_context

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,heads,cu", [
    (100, 4, [0, 0, -1]),                                 # no rows at all
    (100, 4, [0, 100, 0]),
    (6000, 32, [0, 1, 0]),                                # more items than run at once, few with rows
    (6000, 32, [0, 3000, 2999, 6000]),
    (6000, 32, [0, 3000, 6001]),
    (6000, 32, [1, 3000, 6000]),
    (300, 4, list(range(150)) + [148] + list(range(150, 301))),
])
def test_bad_document_ends(n, heads, cu):
    ctx = make_context(heads, heads // 4)
    try:
        q, k, v = make(n, heads, heads // 4)
        ctx.ulysses_attention_forward(q, k, v, cu_seqlens=ints(cu))
        with pytest.raises(RuntimeError, match="cu_seqlens"):
            ctx.check()
        ctx.clear_error()
        check(ctx, q[:300], k[:300], v[:300], heads, heads // 4, cu=[0, 100, 300][:2 + (n > 100)])
    finally:
        ctx.close()


def test_many_documents_are_no_error():
    ctx = make_context(4, 1)
    try:
        q, k, v = make(2000, 4, 1)
        check(ctx, q, k, v, 4, 1, cu=list(range(0, 2001)))
    finally:
        ctx.close()
