"""Attention calls whose document ends make no sense: reported wherever the entry lies, whichever CTA
does an item's work and whether items have rows or not, and the context works on once the error is
cleared."""

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


@pytest.mark.parametrize("n,heads,docs", [(4000, 4, 4000), (4000, 32, 4000), (40, 4, 3001),
                                          (6000, 32, 11)])
def test_one_bad_end_anywhere(n, heads, docs):
    """A single entry below the one before it; there are more and fewer of them than items."""
    ctx = make_context(heads, heads // 4)
    try:
        q, k, v = make(n, heads, heads // 4)
        good = [n * d // docs for d in range(docs + 1)]
        for at in sorted({1, 2, 31, 32, 33, docs // 2, docs - 1, docs}):
            if not 0 < at <= docs:
                continue
            cu = list(good)
            cu[at] = cu[at - 1] - 1
            ctx.ulysses_attention_forward(q, k, v, cu_seqlens=ints(cu))
            with pytest.raises(RuntimeError, match="cu_seqlens"):
                ctx.check()
            ctx.clear_error()
        ctx.ulysses_attention_forward(q, k, v, cu_seqlens=ints(good))
        ctx.check()
    finally:
        ctx.close()
