"""GPU parity of ``ulysses_attention_forward`` against attention in 64 bits."""

import pytest
import torch

from attention_reference import DIM, assert_close, attention
from flash_ulysses_b200 import FlashUlyssesContext

pytestmark = pytest.mark.gpu


def make_context(q_heads, kv_heads):
    return FlashUlyssesContext(rank=0, world_size=1, max_local_tokens=1, hidden_size=64,
                               num_heads=q_heads, num_kv_heads=kv_heads, sp_size=1)


@pytest.fixture(scope="module")
def contexts():
    made = {}

    def get(q_heads, kv_heads):
        if (q_heads, kv_heads) not in made:
            made[q_heads, kv_heads] = make_context(q_heads, kv_heads)
        return made[q_heads, kv_heads]

    yield get
    for ctx in made.values():
        ctx.check()
        ctx.close()


def rows(gen, n, heads, gain=1.0):
    return (torch.randn(n, heads * DIM, generator=gen, device="cuda") * gain).bfloat16()


def make(n, q_heads, kv_heads, seed=0, gain=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return rows(gen, n, q_heads, gain), rows(gen, n, kv_heads), rows(gen, n, kv_heads)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def slopes_of(q_heads):
    return torch.tensor([2.0 ** (-8 * (h + 1) / q_heads) for h in range(q_heads)], device="cuda")


def check(ctx, q, k, v, q_heads, kv_heads, cu=None, prefix=None, causal=True, softcap=0.0,
          slopes=None, scale=None, out=None):
    got = ctx.ulysses_attention_forward(
        q, k, v, cu_seqlens=None if cu is None else ints(cu),
        prefix_lens=None if prefix is None else ints(prefix), causal=causal, softcap=softcap,
        alibi_slopes=slopes, scale=scale, out=out)
    ctx.check()
    want, size = attention(q, k, v, q_heads, kv_heads, cu, prefix, causal,
                           DIM ** -0.5 if scale is None else scale, softcap, slopes)
    assert_close(got[:want.shape[0]], want, size)
    return got


@pytest.mark.parametrize("n", [1, 2, 31, 63, 64, 65, 127, 128, 129, 191, 255, 256, 257, 300, 383,
                               384, 385, 512, 513, 777, 1025])
@pytest.mark.parametrize("causal", [True, False])
def test_lengths(contexts, n, causal):
    check(contexts(4, 1), *make(n, 4, 1, seed=n), 4, 1, causal=causal)


@pytest.mark.parametrize("q_heads,kv_heads", [(1, 1), (8, 8), (8, 2), (8, 1), (32, 8), (3, 1),
                                              (64, 1), (6, 2)])
def test_head_groups(contexts, q_heads, kv_heads):
    check(contexts(q_heads, kv_heads), *make(333, q_heads, kv_heads), q_heads, kv_heads)


@pytest.mark.parametrize("softcap,alibi,prefix,causal", [
    (30.0, False, False, True), (30.0, False, False, False), (0.0, True, False, True),
    (0.0, True, False, False), (0.0, True, True, True), (0.0, False, True, True),
    (5.0, True, True, True), (50.0, True, False, True), (0.5, False, False, True),
])
@pytest.mark.parametrize("cu", [None, (0, 1, 1, 130, 131, 400, 700), (0, 256, 512, 640)])
def test_scores_and_masks(contexts, softcap, alibi, prefix, causal, cu):
    docs = 1 if cu is None else len(cu) - 1
    lens = None
    if prefix:
        lens = [(37 * (d + 3)) % 200 for d in range(docs)]
    check(contexts(8, 2), *make(700, 8, 2, seed=5, gain=3.0), 8, 2, cu=cu, prefix=lens,
          causal=causal, softcap=softcap, slopes=slopes_of(8) if alibi else None)


@pytest.mark.parametrize("cu,n", [
    ([0] + list(range(1, 201)), 200),                    # 200 documents of one row
    ([0, 0, 0, 5, 5, 5], 5),
    ([0, 127, 255, 256, 257, 384, 385, 1000], 1000),
    ([0, 3, 6, 10, 300, 303, 306, 310, 600], 640),
    ([0, 900, 901, 902], 1024),
])
@pytest.mark.parametrize("causal", [True, False])
def test_documents(contexts, cu, n, causal):
    check(contexts(4, 1), *make(n, 4, 1, seed=n), 4, 1, cu=cu, causal=causal)


def test_prefix_lengths_beyond_their_document(contexts):
    check(contexts(4, 1), *make(400, 4, 1), 4, 1, cu=[0, 100, 250, 400], prefix=[100, 149, 0])
    ctx = contexts(4, 1)
    q, k, v = make(400, 4, 1)
    a = ctx.ulysses_attention_forward(q, k, v, cu_seqlens=ints([0, 100, 250, 400]),
                                      prefix_lens=ints([10 ** 9, 200, -5]))
    b = ctx.ulysses_attention_forward(q, k, v, cu_seqlens=ints([0, 100, 250, 400]),
                                      prefix_lens=ints([100, 150, 0]))
    ctx.check()
    assert torch.equal(a, b)


def test_rows_behind_the_last_document_are_left(contexts):
    ctx = contexts(4, 1)
    for n, end in ((300, 200), (300, 257), (129, 1), (64, 63)):
        q, k, v = make(n, 4, 1, seed=n)
        out = torch.full((n, 4 * DIM), 7.0, dtype=torch.bfloat16, device="cuda")
        got = check(ctx, q, k, v, 4, 1, cu=[0, end], out=out)
        assert got is out and bool((out[end:] == 7.0).all())
    out = torch.full((300, 4 * DIM), 7.0, dtype=torch.bfloat16, device="cuda")
    q, k, v = make(300, 4, 1)
    ctx.ulysses_attention_forward(q, k, v, cu_seqlens=ints([0]), out=out)
    ctx.ulysses_attention_forward(q, k, v, cu_seqlens=ints([0, 0, 0]), out=out)
    ctx.check()
    assert bool((out == 7.0).all())


def test_no_rows(contexts):
    q, k, v = make(0, 4, 1)
    assert contexts(4, 1).ulysses_attention_forward(q, k, v).shape == (0, 4 * DIM)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("what", ["k", "v"])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_rows_that_are_not_seen_have_no_part(contexts, bad, what, softcap):
    """Infinities and NaN in later rows, in other documents and behind the last one; the rows that
    do see them get them."""
    n, cu = 640, [0, 150, 300, 301, 610]
    q, k, v = make(n, 4, 1, seed=3)
    x = {"k": k, "v": v}[what]
    x[140, 5] = bad
    x[299] = bad
    x[500, ::3] = bad
    x[610:] = bad
    ctx = contexts(4, 1)
    if what == "v":
        check(ctx, q, k, v, 4, 1, cu=cu, softcap=softcap)
        check(ctx, q, k, v, 4, 1, cu=cu, causal=False, softcap=softcap)
        check(ctx, q, k, v, 4, 1, cu=cu, prefix=[20, 0, 1, 250], softcap=softcap)
        return
    got = ctx.ulysses_attention_forward(q, k, v, cu_seqlens=ints(cu), softcap=softcap)
    ctx.check()
    clean = k.clone()
    clean[~clean.isfinite()] = 0
    want, size = attention(q, clean, v, 4, 1, cu, softcap=softcap)
    sees = torch.zeros(610, dtype=torch.bool, device="cuda")
    sees[140:150] = sees[299] = sees[500:] = True
    assert_close(got[:610][~sees], want[~sees], size[~sees])


def test_largest_scores(contexts):
    """Scores of several hundred: one key takes the whole weight of most rows."""
    check(contexts(4, 1), *make(500, 4, 1, gain=100.0), 4, 1, scale=1.0)
    check(contexts(4, 1), *make(500, 4, 1, gain=100.0), 4, 1, scale=1.0, softcap=30.0)
    check(contexts(4, 1), *make(500, 4, 1), 4, 1, scale=0.0)
    check(contexts(4, 1), *make(500, 4, 1), 4, 1, scale=-0.3)


def test_growing_scores(contexts):
    """Each key scores above all before it, so that the running maximum moves with every tile."""
    n = 900
    q, k, v = make(n, 4, 1)
    q[:, :] = 0.25
    k[:, :] = (torch.arange(n, device="cuda")[:, None] * 0.02).bfloat16()
    check(contexts(4, 1), q, k, v, 4, 1, scale=0.5)
    check(contexts(4, 1), q, k, v, 4, 1, scale=0.5, causal=False)
    check(contexts(4, 1), q, k, v, 4, 1, scale=-0.5)


@pytest.mark.parametrize("slope", [0.0, 1.0, 30.0])
def test_steep_slopes(contexts, slope):
    slopes = torch.full((4,), slope, device="cuda")
    check(contexts(4, 1), *make(400, 4, 1), 4, 1, slopes=slopes)
    check(contexts(4, 1), *make(400, 4, 1), 4, 1, slopes=slopes, causal=False)


def test_strided_rows(contexts):
    """Q, K and V as columns of one packed buffer, output into columns of another."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    n = 300
    packed = torch.randn(n, (8 + 2 * 2 + 1) * DIM, generator=gen, device="cuda").bfloat16()
    q, k, v = packed[:, :1024], packed[:, 1024:1280], packed[:, 1280:1536]
    wide = torch.full((n, 2048), 3.0, dtype=torch.bfloat16, device="cuda")
    out = wide[:, 512:1536]
    got = check(contexts(8, 2), q, k, v, 8, 2, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert bool((wide[:, :512] == 3).all()) and bool((wide[:, 1536:] == 3).all())


def test_offsets_beyond_32_bits(contexts):
    """Row strides that put the last rows more than 2^32 elements behind the first."""
    n, stride = 300, 1 << 24
    big = torch.empty(n * stride, dtype=torch.bfloat16, device="cuda")
    q, k, v = make(n, 4, 1)
    views = []
    for i, x in enumerate((q, k, v, torch.zeros_like(q))):
        view = big.as_strided((n, x.shape[1]), (stride, 1), i * 1024)
        view.copy_(x)
        views.append(view)
    got = contexts(4, 1).ulysses_attention_forward(*views[:3])
    # Views of one buffer overlap as ranges: as an output they are refused.
    with pytest.raises(ValueError, match="overlap"):
        contexts(4, 1).ulysses_attention_forward(*views[:3], out=views[3])
    got2 = contexts(4, 1).ulysses_attention_forward(q, k, v, out=views[3])
    contexts(4, 1).check()
    want, size = attention(q, k, v, 4, 1)
    assert_close(got, want, size)
    assert_close(got2, want, size)


@pytest.mark.parametrize("n,causal,softcap,alibi", [(5000, True, 0.0, False),
                                                    (5000, False, 0.0, False),
                                                    (4999, True, 50.0, True)])
def test_long(contexts, n, causal, softcap, alibi):
    check(contexts(3, 1), *make(n, 3, 1), 3, 1, causal=causal, softcap=softcap,
          slopes=slopes_of(3) if alibi else None)


def test_same_bits_every_time(contexts):
    q, k, v = make(2000, 8, 2)
    ctx = contexts(8, 2)
    cu = ints([0, 700, 1500, 2000])
    first = ctx.ulysses_attention_forward(q, k, v, cu_seqlens=cu)
    for _ in range(5):
        assert torch.equal(ctx.ulysses_attention_forward(q, k, v, cu_seqlens=cu), first)
    ctx.check()


def test_captured_with_other_lengths(contexts):
    """A captured call reads lengths when it is replayed; the same call on a side stream."""
    ctx = contexts(8, 2)
    q, k, v = make(600, 8, 2)
    cu, prefix = ints([0, 100, 600]), ints([50, 0])
    out = torch.zeros(600, 8 * DIM, dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ctx.ulysses_attention_forward(q, k, v, cu_seqlens=cu, prefix_lens=prefix, out=out)
    torch.cuda.current_stream().wait_stream(side)
    want, size = attention(q, k, v, 8, 2, [0, 100, 600], [50, 0])
    assert_close(out, want, size)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ctx.ulysses_attention_forward(q, k, v, cu_seqlens=cu, prefix_lens=prefix, out=out)
    for lens, pre in (([0, 100, 600], [50, 0]), ([0, 333, 500], [0, 166]), ([0, 0, 77], [3, 5])):
        cu.copy_(ints(lens))
        prefix.copy_(ints(pre))
        out.zero_()
        graph.replay()
        ctx.check()
        want, size = attention(q, k, v, 8, 2, lens, pre)
        assert_close(out[:lens[-1]], want, size)
        assert not bool(out[lens[-1]:].any())


@pytest.mark.parametrize("cu", [[1, 50, 100], [0, 80, 60], [0, 50, 101], [-3, 50, 100],
                                [0, 2 ** 31 - 1, 100]])
def test_bad_lengths_are_reported(cu):
    """The call stays inside its tensors; the next one raises until the error is cleared."""
    ctx = make_context(4, 1)
    try:
        q, k, v = make(100, 4, 1)
        ctx.ulysses_attention_forward(q, k, v, cu_seqlens=ints(cu))
        with pytest.raises(RuntimeError, match="cu_seqlens"):
            ctx.check()
        with pytest.raises(RuntimeError, match="earlier call"):
            ctx.ulysses_attention_forward(q, k, v)
        ctx.clear_error()
        check(ctx, q, k, v, 4, 1)
    finally:
        ctx.close()


@pytest.mark.parametrize("softcap", [1e-3, 0.1, 1e3, 3e4, 1e6])
@pytest.mark.parametrize("scale", [None, 1e-4])
def test_any_cap(contexts, softcap, scale):
    """Caps far above the scores leave them as they are, to FP32's precision."""
    check(contexts(4, 1), *make(300, 4, 1, gain=3.0), 4, 1, softcap=softcap, scale=scale)


@pytest.mark.parametrize("softcap", [500.0, 1e5])
def test_one_score_beyond_a_large_cap(contexts, softcap):
    """A key beyond the cap for half of the rows, in the tile of keys far below it."""
    q, k, v = make(300, 4, 1, seed=3)
    k[7] *= 3 * softcap
    k[140] *= softcap
    check(contexts(4, 1), q, k, v, 4, 1, softcap=softcap)
    check(contexts(4, 1), q, k, v, 4, 1, softcap=softcap, causal=False)


@pytest.mark.parametrize("factor", [1e-4, 0.3, 1.0, 1.45, 30.0, -0.7])
@pytest.mark.parametrize("mode", ["causal", "prefix", "full", "documents"])
def test_any_slope(contexts, factor, mode):
    """Slopes from none to ones that leave a row only itself, and a negative one."""
    options = dict(causal=mode != "full", cu=None)
    if mode == "documents":
        options["cu"] = [0, 90, 350, 351, 700]
    if mode == "prefix":
        options.update(cu=[0, 300, 700], prefix=[280, 150])
    slopes = factor * torch.tensor([1.0, 0.5, 0.03, 0.002], device="cuda")
    check(contexts(4, 1), *make(700, 4, 1, seed=11, gain=3.0), 4, 1, slopes=slopes, **options)
    check(contexts(4, 1), *make(700, 4, 1, seed=12, gain=3.0), 4, 1, slopes=slopes, softcap=8.0,
          **options)


@pytest.mark.parametrize("scale", [0.0, 1e-30, -0.1])
def test_slopes_with_any_scale(contexts, scale):
    q, k, v = make(500, 4, 1, seed=13)
    for size in (1.0, 1e-20, 1e20):
        check(contexts(4, 1), q, k, (v.float() * size).bfloat16(), 4, 1, slopes=slopes_of(4),
              scale=scale, cu=[0, 3, 260, 500])


@pytest.mark.parametrize("causal", [True, False])
def test_documents_that_share_a_warp(contexts, causal):
    """Boundaries at every place of a warp's 32 rows, long documents next to short ones."""
    cu = [0, 1, 33, 66, 100, 135, 171, 460, 463, 900, 901, 1000]
    for slopes in (None, slopes_of(4)):
        check(contexts(4, 1), *make(1024, 4, 1, seed=14, gain=2.0), 4, 1, cu=cu, causal=causal,
              slopes=slopes)


@pytest.mark.parametrize("softcap,alibi,prefix,causal", [
    (0.0, False, False, True), (0.0, False, False, False), (30.0, True, True, True),
    (5.0, False, True, True), (0.0, True, False, False), (0.0, True, True, True),
])
@pytest.mark.parametrize("cu,n", [(None, 700), ((0, 1, 1, 130, 131, 400, 700), 700),
                                  ((0, 256, 512, 640), 700), ((0, 300, 310, 600), 641)])
def test_two_tiles_an_item(contexts, softcap, alibi, prefix, causal, cu, n):
    """64 heads: enough tiles of 128 rows for two of them to share an item."""
    lens = None if not prefix else [(37 * (d + 3)) % 200 for d in range(len(cu or (0, 1)) - 1)]
    check(contexts(64, 2), *make(n, 64, 2, seed=15, gain=2.0), 64, 2, cu=cu, prefix=lens,
          causal=causal, softcap=softcap, slopes=slopes_of(64) if alibi else None)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_two_tiles_an_item_and_what_is_not_seen(contexts, bad):
    """Values that rows do not see hold infinities or NaN, in K and in V."""
    q, k, v = make(700, 64, 2, seed=16)
    clean = v.clone()
    v[100:130] = bad
    k[100:130] = bad
    cu = [0, 100, 130, 385, 650]
    ctx = contexts(64, 2)
    got = ctx.ulysses_attention_forward(q, k, v, cu_seqlens=ints(cu))
    ctx.check()
    want, size = attention(q, torch.nan_to_num(k.float()).bfloat16(), clean, 64, 2, cu)
    for a, b in ((0, 100), (130, 650)):
        assert_close(got[a:b], want[a:b], size[a:b])


@pytest.mark.parametrize("n", [1, 127, 128, 129, 255, 256, 257, 500, 513])
def test_two_tiles_an_item_lengths(contexts, n):
    heads = 296 // ((n + 127) // 128) + 1
    check(contexts(heads, 1), *make(n, heads, 1, seed=n), heads, 1)
