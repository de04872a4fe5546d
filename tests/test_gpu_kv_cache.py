"""GPU parity of the 8-bit K/V cache: the append bit for bit, the decode attention against 64
bits."""

import pytest
import torch

from attention_reference import (BLOCK, DIM, ReferenceCache, assert_close, decode, quantise)
from flash_ulysses_b200 import FlashUlyssesContext, KvCache

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


def ints(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def rows(gen, n, heads, gain=1.0):
    return (torch.randn(n, heads * DIM, generator=gen, device="cuda") * gain).bfloat16()


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def poisoned(cache):
    """Everything that no token has been written to holds NaN."""
    cache.k_blocks.view(torch.uint8).fill_(0x7f)
    cache.v_blocks.view(torch.uint8).fill_(0x7f)
    for t in (cache.k_scales, cache.v_scales, cache.k_tail, cache.v_tail):
        t.fill_(float("nan"))
    return cache


def fresh(ctx, max_seqs=4, max_blocks=8, spare=3, seed=0):
    cache = poisoned(ctx.create_kv_cache(max_seqs * max_blocks + spare, max_seqs, max_blocks))
    order = torch.randperm(cache.num_blocks, generator=generator(seed), device="cuda")
    cache.block_table.copy_(order[:max_seqs * max_blocks].view(max_seqs, max_blocks))
    return cache


def assert_holds(cache, reference, slots):
    """The cache's blocks, scales and tails of `slots` bit for bit."""
    for slot in slots:
        k, v = reference.rows[slot]
        n = k.shape[0]
        for x, blocks, scales, tail, swap in ((k, cache.k_blocks, cache.k_scales, cache.k_tail, 0),
                                              (v, cache.v_blocks, cache.v_scales, cache.v_tail, 1)):
            for h in range(reference.kv_heads):
                part = x[:, h * DIM:(h + 1) * DIM]
                for b in range(n // BLOCK):
                    values, scale = quantise(part[b * BLOCK:(b + 1) * BLOCK])
                    at = int(cache.block_table[slot, b])
                    got = blocks[at, h].float().double()
                    got = got.T if swap else got
                    assert torch.equal(torch.nan_to_num(got, 1e9),
                                       torch.nan_to_num(values, 1e9)), (slot, h, b)
                    assert float(scales[at, h]) == scale
                assert torch.equal(tail[slot, h, :n % BLOCK].view(torch.int16),
                                   part[n // BLOCK * BLOCK:].contiguous().view(torch.int16))


def test_append_in_any_pieces(contexts):
    """One call or many: the cache holds the same, whatever the pieces."""
    ctx = contexts(4, 2)
    gen = generator(1)
    k, v = rows(gen, 300, 2), rows(gen, 300, 2)
    reference = ReferenceCache(2)
    reference.append(2, k, v)
    for pieces in ([300], [1] * 300, [63, 1, 64, 65, 107], [64, 64, 64, 64, 44], [10, 130, 160],
                   [127, 173], [62, 3, 235]):
        cache, at = fresh(ctx), 0
        for n in pieces:
            ctx.kv_cache_append(cache, k[at:at + n], v[at:at + n], ints([2]), ints([at + n]),
                                cu_seqlens=ints([0, n]))
            at += n
        ctx.check()
        assert_holds(cache, reference, [2])
        assert bool(cache.k_tail[[0, 1, 3]].isnan().all())


def test_append_ragged_batches(contexts):
    """Batches with empty and padded sequences, rows behind the last one, strided rows."""
    ctx = contexts(8, 2)
    gen = generator(2)
    cache, reference = fresh(ctx, max_seqs=6), ReferenceCache(2)
    lens = [0] * 6
    for step, news in enumerate(([5, 0, 130, 64, 1], [60, 1, 0, 63, 200], [1, 62, 3, 65, 100])):
        slots = [4, 0, 5, 2, 1]
        cu = [0]
        for n in news:
            cu.append(cu[-1] + n)
        packed = rows(gen, cu[-1] + 7, 6)
        k, v = packed[:, 2 * DIM:4 * DIM], packed[:, 4 * DIM:]
        padded = step == 1
        for i, (s, n) in enumerate(zip(slots, news)):
            if padded and i == 3:
                continue
            lens[s] += n
            reference.append(s, k[cu[i]:cu[i + 1]], v[cu[i]:cu[i + 1]])
        given = [-1 if padded and i == 3 else s for i, s in enumerate(slots)]
        ctx.kv_cache_append(cache, k, v, ints(given), ints([lens[s] for s in slots]),
                            cu_seqlens=ints(cu))
    ctx.check()
    assert_holds(cache, reference, slots)


@pytest.mark.parametrize("count", [31, 32, 33, 64, 100, 1025])
def test_append_many_sequences(contexts, count):
    """The search of a work unit's sequence over more of them than a warp looks at at once."""
    ctx = contexts(4, 1)
    gen = generator(count)
    cache, reference = fresh(ctx, max_seqs=count, max_blocks=2), ReferenceCache(1)
    news = [(37 * i * i) % 90 for i in range(count)]
    cu = [0]
    for n in news:
        cu.append(cu[-1] + n)
    k, v = rows(gen, cu[-1] + 3, 1), rows(gen, cu[-1] + 3, 1)
    ctx.kv_cache_append(cache, k, v, ints(range(count)), ints(news), cu_seqlens=ints(cu))
    ctx.check()
    for i in range(count):
        reference.append(i, k[cu[i]:cu[i + 1]], v[cu[i]:cu[i + 1]])
    assert_holds(cache, reference, range(count))


def test_append_single_tokens(contexts):
    """Decode steps of a batch at different places of their blocks, one row padded."""
    ctx = contexts(8, 2)
    gen = generator(3)
    cache, reference = fresh(ctx, max_seqs=5), ReferenceCache(2)
    lens = {0: 0, 1: 60, 3: 62, 4: 127}
    for s, n in lens.items():
        if n:
            k, v = rows(gen, n, 2), rows(gen, n, 2)
            reference.append(s, k, v)
            ctx.kv_cache_append(cache, k, v, ints([s]), ints([n]), cu_seqlens=ints([0, n]))
    for _ in range(70):
        k, v = rows(gen, 5, 2), rows(gen, 5, 2)
        order = [3, 0, -7, 4, 1]
        for i, s in enumerate(order):
            if s >= 0:
                lens[s] += 1
                reference.append(s, k[i:i + 1], v[i:i + 1])
        ctx.kv_cache_append(cache, k, v, ints(order), ints([lens.get(s, 0) for s in order]))
    ctx.check()
    assert_holds(cache, reference, lens)


@pytest.mark.parametrize("gain", [1e-38, 1e-30, 1e-3, 1.0, 448.0, 1e30])
def test_scales(contexts, gain):
    """Powers of two over BF16's range; amounts on either side of 448 times a power."""
    ctx = contexts(4, 2)
    cache, reference = fresh(ctx), ReferenceCache(2)
    k, v = rows(generator(4), 256, 2, gain), rows(generator(5), 256, 2, gain)
    v[64:128] = 0
    k[128:192] = gain
    k[130, 3] = 1.75 * 2.0 ** 5
    k[192:] *= 0
    k[200, 130] = 1.7578125 * 2.0 ** 5
    reference.append(0, k, v)
    ctx.kv_cache_append(cache, k, v, ints([0]), ints([256]), cu_seqlens=ints([0, 256]))
    ctx.check()
    assert_holds(cache, reference, [0])


def test_infinities_and_nan_are_kept_as_nan(contexts):
    ctx = contexts(4, 2)
    cache, reference = fresh(ctx), ReferenceCache(2)
    k, v = rows(generator(6), 128, 2), rows(generator(7), 128, 2)
    k[3, 7], k[70, 200], v[5, 9] = float("inf"), float("-inf"), float("nan")
    v[64:] = float("inf")
    reference.append(1, k, v)
    ctx.kv_cache_append(cache, k, v, ints([1]), ints([128]), cu_seqlens=ints([0, 128]))
    ctx.check()
    assert_holds(cache, reference, [1])


# ------------------------------------------------------------------ decode
def filled(ctx, lens, kv_heads, seed=0, max_blocks=None, gain=1.0):
    """A cache with `lens[i]` tokens in slot `slots[i]`, and what it holds."""
    gen = generator(seed)
    if max_blocks is None:
        max_blocks = max(max(lens), 1) // BLOCK + 1
    cache = fresh(ctx, max_seqs=len(lens) + 2, max_blocks=max_blocks, seed=seed)
    slots = torch.randperm(len(lens) + 2, generator=gen, device="cuda")[:len(lens)].tolist()
    reference = ReferenceCache(kv_heads)
    k, v = rows(gen, sum(lens), kv_heads, gain), rows(gen, sum(lens), kv_heads, gain)
    cu = [0]
    for s, n in zip(slots, lens):
        cu.append(cu[-1] + n)
        reference.append(s, k[cu[-2]:cu[-1]], v[cu[-2]:cu[-1]])
    ctx.kv_cache_append(cache, k, v, ints(slots), ints(lens), cu_seqlens=ints(cu))
    return cache, reference, slots


def check_decode(ctx, cache, reference, slots, lens, q_heads, kv_heads, seed=9, q=None, out=None,
                 gain=1.0, **options):
    if q is None:
        q = rows(generator(seed), len(slots), q_heads, gain)
    got = ctx.kv_cache_attention(cache, q, ints(slots), ints(lens), out=out, **options)
    ctx.check()
    names = dict(scale="scale", softcap="softcap", alibi_slopes="slopes")
    same = {names[n]: x for n, x in options.items()}
    for i, s in enumerate(slots):
        if s < 0:
            continue
        n = lens[i]
        if n == 0:
            assert not bool(got[i].any())
            continue
        whole = reference.rows[s][0].shape[0]
        assert n == whole
        want, size = decode(lambda h: reference.values(s, h), q[i], q_heads, kv_heads, **same)
        assert_close(got[i], want, size)
    return got


LENGTHS = [1, 2, 63, 64, 65, 100, 127, 128, 129, 192, 300, 1000]


@pytest.mark.parametrize("q_heads,kv_heads", [(4, 1), (8, 2), (1, 1), (8, 1), (16, 1), (32, 8),
                                              (17, 1), (64, 1), (8, 8), (3, 1), (24, 2)])
def test_decode_lengths_and_groups(contexts, q_heads, kv_heads):
    ctx = contexts(q_heads, kv_heads)
    cache, reference, slots = filled(ctx, LENGTHS, kv_heads)
    check_decode(ctx, cache, reference, slots, LENGTHS, q_heads, kv_heads)


@pytest.mark.parametrize("n", [1, 64, 100, 4096, 20000])
def test_decode_one_sequence(contexts, n):
    ctx = contexts(4, 1)
    cache, reference, slots = filled(ctx, [n], 1)
    check_decode(ctx, cache, reference, slots, [n], 4, 1)


@pytest.mark.parametrize("softcap,alibi,gain", [(30.0, False, 3.0), (0.0, True, 1.0),
                                                (5.0, True, 3.0), (50.0, False, 1.0),
                                                (0.5, False, 1.0)])
def test_decode_scores(contexts, softcap, alibi, gain):
    ctx = contexts(8, 2)
    lens = [1, 64, 90, 700, 2000]
    cache, reference, slots = filled(ctx, lens, 2)
    slopes = torch.tensor([2.0 ** -(h + 1) for h in range(8)], device="cuda")
    options = dict(alibi_slopes=slopes) if alibi else {}
    check_decode(ctx, cache, reference, slots, lens, 8, 2, softcap=softcap, gain=gain, **options)


@pytest.mark.parametrize("max_blocks", [1, 2, 4, 5])
@pytest.mark.parametrize("q_heads,kv_heads", [(8, 2), (17, 1)])
def test_decode_short_tables(contexts, max_blocks, q_heads, kv_heads):
    """Tables of up to four blocks are not split over warps, longer ones are."""
    ctx = contexts(q_heads, kv_heads)
    lens = [64 * max_blocks, 64 * max_blocks - 1, 1, 63, 0, 64 * max_blocks - 63]
    cache, reference, slots = filled(ctx, lens, kv_heads, max_blocks=max_blocks)
    check_decode(ctx, cache, reference, slots, lens, q_heads, kv_heads)


def test_decode_many_sequences(contexts):
    ctx = contexts(8, 2)
    lens = [(37 * i * i + 11) % 500 for i in range(300)]
    cache, reference, slots = filled(ctx, lens, 2)
    check_decode(ctx, cache, reference, slots, lens, 8, 2)


def test_decode_uneven_lengths(contexts):
    """One long sequence among short ones."""
    ctx = contexts(8, 2)
    lens = [3] * 20 + [30000] + [70] * 20
    cache, reference, slots = filled(ctx, lens, 2)
    check_decode(ctx, cache, reference, slots, lens, 8, 2)


def test_decode_values_of_any_size(contexts):
    """Block scales from 2^-100 up: a value's size is its block's own."""
    ctx = contexts(4, 1)
    lens = [640]
    for gain in (1e-30, 1e-3, 1e3, 1e30):
        gen = generator(3)
        cache, reference = fresh(ctx, max_blocks=16), ReferenceCache(1)
        k, v = rows(gen, 640, 1), rows(gen, 640, 1, gain)
        v[128:192] *= 1e-3
        reference.append(1, k, v)
        ctx.kv_cache_append(cache, k, v, ints([1]), ints([640]), cu_seqlens=ints([0, 640]))
        check_decode(ctx, cache, reference, [1], lens, 4, 1)
    for gain in (1e-20, 1e20):
        gen = generator(3)
        cache, reference = fresh(ctx, max_blocks=16), ReferenceCache(1)
        k, v = rows(gen, 640, 1, gain), rows(gen, 640, 1)
        reference.append(1, k, v)
        ctx.kv_cache_append(cache, k, v, ints([1]), ints([640]), cu_seqlens=ints([0, 640]))
        check_decode(ctx, cache, reference, [1], lens, 4, 1, scale=0.09 / gain)
        q = (rows(generator(8), 1, 4).float() / gain).bfloat16()
        check_decode(ctx, cache, reference, [1], lens, 4, 1, q=q, scale=0.09)


def test_decode_largest_scores(contexts):
    ctx = contexts(4, 1)
    lens = [700, 100]
    cache, reference, slots = filled(ctx, lens, 1)
    check_decode(ctx, cache, reference, slots, lens, 4, 1, scale=1.0, gain=20.0)
    check_decode(ctx, cache, reference, slots, lens, 4, 1, scale=0.0)
    check_decode(ctx, cache, reference, slots, lens, 4, 1, scale=-0.2)


def test_decode_padded_rows_and_repeated_slots(contexts):
    ctx = contexts(8, 2)
    lens = [100, 0, 300]
    cache, reference, slots = filled(ctx, lens, 2)
    order = [slots[2], -1, slots[0], slots[1], slots[2], -5]
    given = [300, 77, 100, 0, 300, 0]
    out = torch.full((6, 8 * DIM), 7.0, dtype=torch.bfloat16, device="cuda")
    got = check_decode(ctx, cache, reference, order, given, 8, 2, out=out)
    assert got is out and bool((out[1] == 7).all()) and bool((out[5] == 7).all())


def test_decode_strided_rows(contexts):
    ctx = contexts(8, 2)
    lens = [100, 65, 300]
    cache, reference, slots = filled(ctx, lens, 2)
    packed = rows(generator(1), 3, 12)
    wide = torch.full((3, 2048), 3.0, dtype=torch.bfloat16, device="cuda")
    check_decode(ctx, cache, reference, slots, lens, 8, 2, q=packed[:, 256:1280],
                 out=wide[:, 8:1032])
    assert bool((wide[:, :8] == 3).all()) and bool((wide[:, 1032:] == 3).all())


def test_decode_nan_stays_in_its_sequence(contexts):
    """A NaN in one sequence's cache, and NaN in all memory that holds no token."""
    ctx = contexts(4, 1)
    lens = [200, 200, 70]
    gen = generator(4)
    cache, reference = fresh(ctx), ReferenceCache(1)
    for s, n in enumerate(lens):
        k, v = rows(gen, n, 1), rows(gen, n, 1)
        if s == 1:
            v[10, 3] = float("nan")
            v[195, 5] = float("nan")
        reference.append(s, k, v)
        ctx.kv_cache_append(cache, k, v, ints([s]), ints([n]), cu_seqlens=ints([0, n]))
    check_decode(ctx, cache, reference, [0, 1, 2], lens, 4, 1)


def test_no_sequences(contexts):
    ctx = contexts(4, 1)
    cache = fresh(ctx)
    none = ints([])
    q, k = rows(generator(0), 0, 4), rows(generator(0), 0, 1)
    assert ctx.kv_cache_attention(cache, q, none, none).shape == (0, 4 * DIM)
    ctx.kv_cache_append(cache, k, k, none, none)
    ctx.kv_cache_append(cache, k, k, none, none, cu_seqlens=ints([0]))
    ctx.check()
    assert bool(cache.k_tail.isnan().all())


def test_offsets_beyond_32_bits():
    """Blocks and tails more than 2^32 bytes into the cache."""
    ctx = make_context(8, 8)
    try:
        cache = ctx.create_kv_cache(70000, 40000, 4)         # 4.6 GB of K blocks, 5.2 GB of tails
        cache.block_table[39999] = ints([69999, 69998, 3, 69000])
        gen = generator(0)
        k, v = rows(gen, 200, 8), rows(gen, 200, 8)
        reference = ReferenceCache(8)
        reference.append(39999, k, v)
        ctx.kv_cache_append(cache, k, v, ints([39999]), ints([200]), cu_seqlens=ints([0, 200]))
        check_decode(ctx, cache, reference, [39999], [200], 8, 8)
        assert_holds(cache, reference, [39999])
    finally:
        ctx.close()


def test_captured_steps_and_two_streams(contexts):
    """A decode step (append, then attention) captured once and replayed while the lengths grow;
    two captured calls that run at the same time."""
    ctx = contexts(8, 2)
    lens = [62, 190, 5]
    cache, reference, slots = filled(ctx, lens, 2, max_blocks=8)
    k, v, q = (rows(generator(i), 3, h) for i, h in ((1, 2), (2, 2), (3, 8)))
    slot_t, len_t = ints(slots), ints(lens)
    out = torch.zeros(3, 8 * DIM, dtype=torch.bfloat16, device="cuda")
    step = torch.cuda.CUDAGraph()
    with torch.cuda.graph(step):
        len_t += 1
        ctx.kv_cache_append(cache, k, v, slot_t, len_t)
        ctx.kv_cache_attention(cache, q, slot_t, len_t, out=out)
    for i in range(70):
        gen = generator(100 + i)
        for t, h in ((k, 2), (v, 2), (q, 8)):
            t.copy_(rows(gen, 3, h))
        step.replay()
        for j, s in enumerate(slots):
            lens[j] += 1
            reference.append(s, k[j:j + 1].clone(), v[j:j + 1].clone())
        if i % 10 == 0 or 60 < lens[0] % 64:
            torch.cuda.synchronize()
            for j, s in enumerate(slots):
                want, size = decode(lambda h: reference.values(s, h), q[j], 8, 2)
                assert_close(out[j], want, size)
    ctx.check()
    assert_holds(cache, reference, slots)

    graphs, outs, want = [], [], []
    for i in range(2):
        qi = rows(generator(50 + i), 3, 8)
        want.append(ctx.kv_cache_attention(cache, qi, slot_t, len_t))
        outs.append(torch.zeros_like(want[i]))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            for _ in range(20):
                ctx.kv_cache_attention(cache, qi, slot_t, len_t, out=outs[i])
        graphs.append((graph, torch.cuda.Stream(), qi))
    torch.cuda.synchronize()
    for graph, stream, _ in graphs:
        with torch.cuda.stream(stream):
            graph.replay()
    ctx.check()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_same_bits_every_time(contexts):
    ctx = contexts(8, 2)
    lens = [3000, 100, 5, 900]
    cache, _, slots = filled(ctx, lens, 2)
    q = rows(generator(2), 4, 8)
    first = ctx.kv_cache_attention(cache, q, ints(slots), ints(lens))
    for _ in range(5):
        assert torch.equal(ctx.kv_cache_attention(cache, q, ints(slots), ints(lens)), first)
    ctx.check()


# ------------------------------------------------------------------ reported errors
def state_of(cache):
    return [t.view(torch.uint8).clone() for t in (
        cache.k_blocks, cache.v_blocks, cache.k_scales, cache.v_scales, cache.k_tail,
        cache.v_tail)]


@pytest.mark.parametrize("slots,lens,cu,match,kept", [
    ([0, 4], [1, 1], None, "outside", [0]),              # no such slot
    ([0, 1], [1, 0], None, "do not fit", [0]),           # a length below the new tokens
    ([0, 1], [1, 513], None, "do not fit", [0]),         # longer than the table
    ([0, 0], [1, 1], None, "twice", [0]),
    ([2, 1, 2], [1, 1, 1], None, "twice", [2, 1]),
    ([0, 1], [1, -5], None, "do not fit", [0]),
    ([0, 1], [1, 1], [0, 1, 3], "do not fit", [0]),      # rows outside the call
    ([0, 1], [1, 1], [0, 1, 0], "do not fit", [0]),
    ([0, 1], [1, 1], [-1, 1, 2], "do not fit", [1]),
])
def test_append_reports_and_skips(slots, lens, cu, match, kept):
    ctx = make_context(4, 1)
    try:
        cache = fresh(ctx)
        before = state_of(cache)
        k, v = rows(generator(1), len(slots), 1), rows(generator(2), len(slots), 1)
        ctx.kv_cache_append(cache, k, v, ints(slots), ints(lens),
                            cu_seqlens=None if cu is None else ints(cu))
        with pytest.raises(RuntimeError, match=match):
            ctx.check()
        with pytest.raises(RuntimeError, match="earlier call"):
            ctx.kv_cache_append(cache, k, v, ints([0, 1, 2][:len(slots)]), ints(lens))
        for t, old, name in zip(state_of(cache), before,
                                ("kb", "vb", "ks", "vs", "k_tail", "v_tail")):
            if name in ("k_tail", "v_tail"):
                for s in range(4):
                    if s not in kept:
                        assert torch.equal(t[s], old[s]), (name, s)
            else:
                assert torch.equal(t, old), name
        for s in kept:
            row = slots.index(s)
            assert torch.equal(cache.k_tail[s, 0, 0], k[row])
    finally:
        ctx.close()


@pytest.mark.parametrize("block", [-1, 35, 2 ** 31 - 1])
def test_blocks_outside_the_cache_are_reported(block):
    ctx = make_context(4, 1)
    try:
        cache = fresh(ctx)
        assert cache.num_blocks == 35
        good = int(cache.block_table[1, 1])
        cache.block_table[1, 1] = block
        before = state_of(cache)
        k, v = rows(generator(1), 200, 1), rows(generator(2), 200, 1)
        ctx.kv_cache_append(cache, k, v, ints([1]), ints([200]), cu_seqlens=ints([0, 200]))
        with pytest.raises(RuntimeError, match="outside"):
            ctx.check()
        mine = [int(cache.block_table[1, b]) for b in (0, 2)]
        others = [b for b in range(35) if b not in mine]
        for t, old in zip(state_of(cache)[:4], before[:4]):
            assert torch.equal(t[others], old[others])
        ctx.clear_error()
        q = rows(generator(3), 1, 4)
        got = ctx.kv_cache_attention(cache, q, ints([1]), ints([200]))
        with pytest.raises(RuntimeError, match="outside"):
            ctx.check()
        assert bool(got.isfinite().all())
        ctx.clear_error()
        cache.block_table[1, 1] = good
        ctx.kv_cache_append(cache, k, v, ints([1]), ints([200]), cu_seqlens=ints([0, 200]))
        reference = ReferenceCache(1)
        reference.append(1, k, v)
        check_decode(ctx, cache, reference, [1], [200], 4, 1)
    finally:
        ctx.close()


@pytest.mark.parametrize("slots,lens,match", [([0, 4], [1, 1], "outside"),
                                              ([0, 1], [1, 513], "do not fit"),
                                              ([0, 1], [1, -1], "do not fit")])
def test_decode_reports_and_skips(slots, lens, match):
    ctx = make_context(4, 1)
    try:
        cache, reference = fresh(ctx), ReferenceCache(1)
        k, v = rows(generator(1), 1, 1), rows(generator(2), 1, 1)
        reference.append(0, k, v)
        ctx.kv_cache_append(cache, k, v, ints([0]), ints([1]))
        out = torch.full((2, 4 * DIM), 7.0, dtype=torch.bfloat16, device="cuda")
        q = rows(generator(3), 2, 4)
        ctx.kv_cache_attention(cache, q, ints(slots), ints(lens), out=out)
        with pytest.raises(RuntimeError, match=match):
            ctx.check()
        assert bool((out[1] == 7).all())
        want, size = decode(lambda h: reference.values(0, h), q[0], 4, 1)
        assert_close(out[0], want, size)
    finally:
        ctx.close()


@pytest.mark.parametrize("softcap", [1e-3, 0.1, 1e3, 3e4, 1e6])
@pytest.mark.parametrize("q_heads,kv_heads", [(8, 2), (12, 1)])
def test_decode_any_cap(contexts, softcap, q_heads, kv_heads):
    """Caps far above the scores leave them as they are, to FP32's precision."""
    ctx = contexts(q_heads, kv_heads)
    lens = [50, 64, 700]
    cache, reference, slots = filled(ctx, lens, kv_heads)
    check_decode(ctx, cache, reference, slots, lens, q_heads, kv_heads, gain=3.0, softcap=softcap)


@pytest.mark.parametrize("softcap", [500.0, 1e5])
def test_decode_one_score_beyond_a_large_cap(contexts, softcap):
    """A key of the unfinished block beyond the cap for half of the rows."""
    ctx = contexts(8, 1)
    gen = generator(21)
    n = 3 * BLOCK + 40
    k, v = rows(gen, n, 1), rows(gen, n, 1)
    k[3 * BLOCK + 5] *= 3 * softcap
    cache, reference = fresh(ctx, max_seqs=2, max_blocks=4, seed=1), ReferenceCache(1)
    reference.append(1, k, v)
    ctx.kv_cache_append(cache, k, v, ints([1]), ints([n]), cu_seqlens=ints([0, n]))
    check_decode(ctx, cache, reference, [1], [n], 8, 1, softcap=softcap)


@pytest.mark.parametrize("lead", [12.0, 17.0, 19.5])
@pytest.mark.parametrize("q_heads", [4, 12])
def test_decode_many_small_weights(contexts, lead, q_heads):
    """One key ahead of all others by `lead`, whose values alone make the output: weights of
    e^-lead keep their precision."""
    ctx = contexts(q_heads, 1)
    n = 10 * BLOCK + 30
    q = torch.zeros(1, q_heads, DIM, device="cuda")
    q[..., 0] = DIM ** 0.5
    q[..., 1] = 2.0 ** -17                               # small next to the row's largest
    k = torch.zeros(n, DIM, device="cuda")
    k[5, 0] = lead
    v = torch.ones(n, DIM, device="cuda")
    v[5] = 0
    q, k, v = q.view(1, -1).bfloat16(), k.bfloat16(), v.bfloat16()
    cache, reference = fresh(ctx, max_seqs=1, max_blocks=11, seed=1), ReferenceCache(1)
    reference.append(0, k, v)
    ctx.kv_cache_append(cache, k, v, ints([0]), ints([n]), cu_seqlens=ints([0, n]))
    check_decode(ctx, cache, reference, [0], [n], q_heads, 1, q=q)


def test_decode_more_sequences_than_a_launch_takes(contexts):
    """Sequences go 1024 to a launch; the launches share their scratch."""
    ctx = contexts(2, 1)
    lens = [1 + (53 * i) % 90 for i in range(1500)]
    lens[1100] = 5000
    cache, reference, slots = filled(ctx, lens, 1)
    check_decode(ctx, cache, reference, slots, lens, 2, 1)
