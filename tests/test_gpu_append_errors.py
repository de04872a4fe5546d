"""What an append does with a call that it has to refuse on the device: everything is reported, and
nothing of a sequence is lost."""

import pytest
import torch

from attention_reference import ReferenceCache
from flash_ulysses_b200 import FlashUlyssesContext
from test_gpu_kv_cache import assert_holds, fresh, generator, ints, rows, state_of

pytestmark = pytest.mark.gpu


@pytest.fixture
def ctx():
    made = FlashUlyssesContext(rank=0, world_size=1, max_local_tokens=1, hidden_size=64,
                               num_heads=8, num_kv_heads=2, sp_size=1)
    yield made
    made.close()


@pytest.mark.parametrize("bad", [0, 1, 2])
@pytest.mark.parametrize("held", [0, 30, 64, 63])
def test_a_call_with_a_block_outside_the_cache_may_be_made_again(ctx, bad, held):
    """The tail's tokens are the only copy of what an unfinished block holds, so a call that cannot
    write one of its blocks must not write over them: with the table put right the same call leaves
    what it would have left at once.  The call's other sequence is written."""
    cache, reference = fresh(ctx), ReferenceCache(2)
    gen = generator(held + bad)
    if held:
        k, v = rows(gen, held, 2), rows(gen, held, 2)
        reference.append(1, k, v)
        ctx.kv_cache_append(cache, k, v, ints([1]), ints([held]), cu_seqlens=ints([0, held]))
    ctx.check()
    n = 3 * 64 + 40 - held % 64
    at = held // 64 + bad
    good = int(cache.block_table[1, at])
    cache.block_table[1, at] = cache.num_blocks
    before = state_of(cache)
    k, v = rows(gen, n + 70, 2), rows(gen, n + 70, 2)
    reference.append(2, k[n:], v[n:])
    ctx.kv_cache_append(cache, k, v, ints([1, 2]), ints([held + n, 70]),
                        cu_seqlens=ints([0, n, n + 70]))
    with pytest.raises(RuntimeError, match="outside"):
        ctx.check()
    ctx.clear_error()
    mine = cache.block_table[1].tolist() + [int(cache.block_table[2, 0])]
    others = [b for b in range(cache.num_blocks) if b not in mine]
    assert good in others
    for t, old in zip(state_of(cache)[:4], before[:4]):
        assert torch.equal(t[others], old[others])
    if held % 64:
        for t, old in zip(state_of(cache)[4:], before[4:]):
            assert torch.equal(t[1], old[1])
    cache.block_table[1, at] = good
    reference.append(1, k[:n], v[:n])
    ctx.kv_cache_append(cache, k[:n], v[:n], ints([1]), ints([held + n]),
                        cu_seqlens=ints([0, n]))
    ctx.check()
    assert_holds(cache, reference, [1, 2])


def test_a_token_that_completes_a_block_outside_the_cache(ctx):
    """The same for a step of single tokens: the row is skipped, the batch's others are not."""
    cache, reference = fresh(ctx), ReferenceCache(2)
    gen = generator(5)
    k, v = rows(gen, 126, 2), rows(gen, 126, 2)
    for slot in (0, 1):
        reference.append(slot, k[63 * slot:63 * slot + 63], v[63 * slot:63 * slot + 63])
    ctx.kv_cache_append(cache, k, v, ints([0, 1]), ints([63, 63]), cu_seqlens=ints([0, 63, 126]))
    ctx.check()
    good = int(cache.block_table[1, 0])
    cache.block_table[1, 0] = -1
    before = state_of(cache)
    k, v = rows(gen, 2, 2), rows(gen, 2, 2)
    ctx.kv_cache_append(cache, k, v, ints([0, 1]), ints([64, 64]))
    with pytest.raises(RuntimeError, match="outside"):
        ctx.check()
    ctx.clear_error()
    for t, old in zip(state_of(cache)[4:], before[4:]):
        assert torch.equal(t[1], old[1])
    cache.block_table[1, 0] = good
    ctx.kv_cache_append(cache, k[1:], v[1:], ints([1]), ints([64]))
    ctx.check()
    for slot in (0, 1):
        reference.append(slot, k[slot:slot + 1], v[slot:slot + 1])
    assert_holds(cache, reference, [0, 1])


@pytest.mark.parametrize("cu,tokens", [([0, 1000, 0, 0], 1000), ([0, 200, 100, 150], 200),
                                       ([0, 10, 5, 10, 15, 20], 20), ([3, 10, 20], 20),
                                       ([0, 5, 21], 20), ([0, -1, 5], 20)])
def test_every_entry_of_cu_seqlens_is_checked(ctx, cu, tokens):
    """Also one that the search for a work unit's sequence passes by.  Slots that the call does not
    name, and blocks that are not theirs, stay as they were."""
    cache = fresh(ctx, max_seqs=8, max_blocks=20)
    count = len(cu) - 1
    before = state_of(cache)
    k, v = rows(generator(1), tokens, 2), rows(generator(2), tokens, 2)
    ctx.kv_cache_append(cache, k, v, ints(range(count)), ints([1000] * count),
                        cu_seqlens=ints(cu))
    with pytest.raises(RuntimeError, match="cu_seqlens"):
        ctx.check()
    ctx.clear_error()
    mine = cache.block_table[:count].flatten().tolist()
    others = [b for b in range(cache.num_blocks) if b not in mine]
    for t, old in zip(state_of(cache)[:4], before[:4]):
        assert torch.equal(t[others], old[others])
    for t, old in zip(state_of(cache)[4:], before[4:]):
        assert torch.equal(t[count:], old[count:])


def test_one_bad_entry_among_many(ctx):
    count = 1000
    cache = fresh(ctx, max_seqs=count, max_blocks=1)
    k, v = rows(generator(1), count, 2), rows(generator(2), count, 2)
    for at in (1, 333, 998):
        cu = list(range(count + 1))
        cu[at], cu[at + 1] = cu[at + 1], cu[at]
        ctx.kv_cache_append(cache, k, v, ints(range(count)), ints([2] * count),
                            cu_seqlens=ints(cu))
        with pytest.raises(RuntimeError, match="cu_seqlens"):
            ctx.check()
        ctx.clear_error()
