"""The append's work units without a GPU: the last one of a call is always to spare."""

import random


def unit_base(first_row, i):
    return first_row // 64 + 2 * i


def test_the_last_unit_never_has_rows():
    """It checks cu_seqlens before it looks for its sequence, so no work of the call waits for
    that: whatever the sequence's place in its block, the unit lies behind every block that its
    rows complete, and it is not the sequence's first, which writes the tail."""
    rng = random.Random(3)
    for _ in range(5000):
        news = [rng.choice([0, 1, 2, 62, 63, 64, 65, 127, 128, 129, rng.randrange(1000)])
                for _ in range(rng.randrange(1, 8))]
        cu = [0]
        for n in news:
            cu.append(cu[-1] + n)
        tokens = max(cu[-1], 1) + rng.choice([0, 0, 1, 63, 100])
        last = unit_base(tokens, len(news)) - 1
        i = len(news) - 1
        assert unit_base(cu[i], i) <= last            # where the search leads
        j = last - unit_base(cu[i], i)
        for start in range(64):
            assert j > 0 and start // 64 + j >= (start + news[i]) // 64
