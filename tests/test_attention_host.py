"""Host side of the attention and cache operators without a GPU: the refusals of every argument,
the cache's own checks, the layout of the C structures, and the append's work units."""

import ctypes
import random
import re
import shutil
import subprocess
from pathlib import Path

import pytest
import torch

from flash_ulysses_b200 import FlashUlyssesContext, KvCache, _C

ROOT = Path(__file__).resolve().parent.parent
HEADER = ROOT / "include" / "flash_ulysses_b200.h"
BF16, I32, F32 = torch.bfloat16, torch.int32, torch.float32


class NoStatus:
    value = 0
    device_ptr = host_ptr = None


@pytest.fixture
def ctx(monkeypatch):
    """A context of 4 query and 2 K/V heads whose tensors are on the CPU; a launch fails."""
    c = object.__new__(FlashUlyssesContext)
    c.world_size, c.sp_size, c.num_heads, c.num_kv_heads, c.head_dim = 1, 1, 4, 2, 128
    c.device, c._status = torch.device("cpu"), NoStatus()

    def launched(*args):
        raise AssertionError("launched")

    for name in ("attention_forward", "kvcache_append", "kvcache_attention"):
        monkeypatch.setattr(_C, name, launched)
    monkeypatch.setattr(_C, "current_stream_handle", lambda index: 0)
    monkeypatch.setattr(_C, "kvcache_attention_workspace", lambda *sizes: 16)
    return c


def q_k_v(n=6):
    return (torch.zeros(n, 512, dtype=BF16), torch.zeros(n, 256, dtype=BF16),
            torch.zeros(n, 256, dtype=BF16))


def test_attention_reaches_the_launch(ctx):
    q, k, v = q_k_v()
    cu, pre = torch.tensor([0, 6], dtype=I32), torch.zeros(1, dtype=I32)
    for extra in ({}, dict(cu_seqlens=cu), dict(cu_seqlens=cu, prefix_lens=pre),
                  dict(prefix_lens=pre), dict(alibi_slopes=torch.zeros(4)), dict(softcap=30),
                  dict(out=torch.zeros(6, 512, dtype=BF16)), dict(scale=0.5, causal=False)):
        with pytest.raises(AssertionError, match="launched"):
            ctx.ulysses_attention_forward(q, k, v, **extra)
    packed = torch.zeros(6, 1024, dtype=BF16)
    with pytest.raises(AssertionError, match="launched"):
        ctx.ulysses_attention_forward(packed[:, :512], packed[:, 512:768], packed[:, 768:])


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(6, 256, dtype=BF16)), dict(q=torch.zeros(6, 512)),
    dict(q=torch.zeros(6, 4, 128, dtype=BF16)), dict(k=torch.zeros(5, 256, dtype=BF16)),
    dict(v=torch.zeros(6, 512, dtype=BF16)), dict(v=torch.zeros(256, 6, dtype=BF16).t()),
    dict(q=torch.zeros(6, 516, dtype=BF16)[:, :512]), dict(k=torch.zeros(6, 264, dtype=BF16)[:, 4:260]),
    dict(q=torch.zeros(1, 512, dtype=BF16).expand(6, 512)),
    dict(cu_seqlens=torch.zeros(3)), dict(cu_seqlens=torch.zeros(3, dtype=torch.int64)),
    dict(cu_seqlens=torch.zeros(0, dtype=I32)), dict(cu_seqlens=torch.zeros(6, dtype=I32)[::2]),
    dict(cu_seqlens=torch.zeros(3, dtype=I32), prefix_lens=torch.zeros(1, dtype=I32)),
    dict(prefix_lens=torch.zeros(1, dtype=I32), causal=False),
    dict(prefix_lens=torch.zeros(2, dtype=I32)),
    dict(alibi_slopes=torch.zeros(2)), dict(alibi_slopes=torch.zeros(4, dtype=BF16)),
    dict(softcap=-1.0), dict(softcap=float("nan")), dict(scale=float("inf")),
    dict(out=torch.zeros(6, 512)), dict(out=torch.zeros(5, 512, dtype=BF16)),
])
def test_attention_refuses(ctx, change):
    q, k, v = q_k_v()
    given = dict(q=q, k=k, v=v)
    given.update(change)
    with pytest.raises(ValueError):
        ctx.ulysses_attention_forward(given.pop("q"), given.pop("k"), given.pop("v"), **given)


def test_attention_refuses_output_over_an_input(ctx):
    q, k, v = q_k_v()
    with pytest.raises(ValueError, match="overlap"):
        ctx.ulysses_attention_forward(q, k, v, out=q)
    packed = torch.zeros(6, 1024, dtype=BF16)
    with pytest.raises(ValueError, match="overlap"):
        ctx.ulysses_attention_forward(q, packed[:, 512:768], v, out=packed[:, :512])


def test_nothing_to_do(ctx):
    """No rows, no documents, no sequences: no launch."""
    q, k, v = q_k_v(0)
    assert ctx.ulysses_attention_forward(q, k, v).shape == (0, 512)
    q, k, v = q_k_v(3)
    out = torch.ones(3, 512, dtype=BF16)
    none = torch.zeros(0, dtype=I32)
    assert ctx.ulysses_attention_forward(q, k, v, cu_seqlens=torch.zeros(1, dtype=I32),
                                         out=out) is out
    cache = KvCache.allocate(3, 2, 2, 2, "cpu")
    ctx.kv_cache_append(cache, k[:0], v[:0], none, none)
    ctx.kv_cache_append(cache, k, v, none, none, cu_seqlens=torch.zeros(1, dtype=I32))
    assert ctx.kv_cache_attention(cache, q[:0], none, none).shape == (0, 512)


def test_earlier_device_error_is_raised(ctx):
    ctx._status = NoStatus()
    ctx._status.value = 5 | (80 << 8)
    q, k, v = q_k_v()
    cache = KvCache.allocate(3, 2, 2, 2, "cpu")
    i = torch.zeros(6, dtype=I32)
    for call in (lambda: ctx.ulysses_attention_forward(q, k, v),
                 lambda: ctx.kv_cache_append(cache, k, v, i, i),
                 lambda: ctx.kv_cache_attention(cache, q, i, i)):
        with pytest.raises(RuntimeError, match="outside the K/V cache"):
            call()


# ------------------------------------------------------------------ cache
def parts(**change):
    c = KvCache.allocate(5, 3, 4, 2, "cpu")
    given = {n: getattr(c, n) for n in ("k_blocks", "v_blocks", "k_scales", "v_scales", "k_tail",
                                        "v_tail", "block_table")}
    given.update(change)
    return given


def test_cache_sizes_and_description():
    c = KvCache.allocate(5, 3, 4, 2, "cpu")
    assert (c.num_blocks, c.max_seqs, c.max_blocks, c.kv_heads) == (5, 3, 4, 2)
    assert c.k_blocks.shape == (5, 2, 64, 128) and c.v_blocks.shape == (5, 2, 128, 64)
    assert c._desc.v_tail == c.v_tail.data_ptr() and c._desc.max_blocks == 4
    assert c._address == ctypes.addressof(c._desc)
    again = KvCache(**parts())
    assert again.kv_heads == 2


@pytest.mark.parametrize("change", [
    dict(k_blocks=torch.zeros(5, 2, 64, 128, dtype=torch.uint8)),
    dict(v_blocks=torch.zeros(5, 2, 64, 128, dtype=torch.uint8).view(torch.float8_e4m3fn)),
    dict(k_scales=torch.zeros(5, 3)), dict(v_scales=torch.zeros(5, 2, dtype=BF16)),
    dict(k_tail=torch.zeros(2, 2, 64, 128, dtype=BF16)),
    dict(v_tail=torch.zeros(3, 2, 128, 64, dtype=BF16).transpose(2, 3)),
    dict(block_table=torch.zeros(3, 4, dtype=torch.int64)),
    dict(block_table=torch.zeros(2, 4, dtype=I32)),
    dict(block_table=torch.zeros(4, 3, dtype=I32).t()),
    dict(block_table=torch.zeros(12, dtype=I32)),
    dict(block_table=torch.zeros(13, dtype=I32)[1:].view(3, 4)),
])
def test_cache_refuses(change):
    with pytest.raises(ValueError):
        KvCache(**parts(**change))


def test_cache_refuses_empty_and_huge():
    with pytest.raises(ValueError):
        KvCache.allocate(0, 3, 4, 2, "cpu")
    with pytest.raises(ValueError):
        KvCache.allocate(1, 1, 1 << 25, 1, "cpu")


def test_append_and_decode_reach_the_launch(ctx):
    cache = KvCache.allocate(5, 3, 4, 2, "cpu")
    q, k, v = q_k_v()
    i = torch.zeros(6, dtype=I32)
    for call in (lambda: ctx.kv_cache_append(cache, k, v, i, i),
                 lambda: ctx.kv_cache_append(cache, k, v, i[:2], i[:2],
                                             cu_seqlens=torch.tensor([0, 2, 6], dtype=I32)),
                 lambda: ctx.kv_cache_attention(cache, q, i, i, softcap=3.0,
                                                alibi_slopes=torch.zeros(4))):
        with pytest.raises(AssertionError, match="launched"):
            call()


@pytest.mark.parametrize("call", [
    lambda c, a, q, k, v, i: c.kv_cache_append(a, k, v[:5], i, i),
    lambda c, a, q, k, v, i: c.kv_cache_append(a, q, v, i, i),
    lambda c, a, q, k, v, i: c.kv_cache_append(a, k, v, i[:5], i[:5]),
    lambda c, a, q, k, v, i: c.kv_cache_append(a, k, v, i, i[:5]),
    lambda c, a, q, k, v, i: c.kv_cache_append(a, k, v, i.long(), i),
    lambda c, a, q, k, v, i: c.kv_cache_append(a, k, v, i, i.float()),
    lambda c, a, q, k, v, i: c.kv_cache_append(a, k, v, i[:2], i[:2], cu_seqlens=i[:2]),
    lambda c, a, q, k, v, i: c.kv_cache_append(a, k, v, i.view(2, 3), i),
    lambda c, a, q, k, v, i: c.kv_cache_append(KvCache.allocate(5, 3, 4, 4, "cpu"), k, v, i, i),
    lambda c, a, q, k, v, i: c.kv_cache_append(KvCache.allocate(5, 3, 4, 2, "meta"), k, v, i, i),
    lambda c, a, q, k, v, i: c.kv_cache_attention(a, k, i, i),
    lambda c, a, q, k, v, i: c.kv_cache_attention(a, q.float(), i, i),
    lambda c, a, q, k, v, i: c.kv_cache_attention(a, q, i[:5], i),
    lambda c, a, q, k, v, i: c.kv_cache_attention(a, q, i, i[:5]),
    lambda c, a, q, k, v, i: c.kv_cache_attention(a, q, i, i, softcap=-2.0),
    lambda c, a, q, k, v, i: c.kv_cache_attention(a, q, i, i, alibi_slopes=torch.zeros(2)),
    lambda c, a, q, k, v, i: c.kv_cache_attention(a, q, i, i, out=q),
    lambda c, a, q, k, v, i: c.kv_cache_attention(a, q, i, i, out=q[:5].clone()),
    lambda c, a, q, k, v, i: c.kv_cache_attention(KvCache.allocate(5, 3, 4, 1, "cpu"), q, i, i),
])
def test_append_and_decode_refuse(ctx, call):
    cache = KvCache.allocate(5, 3, 4, 2, "cpu")
    q, k, v = q_k_v()
    with pytest.raises(ValueError):
        call(ctx, cache, q, k, v, torch.zeros(6, dtype=I32))


# ------------------------------------------------------------------ C ABI
def test_struct_layouts_match_the_header(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no C compiler")
    lines = []
    for cls, name in ((_C.AttentionArgs, "fu_attention_args"), (_C.KvCacheDesc, "fu_kvcache")):
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        for field, *_ in cls._fields_:
            lines.append(f'printf("{name}.{field} %zu\\n", offsetof({name}, {field}));')
    src = tmp_path / "probe.c"
    src.write_text('#include <stdio.h>\n#include "flash_ulysses_b200.h"\nint main(void) {\n'
                   + "\n".join(lines) + "\nreturn 0;\n}\n")
    exe = tmp_path / "probe"
    subprocess.run([gcc, "-I", str(HEADER.parent), str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run(
        [str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    for cls, name in ((_C.AttentionArgs, "fu_attention_args"), (_C.KvCacheDesc, "fu_kvcache")):
        assert int(got[name]) == ctypes.sizeof(cls)
        for field, *_ in cls._fields_:
            assert int(got[f"{name}.{field}"]) == getattr(cls, field).offset, field


def test_constants_and_status_codes_match_the_header():
    text = HEADER.read_text()
    assert int(re.search(r"#define FU_KV_BLOCK (\d+)", text).group(1)) == _C.FU_KV_BLOCK
    for name, code, word in (("LENGTHS", 4, "cu_seqlens"), ("CACHE_RANGE", 5, "block"),
                             ("SLOT_TWICE", 6, "twice")):
        assert re.search(rf"FU_STATUS_{name} = {code}\b", text)
        assert word in _C.decode_status(code)


def args(**change):
    a = _C.AttentionArgs()
    a.q_heads, a.kv_heads, a.tokens, a.docs, a.causal, a.scale = 4, 2, 6, 1, 1, 0.1
    a.q = a.k = a.v = a.out = 4096
    a.q_stride = a.out_stride = 512
    a.k_stride = a.v_stride = 256
    for n, x in change.items():
        setattr(a, n, x)
    return a


@pytest.mark.parametrize("change", [
    dict(q_heads=3), dict(kv_heads=0), dict(tokens=0), dict(tokens=(1 << 30) + 1), dict(docs=0),
    dict(docs=2), dict(causal=0, prefix_lens=4096), dict(softcap=-1.0), dict(scale=float("nan")),
    dict(q=None), dict(out=4098), dict(k=4104), dict(q_stride=504), dict(v_stride=260),
])
def test_c_attention_refuses(change):
    """Refused on the host, before any CUDA call."""
    rc = _C.lib.fu_attention_forward(ctypes.byref(args(**change)), 0, None)
    assert rc == _C.FU_ERR_INVALID and _C.last_error()
    assert _C.lib.fu_attention_forward(None, 0, None) == _C.FU_ERR_INVALID


def description(**change):
    d = _C.KvCacheDesc()
    d.kv_heads, d.num_blocks, d.max_seqs, d.max_blocks = 2, 5, 3, 4
    for n in ("k_blocks", "v_blocks", "k_scales", "v_scales", "k_tail", "v_tail", "block_table"):
        setattr(d, n, 4096)
    for n, x in change.items():
        setattr(d, n, x)
    return d


@pytest.mark.parametrize("cache,change", [
    (dict(kv_heads=0), {}), (dict(max_blocks=1 << 25), {}), (dict(k_tail=None), {}),
    (dict(v_blocks=4104), {}), ({}, dict(tokens=5)), ({}, dict(tokens=0)), ({}, dict(seqs=0)),
    ({}, dict(k=None)), ({}, dict(k_stride=128)), ({}, dict(slots=None)),
    ({}, dict(seq_lens=None)),
])
def test_c_append_refuses(cache, change):
    d = description(**cache)
    a = dict(k=4096, v=4096, k_stride=256, v_stride=256, tokens=6, slots=4096, seq_lens=4096,
             cu=None, seqs=6)
    a.update(change)
    rc = _C.lib.fu_kvcache_append(ctypes.addressof(d), *a.values(), None, None, 0, None)
    assert rc == _C.FU_ERR_INVALID and _C.last_error()


@pytest.mark.parametrize("change", [
    dict(q=None), dict(q_stride=256), dict(out=4100), dict(q_heads=3), dict(seqs=0),
    dict(slots=None), dict(softcap=-1.0), dict(work=None), dict(nbytes=0),
])
def test_c_decode_refuses(change):
    d = description()
    a = dict(q=4096, q_stride=512, out=4096, out_stride=512, q_heads=4, slots=4096, seq_lens=4096,
             seqs=6, scale=0.1, softcap=0.0, slopes=None, work=4096, nbytes=1 << 40)
    a.update(change)
    rc = _C.lib.fu_kvcache_attention(ctypes.addressof(d), *a.values(), None, None, 0, None)
    assert rc == _C.FU_ERR_INVALID and _C.last_error()
    assert _C.lib.fu_kvcache_attention_workspace(0, 3, 2, 1) == 0
    assert _C.lib.fu_kvcache_attention_workspace(0, 4, 2, 0) == 0


# ------------------------------------------------------------------ append units
def unit_base(first_row, i):
    return first_row // 64 + 2 * i


def test_append_units_cover_every_block():
    """Each sequence's units (from its row offset and index alone) are enough for every block its
    rows can touch, wherever in a block they start, and the grid is enough for all."""
    rng = random.Random(0)
    for _ in range(2000):
        news = [rng.choice([0, 1, 2, 62, 63, 64, 65, 127, 128, 129, rng.randrange(1000)])
                for _ in range(rng.randrange(1, 20))]
        cu = [0]
        for n in news:
            cu.append(cu[-1] + n)
        tokens = cu[-1] + rng.choice([0, 1, 100])
        grid = unit_base(tokens, len(news))
        for i, n in enumerate(news):
            first, after = unit_base(cu[i], i), unit_base(cu[i + 1], i + 1)
            assert after <= grid
            for start in range(64):
                touched = (start + n - 1) // 64 + 1 if n else 0
                assert touched <= after - first
        # The kernel's search: the last sequence whose units start at or before the unit.
        for unit in range(grid):
            a, b = 0, len(news)
            while b - a > 1:
                mid = (a + b) // 2
                if unit_base(cu[mid], mid) <= unit:
                    a = mid
                else:
                    b = mid
            assert unit_base(cu[a], a) <= unit
            assert a == len(news) - 1 or unit < unit_base(cu[a + 1], a + 1)


# ------------------------------------------------------------------ decode dealing
def pair_cost(n):
    return 0 if n <= 0 else 1 + 2 * (n // 64) + (4 if n % 64 else 0)


def block_start(b):
    return 0 if b == 0 else 1 + 2 * b


def blocks_before(x):
    return 0 if x <= 0 else 1 if x <= 3 else x // 2


def test_blocks_before_counts_the_starts():
    starts = [block_start(b) for b in range(400)]
    assert all(b - a <= 3 for a, b in zip(starts, starts[1:]))
    for x in range(300):
        assert blocks_before(x) == sum(s < x for s in starts)


def test_decode_deals_every_block_once():
    """The split's arithmetic, restated: every block of every (sequence, pair) goes to one warp,
    a warp has at most one partial of each kind, and the join finds them where they are."""
    rng = random.Random(1)
    for _ in range(400):
        seqs, pairs = rng.choice([1, 2, 3, 10, 50, 200]), rng.choice([1, 2, 8])
        workers = rng.choice([8, 64, 1184])
        lens = [rng.choice([0, 0, 1, 63, 64, 65, 100, 1000, rng.randrange(8000)])
                for _ in range(seqs)]
        first = [0]
        for n in lens:
            first.append(first[-1] + pair_cost(n) * pairs)
        aligned = seqs * pairs <= workers // 4
        over = workers - seqs * pairs if aligned else workers
        share = max(-(-first[-1] // over), 3)
        unit = [0]
        for n in lens:
            nb = -(-n // 64)
            unit.append(unit[-1] + ((block_start(nb - 1) // share + 1) * pairs if nb else 0))
        assert not aligned or unit[-1] <= workers
        got, partial = {}, {}
        for w in range(workers):
            if aligned:
                if w >= unit[-1]:
                    continue
                i = max(k for k in range(seqs) if unit[k] <= w)
                per = block_start(-(-lens[i] // 64) - 1) // share + 1
                pair, part = divmod(w - unit[i], per)
                at = first[i] + pair * pair_cost(lens[i]) + part * share
                end = min(at + share, first[i] + (pair + 1) * pair_cost(lens[i]))
            else:
                at = w * share
                if at >= first[-1]:
                    continue
                end = min(at + share, first[-1])
                i = max(k for k in range(seqs) if first[k] <= at)
            while at < end:
                while first[i + 1] <= at:
                    i += 1
                nb, cost = -(-lens[i] // 64), pair_cost(lens[i])
                pair = (at - first[i]) // cost
                base = first[i] + pair * cost
                b0, b1 = blocks_before(at - base), min(nb, blocks_before(end - base))
                at = base + cost
                for b in range(b0, b1):
                    assert (i, pair, b) not in got
                    got[i, pair, b] = w
                if b0 < b1 and b1 - b0 < nb:
                    assert (w, b0 == 0) not in partial
                    partial[w, b0 == 0] = i, pair
        assert len(got) == sum(-(-n // 64) for n in lens) * pairs
        for i, n in enumerate(lens):
            if n == 0:
                continue
            last = block_start(-(-n // 64) - 1)
            for pair in range(pairs):
                if aligned:
                    per = last // share + 1
                    c0 = unit[i] + pair * per
                    c1 = c0 + per
                else:
                    base = first[i] + pair_cost(n) * pair
                    c0, c1 = base // share, (base + last) // share + 1
                if c1 - c0 == 1:
                    assert got[i, pair, 0] == got[i, pair, -(-n // 64) - 1] == c0
                else:
                    assert all(partial[c, c == c0] == (i, pair) for c in range(c0, c1))


@pytest.mark.parametrize("change", [dict(softcap=1e-4), dict(softcap=1e7), dict(scale=1e31),
                                    dict(scale=2e9, softcap=1.0), dict(scale=float("nan")),
                                    dict(softcap=float("inf"))])
def test_scores_that_leave_the_range_are_refused(ctx, change):
    q, k, v = q_k_v()
    with pytest.raises(ValueError, match="within"):
        ctx.ulysses_attention_forward(q, k, v, **change)
    cache = ctx.create_kv_cache(4, 2, 2)
    i = torch.zeros(6, dtype=I32)
    with pytest.raises(ValueError, match="within"):
        ctx.kv_cache_attention(cache, q, i, i, **change)


def test_a_cache_keeps_its_tensors(ctx):
    cache = ctx.create_kv_cache(4, 2, 2)
    before = cache.block_table
    with pytest.raises(AttributeError, match="copy into them"):
        cache.block_table = torch.zeros(2, 2, dtype=I32)
    assert cache.block_table is before
