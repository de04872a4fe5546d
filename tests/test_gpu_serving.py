"""The operators of a serving step together, as a rank runs them: exchange, attention over packed
prompts, the cache filled from them, output projection; then decode steps over the cache."""

import pytest
import torch

from attention_reference import DIM, ReferenceCache, assert_close, attention, decode
from flash_ulysses_b200 import FlashUlyssesContext, _C
from flash_ulysses_b200.workloads import make_parameters

pytestmark = pytest.mark.gpu

H, HQ, HKV = 1024, 8, 2


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("softcap,alibi", [(0.0, False), (30.0, True)])
def test_prompts_then_decode_steps(softcap, alibi):
    """Each operator's output against 64 bits from what it was given; the projection within the
    0.01/0.01 of its own tests."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    params = make_parameters(H, (HQ + 2 * HKV) * DIM, 4096, seed=5, device="cuda")
    w_o = (torch.randn(H, HQ * DIM, generator=gen, device="cuda") * (HQ * DIM) ** -0.5).bfloat16()
    slopes = torch.tensor([2.0 ** -(h + 1) for h in range(HQ)], device="cuda") if alibi else None
    options = dict(softcap=softcap, alibi_slopes=slopes)
    ctx = FlashUlyssesContext(rank=0, world_size=1, max_local_tokens=256, hidden_size=H,
                              num_heads=HQ, num_kv_heads=HKV, sp_size=1, output_projection=True)
    try:
        cache, reference = ctx.create_kv_cache(12, 4, 4), ReferenceCache(HKV)
        cache.block_table.copy_(ints([[3, 1, 7, 0], [2, 9, 4, 8], [5, 6, 10, 11], [0, 0, 0, 0]]))
        lens, slots = [100, 127, 5], [1, 2, 0]
        cu = [0, 100, 227, 232]
        rows = 240                                         # 8 rows of padding
        x = torch.randn(rows, H, generator=gen, device="cuda").bfloat16()
        x[232:] = 0
        positions = torch.cat([torch.arange(n) for n in lens + [8]]).cuda()

        def project(attn, y):
            want = attn.double() @ w_o.double().T
            assert bool(torch.isclose(y.double(), want, atol=0.01, rtol=0.01).all())

        q, k, v = ctx.ulysses_qkv_forward(x, positions=positions, **params)
        out = torch.zeros(rows, HQ * DIM, dtype=torch.bfloat16, device="cuda")
        attn = ctx.ulysses_attention_forward(q, k, v, cu_seqlens=ints(cu), out=out, **options)
        ctx.kv_cache_append(cache, k, v, ints(slots), ints(lens), cu_seqlens=ints(cu))
        y = ctx.ulysses_o_proj_forward(attn, w_o)
        ctx.check()
        want, size = attention(q, k, v, HQ, HKV, cu, softcap=softcap, slopes=slopes)
        assert_close(attn[:232], want, size)
        assert not bool(attn[232:].any())
        project(attn, y)
        for s, a, b in zip(slots, cu, cu[1:]):
            reference.append(s, k[a:b].clone(), v[a:b].clone())

        slot_t, len_t = ints(slots), ints(lens)
        for _ in range(4):                                 # one sequence completes a block
            x = torch.randn(3, H, generator=gen, device="cuda").bfloat16()
            len_t += 1
            q, k, v = ctx.ulysses_qkv_forward(x, positions=len_t.long() - 1, **params)
            ctx.kv_cache_append(cache, k, v, slot_t, len_t)
            attn = ctx.kv_cache_attention(cache, q, slot_t, len_t, **options)
            y = ctx.ulysses_o_proj_forward(attn, w_o)
            ctx.check()
            for i, s in enumerate(slots):
                reference.append(s, k[i:i + 1].clone(), v[i:i + 1].clone())
                want, size = decode(lambda h: reference.values(s, h), q[i], HQ, HKV,
                                    softcap=softcap, slopes=slopes)
                assert_close(attn[i], want, size)
            project(attn, y)
    finally:
        ctx.close()


def test_decode_equals_the_last_row_of_the_prompt():
    """Without full blocks the cache holds what it was given, so the decode attention of the last
    token and the prompt attention's last row agree up to roundings: both are within one BF16
    rounding and the weights' of the same value."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    ctx = FlashUlyssesContext(rank=0, world_size=1, max_local_tokens=1, hidden_size=64,
                              num_heads=HQ, num_kv_heads=HKV, sp_size=1)
    try:
        cache = ctx.create_kv_cache(1, 1, 1)
        q, k, v = (torch.randn(63, h * DIM, generator=gen, device="cuda").bfloat16()
                   for h in (HQ, HKV, HKV))
        ctx.kv_cache_append(cache, k, v, ints([0]), ints([63]), cu_seqlens=ints([0, 63]))
        prompt = ctx.ulysses_attention_forward(q, k, v)
        last = ctx.kv_cache_attention(cache, q[62:], ints([0]), ints([63]))
        ctx.check()
        want, size = attention(q, k, v, HQ, HKV)
        assert_close(prompt[62:], want[62:], size[62:])
        assert_close(last, want[62:], size[62:])
    finally:
        ctx.close()


def test_both_ways_of_calling(monkeypatch):
    """Tensors are read in C where they fit and in Python where not: the same bits, and the same
    refusals."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    ctx = FlashUlyssesContext(rank=0, world_size=1, max_local_tokens=1, hidden_size=64,
                              num_heads=HQ, num_kv_heads=HKV, sp_size=1)
    assert _C.try_attention is not None
    try:
        def rows(n, h):
            return torch.randn(n, h * DIM, generator=gen, device="cuda").bfloat16()

        q, k, v, one = rows(200, HQ), rows(200, HKV), rows(200, HKV), rows(1, HQ)
        cu, pre = ints([0, 90, 200]), ints([20, 0])
        slopes = torch.rand(HQ, generator=gen, device="cuda")
        slot, length = ints([0]), ints([200])
        caches = [ctx.create_kv_cache(4, 1, 4) for _ in range(2)]
        got = []
        for cache in caches:
            cache.block_table.copy_(ints([[2, 0, 3, 1]]))
            ctx.kv_cache_append(cache, k, v, slot, length, cu_seqlens=ints([0, 200]))
            got.append((
                ctx.ulysses_attention_forward(q, k, v, cu_seqlens=cu, prefix_lens=pre, softcap=20,
                                              alibi_slopes=slopes, scale=0.1),
                ctx.kv_cache_attention(cache, one, slot, length, alibi_slopes=slopes),
                cache.k_blocks.view(torch.uint8), cache.v_tail))
            for name in ("try_attention", "try_append", "try_decode"):
                monkeypatch.setattr(_C, name, None)
        ctx.check()
        assert all(torch.equal(a, b) for a, b in zip(*got))
        monkeypatch.undo()

        cache, i64 = caches[0], slot.long()
        for call in (
                lambda: ctx.ulysses_attention_forward(q.float(), k, v),
                lambda: ctx.ulysses_attention_forward(q, k[:199], v),
                lambda: ctx.ulysses_attention_forward(q, k.cpu(), v),
                lambda: ctx.ulysses_attention_forward(q, k, v, out=q),
                lambda: ctx.ulysses_attention_forward(q, k, v, out=rows(199, HQ)),
                lambda: ctx.ulysses_attention_forward(q, k, v, cu_seqlens=cu.long()),
                lambda: ctx.ulysses_attention_forward(q, k, v, cu_seqlens=cu, prefix_lens=pre[:1]),
                lambda: ctx.ulysses_attention_forward(q, k, v, prefix_lens=pre[:1], causal=False),
                lambda: ctx.ulysses_attention_forward(q, k, v, alibi_slopes=slopes[:4]),
                lambda: ctx.ulysses_attention_forward(q, k, v, softcap=-1.0),
                lambda: ctx.ulysses_attention_forward(q, k, v, scale=float("nan")),
                lambda: ctx.kv_cache_append(cache, k, v, slot, length),
                lambda: ctx.kv_cache_append(cache, k[:1], v[:1], i64, length),
                lambda: ctx.kv_cache_append(cache, k[:1], q[:1], slot, length),
                lambda: ctx.kv_cache_attention(cache, one, slot, length.float()),
                lambda: ctx.kv_cache_attention(cache, q, slot, length),
                lambda: ctx.kv_cache_attention(cache, one, slot, length, out=one),
                lambda: ctx.kv_cache_attention(cache, one.half(), slot, length)):
            with pytest.raises(ValueError):
                call()
        # Tensors that take part in autograd, and their subclasses, are read like any other.
        grad = torch.nn.Parameter(q)
        for x in (grad, q.clone().requires_grad_()):
            assert torch.equal(ctx.ulysses_attention_forward(x, k, v),
                               ctx.ulysses_attention_forward(q, k, v))
        ctx.check()
    finally:
        ctx.close()
