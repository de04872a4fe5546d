"""The attention operators' cases: what they are measured on, and their plain forms.

Three operators belong between the Ulysses exchange and the output projection:

* ``attention``: attention over the exchanged Q/K/V rows of packed documents, with a causal,
  prefix or full mask inside each document, scores capped by a tanh and/or a bias that grows with
  distance;
* ``append``: new K/V rows into a cache that holds every full block of 64 tokens of a head in
  e4m3 with one power-of-two scale, and each sequence's last, unfinished block in BF16;
* ``decode``: attention of one new token per sequence over that cache.

``run`` computes them in plain torch where ``own`` is false, and calls the package where it is
true.  Head counts are those of the package's own configurations: 32/8 heads on one GPU, 8/2, 4/1
(the same split over 4 and 8 GPUs) and 8/1 (64/8 over 8).
"""

import functools
import random

import numpy as np
import torch

own = False

DIM = 128        # head dimension
BLOCK = 64       # tokens of one cache block
E4M3_MAX = 448.0


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One short prompt on one rank of an SP-4 group: an odd length just over one row block.
        dict(name="attention-129", op="attention", tokens=129, q_heads=8, kv_heads=2, docs=1, mix=0,
             pad=0, causal=True, prefix=False, softcap=0.0, alibi=False),
        # A batch of prompts of different lengths packed into one call on a single GPU, the
        # remainder of the 4096 rows being the caller's padding.
        dict(name="attention-packed-4096", op="attention", tokens=4096, q_heads=32, kv_heads=8,
             docs=7, mix=1, pad=37, causal=True, prefix=False, softcap=0.0, alibi=False),
        # A model that caps its scores, one prompt of 8192 tokens split over 4 GPUs by heads.
        dict(name="attention-capped-8192", op="attention", tokens=8192, q_heads=8, kv_heads=2,
             docs=1, mix=0, pad=0, causal=True, prefix=False, softcap=50.0, alibi=False),
        # Prefix language modelling with a distance bias: contexts that are read in both
        # directions, each followed by a causal part.
        dict(name="attention-prefix-8191", op="attention", tokens=8191, q_heads=8, kv_heads=2,
             docs=3, mix=2, pad=0, causal=True, prefix=True, softcap=0.0, alibi=True),
        # A long prompt over 8 GPUs: 8 x 4096 tokens, 4 query heads and one K/V head on each.
        dict(name="attention-32768", op="attention", tokens=32768, q_heads=4, kv_heads=1, docs=1,
             mix=0, pad=0, causal=True, prefix=False, softcap=0.0, alibi=False),
        # One decode step's new tokens, one row for each of 128 sequences.
        dict(name="append-step-128", op="append", seqs=128, new=1, longest=2000, q_heads=8,
             kv_heads=2, mix=3),
        # Five prompts of different lengths written behind what their sequences hold already.
        dict(name="append-prompts-8192", op="append", seqs=5, new=8192, longest=500, q_heads=32,
             kv_heads=8, mix=4),
        # One sequence that has just begun: the cache holds less than two blocks.
        dict(name="decode-1x100", op="decode", seqs=1, longest=100, shortest=100, q_heads=8,
             kv_heads=2, mix=0, softcap=0.0, alibi=False),
        # A batch of a serving step on one GPU, lengths spread from a few tokens to 8192.
        dict(name="decode-64x8192", op="decode", seqs=64, longest=8192, shortest=1, q_heads=32,
             kv_heads=8, mix=5, softcap=0.0, alibi=False),
        # Few sequences with a long context, 8 query heads on one K/V head.
        dict(name="decode-3x131072", op="decode", seqs=3, longest=131072, shortest=100000,
             q_heads=8, kv_heads=1, mix=6, softcap=0.0, alibi=False),
        # Many short conversations on one rank of an SP-4 group, capped scores, distance bias.
        dict(name="decode-256x1500", op="decode", seqs=256, longest=1500, shortest=1, q_heads=8,
             kv_heads=2, mix=7, softcap=30.0, alibi=True),
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return min(high, max(low, round(low * (high / low) ** rng.random())))


def draw(rng):
    q_heads, kv_heads = rng.choice([(32, 8), (8, 2), (4, 1), (8, 1), (16, 4), (8, 8)])
    op = rng.choice(["attention", "attention", "append", "decode", "decode"])
    mix = rng.randrange(1 << 20)
    if op == "attention":
        causal = rng.random() < 0.8
        prefix = causal and rng.random() < 0.3
        pairs = 32768 ** 2 / 2 if causal and not prefix else 32768 ** 2 / 4
        tokens = _spread(rng, 1, int((2 * pairs * 4 / q_heads) ** 0.5))
        docs = min(tokens, rng.choice([1, 1, 2, 5, _spread(rng, 1, 64)]))
        pad = rng.choice([0, 0, rng.randrange(1 + (tokens - docs) // 8)])
        return dict(op=op, tokens=tokens, q_heads=q_heads, kv_heads=kv_heads, docs=docs, mix=mix,
                    pad=pad, causal=causal, prefix=prefix,
                    softcap=rng.choice([0.0, 0.0, 30.0, 50.0]), alibi=rng.random() < 0.3)
    if op == "append":
        seqs = _spread(rng, 1, 256)
        new = 1 if rng.random() < 0.5 else _spread(rng, seqs, max(seqs, 65536 // kv_heads))
        return dict(op=op, seqs=seqs, new=new, longest=_spread(rng, 1, 2000), q_heads=q_heads,
                    kv_heads=kv_heads, mix=mix)
    seqs = _spread(rng, 1, 256)
    longest = _spread(rng, 1, min(131072, 64 * 8192 * 4 // (seqs * kv_heads)))
    return dict(op=op, seqs=seqs, longest=longest, shortest=_spread(rng, 1, longest),
                q_heads=q_heads, kv_heads=kv_heads, mix=mix,
                softcap=rng.choice([0.0, 0.0, 30.0, 50.0]), alibi=rng.random() < 0.3)


def _parts(total, count, mix):
    """`count` positive lengths that add up to `total`, uneven."""
    cuts = sorted(random.Random(mix).sample(range(1, total), count - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def _documents(case):
    """(lengths, prefix lengths) of an attention case's documents."""
    lengths = _parts(case["tokens"] - case["pad"], case["docs"], case["mix"])
    rng = random.Random(case["mix"] + 1)
    return lengths, [rng.randrange(n + 1) if case["prefix"] else 0 for n in lengths]


def _lengths(case):
    """The sequences of a cache case: (tokens held before the call, new tokens)."""
    rng = random.Random(case["mix"] + 2)
    if case["op"] == "decode":
        low, high = case["shortest"], case["longest"]
        return [rng.randint(low, high) for _ in range(case["seqs"] - 1)] + [high], [0] * case["seqs"]
    held = [rng.randint(0, case["longest"]) for _ in range(case["seqs"])]
    new = [1] * case["seqs"] if case["new"] == 1 else _parts(case["new"], case["seqs"], case["mix"])
    return held, new


def work(case):
    hq, hkv = case["q_heads"], case["kv_heads"]
    if case["op"] == "attention":
        lengths, prefix = _documents(case)
        pairs = 0
        for n, p in zip(lengths, prefix):
            pairs += n * n if not case["causal"] else n * (n + 1) // 2 + p * (p - 1) // 2
        rows = sum(lengths)
        return {"bytes": rows * DIM * 2 * (2 * hq + 2 * hkv), "flops": 4 * DIM * hq * pairs}
    held, new = _lengths(case)
    if case["op"] == "append":
        size = 0
        for a, n in zip(held, new):
            full = (a + n) // BLOCK - a // BLOCK
            size += n * DIM * 2                                   # the new rows, read
            size += (a % BLOCK) * DIM * 2 if full else 0          # the unfinished block, read
            size += full * (BLOCK * DIM + 4)                      # finished blocks and scales
            size += min(n, (a + n) % BLOCK) * DIM * 2             # the new unfinished block
        return {"bytes": size * 2 * hkv, "flops": 0}
    size = sum(n // BLOCK * (BLOCK * DIM + 4) + n % BLOCK * DIM * 2 for n in held) * 2 * hkv
    size += case["seqs"] * hq * DIM * 2 * 2
    return {"bytes": size, "flops": 4 * DIM * hq * sum(held)}


# ------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _rows(gen, rows, heads, normed):
    """BF16 rows as they leave the exchange: Q and K behind an RMSNorm with learned gains."""
    x = torch.randn(rows, heads, DIM, device="cuda", generator=gen)
    if normed:
        x = x / x.square().mean(-1, keepdim=True).sqrt()
        x = x * (1 + 0.1 * torch.randn(DIM, device="cuda", generator=gen))
    return x.bfloat16().view(rows, heads * DIM)


def _slopes(case):
    """Distance slopes, a geometric series over this rank's query heads."""
    if not case["alibi"]:
        return None
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / case["q_heads"]) for h in range(case["q_heads"])],
                        device="cuda")


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = _generator(seed)
    hq, hkv = case["q_heads"], case["kv_heads"]
    state = {"case": case}
    if case["op"] == "attention":
        tokens = case["tokens"]
        lengths, prefix = _documents(case)
        state.update(q=_rows(gen, tokens, hq, True), k=_rows(gen, tokens, hkv, True),
                     v=_rows(gen, tokens, hkv, False), slopes=_slopes(case),
                     cu_seqlens=_ints(np.cumsum([0] + lengths).tolist()),
                     prefix_lens=_ints(prefix) if case["prefix"] else None,
                     out=torch.zeros(tokens, hq * DIM, dtype=torch.bfloat16, device="cuda"))
        return state
    held, new = _lengths(case)
    seqs = case["seqs"]
    # Sequences sit in slots in no particular order, their blocks anywhere in the cache.
    order = torch.randperm(seqs + 3, device="cuda", generator=gen)
    blocks = [(a + n + BLOCK - 1) // BLOCK for a, n in zip(held, new)]
    wide, count = max(blocks), sum(blocks) + 5
    slots = order[:seqs].to(torch.int32)
    ids = torch.randperm(count, device="cuda", generator=gen).to(torch.int32)
    table = torch.zeros(seqs + 3, wide, dtype=torch.int32, device="cuda")
    filled = (torch.arange(wide, device="cuda")[None, :]
              < torch.tensor(blocks, device="cuda")[:, None])
    chosen = torch.zeros(seqs, wide, dtype=torch.int32, device="cuda")
    chosen[filled] = ids[:sum(blocks)]
    table[slots.long()] = chosen
    def cache(*shape):
        # Values as quantisation leaves them: the largest of a block in [224, 448].
        x = torch.randn(*shape, device="cuda", generator=gen)
        return (x * 75).clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    def scales():
        return torch.exp2(torch.randint(-8, -5, (count, hkv), device="cuda", generator=gen).float())
    def tail():
        return _rows(gen, (seqs + 3) * BLOCK, hkv, False).view(seqs + 3, BLOCK, hkv, DIM) \
            .transpose(1, 2).contiguous()
    state.update(cache=dict(k_blocks=cache(count, hkv, BLOCK, DIM),
                            v_blocks=cache(count, hkv, DIM, BLOCK),
                            k_scales=scales(), v_scales=scales(), k_tail=tail(), v_tail=tail(),
                            block_table=table),
                 slots=slots, seq_lens=_ints([a + n for a, n in zip(held, new)]))
    if case["op"] == "append":
        rows = sum(new)
        state.update(k=_rows(gen, rows, hkv, True), v=_rows(gen, rows, hkv, False),
                     most_new=max(new),
                     cu_seqlens=None if rows == seqs else _ints(np.cumsum([0] + new).tolist()))
    else:
        state.update(q=_rows(gen, seqs, hq, True), slopes=_slopes(case))
    return state


# ------------------------------------------------------------------ one pass
@functools.lru_cache(maxsize=None)
def _context(q_heads, kv_heads):
    """The context that a rank's program holds (its own projection is not used here)."""
    from flash_ulysses_b200 import FlashUlyssesContext
    return FlashUlyssesContext(rank=0, world_size=1, max_local_tokens=1, hidden_size=64,
                               num_heads=q_heads, num_kv_heads=kv_heads, sp_size=1)


def _cache(state):
    """The cache handle that a program makes once around its cache's tensors."""
    if "handle" not in state:
        from flash_ulysses_b200 import KvCache
        state["handle"] = KvCache(**state["cache"])
    return state["handle"]


def run(state):
    case = state["case"]
    if own:
        ctx = _context(case["q_heads"], case["kv_heads"])
        if case["op"] == "attention":
            return ctx.ulysses_attention_forward(
                state["q"], state["k"], state["v"], cu_seqlens=state["cu_seqlens"],
                prefix_lens=state["prefix_lens"], causal=case["causal"], softcap=case["softcap"],
                alibi_slopes=state["slopes"], out=state["out"])
        cache = _cache(state)
        if case["op"] == "append":
            ctx.kv_cache_append(cache, state["k"], state["v"], state["slots"], state["seq_lens"],
                                cu_seqlens=state["cu_seqlens"])
            return _cache_outputs(state["cache"])
        return ctx.kv_cache_attention(cache, state["q"], state["slots"], state["seq_lens"],
                                      softcap=case["softcap"], alibi_slopes=state["slopes"])
    if case["op"] == "attention":
        return _plain_attention(state)
    if case["op"] == "append":
        return _plain_append(state)
    return _plain_decode(state)


def _cache_outputs(c):
    return {name: c[name] for name in ("k_blocks", "k_scales", "k_tail", "v_blocks", "v_scales",
                                       "v_tail")}


def _plain_scores(case, q, k, slopes, distance, visible):
    """Softmax weights [.., group, rows, keys] of q [.., group, rows, 128] and
    k [.., 1, keys, 128], all FP32."""
    s = q.mul(DIM ** -0.5) @ k.transpose(-1, -2)
    if case["softcap"]:
        s.div_(case["softcap"]).tanh_().mul_(case["softcap"])
    if slopes is not None:
        s.sub_(slopes * distance())
    s.masked_fill_(~visible, float("-inf"))
    s.sub_(s.amax(-1, keepdim=True)).exp_()
    return s.div_(s.sum(-1, keepdim=True))


def _plain_attention(state):
    case = state["case"]
    hq, hkv, rows = case["q_heads"], case["kv_heads"], case["tokens"] - case["pad"]
    def heads(x, h):
        return x[:rows].float().view(rows, h, DIM).transpose(0, 1)
    q = heads(state["q"], hq).view(hkv, hq // hkv, rows, DIM)
    k, v = (heads(state[n], hkv)[:, None] for n in ("k", "v"))
    at = torch.arange(rows, device="cuda", dtype=torch.int32)
    cu = state["cu_seqlens"]
    doc = torch.searchsorted(cu, at, right=True) - 1
    visible = doc[:, None] == doc[None, :]
    if case["causal"]:
        seen = at[None, :] <= at[:, None]
        if state["prefix_lens"] is not None:
            seen |= (at < cu[doc] + state["prefix_lens"][doc])[None, :]
        visible &= seen
    slopes = state["slopes"]
    if slopes is not None:
        slopes = slopes.view(hkv, hq // hkv, 1, 1)
    p = _plain_scores(case, q, k, slopes,
                      lambda: (at[:, None] - at[None, :]).abs().float(), visible)
    out = (p @ v).view(hq, rows, DIM).transpose(0, 1).reshape(rows, hq * DIM)
    state["out"][:rows] = out.bfloat16()
    return state["out"]


def _plain_decode(state):
    case, c = state["case"], state["cache"]
    hq, hkv, seqs = case["q_heads"], case["kv_heads"], case["seqs"]
    slots, lens = state["slots"].long(), state["seq_lens"].long()
    table = c["block_table"][slots].long()
    keys = table.shape[1] * BLOCK
    def whole(blocks, scales, tail, swap):
        # [seqs, heads, keys, 128]: the blocks' values, the tail in place of the last block.
        x = blocks[table].float() * scales[table][..., None, None]
        x = x.transpose(-1, -2) if swap else x
        last = (torch.arange(table.shape[1], device="cuda") == (lens // BLOCK)[:, None])
        x = torch.where(last[:, :, None, None, None], tail[slots].float()[:, None], x)
        return x.transpose(1, 2).reshape(seqs, hkv, 1, keys, DIM)
    k = whole(c["k_blocks"], c["k_scales"], c["k_tail"], False)
    v = whole(c["v_blocks"], c["v_scales"], c["v_tail"], True)
    q = state["q"].float().view(seqs, hkv, hq // hkv, 1, DIM)
    at = torch.arange(keys, device="cuda")
    slopes = state["slopes"]
    if slopes is not None:
        slopes = slopes.view(1, hkv, hq // hkv, 1, 1)
    visible = (at < lens[:, None])[:, None, None, None, :]
    p = _plain_scores(case, q, k, slopes, lambda: (lens[:, None] - 1 - at).abs().float()[
        :, None, None, None, :], visible)
    return (p @ v).reshape(seqs, hq * DIM).bfloat16()


def _plain_quantise(x):
    """(e4m3 values, scales) of blocks [.., tokens, 128]: the scale is the smallest power of two,
    from 2^-126 up, that brings the block's largest value to 448 or less."""
    mantissa, exponent = torch.frexp(x.abs().amax((-1, -2)))
    power = torch.where(mantissa > 0, exponent - 9 + (mantissa > E4M3_MAX / 512).int(), -126)
    scale = ((power.clamp(min=-126) + 127) << 23).int().view(torch.float32)
    return (x / scale[..., None, None]).to(torch.float8_e4m3fn), scale


def _plain_append(state):
    case, c = state["case"], state["cache"]
    hkv, seqs = case["kv_heads"], case["seqs"]
    slots, lens = state["slots"].long(), state["seq_lens"].long()
    rows = state["k"].shape[0]
    cu = state["cu_seqlens"]
    cu = torch.arange(seqs + 1, device="cuda") if cu is None else cu.long()
    at = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(cu, at, right=True) - 1
    start = lens - (cu[1:] - cu[:-1])
    place = start[seq] + at - cu[seq]                    # each new row's place in its sequence
    first = start // BLOCK
    wide = state["most_new"] // BLOCK + 2
    rel = torch.arange(wide, device="cuda")
    done = (first[:, None] + rel + 1) * BLOCK <= lens[:, None]
    ids = c["block_table"][slots[:, None], (first[:, None] + rel).clamp(
        max=c["block_table"].shape[1] - 1)].long()
    last = place >= (lens // BLOCK * BLOCK)[seq]         # rows of blocks that stay unfinished
    for new, blocks, scales, tail, swap in (
            (state["k"], "k_blocks", "k_scales", "k_tail", False),
            (state["v"], "v_blocks", "v_scales", "v_tail", True)):
        new = new.view(rows, hkv, DIM)
        work = torch.zeros(seqs, wide, BLOCK, hkv, DIM, dtype=torch.bfloat16, device="cuda")
        work[:, 0] = c[tail][slots].transpose(1, 2)
        work[seq, place // BLOCK - first[seq], place % BLOCK] = new
        full = work[done].transpose(1, 2).float()        # [blocks, heads, 64, 128]
        values, scale = _plain_quantise(full)
        values = values.view(torch.uint8)
        values = values.transpose(-1, -2) if swap else values
        c[blocks].view(torch.uint8)[ids[done]] = values
        c[scales][ids[done]] = scale
        c[tail][slots[seq[last]], :, place[last] % BLOCK] = new[last]
    return _cache_outputs(c)


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    hq, hkv = case["q_heads"], case["kv_heads"]
    group = hq // hkv

    def softmax_of(scores, head, distance):
        if case["softcap"]:
            scores = case["softcap"] * torch.tanh(scores / case["softcap"])
        if state["slopes"] is not None:
            scores = scores - state["slopes"][head].double() * distance
        return torch.softmax(scores, -1)

    if case["op"] == "attention":
        out = torch.zeros(case["tokens"], hq, DIM, dtype=torch.float64, device="cuda")
        lengths, prefix = _documents(case)
        begin = 0
        for n, p in zip(lengths, prefix):
            at = torch.arange(n, device="cuda")
            for head in range(hq):
                def take(name, h):
                    return state[name][begin:begin + n, h * DIM:(h + 1) * DIM].double()
                for r in range(0, n, 8192):
                    i = at[r:r + 8192, None]
                    s = take("q", head)[r:r + 8192] @ take("k", head // group).T / DIM ** 0.5
                    hidden = (at[None] > i) & (at[None] >= p) if case["causal"] else None
                    if case["softcap"]:
                        s = case["softcap"] * torch.tanh(s / case["softcap"])
                    if state["slopes"] is not None:
                        s = s - state["slopes"][head].double() * (i - at[None]).abs()
                    if hidden is not None:
                        s[hidden] = -torch.inf
                    out[begin + r:begin + min(n, r + 8192), head] = (
                        torch.softmax(s, -1) @ take("v", head // group))
            begin += n
        return out.view(case["tokens"], hq * DIM)

    c = state["cache"]
    held, new = _lengths(case)
    slots = state["slots"].tolist()
    if case["op"] == "decode":
        out = torch.zeros(case["seqs"], hq, DIM, dtype=torch.float64, device="cuda")
        for i, n in enumerate(held):
            ids = c["block_table"][slots[i], :n // BLOCK].long()
            at = torch.arange(n, device="cuda")
            for h in range(hkv):
                k = c["k_blocks"][ids, h].double() * c["k_scales"][ids, h, None, None].double()
                v = c["v_blocks"][ids, h].double() * c["v_scales"][ids, h, None, None].double()
                k = torch.cat([k.reshape(-1, DIM), c["k_tail"][slots[i], h, :n % BLOCK].double()])
                v = torch.cat([v.transpose(1, 2).reshape(-1, DIM),
                               c["v_tail"][slots[i], h, :n % BLOCK].double()])
                for head in range(h * group, (h + 1) * group):
                    q = state["q"][i, head * DIM:(head + 1) * DIM].double()
                    out[i, head] = softmax_of(k @ q / DIM ** 0.5, head, n - 1 - at) @ v
        return out.view(case["seqs"], hq * DIM)

    got = {name: t.double() for name, t in _cache_outputs(c).items()}
    begin = 0
    for i, (a, n) in enumerate(zip(held, new)):
        edge = (a + n) // BLOCK * BLOCK
        for kind in "kv":
            tail = got[kind + "_tail"][slots[i]]
            rows = state[kind][begin:begin + n].double().view(n, hkv, DIM).transpose(0, 1)
            # Everything from the start of the block that was unfinished.
            rows = torch.cat([tail[:, :a % BLOCK], rows], 1)
            low = a // BLOCK * BLOCK
            for b in range(low // BLOCK, edge // BLOCK):
                x = rows[:, b * BLOCK - low:(b + 1) * BLOCK - low]
                for h in range(hkv):
                    scale, top = 2.0 ** -126, float(x[h].abs().max())
                    while scale * E4M3_MAX < top:
                        scale *= 2
                    y = x[h] / scale
                    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
                    y = torch.round(y / step) * step
                    at = int(c["block_table"][slots[i], b])
                    got[kind + "_blocks"][at, h] = y if kind == "k" else y.T
                    got[kind + "_scales"][at, h] = scale
            left = rows[:, edge - low:] if edge > low else rows
            tail[:, :left.shape[1]] = left
        begin += n
    return got
