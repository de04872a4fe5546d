"""Attention and the 8-bit cache in 64 bits, for the tests of the kernels."""

import math

import torch

DIM = 128
BLOCK = 64


def softmax_of(q, k, visible, distance, scale, softcap, slope):
    """Weights [rows, keys] of one head; a row that sees nothing gets zeros."""
    s = (q.double() @ k.double().T) * scale
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    if slope is not None:
        s = s - float(slope) * distance.double()
    s = torch.where(visible, s, torch.full_like(s, -math.inf))
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    return torch.where(visible.any(-1, keepdim=True), p, torch.zeros_like(p))


def weighted(p, visible, v):
    """(p @ v, p @ |v|) where a value that is not seen has no part, and an infinity or NaN that is
    seen with a weight above zero stays one."""
    v = v.double()
    fine = torch.where(v.isfinite(), v, torch.zeros_like(v))
    out = p @ fine
    seen = visible.double()
    nan, pos, neg = (seen @ x.double() > 0 for x in (v.isnan(), v == math.inf, v == -math.inf))
    out = torch.where(pos, torch.full_like(out, math.inf), out)
    out = torch.where(neg, torch.full_like(out, -math.inf), out)
    out = torch.where(nan | (pos & neg), torch.full_like(out, math.nan), out)
    return out, p @ fine.abs()


def attention(q, k, v, q_heads, kv_heads, cu_seqlens=None, prefix_lens=None, causal=True,
              scale=DIM ** -0.5, softcap=0.0, slopes=None):
    """(out, sum of p |v|), both float64 [rows of the documents, q_heads * 128]."""
    cu = [0, q.shape[0]] if cu_seqlens is None else list(cu_seqlens)
    group = q_heads // kv_heads
    out = torch.zeros(cu[-1], q_heads * DIM, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    for d, (a, b) in enumerate(zip(cu, cu[1:])):
        if a == b:
            continue
        at = torch.arange(b - a, device=q.device)
        visible = torch.ones(b - a, b - a, dtype=torch.bool, device=q.device)
        if causal:
            visible = at[None] <= at[:, None]
            if prefix_lens is not None:
                visible = visible | (at[None] < prefix_lens[d])
        distance = (at[:, None] - at[None]).abs()
        for h in range(q_heads):
            cols = slice(h * DIM, (h + 1) * DIM)
            kv = slice(h // group * DIM, (h // group + 1) * DIM)
            p = softmax_of(q[a:b, cols], k[a:b, kv], visible, distance, scale, softcap,
                           None if slopes is None else slopes[h])
            out[a:b, cols], size[a:b, cols] = weighted(p, visible, v[a:b, kv])
    return out, size


def assert_close(got, want, size, weight_eps=2.0 ** -8):
    """|got - want| within one BF16 rounding of the result (2^-8 of it) plus, for every weight,
    its rounding (`weight_eps`) and 2^-10 for the FP32 scores and exponentials: a score is a sum of
    128 products (error at most 128 * 2^-24 of the sum of their magnitudes, some 100 in these
    tests times the scale 0.09, so below 2^-13) and an exponential is good to 2^-12 or better."""
    got = got.double()
    nan = want.isnan()
    assert torch.equal(got.isnan(), nan)
    infinite = want.isinf()
    assert torch.equal(got[infinite], want[infinite])
    fine = ~nan & ~infinite
    tol = 2.0 ** -8 * want.abs() + (weight_eps + 2.0 ** -10) * size + 1e-30
    over = (got - want).abs()[fine] / tol[fine]
    assert over.numel() == 0 or float(over.max()) <= 1.0, \
        f"{int((over > 1).sum())} of {over.numel()} outside, worst {float(over.max()):.2f} x"


# ------------------------------------------------------------------ cache
def quantise(x):
    """(values, scale) of one block: float64 e4m3 values and the power of two."""
    x = x.double()
    fine = torch.where(x.isfinite(), x, torch.zeros_like(x))
    top, scale = float(fine.abs().max()), 2.0 ** -126
    while scale * 448 < top:
        scale *= 2
    y = fine / scale
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    y = torch.round(y / step) * step
    return torch.where(x.isfinite(), y, torch.full_like(y, math.nan)), scale


class ReferenceCache:
    """Every token of every slot in BF16, and what a cache of them holds."""

    def __init__(self, kv_heads):
        self.kv_heads = kv_heads
        self.rows = {}

    def append(self, slot, k, v):
        old = self.rows.get(slot)
        self.rows[slot] = ((k, v) if old is None
                           else (torch.cat([old[0], k]), torch.cat([old[1], v])))

    def values(self, slot, h):
        """(k, v) float64 [tokens, 128] of one head as the cache holds them."""
        got = []
        for x in self.rows[slot]:
            x = x[:, h * DIM:(h + 1) * DIM].double()
            for b in range(x.shape[0] // BLOCK):
                part = x[b * BLOCK:(b + 1) * BLOCK]
                y, scale = quantise(part)
                part.copy_(y * scale)
            got.append(x)
        return got


def decode(cache_values, q, q_heads, kv_heads, scale=DIM ** -0.5, softcap=0.0, slopes=None):
    """(out, sum of p |v|) of one token: cache_values(h) gives (k, v) [tokens, 128]."""
    group = q_heads // kv_heads
    out = torch.zeros(q_heads * DIM, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    for h in range(kv_heads):
        k, v = cache_values(h)
        n = k.shape[0]
        if n == 0:
            continue
        visible = torch.ones(1, n, dtype=torch.bool, device=q.device)
        distance = (n - 1 - torch.arange(n, device=q.device))[None]
        for head in range(h * group, (h + 1) * group):
            cols = slice(head * DIM, (head + 1) * DIM)
            p = softmax_of(q[None, cols], k, visible, distance, scale, softcap,
                           None if slopes is None else slopes[head])
            o, s = weighted(p, visible, v)
            out[cols], size[cols] = o[0], s[0]
    return out, size
