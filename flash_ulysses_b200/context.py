"""Collective receive-buffer ownership and the public QKV interface.

Drop-in for the reference's ``flash_ulysses.context.FlashUlyssesContext``
(joey-shao/flash_ulysses ``flash_ulysses/context.py:9-174``): same constructor
keywords, properties, ``ulysses_qkv_forward`` signature, output aliasing and
``close()`` semantics.  Differences, all deliberate:

* requires an sm_100 GPU (B200) instead of SM90 (context.py:59-60);
* also admits ``sp_size == world_size == 1`` (a self-exchange on one GPU);
  the reference requires ``sp_size >= 2`` (context.py:40);
* receive buffers are plain ``cudaMalloc`` allocations shared through CUDA IPC
  handles exchanged on ``control_group`` instead of ThunderKittens'
  broker-based ``TKParallelTensor``; the exit barrier is fused into the kernel
  and uses per-call epoch flags instead of a separate multicast barrier
  launch;
* a device-side wait that gives up (``timeout_s``, default 30 s) or a
  position outside the RoPE cache sets a status word; the next call (or
  ``check()``) raises ``RuntimeError`` instead of hanging, and
  ``ulysses_qkv_forward(..., check=True)`` raises for the failing call itself.
  A call that starts on the device after an earlier call gave up a wait (one
  queued behind a failed call) stores nothing into any receive buffer and
  waits for no peer.

Added (no counterpart in the reference): ``ulysses_attention_forward`` is the
attention over the exchanged rows, ``kv_cache_append`` and
``kv_cache_attention`` keep an 8-bit K/V cache and attend to it one token per
sequence, and with ``output_projection=True`` ``ulysses_o_proj_forward`` runs
the inverse exchange after attention fused with the attention output
projection.
"""

from __future__ import annotations

import functools

import torch
import torch.distributed as dist

from . import _C
from .kv_cache import KvCache


def _rows(name, t, rows, width, index):
    """(address, row stride) of a BF16 [rows, width] tensor; raises on any other."""
    if t.dtype is not torch.bfloat16 or t.shape != (rows, width) or t.get_device() != index:
        raise ValueError(f"{name} must be a BF16 tensor of shape {(rows, width)} on the "
                         f"context's device")
    row, column = t.stride()
    if rows == 1:
        row = width
    ptr = t.data_ptr()
    if column != 1 or row < width or row % 8 or ptr % 16:
        raise ValueError(f"{name} must be 16-byte aligned with contiguous rows whose stride is a "
                         "multiple of 8 elements")
    return ptr, row


def _vector(name, t, dtype, length, index):
    """Address of a contiguous vector of `length` elements; raises on any other."""
    if (t.dtype is not dtype or t.shape != (length,) or not t.is_contiguous()
            or t.get_device() != index):
        raise ValueError(f"{name} must be a contiguous {dtype} vector of {length} elements on "
                         "the context's device")
    return t.data_ptr()


def _like_rows(t, stride, width):
    """A new contiguous tensor of t's shape."""
    if stride == width:
        return torch.empty_like(t)
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _no_overlap(rows, out, out_stride, out_width, t, stride, width):
    if rows and (out < t + 2 * ((rows - 1) * stride + width)
                 and t < out + 2 * ((rows - 1) * out_stride + out_width)):
        raise ValueError("out must not overlap an input")


def _check_cache(cache, kv_width, device):
    if ((cache.device is not device and cache.device != device)
            or cache.kv_heads * _C.FU_HEAD_DIM != kv_width):
        raise ValueError(f"the cache must hold {kv_width // _C.FU_HEAD_DIM} K/V heads on {device}")


class FlashUlyssesContext:
    """Construct, call and close collectively on one B200 node.

    rank and world_size describe the participating physical GPUs on this node.
    control_group must cover those same participants for lifecycle barriers and
    the exchange of buffer handles.  Calls use the current CUDA stream.  Results
    alias Q/K/V until the next call or close.  Before reuse, every physical rank
    must finish consuming its previous output.
    """

    def __init__(
        self,
        *,
        rank,
        world_size,
        max_local_tokens,
        hidden_size=4096,
        num_heads=32,
        num_kv_heads=8,
        head_dim=128,
        sp_size=2,
        control_group=None,
        timeout_s=30.0,
        output_projection=False,
    ):
        self.rank, self.world_size = rank, world_size
        self.control_group = control_group
        self.hidden_size = hidden_size
        self.num_heads, self.num_kv_heads = num_heads, num_kv_heads
        self.head_dim, self.sp_size = head_dim, sp_size
        self.max_local_tokens = max_local_tokens
        self._op = None
        self._oproj = None
        self._status = None
        self._views = {}
        self.Q = self.K = self.V = self.barrier = None
        self.G = self.o_barrier = None

        if not 1 <= sp_size <= self.world_size <= 8 or self.world_size % sp_size:
            raise ValueError("SP must divide a single-node world of 1 to 8 GPUs")
        if hidden_size <= 0 or hidden_size % 64 or head_dim != 128:
            raise ValueError("Requires hidden_size > 0 divisible by 64 and head_dim=128")
        if (
            num_heads <= 0
            or num_kv_heads <= 0
            or num_heads % num_kv_heads
            or num_heads % self.world_size
            or num_kv_heads % self.world_size
        ):
            raise ValueError("Q heads must divide by KV heads; both must divide by world_size")
        if max_local_tokens <= 0:
            raise ValueError("max_local_tokens must be positive")
        if not 0 <= rank < world_size:
            raise ValueError("rank must be in [0, world_size)")
        self.device = torch.device("cuda", torch.cuda.current_device())
        if torch.cuda.get_device_capability(self.device) != (10, 0):
            raise ValueError("Requires SM100 (B200)")

        group_start = rank // sp_size * sp_size
        self.sp_rank = rank - group_start
        peers = list(range(group_start, group_start + sp_size))
        capacity = sp_size * max_local_tokens

        def parallel(shape, dtype):
            return _C.ParallelTensor(shape, dtype, rank, world_size, False,
                                     group=control_group, peers=peers, device=self.device)

        self.Q = parallel((capacity, self.output_q_heads * head_dim), torch.bfloat16)
        self.K = parallel((capacity, self.output_kv_heads * head_dim), torch.bfloat16)
        self.V = parallel((capacity, self.output_kv_heads * head_dim), torch.bfloat16)
        # Per-rank synchronisation block: epoch flags written by SP peers and a
        # CTA completion counter (layout in include/flash_ulysses_b200.h).
        self.barrier = parallel((_C.FU_SYNC_WORDS,), torch.int32)
        self.barrier.data_.zero_()
        self._status = _C.StatusWord()

        topo = _C.Topology()
        topo.device = self.device.index
        topo.sp_size = sp_size
        topo.sp_rank = self.sp_rank
        topo.q_heads = self.local_q_heads
        topo.kv_heads = self.local_kv_heads
        topo.hidden_size = hidden_size
        topo.capacity_rows = capacity
        for i, r in enumerate(peers):
            topo.q_recv[i] = self.Q.peer_ptr(r)
            topo.k_recv[i] = self.K.peer_ptr(r)
            topo.v_recv[i] = self.V.peer_ptr(r)
            topo.sync[i] = self.barrier.peer_ptr(r)
        topo.status = self._status.device_ptr
        topo.status_host = self._status.host_ptr
        topo.timeout_ns = int(timeout_s * 1e9)
        self._op = _C.QkvOp(topo)

        if output_projection:
            if hidden_size % 256:
                raise ValueError("output_projection requires hidden_size divisible by 256")
            # Gather buffer (peers push this rank's rows of their heads into it)
            # and a separate synchronisation block with per-m-block ready counters.
            self.G = parallel((max_local_tokens, self.local_q_heads * head_dim), torch.bfloat16)
            self.o_barrier = parallel((_C.oproj_sync_words(max_local_tokens),), torch.int32)
            self.o_barrier.data_.zero_()
            otopo = _C.OprojTopology()
            otopo.device = self.device.index
            otopo.sp_size = sp_size
            otopo.sp_rank = self.sp_rank
            otopo.q_heads = self.local_q_heads
            otopo.hidden_size = hidden_size
            otopo.max_local_tokens = max_local_tokens
            for i, r in enumerate(peers):
                otopo.gather[i] = self.G.peer_ptr(r)
                otopo.sync[i] = self.o_barrier.peer_ptr(r)
            otopo.status = self._status.device_ptr
            otopo.status_host = self._status.host_ptr
            otopo.timeout_ns = int(timeout_s * 1e9)
            self._oproj = _C.OprojOp(otopo)

        torch.cuda.current_stream(self.device).synchronize()
        if world_size > 1 or dist.is_initialized():
            dist.barrier(group=control_group)

    @property
    def base_tp_size(self):
        return self.world_size // self.sp_size

    @property
    def local_q_heads(self):
        return self.num_heads // self.base_tp_size

    @property
    def local_kv_heads(self):
        return self.num_kv_heads // self.base_tp_size

    @property
    def output_q_heads(self):
        return self.num_heads // self.world_size

    @property
    def output_kv_heads(self):
        return self.num_kv_heads // self.world_size

    @property
    def packed_width(self):
        return (self.local_q_heads + 2 * self.local_kv_heads) * self.head_dim

    @property
    def epoch(self):
        """Number of calls made so far (the value published to peers)."""
        return self._op.epoch

    @torch.no_grad()
    def ulysses_qkv_forward(
        self,
        hidden_states,
        qkv_weight,
        positions,
        q_norm_weight,
        k_norm_weight,
        rope_cache,
        *,
        q_epsilon=1e-6,
        k_epsilon=1e-6,
        check=False,
        static_weights=False,
        _projection_out=None,
    ):
        """Return BF16 (q, k, v), each with L * sp_size rows.

        Inputs are contiguous CUDA tensors on the current/context device:
        hidden_states BF16 [L, H], qkv_weight BF16 [H, packed_width],
        positions int64 [L], norm weights FP32 [128], and a NeoX RoPE cache
        FP32 [max_position, 128] containing [cos(64), sin(64)]. Positions must
        index the cache. Epsilons must be positive. The caller crops padding.

        ``check=True`` waits for this call to finish on the current stream
        and raises ``RuntimeError`` if it reported a device-side error (a peer
        that never joined it, a position outside the cache), so the caller
        learns that these outputs are invalid; by default errors surface on
        the next call or ``check()``, without a synchronisation per call.

        ``static_weights=True`` is the caller's promise that no kernel that
        may still be running on the current stream writes ``qkv_weight``
        (inference, where weights do not change): the first stages of the
        weight are then read while the previous kernel finishes, which
        shortens decode-sized calls.  Results are the same; without the
        promise holding, a call may read stale weights.

        ``_projection_out`` is test instrumentation: a BF16 [L, packed_width]
        tensor that also receives this rank's BF16 projection ``x @ W``.
        """
        local_tokens = hidden_states.shape[0]
        if not 0 < local_tokens <= self.max_local_tokens:
            raise ValueError("Input length must be within [1, max_local_tokens]")
        if self._status.value:
            raise RuntimeError("an earlier call failed on the device: "
                               + _C.decode_status(self._status.value))
        _C.launch(hidden_states, qkv_weight, positions, q_norm_weight, k_norm_weight,
                  rope_cache, self._op, q_epsilon=q_epsilon, k_epsilon=k_epsilon,
                  flags=_C.FU_FWD_STATIC_WEIGHTS if static_weights else 0,
                  gemm_out=_projection_out)
        if check:
            torch.cuda.current_stream(self.device).synchronize()
            if self._status.value:
                raise RuntimeError("this call failed on the device: "
                                   + _C.decode_status(self._status.value))
        views = self._views.get(local_tokens)
        if views is None:
            output_tokens = local_tokens * self.sp_size
            views = tuple(t.data()[:output_tokens] for t in (self.Q, self.K, self.V))
            self._views = {local_tokens: views}      # row views of the receive buffers
        return views

    @torch.no_grad()
    def ulysses_o_proj_forward(self, attn_output, o_proj_weight, *, out=None):
        """Inverse Ulysses exchange fused with the attention output projection
        (no counterpart in the reference, which stops at the forward exchange).

        ``attn_output`` is this rank's attention output, BF16
        ``[L * sp_size, output_q_heads * 128]`` in the layout of the ``q``
        returned by ``ulysses_qkv_forward`` (rows ``s*L..`` belong to SP member
        ``s``); ``o_proj_weight`` is BF16 ``[hidden_size, local_q_heads * 128]``
        (nn.Linear layout).  Returns BF16 ``[L, hidden_size]`` =
        ``gathered @ o_proj_weight.T`` for this rank's L tokens, written into
        ``out`` when given.  Requires ``output_projection=True`` at
        construction; every rank of the SP group makes the same calls.
        ``attn_output`` is only read during this rank's call.
        """
        if self._oproj is None:
            raise RuntimeError("construct the context with output_projection=True")
        rows = attn_output.shape[0]
        if rows % self.sp_size:
            raise ValueError("attn_output rows must be a multiple of sp_size")
        local_tokens = rows // self.sp_size
        if not 0 < local_tokens <= self.max_local_tokens:
            raise ValueError("Input length must be within [1, max_local_tokens]")
        # The kernel's tensor maps are built from these shapes, so a tensor of
        # another shape, dtype or layout would be read or written out of bounds.
        k = self.local_q_heads * self.head_dim
        for name, t, shape in (
                ("attn_output", attn_output, (rows, self.output_q_heads * self.head_dim)),
                ("o_proj_weight", o_proj_weight, (self.hidden_size, k)),
                ("out", out, (local_tokens, self.hidden_size))):
            if t is None:
                continue
            if (tuple(t.shape) != shape or t.dtype != torch.bfloat16 or not t.is_contiguous()
                    or t.device != self.device):
                raise ValueError(f"{name} must be a contiguous BF16 tensor of shape {shape} "
                                 f"on {self.device}")
        if self._status.value:
            raise RuntimeError("an earlier call failed on the device: "
                               + _C.decode_status(self._status.value))
        if out is None:
            out = torch.empty(local_tokens, self.hidden_size, dtype=torch.bfloat16,
                              device=self.device)
        stream = _C.current_stream_handle(self.device.index)
        self._oproj.forward(attn_output.data_ptr(), o_proj_weight.data_ptr(), local_tokens,
                            out.data_ptr(), 0, stream)
        return out

    # ------------------------------------------------------------ attention
    # These calls are a few microseconds on the GPU at decode sizes, so their
    # checks ask each tensor only once for what they need.
    @functools.cached_property
    def _widths(self):
        """Columns of Q and of K/V rows, and the device index (-1: the CPU)."""
        index = self.device.index
        return (self.output_q_heads * self.head_dim, self.output_kv_heads * self.head_dim,
                -1 if index is None else index)

    @functools.cached_property
    def _head_counts(self):
        return self.output_q_heads, self.output_kv_heads

    @functools.cached_property
    def _default_scale(self):
        return self.head_dim ** -0.5

    @functools.cached_property
    def _attention_scratch(self):
        """Bytes of the decode attention's scratch."""
        return _C.kvcache_attention_workspace(self._widths[2], self.output_q_heads,
                                              self.output_kv_heads, 1)

    def _score_options(self, scale, softcap, alibi_slopes):
        scale = self.head_dim ** -0.5 if scale is None else float(scale)
        softcap = float(softcap)
        if not abs(scale) <= 1e30:
            raise ValueError("scale must be within -1e30 and 1e30")
        if softcap != 0 and not (1e-3 <= softcap <= 1e6 and abs(scale) <= 1e9 * softcap):
            raise ValueError("softcap must be 0, or within 1e-3 and 1e6 and no less than "
                             "1e-9 times the scale")
        slopes = None
        if alibi_slopes is not None:
            slopes = _vector("alibi_slopes", alibi_slopes, torch.float32, self.output_q_heads,
                             self._widths[2])
        return scale, softcap, slopes

    def _raise_earlier(self):
        if self._status.value:
            raise RuntimeError("an earlier call failed on the device: "
                               + _C.decode_status(self._status.value))

    def ulysses_attention_forward(self, q, k, v, *, cu_seqlens=None, prefix_lens=None,
                                  causal=True, scale=None, softcap=0.0, alibi_slopes=None,
                                  out=None):
        """Attention over the exchanged rows (no counterpart in the reference).

        ``q`` is BF16 ``[T, output_q_heads * 128]``, ``k`` and ``v`` BF16
        ``[T, output_kv_heads * 128]``: the layout that ``ulysses_qkv_forward``
        returns, or any tensors with contiguous, 16-byte aligned rows.  Query
        head ``h`` reads K/V head ``h // (q heads / kv heads)``.

        ``cu_seqlens`` (int32, ``[documents + 1]``) packs several documents
        into the rows: document ``d`` is rows ``cu_seqlens[d]`` up to
        ``cu_seqlens[d + 1]``, and a row sees rows of its own document only.
        It starts at 0 and does not decrease; rows behind its last entry are
        not written (undefined if the call makes ``out``) and have no part in
        others.  Without it all rows are one
        document.
        ``causal=True`` lets a row see itself and the rows before it, and with
        ``prefix_lens`` (int32, ``[documents]``, needs ``causal``) also the
        first ``prefix_lens[d]`` rows of its document.

        Scores are ``scale * q.k`` (default ``128 ** -0.5``), then
        ``softcap * tanh(score / softcap)`` if ``softcap`` is positive, then
        less ``alibi_slopes[h] * |i - j|`` if ``alibi_slopes`` (FP32
        ``[output_q_heads]``, this rank's heads) is given.  A ``softcap`` lies
        within 1e-3 and 1e6 and is at least ``1e-9 * abs(scale)``; ``scale`` lies
        within -1e30 and 1e30.  Scores and sums are FP32.  Rows that are not
        seen take no part, whatever they hold.

        Returns BF16 ``[T, output_q_heads * 128]``, the layout that
        ``ulysses_o_proj_forward`` takes, written into ``out`` when given.
        Lengths are read on the device, so a captured call may be replayed
        with other lengths in the same tensors.
        """
        if _C.try_attention is not None and self._widths[2] >= 0:
            to = torch.empty_like(q, memory_format=torch.contiguous_format) if out is None else out
            if _C.try_attention(self._widths[2], *self._head_counts, q, k, v, cu_seqlens,
                                prefix_lens, alibi_slopes, to, causal,
                                self._default_scale if scale is None else scale, softcap,
                                self._status.device_ptr, self._status.host_ptr):
                return to
        # What did not fit, and what there is nothing to launch for.
        rows = q.shape[0]
        q_width, kv_width, index = self._widths
        q_ptr, q_stride = _rows("q", q, rows, q_width, index)
        k_ptr, k_stride = _rows("k", k, rows, kv_width, index)
        v_ptr, v_stride = _rows("v", v, rows, kv_width, index)
        if rows > 1 << 30:
            raise ValueError("at most 2^30 rows")
        scale, softcap, slopes = self._score_options(scale, softcap, alibi_slopes)
        docs, cu, prefix = 1, None, None
        if cu_seqlens is not None:
            docs = cu_seqlens.numel() - 1
            cu = _vector("cu_seqlens", cu_seqlens, torch.int32, max(docs + 1, 1), index)
        if prefix_lens is not None:
            if not causal:
                raise ValueError("prefix_lens needs causal=True")
            prefix = _vector("prefix_lens", prefix_lens, torch.int32, docs, index)
        self._raise_earlier()
        if out is None:
            out = _like_rows(q, q_stride, q_width)
            out_ptr, out_stride = out.data_ptr(), q_width
        else:
            out_ptr, out_stride = _rows("out", out, rows, q_width, index)
            _no_overlap(rows, out_ptr, out_stride, q_width, q_ptr, q_stride, q_width)
            _no_overlap(rows, out_ptr, out_stride, q_width, k_ptr, k_stride, kv_width)
            _no_overlap(rows, out_ptr, out_stride, q_width, v_ptr, v_stride, kv_width)
        if rows == 0 or docs == 0:
            return out
        _C.attention_forward(index, self.output_q_heads, self.output_kv_heads, 1 if causal else 0,
                             rows, q_ptr, k_ptr, v_ptr, out_ptr, q_stride, k_stride, v_stride,
                             out_stride, cu, prefix, slopes, docs, scale, softcap,
                             self._status.device_ptr, self._status.host_ptr, 0, 0,
                             _C.current_stream_handle(index))
        return out

    def create_kv_cache(self, num_blocks, max_seqs, max_blocks):
        """A zeroed :class:`KvCache` for this rank's K/V heads: ``num_blocks``
        blocks of 64 tokens, ``max_seqs`` slots, sequences of up to
        ``max_blocks`` blocks."""
        return KvCache.allocate(num_blocks, max_seqs, max_blocks, self.output_kv_heads,
                                self.device)

    def kv_cache_append(self, cache, k, v, slots, seq_lens, *, cu_seqlens=None):
        """Write new K/V rows into ``cache`` (no counterpart in the reference).

        ``k`` and ``v`` are BF16 ``[T, output_kv_heads * 128]`` as
        ``ulysses_qkv_forward`` returns them.  Without ``cu_seqlens`` each row
        is the next token of one sequence: ``slots`` and ``seq_lens`` (int32,
        ``[T]``) give its slot in the cache and its length, the new token
        included.  With ``cu_seqlens`` (int32, ``[n + 1]``, from 0, not
        decreasing) rows ``cu_seqlens[i]`` up to ``cu_seqlens[i + 1]`` are the
        next tokens of slot ``slots[i]``, whose length becomes ``seq_lens[i]``
        (both ``[n]``); rows behind its last entry are not read.  One that
        decreases is reported, and sequences of the call may then be written
        in part.

        A negative slot is skipped, so a batch may be padded.  Blocks that the
        call completes are written to ``cache.block_table``'s blocks in 8 bits;
        the rest stays in the slot's tail.  A slot may occur only once in a
        call.  Slots, blocks or lengths that do not fit the cache are reported
        like every device-side error, by the next call or ``check()``, and
        nothing is written for them.  Where it was a block, the sequence's
        earlier tokens are kept, and the call may be made again for it with
        the table put right.
        """
        _check_cache(cache, self._widths[1], self.device)
        if _C.try_append is not None and self._widths[2] >= 0:
            if _C.try_append(cache._address, k, v, slots, seq_lens, cu_seqlens,
                             self._status.device_ptr, self._status.host_ptr):
                return
        # What did not fit, and what there is nothing to launch for.
        rows, count = k.shape[0], slots.numel()
        _, kv_width, index = self._widths
        k_ptr, k_stride = _rows("k", k, rows, kv_width, index)
        v_ptr, v_stride = _rows("v", v, rows, kv_width, index)
        if rows > 1 << 30 or count > 1 << 24:
            raise ValueError("at most 2^30 rows and 2^24 sequences")
        slot_ptr = _vector("slots", slots, torch.int32, rows if cu_seqlens is None else count,
                           index)
        lens_ptr = _vector("seq_lens", seq_lens, torch.int32, count, index)
        cu = None
        if cu_seqlens is not None:
            cu = _vector("cu_seqlens", cu_seqlens, torch.int32, count + 1, index)
        self._raise_earlier()
        if rows == 0 or count == 0:
            return
        _C.kvcache_append(cache._address, k_ptr, v_ptr, k_stride, v_stride, rows, slot_ptr,
                          lens_ptr, cu, count, self._status.device_ptr, self._status.host_ptr, 0,
                          _C.current_stream_handle(index))

    def kv_cache_attention(self, cache, q, slots, seq_lens, *, scale=None, softcap=0.0,
                           alibi_slopes=None, out=None):
        """Attention of one token per sequence over ``cache`` (no counterpart
        in the reference).

        ``q`` is BF16 ``[n, output_q_heads * 128]``, row ``i`` the last token of
        the sequence in slot ``slots[i]``, which attends to that sequence's
        first ``seq_lens[i]`` tokens (int32 ``[n]`` each), so append it first.
        Scores as in ``ulysses_attention_forward``.  Returns BF16
        ``[n, output_q_heads * 128]``, written into ``out`` when given.  A row
        with a negative slot is left as it was (undefined if the call makes
        ``out``), one with length 0 is zeroed; a slot may occur more than once.  Slots, blocks and lengths that do not
        fit the cache are reported by the next call or ``check()``.
        """
        _check_cache(cache, self._widths[1], self.device)
        # Scratch from torch's allocator, so calls on other streams and captured
        # graphs each have their own.
        nbytes = self._attention_scratch
        if _C.try_decode is not None and self._widths[2] >= 0:
            to = torch.empty_like(q, memory_format=torch.contiguous_format) if out is None else out
            work = q.new_empty((nbytes + 1) // 2)
            if _C.try_decode(cache._address, self._head_counts[0], q, slots, seq_lens,
                             alibi_slopes, to, work,
                             self._default_scale if scale is None else scale, softcap,
                             self._status.device_ptr, self._status.host_ptr):
                return to
        # What did not fit, and what there is nothing to launch for.
        rows = q.shape[0]
        q_width, kv_width, index = self._widths
        q_ptr, q_stride = _rows("q", q, rows, q_width, index)
        if rows > 1 << 24:
            raise ValueError("at most 2^24 sequences")
        slot_ptr = _vector("slots", slots, torch.int32, rows, index)
        lens_ptr = _vector("seq_lens", seq_lens, torch.int32, rows, index)
        scale, softcap, slopes = self._score_options(scale, softcap, alibi_slopes)
        self._raise_earlier()
        if out is None:
            out = _like_rows(q, q_stride, q_width)
            out_ptr, out_stride = out.data_ptr(), q_width
        else:
            out_ptr, out_stride = _rows("out", out, rows, q_width, index)
            _no_overlap(rows, out_ptr, out_stride, q_width, q_ptr, q_stride, q_width)
        if rows == 0:
            return out
        work = q.new_empty((nbytes + 1) // 2)
        _C.kvcache_attention(cache._address, q_ptr, q_stride, out_ptr, out_stride,
                             self.output_q_heads, slot_ptr, lens_ptr, rows, scale, softcap,
                             slopes, work.data_ptr(), nbytes, self._status.device_ptr,
                             self._status.host_ptr, 0, _C.current_stream_handle(index))
        return out

    def check(self):
        """Synchronise the device and raise if any call reported a device-side error."""
        torch.cuda.synchronize(self.device)
        if self._status.value:
            raise RuntimeError("device-side error: " + _C.decode_status(self._status.value))

    def clear_error(self):
        """Reset the status word, the completion counters and the operators'
        failed marks after a reported error (call only when no launch of this
        context is in flight)."""
        torch.cuda.synchronize(self.device)
        for block in (self.barrier, self.o_barrier):
            if block is not None:
                block.data_[_C.FU_SYNC_COUNTER].zero_()
                block.data_[_C.FU_SYNC_FAILED].zero_()
        torch.cuda.synchronize(self.device)
        self._status.clear()

    def close(self):
        """Collectively release peer mappings after all output consumers finish."""
        torch.cuda.synchronize(self.device)
        if self.world_size > 1 or dist.is_initialized():
            dist.barrier(group=self.control_group)
        self._views = {}
        with torch.cuda.device(self.device):
            if self._op is not None:
                self._op.destroy()
                self._op = None
            if self._oproj is not None:
                self._oproj.destroy()
                self._oproj = None
            for name in ("Q", "K", "V", "barrier", "G", "o_barrier"):
                t = getattr(self, name)
                if t is not None:
                    t.close()
                setattr(self, name, None)
            if self._status is not None:
                self._status.free()
                self._status = None
