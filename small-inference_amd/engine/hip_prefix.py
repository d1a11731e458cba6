"""Decode attention over shared prefixes on MI355X through libsmallinf_hip.so: sequences whose block tables begin with the same
blocks (beams of a request, requests behind one prompt) have the shared keys read once for all of them. The reference shares
no blocks and has no counterpart.

  shared_groups  which sequences of a batch to group, from their block tables
  PrefixPlan     one layer's attention of such a batch, checked once per forward and called for every layer
"""

from __future__ import annotations

import ctypes
import threading

import numpy as np
import torch

from . import _hip
from .hip_decode import QuantKV

MAX_GROUP = 16         # query heads per KV head
MAX_CONTEXT = 1 << 24


def prefix_supported(q_dtype: torch.dtype, pool_dtype: torch.dtype, block_size: int, head_dim: int, group: int,
                     max_context: int = 1) -> bool:
    """Whether PrefixPlan covers this shape (bf16 q; bf16 or INT8 per-token pool; blocks of 16, 32 or 64 tokens, head_dim
    64/128, up to 16 query heads a KV head, contexts up to 2^24 tokens)."""
    return q_dtype == torch.bfloat16 and pool_dtype in (torch.bfloat16, torch.int8) and block_size in (16, 32, 64) and \
        head_dim in (64, 128) and group <= MAX_GROUP and max_context <= MAX_CONTEXT


def shared_groups(tables: list[np.ndarray], context_lens: list[int], block_size: int) -> list[tuple[list[int], int]]:
    """Groups [(rows, tokens)] of a batch whose rows' tables (int arrays of block ids) begin with the same blocks. tokens are
    whole blocks, all of them inside every member's context. A row is in one group at most, so of groups within groups one level
    is taken, that with which the batch reads fewer tokens: what the groups of the other level share is read for every row (64
    requests of 4 beams, 1024 tokens each, behind a common 4096: one group of 256 rows, 266 thousand keys read of 70 thousand)."""
    full = [min(t.shape[0], c // block_size) for t, c in zip(tables, context_lens)]

    def split(rows: list[int], depth: int, level: int = 0) -> tuple[list[tuple[list[int], int]], int]:
        """The groups of rows, which agree in their first `depth` blocks, and the blocks that they save; at most 32 groups
        within each other are looked at."""
        if len(rows) < 2:
            return [], 0
        same = min(full[r] for r in rows)
        if same > depth:
            ids = np.stack([tables[r][depth:same] for r in rows])
            other = np.flatnonzero((ids != ids[0]).any(axis=0))
            if other.size:
                same = depth + int(other[0])
        whole = ([(rows, same * block_size)] if same else []), (len(rows) - 1) * same
        parts: dict[int, list[int]] = {}
        for r in rows if level < 32 else ():
            if full[r] > same:
                parts.setdefault(int(tables[r][same]), []).append(r)
        groups, saved = [], 0
        for part in parts.values():
            g, s = split(part, same, level + 1)
            groups += g
            saved += s
        return (groups, saved) if saved > whole[1] else whole

    by_first: dict[int, list[int]] = {}
    for r, n in enumerate(full):
        if n:
            by_first.setdefault(int(tables[r][0]), []).append(r)
    return [g for rows in by_first.values() for g in split(rows, 0)[0]]


class PrefixPlan:
    """Validated launch parameters of one forward's decode attention over shared prefixes, called for every layer (as
    engine.hip_decode.DecodePlan): building it does every check, calling it swaps in the layer's tensors and launches.

    q [S, Hq, D] bf16 (rows may be strided, last dim contiguous); k_cache, v_cache [Hkv, N, B, D] bf16, or int8 with quant
    (engine.hip_decode.QuantKV of mode 1); block_tables [S, >= ceil(max_context / B)], context_lens [S] int32 (the new token
    included; a sequence of none gets zeros); max_context, known on the host, bounds them. groups [(rows, tokens)]: rows of the
    batch whose tables agree in their first tokens / B entries, tokens whole blocks; a row is in one group at most. Groups
    change the time, not the result: every row attends the positions below its context length, and one whose context is
    shorter than its group's tokens is read by itself. host_context_lens: the lengths as a list, by which the work is
    divided; None: they are read from the device once, which waits for it. Calls can be captured, a plan is built before and has to
    be kept as long as the graph is replayed.

    The workspace is made for the call that needs it, so plans, streams and graphs share none. Calls may be on any stream of the
    device (a plan that is dropped keeps its work list until they have read it). Threads may call one plan at
    the same time: each call fills the parameter block and launches under the plan's lock."""

    def __init__(self, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                 context_lens: torch.Tensor, groups: list[tuple[list[int], int]], scale: float, max_context: int, *,
                 quant: QuantKV | None = None, host_context_lens: list[int] | None = None):
        S, Hq, D = q.shape
        Hkv, N, B, Dk = k_cache.shape
        if D != Dk or Hkv < 1 or Hq % Hkv:
            raise ValueError(f"q {tuple(q.shape)} does not fit pools {tuple(k_cache.shape)}")
        if quant is not None and quant.mode != 1:
            raise ValueError(f"shared prefixes are read from bf16 pools or INT8 pools with per-token scales (QuantKV mode 1), "
                             f"not mode {quant.mode}")
        if q.dtype != torch.bfloat16:
            raise ValueError("the shared-prefix kernel needs bf16 q")
        if context_lens.dtype is not torch.int32 or context_lens.shape != (S,) or not context_lens.is_contiguous():
            raise ValueError(f"context_lens must be a contiguous int32 vector of {S}")
        if block_tables.dtype is not torch.int32 or block_tables.dim() != 2 or block_tables.stride(1) != 1 or \
                block_tables.shape[0] < S or block_tables.shape[1] * B < max_context:
            raise ValueError(f"block_tables {tuple(block_tables.shape)} must be int32 with {S} rows of at least "
                             f"ceil({max_context} / {B}) entries")
        if host_context_lens is not None and (len(host_context_lens) != S or max(host_context_lens, default=0) > max_context):
            raise ValueError("host_context_lens must hold S lengths, none above max_context")
        _hip.require_gpu(q, k_cache, v_cache, block_tables, context_lens)
        if _hip.lib().sipa_capture_id(_hip.stream_of(q)):
            raise ValueError("a PrefixPlan uploads its work list: build it before the graph capture")
        if host_context_lens is None:
            host_context_lens = context_lens.tolist()
        self.shape, self.pool_shape, self.device = (S, Hq, D), tuple(k_cache.shape), q.device
        self.pool_dtype = torch.bfloat16 if quant is None else torch.int8
        self._pool_strides = (N * B * D, B * D, D, 1)  # of a contiguous layer
        self._quantized, self._own_quant = quant is not None, quant
        p = self.params = _hip.PrefixParams(
            struct_size=ctypes.sizeof(_hip.PrefixParams), num_seqs=S, num_q_heads=Hq, num_kv_heads=Hkv, head_dim=D, block_size=B,
            num_blocks=N, max_context=max_context, kv_mode=1 if self._quantized else 0, scale=float(scale),
            block_tables=block_tables.data_ptr(), bt_stride_s=block_tables.stride(0), bt_width=block_tables.shape[1],
            context_lens=context_lens.data_ptr())
        self._ref, self._lib = ctypes.byref(p), _hip.lib()
        starts = np.zeros(len(groups) + 1, dtype=np.int32)
        np.cumsum([len(rows) for rows, _ in groups], out=starts[1:])
        members = np.asarray([r for rows, _ in groups for r in rows], dtype=np.int32)
        tokens = np.asarray([t for _, t in groups], dtype=np.int32)
        lens = None if host_context_lens is None else np.asarray(host_context_lens, dtype=np.int32)
        args = (self._ref, len(groups), starts.ctypes.data, members.ctypes.data, tokens.ctypes.data,
                None if lens is None else lens.ctypes.data)
        with _hip.on_device(self.device):
            _hip.check(self._lib.sipa_prefix_plan(*args, None, 0, ctypes.byref(p.layout)), "prefix plan")
            plan = np.empty(p.layout.plan_ints, dtype=np.int32)
            _hip.check(self._lib.sipa_prefix_plan(*args, plan.ctypes.data, plan.size, ctypes.byref(p.layout)), "prefix plan")
        plan = torch.from_numpy(plan).to(self.device)
        p.plan = plan.data_ptr()
        self._keep = (block_tables, context_lens, plan)
        self._list, self._stream = plan, _hip.stream_of(q)  # the work list, and the stream whose memory it is
        self._ws_bytes = p.layout.workspace_bytes
        self._lock = threading.Lock()
        self._bind(q, k_cache, v_cache, quant)

    def _bind_q(self, q: torch.Tensor) -> None:
        if q.shape != self.shape or q.dtype is not torch.bfloat16 or q.stride(2) != 1 or q.device != self.device:
            raise ValueError("q does not match the plan")
        p = self.params
        p.q, p.q_stride_s, p.q_stride_h = q.data_ptr(), q.stride(0), q.stride(1)
        self._q = q

    def _bind_scales(self, ks: int, ks_dtype, ks_strides, vs: int, vs_dtype, vs_strides) -> None:
        if ks_strides[-1] != 1 or vs_strides[-1] != 1:
            raise ValueError("scales need a contiguous last dim")
        p = self.params
        p.k_scale, p.k_scale_dtype, p.ks_stride_h, p.ks_stride_n = ks, _hip.dtype_code(ks_dtype), *ks_strides[-3:-1]
        p.v_scale, p.v_scale_dtype, p.vs_stride_h, p.vs_stride_n = vs, _hip.dtype_code(vs_dtype), *vs_strides[-3:-1]

    def _check_quant(self, quant: QuantKV | None, lead: tuple) -> None:
        """The scales' shapes, [*lead, Hkv, N, B] each, and place."""
        if (quant is not None) != self._quantized or (quant is not None and quant.mode != 1):
            raise ValueError("quant does not match the plan")
        if quant is not None:
            want = (*lead, *self.pool_shape[:3])
            for t in (quant.k_scale, quant.v_scale):
                if t.shape != want or t.device != self.device:
                    raise ValueError(f"scales must be {want} on {self.device}")

    def _bind(self, q, k_cache, v_cache, quant) -> None:
        """Point the parameters at one layer's tensors."""
        for t in (k_cache, v_cache):
            if t.shape != self.pool_shape or t.dtype is not self.pool_dtype or t.device != self.device or \
                    not t.is_contiguous():
                raise ValueError(f"the pools must be contiguous {self.pool_dtype} {self.pool_shape}, as the plan's")
        self._bind_q(q)
        self._check_quant(quant, ())
        p = self.params
        p.k_cache, p.v_cache = k_cache.data_ptr(), v_cache.data_ptr()
        p.kv_stride_h, p.kv_stride_n = self._pool_strides[:2]
        if quant is not None:
            ks, vs = quant.k_scale, quant.v_scale
            self._bind_scales(ks.data_ptr(), ks.dtype, ks.stride(), vs.data_ptr(), vs.dtype, vs.stride())
        self._k, self._v, self._quant = k_cache, v_cache, quant

    def run_layer(self, layer: int, q: torch.Tensor, k_pools: torch.Tensor, v_pools: torch.Tensor,
                  quant: QuantKV | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        """The attention over layer `layer` of pools [L, Hkv, N, B, D] (quant: scales with a leading layer dimension too):
        the plan called with pools[layer] and the like, without making those views."""
        for t in (k_pools, v_pools):
            if t.shape[1:] != self.pool_shape or t.dtype is not self.pool_dtype or t.device != self.device or \
                    (t.stride()[1:] != self._pool_strides and not _hip.layers_contiguous(t)):
                raise ValueError("the pools do not match the plan")
        self._check_quant(quant, k_pools.shape[:1])
        with self._lock:
            self._bind_q(q)
            p = self.params
            p.k_cache, p.v_cache = _hip.layer_ptr(k_pools, layer), _hip.layer_ptr(v_pools, layer)
            p.kv_stride_h, p.kv_stride_n = self._pool_strides[:2]
            self._k, self._v, self._quant = k_pools, v_pools, quant
            if quant is not None:
                ks, vs = quant.k_scale, quant.v_scale
                self._bind_scales(_hip.layer_ptr(ks, layer), ks.dtype, ks.stride(), _hip.layer_ptr(vs, layer), vs.dtype,
                                  vs.stride())
            return self._run(out)

    def __call__(self, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, quant: QuantKV | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of q over one layer's pools (quant None: the plan's own scales). Returns out ([S, Hq, D] bf16)."""
        with self._lock:
            self._bind(q, k_cache, v_cache, self._own_quant if quant is None else quant)
            return self._run(out)

    def _run(self, out: torch.Tensor | None) -> torch.Tensor:
        p = self.params
        if out is None:
            out = torch.empty(self.shape, dtype=torch.bfloat16, device=self.device)
        elif out.shape != self.shape or out.dtype is not torch.bfloat16 or out.stride(2) != 1 or out.device != self.device:
            raise ValueError("out must be [S, Hq, D] bf16 with a contiguous last dim on q's device")
        if self.shape[0] == 0:
            return out
        p.out, p.out_stride_s, p.out_stride_h = out.data_ptr(), out.stride(0), out.stride(1)
        stream = _hip.stream_of(out)
        if stream != self._stream:
            self._list.record_stream(torch.cuda.current_stream(self.device))
        with _hip.on_device(self.device):
            ws = torch.empty(self._ws_bytes, dtype=torch.uint8, device=self.device)
            p.workspace, p.workspace_bytes = ws.data_ptr(), self._ws_bytes
            rc = self._lib.sipa_prefix_attention(self._ref, stream)
        if rc:
            _hip.check(rc, "prefix attention")
        return out


def paged_prefix_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                           context_lens: torch.Tensor, groups: list[tuple[list[int], int]], scale: float, max_context: int,
                           out: torch.Tensor | None = None, *, quant: QuantKV | None = None,
                           host_context_lens: list[int] | None = None) -> torch.Tensor:
    """One layer's decode attention over shared prefixes: a PrefixPlan built and run once (see there)."""
    plan = PrefixPlan(q, k_cache, v_cache, block_tables, context_lens, groups, scale, max_context, quant=quant,
                      host_context_lens=host_context_lens)
    return plan(q, k_cache, v_cache, out=out)
