"""Drafted trees on MI355X through libsmallinf_hip.so: several tokens drafted ahead for each sequence are verified in one
forward. The reference decodes one token per sequence and step and has no counterpart.

A sequence's nodes stand in the cache behind its `start` cached tokens, node i in the slot of position start + i. A node
has a parent among the nodes before it, or none (-1); it sees the cached tokens, its ancestors and itself, and its rotary
position is start plus the number of its ancestors. Ancestor masks are int64 words [T, ceil(nodes / 64)], node a of the
row's sequence in bit a % 64 of word a // 64.

  TreePlan       one layer's attention of the trees, checked once per forward and called for every layer
  tree_maps      slots, positions, packed block tables and ancestor masks of a forward, from the lengths on the GPU
  commit_tokens  after verification, the accepted nodes' K and V moved to the positions they now have, in all layers
"""

from __future__ import annotations

import ctypes
import struct
import threading
from typing import NamedTuple

import torch

from . import _hip
from .hip_decode import QuantKV

MAX_NODES = 256  # nodes of a sequence: four mask words


class TreeMaps(NamedTuple):
    """A forward's metadata as tree_maps derives it (T rows, S sequences)."""
    positions: torch.Tensor     # [T] int64 rotary position of each node
    slots: torch.Tensor         # [T] int64 slot of each node
    slot_blocks: torch.Tensor   # [T] slot // block_size
    slot_offsets: torch.Tensor  # [T] slot % block_size
    last_rows: torch.Tensor     # [S] int64 row of each sequence's last node
    query_starts: torch.Tensor  # [S + 1] int32 first row of each sequence
    context_lens: torch.Tensor  # [S] int32 cached tokens and nodes
    block_tables: torch.Tensor  # [S, width] int32, -1 padded
    masks: torch.Tensor         # [T, words] int64 ancestor masks


def mask_words(max_nodes: int) -> int:
    """Words of an ancestor mask for trees of up to max_nodes nodes."""
    if not 1 <= max_nodes <= MAX_NODES:
        raise ValueError(f"trees of {max_nodes} nodes; a sequence holds 1 to {MAX_NODES}")
    return -(-max_nodes // 64)


_I32, _I64 = torch.int32, torch.int64
_split = torch.split_with_sizes
# sipa_tree_maps_params and sipa_commit_params as bytes (native alignment): a third of the time that filling a ctypes
# structure takes, in calls whose kernels take a few microseconds
_MAPS = struct.Struct("8iq14Qiq")
_COMMIT = struct.Struct("9i2Q4q2Q4qQq2QqQ")
assert _MAPS.size == ctypes.sizeof(_hip.TreeMapsParams) and _COMMIT.size == ctypes.sizeof(_hip.CommitParams)


def _vector(t: torch.Tensor, n: int, what: str) -> None:
    if t.dtype is not _I32 or t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 vector of {n}")


def tree_maps(tables: torch.Tensor, rows: torch.Tensor, starts: torch.Tensor, counts: torch.Tensor, parents: torch.Tensor,
              block_size: int, width: int, max_nodes: int, out: TreeMaps | None = None, rest_slot: int | None = None) -> TreeMaps:
    """A forward's metadata from device lengths, in one launch (sipa_tree_maps).

    tables [rows, columns] int32: persistent block tables, one row per live sequence (engine.device_tables); rows, starts,
    counts [S] int32: each sequence's table row, cached tokens and nodes; parents [T] int32: each node's parent within its
    sequence, -1 for none, sequences one after the other. width: columns of the packed tables, max_nodes: the largest
    count, both known to the host. T may be more than the counts sum to (a captured step's capacity): rows behind the last
    sequence are left as they are (in tensors made here: undefined, in out: an earlier step's), so none may be stored or
    looked up; with rest_slot, a slot that no sequence has, they get it, position 0 and no ancestors, and a step may store and
    attend all T rows. out: tensors of an earlier call of the same sizes, written again.
    """
    S, T, words = counts.shape[0], parents.shape[0], mask_words(max_nodes)
    _vector(rows, S, "rows"), _vector(starts, S, "starts"), _vector(counts, S, "counts"), _vector(parents, T, "parents")
    table_rows, columns = tables.shape
    table_stride, last = tables.stride()
    if tables.dtype is not _I32 or last != 1:
        raise ValueError("tables must be int32 [rows, columns] with contiguous rows")
    if S < 1 or T < 1 or block_size < 1 or width < 1:
        raise ValueError(f"{S} sequences, {T} nodes, block size {block_size}, width {width}")
    if rest_slot is not None and rest_slot < 0:
        raise ValueError(f"rest_slot {rest_slot}")
    _hip.require_gpu(tables, rows, starts, counts, parents)
    dev = tables.device
    if out is None:
        d64 = torch.empty(T * (4 + words) + S, dtype=_I64, device=dev)
        d32 = torch.empty(S * (width + 2) + 1, dtype=_I32, device=dev)
        pos, slots, blocks, offs, last_rows, masks = _split(d64, (T, T, T, T, S, T * words))
        qs, ctx, bt = _split(d32, (S + 1, S, S * width))
        out = TreeMaps(pos, slots, blocks, offs, last_rows, qs, ctx, bt.view(S, width), masks.view(T, words))
        p64, p32 = d64.data_ptr(), d32.data_ptr()
        at = (p64, p64 + 8 * T, p64 + 16 * T, p64 + 24 * T, p64 + 32 * T, p32, p32 + 4 * (S + 1), p32 + 4 * (2 * S + 1),
              p64 + 32 * T + 8 * S)
    else:
        shapes = ((T,), (T,), (T,), (T,), (S,), (S + 1,), (S,), (S, width), (T, words))
        for i, (t, shape) in enumerate(zip(out, shapes)):
            if t.shape != shape or t.dtype is not (_I32 if 5 <= i <= 7 else _I64) or not t.is_contiguous():
                raise ValueError(f"out.{TreeMaps._fields[i]} must be contiguous {shape}, as a call of these sizes returns")
        _hip.require_gpu(tables, *out)
        at = tuple(t.data_ptr() for t in out)
    p = _MAPS.pack(_MAPS.size, S, T, block_size, width, words, table_rows, columns, table_stride, tables.data_ptr(),
                   rows.data_ptr(), starts.data_ptr(), counts.data_ptr(), parents.data_ptr(), *at, rest_slot is not None,
                   rest_slot or 0)
    with _hip.on_device(dev):
        rc = _hip.lib().sipa_tree_maps(p, _hip.stream_of(tables))
    if rc:
        _hip.check(rc, "tree_maps")
    return out


def commit_tokens(k: torch.Tensor, v: torch.Tensor, block_tables: torch.Tensor, starts: torch.Tensor,
                  accepted: torch.Tensor, num_accepted: torch.Tensor, *, k_scale: torch.Tensor | None = None,
                  v_scale: torch.Tensor | None = None) -> None:
    """Move the accepted nodes' K and V, in place and in all layers, in one launch (sipa_commit_tokens): position
    starts[s] + i takes the rows of position starts[s] + accepted[s, i], for i below num_accepted[s].

    k, v [L, Hkv, N, B, D] (the caches' pools; each layer contiguous), with per-token fp16 scales [L, Hkv, N, B] for INT8
    pools; block_tables [S, columns], starts, num_accepted [S], accepted [S, A] int32 on the device, the accepted nodes of a
    sequence in ascending order, as a path from a root is; entries past num_accepted[s] are not read.
    """
    L, H, N, B, D = k.shape
    S, A = accepted.shape
    if v.shape != k.shape or v.dtype is not k.dtype:
        raise ValueError("K and V pools must have one shape and dtype")
    block = B * D
    ks, vs = k.stride(), v.stride()
    if L < 1 or ks[1:] != (N * block, block, D, 1) or vs[1:] != ks[1:]:
        raise ValueError("each layer of the pools must be contiguous")
    kss = vss = (0, 0)
    ksp = vsp = 0
    if (k_scale is None) != (v_scale is None) or (k_scale is None) == (k.dtype is torch.int8):
        raise ValueError("INT8 pools, and only they, have scales of K and V")
    if k_scale is not None:
        kss, vss = k_scale.stride(), v_scale.stride()
        if k_scale.shape != (L, H, N, B) or v_scale.shape != (L, H, N, B) or k_scale.dtype is not torch.float16 or \
                v_scale.dtype is not torch.float16 or kss[1:] != (N * B, B, 1) or vss[1:] != kss[1:]:
            raise ValueError(f"scales must be fp16 {(L, H, N, B)}, each layer contiguous")
        ksp, vsp = k_scale.data_ptr(), v_scale.data_ptr()
    _vector(starts, S, "starts"), _vector(num_accepted, S, "num_accepted")
    rows, width = block_tables.shape
    bt_stride, last = block_tables.stride()
    if block_tables.dtype is not _I32 or rows < S or last != 1 or width < 1:
        raise ValueError(f"block_tables must be int32 with {S} rows")
    acc_stride, last = accepted.stride()
    if accepted.dtype is not _I32 or (A > 1 and last != 1):
        raise ValueError("accepted must be int32 [S, A] with contiguous rows")
    _hip.require_gpu(k, v, block_tables, starts, accepted, num_accepted, k_scale, v_scale)
    if S == 0 or A == 0:
        return
    size = k.element_size()
    p = _COMMIT.pack(_COMMIT.size, L, H, N, B, D * size, S, A, width, k.data_ptr(), v.data_ptr(), ks[0] * size,
                     ks[1] * size, vs[0] * size, vs[1] * size, ksp, vsp, kss[0], kss[1], vss[0], vss[1],
                     block_tables.data_ptr(), bt_stride, starts.data_ptr(), accepted.data_ptr(), acc_stride,
                     num_accepted.data_ptr())
    with _hip.on_device(k.device):
        rc = _hip.lib().sipa_commit_tokens(p, _hip.stream_of(k))
    if rc:
        _hip.check(rc, "commit_tokens")


def tree_supported(q_dtype: torch.dtype, pool_dtype: torch.dtype, block_size: int, head_dim: int, group: int,
                   max_context: int = 1, max_nodes: int = 1) -> bool:
    """Whether the tree attention kernel covers this shape (bf16 q; bf16 or INT8 per-token pool; blocks of 16, 32 or 64
    tokens, head_dim 64/128, GQA group <= 64, trees of up to MAX_NODES nodes, contexts up to 2097152 tokens for up to 64 rows
    of query heads, 655360 (head_dim 64) or 1179648 (128) for more: the splits that the kernel merges, of 16384 keys each);
    the caches use the gather path otherwise."""
    if not (q_dtype == torch.bfloat16 and pool_dtype in (torch.bfloat16, torch.int8) and block_size in (16, 32, 64) and
            head_dim in (64, 128) and group <= 64 and max_nodes <= MAX_NODES):
        return False
    splits = 128 if max_nodes * group <= 64 else 40 if head_dim == 64 else 72
    return max_context <= splits * 16384


class TreePlan:
    """Validated launch parameters of one forward's tree attention, called for every layer (as engine.hip_decode.DecodePlan
    for decode): building it does every check, calling it swaps in the layer's tensors and launches.

    q [T, Hq, D] bf16 (rows may be strided, last dim contiguous); k_cache, v_cache [Hkv, N, B, D] bf16, or int8 with quant
    (engine.hip_decode.QuantKV of mode 1), one layer of the pool with the nodes' K and V in their slots; block_tables
    [S, >= ceil(max_context / B)], context_lens [S] (cached tokens and nodes), query_starts [S + 1] int32; masks [T, words]
    int64; max_context and max_nodes are the host-known maxima. Row t of sequence s sees the positions below context_lens[s]
    - n_s and the nodes in its mask; a row that sees nothing gets zeros. Rows behind query_starts[S] are left as they are.

    The split workspace is the plan's own: it is made for the stream (and the graph capture) of the call that needs it, so
    plans, streams and graphs share none. Threads may call one plan at the same time: each call fills the parameter block and
    launches under the plan's lock."""

    def __init__(self, q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                 context_lens: torch.Tensor, query_starts: torch.Tensor, masks: torch.Tensor, scale: float, max_context: int,
                 max_nodes: int, *, quant: QuantKV | None = None, num_splits: int | None = None):
        T, Hq, D = q.shape
        Hkv, N, B, Dk = k_cache.shape
        S = context_lens.shape[0]
        if D != Dk or Hkv < 1 or Hq % Hkv:
            raise ValueError(f"q {tuple(q.shape)} does not fit pools {tuple(k_cache.shape)}")
        self.pool_dtype = torch.bfloat16 if quant is None else torch.int8
        if quant is not None and quant.mode != 1:
            raise ValueError(f"drafted trees read bf16 pools or INT8 pools with per-token scales (QuantKV mode 1), not mode "
                             f"{quant.mode}")
        if q.dtype != torch.bfloat16:
            raise ValueError("the tree attention kernel needs bf16 q")
        _vector(context_lens, S, "context_lens"), _vector(query_starts, S + 1, "query_starts")
        if block_tables.dtype is not torch.int32 or block_tables.dim() != 2 or block_tables.stride(1) != 1 or \
                block_tables.shape[0] < S or block_tables.shape[1] * B < max_context:
            raise ValueError(f"block_tables {tuple(block_tables.shape)} must be int32 with {S} rows of at least "
                             f"ceil({max_context} / {B}) entries")
        words = mask_words(max_nodes)
        if masks.dtype is not torch.int64 or masks.dim() != 2 or masks.shape[0] != T or masks.shape[1] < words or \
                not masks.is_contiguous():
            raise ValueError(f"masks must be contiguous int64 [{T}, >= {words}]")
        _hip.require_gpu(q, k_cache, v_cache, block_tables, context_lens, query_starts, masks)
        self.shape, self.pool_shape, self.device = (T, Hq, D), tuple(k_cache.shape), q.device
        self._pool_strides = (N * B * D, B * D, D, 1)  # of a contiguous layer
        self._keep = (block_tables, context_lens, query_starts, masks)
        self._quantized, self._own_quant = quant is not None, quant
        p = self.params = _hip.TreeParams(
            struct_size=ctypes.sizeof(_hip.TreeParams), num_seqs=S, num_tokens=T, num_q_heads=Hq, num_kv_heads=Hkv,
            head_dim=D, block_size=B, num_blocks=N, max_context=max_context, max_nodes=max_nodes, words=masks.shape[1],
            scale=float(scale), block_tables=block_tables.data_ptr(), bt_stride_s=block_tables.stride(0),
            bt_width=block_tables.shape[1], context_lens=context_lens.data_ptr(), query_starts=query_starts.data_ptr(),
            masks=masks.data_ptr(), kv_mode=1 if self._quantized else 0, num_splits=num_splits or 0)
        self._ref, self._lib = ctypes.byref(p), _hip.lib()
        counters = ctypes.c_int64(0)
        with _hip.on_device(self.device):
            n = self._lib.sipa_tree_workspace_bytes(self._ref, ctypes.byref(counters))
        if n < 0:
            _hip.check(n, "tree attention")
        self._ws_bytes, self._counter_bytes = n, counters.value
        self._workspace = self._owner = None
        self._lock = threading.Lock()
        self._bind(q, k_cache, v_cache, quant)

    def _bind_q(self, q: torch.Tensor) -> None:
        if q.shape != self.shape or q.dtype is not torch.bfloat16 or q.stride(2) != 1 or q.device != self.device:
            raise ValueError("q does not match the plan")
        p = self.params
        p.q, p.q_stride_t, p.q_stride_h = q.data_ptr(), q.stride(0), q.stride(1)
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
        p = self.params
        p.k_cache, p.v_cache = k_cache.data_ptr(), v_cache.data_ptr()
        p.kv_stride_h, p.kv_stride_n = self._pool_strides[:2]
        self._check_quant(quant, ())
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
        """Attention of q over one layer's pools (quant None: the plan's own scales). Returns out ([T, Hq, D] bf16)."""
        with self._lock:
            self._bind(q, k_cache, v_cache, self._own_quant if quant is None else quant)
            return self._run(out)

    def _run(self, out: torch.Tensor | None) -> torch.Tensor:
        p = self.params
        if out is None:
            out = torch.empty(self.shape, dtype=torch.bfloat16, device=self.device)
        elif out.shape != self.shape or out.dtype is not torch.bfloat16 or out.stride(2) != 1 or out.device != self.device:
            raise ValueError("out must be [T, Hq, D] bf16 with a contiguous last dim on q's device")
        p.out, p.out_stride_t, p.out_stride_h = out.data_ptr(), out.stride(0), out.stride(1)
        stream = _hip.stream_of(out)
        with _hip.on_device(self.device):
            if self._ws_bytes:
                owner = (stream, self._lib.sipa_capture_id(stream))
                if owner != self._owner:
                    ws = torch.empty(self._ws_bytes, dtype=torch.uint8, device=self.device)
                    ws[:self._counter_bytes].zero_()
                    self._workspace, self._owner = ws, owner
                    p.workspace, p.workspace_bytes = ws.data_ptr(), self._ws_bytes
            rc = self._lib.sipa_tree_attention(self._ref, stream)
        if rc:
            _hip.check(rc, "tree attention")
        return out


def paged_tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                         context_lens: torch.Tensor, query_starts: torch.Tensor, masks: torch.Tensor, scale: float,
                         max_context: int, max_nodes: int, out: torch.Tensor | None = None, *,
                         quant: QuantKV | None = None, num_splits: int | None = None) -> torch.Tensor:
    """One layer's attention of drafted trees: a TreePlan built and run once (see there)."""
    plan = TreePlan(q, k_cache, v_cache, block_tables, context_lens, query_starts, masks, scale, max_context, max_nodes,
                    quant=quant, num_splits=num_splits)
    return plan(q, k_cache, v_cache, out=out)
