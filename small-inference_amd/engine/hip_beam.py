"""Beam search on MI355X through libsmallinf_hip.so: the best continuations over the beams and the vocabulary of every
request, and the copies of blocks of beams that go on from the same one. The reference decodes greedily and has no
counterpart.

A step over the beams of a batch, which share their blocks (engine.block_manager.BlockManager.fork):

  logits = model.forward(...)                      # rows: the beams, one request after the other
  choice = beam_select(logits, scores, beams, n)   # n best (score, beam, token) of each request
  copies = manager.reorder(ids, parents)           # each sequence goes on from the one that was chosen
  cache.copy_blocks(copies)                        # their blocks that are not full yet
"""

from __future__ import annotations

import ctypes
import functools
import itertools
import struct
from array import array
from collections.abc import Sequence
from typing import NamedTuple

import torch

from . import _hip

DTYPES = (torch.bfloat16, torch.float16, torch.float32)
MAX_CANDIDATES = 64
MAX_BEAMS = 1024
# sipa_beam_params and sipa_copy_params as bytes (native alignment), as engine.hip_tree packs its own
_SELECT = struct.Struct("7iPq6Pq")
_COPY = struct.Struct("6i4P4q4q4iPi4x")
assert _SELECT.size == ctypes.sizeof(_hip.BeamParams) and _COPY.size == ctypes.sizeof(_hip.CopyParams)


class BeamChoice(NamedTuple):
    """The best continuations of each request, in descending order; score -inf, beam and token -1 behind the last one."""
    scores: torch.Tensor  # [groups, n] fp32
    beams: torch.Tensor   # [groups, n] int64 row within the group
    tokens: torch.Tensor  # [groups, n] int64


def beam_select(logits: torch.Tensor, scores: torch.Tensor, beams: int | torch.Tensor, candidates: int) -> BeamChoice:
    """The `candidates` (1 .. 64) best continuations over the beams and the vocabulary of each request, in two launches
    (sipa_beam_select): of row r and token v the score is scores[r] + log_softmax(logits[r])[v], equal ones in the order of
    their rows, then tokens. On the GPU a row's log-sum is within 2^-19 of the definition's (exponentials, and sums of eight, in 32
    bits), all after it is in 64 bits: candidates of different rows whose scores are closer than 2^-18 may change places; those of
    one row do not, and rows of equal logits and scores tie. Scores are returned in 32 bits.

    logits [R, V] bf16, fp16 or fp32 with a contiguous last dim (R the beams of all requests); scores [R] fp32; beams: how
    many rows each request has (1 to 1024, dividing R; 1 for the first step, when there is one row a request), or int32
    starts [groups + 1] of requests of different numbers of rows (up to 1024 each). Tokens of logit -inf are never taken,
    nor is any of a row whose score is not finite (a beam that has ended: -inf) or whose logits hold NaN or +inf, or -inf
    alone. CPU tensors are computed by torch operations."""
    if logits.dim() != 2 or logits.dtype not in DTYPES or logits.shape[1] < 1 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits must be [rows, vocab] in bf16, fp16 or fp32 with a contiguous last dim")
    R, V = logits.shape
    if scores.dtype is not torch.float32 or scores.shape != (R,) or not scores.is_contiguous():
        raise ValueError(f"scores must be a contiguous fp32 vector of {R}")
    if not 1 <= candidates <= MAX_CANDIDATES:
        raise ValueError(f"{candidates} candidates (1 to {MAX_CANDIDATES})")
    starts = beams if isinstance(beams, torch.Tensor) else None
    if starts is not None:
        if starts.dtype is not torch.int32 or starts.dim() != 1 or starts.shape[0] < 1 or not starts.is_contiguous():
            raise ValueError("starts of requests must be a contiguous int32 vector")
        groups, beams = starts.shape[0] - 1, 0
    else:
        if not 1 <= beams <= MAX_BEAMS or R % beams:
            raise ValueError(f"{beams} beams a request (1 to {MAX_BEAMS}) in {R} rows")
        groups = R // beams
    devices = {t.device for t in (logits, scores, starts) if t is not None}
    if len(devices) > 1:
        raise ValueError(f"logits, scores and starts must be on one device, got {sorted(map(str, devices))}")
    if not logits.is_cuda:
        return _select_torch(logits, scores, starts, beams, groups, candidates)
    dev, code, n = logits.device, _hip.dtype_code(logits.dtype), candidates
    both = torch.empty(2, groups, n, dtype=torch.int64, device=dev)
    out = BeamChoice(torch.empty(groups, n, dtype=torch.float32, device=dev), both[0], both[1])
    if groups == 0:
        return out
    size = _select_bytes(R, V, groups, beams, n, code)
    at = both.data_ptr()
    with _hip.on_device(dev):
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        p = _SELECT.pack(_SELECT.size, R, V, groups, beams, n, code, logits.data_ptr(), logits.stride(0), scores.data_ptr(),
                         0 if starts is None else starts.data_ptr(), out.scores.data_ptr(), at, at + 8 * groups * n,
                         ws.data_ptr(), size)
        rc = _hip.lib().sipa_beam_select(p, _hip.stream_of(logits))
    if rc:
        _hip.check(rc, "beam_select")
    return out


@functools.lru_cache(maxsize=256)
def _select_bytes(rows: int, vocab: int, groups: int, beams: int, candidates: int, dtype: int) -> int:
    """Workspace bytes of a selection of these sizes."""
    n = _hip.lib().sipa_beam_workspace_bytes(_SELECT.pack(_SELECT.size, rows, vocab, groups, beams, candidates, dtype, 0, 0, 0, 0,
                                                          0, 0, 0, 0, 0))
    if n < 0:
        _hip.check(n, "beam_select")
    return n


def _select_torch(logits, scores, starts, beams: int, groups: int, candidates: int) -> BeamChoice:
    """beam_select() on CPU tensors, group by group."""
    R, V = logits.shape
    bounds = [g * beams for g in range(groups + 1)] if starts is None else starts.clamp(0, R).tolist()
    out = BeamChoice(torch.full((groups, candidates), float("-inf")),
                     *(torch.full((groups, candidates), -1, dtype=torch.int64) for _ in range(2)))
    n = min(candidates, V)
    for g, (a, b) in enumerate(zip(bounds, bounds[1:])):
        b = min(b, a + MAX_BEAMS)
        if a >= b:
            continue
        l = logits[a:b].double()
        value, token = torch.sort(l, dim=-1, descending=True, stable=True)
        value, token = value[:, :n], token[:, :n]
        off = scores[a:b].double() - torch.logsumexp(l, -1)
        score = off[:, None] + value
        score = torch.where(off.isfinite()[:, None] & (value > float("-inf")), score, float("-inf")).reshape(-1)
        best, at = torch.sort(score, descending=True, stable=True)
        k = min(candidates, int((best > float("-inf")).sum()))
        out.scores[g, :k] = best[:k].float()
        out.beams[g, :k], out.tokens[g, :k] = at[:k] // n, token.reshape(-1)[at[:k]]
    return out


def _flat(copies: Sequence[tuple[int, int, int]], blocks: int, block_size: int) -> array:
    """The copies' numbers, one after the other."""
    try:
        flat = array("i", itertools.chain.from_iterable(copies))
    except OverflowError:
        raise ValueError(f"copies past the {blocks} blocks of {block_size} tokens") from None
    if len(flat) != 3 * len(copies) or not set(map(len, copies)) <= {3}:
        raise ValueError("copies must be (src, dst, tokens)")
    return flat


def check_copies(copies: Sequence[tuple[int, int, int]], blocks: int, block_size: int) -> None:
    """ValueError unless copy_blocks takes these copies in pools of `blocks` blocks of block_size tokens."""
    flat = _flat(copies, blocks, block_size)
    _hip.check(_hip.lib().sipa_check_copies(flat.buffer_info()[0], len(copies), blocks, block_size), "copy_blocks")


def copy_blocks(pools: Sequence[torch.Tensor], copies: Sequence[tuple[int, int, int]]) -> None:
    """For each (src, dst, tokens) of copies, the first `tokens` tokens of block src become those of block dst, in every layer
    and head of the pools, in place (sipa_copy_blocks; one launch for 424 copies). No block may be the destination of two
    copies, or of one and the source of another.

    pools: one to four tensors [L, Hkv, N, B, ...], a cache's K, V and their per-token scales, each head's blocks contiguous.
    Blocks of up to 255 tokens on the GPU. The copies are the host's: a graph captures the ones it was given. CPU pools are copied
    by torch operations."""
    P, n = len(pools), len(copies)
    if not 1 <= P <= 4:
        raise ValueError(f"{P} pools (1 to 4)")
    first = pools[0]
    L, H, N, B = lead = first.shape[:4]
    dev, ptrs, st_l, st_h, row_bytes = first.device, [0] * 4, [0] * 4, [0] * 4, [0] * 4
    for i, t in enumerate(pools):
        if t.shape[:4] != lead or t.device != dev:
            raise ValueError(f"the pools must be {(L, H, N, B, '...')} on one device")
        size, st = t.element_size(), t.stride()
        row = 1
        for x, y in zip(t.shape[:3:-1], st[:3:-1]):
            if x > 1 and y != row:
                raise ValueError("each head's blocks must be contiguous")
            row *= x
        if (B > 1 and st[3] != row) or (N > 1 and st[2] != B * row):
            raise ValueError("each head's blocks must be contiguous")
        ptrs[i], st_l[i], st_h[i], row_bytes[i] = t.data_ptr(), st[0] * size, st[1] * size, row * size
    if not n:
        return
    flat = _flat(copies, N, B)
    at = flat.buffer_info()[0]
    if not first.is_cuda:
        _hip.check(_hip.lib().sipa_check_copies(at, n, N, B), "copy_blocks")
        for t in pools:
            for s, d, rows in copies:
                t[:, :, d, :rows] = t[:, :, s, :rows]
        return
    p = _COPY.pack(_COPY.size, L, H, N, B, P, *ptrs, *st_l, *st_h, *row_bytes, at, n)
    with _hip.on_device(dev):
        rc = _hip.lib().sipa_copy_blocks(p, _hip.stream_of(first))
    if rc:
        _hip.check(rc, "copy_blocks")
