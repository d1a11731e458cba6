"""Rules on a forward's logits before a token is taken from them, on MI355X through libsmallinf_hip.so: penalties for tokens
that are already there, biases, and grammar masks. The reference's engine takes the argmax of the raw logits and has no
counterpart.

For row r of sequence s and token v, in fp32 from the logit l to one rounding at the end:
  made = times v occurs among the sequence's generated tokens and on the row's path (a drafted node's ancestors and the node
         itself); seen = made > 0 or v occurs in the prompt
  l = l / repetition if l > 0 else l * repetition        where seen
  l = l - frequency * made - presence                    where made > 0
  l = l + the values the sequence's bias list gives v, added up in the list's order
  l = -inf                                               where the row's grammar state does not allow v

Nothing is kept between calls, so drafts that are rejected leave nothing to undo: the caller's history grows by the tokens
that were accepted.
"""

from __future__ import annotations

import ctypes
import threading

import numpy as np
import torch

from . import _hip

DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def _overlap(logits: torch.Tensor, out: torch.Tensor) -> bool:
    """Whether out [R, V] has rows over each other, or over logits' [R, V] other than as the same rows."""
    R, V = out.shape
    size, so, sl = out.element_size(), out.stride(0), logits.stride(0)
    if R > 1 and so < V:
        return True
    at, start = out.data_ptr(), logits.data_ptr()
    if at >= start + ((R - 1) * sl + V) * size or start >= at + ((R - 1) * so + V) * size or R * V == 0:
        return False
    if at == start and (R == 1 or so == sl):
        return False
    o, l = at + np.arange(R) * (so * size), start + np.arange(R) * (sl * size)
    i = np.searchsorted(l, o)  # each row of out against the rows of logits that start before and behind it
    behind, before = l[np.minimum(i, R - 1)], l[np.maximum(i - 1, 0)]
    return bool((np.abs(behind - o) < V * size).any() or (np.abs(before - o) < V * size).any())


class LogitsRules:
    """The rules of a batch of `num_seqs` sequences over a vocabulary of `vocab` tokens, checked once and applied to any
    number of steps. Tensors on one device; each may be left out:

    history int32, the sequences' tokens one after the other, with history_starts int64 [S + 1]; prompt_lens int32 [S], how
    many of a sequence's tokens are prompt (0); repetition (positive), frequency, presence fp32 [S]; bias_tokens int32 and
    bias_values fp32, with bias_starts int32 [S + 1]; grammar int32 [states, >= ceil(vocab / 32)], bit v % 32 of word v // 32
    set where the state allows token v. Tokens outside the vocabulary (-1 as padding) are ignored, starts
    are clamped to their lists. The tensors are read at
    every apply(), so a program may write new values into them between steps. Threads may call apply() at the same time."""

    def __init__(self, vocab: int, num_seqs: int, *, history: torch.Tensor | None = None,
                 history_starts: torch.Tensor | None = None, prompt_lens: torch.Tensor | None = None,
                 repetition: torch.Tensor | None = None, frequency: torch.Tensor | None = None,
                 presence: torch.Tensor | None = None, bias_tokens: torch.Tensor | None = None,
                 bias_values: torch.Tensor | None = None, bias_starts: torch.Tensor | None = None,
                 grammar: torch.Tensor | None = None):
        if vocab < 1 or num_seqs < 1:
            raise ValueError(f"vocabulary {vocab}, {num_seqs} sequences")
        self.vocab, self.num_seqs = vocab, num_seqs
        self._lock = threading.Lock()  # of the parameter block, from its filling to the launch
        S = num_seqs

        def check(t, dtype, n, what):
            if t is not None and (t.dtype is not dtype or t.dim() != 1 or (n is not None and t.shape[0] != n) or
                                  not t.is_contiguous()):
                raise ValueError(f"{what} must be a contiguous {dtype} vector" + (f" of {n}" if n is not None else ""))

        if (history is None) != (history_starts is None):
            raise ValueError("history needs history_starts, and they it")
        if prompt_lens is not None and history is None:
            raise ValueError("prompt_lens needs a history")
        if len({t is None for t in (bias_tokens, bias_values, bias_starts)}) > 1:
            raise ValueError("bias_tokens, bias_values and bias_starts go together")
        check(history, torch.int32, None, "history")
        check(history_starts, torch.int64, S + 1, "history_starts")
        check(prompt_lens, torch.int32, S, "prompt_lens")
        for t, what in ((repetition, "repetition"), (frequency, "frequency"), (presence, "presence")):
            check(t, torch.float32, S, what)
        check(bias_tokens, torch.int32, None, "bias_tokens")
        check(bias_values, torch.float32, None if bias_tokens is None else bias_tokens.numel(), "bias_values")
        check(bias_starts, torch.int32, S + 1, "bias_starts")
        if grammar is not None and (grammar.dtype is not torch.int32 or grammar.dim() != 2 or grammar.stride(1) != 1 or
                                    grammar.shape[0] < 1 or grammar.shape[1] * 32 < vocab):
            raise ValueError(f"grammar must be int32 [states, >= {-(-vocab // 32)}] with contiguous rows")
        self.history, self.history_starts, self.prompt_lens = history, history_starts, prompt_lens
        self.repetition, self.frequency, self.presence = repetition, frequency, presence
        self.bias_tokens, self.bias_values, self.bias_starts = bias_tokens, bias_values, bias_starts
        self.grammar = grammar
        self._tensors = [t for t in (history, history_starts, prompt_lens, repetition, frequency, presence, bias_tokens,
                                     bias_values, bias_starts, grammar) if t is not None]
        devices = {t.device for t in self._tensors}
        if len(devices) > 1:
            raise ValueError(f"the rules' tensors must be on one device, got {sorted(map(str, devices))}")
        self.device = devices.pop() if devices else None
        p = self._params = _hip.LogitsParams(struct_size=ctypes.sizeof(_hip.LogitsParams), vocab=vocab, num_seqs=S)
        for name in ("history", "history_starts", "prompt_lens", "repetition", "frequency", "presence", "bias_tokens",
                     "bias_values", "bias_starts", "grammar"):
            setattr(p, name, _hip.ptr(getattr(self, name)) or None)
        if history is not None and history.numel() == 0:  # an empty tensor's address is NULL: no token to count
            p.history = p.history_starts = p.prompt_lens = None
        if bias_tokens is not None and bias_tokens.numel() == 0:
            p.bias_tokens = p.bias_values = p.bias_starts = None
        p.history_size = 0 if history is None else history.numel()
        p.num_biases = 0 if bias_tokens is None else bias_tokens.numel()
        if grammar is not None:
            p.grammar_stride, p.grammar_states = grammar.stride(0), grammar.shape[0]

    def check_sequences(self, n: int) -> None:
        """ValueError unless these are the rules of n sequences: rows of other batches would take other sequences' rules."""
        if n != self.num_seqs:
            raise ValueError(f"rules of {self.num_seqs} sequences for a batch of {n}")

    def apply(self, logits: torch.Tensor, *, query_starts: torch.Tensor | None = None, tokens: torch.Tensor | None = None,
              masks: torch.Tensor | None = None, grammar_rows: torch.Tensor | None = None,
              out: torch.Tensor | None = None) -> torch.Tensor:
        """The adjusted logits [R, vocab], in the logits' type (bf16, fp16 or fp32), in one launch (sipa_adjust_logits).

        Row r is of sequence r (there may be fewer rows than sequences), or with query_starts int32 [S + 1] of the sequence
        whose rows query_starts[s] .. query_starts[s + 1] - 1 it is among; rows of no sequence, before or behind them, are
        copied as they are. tokens int64 [R] and masks int64 [R, words] (engine.hip_tree.tree_maps) give each row its path:
        the tokens of the nodes of its sequence whose bits its mask has. grammar_rows int32 [R]: each row's grammar state, -1
        for none. out may be logits itself, and must not overlap it otherwise. CPU tensors are computed by torch
        operations."""
        if logits.dim() != 2 or logits.shape[1] != self.vocab or logits.dtype not in DTYPES or \
                (self.vocab > 1 and logits.stride(1) != 1):
            raise ValueError(f"logits must be [rows, {self.vocab}] in bf16, fp16 or fp32 with a contiguous last dim")
        R = logits.shape[0]
        if query_starts is None and R > self.num_seqs:
            raise ValueError(f"{R} rows of {self.num_seqs} sequences need query_starts")
        if (tokens is None) != (masks is None):
            raise ValueError("a path needs tokens and masks")
        for t, dtype, shape, what in ((query_starts, torch.int32, (self.num_seqs + 1,), "query_starts"),
                                      (tokens, torch.int64, (R,), "tokens"),
                                      (grammar_rows, torch.int32, (R,), "grammar_rows")):
            if t is not None and (t.dtype is not dtype or t.shape != shape or not t.is_contiguous()):
                raise ValueError(f"{what} must be contiguous {dtype} {shape}")
        if masks is not None and (masks.dtype is not torch.int64 or masks.dim() != 2 or masks.shape[0] != R or
                                  not 1 <= masks.shape[1] <= 4 or not masks.is_contiguous()):
            raise ValueError(f"masks must be contiguous int64 [{R}, 1 to 4 words]")
        if grammar_rows is not None and self.grammar is None:
            raise ValueError("grammar_rows without a grammar")
        if out is not None and (out.shape != logits.shape or out.dtype != logits.dtype or
                                (self.vocab > 1 and out.stride(1) != 1)):
            raise ValueError("out must be as logits, with a contiguous last dim")
        if out is not None and _overlap(logits, out):
            raise ValueError("out's rows overlap each other or other rows of the logits (it may be logits itself)")
        dev = logits.device
        if self.device is not None and self.device != dev:
            raise ValueError(f"logits on {dev}, rules on {self.device}")
        if not logits.is_cuda:
            return self._apply_torch(logits, query_starts, tokens, masks, grammar_rows, out)
        _hip.require_gpu(logits, query_starts, tokens, masks, grammar_rows, out)
        if out is None:
            out = torch.empty_like(logits, memory_format=torch.contiguous_format)
        if R == 0:
            return out
        p = self._params
        with self._lock, _hip.on_device(dev):
            p.num_rows, p.dtype = R, _hip.dtype_code(logits.dtype)
            p.words = 0 if masks is None else masks.shape[1]
            p.logits, p.logits_stride, p.out, p.out_stride = logits.data_ptr(), logits.stride(0), out.data_ptr(), out.stride(0)
            p.query_starts, p.tokens, p.masks = _hip.ptr(query_starts), _hip.ptr(tokens), _hip.ptr(masks)
            p.grammar_rows = _hip.ptr(grammar_rows)
            _hip.check(_hip.lib().sipa_adjust_logits(ctypes.byref(p), _hip.stream_of(logits)), "adjust_logits")
        return out

    def _apply_torch(self, logits, query_starts, tokens, masks, grammar_rows, out) -> torch.Tensor:
        """apply() on CPU tensors, row by row."""
        R, V = logits.shape
        qs = list(range(R + 1)) if query_starts is None else query_starts.clamp(0, R).tolist()
        hs = None if self.history is None else self.history_starts.clamp(0, self.history.numel()).tolist()
        bs = None if self.bias_starts is None else self.bias_starts.clamp(0, self.bias_tokens.numel()).tolist()
        words = None if masks is None else masks.tolist()
        result = logits.float()
        if result is logits:
            result = logits.clone()

        def count(of: torch.Tensor) -> torch.Tensor:
            of = of.long()
            return torch.bincount(of[(of >= 0) & (of < V)], minlength=V)

        for s, (a, b) in enumerate(zip(qs, qs[1:])):
            prompt = made = torch.zeros(V, dtype=torch.int64)
            if hs is not None:
                mine = self.history[hs[s]:hs[s + 1]]
                at = 0 if self.prompt_lens is None else max(0, int(self.prompt_lens[s]))
                prompt, made = count(mine[:at]), count(mine[at:])
            bias = torch.zeros(V)
            if bs is not None:
                for v, x in zip(self.bias_tokens[bs[s]:bs[s + 1]].tolist(), self.bias_values[bs[s]:bs[s + 1]]):
                    if 0 <= v < V:
                        bias[v] += x
            for r in range(a, b):
                m = made
                if words is not None:
                    path = [i for i in range(min(b - a, 64 * len(words[r]))) if words[r][i // 64] >> (i % 64) & 1]
                    m = made + count(tokens[[a + i for i in path]])
                l = result[r]
                if self.repetition is not None:
                    rho = self.repetition[s]
                    l = torch.where((m > 0) | (prompt > 0), torch.where(l > 0, l / rho, l * rho), l)
                if self.frequency is not None:
                    l = l - self.frequency[s] * m
                if self.presence is not None:
                    l = l - self.presence[s] * (m > 0)
                if bs is not None:
                    l = l + bias
                if grammar_rows is not None and 0 <= int(grammar_rows[r]) < self.grammar.shape[0]:
                    word = self.grammar[int(grammar_rows[r])]
                    v = torch.arange(V)
                    l = l.masked_fill((word[v // 32] >> (v % 32) & 1) == 0, float("-inf"))
                result[r] = l
        if out is None:
            return result.to(logits.dtype)
        return out.copy_(result)
