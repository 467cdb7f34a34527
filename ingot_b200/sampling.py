"""What follows the lm_head GEMV on the decode path: penalties, biases and grammar masks on the logits, arg-max per row and the sampler's 64 candidates per row
(argmax_rows, Shaders/verify.metal:525-547; TopK64, Shaders/zz_sample.metal and Tests/IngotTests/TopK64Tests.swift)."""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

import torch

from . import capi
from .linear import _DT, _no_cpu, _raw_stream, _stream_ptr

CANDIDATES = 64


def argmax_rows(x: torch.Tensor, rows: int, stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Index of the largest logit of each of the first `rows` rows of x (fp32 [*, n]); ties go to the lower index."""
    if not x.is_cuda:
        _no_cpu()
    if x.dtype != torch.float32:
        raise TypeError("logits are float32")
    ctx = capi.context(x.device.index or 0)
    out = torch.empty(rows, dtype=torch.int32, device=x.device)
    ctx.check(capi.call().argmax_rows(ctx.address, _stream_ptr(stream), x.data_ptr(), x.stride(0), rows, x.shape[1],
                                      out.data_ptr()))
    return out


class TopK64:
    """Scratch sized once for (rows, vocabulary); `encode` enqueues the kernel."""

    def __init__(self, max_rows: int, vocab: int, device: torch.device):
        n = C.c_size_t()
        if capi.lib().iq_topk64_scratch_bytes(max_rows, vocab, C.byref(n)) != 0:
            raise ValueError("TopK64 takes 1..16 rows and up to 262,144 logits per row")
        self.max_rows, self.vocab = max_rows, vocab
        self.scratch = torch.empty(n.value, dtype=torch.uint8, device=device)
        self.ctx = capi.context(device.index or 0)

    def encode(self, x: torch.Tensor, rows: int, temperatures: Sequence[float], stream: Optional[torch.cuda.Stream] = None):
        """Returns (idx int32 [rows, 64], val float32 [rows, 64], z float32 [rows, 2] = (max, sum exp((x - max) / T)))."""
        if not x.is_cuda:
            _no_cpu()
        if x.dtype != torch.float32 or rows > self.max_rows or x.shape[1] != self.vocab:
            raise ValueError("TopK64: float32 logits [rows <= max_rows, vocab]")
        idx = torch.empty(rows, CANDIDATES, dtype=torch.int32, device=x.device)
        val = torch.empty(rows, CANDIDATES, dtype=torch.float32, device=x.device)
        z = torch.empty(rows, 2, dtype=torch.float32, device=x.device)
        t = (C.c_float * len(temperatures))(*temperatures)
        self.ctx.check(capi.call().topk64(self.ctx.address, _stream_ptr(stream), x.data_ptr(), x.stride(0), rows, self.vocab,
                                          C.addressof(t), len(temperatures), idx.data_ptr(), val.data_ptr(), z.data_ptr(),
                                          self.scratch.data_ptr(), self.scratch.numel()))
        return idx, val, z


class LogitRules:
    """Penalties of repeated tokens, biases of tokens and grammar masks for `rows` rows of logits (iq_logits_rules): what a batch's requests ask for, as
    device tensors that the caller fills and changes between steps; `encode` applies them to a step's logits. None: a rule that no row has.

    tokens int32 [rows, capacity], lens int32 [rows]: the conversations so far; prompt_lens int32 [rows]: how much of them is prompt (None: nothing).
    repetition (above 0; 1: none), presence, frequency (0: none) float32 [rows]. bias_offsets int32 [rows + 1], bias_tokens int32 [n], bias_values float32 [n].
    mask int32 or uint32 [masks, at least vocab / 32]: bit t % 32 of word t / 32 allows token t; mask_rows int32 [rows]: a row's mask, -1 for none (None: its own)."""

    MAX_VOCAB, MAX_HISTORY, MAX_LIST = 262144, 1 << 30, 2**31 - 1

    def __init__(self, rows: int, vocab: int, *, tokens=None, lens=None, prompt_lens=None, repetition=None, presence=None, frequency=None, bias_offsets=None,
                 bias_tokens=None, bias_values=None, mask=None, mask_rows=None):
        if rows < 1 or not 1 <= vocab <= self.MAX_VOCAB:
            raise ValueError(f"rows = {rows}, vocab = {vocab} (1 to {self.MAX_VOCAB})")
        if (tokens is None) != (lens is None) or (tokens is None and prompt_lens is not None):
            raise ValueError("a history is tokens and lens (and prompt_lens)")
        if (bias_offsets is None) != (bias_tokens is None) or (bias_tokens is None) != (bias_values is None):
            raise ValueError("biases are offsets, tokens and values")
        if mask is None and mask_rows is not None:
            raise ValueError("mask_rows without masks")
        per_row = {"lens": (lens, torch.int32), "prompt_lens": (prompt_lens, torch.int32), "repetition": (repetition, torch.float32), "presence": (presence, torch.float32),
                   "frequency": (frequency, torch.float32), "mask_rows": (mask_rows, torch.int32)}
        for name, (t, dtype) in per_row.items():
            if t is not None and (t.dtype != dtype or t.dim() != 1 or t.shape[0] < rows or not t.is_contiguous()):
                raise ValueError(f"{name} is {dtype} [at least {rows}], contiguous")
        for name, t in (("bias_offsets", bias_offsets), ("bias_tokens", bias_tokens)):
            if t is not None and (t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous()):
                raise ValueError(f"{name} is int32 in one dimension, contiguous")
        if bias_offsets is not None and bias_offsets.shape[0] < rows + 1:
            raise ValueError(f"bias_offsets has {rows} + 1 entries")
        if bias_values is not None and (bias_values.dtype != torch.float32 or bias_values.shape != bias_tokens.shape or not bias_values.is_contiguous()):
            raise ValueError("bias_values is float32, one per bias token, contiguous")
        if tokens is not None and (tokens.dtype != torch.int32 or tokens.dim() != 2 or tokens.shape[0] < rows or (tokens.shape[1] > 1 and tokens.stride(1) != 1)):
            raise ValueError(f"tokens is int32 [at least {rows}, capacity] with neighbouring elements in a row")
        if mask is not None and (mask.dtype not in (torch.int32, torch.uint32) or mask.dim() != 2 or mask.shape[1] < (vocab + 31) // 32
                                 or (mask.shape[1] > 1 and mask.stride(1) != 1) or mask.shape[0] < (rows if mask_rows is None else 1)):
            raise ValueError(f"mask is int32 [masks, at least {(vocab + 31) // 32}], one per row unless mask_rows tells")
        if tokens is not None and tokens.shape[1] > self.MAX_HISTORY:
            raise ValueError(f"tokens has a capacity of {tokens.shape[1]} (up to {self.MAX_HISTORY})")
        for name, t in (("bias_tokens", bias_tokens), ("mask", mask)):
            if t is not None and t.shape[0] > self.MAX_LIST:
                raise ValueError(f"{name} has {t.shape[0]} entries (up to {self.MAX_LIST})")
        self.rows, self.vocab = rows, vocab
        self._kept = tuple(t for t in (tokens, lens, prompt_lens, repetition, presence, frequency, bias_offsets, bias_tokens, bias_values, mask, mask_rows) if t is not None)
        for t in self._kept:
            if t.device != self._kept[0].device:
                raise ValueError("the tensors are on different devices")
        self.device = self._kept[0].device if self._kept else None
        if self.device is not None and self.device.type != "cuda":
            _no_cpu()
        self._index = None if self.device is None else self.device.index
        at = lambda t: 0 if t is None else t.data_ptr()
        wide = lambda t: 0 if t is None else t.stride(0) if t.shape[0] > 1 else t.shape[1]
        self._c = capi.LogitRules(at(tokens), wide(tokens), at(lens), at(prompt_lens), at(repetition), at(presence), at(frequency), at(bias_offsets), at(bias_tokens),
                                  at(bias_values), at(mask), wide(mask), at(mask_rows), 0 if tokens is None else tokens.shape[1],
                                  0 if bias_tokens is None else bias_tokens.shape[0], 0 if mask is None else mask.shape[0])
        self._at = C.addressof(self._c)

    def __getstate__(self):
        raise TypeError("rules hold device addresses: make new ones from the tensors")

    def _check(self, x, rows, out):
        """Shapes, types and devices, whatever device they are on."""
        if x.dtype not in _DT or (out is not None and out.dtype != torch.float32):
            raise TypeError("logits are float32, float16 or bfloat16, the result float32")
        for name, t in (("x", x), ("out", out)):
            if t is not None and (t.dim() != 2 or t.shape[0] < rows or t.shape[1] != self.vocab or (self.vocab > 1 and t.stride(1) != 1)):
                raise ValueError(f"{name} is [at least {rows}, {self.vocab}] with neighbouring elements in a row, not {tuple(t.shape)}")
        if not 0 <= rows <= self.rows:
            raise ValueError(f"rows = {rows}: these rules are for {self.rows}")
        if (out is not None and out.device != x.device) or (self.device is not None and x.device != self.device):
            raise ValueError("the tensors are on different devices")

    def encode(self, x: torch.Tensor, rows: int, out: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
        """The first `rows` rows of logits x [*, vocab] under the rules, as float32 into out (x itself where that is float32; None: a new tensor)."""
        dev = x.get_device()
        if out is None and dev >= 0:
            with torch.cuda.stream(stream):  # (None: the current one) the memory's stream is the kernel's
                out = torch.empty(x.shape, dtype=torch.float32, device=x.device)
        st = None
        if dev >= 0 and (self._index is None or self._index == dev) and rows <= self.rows:
            # (the other conditions are looked at in csrc/pycall.c, and what fails one is described by _check)
            ctx = capi.context(dev)
            st = capi.call().logits_rules(ctx.address, stream.cuda_stream if stream is not None else _raw_stream(dev), dev, x, out, rows, self.vocab, self._at)
        if st is None:
            self._check(x, rows, out)
            if not x.is_cuda:
                _no_cpu()
            raise ValueError("LogitRules does not take these tensors")
        if st:
            ctx.check(st)
        return out
