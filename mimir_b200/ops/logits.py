"""Penalties for repeated tokens, biases and grammar masks on next-token logits.

The decoding rules of the OpenAI request fields (``presence_penalty``, ``frequency_penalty``,
``logit_bias``), of Transformers' ``repetition_penalty`` and of constrained decoding.  The
reference leaves them to its patched vLLM (``src/mimir/serving/server.py:12-75``).

CUDA: one kernel (``csrc/logits.cu``), one read and one write of the logits.  CPU: PyTorch.
"""
from __future__ import annotations

import math

import torch

from mimir_b200.ops._ext import ext, kernels_enabled


def process_logits(logits, *, tokens=None, token_lens=None, prompt_lens=None, repetition=None, presence=None,
                   frequency=None, bias=None, allowed=None, out=None):
    """float32 ``[rows, vocab]``: ``logits`` (bfloat16, float16 or float32, any row stride) after, in this order,

    * the repetition penalty: a logit of a token of the row is divided by ``repetition[row]`` where it
      is positive and multiplied where not;
    * the frequency and presence penalties: ``- frequency[row] * c - presence[row]`` for a token that was
      generated ``c > 0`` times (tokens from ``prompt_lens[row]`` on);
    * ``bias = (offsets, ids, values)``: row ``r`` adds ``values[i]`` to token ``ids[i]`` for ``i`` in
      ``offsets[r]:offsets[r + 1]`` (equal ids add up; offsets outside the list end at its ends);
    * the mask: -inf where bit ``v % 32`` of word ``v // 32`` of ``allowed[row]`` (int32) is zero, whatever
      the logit was.  A row that allows nothing is all -inf.

    ``tokens`` int32 ``[rows, history]`` holds each row's prompt and generated tokens, the first
    ``token_lens[row]`` of them (all by default); ids outside the vocabulary (padding) count for nothing.
    Penalties are float32 ``[rows]``; lengths and offsets int32.  ``out``: a contiguous float32 tensor for
    the result; the logits themselves where they are one.
    """
    offsets, ids, values = (None, None, None) if bias is None else bias
    if kernels_enabled(logits):
        return ext().process_logits(logits, tokens, token_lens, prompt_lens, repetition, presence, frequency, offsets,
                                    ids, values, allowed, out)
    result = process_logits_reference(logits, tokens, token_lens, prompt_lens, repetition, presence, frequency, offsets,
                                      ids, values, allowed)
    return result if out is None else out.copy_(result)


def process_logits_reference(logits, tokens, token_lens, prompt_lens, repetition, presence, frequency, offsets, ids,
                             values, allowed):
    """PyTorch formulation, a row at a time."""
    if logits.ndim != 2 or not logits.is_floating_point():
        raise ValueError("logits must be [rows, vocab]")
    rows, vocab = logits.shape
    if tokens is None and any(x is not None for x in (token_lens, prompt_lens, repetition, presence, frequency)):
        raise ValueError("lengths and penalties need tokens")
    for name, t, size in (("token_lens", token_lens, rows), ("prompt_lens", prompt_lens, rows),
                          ("repetition", repetition, rows), ("presence", presence, rows),
                          ("frequency", frequency, rows), ("the bias offsets", offsets, rows + 1)):
        if t is not None and t.shape != (size,):
            raise ValueError(f"{name} must be a tensor of {size}")
    if allowed is not None and (allowed.dtype != torch.int32 or allowed.shape != (rows, -(-vocab // 32))):
        raise ValueError("allowed must be int32 [rows, ceil(vocab / 32)]")
    x = logits.float().clone()
    for r in range(rows):
        row = x[r]
        if tokens is not None:
            n = tokens.shape[1] if token_lens is None else int(token_lens[r])
            first = 0 if prompt_lens is None else int(prompt_lens[r])
            held, made = tokens[r, :n].long(), tokens[r, first:n].long()
            held, made = held[(held >= 0) & (held < vocab)], made[(made >= 0) & (made < vocab)]
            if repetition is not None:
                seen = torch.unique(held)
                row[seen] = torch.where(row[seen] > 0, row[seen] / repetition[r], row[seen] * repetition[r])
            seen, count = torch.unique(made, return_counts=True)
            if frequency is not None:
                row[seen] -= frequency[r] * count
            if presence is not None:
                row[seen] -= presence[r]
        if offsets is not None:
            span = slice(max(int(offsets[r]), 0), max(int(offsets[r + 1]), 0))
            ok = (ids[span] >= 0) & (ids[span] < vocab)
            row += torch.zeros_like(row).index_add_(0, ids[span][ok].long(), values[span][ok])
    if allowed is not None:
        v = torch.arange(vocab, device=x.device)
        x = torch.where((allowed[:, v // 32] >> (v % 32).to(torch.int32)) & 1 != 0, x, torch.full_like(x, -math.inf))
    return x
