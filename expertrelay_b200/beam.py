"""Beam search's choice of continuations: the kernels of csrc/er_beam.cu.

The reference decodes greedily (runtime/generate.py); its forward pass gives
one row of logits a sequence. With several sequences in a call (PagedKVCache)
the rows of a text's beams come together, and select picks the continuations.
"""

from __future__ import annotations

import functools

import torch

from . import _lib, kv


@functools.lru_cache(maxsize=1024)
def _bytes(device: int, *sizes: int) -> int:
    """The workspace of a call of these sizes on a device (the current one)."""
    return _lib.lib().er_beam_workspace_bytes(*sizes)


def select(logits: torch.Tensor, scores: torch.Tensor, count: int, *,
           workspace: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The best `count` continuations of every batch, best first: (scores
    float32, beams int32, tokens int32), each [batch, count]. A candidate's
    value is scores[b, i] + log_softmax(logits[b * beams + i])[token]; scores
    [batch, beams] float32, logits [batch * beams, vocab] float32 or bfloat16
    (rows may be strided). Values are compared in 64 bits; ties go to the lower
    beam, then the lower token, and within a beam the higher logit wins. A beam's
    log-sum is good to 2^-20, so candidates of different beams that are closer
    than that may come in either order (equal rows of equal score tie). A beam
    whose score is infinite or NaN, or whose logits hold a NaN or +inf or
    nothing but -inf, offers nothing: its candidates have value -inf, like
    logits of -inf. count: at most 128 and beams x vocab; at most 1024 beams and
    65535 rows. Queued on the device's current stream. workspace: scratch of
    one's own (ValueError names the bytes needed), for one call at a time."""
    if not isinstance(logits, torch.Tensor) or logits.dim() != 2 or logits.dtype not in kv._DTYPES or \
            not logits.is_cuda or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits: expected a [batch * beams, vocab] float32 or bfloat16 CUDA tensor, rows contiguous")
    if not isinstance(scores, torch.Tensor) or scores.dim() != 2:
        raise ValueError("scores: expected [batch, beams] float32")
    kv._need(scores, "scores", torch.float32, logits.device)
    (batch, beams), (rows, vocab) = scores.shape, logits.shape
    if rows != batch * beams:
        raise ValueError(f"logits: {rows} rows for {batch} batches of {beams} beams")
    if rows > 1 and logits.stride(0) < vocab:
        raise ValueError(f"logits: rows of {vocab} by a stride of {logits.stride(0)}")
    if count < 1:
        raise ValueError(f"count: at least 1, got {count}")
    index = logits.device.index
    if torch._C._cuda_getDevice() != index:
        with torch.cuda.device(index):
            return select(logits, scores, count, workspace=workspace)
    lib = _lib.lib()
    best = scores.new_empty((batch, count))
    beams_out, tokens_out = torch.empty((2, batch, count), dtype=torch.int32, device=logits.device).unbind(0)
    need = _bytes(index, batch, beams, vocab, count)
    ws = kv._scratch(need, workspace, logits.device) if need else None
    _lib.check(lib.er_beam_select(logits.data_ptr(), kv._DTYPES[logits.dtype], logits.stride(0) if rows > 1 else vocab,
                                  scores.data_ptr(), batch, beams, vocab, count, best.data_ptr(), beams_out.data_ptr(),
                                  tokens_out.data_ptr(), ws.data_ptr() if need else None, need,
                                  torch._C._cuda_getCurrentRawStream(index)), "er_beam_select")
    return best, beams_out, tokens_out
