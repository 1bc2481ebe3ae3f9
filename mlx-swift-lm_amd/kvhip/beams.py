"""Beam search over device caches: the selection over beams and vocabulary.  Every cache's `reorder` takes the rows it returns."""
from __future__ import annotations

import torch

from . import _lib as L
from .cache import _DT, _ptr, _stream
from .recurrent import _on_current_device


def beam_select(logits, scores=None, count=None, done=None, pad_token=0):
    """The `count` (default: as many as there are beams) best continuations of each batch row's beams: (rows, tokens, scores), each
    [B, count], best first.  logits [B, K, V]; scores [B, K] (float32), what each beam has so far; done [B, K]: beams that offer
    `pad_token` alone, at their own score.  `rows` are rows of the B K logits (int32), an order for `cache.reorder` when count
    is K; a continuation scores scores + log softmax(logits); among equals the lower beam, then the higher logit, then the lower
    token.  Where there are fewer candidates: -1, -1 and minus infinity."""
    if scores is not None and done is None and logits.is_cuda:
        L.init()
        native, entry, workspace = L.native("select", "kvhip_beam_select")  # (of the ordinary form, as one native call)
        out = native(entry, workspace, logits, scores, logits.shape[1] if count is None else count, pad_token) if native and logits.dim() == 3 else None
        if type(out) is int:
            L.check(out)
        if out is not None:
            return out
    if logits.dim() != 3 or logits.dtype not in _DT:
        raise ValueError(f"logits are [B, K, V] in float16, bfloat16 or float32, not {logits.dtype} {tuple(logits.shape)}")
    B, K, V = logits.shape
    count = K if count is None else int(count)
    if scores is not None and (tuple(scores.shape) != (B, K) or scores.dtype != torch.float32):
        raise ValueError(f"scores are float32 {(B, K)}, not {scores.dtype} {tuple(scores.shape)}")
    if done is not None and (tuple(done.shape) != (B, K) or done.dtype not in (torch.bool, torch.uint8)):
        raise ValueError(f"done is bool {(B, K)}, not {done.dtype} {tuple(done.shape)}")
    pitch = logits.stride(1 if K > 1 else 0)  # elements from a row to the next
    if (V > 1 and logits.stride(2) != 1) or (B > 1 and logits.stride(0) != K * pitch):
        logits = logits.contiguous()
        pitch = V
    scores, done = (None if t is None else t.contiguous() for t in (scores, done))
    _on_current_device(logits, scores, done)
    L.init()
    lib = L.load()
    out = torch.empty((3, B, max(count, 0)), dtype=torch.int32, device=logits.device)
    rows, tokens, best = out[0], out[1], out[2].view(torch.float32)
    need = lib.kvhip_beam_select_workspace(B, K, V, _DT[logits.dtype], count)
    scratch = torch.empty(need, dtype=torch.uint8, device=logits.device)
    L.check(lib.kvhip_beam_select(_ptr(logits), pitch, B, K, V, _DT[logits.dtype], None if scores is None else _ptr(scores),
                                  None if done is None else _ptr(done), count, int(pad_token), _ptr(rows), _ptr(tokens), _ptr(best),
                                  _ptr(scratch) if need else None, need, _stream()))
    return rows, tokens, best
