"""Sampling of the next token from logits (host side of ``dkv_sample.hip``).

The generators take the most probable token (the reference's benchmark decodes greedily,
``scripts/benchmark_throughput.py:17-30``; its models inherit transformers' ``generate`` with
temperature, top-k, top-p and min-p). ``sample_tokens`` draws a token per row under these filters from
a uniform number that the caller gives, so a draw can be repeated; it is one launch, or three where
few rows of a large vocabulary are cut among workgroups.
"""

from __future__ import annotations

import torch

from .. import _lib

MAX_VOCAB = 1 << 19


def _setting(value, rows: int, dtype: torch.dtype, device: int, name: str):
    """(pointer of a per-row tensor or None, the value for every row)."""
    if not isinstance(value, torch.Tensor):
        return None, value
    if value.shape != (rows,) or value.dtype != dtype or not value.is_contiguous():
        raise ValueError(f"{name} must be a number or a contiguous ({rows},) {dtype} tensor")
    if value.get_device() != device:
        raise ValueError(f"{name} must be on the logits' device")
    return value.data_ptr(), 0


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, *, temperature=1.0, top_k=0, top_p=1.0,
                  min_p=0.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """A token per row: (rows,) int64.

    ``logits`` (rows, V) in bf16, fp16 or fp32 with unit last stride, V <= 524288; ``u`` (rows,)
    fp32, uniform in [0, 1). Each setting is a number or a (rows,) tensor (``top_k`` int32, the
    others fp32). With w_i = exp((l_i - max l) / temperature), and tokens in the order of their
    logits (of equal ones the lowest index first):

    * ``top_k`` keeps the first k (0, negative or >= V: all);
    * ``top_p`` keeps, of those, the tokens before which less than ``top_p`` of their mass lies
      (1 or more: all);
    * ``min_p`` keeps, of those, the ones with w_i >= ``min_p``.

    The first token is always kept. The result is the first token, in the vocabulary's order, up to
    which the kept mass exceeds u times all of it. ``temperature`` 0 (or below) takes the first
    token. A logit of -inf is never taken, NaN counts as -inf, +inf ones share the mass among
    themselves, and a row with no logit above -inf gives -1. Masses are sums in 64-bit fixed
    point, so the same call gives the same tokens every time."""
    fast = _lib.tensor_calls()
    if fast is not None and out is None:
        dev = logits.get_device()
        if _lib.is_current(dev):
            out = fast.sample_tokens(_lib.stream_on(dev), dev, logits, u, temperature, top_k, top_p,
                                     min_p)
            if out is not None:
                return out
    shape, st = logits.shape, logits.stride()
    if len(shape) != 2 or (shape[1] > 1 and st[1] != 1):
        raise ValueError("logits must be (rows, V) with unit last stride")
    rows, V = shape
    if V == 0:
        raise ValueError("logits have no vocabulary")
    if V > MAX_VOCAB:
        raise NotImplementedError(f"vocabularies of at most {MAX_VOCAB} tokens")
    dev = logits.get_device()
    if (u.shape != (rows,) or u.dtype != torch.float32 or not u.is_contiguous()
            or u.get_device() != dev):
        raise ValueError(f"u must be a contiguous ({rows},) float32 tensor on the logits' device")
    t_ptr, t = _setting(temperature, rows, torch.float32, dev, "temperature")
    k_ptr, k = _setting(top_k, rows, torch.int32, dev, "top_k")
    p_ptr, p = _setting(top_p, rows, torch.float32, dev, "top_p")
    m_ptr, m = _setting(min_p, rows, torch.float32, dev, "min_p")
    stream = _lib.stream_of(logits)
    if out is None:
        out = torch.empty_like(u, dtype=torch.int64)
    elif (out.shape != (rows,) or out.dtype != torch.int64 or not out.is_contiguous()
          or out.get_device() != dev):
        raise ValueError(f"out must be a contiguous ({rows},) int64 tensor on the logits' device")
    lib, code = _lib.calls(), _lib.dtype_code(logits.dtype)
    # a workspace of the call's own, in its stream's order: nothing of it outlives the call
    need = lib.dkv_sample_workspace_bytes(code, rows, V)
    ws = logits.new_empty(need, dtype=torch.uint8) if need else None
    _lib.check(_lib.call_on(
        dev, lib.dkv_sample_tokens, stream, code, logits.data_ptr(), st[0] if rows > 1 else V,
        rows, V, u.data_ptr(), t_ptr, float(t), k_ptr, int(min(max(k, 0), V)), p_ptr, float(p),
        m_ptr, float(m), _lib.ptr(ws), need, out.data_ptr()), "dkv_sample_tokens")
    return out
