"""Sampling of the next token from logits (host side of ``dkv_sample.hip``, ``dkv_logits.hip``).

The generators take the most probable token (the reference's benchmark decodes greedily,
``scripts/benchmark_throughput.py:17-30``; its models inherit transformers' ``generate`` with
temperature, top-k, top-p and min-p). ``sample_tokens`` draws a token per row under these filters from
a uniform number that the caller gives, so a draw can be repeated; it is one launch, or three where
few rows of a large vocabulary are cut among workgroups. ``adjust_logits_`` comes before it where a
request has penalties for the tokens it has seen, biased tokens or a mask of allowed ones.
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


def _rows_of(t: torch.Tensor, rows: int, dtypes: tuple, device: int, name: str) -> int:
    """The row stride of (rows, n), checked."""
    if t.dim() != 2 or t.shape[0] != rows or t.dtype not in dtypes:
        raise ValueError(f"{name} must be ({rows}, n) of {' or '.join(str(d) for d in dtypes)}")
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{name} must have unit last stride")
    if t.get_device() != device:
        raise ValueError(f"{name} must be on the logits' device")
    return t.stride(0) if rows > 1 else t.shape[1]


def adjust_logits_(logits: torch.Tensor, *, tokens: torch.Tensor | None = None, prompt_lens=None,
                   lens=None, repetition=1.0, frequency=0.0, presence=0.0,
                   bias_ids: torch.Tensor | None = None, bias: torch.Tensor | None = None,
                   allowed: torch.Tensor | None = None) -> torch.Tensor:
    """Penalties, biases and a mask on ``logits`` (rows, V), in place; returns them.

    Row b's request has the tokens ``tokens[b, :lens[b]]`` (int32 or int64; ``lens`` a number or a
    (rows,) int32 tensor, all by default), the first ``prompt_lens[b]`` of them given (0 by
    default), the others generated. Settings are numbers or (rows,) fp32 tensors. In this order, for a
    token that is

    * in ``tokens``: x / ``repetition`` where x > 0, else x * ``repetition`` (which must be positive and
      finite: a number is checked, a tensor's entries, which would have to be read back, are not);
    * generated n > 0 times: x - n * ``frequency`` - ``presence``;
    * in ``bias_ids[b]`` ((rows, M) int32): x + its ``bias[b]`` ((rows, M) fp32), several of one token
      added up in their order;
    * not allowed, bit i % 32 of ``allowed[b, i // 32]`` ((rows, >= V / 32) int32) being 0: -infinity.

    In fp32, rounded once to the logits' type (bf16, fp16 or fp32). Ids outside the vocabulary are
    passed over (pad with -1); a row stride may be 0 (one row expanded to all), but for the logits'.
    Logits that nothing concerns are neither read nor written, so the cost goes by the histories' and
    masks' size."""
    fast = _lib.tensor_calls()
    if fast is not None:
        dev = logits.get_device()
        if _lib.is_current(dev) and fast.adjust_logits(
                _lib.stream_on(dev), dev, logits, tokens, prompt_lens, lens, repetition, frequency,
                presence, bias_ids, bias, allowed):
            return logits
    shape, st = logits.shape, logits.stride()
    if len(shape) != 2 or (shape[1] > 1 and st[1] != 1):
        raise ValueError("logits must be (rows, V) with unit last stride")
    rows, V = shape
    if rows > 1 and st[0] < V:
        raise ValueError("rows of logits must not share memory")
    code, dev = _lib.dtype_code(logits.dtype), logits.get_device()
    settings = [_setting(v, rows, torch.float32, dev, name) for v, name in (
        (repetition, "repetition"), (frequency, "frequency"), (presence, "presence"))]
    if not isinstance(repetition, torch.Tensor) and not 0.0 < repetition < float("inf"):
        raise ValueError("repetition must be positive and finite")
    if tokens is None:
        if prompt_lens is not None or lens is not None:
            raise ValueError("prompt_lens and lens need tokens")
        if any(isinstance(v, torch.Tensor) or v != none
               for v, none in ((repetition, 1.0), (frequency, 0.0), (presence, 0.0))):
            raise ValueError("penalties need tokens")
        N, t_ld, size = 0, 0, 4
    else:
        t_ld = _rows_of(tokens, rows, (torch.int32, torch.int64), dev, "tokens")
        N, size = tokens.shape[1], tokens.element_size()
    p_ptr, p = _setting(0 if prompt_lens is None else prompt_lens, rows, torch.int32, dev, "prompt_lens")
    l_ptr, n = _setting(N if lens is None else lens, rows, torch.int32, dev, "lens")
    if (bias_ids is None) != (bias is None):
        raise ValueError("give bias_ids and bias, or neither")
    M = i_ld = b_ld = a_ld = 0
    if bias is not None:
        i_ld = _rows_of(bias_ids, rows, (torch.int32,), dev, "bias_ids")
        b_ld = _rows_of(bias, rows, (torch.float32,), dev, "bias")
        M = bias.shape[1]
        if bias_ids.shape != bias.shape:
            raise ValueError("bias_ids and bias differ in shape")
    if allowed is not None:
        a_ld = _rows_of(allowed, rows, (torch.int32,), dev, "allowed")
        if allowed.shape[1] * 32 < V:
            raise ValueError(f"allowed has {allowed.shape[1]} words for {V} tokens")
    stream = _lib.stream_of(logits)
    _lib.check(_lib.call_on(
        dev, _lib.calls().dkv_adjust_logits, stream, code, logits.data_ptr(),
        st[0] if rows > 1 else V, rows, V, _lib.ptr(tokens), size, t_ld, N, p_ptr,
        min(max(int(p), 0), N), l_ptr, min(max(int(n), 0), N),
        *(x for ptr, v in settings for x in (ptr, float(v) if ptr is None else 1.0)),
        _lib.ptr(bias_ids), i_ld, _lib.ptr(bias), b_ld, M, _lib.ptr(allowed), a_ld),
        "dkv_adjust_logits")
    return logits
