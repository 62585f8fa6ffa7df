"""End-to-end Llama decoder over the compressed cache, and the same model with a dense cache.

The reference runs DynaKV inside HF's Llama (``custom_llama.py:93-323``, the attention module
``compressed_attention.py:204-386``) and times greedy generation with
``benchmark_throughput.py:17-82`` (tokens/s = batch * new tokens / wall time, prefill included).
This module is that model path for this build, written against the kernels directly (no
transformers model classes: their Cache API differs across versions, and the benchmark needs
only the forward math):

* ``RandomLlama``: Llama weights drawn on the device (N(0, 0.02) in bf16 by default) for a
  given shape (config 5: Llama-3-8B -- hidden 4096, 32 layers, 32/8 heads, head dim 128, FFN
  14336, vocab 128256), plus the DynaKV parameters per layer: a random orthogonal 128x128
  spectral basis per KV head for K and for V, the K/V projections merged with the basis
  transposes so that they emit coefficients (the one-time merge of
  ``compressed_attention.py:263-292``), and per-head cutoff heads whose bias ramps over the
  rank so that the retained fraction is close to a target (``retention``).
* ``CompressedLlama.generate``: prefill (cutoff head, packed append, reconstruct-and-attend)
  then greedy decode steps (cutoff head, decode append, routed decode attention). q/k/v and
  gate/up are one concatenated projection each; at decode sizes the projections run on the
  skinny GEMM (``kernels/model_ops.py``), with the residual add and the RMSNorm before them
  folded into its x staging for one or two rows, and the SwiGLU product is one kernel --
  the same stages serve the dense baseline.
* ``PagedLlama.generate``: the same weights over a paged uncompressed cache
  (``kernels/paged.py``), for prompts of different lengths that come and go: prompts go through
  in chunks beside the other requests' single tokens; its pages may be of 8 bits. Generation is
  greedy, or drawn by a ``Sampler`` (``kernels/sampling.py``), which the other generators take too.
* ``DenseLlama.generate``: the uncompressed-cache baseline of the same weights (K/V kept in
  full in a preallocated cache; decode attention by the same split kernel over that cache read
  as a packed cache with all 128 dims per token and an identity basis, prefill attention by
  torch's scaled_dot_product_attention).
"""

from __future__ import annotations

import math
import time
from dataclasses import dataclass, field
from typing import Sequence

import torch
import torch.nn.functional as F
from torch.nn.attention import SDPBackend, sdpa_kernel

from .formats import merge_projection
from .kernels.compressed_cache import CustomDynamicCache
from .kernels.cutoff import CutoffHead
from .kernels.decode import dense_append_, dense_decode_attention, grouped_decode_attention
from .kernels.layer import DecodeLayerPlan
from .kernels.model_ops import linear, rmsnorm_glu, rmsnorm_linear
from .kernels.paged import PagedBatch, PagedKVCache, paged_append, paged_attention
from .kernels.prefill import coef_prefill_attention, rope_dense_
from .kernels.router import KernelPolicy
from .kernels.sampling import adjust_logits_, sample_tokens


@dataclass(frozen=True)
class LlamaShape:
    hidden: int = 4096
    layers: int = 32
    heads: int = 32
    kv_heads: int = 8
    head_dim: int = 128
    ffn: int = 14336
    vocab: int = 128256
    theta: float = 500000.0
    eps: float = 1e-5
    # norms of each query and key head before the rotation (the reference's second model family,
    # custom_qwen3.py): PagedLlama alone takes such a shape
    qk_norm: bool = False


@dataclass
class LayerWeights:
    ln1: torch.Tensor
    w_qkv_c: torch.Tensor  # (H + 2 G Dh, H): q, then the merged K / V coefficient projections
    w_qkv: torch.Tensor    # (H + 2 G Dh, H): q, K, V of the dense baseline
    wq: torch.Tensor       # views of w_qkv_c (wq, wk_c, wv_c) and of w_qkv (wk, wv)
    wk: torch.Tensor       # dense K projection (the baseline)
    wv: torch.Tensor
    wk_c: torch.Tensor     # merged: emits per-head K coefficients
    wv_c: torch.Tensor
    wo: torch.Tensor
    ln2: torch.Tensor
    w_gu: torch.Tensor     # (2 * ffn, hidden): gate and up rows interleaved (2j gate, 2j+1 up)
    w_gate: torch.Tensor   # views of w_gu
    w_up: torch.Tensor
    w_down: torch.Tensor
    k_basis: torch.Tensor  # (G, R, Dh) rank-major
    v_basis: torch.Tensor
    cutoff: CutoffHead = field(repr=False)
    q_norm: torch.Tensor | None = None  # (Dh,) weights of the head norms, where the shape has them
    k_norm: torch.Tensor | None = None


def _orthogonal(n: int, count: int, gen: torch.Generator, device) -> torch.Tensor:
    a = torch.randn(count, n, n, generator=gen, device=device, dtype=torch.float32)
    q, r = torch.linalg.qr(a)
    return q * torch.sign(torch.diagonal(r, dim1=-2, dim2=-1)).unsqueeze(-2)


def ramp_for_retention(D: int, retention: float) -> float:
    """Slope beta of the cutoff bias beta * j / D for which flip(cumsum(softmax)) >= 0.1 keeps
    ``retention * D`` dims when the input term is small: the mass below index D * (1 - r) is
    0.1, i.e. (e^{beta (1-r)} - 1) / (e^{beta} - 1) = 0.1, solved by bisection."""
    lo, hi = 1e-3, 60.0
    target_m = 1.0 - retention
    for _ in range(100):
        mid = 0.5 * (lo + hi)
        frac = math.expm1(mid * target_m) / math.expm1(mid)
        if frac > 0.1:
            lo = mid
        else:
            hi = mid
    return 0.5 * (lo + hi)


class RandomLlama:
    def __init__(self, shape: LlamaShape = LlamaShape(), *, device="cuda", dtype=torch.bfloat16,
                 seed: int = 0, retention: float = 0.47, std: float = 0.02):
        self.shape = shape
        self.dtype = dtype
        self.device = torch.device(device)
        g = torch.Generator(device=self.device)
        g.manual_seed(seed)
        s = shape
        H, Dh, G = s.hidden, s.head_dim, s.kv_heads

        def rnd(*dims):
            return (torch.randn(*dims, generator=g, device=self.device, dtype=torch.float32)
                    * std).to(dtype)

        self.embed = rnd(s.vocab, H)
        self.norm = torch.ones(H, device=self.device, dtype=dtype)
        self.lm_head = rnd(s.vocab, H)
        beta = ramp_for_retention(Dh, retention)
        ramp = (beta * torch.arange(Dh, device=self.device, dtype=torch.float32) / Dh).to(dtype)
        self.layers = []
        for _ in range(s.layers):
            wk, wv = rnd(G * Dh, H), rnd(G * Dh, H)
            Uk = _orthogonal(Dh, G, g, self.device)  # (G, d, r): K_g = U_g c_g
            Uv = _orthogonal(Dh, G, g, self.device)
            # coefficients c_g = U_g^T k_g: the projection merged with the basis transpose (the
            # reference's one-time merge, k_proj <- k_down @ k_proj, per KV group)
            wk_c = merge_projection(wk.float().view(G, Dh, H), Uk.transpose(1, 2))[0]
            wv_c = merge_projection(wv.float().view(G, Dh, H), Uv.transpose(1, 2))[0]
            wk_c, wv_c = wk_c.reshape(G * Dh, H), wv_c.reshape(G * Dh, H)
            cut = [rnd(G, Dh, Dh) for _ in range(2)]
            bias = [ramp.expand(G, Dh).contiguous() for _ in range(2)]
            w_gu = rnd(2 * s.ffn, H)
            wq = rnd(H, H)
            w_qkv_c = torch.cat([wq, wk_c.to(dtype), wv_c.to(dtype)])
            w_qkv = torch.cat([wq, wk, wv])
            GD = G * Dh
            self.layers.append(LayerWeights(
                ln1=torch.ones(H, device=self.device, dtype=dtype), w_qkv_c=w_qkv_c, w_qkv=w_qkv,
                wq=w_qkv_c[:H], wk=w_qkv[H:H + GD], wv=w_qkv[H + GD:],
                wk_c=w_qkv_c[H:H + GD], wv_c=w_qkv_c[H + GD:], wo=rnd(H, H),
                ln2=torch.ones(H, device=self.device, dtype=dtype),
                w_gu=w_gu, w_gate=w_gu[0::2], w_up=w_gu[1::2], w_down=rnd(H, s.ffn),
                k_basis=Uk.transpose(1, 2).contiguous().to(dtype),
                v_basis=Uv.transpose(1, 2).contiguous().to(dtype),
                cutoff=CutoffHead(cut[0], bias[0], cut[1], bias[1], groups=G)))
        if s.qk_norm:  # (drawn last: the other weights are those of the shape without norms)
            for lw in self.layers:
                lw.q_norm, lw.k_norm = 1 + rnd(Dh), 1 + rnd(Dh)


class Sampler:
    """Draws tokens from logits: a generator's replacement for its argmax. The settings are those of
    ``sample_tokens`` and, before them, the penalties of ``adjust_logits_`` over a request's tokens:
    numbers or a tensor with an entry per row (of a batch, or of the requests that are generated for).
    ``bias`` maps tokens to what is added to their logits, for all rows. The uniform numbers come from a generator of
    its own, so a seed gives the same draws for the same logits."""

    _NEUTRAL = dict(repetition=1.0, frequency=0.0, presence=0.0)

    def __init__(self, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, repetition=1.0,
                 frequency=0.0, presence=0.0, bias: dict[int, float] | None = None, seed: int = 0,
                 device="cuda"):
        self.settings = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        # (here, where a tensor may be read back: the operator, which does not, divides by its entries)
        rep = torch.as_tensor(repetition, dtype=torch.float32)
        if not bool(((rep > 0.0) & (rep < float("inf"))).all()):
            raise ValueError("repetition must be positive and finite")
        given = dict(repetition=repetition, frequency=frequency, presence=presence)
        self.penalties = {name: v for name, v in given.items()
                          if torch.is_tensor(v) or v != self._NEUTRAL[name]}
        self._bias = None
        if bias:
            self._bias = (torch.tensor([list(bias)], dtype=torch.int32, device=device),
                          torch.tensor([list(bias.values())], dtype=torch.float32, device=device))
        self._gen = torch.Generator(device=device)
        self._gen.manual_seed(seed)

    def __call__(self, logits: torch.Tensor, *, requests: Sequence[int] | None = None,
                 u: torch.Tensor | None = None, tokens: torch.Tensor | None = None, prompt_lens=None,
                 lens=None, allowed: torch.Tensor | None = None) -> torch.Tensor:
        """``logits`` (..., V) -> tokens (...). ``requests``: the request of each row, whose entries the
        settings' tensors are taken from (else row i has entry i); ``u``: the rows' uniform numbers (else
        the generator's next ones). Penalties need the rows' ``tokens``, with ``prompt_lens`` and
        ``lens``, and ``allowed`` is their mask, as ``adjust_logits_`` takes them (here on a copy of the
        logits). Of a row without a token to take (all NaN or -infinity) token 0, as the tokens are
        looked up next: ``sample_tokens`` tells them by -1."""
        rows = logits.reshape(-1, logits.shape[-1])
        settings = self.settings | self.penalties
        if requests is not None:
            settings = self._of(requests, rows)
        if u is None:
            u = self.uniform(rows.shape[0], logits.device)
        penalties = {name: settings.pop(name) for name in self.penalties}
        if penalties:
            if tokens is None:
                raise ValueError("a sampler with penalties needs the rows' tokens")
            penalties |= dict(tokens=tokens, prompt_lens=prompt_lens, lens=lens)
        if self._bias is not None:
            n = rows.shape[0]
            penalties |= dict(bias_ids=self._bias[0].expand(n, -1), bias=self._bias[1].expand(n, -1))
        if allowed is not None:
            penalties["allowed"] = allowed
        if penalties:
            rows = adjust_logits_(rows.clone(memory_format=torch.contiguous_format), **penalties)
        return sample_tokens(rows, u, **settings).clamp_(min=0).view(logits.shape[:-1])

    def uniform(self, n: int, device) -> torch.Tensor:
        """The generator's next ``n`` numbers."""
        return torch.rand(n, generator=self._gen, device=device)

    def check(self, requests: int) -> None:
        """Raises where a setting's tensor has not an entry for each of so many requests."""
        for name, v in (self.settings | self.penalties).items():
            if torch.is_tensor(v) and v.shape != (requests,):
                raise ValueError(f"{name} must be a number or have an entry for each of the {requests} "
                                 "requests")

    def _of(self, requests: Sequence[int], rows: torch.Tensor) -> dict:
        if len(requests) != rows.shape[0]:
            raise ValueError(f"{len(requests)} requests for {rows.shape[0]} rows of logits")
        at = None
        settings = self.settings | self.penalties
        for name, v in settings.items():
            if not torch.is_tensor(v):
                continue
            if v.dim() != 1 or not all(0 <= r < v.shape[0] for r in requests):
                raise ValueError(f"{name} has no entry for one of the requests {list(requests)}")
            if list(requests) != list(range(v.shape[0])):
                at = _index(requests, v.device) if at is None else at
                settings[name] = v.index_select(0, at)
        return settings



def _index(numbers: Sequence[int], device) -> torch.Tensor:
    """Host numbers as an index on the device (a copy that the host does not wait for)."""
    t = torch.tensor(numbers, dtype=torch.long)
    if torch.device(device).type == "cuda":
        t = t.pin_memory()
    return t.to(device, non_blocking=True)


def _rope_q(q: torch.Tensor, pos0: int, theta: float) -> torch.Tensor:
    """q (B, S, Hq, Dh) -> rotated (B, Hq, S, Dh) contiguous."""
    qh = q.transpose(1, 2).contiguous()
    return rope_dense_(qh, theta=theta, pos0=pos0)


class _Generator:
    takes_qk_norm = False

    def __init__(self, model: RandomLlama):
        if model.shape.qk_norm and not self.takes_qk_norm:
            raise ValueError(f"{type(self).__name__} has no query and key norms")
        self.m = model
        self.s = model.shape

    def _split(self, y: torch.Tensor):
        """The q, K and V column ranges of a fused projection output (views)."""
        H, GD = self.s.hidden, self.s.kv_heads * self.s.head_dim
        return y[..., :H], y[..., H:H + GD], y[..., H + GD:]

    def logits(self, x: torch.Tensor) -> torch.Tensor:
        return rmsnorm_linear(x, None, self.m.norm, self.s.eps, self.m.lm_head)[0]

    def _run(self, x: torch.Tensor, attn, qkv: str) -> torch.Tensor:
        """The decoder layers over the residual stream ``x`` (B, S, hidden); returns the final
        residual stream. ``attn(i, lw, y)`` takes layer i's q/k/v projection output ``y``
        (weight ``getattr(lw, qkv)``) and returns its attention output (B, S, hidden) before the
        output projection. Each residual add and the norm after it are fused into the
        projection that consumes them (decode), or one kernel before it (prefill)."""
        eps = self.s.eps
        delta = None
        for i, lw in enumerate(self.m.layers):
            y, x = rmsnorm_linear(x, delta, lw.ln1, eps, getattr(lw, qkv))
            h, x = rmsnorm_glu(x, linear(attn(i, lw, y), lw.wo), lw.ln2, eps, lw.w_gu)
            delta = linear(h, lw.w_down)
        return x + delta

    def generate(self, prompt: torch.Tensor, new_tokens: int,
                 sampler: Sampler | None = None) -> dict:
        """Greedy decode (or tokens drawn by ``sampler``); returns tokens, timings and cache
        bytes."""
        pick = sampler if sampler is not None else lambda logits: logits.argmax(-1)
        if isinstance(sampler, Sampler) and sampler.penalties:
            pick = self._with_history(sampler, prompt, new_tokens)
        torch.cuda.synchronize(self.m.device)
        t0 = time.perf_counter()
        x = self.prefill(prompt)
        tok = pick(self.logits(x[:, -1:]))  # (B, 1)
        out = [tok]
        torch.cuda.synchronize(self.m.device)
        t1 = time.perf_counter()
        pos = prompt.shape[1]
        for _ in range(new_tokens - 1):
            x = self.decode(tok, pos)
            tok = pick(self.logits(x))
            out.append(tok)
            pos += 1
        torch.cuda.synchronize(self.m.device)
        t2 = time.perf_counter()
        B = prompt.shape[0]
        return {
            "tokens": torch.cat(out, dim=1),
            "prefill_s": t1 - t0,
            "decode_s": t2 - t1,
            "tokens_per_s": B * new_tokens / (t2 - t0),
            "decode_tokens_per_s": B * (new_tokens - 1) / max(t2 - t1, 1e-9),
            "kv_bytes": self.kv_bytes(),
        }


    def _with_history(self, sampler: Sampler, prompt: torch.Tensor, new_tokens: int):
        """Logits (B, 1, V) -> tokens (B, 1), with the prompts' and the generated tokens' penalties."""
        B, S = prompt.shape
        history = torch.zeros(B, S + new_tokens, dtype=torch.long, device=prompt.device)
        history[:, :S] = prompt
        n = S

        def pick(logits):
            nonlocal n
            tok = sampler(logits, tokens=history, prompt_lens=S, lens=n)
            history[:, n:n + 1] = tok
            n += 1
            return tok

        return pick


class CompressedLlama(_Generator):
    """The model over DynaKV's packed cache (per-head layout, rows b*G + g)."""

    def __init__(self, model: RandomLlama, policy: KernelPolicy | None = None,
                 one_call_layers: bool = True):
        super().__init__(model)
        self.policy = policy or KernelPolicy()
        self.cache = CustomDynamicCache()
        self.one_call_layers = one_call_layers
        self.plans: dict = {}

    def _qkv(self, lw, h):
        """``h``: the layer's fused q/k/v projection output (B, S, H + 2 G Dh)."""
        B, S, _ = h.shape
        s = self.s
        q, kc, vc = self._split(h)
        q = q.reshape(B, S, s.heads, s.head_dim)
        kc, vc = kc.contiguous(), vc.contiguous()  # (B, S, G*Dh) coefficients
        k_out, v_out, len_k, len_v, _, _ = lw.cutoff.kv_process_fused(kc, vc)
        G, Dh = s.kv_heads, s.head_dim
        if B == 1:
            # rows b*G + g are strided views (row stride Dh, token stride G*Dh): the appends and
            # the prefill products take the strides, so no transposed copy is made
            rows_k = k_out.view(S, G, Dh).transpose(0, 1)
            rows_v = v_out.view(S, G, Dh).transpose(0, 1)
            lk = len_k.view(S, G).transpose(0, 1)
            lv = len_v.view(S, G).transpose(0, 1)
            return q, rows_k, lk, rows_v, lv
        rows_k = k_out.view(B, S, G, Dh).transpose(1, 2).reshape(B * G, S, Dh)
        rows_v = v_out.view(B, S, G, Dh).transpose(1, 2).reshape(B * G, S, Dh)
        lk = len_k.view(B, S, G).transpose(1, 2).reshape(B * G, S).contiguous()
        lv = len_v.view(B, S, G).transpose(1, 2).reshape(B * G, S).contiguous()
        return q, rows_k, lk, rows_v, lv

    def prefill(self, prompt: torch.Tensor) -> torch.Tensor:
        s = self.s
        self.cache.reset()
        self.plans = {}
        x = F.embedding(prompt, self.m.embed)
        B, S = prompt.shape

        pending = []

        def attn(i, lw, y):
            q, rk, lk, rv, lv = self._qkv(lw, y)
            pending.append((i, rk, lk, rv, lv))
            qh = _rope_q(q, 0, s.theta)
            # the masked coefficients are what the packed cache returns once appended
            a = coef_prefill_attention(qh, rk, rv, lw.k_basis, lw.v_basis, theta=s.theta)
            return a.transpose(1, 2).reshape(B, S, s.hidden)

        x = self._run(x, attn, "w_qkv_c")
        # every layer's appends after the forward pass: one host synchronisation in all
        self.cache.update_sp_prefill_many(pending, s.head_dim)
        return x

    def decode(self, tok: torch.Tensor, pos: int) -> torch.Tensor:
        s = self.s
        x = F.embedding(tok, self.m.embed)  # (B, 1, H)
        B = tok.shape[0]

        def attn(i, lw, y):
            plan = self.plans.get(i)
            if plan is not None and plan.can_step():
                # one call: cutoff head, K+V append, q RoPE, routed attention
                # one projection; q and the coefficients are views into its output
                q, kc, vc = self._split(y.view(B, -1))
                a = plan.step(q.view(B, s.heads, s.head_dim), kc, vc, pos)
            else:
                q, rk, lk, rv, lv = self._qkv(lw, y)
                fk, fv, tk, tv, ok, ov = self.cache.update_sp(rk, lk, rv, lv, s.head_dim, i,
                                                              s.head_dim)
                L = self.cache.get_seq_length_sp(i)
                qh = _rope_q(q, pos, s.theta)[:, :, 0]  # (B, Hq, Dh)
                a = grouped_decode_attention(qh, fk, fv, tk, ok, tv, ov, lw.k_basis, lw.v_basis,
                                             theta=s.theta, route=self.policy.select(L))
                if self.one_call_layers:
                    self.plans[i] = DecodeLayerPlan(self.cache, i, lw.cutoff, lw.k_basis,
                                                    lw.v_basis, batch=B, heads=s.heads,
                                                    theta=s.theta, policy=self.policy)
            return a.reshape(B, 1, s.hidden)

        return self._run(x, attn, "w_qkv_c")

    def kv_bytes(self) -> int:
        """Stored bytes of the packed caches: the used part of each row plus 8 bytes of
        lengths/offsets per token and row."""
        tot = 0
        for slots in (self.cache.key_cache_sp, self.cache.value_cache_sp):
            for c in slots:
                if c is None:
                    continue
                flat, lens, offs, ptr, seq = c[0], c[1], c[2], c[3], c[4]
                tot += int(ptr.sum()) * flat.element_size() + 8 * lens.shape[0] * seq
        return tot


# torch's fused attention kernels only: an input they do not take raises instead of running the
# composite (math) path
_FAST_SDPA = [SDPBackend.FLASH_ATTENTION, SDPBackend.EFFICIENT_ATTENTION]


class DenseLlama(_Generator):
    """The same weights with an uncompressed cache, the reference's baseline (the original model
    with transformers' KV cache, ``scripts/benchmark_throughput.py:17-77``): every token's
    rotated key and its value kept in full (head dim 128 per KV head). A decode step writes the
    new token's rotated key and value and rotates q in one launch (``dkv_dense_append``), then
    runs dense GQA decode attention (``dkv_decode_dense``: no reconstruction, no RoPE in the
    attention, fp32 scores). Prefill attention is torch's fused attention on the rotated keys."""

    def __init__(self, model: RandomLlama, max_len: int = 4096, attention: str = "kernel"):
        """``attention``: "kernel" (``dkv_decode_dense``) or "sdpa" (torch's
        ``scaled_dot_product_attention`` over the cached keys and values, the attention path the
        reference's uncompressed transformers model takes)."""
        super().__init__(model)
        if attention not in ("kernel", "sdpa"):
            raise ValueError("attention must be 'kernel' or 'sdpa'")
        self.max_len = max_len
        self.attention = attention
        self.k = self.v = None
        self.len = 0

    def _kv(self, lw, y, pos0):
        """``y``: the layer's fused q/k/v projection output (B, S, H + 2 G Dh). Returns the
        rotated q (B, Hq, S, Dh) and K (before RoPE) / V as (B, G, S, Dh)."""
        B, S, _ = y.shape
        s = self.s
        q, k, v = self._split(y)
        q = q.reshape(B, S, s.heads, s.head_dim)
        k = k.reshape(B, S, s.kv_heads, s.head_dim).transpose(1, 2)
        v = v.reshape(B, S, s.kv_heads, s.head_dim).transpose(1, 2)
        return _rope_q(q, pos0, s.theta), k, v

    def prefill(self, prompt: torch.Tensor) -> torch.Tensor:
        s = self.s
        B, S = prompt.shape
        dev, dt = self.m.device, self.m.dtype
        G, Dh = s.kv_heads, s.head_dim
        rows = B * G
        # per layer: K and V rows (b*G + g) of max_len tokens x Dh, tokens back to back, and the
        # shared tables of the packed view (128 dims per token, token t at offset 128 t)
        self.k = [torch.empty((rows, self.max_len * Dh), device=dev, dtype=dt)
                  for _ in range(s.layers)]
        self.v = [torch.empty((rows, self.max_len * Dh), device=dev, dtype=dt)
                  for _ in range(s.layers)]
        hpg = s.heads // s.kv_heads
        x = F.embedding(prompt, self.m.embed)

        def attn(i, lw, y):
            qh, k, v = self._kv(lw, y, 0)
            kr = rope_dense_(k.contiguous(), theta=s.theta, pos0=0)
            self.k[i][:, :S * Dh] = kr.reshape(rows, S * Dh)
            self.v[i][:, :S * Dh] = v.reshape(rows, S * Dh)
            with sdpa_kernel(_FAST_SDPA):
                a = F.scaled_dot_product_attention(qh, kr.repeat_interleave(hpg, dim=1),
                                                   v.repeat_interleave(hpg, dim=1),
                                                   is_causal=True)
            return a.transpose(1, 2).reshape(B, S, s.hidden)

        x = self._run(x, attn, "w_qkv")
        self.len = S
        return x

    def decode(self, tok: torch.Tensor, pos: int) -> torch.Tensor:
        """One token: the rotated K and V written at position len (q rotated at ``pos`` in the
        same launch), then dense decode attention over len + 1 tokens."""
        s = self.s
        x = F.embedding(tok, self.m.embed)
        B = tok.shape[0]
        L = self.len
        Dh = s.head_dim

        def attn(i, lw, y):
            y2 = y[:, 0, :]
            dense_append_(y2, self.k[i], self.v[i], q_pos=pos, k_pos=L, heads=s.heads,
                          kv_heads=s.kv_heads, theta=s.theta)
            qh = y2[:, :s.heads * Dh].view(B, s.heads, Dh)
            if self.attention == "sdpa":
                G, hpg = s.kv_heads, s.heads // s.kv_heads
                kk = self.k[i][:, :(L + 1) * Dh].view(B, G, L + 1, Dh)
                vv = self.v[i][:, :(L + 1) * Dh].view(B, G, L + 1, Dh)
                with sdpa_kernel(_FAST_SDPA):
                    a = F.scaled_dot_product_attention(
                        qh.unsqueeze(2), kk.repeat_interleave(hpg, dim=1),
                        vv.repeat_interleave(hpg, dim=1))
                return a.reshape(B, 1, s.hidden)
            a = dense_decode_attention(qh, self.k[i], self.v[i], L + 1)
            return a.reshape(B, 1, s.hidden)

        x = self._run(x, attn, "w_qkv")
        self.len = L + 1
        return x

    def kv_bytes(self) -> int:
        """Stored K and V payload: every token of every (batch, KV head) row at 128 dims."""
        s = self.s
        rows = self.k[0].shape[0] if self.k else 0
        return 2 * s.layers * rows * self.len * s.head_dim * self.m.embed.element_size()


class PagedLlama(_Generator):
    """The same weights over a paged uncompressed cache: requests of different lengths, whose
    prompts go through in chunks beside the other requests' single tokens.

    ``pages`` pages of ``page_size`` tokens per layer are shared by all requests, in the model's type
    or of 8 bits (``cache_dtype=torch.float8_e4m3fn``: half the bytes). ``add`` starts a
    request, ``step`` feeds tokens to some of them and returns the logits after each one's last
    token, ``end`` gives a request's pages back; ``generate`` is the loop over them."""

    takes_qk_norm = True

    def __init__(self, model: RandomLlama, pages: int, page_size: int = 64,
                 cache_dtype: torch.dtype | None = None):
        super().__init__(model)
        s = self.s
        self.cache = PagedKVCache(s.layers, pages, s.kv_heads, page_size=page_size,
                                  dtype=model.dtype if cache_dtype is None else cache_dtype,
                                  device=model.device)

    def add(self) -> int:
        return self.cache.add()

    def end(self, request: int) -> None:
        self.cache.free(request)

    def step(self, feed: list[tuple[int, torch.Tensor]]) -> torch.Tensor:
        """Feed each (request, (n,) tokens), n >= 1; returns (requests, vocab) logits. A step that raises
        leaves the requests as long as they were."""
        if not feed or any(t.dim() != 1 or t.shape[0] < 1 for _, t in feed):
            raise ValueError("a step feeds at least one token to each of its requests")
        before = [(r, self.cache.length(r)) for r, _ in feed]
        batch = self.cache.batch((r, t.shape[0]) for r, t in feed)
        try:
            return self._step(feed, batch)
        except BaseException:
            for r, n in before:
                self.cache.truncate(r, n)
            raise

    def _step(self, feed: list[tuple[int, torch.Tensor]], batch: PagedBatch) -> torch.Tensor:
        s = self.s
        x = F.embedding(torch.cat([t for _, t in feed]), self.m.embed).unsqueeze(0)

        def attn(i, lw, y):
            c = self.cache
            scales = dict(k_scale=c.k_scale[i], v_scale=c.v_scale[i])
            q = paged_append(y[0], c.k[i], c.v[i], batch, heads=s.heads, theta=s.theta,
                             q_norm=lw.q_norm, k_norm=lw.k_norm, eps=s.eps, **scales)
            a = paged_attention(q, c.k[i], c.v[i], batch, **scales)
            return a.view(1, -1, s.hidden)

        x = self._run(x, attn, "w_qkv")[0]
        return self.logits(x[batch.q_start[1:].long() - 1])

    def generate(self, prompts: list[torch.Tensor], new_tokens: int,
                 sampler: Sampler | None = None, chunk: int = 512) -> dict:
        """``new_tokens`` tokens for each of the (n,) prompts (n >= 1), greedily or drawn by
        ``sampler``; a step takes at most ``chunk`` tokens of prompts, in the prompts' order, beside
        a token of each request that is generating. Settings of the sampler with an entry per request
        are the prompts' in their order, and a request's i-th token is drawn by a uniform number of its
        own, whichever requests share its step. Returns the tokens (prompts, new_tokens), the wall time
        and the most pages held."""
        if chunk < 1 or new_tokens < 1 or not prompts:
            raise ValueError("need prompts, a positive chunk and a positive number of tokens")
        if any(p.dim() != 1 or p.shape[0] < 1 for p in prompts):
            raise ValueError("prompts are (n,) tokens, n >= 1")
        pick = self._pick(sampler, prompts, new_tokens)
        torch.cuda.synchronize(self.m.device)
        t0 = time.perf_counter()
        ids: list = [self.add() for _ in prompts]  # None once ended
        fed = [0] * len(prompts)                   # prompt tokens gone through
        out: list[list[torch.Tensor]] = [[] for _ in prompts]
        held = 0
        try:
            while any(len(o) < new_tokens for o in out):
                room, feed, who = chunk, [], []
                for j, p in enumerate(prompts):
                    n = min(room, p.shape[0] - fed[j])
                    if n > 0:
                        feed.append((ids[j], p[fed[j]:fed[j] + n]))
                        room -= n
                        fed[j] += n
                    elif fed[j] == p.shape[0] and len(out[j]) < new_tokens:
                        feed.append((ids[j], out[j][-1]))
                    else:
                        continue
                    who.append(j)
                logits = self.step(feed)
                held = max(held, self.cache.pages - self.cache.free_pages)
                done = [i for i, j in enumerate(who) if fed[j] == prompts[j].shape[0]]
                if not done:  # no request's whole prompt has gone through
                    continue
                if len(done) < len(who):
                    logits = logits.index_select(0, _index(done, logits.device))
                tok = pick(logits, [(who[i], len(out[who[i]])) for i in done])
                for i, j in enumerate(who[i] for i in done):
                    out[j].append(tok[i:i + 1])
                    if len(out[j]) == new_tokens:
                        self.end(ids[j])
                        ids[j] = None
        finally:
            for r in ids:
                if r is not None:
                    self.end(r)
        torch.cuda.synchronize(self.m.device)
        t = time.perf_counter() - t0
        return {"tokens": torch.stack([torch.cat(o) for o in out]), "seconds": t,
                "tokens_per_s": len(prompts) * new_tokens / t, "pages": held}

    def _pick(self, sampler: Sampler | None, prompts: list[torch.Tensor], new_tokens: int):
        """(logits, (request, index of its token) of each row) -> tokens."""
        requests = len(prompts)
        if sampler is None:
            return lambda logits, at: logits.argmax(-1)
        if not isinstance(sampler, Sampler):  # any function of logits
            return lambda logits, at: sampler(logits)
        sampler.check(requests)
        # row i: the numbers of the requests' i-th tokens, drawn when the first of them is
        u = torch.empty(new_tokens, requests, dtype=torch.float32, device=self.m.device)
        drawn = 0
        history = None  # the requests' tokens, where there are penalties for them
        if sampler.penalties:
            sizes = [p.shape[0] for p in prompts]
            history = torch.zeros(requests, max(sizes) + new_tokens, dtype=torch.long,
                                  device=self.m.device)
            for j, p in enumerate(prompts):
                history[j, :sizes[j]] = p

        def pick(logits, at):
            nonlocal drawn
            while drawn <= max(i for _, i in at):
                u[drawn] = sampler.uniform(requests, u.device)
                drawn += 1
            mine = u.view(-1).index_select(0, _index([i * requests + j for j, i in at], u.device))
            who = [j for j, _ in at]
            if history is None:
                return sampler(logits, requests=who, u=mine)
            rows = _index(who + [sizes[j] for j in who] + [sizes[j] + i for j, i in at], u.device)
            rows, first, ends = rows.view(3, -1)
            tok = sampler(logits, requests=who, u=mine, tokens=history.index_select(0, rows),
                          prompt_lens=first.int(), lens=ends.int())
            history[rows, ends] = tok
            return tok

        return pick

    def kv_bytes(self) -> int:
        """Bytes of the pages that requests hold (and of their scales), over all layers."""
        k, scale = self.cache.k[0], self.cache.k_scale[0]
        held = self.cache.pages - self.cache.free_pages
        page = k[0].numel() * k.element_size() + (0 if scale is None else scale[0].numel())
        return 2 * len(self.cache.k) * held * page
