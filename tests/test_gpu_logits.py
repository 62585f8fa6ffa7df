"""``adjust_logits_`` on the GPU against the formula in float64, and its refusals on the CPU.

Tolerance: half a step of the type for the last rounding, and before it fp32 work, half a step (2^-24
relative) of each operand's size per operation: a product or quotient, one product, two differences, a
sum of m biases (m - 1 additions, each of at most the sum of their sizes) and an addition."""
import math

import pytest
import torch

from dynakv_amd import _lib
from dynakv_amd.kernels.sampling import adjust_logits_, sample_tokens

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def reference(x, *, tokens=None, prompt_lens=None, lens=None, repetition=1.0, frequency=0.0,
              presence=0.0, bias_ids=None, bias=None, allowed=None):
    """(result, size of what the fp32 roundings act on, touched), float64 on the CPU."""
    rows, V = x.shape
    dtype = x.dtype
    y = x.double().cpu()
    size, touched = torch.zeros_like(y), torch.zeros_like(y, dtype=torch.bool)
    at = lambda v, b: float(v[b]) if torch.is_tensor(v) else float(v)  # noqa: E731
    for b in range(rows):
        if tokens is not None:
            N = tokens.shape[1]
            n = min(max(int(at(N if lens is None else lens, b)), 0), N)
            first = max(int(at(0 if prompt_lens is None else prompt_lens, b)), 0)
            t = tokens[b, :n].cpu().long()
            inside = (t >= 0) & (t < V)
            seen = torch.unique(t[inside])
            count = torch.bincount(t[first:][inside[first:]], minlength=V).double()
            r, f, p = (at(v, b) for v in (repetition, frequency, presence))
            y[b, seen] = torch.where(y[b, seen] > 0, y[b, seen] / r, y[b, seen] * r)
            size[b, seen] += 2 * y[b, seen].abs()
            y[b] -= torch.where(count > 0, f * count + p, 0.0)
            size[b] += 4 * (f * count).abs() + 2 * abs(p) * (count > 0)
            touched[b, seen] = True
        if bias is not None:
            for i, v in zip(bias_ids[b].tolist(), bias[b].tolist()):
                if 0 <= i < V:
                    y[b, i] += v
                    m = int((bias_ids[b] == i).sum())
                    size[b, i] += (m + 1) * abs(v)
                    touched[b, i] = True
        if allowed is not None:
            w = allowed[b].cpu().long()
            bits = torch.stack([(w >> k) & 1 for k in range(32)], 1).reshape(-1)[:V]
            y[b, bits == 0] = -math.inf
            touched[b, bits == 0] = True
    size += y.abs().nan_to_num(posinf=0.0) * touched
    return y, torch.finfo(dtype).eps / 2 * y.abs().nan_to_num(posinf=0.0) + 2.0**-23 * size, touched


def check(x, **kw):
    x0 = x.clone()
    want, tol, touched = reference(x0, **kw)
    if x.dtype == FP:  # numbers below 2^-14 are 2^-24 apart
        tol = tol + 2.0**-25
    got = adjust_logits_(x, **kw)
    assert got is x
    got = got.double().cpu()
    big = torch.finfo(x.dtype).max
    want = torch.where(want.abs() > big, want.sign() * math.inf, want)
    exact = (got == want) | (got.isnan() & want.isnan())
    good = bool((exact | ((got - want).abs() <= tol)).all())
    assert good
    kept = bool((exact | touched).all())
    assert kept
    return got


def _rows(dev, rows, V, dtype, seed=0, n=0, ids=torch.int64, biases=0, mask=False, settings=True):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, V, generator=g) * 3).to(dtype).to(dev)
    kw = {}
    if n:
        t = (torch.rand(rows, n, generator=g) ** 3 * V).long().clamp(max=V - 1)
        t[torch.rand(rows, n, generator=g) < 0.05] = -1
        t[torch.rand(rows, n, generator=g) < 0.05] = V
        if ids == torch.int64:
            t[torch.rand(rows, n, generator=g) < 0.05] = 2**40 + 1
        kw["tokens"] = t.to(ids).to(dev)
        if settings:
            r = lambda lo, hi: (lo + (hi - lo) * torch.rand(rows, generator=g)).to(dev)  # noqa: E731
            kw["lens"] = torch.randint(-1, n + 3, (rows,), generator=g, dtype=torch.int32).to(dev)
            kw["prompt_lens"] = torch.randint(-1, n + 3, (rows,), generator=g,
                                              dtype=torch.int32).to(dev)
            kw |= dict(repetition=r(0.8, 1.5), frequency=r(-0.2, 0.7), presence=r(-0.2, 0.7))
        else:
            kw |= dict(repetition=1.25, frequency=0.5, presence=0.25, prompt_lens=n // 2)
    if biases:
        i = torch.randint(0, V, (rows, biases), generator=g, dtype=torch.int32)
        i[:, ::5] = i[:, :1]  # one token many times
        i[torch.rand(rows, biases, generator=g) < 0.1] = -1
        i[torch.rand(rows, biases, generator=g) < 0.1] = V
        kw["bias_ids"], kw["bias"] = i.to(dev), (torch.randn(rows, biases, generator=g) * 4).to(dev)
    if mask:
        words = -(-V // 32)
        kw["allowed"] = torch.randint(-2**31, 2**31, (rows, words), generator=g,
                                      dtype=torch.int64).to(torch.int32).to(dev)
        kw["allowed"][0] = -1
        kw["allowed"][-1] = 0
    return x, kw


CASES = {
    # name: rows, V, dtype, history, ids, biases, mask, settings per row
    "one_token_vocab": (2, 1, F32, 3, torch.int64, 2, True, True),
    "all_small": (3, 77, BF, 20, torch.int64, 6, True, True),
    "all_numbers": (3, 1000, FP, 20, torch.int32, 6, True, False),
    "one_row": (1, 32000, BF, 1000, torch.int64, 8, False, True),
    "penalties": (9, 5000, BF, 700, torch.int32, 0, False, True),
    "penalties_fp16": (4, 4097, FP, 2000, torch.int64, 0, False, False),
    "biases": (5, 2049, F32, 0, None, 40, False, False),
    "many_biases": (2, 700, BF, 0, None, 1500, False, False),
    "mask": (4, 50257, F32, 0, None, 0, True, False),
    "mask_bf16": (7, 2111, BF, 0, None, 0, True, False),
    "grammar": (37, 5025, F32, 300, torch.int32, 20, True, True),
    "spans_of_4096": (70, 40000, BF, 50, torch.int64, 0, False, True),
    "spans_of_16384": (260, 40007, FP, 100, torch.int64, 0, True, True),
    "spans_with_biases": (260, 20011, BF, 60, torch.int32, 3, False, True),
    "long_history": (2, 3000, F32, 30000, torch.int64, 0, False, True),
    # histories that are counted by vocabulary, in spans of 2048, 8192 and 16384 tokens
    "long_all": (3, 4100, FP, 7000, torch.int32, 9, True, True),
    "long_spans_of_8192": (80, 40007, BF, 6200, torch.int32, 5, True, True),
    "long_spans_of_16384": (260, 40007, BF, 6200, torch.int64, 0, False, True),
    "largest_table": (2, 50000, BF, 6144, torch.int64, 0, True, True),
    "largest_table_with_biases": (2, 50000, F32, 3000, torch.int64, 72, False, True),
    "every_token_once": (2, 6144, F32, 6144, torch.int64, 0, False, False),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(CASES))
def test_against_the_formula(dev, name):
    rows, V, dtype, n, ids, biases, mask, settings = CASES[name]
    print(f"[gpu] adjust {name}", flush=True)
    x, kw = _rows(dev, rows, V, dtype, seed=len(name), n=n, ids=ids, biases=biases, mask=mask,
                  settings=settings)
    if name == "every_token_once":
        kw["tokens"] = torch.stack([torch.randperm(V, device=dev) for _ in range(rows)])
    check(x, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FP, F32])
def test_logits_that_are_not_finite(dev, dtype):
    """Infinities stay what they are, NaN stays NaN, the mask clears both."""
    print("[gpu] adjust not finite", flush=True)
    x, kw = _rows(dev, 2, 200, dtype, n=40, biases=5, mask=True, seed=3)
    kw["tokens"][:, :3] = torch.tensor([3, 4, 5], device=dev)
    kw["lens"] = kw["prompt_lens"] = None
    kw["bias_ids"][:, 0] = 4
    x[:, 3], x[:, 4], x[:, 5], x[:, 6] = math.inf, -math.inf, math.nan, math.nan
    got = check(x, **kw)
    assert bool((got[1] == -math.inf).all()) and got[0, 3] == math.inf
    assert got[0, 4] == -math.inf and bool(got[0, 5:7].isnan().all())


@pytest.mark.gpu
def test_strides_and_neighbours(dev):
    """Rows inside a larger tensor at odd addresses; what lies around them stays; rows of the other
    inputs apart, or one row expanded to all."""
    print("[gpu] adjust strides", flush=True)
    for dtype in (BF, F32):
        whole = torch.full((6, 3011), 9.0, dtype=dtype, device=dev)
        x, kw = _rows(dev, 6, 2999, dtype, n=50, biases=7, mask=True, seed=8)
        whole[:, 5:3004] = x
        for name in ("tokens", "bias_ids", "bias", "allowed"):
            t = kw[name]
            wide = torch.zeros(t.shape[0], t.shape[1] + 3, dtype=t.dtype, device=dev)
            wide[:, 1:-2] = t
            kw[name] = wide[:, 1:-2]
        got = check(whole[:, 5:3004], **kw)
        assert bool((whole[:, :5] == 9).all()) and bool((whole[:, 3004:] == 9).all())
        for name in ("tokens", "bias_ids", "bias", "allowed"):
            kw[name] = kw[name][2:3].expand(6, -1)
        check(x.clone(), **kw)
        one = x[:1].clone()
        kw = {k: v[:1] for k, v in kw.items()}
        check(one, **kw)
        del got


@pytest.mark.gpu
def test_nothing_to_do(dev):
    """No rows, no history, all of it outside the vocabulary, neutral numbers: the logits stay."""
    print("[gpu] adjust nothing", flush=True)
    x = torch.randn(3, 100, device=dev)
    x0 = x.clone()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    t = i32(*range(30)).view(3, 10)
    adjust_logits_(x)
    adjust_logits_(x, tokens=t, lens=0, repetition=2.0, presence=1.0)
    adjust_logits_(x, tokens=t, lens=i32(0, -4, 0), repetition=2.0)
    adjust_logits_(x, tokens=t + 100, repetition=2.0, frequency=1.0)
    adjust_logits_(x, tokens=t[:, :0], repetition=2.0)
    adjust_logits_(x, tokens=t, prompt_lens=10, frequency=1.0, presence=1.0)
    adjust_logits_(x, bias_ids=t[:, :0], bias=x[:, :0])
    adjust_logits_(x[:0], tokens=t[:0], repetition=2.0)
    assert torch.equal(x, x0)


@pytest.mark.gpu
def test_infinite_penalties_ban_what_was_generated(dev):
    """An infinite frequency or presence penalty takes the generated tokens out and no other."""
    print("[gpu] adjust infinite penalties", flush=True)
    for kw in (dict(frequency=math.inf), dict(presence=math.inf)):
        x = torch.randn(1, 50, device=dev)
        x0 = x.clone()
        t = torch.tensor([[3, 4, 5, 5]], device=dev)
        adjust_logits_(x, tokens=t, prompt_lens=2, **kw)
        assert bool((x[0, 5] == -math.inf)) and torch.equal(x[0, :5], x0[0, :5])
        assert torch.equal(x[0, 6:], x0[0, 6:])


@pytest.mark.gpu
def test_same_bits_every_time_captured_and_on_a_stream(dev):
    """Many biases of one token, repeated calls, a graph replayed with other histories in the same buffers,
    sampling after it in the graph."""
    print("[gpu] adjust graph", flush=True)
    x, kw = _rows(dev, 5, 3000, F32, n=400, biases=90, mask=True, seed=12)
    kw["allowed"][-1] = -1
    first = adjust_logits_(x.clone(), **kw)
    for _ in range(3):
        assert torch.equal(adjust_logits_(x.clone(), **kw), first)
    side = torch.cuda.Stream()
    u = torch.rand(5, device=dev)
    buf = x.clone()
    both = lambda t: sample_tokens(adjust_logits_(t, **kw), u, top_k=50)  # noqa: E731
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        both(buf)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = both(buf)
    torch.cuda.synchronize()
    for rep in range(4):
        other, more = _rows(dev, 5, 3000, F32, n=400, biases=90, mask=True, seed=20 + rep)
        buf.copy_(other)
        for k, v in more.items():
            kw[k].copy_(v)
        kw["allowed"][-1] = -1
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        got, tokens = buf.clone(), out.clone()
        again = other.clone()
        assert torch.equal(both(again), tokens) and torch.equal(again, got)


@pytest.mark.gpu
def test_same_with_and_without_the_tensor_module(dev, monkeypatch):
    print("[gpu] adjust without the tensor module", flush=True)
    calls = []
    for i, kind in enumerate((dict(n=50, settings=False), dict(n=50, ids=torch.int32), dict(biases=4),
                              dict(mask=True), dict(n=30, biases=9, mask=True))):
        calls.append(_rows(dev, 3, 2500, [BF, FP, F32][i % 3], seed=40 + i, **kind))
    calls.append((calls[0][0], dict(tokens=calls[0][1]["tokens"], lens=20, prompt_lens=5,
                                    repetition=2, presence=1)))
    a = [adjust_logits_(x.clone(), **kw) for x, kw in calls]
    monkeypatch.setattr(_lib, "_tensor_calls", None)
    b = [adjust_logits_(x.clone(), **kw) for x, kw in calls]
    for x, y in zip(a, b):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def _refused(match, kind=ValueError, x=None, **kw):
    x = torch.zeros(2, 40) if x is None else x
    with pytest.raises(kind, match=match):
        adjust_logits_(x, **kw)


def test_refusals():
    i32 = lambda *dims: torch.zeros(dims, dtype=torch.int32)  # noqa: E731
    f32 = torch.zeros
    _refused("rows, V", x=f32(40))
    _refused("unit last stride", x=f32(2, 80)[:, ::2])
    _refused("share memory", x=f32(1, 40).expand(2, 40))
    _refused("unsupported dtype", x=torch.zeros(2, 40, dtype=torch.float64))
    _refused("penalties need tokens", repetition=1.5)
    _refused("penalties need tokens", presence=f32(2))
    _refused("need tokens", lens=3)
    _refused("tokens must be", tokens=i32(3, 5))
    _refused("tokens must be", tokens=f32(2, 5))
    _refused("tokens must have unit", tokens=i32(2, 10)[:, ::2])
    _refused("repetition must be positive", tokens=i32(2, 5), repetition=0.0)
    _refused("repetition must be positive", tokens=i32(2, 5), repetition=math.nan)
    _refused("repetition must be a number", tokens=i32(2, 5), repetition=f32(3))
    _refused("frequency must be a number", tokens=i32(2, 5), frequency=i32(2))
    _refused("lens must be a number", tokens=i32(2, 5), lens=torch.zeros(2, dtype=torch.int64))
    _refused("prompt_lens must be a number", tokens=i32(2, 5), prompt_lens=i32(1))
    _refused("bias_ids and bias", bias=f32(2, 3))
    _refused("bias_ids must be", bias=f32(2, 3), bias_ids=torch.zeros(2, 3, dtype=torch.int64))
    _refused("bias must be", bias=torch.zeros(2, 3, dtype=BF), bias_ids=i32(2, 3))
    _refused("differ in shape", bias=f32(2, 3), bias_ids=i32(2, 4))
    _refused("allowed must be", allowed=i32(1, 2))
    _refused("1 words for 40", allowed=i32(2, 1))
    _refused("no CPU path", kind=RuntimeError, tokens=i32(2, 5), repetition=1.5)


def test_c_entry_refusals():
    """The C entry's own checks, which come before anything touches a device."""
    lib = _lib.load()
    base = dict(stream=None, dtype=_lib.DKV_F32, logits=64, ld=40, rows=2, V=40, tokens=64, size=4,
                tld=5, N=5, pl=None, p=0, ln=None, n=5, r=None, ra=1.0, f=None, fa=0.0, pr=None, pa=0.0,
                bi=None, bil=0, b=None, bl=0, M=0, a=None, al=0)
    call = lambda **kw: lib.dkv_adjust_logits(*(base | kw).values())  # noqa: E731
    for kw in (dict(rows=-1), dict(V=-1), dict(N=-1), dict(M=-1), dict(logits=None), dict(ld=39),
               dict(size=2), dict(tld=-1), dict(al=-1), dict(M=3, bi=64), dict(M=3, b=64), dict(ra=0.0),
               dict(ra=math.nan), dict(ra=1e39), dict(ra=1e-50)):
        assert call(**kw) == _lib.DKV_E_ARG, kw
    for kw in (dict(dtype=7), dict(V=2**29, ld=2**29), dict(logits=66)):
        assert call(**kw) == _lib.DKV_E_UNSUPPORTED, kw
    assert call(rows=0) == call(V=0) == call(tokens=None) == _lib.DKV_OK
