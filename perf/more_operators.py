"""Performance cases of serving over a cache held in 8 bits, and of what changes logits before a draw.

A serving step over 8-bit pages takes the requests at hand through these operators: ``append`` norms
(where the model has such norms) and rotates the step's queries and keys and writes keys and values to
the requests' pages as e4m3 codes with a power of two for each 16 tokens and head, ``attend`` lets the
new tokens attend those pages, and ``adjust`` applies a request's penalties, biases and grammar mask to
its logits, in place, before a token is drawn. ``values`` reads pages back as the values they stand for.

A block (16 tokens of a page, one head, keys or values) holds codes c_i and an exponent e: value
c_i 2^e. Appended values y_i get the least e (within the type's range) with max |y_i| <= 448 2^e, or the
block's old e where that is more and the block holds earlier tokens of the request, whose codes are then
rounded again to the new e; c_i is y_i / 2^e rounded to e4m3 (to nearest, ties to even).

``listed`` has the fixed cases, ``draw`` further ones of the same ranges. ``prepare`` builds a
case's inputs from a seed, ``run`` is one pass (plain torch, or the package's operators where
``own`` is set), ``work`` the bytes and operations a pass cannot do without, ``exact`` the same
outputs in float64.
"""

from __future__ import annotations

import math

import torch

own = False

DH = 128            # head dimension
BLOCK = 16          # tokens that share an exponent
THETA = 500000.0
EPS = 1e-6          # of the query and key norms
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# exponents for which every code times 2^e is a number of the type (in bf16 a normal one)
LOWEST = {"bf16": -110, "fp16": -15}
HIGHEST = {"bf16": 119, "fp16": 7}
DEV = "cuda"


# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # one decode step of 64 users in the first turns of their chats (a page each)
        dict(name="append_step", op="append", dtype="bf16", groups=8, heads=32, page=64,
             requests=64, new=1, most=64, ragged=True, norms=False),
        # four 2048-token prompts, with query and key norms
        dict(name="append_prompt", op="append", dtype="bf16", groups=8, heads=32, page=64,
             requests=4, new=2048, most=2048, ragged=False, norms=True),
        # a short request's pages read back
        dict(name="values_few", op="values", dtype="fp16", groups=8, page=16, pool=400, pages=6),
        # a request of 32768 tokens read back, to hand it to a 16-bit cache
        dict(name="values_long", op="values", dtype="bf16", groups=8, page=64, pool=1024, pages=512),
        # the first tokens of one user's chat: a launch whose latency is all there is
        dict(name="attend_tiny", op="attend", dtype="bf16", groups=8, heads=32, page=16,
             requests=1, new=1, most=96, ragged=False, chunks=0),
        # the benchmark's batch: 16 users decoding over up to 8K tokens each
        dict(name="attend_step", op="attend", dtype="bf16", groups=8, heads=32, page=64,
             requests=16, new=1, most=8192, ragged=True, chunks=0),
        # two users decoding over very long documents, odd lengths
        dict(name="attend_long", op="attend", dtype="fp16", groups=8, heads=32, page=128,
             requests=2, new=1, most=131069, ragged=False, chunks=0),
        # prefill of four 2048-token prompts
        dict(name="attend_prompt", op="attend", dtype="bf16", groups=8, heads=32, page=64,
             requests=4, new=2048, most=2048, ragged=False, chunks=0),
        # the later chunks of two long prompts, 16-token pages
        dict(name="attend_chunk", op="attend", dtype="fp16", groups=8, heads=32, page=16,
             requests=2, new=500, most=6001, ragged=True, chunks=0),
        # one user's next token: penalties over what the chat has said, a few biased tokens
        dict(name="adjust_one", op="adjust", dtype="bf16", rows=1, vocab=32000, history=1000,
             ids="int64", penalties=True, biases=8, mask=False),
        # a batch whose answers follow grammars, fp32 logits
        dict(name="adjust_grammar", op="adjust", dtype="fp32", rows=37, vocab=50257, history=300,
             ids="int32", penalties=True, biases=20, mask=True),
        # a large batch with long histories over a large vocabulary
        dict(name="adjust_batch", op="adjust", dtype="bf16", rows=256, vocab=128256, history=4096,
             ids="int64", penalties=True, biases=0, mask=False),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    op = rng.choice(["append", "append", "values", "attend", "attend", "attend", "adjust",
                     "adjust"])
    if op == "adjust":
        kind = rng.choice(["penalties", "penalties", "all", "mask", "biases"])
        return dict(op="adjust", dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                    rows=_log_int(rng, 1, 128), vocab=_log_int(rng, 1000, 128256),
                    history=_log_int(rng, 1, 20000), ids=rng.choice(["int32", "int64"]),
                    penalties=kind in ("penalties", "all"),
                    biases=_log_int(rng, 1, 300) if kind in ("biases", "all") else 0,
                    mask=kind in ("mask", "all"))
    groups, heads = rng.choice([(8, 32), (8, 32), (4, 16), (2, 4), (8, 8), (2, 14)])
    page = rng.choice([16, 32, 64, 128])
    if op == "values":
        return dict(op="values", dtype=rng.choice(["bf16", "fp16", "fp32"]), groups=groups,
                    page=page, pool=_log_int(rng, 300, 800), pages=_log_int(rng, 1, 256))
    base = dict(op=op, dtype=rng.choice(["bf16", "fp16"]), groups=groups, heads=heads, page=page)
    kind = rng.choice(["step", "few", "prompt", "chunk", "mixed"])
    if op == "append":
        # a step's tokens to a batch of prompts, near and far positions
        if kind in ("step", "few", "mixed"):
            return base | dict(requests=_log_int(rng, 1, 64), new=1 if kind == "step" else
                               rng.randint(2, 9), most=_log_int(rng, 64, 100000), ragged=True,
                               norms=rng.random() < 0.5)
        new = _log_int(rng, 33, 2048)
        return base | dict(requests=rng.randint(1, 3), new=new,
                           most=new if kind == "prompt" else new + _log_int(rng, 1, 100000),
                           ragged=rng.random() < 0.5, norms=rng.random() < 0.5)
    if kind in ("step", "few"):
        # single tokens, or a few drafted ones, of one to 16 users over short and long caches
        requests = _log_int(rng, 1, 16)
        new = 1 if kind == "step" else rng.randint(2, 9)
        most = _log_int(rng, 17, 8000 if requests > 2 else 65536)
        return base | dict(requests=requests, new=min(new, most), most=most,
                           ragged=rng.random() < 0.7, chunks=0)
    if kind == "mixed":  # users decoding while one user's prompt goes through in a chunk
        return base | dict(requests=rng.randint(2, 12), new=1, most=_log_int(rng, 600, 4096),
                           ragged=True, chunks=_log_int(rng, 33, 512))
    new = _log_int(rng, 33, 1000)
    return base | dict(requests=rng.randint(1, 2), new=new,
                       most=new if kind == "prompt" else new + _log_int(rng, 1, 3500),
                       ragged=rng.random() < 0.5, chunks=0)


def _lens(case) -> tuple[list[int], list[int]]:
    """(new tokens, tokens with them) of each request, by the case alone: a ragged batch's caches
    hold between a quarter of ``most`` and all of it, its chunks between half of ``new`` and all."""
    new, lens = [], []
    n = case["requests"]
    for b in range(n):
        part = ((b * 0.6180339887) % 1.0) if case["ragged"] and n > 1 else 0.0
        new.append(max(1, round(case["new"] * (1.0 - 0.5 * part))))
        cached = case["most"] - case["new"]
        lens.append(new[b] + round(cached * (1.0 - 0.75 * part)))
    if case.get("chunks"):  # one more request, in the middle, with a chunk of its prompt
        new.insert(n // 2, case["chunks"])
        lens.insert(n // 2, max(case["chunks"], case["most"] // 2))
    return new, lens


def _first_pages(case) -> list[int]:
    """The first page in use of each request: an append reaches no page before its first new token's
    (a window of attention has given them back); attention reads all of them."""
    new, lens = _lens(case)
    if case["op"] == "attend":
        return [0] * len(new)
    return [(m - n) // case["page"] for n, m in zip(new, lens)]


def _pool_pages(case) -> int:
    page = case["page"]
    return sum(-(-m // page) - f for m, f in zip(_lens(case)[1], _first_pages(case))) + 3


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device=DEV)
    g.manual_seed(1_000_003 * (int(seed) + 1))
    return g


def _normal(g, *dims, dtype) -> torch.Tensor:
    return torch.randn(*dims, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def _ints(v) -> torch.Tensor:
    return torch.tensor(v, device=DEV, dtype=torch.int32)


def _times_two(x, e) -> torch.Tensor:
    """x 2^e for whole e, exactly (the power by its bits: a library's may be off by a step)."""
    if x.dtype == torch.float64:
        return x * ((e.long() + 1023) << 52).view(torch.float64)
    return x * ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _batch(case, g) -> dict:
    """The step's plan: page table over pages in the order a pool hands them out after some use
    (any order), row ranges, lengths."""
    new, lens = _lens(case)
    page, first = case["page"], _first_pages(case)
    need = [-(-n // page) for n in lens]
    total = _pool_pages(case)
    ids = torch.randperm(total, generator=g, device=DEV)
    table = torch.full((len(new), max(need)), -1, device=DEV, dtype=torch.int32)
    at = 0
    for b, (f, n) in enumerate(zip(first, need)):
        table[b, f:n] = ids[at:at + n - f].to(torch.int32)
        at += n - f
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    return dict(table=table, q_start=_ints(starts), lens=_ints(lens), rows=starts[-1],
                max_new=max(new), min_new=min(new), max_len=max(lens), pages=total)


def _pool(case, g, pages: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales of a pool in use: normal values, some heads and stretches of text larger than
    others, held with the exponent that their block's largest asks for."""
    h, page = case["groups"], case["page"]
    codes = torch.empty(pages, h, page, DH, device=DEV, dtype=torch.float8_e4m3fn)
    exps = torch.empty(pages, h, page // BLOCK, device=DEV, dtype=torch.int32)
    step = max(1, (1 << 25) // (h * page * DH))
    for p0 in range(0, pages, step):  # (a part at a time: a long cache in fp32 is large)
        n = min(step, pages - p0)
        x = torch.randn(n, h, page // BLOCK, BLOCK * DH, generator=g, device=DEV)
        x *= torch.exp(0.7 * torch.randn(n, h, page // BLOCK, 1, generator=g, device=DEV))
        e = torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True) / 448.0)).to(torch.int32)
        exps[p0:p0 + n] = e[..., 0]
        codes[p0:p0 + n] = _times_two(x, -e).clamp_(-448.0, 448.0).view(
            n, h, page, DH).to(torch.float8_e4m3fn)
    return codes, (exps + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _adjust_inputs(case, g) -> dict:
    rows, vocab, n = case["rows"], case["vocab"], case["history"]
    r = lambda lo, hi: lo + (hi - lo) * torch.rand(rows, generator=g, device=DEV)  # noqa: E731
    s = dict(logits=(torch.randn(rows, vocab, generator=g, device=DEV) * 2.5).to(
        DTYPES[case["dtype"]]))
    if case["penalties"]:
        # a text's tokens: few that come often, many that come once; the prompt, then the answer
        u = torch.rand(rows, n, generator=g, device=DEV)
        s["tokens"] = (u ** 4 * vocab).long().clamp_(max=vocab - 1).to(
            torch.int32 if case["ids"] == "int32" else torch.int64)
        s["history"] = torch.clamp(n * r(0.25, 1.05), min=1, max=n).to(torch.int32)
        s["prompt"] = (s["history"] * r(0.0, 1.0)).to(torch.int32)
        s["repetition"], s["frequency"], s["presence"] = r(0.95, 1.3), r(-0.1, 0.6), r(-0.1, 0.6)
    if case["biases"]:
        m = case["biases"]
        ids = torch.randint(0, vocab, (rows, m), generator=g, device=DEV, dtype=torch.int32)
        ids[:, m // 2:m // 2 + 1] = ids[:, :1]            # a token that is biased twice
        ids[torch.rand(rows, m, generator=g, device=DEV) < 0.1] = -1
        s["bias_ids"] = ids
        s["bias"] = torch.randn(rows, m, generator=g, device=DEV) * 4.0
    if case["mask"]:
        # a grammar allows few tokens (a digit, a bracket), about half, or nearly all (inside a text)
        share = torch.tensor([0.002, 0.5, 0.98], device=DEV)[torch.arange(rows, device=DEV) % 3]
        words = -(-vocab // 32)
        bits = torch.rand(rows, words * 32, generator=g, device=DEV) < share[:, None]
        weight = torch.bitwise_left_shift(torch.ones(32, device=DEV, dtype=torch.int64),
                                          torch.arange(32, device=DEV))
        word = (bits.view(rows, words, 32) * weight).sum(-1)
        s["allowed"] = torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32)
    return s


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case=case)
    if case["op"] == "adjust":
        return s | _adjust_inputs(case, g)
    if case["op"] == "values":
        s["ids"] = torch.randperm(case["pool"], generator=g, device=DEV)[:case["pages"]].to(
            torch.int32)
        s["pages"] = case["pool"]
    else:
        s |= _batch(case, g)
    s["k"], s["k_scale"] = _pool(case, g, s["pages"])
    s["v"], s["v_scale"] = _pool(case, g, s["pages"])
    dt = DTYPES[case["dtype"]]
    if case["op"] == "attend":
        s["q"] = _normal(g, s["rows"], case["heads"], DH, dtype=dt)
    if case["op"] == "append":
        s["qkv"] = _normal(g, s["rows"], (case["heads"] + 2 * case["groups"]) * DH, dtype=dt)
        s["q_norm"] = s["k_norm"] = None
        if case["norms"]:
            s["q_norm"] = (1.0 + 0.1 * torch.randn(DH, generator=g, device=DEV)).to(dt)
            s["k_norm"] = (1.0 + 0.1 * torch.randn(DH, generator=g, device=DEV)).to(dt)
    return s


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _run_own(state)
    return {"append": _plain_append, "values": _plain_values, "attend": _plain_attend,
            "adjust": _plain_adjust}[state["case"]["op"]](state)


def _run_own(s):
    case = s["case"]
    if case["op"] == "adjust":
        from dynakv_amd.kernels.sampling import adjust_logits_
        more = {}
        if case["penalties"]:
            more |= dict(tokens=s["tokens"], prompt_lens=s["prompt"], lens=s["history"],
                         repetition=s["repetition"], frequency=s["frequency"],
                         presence=s["presence"])
        if case["biases"]:
            more |= dict(bias_ids=s["bias_ids"], bias=s["bias"])
        if case["mask"]:
            more |= dict(allowed=s["allowed"])
        return adjust_logits_(s["logits"], **more)
    from dynakv_amd.kernels.paged import PagedBatch, paged_append, paged_attention, paged_values
    scales = dict(k_scale=s["k_scale"], v_scale=s["v_scale"])
    dt = DTYPES[case["dtype"]]
    if case["op"] == "values":
        k, v = paged_values(s["k"], s["v"], **scales, pages=s["ids"], dtype=dt)
        return dict(k=k, v=v)
    batch = PagedBatch(page_table=s["table"], q_start=s["q_start"], lens=s["lens"],
                       rows=s["rows"], max_new=s["max_new"], max_len=s["max_len"],
                       min_new=s["min_new"])
    if case["op"] == "attend":
        return paged_attention(s["q"], s["k"], s["v"], batch, **scales)
    q = paged_append(s["qkv"], s["k"], s["v"], batch, heads=case["heads"], theta=THETA,
                     q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, **scales)
    k, v = paged_values(s["k"], s["v"], **scales, dtype=dt)  # the pool as the values it stands for
    return dict(q=q, k=k, v=v)


def _exponents(scale) -> torch.Tensor:
    return scale.view(torch.uint8).to(torch.int32) - 127


def _held(codes, scale) -> torch.Tensor:
    """fp32 values of pages (n, heads, page, DH)."""
    n, h, page, _ = codes.shape
    x = codes.float().view(n, h, page // BLOCK, BLOCK * DH)
    return _times_two(x, _exponents(scale)[..., None]).view(n, h, page, DH)


def _plain_values(s):
    dt, at = DTYPES[s["case"]["dtype"]], s["ids"].long()
    return dict(k=_held(s["k"][at], s["k_scale"][at]).to(dt),
                v=_held(s["v"][at], s["v_scale"][at]).to(dt))


def _places(s):
    """(request, position) of each row of the step."""
    row = torch.arange(s["rows"], device=DEV)
    req = torch.bucketize(row, s["q_start"][1:].long(), right=True)
    return req, s["lens"][req].long() - s["q_start"][req + 1].long() + row


def _to_e4m3(y):
    """y rounded to the nearest e4m3 value (ties to even), at most 448, in y's own type."""
    e = torch.clamp(torch.frexp(y).exponent - 1, min=-6) - 3  # log2 of the step at y
    return _times_two(torch.round(_times_two(y, -e)), e).clamp(-448.0, 448.0)


def _store(s, codes, scale, y, where, head, slot):
    """The pool's values (fp32) after rows y (rows, heads, DH, in 64 bits: values next to a border
    between two codes) went to page ``where``, slot ``slot``."""
    pages, h, page, _ = codes.shape
    kind = s["case"]["dtype"]
    blocks = page // BLOCK
    b = slot // BLOCK
    # per block: largest new value, first new slot (the page's own slots from 0 on)
    at = (where * h + head) * blocks + b                                    # (rows, heads)
    n = pages * h * blocks
    big = torch.zeros(n, device=DEV, dtype=torch.float64).scatter_reduce_(
        0, at.reshape(-1), y.abs().amax(-1).reshape(-1), "amax")
    first = torch.full((n,), page, device=DEV).scatter_reduce_(
        0, at.reshape(-1), slot.expand_as(at).reshape(-1), "amin")
    m, e = torch.frexp(big / 448.0)
    need = torch.where(m > 0.5, e, e - 1).clamp_(LOWEST[kind], HIGHEST[kind])
    need = torch.where(big > 0, need, LOWEST[kind])
    old = _exponents(scale).reshape(-1)
    old_kept = old.clamp(LOWEST[kind], HIGHEST[kind])
    touched, starts = first < page, first % BLOCK == 0
    new = torch.where(touched, torch.where(starts, need, torch.maximum(need, old_kept)), old)
    lower = torch.where(touched, new - old, 0).view(pages, h, blocks, 1, 1)
    c = codes.float().view(pages, h, blocks, BLOCK, DH)
    earlier = (torch.arange(page, device=DEV).view(blocks, BLOCK, 1)
               < torch.where(touched, first, 0).view(pages, h, blocks, 1, 1))
    c = torch.where(earlier & (lower > 0), _to_e4m3(_times_two(c, -lower)), c)
    x = _times_two(c, new.view(pages, h, blocks, 1, 1)).view(pages, h, page, DH)
    e = new[at][..., None]
    x[where, head, slot] = _times_two(_to_e4m3(_times_two(y, -e)), e).float()
    return x


def _plain_append(s):
    case = s["case"]
    hq, g, page = case["heads"], case["groups"], case["page"]
    dt = DTYPES[case["dtype"]]
    req, pos = _places(s)
    x = s["qkv"].view(s["rows"], hq + 2 * g, DH)
    # (keys in 64 bits: a value next to a border between two codes falls to one side or the other)
    q, k, v = x[:, :hq].float(), x[:, hq:hq + g].double(), x[:, hq + g:].double()
    if s["q_norm"] is not None:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + EPS) * s["q_norm"].float()
        k = k / torch.sqrt(k.square().mean(-1, keepdim=True) + EPS) * s["k_norm"].double()
    j = torch.arange(DH // 2, device=DEV, dtype=torch.float64)
    # far positions times frequencies: the angle in 64 bits
    ang = pos.double()[:, None] * torch.exp(-(2.0 * j / DH) * math.log(THETA))
    c, sn = torch.cos(ang)[:, None], torch.sin(ang)[:, None]

    def turn(t):
        a, b = t[..., : DH // 2], t[..., DH // 2:]
        ct, st = c.to(t.dtype), sn.to(t.dtype)
        return torch.cat([a * ct - b * st, b * ct + a * st], dim=-1)

    where = s["table"][req, pos // page].long()[:, None]
    slot, head = (pos % page)[:, None], torch.arange(g, device=DEV)[None, :]
    return dict(q=turn(q).to(dt),
                k=_store(s, s["k"], s["k_scale"], turn(k), where, head, slot).to(dt),
                v=_store(s, s["v"], s["v_scale"], v, where, head, slot).to(dt))


def _plain_attend(s):
    case = s["case"]
    hq, g, page = case["heads"], case["groups"], case["page"]
    hpg, n_max, l_max = hq // g, s["max_new"], s["max_len"]
    req, pos = _places(s)
    key = torch.arange(l_max, device=DEV)
    where = s["table"][:, key // page].long()                      # (B, L); -1 past the request
    inside = key < s["lens"][:, None]                              # (B, L)

    def pick(codes, scale):                                        # (B, G, L, DH)
        e = torch.where(inside[:, :, None], _exponents(scale)[where, :, key % page // BLOCK], 0)
        c = torch.where(inside[:, :, None, None], codes[where, :, key % page].float(), 0.0)
        return _times_two(c, e[..., None]).transpose(1, 2)

    k, v = pick(s["k"], s["k_scale"]), pick(s["v"], s["v_scale"])
    # rows of the step as (B, G, new token and head of the group, DH), padded to the longest
    at = torch.arange(s["rows"], device=DEV) - s["q_start"][req].long()
    n = s["lens"].numel()
    q = torch.zeros(n, n_max, hq, DH, device=DEV)
    q[req, at] = s["q"].float()
    limit = torch.full((n, n_max), -1, device=DEV)
    limit[req, at] = pos
    q = q.view(n, n_max, g, hpg, DH).transpose(1, 2).reshape(n, g, n_max * hpg, DH)
    dead = key > limit.repeat_interleave(hpg, 1)[:, None, :, None]  # (B, 1, rows, L)
    z = torch.matmul(q, k.transpose(-1, -2).contiguous()).mul_(1.0 / math.sqrt(DH))
    z.masked_fill_(dead, -math.inf)
    m = z.amax(-1, keepdim=True)
    e = z.sub_(torch.where(m == -math.inf, 0.0, m)).exp_()
    o = torch.matmul(e, v) / e.sum(-1, keepdim=True)
    o = o.view(n, g, n_max, hpg, DH).transpose(1, 2).reshape(n, n_max, hq, DH)
    return o[req, at].to(s["q"].dtype)


def _plain_adjust(s):
    case, out = s["case"], s["logits"]
    rows, vocab = out.shape
    x = out.float()
    if case["penalties"]:
        n = s["tokens"].shape[1]
        at, place = s["tokens"].long(), torch.arange(n, device=DEV)[None, :]
        used = place < s["history"][:, None]
        said = used & (place >= s["prompt"][:, None])
        seen = torch.zeros(rows, vocab, device=DEV).scatter_add_(1, at, used.float()) > 0
        count = torch.zeros(rows, vocab, device=DEV).scatter_add_(1, at, said.float())
        r = s["repetition"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
        x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if case["biases"]:
        there = s["bias_ids"] >= 0
        x = x + torch.zeros_like(x).scatter_add_(1, s["bias_ids"].clamp(min=0).long(),
                                                 torch.where(there, s["bias"], 0.0))
    if case["mask"]:
        bit = torch.bitwise_right_shift(s["allowed"][:, :, None], torch.arange(
            32, device=DEV, dtype=torch.int32)) & 1
        x = x.masked_fill(bit.view(rows, -1)[:, :vocab] == 0, -math.inf)
    return out.copy_(x)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case) -> dict:
    if case["op"] == "adjust":
        size, rows, vocab = (4 if case["dtype"] == "fp32" else 2), case["rows"], case["vocab"]
        b = 0.0
        if case["penalties"]:  # ids read; the logits of their tokens read and written
            ids = 0.65 * rows * case["history"]
            b += (4 if case["ids"] == "int32" else 8) * ids + 20 * rows
            b += 2 * size * min(ids, rows * vocab)
        b += rows * case["biases"] * (8 + 2 * size)
        if case["mask"]:       # a bit a token; about half of the logits written
            b += rows * vocab * (0.125 + 0.5 * size)
        return dict(bytes=b, flops=b / 4)
    h = case["groups"]
    per_page = 2 * h * case["page"] * DH                       # values of keys and values
    if case["op"] == "values":
        size = 4 if case["dtype"] == "fp32" else 2
        n = case["pages"] * per_page
        return dict(bytes=(1 + size) * n + n // (BLOCK * DH), flops=n)
    new, lens = _lens(case)
    rows, hq = sum(new), case["heads"]
    if case["op"] == "append":  # and the pool read back
        vals, held = rows * (hq + 2 * h) * DH, _pool_pages(case) * per_page
        return dict(bytes=2 * vals + 2 * rows * hq * DH + 2 * rows * h * DH + 3 * held,
                    flops=(8 if case["norms"] else 4) * vals + held)
    pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(new, lens))
    return dict(bytes=2 * sum(lens) * h * DH + 4 * rows * hq * DH, flops=4 * pairs * hq * DH)


# ---------------------------------------------------------------------------------------------
# float64 results
# ---------------------------------------------------------------------------------------------
def _two_to(e) -> torch.Tensor:
    return _times_two(torch.ones(e.shape, device=DEV, dtype=torch.float64), e)


def _exact_pages(codes, scale) -> torch.Tensor:
    """float64 values of (..., page, DH) codes."""
    two = _two_to(scale.view(torch.uint8).long() - 127)
    return codes.double() * two.repeat_interleave(BLOCK, -1)[..., None]


def _exact_values(s, case):
    at = s["ids"].long()
    return dict(k=_exact_pages(s["k"][at], s["k_scale"][at]),
                v=_exact_pages(s["v"][at], s["v_scale"][at]))


# the e4m3 values from 0 on, in the order of their codes
_GRID = [i / 512.0 for i in range(8)] + [(1.0 + m / 8.0) * 2.0 ** e for e in range(-6, 9)
                                         for m in range(8)][:-1]


def _nearest(y):
    """The nearest of the e4m3 values, of two the one with the even code."""
    grid = torch.tensor(_GRID, device=DEV, dtype=torch.float64)
    a = y.abs().clamp(max=448.0).contiguous()
    low = torch.searchsorted(grid, a, right=True) - 1
    high = torch.clamp(low + 1, max=len(_GRID) - 1)
    below, above = a - grid[low], grid[high] - a
    up = (above < below) | ((above == below) & (high % 2 == 0))
    return torch.where(up, grid[high], grid[low]) * torch.where(y < 0, -1.0, 1.0)


def _exact_append(s, case):
    hq, g, page = case["heads"], case["groups"], case["page"]
    new, lens = _lens(case)
    table = s["table"].tolist()
    lowest, highest = LOWEST[case["dtype"]], HIGHEST[case["dtype"]]
    pools = {}
    for name in ("k", "v"):
        two = _two_to(s[name + "_scale"].view(torch.uint8).long() - 127)
        pools[name] = (s[name].double(), two)
    q_out = torch.empty(s["rows"], hq, DH, device=DEV, dtype=torch.float64)
    freq = torch.tensor([THETA ** (-2.0 * i / DH) for i in range(DH // 2)], device=DEV,
                        dtype=torch.float64)
    at = 0
    for b, (n, total) in enumerate(zip(new, lens)):
        x = s["qkv"][at:at + n].double().view(n, hq + 2 * g, DH)
        y = x[:, :hq + g].clone()
        if s["q_norm"] is not None:
            y /= torch.sqrt((y * y).sum(-1, keepdim=True) / DH + EPS)
            y[:, :hq] *= s["q_norm"].double()
            y[:, hq:] *= s["k_norm"].double()
        ang = torch.arange(total - n, total, device=DEV, dtype=torch.float64)[:, None, None] * freq
        # a pair (j, j + 64) as a complex number, turned by its angle
        z = torch.complex(y[..., : DH // 2], y[..., DH // 2:]) * torch.polar(
            torch.ones_like(ang), ang)
        y = torch.cat([z.real, z.imag], dim=-1)
        q_out[at:at + n] = y[:, :hq]
        for t0 in range((total - n) // BLOCK * BLOCK, total, BLOCK):  # block by block
            lo, hi = max(t0, total - n), min(t0 + BLOCK, total)
            p, i, s0 = table[b][t0 // page], t0 % page // BLOCK, t0 % page
            for name, rows in (("k", y[:, hq:]), ("v", x[:, hq + g:])):
                codes, two = pools[name]
                vals = rows[lo - (total - n):hi - (total - n)].transpose(0, 1)  # (heads, n, DH)
                big = vals.abs().amax((1, 2))
                e = torch.ceil(torch.log2(big / 448.0)).clamp(lowest, highest).long()
                e = torch.where(_two_to(e - 1) * 448.0 >= big, e - 1, e)  # (a logarithm's rounding)
                e = torch.where(_two_to(e) * 448.0 < big, e + 1, e)
                step = _two_to(e.clamp(lowest, highest))
                if lo > t0:
                    was = two[p, :, i].clamp(2.0 ** lowest, 2.0 ** highest)
                    step = torch.maximum(step, was)
                    part = codes[p, :, s0:s0 + lo - t0]
                    codes[p, :, s0:s0 + lo - t0] = _nearest(part * (was / step)[:, None, None])
                codes[p, :, s0 + lo - t0:s0 + hi - t0] = _nearest(vals / step[:, None, None])
                two[p, :, i] = step
        at += n
    out = dict(q=q_out)
    for name, (codes, two) in pools.items():
        out[name] = codes * two.repeat_interleave(BLOCK, -1)[..., None]
    return out


def _exact_attend(s, case):
    hq, g = case["heads"], case["groups"]
    hpg = hq // g
    new, lens = _lens(case)
    out = torch.empty(s["rows"], hq, DH, device=DEV, dtype=torch.float64)
    at = 0
    for b, (n, total) in enumerate(zip(new, lens)):
        ids = s["table"][b][: -(-total // case["page"])].long()
        dead = (torch.arange(total, device=DEV)[None, :]
                > torch.arange(total - n, total, device=DEV)[:, None])
        for h in range(g):
            k = _exact_pages(s["k"][ids, h], s["k_scale"][ids, h]).reshape(-1, DH)[:total]
            v = _exact_pages(s["v"][ids, h], s["v_scale"][ids, h]).reshape(-1, DH)[:total]
            for i in range(h * hpg, (h + 1) * hpg):
                z = (s["q"][at:at + n, i].double() @ k.T) / math.sqrt(DH)
                out[at:at + n, i] = torch.softmax(z.masked_fill(dead, -math.inf), -1) @ v
        at += n
    return out


def _exact_adjust(s, case):
    out = s["logits"].double()
    vocab = case["vocab"]
    for b in range(case["rows"]):
        x = out[b]
        if case["penalties"]:
            ids = s["tokens"][b, :int(s["history"][b])].long()
            count = torch.bincount(ids[int(s["prompt"][b]):], minlength=vocab).double()
            r = float(s["repetition"][b])
            at = torch.unique(ids)
            x[at] = torch.where(x[at] > 0, x[at] / r, x[at] * r)
            x -= float(s["frequency"][b]) * count
            x[count > 0] -= float(s["presence"][b])
        if case["biases"]:
            there = s["bias_ids"][b] >= 0
            x.index_add_(0, s["bias_ids"][b][there].long(), s["bias"][b][there].double())
        if case["mask"]:
            word = s["allowed"][b].long()
            bits = torch.stack([(word >> i) & 1 for i in range(32)], 1).reshape(-1)[:vocab]
            x[bits == 0] = -math.inf
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "values": _exact_values, "attend": _exact_attend,
            "adjust": _exact_adjust}[case["op"]](s, case)
