"""The paged cache's host side, without a device: pages taken and given back, the batch's buffers,
and the refusals of the operators (checked before anything touches a device)."""
import shutil
import subprocess
import sys

import pytest
import torch

from dynakv_amd import _lib
from dynakv_amd.kernels import decode, paged
from dynakv_amd.kernels.paged import PagedBatch, PagedKVCache, paged_append, paged_attention
from dynakv_amd.kernels.sampling import sample_tokens
from dynakv_amd.model import LlamaShape, PagedLlama

BF = torch.bfloat16


def _cache(pages=10, **kw):
    return PagedKVCache(2, pages, 2, page_size=16, device="cpu", **kw)


def test_pages_are_taken_as_tokens_need_them():
    c = _cache()
    a, b = c.add(), c.add()
    batch = c.batch([(a, 17), (b, 16)])
    assert (c.length(a), c.length(b), c.free_pages) == (17, 16, 7)
    assert batch.q_start.tolist() == [0, 17, 33] and batch.lens.tolist() == [17, 16]
    assert (batch.rows, batch.max_new, batch.min_new, batch.max_len) == (33, 17, 16, 17)
    assert batch.page_table.tolist() == [c.page_ids(a), c.page_ids(b) + [-1]]
    batch = c.batch([(b, 1), (a, 1)])  # b needs its second page, a has room
    assert c.free_pages == 6 and batch.page_table.tolist() == [c.page_ids(b), c.page_ids(a)]
    assert len(set(c.page_ids(a) + c.page_ids(b))) == 4
    assert batch.lens.tolist() == [17, 18] and batch.q_start.tolist() == [0, 1, 2]
    assert c.k[0].shape == (10, 2, 16, 128) and len(c.v) == 2


def test_pages_come_back():
    c = _cache(pages=4)
    a, b = c.add(), c.add()
    c.batch([(a, 40), (b, 5)])
    assert c.free_pages == 0
    held = c.page_ids(a)
    c.truncate(a, 33)
    assert c.free_pages == 0 and c.length(a) == 33
    c.truncate(a, 32)
    assert c.free_pages == 1 and c.page_ids(a) == held[:2]
    c.free(a)
    assert c.free_pages == 3
    with pytest.raises(ValueError, match="no request"):
        c.length(a)
    c.batch([(b, 40)])
    assert c.length(b) == 45 and c.free_pages == 1


def test_a_step_that_does_not_fit_changes_nothing():
    c = _cache(pages=3)
    a, b = c.add(), c.add()
    c.batch([(a, 16)])
    with pytest.raises(RuntimeError, match="needs 3 pages, 2 are free"):
        c.batch([(a, 1), (b, 17)])
    assert (c.length(a), c.length(b), c.free_pages) == (16, 0, 2)
    with pytest.raises(ValueError, match="once"):
        c.batch([(a, 1), (a, 1)])
    with pytest.raises(ValueError, match="negative"):
        c.batch([(a, -1)])
    with pytest.raises(ValueError, match="no request"):
        c.batch([(99, 1)])
    with pytest.raises(ValueError):
        c.truncate(a, 17)
    assert (c.length(a), c.free_pages) == (16, 2)


def test_empty_steps():
    c = _cache()
    a = c.add()
    batch = c.batch([])
    assert batch.requests == 0 and batch.rows == 0 and batch.max_new == 0
    batch = c.batch([(a, 0)])
    assert batch.requests == 1 and batch.rows == 0 and batch.page_table.shape == (1, 0)


@pytest.mark.parametrize("kw", [dict(page_size=8), dict(page_size=24), dict(page_size=0),
                                dict(dtype=torch.float32)])
def test_cache_refusals(kw):
    with pytest.raises(ValueError):
        PagedKVCache(1, 4, 2, device="cpu", **kw)
    with pytest.raises(ValueError):
        PagedKVCache(1, 0, 2, device="cpu")


def _batch(B=2, cols=3, **kw):
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    args = dict(rows=4, max_new=2, max_len=20) | kw
    return PagedBatch(torch.zeros(B, cols, dtype=torch.int32), i32(0, 2, 4), i32(20, 7), **args)


def test_batch_refusals():
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    table, start, lens = torch.zeros(2, 3, dtype=torch.int32), i32(0, 2, 4), i32(20, 7)
    ok = dict(rows=4, max_new=2, max_len=20)
    PagedBatch(table, start, lens, **ok)
    for args, kw in (((table, start[:2], lens), ok), ((table[:1], start, lens), ok),
                     ((table.long(), start, lens), ok), ((table, start.float(), lens), ok),
                     ((table.t().contiguous().t(), start, lens), ok),
                     ((table, torch.zeros(6, dtype=torch.int32)[::2], lens), ok),
                     ((table, start, lens), ok | dict(max_new=5)),
                     ((table, start, lens), ok | dict(min_new=3)),
                     ((table, start, lens), ok | dict(max_len=-1))):
        with pytest.raises(ValueError):
            PagedBatch(*args, **kw)


def test_a_batch_is_fixed():
    """Its launch arguments are taken when it is made: only the buffers' contents may change."""
    b = _batch()
    for name, value in (("lens", b.lens.clone()), ("rows", 3), ("max_len", 40), ("other", 1)):
        with pytest.raises(AttributeError):
            setattr(b, name, value)
    assert b.rows == 4 and b.max_len == 20 and b.requests == 2


def _pages(pages=4, heads=2, size=16, dtype=BF):
    return torch.zeros(pages, heads, size, 128, dtype=dtype)


def test_append_refusals():
    b, k = _batch(), _pages()
    qkv = torch.zeros(4, (4 + 4) * 128, dtype=BF)
    call = lambda **kw: paged_append(**(dict(qkv=qkv, k_pages=k, v_pages=k.clone(), batch=b,  # noqa: E731
                                             heads=4, theta=1e4) | kw))
    with pytest.raises(RuntimeError, match="no CPU path"):
        call()
    for kw in (dict(theta=None), dict(inv_freq=[1.0] * 64), dict(theta=0.0), dict(theta=-2.0),
               dict(theta=float("inf")), dict(theta=None, inv_freq=[1.0] * 63),
               dict(theta=None, inv_freq=[float("nan")] * 64),
               dict(heads=8), dict(heads=0), dict(qkv=qkv[:3]), dict(qkv=qkv.half()),
               dict(qkv=qkv.t().contiguous().t()), dict(v_pages=_pages(heads=1)),
               dict(k_pages=_pages(dtype=torch.float16)),
               dict(k_pages=k.transpose(1, 2).contiguous().transpose(1, 2)),
               dict(q_norm=torch.ones(64, dtype=BF)), dict(k_norm=torch.ones(128)),
               dict(eps=-1.0), dict(batch=_batch(max_len=49))):
        with pytest.raises(ValueError):
            call(**kw)
    with pytest.raises(NotImplementedError):
        call(k_pages=_pages(size=24), v_pages=_pages(size=24))


def test_attention_refusals():
    b, k = _batch(), _pages()
    q = torch.zeros(4, 4, 128, dtype=BF)
    call = lambda **kw: paged_attention(**(dict(q=q, k_pages=k, v_pages=k.clone(), batch=b) | kw))  # noqa: E731
    with pytest.raises(RuntimeError, match="no CPU path"):
        call()
    for kw in (dict(q=q[:, :3]), dict(q=q[:, :0]), dict(q=q[:3]), dict(q=q.half()),
               dict(q=q[..., :64]), dict(out_dtype=torch.float16), dict(q=q[0]),
               dict(batch=_batch(max_len=49)), dict(v_pages=_pages(pages=5))):
        with pytest.raises(ValueError):
            call(**kw)


def test_c_entry_refusals():
    """Bad arguments are refused before any launch; empty work is a no-op."""
    lib = _lib.load()
    E, U, OK = _lib.DKV_E_ARG, _lib.DKV_E_UNSUPPORTED, _lib.DKV_OK

    def append(dtype=_lib.DKV_BF16, ps=16, cols=2, ld=2, B=1, T=1, hq=4, hkv=2, dh=128, stride=4096):
        return lib.dkv_paged_append(None, dtype, None, 1024, None, 512, 128, None, None, stride,
                                    2048, 4, ps, None, ld, cols, None, None, B, T, hq, hkv, dh,
                                    None, None, 1e-6, None)

    assert append() == E and append(dtype=0) == U and append(dh=64) == U and append(hq=3) == U
    assert append(B=-1) == E and append(hkv=0) == E and append(ld=1) == E
    assert append(ps=24, cols=0) == U and append(ps=8, cols=0) == U
    assert append(B=0, cols=0) == OK and append(T=0, cols=0) == OK
    assert append(stride=4, cols=0) == U
    # pages on top of each other
    assert append(stride=0, cols=0) == E and append(stride=1024, cols=0) == E

    def attend(dtype=_lib.DKV_BF16, scale=0.1, B=1, T=1, hq=4, hkv=2, new=1, odt=_lib.DKV_BF16):
        return lib.dkv_paged_attention(None, dtype, None, 512, 128, None, None, 4096, 2048, 4, 16,
                                       None, 0, 0, None, None, B, T, hq, hkv, 128, new, 1, 16,
                                       scale, None, 0, None, odt, 512, 128)

    assert attend() == E and attend(dtype=0) == U and attend(hq=34) == U and attend(hq=5) == U
    assert attend(odt=_lib.DKV_F16) == E and attend(B=-1) == E
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert attend(scale=scale) == U
    assert attend(B=0) == OK and attend(T=0) == OK and attend(new=0) == OK


def test_sampling_refusals():
    x, u = torch.zeros(3, 8), torch.zeros(3)
    with pytest.raises(RuntimeError, match="no CPU path"):
        sample_tokens(x, u)
    for args, kw in (((x[0], u), {}), ((x, u[:2]), {}), ((x, u.double()), {}),
                     ((x[:, :0], u), {}), ((x.t().contiguous().t(), u), {}),
                     ((x, u), dict(temperature=torch.ones(2))),
                     ((x, u), dict(top_k=torch.ones(3))),
                     ((x, u), dict(top_p=torch.ones(3, dtype=torch.float64))),
                     ((x, u), dict(min_p=torch.ones(6)[::2]))):
        with pytest.raises(ValueError):
            sample_tokens(*args, **kw)
    with pytest.raises(NotImplementedError):
        sample_tokens(torch.zeros(1, (1 << 19) + 1), u[:1])
    lib = _lib.load()
    call = lambda dt, rows, v, ld=8: lib.dkv_sample_tokens(  # noqa: E731
        None, dt, None, ld, rows, v, None, None, 1.0, None, 0, None, 1.0, None, 0.0, None, 0, None)
    assert call(0, 1, 8) == _lib.DKV_E_ARG and call(0, -1, 8) == _lib.DKV_E_ARG
    assert call(9, 1, 8) == _lib.DKV_E_UNSUPPORTED and call(0, 1, 1 << 20) == _lib.DKV_E_UNSUPPORTED
    assert call(0, 0, 8) == _lib.DKV_OK and call(0, 1, 0) == _lib.DKV_E_ARG


def test_without_the_tensor_module(monkeypatch):
    """What a batch holds for its calls is the same, and so is what is refused."""
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    table = torch.zeros(3, 9, dtype=torch.int32)
    makes = [lambda: PagedBatch(table[:2, :5], start, lens, rows=4, max_new=3, max_len=20, min_new=2),
             lambda: PagedBatch(table[:1, :1], start[:2], lens[:1], rows=0, max_new=0, max_len=0,
                                min_new=0),
             lambda: PagedBatch(table[:0], start[:1], lens[:0], rows=7, max_new=1, max_len=5)]
    start, lens = i32(0, 2, 4), i32(20, 7)
    assert _lib.tensor_calls() is not None  # built here
    fast = [m() for m in makes]
    monkeypatch.setattr(_lib, "_tensor_calls", None)
    for m, f in zip(makes, fast):
        assert m()._args == f._args and m().requests == f.requests
    test_batch_refusals()
    test_append_refusals()
    test_attention_refusals()


def test_tensor_module_of_another_torch(monkeypatch, tmp_path):
    """It is left alone: the operators make their calls by themselves."""
    monkeypatch.setattr(_lib, "_tensor_calls", False)
    monkeypatch.setattr(torch, "__version__", "1.0.0")
    assert _lib.tensor_calls() is None
    monkeypatch.setattr(_lib, "_tensor_calls", False)
    monkeypatch.setattr(_lib, "LIB_PATH", tmp_path / "none.so")
    assert _lib.tensor_calls() is None
    _batch()


@pytest.mark.parametrize("heads,kv", [(32, 8), (16, 1), (8, 8)])
def test_requests_without_new_tokens_need_no_workspace(heads, kv):
    """A chunk beside requests that have no token in the step: the records are those of the requests
    that can have rows, by the step's rows and the least number of new tokens."""
    floats = lambda B, T, new, least: _lib.load().dkv_paged_workspace_floats(  # noqa: E731
        B, T, heads, kv, new, least, 32768)
    alone = floats(1, 64, 64, 64)
    assert alone > 16384
    for B in (2, 64, 1024):
        assert floats(B, 64, 64, 64) == alone
        # single tokens are allowed: requests of more than 16 rows are still few
        few = 64 // (16 // (heads // kv) + 1)
        assert floats(B, 64, 64, 1) <= floats(1, 64, 64, 1) * (1 + few) + 256 * 16 * 130


def test_the_attention_has_a_workspace_of_its_own(monkeypatch):
    """Other operators' calls, which another thread may make between its two launches, do not write
    there."""
    monkeypatch.setattr(_lib, "call_on", lambda device, fn, *args: False)  # no capture
    monkeypatch.setattr(paged, "_WORKSPACES", {}, raising=False)
    q = torch.zeros(1, 1, 128, dtype=BF)
    mine = paged._attention_workspace(q, 77, 1 << 17)
    assert mine is paged._attention_workspace(q, 77, 1 << 16) and not mine.any()
    assert mine.data_ptr() != decode.workspace(q.device, 77, 1 << 17).data_ptr()
    assert mine is not paged._attention_workspace(q, 78, 1 << 16)
    decode._WS_CACHE.pop((q.device.index, 77))


def test_outputs_on_top_of_inputs_or_themselves():
    """An output may be its operator's queries, place for place, or memory that no row of theirs and no
    other row of its own has: anything else is refused, as rows are written while others are read. (No
    call here gets to its launch: weights off their alignment, or no workspace, are refused next.)"""
    lib = _lib.load()
    E, U, WS = _lib.DKV_E_ARG, _lib.DKV_E_UNSUPPORTED, _lib.DKV_E_WORKSPACE
    at, far = 1 << 32, (1 << 32) + (1 << 24)

    def append(q_out, q_st, q_sh, T=4, hq=4):  # a projection of (T, 1024), 8 heads
        return lib.dkv_paged_append(None, _lib.DKV_BF16, at, 1024, q_out, q_st, q_sh, at << 1, at << 2,
                                    4096, 2048, 4, 16, at << 3, 2, 2, at << 3, at << 3, 1, T, hq,
                                    (8 - hq) // 2, 128, at + 2, None, 1e-6, at)

    for q_out, st, sh in ((at, 1024, 128), (far, 512, 128), (far, 128, 512), (far, 640, 128),
                          (far, 1024, 256), (at - 4096, 512, 128), (at + 8192, 512, 128)):
        assert append(q_out, st, sh) == U, (q_out - at, st, sh)
    for q_out, st, sh in ((at + 16, 1024, 128), (at + 2048, 1024, 128), (at + 1024, 1024, 128),
                          (at - 256, 1024, 128), (at, 512, 128), (at, 1024, 256), (at - 4080, 512, 128),
                          (at + 8176, 512, 128), (far, 128, 128), (far, 256, 128), (far, 384, 384),
                          (far, 504, 128), (far, 128, 504)):
        assert append(q_out, st, sh) == E, (q_out - at, st, sh)
    assert append(at, 8, 128, T=1) == E and append(at, 512, 128, T=1) == U  # (a row is a row)
    assert append(at + 256, 512, 128, T=1) == E

    def attend(out, o_st, o_sh, q_st=512, q_sh=128, T=4, hq=4, odt=_lib.DKV_BF16):
        return lib.dkv_paged_attention(None, _lib.DKV_BF16, at, q_st, q_sh, at << 1, at << 2, 4096,
                                       2048, 4, 16, at << 3, 4096, 4096, at << 3, at << 3, 1, T, hq, 2,
                                       128, T, 1, 65536, 0.1, None, 0, out, odt, o_st, o_sh)

    f32 = _lib.DKV_F32
    for args in ((at, 512, 128), (far, 512, 128), (far, 128, 512), (far, 512, 128, 512, 128, 4, 4, f32),
                 (far, 512, 128, 0, 0), (at, 1024, 128, 1024), (at + 1024, 1024, 128, 1024),
                 (at, 1024, 256, 1024, 256), (at + 256, 1024, 256, 1024, 256), (at, 128, 512, 128, 512),
                 (at + 4096, 512, 128), (at - 4096, 512, 128), (at, 77, 128, 96, 128, 1)):
        assert attend(*args) == WS, args
    for args in ((at + 16, 512, 128), (at + 256, 512, 128), (at + 1024, 512, 128), (at - 256, 512, 128),
                 (at, 512, 128, 512, 128, 4, 4, f32), (at, 1024, 128), (at, 128, 512),
                 (at + 1008, 1024, 128, 1024), (at, 512, 128, 0, 0), (at + 4080, 512, 128),
                 (far, 0, 128), (far, 256, 128), (far, 128, 256), (far, 504, 128)):
        assert attend(*args) == E, args


_RECORDER = r"""
#include <pthread.h>
#include <stddef.h>
#include <stdint.h>
#include <time.h>
typedef struct { uint32_t x, y, z; } dims;
static pthread_mutex_t lock = PTHREAD_MUTEX_INITIALIZER;
static const void* seen[4096];
static int n;
int hipGetLastError(void) { return 0; }
int __hipPushCallConfiguration(dims grid, dims block, size_t lds, void* stream) { return 0; }
int __hipPopCallConfiguration(dims* grid, dims* block, size_t* lds, void** stream) { return 0; }
/* a launch takes a millisecond; its first argument's first member, q, tells the call */
int hipLaunchKernel(const void* f, dims grid, dims block, void** args, size_t lds, void* stream) {
  pthread_mutex_lock(&lock);
  if (n < 4096) seen[n++] = *(const void**)args[0];
  pthread_mutex_unlock(&lock);
  struct timespec t = {0, 1000000};
  nanosleep(&t, 0);
  return 0;
}
int launches(const void** out) {
  for (int i = 0; i < n; ++i) out[i] = seen[i];
  return n;
}
"""

_THREADS = r"""
import ctypes, sys, threading
rec = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)  # found before the runtime's own
lib = ctypes.CDLL(sys.argv[2])
L, F = ctypes.c_longlong, ctypes.c_float
lib.dkv_paged_workspace_floats.restype = L
floats = lib.dkv_paged_workspace_floats(1, 64, 32, 8, 64, 64, 32768)
assert floats > 16384 and lib.dkv_paged_workspace_floats(1, 1, 32, 8, 1, 1, 32768) > 16384
P = ctypes.c_void_p

def calls(q, workspace, times, new):
    for _ in range(times):
        rc = lib.dkv_paged_attention(
            P(0), 2, P(q), L(4096), L(128), P(1 << 30), P(1 << 31), L(65536), L(8192), 1000, 64,
            P(1 << 20), L(512), 512, P(1 << 21), P(1 << 22), 1, new, 32, 8, 128, new, new, 32768, F(0.1),
            P(workspace), L(floats), P(1 << 23), 2, L(4096), L(128))
        assert rc == 0, rc

# threads on one stream share its workspace: 1 .. 3 make two launches a call, 4 and 5 one
threads = [threading.Thread(target=calls, args=((i + 1) << 32, 1 << 24, 8, 64 if i < 3 else 1))
           for i in range(5)]
for t in threads: t.start()
for t in threads: t.join()
seen = (P * 4096)()
n = rec.launches(seen)
assert n == 3 * 8 * 2 + 2 * 8, n
order = [(s or 0) >> 32 for s in seen[:n]]
i = 0
while i < n:
    two = order[i] <= 3
    assert not two or order[i] == order[i + 1], order
    i += 2 if two else 1
print("together")
"""


def test_launches_of_a_call_stay_together(tmp_path):
    """Calls of one stream share its workspace, from any thread: what a call's first launch leaves there
    its second one reads, so no other call's launch may come between them. Launches are recorded in place
    of being made, in a process of its own."""
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    (tmp_path / "rec.c").write_text(_RECORDER)
    rec = tmp_path / "librec.so"
    subprocess.run([cc, "-shared", "-fPIC", "-O1", str(tmp_path / "rec.c"), "-o", str(rec), "-lpthread"],
                   check=True)
    run = subprocess.run([sys.executable, "-c", _THREADS, str(rec), str(_lib.LIB_PATH)],
                         capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and "together" in run.stdout, run.stdout + run.stderr


class _Weights:
    """What a PagedLlama takes of a model before its first kernel."""

    shape = LlamaShape(hidden=256, layers=2, heads=2, kv_heads=2, head_dim=128, ffn=64, vocab=50)
    dtype, device = BF, torch.device("cpu")
    embed = torch.zeros(50, 256, dtype=BF)
    layers: list = []


def test_a_step_that_fails_changes_nothing():
    """Tokens that cannot be looked up (floats here): the requests have the lengths and pages they
    had, so that the step can be given again."""
    p = PagedLlama(_Weights(), pages=8, page_size=16)
    a, b = p.add(), p.add()
    p.cache.batch([(a, 20)])
    ids = p.cache.page_ids(a)
    for tokens in ([torch.zeros(5), torch.zeros(40)], [torch.zeros(5, dtype=torch.long), torch.ones(40)]):
        with pytest.raises(Exception):
            p.step([(a, tokens[0]), (b, tokens[1])])
        assert (p.cache.length(a), p.cache.length(b), p.cache.free_pages) == (20, 0, 6)
        assert p.cache.page_ids(a) == ids
    with pytest.raises(ValueError, match="no request"):
        p.step([(a, torch.zeros(1)), (9, torch.zeros(1))])
    with pytest.raises(ValueError, match="once"):
        p.step([(a, torch.zeros(1)), (a, torch.zeros(1))])
    with pytest.raises(RuntimeError, match="pages"):
        p.step([(a, torch.zeros(200))])
    assert (p.cache.length(a), p.cache.free_pages) == (20, 6)


def test_attention_scale_too_large_for_its_logarithm():
    """The scores are in units of log2: a scale whose product with log2(e) is past fp32 is refused (the
    call that is not is refused next, for its lack of a workspace)."""
    at = 1 << 32
    attend = lambda scale: _lib.load().dkv_paged_attention(  # noqa: E731
        None, _lib.DKV_BF16, at, 512, 128, at << 1, at << 2, 4096, 2048, 4, 16, at << 3, 4096, 4096,
        at << 3, at << 3, 1, 4, 4, 2, 128, 4, 1, 65536, scale, None, 0, at, _lib.DKV_BF16, 512, 128)
    assert attend(2.3e38) == _lib.DKV_E_WORKSPACE and attend(1e-30) == _lib.DKV_E_WORKSPACE
    assert attend(2.4e38) == _lib.DKV_E_UNSUPPORTED and attend(3.4e38) == _lib.DKV_E_UNSUPPORTED


def test_attention_workspace_alignment():
    """Records are read and written 8 and 16 bytes at a time: a workspace that is not aligned to 16 is
    refused (before one that is too small, as all of these are)."""
    at = 1 << 32
    attend = lambda ws: _lib.load().dkv_paged_attention(  # noqa: E731
        None, _lib.DKV_BF16, at, 512, 128, at << 1, at << 2, 4096, 2048, 4, 16, at << 3, 4096, 4096,
        at << 3, at << 3, 1, 4, 4, 2, 128, 4, 1, 65536, 0.1, ws, 0, at, _lib.DKV_BF16, 512, 128)
    assert attend(at) == _lib.DKV_E_WORKSPACE and attend(None) == _lib.DKV_E_WORKSPACE
    for off in (2, 4, 8):
        assert attend(at + off) == _lib.DKV_E_UNSUPPORTED
