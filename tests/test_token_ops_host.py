"""The operators on token ids, as far as the CPU can check them: what the C ABI refuses, the workspace sizes, and the paged
cache's arithmetic (the functions the kernels call, run one request after the other) against a plain statement of it."""
import ctypes as C
import random

import numpy as np
import pytest

from tests import token_ops_ref as ref
from tests.hostshim import HostShim
from tokenizer_amd import capi

_P, _I, _U, _Q = C.c_void_p, C.c_int, C.c_uint32, C.c_uint64


class EmbedArgs(C.Structure):
    _fields_ = [("ids", _P), ("n", _Q), ("n_dev", _P), ("table", _P), ("dtype", _I), ("rows", _Q), ("dim", _Q), ("stride", _Q), ("out", _P),
                ("out_dtype", _I), ("out_stride", _Q), ("scale", C.c_float)]


class GradArgs(C.Structure):
    _fields_ = [("ids", _P), ("n", _Q), ("n_dev", _P), ("grad", _P), ("dtype", _I), ("grad_stride", _Q), ("rows", _Q), ("dim", _Q), ("table", _P),
                ("table_dtype", _I), ("table_stride", _Q), ("scale", C.c_float), ("accumulate", _I), ("work", _P), ("work_bytes", _Q)]


class CacheArgs(C.Structure):
    _fields_ = [("off", _P), ("keep", _P), ("n", _Q), ("len", _P), ("held", _P), ("page", _U), ("n_pages", _U), ("table", _P),
                ("table_stride", _Q), ("max_pages", _Q), ("free_pages", _P), ("n_free", _P), ("len_out", _P), ("held_out", _P),
                ("n_free_out", _P), ("slots", _P), ("pos", _P), ("cap", _Q), ("status", _P), ("work", _P), ("work_bytes", _Q)]


class VerifyArgs(C.Structure):
    _fields_ = [("draft", _P), ("off", _P), ("n", _Q), ("n_draft", _Q), ("max_draft", _U), ("target", _P), ("dtype", _I), ("target_stride", _Q),
                ("q", _P), ("q_stride", _Q), ("vocab", _Q), ("u_accept", _P), ("u_draw", _P), ("out", _P), ("accepted", _P), ("work", _P),
                ("work_bytes", _Q)]


@pytest.fixture(scope="module")
def lib():
    L = HostShim().lib
    for f in ("embed", "embed_grad", "verify"):
        getattr(L, "l3t_check_" + f).restype = C.c_char_p
        getattr(L, "l3t_check_" + f).argtypes = [_P]
    L.l3t_check_cache.restype = C.c_char_p
    L.l3t_check_cache.argtypes = [_P, _I]
    for f, k in (("grad", 2), ("cache", 1), ("verify", 2)):
        getattr(L, "l3t_%s_work" % f).restype = _Q
        getattr(L, "l3t_%s_work" % f).argtypes = [_Q] * k
    L.l3t_cache_slots.argtypes = L.l3t_cache_trim.argtypes = [_P]
    L.l3t_cache_slots.restype = L.l3t_cache_trim.restype = None
    return L


# an address that is never read: the checks look at pointers only
AT = 0x10000

EMBED = dict(ids=AT, n=10, n_dev=None, table=AT, dtype=2, rows=100, dim=64, stride=64, out=AT, out_dtype=2, out_stride=64, scale=1.0)
GRAD = dict(ids=AT, n=10, n_dev=None, grad=AT, dtype=2, grad_stride=64, rows=100, dim=64, table=AT, table_dtype=0, table_stride=64, scale=1.0,
            accumulate=1, work=AT, work_bytes=1 << 30)
SLOTS = dict(off=AT, keep=None, n=4, len=AT, held=AT, page=16, n_pages=100, table=AT, table_stride=8, max_pages=8, free_pages=AT, n_free=AT,
             len_out=AT, held_out=AT, n_free_out=AT, slots=AT, pos=AT, cap=64, status=AT, work=AT, work_bytes=1 << 20)
TRIM = dict(SLOTS, off=None, keep=AT, slots=None, pos=None, cap=0)
VERIFY = dict(draft=AT, off=AT, n=4, n_draft=8, max_draft=4, target=AT, dtype=0, target_stride=1000, q=AT, q_stride=1000, vocab=1000, u_accept=AT,
              u_draw=AT, out=AT, accepted=AT, work=AT, work_bytes=1 << 20)


def _check(lib, kind, **change):
    cls, good, f = {"embed": (EmbedArgs, EMBED, lib.l3t_check_embed), "grad": (GradArgs, GRAD, lib.l3t_check_embed_grad),
                    "slots": (CacheArgs, SLOTS, lambda a: lib.l3t_check_cache(a, 0)), "trim": (CacheArgs, TRIM, lambda a: lib.l3t_check_cache(a, 1)),
                    "verify": (VerifyArgs, VERIFY, lib.l3t_check_verify)}[kind]
    return f(C.byref(cls(**dict(good, **change))))


ACCEPTED = [
    ("embed", {}), ("embed", dict(n=0, ids=None, table=None, out=None)), ("embed", dict(table=AT + 2, out=AT + 6, stride=65, out_stride=67)),
    ("embed", dict(n_dev=AT + 8, rows=2 ** 31 - 1, dim=1, stride=1, out_stride=1)), ("embed", dict(dim=1 << 24, stride=1 << 24, out_stride=1 << 24)),
    ("grad", {}), ("grad", dict(n=0, ids=None, grad=None, work=None, work_bytes=0, accumulate=0)), ("grad", dict(dtype=0, table_dtype=1)),
    ("slots", {}), ("slots", dict(n=0, len=None, held=None, table=None, len_out=None, held_out=None)), ("slots", dict(cap=0, slots=None, pos=None)),
    ("slots", dict(page=1)), ("slots", dict(page=12)),
    ("trim", {}), ("trim", dict(n=0, len=None, held=None, table=None, len_out=None, held_out=None, keep=None)),
    ("verify", {}), ("verify", dict(q=None, q_stride=0)), ("verify", dict(n=0, off=None, target=None, u_draw=None, out=None, accepted=None, work=None)),
    ("verify", dict(n_draft=0, draft=None, u_accept=None, max_draft=0)), ("verify", dict(dtype=2, target=AT + 2, q=AT + 2, target_stride=1001)),
]

REFUSED = [
    ("embed", dict(dtype=3), "type"), ("embed", dict(out_dtype=-1), "type"), ("embed", dict(n=2 ** 31), "split"), ("embed", dict(rows=0), "n_rows"),
    ("embed", dict(rows=2 ** 31), "n_rows"), ("embed", dict(dim=0), "dim"), ("embed", dict(dim=(1 << 24) + 1, stride=1 << 25, out_stride=1 << 25), "dim"),
    ("embed", dict(stride=63), "stride"), ("embed", dict(out_stride=63), "stride"), ("embed", dict(stride=2 ** 31), "stride"),
    ("embed", dict(ids=None), "null"), ("embed", dict(table=None), "null"), ("embed", dict(out=None), "null"), ("embed", dict(ids=AT + 2), "aligned"),
    ("embed", dict(n_dev=AT + 4), "aligned"), ("embed", dict(table=AT + 1), "aligned"), ("embed", dict(dtype=0, table=AT + 2), "aligned"),
    ("embed", dict(out_dtype=0, out=AT + 2), "aligned"),
    ("grad", dict(dtype=7), "type"), ("grad", dict(table_dtype=3), "type"), ("grad", dict(n=2 ** 24 + 1), "split"), ("grad", dict(rows=0), "n_rows"), ("grad", dict(rows=2 ** 28 + 1), "n_rows"),
    ("grad", dict(dim=0), "dim"), ("grad", dict(grad_stride=10), "stride"), ("grad", dict(table_stride=10), "stride"), ("grad", dict(accumulate=2), "accumulate"),
    ("grad", dict(table=None), "null"), ("grad", dict(ids=None), "null"), ("grad", dict(grad=None), "null"), ("grad", dict(work=None), "null"),
    ("grad", dict(table=AT + 2), "aligned"), ("grad", dict(grad=AT + 1), "aligned"), ("grad", dict(work=AT + 8), "16 bytes"),
    ("grad", dict(work_bytes=100), "too small"), ("grad", dict(n=0, table=None), "null"),
    ("slots", dict(n=(1 << 20) + 1), "split"), ("slots", dict(page=0), "page_size"), ("slots", dict(page=(1 << 20) + 1), "page_size"),
    ("slots", dict(n_pages=0), "n_pages"), ("slots", dict(n_pages=2 ** 31), "n_pages"), ("slots", dict(max_pages=0), "max_pages"),
    ("slots", dict(table_stride=7), "table_stride"), ("slots", dict(cap=2 ** 31), "cap"), ("slots", dict(slots=None), "null"), ("slots", dict(pos=None), "null"),
    ("slots", dict(slots=AT + 4), "aligned"), ("slots", dict(work_bytes=64), "too small"), ("slots", dict(work=AT + 4), "16 bytes"),
] + [(k, {f: None}, "null") for k in ("slots", "trim") for f in ("len", "held", "table", "free_pages", "n_free", "len_out", "held_out", "n_free_out",
                                                                "status", "work")] + [
    (k, {f: AT + 2}, "aligned") for k in ("slots", "trim") for f in ("len", "held", "table", "free_pages", "n_free", "len_out", "held_out", "n_free_out",
                                                                    "status")] + [
    ("slots", dict(off=None), "null"), ("slots", dict(off=AT + 4), "aligned"), ("trim", dict(keep=None), "null"), ("trim", dict(keep=AT + 1), "aligned"),
    ("slots", dict(off=None, n=0), "null"),
    ("verify", dict(dtype=3), "type"), ("verify", dict(n=(1 << 20) + 1), "split"), ("verify", dict(n_draft=2 ** 31), "split"),
    ("verify", dict(max_draft=65536), "max_draft"), ("verify", dict(vocab=0), "vocab"), ("verify", dict(target_stride=999), "stride"),
    ("verify", dict(q_stride=999), "stride"), ("verify", dict(dtype=0, target=AT + 2), "aligned"), ("verify", dict(q=AT + 1), "aligned"),
    ("verify", dict(work=AT + 8), "16 bytes"), ("verify", dict(work_bytes=32), "too small"),
] + [("verify", {f: None}, "null") for f in ("draft", "off", "target", "u_accept", "u_draw", "out", "accepted", "work")]


@pytest.mark.parametrize("kind, change", ACCEPTED)
def test_accepted(lib, kind, change):
    assert _check(lib, kind, **change) is None


@pytest.mark.parametrize("kind, change, word", REFUSED)
def test_refused(lib, kind, change, word):
    said = _check(lib, kind, **change)
    assert said and word in said.decode(), said


def test_null_context_is_refused():
    L = capi.load_library()
    assert L.l3_embed(None, None, 0, None, None, 0, 1, 1, 1, 1.0, None, 0, 1, None) == capi.L3_E_INVALID_ARG
    assert L.l3_embed_grad(None, None, 0, None, None, 0, 1, 1, 1, 1.0, None, 0, 1, 0, None, 0, None) == capi.L3_E_INVALID_ARG
    assert L.l3_cache_slots(None, *[None, 0, None, None, 1, 1, None, 1, 1] + [None] * 7 + [0, None, None, 0, None]) == capi.L3_E_INVALID_ARG
    assert L.l3_cache_trim(None, *[None, 0, None, None, 1, 1, None, 1, 1] + [None] * 7 + [0, None]) == capi.L3_E_INVALID_ARG
    assert L.l3_verify_draft(None, None, None, 0, 0, 0, None, 0, 1, None, 1, 1, None, None, None, None, None, 0, None) == capi.L3_E_INVALID_ARG


def test_workspace_sizes(lib):
    """The library's answers are the checks' own sizes; 0 stands for sizes that no call takes."""
    L = capi.load_library()
    for n, dim in ((0, 1), (1, 1), (64, 4096), (65536, 4096), (2 ** 24, 8)):
        assert L.l3_embed_grad_workspace(n, dim) == lib.l3t_grad_work(n, dim) > 0
        need = lib.l3t_grad_work(n, dim)
        assert _check(lib, "grad", n=n, dim=dim, grad_stride=dim, table_stride=dim, work_bytes=need) is None
        if n:
            assert _check(lib, "grad", n=n, dim=dim, grad_stride=dim, table_stride=dim, work_bytes=need - 1)
    for n in (0, 1, 1024, 1 << 20):
        assert L.l3_cache_workspace(n) == lib.l3t_cache_work(n) > 0
    for n, v in ((0, 5), (1, 1), (3, 128256)):
        assert L.l3_verify_workspace(n, v) == lib.l3t_verify_work(n, v) > 0
    assert L.l3_embed_grad_workspace(2 ** 24 + 1, 8) == 0 == L.l3_cache_workspace(2 ** 20 + 1) == L.l3_verify_workspace(1, 2 ** 31)
    with pytest.raises(capi.L3Error):
        capi.cache_workspace(2 ** 20 + 1)


def test_a_workspace_for_the_largest_batch_is_enough_for_all(lib):
    """Sizes never shrink as n or dim grow (a smaller batch on the largest one's workspace must not be refused), and hold what the
    kernels lay out in them."""
    lib.l3t_grad_pieces.restype, lib.l3t_grad_pieces.argtypes = None, [_Q, _Q, _P]
    rng = random.Random(2)
    edges = {m + d for m in (512, 1024, 2048, 4096, 4600, 8192, 18400, 18432, 36864, 65536, 69632, 135168, 262144, 1 << 20, 1 << 24) for d in (-1, 0, 1)}
    # (where the chunk changes: n * ceil(dim / 512) at 9, 17 and 33 times 4,096)
    edges |= {-(-k * 4096 // t) + d for k in (9, 17, 33) for t in range(1, 34) for d in (-1, 0, 1)}
    ns = sorted({n for n in edges | set(range(0, 3000, 37)) | {int(10 ** rng.uniform(0, 7.22)) for _ in range(300)} if 0 <= n <= 1 << 24})
    dims = sorted({1, 7, 8, 9, 64, 511, 512, 513, 1001, 1024, 1025, 2048, 4095, 4096, 4097, 8192, 16000, 65536, 1 << 20, 1 << 24})
    pieces = np.zeros(4, np.uint64)
    below = [0] * len(ns)
    for dim in dims:
        size = [lib.l3t_grad_work(n, dim) for n in ns]
        assert all(a <= b for a, b in zip(size, size[1:])), dim
        assert all(a <= b for a, b in zip(below, size)), dim
        below = size
        for n in ns:
            lib.l3t_grad_pieces(n, dim, pieces.ctypes.data)
            assert pieces[0] <= pieces[1] and pieces[2] <= pieces[3] == lib.l3t_grad_work(n, dim), (n, dim)
    for n, dim in ((4600, 4096), (18400, 1024), (65536, 64), (262144, 64), (512, 2048)):
        assert _check(lib, "grad", n=n, dim=dim, grad_stride=dim, table_stride=dim, work_bytes=lib.l3t_grad_work(2 * n, dim)) is None
    ns = sorted({int(2 ** rng.uniform(0, 20)) for _ in range(500)} | {0, 1, 1023, 1024, 1025, 1 << 20})
    size = [lib.l3t_cache_work(n) for n in ns]
    assert all(a <= b for a, b in zip(size, size[1:]))
    below = [0] * len(ns)
    for vocab in (1, 2047, 2048, 2049, 128256, 2 ** 31 - 1):
        size = [lib.l3t_verify_work(n, vocab) for n in ns]
        assert all(a <= b for a, b in zip(size, size[1:])) and all(a <= b for a, b in zip(below, size))
        below = size


# ---- error texts --------------------------------------------------------------------------------------------------
@pytest.fixture
def texts(lib):
    """make() -> (assign(text), leave(what, more), text()) of a context's error texts"""
    lib.l3t_err_new.restype, lib.l3t_err_delete.argtypes = _P, [_P]
    lib.l3t_err_assign.argtypes, lib.l3t_err_leave.argtypes = [_P, C.c_char_p], [_P, C.c_char_p, C.c_char_p]
    lib.l3t_err_text.restype, lib.l3t_err_text.argtypes = _P, [_P]
    made = []

    def make():
        e = lib.l3t_err_new()
        made.append(e)
        return lambda t: lib.l3t_err_assign(e, t), lambda w, m=b"": lib.l3t_err_leave(e, w, m), lambda: C.string_at(lib.l3t_err_text(e)), e
    yield make
    for e in made:
        lib.l3t_err_delete(e)


def test_error_texts_of_one_thread(lib, texts):
    """The last error of the thread's own calls, whatever kind of call it was; nothing that was handed out changes."""
    assign, leave, text, e = texts()
    assign2, leave2, text2, _ = texts()
    assert text() == text2() == b""
    assign(b"encode")
    assert text() == b"encode"
    first = lib.l3t_err_text(e)
    leave(b"launch: ", b"reason")
    leave2(b"other")
    assert text() == b"launch: reason" and text2() == b"other"
    leave(b"again")
    assert text() == b"again"
    for i in range(3000):
        assign(b"encode %d" % (i % 50))
    assert text() == b"encode 49" and text2() == b"other" and C.string_at(first) == b"encode"
    assign2(b"")
    assert text2() == b""


def test_error_texts_of_many_contexts(lib, texts):
    """A thread has the texts of as many contexts at once as one handle over several GPUs has."""
    all_of = [texts() for _ in range(64)]
    for turn in range(3):
        for i, (_, leave, _, _) in enumerate(all_of):
            leave(b"%d of " % i, b"%d" % turn)
        assert [t() for _, _, t, _ in all_of] == [b"%d of %d" % (i, turn) for i in range(64)]
    assign, leave, text, _ = texts()
    leave(b"one more")
    assert text() == b"one more" and sum(t() == b"" for _, _, t, _ in all_of) == 1
    all_of[5][0](b"encode")
    assert all_of[5][2]() == b"encode" and text() == b"one more"


def test_error_texts_of_a_context_are_not_the_next_ones(lib, texts):
    """A context that comes to lie where one was destroyed has none of its texts."""
    for _ in range(200):
        e = lib.l3t_err_new()
        assert C.string_at(lib.l3t_err_text(_P(e))) == b""
        lib.l3t_err_leave(_P(e), b"gone", b"")
        lib.l3t_err_delete(_P(e))


def test_error_texts_of_threads_that_fail_at_the_same_time(lib, texts):
    """Operators that are refused on several threads of one context while encode calls fail on another: everyone reads their own."""
    import threading
    assign, leave, text, e = texts()
    wrong, stop = [], threading.Event()

    def refused(k):
        for i in range(4000):
            mine = b"thread %d, call %d " % (k, i % 7) + b"x" * (20 * k)
            leave(b"", mine)
            if text() != mine:
                wrong.append((k, i))

    def encodes():
        i = 0
        while not stop.is_set():
            i += 1
            assign(b"batch %d: too large" % (i % 5))
            if not text().startswith(b"batch"):
                wrong.append(("encode", i))

    threads = [threading.Thread(target=refused, args=(k,)) for k in range(4)]
    side = threading.Thread(target=encodes)
    side.start()
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    stop.set()
    side.join()
    assert not wrong, wrong[:5]
    assert text().startswith(b"batch")        # this thread had no refused call


# ---- the paged cache ----------------------------------------------------------------------------------------------
def random_cache(rng, n, page, max_pages, n_pages, full=0.5):
    """A sane state: (length, held, table, free, n_free); entries that mean nothing hold -5."""
    pages = list(range(n_pages))
    rng.shuffle(pages)
    length, held, table = [], [], []
    for _ in range(n):
        h = min(rng.randint(0, max_pages), int(len(pages) * full))
        mine = [pages.pop() for _ in range(h)]
        held.append(h)
        # some hold more pages than their tokens need, as after a trim that kept none of the drafted tokens' pages back
        length.append(rng.randint(0, h * page))
        table.append(mine + [-5] * (max_pages - h))
    return length, held, table, pages + [-5] * (n_pages - len(pages)), len(pages)


def _run_host(lib, state, kind, arg, cap=0):
    length, held, table, free, n_free, page, n_pages, max_pages = state
    n = len(length)
    L, H = np.array(length, np.int32), np.array(held, np.int32)
    T = np.array(table, np.int32).reshape(n, max_pages)
    F, N = np.array(free, np.int32), np.array([n_free], np.int32)
    slots, pos, status = np.full(cap + 1, -7, np.int64), np.full(cap + 1, -7, np.int32), np.full(1, 77, np.uint32)
    A = np.array(arg, np.uint64 if kind == "slots" else np.int32)
    args = CacheArgs(off=A.ctypes.data if kind == "slots" else None, keep=A.ctypes.data if kind == "trim" else None, n=n, len=L.ctypes.data,
                     held=H.ctypes.data, page=page, n_pages=n_pages, table=T.ctypes.data, table_stride=max_pages, max_pages=max_pages,
                     free_pages=F.ctypes.data, n_free=N.ctypes.data, len_out=L.ctypes.data, held_out=H.ctypes.data, n_free_out=N.ctypes.data,
                     slots=slots.ctypes.data, pos=pos.ctypes.data, cap=cap, status=status.ctypes.data, work=AT, work_bytes=1 << 40)
    (lib.l3t_cache_slots if kind == "slots" else lib.l3t_cache_trim)(C.byref(args))
    return L.tolist(), H.tolist(), T.tolist(), F.tolist(), int(N[0]), slots.tolist(), pos.tolist(), int(status[0])


@pytest.mark.parametrize("seed", range(40))
def test_cache_arithmetic(lib, seed):
    rng = random.Random(seed)
    page, max_pages, n = rng.choice([1, 2, 3, 16, 17]), rng.randint(1, 9), rng.randint(1, 12)
    n_pages = rng.randint(1, 40)
    length, held, table, free, n_free = random_cache(rng, n, page, max_pages, n_pages)
    if rng.random() < 0.3:      # requests and counts that cannot be, pages outside the pool
        i = rng.randrange(n)
        length[i], held[i] = rng.choice([(-1, 0), (5, -1), (held[i] * page + 1, held[i]), (0, max_pages + 1)])
    if rng.random() < 0.3:
        n_free = rng.choice([-1, n_pages + 1, n_free // 2])
    if rng.random() < 0.3:
        free[rng.randrange(n_pages)] = rng.choice([-1, n_pages, 2 ** 31 - 1])
    new = [rng.choice([0, 1, 1, rng.randint(0, 3 * page)]) for _ in range(n)]
    off = [0] + np.cumsum(new).tolist()
    cap = off[-1] + rng.randint(-2, 3) if off[-1] > 2 else off[-1]
    if rng.random() < 0.2 and n > 1:
        off[rng.randrange(1, n)] = 0 if rng.random() < 0.5 else off[-1] + 5
        off[-1] = max(off)
    state = (length, held, table, free, n_free, page, n_pages, max_pages)
    model = ref.Cache(*state)
    slots, pos = [-7] * (cap + 1), [-7] * (cap + 1)
    status = model.slots(off, cap, slots, pos)
    got = _run_host(lib, state, "slots", off, cap)
    assert got == (model.length, model.held, model.table, model.free, model.n_free, slots, pos, status)
    keep = [rng.choice([-1, 0, rng.randint(0, max(0, L)), max(0, L), max(0, L) + 5, max(0, L - 1)]) for L in model.length]
    if rng.random() < 0.2:
        model.n_free = min(n_pages, max(0, model.n_free) + rng.randint(0, 10))     # a pool that is too full
    state = (list(model.length), list(model.held), [list(r) for r in model.table], list(model.free), model.n_free, page, n_pages, max_pages)
    status = model.trim(keep)
    got = _run_host(lib, state, "trim", keep)
    assert got[:5] == (model.length, model.held, model.table, model.free, model.n_free) and got[7] == status


class PlanRec(C.Structure):
    _fields_ = [("before", _Q), ("len", C.c_int32), ("held", C.c_int32), ("delta", C.c_int32), ("new_len", C.c_int32), ("flags", _U), ("pad", _U)]


class Owner(C.Structure):
    _fields_ = [("first", _U), ("end", _U), ("next", _U), ("len", C.c_int32), ("held", C.c_int32)]


@pytest.mark.parametrize("seed", range(12))
def test_records_of_another_call_lead_nowhere(lib, seed):
    """Whatever a workspace holds that another call has written over, and whatever offsets stand beside it: what is served lies inside the
    table and the pool.  Numbers near the borders of the sizes and of the types, all of them mixed."""
    for f in ("slots", "trim"):
        getattr(lib, "l3t_%s_served_within" % f).argtypes = [_P, _P, _Q, _Q]
    lib.l3t_owner_of.restype, lib.l3t_owner_of.argtypes = None, [_P, _P, _Q, _Q, _Q, _Q, _P]
    rng = random.Random(seed)
    served = [0, 0, 0]
    for _ in range(30000):
        page, max_pages, n_pages = rng.choice([1, 3, 16, 1 << 20]), rng.choice([1, 5, 4096, 2 ** 31 - 1]), rng.choice([1, 40, 2 ** 20, 2 ** 31 - 1])
        near = lambda *of: max(0, rng.choice(of) + rng.choice([-1, 0, 0, 1, 2])) % 2 ** 64  # noqa: E731
        i32 = lambda *of: max(-2 ** 31, min(2 ** 31 - 1, rng.choice(of) + rng.choice([-1, 0, 0, 1])))  # noqa: E731
        A = CacheArgs(n=3, page=page, n_pages=n_pages, max_pages=max_pages, table_stride=max_pages, cap=100)
        held = i32(0, 0, 1, max_pages, 2 ** 31 - 1, -2 ** 31)
        r = PlanRec(len=i32(0, 5, min(2 ** 31 - 1, max(held, 0) * page), 2 ** 31 - 1, -7), held=held, delta=i32(0, 0, 1, 3, held, max_pages - max(held, 0), n_pages, -4),
                    flags=rng.choice([0, 0, 0, 0, 4, 2 ** 31]))
        left = near(0, n_pages, n_pages // 2, n_pages, 2 ** 63)
        before = near(0, 0, left, left - max(r.delta, 0), n_pages - left - max(r.delta, 0), 2 ** 64 - max(r.delta, 0) - 1, 2 ** 64 - 1)
        if lib.l3t_trim_served_within(C.byref(A), C.byref(r), before, left) and r.delta:
            served[0] += 1
            assert 0 < r.delta <= r.held <= max_pages and left + before + r.delta <= n_pages
        if lib.l3t_slots_served_within(C.byref(A), C.byref(r), before, left):
            served[1] += 1
            assert 0 <= r.held <= r.held + r.delta <= max_pages and r.delta >= 0
            assert r.delta == 0 or before + r.delta <= left <= n_pages
        first = near(0, 7, 99, 2 ** 32, 2 ** 63)
        end = near(first, first + 1, first + page * max(r.delta, 0), first + page * (max(r.held, 0) + max(r.delta, 0)) - max(r.len, 0), 0, 2 ** 64 - 1,
                   first + 2 ** 64 - max(r.len, 0))
        w = Owner()
        lib.l3t_owner_of(C.byref(A), C.byref(r), first, end, before, left, C.byref(w))
        if w.held >= 0 and w.first < w.end:
            served[2] += 1
            for t in (w.first, w.end - 1):
                q = w.len + t - w.first
                assert 0 <= q < 2 ** 31 and q // page < r.held + r.delta <= max_pages, (r.len, r.held, r.delta, first, end)
                fresh = q // page - r.held
                assert fresh < 0 or 0 <= w.next - 1 - fresh < n_pages
    assert min(served) > 100, served


class Verdict(C.Structure):
    _fields_ = [("state", C.c_int32), ("a", _U), ("p_row", _Q), ("q_row", _Q), ("token", C.c_int32), ("pad", C.c_int32)]


def test_verdicts_of_another_call_lead_nowhere(lib):
    A = VerifyArgs(n=3, n_draft=10, max_draft=4)
    for state in (1, 2, 3, -1):
        for a in (0, 4, 5, 2 ** 32 - 1):
            for p in (0, 12, 13, 2 ** 64 - 1):
                for q in (0, 9, 10, 2 ** 64 - 1):
                    got = lib.l3t_verdict_within(C.byref(A), C.byref(Verdict(state=state, a=a, p_row=p, q_row=q, token=7)))
                    assert bool(got) == (a <= 4 and p < 13 and (state != 2 or q < 10))


def test_division_by_the_page_size(lib):
    """The product that stands for x / page, next to multiples of every page size up to 600 and of others up to 2^20."""
    lib.l3t_page_div.restype, lib.l3t_page_div.argtypes = _U, [_U, _U]
    rng = random.Random(1)
    for page in [*range(1, 600), 1023, 1024, 1025, 65535, 65536, 65537, (1 << 20) - 1, 1 << 20] + [rng.randint(600, 1 << 20) for _ in range(200)]:
        top = (2 ** 31 - 1) // page
        for k in {0, 1, 2, top // 3, top - 1, top, rng.randint(0, top)}:
            for x in (k * page - 1, k * page, k * page + 1, 2 ** 31 - 1):
                if 0 <= x < 2 ** 31:
                    assert lib.l3t_page_div(x, page) == x // page, (x, page)


def test_positions_end_at_31_bits(lib):
    """A request that would pass 2^31 - 1 tokens is not served, whatever max_pages allows."""
    page, max_pages = 1 << 20, 4096
    table = [[0] * 2048 + [-5] * 2048]
    state = ([(1 << 31) - 2], [2048], table, [1, 2], 2, page, 4096, max_pages)
    one = _run_host(lib, state, "slots", [0, 1], 1)
    assert one[0] == [(1 << 31) - 1] and one[6][0] == (1 << 31) - 2 and one[5][0] == (1 << 20) - 2 and one[7] == 0
    two = _run_host(lib, state, "slots", [0, 2], 2)
    assert two[0] == [(1 << 31) - 2] and two[5][:2] == [-1, -1] and two[7] == ref.ROW
