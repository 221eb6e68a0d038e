"""Host side of the serving operators: exported symbols, argument refusals (which come before the device is looked at)
and the tree masks."""
import ctypes
import math

import numpy as np
import pytest
import torch

import servref
from conftest import has_gpu
from kvc_b200 import attn, lib as kvclib, pages
from test_library_cpu import declared_functions


@pytest.mark.parametrize("header,listed", [("kvc-pages.h", "PAGES_SYMBOLS"), ("kvc-attn.h", "ATTN_SYMBOLS")])
def test_symbols(kvc, header, listed):
    names = declared_functions(header)
    assert sorted(getattr(kvclib, listed)) == names
    for n in names:
        assert hasattr(kvc["_lib"], n)


def cache_desc(**kw):
    """A description over host memory: enough for the checks, which read no device memory."""
    d = dict(n_layers=2, n_pages=8, page_size=16, n_slots=4, max_pages=4, n_head_kv=2, d_k=64, d_v=64, k_type=8, v_type=8,
             k_row_bytes=2 * 68, v_row_bytes=2 * 68)
    buf = (ctypes.c_uint8 * 65536)()
    at = (ctypes.addressof(buf) + 255) // 256 * 256
    for f in ("K", "V", "page_table", "seq_len", "ref_count", "status"):
        d[f] = at
    d["beta"] = None
    d.update(kw)
    c = pages.PageCacheDesc(**d)
    c._buf = buf
    return c


NODEV = -10


def ok_code():
    return 0 if has_gpu() else NODEV


BAD_CACHES = [
    (dict(K=None), -1), (dict(V=None), -1), (dict(page_table=None), -1), (dict(seq_len=None), -1),
    (dict(ref_count=None), -1), (dict(status=None), -1), (dict(n_layers=0), -2), (dict(n_pages=0), -2),
    (dict(page_size=0), -2), (dict(n_slots=-1), -2), (dict(max_pages=0), -2), (dict(n_head_kv=0), -2), (dict(d_k=0), -2),
    (dict(k_type=7), -2), (dict(v_type=30), -2), (dict(k_row_bytes=100), -4), (dict(v_row_bytes=2 * 68 + 34), -4),
    (dict(d_k=40), -4), (dict(n_pages=2 ** 30, page_size=4), -13), (dict(max_pages=2 ** 30, page_size=4), -13),
    (dict(n_layers=65536), -13),
]


@pytest.mark.parametrize("field", ["K", "V", "beta", "page_table", "seq_len", "ref_count", "status"])
def test_cache_arrays_off_their_elements(kvc, field):
    c = cache_desc(k_type=0, k_row_bytes=512, v_type=0, v_row_bytes=512)
    at = c.K
    setattr(c, field, at + 2)
    one = pages.ids([0])
    assert kvc["_lib"].kvc_pages_free(ctypes.addressof(c), one, 1, at, 1 << 20, None) == -13
    assert kvc["_lib"].kvc_pages_workspace(ctypes.addressof(c)) == 0


def test_call_arrays_off_their_elements(kvc):
    L, c = kvc["_lib"], cache_desc(beta=None)
    c.beta = c.K
    ref, at, odd, one = ctypes.addressof(c), c.K, c.K + 2, pages.ids([0])
    ws = (at, L.kvc_pages_workspace(ref))
    assert ws[1] > 0
    assert L.kvc_pages_copy(ref, odd, at, 1, None) == -13 and L.kvc_pages_copy(ref, at, odd, 1, None) == -13
    for call in (L.kvc_pages_write, L.kvc_pages_read):
        assert call(ref, one, one, pages.ids([1]), 1, None, None, odd, None) == -13
    good = dict(base=at, keep_n=at, keep=at, beta=at)
    for name in good:
        a = dict(good, **{name: odd})
        assert L.kvc_pages_compact(ref, one, one, 1, a["base"], a["keep_n"], a["keep"], 4, 0, None, a["beta"], *ws, None) == -13
    for name in ("lse", "cu", "seqs", "mask"):
        t = tree_desc(c, **{name: odd})
        assert L.kvc_attn_tree(ref, ctypes.addressof(t), None, 0, None) == -13
    for name in ("lse", "cu_q", "cu_k"):
        d = dict(q=4096, k=4096, v=4096, out=4096, lse=4096, cu_q=4096, cu_k=4096, type=1, n_seqs=1, total_q=4, total_k=4,
                 n_head=4, n_head_kv=2, d_k=64, d_v=64, causal=1, scale=0.1, q_stride=256, q_head_stride=64, k_stride=128,
                 k_head_stride=64, v_stride=128, v_head_stride=64)
        p = attn.PromptDesc(**dict(d, **{name: 4098}))
        assert L.kvc_attn_prompt(ctypes.addressof(p), None) == -13


@pytest.mark.parametrize("kw,code", BAD_CACHES)
def test_cache_refusals(kvc, kw, code):
    c, L = cache_desc(**kw), kvc["_lib"]
    ref = ctypes.addressof(c)
    assert L.kvc_pages_workspace(ref) == 0
    one = pages.ids([0])
    assert L.kvc_pages_free(ref, one, 1, None, 0, None) == code
    assert L.kvc_pages_copy(ref, None, None, 0, None) == code
    t = attn.TreeDesc()
    assert L.kvc_attn_tree(ref, ctypes.addressof(t), None, 0, None) == code


@pytest.mark.parametrize("kw", [dict(n_pages=2 ** 31 - 1, page_size=1), dict(max_pages=2 ** 31 - 1, page_size=1),
                                dict(n_pages=1, page_size=2 ** 31 - 1, max_pages=1)])
def test_cache_sizes_leave_room_for_a_step(kvc, kw):
    """Scans and grids step past the last page and row; their numbers are 32-bit."""
    c, L = cache_desc(**kw), kvc["_lib"]
    assert L.kvc_pages_free(ctypes.addressof(c), pages.ids([0]), 1, None, 0, None) == -13
    small = {k: v - 65536 if v > 1 else v for k, v in kw.items()}
    assert L.kvc_pages_free(ctypes.addressof(cache_desc(**small)), pages.ids([0]), 1, None, 0, None) == -1    # no workspace


def test_page_call_refusals(kvc):
    L, c = kvc["_lib"], cache_desc()
    ref = ctypes.addressof(c)
    size = L.kvc_pages_workspace(ref)
    assert size > 0
    ws = (c.K, size)
    ids = pages.ids
    fork = lambda s, d, n=None, w=ws: L.kvc_pages_fork(ref, s, d, len(s) if n is None else n, *w, None)  # noqa: E731
    assert fork(ids([0]), ids([0])) == -2                      # onto itself
    assert fork(ids([0, 0]), ids([1, 1])) == -2                # one destination twice
    assert fork(ids([0, 1]), ids([1, 2])) == -2                # a destination that is a source
    assert fork(ids([0]), ids([4])) == -2 and fork(ids([-1]), ids([1])) == -2
    assert fork(ids([0]), ids([1]), n=-1) == -2 and fork(ids([0]), ids([1]), n=257) == -2
    assert L.kvc_pages_fork(ref, None, None, 1, *ws, None) == -1
    assert fork(ids([0]), ids([1]), w=(None, size)) == -1
    assert fork(ids([0]), ids([1]), w=(c.K, size - 1)) == -13
    assert fork(ids([0]), ids([1]), w=(c.K + 4, size)) == -13
    assert L.kvc_pages_reserve(ref, ids([1, 1]), ids([1, 1]), 2, *ws, None) == -2
    assert L.kvc_pages_reserve(ref, ids([1]), ids([-1]), 1, *ws, None) == -2
    assert L.kvc_pages_reserve(ref, ids([1]), None, 1, *ws, None) == -1
    assert L.kvc_pages_free(ref, ids([2, 2]), 2, *ws, None) == -2
    comp = lambda s, d, b=c.K, k=c.K, i=c.K, ld=4, beta=None: L.kvc_pages_compact(  # noqa: E731
        ref, ids(s), ids(d), len(s), b, k, i, ld, 0, None, beta, *ws, None)
    assert comp([0, 1], [2, 2]) == -2 and comp([0], [9]) == -2 and comp([0], [0], ld=-1) == -2
    assert comp([0], [0], b=None) == -1 and comp([0], [0], k=None) == -1 and comp([0], [0], i=None) == -1
    assert comp([0], [0], beta=c.K) == -1                      # a cache without beta
    for call in (L.kvc_pages_write, L.kvc_pages_read):
        assert call(ref, ids([0]), ids([-1]), ids([1]), 1, None, None, None, None) == -2
        assert call(ref, ids([0]), ids([0]), ids([-1]), 1, None, None, None, None) == -2
        assert call(ref, ids([0]), ids([2 ** 31 - 1]), ids([1]), 1, None, None, None, None) == -2
        assert call(ref, ids([4]), ids([0]), ids([1]), 1, None, None, None, None) == -2
        assert call(ref, ids([0]), ids([0]), ids([1]), 1, None, None, c.K, None) == -1
    assert L.kvc_pages_write(ref, ids([0, 0]), ids([0, 3]), ids([4, 4]), 2, None, None, None, None) == -2   # one row twice
    assert L.kvc_pages_copy(ref, None, None, 1, None) == -1
    assert L.kvc_pages_copy(ref, None, None, -1, None) == -2
    assert fork(ids([]), ids([])) == ok_code()
    assert L.kvc_pages_copy(ref, None, None, 0, None) == ok_code()


def test_ids_are_ints():
    """Host lists of any integer type become C ints; only an array of these is passed on as it is."""
    given = (ctypes.c_int * 3)(1, 2, 3)
    assert pages.ids(given) is given
    for values in ([1, 2, 3], (ctypes.c_int64 * 3)(1, 2, 3), np.array([1, 2, 3]), torch.tensor([1, 2, 3]), (1, 2, 3)):
        got = pages.ids(values)
        assert isinstance(got, ctypes.Array) and got._type_ is ctypes.c_int and list(got) == [1, 2, 3]


def tree_desc(c, **kw):
    d = dict(q=c.K, out=c.K, lse=None, cu=c.K, seqs=c.K, mask=None, q_type=1, mask_words=0, n_seqs=1, total=1, max_nodes=1,
             n_head=4, layer=0, scale=0.1, q_stride=4 * 64)
    d.update(kw)
    return attn.TreeDesc(**d)


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), -1), (dict(out=None), -1), (dict(cu=None), -1), (dict(seqs=None), -1), (dict(n_seqs=-1), -2),
    (dict(total=-1), -2), (dict(max_nodes=-1), -2), (dict(n_head=3), -2), (dict(n_head=0), -2), (dict(layer=2), -2),
    (dict(layer=-1), -2), (dict(mask_words=-1), -2), (dict(q_type=8), -2), (dict(q_stride=255), -2),
    (dict(total=2 ** 30), -13),
])
def test_tree_refusals(kvc, kw, code):
    c = cache_desc()
    t = tree_desc(c, **kw)
    rc = ctypes.c_int(0)
    assert kvc["_lib"].kvc_attn_tree(ctypes.addressof(c), ctypes.addressof(t), None, 0, None) == code
    assert kvc["_lib"].kvc_attn_tree_workspace(ctypes.addressof(c), ctypes.addressof(t), ctypes.addressof(rc)) == 0
    assert rc.value == code


def test_tree_refuses_head_sizes(kvc):
    for kw in (dict(d_k=512, k_row_bytes=2 * 16 * 34), dict(n_head_kv=2, d_k=48, k_row_bytes=3 * 34)):
        c = cache_desc(**kw)                                   # beyond 256; heads that begin inside a block
        t = tree_desc(c, q_stride=4 * c.d_k)
        assert kvc["_lib"].kvc_attn_tree(ctypes.addressof(c), ctypes.addressof(t), None, 0, None) == -13
    assert kvc["_lib"].kvc_attn_tree(ctypes.addressof(cache_desc()), None, None, 0, None) == -1


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(out=None), -1), (dict(cu_q=None), -1),
    (dict(cu_k=None), -1), (dict(type=8), -2), (dict(n_seqs=-1), -2), (dict(total_q=-1), -2), (dict(total_k=-1), -2),
    (dict(n_head=3), -2), (dict(n_head=0), -2), (dict(n_head_kv=0), -2), (dict(d_k=0), -2), (dict(d_v=-8), -2),
    (dict(q_stride=-1), -2), (dict(v_head_stride=-64), -2), (dict(d_k=264), -13), (dict(d_v=300), -13), (dict(q=1), -13),
    (dict(total_q=2 ** 30), -13),
])
def test_prompt_refusals(kvc, kw, code):
    d = dict(q=4096, k=4096, v=4096, out=4096, lse=None, cu_q=4096, cu_k=4096, type=1, n_seqs=1, total_q=4, total_k=4,
             n_head=4, n_head_kv=2, d_k=64, d_v=64, causal=1, scale=0.1, q_stride=256, q_head_stride=64, k_stride=128,
             k_head_stride=64, v_stride=128, v_head_stride=64)
    d.update(kw)
    p = attn.PromptDesc(**d)
    assert kvc["_lib"].kvc_attn_prompt(ctypes.addressof(p), None) == code
    assert kvc["_lib"].kvc_attn_prompt(None, None) == -1


def test_tree_mask():
    m = attn.tree_mask([[-1, 0, 0, 2], [-1], [-1] + list(range(39))])
    assert m.shape == (45, 2)
    see = [[bool((int(m[i, j // 32]) >> (j % 32)) & 1) for j in range(64)] for i in range(45)]
    want = [{0}, {0, 1}, {0, 2}, {0, 2, 3}, {0}] + [set(range(i + 1)) for i in range(40)]
    assert [{j for j in range(64) if row[j]} for row in see] == want
    with pytest.raises(ValueError):
        attn.tree_mask([[-1, 1]])


def test_reference_formats_agree_with_the_codecs(kvc):
    """The tests' own decoding of stored rows is the library's."""
    from kvc_b200 import abi
    x = np.random.default_rng(1).standard_normal((6, 64)).astype(np.float32)
    for kind in (0, 1, 2, 3, 8):
        raw = abi.quantize_rows(kvc, x, kind)
        want = abi.dequantize_rows(kvc, raw, kind, 64)
        got = servref.decode(torch.from_numpy(raw), kind).float().numpy()
        np.testing.assert_allclose(got, want, rtol=2.0 ** -23, atol=0)
        raw = servref.encode(torch.from_numpy(x), kind)
        assert raw.shape[1] == servref.row_bytes(kind, 64)
        near = np.abs(abi.dequantize_rows(kvc, raw.numpy(), kind, 64) - x).max()
        assert near <= {0: 0, 1: 2 ** -9, 8: 0.05, 2: 0.6, 3: 0.4}[kind]


def test_reference_attention():
    q = torch.tensor([[1.0, 0.0]])
    K, V = torch.tensor([[0.0, 0.0], [1.0, 0.0]]).double(), torch.tensor([[2.0], [4.0]]).double()
    o, lse = servref.attend(q, K, V, None, torch.ones(1, 2, dtype=torch.bool), 1.0)
    assert abs(float(o) - (2 + 4 * math.e) / (1 + math.e)) < 1e-12 and abs(float(lse) - math.log(1 + math.e)) < 1e-12
    o, lse = servref.attend(q, K, V * math.nan, None, torch.zeros(1, 2, dtype=torch.bool), 1.0)
    assert float(o) == 0.0 and float(lse) == -math.inf
