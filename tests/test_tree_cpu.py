"""Argument checks of the draft-tree C entries (they run on the host before any launch) and the operators' presence."""
import ctypes
import os

import pytest

from _util import LIB, ROOT, G9AttnBatch, capi

pytestmark = pytest.mark.skipif(not os.path.exists(LIB), reason="library not built")
INVALID = 1


class G9KvCache(ctypes.Structure):
    _fields_ = [("k", ctypes.c_void_p), ("k_page_stride", ctypes.c_int64), ("k_tok_stride", ctypes.c_int64),
                ("k_head_stride", ctypes.c_int64), ("v", ctypes.c_void_p), ("v_page_stride", ctypes.c_int64),
                ("v_tok_stride", ctypes.c_int64), ("v_head_stride", ctypes.c_int64), ("v_mode", ctypes.c_int),
                ("num_blocks", ctypes.c_int), ("block_size", ctypes.c_int), ("num_heads_kv", ctypes.c_int)]


def cache(**over):
    c = G9KvCache(k=1 << 20, k_page_stride=16 * 2 * 136, k_tok_stride=2 * 136, k_head_stride=136, v=2 << 20,
                  v_page_stride=16 * 2 * 136, v_tok_stride=0, v_head_stride=16 * 136, v_mode=3, num_blocks=8, block_size=16,
                  num_heads_kv=2)
    for k, v in over.items():
        setattr(c, k, v)
    return c


def batch(**over):
    b = G9AttnBatch()
    b.q, b.q_dtype, b.q_tok_stride, b.q_head_stride = 1 << 20, 1, 6 * 128, 128
    b.q_start, b.seq_q, b.out, b.out_dtype = 2 << 20, 4, 3 << 20, 1
    b.o_tok_stride, b.o_head_stride = 6 * 128, 128
    b.k_cache, b.k_page_stride, b.k_tok_stride, b.k_head_stride = 4 << 20, 16 * 2 * 136, 2 * 136, 136
    b.v_cache, b.v_page_stride, b.v_tok_stride, b.v_head_stride = 5 << 20, 16 * 2 * 136, 0, 16 * 136
    b.v_fmt, b.block_table, b.max_blocks, b.block_size = 3, 6 << 20, 4, 16
    b.kv_len, b.max_kv, b.num_seqs, b.num_heads_q, b.num_heads_kv, b.head_dim = 7 << 20, 64, 2, 6, 2, 128
    b.scale, b.num_blocks, b.flags = 0.1, 8, 1
    for k, v in over.items():
        setattr(b, k, v)
    return b


def test_tree_attention_refuses_bad_batches():
    lib = capi()
    size = lib.gfx906_fa_tree_attention_workspace_size
    size.restype, size.argtypes = ctypes.c_size_t, [ctypes.POINTER(G9AttnBatch)]
    run = lib.gfx906_fa_tree_attention
    run.argtypes = [ctypes.POINTER(G9AttnBatch), ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_void_p, ctypes.c_size_t,
                    ctypes.c_void_p]

    def call(b, mask=1 << 24, words=1, ws=1 << 26, n=1 << 40):
        return run(ctypes.byref(b), mask, words, words, ws, n, None)

    assert size(ctypes.byref(batch())) > 0
    assert size(ctypes.byref(batch(block_size=8))) == 0            # the row kernel needs no workspace
    assert size(ctypes.byref(batch(k_tok_stride=2 * 136 + 2))) == 0
    for over in (dict(head_dim=64), dict(num_heads_q=5), dict(num_heads_kv=0), dict(block_size=0), dict(q_dtype=3),
                 dict(out_dtype=4), dict(out_dtype=3), dict(v_fmt=4), dict(q_abs=1 << 20), dict(mask=1 << 20), dict(flags=3),
                 dict(k_cache=(4 << 20) + 1), dict(v_head_stride=16 * 136 + 1), dict(out=(3 << 20) + 2), dict(o_tok_stride=769),
                 dict(num_seqs=-1), dict(seq_q=-1), dict(max_kv=-1)):
        assert call(batch(**over)) == INVALID, over
    assert call(batch(), words=0) == INVALID
    assert call(batch(), mask=None) == INVALID
    assert call(batch(kv_len=None)) == INVALID
    assert call(batch(), ws=None) == INVALID
    assert call(batch(), n=64) == INVALID
    assert call(batch(num_seqs=0)) == 0 and call(batch(seq_q=0)) == 0


def test_kv_entries_refuse_bad_arguments():
    lib = capi()
    i64, p, i = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int
    mask = lib.gfx906_fa_tree_mask
    mask.argtypes = [p, p, p, i, i, i, p, p, p]
    ok = [1 << 20, 1 << 20, 1 << 20, 2, 4, 1, 1 << 20, 1 << 20, None]
    for at, bad in ((0, None), (1, None), (2, None), (3, -1), (3, 0), (4, -1), (5, 0), (6, None)):
        a = list(ok)
        a[at] = bad
        assert mask(*a) == INVALID, at
    assert mask(None, None, None, 0, 0, 1, None, None, None) == 0

    read = lib.gfx906_fa_read_kv
    read.argtypes = [ctypes.POINTER(G9KvCache), i, p, i, p, p, i, p]
    for c in (cache(k=None), cache(block_size=0), cache(num_heads_kv=0), cache(k_tok_stride=273), cache(v=None), cache(v_mode=4),
              cache(v_head_stride=2177)):
        assert read(ctypes.byref(c), 0, 1 << 20, 4, 1 << 20, 1 << 20, 1, None) == INVALID
    assert read(ctypes.byref(cache()), 0, None, 4, 1 << 20, 1 << 20, 1, None) == INVALID
    assert read(ctypes.byref(cache()), 0, 1 << 20, 4, (1 << 20) + 8, 1 << 20, 1, None) == INVALID
    assert read(ctypes.byref(cache()), 0, 1 << 20, 4, 1 << 20, 1 << 20, 3, None) == INVALID
    assert read(ctypes.byref(cache(v_mode=0)), 0, 1 << 20, 4, 1 << 20, 1 << 20, 1, None) == INVALID
    assert read(ctypes.byref(cache()), 0, None, 0, None, None, 1, None) == 0

    move = lib.gfx906_fa_move_kv
    move.argtypes = [p, p, i, ctypes.POINTER(G9KvCache), p, p, i, i, p]
    one = (ctypes.c_void_p * 1)(1 << 20)
    odd = (ctypes.c_void_p * 1)((1 << 20) + 1)
    null = (ctypes.c_void_p * 1)(None)
    args = lambda k=one, v=one, c=None, s=1 << 20, g=2, n=3: (k, v, 1, ctypes.byref(c or cache()), s, 1 << 20, g, n, None)  # noqa: E731
    for a in (args(k=odd), args(v=odd), args(k=null), args(v=None), args(s=None), args(n=900), args(g=-1), args(c=cache(num_blocks=0)),
              args(c=cache(v_head_stride=2177)), args(c=cache(v_mode=7))):
        assert move(*a) == INVALID
    assert move(*args(g=0)) == 0

    pages = lib.gfx906_fa_copy_pages
    pages.argtypes = [p, i, i64, i64, i64, p, p, i, p]
    for a in ((one, 1, 8, 4096, 4095, 1 << 20, 1 << 20, 2), (odd, 1, 8, 4096, 4096, 1 << 20, 1 << 20, 2),
              (null, 1, 8, 4096, 4096, 1 << 20, 1 << 20, 2), (one, 1, 8, 4096, 4096, None, 1 << 20, 2),
              (one, 1, 8, 4096, -2, 1 << 20, 1 << 20, 2), (one, -1, 8, 4096, 4096, 1 << 20, 1 << 20, 2)):
        assert pages(*a, None) == INVALID, a
    assert pages(one, 1, 8, 4096, 4096, None, None, 0, None) == 0

    store = lib.gfx906_fa_norm_rope_store_kv
    f = ctypes.c_float
    store.argtypes = [p, i, i64, i64, i, p, i, i64, i64, p, i, i64, i64, p, i, p, i, f, p, p, i, i, i64, i, p, ctypes.POINTER(G9KvCache),
                      p, i64, i64, p, i64, i64, i, p]
    base = dict(q=1 << 20, qdt=1, qt=768, qh=128, hq=6, k=1 << 20, kdt=1, kt=256, kh=128, v=1 << 20, vdt=1, vt=256, vh=128, qw=None, qwd=0,
                kw=None, kwd=0, eps=1e-6, pos=1 << 20, cs=1 << 20, csd=2, rot=128, mp=100, neox=1, slots=1 << 20, c=cache(),
                qo=1 << 20, qot=768, qoh=128, ko=None, kot=0, koh=0, n=4)
    for over in (dict(k=None), dict(pos=None), dict(cs=None), dict(slots=None), dict(rot=24), dict(rot=144), dict(rot=0), dict(mp=0),
                 dict(kdt=3), dict(csd=-1), dict(hq=0), dict(qo=None), dict(v=None), dict(n=-1), dict(c=cache(k=None)),
                 dict(c=cache(v_mode=1), vdt=2)):
        a = {**base, **over}
        a["c"] = ctypes.byref(a["c"])
        assert store(*a.values(), None) == INVALID, over
    a = {**base, "n": 0, "c": ctypes.byref(base["c"])}
    assert store(*a.values(), None) == 0


def test_operators_are_exposed():
    if not os.path.exists(os.path.join(ROOT, "gfx906-fa-vllm_b200", "gfx906_fa.so")):
        pytest.skip("extension not built")
    import gfx906_fa
    for name in ("tree_mask", "norm_rope_store_kv", "read_kv", "tree_attention", "move_kv", "copy_pages"):
        assert gfx906_fa.__dict__[name].__doc__
