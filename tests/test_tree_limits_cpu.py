"""Sizes whose products do not fit 32 bits, and missing arrays, are refused on the host, before any launch."""
import ctypes
import os

import pytest

from _util import LIB, G9AttnBatch, capi
from test_tree_cpu import INVALID, G9KvCache, batch, cache

pytestmark = pytest.mark.skipif(not os.path.exists(LIB), reason="library not built")


@pytest.mark.parametrize("mode", [0, 1, 2, 3])
@pytest.mark.parametrize("per", [1000, 2 ** 24, 2 ** 26, 2 ** 27, 2 ** 28, 2 ** 29, 2 ** 30, 2 ** 31 - 1, 0x0f0f0f0f, 0x1e1e1e1e])
def test_move_groups_that_no_shared_memory_holds(per, mode):
    """16 * per and per * (136 + V row) wrap to small or negative 32-bit numbers for some of these."""
    move = capi().gfx906_fa_move_kv
    i, p = ctypes.c_int, ctypes.c_void_p
    move.argtypes = [p, p, i, ctypes.POINTER(G9KvCache), p, p, i, i, p]
    one = (ctypes.c_void_p * 1)(1 << 20)
    c = cache(v_mode=mode, v_tok_stride=512)
    assert move(one, one, 1, ctypes.byref(c), 1 << 20, 1 << 20, 1, per, None) == INVALID


def test_counts_from_offsets_need_the_offsets():
    """G9_F_CU_SEQLENS takes a sequence's drafts from q_start, which must then be there."""
    run = capi().gfx906_fa_tree_attention
    run.argtypes = [ctypes.POINTER(G9AttnBatch), ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_void_p, ctypes.c_size_t,
                    ctypes.c_void_p]
    size = capi().gfx906_fa_tree_attention_workspace_size
    size.restype, size.argtypes = ctypes.c_size_t, [ctypes.POINTER(G9AttnBatch)]
    for over in (dict(), dict(block_size=8)):                  # either kernel
        b = batch(q_start=None, flags=1, **over)
        assert run(ctypes.byref(b), 1 << 24, 1, 1, 1 << 26, 1 << 40, None) == INVALID
        assert size(ctypes.byref(b)) == 0
    assert size(ctypes.byref(batch(q_start=None, flags=1, n_q=1 << 20))) > 0
    assert size(ctypes.byref(batch(q_start=None, flags=0))) > 0
