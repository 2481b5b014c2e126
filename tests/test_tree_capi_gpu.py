"""The draft-tree C entries called as a C program calls them: forms that the torch operators do not use."""
import ctypes

import numpy as np
import pytest
import torch

from _tree import dequant_rows
from _util import capi
from test_tree_cpu import G9KvCache

pytestmark = pytest.mark.gpu
dev = "cuda"
D, BS, F32 = 128, 16, 2


def q8_cache(NB, Hkv, bs, seed):
    """Random whole numbers under scales of either sign of exponent: K rows [NB, bs, Hkv, 136]."""
    rng = np.random.default_rng(seed)
    rows = rng.integers(0, 256, (NB, bs, Hkv, 4, 34), dtype=np.uint8)
    rows[..., :2] = rng.uniform(1e-4, 4, (NB, bs, Hkv, 4, 1)).astype(np.float16).view(np.uint8)
    return rows.reshape(NB, bs, Hkv, 136)


@pytest.mark.parametrize("mode", [0, 1, 2, 3])
@pytest.mark.parametrize("N,Hkv", [(1, 1), (3, 1), (8, 1), (3, 2), (61, 3), (64, 8)])
def test_read_kv_of_keys_alone(N, Hkv, mode):
    """value_out NULL: keys only, whatever the number of rows and whatever the cache holds of V (with mode 0: nothing)."""
    NB = -(-N // BS) + 1
    rows = q8_cache(NB, Hkv, BS, N + Hkv)
    kc = torch.from_numpy(rows).to(dev)
    vc = torch.zeros((NB, BS, Hkv, 256), dtype=torch.uint8, device=dev)        # room for every layout
    vrow = {0: 0, 1: 256, 2: 136, 3: 136}[mode]
    c = G9KvCache(k=kc.data_ptr(), k_page_stride=BS * Hkv * 136, k_tok_stride=Hkv * 136, k_head_stride=136,
                  v=vc.data_ptr() if mode else None, v_page_stride=BS * Hkv * vrow, v_tok_stride=0 if mode == 3 else Hkv * vrow,
                  v_head_stride=BS * 136 if mode == 3 else vrow, v_mode=mode, num_blocks=NB, block_size=BS, num_heads_kv=Hkv)
    slots = torch.randperm(NB * BS, generator=torch.Generator().manual_seed(N))[:N]
    out = torch.full((N + 4, Hkv, D), 7.0, device=dev)
    read = capi().gfx906_fa_read_kv
    read.argtypes = [ctypes.POINTER(G9KvCache), ctypes.c_int, ctypes.c_void_p, ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p,
                     ctypes.c_int, ctypes.c_void_p]
    on_gpu = slots.to(dev)
    assert read(ctypes.byref(c), 1, on_gpu.data_ptr(), N, out.data_ptr(), None, F32, torch.cuda.current_stream().cuda_stream) == 0
    got = out.cpu().numpy()
    want = dequant_rows(rows.reshape(NB * BS, Hkv, 136)[slots.numpy()]).astype(np.float32)
    assert np.array_equal(got[:N], want)
    assert (got[N:] == 7.0).all()
    assert not vc.any()
