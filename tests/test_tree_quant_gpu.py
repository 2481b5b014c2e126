"""norm_rope_store_kv's division-free quantiser over every finite 16-bit maximum."""
import numpy as np
import pytest
import torch

import oracle as O
from _util import to_np
from test_tree_kv_gpu import caches, check_cache

pytestmark = pytest.mark.gpu
dev = "cuda"


@pytest.mark.parametrize("mode", [2, 3])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_every_16bit_maximum(dtype, mode):
    """Every finite value is the maximum of one 32-element block, whose other elements are that value times k / 31, as keys
    (no weights, an angle of zero: they are quantised as they come) and as values: the oracle's bytes (IEEE division, rintf)."""
    import gfx906_fa
    bits = np.arange(65536, dtype=np.uint32).astype(np.uint16)
    v = bits.view(np.float16).astype(np.float32) if dtype == torch.float16 else O.bf16_bits_to_f32(bits)
    v = v[np.isfinite(v)]
    v = np.concatenate([v, np.zeros(-len(v) % 512, np.float32)])              # whole tokens of 8 heads x 4 blocks
    # the largest element stands at another place in each block
    order = (np.arange(32)[None] + np.arange(len(v))[:, None]) % 32
    rows = torch.from_numpy(v[:, None] * (order[:, ::-1].astype(np.float32) / 31.0)).to(dtype).view(-1, 8, 128)
    T = rows.shape[0]
    kc, vc = caches(-(-T // 16), 8, mode, dtype)
    x = rows.to(dev)
    cs = torch.cat([torch.ones((1, 64)), torch.zeros((1, 64))], 1).to(dev)
    ko = torch.empty_like(x)
    gfx906_fa.norm_rope_store_kv(None, x, x.flip(0).contiguous(), None, None, 0.0, torch.zeros(T, dtype=torch.int64, device=dev), cs,
                                 True, torch.arange(T, device=dev), kc, vc, mode, key_out=ko)
    assert torch.equal(ko.float(), x.float())
    check_cache(kc, vc, mode, x, rows.flip(0).contiguous(), torch.arange(T), dtype)
    assert gfx906_fa.device_error(True) == 0
