"""tree_attention keeps the range of bf16 values."""
import pytest
import torch

import numpy as np

from _paged import assert_close
from _tree import TreeCase

pytestmark = pytest.mark.gpu
dev = "cuda"


@pytest.mark.parametrize("lens,n_q,Hq,Hkv", [([300, 40], [8, 5], 12, 2),      # one row tile
                                             ([200, 90], [40, 33], 48, 8),    # two
                                             ([20011], [16], 12, 2)])         # cut into ranges that are joined
def test_bf16_values_keep_their_range(lens, n_q, Hq, Hkv):
    """Dim d of every value is scaled by 2^k_d, k_d from -100 to 100: the output is the unscaled one times 2^k_d, to the same
    relative accuracy (2e-3 + 1e-2 |o| of the unscaled output)."""
    import gfx906_fa
    case = TreeCase(lens, n_q, Hq, Hkv, "bf16", seed=1, dtype=torch.bfloat16)
    ref = case.reference()
    k = torch.linspace(-100, 100, 128).round()
    case.v_cache.mul_(torch.exp2(k).to(dev).bfloat16())                        # exact: powers of two
    out = torch.empty(case.q.shape, device=dev)
    case.run(out=out)
    assert_close((out.double().cpu() * torch.exp2(-k.double())).numpy(), ref, what="scaled values")
    small = torch.empty_like(case.q)
    case.run(out=small)
    assert_close((small.double().cpu() * torch.exp2(-k.double())).numpy(), ref, what="bf16 output")
    assert gfx906_fa.device_error(True) == 0


def test_bf16_values_do_not_depend_on_the_caches_alignment():
    """Values of 1e5 and 1e-9 read by the tensor-core kernel and by the one for rows on 2-byte boundaries."""
    case = TreeCase([200, 333], [6, 9], 12, 2, "bf16", seed=2, dtype=torch.bfloat16)
    for scale in (1e5, 1e-9):
        value = case.v_cache.clone()
        case.v_cache = value * scale
        out = torch.empty(case.q.shape, device=dev)
        case.run(out=out)
        wide = torch.zeros((*value.shape[:3], 129), dtype=torch.bfloat16, device=dev)
        wide[..., :128] = case.v_cache
        case.v_cache = wide[..., :128]
        other = torch.empty(case.q.shape, device=dev)
        case.run(out=other)
        assert_close((out / scale).cpu().numpy(), (other / scale).cpu().numpy(), what=f"{scale}")
        case.v_cache = value


def test_an_infinite_bf16_value_stays_infinite():
    """In a tile that every row sees whole, also where every weight is exactly 1 (equal scores: keys of zero)."""
    for keys in (1.0, 0.0):
        case = TreeCase([400], [9], 12, 2, "bf16", seed=4, dtype=torch.bfloat16)
        if keys == 0:
            case.k_cache.zero_()
        page = case.block_table[0].tolist()
        for pos, d, x in ((5, 3, float("inf")), (140, 40, -float("inf")), (141, 90, float("nan")), (6, 91, float("inf")),
                          (142, 91, -float("inf"))):
            case.v_cache[page[pos // 16], pos % 16, :, d] = x
        out = case.run().float().cpu()
        assert (out[..., 3] == float("inf")).all() and (out[..., 40] == -float("inf")).all()
        assert out[..., 90:92].isnan().all()
        rest = [d for d in range(128) if d not in (3, 40, 90, 91)]
        assert_close(out[..., rest].numpy(), case.reference()[..., rest], what="the other elements")
