"""tree_attention of values that are not finite: element d of a row's output is what element d of the values it sees makes of it,
whichever tile of keys they stand in.  Tolerance of the finite elements: the attention kernels' own 2e-3 + 1e-2 |ref|."""
import numpy as np
import pytest
import torch

from _paged import assert_close
from _tree import TreeCase

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("v_fmt", ["f16", "bf16", "q8", "q8t"])
@pytest.mark.parametrize("ctx,n,kw", [(100, 12, {}), (290, 7, {}), (290, 60, {}), (9000, 12, {}), (700, 12, dict(sliding_window=300)),
                                      (3, 40, {})])
def test_only_their_own_elements(ctx, n, kw, v_fmt):
    """Infinities of both signs and NaN in a few elements of context keys and drafts: in tiles every row sees whole, in the one with
    the drafts, and in the one where windows begin."""
    dtype = torch.bfloat16 if v_fmt == "bf16" else torch.float16
    case = TreeCase([ctx + n, 90], [n, 5], 12, 2, v_fmt, seed=ctx + n, dtype=dtype)
    table = case.block_table.numpy()
    lo = max(0, ctx + 2 - kw.get("sliding_window", ctx + 2))
    at = sorted({min(lo + 1, ctx - 1), ctx // 2, ctx - 1, ctx, ctx + n // 2, ctx + n - 1})
    for i, pos in enumerate(at):
        page, off, h = int(table[0, pos // 16]), pos % 16, i % 2
        if v_fmt in ("f16", "bf16"):
            for k, x in enumerate((INF, -INF, NAN)):
                case.v_cache[page, off, h, 7 * i + 31 * k] = x
            case.v_cache[page, off, h, 100] = INF if i < 2 else -INF           # two signs meet: NaN
        elif v_fmt == "q8":
            block = case.v_cache[page, off, h].view(4, 34)[i % 4]
            block[:2] = torch.tensor([0x00, 0x7c], dtype=torch.uint8)         # a scale of infinity: a block of +-inf and, at 0, NaN
        else:
            scale = 2 * (i % 4 * 16 + off)
            case.v_cache[page, h, scale:scale + 2] = torch.tensor([0x00, 0x7c], dtype=torch.uint8)
    with np.errstate(invalid="ignore"):
        want = case.reference(**{"window": kw.get("sliding_window", 0)})
    got = case.run(**kw).double().cpu().numpy()
    assert not np.isfinite(want).all() and np.isfinite(want).any()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.isposinf(got), np.isposinf(want)) and np.array_equal(np.isneginf(got), np.isneginf(want))
    ok = np.isfinite(want)
    assert_close(np.where(ok, got, 0), np.where(ok, want, 0), what=f"{v_fmt} {ctx} {n}")
