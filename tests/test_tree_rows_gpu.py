"""tree_attention where the last warp, the last row tile or the last row group is partly filled: rows past the group skip what the
rows beside them do between two accesses of the warp's tensor memory.  Tolerance: the attention kernels' own 2e-3 + 1e-2 |ref|."""
import pytest
import torch

from _paged import assert_close
from _tree import TreeCase

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("v_fmt", ["q8t", "bf16"])
@pytest.mark.parametrize("n,G", [(1, 1), (31, 1), (33, 1), (63, 1), (97, 1), (127, 1), (129, 1), (161, 1), (3, 7), (13, 16), (17, 16),
                                 (257, 1), (43, 6)])
def test_partly_filled_warps(n, G, v_fmt):
    """A long context (ranges that are cut, partial rows), and one inside a single tile (rows written at once), with everything
    that changes scores lane by lane: masks, a window, a cap, sinks."""
    import gfx906_fa
    dtype = torch.bfloat16 if v_fmt == "bf16" else torch.float16
    kw = dict(softcap=20.0, sliding_window=400, sinks=torch.linspace(-1, 1, 2 * G, device="cuda"))
    for lens in ([1500 + n, n + 9], [n]):
        case = TreeCase(lens, [n] * len(lens), 2 * G, 2, v_fmt, seed=n + G, dtype=dtype)
        ref = case.reference(softcap=20.0, window=400, sinks=kw["sinks"].cpu().numpy())
        assert_close(case.run(**kw).float().cpu().numpy(), ref, what=f"{n} x {G}, {lens}")
        assert_close(case.run().float().cpu().numpy(), case.reference(), what=f"{n} x {G}, {lens}, plain")
    assert gfx906_fa.device_error(True) == 0
