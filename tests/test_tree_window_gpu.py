"""tree_attention's sliding window among the drafts: a draft at distance `window` or more along the token's own path is hidden, as
paged_attention hides the key at that distance.  Tolerance: the attention kernels' own 2e-3 + 1e-2 |ref|."""
import numpy as np
import pytest
import torch

import gfx906_fa_paged
from _paged import assert_close
from _tree import TreeCase, ancestors, random_parents, tree_reference

pytestmark = pytest.mark.gpu
dev = "cuda"


def check(case, seen, window, what):
    """`seen`: what each draft sees of the drafts once the window is taken into account."""
    import gfx906_fa
    out = case.run(sliding_window=window).float().cpu().numpy()
    assert_close(out, tree_reference(case, case.q.cpu().double().numpy(), case.n_q, seen, window=window), what=what)
    assert gfx906_fa.device_error(True) == 0


@pytest.mark.parametrize("v_fmt,bs", [("q8t", 16), ("f16", 16), ("bf16", 16), ("q8", 16), ("q8t", 8)])
@pytest.mark.parametrize("window", [1, 4, 10, 11, 12, 40])
def test_a_chain_is_the_causal_window(window, v_fmt, bs):
    """A chain through forward_paged: what paged_attention gives, and what the rule gives in 64 bits."""
    import gfx906_fa
    n = 11
    dtype = torch.bfloat16 if v_fmt == "bf16" else torch.float16
    case = TreeCase([900, 33, n], [n] * 3, 12, 2, v_fmt, bs=bs, seed=window, dtype=dtype, seen=[np.tril(np.ones((n, n), bool))] * 3)
    i = np.arange(n)
    check(case, [(i[:, None] >= i) & (i[:, None] - i < window)] * 3, window, f"chain, window {window}")
    out = gfx906_fa_paged.forward_paged(case.q, None, case.v_cache, case.bt, case.lens, case.start, n, 900, scale=case.scale,
                                        key_cache_q8=case.k_cache, tree_mask=case.mask, sliding_window=window)
    ref = gfx906_fa.paged_attention(case.q, case.k_cache, case.v_cache, case.bt, case.lens, case.start, n, 900, case.scale,
                                    sliding_window=window)
    assert_close(out.view(3 * n, 12, 128).cpu().numpy(), ref.float().cpu().numpy(), what="paged_attention")


@pytest.mark.parametrize("v_fmt,bs", [("q8t", 16), ("f16", 16), ("f16", 8)])
@pytest.mark.parametrize("window,n", [(3, 20), (33, 90), (64, 100), (31, 70)])
def test_trees_deeper_than_the_window(window, n, v_fmt, bs):
    """Distances are differences of depth, however the siblings stand between a draft and its ancestors."""
    rng = np.random.default_rng(window + n)
    n_q, seen = [n, n // 2, 1], []
    parents = [random_parents(k, rng, reach=2) for k in n_q]
    for p in parents:
        full = ancestors(p)
        depth = full.sum(1)
        assert len(p) < n or depth.max() > window
        seen.append(full & (depth[:, None] - depth[None] < window))
    case = TreeCase([n + 300, n // 2 + 5, 200], n_q, 12, 2, v_fmt, bs=bs, seed=n, dtype=torch.float16,
                    seen=[ancestors(p) for p in parents])
    check(case, seen, window, f"{n} drafts, window {window}")


@pytest.mark.parametrize("window", [1, 7, 20])
def test_any_bits_keep_the_last_ones(window):
    """Bits that are no tree: a row's distances are ranks among the drafts it selects, of which the last `window` stay."""
    rng = np.random.default_rng(window)
    full = [rng.random((70, 70)) < 0.4, rng.random((9, 9)) < 0.5, np.zeros((4, 4), bool)]
    seen = [f & (np.cumsum(f[:, ::-1], 1)[:, ::-1] <= window) for f in full]
    case = TreeCase([370, 9, 60], [70, 9, 4], 12, 2, "q8t", seed=window, seen=full)
    check(case, seen, window, f"any bits, window {window}")


@pytest.mark.parametrize("bs", [16, 8])
def test_a_window_wider_than_any_length_hides_nothing(bs):
    """Sequences of which the cache holds fewer rows than they drafted stand before position 0; with the widest window too."""
    case = TreeCase([12, 40, 300], [12, 40, 9], 12, 2, "q8t", bs=bs, seed=3)
    case.lens = torch.tensor([3, 0, 300], dtype=torch.int32, device=dev)
    ref = case.run()
    assert torch.isfinite(ref).all() and ref[52:].any()
    assert torch.equal(case.run(sliding_window=2 ** 31 - 1), ref)
    assert torch.equal(case.run(sliding_window=2 ** 31 - 20), ref)
