"""One attention layer of draft-tree speculation over the paged Q8_0 cache, end to end.

A toy drafter proposes a tree of tokens for each of a few sequences; the target layer verifies all of them in one pass, the accepted
path of each tree is kept, and one sequence is forked:

  tree_mask           parent links -> ancestor bits and rotary positions
  norm_rope_store_kv  QK norm + rotation, drafts' keys and values into the cache
  tree_attention      every draft against its context and its own ancestors
  move_kv             the accepted path's rows moved behind the context
  copy_pages          the fork's last, partly filled page

The last step shows that nothing was lost: the next token attends over the compacted cache with the plain decode kernel, and gives
what the accepted leaf's own row gave.

    python examples/tree_verify.py            # needs a B200 and the built extension
"""
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gfx906-fa-vllm_b200"))

import gfx906_fa  # noqa: E402
from gfx906_fa_paged import forward_paged, kv_cache_views  # noqa: E402

HQ, HKV, D, BS = 48, 8, 128, 16


class Layer:
    """Projections of a token's hidden state to the packed q, k, v a model hands its attention."""

    def __init__(self, hidden, g, dev):
        self.w = (torch.randn((hidden, (HQ + 2 * HKV) * D), generator=g) / hidden ** 0.5).bfloat16().to(dev)
        self.q_norm = (1 + 0.1 * torch.randn(D, generator=g)).bfloat16().to(dev)
        self.k_norm = (1 + 0.1 * torch.randn(D, generator=g)).bfloat16().to(dev)
        inv = 1.0 / (1e6 ** (torch.arange(0, D, 2) / D))
        angle = torch.outer(torch.arange(4096), inv)
        self.cos_sin = torch.cat([angle.cos(), angle.sin()], -1).float().to(dev)

    def store(self, x, positions, slots, k_cache, v_cache):
        """Rotated queries of x [T, hidden]; its keys and values go into the cache."""
        qkv = (x @ self.w).view(-1, HQ + 2 * HKV, D)
        q, k, v = qkv.split([HQ, HKV, HKV], 1)
        gfx906_fa.norm_rope_store_kv(q, k, v, self.q_norm, self.k_norm, 1e-6, positions, self.cos_sin, True, slots, k_cache, v_cache,
                                     3 if v_cache.dim() == 3 else 1)
        return q


def main(v_fmt="q8_0", seed=0):
    dev = "cuda"
    g = torch.Generator().manual_seed(seed)
    hidden, context = 256, [700, 33, 1500]
    B, drafts = len(context), 20
    layer = Layer(hidden, g, dev)

    pages = [(n + drafts + BS) // BS + 1 for n in context]
    num_pages = sum(pages) + 2 + max(pages)
    kv = torch.zeros((num_pages, 2, BS, HKV, D), dtype=torch.bfloat16, device=dev)
    k_cache, v_cache = kv_cache_views(kv, v_fmt)
    free = (torch.randperm(num_pages - 1, generator=g) + 1).tolist()          # page 0 stays unused
    table = torch.zeros((B, max(pages)), dtype=torch.int32)
    for b, n in enumerate(pages):
        table[b, :n] = torch.tensor([free.pop() for _ in range(n)])
    table_d = table.to(dev)

    def slot(b, i):
        return int(table[b, i // BS]) * BS + i % BS

    def slots(spans):
        return torch.tensor([slot(b, i) for b, (lo, hi) in enumerate(spans) for i in range(lo, hi)], device=dev)

    # ---- the prompts -------------------------------------------------------------------
    x = torch.randn((sum(context), hidden), generator=g).bfloat16().to(dev)
    pos = torch.cat([torch.arange(n) for n in context]).to(dev)
    layer.store(x, pos, slots([(0, n) for n in context]), k_cache, v_cache)

    # ---- a tree of drafts per sequence ---------------------------------------------------
    parents = torch.cat([torch.tensor([max(-1, i - 1 - int(torch.randint(0, 4, (1,), generator=g))) for i in range(drafts)])
                         for _ in context]).to(torch.int32).to(dev)
    start = torch.arange(0, (B + 1) * drafts, drafts, dtype=torch.int32, device=dev)
    lens = torch.tensor([n + drafts for n in context], dtype=torch.int32, device=dev)
    mask, pos = gfx906_fa.tree_mask(parents, start, lens, drafts)
    x = torch.randn((B * drafts, hidden), generator=g).bfloat16().to(dev)
    q = layer.store(x, pos, slots([(n, n + drafts) for n in context]), k_cache, v_cache)
    out = forward_paged(q, None, v_cache, table_d, lens, start, drafts, int(lens.max()), key_cache_q8=k_cache,
                        out=torch.empty((B * drafts, HQ, D), dtype=torch.bfloat16, device=dev), tree_mask=mask)

    # ---- accept a path: here, from the root to each tree's last token -----------------------
    up = parents.view(B, drafts).tolist()
    paths = []
    for b in range(B):
        path, i = [], drafts - 1
        while i >= 0:
            path.append(i)
            i = up[b][i]
        paths.append(path[::-1])
    most = max(map(len, paths))
    src = torch.tensor([[slot(b, context[b] + i) for i in p] + [-1] * (most - len(p)) for b, p in enumerate(paths)], device=dev)
    dst = torch.tensor([[slot(b, context[b] + i) for i in range(len(p))] + [-1] * (most - len(p)) for b, p in enumerate(paths)],
                       device=dev)
    leaf_k, leaf_v = gfx906_fa.read_kv(k_cache, v_cache, torch.stack([src[b, len(p) - 1] for b, p in enumerate(paths)]), torch.float32)
    gfx906_fa.move_kv([k_cache], [v_cache], src.flatten(), dst.flatten(), most)
    kept = torch.tensor([n + len(p) for n, p in zip(context, paths)], dtype=torch.int32, device=dev)
    moved_k, moved_v = gfx906_fa.read_kv(k_cache, v_cache, torch.stack([dst[b, len(p) - 1] for b, p in enumerate(paths)]), torch.float32)
    assert torch.equal(leaf_k, moved_k) and torch.equal(leaf_v, moved_v)

    # ---- fork sequence 0: its full pages are shared, the last one is copied -------------------
    last = (int(kept[0]) - 1) // BS
    fork = table[0].clone()
    fork[last] = free.pop()
    gfx906_fa.copy_pages([kv], table[0, last:last + 1].long().to(dev), fork[last:last + 1].long().to(dev))

    # ---- the accepted leaves again, as plain decode over the compacted caches and the fork ------
    leaves = torch.tensor([b * drafts + p[-1] for b, p in enumerate(paths)] + [paths[0][-1]], device=dev)
    again = torch.empty((B + 1, HQ, D), dtype=torch.bfloat16, device=dev)
    forward_paged(q[leaves], None, v_cache, torch.cat([table, fork[None]]).to(dev), torch.cat([kept, kept[:1]]),
                  torch.arange(B + 2, dtype=torch.int32, device=dev), 1, int(kept.max()), key_cache_q8=k_cache, out=again)
    worst = float((again.float() - out[leaves].float()).abs().max())
    print(f"{B} sequences, {drafts} drafts each, accepted {[len(p) for p in paths]}; tree row against decode over the "
          f"compacted cache: largest difference {worst:.2e}")
    assert worst < 1e-2 and gfx906_fa.device_error(True) == 0
    return worst


if __name__ == "__main__":
    for fmt in ("q8_0", "fp16"):
        main(fmt)
