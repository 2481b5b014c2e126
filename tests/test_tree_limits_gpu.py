"""Counts that do not fit 32 bits are refused, not cut to what is left of them."""
import pytest
import torch

pytestmark = pytest.mark.gpu
dev = "cuda"
N = 2 ** 32                                                    # 32-bit: 0, which would be a call that does nothing


def refuses(fn, *a, **kw):
    with pytest.raises(RuntimeError, match="2147483647"):
        fn(*a, **kw)


def test_counts_past_32_bits_are_refused():
    import gfx906_fa
    if torch.cuda.mem_get_info()[0] < 60 * 2 ** 30:
        pytest.skip("needs 60 GB")
    kc = torch.zeros((4, 16, 1, 136), dtype=torch.uint8, device=dev)
    vc = torch.zeros((4, 16, 1, 128), dtype=torch.bfloat16, device=dev)
    long = torch.empty(N, dtype=torch.int64, device=dev)       # never read
    refuses(gfx906_fa.read_kv, kc, vc, long, torch.float16)
    refuses(gfx906_fa.move_kv, [kc], [vc], long, long, 1)
    refuses(gfx906_fa.move_kv, [kc], [vc], long, long, N)
    refuses(gfx906_fa.copy_pages, [kc], long, long)
    key = torch.zeros((1, 1, 128), dtype=torch.bfloat16, device=dev).expand(N, 1, 128)
    refuses(gfx906_fa.norm_rope_store_kv, None, key, key, None, None, 0.0, long, torch.ones((1, 128), device=dev), True, long, kc, vc, 1)
    links = long.view(torch.int32)[:N]
    refuses(gfx906_fa.tree_mask, links, torch.zeros(2, dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev), 8)
