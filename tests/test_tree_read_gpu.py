"""read_kv of consecutive slots, and of page sizes and records that go element by element, against the oracle's bytes."""
import numpy as np
import pytest
import torch

import oracle as O
from _tree import dequant_rows
from _util import to_np

pytestmark = pytest.mark.gpu
dev = "cuda"
D = 128


def stored(T, Hkv, bs, mode, seed, shift=0):
    """A cache of T tokens of random keys and values in shuffled pages, with what its rows stand for: [NB * bs, Hkv, D] float64.
    `shift`: bytes the page-transposed records stand off their natural place."""
    import gfx906_fa
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((2, T, Hkv, D), generator=g).half()
    NB = -(-T // bs) + 2
    pages = torch.randperm(NB, generator=g)
    at = torch.arange(T)
    slots = pages[at // bs] * bs + at % bs
    kc = torch.zeros((NB, bs, Hkv, 136), dtype=torch.uint8, device=dev)
    if mode == 3:
        raw = torch.zeros((NB, Hkv, bs * 136 + 2 * shift), dtype=torch.uint8, device=dev)
        vc = raw[..., shift:shift + bs * 136]
    else:
        vc = torch.zeros((NB, bs, Hkv, 136) if mode == 2 else (NB, bs, Hkv, D), dtype=torch.uint8 if mode == 2 else torch.float16,
                         device=dev)
    dense = torch.zeros((NB, Hkv, bs * 136), dtype=torch.uint8, device=dev) if mode == 3 else vc
    gfx906_fa.store_kv(x[0].to(dev), x[1].to(dev), slots.to(dev), kc, dense, mode)
    if mode == 3:
        vc.copy_(dense)
    want = []
    for src, q8 in ((x[0], True), (x[1], mode != 1)):
        rows = np.zeros((NB, bs, Hkv, 136), np.uint8)
        full = np.zeros((NB * bs, Hkv, D))
        if q8:
            O.reshape_and_cache(to_np(src), slots.numpy(), rows)
            full[slots.numpy()] = dequant_rows(rows.reshape(NB * bs, Hkv, 136))[slots.numpy()]
        else:
            full[slots.numpy()] = src.double().numpy()
        want.append(full)
    return kc, vc, slots, want


def check(kc, vc, ask, want, dtype):
    import gfx906_fa
    got = gfx906_fa.read_kv(kc, vc, ask.to(dev), dtype)
    keep = (ask >= 0).numpy()[:, None, None]
    for name, x, w in zip(("keys", "values"), got, want):
        w = torch.from_numpy(np.where(keep, w[ask.clamp(min=0).numpy()], 0.0)).float().to(dtype)    # whole number * fp16: exact in fp32
        assert torch.equal(x.cpu(), w), name
    assert gfx906_fa.device_error(True) == 0


@pytest.mark.parametrize("mode", [1, 2, 3])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bs", [16, 32, 8, 48])
def test_consecutive_slots(bs, dtype, mode):
    kc, vc, slots, want = stored(160, 3, bs, mode, seed=bs + mode)
    for first in (0, 5, 15):
        for n in (1, 16, 33, 100, 144):
            ask = slots[first:first + n].clone()
            check(kc, vc, ask, want, dtype)
            if n > 16:
                ask[n // 2] = -1                            # a hole in the run
                check(kc, vc, ask, want, dtype)
                check(kc, vc, ask.flip(0), want, dtype)     # no runs at all
                check(kc, vc, torch.cat([ask[:7], ask[3:n]]), want, dtype)      # runs that start and end anywhere, rows twice


@pytest.mark.parametrize("shift", [2, 8, 16])
def test_records_off_their_boundaries(shift):
    kc, vc, slots, want = stored(70, 2, 16, 3, seed=shift, shift=shift)
    assert vc.stride(1) != vc.shape[2]
    check(kc, vc, slots, want, torch.float32)
    check(kc, vc, slots[torch.randperm(70, generator=torch.Generator().manual_seed(1))], want, torch.float16)


def test_values_of_far_slots():
    """Page-transposed values at byte offsets past 32 bits, against the oracle."""
    import gfx906_fa
    from gfx906_fa_paged import kv_cache_views
    kv = torch.empty((72000, 2, 16, 8, D), dtype=torch.bfloat16, device=dev)
    k, v = kv_cache_views(kv, "q8_0")
    x = torch.randn((2, 40, 8, D), generator=torch.Generator().manual_seed(5)).bfloat16()
    slots = torch.arange(71990 * 16 + 3, 71990 * 16 + 43)
    gfx906_fa.store_kv(x[0].to(dev), x[1].to(dev), slots.to(dev), k, v, 3)
    got = gfx906_fa.read_kv(k, v, slots.to(dev), torch.float32)
    for src, y in zip(x, got):
        rows = np.zeros((3, 16, 8, 136), np.uint8)
        O.reshape_and_cache(to_np(src), slots.numpy() - 71990 * 16, rows, dtype="bf16")
        assert torch.equal(y.cpu(), torch.from_numpy(dequant_rows(rows.reshape(-1, 8, 136)[3:43])).float())
