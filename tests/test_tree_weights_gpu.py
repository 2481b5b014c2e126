"""tree_attention rounds a softmax weight to 16 bits once."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
dev = "cuda"
D, BS = 128, 16


@pytest.mark.parametrize("drafts", [64, 160])                  # one row tile, two
@pytest.mark.parametrize("v_fmt", ["q8t", "f16", "bf16"])
def test_weights_are_rounded_once(v_fmt, drafts):
    """The maximum rises by more than the lazy threshold between the halves of a key tile, after the first half's weights are
    written.  Keys are 127 * 2^-7 in one element of a Q8_0 block of their own, so scores are exact; a row's 64 keys of the first half
    have one score, so their rounding errors do not average out, and they alone have the value 1.  The output is then
    off by the weight's own rounding, 2^-11 of it, and by what fp32 and ex2.approx leave: 2^-16 bounds a dozen steps
    of 2^-24 on scores up to 18.  More kv heads than SMs: no CTA range cuts the sequence, whatever the card."""
    import gfx906_fa
    H, L, c = 160, 4 * 128, 127 * 2.0 ** -7
    NB = (L + drafts) // BS + 1
    g = torch.Generator().manual_seed(drafts)
    key = torch.zeros((L, H, D))
    # tiles 0 and 2 go to one stream of key tiles (or all to one): level 0, then `low` and `high`; tiles 1 and 3 lie far below
    key[:128, :, 64] = c
    key[128:256, :, 96] = c
    key[256:320, :, 0] = c
    key[320:384, :, 32] = c
    key[384:, :, 96] = c
    value = torch.zeros((L, H, D))
    value[256:320] = 1.0
    vdt = torch.bfloat16 if v_fmt == "bf16" else torch.float16
    slots = torch.arange(L, device=dev)
    kc = torch.zeros((NB, BS, H, 136), dtype=torch.uint8, device=dev)
    vc = (torch.zeros((NB, H, BS * 136), dtype=torch.uint8, device=dev) if v_fmt == "q8t" else
          torch.zeros((NB, BS, H, D), dtype=vdt, device=dev))
    gfx906_fa.store_kv(key.to(vdt).to(dev), value.to(vdt).to(dev), slots, kc, vc, 3 if v_fmt == "q8t" else 1)
    q = torch.zeros((drafts, H, D))
    q[..., 0] = 3 + 4.5 * torch.rand((drafts, H), generator=g)               # log2 of the first half's weights against level 0
    q[..., 32] = 8.2 + 0.9 * torch.rand((drafts, H), generator=g)
    q[..., 96] = -40.0
    q = q.half()
    scale = float(np.log(2.0))
    mask = torch.zeros((drafts, (drafts + 31) // 32), dtype=torch.int32, device=dev)
    out = torch.empty((drafts, H, D), device=dev)
    gfx906_fa.tree_attention(q.to(dev), kc, vc, torch.arange(NB, dtype=torch.int32, device=dev)[None],
                             torch.tensor([L + drafts], dtype=torch.int32, device=dev),
                             torch.tensor([0, drafts], dtype=torch.int32, device=dev), mask, drafts, L + drafts, scale, out=out)
    # values of 1 as the cache holds them: Q8_0 stores 127 * fp16(1 / 127), rounded to fp16 by the kernel
    one = float(np.float16(127 * np.float64(np.float16(1 / 127)))) if v_fmt == "q8t" else 1.0
    low, high, far = (2.0 ** (q[..., e].double().numpy() * c) for e in (0, 32, 96))
    want = one * 64 * low / (64 * low + 64 * high + 128 + 256 * far)
    got = out.double().cpu().numpy()
    assert np.array_equal(got, np.broadcast_to(got[..., :1], got.shape))
    off = np.abs(got[..., 0] / want - 1)
    assert off.max() <= 2.0 ** -11 + 2.0 ** -16, f"{off.max() * 2 ** 11:.3f} of 2^-11"
    assert gfx906_fa.device_error(True) == 0
