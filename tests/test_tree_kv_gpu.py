"""tree_mask, norm_rope_store_kv, read_kv, move_kv and copy_pages against plain forms."""
import numpy as np
import pytest
import torch

import oracle as O
from _tree import ancestors, dequant_rows, pack_bits, random_parents
from _util import to_np

pytestmark = pytest.mark.gpu
dev = "cuda"
D, BS = 128, 16


# ---------------------------------------------------------------- tree_mask
@pytest.mark.parametrize("n", [[1], [16], [5, 0, 32, 33, 1], [64] * 40, [200, 3], [700]])
def test_tree_mask(n):
    import gfx906_fa
    rng = np.random.default_rng(sum(n))
    parents = [random_parents(k, rng, reach=6) for k in n]
    start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
    lens = (rng.integers(0, 5000, len(n)) + np.array(n)).astype(np.int32)
    flat = np.array(sum(parents, []), np.int32)
    mask, pos = gfx906_fa.tree_mask(torch.from_numpy(flat).to(dev), torch.from_numpy(start).to(dev),
                                    torch.from_numpy(lens).to(dev), max(n))
    words = -(-max(n) // 32)
    seen = [ancestors(p) for p in parents]
    want = np.concatenate([pack_bits(s, words) for s in seen if s.size])
    assert mask.dtype == torch.int32 and np.array_equal(mask.cpu().numpy(), want)
    depth = np.concatenate([s.sum(1) - 1 for s in seen if s.size])
    base = np.repeat(lens - np.array(n), n)
    assert pos.dtype == torch.int64 and np.array_equal(pos.cpu().numpy(), base + depth)
    assert gfx906_fa.device_error(True) == 0


def test_tree_mask_cuts_bad_links_and_zeroes_padding():
    import gfx906_fa
    parents = torch.tensor([0, 5, 1, -7, 0, 0], dtype=torch.int32, device=dev)       # drafts 0 and 1 link to themselves / forward
    start = torch.tensor([0, 4], dtype=torch.int32, device=dev)
    mask, pos = gfx906_fa.tree_mask(parents, start, torch.tensor([14], dtype=torch.int32, device=dev), 4)
    assert mask.cpu().flatten().tolist() == [1, 2, 6, 8, 0, 0]
    assert pos.cpu().tolist() == [10, 10, 11, 10, 0, 0]
    assert gfx906_fa.device_error(True) == 8
    empty = gfx906_fa.tree_mask(parents[:0], start[:1], torch.empty(0, dtype=torch.int32, device=dev), 4)
    assert empty[0].shape == (0, 1) and empty[1].shape == (0,)


# ---------------------------------------------------------------- norm + rope + store
def cos_sin(max_pos, rot, base=1e4):
    inv = 1.0 / (base ** (torch.arange(0, rot, 2, dtype=torch.float64) / rot))
    f = torch.outer(torch.arange(max_pos, dtype=torch.float64), inv)
    return torch.cat([f.cos(), f.sin()], -1)


def norm_rope_reference(x, w, eps, pos, cs, neox):
    y = x.double()
    if w is not None:
        y = y / torch.sqrt((y ** 2).mean(-1, keepdim=True) + eps) * w.double()
    rot = cs.shape[1]
    c, s = cs[pos].double()[:, None, :rot // 2], cs[pos].double()[:, None, rot // 2:]
    j = torch.arange(rot // 2)
    a, b = (j, j + rot // 2) if neox else (2 * j, 2 * j + 1)
    out = y.clone()
    out[..., a] = y[..., a] * c - y[..., b] * s
    out[..., b] = y[..., b] * c + y[..., a] * s
    return out


def close(got, want, dtype):
    """|fp32 - exact| <= 2^-20 of the row's largest element (a dozen roundings of 2^-24, which a rotation's cancellation keeps
    relative to the larger element), then one rounding to the type: half a step, 2^-8 (bf16), 2^-11 (fp16) or 2^-24 of the
    value, or half of fp16's smallest step."""
    half = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}[dtype]
    want = want.numpy()
    off = np.abs(got.double().cpu().numpy() - want)
    fp32 = 2.0 ** -20 * np.abs(want).max(-1, keepdims=True)
    assert (off <= half * (np.abs(want) + fp32) + fp32 + 2.0 ** -25).all(), off.max()


def store_case(T, Hq, Hkv, dtype, seed, bs=BS):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn((T, Hq + 2 * Hkv, D), generator=g) * 3).to(dtype)
    w = (1 + 0.3 * torch.randn((2, D), generator=g))
    pos = torch.randint(0, 4000, (T,), generator=g)
    NB = -(-T // bs) + 3
    slots = torch.randperm(NB * bs, generator=g)[:T]
    slots[::7] = -1
    return qkv, w, pos, slots, NB


def caches(NB, Hkv, mode, dtype, bs=BS):
    kc = torch.zeros((NB, bs, Hkv, 136), dtype=torch.uint8, device=dev)
    vc = {1: lambda: torch.zeros((NB, bs, Hkv, D), dtype=dtype, device=dev),
          2: lambda: torch.zeros((NB, bs, Hkv, 136), dtype=torch.uint8, device=dev),
          3: lambda: torch.zeros((NB, Hkv, bs * 136), dtype=torch.uint8, device=dev)}[mode]()
    return kc, vc


def check_cache(kc, vc, mode, key, value, slots, dtype, bs=BS):
    """The cache holds the oracle's bytes of the key as it was rounded, and of the value."""
    tag = "bf16" if dtype == torch.bfloat16 else None
    want = np.zeros(tuple(kc.shape), np.uint8)
    O.reshape_and_cache(to_np(key), slots.numpy(), want, dtype=tag)
    assert np.array_equal(to_np(kc), want), "keys"
    if mode == 1:
        want = np.zeros(tuple(vc.shape), np.uint16)
        O.store_v16(to_np(value).view(np.uint16), slots.numpy(), want)
        assert np.array_equal(to_np(vc).view(np.uint16), want), "16-bit values"
    else:
        want = np.zeros(tuple(vc.shape), np.uint8)
        if mode == 2:
            O.reshape_and_cache(to_np(value), slots.numpy(), want, dtype=tag)
        else:
            O.store_v_q8t(to_np(value), slots.numpy(), want, bs, dtype=tag)
        assert np.array_equal(to_np(vc), want), "Q8_0 values"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("rot,mode,T,Hq,Hkv", [(128, 3, 77, 48, 8), (64, 1, 77, 48, 8), (96, 2, 1, 6, 1), (16, 3, 33, 9, 3),
                                               (32, 1, 700, 4, 4), (112, 3, 5, 14, 2)])
def test_norm_rope_store(dtype, neox, rot, mode, T, Hq, Hkv):
    import gfx906_fa
    qkv, w, pos, slots, NB = store_case(T, Hq, Hkv, dtype, seed=rot + T + mode)
    cs = cos_sin(4000, rot).to(dtype if neox else torch.float32)
    kc, vc = caches(NB, Hkv, mode, dtype)
    d = qkv.to(dev)
    q, k, v = d[:, :Hq], d[:, Hq:Hq + Hkv], d[:, Hq + Hkv:]
    before = d.clone()
    qo = torch.empty((T, Hq, D), dtype=dtype, device=dev)
    ko = torch.empty((T, Hkv, D), dtype=dtype, device=dev)
    wq, wk = w[0].to(dtype), w[1]                       # weights of either type
    gfx906_fa.norm_rope_store_kv(q, k, v, wq.to(dev), wk.to(dev), 1e-6, pos.to(dev), cs.to(dev), neox, slots.to(dev), kc, vc,
                                 mode, query_out=qo, key_out=ko)
    assert torch.equal(d, before), "inputs are left alone"
    close(qo, norm_rope_reference(qkv[:, :Hq], wq, 1e-6, pos, cs, neox), dtype)
    close(ko, norm_rope_reference(qkv[:, Hq:Hq + Hkv], wk, 1e-6, pos, cs, neox), dtype)
    check_cache(kc, vc, mode, ko, qkv[:, Hq + Hkv:].contiguous(), slots, dtype)
    # in place, without a key output
    gfx906_fa.norm_rope_store_kv(q, k, v, wq.to(dev), wk.to(dev), 1e-6, pos.to(dev), cs.to(dev), neox, slots.to(dev), kc, vc, mode)
    assert torch.equal(q, qo) and torch.equal(d[:, Hq:], before[:, Hq:])
    assert gfx906_fa.device_error(True) == 0


@pytest.mark.parametrize("mode", [1, 3])
@pytest.mark.parametrize("first", [0, 5])
@pytest.mark.parametrize("T,bs", [(16, 16), (100, 16), (70, 32), (40, 8)])
def test_store_of_consecutive_slots(T, bs, first, mode):
    """A prompt's slots run through whole pages: every page size and start offset."""
    import gfx906_fa
    qkv, w, pos, _, _ = store_case(T, 4, 2, torch.bfloat16, seed=T + first)
    NB = -(-(T + first) // bs) + 1
    pages = torch.randperm(NB, generator=torch.Generator().manual_seed(T))
    at = torch.arange(T) + first
    slots = pages[at // bs] * bs + at % bs
    slots[T // 2] = -1                                  # a hole in the run
    kc, vc = caches(NB, 2, mode, torch.bfloat16, bs)
    d, ko = qkv.to(dev), torch.empty((T, 2, D), dtype=torch.bfloat16, device=dev)
    gfx906_fa.norm_rope_store_kv(d[:, :4], d[:, 4:6], d[:, 6:], w[0].to(dev), w[1].to(dev), 1e-5, pos.to(dev),
                                 cos_sin(4000, 128).float().to(dev), True, slots.to(dev), kc, vc, mode, key_out=ko)
    check_cache(kc, vc, mode, ko, qkv[:, 6:].contiguous(), slots, torch.bfloat16, bs)


def test_without_norm_it_is_the_rope_store():
    """No weights: the bytes of rope_store_kv, whose rotation the oracle pins."""
    import gfx906_fa
    T, Hq, Hkv, dtype = 50, 12, 4, torch.bfloat16
    qkv, _, pos, slots, NB = store_case(T, Hq, Hkv, dtype, seed=1)
    cs = cos_sin(4000, 64).float().to(dev)
    out = []
    for fn in ("rope", "norm"):
        d = qkv.to(dev)
        kc, vc = caches(NB, Hkv, 3, dtype)
        q, k, v = d[:, :Hq], d[:, Hq:Hq + Hkv], d[:, Hq + Hkv:]
        if fn == "rope":
            gfx906_fa.rope_store_kv(q, k, v, pos.to(dev), cs, True, slots.to(dev), kc, vc, 3)
        else:
            gfx906_fa.norm_rope_store_kv(q, k, v, None, None, 0.0, pos.to(dev), cs, True, slots.to(dev), kc, vc, 3, key_out=k)
        out.append((d, kc, vc))
    for a, b in zip(*out):
        assert torch.equal(a, b)


def test_fp32_unaligned_rows_and_keys_only():
    import gfx906_fa
    T, Hkv = 21, 3
    g = torch.Generator().manual_seed(2)
    k = torch.randn((T, Hkv * 131 + 1), generator=g)
    w = torch.rand(D, generator=g) + 0.5
    pos, slots = torch.arange(T), torch.arange(T) + 3
    cs = cos_sin(64, 32)
    d = k.to(dev)
    key = d[:, 1:].view(T, Hkv, 131)[..., :D]
    kc, vc = caches(3, Hkv, 2, torch.float16)
    ko = torch.empty((T, Hkv, D), device=dev)
    gfx906_fa.norm_rope_store_kv(None, key, key, None, w.to(dev), 1e-6, pos.to(dev), cs.float().to(dev), False, slots.to(dev),
                                 kc, vc, 2, key_out=ko)
    close(ko, norm_rope_reference(k[:, 1:].reshape(T, Hkv, 131)[..., :D], w, 1e-6, pos, cs.float(), False), torch.float32)
    check_cache(kc, vc, 2, ko, key.cpu().contiguous(), slots, torch.float32)
    # K only, into a cache whose rows sit on 2-byte boundaries
    raw = torch.zeros(3 * BS * Hkv * 138 + 2, dtype=torch.uint8, device=dev)
    odd = raw[2:].view(3, BS, Hkv, 138)[..., :136]
    gfx906_fa.norm_rope_store_kv(None, key, key, None, w.to(dev), 1e-6, pos.to(dev), cs.float().to(dev), False, slots.to(dev),
                                 odd, odd, 0)
    assert torch.equal(odd, kc)


def test_bad_slots_and_positions_are_reported():
    import gfx906_fa
    qkv, w, pos, slots, NB = store_case(20, 4, 2, torch.bfloat16, seed=3)
    kc, vc = caches(NB, 2, 3, torch.bfloat16)
    d = qkv.to(dev)
    args = (w[0].to(dev), w[1].to(dev), 1e-6)
    cs = cos_sin(4000, 128).float().to(dev)
    slots[5] = NB * BS + 3
    gfx906_fa.norm_rope_store_kv(d[:, :4], d[:, 4:6], d[:, 6:], *args, pos.to(dev), cs, True, slots.to(dev), kc, vc, 3)
    assert gfx906_fa.device_error(True) == 8
    slots[5] = -1
    pos[3] = 4000
    gfx906_fa.norm_rope_store_kv(d[:, :4], d[:, 4:6], d[:, 6:], *args, pos.to(dev), cs, True, slots.to(dev), kc, vc, 3)
    assert gfx906_fa.device_error(True) == 8


def test_a_zero_row_stays_zero():
    import gfx906_fa
    kc, vc = caches(1, 1, 3, torch.bfloat16)
    z = torch.zeros((1, 1, D), dtype=torch.bfloat16, device=dev)
    one = torch.ones(D, device=dev)
    qo = torch.ones_like(z)
    gfx906_fa.norm_rope_store_kv(z, z, z, one, one, 1e-6, torch.zeros(1, dtype=torch.int64, device=dev),
                                 cos_sin(4, 128).float().to(dev), True, torch.zeros(1, dtype=torch.int64, device=dev), kc, vc, 3,
                                 query_out=qo)
    assert not qo.any() and not kc.any() and not vc.any()


def test_norm_store_refusals():
    import gfx906_fa
    qkv, w, pos, slots, NB = store_case(20, 4, 2, torch.bfloat16, seed=4)
    kc, vc = caches(NB, 2, 3, torch.bfloat16)
    d = qkv.to(dev)
    base = dict(query=d[:, :4], key=d[:, 4:6], value=d[:, 6:], q_weight=w[0].to(dev), k_weight=w[1].to(dev), eps=1e-6,
                positions=pos.to(dev), cos_sin_cache=cos_sin(4000, 128).float().to(dev), is_neox=True, slot_mapping=slots.to(dev),
                k_cache=kc, v_cache=vc, v_mode=3)
    half = torch.zeros((NB, BS, 2, D), dtype=torch.float16, device=dev)
    for over in (dict(key=qkv[:, 4:6]), dict(key=d[:, 4:6, :64]), dict(q_weight=w[0, :64].to(dev)), dict(k_weight=w[1]),
                 dict(positions=pos[:5].to(dev)), dict(positions=pos.int().to(dev)), dict(slot_mapping=slots[:3].to(dev)),
                 dict(cos_sin_cache=cos_sin(4000, 24).float().to(dev)), dict(cos_sin_cache=cos_sin(4000, 144).float().to(dev)),
                 dict(v_mode=1), dict(v_mode=4), dict(v_cache=half, v_mode=1), dict(k_cache=kc[..., :130]), dict(k_cache=kc[:, :, :1]),
                 dict(value=d[:5, 6:]), dict(query_out=torch.empty((20, 4, D), device=dev)),
                 dict(key_out=torch.empty((19, 2, D), dtype=torch.bfloat16, device=dev))):
        with pytest.raises(RuntimeError):
            gfx906_fa.norm_rope_store_kv(**{**base, **over})
    gfx906_fa.norm_rope_store_kv(**base)


# ---------------------------------------------------------------- read_kv
@pytest.mark.parametrize("mode", [1, 2, 3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("N,Hkv,bs", [(1, 1, 16), (61, 8, 16), (300, 3, 32)])
def test_read_kv(mode, dtype, N, Hkv, bs):
    import gfx906_fa
    g = torch.Generator().manual_seed(N + mode)
    vdt = torch.bfloat16 if dtype == torch.bfloat16 else torch.float16
    x = torch.randn((2, N, Hkv, D), generator=g).to(vdt)
    NB = -(-N // bs) + 2
    slots = torch.randperm(NB * bs, generator=g)[:N]
    kc, vc = caches(NB, Hkv, mode, vdt, bs)
    gfx906_fa.store_kv(x[0].to(dev), x[1].to(dev), slots.to(dev), kc, vc, mode)
    ask = slots.clone()
    ask[::5] = -1
    k, v = gfx906_fa.read_kv(kc, vc, ask.to(dev), dtype)
    tag = "bf16" if vdt == torch.bfloat16 else None
    rows = np.zeros((NB, bs, Hkv, 136), np.uint8)
    keep = (ask >= 0)[:, None, None]
    for got, src, q8 in ((k, x[0], True), (v, x[1], mode != 1)):
        want = src.double()
        if q8:
            O.reshape_and_cache(to_np(src), slots.numpy(), rows, dtype=tag)
            want = torch.from_numpy(dequant_rows(rows.reshape(NB * bs, Hkv, 136)[slots.numpy()]))
        want = (want * keep).float().to(dtype)         # whole number * 16-bit scale: exact in fp32
        assert got.dtype == dtype and torch.equal(got.cpu(), want)
    assert gfx906_fa.device_error(True) == 0


def test_read_kv_edges_and_refusals():
    import gfx906_fa
    kc, vc = caches(3, 2, 3, torch.bfloat16)
    none = torch.empty(0, dtype=torch.int64, device=dev)
    assert gfx906_fa.read_kv(kc, vc, none, torch.float16)[0].shape == (0, 2, D)
    k, v = gfx906_fa.read_kv(kc, vc, torch.tensor([48, 0], device=dev), torch.float32)
    assert not k.any() and gfx906_fa.device_error(True) == 8
    for bad in ((kc, vc, none.int(), torch.float16), (kc, vc, none, torch.int32), (kc[..., :100], vc, none, torch.float16),
                (kc, vc[:2], none, torch.float16), (kc, vc, none.cpu(), torch.float16)):
        with pytest.raises(RuntimeError):
            gfx906_fa.read_kv(*bad)


# ---------------------------------------------------------------- move_kv
def layer_views(L, NB, Hkv, mode, dtype=torch.bfloat16, bs=BS, seed=0):
    """L layers of the backend's allocation filled with random bytes, and their views."""
    from gfx906_fa_paged import kv_cache_views
    g = torch.Generator(device=dev).manual_seed(seed)
    raw = torch.randint(0, 256, (L, NB, 2 * bs * Hkv * D * 2), dtype=torch.uint8, device=dev, generator=g)
    kv = [raw[i].view(dtype).view(NB, 2, bs, Hkv, D) for i in range(L)]
    if mode == 2:
        half = bs * Hkv * 136
        k = [raw[i][:, :half].view(NB, bs, Hkv, 136) for i in range(L)]
        v = [raw[i][:, half:2 * half].view(NB, bs, Hkv, 136) for i in range(L)]
    else:
        views = [kv_cache_views(x, "q8_0" if mode == 3 else "fp16") for x in kv]
        k, v = [x[0] for x in views], [x[1] for x in views]
    return raw, kv, k, v


def plain_move(raw, L, Hkv, mode, pairs, bs=BS):
    """Bytes after every group's rows were read and then written, one row at a time."""
    out = raw.cpu().numpy().copy()
    half = bs * Hkv * 136
    for layer in range(L):
        x = out[layer]
        k = x[:, :half].reshape(-1, bs, Hkv, 136)
        groups = []
        for group in pairs:
            held = []
            for s, d in group:
                if s < 0 or d < 0:
                    continue
                pg, o = divmod(s, bs)
                if mode == 1:
                    v = x[:, x.shape[1] // 2:].reshape(-1, bs, Hkv, 256)[pg, o].copy()
                elif mode == 2:
                    v = x[:, half:2 * half].reshape(-1, bs, Hkv, 136)[pg, o].copy()
                else:
                    rec = x[:, half:2 * half].reshape(-1, Hkv, bs * 136)[pg]
                    v = (rec[:, :8 * bs].reshape(Hkv, 4, bs, 2)[:, :, o].copy(), rec[:, 8 * bs:].reshape(Hkv, D, bs)[:, :, o].copy())
                held.append((d, k[pg, o].copy(), v))
            groups.append(held)
        for held in groups:
            for d, kr, v in held:
                pg, o = divmod(d, bs)
                kk = x[pg, :half].reshape(bs, Hkv, 136)
                kk[o] = kr
                x[pg, :half] = kk.reshape(-1)
                if mode == 1:
                    vv = x[pg, x.shape[1] // 2:].reshape(bs, Hkv, 256)
                    vv[o] = v
                    x[pg, x.shape[1] // 2:] = vv.reshape(-1)
                elif mode == 2:
                    vv = x[pg, half:2 * half].reshape(bs, Hkv, 136)
                    vv[o] = v
                    x[pg, half:2 * half] = vv.reshape(-1)
                else:
                    rec = x[pg, half:2 * half].reshape(Hkv, bs * 136).copy()
                    sc = rec[:, :8 * bs].reshape(Hkv, 4, bs, 2).copy()
                    sc[:, :, o] = v[0]
                    w = rec[:, 8 * bs:].reshape(Hkv, D, bs).copy()
                    w[:, :, o] = v[1]
                    x[pg, half:2 * half] = np.concatenate([sc.reshape(Hkv, -1), w.reshape(Hkv, -1)], 1).reshape(-1)
    return out


@pytest.mark.parametrize("mode", [1, 2, 3])
@pytest.mark.parametrize("L,Hkv,groups,per,bs", [(1, 1, 1, 1, 16), (3, 8, 5, 6, 16), (2, 3, 2, 40, 16), (70, 2, 2, 3, 32),
                                                 (2, 8, 1, 130, 8)])
def test_move_kv(mode, L, Hkv, groups, per, bs):
    import gfx906_fa
    rng = np.random.default_rng(per)
    tree = 2 * per + 3
    npg = -(-(tree + 5) // bs) + 1
    NB = groups * npg + 1
    raw, _, k, v = layer_views(L, NB, Hkv, mode, bs=bs, seed=per)
    pages = rng.permutation(NB)[:groups * npg].reshape(groups, npg)
    pairs = []
    for g in range(groups):
        slot = lambda i: int(pages[g, (i + 5) // bs]) * bs + (i + 5) % bs  # noqa: E731,B023
        keep = sorted(rng.choice(tree, per, replace=False))
        if g == 1:                                      # a reversal: every row is overwritten before a serial move would read it
            group = [(slot(i), slot(per - 1 - i)) for i in range(per)]
        else:
            group = [(slot(int(i)), slot(j)) for j, i in enumerate(keep)]
            if per > 2:
                group[-1] = (-1, slot(per - 1))
                group[-2] = (group[-2][0], -1)
        pairs.append(group)
    src = torch.tensor([p[0] for g in pairs for p in g], device=dev)
    dst = torch.tensor([p[1] for g in pairs for p in g], device=dev)
    want = plain_move(raw, L, Hkv, mode, pairs, bs)
    gfx906_fa.move_kv(k, v, src, dst, per)
    assert np.array_equal(raw.cpu().numpy(), want)
    assert gfx906_fa.device_error(True) == 0


def test_move_kv_keys_only_and_edges():
    import gfx906_fa
    raw, _, k, v = layer_views(2, 4, 2, 3)
    before = raw.clone()
    one = torch.tensor([3], device=dev)
    gfx906_fa.move_kv([], [], one, one, 1)
    gfx906_fa.move_kv(k, v, one[:0], one[:0], 1)
    gfx906_fa.move_kv(k, v, one, one, 1)                # onto itself
    gfx906_fa.move_kv(k, v, one, one + 64, 1)           # past the cache
    assert gfx906_fa.device_error(True) == 8
    assert torch.equal(raw, before)
    gfx906_fa.move_kv(k, [], one, one + 20, 1)
    assert torch.equal(k[1][1, 7], k[1][0, 3])
    assert torch.equal(raw[:, :, 2 * BS * 136:], before[:, :, 2 * BS * 136:])
    for bad in ((k, v[:1], one, one, 1), (k, v, one, one.repeat(2), 1), (k, v, one.int(), one.int(), 1), (k, v, one, one, 0),
                (k, v, one.repeat(3), one.repeat(3), 2), ([k[0], k[1][:2]], v, one, one, 1), (k, v, one.repeat(900), one.repeat(900), 900)):
        with pytest.raises(RuntimeError):
            gfx906_fa.move_kv(*bad)


# ---------------------------------------------------------------- copy_pages
@pytest.mark.parametrize("L,Hkv,bs,n", [(1, 1, 16, 1), (3, 8, 16, 9), (70, 2, 16, 4), (2, 3, 48, 5)])
def test_copy_pages(L, Hkv, bs, n):
    import gfx906_fa
    NB = 2 * n + 3
    raw, kv, _, _ = layer_views(L, NB, Hkv, 1, bs=bs, seed=n)
    at = torch.randperm(NB, generator=torch.Generator().manual_seed(n))
    src, dst = at[:n].clone(), at[n:2 * n].clone()
    if n > 3:
        src[1], dst[2] = -1, -1
    want = raw.clone()
    for s, d in zip(src.tolist(), dst.tolist()):
        if s >= 0 and d >= 0:
            want[:, d] = raw[:, s]
    gfx906_fa.copy_pages(kv, src.to(dev), dst.to(dev))
    assert torch.equal(raw, want)
    assert gfx906_fa.device_error(True) == 0


def test_copy_pages_odd_sizes_strides_and_refusals():
    import gfx906_fa
    base = torch.randint(0, 256, (6, 1002), dtype=torch.uint8, device=dev)
    view = base[:, 2:1000]                              # 998 bytes a page, 1002 apart, on 2-byte boundaries
    want = base.clone()
    want[4, 2:1000] = base[1, 2:1000]
    one, four = torch.tensor([1], device=dev), torch.tensor([4], device=dev)
    gfx906_fa.copy_pages([view], one, four)
    assert torch.equal(base, want)
    gfx906_fa.copy_pages([view], one, four + 2)
    assert gfx906_fa.device_error(True) == 2
    gfx906_fa.copy_pages([], one, four)
    gfx906_fa.copy_pages([view], one[:0], four[:0])
    gfx906_fa.copy_pages([view], four, four)
    assert torch.equal(base, want)
    for bad in (([view], one.int(), four.int()), ([view], one, four.repeat(2)), ([view, base], one, four), ([view.cpu()], one, four),
                ([base.view(6, 3, 334)[:, :, :300]], one, four), ([base[:, 1:1000]], one, four)):
        with pytest.raises(RuntimeError):
            gfx906_fa.copy_pages(*bad)


@pytest.mark.parametrize("mode", [1, 3])
def test_slots_past_four_gigabytes(mode):
    """Store, read back, move and copy at the end of a cache whose byte offsets need more than 32 bits."""
    import gfx906_fa
    from gfx906_fa_paged import kv_cache_views
    kv = torch.empty((72000, 2, BS, 8, D), dtype=torch.bfloat16, device=dev)
    k, v = kv_cache_views(kv, "q8_0" if mode == 3 else "fp16")
    qkv, w, pos, _, _ = store_case(40, 8, 8, torch.bfloat16, seed=5)
    d = qkv.to(dev)
    slots = torch.arange(71990 * BS + 3, 71990 * BS + 43)
    ko = torch.empty((40, 8, D), dtype=torch.bfloat16, device=dev)
    gfx906_fa.norm_rope_store_kv(d[:, :8], d[:, 8:16], d[:, 16:], w[0].to(dev), w[1].to(dev), 1e-6, pos.to(dev),
                                 cos_sin(4000, 128).float().to(dev), True, slots.to(dev), k, v, mode, key_out=ko)
    rows = np.zeros((3, BS, 8, 136), np.uint8)
    O.reshape_and_cache(to_np(ko), slots.numpy() - 71990 * BS, rows, dtype="bf16")
    want = torch.from_numpy(dequant_rows(rows.reshape(-1, 8, 136)[3:43])).float().to(dev)
    got_k, got_v = gfx906_fa.read_kv(k, v, slots.to(dev), torch.float32)
    assert torch.equal(got_k, want)
    if mode == 1:
        assert torch.equal(got_v, qkv[:, 16:].float().to(dev))
    gfx906_fa.move_kv([k], [v], slots[20:30].to(dev), slots[:10].to(dev), 10)
    moved = gfx906_fa.read_kv(k, v, slots[:10].to(dev), torch.float32)
    assert torch.equal(moved[0], want[20:30]) and torch.equal(moved[1], got_v[20:30])
    gfx906_fa.copy_pages([kv], torch.tensor([71991], device=dev), torch.tensor([71999], device=dev))
    assert torch.equal(kv.view(torch.uint8)[71999], kv.view(torch.uint8)[71991])
    assert gfx906_fa.device_error(True) == 0
