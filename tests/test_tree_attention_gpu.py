"""gfx906_fa.tree_attention against a plain 64-bit form over the dequantised cache.

Tolerance: |out - ref| <= 2e-3 + 1e-2 |ref|, the attention kernels' own bar: keys, values and weights are rounded to 16
bits once (2^-11 each for fp16, 2^-9 for bf16 values and output), a score of magnitude s moves its weight by s * 2^-11."""
import numpy as np
import pytest
import torch

import gfx906_fa_paged
from _paged import assert_close
from _tree import TreeCase

pytestmark = pytest.mark.gpu
dev = "cuda"


def check(case, what, out=None, **kw):
    import gfx906_fa
    out = case.run(**kw) if out is None else out
    ref = {"softcap": kw.get("softcap", 0.0), "window": kw.get("sliding_window", 0), "sinks": kw.get("sinks")}
    assert_close(out.float().cpu().numpy(), case.reference(**ref), what=what)
    assert gfx906_fa.device_error(True) == 0
    return out


@pytest.mark.parametrize("v_fmt", ["q8t", "f16", "bf16", "q8"])
@pytest.mark.parametrize("lens,n_q", [
    ([300], [8]),                                    # one sequence, one row tile
    ([17, 129, 1000, 640], [1, 16, 5, 21]),          # ragged, pages that end inside a tile
    ([64, 200, 33], [64, 60, 33]),                   # no context at all, and several row tiles
])
def test_formats_and_lengths(v_fmt, lens, n_q):
    dtype = torch.bfloat16 if v_fmt == "bf16" else torch.float16
    check(TreeCase(lens, n_q, 48, 8, v_fmt, seed=len(lens), dtype=dtype), f"{v_fmt} {lens}")


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (6, 1), (2, 2), (7, 7), (12, 3), (40, 4), (16, 16), (9, 9)])
def test_head_layouts(Hq, Hkv):
    check(TreeCase([150, 700], [9, 13], Hq, Hkv, "q8t", seed=Hq), f"heads {Hq}/{Hkv}")


@pytest.mark.parametrize("v_fmt", ["q8t", "f16"])
@pytest.mark.parametrize("bs", [8, 16, 32, 48])
def test_page_sizes(bs, v_fmt):
    check(TreeCase([3 * bs + 5, 500], [7, 12], 12, 2, v_fmt, bs=bs, seed=bs, dtype=torch.float16), f"pages of {bs}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_query_and_output_types(dtype):
    case = TreeCase([400, 90], [10, 10], 12, 2, "q8t", seed=3, dtype=dtype)
    check(case, f"{dtype}")
    for o in (torch.float32, torch.float16, torch.bfloat16):
        out = torch.full((20, 12, 128), 7.0, dtype=o, device=dev)
        assert case.run(out=out) is not None
        assert_close(out.float().cpu().numpy(), case.reference(), what=f"{dtype} -> {o}")


def test_strided_query_and_output():
    case = TreeCase([400, 90], [10, 3], 12, 2, "q8t", seed=4)
    wide = torch.zeros((13, 20, 136), dtype=torch.bfloat16, device=dev)
    wide[:, 4:16, :128] = case.q
    out = torch.zeros((13, 12, 131 * 2), dtype=torch.bfloat16, device=dev)
    assert_close(case.run(q=wide[:, 4:16, :128], out=out[..., :128])[:13].float().cpu().numpy(), case.reference(), what="strided")
    assert not out[..., 128:].any()


@pytest.mark.parametrize("v_fmt", ["q8t", "f16"])
def test_long_context_is_split(v_fmt):
    check(TreeCase([20011, 3], [16, 3], 12, 2, v_fmt, seed=5, dtype=torch.float16), "long context")


@pytest.mark.parametrize("n", [31, 32, 33, 64, 65, 100])
def test_word_boundaries_of_the_bit_rows(n):
    check(TreeCase([n + 70, n], [n, n], 6, 1, "q8t", seed=n), f"{n} drafts")


@pytest.mark.parametrize("v_fmt", ["q8t", "f16"])
@pytest.mark.parametrize("kw", [dict(softcap=20.0), dict(sliding_window=100), dict(sliding_window=300, softcap=15.0),
                                dict(sliding_window=33)])
def test_softcap_and_window(kw, v_fmt):
    check(TreeCase([450, 129, 60, 2000], [12, 5, 30, 40], 12, 2, v_fmt, seed=6, dtype=torch.float16), str(kw), **kw)


def test_sinks():
    sinks = torch.linspace(-3, 3, 12, device=dev)
    case = TreeCase([450, 129, 20], [12, 5, 20], 12, 2, "q8t", seed=7)
    out = case.run(sinks=sinks)
    assert_close(out.float().cpu().numpy(), case.reference(sinks=sinks.cpu().numpy()), what="sinks")
    long = TreeCase([15000], [12], 12, 2, "q8t", seed=7)
    out = long.run(sinks=sinks)
    assert_close(out.float().cpu().numpy(), long.reference(sinks=sinks.cpu().numpy()), what="sinks, split")


def test_rows_that_see_nothing():
    """No context and empty bit rows: zeros, with and without a sink; with a context the row sees just that."""
    seen = [np.zeros((6, 6), bool), np.eye(5, dtype=bool)]
    seen[0][2, 0] = seen[0][2, 2] = True
    case = TreeCase([6, 140], [6, 5], 12, 2, "q8t", seed=8, seen=seen)
    out = check(case, "empty rows")
    assert not out[[0, 1, 3, 4, 5]].any()
    assert not case.run(sinks=torch.ones(12, device=dev))[[0, 1, 3, 4, 5]].any()
    hidden = TreeCase([100], [4], 12, 2, "f16", seed=8, seen=[np.zeros((4, 4), bool)], dtype=torch.float16)
    check(hidden, "context only")


def test_arbitrary_bits_and_bits_past_the_tree():
    rng = np.random.default_rng(0)
    seen = [rng.random((40, 40)) < 0.3, rng.random((9, 9)) < 0.5]
    case = TreeCase([340, 109], [40, 9], 12, 2, "q8t", seed=9, seen=seen)
    check(case, "any bits")
    case.mask[40:, 0] |= -512                          # every bit from draft 9 on
    case.mask[40:, 1] = -1
    check(case, "bits past the tree are ignored")
    wide = torch.full((49, 5), -1, dtype=torch.int32, device=dev)
    wide[:, 1:3] = case.mask
    case.mask = wide[:, 1:3]
    check(case, "strided rows")


@pytest.mark.parametrize("v_fmt", ["q8t", "f16", "bf16", "q8"])
def test_cache_rows_past_the_end_and_masked_drafts_may_hold_anything(v_fmt):
    """Slots past the sequence and drafts outside a row's path hold NaN and infinity: no row that does not see them changes."""
    import gfx906_fa
    dtype = torch.bfloat16 if v_fmt == "bf16" else torch.float16
    seen = [np.tril(np.ones((6, 6), bool)), np.tril(np.ones((3, 3), bool))]
    seen[0][:, 2] = False
    seen[0][2, 2] = True                             # draft 2: a branch of its own
    case = TreeCase([86, 13], [6, 3], 12, 2, v_fmt, seed=10, dtype=dtype, seen=seen)
    ref = case.reference()
    bad_k = torch.full((1, 2, 128), 60000.0, dtype=dtype, device=dev)
    bad_v = torch.full((1, 2, 128), float("inf"), dtype=dtype, device=dev)
    mode = {"q8t": 3, "q8": 2}.get(v_fmt, 1)
    bt = case.block_table.numpy()

    def poison(b, pos):
        slot = torch.tensor([int(bt[b, pos // 16]) * 16 + pos % 16], device=dev)
        gfx906_fa.store_kv(bad_k, bad_v, slot, case.k_cache, case.v_cache, mode)
        k = case.k_cache.view(-1, 2, 136)            # a NaN scale as well
        k[slot, :, :2] = 255

    for pos in range(86, 96):
        poison(0, pos)
    for pos in range(13, 16):
        poison(1, pos)
    assert_close(case.run().float().cpu().numpy(), ref, what="past the end")
    poison(0, 80 + 2)
    out = case.run().float().cpu().numpy()
    rows = [0, 1, 3, 4, 5, 6, 7, 8]
    assert_close(out[rows], ref[rows], what="masked draft")
    assert not np.isfinite(out[2]).any(axis=-1).all()


def test_no_drafts_and_empty_batches():
    import gfx906_fa
    case = TreeCase([200, 90, 40], [5, 0, 7], 12, 2, "q8t", seed=11)
    check(case, "a sequence without drafts")
    out = gfx906_fa.tree_attention(case.q[:0], case.k_cache, case.v_cache, case.bt, case.lens,
                                   torch.zeros(4, dtype=torch.int32, device=dev), case.mask[:0], 5, 200, case.scale)
    assert out.shape == (0, 12, 128)


def test_rows_beyond_the_batch_are_left_alone():
    case = TreeCase([200], [5], 12, 2, "q8t", seed=12)
    out = torch.full((9, 12, 128), 3.0, dtype=torch.bfloat16, device=dev)
    case.run(out=out)
    assert (out[5:] == 3.0).all()


def test_bad_pages_are_dropped_and_reported():
    import gfx906_fa
    for bad in (-1, 10 ** 6):
        case = TreeCase([200, 300], [5, 9], 12, 2, "q8t", seed=13)
        case.block_table[1, 4] = bad
        case.block_table[1, 11] = bad
        case.bt = case.block_table.to(dev)
        out = case.run()
        assert_close(out.float().cpu().numpy(), case.reference(), what=f"page {bad}")
        assert gfx906_fa.device_error(True) == 2


def test_one_draft_equals_decode():
    import gfx906_fa
    case = TreeCase([900, 33, 5000], [1, 1, 1], 48, 8, "q8t", seed=14)
    ref = gfx906_fa.paged_attention(case.q, case.k_cache, case.v_cache, case.bt, case.lens, case.start, 1, 5000, case.scale)
    assert_close(case.run().float().cpu().numpy(), ref.float().cpu().numpy(), what="decode")


def test_chain_through_forward_paged():
    import gfx906_fa
    n = 11
    case = TreeCase([900, 33], [n, n], 12, 2, "q8t", seed=15, seen=[np.tril(np.ones((n, n), bool))] * 2)
    ref = gfx906_fa.paged_attention(case.q, case.k_cache, case.v_cache, case.bt, case.lens, case.start, n, 900, case.scale)
    out = gfx906_fa_paged.forward_paged(case.q, None, case.v_cache, case.bt, case.lens, case.start, n, 900, scale=case.scale,
                                        key_cache_q8=case.k_cache, tree_mask=case.mask)
    assert out.dtype == torch.float32 and out.shape == (2 * n, 12 * 128)
    assert_close(out.view(2 * n, 12, 128).cpu().numpy(), ref.float().cpu().numpy(), what="chain")


def test_fp8_output():
    case = TreeCase([200, 90], [5, 4], 12, 2, "q8t", seed=16)
    scale = torch.tensor([0.01], device=dev)
    out = torch.empty((9, 12, 128), dtype=torch.float8_e4m3fn, device=dev)
    case.run(out=out, output_scale=scale)
    ref = np.clip(case.reference() / 0.01, -448, 448)
    # e4m3 keeps 4 significant bits (half a step: 2^-4 of the value, 2^-10 below the smallest normal) on top of the kernel's
    # own 2e-3 + 1e-2 |o|, which the scale of 0.01 makes 0.2 + 1e-2 |ref|
    bound = np.abs(ref) * (1 / 16 + 1e-2 * 17 / 16) + 0.2 * 17 / 16 + 2.0 ** -10
    assert (np.abs(out.float().cpu().numpy() - ref) <= bound).all()


def test_another_stream_and_a_captured_graph():
    case = TreeCase([3000, 90], [16, 4], 12, 2, "q8t", seed=17)
    ref = case.reference()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = case.run()
    torch.cuda.current_stream().wait_stream(s)
    assert_close(side.float().cpu().numpy(), ref, what="side stream")
    out = torch.empty_like(case.q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        case.run(out=out)
    for _ in range(2):
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert_close(out.float().cpu().numpy(), ref, what="graph")


def test_the_same_call_gives_the_same_bits():
    case = TreeCase([20000, 700, 90], [16, 30, 4], 48, 8, "q8t", seed=18)
    a = case.run()
    assert torch.equal(a, case.run())


def test_refusals():
    import gfx906_fa
    case = TreeCase([200, 90], [5, 4], 12, 2, "q8t", seed=19)

    def call(**over):
        a = dict(query=case.q, key_cache_q8=case.k_cache, value_cache=case.v_cache, block_table=case.bt, seq_lens=case.lens,
                 query_start_loc=case.start, tree_mask=case.mask, max_query_len=5, max_seq_len=200, scale=case.scale)
        return gfx906_fa.tree_attention(**{**a, **over})

    for over in (dict(query=case.q.cpu()), dict(query=case.q[..., :64]), dict(query=case.q[:, :11]),
                 dict(tree_mask=case.mask.long()), dict(tree_mask=case.mask[:3]), dict(tree_mask=case.mask.cpu()),
                 dict(max_query_len=33), dict(query_start_loc=case.start[:2]), dict(seq_lens=case.lens.long()),
                 dict(block_table=case.bt[:1]), dict(out=torch.empty((3, 12, 128), device=dev)),
                 dict(out=torch.empty((9, 12, 128), dtype=torch.float8_e4m3fn, device=dev)), dict(softcap=-1.0),
                 dict(sliding_window=-1), dict(sinks=torch.zeros(3, device=dev)), dict(max_seq_len=-1),
                 dict(value_cache=case.v_cache[:-1])):
        with pytest.raises(RuntimeError):
            call(**over)
    call()


def test_many_short_sequences():
    """More sequences than a prefix-sum chunk, some without drafts."""
    rng = np.random.default_rng(20)
    n_q = [int(x) for x in rng.integers(0, 5, 1100)]
    lens = [n + int(x) for n, x in zip(n_q, rng.integers(0, 40, 1100))]
    check(TreeCase(lens, n_q, 4, 2, "q8t", seed=20), "1100 sequences")


@pytest.mark.parametrize("v_fmt", ["q8t", "f16"])
@pytest.mark.parametrize("rows", [16, 40])
def test_scores_that_jump(rows, v_fmt):
    """Every 64 keys score at a level of their own, up to 15 nats apart, so that the running maximum rises by more than the
    lazy threshold in first and second halves of tiles: the accumulator, and weights already written, are scaled down.
    (15 nats of score err by 15 * 2^-12 from the keys' rounding, the same way in every element: 0.4 %.)"""
    import gfx906_fa
    B, L = 60, 1500
    case = TreeCase([L] * B, [rows] * B, 6, 1, v_fmt, seed=21, dtype=torch.float16)
    g = torch.Generator().manual_seed(1)
    level = (torch.rand((B, L // 64 + 1), generator=g) * 1.3).repeat_interleave(64, 1)[:, :L]
    key = (level.reshape(-1, 1, 1) * torch.ones(B * L, 1, 128)).half()
    val = torch.randn((B * L, 1, 128), generator=g).half()
    pos = torch.arange(L)
    slots = (case.block_table[:, pos // 16].long() * 16 + pos % 16).flatten()
    gfx906_fa.store_kv(key.to(dev), val.to(dev), slots.to(dev), case.k_cache, case.v_cache, 3 if v_fmt == "q8t" else 1)
    case.q = (1 + 0.05 * torch.randn(case.q.shape, generator=g)).half().to(dev)
    check(case, "jumps")


def test_lengths_past_the_table_or_the_bound_are_clamped():
    case = TreeCase([300, 200], [4, 4], 12, 2, "q8t", seed=22)
    short = TreeCase([304, 200], [4, 4], 12, 2, "q8t", seed=22)
    lens = short.lens.clone()
    lens[0] = 5000                                     # the table holds 19 pages: 304 keys
    case = short
    case.lens = lens
    assert_close(case.run().float().cpu().numpy(), case.reference(), what="clamped to the table")


@pytest.mark.parametrize("bits", [1, 2])
def test_caches_the_tensor_core_kernel_cannot_read(bits):
    """Rows on 2-byte boundaries only."""
    case = TreeCase([210, 40], [9, 5], 12, 2, "q8", seed=23)
    ref = case.reference()
    for name in ("k_cache", "v_cache"):
        c = getattr(case, name)
        wide = torch.zeros((*c.shape[:3], 138), dtype=torch.uint8, device=dev)
        wide[..., :136] = c
        if bits == 1 or name == "k_cache":
            setattr(case, name, wide[..., :136])
    assert_close(case.run().float().cpu().numpy(), ref, what="2-byte rows")


def test_backend_cache_views():
    """The views of one vLLM allocation: K rows and V records share each page's K half."""
    import gfx906_fa
    for v_fmt, mode, fmt in (("q8_0", 3, "q8t"), ("fp16", 1, "bf16")):
        case = TreeCase([500, 77], [12, 7], 16, 8, fmt, seed=24)
        ref = case.reference()
        kv = torch.full((case.NB, 2, 16, 8, 128), float("nan"), dtype=torch.bfloat16, device=dev)
        k, v = gfx906_fa_paged.kv_cache_views(kv, v_fmt)
        k.copy_(case.k_cache)
        v.copy_(case.v_cache)
        case.k_cache, case.v_cache = k, v
        assert_close(case.run().float().cpu().numpy(), ref, what=v_fmt)
        assert gfx906_fa.device_error(True) == 0


def test_a_visible_key_that_is_not_a_number_shows():
    import gfx906_fa
    case = TreeCase([700], [6], 6, 1, "q8t", seed=25)
    slot = int(case.block_table[0, 3]) * 16 + 5
    case.k_cache.view(-1, 136)[slot, :2] = 255         # a NaN scale in the context
    assert np.isnan(case.run().float().cpu().numpy()).all()
    assert gfx906_fa.device_error(True) == 0


def test_zero_and_negative_scale():
    for scale in (0.0, -0.05):
        case = TreeCase([333, 20], [6, 9], 12, 2, "q8t", seed=26)
        import gfx906_fa
        out = gfx906_fa.tree_attention(case.q, case.k_cache, case.v_cache, case.bt, case.lens, case.start, case.mask, 9, 333, scale)
        type(case).scale = property(lambda self, s=scale: s)
        try:
            assert_close(out.float().cpu().numpy(), case.reference(), what=f"scale {scale}")
        finally:
            del type(case).scale


@pytest.mark.parametrize("v_fmt", ["q8t", "f16"])
def test_pages_past_four_gigabytes(v_fmt):
    """The same pages at the end of a cache whose byte offsets need more than 32 bits."""
    case = TreeCase([900, 130], [16, 9], 48, 8, v_fmt, seed=27, dtype=torch.float16)
    ref = case.reference()
    kv = torch.empty((72000, 2, 16, 8, 128), dtype=torch.float16, device=dev)         # 65536 bytes a page
    k, v = gfx906_fa_paged.kv_cache_views(kv, "q8_0" if v_fmt == "q8t" else "fp16")
    first = kv.shape[0] - case.NB
    assert first * 65536 > 2 ** 32
    k[first:] = case.k_cache
    v[first:] = case.v_cache
    case.k_cache, case.v_cache = k, v
    case.bt = torch.where(case.bt >= 0, case.bt + first, case.bt)
    assert_close(case.run().float().cpu().numpy(), ref, what="far pages")


@pytest.mark.parametrize("v_fmt", ["q8_0", "fp16"])
def test_backend_forward_with_a_tree(v_fmt):
    """Gfx906FAImpl.forward takes the bit rows from its metadata; the legacy mode, which has no Q8_0 cache, refuses them."""
    pytest.importorskip("vllm")
    import gfx906_fa_backend as be
    case = TreeCase([500, 77], [12, 7], 48, 8, "q8t" if v_fmt == "q8_0" else "bf16", seed=28)
    kv = torch.zeros((case.NB, 2, 16, 8, 128), dtype=torch.bfloat16, device=dev)
    k, v = gfx906_fa_paged.kv_cache_views(kv, v_fmt)
    k.copy_(case.k_cache)
    v.copy_(case.v_cache)
    impl = be.Gfx906FAImpl(num_heads=48, head_size=128, scale=case.scale, num_kv_heads=8, alibi_slopes=None, sliding_window=None,
                           kv_cache_dtype="auto")
    impl._v_fmt, impl._legacy = v_fmt, False
    meta = be.Gfx906FAMetadata(num_actual_tokens=19, max_query_len=12, max_seq_len=500, query_start_loc=case.start,
                               seq_lens=case.lens, block_table=case.bt, slot_mapping=torch.zeros(19, dtype=torch.int64, device=dev),
                               tree_mask=case.mask)
    out = torch.zeros((19, 48 * 128), dtype=torch.bfloat16, device=dev)
    impl.forward(None, case.q, None, None, kv, meta, output=out)
    assert_close(out.view(19, 48, 128).float().cpu().numpy(), case.reference(), what="backend")
    impl._legacy = True
    with pytest.raises(NotImplementedError):
        impl.forward(None, case.q, None, None, kv, meta, output=out)
