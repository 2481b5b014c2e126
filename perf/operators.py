"""Measured cases of the draft-tree operators: what one verify step of tree speculation runs over the paged Q8_0 cache.

  tree_mask           parent links of the drafted tokens -> ancestor bit rows and rotary positions
  norm_rope_store_kv  per-head RMS norm + rotation of queries and keys, Q8_0 store of keys and values (read_kv reads the rows back)
  tree_attention      attention of the drafted tokens over their context and their own ancestors
  move_kv             cache rows of the accepted path moved together, every layer at once
  copy_pages          pages copied for a forked sequence, every layer at once

`own` False: plain torch in 32 bits.  `own` True: the calls a user makes of `gfx906_fa`.  Page 0 of every cache is the null
page, as vLLM keeps it: no sequence owns it."""
import os
import sys

import torch

own = False

D = 128                      # head size
RB = D // 32 * 34            # bytes of a Q8_0 row
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
DEV = "cuda"


def _ops():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gfx906-fa-vllm_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import gfx906_fa
    return gfx906_fa


# ------------------------------------------------------------------ cases
def listed():
    return [
        # ancestor bits of one sequence's 16-token draft tree: pure launch latency
        dict(name="mask one", op="mask", seqs=1, tokens=16, ctx=900),
        # a serving batch: 256 sequences, up to 64 drafts each, ragged
        dict(name="mask batch", op="mask", seqs=256, tokens=64, ctx=4000),
        # one sequence's 16 drafts of a 48/8-head layer: the smallest store
        dict(name="store one", op="store", tokens=16, run=16, hq=48, hkv=8, rot=128, neox=True, v="q8t", dtype="bf16", ctx=8000),
        # 64 sequences of up to 33 drafts, GPT-J pairs over half the head, 16-bit V, odd token count
        dict(name="store batch", op="store", tokens=2111, run=33, hq=48, hkv=8, rot=64, neox=False, v="v16", dtype="fp16", ctx=32768),
        # a prompt chunk that fills the cache before drafting starts
        dict(name="store prompt", op="store", tokens=16384, run=16384, hq=48, hkv=8, rot=128, neox=True, v="q8t", dtype="bf16", ctx=32768),
        # one sequence, short context, small tree: latency of one layer
        dict(name="attention one", op="attention", seqs=1, lo=2047, hi=2047, tokens=8, hq=48, hkv=8, v="q8t", dtype="bf16",
             softcap=0.0, window=0),
        # a decode batch with 16-token trees, contexts of 1K to 32K
        dict(name="attention batch", op="attention", seqs=32, lo=1024, hi=32768, tokens=16, hq=48, hkv=8, v="q8t", dtype="bf16",
             softcap=0.0, window=0),
        # wide trees (up to 60 drafts, 360 rows a kv head), 16-bit V, ragged
        dict(name="attention wide", op="attention", seqs=8, lo=4001, hi=16383, tokens=60, hq=48, hkv=8, v="v16", dtype="fp16",
             softcap=0.0, window=0),
        # one sequence keeps up to 5 of 16 drafts in a 32-layer model
        dict(name="move one", op="move", seqs=1, tokens=16, keep=5, layers=32, hkv=8, v="q8t", ctx=900),
        # 128 sequences keep up to 8 of 48 drafts each, 16-bit V
        dict(name="move batch", op="move", seqs=128, tokens=48, keep=8, layers=32, hkv=8, v="v16", ctx=300),
        # a fork copies the last, partly filled page of one sequence in 32 layers
        dict(name="pages one", op="pages", pages=1, pool=64, layers=32, hkv=8),
        # a beam step or a swap: 500 pages in 16 layers
        dict(name="pages many", op="pages", pages=500, pool=1200, layers=16, hkv=8),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["mask", "store", "store", "attention", "attention", "attention", "move", "pages"])
    hkv = rng.choice([1, 2, 4, 8])
    if op == "mask":
        return dict(op=op, seqs=_log(rng, 1, 256), tokens=_log(rng, 2, 64), ctx=_log(rng, 64, 32768))
    if op == "store":
        tokens = _log(rng, 1, 16384)
        return dict(op=op, tokens=tokens, run=_log(rng, 1, tokens) if tokens > 1 else 1, hq=hkv * rng.randint(1, 6), hkv=hkv, rot=rng.choice([32, 64, 96, 128]),
                    neox=rng.random() < 0.6, v=rng.choice(["q8t", "v16"]), dtype=rng.choice(["bf16", "fp16"]),
                    ctx=_log(rng, 512, 32768))
    if op == "attention":
        hi = _log(rng, 65, 32768)
        seqs = max(1, min(_log(rng, 1, 96), 32 * 32768 // hi))
        lo = max(1, int(hi * rng.random()))
        tokens = max(1, min(_log(rng, 1, 64), 16 * 32 * 32768 // (seqs * hi), hi))
        return dict(op=op, seqs=seqs, lo=max(lo, tokens), hi=hi, tokens=tokens, hq=hkv * rng.randint(1, 6), hkv=hkv,
                    v=rng.choice(["q8t", "v16"]), dtype=rng.choice(["bf16", "fp16"]), softcap=rng.choice([0.0, 0.0, 0.0, 30.0]),
                    window=rng.choice([0, 0, 0, _log(rng, 200, 8000)]))
    if op == "move":
        tokens = _log(rng, 4, 64)
        return dict(op=op, seqs=_log(rng, 1, 128), tokens=tokens, keep=rng.randint(1, max(2, tokens // 4)),
                    layers=rng.choice([8, 16, 32]), hkv=hkv, v=rng.choice(["q8t", "v16"]), ctx=_log(rng, 16, 300))
    pages = _log(rng, 1, 500)
    return dict(op=op, pages=pages, pool=2 * pages + rng.randint(8, 200), layers=_log(rng, 4, 16), hkv=hkv)


# ------------------------------------------------------------------ shapes that follow from a case alone
def _spread(lo, hi, n, mul=7):
    """n whole numbers of lo..hi, evenly spread, in a mixed order that depends on nothing else."""
    if n == 1:
        return [hi]
    while n % mul == 0:
        mul += 2
    return [lo + (hi - lo) * ((i * mul) % n) // (n - 1) for i in range(n)]


def _lens(case):
    """(drafts, length with the drafts) of each sequence."""
    n = _spread(max(1, case["tokens"] // 2), case["tokens"], case["seqs"], 5)
    if case["op"] == "attention":
        total = _spread(case["lo"], case["hi"], case["seqs"])
    else:
        total = [c + k for c, k in zip(_spread(max(1, case["ctx"] // 2), case["ctx"], case["seqs"]), n)]
    return n, total


def _starts(n):
    at = [0]
    for x in n:
        at.append(at[-1] + x)
    return at


def work(case):
    op = case["op"]
    if op == "mask":
        n, _ = _lens(case)
        words = -(-max(n) // 32)
        return {"bytes": sum(n) * (4 + 4 * words + 8) + 8 * len(n), "flops": sum(n)}
    if op == "store":
        t, hq, hkv = case["tokens"], case["hq"], case["hkv"]
        v = RB if case["v"] == "q8t" else 2 * D
        stored = t * hkv * (RB + v)
        # queries in and out, keys and values in, the cache rows out, and the same rows read back as 16-bit values
        return {"bytes": t * (2 * hq + 2 * hkv) * 2 * D + stored * 2 + t * hkv * 4 * D + t * 24,
                "flops": t * (hq + hkv) * D * 8}
    if op == "attention":
        n, total = _lens(case)
        v = RB if case["v"] == "q8t" else 2 * D
        window = case["window"] or 1 << 30
        seen = [min(L, window + k) for k, L in zip(n, total)]
        pairs = sum(k * min(L - k + 1, window) for k, L in zip(n, total))
        return {"bytes": sum(seen) * case["hkv"] * (RB + v) + sum(n) * case["hq"] * 4 * D + sum(-(-L // 16) * 4 for L in total),
                "flops": 4 * D * case["hq"] * pairs}
    if op == "move":
        n, _ = _lens(case)
        v = RB if case["v"] == "q8t" else 2 * D
        rows = sum(min(case["keep"], k) for k in n)
        return {"bytes": rows * case["layers"] * case["hkv"] * (RB + v) * 2 + rows * 16, "flops": 0}
    return {"bytes": 2 * case["pages"] * case["layers"] * 2 * 16 * case["hkv"] * D * 2 + case["pages"] * 16, "flops": 0}


# ------------------------------------------------------------------ inputs
def _views(kv, v):
    """The framework's views of one KV allocation [NB, 2, 16, Hkv, D]: Q8_0 K rows, and V in the V half (v16) or as
    page-transposed Q8_0 records behind the K rows (q8t)."""
    nb, _, bs, hkv, d = kv.shape
    raw = kv.view(torch.uint8).view(nb, -1)
    k = raw[:, :bs * hkv * RB].view(nb, bs, hkv, RB)
    return k, raw[:, bs * hkv * RB:2 * bs * hkv * RB].view(nb, hkv, bs * RB) if v == "q8t" else kv[:, 1]


def _quantise(x):
    """Q8_0 of x [..., D]: whole numbers [..., D/32, 32] as int8, scales [..., D/32] as fp16."""
    b = x.float().reshape(*x.shape[:-1], D // 32, 32)
    d = b.abs().amax(-1) / 127.0
    inv = torch.where(d > 0, 1.0 / d, torch.zeros_like(d))
    return (b * inv[..., None]).round().clamp(-128, 127).to(torch.int8), d.half()


def _bytes_k(q, d):
    return torch.cat([d[..., None].view(torch.uint8), q.view(torch.uint8)], -1).flatten(-2)


def _fill(kv, v, g):
    """Keys (a few loud channels, as models have them) and values of every page, 1024 pages at a time."""
    k, vv = _views(kv, v)
    nb, bs, hkv = k.shape[:3]
    loud = torch.ones(D, device=DEV)
    loud[::17] = 3.0
    for i in range(0, nb, 1024):
        n = min(1024, nb - i)
        x = torch.randn((n, bs, hkv, D), device=DEV, generator=g) * loud
        k[i:i + n] = _bytes_k(*_quantise(x))
        x = torch.randn((n, bs, hkv, D), device=DEV, generator=g)
        if v == "q8t":
            q, d = _quantise(x)
            vv[i:i + n, :, :128] = d.permute(0, 2, 3, 1).contiguous().view(torch.uint8).flatten(-2)
            vv[i:i + n, :, 128:] = q.flatten(-2).permute(0, 2, 3, 1).contiguous().view(torch.uint8).flatten(-2)
        else:
            vv[i:i + n] = x.to(vv.dtype)


def _trees(n, seed):
    """Parents of each sequence's drafts (-1: the tree's root hangs on the last context token): most drafts hang on one of
    the last few, as ranked expansions of a small beam do."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for k in n:
        back = (torch.rand(k, generator=g) ** 2 * 6).long() + 1
        out.append((torch.arange(k) - back).clamp(min=-1))
    return torch.cat(out).to(torch.int32)


def _bits(parents, at):
    """Ancestor-or-self bit rows [T, words] of the trees, on the host."""
    words = -(-max(b - a for a, b in zip(at, at[1:])) // 32)
    rows, p = [], parents.tolist()
    for a, b in zip(at, at[1:]):
        seen = []
        for i in range(b - a):
            seen.append((seen[p[a + i]] if p[a + i] >= 0 else 0) | 1 << i)
        rows += [[(r >> 32 * w & 0xffffffff) - (r >> 32 * w & 0x80000000) * 2 for w in range(words)] for r in seen]
    return torch.tensor(rows, dtype=torch.int32)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op = case["op"]
    s = {"case": case}
    if op == "mask":
        n, total = _lens(case)
        s |= {"parents": _trees(n, seed).to(DEV), "start": torch.tensor(_starts(n), dtype=torch.int32, device=DEV),
              "lens": torch.tensor(total, dtype=torch.int32, device=DEV), "most": max(n)}
        return s
    if op == "store":
        t, hq, hkv, dt = case["tokens"], case["hq"], case["hkv"], DTYPES[case["dtype"]]
        qkv = torch.randn((t, hq + 2 * hkv, D), device=DEV, generator=g).to(dt)       # the projection's output, split in views
        weights = 1 + 0.2 * torch.randn((2, D), device=DEV, generator=g)
        inv = 1.0 / (1e6 ** (torch.arange(0, case["rot"], 2, device=DEV, dtype=torch.float32) / case["rot"]))
        angle = torch.outer(torch.arange(case["ctx"], device=DEV, dtype=torch.float32), inv)
        # runs of `run` tokens, one a sequence: each starts somewhere inside a page of its own and goes on through its next pages
        run, runs = case["run"], -(-t // case["run"])
        per = -(-(run + 15) // 16)
        first = torch.randint(0, 16, (runs,), device=DEV, generator=g)
        base = torch.randint(0, max(1, case["ctx"] - run), (runs,), device=DEV, generator=g)
        of, at = torch.arange(t, device=DEV) // run, torch.arange(t, device=DEV) % run
        nb = runs * per + 1
        pages = torch.randperm(nb - 1, device=DEV, generator=g) + 1
        at_slot = first[of] + at
        kv = torch.zeros((nb, 2, 16, hkv, D), dtype=dt, device=DEV)
        k, v = _views(kv, case["v"])
        slots = pages[of * per + at_slot // 16] * 16 + at_slot % 16
        s |= {"q": qkv[:, :hq], "k": qkv[:, hq:hq + hkv], "v": qkv[:, hq + hkv:], "wq": weights[0].to(dt), "wk": weights[1].to(dt),
              "pos": (base[of] + at) % case["ctx"], "cs": torch.cat([angle.cos(), angle.sin()], -1).to(dt),
              "slots": slots, "kc": k, "vc": v, "q_out": torch.empty((t, hq, D), dtype=dt, device=DEV)}
        return s
    if op == "attention":
        n, total = _lens(case)
        at, dt = _starts(n), DTYPES[case["dtype"]]
        pages = [-(-L // 16) for L in total]
        kv = torch.empty((sum(pages) + 1, 2, 16, case["hkv"], D), dtype=dt, device=DEV)
        _fill(kv, case["v"], g)
        own_pages = torch.randperm(sum(pages), device=DEV, generator=g).to(torch.int32) + 1
        table = torch.zeros((len(n), max(pages)), dtype=torch.int32, device=DEV)
        for b, (a, k) in enumerate(zip(_starts(pages), pages)):
            table[b, :k] = own_pages[a:a + k]
        k, v = _views(kv, case["v"])
        s |= {"q": torch.randn((sum(n), case["hq"], D), device=DEV, generator=g).to(dt), "kc": k, "vc": v, "table": table,
              "lens": torch.tensor(total, dtype=torch.int32, device=DEV), "start": torch.tensor(at, dtype=torch.int32, device=DEV),
              "mask": _bits(_trees(n, seed), at).to(DEV), "most": max(n), "longest": max(total), "scale": D ** -0.5,
              "out": torch.empty((sum(n), case["hq"], D), dtype=dt, device=DEV)}
        return s
    if op == "move":
        n, total = _lens(case)
        pages = [-(-L // 16) for L in total]
        kv = torch.randint(-2 ** 31, 2 ** 31 - 1, (case["layers"], sum(pages) + 1, 16 * case["hkv"] * D), dtype=torch.int32, device=DEV,
                           generator=g)
        own_pages = torch.randperm(sum(pages), device=DEV, generator=g).cpu() + 1
        host = torch.Generator().manual_seed(seed)
        src, dst, first = [], [], _starts(pages)
        for b, (k, L) in enumerate(zip(n, total)):
            keep = min(case["keep"], k)
            path = torch.randperm(k, generator=host)[:keep].sort().values.tolist()
            row = own_pages[first[b]:first[b + 1]]
            slot = lambda i: int(row[i // 16]) * 16 + i % 16  # noqa: E731
            kept = keep - (b % 3 == 2)                           # a shorter path: its row is padded with -1
            src += [slot(L - k + i) for i in path[:kept]] + [-1] * (case["keep"] - kept)
            dst += [slot(L - k + i) for i in range(kept)] + [-1] * (case["keep"] - kept)
        layers = [x.view(torch.bfloat16).view(-1, 2, 16, case["hkv"], D) for x in kv]
        views = [_views(x, case["v"]) for x in layers]
        s |= {"kv": kv, "kc": [k for k, _ in views], "vc": [v for _, v in views], "src": torch.tensor(src, device=DEV),
              "dst": torch.tensor(dst, device=DEV), "per": case["keep"]}
        return s
    kv = torch.randint(-2 ** 31, 2 ** 31 - 1, (case["layers"], case["pool"], 16 * case["hkv"] * D), dtype=torch.int32, device=DEV,
                       generator=g)
    at = torch.randperm(case["pool"] - 1, device=DEV, generator=g) + 1
    s |= {"kv": kv, "caches": [x.view(torch.bfloat16).view(-1, 2, 16, case["hkv"], D) for x in kv],
          "src": at[:case["pages"]].contiguous(), "dst": at[case["pages"]:2 * case["pages"]].contiguous()}
    return s


# ------------------------------------------------------------------ plain forms
def _plain_mask(s):
    """Ancestor closure by doubling: after i steps `reach` holds the ancestors up to 2^i - 1 links away."""
    start, lens, most, words = s["start"].long(), s["lens"].long(), s["most"], -(-s["most"] // 32)
    n = start[1:] - start[:-1]
    t = torch.arange(s["parents"].numel(), device=DEV)
    b = torch.bucketize(t, start[1:], right=True)
    i = t - start[b]
    up = torch.zeros((n.numel(), most + 1, most + 1), device=DEV)              # column `most` stands for the context
    parent = s["parents"].long()
    up[b, i, torch.where(parent < 0, most, parent)] = 1
    reach = torch.eye(most + 1, device=DEV).expand_as(up)
    for _ in range(most.bit_length()):
        reach = ((reach + up @ reach) > 0).float()
        up = up @ up
    seen = reach[b, i][:, :most] > 0
    depth = seen.sum(-1) - 1
    bit = torch.arange(words * 32, device=DEV)
    seen = torch.cat([seen, seen.new_zeros((t.numel(), words * 32 - most))], 1)
    packed = (seen.long() << bit % 32).view(-1, words, 32).sum(-1)
    return torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32), (lens - n)[b] + depth


def _norm_rope(x, w, pos, cs, neox):
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.float()
    rot = cs.shape[1]
    c, z = cs[pos].float()[:, None, :rot // 2], cs[pos].float()[:, None, rot // 2:]
    head, rest = x[..., :rot], x[..., rot:]
    a, b = (head[..., :rot // 2], head[..., rot // 2:]) if neox else (head[..., 0::2], head[..., 1::2])
    y = torch.stack([a * c - b * z, b * c + a * z], -2 if neox else -1).flatten(-2)
    return torch.cat([y, rest], -1)


def _dequant_k(rows):
    b = rows.unflatten(-1, (D // 32, 34))
    return (b[..., 2:].contiguous().view(torch.int8).float() * b[..., :2].contiguous().view(torch.float16).float()).flatten(-2)


def _plain_store(s):
    case, dt = s["case"], s["q"].dtype
    q = _norm_rope(s["q"], s["wq"], s["pos"], s["cs"], case["neox"]).to(dt)
    k = _norm_rope(s["k"], s["wk"], s["pos"], s["cs"], case["neox"]).to(dt)
    page, off = s["slots"] // 16, s["slots"] % 16
    s["kc"][page, off] = _bytes_k(*_quantise(k))
    k = _dequant_k(s["kc"][page, off]).to(dt)
    if case["v"] != "q8t":
        s["vc"][page, off] = s["v"]
        return q, k, s["vc"][page, off]
    w, d = _quantise(s["v"])
    scales = s["vc"][..., :128].unflatten(-1, (4, 16, 2))
    whole = s["vc"][..., 128:].unflatten(-1, (D, 16))
    scales[page, :, :, off] = d[..., None].view(torch.uint8)
    whole[page, :, :, off] = w.flatten(-2).view(torch.uint8)
    d = scales[page, :, :, off].contiguous().view(torch.float16).float()
    w = whole[page, :, :, off].contiguous().view(torch.int8).float().unflatten(-1, (4, 32))
    return q, k, (w * d).flatten(-2).to(dt)


def _plain_attention(s):
    case, start, lens = s["case"], s["start"].long(), s["lens"].long()
    seqs, hkv, group = lens.numel(), case["hkv"], case["hq"] // case["hkv"]
    table = s["table"].long()
    k = _dequant_k(s["kc"][table]).flatten(1, 2)                              # [B, L, Hkv, D]
    if case["v"] == "q8t":
        rec = s["vc"][table]                                                  # [B, pages, Hkv, record]
        d = rec[..., :128].contiguous().view(torch.float16).float().unflatten(-1, (4, 1, 16))
        v = rec[..., 128:].view(torch.int8).float().unflatten(-1, (4, 32, 16)) * d
        v = v.flatten(-3, -2).permute(0, 1, 4, 2, 3).flatten(1, 2)
    else:
        v = s["vc"][table].float().flatten(1, 2)
    n = start[1:] - start[:-1]
    most, longest = s["most"], k.shape[1]
    i = torch.arange(most, device=DEV)
    t = (start[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)                 # [B, most]
    q = s["q"][t].float().unflatten(2, (hkv, group))
    bits = s["mask"][t]                                                       # [B, most, words]
    tree = (bits[..., i // 32] >> i % 32 & 1) > 0                             # [B, most, most]
    depth = tree.sum(-1) - 1
    ctx = (lens - n)[:, None, None]
    key = torch.arange(longest, device=DEV)
    draft = (key - ctx).clamp(0, most - 1).expand(seqs, most, longest)
    near = ctx + depth[..., None] - key < (case["window"] or 1 << 30)
    seen = torch.where(key < ctx, near, tree.gather(-1, draft) & (key < lens[:, None, None]))
    score = torch.einsum("bnhgd,blhd->bhgnl", q, k) * s["scale"]
    if case["softcap"]:
        score = case["softcap"] * torch.tanh(score / case["softcap"])
    seen = seen[:, None, None]
    score = torch.where(seen, score, torch.full_like(score, -torch.inf))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top > -torch.inf, top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    o = torch.einsum("bhgnl,blhd->bnhgd", p, v).flatten(2, 3)
    there = torch.bucketize(torch.arange(s["q"].shape[0], device=DEV), start[1:], right=True)
    return o[there, torch.arange(s["q"].shape[0], device=DEV) - start[there]].to(s["q"].dtype)


def _plain_move(s):
    case = s["case"]
    skip = (s["src"] < 0) | (s["dst"] < 0)
    src, dst = (torch.where(skip, torch.zeros_like(x), x) for x in (s["src"], s["dst"]))      # skipped: the null page's slot 0 to itself
    raw = s["kv"].view(torch.uint8)
    half = 16 * case["hkv"] * RB
    k = raw[..., :half].unflatten(-1, (16, case["hkv"], RB))
    k[:, dst // 16, dst % 16] = k[:, src // 16, src % 16]
    if case["v"] != "q8t":
        v = raw[..., raw.shape[-1] // 2:].unflatten(-1, (16, case["hkv"], 2 * D))
        v[:, dst // 16, dst % 16] = v[:, src // 16, src % 16]
        return s["kv"]
    rec = raw[..., half:2 * half].unflatten(-1, (case["hkv"], 16 * RB))
    scales, whole = rec[..., :128].unflatten(-1, (4, 16, 2)), rec[..., 128:].unflatten(-1, (D, 16))
    scales[:, dst // 16, :, :, dst % 16] = scales[:, src // 16, :, :, src % 16]
    whole[:, dst // 16, :, :, dst % 16] = whole[:, src // 16, :, :, src % 16]
    return s["kv"]


def _plain_pages(s):
    s["kv"][:, s["dst"]] = s["kv"][:, s["src"]]
    return s["kv"]


# ------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        return {"mask": _plain_mask, "store": _plain_store, "attention": _plain_attention, "move": _plain_move, "pages": _plain_pages}[op](s)
    fa = _ops()
    if op == "mask":
        return fa.tree_mask(s["parents"], s["start"], s["lens"], s["most"])
    if op == "store":
        mode = 3 if case["v"] == "q8t" else 1
        fa.norm_rope_store_kv(s["q"], s["k"], s["v"], s["wq"], s["wk"], 1e-6, s["pos"], s["cs"], case["neox"], s["slots"], s["kc"],
                              s["vc"], mode, query_out=s["q_out"])
        k, v = fa.read_kv(s["kc"], s["vc"], s["slots"], s["q"].dtype)
        return s["q_out"], k, v
    if op == "attention":
        return fa.tree_attention(s["q"], s["kc"], s["vc"], s["table"], s["lens"], s["start"], s["mask"], s["most"], s["longest"],
                                 s["scale"], out=s["out"], softcap=case["softcap"], sliding_window=case["window"])
    if op == "move":
        fa.move_kv(s["kc"], s["vc"], s["src"], s["dst"], s["per"])
        return s["kv"]
    fa.copy_pages(s["caches"], s["src"], s["dst"])
    return s["kv"]


# ------------------------------------------------------------------ 64 bits
def _exact_norm_rope(x, w, pos, cs, neox):
    y = x.double()
    y = y / ((y ** 2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
    half = cs.shape[1] // 2
    j = torch.arange(half, device=DEV)
    a, b = (j, j + half) if neox else (2 * j, 2 * j + 1)
    c, z = cs[pos][:, None, :half].double(), cs[pos][:, None, half:].double()
    out = y.clone()
    out[..., a] = y[..., a] * c - y[..., b] * z
    out[..., b] = y[..., a] * z + y[..., b] * c
    return out


def _exact_q8(x):
    """What x [..., D] stands for once it is held as Q8_0."""
    b = x.double().unflatten(-1, (D // 32, 32))
    top = b.abs().amax(-1, keepdim=True)
    whole = (b * 127 / top.clamp(min=1e-300)).round()
    return (whole * (top / 127).half().double()).flatten(-2)


def exact(case, seed):
    if case["op"] not in ("store", "attention"):
        return None                                                # bits, positions and moved bytes: whole numbers
    s = prepare(case, seed)
    if case["op"] == "store":
        q = _exact_norm_rope(s["q"], s["wq"], s["pos"], s["cs"], case["neox"])
        k = _exact_norm_rope(s["k"], s["wk"], s["pos"], s["cs"], case["neox"])
        return q, _exact_q8(k.to(s["q"].dtype)), _exact_q8(s["v"]) if case["v"] == "q8t" else s["v"].double()
    out = []
    start, lens = s["start"].tolist(), s["lens"].tolist()
    for b, length in enumerate(lens):
        a, z = start[b], start[b + 1]
        n, ctx = z - a, length - (z - a)
        pages = s["table"][b, :-(-length // 16)].long()
        raw = s["kc"][pages].reshape(-1, case["hkv"], 4, 34)[:length]
        k = raw[..., 2:].contiguous().view(torch.int8).double() * raw[..., :2].contiguous().view(torch.float16).double()
        k = k.flatten(-2)
        if case["v"] == "q8t":
            rec = s["vc"][pages]
            d = rec[..., :128].contiguous().view(torch.float16).double().view(-1, case["hkv"], 4, 16).repeat_interleave(32, 2)
            v = rec[..., 128:].contiguous().view(torch.int8).double().view(-1, case["hkv"], D, 16) * d
            v = v.permute(0, 3, 1, 2).reshape(-1, case["hkv"], D)[:length]
        else:
            v = s["vc"][pages].reshape(-1, case["hkv"], D)[:length].double()
        words = s["mask"][a:z].tolist()
        seen = torch.ones((n, length), dtype=torch.bool)
        for i, row in enumerate(words):
            on = [row[j // 32] >> j % 32 & 1 for j in range(n)]
            seen[i, ctx:] = torch.tensor(on, dtype=torch.bool)
            if case["window"]:
                seen[i, :max(0, min(ctx, ctx + sum(on) - 1 - case["window"] + 1))] = False
        seen = seen.to(DEV)
        rows = []
        for h in range(case["hq"]):
            kv_h = h // (case["hq"] // case["hkv"])
            x = s["q"][a:z, h].double() @ k[:, kv_h].T * s["scale"]
            x = case["softcap"] * torch.tanh(x / case["softcap"]) if case["softcap"] else x
            rows.append(torch.softmax(x.masked_fill(~seen, -torch.inf), -1) @ v[:, kv_h])
        out.append(torch.stack(rows, 1))
    return torch.cat(out)
