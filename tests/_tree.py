"""Plain 64-bit forms of the draft-tree operators and builders of their cases (no test functions here)."""
import numpy as np
import torch

from _paged import PagedCase


def random_parents(n, rng, reach=4):
    """Parent index of each of n drafts (-1: the context)."""
    return [max(-1, i - 1 - int(rng.integers(0, reach))) for i in range(n)]


def ancestors(parents):
    """bool [n, n]: draft j is i or an ancestor of i."""
    n = len(parents)
    seen = np.zeros((n, n), bool)
    for i in range(n):
        j = i
        while j >= 0:
            seen[i, j] = True
            j = parents[j]
    return seen


def pack_bits(seen, words):
    """bool [n, m] -> int32 [n, words]."""
    out = np.zeros((seen.shape[0], words), np.uint32)
    for j in range(seen.shape[1]):
        out[:, j // 32] |= seen[:, j].astype(np.uint32) << np.uint32(j % 32)
    return out.view(np.int32)


def dequant_rows(rows):
    """Q8_0 bytes [..., D/32*34] -> float64 [..., D]."""
    b = np.ascontiguousarray(rows).reshape(*rows.shape[:-1], -1, 34)
    d = np.ascontiguousarray(b[..., :2]).view(np.float16).astype(np.float64)
    return (np.ascontiguousarray(b[..., 2:]).view(np.int8).astype(np.float64) * d).reshape(*rows.shape[:-1], -1)


def dense_kv(case, b):
    """float64 keys and values [L, Hkv, D] of sequence b of a PagedCase, and which keys lie on readable pages."""
    L, bs, D = int(case.seq_lens[b]), case.bs, case.D
    pages = case.block_table.numpy()[b][:(L + bs - 1) // bs]
    ok = np.repeat((pages >= 0) & (pages < case.NB), bs)[:L]
    safe = np.where((pages >= 0) & (pages < case.NB), pages, 0)
    k = dequant_rows(case.k_cache.cpu().numpy()[safe]).reshape(-1, case.Hkv, D)[:L]
    vc = case.v_cache.cpu()
    if case.v_fmt == "q8t":
        rec = vc.numpy()[safe]
        sc = np.ascontiguousarray(rec[..., :2 * (D // 32) * bs]).view(np.float16).astype(np.float64)
        sc = sc.reshape(len(safe), case.Hkv, D // 32, 1, bs)
        q = np.ascontiguousarray(rec[..., 2 * (D // 32) * bs:]).view(np.int8).astype(np.float64)
        v = q.reshape(len(safe), case.Hkv, D // 32, 32, bs) * sc
        v = v.reshape(len(safe), case.Hkv, D, bs).transpose(0, 3, 1, 2).reshape(-1, case.Hkv, D)[:L]
    elif case.v_fmt == "q8":
        v = dequant_rows(vc.numpy()[safe]).reshape(-1, case.Hkv, D)[:L]
    else:
        v = vc.double().numpy()[safe].reshape(-1, case.Hkv, D)[:L]
    return k, v, ok


def tree_reference(case, q, n_q, seen, softcap=0.0, window=0, sinks=None):
    """float64 [T, Hq, D]: q float64 [T, Hq, D], seen: list of bool [n, n] per sequence."""
    T, Hq, D = q.shape
    G = Hq // case.Hkv
    out = np.zeros((T, Hq, D))
    t0 = 0
    for b, n in enumerate(n_q):
        L = int(case.seq_lens[b])
        ctx = L - n
        if n == 0:
            continue
        k, v, ok = dense_kv(case, b)
        vis = np.ones((n, L), bool)
        vis[:, ctx:] = seen[b]
        if window:
            depth = seen[b].sum(1) - 1
            vis[:, :ctx] = ctx + depth[:, None] - np.arange(ctx)[None] < window
        vis &= ok[None]
        for h in range(Hq):
            with np.errstate(invalid="ignore", over="ignore"):
                s = q[t0:t0 + n, h] @ k[:, h // G].T * case.scale
                if softcap:
                    s = softcap * np.tanh(s / softcap)
            s = np.where(vis, s, -np.inf)
            top = s.max(1, keepdims=True)
            p = np.where(vis, np.exp(s - np.where(np.isfinite(top), top, 0)), 0.0)
            z = p.sum(1, keepdims=True)
            if sinks is not None:
                z = z + np.where(vis.any(1, keepdims=True), np.exp(float(sinks[h]) - np.where(np.isfinite(top), top, 0)), 0)
            p = np.divide(p, z, out=np.zeros_like(p), where=z > 0)
            for i in range(n):                       # a key that is not seen contributes nothing, whatever it holds
                out[t0 + i, h] = p[i][vis[i]] @ v[vis[i], h // G]
        t0 += n
    return out


class TreeCase(PagedCase):
    """Paged cache + queries + trees: lens counts each sequence's n_q drafts."""

    def __init__(self, lens, n_q, Hq, Hkv, v_fmt="q8t", bs=16, seed=0, dtype=torch.bfloat16, seen=None, kv_scale=1.0,
                 device="cuda"):
        super().__init__(lens, Hkv, bs=bs, v_fmt=v_fmt, seed=seed, device=device, kv_scale=kv_scale)
        rng = np.random.default_rng(seed)
        self.n_q, self.Hq = list(n_q), Hq
        self.seen = seen or [ancestors(random_parents(n, rng)) for n in n_q]
        self.words = max(1, -(-max(max(n_q), 1) // 32))
        T = sum(n_q)
        bits = [pack_bits(s, self.words) for s, n in zip(self.seen, n_q) if n]
        self.mask = torch.from_numpy(np.concatenate(bits) if bits else np.zeros((0, self.words), np.int32)).to(device)
        g = torch.Generator().manual_seed(seed + 1)
        self.q = torch.randn((T, Hq, self.D), generator=g).to(dtype).to(device)
        self.start = torch.tensor(np.concatenate([[0], np.cumsum(n_q)]), dtype=torch.int32, device=device)
        self.bt = self.block_table.to(device)
        self.lens = torch.from_numpy(self.seq_lens).to(device)

    def run(self, q=None, **kw):
        import gfx906_fa
        return gfx906_fa.tree_attention(self.q if q is None else q, self.k_cache, self.v_cache, self.bt, self.lens,
                                        self.start, self.mask, max(self.n_q), int(max(self.seq_lens)), self.scale, **kw)

    def reference(self, **kw):
        return tree_reference(self, self.q.cpu().double().numpy(), self.n_q, self.seen, **kw)
