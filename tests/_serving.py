"""64-bit CPU forms of the serving operators over the compressed cache (tree attention, attention mass, key selection, cache
compaction), seeded cases for them, and the bounds their kernels are held to.

Bounds.  With S = scale * max_n sum_d |q_d k_nd| over the keys a row sees, its scores come from fp32 sums of 128 products (the
query enters as two fp16 terms, off by 2^-22 of its value): off by at most 64 steps of 2^-24 S each way, d = 2^-18 S, plus
2^-20 for the exponential and the base-2 argument, plus cap * 2^-20 where scores are capped (the capping function's own error
is below 2^-21 of the cap).  Then
  lse   off by d + 2^-22 |lse|
  out   probabilities are off by 2 d and rounded to fp16 (2^-11): (2^-11 + 2 d) sum_n p_n |v_n| in the rotated frame, which the
        rotation back spreads over the row as at most sum_d(.) / sqrt(128); the result is rounded to fp16 (2^-11 |out|, and
        2^-25 where fp16 is subnormal).  A 4-bit value row is fp16(level) * norm in the kernel and fp16(level * norm) here: either
        rounding is off by at most half a step, 2^-11 of the value, so the two differ by at most 2^-10 |v|; where a row is
        subnormal, by at most 2 * 2^-25 a coordinate, which spreads to less than 2^-20
  mass  every term off by 2 d of its value, and the sum of R terms by R 2^-24 of it
"""
from __future__ import annotations

import math

import torch

from oracle import cda_oracle as O
from tests import _cases as Cs


def random_tree(gen, n, chain=0.5):
    """Ancestor masks (n,) int64 of a random tree: draft i continues i - 1 or branches off any earlier draft or the context."""
    masks = []
    for i in range(n):
        if i and float(torch.rand(1, generator=gen)) < chain:
            parent = i - 1
        else:
            parent = int(torch.randint(-1, i, (1,), generator=gen)) if i else -1
        masks.append((masks[parent] if parent >= 0 else 0) | (1 << i))
    return masks


def signed(m):
    return m - (1 << 64) if m >> 63 else m


def attend_case(lens, q_lens, *, H_kv=2, group=4, k_bits=4, v_bits=4, block_size=16, seed=0, tree=True, masks=None, softcap=None,
                window=None, alibi=False, scale=None):
    c = Cs.paged_case(lens, H_kv=H_kv, group=group, k_bits=k_bits, v_bits=v_bits, block_size=block_size, seed=seed)
    gen = torch.Generator().manual_seed(seed + 77)
    T = sum(q_lens)
    c["Q"] = Cs.rows(gen, T, H_kv * group)
    c["q_lens"] = list(q_lens)
    c["cu"] = torch.tensor([0] + list(q_lens)).cumsum(0).to(torch.int32)
    if masks is None and tree:
        masks = [m for n in q_lens for m in random_tree(gen, n)]
    c["masks"] = masks
    c["tree_mask"] = None if masks is None else torch.tensor([signed(m) for m in masks], dtype=torch.int64)
    c["slopes"] = torch.exp2(-8.0 * torch.arange(1, H_kv * group + 1) / (H_kv * group)).float() if alibi else None
    c.update(softcap=softcap, window=window, scale=scale if scale is not None else 1 / math.sqrt(128))
    return c


def sequence_scores(c, b):
    """(scores (H_kv, T, G, N) float64 with -inf where a key is not seen, S (H_kv, T, G): the bound's largest sum of products)."""
    n, lo, hi = int(c["seq_lens"][b]), int(c["cu"][b]), int(c["cu"][b + 1])
    T, G, H = hi - lo, c["group"], c["H_kv"]
    ctx = n - T
    Ks, _ = O.gather_sequence(c["cache"], c["block_table"][b], n, c["block_size"], c["k_bits"], c["v_bits"])
    K = O.decode_rotated(Ks, c["cb_K"])[0].double()                                    # (H, N, 128), fp16 rows by the format
    had = O.sylvester_hadamard(128).double()
    had = torch.sign(had) / math.sqrt(128.0)
    q = (c["Q"][lo:hi].double() @ had).view(T, H, G, 128).permute(1, 0, 2, 3)
    x = torch.einsum("htgd,hnd->htgn", q, K) * c["scale"]
    S = torch.einsum("htgd,hnd->htgn", q.abs(), K.abs()).amax(-1) * abs(c["scale"]) if n else torch.zeros(H, T, G).double()
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    masks = c["masks"][lo:hi] if c["masks"] is not None else [(1 << (t + 1)) - 1 for t in range(T)]
    depth = [max(bin(m).count("1") - 1, 0) for m in masks]
    pos_k = list(range(ctx)) + [ctx + d for d in depth]
    for t in range(T):
        for k in range(n):
            seen = k < ctx or (masks[t] >> (k - ctx)) & 1
            if c["window"] and ctx + depth[t] - pos_k[k] >= c["window"]:
                seen = False
            if not seen:
                x[:, t, :, k] = -math.inf
    if c["slopes"] is not None:
        apart = torch.tensor(pos_k).double()[None, :] - (ctx + torch.tensor(depth).double())[:, None]
        x = x + c["slopes"].double().view(H, 1, G, 1) * apart[None, :, None, :]
    return x, S, had


def score_bound(c, x, S):
    d = S * 2.0 ** -18 + 2.0 ** -20 + (c["softcap"] or 0.0) * 2.0 ** -20
    if c["slopes"] is not None:                                       # the bias and its sum with the score, rounded once each
        d = d + torch.nan_to_num(x, neginf=0.0).abs().amax(-1) * 2.0 ** -22
    return d


def tree_reference(c):
    """(out (T, H_q, 128), its bound, lse (T, H_q), its bound), float64."""
    T, Hq = c["Q"].shape[0], c["Q"].shape[1]
    out, tol = torch.zeros(T, Hq, 128).double(), torch.zeros(T, Hq, 128).double()
    lse, ltol = torch.full((T, Hq), -math.inf).double(), torch.zeros(T, Hq).double()
    for b in range(len(c["q_lens"])):
        lo, hi = int(c["cu"][b]), int(c["cu"][b + 1])
        if hi == lo:
            continue
        x, S, had = sequence_scores(c, b)
        n = int(c["seq_lens"][b])
        _, Vs = O.gather_sequence(c["cache"], c["block_table"][b], n, c["block_size"], c["k_bits"], c["v_bits"])
        V = O.decode_rotated(Vs, c["cb_V"])[0].double()
        z = torch.logsumexp(x, -1)
        p = torch.nan_to_num(torch.exp(x - z[..., None]))
        d = score_bound(c, x, S)
        o = torch.einsum("htgn,hnd->htgd", p, V) @ had
        spread = torch.einsum("htgn,hnd->htgd", p, V.abs()).sum(-1, keepdim=True) / math.sqrt(128.0)
        rows = 2.0 ** -10 if c["v_bits"] == 4 else 0.0
        t = 2.0 ** -11 * o.abs() + (2.0 ** -11 + rows + 2 * d[..., None]) * spread + 2.0 ** -25 + (2.0 ** -20 if rows else 0.0)
        back = lambda y: y.permute(1, 0, 2, 3).reshape(hi - lo, Hq, -1)  # noqa: E731
        out[lo:hi], tol[lo:hi] = back(o), back(t)
        lse[lo:hi], ltol[lo:hi] = back(z[..., None])[..., 0], back((d + torch.nan_to_num(z, neginf=0.0).abs() * 2.0 ** -22)[..., None])[..., 0]
    return out, tol, lse, ltol


def mass_reference(c, lse, mass, weights=None):
    """(mass + what the rows add, bound), float64."""
    got, tol = mass.double().clone(), torch.zeros_like(mass).double()
    for b in range(len(c["q_lens"])):
        lo, hi = int(c["cu"][b]), int(c["cu"][b + 1])
        if hi == lo:
            continue
        x, S, _ = sequence_scores(c, b)
        H, T, G, n = x.shape
        z = lse[lo:hi].double().view(T, H, G).permute(1, 0, 2)
        w = torch.ones(T).double() if weights is None else weights[lo:hi].double()
        p = torch.where(torch.isinf(x) | torch.isinf(z)[..., None], torch.zeros(()).double(), torch.exp(x - z[..., None])) * w[None, :, None, None]
        d = score_bound(c, x, S) + torch.nan_to_num(z, neginf=0.0).abs() * 2.0 ** -22
        got[b, :, :n] += p.sum(dim=(1, 2))
        tol[b, :, :n] += (p.abs() * 2 * d[..., None]).sum(dim=(1, 2)) + p.abs().sum(dim=(1, 2)) * (T * G) * 2.0 ** -24
    return got, tol + got.abs() * 2.0 ** -23 + 1e-37


def select_reference(mass, lens, budget, sink, recent):
    B, H, M = mass.shape
    keep = torch.full((B, H, budget), -1, dtype=torch.int32)
    for b in range(B):
        n = min(int(lens[b]), M)
        for h in range(H):
            if n <= budget:
                chosen = list(range(n))
            else:
                row = [(-math.inf if math.isnan(v) else v) for v in mass[b, h, :n].tolist()]
                middle = sorted(range(sink, n - recent), key=lambda i: (-row[i], i))[:budget - sink - recent]
                chosen = sorted(list(range(sink)) + middle + list(range(n - recent, n)))
            keep[b, h, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
    return keep, torch.tensor([min(int(x), budget) for x in lens], dtype=torch.int32)


def compact_reference(cache, table, lens, keep, block_size, start=None, mass=None):
    """Copies of (cache, mass) after the moves, one destination after another from a copy of the old state."""
    new, new_mass = cache.clone(), None if mass is None else mass.clone()
    B, H, K = keep.shape[0], cache.shape[1], keep.shape[2]
    place = lambda b, t: int(table[b, t // block_size]) * block_size + t % block_size  # noqa: E731
    for b in range(B):
        s0, n = (0 if start is None else int(start[b])), int(lens[b])
        for h in range(H):
            for i in range(K):
                src, dst = int(keep[b, h if keep.shape[1] > 1 else 0, i]), s0 + i
                ok = dst <= src < n
                if ok:
                    new[place(b, dst), h] = cache[place(b, src), h]
                if mass is not None and dst < mass.shape[2]:
                    new_mass[b, h, dst] = mass[b, h, src] if ok and src < mass.shape[2] else 0.0
            if mass is not None:
                new_mass[b, h, s0 + K:max(n, s0 + K)] = 0.0
    return new, new_mass
