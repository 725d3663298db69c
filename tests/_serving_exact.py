"""Bounds of the tree attention kernel that follow from the cache format alone, without room for a value row that is rounded in
another way.  With d the error of a score (``_serving.score_bound``) and |v| the absolute values of the rows fp16(level * norm):

  out   a probability is off by 2 d of its value and rounded to fp16 once: by 2^-11 of it, or, where fp16 is subnormal, by 2^-25
        on the kernel's scale, on which the largest probability of a row's first tile is 2^10 and so its sum at least that: 2^-35
        of the sum, for each of the keys it sees.  Together (2^-11 + 2 d) sum_n p_n |v_n| + 2^-35 sum_n |v_n|, which the
        rotation back spreads over the row as at most sum_d(.) / sqrt(128); the result is rounded to fp16 (2^-11 |out|, and
        2^-25 where fp16 is subnormal), after fp32 sums and a rotation in fp32 (below 2^-18 of the same spread)
  own   a row that sees a single key has the probability 1, which fp16 holds: only the result's rounding and 2^-18 remain
"""
from __future__ import annotations

import math

import torch

from oracle import cda_oracle as O
from tests import _serving as S


def tree_bounds(c, own=False):
    """(out, bound), (T, H_q, 128) float64."""
    T, Hq = c["Q"].shape[0], c["Q"].shape[1]
    out, tol = torch.zeros(T, Hq, 128).double(), torch.zeros(T, Hq, 128).double()
    for b in range(len(c["q_lens"])):
        lo, hi = int(c["cu"][b]), int(c["cu"][b + 1])
        if hi == lo:
            continue
        x, reach, had = S.sequence_scores(c, b)
        n = int(c["seq_lens"][b])
        _, Vs = O.gather_sequence(c["cache"], c["block_table"][b], n, c["block_size"], c["k_bits"], c["v_bits"])
        V = O.decode_rotated(Vs, c["cb_V"])[0].double()
        z = torch.logsumexp(x, -1)
        p = torch.nan_to_num(torch.exp(x - z[..., None]))
        V = torch.where(torch.isfinite(V), V, torch.zeros(()).double())          # (keys that no checked row sees)
        o = torch.einsum("htgn,hnd->htgd", p, V) @ had
        spread = torch.einsum("htgn,hnd->htgd", p, V.abs()).sum(-1, keepdim=True) / math.sqrt(128.0)
        t = 2.0 ** -11 * o.abs() + 2.0 ** -18 * spread + 2.0 ** -25
        if not own:
            d = S.score_bound(c, x, reach)
            seen = torch.einsum("htgn,hnd->htgd", (~torch.isinf(x)).double(), V.abs()).sum(-1, keepdim=True) / math.sqrt(128.0)
            t = t + (2.0 ** -11 + 2 * d[..., None]) * spread + 2.0 ** -35 * seen
        back = lambda y: y.permute(1, 0, 2, 3).reshape(hi - lo, Hq, -1)  # noqa: E731
        out[lo:hi], tol[lo:hi] = back(o), back(t)
    return out, tol


def norm_bytes(c, side):
    """Byte range of a slot's K (0) or V (1) norm."""
    at = 16 * (c["k_bits"] + c["v_bits"]) + 4 * side
    return slice(at, at + 4)


def slot_of(c, b, t):
    return int(c["block_table"][b, t // c["block_size"]]) * c["block_size"] + t % c["block_size"]


def set_norm(c, b, t, side, value, head=slice(None)):
    """Sets the K (0) or V (1) norm of token t of sequence b."""
    raw = torch.tensor([value], dtype=torch.float32).view(torch.uint8)
    c["cache"][slot_of(c, b, t), head, norm_bytes(c, side)] = raw
