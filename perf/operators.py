"""Measured cases of the serving operators around the compressed paged KV cache: attention of drafted tokens, the
accumulated attention weight of cached keys, the choice of the keys to keep, and the compaction of the cache.

``listed()`` and ``draw()`` name cases, ``prepare()`` makes what a serving program has in hand, ``run()`` makes one pass --
in plain torch, or through ``sub0_b200.ops`` when ``own`` is set -- ``work()`` counts what a pass cannot do without and
``exact()`` gives the same outputs in 64 bits.

A cache slot (one token, one KV head) holds packed codebook indices of K and of V and two fp32 norms.  What a slot stands
for is the rotated-frame row ``fp16(level * norm)``; that rounding belongs to the format, like the codes themselves, and so
appears in every form below.
"""
import math

import torch

own = False

D = 128
# the default 16- and 4-level tables, as IEEE-754 bit patterns
LEVELS = {
    4: (0xbf700000, 0xbf500000, 0xbf300000, 0xbf100000, 0xbe401459, 0xbdf4d0d9, 0xbd8ead6c, 0xbcdadd51,
        0x3c4ec2dc, 0x3d546849, 0x3dbfc3a0, 0x3e117705, 0x3e560388, 0x3f300000, 0x3f500000, 0x3f700000),
    2: (0xbf400000, 0xbd8fba69, 0x3d91f2a4, 0x3f400000),
}
OUTLIER_CHANNELS = (3, 37, 64, 101)


# ---- cases ------------------------------------------------------------------------------------------------------------

def _tree(name, batch, tokens, context, group=4, heads=8, k_bits=4, v_bits=4, page=16, drafted=True, ragged=True, softcap=0.0,
          window=0, alibi=False):
    return {"name": name, "op": "tree", "batch": batch, "tokens": tokens, "context": context, "group": group, "heads": heads,
            "k_bits": k_bits, "v_bits": v_bits, "page": page, "drafted": drafted, "ragged": ragged, "softcap": softcap,
            "window": window, "alibi": alibi}


def _mass(name, batch, tokens, context, **more):
    return dict(_tree(name, batch, tokens, context, **more), op="mass")


def _select(name, batch, heads, context, budget, sink, recent):
    return {"name": name, "op": "select", "batch": batch, "heads": heads, "context": context, "budget": budget, "sink": sink,
            "recent": recent}


def _compact(name, batch, heads, context, kept, k_bits=4, v_bits=4, page=16, tokens=0):
    return {"name": name, "op": "compact", "batch": batch, "heads": heads, "context": context, "kept": kept, "k_bits": k_bits,
            "v_bits": v_bits, "page": page, "tokens": tokens}


def listed():
    return [
        # one user, a tree of eight drafts behind a short chat: latency
        _tree("tree one chat", 1, 8, 1000),
        # a batch of users with trees of sixteen drafts and contexts of all lengths
        _tree("tree batch", 16, 16, 16384),
        # wide trees of 64 drafts, eight query heads per KV head, values in 2 bits
        _tree("tree wide", 4, 64, 32768, group=8, v_bits=2, ragged=False),
        # one user behind a very long document
        _tree("tree long", 1, 32, 131072, ragged=False),
        # chains of up to four tokens (no tree) of a model that caps its scores and slides its window, 2-bit cache
        _tree("chain capped", 32, 4, 4096, k_bits=2, v_bits=2, drafted=False, softcap=50.0, window=1500),
        # after each decode step: what the new token gave to every key
        _mass("mass decode", 32, 1, 16384, drafted=False, ragged=False),
        # after a prompt: what its last 64 tokens gave to every key
        _mass("mass prompt end", 2, 64, 30000, drafted=False),
        # a short chat after one accepted tree, capped scores, eight query heads per KV head
        _mass("mass small", 1, 5, 700, group=8, softcap=30.0),
        # a short chat that is cut to 512 keys
        _select("select small", 1, 8, 2000, 512, 4, 64),
        # a full batch of long contexts cut to 4096 keys
        _select("select batch", 32, 8, 65536, 4096, 4, 256),
        # the cache of a batch moved together after such a choice, another one per KV head
        _compact("compact evicted", 16, 8, 16384, 4096),
        # the accepted path of every tree of a batch moved to the end of its context
        _compact("compact accepted", 64, 8, 2000, 6, tokens=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "mass", "select", "compact"])
    if op in ("tree", "mass"):
        group, heads = rng.choice([1, 2, 3, 4, 4, 5, 8, 8]), rng.choice([1, 2, 4, 8, 8])
        k_bits, v_bits = rng.choice([(4, 4), (4, 4), (4, 2), (2, 2)])
        drafted = rng.random() < 0.6
        tokens = _log(rng, 1, 64) if drafted or op == "mass" else _log(rng, 1, 150)
        batch = _log(rng, 1, 48)
        most = min(131072, int(3.0e8 / (batch * heads * max(group * tokens, 8))), int(4.0e6 / (batch * heads)))
        context = _log(rng, min(2, max(most, 1)), max(most, 2))
        c = _tree("", batch, tokens, context, group=group, heads=heads, k_bits=k_bits, v_bits=v_bits, page=rng.choice([16, 16, 32, 48]),
                  drafted=drafted, ragged=rng.random() < 0.7, softcap=rng.choice([0.0, 0.0, 30.0, 50.0]),
                  window=rng.choice([0, 0, max(1, context // 3)]), alibi=rng.random() < 0.2)
        c["op"] = op
    elif op == "select":
        batch, heads = _log(rng, 1, 32), rng.choice([1, 2, 4, 8])
        context = _log(rng, 50, 65536)
        budget = _log(rng, 4, context - context // 8)
        sink = rng.randint(0, min(8, budget // 4))
        c = _select("", batch, heads, context, budget, sink, rng.randint(0, min(256, budget // 2)))
    else:
        batch, heads = _log(rng, 1, 64), rng.choice([1, 2, 4, 8])
        k_bits, v_bits = rng.choice([(4, 4), (4, 2), (2, 2)])
        if rng.random() < 0.4:
            tokens = rng.randint(1, 64)
            c = _compact("", batch, heads, _log(rng, 1, 4000), rng.randint(1, tokens), k_bits, v_bits, rng.choice([16, 32, 48]), tokens)
        else:
            context = _log(rng, 1, min(100000, 262144 // batch))
            c = _compact("", batch, heads, context, _log(rng, 1, context), k_bits, v_bits, rng.choice([16, 32, 48]))
    del c["name"]
    return c


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _hadamard(dtype, device):
    i = torch.arange(D, device=device)
    bits = i[:, None] & i[None, :]
    sign = torch.ones(D, D, dtype=torch.float64, device=device)
    for b in range(7):
        sign = sign * (1 - 2 * ((bits >> b) & 1)).double()
    return (sign / math.sqrt(D)).to(dtype)


def _levels(bits, device):
    return torch.tensor(LEVELS[bits], dtype=torch.int64).to(torch.int32).view(torch.float32).clone().to(device)


def _encode(rows, levels, bits, hadamard):
    """(packed indices (n, 16 * bits) uint8, norms (n,)) of fp32 rows (n, 128): the format's encoder."""
    rot = (rows @ hadamard).half().float()
    norm = rot.norm(dim=-1).clamp_min(1e-12)
    unit = (rot / norm[:, None]).clamp(-1.0, 1.0)
    idx = torch.bucketize(unit, (levels[1:] + levels[:-1]) / 2).to(torch.uint8)
    per = 8 // bits
    idx = idx.view(rows.shape[0], D // per, per)
    packed = torch.zeros_like(idx[..., 0])
    for k in range(per):
        packed |= idx[..., k] << (bits * (per - 1 - k))
    return packed, norm


def _fill_cache(gen, slots, heads, k_bits, v_bits, device):
    """A cache whose every slot holds an encoded pair of K and V rows: N(0, 1), four K channels eight times as large."""
    width = 16 * k_bits + 16 * v_bits + 16
    hadamard = _hadamard(torch.float32, device)
    cache = torch.zeros(slots, heads, width, dtype=torch.uint8, device=device)
    flat, kb, vb = cache.view(slots * heads, width), 16 * k_bits, 16 * v_bits
    step = 1 << 20
    for at in range(0, slots * heads, step):
        n = min(step, slots * heads - at)
        k, v = torch.randn(2, n, D, generator=gen, device=device)
        k[:, list(OUTLIER_CHANNELS)] *= 8.0
        for rows, bits, put, norm_at in ((k, k_bits, 0, kb + vb), (v, v_bits, kb, kb + vb + 4)):
            packed, norm = _encode(rows, _levels(bits, device), bits, hadamard)
            flat[at:at + n, put:put + 16 * bits] = packed
            flat[at:at + n, norm_at:norm_at + 4] = norm.view(torch.uint8).view(n, 4)
    return cache


def _trees(rng, tokens):
    """Ancestor masks of one random tree of ``tokens`` drafts: bit j of mask i is set when draft i may see draft j."""
    masks = []
    for i in range(tokens):
        parent = int(torch.randint(-1, i, (1,), generator=rng)) if i else -1
        masks.append((masks[parent] if parent >= 0 else 0) | (1 << i))
    return [m - (1 << 64) if m >> 63 else m for m in masks]


def _lengths(case):
    """Drafted tokens and whole lengths of every sequence: the case's own, whatever the seed."""
    B, T, N = case["batch"], case["tokens"], case["context"]
    rng = torch.Generator().manual_seed(1000003 * B + 1009 * T + N)
    if case["ragged"] and B > 1:
        q = torch.randint(1, T + 1, (B,), generator=rng).tolist()
        n = [int(x) for x in torch.exp(torch.rand(B, generator=rng) * math.log(8.0) + math.log(max(N, 8) / 8.0)).tolist()]
        q[0], n[0] = T, N
    else:
        q, n = [T] * B, [N] * B
    return q, [a + min(b, N) for a, b in zip(q, n)]


def _table(rng, lens, page, device):
    blocks = [-(-n // page) for n in lens]
    total = sum(blocks)
    order = torch.randperm(total, generator=rng).to(torch.int32)
    table = torch.zeros(len(lens), max(blocks), dtype=torch.int32)
    at = 0
    for b, n in enumerate(blocks):
        table[b, :n] = order[at:at + n]
        at += n
    return table.to(device), total * page


def prepare(case, seed):
    dev = torch.device("cuda")
    rng, gen = torch.Generator().manual_seed(seed), torch.Generator(device=dev).manual_seed(seed)
    op, B, H = case["op"], case["batch"], case["heads"]
    fixed = torch.Generator().manual_seed(1000003 * B + case["context"])
    s = {"op": op, "case": case}
    if op in ("tree", "mass"):
        q, n = _lengths(case)
        G, T = case["group"], sum(q)
        s["table"], slots = _table(rng, n, case["page"], dev)
        s["cache"] = _fill_cache(gen, slots, H, case["k_bits"], case["v_bits"], dev)
        s["lens"] = torch.tensor(n, dtype=torch.int32, device=dev)
        s["cu"] = torch.tensor([0] + q, dtype=torch.int32).cumsum(0).to(torch.int32).to(dev)
        s["max_q"], s["max_n"] = max(q), max(n)
        s["Q"] = torch.randn(T, H * G, D, generator=gen, device=dev).half()
        s["mask"] = torch.tensor([m for t in q for m in _trees(rng, t)], dtype=torch.int64).to(dev) if case["drafted"] else None
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, H * G + 1, device=dev) / (H * G)).float() if case["alibi"] else None
        s["cb_K"], s["cb_V"] = _levels(case["k_bits"], dev), _levels(case["v_bits"], dev)
        if op == "tree":
            s["out"] = torch.zeros_like(s["Q"])
            s["lse"] = torch.zeros(T, H * G, device=dev)
        else:
            s["mass"] = torch.rand(B, H, s["max_n"] + 100, generator=gen, device=dev) * 0.01
            live = torch.arange(s["mass"].shape[2], device=dev)[None, :] < s["lens"][:, None] - (s["cu"][1:] - s["cu"][:-1])[:, None]
            s["mass"] *= live[:, None]
            # the attention that came before left its log-sum-exp; drafts that were not accepted count nothing
            s["lse"] = _log_sum_exp(s)
            s["weights"] = (torch.rand(T, generator=gen, device=dev) < 0.5).float() if case["drafted"] else None
    elif op == "select":
        N = case["context"]
        n = [N] + [int(x) for x in torch.randint(max(1, N // 2), N + 1, (B - 1,), generator=fixed).tolist()]
        s["lens"] = torch.tensor(n, dtype=torch.int32, device=dev)
        # accumulated weights spread over orders of magnitude, and some keys that no query has looked at
        s["mass"] = torch.exp(2.5 * torch.randn(B, H, N, generator=gen, device=dev) - 3.0)
        s["mass"] *= torch.rand(B, H, N, generator=gen, device=dev) > 0.1
    else:
        N, K, T = case["context"], case["kept"], case["tokens"]
        n = [N + T] + [int(x) + T for x in torch.randint(max(1, N // 2), N + 1, (B - 1,), generator=fixed).tolist()]
        s["table"], slots = _table(rng, n, case["page"], dev)
        width = 16 * case["k_bits"] + 16 * case["v_bits"] + 16
        s["cache"] = torch.randint(0, 256, (slots, H, width), generator=gen, device=dev, dtype=torch.uint8)
        s["lens"] = torch.tensor(n, dtype=torch.int32, device=dev)
        if T:  # an accepted path: ascending drafts of each sequence, the same for every KV head
            keys = torch.rand(B, 1, T, generator=gen, device=dev)
            first = s["start"] = s["lens"] - T
            took = torch.randint(1, K + 1, (B,), generator=gen, device=dev)
            s["mass"] = None
        else:  # keys kept by each KV head
            keys = torch.rand(B, H, N, generator=gen, device=dev)
            keys = torch.where(torch.arange(N, device=dev) < s["lens"][:, None, None], keys, 2.0)
            s["start"], first = None, torch.zeros_like(s["lens"])
            took = s["lens"].clamp_max(K)
            s["mass"] = torch.rand(B, H, N, generator=gen, device=dev)
        pick = keys.argsort(dim=-1)[..., :K]
        live = torch.arange(K, device=dev) < took[:, None, None]
        pick = torch.where(live, pick, 1 << 30).sort(dim=-1).values
        s["keep"] = torch.where(live, pick + first[:, None, None], -1).to(torch.int32).contiguous()
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------------

def _side(s, bits, at, norm_at, levels):
    """The rows of one side of the cache, (B, H, N, 128) fp32."""
    page, N = s["case"]["page"], s["max_n"]
    pos = torch.arange(N, device=levels.device)
    slot = s["table"].long()[:, pos // page] * page + pos % page
    raw = s["cache"][slot][..., at:at + 16 * bits]
    norm = s["cache"][slot][..., norm_at:norm_at + 4].contiguous().view(torch.float32)
    shift = torch.arange(8 - bits, -1, -bits, device=levels.device, dtype=torch.uint8)
    idx = (raw[..., None] >> shift) & ((1 << bits) - 1)
    rows = levels[idx.flatten(-2).int()] * norm
    return rows.half().float().transpose(1, 2)


def _scores(s):
    """Scores (B, H, T, G, N) of every drafted token of every sequence, minus infinity where a key is not seen, and the places
    (B, T) of the tokens in Q."""
    c = s["case"]
    kb, vb = c["k_bits"], c["v_bits"]
    H, G, T, N = c["heads"], c["group"], s["max_q"], s["max_n"]
    K = _side(s, kb, 0, 16 * kb + 16 * vb, s["cb_K"])
    dev = K.device
    q_len = (s["cu"][1:] - s["cu"][:-1]).long()
    lens = s["lens"].long()
    t = torch.arange(T, device=dev)
    live = t < q_len[:, None]
    place = torch.where(live, s["cu"][:-1].long()[:, None] + t, 0)
    Q = (s["Q"].float() @ _hadamard(torch.float32, dev))[place].view(-1, T, H, G, D).permute(0, 2, 1, 3, 4)
    x = (Q.reshape(-1, H, T * G, D) @ K.transpose(2, 3)).view(-1, H, T, G, N) * (1.0 / math.sqrt(D))
    if c["softcap"]:
        x = c["softcap"] * torch.tanh(x / c["softcap"])
    n = torch.arange(N, device=dev)
    context = (lens - q_len)[:, None]
    if s["mask"] is None:
        pos_q, pos_k = context + t, n.expand(len(lens), N)
        seen = n <= pos_q[..., None]
    else:
        mask = s["mask"][place]
        depth = torch.where(live, sum((mask >> j) & 1 for j in range(min(T, 64))) - 1, 0).clamp_min(0)
        draft = n - context
        pos_q = context + depth
        pos_k = torch.where(draft < 0, n, context + depth.gather(1, draft.clamp(0, T - 1)))
        seen = (draft < 0)[:, None] | ((mask[..., None] >> draft.clamp(0, 63)[:, None]) & 1).bool()
    seen = seen & (n < lens[:, None])[:, None] & live[..., None]
    if c["window"]:
        seen = seen & (pos_q[..., None] - pos_k[:, None] < c["window"])
    if s["slopes"] is not None:
        x = x + s["slopes"].view(H, 1, G, 1) * (pos_k[:, None] - pos_q[..., None])[:, None, :, None].float()
    return x.masked_fill(~seen[:, None, :, None], float("-inf")), place, live


def _softmax_parts(x):
    top = x.amax(dim=-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)
    p = torch.exp(x - top)
    return p, p.sum(dim=-1), top.squeeze(-1)


def _log_sum_exp(s):
    x, place, live = _scores(s)
    _, total, top = _softmax_parts(x)
    return (torch.log(total) + top).permute(0, 2, 1, 3).flatten(2)[live]


def _run_tree(s):
    c = s["case"]
    x, place, live = _scores(s)
    p, total, top = _softmax_parts(x)
    V = _side(s, c["v_bits"], 16 * c["k_bits"], 16 * c["k_bits"] + 16 * c["v_bits"] + 4, s["cb_V"])
    B, H, T, G, N = p.shape
    o = (p.view(B, H, T * G, N) @ V).view(B, H, T, G, D) / total.clamp_min(1e-30)[..., None]
    o = o @ _hadamard(torch.float32, o.device)
    s["out"][place[live]] = o.permute(0, 2, 1, 3, 4).flatten(2, 3)[live].half()
    s["lse"][place[live]] = (torch.log(total) + top).permute(0, 2, 1, 3).flatten(2)[live]
    return {"out": s["out"], "lse": s["lse"]}


def _run_mass(s):
    x, place, live = _scores(s)
    B, H, T, G, N = x.shape
    lse = s["lse"][place].view(B, T, H, G).permute(0, 2, 1, 3)[..., None]
    p = torch.where(x == float("-inf"), 0.0, torch.exp(x - lse))
    if s["weights"] is not None:
        p = p * s["weights"][place][:, None, :, None, None]
    s["mass"][..., :N] += p.sum(dim=(2, 3))
    return s["mass"]


def _run_select(s):
    c = s["case"]
    N, K, dev = c["context"], c["budget"], s["mass"].device
    lens = s["lens"].long()[:, None, None]
    n = torch.arange(N, device=dev)
    m = torch.where(torch.isnan(s["mass"]), float("-inf"), s["mass"])
    # 0: the first and last keys, kept whatever their weight; 1: by weight; 2: behind the end
    rank = torch.where(n >= lens, 2, torch.where((n < c["sink"]) | (n >= lens - c["recent"]), 0, 1))
    by_weight = m.sort(dim=-1, descending=True, stable=True).indices
    order = by_weight.gather(-1, rank.expand_as(m).gather(-1, by_weight).sort(dim=-1, stable=True).indices)[..., :K]
    live = torch.arange(order.shape[-1], device=dev) < lens
    keep = torch.where(live, order, 1 << 30).sort(dim=-1).values
    keep = torch.where(live, keep, -1)
    keep = torch.cat([keep, keep.new_full((*keep.shape[:2], max(0, K - keep.shape[-1])), -1)], dim=-1)
    return {"keep": keep.to(torch.int32), "lens": s["lens"].clamp_max(K)}


def _run_compact(s):
    c, keep = s["case"], s["keep"].long()
    B, _, K = keep.shape
    dev, page, H = keep.device, c["page"], c["heads"]
    start = s["start"].long() if s["start"] is not None else torch.zeros(B, dtype=torch.long, device=dev)
    dst = (start[:, None, None] + torch.arange(K, device=dev)).expand(B, H, K)
    src = keep.expand(B, H, K)
    move = src >= 0
    b, h, _ = torch.nonzero(move, as_tuple=True)
    place = lambda n: s["table"].long()[b, n // page] * page + n % page  # noqa: E731
    rows = s["cache"][place(src[move]), h]
    s["cache"][place(dst[move]), h] = rows
    if s["mass"] is None:
        return s["cache"]
    kept = torch.where(move, s["mass"].gather(-1, src.clamp_min(0)), 0.0)
    live = torch.arange(s["mass"].shape[-1], device=dev) < s["lens"][:, None, None]
    s["mass"].copy_(torch.where(live, 0.0, s["mass"]))
    s["mass"].scatter_(-1, dst, kept)
    return {"cache": s["cache"], "mass": s["mass"]}


# ---- one pass ---------------------------------------------------------------------------------------------------------

def run(s):
    if not own:
        return {"tree": _run_tree, "mass": _run_mass, "select": _run_select, "compact": _run_compact}[s["op"]](s)
    from sub0_b200 import ops
    c = s["case"]
    if s["op"] == "tree":
        ops.tree_attention(s["Q"], s["cache"], s["table"], s["lens"], s["out"], cb_K=s["cb_K"], cb_V=s["cb_V"],
                           block_size=c["page"], cu_seqlens_q=s["cu"], max_query_len=s["max_q"], max_seq_len=s["max_n"],
                           tree_mask=s["mask"], softcap=c["softcap"] or None, window=c["window"] or None,
                           alibi_slopes=s["slopes"], lse=s["lse"])
        return {"out": s["out"], "lse": s["lse"]}
    if s["op"] == "mass":
        ops.attention_mass(s["Q"], s["cache"], s["table"], s["lens"], s["lse"], s["mass"], cb_K=s["cb_K"],
                           block_size=c["page"], cu_seqlens_q=s["cu"], max_query_len=s["max_q"], max_seq_len=s["max_n"],
                           tree_mask=s["mask"], softcap=c["softcap"] or None, window=c["window"] or None,
                           alibi_slopes=s["slopes"], weights=s["weights"])
        return s["mass"]
    if s["op"] == "select":
        keep, lens = ops.select_keys(s["mass"], s["lens"], c["budget"], sink=c["sink"], recent=c["recent"])
        return {"keep": keep, "lens": lens}
    ops.compact_cache(s["cache"], s["table"], s["lens"], s["keep"], block_size=c["page"], start=s["start"], mass=s["mass"])
    return s["cache"] if s["mass"] is None else {"cache": s["cache"], "mass": s["mass"]}


# ---- what a pass cannot do without ------------------------------------------------------------------------------------

def work(case):
    op, B, H = case["op"], case["batch"], case["heads"]
    if op in ("tree", "mass"):
        # mean lengths of _lengths(): contexts spread evenly over the logarithm of a factor of eight, drafts over 1 .. T
        spread = case["ragged"] and B > 1
        q = (case["tokens"] + (B - 1) * (case["tokens"] + 1) / 2) / B if spread else case["tokens"]
        n = case["context"] * (1 + (B - 1) * 0.875 / math.log(8.0)) / B if spread else case["context"]
        seen = min(n, case["window"]) if case["window"] else n
        rows, keys = B * H * case["group"] * q, B * H * (min(n, seen) + q)
        q_bytes = rows * D * 2
        if op == "tree":
            return {"bytes": keys * (16 * case["k_bits"] + 16 * case["v_bits"] + 8) + 2 * q_bytes + 4 * rows,
                    "flops": 4.0 * D * rows * (seen + q / 2)}
        return {"bytes": keys * (16 * case["k_bits"] + 4 + 8) + q_bytes + 4 * rows, "flops": 2.0 * D * rows * (seen + q / 2)}
    if op == "select":
        n = case["context"] * (1 + (B - 1) * 0.75) / B
        return {"bytes": 4.0 * B * H * (n + case["budget"]), "flops": B * H * n}
    width = 16 * case["k_bits"] + 16 * case["v_bits"] + 8
    n = case["context"] * (1 + (B - 1) * 0.75) / B
    if case["tokens"]:
        moved, lists, weights = B * H * (1 + case["kept"]) / 2, B * case["kept"], 0
    else:
        moved = lists = B * H * min(n, case["kept"])
        weights = moved + B * H * n
    return {"bytes": 2.0 * moved * width + 4 * lists + 4 * weights, "flops": 0.0}


# ---- 64 bits ----------------------------------------------------------------------------------------------------------

def _stored(s, b, bits, at, norm_at, levels):
    """Rows of one side of sequence b in 64 bits, (N, H, 128)."""
    page, n = s["case"]["page"], int(s["lens"][b])
    blocks = s["table"][b, :-(-n // page)].long()
    raw = s["cache"].view(-1, page, *s["cache"].shape[1:])[blocks].flatten(0, 1)[:n]
    code = raw[..., at:at + 16 * bits].long()
    parts = [code.bitwise_right_shift(8 - bits * (k + 1)).remainder(1 << bits) for k in range(8 // bits)]
    norm = raw[..., norm_at:norm_at + 4].clone().view(torch.float32)
    return torch.mul(levels[torch.stack(parts, -1).flatten(-2)], norm).half().double()


def _exact_scores(s, b):
    """64-bit scores (H, T * G, N) of sequence b, one key after another by the rule that says who sees whom."""
    c = s["case"]
    H, G = c["heads"], c["group"]
    lo, hi, n = int(s["cu"][b]), int(s["cu"][b + 1]), int(s["lens"][b])
    T, ctx = hi - lo, n - (hi - lo)
    kb, vb = c["k_bits"], c["v_bits"]
    k = _stored(s, b, kb, 0, 16 * (kb + vb), s["cb_K"])
    q = s["Q"][lo:hi].double().matmul(_hadamard(torch.float64, k.device)).view(T, H, G, D)
    x = torch.einsum("thgd,nhd->htgn", q, k).div_(math.sqrt(D))
    if c["softcap"]:
        x = x.div_(c["softcap"]).tanh_().mul_(c["softcap"])
    see = torch.ones(T, n, dtype=torch.bool)
    pos_q, pos_k = torch.arange(ctx, n), torch.arange(n)
    if s["mask"] is None:
        for t in range(T):
            see[t, ctx + t + 1:] = False
    else:
        masks = [int(m) & ((1 << 64) - 1) for m in s["mask"][lo:hi]]
        for t in range(T):
            pos_q[t] = ctx + max(bin(masks[t]).count("1") - 1, 0)
            see[t, ctx:] = torch.tensor([bool(masks[t] >> j & 1) for j in range(T)])
        pos_k[ctx:] = pos_q
    apart = pos_q[:, None] - pos_k[None, :]
    if c["window"]:
        see &= apart < c["window"]
    if s["slopes"] is not None:
        x -= s["slopes"].double().view(H, 1, G, 1) * apart.double().to(x.device)[None, :, None, :]
    x.masked_fill_(~see.to(x.device)[None, :, None, :], float("-inf"))
    return x.flatten(1, 2), lo, hi


def exact(case, seed):
    if case["op"] in ("select", "compact"):
        return None   # whole numbers and bytes that are moved: nothing is computed in floating point
    rows = case["batch"] * case["heads"] * case["group"] * case["tokens"]
    if rows * case["context"] > 1.2e9:
        return None
    s = prepare(case, seed)
    H, G = case["heads"], case["group"]
    if case["op"] == "tree":
        out = torch.zeros(s["Q"].shape, dtype=torch.float64, device=s["Q"].device)
        lse = torch.zeros(s["lse"].shape, dtype=torch.float64, device=out.device)
        had = _hadamard(torch.float64, out.device)
        kb, vb = case["k_bits"], case["v_bits"]
        for b in range(case["batch"]):
            x, lo, hi = _exact_scores(s, b)
            v = _stored(s, b, vb, 16 * kb, 16 * (kb + vb) + 4, s["cb_V"])
            z = torch.logsumexp(x, dim=-1)
            p = torch.softmax(x, dim=-1).nan_to_num_(0.0)
            o = torch.einsum("hrn,nhd->hrd", p, v).matmul(had)
            out[lo:hi] = o.view(H, hi - lo, G, D).transpose(0, 1).flatten(1, 2)
            lse[lo:hi] = z.view(H, hi - lo, G).transpose(0, 1).flatten(1, 2)
        return {"out": out, "lse": lse}
    mass = s["mass"].double()
    for b in range(case["batch"]):
        x, lo, hi = _exact_scores(s, b)
        z = s["lse"][lo:hi].double().view(hi - lo, H, G).transpose(0, 1).flatten(1, 2)
        p = torch.where(torch.isinf(x), 0.0, torch.exp(x - z[..., None])).view(H, hi - lo, G, -1)
        if s["weights"] is not None:
            p = p * s["weights"][lo:hi].double()[None, :, None, None]
        mass[b, :, :p.shape[-1]] += p.sum(dim=(1, 2))
    return mass
