"""The serving operators over the compressed cache on the GPU, against their 64-bit forms (tests/_serving.py)."""
import math

import pytest
import torch

from tests import _serving as S

pytestmark = pytest.mark.gpu
DEV = "cuda"


def on(t):
    return None if t is None else t.to(DEV)


def call_args(c):
    return dict(cb_K=on(c["cb_K"]), block_size=c["block_size"], cu_seqlens_q=on(c["cu"]), max_query_len=max(c["q_lens"] + [0]),
                max_seq_len=int(c["seq_lens"].max()), tree_mask=on(c["tree_mask"]), scale=c["scale"], softcap=c["softcap"],
                alibi_slopes=on(c["slopes"]), window=c["window"])


def run_tree(c, lse=True, pad=3, **more):
    from sub0_b200 import ops
    T, Hq = c["Q"].shape[0], c["Q"].shape[1]
    Q = torch.cat([c["Q"], torch.full((pad, Hq, 128), float("nan"), dtype=torch.float16)])     # rows behind the last sequence
    out = torch.full(Q.shape, 7.0, dtype=torch.float16, device=DEV)
    z = torch.full(Q.shape[:2], 7.0, device=DEV) if lse else None
    a = call_args(c)
    if a["tree_mask"] is not None:
        a["tree_mask"] = torch.cat([a["tree_mask"], a["tree_mask"].new_full((pad,), -1)])
    a.update(more)
    ops.tree_attention(on(Q), on(c["cache"]), on(c["block_table"]), on(c["seq_lens"]), out, cb_V=on(c["cb_V"]), lse=z, **a)
    assert ops.kv_status() == 0
    assert bool((out[T:] == 7.0).all()) and (z is None or bool((z[T:] == 7.0).all()))
    return out[:T], None if z is None else z[:T]


def check_tree(c, out, lse):
    want, tol, wz, ztol = S.tree_reference(c)
    off = ((out.double().cpu() - want).abs() / tol).max() if want.numel() else torch.tensor(0.0)
    assert float(off) <= 1.0, f"out is {float(off):.2f} bounds off"
    z = lse.double().cpu()
    assert torch.equal(torch.isinf(z), torch.isinf(wz))
    live = ~torch.isinf(wz)
    if bool(live.any()):
        zo = float(((z - wz).abs()[live] / ztol[live]).max())
        assert zo <= 1.0, f"lse is {zo:.2f} bounds off"


TREES = {
    "one token": dict(lens=[1], q_lens=[1]),
    "only drafts": dict(lens=[5, 1, 64], q_lens=[5, 1, 64]),
    "tile edges": dict(lens=[127, 128, 129, 256, 257], q_lens=[3, 3, 3, 1, 2], H_kv=1),
    "drafts across a tile": dict(lens=[140, 300], q_lens=[40, 64]),
    "ragged, empty sequence": dict(lens=[700, 0, 33, 1290], q_lens=[7, 0, 1, 16]),
    "group 1": dict(lens=[200, 77], q_lens=[9, 2], group=1, H_kv=3),
    "group 3": dict(lens=[333], q_lens=[11], group=3),
    "group 8, 512 rows": dict(lens=[260], q_lens=[64], group=8, H_kv=1),
    "group 16": dict(lens=[150, 90], q_lens=[3, 8], group=16, H_kv=1),
    "k4v2": dict(lens=[500, 61], q_lens=[12, 5], v_bits=2),
    "k2v2, page 48": dict(lens=[301, 96], q_lens=[6, 33], k_bits=2, v_bits=2, block_size=48),
    "k2v4, page 32": dict(lens=[301], q_lens=[6], k_bits=2, v_bits=4, block_size=32),
    "chain": dict(lens=[400, 90], q_lens=[30, 4], tree=False),
    "long chain": dict(lens=[420, 600], q_lens=[150, 333], tree=False, H_kv=1),
    "capped": dict(lens=[400, 130], q_lens=[10, 4], softcap=20.0),
    "capped steeply": dict(lens=[300], q_lens=[10], softcap=1.5, scale=1.0),
    "window": dict(lens=[700, 90], q_lens=[9, 40], window=64),
    "window of one": dict(lens=[300, 20], q_lens=[9, 20], window=1, tree=False),
    "window, chain": dict(lens=[900], q_lens=[200], window=130, tree=False, H_kv=1),
    "alibi": dict(lens=[500, 40], q_lens=[8, 12], alibi=True),
    "all modifiers": dict(lens=[513, 129], q_lens=[17, 5], alibi=True, softcap=30.0, window=200, k_bits=2, v_bits=2),
    "steep scores": dict(lens=[600], q_lens=[8], scale=2.0),
}


@pytest.mark.parametrize("name", TREES)
def test_tree_attention(name):
    c = S.attend_case(seed=len(name), **TREES[name])
    check_tree(c, *run_tree(c))


def test_rows_that_see_nothing_are_zero():
    c = S.attend_case([3, 90, 4], [3, 2, 4], masks=[0, 1, 0, 0, 0, 8, 0, 2, 1], seed=5)
    out, lse = run_tree(c)
    check_tree(c, out, lse)
    assert bool((out[0] == 0).all()) and bool(torch.isinf(lse[0]).all()) and bool((out[2] == 0).all()) and bool((out[6] == 0).all())


def test_late_dominant_keys_move_the_reference():
    """Scores that climb by hundreds along the sequence, so that every tile's largest is far above what came before it, and
    fall again."""
    c = S.attend_case([1200, 900], [6, 3], seed=3, scale=1.0)
    kb = 16 * (c["k_bits"] + c["v_bits"])
    for b, n in enumerate([1200, 900]):
        for t in range(n):
            slot = int(c["block_table"][b, t // 16]) * 16 + t % 16
            norm = c["cache"][slot, :, kb:kb + 4].contiguous().view(torch.float32)
            f = 0.01 + (t if t < 800 else 1200 - t) / 400.0
            c["cache"][slot, :, kb:kb + 4] = (norm * f).view(torch.uint8).view(-1, 4)
    check_tree(c, *run_tree(c))


def test_single_token_chain_agrees_with_decode():
    from sub0_b200 import ops
    c = S.attend_case([4096, 5000], [1, 1], tree=False, seed=9)
    out, lse = run_tree(c)
    ref, rz = torch.empty_like(out), torch.empty_like(lse)
    ops.decode(on(c["Q"]), on(c["cache"]), on(c["block_table"]), on(c["seq_lens"]), ref, cb_K=on(c["cb_K"]), cb_V=on(c["cb_V"]),
               block_size=16, max_seq_len=5000, lse=rz)
    assert float((out.float() - ref.float()).abs().max()) < 2e-3 and float((lse - rz).abs().max()) < 2e-2


def test_tree_attention_is_reproducible_and_survives_a_dirty_workspace():
    from sub0_b200 import ops
    c = S.attend_case([900, 64, 2000], [13, 2, 9], seed=2)
    first, z = run_tree(c)
    need = ops.tree_attention_workspace_bytes(8, 2, 13)
    for fill in (0x00, 0xFF):
        ws = torch.full((need + 16,), fill, dtype=torch.uint8, device=DEV)
        again, z2 = run_tree(c, workspace=ws[:need])
        assert torch.equal(again, first) and torch.equal(z, z2)
        assert bool((ws[need:] == fill).all())
    no_lse, _ = run_tree(c, lse=False)
    assert torch.equal(no_lse, first)


def test_lengths_that_do_not_fit_are_skipped_and_reported():
    from sub0_b200 import ops
    c = S.attend_case([50, 60, 40], [5, 4, 3], seed=1)
    sl = c["seq_lens"].clone()
    sl[1] = 3                                                          # fewer tokens than new tokens
    out = torch.full_like(c["Q"], 7.0, device=DEV)
    a = call_args(c)
    ops.kv_clear_status()
    ops.tree_attention(on(c["Q"]), on(c["cache"]), on(c["block_table"]), on(sl), out, cb_V=on(c["cb_V"]), **a)
    assert ops.kv_status() == ops.KV_LENGTHS
    ops.kv_clear_status()
    want, tol, _, _ = S.tree_reference(c)
    o = out.double().cpu()
    assert bool((o[5:9] == 7.0).all())
    for r in (slice(0, 5), slice(9, 12)):
        assert bool(((o[r] - want[r]).abs() <= tol[r]).all())


def test_bad_block_is_reported_not_followed():
    from sub0_b200 import ops
    c = S.attend_case([80, 90], [3, 3], seed=1)
    bt = c["block_table"].clone()
    bt[1, 2] = 1 << 30
    bt[0, 1] = -5
    ops.kv_clear_status()
    out = torch.empty_like(c["Q"], device=DEV)
    mass, lse = torch.zeros(2, 2, 90, device=DEV), torch.zeros(6, 8, device=DEV)
    ops.tree_attention(on(c["Q"]), on(c["cache"]), on(bt), on(c["seq_lens"]), out, cb_V=on(c["cb_V"]), **call_args(c))
    assert ops.kv_status() == ops.KV_BAD_BLOCK
    ops.kv_clear_status()
    ops.attention_mass(on(c["Q"]), on(c["cache"]), on(bt), on(c["seq_lens"]), lse, mass, **call_args(c))
    assert ops.kv_status() == ops.KV_BAD_BLOCK
    ops.kv_clear_status()


# ---- attention mass ---------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("name", TREES)
def test_attention_mass(name):
    from sub0_b200 import ops
    c = S.attend_case(seed=len(name), **TREES[name])
    _, _, lse, _ = S.tree_reference(c)
    lse = lse.float()
    gen = torch.Generator().manual_seed(4)
    B, n = len(c["q_lens"]), int(c["seq_lens"].max())
    start = torch.rand(B, c["H_kv"], n + 5, generator=gen)
    for weights in (None, torch.rand(c["Q"].shape[0], generator=gen).round()):
        mass = on(start).clone()
        ops.attention_mass(on(c["Q"]), on(c["cache"]), on(c["block_table"]), on(c["seq_lens"]), on(lse), mass, weights=on(weights), **call_args(c))
        assert ops.kv_status() == 0
        want, tol = S.mass_reference(c, lse, start, weights)
        off = float(((mass.double().cpu() - want).abs() / tol).max())
        assert off <= 1.0, f"mass is {off:.2f} bounds off"
        assert torch.equal(mass[..., n:].cpu(), start[..., n:])
        again = on(start).clone()
        ops.attention_mass(on(c["Q"]), on(c["cache"]), on(c["block_table"]), on(c["seq_lens"]), on(lse), again, weights=on(weights), **call_args(c))
        assert torch.equal(again, mass)


def test_mass_of_rows_without_keys():
    from sub0_b200 import ops
    c = S.attend_case([3, 90], [3, 2], masks=[0, 1, 0, 0, 3], seed=5)
    _, _, lse, _ = S.tree_reference(c)
    mass = torch.zeros(2, 2, 90, device=DEV)
    ops.attention_mass(on(c["Q"]), on(c["cache"]), on(c["block_table"]), on(c["seq_lens"]), on(lse.float()), mass, **call_args(c))
    want, tol = S.mass_reference(c, lse.float(), torch.zeros(2, 2, 90))
    assert bool(((mass.double().cpu() - want).abs() <= tol).all())
    assert abs(float(mass.sum()) - float((~torch.isinf(lse)).sum())) < 1e-3      # every live row gives away one


# ---- key selection ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("lens,budget,sink,recent", [([1], 1, 0, 0), ([1, 5, 0], 4, 1, 1), ([2, 3, 4, 5], 3, 0, 3), ([100, 37], 37, 4, 8),
                                                     ([513, 512, 511], 256, 0, 0), ([2000], 1999, 4, 0), ([2000], 1, 0, 0),
                                                     ([5000, 4097], 700, 4, 64), ([40000], 9000, 4, 100), ([9], 6, 6, 0), ([9], 6, 2, 4)])
def test_select_keys(lens, budget, sink, recent):
    from sub0_b200 import ops
    gen = torch.Generator().manual_seed(budget)
    M = max(lens) + 3
    for kind in ("spread", "ties", "odd"):
        mass = torch.exp(3 * torch.randn(len(lens), 3, M, generator=gen))
        if kind == "ties":
            mass = mass.round()                                        # many equal weights, most of them 0
        if kind == "odd":
            pick = torch.rand(mass.shape, generator=gen)
            mass[pick < 0.1] = float("nan")
            mass[(pick >= 0.1) & (pick < 0.2)] = -0.0
            mass[(pick >= 0.2) & (pick < 0.3)] = 0.0
            mass[(pick >= 0.3) & (pick < 0.4)] = float("inf")
            mass[(pick >= 0.4) & (pick < 0.5)] = float("-inf")
            mass[(pick >= 0.5) & (pick < 0.6)] *= -1
            mass[(pick >= 0.6) & (pick < 0.7)] *= 1e-41
        keep, new = ops.select_keys(on(mass), on(torch.tensor(lens)), budget, sink=sink, recent=recent)
        want, want_new = S.select_reference(mass, lens, budget, sink, recent)
        assert torch.equal(keep.cpu(), want) and torch.equal(new.cpu(), want_new), kind
    assert ops.kv_status() == 0


def test_select_keys_of_too_long_a_sequence_is_cut_and_reported():
    from sub0_b200 import ops
    mass = torch.rand(1, 1, 20)
    keep, new = ops.select_keys(on(mass), on(torch.tensor([25])), 8)
    assert ops.kv_status() == ops.KV_LENGTHS
    ops.kv_clear_status()
    assert torch.equal(keep.cpu(), S.select_reference(mass, [20], 8, 0, 0)[0]) and int(new) == 8


# ---- compaction -------------------------------------------------------------------------------------------------------

def compact_case(lens, K, *, H=2, k_bits=4, v_bits=4, block_size=16, seed=0, shared=False, tail=None):
    gen = torch.Generator().manual_seed(seed)
    blocks = [-(-n // block_size) for n in lens]
    order = torch.randperm(sum(blocks) + 2, generator=gen).to(torch.int32)
    table = torch.zeros(len(lens), max(max(blocks), 1), dtype=torch.int32)
    at = 0
    for b, n in enumerate(blocks):
        table[b, :n] = order[at:at + n]
        at += n
    width = 16 * (k_bits + v_bits) + 16
    cache = torch.randint(0, 256, ((sum(blocks) + 2) * block_size, H, width), generator=gen, dtype=torch.uint8)
    start = None if tail is None else torch.tensor([max(n - tail, 0) for n in lens], dtype=torch.int32)
    keep = torch.full((len(lens), 1 if shared else H, K), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        for h in range(keep.shape[1]):
            s0 = 0 if start is None else int(start[b])
            pick = (torch.randperm(n - s0, generator=gen)[:K] + s0).sort().values
            keep[b, h, :pick.numel()] = pick.to(torch.int32)
    return cache, table, torch.tensor(lens, dtype=torch.int32), keep, start, torch.rand(len(lens), H, max(lens) + 4, generator=gen)


@pytest.mark.parametrize("case", [dict(lens=[1], K=1), dict(lens=[40, 0, 7], K=5), dict(lens=[700, 300], K=290), dict(lens=[3000, 2900], K=2800),
                                  dict(lens=[5000], K=1500, H=1), dict(lens=[400, 90], K=100, H=3, v_bits=2),
                                  dict(lens=[400, 90], K=100, k_bits=2, v_bits=2, block_size=48),
                                  dict(lens=[400, 90, 16], K=6, shared=True, tail=16), dict(lens=[20000], K=19000, H=1)])
@pytest.mark.parametrize("with_mass", [True, False])
def test_compact_cache(case, with_mass):
    from sub0_b200 import ops
    cache, table, lens, keep, start, mass = compact_case(**case)
    want, want_mass = S.compact_reference(cache, table, lens, keep, case.get("block_size", 16), start, mass if with_mass else None)
    got, got_mass = on(cache), on(mass) if with_mass else None
    ops.compact_cache(got, on(table), on(lens), on(keep), block_size=case.get("block_size", 16), start=on(start), mass=got_mass)
    assert ops.kv_status() == 0
    assert torch.equal(got.cpu(), want)
    if with_mass:
        assert torch.equal(got_mass.cpu(), want_mass)


def test_compact_cache_takes_repeats_and_gaps_and_refuses_what_breaks_the_rule():
    from sub0_b200 import ops
    cache, table, lens, keep, _, mass = compact_case([600, 300], 200, seed=8)
    keep = torch.arange(200, dtype=torch.int32).expand(2, 2, 200).contiguous()
    keep[0, 0] = 599                                                   # the same key everywhere
    keep[0, 1] = torch.flip(torch.arange(300, 500, dtype=torch.int32), (0,))       # descending, but behind every destination
    keep[1, 0, ::3] = -1                                               # gaps
    keep[1, 1, 7:] += 1
    want, want_mass = S.compact_reference(cache, table, lens, keep, 16, None, mass)
    got, got_mass = on(cache), on(mass)
    ops.compact_cache(got, on(table), on(lens), on(keep), block_size=16, mass=got_mass)
    assert ops.kv_status() == 0 and torch.equal(got.cpu(), want) and torch.equal(got_mass.cpu(), want_mass)
    for bad in (5, 600, 1 << 30):                                      # in front of its destination, behind the end
        broken = keep.clone()
        broken[0, 0, 10] = bad
        want, want_mass = S.compact_reference(cache, table, lens, broken, 16, None, mass)
        got, got_mass = on(cache), on(mass)
        ops.compact_cache(got, on(table), on(lens), on(broken), block_size=16, mass=got_mass)
        assert ops.kv_status() == ops.KV_BAD_KEEP
        ops.kv_clear_status()
        assert torch.equal(got.cpu(), want) and torch.equal(got_mass.cpu(), want_mass)


# ---- together ---------------------------------------------------------------------------------------------------------

def test_speculative_steps_with_eviction():
    """Three rounds as a serving loop runs them: drafts are encoded behind the context, the tree attends, the accepted path is
    moved behind the context and counted, the cache is cut to its budget.  The state is followed by the 64-bit forms."""
    from sub0_b200 import ops
    gen = torch.Generator().manual_seed(11)
    H, G, bs, drafts, budget = 2, 4, 16, 12, 160
    c = S.attend_case([200, 150], [drafts, drafts], seed=21)
    blocks = -(-260 // bs)
    cache = torch.zeros(2 * blocks * bs, H, 144, dtype=torch.uint8)
    table = torch.randperm(2 * blocks, generator=gen).to(torch.int32).view(2, blocks)
    for b, n in enumerate([200, 150]):
        for t in range(n):
            cache[int(table[b, t // bs]) * bs + t % bs] = c["cache"][int(c["block_table"][b, t // bs]) * bs + t % bs]
    c["cache"], c["block_table"] = cache, table
    d_cache, d_table = on(cache), on(table)
    ctx = [200 - drafts, 150 - drafts]
    mass = torch.zeros(2, H, 260, device=DEV)
    for step in range(3):
        c["seq_lens"] = torch.tensor([n + drafts for n in ctx], dtype=torch.int32)
        if step:
            K, V = S.Cs.rows(gen, 2 * drafts, H, outliers=True), S.Cs.rows(gen, 2 * drafts, H)
            slots = torch.tensor([int(table[b, t // bs]) * bs + t % bs for b in range(2) for t in range(ctx[b], ctx[b] + drafts)], dtype=torch.int32)
            ops.paged_encode(on(K), on(V), on(slots), d_cache, on(c["cb_K"]), on(c["cb_V"]))
        c["Q"] = S.Cs.rows(gen, 2 * drafts, H * G)
        c["masks"] = [m for _ in range(2) for m in S.random_tree(gen, drafts)]
        c["tree_mask"] = torch.tensor(c["masks"], dtype=torch.int64)
        c["cache"] = d_cache.cpu()
        a = call_args(c)
        out, lse = torch.empty(2 * drafts, H * G, 128, dtype=torch.float16, device=DEV), torch.empty(2 * drafts, H * G, device=DEV)
        ops.tree_attention(on(c["Q"]), d_cache, d_table, on(c["seq_lens"]), out, cb_V=on(c["cb_V"]), lse=lse, **a)
        check_tree(c, out, lse)
        path = [[j for j in range(drafts) if c["masks"][b * drafts + 9] >> j & 1] for b in range(2)]   # accepted: draft 9 and its ancestors
        weights = torch.zeros(2 * drafts)
        keep = torch.full((2, 1, drafts), -1, dtype=torch.int32)
        for b in range(2):
            keep[b, 0, :len(path[b])] = torch.tensor([ctx[b] + j for j in path[b]], dtype=torch.int32)
            weights[[b * drafts + j for j in path[b]]] = 1.0
        before = mass.cpu()
        ops.attention_mass(on(c["Q"]), d_cache, d_table, on(c["seq_lens"]), lse, mass, weights=on(weights), **a)
        want, tol = S.mass_reference(c, lse.cpu(), before, weights)
        assert bool(((mass.double().cpu() - want).abs() <= tol).all())
        starts = torch.tensor(ctx, dtype=torch.int32)
        moved, moved_mass = S.compact_reference(c["cache"], table, c["seq_lens"], keep, bs, starts, mass.cpu())
        ops.compact_cache(d_cache, d_table, on(c["seq_lens"]), on(keep), block_size=bs, start=on(starts), mass=mass)
        assert torch.equal(d_cache.cpu(), moved) and torch.equal(mass.cpu(), moved_mass)
        lens = torch.tensor([ctx[b] + len(path[b]) for b in range(2)], dtype=torch.int32)
        want_keep, want_lens = S.select_reference(mass.cpu(), lens, budget, 4, 16)
        cut, cut_mass = S.compact_reference(d_cache.cpu(), table, lens, want_keep, bs, None, mass.cpu())
        kept, new_lens = ops.evict(d_cache, d_table, on(lens), mass, budget, block_size=bs, sink=4, recent=16)
        assert torch.equal(kept.cpu(), want_keep) and torch.equal(new_lens.cpu(), want_lens)
        assert torch.equal(d_cache.cpu(), cut) and torch.equal(mass.cpu(), cut_mass)
        ctx = new_lens.tolist()
    assert ops.kv_status() == 0


def test_captured_and_replayed_beside_an_eager_call():
    """Two graphs and an eager call on another stream share nothing: each gives its own result."""
    from sub0_b200 import ops
    cases = [S.attend_case([700, 90], [9, 3], seed=31), S.attend_case([1500], [20], seed=32), S.attend_case([333, 64], [2, 30], seed=33)]
    graphs, outs = [], []
    want = [run_tree(c)[0] for c in cases]
    dev = [{k: on(c[k]) for k in ("Q", "cache", "block_table", "seq_lens", "cb_V")} | call_args(c) for c in cases]

    def call(d, out):
        a = {k: v for k, v in d.items() if k not in ("Q", "cache", "block_table", "seq_lens")}
        ops.tree_attention(d["Q"], d["cache"], d["block_table"], d["seq_lens"], out, **a)
    for d in dev[:2]:
        out = torch.zeros_like(d["Q"])
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            call(d, out)
        graphs.append(g)
        outs.append(out)
    side = [torch.cuda.Stream() for _ in range(3)]
    eager = torch.zeros_like(dev[2]["Q"])
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, side):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(side[2]):
            call(dev[2], eager)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[2])
    assert ops.kv_status() == 0


@pytest.mark.parametrize("B,N,group,k_bits,v_bits", [(16, 16384, 4, 4, 4), (3, 70000, 8, 4, 2), (40, 5000, 1, 2, 2)])
def test_many_tiles_per_cta(B, N, group, k_bits, v_bits):
    """Sizes at which every ring and buffer of the kernels wraps many times.  Each row's weights sum to one, so a sequence and KV
    head give away as many as it has rows; a chain of one token is a decode step."""
    from sub0_b200 import ops, synth
    w = synth.build_decode_workload(B, N, group=group, k_bits=k_bits, v_bits=v_bits)
    cu = torch.arange(B + 1, dtype=torch.int32, device=DEV)
    out, lse, ref = torch.empty_like(w.Q), torch.empty(w.Q.shape[:2], device=DEV), torch.empty_like(w.Q)
    a = dict(cb_K=w.cb_K, block_size=16, cu_seqlens_q=cu, max_query_len=1, max_seq_len=N)
    ops.tree_attention(w.Q, w.cache, w.block_table, w.seq_lens, out, cb_V=w.cb_V, lse=lse, **a)
    ops.decode(w.Q, w.cache, w.block_table, w.seq_lens, ref, cb_K=w.cb_K, cb_V=w.cb_V, block_size=16, max_seq_len=N)
    assert float(((out.float() - ref.float()).abs() / (1e-3 + 2e-3 * ref.float().abs())).max()) < 2.0
    mass = torch.zeros(B, 8, N, device=DEV)
    ops.attention_mass(w.Q, w.cache, w.block_table, w.seq_lens, lse, mass, **a)
    # a sum of N terms that are off by 2^-16 of their value at most (scores of size 2^2 summed in fp32), and lse by as much
    assert float((mass.double().sum(-1) - group).abs().max()) < group * 2.0 ** -15
    T = 12                                                             # the same cache under longer chunks, rows in several blocks
    gen = torch.Generator(device=DEV).manual_seed(1)
    Q = torch.randn(B * T, 8 * group, 128, generator=gen, device=DEV).half()
    out, lse = torch.empty_like(Q), torch.empty(Q.shape[:2], device=DEV)
    a.update(cu_seqlens_q=cu * T, max_query_len=T)
    ops.tree_attention(Q, w.cache, w.block_table, w.seq_lens, out, cb_V=w.cb_V, lse=lse, **a)
    mass.zero_()
    ops.attention_mass(Q, w.cache, w.block_table, w.seq_lens, lse, mass, **a)
    assert float((mass.double().sum(-1) - group * T).abs().max()) < group * T * 2.0 ** -15
    pre = torch.empty_like(Q)
    if group in (1, 4, 8):
        ops.prefill_varlen(Q, w.cache, w.block_table, cu * T, w.seq_lens, pre, cb_K=w.cb_K, cb_V=w.cb_V, block_size=16, max_query_len=T, max_seq_len=N)
        assert float(((out.float() - pre.float()).abs() / (1e-3 + 2e-3 * pre.float().abs())).max()) < 2.0
    assert ops.kv_status() == 0


def check_mass(c, lse):
    from sub0_b200 import ops
    start = torch.zeros(len(c["q_lens"]), c["H_kv"], int(c["seq_lens"].max()))
    mass = on(start).clone()
    ops.attention_mass(on(c["Q"]), on(c["cache"]), on(c["block_table"]), on(c["seq_lens"]), on(lse), mass, **call_args(c))
    assert ops.kv_status() == 0
    want, tol = S.mass_reference(c, lse, start)
    off = float(((mass.double().cpu() - want).abs() / tol).max())
    assert off <= 1.0, f"mass is {off:.2f} bounds off"


@pytest.mark.parametrize("H_kv", [1, 3, 6, 7, 11, 12, 16, 33])
def test_numbers_of_heads(H_kv):
    """Neighbouring CTAs walk the heads of a token together, in teams of the largest divisor up to eight."""
    c = S.attend_case([300, 5, 0, 900, 129], [3, 5, 0, 2, 1], H_kv=H_kv, group=2, seed=H_kv)
    check_tree(c, *run_tree(c))
    check_mass(c, S.tree_reference(c)[2].float())


@pytest.mark.parametrize("rows", [1, 2, 5, 16])
def test_many_pieces_per_cta(rows):
    """Hundreds of short sequences, some empty: a CTA starts and ends dozens of pieces, most of a single tile."""
    gen = torch.Generator().manual_seed(rows)
    lens = [int(v) for v in torch.randint(0, 300, (700,), generator=gen)]
    lens[::5] = [v % 7 for v in lens[::5]]
    q_lens = [min(v, 1 + int(r)) for v, r in zip(lens, torch.randint(0, rows, (700,), generator=gen))]
    c = S.attend_case(lens, q_lens, H_kv=4, group=4, seed=rows)
    check_tree(c, *run_tree(c))
    check_mass(c, S.tree_reference(c)[2].float())


@pytest.mark.parametrize("max_q,more", [(17, 0), (40, 1000), (64, 500000)])
def test_limits_above_the_lengths(max_q, more):
    """Callers give bounds, not lengths: the call may then use larger row blocks and has idle ones."""
    from sub0_b200 import ops
    c = S.attend_case([700, 0, 33, 1290], [7, 0, 1, 16], seed=9)
    wide = (int(c["seq_lens"].max()) + more + 15) // 16
    c["block_table"] = torch.cat([c["block_table"], torch.full((4, max(0, wide - c["block_table"].shape[1])), -1, dtype=torch.int32)], 1)
    a = dict(max_query_len=max_q, max_seq_len=int(c["seq_lens"].max()) + more)
    out, lse = run_tree(c, **a)
    check_tree(c, out, lse)
    z = S.tree_reference(c)[2].float()
    mass = torch.zeros(4, c["H_kv"], a["max_seq_len"], device=DEV)
    ops.attention_mass(on(c["Q"]), on(c["cache"]), on(c["block_table"]), on(c["seq_lens"]), on(z), mass, **{**call_args(c), **a})
    want, tol = S.mass_reference(c, z, torch.zeros(mass.shape))
    assert bool(((mass.double().cpu() - want).abs() <= tol).all()) and ops.kv_status() == 0


def test_two_streams_at_once():
    """Calls of different sizes interleaved on two streams, each several times: bit for bit what the calls give alone."""
    from sub0_b200 import ops
    cases = [S.attend_case([700, 5000, 33], [7, 16, 1], seed=1), S.attend_case([9000, 300], [40, 3], group=8, v_bits=2, seed=2)]
    calls = []
    for c in cases:
        a = call_args(c)
        tensors = [on(c[k]) for k in ("Q", "cache", "block_table", "seq_lens", "cb_V")]
        calls.append((a, tensors, torch.empty_like(tensors[0]), torch.empty(tensors[0].shape[:2], device=DEV),
                      torch.zeros(len(c["q_lens"]), c["H_kv"], a["max_seq_len"], device=DEV)))

    def run(a, tensors, out, lse, mass):
        Q, cache, table, lens, cb_V = tensors
        ops.tree_attention(Q, cache, table, lens, out, cb_V=cb_V, lse=lse, **a)
        mass.zero_()
        ops.attention_mass(Q, cache, table, lens, lse, mass, **a)

    alone = []
    for call in calls:
        run(*call)
        torch.cuda.synchronize()
        alone.append([t.clone() for t in call[2:]])
        for t in call[2:]:
            t.fill_(3.0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for stream, call in zip(streams, calls):
            with torch.cuda.stream(stream):
                run(*call)
    torch.cuda.synchronize()
    assert ops.kv_status() == 0
    for call, want in zip(calls, alone):
        for got, w in zip(call[2:], want):
            assert torch.equal(got, w)


def test_refusals_on_the_gpu():
    """Arguments that the front end refuses before anything is launched."""
    from sub0_b200 import ops
    c = S.attend_case([50], [5], seed=1)
    a, out = call_args(c), torch.empty_like(c["Q"], device=DEV)
    pos = (on(c["Q"]), on(c["cache"]), on(c["block_table"]), on(c["seq_lens"]))
    tree = lambda **kw: ops.tree_attention(*pos, kw.pop("out", out), cb_V=on(c["cb_V"]), **{**a, **kw})  # noqa: E731
    for kw in (dict(softcap=0.0), dict(softcap=-1.0), dict(softcap=math.inf), dict(window=0), dict(out=out.float()), dict(out=out.cpu()),
               dict(tree_mask=a["tree_mask"][:4]), dict(tree_mask=a["tree_mask"].int()), dict(alibi_slopes=torch.ones(3, device=DEV)),
               dict(lse=torch.zeros(5, 8)), dict(lse=torch.zeros(5, 7, device=DEV)), dict(cu_seqlens_q=a["cu_seqlens_q"][:1]),
               dict(workspace=torch.zeros(16, dtype=torch.uint8, device=DEV)), dict(max_seq_len=1 << 20), dict(block_size=24)):
        with pytest.raises((ValueError, TypeError)):
            tree(**kw)
    with pytest.raises(NotImplementedError):
        tree(max_query_len=65)
    mass, lse = torch.zeros(1, 2, 50, device=DEV), torch.zeros(5, 8, device=DEV)
    for m, z in ((mass[..., :49].contiguous(), lse), (mass.double(), lse), (mass[:, :1].contiguous(), lse), (mass, lse[:4])):
        with pytest.raises(ValueError):
            ops.attention_mass(*pos, z, m, **a)
    with pytest.raises(ValueError):
        ops.select_keys(mass, on(c["seq_lens"]), 4, sink=3, recent=2)
    with pytest.raises(ValueError):
        ops.compact_cache(pos[1], pos[2], pos[3], torch.zeros(1, 3, 4, dtype=torch.int32, device=DEV), block_size=16)
    assert ops.kv_status() == 0


def test_views_orders_and_other_index_types():
    """Strided queries, 64-bit lengths and tables, a 4-d cache in the type vLLM allocates."""
    from sub0_b200 import ops
    c = S.attend_case([130, 77], [7, 3], seed=6)
    a = call_args(c)
    wide = torch.zeros(10, 16, 128, dtype=torch.float16, device=DEV)
    wide[:, ::2] = on(c["Q"])
    cache = on(c["cache"]).view(-1, 16, 2, 144).view(torch.float16)
    out, lse = torch.empty_like(c["Q"], device=DEV), torch.empty(10, 8, device=DEV)
    a["cu_seqlens_q"] = a["cu_seqlens_q"].long()
    ops.tree_attention(wide[:, ::2], cache, on(c["block_table"]).long(), on(c["seq_lens"]).long(), out, cb_V=on(c["cb_V"]), lse=lse, **a)
    check_tree(c, out, lse)


def test_backend_caps_scores_of_decodes_and_prompts():
    from sub0_b200.vllm_integration.cda_attn_v2 import get_backend_classes
    from tests.test_gpu_vllm_backend import metadata, vllm_cache
    _, Impl, _, Metadata = get_backend_classes()
    for q_lens in ([1, 1, 45, 130], [1, 1, 1, 1]):
        c = S.attend_case([200, 90, 300, 130], q_lens, tree=False, softcap=12.0, seed=17)
        impl = Impl(8, 128, c["scale"], num_kv_heads=2, logits_soft_cap=12.0)
        md, _ = metadata(Metadata, q_lens, c)
        n = sum(q_lens)
        out = torch.full((n + 2, 1024), float("nan"), dtype=torch.float16, device=DEV)
        q = torch.zeros(n + 2, 1024, dtype=torch.float16, device=DEV)
        q[:n] = on(c["Q"]).view(n, -1)
        impl.forward(None, q, None, None, vllm_cache(c), md, output=out)
        want, tol, wz, _ = S.tree_reference(c)
        assert bool(((out[:n].double().cpu().view(n, 8, 128) - want).abs() <= tol).all()) and bool(out[n:].isnan().all())
    o, z = impl.forward_decode_with_lse(q, vllm_cache(c), md)
    check_tree(c, o, z)
