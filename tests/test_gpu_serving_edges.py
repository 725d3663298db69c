"""The serving operators at the edges of their rules: where a kernel's shortcut, range or early exit could answer something else."""
import math

import pytest
import torch

from tests import _serving as S
from tests import _serving_exact as X
from tests.test_gpu_serving_ops import DEV, call_args, check_mass, check_tree, compact_case, on, run_tree

pytestmark = pytest.mark.gpu


def worst(got, want, tol, rows=slice(None)):
    return float(((got.double().cpu() - want).abs() / tol)[rows].max())


# ---- masks ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("group,window", [(4, 70), (4, 200), (8, 130), (1, 300)])
def test_mask_bits_that_name_no_token_move_the_window(group, window):
    """Bits at and above the number of new tokens show no key, but they count for the depth and with it for the window: rows then
    stand up to 63 positions behind the last token's place, and tiles that every other row sees whole hold keys they do not."""
    stray = [-1, (1 << 63) | 1, ((1 << 40) - 1), 0b1011]
    c = S.attend_case([700, 390, 1000], [4, 4, 4], group=group, window=window, masks=[m & (2 ** 64 - 1) for m in stray * 3], seed=group + window)
    check_tree(c, *run_tree(c))
    check_mass(c, S.tree_reference(c)[2].float())


# ---- probabilities and value rows -------------------------------------------------------------------------------------

def sink_case(v_bits, B, n, T, seed):
    """Key 0 of every sequence draws nearly all attention and has a value row of almost zero: what is left of the output are the
    other keys, each some 2^25 below it, with one value row among them so that what is lost of them does not average out."""
    c = S.attend_case([n] * B, [T] * B, v_bits=v_bits, tree=False, seed=seed)
    had = torch.sign(S.O.sylvester_hadamard(128).double()) / math.sqrt(128.0)
    for b in range(B):
        Ks, _ = S.O.gather_sequence(c["cache"], c["block_table"][b], 1, c["block_size"], 4, v_bits)
        k = S.O.decode_rotated(Ks, c["cb_K"])[0].double()[:, 0] @ had             # (H_kv, 128), where Q lives
        k[:, list(S.Cs.OUTLIER_CHANNELS)] = 0.0                       # (channels in which all keys are large)
        unit = (k / k.norm(dim=-1, keepdim=True)).repeat_interleave(c["group"], 0)
        c["Q"][b * T:(b + 1) * T] = (18.0 * unit + 0.1 * c["Q"][b * T:(b + 1) * T].double()).half()
        slots = torch.tensor([X.slot_of(c, b, t) for t in range(1, n)])
        for part in (slice(64, 64 + 16 * v_bits), X.norm_bytes(c, 1)):
            c["cache"][slots, :, part] = c["cache"][slots[0], :, part]
        X.set_norm(c, b, 0, 1, 1e-9)
    return c


@pytest.mark.parametrize("v_bits,B,n,T", [(2, 40, 1500, 1), (2, 12, 1500, 32), (4, 40, 1500, 1), (2, 1, 700, 6)])
def test_small_terms_behind_a_dominant_key(v_bits, B, n, T):
    c = sink_case(v_bits, B, n, T, seed=B)
    out, lse = run_tree(c)
    want, tol = X.tree_bounds(c)
    off = worst(out, want, tol)
    assert off <= 1.0, f"out is {off:.2f} bounds off"


@pytest.mark.parametrize("k_bits,v_bits", [(4, 4), (4, 2), (2, 4), (2, 2)])
@pytest.mark.parametrize("group", [1, 4, 8])
def test_value_rows_are_the_formats(k_bits, v_bits, group):
    """Rows that see a single key give its value row fp16(level * norm), rotated back: rounded once, when it is written."""
    c = S.attend_case([64, 1, 33], [64, 1, 33], k_bits=k_bits, v_bits=v_bits, group=group, seed=group, masks=[1 << t for n in (64, 1, 33) for t in range(n)])
    out, _ = run_tree(c)
    want, tol = X.tree_bounds(c, own=True)
    off = worst(out, want, tol)
    assert off <= 1.0, f"out is {off:.2f} bounds off"


@pytest.mark.parametrize("name", ["ragged, empty sequence", "drafts across a tile", "group 8, 512 rows", "long chain", "all modifiers", "k2v4, page 32"])
def test_tree_attention_within_the_formats_bound(name):
    from tests.test_gpu_serving_ops import TREES
    c = S.attend_case(seed=len(name), **TREES[name])
    out, _ = run_tree(c)
    want, tol = X.tree_bounds(c)
    off = worst(out, want, tol)
    assert off <= 1.0, f"out is {off:.2f} bounds off"


@pytest.mark.parametrize("k_bits,v_bits", [(4, 4), (4, 2), (2, 2), (2, 4)])
@pytest.mark.parametrize("group", [2, 8])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf, 3.0e5, 2.0e6])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(k_bits, v_bits, group, value):
    """A NaN or infinite norm, or one whose rows come near fp16's end or beyond it, in a draft that only some rows see, and in a
    context key behind the window: rows that do not see the key are as they would be, rows that do are NaN where its value row
    is not finite; log-sum-exp does not know values."""
    T = 8
    masks = [(1 << t) | 1 for t in range(T)]                          # a root and seven siblings
    c = S.attend_case([400, 150], [T, T], k_bits=k_bits, v_bits=v_bits, group=group, window=100, masks=masks * 2, seed=3)
    for b, n in enumerate((400, 150)):
        X.set_norm(c, b, n - T + 5, 1, value)                         # the sixth draft, seen by itself alone
        X.set_norm(c, b, n - T - 101, 1, value)                       # behind every row's window
        X.set_norm(c, b, n - T - 128 if b == 0 else 0, 1, value)
    out, lse = run_tree(c)
    want, tol = X.tree_bounds(c)
    finite = torch.ones(2 * T, 2, dtype=torch.bool)                   # (row, KV head): all values that it sees are
    for b, n in enumerate((400, 150)):
        _, Vs = S.O.gather_sequence(c["cache"], c["block_table"][b], n, 16, k_bits, v_bits)
        finite[b * T + 5] = S.O.decode_rotated(Vs, c["cb_V"])[0][:, n - T + 5].isfinite().all(-1)
    assert bool(finite[5].all()) == (value == 3.0e5)                  # (rows of encoded values: levels up to 0.21 of the norm)
    seen = finite.repeat_interleave(group, 1)
    assert worst(out, want, tol, seen) <= 1.0
    assert not bool(out.cpu()[~seen].isfinite().any())
    _, _, wz, ztol = S.tree_reference(c)
    assert float(((lse.double().cpu() - wz).abs() / ztol).max()) <= 1.0


@pytest.mark.parametrize("k_bits", [4, 2])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_keys_that_are_not_finite_reach_the_rows_that_see_them(k_bits, value):
    from sub0_b200 import ops
    T = 6
    masks = [(1 << t) | 1 for t in range(T)]
    c = S.attend_case([300], [T], k_bits=k_bits, masks=masks, seed=4)
    want, tol = X.tree_bounds(c)                                      # of the other rows, which do not see the fourth draft
    z = S.tree_reference(c)[2].float()
    X.set_norm(c, 0, 300 - T + 3, 0, value)
    out, lse = run_tree(c)
    rest = [t for t in range(T) if t != 3]
    assert worst(out, want, tol, rest) <= 1.0 and not bool(out[3].isfinite().any())
    z[3] = 0.0
    weights = torch.ones(T)
    mass = torch.zeros(1, 2, 300, device=DEV)
    ops.attention_mass(on(c["Q"]), on(c["cache"]), on(c["block_table"]), on(c["seq_lens"]), on(z), mass, weights=on(weights), **call_args(c))
    assert ops.kv_status() == 0
    bad = torch.zeros(300, dtype=torch.bool)
    bad[300 - T + 3] = True
    assert bool(mass[..., ~bad].isfinite().all())


@pytest.mark.parametrize("T,group", [(1, 8), (4, 4), (16, 8)])
def test_mass_gives_away_what_the_rows_have(T, group):
    """Every row gives away one, up to the roundings of single terms, which average out, and a bias: the tensor cores cut sums off
    towards zero.  A score of eight steps of 16 products loses on average half a last place (2^-24) of the partial sum in each,
    and partial sums average at half of the score: 2^-23 |x| at most eight halves of it, 2^-22 |x|, weighted as the rows weigh
    their keys.  2^-23 is left for what does not average out of some thousand terms."""
    from sub0_b200 import ops
    c = S.attend_case([3000, 2500, 2000], [T] * 3, H_kv=4, group=group, tree=False, seed=T)
    z = S.tree_reference(c)[2].float()
    mass = torch.zeros(3, 4, 3000, device=DEV)
    ops.attention_mass(on(c["Q"]), on(c["cache"]), on(c["block_table"]), on(c["seq_lens"]), on(z), mass, **call_args(c))
    gain, reach = mass.double().sum().item(), 0.0
    exact = 0.0                                                       # with the log-sum-exp as the call got it, in 32 bits
    for b in range(3):
        x, _, _ = S.sequence_scores(c, b)
        p = torch.nan_to_num(torch.exp(x - z[b * T:(b + 1) * T].double().view(T, 4, group).permute(1, 0, 2)[..., None]))
        exact += p.sum().item()
        reach += (p * torch.nan_to_num(x, neginf=0.0).abs()).sum().item()
    assert abs(gain - exact) <= 2.0 ** -22 * reach + 2.0 ** -23 * exact, f"{(gain - exact) / exact:.2e} of {reach / exact:.2f}"


# ---- limits and status ------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("max_q", [1 << 16, 1 << 23])
def test_query_limits_far_above_the_chunks(max_q):
    """Hundreds of short sequences under a limit that would allow each of them hundreds of thousands of row blocks."""
    c = S.attend_case([40] * 250 + [300], [1] * 250 + [40], H_kv=1, group=8, tree=False, seed=2)
    out, lse = run_tree(c, max_query_len=max_q)
    check_tree(c, out, lse)


@pytest.mark.parametrize("T,group", [(1, 4), (8, 4), (8, 8), (32, 4)])
def test_waits_that_run_out_end_the_calls_cleanly(T, group):
    """One signal of CTA 0 is kept back and the limit of the waits cut to 5 ms, in shares of more tiles than a ring has stages: the
    CTA gives up, what it had to write stays as it was, all else is right, and so is the next call."""
    from sub0_b200 import ops
    B, n = 12, 4000
    c = S.attend_case([n] * B, [T] * B, H_kv=4, group=group, tree=False, seed=T)
    want, tol = X.tree_bounds(c)
    z = S.tree_reference(c)[2].float()
    start = torch.rand(B, 4, n, generator=torch.Generator().manual_seed(1))
    gain, mtol = S.mass_reference(c, z, start)
    dev, cb_V, a = [on(c[k]) for k in ("Q", "cache", "block_table", "seq_lens")], on(c["cb_V"]), call_args(c)

    def tree():
        out = torch.full_like(dev[0], 7.0)
        ops.tree_attention(*dev, out, cb_V=cb_V, **a)
        return out

    def mass():
        got = on(start).clone()
        ops.attention_mass(*dev, on(z), got, **a)
        return got

    ops.kv_clear_status()
    for run, right, bound, before in ((tree, want, tol, torch.full_like(want, 7.0)), (mass, gain, mtol, start.double())):
        try:
            ops.kv_debug(wait_limit_us=5000, withhold_first_k_arrive=True)
            got = run()
            assert ops.kv_status() == ops.KV_WAIT_GAVE_UP
        finally:
            ops.kv_debug()
            ops.kv_clear_status()
        g = got.double().cpu()
        left = g == before
        assert bool(left.any()) and bool((left | ((g - right).abs() <= bound)).all())
        assert not bool(left[-1].any())                               # (the last CTAs' work)
        assert worst(run(), right, bound) <= 1.0 and ops.kv_status() == 0


def busy(milliseconds=60):
    torch.cuda._sleep(int(milliseconds * 1.9e6))


def test_status_waits_for_other_streams():
    """A call on a side stream, still queued behind long work, has reported by the time its status is read, and a status that
    is cleared stays clear of it."""
    from sub0_b200 import ops
    c = S.attend_case([50, 60], [5, 4], seed=1)
    sl = c["seq_lens"].clone()
    sl[1] = 3
    dev = [on(c["Q"]), on(c["cache"]), on(c["block_table"]), on(sl)]
    out, a, cb_V = torch.empty_like(dev[0]), call_args(c), on(c["cb_V"])
    mass = torch.rand(1, 1, 20, device=DEV)
    long = on(torch.tensor([25], dtype=torch.int32))
    side = torch.cuda.Stream()
    calls = (lambda: ops.tree_attention(*dev, out, cb_V=cb_V, **a), lambda: ops.select_keys(mass, long, 8))
    for call in calls:                                                # (once, so that nothing is loaded behind the busy stream)
        call()
    assert ops.kv_status() == ops.KV_LENGTHS
    ops.kv_clear_status()
    for call in calls:
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            busy()
            call()
        assert ops.kv_status() == ops.KV_LENGTHS
        ops.kv_clear_status()
        assert ops.kv_status() == 0
        with torch.cuda.stream(side):
            busy()
            call()
        ops.kv_clear_status()
        torch.cuda.synchronize()
        assert ops.kv_status() == 0
    ops.kv_clear_status()


def test_prefill_status_waits_for_other_streams():
    from sub0_b200 import ops
    from tests import _cases as Cs
    from tests.test_gpu_prefill import prefill_inputs
    case = Cs.paged_case([70], H_kv=1, group=4, seed=2)
    Q, cu = prefill_inputs(case, [5], 3)
    out = torch.empty_like(Q, device=DEV)
    dev = [on(Q), on(case["cache"]), on(case["block_table"]), on(cu), on(torch.tensor([3], dtype=torch.int32)), out]
    cb_K, cb_V = on(case["cb_K"]), on(case["cb_V"])
    call = lambda: ops.prefill_varlen(*dev, cb_K=cb_K, cb_V=cb_V, block_size=16, max_query_len=5, max_seq_len=70)  # noqa: E731
    call()
    assert ops.prefill_status() == ops.PREFILL_QLEN_EXCEEDS_SEQLEN
    ops.prefill_clear_status()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        busy()
        call()
    assert ops.prefill_status() == ops.PREFILL_QLEN_EXCEEDS_SEQLEN
    ops.prefill_clear_status()
    assert ops.prefill_status() == 0
    with torch.cuda.stream(side):
        busy()
        call()
    ops.prefill_clear_status()
    torch.cuda.synchronize()
    assert ops.prefill_status() == 0 and ops.prefill_fault() is False


# ---- selection and compaction -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,M,n,budget", [(1, 300000, 300000, 5000), (2, 270001, 269000, 200000), (90, 20000, 19990, 700), (3, 262144, 262144, 1)])
def test_select_keys_of_rows_that_do_not_fit_on_chip(rows, M, n, budget):
    """Slices of more than 32768 keys are read again in every pass; with more rows than half the SMs a row keeps few CTAs."""
    from sub0_b200 import ops
    gen = torch.Generator().manual_seed(M)
    lens = [n] + [int(v) for v in torch.randint(n // 2, n, (rows - 1,), generator=gen)]
    for ties in (False, True):
        mass = torch.exp(2 * torch.randn(rows, 1, M, generator=gen))
        mass = (8 * mass).round() if ties else mass
        keep, new = ops.select_keys(on(mass), on(torch.tensor(lens)), budget, sink=1 if budget > 1 else 0, recent=min(64, budget // 2))
        order = torch.arange(M)
        want = torch.full((rows, 1, budget), -1, dtype=torch.int32)
        for b, m in enumerate(lens):
            row = mass[b, 0, :m].clone()
            row[:1 if budget > 1 else 0] = math.inf
            row[m - min(64, budget // 2):] = math.inf
            if m > budget:
                pick = torch.sort(row, descending=True, stable=True).indices[:budget].sort().values
            else:
                pick = order[:m]
            want[b, 0, :pick.numel()] = pick.to(torch.int32)
        assert torch.equal(keep.cpu(), want) and new.cpu().tolist() == [min(m, budget) for m in lens]
    assert ops.kv_status() == 0


@pytest.mark.parametrize("shared", [False, True])
def test_compaction_skips_bad_blocks_with_their_weights(shared):
    """Slots whose block, at either end of the move, lies outside the cache stay as they are; a place that no slot came to has the
    weight 0."""
    from sub0_b200 import ops
    cache, table, lens, keep, _, mass = compact_case([600, 300], 200, seed=8, shared=shared)
    bad = table.clone()
    bad[0, 3], bad[0, 20], bad[1, 0], bad[1, 9] = 1 << 30, -1, cache.shape[0] // 16, -7
    keep[0, 0, :5] = torch.arange(5, dtype=torch.int32)               # slots that stay where they are: in a good block,
    keep[1, 0, :5] = torch.arange(5, dtype=torch.int32)               # in a bad one
    want, want_mass = cache.clone(), mass.clone()
    ok = lambda b, t: 0 <= int(bad[b, t // 16]) < cache.shape[0] // 16  # noqa: E731
    place = lambda b, t: int(bad[b, t // 16]) * 16 + t % 16  # noqa: E731
    for b in range(2):
        for h in range(2):
            for i in range(200):
                src = int(keep[b, 0 if shared else h, i])
                moved = src >= 0 and ok(b, src) and ok(b, i)
                if moved:
                    want[place(b, i), h] = cache[place(b, src), h]
                want_mass[b, h, i] = mass[b, h, src] if moved else 0.0
            want_mass[b, h, 200:int(lens[b])] = 0.0
    for with_mass in (True, False):
        got, got_mass = on(cache), on(mass) if with_mass else None
        ops.compact_cache(got, on(bad), on(lens), on(keep), block_size=16, mass=got_mass)
        assert ops.kv_status() == ops.KV_BAD_BLOCK
        ops.kv_clear_status()
        assert torch.equal(got.cpu(), want)
        if with_mass:
            assert torch.equal(got_mass.cpu(), want_mass)


# ---- backend ----------------------------------------------------------------------------------------------------------

def test_backend_caps_scores_of_long_prompts_beside_decodes():
    from sub0_b200.vllm_integration.cda_attn_v2 import get_backend_classes
    from tests.test_gpu_vllm_backend import metadata, vllm_cache
    _, Impl, _, Metadata = get_backend_classes()
    q_lens = [1, 1, 700, 300]
    c = S.attend_case([900, 33, 700, 650], q_lens, tree=False, softcap=15.0, seed=23)
    impl = Impl(8, 128, c["scale"], num_kv_heads=2, logits_soft_cap=15.0)
    md, _ = metadata(Metadata, q_lens, c)
    n = sum(q_lens)
    out = torch.full((n, 1024), float("nan"), dtype=torch.float16, device=DEV)
    impl.forward(None, on(c["Q"]).view(n, -1), None, None, vllm_cache(c), md, output=out)
    want, tol = X.tree_bounds(c)
    assert worst(out.view(n, 8, 128), want, tol) <= 1.0
