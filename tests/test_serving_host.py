"""CPU-only checks of the serving operators' boundary: what the C entry points and the Python front end refuse, before any GPU is
touched, and the host side of the backend's capped scores."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from sub0_b200 import build
    build.build()
    from sub0_b200 import _lib
    return _lib


@pytest.fixture(scope="module")
def al():
    buf = (C.c_char * 4096)()
    al.keep = buf
    return (C.addressof(buf) + 15) // 16 * 16


def attend(**kw):
    a = dict(T=4, B=2, H_q=8, H_kv=2, bs=16, stride=8, max_q=3, max_n=100, slots=256, width=144, kb=4, vb=4, scale=0.1, cap=0.0, window=0)
    a.update(kw)
    return (a["T"], a["B"], a["H_q"], a["H_kv"], a["bs"], a["stride"], a["max_q"], a["max_n"], a["slots"], a["width"], a["kb"], a["vb"],
            a["scale"], a["cap"], a["window"], None)


REFUSED = [(dict(B=-1), "BAD_ARG"), (dict(T=-1), "BAD_ARG"), (dict(window=-1), "BAD_ARG"), (dict(cap=-1.0), "BAD_ARG"),
           (dict(cap=float("inf")), "BAD_ARG"), (dict(cap=float("nan")), "BAD_ARG"), (dict(scale=float("inf")), "BAD_ARG"),
           (dict(kb=8), "UNSUPPORTED"), (dict(H_q=7), "BAD_SHAPE"), (dict(H_q=130), "UNSUPPORTED"), (dict(width=112), "BAD_SHAPE"),
           (dict(bs=24), "BAD_SHAPE"), (dict(stride=6), "BAD_SHAPE"), (dict(slots=8), "BAD_SHAPE"), (dict(slots=1 << 32), "N_TOO_LARGE")]


@pytest.mark.parametrize("what,code", REFUSED)
def test_attention_refusals(lib, al, what, code):
    want = getattr(lib, "CDA_ERR_" + code)
    L = lib.lib
    need = L.cda_b200_tree_attention_workspace_bytes(8, 2, 3, -1)
    assert L.cda_b200_tree_attention(al, al, al, al, al, al, al, None, None, al, None, al, need, *attend(**what)) == want
    assert L.cda_b200_attention_mass(al, al, al, al, al, al, None, None, al, None, al, 100, *attend(**what)) == want


def test_chunks_of_too_many_rows_are_refused(lib, al):
    L = lib.lib
    for max_q, want in (((1 << 24) + 1, lib.CDA_ERR_N_TOO_LARGE), ((1 << 24), lib.CDA_ERR_WORKSPACE)):
        assert L.cda_b200_tree_attention(al, al, al, al, al, al, al, None, None, al, None, al, 0, *attend(max_q=max_q)) == want
    assert L.cda_b200_attention_mass(al, al, al, al, al, al, None, None, al, None, al, 100, *attend(max_q=(1 << 24) + 1)) == lib.CDA_ERR_N_TOO_LARGE


def test_attention_refusals_of_pointers_and_workspace(lib, al):
    L = lib.lib
    need = L.cda_b200_tree_attention_workspace_bytes(8, 2, 3, -1)
    tree = lambda *p, ws=al, wsb=need, **kw: L.cda_b200_tree_attention(*p, ws, wsb, *attend(**kw))  # noqa: E731
    ok = [al, al, al, al, al, al, al, None, None, al, None]
    for i in (0, 1, 2, 3, 4, 5, 6, 9):
        assert tree(*[None if k == i else p for k, p in enumerate(ok)]) == lib.CDA_ERR_BAD_ARG
    for i in (0, 1, 9):
        assert tree(*[al + 8 if k == i else p for k, p in enumerate(ok)]) == lib.CDA_ERR_BAD_ALIGN
    assert tree(*ok, wsb=need - 1) == lib.CDA_ERR_WORKSPACE and tree(*ok, ws=None) == lib.CDA_ERR_WORKSPACE
    assert tree(*ok, ws=al + 8) == lib.CDA_ERR_BAD_ALIGN
    masked = [al, al, al, al, al, al, al, al, None, al, None]
    assert tree(*masked, max_q=65) == lib.CDA_ERR_UNSUPPORTED                       # a tree has at most 64 tokens
    assert tree(*ok, B=0) == tree(*ok, T=0) == tree(*ok, max_q=0) == tree(*ok, max_n=0) == lib.CDA_OK   # nothing to do
    mass = lambda *p, stride=100, **kw: L.cda_b200_attention_mass(*p, stride, *attend(**kw))  # noqa: E731
    good = [al, al, al, al, al, al, None, None, al, None, al]
    for i in (0, 1, 2, 3, 4, 5, 8, 10):
        assert mass(*[None if k == i else p for k, p in enumerate(good)]) == lib.CDA_ERR_BAD_ARG
    assert mass(*good, stride=99) == lib.CDA_ERR_BAD_SHAPE
    assert mass(*good, B=0) == lib.CDA_OK
    assert L.cda_b200_tree_attention_workspace_bytes(8, 2, 64, -1) >= L.cda_b200_tree_attention_workspace_bytes(8, 2, 1, -1) > 0


def test_eviction_refusals(lib, al):
    L = lib.lib
    sel = lambda m=al, s=al, k=al, n=al, B=2, H=2, M=50, budget=8, sink=1, recent=2: L.cda_b200_select_keys(m, s, k, n, B, H, M, budget, sink, recent, None)  # noqa: E731
    for kw in (dict(B=-1), dict(H=0), dict(M=-1), dict(budget=0), dict(sink=-1), dict(recent=-1), dict(m=None), dict(s=None), dict(k=None), dict(n=None)):
        assert sel(**kw) == lib.CDA_ERR_BAD_ARG
    assert sel(sink=7) == lib.CDA_ERR_BAD_SHAPE and sel(M=1 << 31) == lib.CDA_ERR_N_TOO_LARGE and sel(B=0) == lib.CDA_OK
    cmp_ = lambda c=al, t=al, s=al, k=al, st=None, m=None, M=0, B=2, H=2, K=4, heads=2, bs=16, stride=8, slots=256, W=144: \
        L.cda_b200_compact_cache(c, t, s, k, st, m, M, B, H, K, heads, bs, stride, slots, W, None)  # noqa: E731
    for kw in (dict(B=-1), dict(K=-1), dict(H=0), dict(slots=-1), dict(m=al, M=-1), dict(c=None), dict(t=None), dict(s=None), dict(k=None)):
        assert cmp_(**kw) == lib.CDA_ERR_BAD_ARG
    for kw in (dict(W=128), dict(bs=20), dict(heads=3)):
        assert cmp_(**kw) == lib.CDA_ERR_BAD_SHAPE
    assert cmp_(c=al + 8) == lib.CDA_ERR_BAD_ALIGN and cmp_(B=0) == cmp_(K=0) == lib.CDA_OK


def test_front_end_wants_cuda_tensors(lib):
    from sub0_b200 import ops
    z = torch.zeros
    Q, cache, bt, sl, cu, cb = z(4, 8, 128).half(), z(64, 2, 144, dtype=torch.uint8), z(1, 4, dtype=torch.int32), z(1, dtype=torch.int32), z(2, dtype=torch.int32), z(16)
    a = dict(cb_K=cb, block_size=16, cu_seqlens_q=cu, max_query_len=4, max_seq_len=64)
    with pytest.raises(ValueError):
        ops.tree_attention(Q, cache, bt, sl, Q, cb_V=cb, **a)
    with pytest.raises(ValueError):
        ops.attention_mass(Q, cache, bt, sl, z(4, 8), z(1, 2, 64), **a)
    with pytest.raises(ValueError):
        ops.select_keys(z(1, 2, 64), sl, 8)
    with pytest.raises(ValueError):
        ops.compact_cache(cache, bt, sl, z(1, 2, 4, dtype=torch.int32), block_size=16)


def test_reference_forms_agree_with_the_oracle():
    """The 64-bit forms that the GPU tests use, against the framework's own oracle where the two overlap: a causal chunk."""
    from oracle import cda_oracle as O
    from tests import _serving as S
    c = S.attend_case([70, 33], [9, 4], tree=False, seed=3)
    out, _, lse, _ = S.tree_reference(c)
    want = O.paged_prefill(c["Q"], c["cache"], c["block_table"], c["cu"], c["seq_lens"], cb_K=c["cb_K"], cb_V=c["cb_V"], group=4, block_size=16)
    assert float((out - want.double()).abs().max()) < 4e-3
    gain, _ = S.mass_reference(c, lse.float(), torch.zeros(2, 2, 70))
    assert float((gain.sum(-1) - torch.tensor([[36.0], [16.0]]).double()).abs().max()) < 1e-4       # rows x group, one each


def test_backend_takes_capped_scores():
    from sub0_b200.vllm_integration import cda_attn_v2 as V
    _, Impl, _, Metadata = V.get_backend_classes()
    assert Impl(8, 128, 0.1, num_kv_heads=2).logits_soft_cap is None and Impl(8, 128, 0.1, num_kv_heads=2, logits_soft_cap=0.0).logits_soft_cap is None
    impl = Impl(8, 128, 0.1, num_kv_heads=2, logits_soft_cap=30)
    assert impl.logits_soft_cap == 30.0
    md = Metadata(num_actual_tokens=1, num_reqs=1, max_query_len=1, max_seq_len=1, query_start_loc=None, seq_lens=None, block_table=None,
                  slot_mapping=None, dcp_world_size=2)
    with pytest.raises(NotImplementedError):
        impl.forward(None, torch.zeros(1, 1024).half(), None, None, torch.zeros(1, 16, 2, 72).half(), md, output=torch.zeros(1, 1024).half())
