"""Host side of the backend's capped scores: what a batch becomes on its way to the kernel (no GPU)."""
import pytest
import torch

from sub0_b200.vllm_integration import cda_attn_v2 as V


def recorded(monkeypatch, q_lens, counts=True):
    from sub0_b200 import ops
    calls = []
    monkeypatch.setattr(ops, "tree_attention", lambda Q, cache, table, lens, out, **kw: calls.append((Q, table, lens, out, kw)))
    _, Impl, _, Metadata = V.get_backend_classes()
    impl = Impl(8, 128, 0.1, num_kv_heads=2, logits_soft_cap=30.0)
    n, B = sum(q_lens), len(q_lens)
    nd = sum(1 for q in q_lens if q == 1)
    md = Metadata(num_actual_tokens=n, num_reqs=B, max_query_len=max(q_lens), max_seq_len=500,
                  query_start_loc=torch.tensor([0] + q_lens).cumsum(0).to(torch.int32), seq_lens=torch.arange(100, 100 + B, dtype=torch.int32),
                  block_table=torch.arange(B * 4, dtype=torch.int32).view(B, 4), slot_mapping=None, num_decodes=nd if counts else 0,
                  num_prefills=B - nd if counts else 0, num_decode_tokens=nd if counts else 0, num_prefill_tokens=n - nd if counts else 0)
    output = torch.zeros(n + 1, 1024, dtype=torch.float16)
    query = torch.arange(n + 1, dtype=torch.float16)[:, None].expand(n + 1, 1024).contiguous()
    impl.forward(None, query, None, None, torch.zeros(3, 16, 2, 72, dtype=torch.float16), md, output=output)
    return calls, md, output


@pytest.mark.parametrize("counts", [True, False])
def test_decodes_and_chunks_go_in_calls_of_their_own(monkeypatch, counts):
    calls, md, output = recorded(monkeypatch, [1, 1, 1, 45, 7], counts)
    assert [c[4]["max_query_len"] for c in calls] == [1, 45]
    (Q, table, lens, out, kw), (Q2, table2, lens2, out2, kw2) = calls
    assert Q.shape == (3, 8, 128) and Q2.shape == (52, 8, 128) and float(Q2[0, 0, 0]) == 3.0
    assert torch.equal(table, md.block_table[:3]) and torch.equal(table2, md.block_table[3:])
    assert torch.equal(lens, md.seq_lens[:3]) and torch.equal(lens2, md.seq_lens[3:])
    assert kw["cu_seqlens_q"].tolist() == [0, 1, 2, 3] and kw2["cu_seqlens_q"].tolist() == [0, 45, 52]
    assert out.data_ptr() == output.data_ptr() and out2.data_ptr() == output[3:].data_ptr()
    assert all(k["softcap"] == 30.0 and k["scale"] == 0.1 and k["max_seq_len"] == 500 and k["block_size"] == 16 for k in (kw, kw2))


@pytest.mark.parametrize("q_lens", [[1, 1, 1], [9, 30], [1]])
def test_batches_of_one_kind_stay_one_call(monkeypatch, q_lens):
    calls, md, _ = recorded(monkeypatch, q_lens)
    assert len(calls) == 1 and calls[0][4]["max_query_len"] == max(q_lens)
    assert calls[0][4]["cu_seqlens_q"].tolist() == md.query_start_loc.tolist() and calls[0][0].shape[0] == sum(q_lens)
