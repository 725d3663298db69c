"""Sizes at the end of what the serving operators' 32-bit places hold: refused before anything is launched (no GPU)."""
import pytest
import torch

from tests.test_serving_host import al, attend, lib  # noqa: F401  (fixtures)


def test_lists_whose_places_would_wrap_are_refused(lib, al):  # noqa: F811
    L = lib.lib
    for budget in (2 ** 31 - 1, 0x7fff0001):
        assert L.cda_b200_select_keys(al, al, al, al, 1, 1, 50, budget, 0, 0, None) == lib.CDA_ERR_N_TOO_LARGE
        assert L.cda_b200_compact_cache(al, al, al, al, None, None, 0, 1, 1, budget, 1, 16, 8, 256, 144, None) == lib.CDA_ERR_N_TOO_LARGE


def test_sequences_whose_places_would_wrap_are_refused(lib, al):  # noqa: F811
    L = lib.lib
    need = L.cda_b200_tree_attention_workspace_bytes(8, 2, 3, -1)
    huge = attend(max_n=2 ** 31 - 1, stride=1 << 28)
    assert L.cda_b200_tree_attention(al, al, al, al, al, al, al, None, None, al, None, al, need, *huge) == lib.CDA_ERR_N_TOO_LARGE
    assert L.cda_b200_attention_mass(al, al, al, al, al, al, None, None, al, None, al, 1 << 31, *huge) == lib.CDA_ERR_N_TOO_LARGE


@pytest.mark.parametrize("v", [2 ** 31, 2 ** 32 + 8, -2 ** 31 - 1])
def test_numbers_that_would_reach_the_library_as_others_are_refused(v):
    from sub0_b200 import ops
    with pytest.raises(ValueError):
        ops._int(v, "budget")
    assert ops._int(2 ** 31 - 1, "budget") == 2 ** 31 - 1 and ops._int(torch.tensor(7), "budget") == 7
