"""The serving operators at the edges of their rules: where a kernel's shortcut, range or early exit could answer something else."""
import math

import pytest
import torch

from tests import _serving as S
from tests import _serving_exact as X
from tests.test_gpu_serving_ops import check_mass, check_tree, run_tree

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
