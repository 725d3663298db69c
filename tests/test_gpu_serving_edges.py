"""The serving operators at the edges of their rules: where a kernel's shortcut, range or early exit could answer something else."""
import pytest

from tests import _serving as S
from tests.test_gpu_serving_ops import check_mass, check_tree, run_tree

pytestmark = pytest.mark.gpu


# ---- masks ------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("group,window", [(4, 70), (4, 200), (8, 130), (1, 300)])
def test_mask_bits_that_name_no_token_move_the_window(group, window):
    """Bits at and above the number of new tokens show no key, but they count for the depth and with it for the window: rows then
    stand up to 63 positions behind the last token's place, and tiles that every other row sees whole hold keys they do not."""
    stray = [-1, (1 << 63) | 1, ((1 << 40) - 1), 0b1011]
    c = S.attend_case([700, 390, 1000], [4, 4, 4], group=group, window=window, masks=[m & (2 ** 64 - 1) for m in stray * 3], seed=group + window)
    check_tree(c, *run_tree(c))
    check_mass(c, S.tree_reference(c)[2].float())
