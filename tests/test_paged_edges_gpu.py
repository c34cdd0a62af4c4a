"""GPU: calls of the paged KV cache at the edges of what its contract allows, against the plain
64-bit forms."""
import pytest
import torch

from tests import paged_ref as ref
from tests.test_paged_gpu import _check_attn

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


# ------------------------------------------------------------------ records of two query tiles

@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("behind", [300, 5000])
@pytest.mark.parametrize("group,tokens", [(3, (43, 44, 48, 51, 84, 85)), (5, (26, 27, 28, 50, 51)), (6, (22, 23, 42)),
                                          (7, (19, 20, 21, 36)), (12, (11, 12, 20)), (33, (4, 5, 6)), (100, (2, 3))])
def test_attn_one_sequence_with_groups_that_do_not_divide_a_tile(dev, group, tokens, behind, D):
    """A chunk of one sequence that fills one query tile and part of a second one, its slots shared
    out to many CTAs: every row of both tiles comes back from the records."""
    for T in tokens:
        _check_attn(ref.make(dev, [T], [T + behind], hkv=2, group=group, D=D, page=64, dtype=F16, seed=T))
