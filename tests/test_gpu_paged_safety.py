"""What the paged cache's operators do where a caller or the cache's contents go wrong: values
that no row sees, bounds that are too small, tokens that belong to nobody, memory that overlaps.

Tolerances are those of test_gpu_paged.py (derived there)."""

import math

import pytest
import torch

from test_gpu_paged import BF16, F16, F32, check, make, restate, run
from wisp_b200 import paged
from wisp_b200.lib import WispError

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------ hidden values
@pytest.mark.parametrize("dim,cache", [(64, F16), (128, BF16)])
@pytest.mark.parametrize("heads,window,sinks", [((8, 2), 0, 0), ((4, 4), 100, 70)])
def test_two_row_tiles_behind_one_tile_of_hidden_nans(cuda, dim, cache, heads, window, sinks):
    """Row tiles of more than 128 rows share each V tile: infinities and NaNs that no row sees
    (the ends of pages) are taken out of it before either half's product reads it."""
    for fill in (math.nan, math.inf):
        args = make([(260, 300), (129, 129), (64, 1000), (200, 333)], heads=heads, dim=dim,
                    page=48, cache=cache, fill=fill)
        first, _ = run(args, window=window, sinks=sinks)
        for _ in range(20):
            again = paged.attention(*args, window=window, sinks=sinks)
            assert torch.equal(again, first)
