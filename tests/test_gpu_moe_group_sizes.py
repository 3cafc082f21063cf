"""Routing with groups that end inside a lane's experts (csrc/moe.hip): a lane
holds two experts above 64 of them and four above 128, and its list of keys may
then belong to two groups, of which only one is kept.  Compared as in
test_gpu_moe.py."""
import numpy as np
import pytest

import _mx4ref as R
import bitsqz_amd as B
from test_gpu_moe import check_route
from test_gpu_mx4 import normal, stored

pytestmark = pytest.mark.gpu

# experts, groups, kept, k: groups of 45, 65, 9, 25, 25, 3, 125, 50 and 33 experts
SHAPES = [(180, 4, 2, 8), (130, 2, 1, 8), (72, 8, 3, 6), (100, 4, 2, 6), (200, 8, 4, 8), (150, 50, 20, 9), (250, 2, 1, 5),
          (100, 2, 1, 7), (66, 2, 1, 33)]


def case(type, experts, groups, kept, k, biased):
    rng = np.random.default_rng(experts * groups + kept)
    x = normal(rng, 300, experts, outliers=False) * 1.5
    # tokens with closed experts: every third, all of the first group, all but one
    # of each group, and all
    each = experts // groups
    x[3, ::3], x[4, :each], x[6] = -np.inf, -np.inf, -np.inf
    x[5, np.arange(experts) % each != each - 1] = -np.inf
    raw, x = stored(x, type)
    bias = np.round(rng.standard_normal(experts) * 50).astype(np.float32) * np.float32(0.002) if biased else None
    return raw, x, bias


@pytest.mark.parametrize("type", [B.TYPE_F32, B.TYPE_BF16])
@pytest.mark.parametrize("experts,groups,kept,k", SHAPES)
@pytest.mark.parametrize("biased,sigmoid", [(False, False), (True, True)])
def test_groups_that_end_inside_a_lane(type, experts, groups, kept, k, biased, sigmoid):
    raw, x, bias = case(type, experts, groups, kept, k, biased)
    ids, weights = check_route(raw, x, type, k, bias, sigmoid, groups, kept)
    # whatever the keys' distances: experts of at most `kept` groups, none twice
    for row in ids:
        row = row[row >= 0]
        assert len(set(row.tolist())) == len(row) and len(set((row // (experts // groups)).tolist())) <= kept
    assert (ids[6] == -1).all() and (weights[6] == 0).all()
