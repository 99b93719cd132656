"""The routed layers' values where a form could lose them: an output column much
larger than its neighbours, codes at exact ties, infinite scales and weights, and
adapter sums whose last bits count.  Every form has to give the definition's
value, whatever the number of rows that chose it."""
from __future__ import annotations

import numpy as np
import pytest

from inferrous_amd import CudaContext, load
from test_gpu_routed import Experts, close_bf16

pytestmark = pytest.mark.gpu

F32 = np.float32
INF = np.inf


@pytest.fixture(scope="module")
def env():
    ctx = CudaContext(0)
    return load(ctx), ctx.new_stream(), ctx


# Rows at which experts_mlp runs slot by slot, and expert by expert in tiles of 32, 64, 128
# and 256 rows.
ROWS = [1, 5, 70, 130, 300, 900]


@pytest.mark.parametrize("m", ROWS)
def test_experts_large_columns_cost_their_neighbours_nothing(env, m):
    """Columns 3000 and 100,000 times their neighbours: an output column depends on
    its own scale alone, so the others keep the bound that they had without."""
    c = Experts(m, 2, 3, 192, 144, seed=m)
    want, err = c.want()
    c.sd[:, 5] *= 3000.0
    c.sd[:, 70] *= 1e5
    rest = np.setdiff1d(np.arange(192), [5, 70])
    close_bf16(c.run(env)[:, rest], want[:, rest], err[:, rest])
