"""The 8-bit linear layers on the GPU, more of their paths bit for bit against the oracle: 17 to 32 rows whose workgroups take
several units of columns, and rows whose neighbours hold the largest values."""
import numpy as np
import pytest

import test_gpu_linear8 as cases
from test_gpu_linear8 import L, dev, host, rows, weights  # noqa: F401

pytestmark = pytest.mark.gpu

WIDE = [(17, 200, 8300), (32, 700, 9001), (31, 1500, 16500), (20, 64, 49152)]


@pytest.mark.parametrize("n,k,m", WIDE, ids=str)
@pytest.mark.parametrize("form", ["plain", "bias", "residual", "both"])
def test_columns_unit_by_unit(L, n, k, m, form):  # noqa: F811
    """Two fragments of rows, more columns than the workgroups take at once: the sums cleared, the weights, the parameters and the
    residual loaded for each unit."""
    cases.test_linear(L, n, k, m, form)


@pytest.mark.parametrize("n,k,m", [(17, 200, 8300), (32, 700, 9001)], ids=str)
@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
def test_gate_unit_by_unit(L, oracle_lib, n, k, m, act):  # noqa: F811
    cases.test_gated(L, oracle_lib, n, k, m, act)


@pytest.mark.parametrize("n,k,m", [(1, 1, 33), (1, 16, 33), (3, 17, 40), (16, 960, 96), (16, 961, 96), (9, 1023, 300), (30, 64, 40),
                                   (40, 63, 64), (64, 256, 64), (100, 960, 200), (77, 1001, 90), (200, 1536, 64), (300, 4096, 64)], ids=str)
@pytest.mark.parametrize("at", [0, 1, 2, 3])
def test_neighbours_of_rows_do_not_count(L, n, k, m, at):  # noqa: F811
    """Rows at each offset from a word whose neighbours on both sides are the lowest and highest int16: no maximum, no code, no sum
    has them, from x and from codes."""
    import torch
    from oracle import linear8 as O
    rng = np.random.default_rng([n, k, at])
    x, (w, mult) = rows(rng, n, k, 20), weights(rng, k, m)
    weight = L.Weight8(dev(w), dev(mult))
    for pad in (4, 5):
        wide = torch.full((n, k + pad), -32768, dtype=torch.int16, device="cuda")
        wide[:, 1::2] = 32767
        xv = wide[:, at:at + k]
        xv.copy_(dev(x))
        want, out = O.linear(x, w, mult), torch.zeros(n, m, dtype=torch.int16, device="cuda")
        np.testing.assert_array_equal(host(L.linear8(xv, weight, out)), want)
        out.zero_()
        np.testing.assert_array_equal(host(L.linear8(L.quant_rows(xv), weight, out)), want)
