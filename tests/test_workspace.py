"""How the device's workspace grows (cm_host_workspace_growth), without a GPU: outgrown buffers are kept, so requests that
grow a little at a time must not add up."""
import os

import pytest


@pytest.fixture(scope="module")
def growth():
    from cormorant_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        pytest.fail("libcormo_hip.so is not built (run __graft_entry__.build())")
    return _lib.lib().cm_host_workspace_growth


def run(growth, requests):
    held, retired, times = 0, 0, 0
    for need in requests:
        if need > held:
            size = growth(held, need)
            assert size >= need and size >= 2 * held and size % (1 << 21) == 0
            retired, held, times = retired + held, size, times + 1
            assert retired <= held
    return held, retired, times


def test_a_servers_steps(growth):
    """The kept scores of 64 tokens of 32 heads, their tables widened by a page of 16 rows at a time: 250 MB at the end.
    Buffers just large enough were 120 and more, 16 GB together."""
    requests = [64 * 32 * 2 * cap for cap in range(2064, 65537, 16)]
    held, retired, times = run(growth, requests)
    assert held < 2 * requests[-1] + (1 << 22) and times <= 7


@pytest.mark.parametrize("first", [1, 1 << 21, (1 << 21) + 1, 3 << 30])
def test_first_and_jumps(growth, first):
    assert growth(0, first) == -(-first // (1 << 21)) << 21              # nothing held: what the call needs
    held, retired, times = run(growth, [first, first + 1, 10 * first, 10 * first + 1, 200 * first])
    assert times <= 5 and held <= 400 * first + (1 << 24)
