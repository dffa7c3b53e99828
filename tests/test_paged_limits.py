"""What the paged cache's Python layer refuses before a C type could drop bits of it, without a GPU."""
from types import SimpleNamespace

import pytest

from cormorant_amd import paged as P
from cormorant_amd.graph import PagedAttentionNode, SchedulerError, TensorInfo, paged_pool


@pytest.mark.parametrize("window", [-1, 1 << 30, 1 << 32, (1 << 32) + 5, 1 << 64])
def test_windows(window):
    """A window of 2^32 + 5 keys would reach the library as one of 5."""
    cache, batch = SimpleNamespace(kv_heads=2, head_dim=64), SimpleNamespace(tokens=1)
    with pytest.raises(ValueError, match="window"):
        P.paged_attention(cache, batch, None, None, 4, 1 << 23, 20 | 14 << 8, window=window)
    T = TensorInfo
    ins = [T("q", [4, 128], exp=8), paged_pool("pool", 4, 16, 1, 64), T("qs", [3], kind="i32"), T("kl", [2], kind="i32"),
           T("tb", [2, 2], kind="i32")]
    with pytest.raises(SchedulerError, match="window"):
        PagedAttentionNode(ins, T("o", [4, 128], exp=8), heads=2, kv_heads=1, head_dim=64, page=16, window=window)


@pytest.mark.parametrize("eps", [-1, (1 << 61) + 1, 1 << 63, (1 << 64) + 5])
def test_eps(eps):
    """An eps of 2^64 + 5 would reach the library as 5."""
    import torch
    table, entry = torch.zeros(4, 32, dtype=torch.int32), torch.zeros(16, dtype=torch.uint8)
    for kw in (dict(eps_q=eps), dict(eps_k=eps)):
        with pytest.raises(ValueError, match="eps"):
            P.PagedPrep(table, entry, entry, **kw)


def test_o_apart_from_q():
    """The many-row kernels read q again after other workgroups have written o."""
    import torch
    rows = SimpleNamespace(dtype=torch.int16, is_cuda=True, shape=(3, 256), stride=lambda: (256, 1), data_ptr=lambda: 4096)
    cache, batch = SimpleNamespace(kv_heads=2, head_dim=64), SimpleNamespace(tokens=3)
    with pytest.raises(ValueError, match="o is q"):
        P.paged_attention(cache, batch, rows, rows, 4, 1 << 23, 20 | 14 << 8)
