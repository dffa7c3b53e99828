"""The paged cache's calls at the ends of what their contract allows: lengths that no table holds, the workspace that small
decode steps use, serving entries that share their weights."""
import numpy as np
import pytest

from test_gpu_paged import Case, check_prep, check_read, dev, paged, regs  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("lengths", [(2 ** 31 - 1, 2 ** 31 - 1), (40, 2 ** 31 - 64), (2 ** 30 + 1, 2 ** 31 - 200), (2 ** 31 - 1, 40)])
def test_lengths_past_every_table(paged, lengths, hd, int8):  # noqa: F811
    """kv_len up to 2^31 - 1, in front of more rows of padding than the table has: nothing of such a sequence is
    written, its rows are read back as 0, the other's as they are.  Its tokens attend to every row of the table."""
    import torch
    rng = np.random.default_rng(hd)
    c = Case(rng, [40, 30], [5, 3], hd=hd, int8=int8, tail=1500)
    c.kv_len = np.array(lengths, np.int32)
    cache, batch = check_prep(paged, c, rng, hd, False, False, True, rows=70)
    check_read(paged, c, cache, batch)
    attends_to_the_table(paged, c, lengths)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,wide", [((1, 1), 150), ((60, 3), 4000)])
def test_lengths_past_long_tables(paged, new, wide, hd, int8):  # noqa: F811
    """The attention's other two ways."""
    c = Case(np.random.default_rng(wide), [70, 64], list(new), kv=4, hd=hd, int8=int8, tail=1, wide=wide)
    attends_to_the_table(paged, c, (2 ** 31 - 1, 64))


def attends_to_the_table(P, c, lengths):
    """The tokens of a sequence longer than its table: the same keys as at a length whose new tokens stand just past it."""
    import torch
    cap = c.table.shape[1] * c.page
    q, o, want = dev(c.q), *(torch.zeros((c.T, c.heads * c.hd), dtype=torch.int16, device="cuda") for _ in range(2))
    for kv, out in ((lengths, o), ([cap + n if x > cap else x for x, n in zip(lengths, c.new)], want)):
        c.kv_len = np.array(kv, np.int32)
        cache, batch = c.device(P)
        P.paged_attention(cache, batch, q, out, c.heads, *regs(c.hd))
    assert torch.equal(o, want) and o[:c.new[0]].any()
