"""Attention (strata_cuda_attention_dev) of tokens at and behind the table's reach: positions behind it have no place, and what
tokens there see of the positions that have is the mask's, as everywhere. The cases, the formula in 64 bits and the tolerances are
test_attention_gpu.py's."""
import pytest

import strata_cuda as sc

from test_attention_gpu import Case, ctx, torch  # noqa: F401

pytestmark = pytest.mark.gpu


def behind(c, lens):
    """The sequences' lengths, the call's tokens included, wherever their pages end."""
    c.len.copy_(torch.tensor(lens))
    return c


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("sinks", [0, 5])
@pytest.mark.parametrize("window", [1, 36, 37, 63, 64, 65, 99, 100, 101, 128, (1 << 31) - 1, 1 << 31, 1 << 40])
def test_windows_around_the_table(ctx, window, sinks, dtype):  # noqa: F811
    """A table of 64 positions; windows below, at and above it, and lengths inside, at and behind it."""
    lens = [64, 65, 100, 127, 163]
    behind(Case([1] * 5, [63] * 5, 4, 2, 64, 16, dtype, window, sinks, width=4, uniform=1), lens).check(ctx)
    behind(Case([20] * 5, [44] * 5, 4, 2, 64, 16, dtype, window, sinks, width=4, uniform=20), lens).check(ctx)


@pytest.mark.parametrize("sinks", [0, 70])
@pytest.mark.parametrize("window", [500, 1023, 1024, 1025, 1300, 1324, 1 << 31])
def test_windows_around_the_table_in_tiles(ctx, window, sinks):  # noqa: F811
    n = 600
    c = Case([n, n, n], [1024 - n] * 3, 4, 2, 128, 64, "bf16", window, sinks, width=16, uniform=n)
    behind(c, [1024, 1324, 2000]).check(ctx)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window", [(1 << 31) - 3, (1 << 31) - 2, (1 << 31) - 1])
def test_the_last_positions_of_all(ctx, window, dtype):  # noqa: F811
    """Lengths of 2^31 - 1 over a table of 64 positions: the window's begin is next to the first of them."""
    behind(Case([1, 20], [63, 44], 4, 2, 64, 16, dtype, window, 0, width=4), [(1 << 31) - 1] * 2).check(ctx)
    if dtype == "bf16":
        behind(Case([600, 600], [104, 104], 4, 2, 64, 16, dtype, window, 0, width=44), [(1 << 31) - 1, 5]).check(ctx)


@pytest.mark.parametrize("lens,past,window,dtype", [([1], 639, 0, "bf16"), ([1], 639, 200, "bf16"), ([1], 634, 200, "f32"), ([30], 610, 200, "f32"), ([600], 360, 300, "bf16"),
                                                    ([600], 355, 300, "bf16")], ids=str)
def test_the_largest_table(ctx, lens, past, window, dtype):  # noqa: F811
    """The largest reach there is, 2^31 - 16 positions in pages of 16, whose last pages hold the sequence (the others are none):
    tiles that end at 2^31. What is seen is as behind `past` tokens, and so is the result."""
    width = (1 << 27) - 1
    c = Case(lens, [past], 4, 2, 64, 16, dtype, window)
    want, tol = c.want()
    table = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    table[0, width - c.width:] = c.table[0]
    c.len.add_((width - c.width) * 16)
    c.cache = sc.KvCache(c.k.data_ptr(), c.v.data_ptr(), table.data_ptr(), c.len.data_ptr(), n_pages=c.pages, page_size=16, n_kv_head=2, head_dim=64, max_pages=width)
    c.run(ctx)
    torch.cuda.synchronize()
    got = c.obuf[: c.total].unflatten(1, (4, 64)).double()
    assert ((got - want).abs() <= tol).all()
