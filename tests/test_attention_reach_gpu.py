"""Attention (strata_cuda_attention_dev) of tokens behind the table's reach: their positions have no place, and what they see
of the positions that have is the mask's, as everywhere. The cases, the formula in 64 bits and the tolerances are
test_attention_gpu.py's."""
import pytest

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
