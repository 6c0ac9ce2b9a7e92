"""Which way the gated delta rule reads a call, as far as its workspace shows (0: token by token), without a device."""
import pytest

import strata_cuda as sc


def work(lens, heads=32, dk=128, dv=128):
    off = [0]
    for n in lens:
        off.append(off[-1] + n)
    return sc.gated_delta_work_bytes(sc.GatedDelta(len(lens), heads // 2, heads, dk, dv, offsets=off))


@pytest.mark.parametrize("lens", [[17], [19], [16, 18, 3], [20], [17] * 9, [100, 1, 1], [1] * 40 + [90]])
@pytest.mark.parametrize("empty", [1, 7, 300])
def test_empty_sequences_change_nothing(lens, empty):
    for mixed in ([0] * empty + lens, lens + [0] * empty, [n for v in lens for n in [v] + [0] * empty]):
        assert work(mixed) == work(lens)


def test_few_short_sequences_are_read_token_by_token():
    assert work([16]) == work([19]) == 0 and work([20]) > 0
    assert work([16] * 9) > 0 and work([15] * 9) == 0
