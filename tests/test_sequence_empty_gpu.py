"""Steps in which no sequence has a token: empty tensors have no address."""
import pytest

import strata_cuda as sc

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = sc.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("lens", [dict(seq_len=0), dict(offsets=[0, 0, 0]), dict(offsets=[5, 5, 5])], ids=str)
def test_nothing_to_do(ctx, lens):
    none = torch.empty(0, 64, device="cuda")
    assert none.data_ptr() == 0
    conv_state, state = torch.randn(2, 3, 64, device="cuda"), torch.randn(2, 2, 16, 16, device="cuda")
    kept = conv_state.clone(), state.clone()
    s = torch.cuda.current_stream().cuda_stream or 1
    w = torch.randn(64, 4, device="cuda")
    ctx.short_conv_dev(sc.ShortConv(2, 64, 4, **lens), none.data_ptr(), w.data_ptr(), 0, conv_state.data_ptr(), none.data_ptr(), s)
    shape = sc.GatedDelta(2, 1, 2, 16, 16, **lens)
    assert sc.gated_delta_work_bytes(shape) == 0
    p = none.data_ptr()
    ctx.gated_delta_dev(shape, p, p, p, p, p, 0, 0, state.data_ptr(), p, 0, 0, s)
    torch.cuda.synchronize()
    assert torch.equal(conv_state, kept[0]) and torch.equal(state, kept[1])


def test_bad_shapes_are_refused_all_the_same(ctx):
    for shape in (sc.ShortConv(2, 0, 4, seq_len=0), sc.ShortConv(2, 64, 9, seq_len=0), sc.ShortConv(2, 64, 4, seq_len=0, dtype=sc.F16)):
        with pytest.raises(sc.BackendError):
            ctx.short_conv_dev(shape, 0, 0, 0, 0, 0)
    with pytest.raises(sc.BackendError):
        ctx.gated_delta_dev(sc.GatedDelta(2, 1, 2, 300, 16, seq_len=0), 0, 0, 0, 0, 0, 0, 0, 0, 0)
    with pytest.raises(sc.BackendError):  # a token after all
        ctx.gated_delta_dev(sc.GatedDelta(2, 1, 2, 16, 16, offsets=[0, 0, 1]), 0, 0, 0, 0, 0, 0, 0, 0, 0)
