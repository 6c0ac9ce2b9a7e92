"""The attention operators between work on other streams: their kernels begin while the kernel before them in the stream ends,
and still see what an event says they wait for, by calls and captured; and work that waits for them sees all they wrote."""
import pytest

import strata_cuda as sc
from test_attention_gpu import Case, ctx, torch  # noqa: F401

pytestmark = pytest.mark.gpu


class Both:
    """An append, attention over it and scored tokens, whose inputs another stream writes late."""

    def __init__(self, ctx, dtype, n, past):  # noqa: F811
        self.ctx, (hq, hkv, d) = ctx, (8, 2, 64)
        self.c = c = Case([n, n], [past, 40], hq, hkv, d, 16, dtype)
        self.rows = rows = 2 * n
        self.inputs = [torch.randn(rows, hq, d, device="cuda"), torch.randn(rows, hkv, d, device="cuda"), torch.randn(rows, hkv, d, device="cuda"),
                       torch.randn(rows, 5003, device="cuda")]
        self.late = [x.clone() for x in self.inputs]
        self.q = torch.zeros(rows, hq, d, dtype=c.qbuf.dtype, device="cuda")
        self.o = torch.zeros_like(self.q)
        self.lp, self.ent = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
        self.targets = torch.arange(rows, dtype=torch.int32, device="cuda")
        self.append = sc.KvAppend(2, hq, d, offsets=c.offsets, q_dtype=c.code)
        self.attend = sc.Attention(2, hq, c.scale, offsets=c.offsets, dtype=c.code)
        self.slow = torch.randn(4096, 4096, device="cuda")
        self.copies = None

    def write(self):
        """What takes a while, then the inputs."""
        x = self.slow
        for _ in range(3):
            x = x @ self.slow
        for dst, src in zip(self.late, self.inputs):
            dst.copy_(src)
        return x

    def calls(self, s):
        c, (q, k, v, logits) = self.c, self.late
        self.ctx.kv_append_dev(self.append, c.cache, q.data_ptr(), k.data_ptr(), v.data_ptr(), self.q.data_ptr(), s)
        self.ctx.attention_dev(self.attend, c.cache, self.q.data_ptr(), self.o.data_ptr(), c.work.data_ptr(), c.work.numel(), s)
        self.ctx.logprobs_dev(logits.data_ptr(), self.rows, 5003, self.targets.data_ptr(), self.lp.data_ptr(), self.ent.data_ptr(), stream=s)

    def outputs(self):
        return [self.q, self.o, self.lp, self.ent, torch.nan_to_num(self.c.k), torch.nan_to_num(self.c.v)]

    def step(self, main, other, third):
        """Inputs by `other`, the calls on `main` behind them, the outputs' copies on `third`."""
        other.wait_stream(main)
        with torch.cuda.stream(other):
            self.write()
        self.calls(main.cuda_stream)  # of what is there before: the kernel that the waiting calls come behind
        main.wait_stream(other)
        self.calls(main.cuda_stream)
        third.wait_stream(main)
        with torch.cuda.stream(third):
            copies = [x.clone() for x in self.outputs()]
        main.wait_stream(third)
        return copies

    def spoil(self):
        for x in self.late:
            x.fill_(0.25)
        for x in (self.q, self.o, self.lp, self.ent):
            x.fill_(9.0)


@pytest.mark.parametrize("dtype,n", [("bf16", 1), ("f32", 1), ("f32", 30), ("bf16", 300)])
def test_calls_between_events(ctx, dtype, n):  # noqa: F811
    b = Both(ctx, dtype, n, 700)
    b.write()
    torch.cuda.synchronize()
    b.calls(torch.cuda.current_stream().cuda_stream or 1)
    torch.cuda.synchronize()
    want = [x.clone() for x in b.outputs()]
    main, other, third = (torch.cuda.Stream() for _ in range(3))
    torch.cuda.synchronize()
    for _ in range(3):
        b.spoil()
        torch.cuda.synchronize()
        with torch.cuda.stream(main):
            got = b.step(main, other, third)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=main):
        copies = b.step(main, other, third)
    for _ in range(3):
        b.spoil()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(copies, want))
