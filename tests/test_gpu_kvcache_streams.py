"""The prompts' kernels of kvcache_attention (plan, tiles, join) captured, replayed with other sequences in the same arrays, on several
streams at once and beside the tensor-core matmul."""
import numpy as np
import pytest
import torch

import kvcache_plain as P

pytestmark = pytest.mark.gpu
ROWS, BATCH = 700, 6
# (lens, new): the numbers of rows a sequence has, and of the groups of rows that the kernels plan, differ from replay to replay
STEPS = [([700, 0, 0, 0, 0, 0], [700, 0, 0, 0, 0, 0]), ([300, 1000, 77, 1, 512, 64], [300, 140, 77, 1, 65, 64]), ([1] * 6, [1] * 6),
         ([0] * 6, [0] * 6), ([2000, 1500, 900, 333, 129, 128], [1, 1, 500, 100, 2, 96]), ([120, 120, 115, 115, 115, 115], [120, 120, 115, 115, 115, 115])]


@pytest.fixture(scope="module")
def TF():
    from deepx_b200 import tensorfunc
    return tensorfunc


def status():
    from deepx_b200 import _native as N
    N.check(N.lib.dx_kvcache_status(None))
    N.check(N.lib.dx_matmul_status(None))


def matmul(A, B, C):
    """Without scratch memory, so that no stream of these tests takes one of the library's banks of counters."""
    from deepx_b200 import _native as N
    N.check(N.lib.dx_matmul(N.BF16, A.data_ptr(), B.data_ptr(), C.data_ptr(), 1, A.shape[0], B.shape[1], A.shape[1], torch.cuda.current_stream().cuda_stream))


class Prompts:
    """Room for ROWS new tokens of BATCH sequences up to 2000 tokens, in fixed arrays; `set` puts another step's sequences into them."""

    def __init__(self, seed, heads, q_heads, dim, fmt):
        self.b = P.Batch(seed, [2000] * BATCH, [0] * BATCH, heads, dim, 16, fmt).fill([2000] * BATCH)
        self.b.table = self.b.host_table.int().cuda()
        self.Q = self.b.rand(ROWS, q_heads, dim, dtype=torch.bfloat16)
        self.Out, self.eager = torch.empty_like(self.Q), torch.empty_like(self.Q)
        self.scale = dim ** -0.5

    def set(self, lens, new):
        self.b.lens, self.b.new = lens, new
        self.b.host_starts = [0] + [int(x) for x in np.cumsum(new)]
        self.b.starts.copy_(torch.tensor(self.b.host_starts, dtype=torch.int32))
        self.b.length.copy_(torch.tensor(lens, dtype=torch.int32))
        for x in (self.Out, self.eager):
            x.fill_(3.0)

    def call(self, TF, out):
        TF.kvcache_attention(self.Q, *self.b.cache(), *self.b.seqs(), self.scale, 0, 0, out, self.b.flag)

    def check(self):
        want, bound = P.attention_rows(self.b, self.Q, self.scale)
        n = self.b.host_starts[-1]
        off = (self.Out[:n].double() - want[:n]).abs()
        assert bool((off <= bound[:n] + P.half_step(torch.bfloat16) * (want[:n].abs() + bound[:n]) + torch.finfo(torch.bfloat16).tiny).all())
        assert bool((self.Out[n:] == 3).all()), "rows behind the last sequence changed"


def capture(call):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    return graph


@pytest.mark.parametrize("dim", [64, 128])
def test_captured_prompts_replay_with_other_sequences(TF, dim):
    """Two captured calls replayed at once on two streams, a matmul on a third between them, an eager call of each afterwards."""
    both = [Prompts(50, 2, 8, dim, "int8"), Prompts(51, 1, 5, dim, "e4m3")]
    for p in both:
        p.set(*STEPS[0])
    graphs = [capture(lambda p=p: p.call(TF, p.Out)) for p in both]
    streams = [torch.cuda.Stream() for _ in range(3)]
    A, B = (torch.randn(1024, 1024, device="cuda").bfloat16() for _ in "ab")
    C, D = torch.empty_like(A), torch.empty_like(A)
    matmul(A, B, D)
    for i, step in enumerate(STEPS * 2):
        for p, other in zip(both, (step, STEPS[(i + 1) % len(STEPS)])):
            p.set(*other)
        C.zero_()
        torch.cuda.synchronize()
        for _ in range(3):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
            with torch.cuda.stream(streams[2]):
                matmul(A, B, C)
        torch.cuda.synchronize()
        assert torch.equal(C, D)
        for p in both:
            p.check()
            p.call(TF, p.eager)
            assert torch.equal(p.eager, p.Out) and int(p.b.flag) == 0
    status()


@pytest.mark.parametrize("dim", [64, 128])
def test_prompts_on_streams_at_once(TF, dim):
    """Eager calls, each with scratch of its own, on three streams, with matmuls in front of and behind them on the same streams."""
    many = [Prompts(52 + i, 1, 4, dim, "int8") for i in range(3)]
    want = []
    for i, p in enumerate(many):
        p.set(*STEPS[(1, 4, 0)[i]])
        p.call(TF, p.eager)
        want.append(p.eager.clone())
    A, B = (torch.randn(512, 4096, device="cuda").bfloat16() for _ in "ab")
    C = [torch.empty(512, 512, dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    Bt = B.T.contiguous()
    matmul(A, Bt, C[3])
    streams = [torch.cuda.Stream() for _ in many]
    torch.cuda.synchronize()
    for _ in range(10):
        for p, stream, c in zip(many, streams, C):
            with torch.cuda.stream(stream):
                matmul(A, Bt, c)
                p.call(TF, p.Out)
    torch.cuda.synchronize()
    for p, w, c in zip(many, want, C):
        assert torch.equal(p.Out, w) and torch.equal(c, C[3])
        p.check()
    status()


def test_compiled_prompts_replay(TF):
    """A compiled program of a prompt's attention behind a matmul, replayed with other sequences in the same tensors."""
    from deepx_b200.executor import Executor
    from helpers import to_np
    p = Prompts(55, 2, 8, 64, "int8")
    p.set(*STEPS[0])
    ex = Executor(0)
    try:
        for name, x in (("q", p.Q), ("a", torch.eye(512).bfloat16())):
            ex.put(name, to_np(x.cpu()))
        for name, x in (("kc", p.b.k), ("vc", p.b.v), ("ks", p.b.ks.nan_to_num(1.0)), ("vs", p.b.vs.nan_to_num(1.0)), ("starts", p.b.starts), ("lens", p.b.length), ("table", p.b.table)):
            ex.put(name, x.cpu().numpy())
        ex.new("c", "bfloat16", (512, 512))
        ex.new("out", "bfloat16", tuple(p.Q.shape))
        line = ("kvcache_attention(tensor<bfloat16>:q, tensor<int8>:kc, tensor<int8>:vc, tensor<float32>:ks, tensor<float32>:vs, tensor<int32>:starts, "
                "tensor<int32>:lens, tensor<int32>:table, var<float32>:0.125, var<int32>:0, var<int32>:0, var<string>:int8)->(tensor<bfloat16>:out)")
        prog = ex.compile("matmul(tensor<bfloat16>:a, tensor<bfloat16>:a)->(tensor<bfloat16>:c)\n" + line)
        for step in STEPS:
            p.set(*step)
            ex.upload("starts", p.b.starts.cpu().numpy())
            ex.upload("lens", p.b.length.cpu().numpy())
            prog.run()
            ex.sync()
            p.call(TF, p.eager)
            n = p.b.host_starts[-1]
            got = np.asarray(ex.download("out")).view(np.uint16)
            assert np.array_equal(got[:n], to_np(p.eager.cpu()).view(np.uint16)[:n])
    finally:
        ex.close()
    status()
