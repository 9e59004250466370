"""The operators of a serving step without a stream argument: they run on torch's current stream, as the torch operations around
them do."""
import numpy as np
import pytest

import serving_oracle as so
from test_gpu_serving import E4M3, HALF_STEP, gpu, i32, torch  # noqa: F401  (fixtures)

pytestmark = pytest.mark.gpu


class Step:
    """Buffers of a step of two requests, and the four calls; `out` names what they write."""
    page, dim, heads, group, columns, hidden = 16, 64, 2, 2, 64, 128

    def __init__(self, torch, gpu):  # noqa: F811
        rs = np.random.RandomState(2)
        page, dim, heads, group, n = self.page, self.dim, self.heads, self.group, self.columns
        self.tables, self.write = gpu("PageTable", page_size=page), gpu("CacheWrite", head_dim=dim, page_size=page, dtype="bf16")
        self.attend, self.project = gpu("CacheAttention", head_dim=dim, page_size=page, dtype="bf16"), gpu("Matvec4", group=n, dtype="bf16")
        self.rows = rows = heads * (group + 2)
        half = dict(dtype=torch.bfloat16, device="cuda")
        self.x = torch.zeros((8, self.hidden), **half)
        self.codes = torch.from_numpy(rs.randint(0, 256, (rows * dim, self.hidden // 2)).astype(np.uint8)).cuda()
        self.scales = torch.full((self.hidden // n, rows * dim), 0.01, **half)
        self.cached, self.added, self.free, self.count = i32(torch, [0, 0]), i32(torch, [0, 0]), i32(torch, rs.permutation(12)), i32(torch, [12])
        self.out = dict(qkv=torch.zeros((8, rows, dim), **half), table=i32(torch, np.full((2, 4), -1)), lengths=i32(torch, [0, 0]), starts=i32(torch, [0] * 3),
                        slots=i32(torch, [0] * 8), counts=i32(torch, [0, 0]), kc=torch.zeros((12, heads, page, dim), dtype=torch.uint8, device="cuda"),
                        vc=torch.zeros((12, heads, page, dim), dtype=torch.uint8, device="cuda"), ks=torch.ones((12, heads), device="cuda"),
                        vs=torch.ones((12, heads), device="cuda"), o=torch.zeros((8, heads * group, dim), **half))
        torch.cuda.synchronize()

    def inputs(self, torch, seed):  # noqa: F811
        """Fresh inputs, written by torch on its current stream."""
        rs = np.random.RandomState(seed)
        x, added = torch.from_numpy(rs.normal(size=(8, self.hidden))).bfloat16(), rs.randint(1, 5, 2)
        return x.cuda(), i32(torch, added)

    def __call__(self, **kw):
        o, h = self.out, self.heads * self.group
        self.project(self.x, self.codes, self.scales, o["qkv"].view(8, -1), **kw)
        self.tables(self.cached, self.added, self.free, self.count, o["table"], o["lengths"], o["starts"], o["slots"], o["counts"], **kw)
        self.write(o["qkv"][:, h:h + self.heads], o["qkv"][:, h + self.heads:], o["slots"], o["kc"], o["vc"], o["ks"], o["vs"], **kw)
        self.attend(o["qkv"][:, :h], o["kc"], o["vc"], o["ks"], o["vs"], o["table"], o["lengths"], o["starts"], o["o"], 0.125, max_queries=8, max_length=64, **kw)

    def state(self):
        return {n: t.clone() for n, t in self.out.items()}


def test_runs_on_the_current_stream(torch, gpu):  # noqa: F811
    """Inputs that arrive late on a stream of the caller's."""
    step = Step(torch, gpu)
    x, added = step.inputs(torch, 1)
    torch.cuda.synchronize()
    step.x.copy_(x), step.added.copy_(added)
    step()
    torch.cuda.synchronize()
    want = step.state()
    for t in (step.x, step.added, *step.out.values()):
        t.zero_()
    work = torch.zeros((4096, 4096), device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(20):  # some milliseconds in front of the inputs
            torch.mm(work, work, out=torch.empty_like(work))
        step.out["table"].fill_(-1)
        step.x.copy_(x), step.added.copy_(added)
        step()
        got = step.state()
    side.synchronize()
    assert int(want["counts"][0]) == 10
    for name in ("qkv", "table", "lengths", "starts", "slots", "counts", "o"):
        assert torch.equal(got[name][:int(want["starts"][2])] if name == "o" else got[name], want[name][:int(want["starts"][2])] if name == "o" else want[name]), name


def test_captured_without_a_stream(torch, gpu):  # noqa: F811
    """The step recorded on the stream that torch captures, and replayed in turn with eager steps on the default stream."""
    step = Step(torch, gpu)
    step()  # adds nothing
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    start = step.state()
    for seed in range(4):
        x, added = step.inputs(torch, seed)
        results = []
        for run in (graph.replay, step):
            for name, t in step.out.items():
                t.copy_(start[name])
            step.x.copy_(x), step.added.copy_(added)
            run()
            torch.cuda.synchronize()
            results.append(step.state())
        assert int(results[0]["starts"][2]) == int(added.sum()) and float(results[0]["o"][0].abs().max()) > 0
        assert all(torch.equal(results[0][name], results[1][name]) for name in start)


def test_stream_argument_is_taken(torch, gpu):  # noqa: F811
    """A stream that is named is the one that is used, 0 as the default stream, whatever torch's current one is."""
    step = Step(torch, gpu)
    x, added = step.inputs(torch, 5)
    step.x.copy_(x), step.added.copy_(added)
    torch.cuda.synchronize()
    graph, side, other = torch.cuda.CUDAGraph(), torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(other):
        step(stream=side.cuda_stream)
        step(stream=0)
    torch.cuda.synchronize()
    want = step.state()
    with torch.cuda.graph(graph, stream=side):
        step(stream=side.cuda_stream)
    for t in step.out.values():
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(step.out["qkv"], want["qkv"]) and torch.equal(step.out["lengths"], want["lengths"])
