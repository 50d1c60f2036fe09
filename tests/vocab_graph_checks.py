"""The C entry points over a vocabulary captured into HIP graphs and replayed: run by test_gpu_vocab_graphs.py in a process that
imports torch first."""
import ctypes

import torch

from tests.test_vocab_host import BF16, F32, I32, I64, AdjustArgs, DistillArgs, EmbedArgs, EmbedGradArgs, lib

V, W, N, K = 5001, 67, 700, 9


class Step:
    """One pass through every operator on buffers of its own; the gradient's scratch may be another's."""

    def __init__(self, L, seed, tokens=N, scratch=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.L, self.g, self.n = L, g, tokens
        new = lambda *s, dt=torch.float32: torch.zeros(s, dtype=dt, device="cuda")
        self.table, self.dy = new(V, W), new(tokens, W)
        self.ids = new(tokens, dt=torch.int64)
        self.z, self.index, self.top = new(40, V, dt=torch.bfloat16), new(40, K, dt=torch.int32), new(40, K)
        self.labels, self.dloss = new(40, dt=torch.int64), new(40)
        self.history, self.lengths = new(40, 300, dt=torch.int32), new(40, dt=torch.int32)
        self.bias, self.allowed = new(40, K), new(40, (V + 31) // 32, dt=torch.int32)
        self.y, self.dtable, self.loss, self.sums = new(tokens, W, dt=torch.bfloat16), new(V, W), new(40), new(40, 3)
        self.dz, self.out = new(40, V, dt=torch.bfloat16), new(40, V)
        p = lambda t: t.data_ptr()
        self.embed = EmbedArgs(F32, BF16, I64, 2.0, tokens, V, W, p(self.table), W, 1, p(self.ids), p(self.y))
        self.grad = EmbedGradArgs(F32, F32, I64, 0, 0.5, tokens, V, W, p(self.dy), W, p(self.ids), p(self.dtable))
        need = L.musapy_embedding_grad_scratch_v1(ctypes.byref(self.grad))
        self.scratch = new(need // 4 + 4) if scratch is None else scratch
        assert self.scratch.numel() * 4 >= need
        self.distill = DistillArgs(BF16, I32, F32, I64, 2.0, 0.5, 40, V, K, p(self.z), V, p(self.index), K, p(self.top), K,
                                   p(self.labels), p(self.loss), p(self.sums), p(self.dloss), 1, p(self.dz))
        self.adjust = AdjustArgs(BF16, F32, I32, I32, F32, I32, 1, 40, V, 300, K, p(self.z), V, p(self.history), 300, p(self.lengths),
                                 None, None, None, 1.2, 0.3, 0.1, p(self.bias), K, p(self.index), K, p(self.allowed),
                                 self.allowed.shape[1], p(self.out))

    def inputs(self):
        r = lambda lo, hi, like: like.copy_(torch.randint(lo, hi, like.shape, device="cuda", generator=self.g))
        for t in (self.table, self.dy, self.top, self.dloss, self.bias, self.z):
            t.copy_(torch.randn(t.shape, device="cuda", generator=self.g))
        r(-1, V + 1, self.ids)
        self.ids[: self.n // 3] = 7
        r(-1, V, self.index), r(-1, V, self.labels), r(0, 200, self.history), r(0, 301, self.lengths), r(-(1 << 31), 1 << 31, self.allowed)

    def run(self):
        s = torch.cuda.current_stream().cuda_stream
        b, L = ctypes.byref, self.L
        rc = [L.musapy_embedding_v1(b(self.embed), s),
              L.musapy_embedding_grad_v1(b(self.grad), self.scratch.data_ptr(), self.scratch.numel() * 4, s),
              L.musapy_distill_loss_v1(b(self.distill), None, 0, s), L.musapy_distill_loss_grad_v1(b(self.distill), s),
              L.musapy_adjust_logits_v1(b(self.adjust), s)]
        assert rc == [0] * 5, (rc, L.musapy_kernels_take_error())

    def results(self):
        return [t.clone() for t in (self.y, self.dtable, self.loss, self.sums, self.dz, self.out)]


def captured(step):
    step.inputs()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.run()
    return graph


def same(a, b):
    return all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))


def check_replays():
    """Replays on new inputs, with eager work between them, give bit for bit what the eager calls give."""
    L = lib()
    for tokens in (50, 100, N, 9000, 17000, 40000):  # without an order, by rank, by blocks, by digits
        step = Step(L, tokens, tokens)
        graph = captured(step)
        for k in range(4):
            step.inputs()
            graph.replay()
            got = step.results()
            for t in (step.y, step.dtable, step.dz, step.out):
                t.fill_(float("nan"))
            step.run()
            assert same(got, step.results()), (tokens, k)
            if k % 2:
                torch.cuda.synchronize()


def check_two_graphs_on_one_scratch():
    """Graphs of a stream that share the gradient's scratch: it may hold anything."""
    L = lib()
    a = Step(L, 1, 40000)
    b = Step(L, 2, N, a.scratch)
    graphs = captured(a), captured(b)
    for k in range(4):
        a.inputs(), b.inputs()
        graphs[k % 2].replay()
        graphs[1 - k % 2].replay()
        a.scratch.fill_(float("nan"))
        got = a.results(), b.results()
        a.run(), b.run()
        assert same(got[0], a.results()) and same(got[1], b.results()), k


if __name__ == "__main__":
    for check in (check_replays, check_two_graphs_on_one_scratch):
        check()
        print(check.__name__, "ok", flush=True)
