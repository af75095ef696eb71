"""A step of several answers to common prompts with 8-bit weights: rows quantised, queries, attention behind the shared positions, the product back into the residual, logits, the next tokens and how
likely they are. Each operator is checked against 64 bits on what the one before it left; then the whole step is captured, replayed with other inputs and compared with its own calls, bit for bit.

Tolerances: codes and scales as IEEE says; a product of codes is exact but for the five roundings of its scales and sums (half a unit each, of the sizes added up); attention as where it is tested
by itself (2^-24 * 44 of a value, three times that over a row's norm); a log probability is off by the roundings of the maximum's difference, of the logarithm and of their difference:
2^-24 * (2 * 40 + 4 * 2) = 5.3e-6 for logits within 40 of each other."""
import pytest
import torch
from answers_testlib import SharedStep, codes_of, logprobs_of

pytestmark = pytest.mark.gpu
D, VOCAB, TOP = 512, 1000, 5


class _Step:
    def __init__(self, dim, groups, seed):
        from simplellminference_b200.config import BF16
        from simplellminference_b200.seqops import Ops
        self.ops, self.s, self.dim, self.heads, self.kv_heads = Ops(BF16), SharedStep(groups, D // dim, 2, dim, seed=seed), dim, D // dim, 2
        self.T = T = self.s.n_tokens
        g = torch.Generator().manual_seed(seed)
        self.w = {name: torch.randn(n, D, generator=g).to(torch.bfloat16) / 16 for name, n in (("q", D), ("o", D), ("head", VOCAB))}
        self.w8 = {}
        for name, w in self.w.items():
            codes, scale, w = torch.empty(w.shape, dtype=torch.int8, device="cuda"), torch.empty(w.shape[0], device="cuda"), w.cuda()
            self.ops.quantise_rows(w.data_ptr(), True, D, codes.data_ptr(), D, scale, w.shape[0], D, torch.cuda.current_stream().cuda_stream)
            torch.cuda.synchronize()
            self.w8[name] = (codes, scale)
        self.k, self.v = self.s.k.cuda(), self.s.v.cuda()
        self.x, self.u = torch.empty(T, D, device="cuda"), torch.empty(T, device="cuda")
        self.codes = {name: (torch.empty(T, D, dtype=torch.int8, device="cuda"), torch.empty(T, device="cuda")) for name in self.w}
        self.q, self.att, self.y, self.logits = (torch.empty(T, n, device="cuda") for n in (D, D, D, VOCAB))
        self.idx, self.rank, self.best = (torch.empty(n, dtype=torch.int32, device="cuda") for n in ((T,), (T,), (T, TOP)))
        self.logprob, self.entropy, self.best_lp = (torch.empty(n, device="cuda") for n in ((T,), (T,), (T, TOP)))
        self.ws = torch.empty(self.ops.attention_shared_ws_bytes(self.s.b, len(groups), self.heads, 2, dim, dim), dtype=torch.uint8, device="cuda")
        self.results = ("q", "att", "y", "logits", "idx", "rank", "best", "logprob", "entropy", "best_lp")

    def set(self, seed):
        g = torch.Generator().manual_seed(seed)
        self.x.copy_(torch.randn(self.T, D, generator=g))
        self.u.copy_(torch.rand(self.T, generator=g))

    def linear(self, x, name, out, st, accumulate=False):
        (codes, scale), (w, ws) = self.codes[name], self.w8[name]
        self.ops.quantise_rows(x.data_ptr(), False, D, codes.data_ptr(), D, scale, self.T, D, st)
        self.ops.linear8(codes.data_ptr(), D, scale, w, D, ws, None, out.data_ptr(), out.shape[1], self.T, out.shape[1], D, st, accumulate=accumulate)

    def run(self):
        st, s = torch.cuda.current_stream().cuda_stream, self.s
        self.linear(self.x, "q", self.q, st)
        self.ops.attention_shared(s.b, s.group_len.numel(), s.group_start, s.group_len, self.q.data_ptr(), D, self.heads, 2, self.dim, self.dim, self.dim ** -0.5, self.k, self.v, s.n_pages, self.ws, st,
                                  out=self.att, ldo=D)
        self.y.copy_(self.x)
        self.linear(self.att, "o", self.y, st, accumulate=True)
        self.linear(self.y, "head", self.logits, st)
        self.ops.sample_rows(self.logits.data_ptr(), VOCAB, self.T, VOCAB, None, None, None, None, self.u, self.idx, st)
        self.ops.token_logprobs(self.logits.data_ptr(), VOCAB, self.T, VOCAB, self.idx, st, logprob=self.logprob, entropy=self.entropy, rank=self.rank, top=TOP, top_idx=self.best, top_logprob=self.best_lp)

    def check(self):
        torch.cuda.synchronize()
        self.ops._ck(self.ops.lib.sllm_status())

        def product(x, name, out, before=None):
            codes, scale = (t.cpu() for t in self.codes[name])
            want, ws = codes_of(x.cpu())
            assert torch.equal(codes, want) and torch.equal(scale, ws)
            w, w_scale = codes_of(self.w[name])
            v = (codes.double() @ w.double().T) * scale.double()[:, None] * w_scale.double()
            size = v.abs()
            if before is not None:
                v, size = v + before.cpu().double(), size + before.cpu().double().abs()
            assert ((out.cpu().double() - v).abs() <= 5 * 2.0 ** -24 * size).all()

        product(self.x, "q", self.q)
        self.s.q = self.q.cpu()
        want, got = self.s.want(), self.att.cpu().double()
        assert (got - want).norm() <= 8e-6 * want.norm()
        product(self.att, "o", self.y, self.x)
        product(self.y, "head", self.logits)
        logits, idx = self.logits.cpu(), self.idx.cpu()
        assert (logits.amax(1) - logits.amin(1)).max() < 40 and ((idx >= 0) & (idx < VOCAB)).all()
        logprob, rank, entropy, best, best_lp = logprobs_of(logits, idx.long(), TOP)
        assert (self.logprob.cpu().double() - logprob).abs().max() <= 5.3e-6 and (self.best_lp.cpu().double() - best_lp).abs().max() <= 5.3e-6
        assert torch.equal(self.rank.cpu().long(), rank.long()) and torch.equal(self.best.cpu().long(), best)
        assert (self.entropy.cpu().double() - entropy).abs().max() <= 3e-5             # (a sum of 1000 such numbers by their weights, and of the weights' own roundings times them)

    def left(self):
        torch.cuda.synchronize()
        return [getattr(self, name).clone() for name in self.results]


STEPS = {"answers": [(200, [(i * 7 % 50, 1) for i in range(6)]), (0, [(33, 1)])], "one": [(64, [(0, 1)])], "portions and answers": [(300, [(0, 40), (3, 1), (90, 1)]), (31, [(5, 3), (0, 17)])]}


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("groups", list(STEPS.values()), ids=list(STEPS))
def test_a_step(groups, dim):
    step = _Step(dim, groups, 3)
    for seed in (1, 2):
        step.set(seed)
        step.run()
        step.check()


@pytest.mark.parametrize("groups", list(STEPS.values()), ids=list(STEPS))
def test_captured_and_replayed(groups):
    step = _Step(128, groups, 4)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step.set(5)
        step.run()
    want = step.left()
    step.set(6)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g, stream=side):
        step.run()
        step.run()                   # twice: the second's first kernels may start while the first's last are at work
    step.ops.overlap(g.raw_cuda_graph())
    g.instantiate()
    g.replay()
    step.check()
    step.set(5)
    torch.cuda.synchronize()
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(want, step.left()))


def test_two_steps_at_once():
    """On two streams, a workspace each: what either leaves is what it leaves alone."""
    steps = [_Step(128, STEPS["portions and answers"], 7), _Step(64, STEPS["answers"], 8)]
    want = []
    for i, step in enumerate(steps):
        step.set(10 + i)
        torch.cuda.synchronize()
        step.run()
        want.append(step.left())
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for step, st in zip(steps, streams):
            with torch.cuda.stream(st):
                step.run()
    for step, was in zip(steps, want):
        assert all(torch.equal(a, b) for a, b in zip(was, step.left()))
