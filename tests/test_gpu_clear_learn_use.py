"""GPU tests of the operators that score and train as programs use them: on a stream of their own, in recorded graphs that are
replayed, two calls at once with workspaces of their own, the same inputs twice."""
import pytest

from engine_loader import load_module

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def ops():
    return load_module("clear_ops")


def normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def workspace(need):
    return torch.full((need,), 255, dtype=torch.uint8, device="cuda") if need else None


class Step:
    """one call of every operator on buffers of its own, outputs set to 7 first; long rows and few lanes, so that every one of
    them takes its workspace"""

    def __init__(self, seed, kind=torch.bfloat16):
        c, gen = ops(), torch.Generator(device="cuda").manual_seed(seed)
        rows, d, vocab, self.n = 600, 256, 40000, 3000
        self.x, self.dy = normal(gen, rows, d).to(kind), normal(gen, rows, d).to(kind)
        self.w, self.b = normal(gen, d), normal(gen, d)
        self.z, self.v, self.dh = (normal(gen, 1, self.n, 96).to(kind) for _ in range(3))
        self.state = normal(gen, 1, 96)
        self.tokens = torch.randint(-1, 70, (rows,), generator=gen, device="cuda")
        self.many = torch.randint(0, 500, (9000,), generator=gen, device="cuda")
        self.dmany = normal(gen, 9000, 64).to(kind)
        self.logits = (3 * normal(gen, 20, vocab)).to(kind)
        self.weights = normal(gen, 20)
        self.param, self.grad = normal(gen, 5000), normal(gen, 5000).to(kind)
        like = torch.empty_like
        self.out = {"y": like(self.x), "mean": torch.empty(rows, device="cuda"), "rstd": torch.empty(rows, device="cuda"),
                    "dx": like(self.x), "dw": like(self.w), "db": like(self.w), "h": like(self.z), "last": like(self.state),
                    "dz": like(self.z), "dv": like(self.z), "dstate": like(self.state), "rows": like(self.x),
                    "few": torch.empty((70, d), device="cuda"), "table": torch.empty((500, 64), device="cuda"),
                    "logprobs": torch.empty(20, device="cuda"), "entropy": torch.empty(20, device="cuda"),
                    "stats": torch.empty((20, 2), device="cuda"), "top": torch.empty((20, 7), dtype=torch.int64, device="cuda"),
                    "top_logprobs": torch.empty((20, 7), device="cuda"), "dlogits": like(self.logits)}
        self.table = normal(gen, 70, d)
        self.work = [workspace(n) for n in (c.layer_norm_workspace(self.x), c.gated_recurrence_workspace(self.z),
                                            c.embedding_gradient_workspace(self.many, self.out["table"]),
                                            c.token_logprobs_workspace(self.logits, 7))]
        assert all(w is not None for w in self.work)
        self.saved = workspace(c.gated_recurrence_saved(self.z))
        self.step, self.lr = torch.ones(1, dtype=torch.int32, device="cuda"), torch.full((1,), 0.01, device="cuda")
        self.params = [self.param.clone(), self.param.clone()]
        self.adamw = c.AdamW(self.params[:1], bits=32), c.AdamW(self.params[1:], bits=8)

    def clear(self):
        for t in self.out.values():
            t.fill_(7)

    def run(self):
        c, o = ops(), self.out
        c.layer_norm(self.x, self.w, self.b, o["y"], o["mean"], o["rstd"])
        c.layer_norm_backward(self.dy, self.x, self.w, o["mean"], o["rstd"], o["dx"], o["dw"], o["db"], workspace=self.work[0])
        c.gated_recurrence(self.z, self.v, self.state, o["last"], o["h"], saved=self.saved, workspace=self.work[1])
        c.gated_recurrence_backward(self.z, self.v, self.saved, self.dh, self.state, o["dz"], o["dv"], o["dstate"], workspace=self.work[1])
        c.embedding(self.tokens, self.table, o["rows"])
        c.embedding_gradient(self.tokens, self.dy, o["few"])
        c.embedding_gradient(self.many, self.dmany, o["table"], workspace=self.work[2])
        c.token_logprobs(self.logits, self.tokens[:20], o["logprobs"], o["entropy"], o["stats"], o["top"], o["top_logprobs"], workspace=self.work[3])
        c.token_logprobs_gradient(self.logits, self.tokens[:20], o["stats"], self.weights, o["dlogits"], self.weights, o["entropy"])

    def learn(self):
        for a in self.adamw:
            a.step([self.grad], lr=self.lr, step=self.step, seed=3)
        self.step += 1

    def results(self):
        return [t.clone() for t in self.out.values()]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_recorded_step_replays():
    """every replay gives what eager calls give, with eager work and waits in between"""
    s = Step(1)
    s.clear()
    s.run()
    want = s.results()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.run()
    for _ in range(4):
        s.clear()
        graph.replay()
        torch.cuda.synchronize()
        assert same(s.results(), want)
        s.clear()
        s.run()
        assert same(s.results(), want)


def test_a_recorded_optimizer_follows_its_step_and_rate():
    eager, recorded = Step(2), Step(2)
    graph = torch.cuda.CUDAGraph()
    kept = [t.clone() for t in recorded.params]
    with torch.cuda.graph(graph):
        recorded.learn()
    assert same(recorded.params, kept) and recorded.step.item() == 1
    for i in range(4):
        for s in (eager, recorded):
            s.lr.fill_(0.01 / (i + 1))
        eager.learn()
        graph.replay()
        torch.cuda.synchronize()
        assert same(eager.params, recorded.params) and not same(recorded.params, kept)
        for a, b in zip(eager.adamw, recorded.adamw):
            assert all(same([x.float() for x in p], [x.float() for x in q]) for p, q in zip(a.states, b.states))
        kept = [t.clone() for t in recorded.params]


def test_two_steps_at_once_on_streams_of_their_own():
    """each with its workspaces, while the null stream is busy"""
    steps = Step(3), Step(4)
    want = []
    for s in steps:
        s.clear()
        s.run()
        want.append(s.results())
        s.clear()
    torch.cuda.synchronize()
    big, streams = torch.zeros((4096, 4096), device="cuda"), [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(8):
        big @ big
    for _ in range(3):
        for s, stream in zip(steps, streams):
            with torch.cuda.stream(stream):
                s.run()
    for stream in streams:
        stream.synchronize()
    assert all(same(s.results(), w) for s, w in zip(steps, want))
    torch.cuda.synchronize()


def test_a_stream_that_is_given_is_the_one_that_is_used():
    c, s, side = ops(), Step(5), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        s.x.fill_(1.0)
    c.layer_norm(s.x, None, s.b, s.out["y"], stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(s.out["y"], s.b.to(s.x.dtype).expand_as(s.x))


def test_the_model_learns_on_a_stream_of_its_own():
    learn = load_module("clear_learn")
    tokens = torch.randint(0, 500, (4, 60), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    ends = []
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            model = learn.Learner(layers=1, d=64, vocab=500, seed=2, dtype=torch.float32)
            losses = [model.learn(tokens) for _ in range(3)]
            stream.synchronize()
        ends.append((torch.stack(losses), [w.clone() for w in model.matrices]))
        torch.cuda.synchronize()
    assert torch.equal(ends[0][0], ends[1][0]) and same(ends[0][1], ends[1][1])
