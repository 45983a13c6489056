"""The training-step operators in a CUDA graph, from two threads, and in a compiled model."""

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def operators():
    """name -> (inputs that may change, function of them)."""
    import spark_gpt_b200 as b200
    torch.manual_seed(0)
    bias = 0.1 * torch.randn(256, device=DEV)
    w, b = torch.randn(1024, device=DEV), torch.randn(1024, device=DEV)
    tok = torch.randint(50257, (8,), device=DEV)
    return {
        "route one token": (torch.randn(1, 256, device=DEV),
                            lambda x: b200.route_experts(x, 8, bias=bias, num_groups=8, kept_groups=4)),
        "norm": (torch.randn(4, 1024, device=DEV).to(BF16), lambda x: (b200.layer_norm(x, w, b),)),
        "norm of odd rows": (torch.randn(300, 1001, device=DEV).to(BF16), lambda x: (b200.layer_norm(x),)),
        "report": (torch.randn(8, 131072, device=DEV),
                   lambda x: tuple(b200.token_logprobs(x, tok, top=20))),
        "report of rows": (torch.randn(8, 50257, device=DEV).to(BF16),
                           lambda x: tuple(b200.token_logprobs(x, tok, top=5))),
        "balance": (torch.randn(256, device=DEV), lambda x: (b200.balance_bias(x, ids, 0.01),)),
        "norm and clip": (torch.randn(100_000, device=DEV),
                          lambda x: (b200.clip_grads([x[:7], x[8:]], 1.0, out=[c, d]), c, d)),
    }


ids = c = d = None


@pytest.fixture(autouse=True)
def buffers():
    global ids, c, d
    ids = torch.randint(256, (20000,), device=DEV)
    c, d = torch.zeros(7, device=DEV), torch.zeros(99_992, device=DEV)


@pytest.mark.parametrize("name", list(operators()) if torch.cuda.is_available() else ["none"])
def test_replayed_from_a_graph(name):
    """New inputs in the same place: the replay gives the bits of a call."""
    x, f = operators()[name]
    f(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f(x)
    for _ in range(3):
        x.copy_(torch.randn_like(x, dtype=F32))
        graph.replay()
        got = [t.clone() for t in out]
        for a, b in zip(got, f(x)):
            assert torch.equal(a, b)


def test_a_training_step_replayed_from_a_graph():
    import spark_gpt_b200 as b200
    norm = b200.LayerNorm(256).to(DEV)
    head = torch.nn.Parameter(torch.randn(259, 256, device=DEV) * 0.05)
    params = [*norm.parameters(), head]
    x = torch.randn(512, 256, device=DEV).to(BF16)
    tok = torch.randint(259, (512,), device=DEV)

    def step():
        for p in params:
            p.grad = None
        r = b200.token_logprobs(norm(x) @ head.to(BF16).T, tok)
        (-(r.logprob + 0.01 * r.entropy).sum()).backward()
        return b200.clip_grad_norm_(params, 0.5)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n = step()
    held = [p.grad for p in params]
    x.copy_(torch.randn_like(x, dtype=F32))
    graph.replay()
    got = [n.clone(), *(g.clone() for g in held)]
    want = [step(), *(p.grad for p in params)]
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_two_threads_at_once():
    """Each on a stream of its own: the bits of calls made one after the other."""
    ops = operators()
    names = [n for n in ops if n != "norm and clip"]
    want = {n: [t.clone() for t in ops[n][1](ops[n][0])] for n in names}
    torch.cuda.synchronize()
    wrong = []

    def work(order):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                for n in order:
                    x, f = ops[n]
                    got = f(x)
                    stream.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[n])):
                        wrong.append(n)
    threads = [threading.Thread(target=work, args=(o,)) for o in (names, names[::-1])]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


class Block(torch.nn.Module):
    def __init__(self, H=256, E=60, V=259):
        import spark_gpt_b200 as b200
        from tests.test_gpu_step_edges import moe
        super().__init__()
        self.norm = b200.LayerNorm(H).to(DEV)
        self.moe = moe(H, E, 4, 128)

    def forward(self, x, tokens):
        import spark_gpt_b200 as b200
        out, logits, sel = self.moe(self.norm(x))
        r = b200.token_logprobs(out, tokens, top=3)
        w, s = b200.route_experts(out[:, :40], 4, num_groups=4, kept_groups=2)
        return out, logits, sel, r.logprob, r.entropy, r.top_ids, w, s


def test_compiled_model_gives_the_same_bits():
    """The operators run outside the graphs of a compiled model (a break before and behind each), with
    their gradients."""
    torch._dynamo.reset()
    m = Block()
    x = torch.randn(70, 256, device=DEV).to(BF16)
    tokens = torch.randint(256, (70,), device=DEV)

    def run(f, grad):
        m.zero_grad()
        with torch.set_grad_enabled(grad):
            xl = x.clone().requires_grad_(grad)
            out = f(xl, tokens)
        if not grad:
            return list(out)
        torch.autograd.backward([out[0].sum(), out[3].sum(), out[4].sum(), (out[6] * out[7]).sum()])
        return [*out, xl.grad, *(p.grad.clone() for p in m.parameters())]

    compiled = torch.compile(m, dynamic=False)
    for grad in (True, False):
        for _ in range(2):
            for a, b in zip(run(m, grad), run(compiled, grad)):
                assert a.shape == b.shape and torch.equal(a, b)


def test_compiled_step_functions():
    import spark_gpt_b200 as b200
    torch._dynamo.reset()
    ps = [torch.nn.Parameter(torch.zeros(n, device=DEV)) for n in (100, 33)]
    bias = torch.randn(64, device=DEV)
    sel = torch.randint(64, (100, 4), device=DEV)

    def step(scale):
        for p in ps:
            p.grad = torch.full_like(p, 2.0) * scale
        norm = b200.clip_grad_norm_(ps, 1.0)
        return norm, b200.grad_norm([p.grad for p in ps]), b200.balance_bias(bias, sel, 0.5) + 0.0

    want = [*step(3.0), *(p.grad for p in ps)]
    got = [*torch.compile(step)(3.0), *(p.grad for p in ps)]
    for a, b in zip(want, got):
        assert torch.equal(a, b)
