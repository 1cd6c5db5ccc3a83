"""spn4cir_amd.optim.AdamW.step() in a graph: replays train as eager steps do."""
import pytest
import torch

pytestmark = pytest.mark.gpu
HP = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.02)
SHAPES = [(37, 16), (16,), (64, 130), (5,), (1,), (4100, 3)]


@pytest.fixture(scope="module")
def optim():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from spn4cir_amd import optim as o
    return o


def make(seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(s, generator=g).cuda()) for s in SHAPES]


def groups(ps):
    return [dict(params=ps[0::2]), dict(params=ps[1::2], weight_decay=0.0, lr=3e-3)]


def gradients(ps, seed):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(p.shape, generator=g) * 0.1).cuda() for p in ps]


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("warm", ["init_state", "step"])
def test_replays_train(optim, bits, warm):
    """Captured after init_state(), or after a step; then replays with other gradients and eager work between them: the parameters and moments
    of as many eager steps."""
    a, b = make(), make()
    oa, ob = optim.AdamW(groups(a), state_bits=bits, **HP), optim.AdamW(groups(b), state_bits=bits, **HP)
    for p, q, x in zip(a, b, gradients(a, 0)):
        p.grad, q.grad = x.clone(), x.clone()
    done = 0
    if warm == "init_state":
        oa.init_state()
    else:
        oa.step(), ob.step()
        done = 1
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        oa.step()
    for t in range(5):
        for p, q, x in zip(a, b, gradients(a, 1 + t)):
            p.grad.copy_(x), q.grad.copy_(x)
        torch.cuda.synchronize()
        graph.replay()
        ob.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(a, b)), t
        assert float(oa.state[a[0]]["step"]) == done + t + 1
    for p, q in zip(a, b):
        assert all(torch.equal(oa.state[p][k], ob.state[q][k]) for k in ("exp_avg", "exp_avg_sq"))


def test_an_8_bit_first_step_under_capture_is_refused(optim):
    """The refusal leaves the optimizer as it was: the next step is the eager first one."""
    a, b = make(), make()
    oa, ob = optim.AdamW(groups(a), state_bits=8, **HP), optim.AdamW(groups(b), state_bits=8, **HP)
    for p, q, x in zip(a, b, gradients(a, 0)):
        p.grad, q.grad = x.clone(), x.clone()
    graph, other = torch.cuda.CUDAGraph(), torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        other.add_(1.0)
        with pytest.raises(RuntimeError, match="init_state"):
            oa.step()
    oa.step(), ob.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and float(oa.state[a[0]]["step"]) == 1.0


@pytest.mark.parametrize("bits", [8, 32])
def test_a_loaded_state_leaves_an_older_graph_its_memory(optim, bits):
    """A graph captured before load_state_dict() goes on with the moments, counter and tables it was captured with, whatever is allocated
    afterwards; it is the twin that was never loaded."""
    a, b = make(), make()
    oa, ob = optim.AdamW(groups(a), state_bits=bits, **HP), optim.AdamW(groups(b), state_bits=bits, **HP)
    for p, q, x in zip(a, b, gradients(a, 0)):
        p.grad, q.grad = x.clone(), x.clone()
    oa.step(), ob.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        oa.step()
    oa.load_state_dict(oa.state_dict())
    junk = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for n in (64, 512, 1000, 4096, 20000, 100000) for _ in range(20)]
    for _ in range(3):
        torch.cuda.synchronize()
        graph.replay()
        ob.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert all(bool((t == 255).all()) for t in junk)


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("sizes", [(0,), (0, 0), (0, 5)])
def test_parameters_without_elements(optim, bits, sizes):
    """Alone, together and beside others; eager, and captured before any plan exists."""
    from spn4cir_amd import ops
    ps = [torch.nn.Parameter(torch.ones(n, device="cuda")) for n in sizes]
    for p in ps:
        p.grad = torch.ones_like(p)
    plan = ops.AdamWPlan([p.data.clone() for p in ps], state_bits=bits)
    ops.adamw_multi(plan, [p.grad for p in ps], 1, HP)
    assert all(t.numel() == sum((n + 127) // 128 * 128 for n in sizes) for t in plan.moments())
    o = optim.AdamW(ps, state_bits=bits, **HP)
    o.init_state()
    graph, other = torch.cuda.CUDAGraph(), torch.zeros(4, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        other.add_(1.0)
        o.step()
    o.step()
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    assert float(o._step_dev) == 2.0 and all(bool((p < 1.0 - HP["lr"]).all()) for p in ps)


def test_a_flat_run_whose_data_is_replaced(optim):
    """Views of one buffer with their gradients in another; one view, then all of them, move: the bits of tensors that were always separate."""
    def flat(seed):
        buf, out, at = torch.zeros(sum(torch.Size(s).numel() for s in SHAPES), device="cuda"), [], 0
        for p in make(seed):
            out.append(buf[at:at + p.numel()].view(p.shape).copy_(p.detach()))
            at += p.numel()
        return out
    a, b = [torch.nn.Parameter(x) for x in flat(0)], make()
    g = flat(1)
    for p, q, x in zip(a, b, g):
        p.grad, q.grad = x, x.clone()
    oa, ob = optim.AdamW(a, **HP), optim.AdamW(b, **HP)
    for t in range(4):
        if t == 1:
            a[2].data = a[2].data.clone()
        if t == 3:
            for p, x in zip(a, flat(2)):
                p.data = x.copy_(p.data)
        oa.step(), ob.step()
        assert all(torch.equal(p, q) for p, q in zip(a, b)), t


@pytest.mark.parametrize("bits", [8, 32])
def test_a_frozen_parameter_in_front_elsewhere(optim, bits):
    """A frozen parameter of another device (host memory) in front of the trained ones decides nothing."""
    a, b = make(), make()
    for p, q, x in zip(a, b, gradients(a, 0)):
        p.grad, q.grad = x.clone(), x.clone()
    frozen = torch.nn.Parameter(torch.ones(7), requires_grad=False)
    oa, ob = optim.AdamW([frozen] + a, state_bits=bits, **HP), optim.AdamW(b, state_bits=bits, **HP)
    oa.step(), ob.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and bool((frozen == 1).all()) and oa.state[a[0]]["step"].is_cuda
