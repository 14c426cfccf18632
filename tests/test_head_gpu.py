"""top_logits, distill_loss, distill_loss_grad and linear_act at their seams: the C++ host path against the autograd
functions behind it, autograd's rules, graphs, tracing, bounded waits, and the example that runs them together."""
import ctypes
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def head(seed=1, m=130, k=72, n=300, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)
    return normal(m, k), normal(n, k) / 8, normal(n), normal(m, n)


@pytest.fixture
def launches():
    from ddfnet_b200 import _lib
    before = _lib.load().ddf_b200_launch_count()
    return lambda: _lib.load().ddf_b200_launch_count() - before


def test_both_host_paths_agree(launches):
    from ddfnet_b200 import distill_loss, linear_act, top_logits
    from ddfnet_b200.distill import DistillFunction
    from ddfnet_b200.linear import LinearActFunction
    x, w, b, r = (t.requires_grad_() for t in head())
    for act, after in (("none", False), ("relu", False), ("relu", True), ("gelu", False), ("silu", True)):
        y = linear_act(x, w, b, r, activation=act, add="after" if after else "before")
        z = LinearActFunction.apply(x, w, b, r, act, after)
        assert torch.equal(y, z) and "LinearActFunctionBackward" in type(y.grad_fn).__name__ + y.grad_fn.name()
        up = torch.randn_like(y)
        for a, c in zip(torch.autograd.grad(y, (x, w, b, r), up), torch.autograd.grad(z, (x, w, b, r), up)):
            assert torch.equal(a, c)
    teacher = torch.randn(50, 700, device="cuda")
    targets = top_logits(teacher, 9, temperature=2.0)
    s = (teacher + torch.randn_like(teacher)).requires_grad_()
    for reduction in ("none", "sum", "mean"):
        for rest in (targets.rest, None):
            a = distill_loss(s, targets.values, targets.indices, rest, temperature=2.0, reduction=reduction)
            c = DistillFunction.apply(s, targets.values, targets.indices, rest, 2.0, reduction)
            up = torch.rand_like(a)
            assert torch.equal(a, c)
            assert torch.equal(torch.autograd.grad(a, s, up)[0], torch.autograd.grad(c, s, up)[0])
    assert launches() > 0


def test_autograd_rules():
    from ddfnet_b200 import distill_loss, linear_act, top_logits
    x, w, b, r = (t.requires_grad_() for t in head())
    y = linear_act(x, w, b, activation="relu")
    loss = distill_loss(y, *top_logits(r.detach(), 5))
    loss.backward(retain_graph=True)
    first = x.grad.clone()
    loss.backward()
    assert torch.equal(x.grad, first + first)
    with pytest.raises(RuntimeError, match="second time"):
        loss.backward()
    for change in (lambda: w.data.add_(0), lambda: w.mul_(1)):
        y = linear_act(x, w, activation="silu")
        with torch.no_grad():
            change()
        if change.__code__.co_names[0] == "data":
            torch.autograd.grad(y.sum(), x)
        else:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                torch.autograd.grad(y.sum(), x)
    with torch.no_grad():
        assert not linear_act(x, w).requires_grad
    assert not top_logits(x, 3).values.requires_grad
    # an output that did not reach the loss
    y = linear_act(x, w, b)
    z = distill_loss(y.detach().requires_grad_(), *top_logits(r.detach(), 5))
    assert torch.autograd.grad(y.float().mean() * 0 + z * 0, (x, b))[0].abs().sum() == 0


def test_hooks_profiler_and_views():
    from ddfnet_b200 import linear_act
    x, w, b, _ = (t.requires_grad_() for t in head())
    with torch.profiler.profile() as seen:
        linear_act(x, w, b).sum().backward()
    names = {e.name for e in seen.events()}
    assert "LinearActFunction" in names and any("LinearActFunctionBackward" in n for n in names)
    y = linear_act(x.view(13, 10, 72), w, b)
    assert y.shape == (13, 10, 300)
    got = []
    y.register_hook(got.append)
    y[:, ::2].sum().backward()
    assert got[0].shape == y.shape


def test_cuda_graph():
    from ddfnet_b200 import distill_loss_grad, linear_act, top_logits
    x, w, b, r = head(m=257, k=2048, n=1000)
    t = top_logits(r, 8)

    def step():
        y = linear_act(x, w, b, activation="gelu")
        return (y, *distill_loss_grad(y, *t))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    x.copy_(head(seed=2, m=257, k=2048, n=1000)[0])
    graph.replay()
    assert all(torch.equal(a, c) for a, c in zip(out, step()))


def test_a_traced_call_runs_on_new_inputs():
    from ddfnet_b200 import linear_act
    x, w, b, _ = head()
    with torch.no_grad():
        traced = torch.jit.trace(lambda t: linear_act(t, w, b, activation="relu"), (x,), check_trace=False)
        z = head(seed=3)[0]
        assert torch.equal(traced(z), linear_act(z, w, b, activation="relu"))


def test_many_streams_at_once():
    from ddfnet_b200 import linear_act, top_logits
    inputs = [head(seed=i, m=64, k=4096, n=512) for i in range(6)]
    want = [(linear_act(x, w, b), top_logits(r, 7)) for x, w, b, r in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in inputs]
    for _ in range(20):
        got = []
        for s, (x, w, b, r) in zip(streams, inputs):
            with torch.cuda.stream(s):
                got.append((linear_act(x, w, b), top_logits(r, 7)))
        torch.cuda.synchronize()
        for (y, t), (yw, tw) in zip(got, want):
            assert torch.equal(y, yw) and all(torch.equal(a, c) for a, c in zip(t, tw))


def test_a_residual_keeps_up_with_its_piece():
    """The residual's copies run ahead of the pieces they belong to: many tiles a block, every tile width, over and over."""
    from ddfnet_b200 import linear_act
    for m, k, n in ((2500, 512, 2048), (9000, 64, 512), (700, 1024, 96)):
        x, w, b, r = head(m=m, k=k, n=n)
        want = (x.double() @ w.double().t() + r.double()).clamp(min=0)
        for _ in range(40):
            y = linear_act(x, w, None, r, activation="relu")
            assert ((y.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-3).all()


@pytest.mark.parametrize("rows,inputs,outputs", [(300, 256, 512), (64, 4096, 256)])
def test_bounded_waits(rows, inputs, outputs):
    """A product whose operands never arrive: fault 6, the device stays usable, the next call is right."""
    from ddfnet_b200 import _lib, linear_act
    from ddfnet_b200.linear import _args
    L = _lib.load()
    assert L.ddf_b200_take_fault() == 0
    x, w, b, _ = head(m=rows, k=inputs, n=outputs)
    want = linear_act(x, w, b)
    args = _args(x, w, b, None, "none", False)
    size = L.ddf_b200_linear_workspace(ctypes.byref(args))
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    y = torch.full_like(want, 7.0)
    stream = torch.cuda.current_stream().cuda_stream
    call = lambda cycles, starve: L.ddf_b200_linear_waitlimit(ctypes.byref(args), y.data_ptr(), ws.data_ptr(), size, cycles, starve, stream)
    assert call(2_000_000, 1) == 0
    assert L.ddf_b200_take_fault() == 6 and L.ddf_b200_take_fault() == 0
    assert call(2_000_000_000, 0) == 0
    torch.cuda.synchronize()
    assert torch.equal(y, want) and torch.equal(linear_act(x, w, b), want)
    assert L.ddf_b200_take_fault() == 0


def test_example():
    spec = importlib.util.spec_from_file_location("distill_resnet", os.path.join(ROOT, "examples", "distill_resnet.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    losses = module.train(steps=8, batch=16, image=64, k=10, teacher="ddf_add_resnet50", classes=200)
    assert all(loss == loss and loss > 0 for loss in losses) and losses[-1] < 0.9 * losses[0]


def test_no_wait_ran_out():
    from ddfnet_b200 import take_fault
    assert take_fault() == 0
