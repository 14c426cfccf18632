"""linear_act against its definition in 64 bits.

Tolerances.  A sum of K float products of 2-byte numbers is within about sqrt(K) 2^-24 of its summands' norm: with
inputs of unit variance and weights of variance 1 / K, 2e-6 sqrt(K) / 8 at most for the sizes here.  What counts is the
rounding to the type, u = 2^-11 or 2^-8 relative.  Gradients: gz is an operand rounded to the type (u relative, each
on its own), the activation's input likewise, whose error enters by the slope's own slope (at most 1.1 for the
activations here): a sum over n of them is off by 3 u times the root of the sum of squares, at most.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def inputs(m, k, n, dtype, seed, bias=True, residual=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=g, device="cuda")
    return (normal(m, k).to(dtype), (normal(n, k) / math.sqrt(k)).to(dtype), normal(n).to(dtype) if bias else None,
            normal(m, n).to(dtype) if residual else None, normal(m, n).to(dtype))


def act64(z, act):
    if act == "relu":
        return z.clamp(min=0), (z > 0).double()
    if act == "gelu":
        phi = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


def linear64(x, w, b, r, act, add, gy=None):
    x, w, b, r, gy = (t.detach().double() if t is not None else None for t in (x, w, b, r, gy))
    z = x @ w.t()
    z = z + b if b is not None else z
    z = z + r if r is not None and add == "before" else z
    y, slope = act64(z, act)
    y = y + r if r is not None and add == "after" else y
    if gy is None:
        return y
    gz = gy * slope
    grads = {"x": gz @ w, "weight": gz.t() @ x, "bias": gz.sum(0) if b is not None else None,
             "residual": (gz if add == "before" else gy) if r is not None else None}
    # roots of the sums of squares that the gradients' errors are relative to
    scales = {"x": (gy.square() @ w.square()).sqrt(), "weight": (gy.square().t() @ x.square()).sqrt(),
              "bias": gy.square().sum(0).sqrt(), "residual": gy.abs()}
    return y, grads, scales


def check_forward(y, want, dtype, k):
    u = UNIT[dtype]
    off = (y.double() - want).abs()
    bound = u * want.abs() + 4e-7 * math.sqrt(k) + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert y.dtype == dtype and (off <= bound).all(), (off / bound).max().item()


def check_grads(got, grads, scales, dtype):
    u = UNIT[dtype]
    for name, g in got.items():
        off = (g.double() - grads[name]).abs()
        # 3 u of one standard deviation is the rounding's; the largest of some 10^6 normal errors is 5 of them
        bound = u * grads[name].abs() + 5 * u * scales[name] + 1e-6
        assert g.dtype == dtype and (off <= bound).all(), (name, (off / bound).max().item())
        rel = (off.square().sum() / grads[name].square().sum().clamp(min=1e-12)).sqrt().item()
        assert rel <= 3 * u, (name, rel)


FORWARD = [(1, 1, 1), (1, 8, 3), (1, 2048, 1000), (2, 100, 33), (3, 576, 64), (4, 4096, 130), (4, 77, 1000), (5, 64, 64), (7, 8, 16),
           (33, 4096, 512), (127, 63, 65), (128, 64, 256), (129, 65, 257), (300, 1000, 1000), (1024, 128, 512), (1, 8191, 17),
           (200, 8200, 72), (5000, 24, 40), (2500, 512, 2048)]


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("m,k,n", FORWARD)
def test_forward(m, k, n, dt):
    from ddfnet_b200 import linear_act
    x, w, b, r, _ = inputs(m, k, n, DTYPES[dt], m + k + n)
    for act, add, bias, residual in (("none", "before", None, None), ("relu", "before", b, r), ("silu", "after", b, r),
                                     ("gelu", "before", None, r), ("relu", "after", b, None)):
        with torch.no_grad():
            y = linear_act(x, w, bias, residual, activation=act, add=add)
        check_forward(y, linear64(x, w, bias, residual, act, add), DTYPES[dt], k)


TRAIN = [(1, 1, 1), (1, 64, 10), (3, 100, 33), (64, 64, 64), (100, 577, 203), (257, 128, 1000), (1001, 72, 130), (300, 2048, 96),
         (5000, 64, 256), (20000, 40, 24), (512, 1024, 2048)]


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("m,k,n", TRAIN)
def test_gradients(m, k, n, dt):
    from ddfnet_b200 import linear_act
    x, w, b, r, gy = inputs(m, k, n, DTYPES[dt], m * 3 + k + n)
    for act, add, bias, residual in (("none", "before", b, None), ("relu", "before", b, r), ("silu", "after", b, r),
                                     ("gelu", "before", None, r), ("relu", "after", b, r), ("none", "after", None, r)):
        args = {name: t.detach().requires_grad_() for name, t in
                (("x", x), ("weight", w), ("bias", bias), ("residual", residual)) if t is not None}
        y = linear_act(args["x"], args["weight"], args.get("bias"), args.get("residual"), activation=act, add=add)
        want, grads, scales = linear64(x, w, bias, residual, act, add, gy)
        check_forward(y, want, DTYPES[dt], k)
        got = dict(zip(args, torch.autograd.grad(y, list(args.values()), gy)))
        if act == "relu":  # where z rounds to the other side of 0 the slope is a matter of that rounding
            z = linear64(x, w, bias, residual if add == "before" else None, "none", "before")
            gy = torch.where(z.abs() < 1e-5, 0.0, gy).to(gy.dtype)
            got = dict(zip(args, torch.autograd.grad(
                linear_act(*(args.get(a) for a in ("x", "weight", "bias", "residual")), activation=act, add=add),
                list(args.values()), gy)))
            _, grads, scales = linear64(x, w, bias, residual, act, add, gy)
        check_grads(got, grads, scales, DTYPES[dt])


def test_some_gradients_only():
    from ddfnet_b200 import linear_act
    x, w, b, r, gy = inputs(200, 96, 136, torch.bfloat16, 5)
    full = [t.detach().requires_grad_() for t in (x, w, b, r)]
    want = torch.autograd.grad(linear_act(*full, activation="silu"), full, gy)
    for i in range(4):
        args = [t.detach() for t in (x, w, b, r)]
        args[i].requires_grad_()
        got, = torch.autograd.grad(linear_act(*args, activation="silu"), [args[i]], gy)
        assert torch.equal(got, want[i])


def test_gradient_against_differences():
    """A directional derivative in float64 sums of the float16 outputs: with steps of 2^-4 along a unit-norm direction
    each of m n outputs is off by at most 2^-11 |y| u, the sum's error by their root sum of squares."""
    from ddfnet_b200 import linear_act
    m, k, n = 64, 128, 96
    x, w, b, r, gy = inputs(m, k, n, torch.float16, 9)
    for act in ("gelu", "silu", "none"):
        args = [t.detach().requires_grad_() for t in (x, w, b, r)]
        grads = torch.autograd.grad(linear_act(*args, activation=act), args, gy)
        for i in range(4):
            d = torch.randn(args[i].shape, generator=torch.Generator().manual_seed(i)).cuda().half()
            h = 2.0 ** -4
            both = []
            for s in (h, -h):
                moved = [t.detach() for t in (x, w, b, r)]
                moved[i] = moved[i] + s * d
                both.append((moved[i], (linear_act(*moved, activation=act).double() * gy.double()).sum()))
            step = both[0][0].double() - both[1][0].double()  # as rounded
            slope = (grads[i].double() * step).sum()
            # rounding of the outputs, twice; rounding of the gradient; curvature of the activation at this step
            y = linear64(x, w, b, r, act, "before")
            noise = 4 * 2.0 ** -11 * ((y * gy.double()).square().sum().sqrt() * 2 + (grads[i].double() * step).square().sum().sqrt())
            z_step = (lambda: step @ w.double().t(), lambda: x.double() @ step.t(), lambda: step.expand(m, n), lambda: step)[i]()
            curve = (z_step.abs() ** 3 * gy.double().abs()).sum() / 24 * 1.2
            assert abs((both[0][1] - both[1][1] - slope).item()) <= (noise + curve).item()


@pytest.mark.parametrize("dt", list(DTYPES))
def test_layouts(dt):
    """Rows inside wider ones, odd offsets, transposed weights, leading dimensions, channels_last pixels, expanded
    upstream gradients, another stream."""
    from ddfnet_b200 import linear_act
    dtype = DTYPES[dt]
    x, w, b, r, gy = inputs(150, 200, 120, dtype, 3)
    for m in (2, 150):
        for xs, ws, rs in ((x[:m, :96], w[:, :96], r[:m]), (x[:m, 1:98], w[:, 1:98], r[:m, :]), (x[:m, 8:104], w[:, 3:99], r[:m]),
                           (x[:m].t().contiguous().t(), w.t().contiguous().t(), r[:m].t().contiguous().t()),
                           (x[:m, 5:6], w[:, 5:6], r[:m]), (x[:1].expand(m, -1), w, r[:1].expand(m, -1))):
            xg, wg, rg = (t.detach().requires_grad_() for t in (xs, ws, rs))
            y = linear_act(xg, wg, b, rg, activation="silu")
            check_forward(y, linear64(xs, ws, b, rs, "silu", "before"), dtype, 200)
            if m > 2:  # (two rows take another order of the sum where 16 bytes do not divide them)
                plain = [t.detach().contiguous().requires_grad_() for t in (xs, ws, rs)]
                up = gy[:1].expand(m, -1)
                got = [y, *torch.autograd.grad(y, (xg, wg, rg), up)]
                want = linear_act(*plain[:2], b, plain[2], activation="silu")
                want = [want, *torch.autograd.grad(want, plain, up.contiguous())]
                assert all(torch.equal(u, v) for u, v in zip(got, want))
    image = torch.randn(3, 64, 9, 7, device="cuda").to(dtype).contiguous(memory_format=torch.channels_last)
    wide = torch.randn(40, 64, device="cuda").to(dtype) / 8
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        y = linear_act(image.permute(0, 2, 3, 1), wide, activation="relu")
    stream.synchronize()
    assert y.shape == (3, 9, 7, 40)
    want = torch.einsum("bchw,nc->bhwn", image.double(), wide.double()).clamp(min=0)
    check_forward(y, want, dtype, 64)


def test_extreme_values():
    """Infinities, NaN and overflow come out where the definition has them."""
    from ddfnet_b200 import linear_act
    for m in (3, 140):
        x, w, b, r, _ = inputs(m, 70, 50, torch.float16, 4)
        x[0] = 0
        x[0, 3] = float("inf")
        x[1, 5] = float("nan")
        x[2] = 6e4
        w[:, 3] = torch.where(torch.arange(50, device="cuda") % 2 == 0, 1.0, -1.0).half()
        y = linear_act(x, w, b, r, activation="relu")
        want = linear64(x, w, b, r, "relu", "before").half()
        assert torch.equal(y[:2].isnan(), want[:2].isnan()) and y[1].isnan().all()
        assert torch.equal(y[0] == float("inf"), want[0] == float("inf"))
        rows = torch.arange(m, device="cuda") != 1
        assert torch.equal(y[rows].isinf(), want[rows].isinf())


def test_autocast_empty_and_repeatable():
    from ddfnet_b200 import linear_act
    x, w, b, r, gy = inputs(700, 256, 320, torch.bfloat16, 6)
    w32 = w.float().requires_grad_()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = linear_act(x.float(), w32, b.float(), activation="gelu")
    assert y.dtype == torch.bfloat16 and torch.equal(y, linear_act(x, w, b, activation="gelu"))
    y.backward(gy)
    assert w32.grad.dtype == torch.float32
    runs = []
    for _ in range(2):
        args = [t.detach().requires_grad_() for t in (x, w, b, r)]
        y = linear_act(*args, activation="silu", add="after")
        runs.append([y, *torch.autograd.grad(y, args, gy)])
    assert all(torch.equal(a, c) for a, c in zip(*runs))
    args = [t.detach().requires_grad_() for t in (x[:0], w, b, r[:0])]
    y = linear_act(*args, activation="relu")
    assert y.shape == (0, 320)
    grads = torch.autograd.grad(y, args, y.detach())
    assert grads[0].shape == (0, 256) and (grads[1] == 0).all() and (grads[2] == 0).all()


def test_refusals():
    from ddfnet_b200 import linear_act
    x, w, b, r, _ = inputs(4, 32, 16, torch.float16, 1)
    for args, kw, error in (((x.cpu(), w), {}, ValueError), ((x.float(), w.float()), {}, TypeError), ((x, w.bfloat16()), {}, TypeError),
                            ((x, w.t()), {}, ValueError), ((x, w, b[:3]), {}, ValueError), ((x, w, b, r[:2]), {}, ValueError),
                            ((x, w, b.float()), {}, TypeError), ((x, w.cpu()), {}, ValueError), ((x, w[:0]), {}, ValueError),
                            ((x[:, :0], w[:, :0]), {}, ValueError), ((x, w), {"activation": "tanh"}, ValueError),
                            ((x, w, b, r), {"add": "between"}, ValueError), ((x, w, b, r[:1]), {}, ValueError)):
        with pytest.raises(error):
            linear_act(*args, **kw)


def test_no_wait_ran_out():
    from ddfnet_b200 import take_fault
    assert take_fault() == 0
