"""top_logits, distill_loss and distill_loss_grad against their definitions in 64 bits on the CPU.

Tolerances.  The kernels' exponentials are within 2^-22 relative, exponents are rounded once at the size of the
difference from the row's maximum, sums of n terms lose about log2(n) roundings of 2^-24: a share q of the softmax
is within 4e-6 relative for differences up to 20.  Errors of log q enter the loss multiplied by p - q, hence the
absolute part, which goes with T^2; the gradient's listed entries p expm1(-d) have an error of p times that of d.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
INF = float("inf")
LOWEST = {torch.float32: -3.4028234663852886e38, torch.float16: -65504.0, torch.bfloat16: -3.3895313892515355e38}


def logits_of(rows, classes, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, classes, generator=g) * spread).to(dtype)


# ------------------------------------------------------------------ definitions in 64 bits
def top64(x, k, t):
    x = x.double()
    order = x.sort(dim=-1, descending=True, stable=True)[1][..., :k]
    others = x.clone()
    others.scatter_(-1, order, -INF)
    return order, (others / t).logsumexp(-1)


def distill64(x, values, indices, rest, t):
    """(losses, d losses / d x, counted) row by row, class by class."""
    n, v = x.shape
    x, values = x.double(), values.double()
    losses, grad, counted = torch.zeros(n, dtype=torch.float64), torch.zeros(n, v, dtype=torch.float64), []
    for r in range(n):
        listed = {}
        for a, j in zip(values[r].tolist(), indices[r].tolist()):
            if 0 <= j < v:
                listed.setdefault(j, []).append(a / t)
        a_rest = rest[r].item() if rest is not None else -INF
        everything = [a for some in listed.values() for a in some] + [a_rest]
        counted.append(bool(listed) and not max(everything) == -INF)
        if not counted[-1]:
            continue
        logp = torch.tensor(everything, dtype=torch.float64).log_softmax(0).exp().tolist()
        p, at = {}, 0
        for j, some in listed.items():
            p[j] = sum(logp[at:at + len(some)])
            at += len(some)
        p_rest = logp[-1]
        s = x[r] / t
        logq = s.log_softmax(0)
        mask = torch.ones(v, dtype=torch.bool)
        mask[list(listed)] = False
        logq_rest = logq[mask].logsumexp(0) if mask.any() else torch.tensor(-INF, dtype=torch.float64)
        loss = p_rest * (math.log(p_rest) - logq_rest.item()) if p_rest > 0 else 0.0
        for j, pj in p.items():
            if pj > 0:
                loss += pj * (math.log(pj) - logq[j].item())
        losses[r] = loss * t * t
        q_rest = logq_rest.exp()
        if mask.any():
            # (not exp(s - logsumexp): the sum's logarithm would vanish beside the type's lowest value)
            e = (s - s[mask].max()).exp() if s[mask].max() > -INF else torch.zeros(v, dtype=torch.float64)
            grad[r] = t * (q_rest - p_rest) * e / e[mask].sum().clamp(min=1e-300)
        for j, pj in p.items():
            grad[r, j] = t * (logq[j].exp() - pj)
    return losses, grad, torch.tensor(counted)


def check_grad(got, want, t, upstream, dtype):
    """upstream: largest factor of a row's gradient."""
    got = got.detach().double().cpu()
    unit = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    bound = want.abs() * (unit + 1e-5) + upstream * t * 1e-6 + tiny
    off = (got - want).abs()
    assert got.shape == want.shape and (off <= bound).all(), (off / bound).max().item()


def check_loss(got, want, t):
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    off = (got - want).abs()
    assert (off <= 1e-5 * want.abs() + 4e-6 * t * t).all(), (got, want)


# ------------------------------------------------------------------ top logits
SIZES = [(1, 1, 1), (3, 2, 2), (2, 7, 3), (5, 31, 31), (4, 100, 20), (9, 1000, 20), (3, 1009, 128), (2, 1025, 129),
         (2, 4099, 256), (3, 32003, 64), (1, 65536, 40), (2, 131075, 33), (160, 40000, 17), (11, 474, 111), (69, 1000, 116), (40, 1000, 256),
         (160, 8000, 200)]


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("rows,classes,k", SIZES)
def test_top_logits(rows, classes, k, dt):
    from ddfnet_b200 import top_logits
    x = logits_of(rows, classes, DTYPES[dt], rows + classes + k)
    for t in (1.0, 2.5):
        top = top_logits(x.cuda(), k, temperature=t)
        order, rest = top64(x, k, t)
        assert top.indices.dtype == torch.int64 and torch.equal(top.indices.cpu(), order)
        assert top.values.dtype == x.dtype and torch.equal(top.values.cpu(), x.gather(1, order))
        check_rest(top.rest, rest)


def check_rest(got, want):
    got = got.double().cpu()
    assert torch.equal(got == -INF, want == -INF) and torch.equal(got.isnan(), want.isnan())
    fin = torch.isfinite(want)
    assert ((got - want).abs()[fin] <= 4e-6 + 2e-7 * want.abs()[fin]).all()


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("classes,k", [(40, 40), (1000, 7), (3000, 100), (50001, 65)])
def test_top_logits_ties(classes, k, dt):
    """Few distinct values, one value, masked rows, signed zeros, NaN and infinities."""
    from ddfnet_b200 import top_logits
    x = logits_of(9, classes, DTYPES[dt], 5)
    x[0] = x[0].round()
    x[1] = 0.25
    x[2] = -INF
    x[3] = -INF
    x[3, classes // 3::max(1, classes // 5)] = 1.5
    x[4] = LOWEST[DTYPES[dt]]
    x[5] = torch.where(torch.arange(classes) % 2 == 0, 0.0, -0.0)
    x[6, classes // 2] = float("nan")
    x[7, ::max(1, classes // 3)] = INF
    x[8] = torch.arange(classes, 0, -1).clamp(max=7)
    top = top_logits(x.cuda(), k, temperature=2.0)
    order, rest = top64(x, k, 2.0)
    assert torch.equal(top.indices.cpu(), order)
    want = x.gather(1, order)
    assert torch.equal(top.values.cpu().nan_to_num(99.0), want.nan_to_num(99.0))
    finite = [0, 1, 2, 3, 4, 5, 6, 8]
    if k > 4:
        finite.append(7)
    check_rest(top.rest[finite], rest[finite])


@pytest.mark.parametrize("dt", list(DTYPES))
def test_top_logits_layouts(dt):
    """Rows that begin inside 16 bytes, wider rows, other strides, leading dimensions, another stream."""
    from ddfnet_b200 import top_logits
    wide = logits_of(6, 1205, DTYPES[dt], 8).cuda()
    for x in (wide[:, 3:1104], wide[:, :1000], wide[::2, 5:], wide.t(), wide[:1].expand(4, -1), wide.view(2, 3, 1205)):
        top = top_logits(x, 6)
        order, rest = top64(x.cpu(), 6, 1.0)
        assert torch.equal(top.indices.cpu(), order)
        check_rest(top.rest, rest)
    flat = torch.zeros(1 + 3 * 977, dtype=DTYPES[dt], device="cuda")
    flat[1:] = wide.reshape(-1)[:3 * 977]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        top = top_logits(flat[1:].view(3, 977), 11)
    stream.synchronize()
    assert torch.equal(top.indices.cpu(), top64(flat[1:].view(3, 977).cpu(), 11, 1.0)[0])
    empty = top_logits(wide[:0], 4)
    assert empty.values.shape == (0, 4) and empty.rest.shape == (0,)


# ------------------------------------------------------------------ the loss
def targets(x, k, t, with_rest, seed, dtype=None):
    """Targets of a teacher near the student, as top_logits leaves them."""
    g = torch.Generator().manual_seed(seed)
    teacher = (x.double() + torch.randn(x.shape, generator=g, dtype=torch.float64)).to(dtype or x.dtype)
    order, rest = top64(teacher, k, t)
    return teacher.gather(1, order), order, rest.float() if with_rest else None


def to_cuda(*tensors):
    return [t.cuda() if t is not None else None for t in tensors]


LOSS_SIZES = [(1, 1, 1), (2, 2, 1), (3, 9, 4), (5, 100, 100), (130, 1000, 20), (3, 1017, 3), (3, 1025, 256),
              (2, 5003, 30), (4, 32003, 64), (1, 128000, 20), (2, 300007, 33)]


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("rows,classes,k", LOSS_SIZES)
def test_loss_and_gradient(rows, classes, k, dt):
    from ddfnet_b200 import distill_loss, distill_loss_grad
    dtype = DTYPES[dt]
    x = logits_of(rows, classes, dtype, rows + classes)
    for t, with_rest, reduction in ((1.0, False, "none"), (2.0, True, "mean"), (3.0, True, "sum")):
        values, indices, rest = targets(x, k, t, with_rest, k)
        if rows > 2:
            indices[1] = -1                     # a row that is left out
            indices[2, k // 2:] = classes + 5   # fewer entries
        losses, grad, counted = distill64(x, values, indices, rest, t)
        g = torch.Generator().manual_seed(3)
        upstream = torch.rand(rows, generator=g) + 0.5 if reduction == "none" else torch.tensor(0.75)
        count = max(1, int(counted.sum())) if reduction == "mean" else 1
        want_loss = losses if reduction == "none" else losses.sum() / count
        xd = x.cuda().requires_grad_()
        v, i, r = to_cuda(values, indices, rest)
        loss = distill_loss(xd, v, i, r, temperature=t, reduction=reduction)
        assert loss.dtype == torch.float32
        check_loss(loss, want_loss, t * (rows if reduction == "sum" else 1))
        loss.backward(upstream.cuda())
        factor = (upstream.double() / count).reshape(-1, 1).expand(rows, 1)
        check_grad(xd.grad, grad * factor, t, 1.5 / count, dtype)
        assert (xd.grad[~counted.cuda()] == 0).all()
        one, g1 = distill_loss_grad(x.cuda(), v, i.int(), r, temperature=t, reduction=reduction, scale=0.75)
        check_loss(one, want_loss, t * (rows if reduction == "sum" else 1))
        check_grad(g1, grad * (0.75 / count), t, 0.75 / count, dtype)


def test_near_teacher_keeps_its_digits():
    """A student that is its teacher but for 1e-3: the loss is of the order 1e-7, the gradient of 1e-4."""
    from ddfnet_b200 import distill_loss
    teacher = logits_of(64, 1000, torch.float32, 1)
    g = torch.Generator().manual_seed(2)
    x = teacher + 1e-3 * torch.randn(64, 1000, generator=g)
    order, rest = top64(teacher, 20, 1.0)
    values = teacher.gather(1, order)
    want, grad, _ = distill64(x, values, order, rest.float(), 1.0)
    xd = x.cuda().requires_grad_()
    loss = distill_loss(xd, values.cuda(), order.cuda(), rest.float().cuda(), reduction="none")
    # d = log(p / q) is some 1e-3 with an error of 1e-6: losses, quadratic in d, are within a few per mille
    assert ((loss.double().cpu() - want).abs() <= 5e-3 * want + 1e-12).all()
    loss.sum().backward()
    assert ((xd.grad.double().cpu() - grad).abs() <= 1e-6 * (1 + grad.abs())).all()


def test_nearly_one_class():
    """One class has all but 1e-6: log1p keeps what 1 + x would lose."""
    from ddfnet_b200 import distill_loss
    x = torch.zeros(1, 1000)
    x[0, 17] = 21.0
    values, indices = torch.tensor([[3.0]]), torch.tensor([[17]])
    want, grad, _ = distill64(x, values, indices, None, 1.0)
    xd = x.cuda().requires_grad_()
    loss = distill_loss(xd, values.cuda(), indices.cuda())
    assert abs(loss.item() - want.item()) <= 1e-5 * want.item()
    loss.backward()
    assert ((xd.grad.double().cpu() - grad).abs() <= 2e-5 * grad.abs()).all()


@pytest.mark.parametrize("dt", list(DTYPES))
@pytest.mark.parametrize("classes", [50, 1000, 9001])
def test_masks_and_empty_rows(classes, dt):
    from ddfnet_b200 import distill_loss, distill_loss_grad
    dtype, t, k = DTYPES[dt], 2.0, 5
    x = logits_of(9, classes, dtype, 12)
    values, indices, rest = targets(x, k, t, True, 4)
    x[0, indices[0, 0] + 1:] = -INF          # masked classes
    x[1] = LOWEST[dtype]                     # a row of the type's lowest value
    x[2, ::2] = LOWEST[dtype]
    values[3, 2:] = -INF                     # listed, without mass
    values[4] = -INF                         # ... all of them, and no rest: not counted
    rest[4] = -INF
    indices[5] = -7                          # no entry, whatever `rest` says
    values[6] = LOWEST[dtype]                # uniform over the list
    rest[6] = -INF
    x[7].fill_(-INF)                         # only the listed classes are possible
    x[7, indices[7]] = 1.0
    rest[7] = -INF
    indices[8, 3] = indices[8, 1]            # a class listed twice, and thrice
    indices[8, 4] = indices[8, 1]
    keep = torch.tensor([1, 2, 3, 4, 5, 6, 7, 8])  # (row 0's loss is infinite: checked by itself)
    want, grad, counted = distill64(x[keep], values[keep], indices[keep], rest[keep], t)
    v, i, r = to_cuda(values[keep], indices[keep], rest[keep])
    xd = x[keep].cuda().requires_grad_()
    loss = distill_loss(xd, v, i, r, temperature=t, reduction="none")
    check_loss(loss, want, t)
    loss.sum().backward()
    check_grad(xd.grad, grad, t, 1.0, dtype)
    one, g1 = distill_loss_grad(x[keep].cuda(), v, i, r, temperature=t)
    check_loss(one, want.sum() / counted.sum(), t)
    check_grad(g1, grad / counted.sum(), t, 1.0, dtype)
    x0 = x[:1].cuda().requires_grad_()
    loss = distill_loss(x0, *to_cuda(values[:1], indices[:1], rest[:1]), temperature=t)
    loss.backward()
    share = x0.detach().double().cpu()[0] / t
    assert loss.item() == INF or distill64(x[:1], values[:1], indices[:1], rest[:1], t)[0].isfinite()
    masked = (x[0] == -INF)
    masked[indices[0]] = False
    assert (x0.grad[0].cpu()[masked] == 0).all() and torch.isfinite(x0.grad).all() and share.shape[0] == classes
    # no row counts
    none = torch.full_like(i, -1)
    xd = x[keep].cuda().requires_grad_()
    loss = distill_loss(xd, v, none, r)
    loss.backward()
    assert loss.item() == 0 and (xd.grad == 0).all()
    one, g1 = distill_loss_grad(xd.detach(), v, none, r)
    assert one.item() == 0 and (g1 == 0).all()


def test_nan_is_not_hidden():
    from ddfnet_b200 import distill_loss
    for classes in (300, 5000):
        x = logits_of(3, classes, torch.float32, 9)
        values, indices, rest = targets(x, 4, 1.0, True, 4)
        for where in ("student", "listed", "teacher", "infinite"):
            a, b = x.clone(), values.clone()
            if where == "student":
                a[1, classes // 2] = float("nan")
            elif where == "listed":
                a[1, indices[1, 2]] = float("nan")
            elif where == "teacher":
                b[1, 3] = float("nan")
            else:
                a[1, classes // 2] = INF
            ad = a.cuda().requires_grad_()
            loss = distill_loss(ad, *to_cuda(b, indices, rest), reduction="none")
            assert loss[1].isnan() and torch.isfinite(loss[[0, 2]]).all()
            loss.sum().backward()
            assert ad.grad[1].isnan().any() and torch.isfinite(ad.grad[[0, 2]]).all()


def test_layouts_and_types_of_targets():
    from ddfnet_b200 import distill_loss, distill_loss_grad
    wide = logits_of(8, 2100, torch.bfloat16, 31)
    for x in (wide[:, 3:1904], wide[:, :900], wide[::2, 1:], wide[:, :600].reshape(2, 4, 600), wide[:, ::3]):
        flat = x.reshape(-1, x.shape[-1])
        values, indices, rest = targets(flat, 7, 1.0, True, 2, torch.float32)
        want, grad, _ = distill64(flat, values, indices, rest, 1.0)
        lead = x.shape[:-1]
        v, i, r = (a.reshape(*lead, *a.shape[1:]).cuda() for a in (values, indices, rest.double()))
        xd = wide.cuda().as_strided(x.size(), x.stride(), x.storage_offset()).requires_grad_()
        loss = distill_loss(xd, v, i, r, reduction="none")
        check_loss(loss.reshape(-1), want, 1.0)
        loss.backward(torch.ones((), device="cuda").expand(lead))
        check_grad(xd.grad.reshape(grad.shape), grad, 1.0, 1.0, torch.bfloat16)
        one, g1 = distill_loss_grad(xd.detach(), v.half().float(), i.int(), r, reduction="none")
        assert one.shape == lead and g1.shape == x.shape and g1.is_contiguous()


def test_gradient_against_differences():
    """Directional derivatives: the loss is within 1e-6, a central difference over 2 h = 0.1 within that / 0.1 plus its
    third-order term h^2 / 6 times the third derivative (below 1 along a unit direction)."""
    from ddfnet_b200 import distill_loss
    for classes, k in ((40, 5), (1500, 9)):
        x = logits_of(1, classes, torch.float32, 77)
        values, indices, rest = to_cuda(*targets(x, k, 1.0, True, 5))
        xd = x.cuda().requires_grad_()
        distill_loss(xd, values, indices, rest).backward()
        for seed in range(3):
            d = torch.randn(1, classes, generator=torch.Generator().manual_seed(seed)).cuda()
            d /= d.norm()
            up, down = (distill_loss(x.cuda() + s * 0.05 * d, values, indices, rest).item() for s in (1, -1))
            assert abs((up - down) / 0.1 - (xd.grad * d).sum().item()) <= 1e-5 + 0.05 ** 2 / 6


def test_large_offsets():
    """Rows that lie past 2^31 elements from the first."""
    from ddfnet_b200 import distill_loss_grad, top_logits
    rows, classes = 3, 1 << 30
    x = torch.empty(0, dtype=torch.float16, device="cuda")
    x.resize_(((rows - 1) * classes + 1000,))
    y = x.as_strided((rows, 1000), (classes, 1))
    small = logits_of(rows, 1000, torch.float16, 3)
    y.copy_(small)
    top = top_logits(y, 9)
    order, rest = top64(small, 9, 1.0)
    assert torch.equal(top.indices.cpu(), order)
    loss, grad = distill_loss_grad(y, *top)
    want, g64, _ = distill64(small, small.gather(1, order), order, rest.float(), 1.0)
    check_loss(loss, want.sum() / rows, 1.0)
    check_grad(grad, g64 / rows, 1.0, 1.0, torch.float16)


def test_results_repeat_and_empty_batches():
    from ddfnet_b200 import distill_loss, distill_loss_grad
    x = logits_of(500, 3000, torch.float32, 1).cuda().requires_grad_()
    values, indices, rest = to_cuda(*targets(x.detach().cpu(), 30, 1.0, True, 2))
    runs = []
    for _ in range(2):
        loss = distill_loss(x, values, indices, rest)
        runs.append((loss, torch.autograd.grad(loss, x)[0], *distill_loss_grad(x, values, indices, rest)))
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    none = distill_loss(x[:0], values[:0], indices[:0], rest[:0])
    none.backward()
    assert none.item() == 0
    assert distill_loss_grad(x[:0], values[:0], indices[:0], rest[:0], reduction="none")[0].shape == (0,)


def test_refusals():
    from ddfnet_b200 import distill_loss, distill_loss_grad, top_logits
    x = torch.randn(3, 50, device="cuda")
    v, i, r = top_logits(x, 4)
    for bad in (lambda: top_logits(x.cpu(), 4), lambda: top_logits(x, 0), lambda: top_logits(x, 51),
                lambda: top_logits(x, 4, temperature=0.0), lambda: top_logits(torch.randn(2, 999, device="cuda"), 257)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        top_logits(x.double(), 4)
    for call in (distill_loss, distill_loss_grad):
        for args, error in (((x, v, i[:, :3], r), ValueError), ((x, v[:2], i[:2], r), ValueError),
                            ((x, v, i, r[:2]), ValueError), ((x, v.cpu(), i, r), ValueError),
                            ((x, v.requires_grad_(), i, r), ValueError), ((x, v.detach(), i.float(), r), TypeError),
                            ((x.double(), v.detach(), i, r), TypeError), ((x.cpu(), v.detach(), i, r), ValueError)):
            with pytest.raises(error):
                call(*args)
        v = v.detach()
        with pytest.raises(ValueError):
            call(x, v, i, r, temperature=-1.0)
        with pytest.raises(ValueError):
            call(x, v, i, r, reduction="batchmean")
