"""Classes switched off by large finite logits, and rows whose values lie far from zero: class_log_probs and
MaskedDistillationLoss against their definitions in 64 bits, in every form of the kernels.

Tolerances as in test_gpu_class_distributions, with the term's roundings counted one by one: log2(e) / T is off by U / 4 and U, the
multiply-add, the difference and the product with ln 2 by U each, ln 2 itself by less than U / 4, so 5 U of |log p|; log2 s of a row whose reference
exponent is off by up to 1/2 adds 2 U.  The definitions below subtract the maximum first, of all classes and of those that a
teacher does not keep: in 64 bits too, -1e30 would swallow the logarithm of the sum beside it.  The exponential instruction gives 0 for
results below 2^-126: a probability there is off by itself, by less than FLUSHED, and its gradient by that times what stands beside it."""
import math

import pytest
import torch

from tests.test_gpu_class_distributions import CHAIN, DTYPES, NINF, U, classes, close, half_step, loss_module, scores, teacher_top
from tests.test_gpu_class_distributions import M  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu

FILLS = [-1e5, -1e7, -1.2e7, -1e9, -1e10, -1e15, -1e30, -1e37]
FLUSHED = 2.0 ** -125
ids = dict(ids=lambda v: f"{v:g}" if isinstance(v, float) else str(v))


def centred(x):
    """x - max over dimension 1; -inf where there is nothing."""
    top = x.amax(1, keepdim=True)
    return x - torch.where(top == NINF, 0.0, top)


def check_scores(M, z, target, k, temperature):
    leaf = z.detach().clone().requires_grad_(True)
    out = M.class_log_probs(leaf, target, top_k=k, temperature=temperature)
    x, t = z.detach().double().cpu(), target.cpu()
    c = x.shape[1]
    d = centred(x) / temperature
    s = d.exp().sum(1, keepdim=True)
    logp = d - s.log()
    p = logp.exp()
    finite = torch.where(p > 0, logp, 0.0)
    h = -(p * finite).sum(1)
    tol = lambda v: 5 * U * v.abs() + 6 * U * (math.log(c) + 1) + CHAIN  # noqa: E731
    lp = logp.gather(1, t.unsqueeze(1)).squeeze(1)
    close(out.log_prob, lp, tol(lp), "log_prob")
    close(out.entropy, h, 2 * tol(h + math.log(c)), "entropy")
    if k:
        order = torch.sort(x.movedim(1, -1), dim=-1, descending=True, stable=True).indices[..., :k].movedim(-1, 1)
        assert torch.equal(out.top_class.cpu(), order)
        want = logp.gather(1, order)
        close(out.top_log_prob, want, tol(want), "top_log_prob")
    g = torch.Generator().manual_seed(5)
    gl, gh = (torch.randn(target.shape, generator=g) for _ in range(2))
    (got,) = torch.autograd.grad(out[:2], leaf, (gl.cuda(), gh.cuda()))
    gl, gh = gl.double().unsqueeze(1), gh.double().unsqueeze(1)
    hot = torch.zeros_like(p).scatter_(1, t.unsqueeze(1), 1.0)
    lph = finite + h.unsqueeze(1)
    want = (gl * (hot - p) - gh * p * lph) / temperature
    size = (gl.abs() * hot + p * (gl.abs() + gh.abs() * (lph.abs() + 1 + math.log(c)))) / temperature
    flushed = FLUSHED * (gl.abs() + gh.abs() * (lph.abs() + 1)) / temperature
    close(got, want, half_step(z.dtype, want) + size * (2 * CHAIN + 20 * U * (1 + math.log(c))) + flushed, "grad")


def distil(z, cls, val, temperature, log_probs):
    """(weighted losses of the positions, their sizes, gradient, its size) of the mean over all positions."""
    x, cls, val = z.detach().double().cpu(), cls.cpu().long(), val.double().cpu()
    b, c = x.shape[:2]
    ok = (cls >= 0) & (cls < c)
    v = torch.where(ok, val, NINF)
    if log_probs:
        lq = v
    else:
        e = centred(v) / temperature
        lq = torch.where(v == NINF, NINF, e - e.exp().sum(1, keepdim=True).log())
    q = lq.exp()
    d = centred(x) / temperature
    logp = d - d.exp().sum(1, keepdim=True).log()
    p = logp.exp()
    at = torch.where(ok, cls, 0)
    mine = logp.gather(1, at)
    rows = torch.where(q > 0, q * (lq - mine), 0.0).sum(1)
    sizes = torch.where(q > 0, q * (lq.abs() + mine.abs() + 1 + math.log(c)), 0.0).sum(1) + 1
    hot = torch.zeros_like(x).scatter_add_(1, at, q)
    mass = q.sum(1, keepdim=True)
    grad, gsize = p * mass - hot, p * mass + hot
    if log_probs:
        kept = torch.zeros(b, c + 1, *x.shape[2:], dtype=torch.bool).scatter_(1, torch.where(ok, cls, c), True)[:, :c]
        other = torch.where(kept, NINF, x)
        some = (other > NINF).any(1, keepdim=True)
        top = torch.where(some, other.amax(1, keepdim=True), 0.0)
        o = (other - top) / temperature
        share = torch.where(some, o.exp() / o.exp().sum(1, keepdim=True), 0.0)
        left = torch.where(some, (top - x.amax(1, keepdim=True)) / temperature + o.exp().sum(1, keepdim=True).log() - d.exp().sum(1, keepdim=True).log(), 0.0)
        r = torch.where(some, (1 - mass).clamp(min=0), 0.0)
        rows = rows + torch.xlogy(r, r).squeeze(1) - (r * left).squeeze(1)
        sizes = sizes + (r * (left.abs() + 1)).squeeze(1)
        grad = grad + p * r - r * share
        gsize = gsize + p * r + r * share
    n = x.numel() // c
    return rows * temperature ** 2 / n, sizes * temperature ** 2 / n, grad * temperature / n, gsize * temperature / n


def check_loss(M, z, cls, val, temperature, log_probs):
    leaf = z.detach().clone().requires_grad_(True)
    loss = loss_module(M, 1, temperature, log_probs)(leaf, (cls, val))
    (grad,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    (scaled,) = torch.autograd.grad(loss, leaf, torch.tensor(-3.0, device="cuda"))
    rows, sizes, want, gsize = distil(z, cls, val, temperature, log_probs)
    c = z.shape[1]
    rel = 2 * CHAIN + 20 * U * (1 + math.log(c)) + (cls.shape[1] + 16) * U
    close(loss, rows.sum(), sizes.sum() * rel, "loss")
    flushed = 2 * FLUSHED * temperature * c / z.numel()  # (of p (Q + r) and of the rest's share)
    close(grad, want, half_step(z.dtype, want) + gsize * (rel + 8 * U * 30) + flushed, "grad")
    close(scaled, -3 * want, half_step(z.dtype, 3 * want) + 3 * gsize * (rel + 8 * U * 30) + 3 * flushed, "grad, upstream -3")


def filled(shape, dtype, fill, seed):
    """Seven samples: where the fill leaves every other class, one, none, the last three, the first half; ordinary logits beside one
    peak as far above as the fill is below; two fills."""
    z = scores(shape, dtype, seed)
    c = shape[1]
    z[0, 1::2] = fill
    z[1] = fill; z[1, c - 2] = -4.0
    z[2] = fill
    z[3, : c - 3] = fill
    z[4, c // 2:] = fill
    z[5, c // 3] = -fill
    z[6] = fill; z[6, ::3] = 2 * fill
    return z


# one wave, a workgroup, split over workgroups, several tiles a workgroup; maps in registers, in the LDS, in a few slices and in many
SCORE_SHAPES = [(7, 70), (7, 700), (7, 3000), (7, 40007), (7, 300011), (7, 70, 3, 5), (7, 150, 3, 5), (7, 1700, 3, 5), (7, 9000, 3, 5)]
# held by one wave and by a workgroup, slices, several tiles a slice; maps in the LDS and in slices
LOSS_SHAPES = [(7, 700), (7, 3001), (7, 40007), (7, 600011), (7, 70, 3, 5), (7, 1300, 3, 5)]


@pytest.mark.parametrize("fill", FILLS, **ids)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SCORE_SHAPES, ids=str)
def test_log_probs_beside_finite_fills(M, shape, dtype, fill):
    z = filled(shape, dtype, fill, seed=shape[1])
    target = classes(shape[:1] + shape[2:], shape[1], seed=4)
    target[1] = shape[1] - 2
    for k, temperature in ((8, 1.0), (0, 0.7), (64, 0.5), (3, 2.0)):
        if k < 64 or shape[1] < 100000:
            check_scores(M, z, target, k, temperature)


@pytest.mark.parametrize("fill", FILLS, **ids)
@pytest.mark.parametrize("log_probs", [False, True], ids=["logits", "log_probs"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", LOSS_SHAPES, ids=str)
def test_distillation_beside_finite_fills(M, shape, dtype, log_probs, fill):
    z = filled(shape, dtype, fill, seed=shape[1] + 1)
    for temperature in (1.0, 0.5, 2.0):
        cls, val = teacher_top(shape, 9, 5, log_probs, temperature)
        cls[3, 4:] = -1
        check_loss(M, z, cls, val, temperature, log_probs)
        only = torch.full_like(z, fill).scatter(1, cls.clamp(min=0), scores(shape, dtype, 6))  # none but kept classes left
        check_loss(M, only, cls, val, temperature, log_probs)
        if shape[1] < 100000:
            for i in range(7):
                check_loss(M, z[i:i + 1], cls[i:i + 1], val[i:i + 1], temperature, log_probs)


# walked rows, a register kernel's maps: many rows or tiles of a few kinds
@pytest.mark.parametrize("fill", [-1e7, -1e9, -1e10, -1e30], **ids)
@pytest.mark.parametrize("log_probs", [False, True], ids=["logits", "log_probs"])
@pytest.mark.parametrize("rows,c,dtype", [(2100, 2049, "bf16"), (2100, 9000, "bf16"), (2100, 3001, "f32"), (300, 33000, "bf16"), (300, 33000, "f32"),
                                          (300, 9000, "f32"), (300, 20000, "bf16")], **ids)
def test_distillation_of_many_rows_beside_finite_fills(M, rows, c, dtype, log_probs, fill):
    base = filled((8, c), dtype, fill, seed=c)
    cls, val = teacher_top((8, c), 9, 5, log_probs, 1.5)
    base[7] = fill
    base[7, cls[7]] = 1.0
    which = (torch.arange(rows) % 8).cuda()
    leaf = base[which].requires_grad_(True)
    loss = loss_module(M, 1, 1.5, log_probs)(leaf, (cls[which], val[which]))
    (grad,) = torch.autograd.grad(loss, leaf)
    each, sizes, want, gsize = distil(base, cls, val, 1.5, log_probs)
    times = torch.bincount(which.cpu(), minlength=8).double()
    rel = 2 * CHAIN + 20 * U * (1 + math.log(c)) + 25 * U
    close(loss, (each * times).sum() * 8 / rows, (sizes * times).sum() * 8 / rows * (rel + 2 * 16 * U), "loss")
    want, gsize = want * 8 / rows, gsize * 8 / rows
    first = grad[:8]
    close(first, want, half_step(base.dtype, want) + gsize * (rel + 8 * U * 30), "grad")
    assert torch.equal(grad, first[which]), "one row, two gradients"


@pytest.mark.parametrize("fill", [-1e7, -1e9, -1e10, -1e30], **ids)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("c", [31, 60, 100, 133])
def test_maps_in_registers_beside_finite_fills(M, c, dtype, fill):
    z = scores((530, c, 4, 6), dtype, seed=c)
    z[:7] = filled((7, c, 4, 6), dtype, fill, seed=c + 1)
    check_scores(M, z, classes((530, 4, 6), c, 4), 8, 0.7)
    for log_probs in (False, True):
        cls, val = teacher_top(tuple(z.shape), 9, 5, log_probs, 1.5)
        z[7] = fill
        z[7].scatter_(0, cls[7], scores((9, 4, 6), dtype, 6))
        z[8, :, 1] = fill                       # (beside ordinary positions of the same wave)
        z[9, :, 2, 3:] = fill
        check_loss(M, z, cls, val, 1.5, log_probs)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(7, 700), (7, 3000), (7, 40007), (7, 70, 3, 5), (7, 150, 3, 5), (7, 1700, 3, 5)], ids=str)
def test_temperatures_far_from_one(M, shape, dtype):
    """Low ones leave every row beyond the reference exponents' range, high ones make it uniform."""
    z = scores(shape, dtype, seed=shape[1])
    target = classes(shape[:1] + shape[2:], shape[1], seed=4)
    for temperature in (1e-36, 1e-20, 1e-6, 1e-3, 1e6, 1e30):
        check_scores(M, z, target, 5, temperature)
    for temperature in (1e-15, 1e-3, 1e6):
        for log_probs in (False, True):
            check_loss(M, z, *teacher_top(shape, 6, 5, log_probs, temperature), temperature, log_probs)


@pytest.mark.parametrize("shape", [(7, 700), (7, 40007), (7, 70, 3, 5), (7, 1700, 3, 5)], ids=str)
def test_large_gradients_of_the_entropy(M, shape):
    """Classes without any probability have no gradient, however large the one that arrives: 1e36 times a bounded logarithm (128 ln 2)
    is below 3.4e38."""
    z = filled(shape, "f32", -1e30, 3)
    leaf = z.clone().requires_grad_(True)
    out = M.class_log_probs(leaf, torch.zeros_like(z[:, 0], dtype=torch.long))
    (got,) = torch.autograd.grad(out.entropy, leaf, torch.full_like(out.entropy, 1e36))
    (unit,) = torch.autograd.grad(M.class_log_probs(leaf, torch.zeros_like(z[:, 0], dtype=torch.long)).entropy, leaf, torch.ones_like(out.entropy))
    assert torch.isfinite(got).all() and (got[z == -1e30][unit[z == -1e30] == 0] == 0).all()
    want = unit.double().cpu() * 1e36
    close(got, want, want.abs() * 64 * U + 1e36 * (2 * CHAIN + 20 * U * (1 + math.log(shape[1]))) * torch.softmax(z.double().cpu(), 1) * (2 + 2 * math.log(shape[1])), "grad")


@pytest.mark.parametrize("shape", [(3, 300, 8, 12), (40, 20000), (530, 60, 4, 6), (2, 1111, 8, 12)], ids=str)
def test_fills_in_captured_graphs(M, shape):
    """Rows beyond the reference exponents in one replay and not in the next: what a call finds out about its rows stays in that call
    (forms with more than 64 KiB of LDS, in registers and in slices among them)."""
    z = scores(shape, "f32", 1).requires_grad_(True)
    target = classes(shape[:1] + shape[2:], shape[1], 3)
    cls, val = teacher_top(shape, 9, 5, True, 1.0)
    fn = loss_module(M, 1, 1.0, True)

    def step():
        loss = fn(z, (cls, val)) * 0.5
        out = M.class_log_probs(z, target, top_k=20)
        (grad,) = torch.autograd.grad(loss + out.entropy.mean(), z)
        return [loss.detach(), out.log_prob.detach(), out.top_class, grad]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        new = scores(shape, "f32", 20 + i)
        if i % 2 == 0:
            new[0] = -1e9
            new[1:] = torch.full_like(new[1:], -1e30).scatter(1, cls[1:], new[1:].gather(1, cls[1:]))
        with torch.no_grad():
            z.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, step())), i
        assert all(torch.isfinite(t).all() for t in got), i
