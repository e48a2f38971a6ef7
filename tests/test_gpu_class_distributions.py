"""Log probabilities with entropy and alternatives (class_log_probs) and distillation from a teacher's top classes
(MaskedDistillationLoss) against plain 64-bit implementations of their definitions.

Tolerances are counted, not tried.  U = 2^-24 is half a step of fp32.  A log probability is (z - m) c - log2 s, times ln 2: three
roundings of a term up to |log p| + log C, and a sum of C terms whose longest chain of additions is taken as 512 links, so its
relative error is below (512 + 16) U (16: the exponentials' own error and the joins).  A gradient adds half a step of the
logits' type (relative) to the same relative errors of its terms."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
CHAIN = 528 * U
NINF = float("-inf")
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half_step(dtype, ref):
    """Half a step of `dtype` at `ref`: relative, and absolute below the smallest normal number."""
    fi = torch.finfo(dtype)
    return torch.clamp(fi.eps / 2 * ref.abs(), min=fi.tiny * fi.eps / 2)


@pytest.fixture(scope="module")
def M():
    assert torch.cuda.is_available(), "GPU tests need a GPU"
    import multimae_amd
    from multimae_amd import ops
    ops._L()
    return multimae_amd


def scores(shape, dtype, seed, scale=3.0, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(DTYPES[dtype]).to(device)


def classes(shape, c, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, c, shape, generator=g).cuda()


# ------------------------------------------------------------------------------------------------ definitions in 64 bits
def log_softmax64(x):
    """log softmax over dimension 1 as differences from the maximum (which would swallow log C at the type's lowest value); all
    -inf where every logit is."""
    top = x.amax(1, keepdim=True)
    d = x - torch.where(top == NINF, 0.0, top)
    s = d.exp().sum(1, keepdim=True)
    return torch.where(s == 0, NINF, d - s.log())


def reference(z, target, k, temperature):
    """(log p, log p of the target, entropy, top log p, top classes) of z [B, C, ...] in float64 on the CPU."""
    z = z.detach().double().cpu()
    target = target.cpu()
    logp = log_softmax64(z / temperature)
    ok = (target >= 0) & (target < z.shape[1])
    lp = torch.where(ok, logp.gather(1, torch.where(ok, target, 0).unsqueeze(1)).squeeze(1), 0.0)
    p = logp.exp()
    h = -torch.where(p > 0, p * logp, torch.where(p.isnan(), math.nan, 0.0)).sum(1)
    rows = torch.where(z.isnan(), math.inf, z).movedim(1, -1)
    nan = z.isnan().movedim(1, -1)
    order = torch.sort(rows, dim=-1, descending=True, stable=True).indices
    if nan.any():  # NaN first, then +inf
        order = order.gather(-1, torch.sort(nan.gather(-1, order).int(), dim=-1, descending=True, stable=True).indices)
    top = order[..., :k].movedim(-1, 1)
    return logp, lp, h, logp.gather(1, top), top


def reference_grad(z, target, temperature, gl, gh):
    logp, _, h, _, _ = reference(z, target, 0, temperature)
    gl, gh, target = gl.double().cpu().unsqueeze(1), gh.double().cpu().unsqueeze(1), target.cpu().unsqueeze(1)
    c = z.shape[1]
    p = logp.exp()
    ok = (target >= 0) & (target < c)
    gl = torch.where(ok, gl, 0.0)
    hot = torch.zeros_like(p).scatter_(1, torch.where(ok, target, 0), ok.double())
    lph = torch.where(p > 0, logp, 0.0) + h.unsqueeze(1)
    grad = (gl * (hot - p) - gh * p * lph) / temperature
    # every term with the relative error of its probability (an exponential of a log probability: its absolute error)
    size = (gl.abs() * hot + p * (gl.abs() + gh.abs() * (lph.abs() + 1 + math.log(c)))) / temperature
    return grad, size


def close(got, want, tol, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(got.isnan(), want.isnan()), (what, "NaN")
    ends = want.isinf()
    assert torch.equal(got[ends], want[ends]) and not got[~ends].isinf().any(), (what, "inf")
    ok = ~(want.isnan() | ends)
    bad = ((got - want).abs() - tol.expand_as(want))[ok]
    assert not (bad > 0).any(), (what, "off by", bad.max().item(), "more than the tolerance; error", (got - want)[ok].abs().max().item())


def check_log_probs(M, z, target, k, temperature, backward=True):
    z = z.detach()
    leaf = z.requires_grad_(backward)
    out = M.class_log_probs(leaf, target, top_k=k, temperature=temperature)
    logp, lp, h, top_lp, top = reference(z, target, k, temperature)
    c = z.shape[1]
    tol = lambda v: 4 * U * (v.abs().nan_to_num(0, 0, 0) + math.log(c) + 1) + CHAIN  # noqa: E731
    close(out.log_prob, lp, tol(lp), "log_prob")
    # H = log2 s - t / s: the same errors, on terms of size H + log C
    close(out.entropy, h, 2 * tol(h + math.log(c)), "entropy")
    if k:
        assert torch.equal(out.top_class.cpu(), top), "top_class"
        close(out.top_log_prob, top_lp, tol(top_lp), "top_log_prob")
    else:
        assert out.top_class is None and out.top_log_prob is None
    if not backward:
        return out
    g = torch.Generator().manual_seed(5)
    gl, gh = (torch.randn(target.shape, generator=g).cuda() for _ in range(2))
    for pair in ((gl, gh), (gl, None), (None, gh)):
        outs = [t for t, d in zip(out[:2], pair) if d is not None]
        (got,) = torch.autograd.grad(outs, leaf, [d for d in pair if d is not None], retain_graph=True)
        zero = torch.zeros_like(gl)
        want, size = reference_grad(z, target, temperature, *(zero if d is None else d for d in pair))
        assert got.dtype == z.dtype
        want = torch.where(torch.isinf(logp.amax(1, keepdim=True)) & ~z.isnan().any(1, keepdim=True).cpu(), 0.0, want)
        err = half_step(z.dtype, want) + size.nan_to_num(0) * (2 * CHAIN + 16 * U * (1 + math.log(c)))
        close(got, want, err, f"grad {[d is not None for d in pair]}")
    return out


# ------------------------------------------------------------------------------------------------ log probabilities
ROWS = [(1, 1), (1, 2), (3, 5), (64, 63), (65, 64), (130, 133), (7, 511), (5, 512), (6, 513), (4, 1000), (3, 2049), (2, 8191), (2, 8192),
        (3, 8200), (1, 16387), (2, 50001), (1, 131072), (3, 150016), (1, 262147)]
MAPS = [(2, 133, 56, 56), (1, 5, 4, 4), (3, 7, 1, 1), (2, 150, 5, 7), (1, 1000, 3, 5), (2, 40, 11), (1, 2, 1, 130), (1, 6007, 2, 3), (4, 257, 9),
        (1, 1, 8, 8), (2, 700, 1, 65), (2, 640, 6, 7), (1, 641, 70), (1, 321, 70), (1, 32000, 66), (1, 5001, 1, 3)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", ROWS + MAPS, ids=str)
def test_log_probs_of_rows_and_maps(M, shape, dtype):
    z = scores(shape, dtype, seed=sum(shape))
    target = classes(shape[:1] + shape[2:], shape[1], seed=1)
    for k, temperature in ((min(8, shape[1]), 1.0), (0, 0.7), (min(64, shape[1]), 2.5)):
        check_log_probs(M, z, target, k, temperature, backward=k != 0)


@pytest.mark.parametrize("shape", [(6, 70), (6, 700), (6, 9000), (6, 40007), (6, 70, 3, 5), (6, 1700, 3, 5)], ids=str)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_log_probs_of_masked_rows(M, shape, dtype):
    """-inf and the type's lowest value in masked places, rows with one class or none left, NaN and +inf."""
    z = scores(shape, dtype, seed=3)
    low = torch.finfo(z.dtype).min
    c = shape[1]
    z[0, 1::2] = NINF                      # every other class
    z[1] = NINF; z[1, c - 2] = -4.0        # one left
    z[2] = NINF                            # none left
    z[3] = low                             # all at the lowest value: uniform
    z[4, : c - 3] = low                    # three above it
    z[5, c // 2:] = NINF                   # the upper half
    target = classes(shape[:1] + shape[2:], c, seed=4)
    target[0] = 0; target[1] = c - 2; target[4] = c - 1
    for k in (3, min(64, c)):
        out = check_log_probs(M, z, target, k, 1.0)
        check_log_probs(M, z, target, k, 3.0, backward=False)
    assert (out.entropy[2] == 0).all() and (out.log_prob[2] == NINF).all()
    close(out.entropy[3], torch.full(out.entropy[3].shape, math.log(c), dtype=torch.float64), torch.tensor(2 * CHAIN), "uniform")
    z[0, 3] = float("nan"); z[0, 4] = float("inf"); z[5, 0] = float("inf")
    out = M.class_log_probs(z, target, top_k=5)
    assert out.entropy[0].isnan().all() and out.log_prob[0].isnan().all() and out.entropy[5].isnan().all()
    assert torch.equal(out.top_class.cpu(), reference(z, target, 5, 1.0)[4])
    assert not out.entropy[1:5].isnan().any()


@pytest.mark.parametrize("shape", [(3, 70), (3, 700), (3, 9000), (2, 40007), (3, 140, 3, 5), (3, 1400, 3, 5)], ids=str)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_equal_logits_rank_by_the_lower_class(M, shape, dtype):
    few = classes(shape, 4, seed=8).to(DTYPES[dtype]) - 1.0        # four levels, one of them zero
    signed = torch.where(few == 0, few * classes(shape, 3, seed=9).sub(1).to(few.dtype), few)  # both zeros
    constant = torch.full_like(few, 2.5)
    ramp = torch.arange(shape[1], device="cuda").to(few.dtype).view((1, -1) + (1,) * (len(shape) - 2)).expand(shape).contiguous() / 64
    stripes = torch.where(torch.arange(shape[1], device="cuda") % 2048 < 8, 5.0, -1.0).to(few.dtype).view(ramp[:1].shape[0:1] + (-1,) + (1,) * (len(shape) - 2)).expand(shape).contiguous()
    stripes = stripes + few * 0.25
    target = classes(shape[:1] + shape[2:], shape[1], seed=2)
    for z in (few, signed, constant, ramp, -ramp, stripes):
        for k in (1, 7, 64):
            check_log_probs(M, z, target, k, 1.0, backward=False)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("c", [5, 100, 1000, 2049, 4095, 8191])
def test_log_probs_of_many_rows(M, c, dtype):
    """A wave a row; lists of any length from a tile that fills few lanes, levels with many equal values, mostly -inf."""
    z = scores((2051, c), dtype, seed=c)
    z[3] = torch.randint(0, 3, (c,), generator=torch.Generator().manual_seed(1)).to(z.dtype)
    z[4] = -z[3]
    z[5, 3:] = NINF
    z[6] = NINF
    z[7] = torch.finfo(z.dtype).min
    z[8, : c // 2] = torch.finfo(z.dtype).min
    z[9] = 0.0; z[9, 1::3] = -0.0
    target = classes((2051,), c, 1)
    for k in (0, 5, 16, 33, 64):
        check_log_probs(M, z, target, min(k, c), 1.5, backward=k in (0, 33))


def test_targets_outside_the_classes_are_ignored(M):
    for shape in ((6, 50), (6, 5000), (6, 50, 2, 3)):
        z = scores(shape, "f32", seed=1)
        target = classes(shape[:1] + shape[2:], shape[1], seed=2)
        target[0], target[1], target[2], target[3] = -100, shape[1], -1, 2 ** 40
        out = check_log_probs(M, z, target, 2, 1.0)
        assert (out.log_prob[:4] == 0).all() and (out.entropy > 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_log_probs_of_strided_logits(M, dtype):
    wide = scores((9, 1300), dtype, seed=1)
    target = classes((9,), 1001, seed=2)
    check_log_probs(M, wide[:, 3:1004], target, 5, 1.0)                     # rows further apart, odd offsets
    check_log_probs(M, wide[::2, :70], classes((5,), 70, 3), 5, 1.0)
    check_log_probs(M, wide.t()[:77].t(), classes((9,), 77, 3), 5, 1.0)     # (the same rows, cut)
    check_log_probs(M, wide.t(), classes((1300,), 9, 3), 5, 1.0)            # classes far apart: copied
    check_log_probs(M, wide[:1].expand(4, 1300), classes((4,), 1300, 3), 5, 1.0)
    large = scores((4, 1001, 3, 5), dtype, seed=4)
    check_log_probs(M, large[::2], classes((2, 3, 5), 1001, 5), 5, 1.0)
    check_log_probs(M, large[:, 3:], classes((4, 3, 5), 998, 5), 5, 1.0)
    maps = scores((4, 20, 6, 9), dtype, seed=4)
    t = classes((4, 6, 9), 20, 5)
    check_log_probs(M, maps.contiguous(memory_format=torch.channels_last), t, 5, 1.0)
    check_log_probs(M, maps[::2], t[::2], 5, 1.0)                           # samples further apart
    check_log_probs(M, maps[:, 3:15], classes((4, 6, 9), 12, 6), 5, 1.0)
    check_log_probs(M, maps[..., 1:7], t[..., 1:7], 5, 1.0)
    flat = scores((4 * 333 + 1,), dtype, seed=6)
    check_log_probs(M, flat[1:].view(4, 333), classes((4,), 333, 7), 5, 1.0)  # odd storage offset


def test_log_probs_of_nothing_and_refusals(M):
    from multimae_amd._lib import MmaeError
    out = M.class_log_probs(torch.empty(0, 9, device="cuda"), torch.empty(0, dtype=torch.long, device="cuda"), top_k=3)
    assert out.log_prob.shape == (0,) and out.top_class.shape == (0, 3)
    out = M.class_log_probs(torch.empty(2, 9, 0, 4, device="cuda", requires_grad=True), torch.empty(2, 0, 4, dtype=torch.long, device="cuda"))
    out.entropy.sum().backward()
    z, t = torch.randn(4, 9, device="cuda"), torch.zeros(4, dtype=torch.long, device="cuda")
    for bad in (lambda: M.class_log_probs(z, t, top_k=10), lambda: M.class_log_probs(z, t, top_k=-1), lambda: M.class_log_probs(z, t[:3]),
                lambda: M.class_log_probs(z.double(), t), lambda: M.class_log_probs(z, t.cpu()), lambda: M.class_log_probs(z.cpu(), t.cpu()),
                lambda: M.class_log_probs(z, t, temperature=0.0), lambda: M.class_log_probs(z, t, temperature=float("nan")),
                lambda: M.class_log_probs(z, t, temperature=float("inf")), lambda: M.class_log_probs(z[0], t[0]),
                lambda: M.class_log_probs(z[:, :0], t), lambda: M.class_log_probs(torch.randn(2, 99, device="cuda"), t[:2], top_k=65)):
        with pytest.raises(MmaeError):
            bad()


def test_log_prob_gradient_against_differences(M):
    """Central differences of f = sum(a log_prob + b entropy) along random directions, in fp32 calls: the truncation is below
    h^2 / 6 |f'''| (f''' < 40 |direction|_inf^3 sum |a| + |b| (1 + log C) here), the rounding 2 tol(f) / (2 h)."""
    for shape in ((3, 40), (2, 3000), (2, 30, 2, 2)):
        z = scores(shape, "f32", seed=1, scale=1.0)
        target = classes(shape[:1] + shape[2:], shape[1], seed=2)
        a, b = torch.randn(2, *target.shape, generator=torch.Generator().manual_seed(3)).cuda()
        leaf = z.clone().requires_grad_(True)
        out = M.class_log_probs(leaf, target)
        (grad,) = torch.autograd.grad((out.log_prob, out.entropy), leaf, (a, b))

        def f(x):
            o = M.class_log_probs(x, target)
            return (a.double() * o.log_prob.double() + b.double() * o.entropy.double()).sum()
        logc = math.log(shape[1])
        weight = (a.abs() + b.abs() * (1 + logc)).double().sum().item()
        tol_f = (4 * U * (8 + 3 * logc) + 2 * CHAIN) * weight
        for seed in range(3):
            d = torch.randn(shape, generator=torch.Generator().manual_seed(10 + seed)).cuda().clamp(-1, 1)
            h = 0.02
            slope = (f(z + h * d) - f(z - h * d)) / (2 * h)
            assert abs(slope.item() - (grad.double() * d.double()).sum().item()) < tol_f / h + 40 * weight * h * h / 6


def test_log_probs_beyond_32_bit_offsets(M):
    """More than 2^31 logits in one call: the last rows, forward and backward, are those of the rows alone."""
    n, c = 16500, 131072
    z = torch.zeros(n, c, dtype=torch.bfloat16, device="cuda")
    last = scores((3, c), "bf16", seed=1)
    z[-3:] = last
    target = torch.full((n,), c - 1, device="cuda")
    leaf = z.requires_grad_(True)
    out = M.class_log_probs(leaf, target, top_k=4)
    (grad,) = torch.autograd.grad((out.log_prob, out.entropy), leaf, (torch.ones(n, device="cuda"),) * 2)
    few = last.clone().requires_grad_(True)
    want = M.class_log_probs(few, target[-3:], top_k=4)
    (want_grad,) = torch.autograd.grad((want.log_prob, want.entropy), few, (torch.ones(3, device="cuda"),) * 2)
    assert torch.equal(out.top_class[-3:], want.top_class) and torch.equal(out.top_class[:-3, 0], torch.zeros_like(target[:-3]))
    close(out.log_prob[-3:], want.log_prob.double().cpu(), torch.tensor(2 * CHAIN), "log_prob")
    close(grad[-3:], want_grad.double().cpu(), 2 * half_step(torch.bfloat16, want_grad.double().cpu()), "grad")
    assert torch.isfinite(out.entropy).all() and (out.entropy[:-3] - math.log(c)).abs().max().item() < 2 * CHAIN + 4 * U * 3 * math.log(c)


# ------------------------------------------------------------------------------------------------ distillation
def reference_distill(z, cls, val, mask, patch, temperature, log_probs):
    """(loss, sum of |terms| of the loss, gradient, sum of |terms| of the gradient) in float64 on the CPU."""
    z, cls, val = z.detach().double().cpu(), cls.cpu().long(), val.double().cpu()
    b, c = z.shape[:2]
    space = z.shape[2:]
    logp = log_softmax64(z / temperature)
    empty = (z == NINF).all(1, keepdim=True)
    ok = (cls >= 0) & (cls < c)
    at = torch.where(ok, cls, 0)
    v = torch.where(ok, val, NINF)
    if log_probs:
        lq = v
    else:
        some = torch.logsumexp(v / temperature, 1, keepdim=True)
        lq = torch.where(some == NINF, NINF, v / temperature - some)
    q = lq.exp()
    terms = torch.where(q > 0, q * (lq - logp.gather(1, at)), 0.0)
    hot = torch.zeros_like(z).scatter_add_(1, at, q)
    p = logp.exp()
    mass = q.sum(1, keepdim=True)
    grad_p, rest_term, size = p * mass, torch.zeros_like(mass), torch.zeros_like(z)
    if log_probs:
        kept = torch.zeros(b, c + 1, *space, dtype=torch.bool).scatter_(1, torch.where(ok, cls, c), True)[:, :c]
        left = torch.logsumexp(torch.where(kept, NINF, logp), 1, keepdim=True)
        r = (1 - mass).clamp(min=0)
        r = torch.where(left == NINF, 0.0, r)
        rest_term = torch.where(r > 0, r * (r.clamp(min=1e-300).log() - torch.where(r > 0, left, 0.0)), 0.0)
        share = torch.where(kept | (r == 0), 0.0, (logp - torch.where(left == NINF, 0.0, left)).exp())
        grad_p = p * (mass + r) - r * share
        size = r * share
    if mask is None:
        w = torch.full((b,) + space, 1.0 / (z.numel() / c), dtype=torch.float64)
    else:
        m = (mask.cpu() != 0).double()
        m = m.view(b, space[0] // patch, space[1] // patch).repeat_interleave(patch, 1).repeat_interleave(patch, 2) if patch > 1 else m.view((b,) + space)
        count = m.reshape(b, -1).sum(1)
        w = m * (torch.where(count > 0, 1 / count.clamp(min=1), 0.0) / (count > 0).sum().clamp(min=1)).view((b,) + (1,) * len(space))
    rows = terms.sum(1) + rest_term.squeeze(1)
    sizes = torch.where(q > 0, q * (lq.abs() + logp.gather(1, at).abs() + 1 + math.log(c)), 0.0).sum(1) + rest_term.abs().squeeze(1) + 1
    t2 = temperature * temperature
    loss = torch.where(w > 0, rows * w, 0.0).sum() * t2
    sw = (w * temperature).unsqueeze(1)
    grad = torch.where((sw > 0) & ~empty, (grad_p - hot) * sw, 0.0)
    gsize = (p * mass + hot + size) * sw
    return loss, (torch.where(w > 0, sizes.nan_to_num(0, 0, 0) * w, 0.0)).sum() * t2, grad, gsize.nan_to_num(0)


def loss_module(M, patch, temperature, log_probs):
    return M.MaskedDistillationLoss(patch_size=16, stride=16 // patch, temperature=temperature, teacher="log_probs" if log_probs else "logits")


def check_distill(M, z, cls, val, mask=None, patch=1, temperature=1.0, log_probs=False):
    leaf = z.detach().requires_grad_(True)
    loss = loss_module(M, patch, temperature, log_probs)(leaf, (cls, val), mask=mask)
    want, size, want_grad, grad_size = reference_distill(z, cls, val, mask, patch, temperature, log_probs)
    c = z.shape[1]
    rel = 2 * CHAIN + 16 * U * (1 + math.log(c)) + (cls.shape[1] + 16) * U
    close(loss, want, size * rel, "loss")
    (grad,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    assert grad.dtype == z.dtype
    # a gradient is a difference of probabilities, each with its relative error (the teacher's: |log q| of absolute error)
    tol = half_step(z.dtype, want_grad) + grad_size * (rel + 8 * U * 30)
    close(grad, want_grad, tol, "grad")
    # another upstream gradient, the second backward pass of the same graph
    (grad3,) = torch.autograd.grad(loss, leaf, torch.tensor(-3.0, device="cuda"))
    close(grad3, -3 * want_grad, half_step(z.dtype, 3 * want_grad) + 3 * grad_size * (rel + 8 * U * 30), "grad, upstream -3")
    return loss, grad


def teacher_top(shape, k, seed, log_probs, temperature, value_dtype="f32", class_dtype=torch.int64):
    t = scores(shape, "f32", seed)
    v, i = torch.topk(t, min(k, shape[1]), dim=1)
    if log_probs:
        v = v / temperature - torch.logsumexp(t / temperature, 1, keepdim=True)
    return i.to(class_dtype).contiguous(), v.to(DTYPES[value_dtype]).contiguous()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("log_probs", [False, True], ids=["logits", "log_probs"])
@pytest.mark.parametrize("shape", ROWS + MAPS, ids=str)
def test_distillation_of_rows_and_maps(M, shape, log_probs, dtype):
    z = scores(shape, dtype, seed=sum(shape) + 1)
    for n, (k, t) in enumerate(((8, 2.0), (64, 1.0), (1, 0.6))):
        cls, val = teacher_top(shape, k, 7 + n, log_probs, t, ("f32", "bf16", "f16")[n], (torch.int64, torch.int32)[n % 2])
        check_distill(M, z, cls, val, temperature=t, log_probs=log_probs)


@pytest.mark.parametrize("log_probs", [False, True], ids=["logits", "log_probs"])
@pytest.mark.parametrize("shape,patch", [((5, 133, 56, 56), 4), ((4, 12, 8, 4), 4), ((3, 150, 6, 10), 2), ((4, 9, 5, 3), 1), ((130, 40), 1),
                                         ((33, 3000), 1), ((9, 20000), 1), ((6, 21, 50), 1), ((4, 1500, 6, 10), 2), ((4, 900, 130), 1)], ids=str)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_distillation_with_a_mask(M, shape, patch, log_probs, dtype):
    z = scores(shape, dtype, seed=2)
    cls, val = teacher_top(shape, 6, 3, log_probs, 1.5)
    space = shape[2:]
    tokens = math.prod(space) // (patch * patch)
    mask = (classes((shape[0], tokens), 4, 5) > 0).long() * 2 - 0  # any nonzero value counts
    mask[1] = 0                                                   # a sample without a position in the loss
    z[2 if len(shape) > 2 else 1] = float("nan") if len(shape) == 2 else z[2]
    z[1] = float("nan")                                           # outside the loss: not looked at
    loss, grad = check_distill(M, z, cls, val, mask, patch, 1.5, log_probs)
    assert torch.isfinite(loss) and torch.isfinite(grad).all() and (grad[1] == 0).all()
    fn = loss_module(M, patch, 1.5, log_probs)
    assert torch.equal(fn(z, (cls, val), mask=mask != 0), loss.detach())
    zero, none = check_distill(M, z, cls, val, torch.zeros_like(mask), patch, 1.5, log_probs)
    assert zero.item() == 0 and (none == 0).all()


@pytest.mark.parametrize("log_probs", [False, True], ids=["logits", "log_probs"])
@pytest.mark.parametrize("shape", [(7, 70), (7, 3000), (7, 40007), (7, 70, 2, 3), (7, 1300, 2, 3)], ids=str)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_distillation_padding_duplicates_and_masked_classes(M, shape, log_probs, dtype):
    c = shape[1]
    z = scores(shape, dtype, seed=4)
    cls, val = teacher_top(shape, 9, 5, log_probs, 1.0)
    cls[0, 3:] = -1                                    # padding
    cls[1, ::2] = c + 5
    cls[2] = -100                                      # nothing kept
    cls[3, 4] = cls[3, 2]; cls[3, 8] = cls[3, 2]       # listed three times
    val[4, 5:] = NINF                                  # no mass there
    z[5, : c // 2] = NINF                              # classes switched off for the student, none of them kept
    cls[5] = torch.where(cls[5] < c // 2, cls[5] + (c + 1) // 2, cls[5]).clamp(max=c - 1)
    z[6] = torch.finfo(z.dtype).min                    # uniform at the lowest value
    loss, grad = check_distill(M, z, cls, val, log_probs=log_probs)
    assert torch.isfinite(loss)
    if not log_probs:
        assert (grad[2] == 0).all()
    z[0] = NINF                                        # no class left: an infinite divergence, no gradient
    loss, grad = check_distill(M, z, cls, val, log_probs=log_probs)
    assert loss.item() == math.inf and (grad[0] == 0).all() and torch.isfinite(grad).all()


def test_distillation_with_every_class_kept(M):
    """The rest has no classes: its term is left out, whatever mass rounding leaves it; more kept entries than classes."""
    for shape in ((5, 12), (5, 12, 3, 2)):
        z = scores(shape, "f32", seed=1)
        cls, val = teacher_top(shape, 12, 2, True, 1.0)
        check_distill(M, z, cls, val, log_probs=True)
        pad = torch.full_like(cls, -1)
        check_distill(M, z, torch.cat([cls, pad], 1), torch.cat([val, val], 1), log_probs=True)
    # all but one kept, the student's rest vanishing beside them
    z = torch.zeros(2, 9, device="cuda"); z[:, 8] = -60.0
    cls = torch.arange(8, device="cuda").expand(2, 8).contiguous()
    val = torch.full((2, 8), math.log(0.12), device="cuda")
    check_distill(M, z, cls, val, log_probs=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_distillation_of_strided_logits(M, dtype):
    wide = scores((9, 1300), dtype, seed=1)
    for z in (wide[:, 3:1004], wide[::2, :70], wide.t()[:40], wide[:1].expand(4, 1300), wide.view(-1)[1:1 + 4 * 333].view(4, 333)):
        check_distill(M, z, *teacher_top(tuple(z.shape), 5, 2, True, 1.0), log_probs=True)
    maps = scores((4, 20, 6, 9), dtype, seed=4)
    for z in (maps.contiguous(memory_format=torch.channels_last), maps[::2], maps[:, 3:15], maps[..., 1:7]):
        cls, val = teacher_top(tuple(z.shape), 5, 2, False, 1.0)
        check_distill(M, z, cls, val)
        check_distill(M, z, cls.contiguous(memory_format=torch.channels_last), val)


def test_distillation_refusals(M):
    from multimae_amd import ops
    from multimae_amd._lib import MmaeError
    z = torch.randn(4, 9, 8, 8, device="cuda")
    cls, val = teacher_top(tuple(z.shape), 3, 1, False, 1.0)
    mask = torch.ones(4, 4, dtype=torch.long, device="cuda")
    fn = M.MaskedDistillationLoss(16, 4)
    assert torch.isfinite(fn(z, (cls, val), mask=mask))
    many = torch.zeros(4, 65, 8, 8, device="cuda")
    for bad in (lambda: fn(z, (cls[:, :2], val)), lambda: fn(z, (cls.float(), val)), lambda: fn(z, (cls, val.double())), lambda: fn(z, (many.long(), many)),
                lambda: fn(z, (cls[:, :0], val[:, :0])), lambda: fn(z, (cls.cpu(), val)), lambda: fn(z, (cls, val), mask=mask[:, :3]),
                lambda: fn(z.cpu(), (cls.cpu(), val.cpu())), lambda: fn(z[:, :, :6], (cls[:, :, :6], val[:, :, :6]), mask=mask),
                lambda: M.MaskedDistillationLoss(16, 4, temperature=0.0)(z, (cls, val)), lambda: fn(z[:0], (cls[:0], val[:0])),
                lambda: fn(z.double(), (cls, val)), lambda: ops.distill(z, cls, val, d_logits=torch.empty(4, 9, 8, 8, device="cuda").bfloat16()),
                lambda: ops.Distillation(z, cls, val).scale(torch.empty_like(z), torch.ones(2, device="cuda"))):
        with pytest.raises(MmaeError):
            bad()
    with pytest.raises(ValueError):
        M.MaskedDistillationLoss(teacher="probs")


def test_distillation_gradient_against_differences(M):
    """Central differences along random directions; the third derivative of a log-sum-exp along d is below 2 |d|_inf^3, twice
    of them with the rest, times T^2 / T^3."""
    for shape, log_probs in (((3, 40), False), ((3, 40), True), ((2, 3000), True), ((2, 30, 2, 2), True)):
        t = 1.3
        z = scores(shape, "f32", seed=1, scale=1.0)
        cls, val = teacher_top(shape, 6, 2, log_probs, t)
        fn = loss_module(M, 1, t, log_probs)
        leaf = z.clone().requires_grad_(True)
        (grad,) = torch.autograd.grad(fn(leaf, (cls, val)), leaf)
        _, size, _, _ = reference_distill(z, cls, val, None, 1, t, log_probs)
        tol = size.item() * (2 * CHAIN + 16 * U * (1 + math.log(shape[1])) + 32 * U)
        for seed in range(3):
            d = torch.randn(shape, generator=torch.Generator().manual_seed(10 + seed)).cuda().clamp(-1, 1)
            h = 0.05
            slope = (fn(z + h * d, (cls, val)).double() - fn(z - h * d, (cls, val)).double()) / (2 * h)
            assert abs(slope.item() - (grad.double() * d.double()).sum().item()) < tol / h + 4 / t * h * h / 6


def test_distillation_beyond_32_bit_offsets(M):
    n, c = 16500, 131072
    z = torch.zeros(n, c, dtype=torch.bfloat16, device="cuda")
    last = scores((3, c), "bf16", seed=1)
    z[-3:] = last
    cls, val = teacher_top((3, c), 4, 2, True, 1.0)
    all_cls = torch.full((n, 4), -1, device="cuda"); all_cls[-3:] = cls
    all_val = torch.zeros(n, 4, device="cuda"); all_val[-3:] = val
    mask = torch.zeros(n, dtype=torch.long, device="cuda"); mask[-3:] = 1
    leaf = z.requires_grad_(True)
    loss = M.MaskedDistillationLoss(teacher="log_probs")(leaf, (all_cls, all_val), mask=mask)
    (grad,) = torch.autograd.grad(loss, leaf)
    few = last.clone().requires_grad_(True)
    want = M.MaskedDistillationLoss(teacher="log_probs")(few, (cls, val))
    (want_grad,) = torch.autograd.grad(want, few)
    assert abs(loss.item() - want.item()) < abs(want.item()) * 4 * CHAIN
    close(grad[-3:], want_grad.double().cpu(), 2 * half_step(torch.bfloat16, want_grad.double().cpu()), "grad")
    assert (grad[:-3] == 0).all()


def check_repeated(M, base, cls, val, rows, log_probs, temperature=1.0):
    """Many rows, repetitions of a few (the oracle's work is that of the few), a third of them outside the loss and NaN there."""
    n = base.shape[0]
    which = torch.arange(rows) % n
    mask = (torch.rand(rows, generator=torch.Generator().manual_seed(1)) > 0.33).long()
    mask[rows - 1] = 1
    z = base[which.cuda()]
    z[mask.cuda() == 0] = float("nan")
    leaf = z.requires_grad_(True)
    fn = loss_module(M, 1, temperature, log_probs)
    loss = fn(leaf, (cls[which.cuda()], val[which.cuda()]), mask=mask.view(-1, 1).cuda())
    (grad,) = torch.autograd.grad(loss, leaf, retain_graph=True)
    (scaled,) = torch.autograd.grad(loss, leaf, torch.tensor(-3.0, device="cuda"))
    with torch.no_grad():
        alone = fn(leaf, (cls[which.cuda()], val[which.cuda()]), mask=mask.view(-1, 1).cuda())
    c, count = base.shape[1], mask.sum().item()
    rel = 2 * CHAIN + 16 * U * (1 + math.log(c)) + (cls.shape[1] + 16) * U
    total, sizes = 0.0, 0.0
    for j in range(n):
        want, size, want_grad, grad_size = reference_distill(base[j:j + 1], cls[j:j + 1], val[j:j + 1], None, 1, temperature, log_probs)
        times = (mask[which == j] != 0).sum().item()
        total, sizes = total + want * times / count, sizes + size * times / count
        at = ((which == j) & (mask != 0)).nonzero().view(-1)
        mine = grad[at.cuda()]
        assert torch.equal(mine, mine[:1].expand_as(mine)), ("one row, two gradients", j)
        size = grad_size * (rel + 8 * U * 30)
        close(mine[:1], want_grad / count, half_step(base.dtype, want_grad / count) + size / count, f"grad of row {j}")
        mine = scaled[at.cuda()]
        assert torch.equal(mine, mine[:1].expand_as(mine)), ("one row, two gradients, upstream -3", j)
        close(mine[:1], -3 * want_grad / count, half_step(base.dtype, 3 * want_grad / count) + 3 * size / count, f"grad of row {j}, upstream -3")
    assert (grad[(mask == 0).cuda()] == 0).all() and (scaled[(mask == 0).cuda()] == 0).all()
    for got in (loss, alone):
        close(got, total, torch.as_tensor(sizes * (rel + 2 * 16 * U)), "loss")


MANY_ROWS = [(2100, c, d) for d in ("bf16", "f16") for c in (2049, 4095, 4104, 8191, 9000, 16384, 20001, 32768)] \
    + [(2100, c, "f32") for c in (2049, 3001, 4096)] \
    + [(600, c, "bf16") for c in (32769, 49152, 50001, 70000, 90007, 100000, 114696, 131072)] \
    + [(300, c, "f32") for c in (32770, 50001, 65536)]


@pytest.mark.parametrize("log_probs", [False, True], ids=["logits", "log_probs"])
@pytest.mark.parametrize("rows,c,dtype", MANY_ROWS, ids=str)
def test_distillation_of_many_rows(M, rows, c, dtype, log_probs):
    """More rows than the card takes at once: masked classes, padding, duplicates, empty rows and rows at the lowest value among
    them, so that one kind follows another."""
    base = scores((8, c), dtype, seed=c)
    cls, val = teacher_top((8, c), 9, 5, log_probs, 1.5)
    cls[0, 3:] = -1
    cls[1, ::2] = c + 5
    cls[2] = -100
    cls[3, 4] = cls[3, 2]; cls[3, 8] = cls[3, 2]
    cls[3, 0], cls[3, 1], cls[3, 3] = 0, c - 1, (c // 2048) * 2048 - 1    # the ends, and where the pieces meet
    val[4, 5:] = NINF
    base[5, : c // 2] = NINF
    cls[5] = torch.where(cls[5] < c // 2, cls[5] + (c + 1) // 2, cls[5]).clamp(max=c - 1)
    base[6] = torch.finfo(base.dtype).min
    check_repeated(M, base, cls, val, rows, log_probs, 1.5)
    base[1] = NINF
    fn = loss_module(M, 1, 1.5, log_probs)
    leaf = base[(torch.arange(rows) % 8).cuda()].requires_grad_(True)
    loss = fn(leaf, (cls.repeat(rows // 8 + 1, 1)[:rows], val.repeat(rows // 8 + 1, 1)[:rows]))
    (grad,) = torch.autograd.grad(loss, leaf)
    # (a row without a class left: no gradient, and an infinite loss wherever the teacher's mass is above zero)
    assert loss.item() == math.inf and (grad[1::8] == 0).all() and torch.isfinite(grad).all()


@pytest.mark.parametrize("log_probs", [False, True], ids=["logits", "log_probs"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("c", [1, 7, 32, 33, 64, 65, 104, 105, 133, 136, 137])
def test_distillation_of_many_small_maps(M, c, dtype, log_probs):
    """As many tiles of positions as the card has waves, few classes: masks with NaN outside, padding, duplicates, -inf and the
    lowest value, up to 16 kept classes and more."""
    shape = (530, c, 4, 6)
    z = scores(shape, dtype, seed=c)
    mask = (classes((530, 6), 4, 5) > 0).long()
    mask[7] = 0
    for k in (min(16, c), min(3, c), min(17, c)):
        cls, val = teacher_top(shape, k, 3, log_probs, 1.5, "bf16" if k == 3 else "f32", torch.int32 if k == 3 else torch.int64)
        cls[0, k // 2:] = -1
        cls[1] = c
        cls[2, -1] = cls[2, 0]; cls[2, k // 2] = cls[2, 0]
        val[3, k // 2:] = NINF
        z[4] = torch.finfo(z.dtype).min
        z[5, c // 2:] = torch.finfo(z.dtype).min
        z[6, 1::2] = torch.finfo(z.dtype).min
        check_distill(M, z, cls, val, None, 1, 1.5, log_probs)
        off = (mask == 0).view(530, 1, 2, 3).repeat_interleave(2, 2).repeat_interleave(2, 3).expand(shape)
        check_distill(M, torch.where(off, float("nan"), z), cls, val, mask, 2, 1.5, log_probs)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_distillation_of_large_maps(M, dtype):
    shape = (5, 133, 90, 91)
    for log_probs in (False, True):
        check_distill(M, scores(shape, dtype, 1), *teacher_top(shape, 8, 2, log_probs, 2.0), temperature=2.0, log_probs=log_probs)


def test_scaling_needs_a_gradient_to_scale(M):
    from multimae_amd import ops
    from multimae_amd._lib import MmaeError
    z = scores((300, 40000), "bf16", 1)
    call = ops.Distillation(z, *teacher_top((300, 40000), 8, 2, True, 1.0), log_probs=True)
    one, two, d = torch.ones((), device="cuda"), torch.full((), 2.0, device="cuda"), torch.empty_like(z)
    with pytest.raises(MmaeError):
        call.scale(d, one)
    loss = call.run()
    with pytest.raises(MmaeError):
        call.scale(d, one)
    assert torch.equal(call.run(d), loss) or abs(call.run(d).item() - loss.item()) < 4 * CHAIN * (abs(loss.item()) + 1)
    first = d.clone()
    assert torch.equal(call.scale(d, one), first)
    assert torch.equal(call.scale(d, two), 2 * first)  # (a power of two: exact; none of the gradients is subnormal in bf16)
    call.run()
    with pytest.raises(MmaeError):
        call.scale(d, one)


# ------------------------------------------------------------------------------------------------ as they are used
def test_class_distribution_calls_are_bitwise_reproducible_and_stay_in_their_buffers(M):
    from multimae_amd import ops
    for shape in ((5, 133, 9, 7), (300, 133), (40, 3000), (3, 100003), (3, 2000, 9, 9)):
        z = scores(shape, "bf16", seed=1)
        target = classes(shape[:1] + shape[2:], shape[1], 2)
        cls, val = teacher_top(shape, 8, 3, True, 1.0)
        room = torch.full((z.numel() + 64,), 7.0, dtype=z.dtype, device="cuda")
        d = room[32:32 + z.numel()].view(shape)
        first = None
        for _ in range(3):
            out = ops.class_log_probs(z, target, 8)
            g = ops.class_log_probs_bwd(z, target, out[1], out[4], out[0], out[1])
            loss = ops.distill(z, cls, val, log_probs=True, d_logits=d)
            now = [t.clone() for t in (*out, g, loss, d)]
            first = first or now
            assert all(torch.equal(a, b) for a, b in zip(first, now))
        assert (room[:32] == 7).all() and (room[-32:] == 7).all()


def test_class_distributions_on_another_stream_and_two_at_once(M):
    z = scores((64, 30000), "bf16", seed=1)
    target = classes((64,), 30000, 2)
    cls, val = teacher_top((64, 30000), 8, 3, True, 1.0)
    fn = M.MaskedDistillationLoss(teacher="log_probs")
    want = M.class_log_probs(z, target, top_k=8), fn(z, (cls, val))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append((M.class_log_probs(z, target, top_k=8), fn(z, (cls, val))))
    torch.cuda.synchronize()
    for out, loss in got:
        assert all(torch.equal(a, b) for a, b in zip(out, want[0])) and torch.equal(loss, want[1])


@pytest.mark.parametrize("shape", [(40, 133), (24, 9000), (2, 140000), (3, 133, 8, 12), (2, 1111, 8, 12)], ids=str)
def test_class_distributions_in_captured_graphs(M, shape):
    """A teacher's alternatives, the student's loss and its gradient captured as one graph, two such graphs, replayed in turn
    with new logits and eager calls in between."""
    teacher, z = scores(shape, "bf16", seed=1), scores(shape, "bf16", seed=2).requires_grad_(True)
    target = classes(shape[:1] + shape[2:], shape[1], 3)
    fn = M.MaskedDistillationLoss(teacher="log_probs")

    def step(scale):
        t = M.class_log_probs(teacher, target, top_k=8)
        loss = fn(z, (t.top_class, t.top_log_prob)) * scale
        s = M.class_log_probs(z, target)
        (grad,) = torch.autograd.grad(loss + s.entropy.mean(), z)
        return [t.top_class, t.top_log_prob, loss.detach(), s.log_prob.detach(), grad]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(1.0)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for scale in (1.0, 0.25):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step(scale)
        graphs.append((g, outs, scale))
    for i in range(4):
        with torch.no_grad():
            teacher.copy_(scores(shape, "bf16", seed=20 + i))
            z.copy_(scores(shape, "bf16", seed=30 + i))
        for g, outs, scale in graphs:
            g.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in outs]
            assert all(torch.equal(a, b) for a, b in zip(got, step(scale))), (i, scale)


def test_outputs_can_be_changed_in_place_and_one_of_them_used(M):
    z = scores((5, 200), "f32", seed=1).requires_grad_(True)
    target = classes((5,), 200, 2)
    out = M.class_log_probs(z, target, top_k=3)
    out.log_prob.mul_(2.0)
    (got,) = torch.autograd.grad(out.log_prob.sum(), z)
    p = torch.softmax(z.detach().double(), 1)
    want = -2 * p
    want[torch.arange(5), target] += 2
    close(got, want.cpu(), 2 * U * want.abs().cpu() + 2 * CHAIN, "grad")
    assert not out.top_class.requires_grad and not out.top_log_prob.requires_grad
    with torch.no_grad():
        assert not M.class_log_probs(z, target).log_prob.requires_grad
        assert not M.MaskedDistillationLoss()(z, (target.view(5, 1), torch.zeros(5, 1, device="cuda"))).requires_grad


@pytest.mark.parametrize("shape", [(40, 133), (24, 9000), (700, 40007), (3, 133, 8, 12), (2, 1111, 8, 12), (5, 21, 50)], ids=str)
def test_timed_calls_go_through_the_python_nodes_with_the_same_results(M, shape, monkeypatch):
    from multimae_amd import functional, ops
    target = classes(shape[:1] + shape[2:], shape[1], 3)
    cls, val = teacher_top(shape, 8, 2, True, 1.5)
    mask = torch.ones(shape[0], math.prod(shape[2:]), dtype=torch.long, device="cuda")
    mask[1] = 0
    fn = loss_module(M, 1, 1.5, True)
    rows = []
    for profile in (None, []):
        monkeypatch.setattr(ops, "PROFILE", profile)
        z = scores(shape, "bf16", 1).requires_grad_(True)
        out = M.class_log_probs(z, target, top_k=5, temperature=1.5)
        (g,) = torch.autograd.grad(out[:2], z, [torch.ones_like(out.entropy), out.entropy.detach()], retain_graph=True)
        loss = fn(z, (cls, val), mask=mask)
        mine = []
        for up in (1.0, 1.0, 0.3):
            mine += torch.autograd.grad(loss, z, torch.tensor(up, device="cuda"), retain_graph=True)
        assert mine[0].data_ptr() != mine[1].data_ptr()
        marked = fn(z, (cls, val), mask=mask)
        functional.mark_unit_upstream([marked])
        (unit,) = torch.autograd.grad(marked, z, torch.tensor(5.0, device="cuda"))  # (taken at its word)
        with torch.no_grad():
            plain = (*M.class_log_probs(z, target, top_k=3), fn(z, (cls, val), mask=mask))
        rows.append([*out, g, loss, *mine, unit, *plain])
        assert (type(loss.grad_fn).__name__ == "DistillFnBackward") == (profile is not None)
    assert all(torch.equal(a, b) for a, b in zip(*rows)) and torch.equal(rows[0][9], rows[0][6])  # (unit, the first of mine)


def test_the_teacher_has_no_gradient(M, monkeypatch):
    from multimae_amd import ops
    z = scores((6, 500), "f32", 1)
    cls, val = teacher_top((6, 500), 4, 2, False, 1.0)
    fn = M.MaskedDistillationLoss()
    for profile in (None, []):
        monkeypatch.setattr(ops, "PROFILE", profile)
        leaf, teacher = z.clone().requires_grad_(True), val.clone().requires_grad_(True)
        assert not fn(z, (cls, teacher)).requires_grad
        fn(leaf, (cls, teacher)).backward()
        assert leaf.grad is not None and teacher.grad is None


def test_what_a_call_points_to_lives_as_long_as_it_is_needed(M):
    """ops.Distillation keeps its arguments; a loss that is kept after the backward pass keeps none of them."""
    import gc
    from multimae_amd import ops
    z = scores((300, 40000), "bf16", 1)
    cls, val = teacher_top((300, 40000), 8, 2, True, 1.0)
    d = torch.empty_like(z)
    want = ops.distill(z, cls, val, log_probs=True, d_logits=d)
    call = ops.Distillation(z.clone(), cls.clone(), val.clone(), log_probs=True)
    trash = [torch.full_like(t, 1) for t in (z, cls, val)]
    got = torch.empty_like(z)
    assert torch.equal(call.run(got), want) and torch.equal(got, d)
    trash += [torch.full_like(t, 1) for t in (z, cls, val)]
    assert torch.equal(call.scale(got, torch.ones((), device="cuda")), d)
    del call, trash, got
    gc.collect()
    fn = M.MaskedDistillationLoss(teacher="log_probs")
    leaf = z.clone().requires_grad_(True)  # (the graph keeps its leaf, and the leaf its gradient: not what is counted)
    before = torch.cuda.memory_allocated()
    loss = fn(leaf * 1.0, (cls.clone(), val.clone()))
    loss.backward()
    with pytest.raises(RuntimeError):  # the graph is freed
        loss.backward()
    leaf.grad = None
    gc.collect()
    assert torch.cuda.memory_allocated() - before < 4096  # the loss itself
    # changed since: refused, as for any tensor that autograd saved
    leaf = z.clone().requires_grad_(True)
    x = leaf * 1.0
    loss = fn(x, (cls, val))
    x.mul_(2.0)
    with pytest.raises(RuntimeError):
        loss.backward()


def test_gradients_of_gradients_are_refused_and_other_gradient_types_taken(M):
    z = scores((6, 500), "bf16", 1).requires_grad_(True)
    target = classes((6,), 500, 2)
    loss = M.MaskedDistillationLoss()(z, (target.view(6, 1), torch.zeros(6, 1, device="cuda")))
    out = M.class_log_probs(z, target)
    for value in (loss, out.entropy.sum()):
        (first,) = torch.autograd.grad(value, z, retain_graph=True)
        (grad,) = torch.autograd.grad(value, z, create_graph=True)
        assert torch.equal(grad, first)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(grad.sum(), z)
    # gradients that are expanded, strided or of another type
    gl = torch.randn(12, generator=torch.Generator().manual_seed(3)).cuda()[::2]
    (want,) = torch.autograd.grad(out.log_prob, z, gl.contiguous(), retain_graph=True)
    (got,) = torch.autograd.grad(out.log_prob, z, gl, retain_graph=True)
    assert torch.equal(got, want)
    half = gl.bfloat16()
    (want,) = torch.autograd.grad(out.log_prob, z, half.float(), retain_graph=True)
    (got,) = torch.autograd.grad(out.log_prob, z, half, retain_graph=True)
    assert torch.equal(got, want)
    (want,) = torch.autograd.grad(loss, z, torch.tensor(0.5, device="cuda"), retain_graph=True)
    (got,) = torch.autograd.grad(loss, z, torch.tensor(0.5, device="cuda", dtype=torch.float64))
    assert torch.equal(got, want)


def test_a_teacher_labels_and_the_pretraining_step_distils(M):
    """As they are used together: the teacher decoder's alternatives become the target of the semseg task in PretrainStep, with
    the semseg domain's mask; the gradients are those of the plain definition through the same model."""
    from multimae_amd.builders import build_multimae
    from multimae_amd.train import PretrainStep
    torch.manual_seed(0)

    def build():
        torch.manual_seed(1)
        return build_multimae(in_domains=("rgb", "depth", "semseg"), out_domains=("semseg",), image_size=64, extra_norm_pix_loss=False,
                              decoder_depth=1).cuda()
    g = torch.Generator().manual_seed(2)
    B = 4
    batch = {"rgb": torch.randn(B, 3, 64, 64, generator=g).cuda(), "depth": torch.randn(B, 1, 64, 64, generator=g).cuda(),
             "semseg": torch.randint(0, 133, (B, 16, 16), generator=g).cuda()}
    teacher = scores((B, 133, 16, 16), "f32", seed=3)
    labels = M.class_log_probs(teacher, batch["semseg"], top_k=8, temperature=2.0)
    batch["semseg_teacher"] = (labels.top_class, labels.top_log_prob)
    fn = M.MaskedDistillationLoss(16, 4, temperature=2.0, teacher="log_probs")
    grads = {}
    for name, loss_fn in (("kernel", fn), ("plain", None)):
        masks_seen = []

        def plain(pred, target, mask=None):
            cls, val = target
            x = torch.log_softmax(pred.float() / 2.0, 1)
            q = val.exp()
            kept = torch.zeros_like(x, dtype=torch.bool).scatter_(1, cls, True)
            r = (1 - val.double().exp().sum(1)).clamp(min=0).float()
            rows = (q * (val - x.gather(1, cls))).sum(1) + r * (r.log() - torch.logsumexp(x.masked_fill(kept, NINF), 1))
            m = mask.view(-1, 4, 4).repeat_interleave(4, 1).repeat_interleave(4, 2).float()
            count = m.sum((1, 2))
            per = (rows * m).sum((1, 2)) / count.clamp(min=1)
            masks_seen.append(mask)
            return 4.0 * per[count > 0].mean()
        torch.manual_seed(7)
        model = build()
        step = PretrainStep(model, {"semseg": (loss_fn or plain, "semseg_teacher", "semseg")}, num_encoded_tokens=12, lr=0.0, weight_decay=0.0,
                            keep_grads=True)
        torch.manual_seed(9)
        loss, tasks, _ = step(batch)
        grads[name] = (loss.item(), torch.cat([p.grad.flatten() for p in model.parameters() if p.grad is not None]).clone())
    (a, ga), (b, gb) = grads["kernel"], grads["plain"]
    # one loss on the same bf16 predictions, in fp32 on both sides; the gradients pass through the same bf16 kernels, whose
    # input differs by one rounding of d_logits: half a step of bf16 (2^-8) at every operand along the way
    assert abs(a - b) < 1e-5 * abs(b), (a, b)
    assert ((ga - gb).norm() / gb.norm()).item() < 2.0 ** -7
