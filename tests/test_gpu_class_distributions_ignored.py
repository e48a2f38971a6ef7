"""Positions that a call leaves out, whatever stands there."""
import pytest
import torch

from tests.test_gpu_class_distributions import M, classes, scores  # noqa: F401  (M: the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", [(9, 70), (9, 2049), (9, 40007), (9, 70, 3, 5), (9, 1700, 3, 5), (9, 33, 70)], ids=str)
def test_ignored_positions_have_no_gradient_whatever_their_logits(M, shape, dtype):  # noqa: F811
    """A target outside the classes: a log probability of 0 without a gradient, with NaN, infinities or nothing left among the logits,
    for the log probability alone and with an entropy whose gradient is 0 there."""
    z = scores(shape, dtype, 1)
    target = classes(shape[:1] + shape[2:], shape[1], 2)
    want = torch.autograd.grad(M.class_log_probs(z.requires_grad_(True), target).log_prob.sum(), z)[0]
    z = z.detach().clone()
    out = torch.zeros_like(target, dtype=torch.bool)
    for n, (i, bad, first) in enumerate(((1, float("nan"), 3), (2, float("inf"), 0), (3, float("-inf"), 0), (4, -1e30 if dtype != "f16" else -6e4, 0), (6, float("nan"), 0))):
        z[i, first:] = bad
        target[i] = (-100, shape[1], -1, 2 ** 40, -2 ** 40)[n]
        out[i] = True
    if len(shape) > 2:  # single positions of a wave
        z[8, 1, ..., ::2] = float("nan")
        target[8, ..., ::2] = -100
        out[8, ..., ::2] = True
    z.requires_grad_(True)
    got = M.class_log_probs(z, target)
    assert (got.log_prob[out] == 0).all() and torch.isfinite(got.log_prob).all()
    (alone,) = torch.autograd.grad(got.log_prob.sum(), z, retain_graph=True)
    zero = torch.zeros_like(got.entropy)
    (beside,) = torch.autograd.grad((got.log_prob, got.entropy), z, (torch.ones_like(zero), zero))
    keep = ~out.unsqueeze(1).expand(shape)
    for grad in (alone, beside):
        assert (grad[~keep] == 0).all() and torch.equal(grad[keep], want[keep])
