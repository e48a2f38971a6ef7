"""What the class distributions' C entries and their Python faces refuse before anything is launched: no GPU needed, and no
pointer is followed."""
import pytest
import torch

from multimae_amd import _lib

EINVAL, ESHAPE, EWORKSPACE = -1, -2, -3
P = 4096  # an address that is never read
INF, NAN = float("inf"), float("nan")

# arguments of a call that would be launched, by name
LOG_PROBS = dict(logits=P, dtype=0, outer=4, classes=100, inner=1, ld=100, target=P, top_k=5, temperature=1.0, log_prob=P, entropy=P,
                 row_max=P, row_log_sum=P, top_log_prob=P, top_class=P, workspace=None, workspace_bytes=0, stream=None)
BACKWARD = dict(logits=P, dtype=0, outer=4, classes=100, inner=1, ld=100, target=P, temperature=1.0, entropy=P, row_max=P, row_log_sum=P,
                d_log_prob=P, d_entropy=None, d_logits=P, stream=None)
DISTILL = dict(logits=P, dtype=0, outer=4, classes=100, inner=16, ld=1600, top_class=P, class_bytes=8, top_value=P, value_dtype=0, k=5, kind=1,
               temperature=1.0, mask=P, width=4, patch=2, upstream=None, again=0, skip_unit=0, loss=P, d_logits=P, workspace=P,
               workspace_bytes=1 << 20, stream=None)
COMMON = [(dict(logits=None), EINVAL, "null"), (dict(dtype=3), EINVAL, "dtype"), (dict(dtype=-1), EINVAL, "dtype"), (dict(outer=0), ESHAPE, "empty"),
          (dict(classes=0), ESHAPE, "empty"), (dict(inner=-1), ESHAPE, "empty"), (dict(ld=99), ESHAPE, "samples"),
          (dict(classes=(1 << 30) + 1, ld=1 << 40), ESHAPE, "classes"), (dict(outer=1 << 20, inner=1 << 12, ld=1 << 20), ESHAPE, "positions"),
          (dict(temperature=0.0), EINVAL, "temperature"), (dict(temperature=-1.0), EINVAL, "temperature"), (dict(temperature=INF), EINVAL, "temperature"),
          (dict(temperature=NAN), EINVAL, "temperature"), (dict(outer=1 << 27, inner=1, ld=1 << 20), ESHAPE, "launch")]
CASES = [("mmae_class_log_probs", LOG_PROBS, c) for c in COMMON + [
    (dict(target=None), EINVAL, "null"), (dict(log_prob=None), EINVAL, "null"), (dict(entropy=None), EINVAL, "null"),
    (dict(row_max=None), EINVAL, "null"), (dict(row_log_sum=None), EINVAL, "null"), (dict(top_class=None), EINVAL, "null"),
    (dict(top_log_prob=None), EINVAL, "null"), (dict(top_k=-1), ESHAPE, "top"), (dict(top_k=65), ESHAPE, "top"),
    (dict(classes=4, ld=4), ESHAPE, "top"), (dict(classes=100000, ld=100000), EWORKSPACE, "workspace"),
    (dict(classes=100000, ld=100000, workspace=None, workspace_bytes=1 << 30), EWORKSPACE, "workspace")]]
CASES += [("mmae_class_log_probs_bwd", BACKWARD, c) for c in COMMON + [
    (dict(target=None), EINVAL, "null"), (dict(entropy=None), EINVAL, "null"), (dict(row_max=None), EINVAL, "null"),
    (dict(row_log_sum=None), EINVAL, "null"), (dict(d_logits=None), EINVAL, "null"), (dict(outer=1 << 25, classes=4096, ld=4096), ESHAPE, "launch")]]
CASES += [("mmae_distill", DISTILL, c) for c in COMMON[:-1] + [
    (dict(outer=1 << 27, inner=1, ld=1 << 20, mask=None, workspace_bytes=1 << 40), ESHAPE, "launch"),
    (dict(top_class=None), EINVAL, "null"), (dict(top_value=None), EINVAL, "null"), (dict(workspace=None), EINVAL, "null"),
    (dict(loss=None, d_logits=None), EINVAL, "null"), (dict(class_bytes=2), EINVAL, "classes of"), (dict(value_dtype=3), EINVAL, "value"),
    (dict(k=0), ESHAPE, "kept"), (dict(k=65), ESHAPE, "kept"), (dict(kind=2), EINVAL, "kind"), (dict(patch=0), ESHAPE, "patches"),
    (dict(patch=3), ESHAPE, "patches"), (dict(width=3), ESHAPE, "patches"), (dict(width=0), ESHAPE, "patches"), (dict(width=8, patch=4), ESHAPE, "patches"),
    (dict(workspace_bytes=16), EWORKSPACE, "workspace"), (dict(again=1), EINVAL, "first call")]]


@pytest.mark.parametrize("name,args,case", CASES, ids=lambda v: v if isinstance(v, str) else "-".join(v[0]) if isinstance(v, tuple) else "")
def test_calls_are_refused_on_the_host(name, args, case):
    change, code, word = case
    lib = _lib.load()
    assert getattr(lib, name)(*{**args, **change}.values()) == code
    message = lib.mmae_last_error().decode()
    assert word in message and name[5:].split("_")[0] in message, message


def test_workspaces():
    lib = _lib.load()
    assert lib.mmae_class_log_probs_workspace_bytes(0, 4, 100, 1, 5) == 0         # a row is one wave's
    assert lib.mmae_class_log_probs_workspace_bytes(0, 1, 100000, 1, 64) > lib.mmae_class_log_probs_workspace_bytes(0, 1, 100000, 1, 0) > 0
    assert lib.mmae_class_log_probs_workspace_bytes(1, 4096, 100000, 1, 5) == 0   # a row is one workgroup's
    assert lib.mmae_class_log_probs_workspace_bytes(0, 2, 133, 64, 5) == 0        # a map's tile fits
    assert lib.mmae_class_log_probs_workspace_bytes(0, 2, 32000, 64, 5) >= 2 * 64 * (16 + 5 * 8)
    assert lib.mmae_distill_workspace_bytes(0, 2, 32000, 64, 5) > lib.mmae_distill_workspace_bytes(0, 2, 133, 64, 5)
    for bad in ((0, 1, 1, 0), (1, 0, 1, 0), (1, 1, 1, -1)):
        assert lib.mmae_class_log_probs_workspace_bytes(0, *bad) == 0
    assert lib.mmae_distill_workspace_bytes(0, 0, 1, 1, 1) == 0
    for rows in (1, 1000):
        for classes in (10, 5000, 300000):
            assert lib.mmae_distill_workspace_bytes(1, rows, classes, 1, 8) >= 4 * (4 + 2 * rows)


def test_the_nodes_leave_what_they_do_not_take():
    """Anything but contiguous tensors on the GPU is answered with None, before anything is launched."""
    from multimae_amd import _nodes
    z, t, v = torch.randn(4, 9), torch.zeros(4, dtype=torch.long), torch.zeros(4, 1)
    assert _nodes.class_log_probs(z, t, 2, 1.0) is None
    assert _nodes.distill(z, t.view(4, 1), v, None, 1, 1.0, False) is None
    assert not _nodes.mark_unit_upstream(z) and not _nodes.mark_unit_upstream(z.requires_grad_(True).sum())


def test_the_entry_points_take_tensors_on_the_gpu_only():
    import multimae_amd as M
    z, t = torch.randn(4, 9), torch.zeros(4, dtype=torch.long)
    for bad in (lambda: M.class_log_probs(z, t), lambda: M.class_log_probs(z.requires_grad_(True), t, top_k=2),
                lambda: M.MaskedDistillationLoss()(z, (t.view(4, 1), torch.zeros(4, 1)))):
        with pytest.raises(_lib.MmaeError, match="GPU"):
            bad()
    with pytest.raises(ValueError, match="teacher"):
        M.MaskedDistillationLoss(teacher="probs")
