"""The autograd nodes of the class distributions without a GPU: the launches are recorded instead of made, so no address is followed."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from multimae_amd import functional, ops


@pytest.fixture
def launches(monkeypatch):
    """(name, arguments) of every launch; tensors on the CPU are taken."""
    seen = []
    monkeypatch.setattr(ops, "_launch", lambda what, fn, device, nbytes, *args: seen.append((what, args)))
    monkeypatch.setattr(ops, "_req", lambda t, *a, **k: t)
    monkeypatch.setattr(ops, "_beside", lambda t, *a: t)
    return seen


def distill_args():
    logits = torch.randn(6, 40)[:, 3:33].requires_grad_(True)  # rows further apart: the Python node
    return logits, torch.randint(0, 30, (6, 4)), torch.randn(6, 4), torch.ones(6, 1, dtype=torch.long)


def strided(t):
    """t with its elements two apart."""
    return torch.stack([t, t], -1)[..., 0]


class Unpacked(torch.autograd.graph.saved_tensors_hooks):
    """Saved tensors live elsewhere when they come back, in the layout that `like` gives them."""

    def __init__(self, like=torch.clone):
        self.given = []

        def unpack(t):
            self.given.append(like(t))
            return self.given[-1]
        super().__init__(lambda t: t.detach().clone(), unpack)


def test_distillation_backward_points_to_the_unpacked_tensors(launches):
    logits, cls, val, mask = distill_args()
    hooks = Unpacked()
    with hooks:
        loss = functional.distill(logits, cls, val, mask, 1, 1.0, True)
    for again in range(2):
        hooks.given.clear()
        torch.autograd.grad(loss, logits, torch.tensor(3.0), retain_graph=True)
        args = launches[-1][1]
        at = {t.data_ptr() for t in hooks.given}
        assert len(hooks.given) == 5
        for place, what in ((0, "logits"), (6, "classes"), (8, "values"), (13, "mask"), (-2, "workspace")):
            assert args[place] in at, (what, again)
        assert args[5] == hooks.given[0].stride(0)


def test_distillation_backward_after_recomputation_points_to_the_recomputed_tensors(launches):
    logits, cls, val, mask = distill_args()
    made = []

    def body(x):
        made.append((x * 2.0).t().contiguous().t()[:, :29])
        return functional.distill(made[-1], cls % 29, val, mask, 1, 1.0, False)
    loss = checkpoint(body, logits, use_reentrant=False)
    made.clear()  # what the first forward pass made is gone
    torch.autograd.grad(loss, logits, torch.tensor(3.0))
    first, again, last = (args[0] for _, args in launches)
    assert len(made) == 1 and last == again != first


def test_backward_passes_take_any_layout_from_the_hooks(launches):
    logits, cls, val, mask = distill_args()
    hooks = Unpacked(strided)
    target = torch.randint(0, 30, (6,))
    with hooks:
        loss = functional.distill(logits, cls, val, mask, 1, 1.0, True)
        log_prob, entropy, _, _ = functional.class_log_probs(logits, target, 0, 1.0)
    contiguous = []
    launch = ops._launch

    def look(what, fn, device, nbytes, *args):  # (while the tensors live)
        import ctypes
        if what == "class_log_probs_bwd":
            contiguous.append([ctypes.c_int64.from_address(args[6] + 8 * i).value for i in range(6)] == target.tolist())
            contiguous.append([ctypes.c_float.from_address(args[0] + 4 * i).value for i in range(30)] == logits[0].tolist())
        elif what == "distill":
            contiguous.append([ctypes.c_int64.from_address(args[6] + 8 * i).value for i in range(24)] == cls.flatten().tolist())
            contiguous.append([ctypes.c_float.from_address(args[8] + 4 * i).value for i in range(24)] == val.flatten().tolist())
        launch(what, fn, device, nbytes, *args)
    ops._launch = look
    torch.autograd.grad(loss, logits, torch.tensor(3.0))
    torch.autograd.grad((log_prob, entropy), logits, (torch.ones(6), torch.ones(6)))
    assert contiguous == [True] * 4


def test_forward_mode_and_tracing_are_refused_by_name():
    """Neither sees the kernels: a derivative of zero, a graph that holds nothing but the outputs' allocations."""
    import multimae_amd as M
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx
    from multimae_amd._lib import MmaeError
    z, t, v = torch.randn(6, 30), torch.randint(0, 30, (6,)), torch.randn(6, 1)
    calls = [lambda x: M.class_log_probs(x, t).log_prob, lambda x: M.MaskedDistillationLoss()(x, (t.view(6, 1), v))]
    for call in calls:
        with forward_ad.dual_level():
            with pytest.raises(MmaeError, match="forward-mode"):
                call(forward_ad.make_dual(z, torch.ones_like(z)))
            with pytest.raises(MmaeError, match="GPU"):  # (no tangent: an ordinary call)
                call(z)
        with pytest.raises(MmaeError, match="traced"):
            torch.jit.trace(call, z, check_trace=False)
        with pytest.raises(MmaeError, match="traced"):
            make_fx(call)(z)
        with pytest.raises(MmaeError, match="GPU"):
            call(z)


def test_without_the_module_the_python_nodes_serve(launches, monkeypatch, recwarn):
    import sys

    import multimae_amd
    monkeypatch.setitem(sys.modules, "multimae_amd._nodes", None)  # (an import error)
    monkeypatch.delattr(multimae_amd, "_nodes", raising=False)
    monkeypatch.setattr(functional, "_node_module", False)
    logits, cls, val, mask = distill_args()
    for _ in range(2):
        loss = functional.distill(logits, cls, val, mask, 1, 1.0, True)
        functional.mark_unit_upstream([loss, logits.sum()])
        functional.class_log_probs(logits, cls[:, 0], 2, 1.0)
    assert [what for what, _ in launches] == ["distill", "class_log_probs"] * 2
    assert type(loss.grad_fn).__name__ == "DistillFnBackward" and loss.grad_fn.unit_upstream
    assert sum("_nodes" in str(w.message) for w in recwarn) == 1
