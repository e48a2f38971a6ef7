"""Measured calls of the class-distribution operators: log probabilities with entropy and top alternatives, and distillation
from a teacher's top classes.

`own` chooses between the operators' plain form (elementary torch operations in 32 bits) and the framework's entry points
`multimae_amd.class_log_probs` and `multimae_amd.MaskedDistillationLoss`.  The class dimension is dimension 1, as in
torch's cross entropy: rows [N, C], or class maps [N, C, H, W]."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SCALE = 4  # patch_size // stride_level of the class map: 16 / 4


def _case(name, op, n, c, h=0, w=0, k=0, dtype="bf16", temperature=1.0, teacher="", masked=False, pad=0):
    """op: log_probs (values only), log_probs_step (values, and gradients of the log probability and the entropy), distill
    (loss and gradient).  h = w = 0: rows.  pad: classes at the end that are switched off (logit -inf), as in a vocabulary
    rounded up for the matrix product.  masked: positions outside the loss, one sample without any position in it."""
    return {"name": name, "op": op, "n": n, "c": c, "h": h, "w": w, "k": k, "dtype": dtype, "temperature": temperature,
            "teacher": teacher, "masked": masked, "pad": pad}


def listed():
    return [
        # one generated token's probability and its alternatives: only latency counts
        _case("logprob_1x32000", "log_probs", 1, 32000, k=5),
        # the tokens of a batch of streams, one each, over a large vocabulary
        _case("logprob_24x131072", "log_probs", 24, 131072, k=20),
        # scoring a prompt from fp32 logits, an odd vocabulary with switched-off classes, away from temperature 1
        _case("logprob_2047x50001_f32", "log_probs", 2047, 50001, k=8, dtype="f32", temperature=0.7, pad=40),
        # scoring a long prompt over the largest vocabulary: the largest call
        _case("logprob_4096x150016", "log_probs", 4096, 150016, k=8),
        # a training step that weights log probabilities and entropies, odd sizes
        _case("logprob_step_4095x64007", "log_probs_step", 4095, 64007, k=0),
        # the same for a classifier's few short rows
        _case("logprob_step_512x1000_f32", "log_probs_step", 512, 1000, k=5, dtype="f32"),
        # a teacher labels a batch of this repository's class maps (133 classes, 56 x 56) with its top classes
        _case("logprob_map_256x133x56x56_f32", "log_probs", 256, 133, 56, 56, k=8, dtype="f32"),
        # a training step on class maps of 384 x 384 images at stride 4
        _case("logprob_step_map_32x133x96x96", "log_probs_step", 32, 133, 96, 96, k=4),
        # distillation on a handful of rows
        _case("distill_16x32000", "distill", 16, 32000, k=16, temperature=2.0, teacher="logits"),
        # distillation over a large vocabulary against the teacher's top log probabilities and the rest they leave
        _case("distill_4096x128000_rest", "distill", 4096, 128000, k=32, teacher="log_probs"),
        # fp32, odd sizes, many kept classes, some rows outside the loss
        _case("distill_1023x50001_f32", "distill", 1023, 50001, k=64, dtype="f32", temperature=1.5, teacher="logits", masked=True),
        # this repository's class-map batch, the fp32 decoder's output, half of the patches in the loss
        _case("distill_map_256x133x56x56_f32", "distill", 256, 133, 56, 56, k=8, dtype="f32", temperature=2.0, teacher="logits",
              masked=True),
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["log_probs", "log_probs_step", "distill"])
    dtype = rng.choice(["bf16", "bf16", "f32", "f16"])
    temperature = rng.choice([1.0, 1.0, 0.5 + rng.random() * 2.5])
    teacher = rng.choice(["logits", "log_probs"]) if op == "distill" else ""
    masked = op == "distill" and rng.random() < 0.5
    most = 250_000_000  # logits of one call
    if rng.random() < 0.6:  # rows
        c = _log_uniform(rng, 20, 150_000)
        n = _log_uniform(rng, 1, max(1, min(8192, most // c)))
        h = w = 0
    else:  # class maps, whole patches on a side
        c = _log_uniform(rng, 5, 400)
        h, w = SCALE * rng.randint(2, 24), SCALE * rng.randint(2, 24)
        n = _log_uniform(rng, 1, max(1, min(256, most // (c * h * w))))
    most_k = min(64 if op == "distill" else 32, c // 2)
    k = _log_uniform(rng, 1, most_k)
    if op != "distill" and rng.random() < 0.3:
        k = 0
    pad = rng.randint(1, c // 8) if not h and c >= 64 and rng.random() < 0.4 else 0
    return _case("", op, n, c, h, w, k, dtype, temperature, teacher, masked, pad)


def prepare(case, seed):
    """Logits with one pronounced class at most positions, and what goes with them: the given classes and the gradients that
    arrive (log_probs), or the teacher's top classes and the patch mask (distill)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    n, c, h, w, k = case["n"], case["c"], case["h"], case["w"], case["k"]
    dtype = DTYPES[case["dtype"]]
    space = (h, w) if h else ()
    live = c - case["pad"]

    def scores(start=None):
        x = torch.randn(n, c, *space, device="cuda", generator=g)
        x.mul_(2.0)
        if start is not None:
            x.add_(start.float(), alpha=0.5)
        return x
    named = torch.randint(0, live, (n, 1) + space, device="cuda", generator=g)
    x = scores()
    x.scatter_add_(1, named, 10.0 * torch.rand(n, 1, *space, device="cuda", generator=g))
    if case["pad"]:
        x[:, live:] = float("-inf")
    logits = x.to(dtype)
    del x
    state = dict(case, logits=logits)
    if case["op"] == "distill":
        t = scores(logits)
        top = torch.topk(t, k, dim=1)
        state["top_class"] = top.indices.contiguous()
        if case["teacher"] == "logits":
            state["top_value"] = top.values.contiguous()
        else:
            t.div_(case["temperature"])
            state["top_value"] = (top.values / case["temperature"] - torch.logsumexp(t, dim=1, keepdim=True)).contiguous()
        state["mask"] = None
        if case["masked"]:
            tokens = (h // SCALE) * (w // SCALE) if h else 1
            mask = (torch.rand(n, tokens, device="cuda", generator=g) < 0.5).long()
            if n > 1:
                mask[0] = 0
            mask[-1, 0] = 1
            state["mask"] = mask if h else mask.view(n)
    else:
        state["target"] = torch.where(torch.rand(n, *space, device="cuda", generator=g) < 0.75, named.squeeze(1),
                                      torch.randint(0, live, (n,) + space, device="cuda", generator=g))
        if case["op"] == "log_probs_step":
            state["d_log_prob"] = torch.randn(n, *space, device="cuda", generator=g)
            state["d_entropy"] = torch.randn(n, *space, device="cuda", generator=g) * 0.1
    if case["op"] != "log_probs":
        logits.requires_grad_(True)
    return state


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain_distill(state) if state["op"] == "distill" else _plain_log_probs(state)


def _own(state):
    import multimae_amd as M
    logits = state["logits"]
    if state["op"] == "distill":
        loss_fn = M.MaskedDistillationLoss(patch_size=16, stride=4, temperature=state["temperature"], teacher=state["teacher"])
        loss = loss_fn(logits, (state["top_class"], state["top_value"]), mask=state["mask"])
        return {"loss": loss.detach(), "grad": torch.autograd.grad(loss, logits)[0]}
    out = M.class_log_probs(logits, state["target"], top_k=state["k"], temperature=state["temperature"])
    found = {"log_prob": out.log_prob.detach(), "entropy": out.entropy.detach()}
    if state["k"]:
        found["top_log_prob"], found["top_class"] = out.top_log_prob, out.top_class
    if state["op"] == "log_probs_step":
        found["grad"] = torch.autograd.grad((out.log_prob, out.entropy), logits, (state["d_log_prob"], state["d_entropy"]))[0]
    return found


def _log_softmax(x):
    """(log p, p) along dimension 1."""
    d = x - x.amax(1, keepdim=True)
    e = d.exp()
    s = e.sum(1, keepdim=True)
    return d - s.log(), e / s


def _plain_log_probs(state):
    z = state["logits"].float()
    k, c, t = state["k"], state["c"], state["temperature"]
    logp, p = _log_softmax(z / t)
    target = state["target"].unsqueeze(1)
    finite = torch.where(p > 0, logp, torch.zeros_like(logp))
    entropy = -(p * finite).sum(1)
    found = {"log_prob": logp.gather(1, target).squeeze(1), "entropy": entropy}
    if k:
        # value and inverted class in one integer: equal values rank by the lower class
        b = (z + 0.0).view(torch.int32).long()
        b = torch.where(b < 0, b ^ 0x7FFFFFFF, b)
        place = torch.arange(c - 1, -1, -1, device=z.device).view((1, c) + (1,) * (z.dim() - 2))
        best = ((b << 32) + place).topk(k, dim=1).values
        found["top_class"] = c - 1 - (best & 0xFFFFFFFF)
        found["top_log_prob"] = logp.gather(1, found["top_class"])
        found = {key: found[key] for key in ("log_prob", "entropy", "top_log_prob", "top_class")}
    if state["op"] == "log_probs_step":
        gl, gh = state["d_log_prob"].unsqueeze(1), state["d_entropy"].unsqueeze(1)
        grad = -p * (gl + gh * (finite + entropy.unsqueeze(1)))
        grad.scatter_add_(1, target, gl)
        found["grad"] = (grad / t).to(state["logits"].dtype)
    return found


def _plain_distill(state):
    z = state["logits"].float()
    t, ids, values = state["temperature"], state["top_class"], state["top_value"].float()
    x = z / t
    logp, p = _log_softmax(x)
    lp = logp.gather(1, ids)
    if state["teacher"] == "logits":
        lq, q = _log_softmax(values / t)
        loss = (q * (lq - lp)).sum(1)
        grad = p
    else:
        lq, q = values, values.exp()
        loss = (q * (lq - lp)).sum(1)
        total = values.double().exp().sum(1)  # 64 bits: the rest is what a sum near 1 leaves
        rq = (1.0 - total).clamp(min=0.0)
        kept = torch.zeros_like(z, dtype=torch.bool).scatter_(1, ids, True)
        other = torch.where(kept, torch.full_like(x, float("-inf")), x)
        rest_logp, rest_p = _log_softmax(other)
        log_rest = (logp.gather(1, other.argmax(1, keepdim=True)) - rest_logp.amax(1, keepdim=True)).squeeze(1)
        loss = loss + torch.where(rq > 0, rq * (rq.log() - log_rest), torch.zeros_like(rq)).float()
        grad = p * (total + rq).float().unsqueeze(1) - rest_p * rq.float().unsqueeze(1)
    grad = grad.scatter_add(1, ids, -q)
    weight = _weights(state, z)
    loss = (loss * weight).sum() * (t * t)
    return {"loss": loss, "grad": (grad * (weight * t).unsqueeze(1)).to(state["logits"].dtype)}


def _weights(state, z):
    """What each position's loss counts: the mean over a sample's positions in the loss, then over the samples that have any."""
    n, space = z.shape[0], z.shape[2:]
    mask = state["mask"]
    if mask is None:
        m = torch.ones((n,) + space, device=z.device)
    elif len(space) == 2:
        h, w = space
        m = mask.float().view(n, h // SCALE, 1, w // SCALE, 1).expand(n, h // SCALE, SCALE, w // SCALE, SCALE).reshape(n, h, w)
    else:
        m = mask.float().view((n,) + space)
    count = m.reshape(n, -1).sum(1)
    share = torch.where(count > 0, 1.0 / count, torch.zeros_like(count)) / (count > 0).sum().clamp(min=1)
    return m * share.view((n,) + (1,) * len(space))


def work(case):
    positions = case["n"] * max(1, case["h"] * case["w"])
    size = 4 if case["dtype"] == "f32" else 2
    logits = positions * case["c"]
    k = positions * case["k"]
    if case["op"] == "distill":  # logits, classes and values in; gradient out
        return {"bytes": 2 * logits * size + k * 12, "flops": 8 * logits}
    read = logits * size + positions * 16 + k * 12  # logits and classes in; log probability, entropy and top classes out
    if case["op"] == "log_probs":
        return {"bytes": read, "flops": 6 * logits}
    return {"bytes": read + logits * size + positions * 8, "flops": 11 * logits}  # two gradients in, one out


def exact(case, seed):
    """The definitions in 64 bits: torch's log_softmax, a stable sort and, for the gradients, differentiation."""
    state = prepare(case, seed)
    t, k = case["temperature"], case["k"]
    logits = state["logits"].detach()
    n = logits.shape[0]
    per = max(1, 40_000_000 // (logits.numel() // n))
    found = {}
    if case["op"] == "distill":
        mask = state["mask"]
        if mask is None:
            scale = torch.full(logits.shape[:1] + logits.shape[2:], 1.0 / (logits.numel() // case["c"]), dtype=torch.float64, device="cuda")
        else:
            m = mask.double()
            if case["h"]:
                m = m.view(n, case["h"] // SCALE, case["w"] // SCALE).repeat_interleave(SCALE, 1).repeat_interleave(SCALE, 2)
            flat = m.view(n, -1)
            some = flat.sum(1) > 0
            scale = torch.where(some[:, None], flat / flat.sum(1, keepdim=True).clamp(min=1), 0.0).div(some.sum()).view(m.shape)
    for a in range(0, n, per):
        x = logits[a:a + per].double().requires_grad_(case["op"] != "log_probs")
        logp = torch.log_softmax(x / t, 1)
        if case["op"] == "distill":
            ids, v = state["top_class"][a:a + per], state["top_value"][a:a + per].double()
            lq = torch.log_softmax(v / t, 1) if case["teacher"] == "logits" else v
            rows = (lq.exp() * (lq - logp.gather(1, ids))).sum(1)
            if case["teacher"] == "log_probs":
                rq = (1 - lq.exp().sum(1)).clamp(min=0)
                left = torch.logsumexp(logp.scatter(1, ids, float("-inf")), 1)
                rows = rows + torch.xlogy(rq, rq) - rq * left
            loss = (rows * scale[a:a + per]).sum() * t * t
            part = {"loss": loss.detach().view(1), "grad": torch.autograd.grad(loss, x)[0]}
        else:
            lp = logp.gather(1, state["target"][a:a + per, None]).squeeze(1)
            h = -(logp.exp() * torch.where(logp > -math.inf, logp, 0.0)).sum(1)
            part = {"log_prob": lp.detach(), "entropy": h.detach()}
            if k:
                order = torch.sort(x.detach().movedim(1, -1), dim=-1, descending=True, stable=True).indices[..., :k].movedim(-1, 1)
                part["top_log_prob"], part["top_class"] = logp.detach().gather(1, order), order
            if case["op"] == "log_probs_step":
                part["grad"] = torch.autograd.grad((lp, h), x, (state["d_log_prob"][a:a + per].double(), state["d_entropy"][a:a + per].double()))[0]
        for key, value in part.items():
            found.setdefault(key, []).append(value)
    found = {key: torch.cat(parts) for key, parts in found.items()}
    if "loss" in found:
        found["loss"] = found["loss"].sum()
    return found
