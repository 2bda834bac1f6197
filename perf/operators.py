"""The operators at the end of a language-model training step, as they are measured: the linear softmax cross entropy
(scoring and training) and the global gradient norm with clipping. Shapes are those of this repository's Pythia models
(hidden 512 to 2048, vocabulary 50304, its benchmark and test batches) and of its small test models."""
import math

import torch

own = False

VOCAB = 50304          # the models' (padded) vocabulary
TOKENIZER = 50277      # the ids a tokenizer of theirs produces: an odd row count


def listed():
    return [
        # scoring (loss of every token, no gradient)
        # one token: the log-probability of one continuation, where latency counts
        dict(name="score 1 bf16", op="score", n=1, d=1024, v=VOCAB, dtype="bf16", ignored=0.0),
        # 4 prompts of 128 tokens (127 predictions each) in float32 on the smallest model's width
        dict(name="score 4x127 f32", op="score", n=508, d=512, v=VOCAB, dtype="f32", ignored=0.0),
        # a padded evaluation batch: 8 sequences of 512, a quarter of the places padding
        dict(name="score 8x511 bf16 padded", op="score", n=4088, d=1024, v=VOCAB, dtype="bf16", ignored=0.25),
        # the long-context evaluation of the 1B width: 8 sequences of 2048
        dict(name="score 8x2047 bf16", op="score", n=16376, d=2048, v=VOCAB, dtype="bf16", ignored=0.0),
        # training (loss and both gradients)
        # the test model: 2 sequences of 24 tokens, hidden 128, vocabulary 1024
        dict(name="train 2x23 f32 tiny", op="train", n=46, d=128, v=1024, dtype="f32", ignored=0.0, reduction="mean"),
        # float32 training at the 410M width (what trainable models run in), answers only: a third of the tokens kept out
        dict(name="train 8x255 f32", op="train", n=2040, d=1024, v=VOCAB, dtype="f32", ignored=0.33, reduction="mean"),
        # an odd batch over the tokenizer's odd id range, each token with a weight of its own
        dict(name="train 1021 bf16 weighted", op="train", n=1021, d=768, v=TOKENIZER, dtype="bf16", ignored=0.05,
             reduction="none"),
        # bf16 training, 410M width, 8192 tokens a step
        dict(name="train 8192 bf16 d1024", op="train", n=8192, d=1024, v=VOCAB, dtype="bf16", ignored=0.0,
             reduction="mean"),
        # bf16 training, 1B width: the largest
        dict(name="train 8192 bf16 d2048", op="train", n=8192, d=2048, v=VOCAB, dtype="bf16", ignored=0.0,
             reduction="mean"),
        # clipping (gradients of a whole model into the optimizer's float32 buffer)
        # the test model's gradients: two dozen small tensors, where latency counts
        dict(name="clip tiny f32", op="clip", layers=2, d=128, ff=512, support=64, v=1024, dtype="f32", max_norm=0.5),
        # the 70M model, float32, half of each FFN's support kept
        dict(name="clip 70M f32", op="clip", layers=6, d=512, ff=2048, support=256, v=VOCAB, dtype="f32",
             max_norm=1.0),
        # the 1B model's gradients in bf16; the norm is below the limit, so the factor is one
        dict(name="clip 1B bf16", op="clip", layers=16, d=2048, ff=8192, support=410, v=VOCAB, dtype="bf16",
             max_norm=1e6),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("score", "score", "train", "train", "clip"))
    dtype = rng.choice(("bf16", "f32"))
    if op == "clip":
        d = 8 * _log_int(rng, 8, 128)
        return dict(op=op, layers=_log_int(rng, 1, 24), d=d, ff=4 * d,
                    support=rng.randint(1, d // 2), v=_log_int(rng, 500, VOCAB), dtype=dtype,
                    max_norm=rng.choice((0.1, 1.0, 1e6)))
    n = _log_int(rng, 1, 16384 if op == "score" else 8192)
    d = 8 * _log_int(rng, 8, 256)
    v = _log_int(rng, 500, 60000)
    case = dict(op=op, n=n, d=d, v=min(v, 8192 * VOCAB // n), dtype=dtype,
                ignored=rng.choice((0.0, 0.1, round(rng.uniform(0, 0.9), 3))))
    if op == "train":
        case["reduction"] = rng.choice(("mean", "sum", "none"))
    return case


def _type(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _kept(case):
    return case["n"] - int(case["n"] * case["ignored"])


def _shapes(case):
    """The gradients of a model with HFFN FFNs: embeddings, per block two norms, the attention's two projections and
    the FFN's compact arrays (support entries per neuron on both sides), the last norm and the head."""
    d, f, s, v = case["d"], case["ff"], case["support"], case["v"]
    block = [(d,)] * 4 + [(3 * d, d), (3 * d,), (d, d), (d,), (f * s,), (f,), (f * s,), (d,)]
    return [(v, d)] + block * case["layers"] + [(d,), (d,), (v, d)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _type(case)
    if case["op"] == "clip":
        shapes = _shapes(case)
        # every tensor at a scale of its own: gradients of embeddings, norms and projections differ by decades
        scales = torch.rand(len(shapes), generator=torch.Generator().manual_seed(seed))
        scales = torch.pow(10.0, -1 - 3 * scales).tolist()
        grads = [torch.randn(s, generator=g, device="cuda").mul_(k).to(dtype) for s, k in zip(shapes, scales)]
        # the optimizer's flat float32 gradient buffer; each tensor's place starts on a multiple of 64 entries
        places = [-(-x.numel() // 64) * 64 for x in grads]
        flat = torch.zeros(sum(places), device="cuda")
        views = [p[:x.numel()].view_as(x) for p, x in zip(flat.split(places), grads)]
        return dict(case=case, grads=grads, flat=flat, views=views)
    n, d, v = case["n"], case["d"], case["v"]
    # a head whose logits spread by about 2, and hidden states that lean towards their target's row by a varying
    # degree, so that some tokens are well predicted and others are not; targets are more often low ids
    weight = torch.randn(v, d, generator=g, device="cuda").mul_(2 / math.sqrt(d)).to(dtype)
    targets = (torch.rand(n, generator=g, device="cuda").pow(3) * v).long().clamp(max=v - 1)
    lean = torch.rand(n, 1, generator=g, device="cuda") * 3
    hidden = (torch.randn(n, d, generator=g, device="cuda") + lean * weight[targets].float()).to(dtype)
    skipped = torch.randperm(n, generator=g, device="cuda")[:n - _kept(case)]
    targets[skipped] = -100
    state = dict(case=case, hidden=hidden, weight=weight, targets=targets)
    if case["op"] == "train":
        hidden.requires_grad_(True)
        weight.requires_grad_(True)
        if case["reduction"] == "none":
            state["upstream"] = torch.randn(n, generator=g, device="cuda") / n
    return state


def _losses(hidden, weight, targets):
    """Plain form, float32: every token's loss and what its gradient needs."""
    keep = targets >= 0
    h, w = hidden.float(), weight.float()
    h = torch.where(keep[:, None], h, torch.zeros_like(h))
    z = h @ w.t()
    z = z - z.amax(1, keepdim=True)
    at = targets.clamp(min=0)[:, None]
    picked = z.gather(1, at).squeeze(1)
    z = z.exp_()
    total = z.sum(1)
    losses = torch.where(keep, total.log() - picked, torch.zeros_like(total))
    return losses, h, w, z, total, keep, at


def _score(state):
    return _losses(state["hidden"], state["weight"], state["targets"])[0]


def _train(state):
    reduction = state["case"]["reduction"]
    with torch.no_grad():
        losses, h, w, z, total, keep, at = _losses(state["hidden"], state["weight"], state["targets"])
        kept = keep.sum().clamp(min=1)
        if reduction == "none":
            loss, c = losses, state["upstream"]
        elif reduction == "sum":
            loss, c = losses.sum(), torch.ones_like(losses)
        else:
            loss, c = losses.sum() / kept, torch.ones_like(losses) / kept
        c = torch.where(keep, c, torch.zeros_like(c))
        g = z.mul_((c / total)[:, None])
        g.scatter_add_(1, at, -c[:, None])
        return loss, (g @ w).to(state["hidden"].dtype), (g.t() @ h).to(state["weight"].dtype)


def _clip(state):
    grads, max_norm = state["grads"], state["case"]["max_norm"]
    norm = torch.stack([x.float().square().sum() for x in grads]).sum().sqrt()
    factor = (max_norm / (norm + 1e-6)).clamp(max=1.0)
    [view.copy_(x.float() * factor) for view, x in zip(state["views"], grads)]
    return norm, state["flat"]


def run(state):
    op = state["case"]["op"]
    if not own:
        return {"score": _score, "train": _train, "clip": _clip}[op](state)
    if op == "clip":
        from hffn_b200.grad_clip import clip_grad_norm
        norm = clip_grad_norm(state["grads"], state["case"]["max_norm"], out=state["views"])
        return norm, state["flat"]
    from hffn_b200.losses import linear_cross_entropy
    hidden, weight, targets = state["hidden"], state["weight"], state["targets"]
    if op == "score":
        with torch.no_grad():
            return linear_cross_entropy(hidden, weight, targets, reduction="none")
    loss = linear_cross_entropy(hidden, weight, targets, reduction=state["case"]["reduction"])
    grad_hidden, grad_weight = torch.autograd.grad(loss, (hidden, weight), state.get("upstream"))
    return loss.detach(), grad_hidden, grad_weight


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "clip":
        entries = sum(math.prod(s) for s in _shapes(case))
        return dict(bytes=entries * (size + 4) + 4, flops=3 * entries)
    n, d, v, kept = case["n"], case["d"], case["v"], _kept(case)
    product = 2 * kept * d * v
    if case["op"] == "score":
        return dict(bytes=size * d * (kept + v) + 8 * n + 4 * n, flops=product)
    per_token = 8 * n if case["reduction"] == "none" else 4      # losses out and upstream in, or one loss
    return dict(bytes=size * d * (kept + n + 2 * v) + 8 * n + per_token, flops=3 * product)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "clip":
        norm = math.sqrt(sum(float((x.double() ** 2).sum()) for x in state["grads"]))
        factor = min(1.0, case["max_norm"] / (norm + 1e-6))
        flat = torch.zeros_like(state["flat"], dtype=torch.float64)
        at = 0
        for x in state["grads"]:
            flat[at:at + x.numel()] = x.double().reshape(-1) * factor
            at += -(-x.numel() // 64) * 64
        return norm, flat
    targets = state["targets"]
    rows = (targets != -100).nonzero().squeeze(1)
    n, d, v = case["n"], case["d"], case["v"]
    with torch.no_grad():
        h, w, t = state["hidden"].double()[rows], state["weight"].double(), targets[rows]
        logits = torch.mm(h, w.T)
        lse = torch.logsumexp(logits, 1)
        losses = torch.zeros(n, dtype=torch.float64, device="cuda")
        losses[rows] = lse - logits[torch.arange(len(rows), device="cuda"), t]
        if case["op"] == "score":
            return losses
        probabilities = logits.sub_(lse[:, None]).exp_()
        probabilities[torch.arange(len(rows), device="cuda"), t] -= 1
        if case["reduction"] == "none":
            loss, upstream = losses, state["upstream"].double()[rows]
        else:
            share = max(1, len(rows)) if case["reduction"] == "mean" else 1
            loss, upstream = losses.sum() / share, torch.full((len(rows),), 1 / share, dtype=torch.float64, device="cuda")
        probabilities *= upstream[:, None]
        grad_hidden = torch.zeros(n, d, dtype=torch.float64, device="cuda")
        grad_hidden[rows] = torch.mm(probabilities, w)
        return loss, grad_hidden, torch.mm(probabilities.T, h)
