"""GPU: the linear softmax cross entropy (``hffn_b200.losses``) against its definition in float64.

Every bound is elementwise and derived, not fitted. Notation: u = 2^-24 (half a step of float32), r the half step of
the storage type (bfloat16 2^-8; float32: the operands of the products are held as two fp16 parts, whose
representation and dropped low-by-low product are within r = 2^-20 of a product, then rounded once to float32).
- A product summed over k terms in float32 is within acc(k) = (k / 16 + 32) 2^-23 of the sum of its terms' absolute
  values (the tensor core adds 16 products at a time and truncates; one step each, and the sums within one add).
- A logit is within dz = (acc(d) + [float32: r]) sum_i |h_i w_i| of the exact one; every exponential's argument and the
  log sum are within the largest dz of a row plus rounding of a value of size |z|: e_t = 2 max_v dz + 8 u (max |z| + 1
  + log V).
- loss_t is within e_t + u (|lse| + |z|).
- g = c (p - [target]) is within |c| p (e^{e_t} - 1 + 2^-20) + r |g| (its storage) of the exact one, and a gradient
  sum_k g x is within sum_k |delta g| |x| + (acc(k) + [float32: r]) sum_k |g x| + r |result|.
- Two fp16 parts hold an entry of float32 operands (hidden states, head, c h and p - [target]) to 2^-39 of the largest
  entry of its operand at worst (the end of fp16's range), which adds that much per entry to every product.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
IGNORE = -100


def make(n, d, v, dtype, seed=0, ignored=0.0, scale=2.0, ignore_index=IGNORE):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = (torch.randn(v, d, generator=g, device="cuda") * scale / math.sqrt(d)).to(dtype)
    targets = torch.randint(0, v, (n,), generator=g, device="cuda")
    lean = torch.rand(n, 1, generator=g, device="cuda") * 3
    h = (torch.randn(n, d, generator=g, device="cuda") + lean * w[targets].float()).to(dtype)
    if ignored:
        targets[torch.rand(n, generator=g, device="cuda") < ignored] = ignore_index
    return h, w, targets


def acc(k):
    return (k / 16 + 32) * 2.0 ** -23


def reference(h, w, targets, c, ignore_index=IGNORE):
    """Losses and both gradients in float64 for upstream gradients ``c`` [n] (0 where ignored), and their bounds."""
    fp32 = h.dtype == torch.float32
    store = 2.0 ** -20 if fp32 else 2.0 ** -8
    split = 2.0 ** -20 if fp32 else 0.0
    out_r = U if fp32 else 2.0 ** -8
    n, d = h.shape
    v = w.shape[0]
    keep = targets != ignore_index
    h64 = torch.where(keep[:, None], h, torch.zeros_like(h)).double()
    w64 = w.double()
    z = h64 @ w64.T
    held = 2.0 ** -39 if fp32 else 0.0          # of the largest entry of an operand
    h_held, w_held = held * h64.abs().amax(), held * w64.abs().amax()
    dz = (acc(d) + split) * (h64.abs() @ w64.abs().T).amax(1) + h_held * w64.abs().sum(1).amax() \
        + w_held * h64.abs().sum(1)
    lse = torch.logsumexp(z, 1)
    picked = z.gather(1, targets.clamp(min=0)[:, None]).squeeze(1)
    losses = torch.where(keep, lse - picked, 0.0)
    e = 2 * dz + 8 * U * (z.abs().amax(1) + 1 + math.log(v))
    loss_bound = torch.where(keep, e + 2 * U * (lse.abs() + picked.abs()), 0.0)
    p = (z - lse[:, None]).exp()
    g = p.clone()
    g.scatter_add_(1, targets.clamp(min=0)[:, None], torch.full((n, 1), -1.0, dtype=torch.float64, device="cuda"))
    c64 = torch.where(keep, c.double(), 0.0)
    g = g * c64[:, None]
    dg = c64.abs()[:, None] * ((torch.expm1(e) + 2.0 ** -20)[:, None] * p + held) + (store + 4 * U) * g.abs()
    dg = torch.where(keep[:, None], dg, 0.0)
    dh, dw = g @ w64, g.T @ h64
    k_n = max(1, int(keep.sum()))
    dh_bound = dg @ w64.abs() + (acc(v) + split) * (g.abs() @ w64.abs()) + out_r * dh.abs()
    dh_bound += w_held * g.abs().sum(1, keepdim=True)
    dw_bound = dg.T @ h64.abs() + (acc(k_n) + split) * (g.abs().T @ h64.abs()) + out_r * dw.abs()
    ch = held * (c64[:, None] * h64).abs().amax()
    unit = torch.where(c64 == 0, 0.0, 1 / torch.where(c64 == 0, 1.0, c64.abs()))
    dw_bound += ch * (g.abs() * unit[:, None]).sum(0)[:, None]
    return (losses, loss_bound), (dh, 1.01 * dh_bound + 1e-30), (dw, 1.01 * dw_bound + 1e-30)


def within(actual, expected, what):
    value, bound = expected
    assert actual.shape == value.shape, what
    off = (actual.double() - value).abs()
    assert bool(torch.isfinite(actual).all()), what
    worst = (off / (bound + 1e-300)).max()
    assert bool((off <= bound).all()), f"{what}: {float(worst)} of the bound, off by {float(off.max())}"


def check(h, w, targets, reduction="none", seed=3, ignore_index=IGNORE):
    from hffn_b200.losses import linear_cross_entropy
    n = h.shape[0]
    kept = max(1, int((targets != ignore_index).sum()))
    if reduction == "none":
        c = torch.randn(n, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")
    else:
        c = torch.full((n,), 1.0 / kept if reduction == "mean" else 1.0, dtype=torch.float64, device="cuda")
    expected_losses, expected_dh, expected_dw = reference(h, w, targets, c, ignore_index)
    h, w = h.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = linear_cross_entropy(h, w, targets, ignore_index=ignore_index, reduction=reduction)
    assert loss.dtype == torch.float32
    dh, dw = torch.autograd.grad(loss, (h, w), c if reduction == "none" else None)
    assert dh.dtype == h.dtype and dw.dtype == w.dtype
    if reduction == "none":
        within(loss.detach(), expected_losses, "losses")
    else:
        share = kept if reduction == "mean" else 1
        total, bound = expected_losses[0].sum() / share, expected_losses[1].sum() / share
        within(loss.detach(), (total, bound + U * total.abs()), "loss")
    within(dh, expected_dh, "grad_hidden")
    within(dw, expected_dw, "grad_weight")
    with torch.no_grad():                                  # without a backward
        scored = linear_cross_entropy(h, w, targets, ignore_index=ignore_index, reduction="none")
    within(scored, expected_losses, "scored losses")
    return loss.detach(), dh, dw


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    from hffn_b200.losses import device_errors
    assert device_errors() == 0


BOTH = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
SHAPES = [(9000, 8, 300), (40, 4104, 600), (3, 8, 140001), (2, 32768, 40), (1, 8, 1), (1, 64, 2), (2, 72, 7),
          (46, 128, 1024), (31, 136, 255), (64, 64, 256), (255, 200, 257),
          (256, 512, 1000), (257, 1024, 2049), (700, 328, 4099), (1, 1024, 50304), (9, 2048, 5001), (1021, 768, 3001)]


@BOTH
@pytest.mark.parametrize("n,d,v", SHAPES)
def test_against_float64(n, d, v, dtype):
    check(*make(n, d, v, dtype, seed=n + v))


@BOTH
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 8, 9, 17, 32, 33])
@pytest.mark.parametrize("d,v", [(8, 3), (520, 1027), (2048, 700), (4096, 300)])
def test_few_rows(n, d, v, dtype):
    check(*make(n, d, v, dtype, seed=n + d, ignored=0.2))


@BOTH
@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("ignored", [0.0, 0.3])
def test_reductions(reduction, ignored, dtype):
    check(*make(190, 128, 1500, dtype, seed=5, ignored=ignored), reduction=reduction)


@BOTH
@pytest.mark.parametrize("ignored", [0.1, 0.9])
@pytest.mark.parametrize("n", [3, 256, 515])
def test_ignored_rows(n, ignored, dtype):
    h, w, t = make(n, 96, 777, dtype, seed=n, ignored=ignored)
    t[0] = IGNORE
    losses, dh, _ = check(h, w, t)
    gone = t == IGNORE
    assert bool((losses[gone] == 0).all()) and bool((dh[gone] == 0).all())


@BOTH
def test_several_pieces_of_the_vocabulary(dtype):
    """Enough tokens that g is held in several pieces (float32: from 1334 tokens of 50304 ids)."""
    check(*make(6200, 64, 50304, dtype, seed=8, ignored=0.05), reduction="mean")


@BOTH
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_every_row_ignored(reduction, dtype):
    from hffn_b200.losses import linear_cross_entropy
    h, w, t = make(300, 64, 500, dtype)
    h[:] = float("nan")
    t[:] = IGNORE
    h.requires_grad_(True), w.requires_grad_(True)
    loss = linear_cross_entropy(h, w, t, reduction=reduction)
    dh, dw = torch.autograd.grad(loss.sum(), (h, w))
    for x in (loss, dh, dw):
        assert bool((x == 0).all())


@BOTH
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf")])
def test_what_ignored_rows_hold_reaches_nothing(poison, dtype):
    h, w, t = make(333, 72, 900, dtype, seed=2, ignored=0.4)
    clean = check(h, w, t)
    h = h.clone()
    h[t == IGNORE] = poison
    dirty = check(h, w, t)
    for a, b in zip(clean, dirty):
        assert torch.equal(a, b)


@BOTH
def test_a_row_that_is_not_finite_stays_alone(dtype):
    from hffn_b200.losses import linear_cross_entropy
    h, w, t = make(40, 64, 300, dtype, seed=4)
    h = h.clone()
    h[7, 3] = float("nan")
    h[20, 0] = float("inf")
    h.requires_grad_(True)
    losses = linear_cross_entropy(h, w, t, reduction="none")
    (dh,) = torch.autograd.grad(losses.sum(), h)
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[[7, 20]] = True
    assert not bool(torch.isfinite(losses[bad]).any())
    assert bool(torch.isfinite(losses[~bad]).all()) and bool(torch.isfinite(dh[~bad]).all())
    expected = reference(h.detach()[~bad], w, t[~bad], torch.ones(38, device="cuda"))
    within(losses.detach()[~bad], expected[0], "losses")
    within(dh[~bad], expected[1], "grad_hidden")


@BOTH
def test_targets_out_of_range_give_nan_and_no_gradient(dtype):
    from hffn_b200.losses import linear_cross_entropy
    h, w, t = make(50, 64, 300, dtype, seed=6)
    t[3], t[11], t[49] = 300, -1, 2 ** 40
    bad = torch.zeros(50, dtype=torch.bool, device="cuda")
    bad[[3, 11, 49]] = True
    h.requires_grad_(True), w.requires_grad_(True)
    losses = linear_cross_entropy(h, w, t, reduction="none")
    dh, dw = torch.autograd.grad(losses, (h, w), torch.ones_like(losses))
    assert bool(torch.isnan(losses[bad]).all()) and bool((dh[bad] == 0).all())
    expected = reference(h.detach()[~bad], w.detach(), t[~bad], torch.ones(47, device="cuda"))
    within(losses.detach()[~bad], expected[0], "losses")
    within(dh[~bad], expected[1], "grad_hidden")
    within(dw, expected[2], "grad_weight")
    assert bool(torch.isnan(linear_cross_entropy(h, w, t)))


@BOTH
def test_ignore_index_can_be_an_id(dtype):
    h, w, t = make(120, 64, 50, dtype, seed=7)
    check(h, w, t, ignore_index=int(t[5]))


@BOTH
@pytest.mark.parametrize("size", [1e-6, 40.0, 3000.0])
def test_logits_of_every_size(size, dtype):
    h, w, t = make(60, 128, 700, dtype, seed=9, scale=size)
    h = torch.randn(60, 128, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    check(h, w, t)


@BOTH
@pytest.mark.parametrize("h_size,w_size", [(0.0, 1.0), (1.0, 0.0), (0.0, 0.0), (1e-25, 1e-25), (1e25, 1e-25),
                                           (1e-25, 1e25)])
def test_operands_of_every_size(h_size, w_size, dtype):
    h, w, t = make(60, 128, 700, dtype, seed=27)
    check((h.float() * h_size).to(dtype), (w.float() * w_size).to(dtype), t)


@BOTH
def test_rows_of_very_different_sizes(dtype):
    """Hidden rows, head rows and upstream gradients over several decades."""
    h, w, t = make(130, 128, 600, dtype, seed=10)
    g = torch.Generator(device="cuda").manual_seed(2)
    w = (w.float() * torch.pow(10.0, -3 * torch.rand(600, 1, generator=g, device="cuda"))).to(dtype)
    h = (h.float() * torch.pow(10.0, 2 - 4 * torch.rand(130, 1, generator=g, device="cuda"))).to(dtype)
    h[5] = 0
    w[17] = 0
    check(h, w, t)


@BOTH
def test_shapes_and_strides(dtype):
    from hffn_b200.losses import linear_cross_entropy
    h, w, t = make(6 * 33, 64, 500, dtype, seed=11)
    plain = linear_cross_entropy(h, w, t, reduction="none")
    wide = torch.full((6 * 33, 80), float("nan"), dtype=dtype, device="cuda")
    wide[:, 8:72] = h
    assert torch.equal(linear_cross_entropy(wide[:, 8:72], w, t, reduction="none"), plain)          # a row stride
    odd = torch.zeros(6 * 33 * 64 + 1, dtype=dtype, device="cuda")[1:].view(-1, 64).copy_(h)         # odd address
    assert torch.equal(linear_cross_entropy(odd, w, t, reduction="none"), plain)
    turned = h.t().contiguous().t()                                                                  # inner stride
    assert torch.equal(linear_cross_entropy(turned, w, t, reduction="none"), plain)
    cube, ids = h.view(6, 33, 64), t.view(6, 33)
    shifted = linear_cross_entropy(cube[:, :-1], w, ids[:, 1:], reduction="none")
    assert shifted.shape == (6, 32)
    same = linear_cross_entropy(cube[:, :-1].reshape(-1, 64), w, ids[:, 1:].reshape(-1), reduction="none")
    assert torch.equal(shifted.reshape(-1), same)
    one = linear_cross_entropy(h[3], w, t[3], reduction="none")                                      # a single token
    assert one.shape == () and abs(float(one - plain[3])) <= 1e-5 * float(plain[3])
    repeated = linear_cross_entropy(h[:1].expand(5, 64), w, t[:1].expand(5), reduction="none")       # no stride
    assert torch.equal(repeated, linear_cross_entropy(h[:1].repeat(5, 1), w, t[:1].repeat(5), reduction="none"))


@BOTH
def test_a_broadcast_row_collects_every_gradient(dtype):
    from hffn_b200.losses import linear_cross_entropy
    h, w, t = make(20, 64, 300, dtype, seed=12)
    row = h[:1].clone().requires_grad_(True)
    (collected,) = torch.autograd.grad(linear_cross_entropy(row.expand(20, 64), w, t, reduction="sum"), row)
    rows = h[:1].repeat(20, 1).requires_grad_(True)
    (each,) = torch.autograd.grad(linear_cross_entropy(rows, w, t, reduction="sum"), rows)
    assert torch.equal(collected, each.sum(0, keepdim=True))


@BOTH
def test_one_gradient_alone(dtype):
    from hffn_b200.losses import linear_cross_entropy
    h, w, t = make(77, 64, 400, dtype, seed=13)
    hg, wg = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    both = torch.autograd.grad(linear_cross_entropy(hg, wg, t), (hg, wg))
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(hg, w, t), hg)[0], both[0])
    assert torch.equal(torch.autograd.grad(linear_cross_entropy(h, wg, t), wg)[0], both[1])


@BOTH
def test_same_bits_on_every_call(dtype):
    h, w, t = make(600, 256, 9000, dtype, seed=14, ignored=0.1)
    first = check(h, w, t)
    for _ in range(2):
        for a, b in zip(first, check(h, w, t)):
            assert torch.equal(a, b)


def test_gradients_against_differences():
    """A directional derivative of the summed loss in float32 by central differences: the loss is within its own bound
    at both ends (divided by the step), and the third derivative of a log sum of exponentials along a direction that
    moves the logits by at most R per unit is at most (2 R)^3 per row."""
    from hffn_b200.losses import linear_cross_entropy
    h, w, t = make(24, 64, 200, torch.float32, seed=15)
    g = torch.Generator(device="cuda").manual_seed(3)
    uh, uw = torch.randn(24, 64, generator=g, device="cuda"), torch.randn(200, 64, generator=g, device="cuda") / 8
    hg, wg = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dh, dw = torch.autograd.grad(linear_cross_entropy(hg, wg, t, reduction="sum"), (hg, wg))
    for direction, grad, at in ((uh, dh, 0), (uw, dw, 1)):
        step = 2.0 ** -7
        ends, bound = [], 0.0
        for sign in (1, -1):
            hh, ww = (h + sign * step * direction, w) if at == 0 else (h, w + sign * step * direction)
            ends.append(linear_cross_entropy(hh, ww, t, reduction="none").double().sum())
            bound += float(reference(hh, ww, t, torch.ones(24, device="cuda"))[0][1].sum())
        moved = (direction.double() @ w.double().T) if at == 0 else (h.double() @ direction.double().T)
        curvature = float((2 * moved.abs().amax(1)).pow(3).sum()) * step ** 2 / 6
        # perturbed inputs are rounded to float32 once: half a step of entries below 16
        rounding = 16 * U * float(grad.double().abs().sum()) / step
        slope = float((ends[0] - ends[1]) / (2 * step))
        assert abs(slope - float((grad.double() * direction.double()).sum())) <= bound / (2 * step) + curvature + rounding


@BOTH
def test_another_stream_and_two_at_once(dtype):
    from hffn_b200.losses import linear_cross_entropy
    a, b = make(500, 128, 3000, dtype, seed=16), make(333, 64, 5000, dtype, seed=17, ignored=0.2)

    def grads(case):
        h, w = case[0].detach().requires_grad_(True), case[1].detach().requires_grad_(True)
        loss = linear_cross_entropy(h, w, case[2])
        return (loss.detach(), *torch.autograd.grad(loss, (h, w)))

    expected = [grads(a), grads(b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        results = []
        for stream, case in zip(streams, (a, b)):
            with torch.cuda.stream(stream):
                results.append(grads(case))
        torch.cuda.synchronize()
        for got, want in zip(results, expected):
            assert all(torch.equal(x, y) for x, y in zip(got, want))


@BOTH
@pytest.mark.parametrize("through_autograd", [False, True])
@pytest.mark.parametrize("n", [1, 12, 400])
def test_captured_and_replayed(n, through_autograd, dtype):
    """A captured loss with its gradients, replayed on other inputs with another number of kept rows, two graphs in
    turn. Outside autograd also while an eager graph of the same leaves lives."""
    from hffn_b200.losses import linear_cross_entropy, linear_cross_entropy_gradients
    h, w, t = make(n, 128, 2000, dtype, seed=18, ignored=0.1)
    h, w = h.requires_grad_(True), w.requires_grad_(True)
    eager = None if through_autograd else linear_cross_entropy(h, w, t)

    def step(reduction):
        if not through_autograd:
            return linear_cross_entropy_gradients(h, w, t, reduction=reduction)
        loss = linear_cross_entropy(h, w, t, reduction=reduction)
        return (loss.detach(), *torch.autograd.grad(loss, (h, w)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step("mean"), step("sum")
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for reduction in ("mean", "sum"):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(reduction))
        graphs.append(graph)
    for seed, ignored in ((19, 0.6), (20, 0.0), (21, 1.0)):
        h2, w2, t2 = make(n, 128, 2000, dtype, seed=seed, ignored=ignored)
        with torch.no_grad():
            h.copy_(h2), w.copy_(w2), t.copy_(t2)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for reduction, got in zip(("mean", "sum"), outs):
            assert all(torch.equal(x, y) for x, y in zip(got, step(reduction)))
    assert eager is None or bool(torch.isfinite(eager))


@BOTH
def test_gradients_outside_autograd(dtype):
    from hffn_b200.losses import linear_cross_entropy_gradients
    h, w, t = make(96, 64, 700, dtype, seed=22, ignored=0.2)
    c = torch.randn(96, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    for a, b in zip(check(h, w, t), linear_cross_entropy_gradients(h, w, t, c, reduction="none")):
        assert torch.equal(a, b)
    cube = linear_cross_entropy_gradients(h.view(4, 24, 64), w, t.view(4, 24))
    assert cube[1].shape == (4, 24, 64) and cube[0].shape == ()
    for a, b in zip(check(h, w, t, "mean"), cube):
        assert torch.equal(a, b.view(a.shape))
    with pytest.raises(ValueError):
        linear_cross_entropy_gradients(h, w, t, c[:5], reduction="none")
    with pytest.raises(ValueError):
        linear_cross_entropy_gradients(h, w, t, c)


@pytest.mark.parametrize("n", [1, 20])
def test_offsets_past_32_bits(n):
    """A head of 2.2e9 entries: the losses against float32 sums over the head in stretches (whose own errors are far
    below the bound), and the last rows of its gradient, where the targets lie."""
    from hffn_b200.losses import linear_cross_entropy
    v, d = 1_060_003, 2056
    g = torch.Generator(device="cuda").manual_seed(24)
    w = torch.empty(v, d, dtype=torch.bfloat16, device="cuda").normal_(0, 2 / math.sqrt(d), generator=g)
    h = torch.randn(n, d, generator=g, device="cuda").bfloat16()
    t = torch.arange(v - n, v, device="cuda")
    z = torch.cat([h.double() @ part.double().T for part in w.split(100_000)], 1)
    lse = torch.logsumexp(z, 1)
    dz = acc(d) * max(float((h.double().abs() @ part.double().abs().T).max()) for part in w.split(100_000))
    e = 2 * dz + 8 * U * (float(z.abs().max()) + 1 + math.log(v))
    h.requires_grad_(True), w.requires_grad_(True)
    losses = linear_cross_entropy(h, w, t, reduction="none")
    expected = lse - z[torch.arange(n), t]
    assert float((losses.detach().double() - expected).abs().max()) <= e + 2 * U * float(lse.max() + z.abs().max())
    dh, dw = torch.autograd.grad(losses.sum(), (h, w))
    h, w = h.detach(), w.detach()
    p = (z[:, -1000:] - lse[:, None]).exp()
    p[torch.arange(n), t - (v - 1000)] -= 1
    exact = p.T @ h.double()
    bound = (2 * 2.0 ** -8 + 2 * math.expm1(e)) * (p.abs().T @ h.double().abs()) + 1e-30
    assert bool(((dw[-1000:].double() - exact).abs() <= bound).all())
    assert bool(torch.isfinite(dw[:: 1000]).all()) and bool(torch.isfinite(dh).all())
    del z, dw
    torch.cuda.empty_cache()


@BOTH
def test_one_token_of_every_kind(dtype):
    from hffn_b200.losses import linear_cross_entropy
    h, w, t = make(1, 64, 300, dtype, seed=25)
    check(h, w, t)
    for bad, expected in ((IGNORE, 0.0), (300, math.nan), (-7, math.nan)):
        hg, wg = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
        for reduction in ("none", "mean", "sum"):
            loss = linear_cross_entropy(hg, wg, torch.full_like(t, bad), reduction=reduction)
            dh, dw = torch.autograd.grad(loss.sum(), (hg, wg))
            assert bool((dh == 0).all()) and bool((dw == 0).all())
            assert bool(torch.isnan(loss).all()) if math.isnan(expected) else bool((loss == expected).all())
    h[0, 3] = float("inf")
    assert not bool(torch.isfinite(linear_cross_entropy(h, w, t)))


@BOTH
def test_two_backwards_of_one_forward(dtype):
    from hffn_b200.losses import linear_cross_entropy
    for n in (3, 70):
        h, w, t = make(n, 64, 900, dtype, seed=26)
        h.requires_grad_(True), w.requires_grad_(True)
        loss = linear_cross_entropy(h, w, t)
        first = torch.autograd.grad(loss, (h, w), retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(loss, (h, w))))


def test_second_derivatives_are_refused():
    from hffn_b200.losses import linear_cross_entropy
    h, w, t = make(20, 64, 300, torch.float32)
    h.requires_grad_(True)
    (dh,) = torch.autograd.grad(linear_cross_entropy(h, w, t), h, create_graph=True)
    with pytest.raises(RuntimeError):
        dh.sum().backward()


def test_from_a_thread_that_has_made_no_cuda_call():
    import threading
    from hffn_b200.losses import linear_cross_entropy_gradients
    h, w, t = make(50, 64, 300, torch.float32, seed=23)
    expected, got = linear_cross_entropy_gradients(h, w, t), []
    thread = threading.Thread(target=lambda: got.extend(linear_cross_entropy_gradients(h, w, t)))
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert len(got) == 3 and all(torch.equal(a, b) for a, b in zip(expected, got))


def test_a_weight_changed_before_the_backward_is_noticed():
    from hffn_b200.losses import linear_cross_entropy
    h, w, t = make(20, 64, 300, torch.float32)
    h.requires_grad_(True)
    loss = linear_cross_entropy(h, w, t)
    w.add_(1.0)
    with pytest.raises(RuntimeError):
        loss.backward()


def test_refusals():
    from hffn_b200.losses import linear_cross_entropy
    h, w, t = make(20, 64, 300, torch.float32)
    for bad in (lambda: linear_cross_entropy(h, w, t, reduction="avg"),
                lambda: linear_cross_entropy(h.half(), w.half(), t),
                lambda: linear_cross_entropy(h.bfloat16(), w, t),
                lambda: linear_cross_entropy(h, w, t.int()),
                lambda: linear_cross_entropy(h, w, t.cpu()),
                lambda: linear_cross_entropy(h, w, t[:19]),
                lambda: linear_cross_entropy(h[:, :60], w[:, :60].contiguous(), t),
                lambda: linear_cross_entropy(h[:, :56], w[:, :56], t),
                lambda: linear_cross_entropy(h, torch.zeros(300 * 64 + 1, device="cuda")[1:].view(300, 64), t),
                lambda: linear_cross_entropy(torch.zeros(20, 32776, device="cuda"), torch.zeros(3, 32776, device="cuda"), t),
                lambda: linear_cross_entropy(h, w[:0], t),
                lambda: linear_cross_entropy(h[:0], w, t[:0])):
        with pytest.raises(ValueError):
            bad()


@BOTH
@pytest.mark.parametrize("n", [1, 2, 8, 16, 17])
@pytest.mark.parametrize("row", [0, 1, 777, 5002])
def test_a_head_row_that_is_not_a_number_reaches_every_loss(row, n, dtype):
    """Whatever kernel the number of tokens takes, and whichever lane comes upon the row first."""
    from hffn_b200.losses import linear_cross_entropy
    h, w, t = make(n, 64, 5003, dtype, seed=28)
    w, t = w.clone(), torch.full_like(t, 5)
    w[row, 9] = float("nan")
    assert bool(torch.isnan(linear_cross_entropy(h, w, t, reduction="none")).all())
    h.requires_grad_(True)
    losses = linear_cross_entropy(h, w, t, reduction="none")
    (dh,) = torch.autograd.grad(losses.sum(), h)
    assert bool(torch.isnan(losses).all()) and bool(torch.isnan(dh).any(1).all())


@BOTH
@pytest.mark.parametrize("n", [1, 12, 70])
@pytest.mark.parametrize("size", [1e-3, 1e-4, 1e-5, 1e-7])
def test_well_predicted_tokens(size, n, dtype):
    """Losses of about `size` at a target's logit of 20 to 40: p - 1 is a small difference, of which every digit counts.
    With the odds o = sum_{v != target} exp(z_v - z_target), loss = log(1 + o) and g_target = -o / (1 + o); every
    difference of two logits is within 2 dz of the exact one (dz: of the largest logit's terms, since all of K may stay in
    one accumulator in the backward), so o, the loss and every entry of g are within expm1(2 dz) of themselves, plus at
    most 2^-18 of float32's own roundings (exponents' arguments of at most 64 are within 2^-18 of exact; sums and
    functions are far closer), plus the storage of g and of the result."""
    from hffn_b200.losses import linear_cross_entropy
    d, v = 2048, 5000
    g = torch.Generator(device="cuda").manual_seed(29)
    w = (torch.randn(v, d, generator=g, device="cuda") / math.sqrt(d)).to(dtype)
    t = torch.randint(0, v, (n,), generator=g, device="cuda")
    noise = torch.randn(n, d, generator=g, device="cuda")
    # about (log V + 1/2 - log size) / |w_t|^2 of the target's row: the odds come out near `size`
    h = (noise + (math.log(v) + 0.5 - math.log(size)) * w[t].float()).to(dtype)
    z = h.double() @ w.double().T
    at = t[:, None]
    difference = z - z.gather(1, at)
    odds = difference.exp().scatter(1, at, 0.0).sum(1)
    assert float(odds.max()) < 100 * size and float(z.gather(1, at).min()) > 8
    fp32 = dtype == torch.float32
    dz = (acc(d) + (2.0 ** -20 if fp32 else 0.0)) * (h.double().abs() @ w.double().abs().T).amax(1)
    relative = torch.expm1(2 * dz) + 2.0 ** -18
    exact = torch.log1p(odds)
    h.requires_grad_(True), w.requires_grad_(True)
    losses = linear_cross_entropy(h, w, t, reduction="none")
    assert bool(((losses.detach().double() - exact).abs() <= relative * exact).all())
    with torch.no_grad():
        scored = linear_cross_entropy(h, w, t, reduction="none")
    assert bool(((scored.double() - exact).abs() <= relative * exact).all())
    dh, dw = torch.autograd.grad(losses.sum(), (h, w))
    h, w = h.detach().double(), w.detach().double()
    p = difference.exp() / (1 + odds)[:, None]
    p.scatter_(1, at, -(odds / (1 + odds))[:, None])
    held = 2.0 ** -39 if fp32 else 0.0
    dg = p.abs() * (2 * relative + (2.0 ** -20 if fp32 else 2.0 ** -8))[:, None] + held
    r = U if fp32 else 2.0 ** -8
    split = 2.0 ** -20 if fp32 else 0.0
    for got, want, bound in (
            (dh, p @ w, dg @ w.abs() + (acc(v) + split) * (p.abs() @ w.abs())
             + held * w.abs().amax() * p.abs().sum(1)[:, None]),
            (dw, p.T @ h, dg.T @ h.abs() + (acc(n) + split) * (p.abs().T @ h.abs())
             + held * h.abs().amax() * p.abs().sum(0)[:, None])):
        assert bool(((got.double() - want).abs() <= 1.01 * (bound + r * want.abs()) + 1e-30).all())


@pytest.mark.parametrize("size", [1e6, 1e12, 1e20, 3e38])
@pytest.mark.parametrize("n", [20, 300])
def test_a_huge_hidden_row_leaves_the_others_alone(n, size):
    """float32: one kept row of any finite size changes nothing of the other tokens' losses and of their rows of
    grad_hidden, scoring and training alike."""
    from hffn_b200.losses import linear_cross_entropy
    h, w, t = make(n, 128, 900, torch.float32, seed=30)
    others = torch.arange(n, device="cuda") != 7
    huge = h.clone()
    huge[7] = torch.sign(h[7]) * size * torch.rand(128, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    expected = reference(h, w, t, others.float())
    for hidden in (h, huge):
        scored = linear_cross_entropy(hidden, w, t, reduction="none")
        hidden = hidden.detach().requires_grad_(True)
        losses = linear_cross_entropy(hidden, w, t, reduction="none")
        (dh,) = torch.autograd.grad(losses, hidden, others.float())
        for got in (scored, losses.detach()):
            within(got[others], [x[others] for x in expected[0]], "losses")
        within(dh[others], [x[others] for x in expected[1]], "grad_hidden")


@pytest.mark.parametrize("size", [1e6, 1e12, 1e20, -float(torch.finfo(torch.float32).min) / 2])
@pytest.mark.parametrize("n", [5, 20, 300])
def test_a_huge_head_row_leaves_the_losses_alone(n, size):
    """float32: an id that its row puts far out of reach (its logits are of -`size`) changes no loss, scoring and training
    alike, nor the other rows of grad_weight."""
    from hffn_b200.losses import linear_cross_entropy
    h, w, t = make(n, 128, 900, torch.float32, seed=31)
    h, w, t = h.clone(), w.clone(), torch.where(t == 400, 401, t)
    h[:, 5] = 1.0 + h[:, 5].abs()
    others = torch.arange(900, device="cuda") != 400
    w[400] = 0
    w[400, 5] = -1.0
    w[400] *= size
    rest = w[others].contiguous()
    expected = reference(h, rest, t - (t > 400).long(), torch.ones(n, device="cuda"))
    with torch.no_grad():
        within(linear_cross_entropy(h, w, t, reduction="none"), expected[0], "scored losses")
    w.requires_grad_(True)
    losses = linear_cross_entropy(h, w, t, reduction="none")
    (dw,) = torch.autograd.grad(losses.sum(), w)
    within(losses.detach(), expected[0], "losses")
    within(dw[others], expected[2], "grad_weight")
    assert bool((dw[400] == 0).all())


@BOTH
@pytest.mark.parametrize("of", ["hidden", "weight"])
def test_forward_mode_derivatives_are_refused(of, dtype):
    """A tangent is never dropped without a word, with or without gradients."""
    import torch.autograd.forward_ad as forward_ad
    from hffn_b200.losses import linear_cross_entropy, linear_cross_entropy_gradients
    h, w, t = make(20, 64, 300, dtype)
    plain = linear_cross_entropy(h, w, t)
    for grads in (False, True):
        with forward_ad.dual_level(), torch.set_grad_enabled(grads):
            assert torch.equal(linear_cross_entropy(h, w, t), plain)            # no tangent: as ever
            hh = forward_ad.make_dual(h, torch.ones_like(h)) if of == "hidden" else h
            ww = forward_ad.make_dual(w, torch.ones_like(w)) if of == "weight" else w
            with pytest.raises(ValueError):
                linear_cross_entropy(hh, ww, t)
            with pytest.raises(ValueError):
                linear_cross_entropy_gradients(hh, ww, t)


def test_one_token_takes_little_memory():
    """float32, a few tokens: the head is read as it is, so nothing of its size is allocated for a loss, and nothing of it
    is kept for the backward."""
    from hffn_b200.losses import linear_cross_entropy
    h, w, t = make(4, 1024, 20000, torch.float32, seed=32)
    linear_cross_entropy(h, w, t)
    torch.cuda.synchronize()
    for hidden in (h, h.detach().requires_grad_(True)):
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        loss = linear_cross_entropy(hidden, w, t)
        assert torch.cuda.max_memory_allocated() - before < w.numel()
        del loss


@BOTH
@pytest.mark.parametrize("wanted", [(True, True), (True, False), (False, True)])
def test_no_gradient_from_a_wait_that_ran_out(wanted, dtype):
    """A kernel whose wait runs out marks its call's state and leaves its tiles; the gradients are then NaN, not what the
    tiles hold. The mark (the fifth word of the state) is set by hand here."""
    from hffn_b200.losses import _backward, _forward
    h, w, t = make(90, 64, 700, dtype, seed=33, ignored=0.2)
    loss, state = _forward(h, w, t, IGNORE, "mean")
    c = torch.ones_like(loss)
    assert all(x is None or bool(torch.isfinite(x).all()) for x in _backward(w, state, 90, "mean", c, *wanted))
    state[16:20].view(torch.int32).fill_(1)
    dh, dw = _backward(w, state, 90, "mean", c, *wanted)
    assert (dh is not None, dw is not None) == wanted
    assert dh is None or torch.equal(torch.isnan(dh).all(1), t != IGNORE) and bool((dh[t == IGNORE] == 0).all())
    assert dw is None or bool(torch.isnan(dw).all())
    again, state = _forward(h, w, t, IGNORE, "mean")
    assert torch.equal(again, loss) and bool(torch.isfinite(_backward(w, state, 90, "mean", c)[1]).all())


@BOTH
@pytest.mark.parametrize("h_size,w_size", [(1e-37, 1e36), (1e36, 1e-37), (1e-30, 1e35), (1e35, 1e-30)])
def test_operands_at_the_ends_of_float32(h_size, w_size, dtype):
    """Ordinary logits of operands whose own scales leave float32 when either is applied before the other."""
    from hffn_b200.losses import linear_cross_entropy
    h, w, t = make(60, 128, 700, dtype, seed=34)
    h, w = (h.float() * h_size).to(dtype), (w.float() * w_size).to(dtype)
    h64, w64 = h.double(), w.double()
    z = h64 @ w64.T
    # an entry at 2^-126 and below keeps fewer bits than 22: a scale is at most 2^110, which leaves it to 2^-25 / 2^110
    held = 2.0 ** -135 if dtype == torch.float32 else 0.0
    dz = ((acc(128) + 2.0 ** -20) * (h64.abs() @ w64.abs().T) + held * w64.abs().sum(1) + held * h64.abs().sum(1)[:, None])
    e = 2 * dz.amax(1) + 8 * U * (z.abs().amax(1) + 1 + math.log(700))
    exact = torch.logsumexp(z, 1) - z.gather(1, t[:, None]).squeeze(1)
    bound = e + 2 * U * (z.abs().amax(1) * 2 + math.log(700))
    with torch.no_grad():
        within(linear_cross_entropy(h, w, t, reduction="none"), (exact, bound), "scored losses")
    h.requires_grad_(True)
    losses = linear_cross_entropy(h, w, t, reduction="none")
    within(losses.detach(), (exact, bound), "losses")
    (dh,) = torch.autograd.grad(losses.sum(), h)
    p = torch.softmax(z, 1).scatter_add(1, t[:, None], torch.full((60, 1), -1.0, dtype=torch.float64, device="cuda"))
    r = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -20
    size = p.abs() @ w64.abs()
    limit = size * (2 * r + 2 * float(torch.expm1(e).max()) + acc(700)) + 2.0 ** -38 * w64.abs().sum(0)
    assert bool(((dh.double() - p @ w64).abs() <= 1.01 * limit + 1e-37).all())
