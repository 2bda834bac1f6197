"""GPU: the global gradient norm and clipping (``hffn_b200.grad_clip``) against float64.

The norm is a float64 sum rounded once to float32 (2^-24 relative, and the square root's own rounding: 2^-23 together). The
factor is a float32 sum and division of it (3 roundings, 2^-24 each, and the norm's 2^-23), a scaled entry one more
rounding and, in bfloat16, half a step of 2^-8."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def norm64(tensors):
    return math.sqrt(sum(float((t.double() ** 2).sum()) for t in tensors))


def make(shapes, dtype, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(s, generator=g, device="cuda") * scale * 10.0 ** -(i % 4)).to(dtype)
            for i, s in enumerate(shapes)]


def check_scaled(outs, before, norm, max_norm):
    factor = min(1.0, max_norm / (norm + 1e-6))
    for out, x in zip(outs, before):
        expected = x.double() * factor
        relative = 6 * U + (2.0 ** -8 if out.dtype == torch.bfloat16 else 0.0)
        assert bool(((out.double() - expected).abs() <= relative * expected.abs() + 1e-44).all())


LISTS = [[(1,)], [(7,), (3, 5), (1,)], [(8192,), (8193,), (8191,)], [(1000, 1000), (33,), (0,), (50304, 64), (5,)],
         [(129,)] * 70, [(i + 1,) for i in range(1003)]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shapes", LISTS, ids=range(len(LISTS)))
def test_norm_and_clip(shapes, dtype):
    from hffn_b200.grad_clip import clip_grad_norm, grad_norm
    tensors = make(shapes, dtype, seed=len(shapes))
    before = [t.clone() for t in tensors]
    norm = norm64(tensors)
    for max_norm in (2 * norm, norm / 3):
        got = grad_norm(tensors)
        assert got.dtype == torch.float32 and got.shape == () and abs(float(got) - norm) <= 2 * U * norm
        again = clip_grad_norm(tensors, max_norm)
        assert torch.equal(again, got)
        if max_norm > norm + 1e-5:
            assert all(torch.equal(a, b) for a, b in zip(tensors, before))
        else:
            check_scaled(tensors, before, norm, max_norm)


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("share", [0.25, 4.0])
def test_into_other_tensors(dtype, out_dtype, share):
    from hffn_b200.grad_clip import clip_grad_norm
    tensors = make([(300, 70), (17,), (9000,), (1, 1)], dtype, seed=3)
    before = [t.clone() for t in tensors]
    arena = torch.full((300 * 70 + 17 + 9000 + 1 + 4 * 3,), 7.0, device="cuda").to(out_dtype)
    outs, at = [], 3                               # odd places in one arena, with a gap after each
    for t in tensors:
        outs.append(arena[at:at + t.numel()].view_as(t))
        at += t.numel() + 3
    norm = norm64(tensors)
    clip_grad_norm(tensors, share * norm, out=outs)
    check_scaled(outs, before, norm, share * norm)
    assert all(torch.equal(a, b) for a, b in zip(tensors, before))
    outside = torch.ones_like(arena, dtype=torch.bool)
    at = 3
    for t in tensors:
        outside[at:at + t.numel()] = False
        at += t.numel() + 3
    assert bool((arena[outside] == 7).all())


def test_mixed_types_layouts_and_places():
    from hffn_b200.grad_clip import clip_grad_norm
    a = make([(64, 33)], torch.float32, 1)[0].t()                       # a transposed gradient
    b = make([(4, 5, 6)], torch.bfloat16, 2)[0].permute(2, 0, 1)
    c = torch.randn(1001, device="cuda")[1:]                            # an odd address
    d = make([(2001,)], torch.bfloat16, 3)[0][1:]
    tensors = [a, b, c, d]
    before = [t.clone() for t in tensors]
    norm = norm64(tensors)
    assert abs(float(clip_grad_norm(tensors, norm / 2)) - norm) <= 2 * U * norm
    check_scaled(tensors, before, norm, norm / 2)


@pytest.mark.parametrize("size", [1e-30, 1e-22, 1e19, 1e30])
def test_entries_whose_squares_leave_float32(size):
    from hffn_b200.grad_clip import grad_norm
    for dtype in (torch.float32, torch.bfloat16):
        x = (torch.randn(5000, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") * size).to(dtype)
        assert abs(float(grad_norm([x])) - norm64([x])) <= 2 * U * norm64([x])


def test_long_sums():
    from hffn_b200.grad_clip import grad_norm
    x = torch.full((50_000_001,), 0.1, device="cuda")
    assert abs(float(grad_norm([x])) - norm64([x])) <= 2 * U * norm64([x])


@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_not_finite(value):
    """As torch.nn.utils.clip_grad_norm_: the factor is 0 or NaN."""
    from hffn_b200.grad_clip import clip_grad_norm
    tensors = make([(100,), (50,)], torch.float32)
    tensors[1][7] = value
    twins = [torch.nn.Parameter(t.clone()) for t in tensors]
    for p, t in zip(twins, tensors):
        p.grad = t.clone()
    theirs = torch.nn.utils.clip_grad_norm_(twins, 1.0, foreach=False)
    ours = clip_grad_norm(tensors, 1.0)
    assert bool(torch.isnan(ours) == torch.isnan(theirs)) and (bool(torch.isnan(ours)) or bool(ours == theirs))
    for t, p in zip(tensors, twins):
        assert torch.equal(torch.isnan(t), torch.isnan(p.grad))
        assert torch.equal(torch.nan_to_num(t), torch.nan_to_num(p.grad))


def test_zero_limit_zero_gradients_and_nothing():
    from hffn_b200.grad_clip import clip_grad_norm, grad_norm
    tensors = make([(100,), (50,)], torch.float32)
    clip_grad_norm(tensors, 0.0)
    assert all(bool((t == 0).all()) for t in tensors)
    assert float(clip_grad_norm(tensors, 1.0)) == 0.0 and all(bool((t == 0).all()) for t in tensors)
    assert float(grad_norm([])) == 0.0 and float(clip_grad_norm([], 1.0)) == 0.0
    empty = [torch.empty(0, device="cuda"), torch.empty(3, 0, device="cuda")]
    assert float(clip_grad_norm(empty, 1.0)) == 0.0


def test_a_tensor_alone():
    from hffn_b200.grad_clip import clip_grad_norm, grad_norm
    x = make([(30, 7)], torch.float32, 5)[0]
    before = x.clone()
    norm = norm64([x])
    assert abs(float(grad_norm(x)) - norm) <= 2 * U * norm
    clip_grad_norm(x, norm / 5)
    check_scaled([x], [before], norm, norm / 5)
    point = torch.tensor(-3.0, device="cuda")
    assert float(grad_norm(point)) == 3.0


def test_same_bits_streams_and_capture():
    from hffn_b200.grad_clip import clip_grad_norm
    tensors = make([(2000, 300), (77,), (5, 5)], torch.float32, 4)
    outs = [torch.empty_like(t) for t in tensors]
    norm = clip_grad_norm(tensors, 0.5, out=outs)
    first = [o.clone() for o in outs]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        assert torch.equal(clip_grad_norm(tensors, 0.5, out=outs), norm)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, outs))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = clip_grad_norm(tensors, 0.5, out=outs)
    for t in tensors:
        t.mul_(-3.0)
    graph.replay()
    replayed = [o.clone() for o in outs]
    assert torch.equal(clip_grad_norm(tensors, 0.5, out=outs), captured)
    assert all(torch.equal(a, b) for a, b in zip(replayed, outs))


def test_autograd_sees_the_write():
    from hffn_b200.grad_clip import clip_grad_norm
    x = torch.randn(10, device="cuda")
    w = torch.randn(10, device="cuda", requires_grad=True)
    y = (w * x).sum()
    clip_grad_norm([x], 0.1)
    with pytest.raises(RuntimeError):
        y.backward()


def test_refusals():
    from hffn_b200.grad_clip import clip_grad_norm, grad_norm
    x, y = torch.randn(100, device="cuda"), torch.randn(100, device="cuda")
    kept = x.clone()
    for bad in (lambda: grad_norm([x, x.cpu()]),
                lambda: grad_norm([x.half()]),
                lambda: grad_norm([x[::2]]),
                lambda: grad_norm([x[:1].expand(5)]),
                lambda: clip_grad_norm([x, x], 1.0),                       # the same tensor twice
                lambda: clip_grad_norm([x, x[50:]], 1.0),
                lambda: clip_grad_norm([x[:50], x[50:]], 1.0, out=[y[:50], y[49:99]]),
                lambda: clip_grad_norm([x[:50], x[50:]], 1.0, out=[x[50:], x[:50]]),
                lambda: clip_grad_norm([x[:50]], 1.0, out=[x[1:51]]),
                lambda: clip_grad_norm([x], 1.0, out=[y[:99]]),
                lambda: clip_grad_norm([x], 1.0, out=[]),
                lambda: clip_grad_norm([x], 1.0, out=[y.cpu()]),
                lambda: clip_grad_norm([x], -1.0),
                lambda: clip_grad_norm([x], float("nan"))):
        with pytest.raises(ValueError):
            bad()
    torch.cuda.synchronize()
    assert torch.equal(x, kept)
    halves = [x[:50], x[50:]]                    # neighbours in memory are no overlap
    clip_grad_norm(halves, 1e9)
    assert torch.equal(x, kept)
    assert abs(float(grad_norm([x, x])) - math.sqrt(2) * norm64([x])) <= 3 * U * 2 * norm64([x])   # reading twice is fine
