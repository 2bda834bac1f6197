"""GPU: the loss, the gradient norm, the clipping and the updates together, as a Pythia training step uses them
(``pythia.causal_lm_loss``, ``HFFNTrainRuntime.clip_grad_norm``, ``pythia.train_step``).

The loss equals the cross entropy of the model's own logits: both are float32 evaluations of the same function, each
token's logit and log sum within acc(128) = 8.6e-6 of sum |h w| (the tensor cores' accumulation, as in the loss's own
tests; the library's is closer), which the hidden states (LayerNorm: norm sqrt(128)) and the head's initialisation
(0.02) keep below 128 x 0.8 x 0.02: 4e-5 on losses of about 7. Gradients are held to the bar of the model's training
tests, 1e-4 of their scale. The step is compared bit for bit with the same calls made one by one.
"""
import copy
import math

import pytest
import torch
import torch.nn.functional as F

from hffn_b200 import pythia

pytestmark = pytest.mark.gpu

SMALL = dict(pythia.PYTHIA_410M, hidden_size=128, num_hidden_layers=2, num_attention_heads=4, intermediate_size=512,
             vocab_size=1024, max_position_embeddings=128)


@pytest.fixture(scope="module")
def tiny(tmp_path_factory):
    root = tmp_path_factory.mktemp("pythia_loss")
    pythia.make_random_pythia(root / "model", root / "export", SMALL, support=64, seed=31)
    return root


def load(tiny, **options):
    return pythia.load_pythia(tiny / "model", tiny / "export", "hffn", "cuda", trainable=True, **options)


def batch(seed=5, ignored=0.3):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, SMALL["vocab_size"], (3, 25), generator=g)
    labels = ids.clone()
    labels[torch.rand(3, 25, generator=g) < ignored] = -100
    return ids.cuda(), labels.cuda()


def logits_loss(model, ids, labels):
    logits = model(input_ids=ids).logits
    return F.cross_entropy(logits[:, :-1].reshape(-1, logits.shape[-1]), labels[:, 1:].reshape(-1))


def relative(a, b):
    return float((a.double() - b.double()).abs().max() / max(float(b.double().abs().max()), 1e-30))


def compact(model):
    train = model.hffn_train
    return [g for index in range(len(train.steps)) for g in train.gradients(index).values()]


def test_loss_and_gradients_equal_those_of_the_logits(tiny):
    ours, theirs = load(tiny), load(tiny)
    ids, labels = batch()
    loss, expected = pythia.causal_lm_loss(ours, ids, labels), logits_loss(theirs, ids, labels)
    assert abs(float(loss.detach()) - float(expected.detach())) <= 1e-4
    loss.backward()
    expected.backward()
    named = dict(theirs.named_parameters())
    compared = 0
    for name, p in ours.named_parameters():
        assert relative(p.grad, named[name].grad) <= 1e-4, name
        compared += 1
    assert compared > 10
    for a, b in zip(compact(ours), compact(theirs)):
        assert relative(a, b) <= 1e-4


@pytest.mark.parametrize("arm,dtype", [("hffn", torch.float32), ("hffn", torch.bfloat16), ("dense", torch.float32)])
def test_scoring(tiny, arm, dtype):
    """bfloat16: the model's own logits are rounded to 2^-8 of values below 2 (the fused loss's are not): 2 x 2^-8 x 2."""
    model = pythia.load_pythia(tiny / "model", tiny / "export", arm, "cuda", dtype)
    ids, labels = batch(6)
    with torch.no_grad():
        losses = pythia.causal_lm_loss(model, ids, labels, reduction="none")
        logits = model(input_ids=ids).logits.double()
    assert losses.shape == ids.shape and not losses.requires_grad
    expected = torch.zeros_like(losses, dtype=torch.float64)
    expected[:, :-1] = F.cross_entropy(logits[:, :-1].transpose(1, 2), labels[:, 1:], reduction="none")
    bound = 1e-4 if dtype == torch.float32 else 2 * 2.0 ** -8 * max(2.0, float(logits.abs().max()))
    assert float((losses.double() - expected).abs().max()) <= bound
    assert bool((losses[:, -1] == 0).all())


def test_norm_and_clipping_over_all_gradients(tiny):
    model = load(tiny)
    ids, labels = batch(7)
    pythia.causal_lm_loss(model, ids, labels).backward()
    others = [p.grad for p in model.parameters() if p.grad is not None]
    every = compact(model) + others
    before = [g.clone() for g in every]
    norm = math.sqrt(sum(float((g.double() ** 2).sum()) for g in before))
    got = model.hffn_train.clip_grad_norm(norm / 4, others)
    assert abs(float(got) - norm) <= 2.0 ** -23 * norm
    for g, b in zip(every, before):
        expected = b.double() * ((norm / 4) / (norm + 1e-6))
        assert bool(((g.double() - expected).abs() <= 6 * 2.0 ** -24 * expected.abs() + 1e-44).all())
    first = [g.clone() for g in model.hffn_train.gradients(0).values()]
    second = [g.clone() for g in model.hffn_train.gradients(1).values()]
    model.hffn_train.clip_grad_norm(1e-6, layers=[1])                      # one layer alone
    assert all(torch.equal(a, b) for a, b in zip(first, model.hffn_train.gradients(0).values()))
    assert not any(torch.equal(a, b) for a, b in zip(second, model.hffn_train.gradients(1).values()))


@pytest.mark.parametrize("max_norm", [None, 0.05])
def test_train_step_equals_its_parts(tiny, max_norm):
    whole, parts = load(tiny), load(tiny)
    optimizers = [torch.optim.AdamW(m.parameters(), lr=1e-3) for m in (whole, parts)]
    for seed in (8, 9):
        ids, labels = batch(seed)
        loss, norm = pythia.train_step(whole, optimizers[0], ids, labels, max_norm=max_norm)
        optimizers[1].zero_grad()
        expected = pythia.causal_lm_loss(parts, ids, labels)
        expected.backward()
        others = [p.grad for p in parts.parameters()]
        expected_norm = parts.hffn_train.clip_grad_norm(math.inf if max_norm is None else max_norm, others)
        if max_norm is not None:
            assert float(expected_norm) > max_norm
        optimizers[1].step()
        for index in range(SMALL["num_hidden_layers"]):
            parts.hffn_train.adamw(index)
        assert torch.equal(loss, expected.detach()) and torch.equal(norm, expected_norm)
    for a, b in zip(whole.parameters(), parts.parameters()):
        assert torch.equal(a, b)
    for index in range(SMALL["num_hidden_layers"]):
        for a, b in zip(whole.hffn_train.parameters(index).values(), parts.hffn_train.parameters(index).values()):
            assert torch.equal(a, b)
    assert whole.hffn_train.steps == [2, 2]


def test_nothing_to_train_on_changes_no_gradient(tiny):
    model = load(tiny)
    ids, labels = batch(10)
    labels = torch.full_like(labels, -100)
    pythia.causal_lm_loss(model, ids, labels).backward()
    assert float(model.hffn_train.clip_grad_norm(1.0, [p.grad for p in model.parameters()])) == 0.0


def test_refusals(tiny):
    model = load(tiny)
    ids, labels = batch(11)
    with pytest.raises(ValueError):
        pythia.causal_lm_loss(model, ids, labels[:, :-1])
    with pytest.raises(ValueError):
        pythia.causal_lm_loss(model, ids[0])
    dense = pythia.load_pythia(tiny / "model", tiny / "export", "dense", "cuda")
    with pytest.raises(ValueError):
        pythia.train_step(dense, None, ids)
    shared = model.hffn_train.gradients(0)["up_val"]
    with pytest.raises(ValueError):
        model.hffn_train.clip_grad_norm(1.0, [shared])                     # the same gradient twice
    assert copy.copy(model.hffn_train.steps) == [0, 0]


def test_no_limit_writes_no_gradient(tiny):
    """max_norm=None is the norm only: gradients that are not finite stay where they are, the others as they were."""
    whole, parts = load(tiny), load(tiny)
    ids, labels = batch(12)
    for model in (whole, parts):
        weight = model.gpt_neox.layers[0].attention.dense.weight
        weight.register_hook(lambda g: g.index_put((torch.tensor(3, device="cuda"), torch.tensor(4, device="cuda")),
                                                   torch.tensor(float("inf"), device="cuda")))
    still = torch.optim.SGD(whole.parameters(), lr=0.0)
    loss, norm = pythia.train_step(whole, still, ids, labels)
    pythia.causal_lm_loss(parts, ids, labels).backward()
    assert math.isinf(float(norm)) and math.isfinite(float(loss))
    for a, b in zip(whole.parameters(), parts.parameters()):
        assert torch.equal(a.grad, b.grad)
    for a, b in zip(compact(whole), compact(parts)):
        assert torch.equal(a, b)


def test_a_parameter_outside_the_optimizer_adds_up_nothing(tiny):
    """Every step's gradients are that step's own, whatever the optimizer holds."""
    model = load(tiny)
    held = [p for name, p in model.named_parameters() if "embed" not in name]
    optimizer = torch.optim.SGD(held, lr=0.0)
    model.hffn_train.lr = 0.0
    ids, labels = batch(13)
    _, first = pythia.train_step(model, optimizer, ids, labels)
    grads = [p.grad.clone() for p in model.parameters()]
    _, second = pythia.train_step(model, optimizer, ids, labels)
    assert torch.equal(first, second)
    assert all(torch.equal(p.grad, g) for p, g in zip(model.parameters(), grads))


def test_ffns_below_frozen_parameters_get_their_gradients(tiny):
    """An FFN whose input carries no gradient has gradients of its own all the same: none is left from an earlier step."""
    whole, frozen = load(tiny), load(tiny)
    ids, labels = batch(14)
    frozen.requires_grad_(False)
    frozen.embed_out.weight.requires_grad_(True)
    for model in (whole, frozen):
        for index in range(SMALL["num_hidden_layers"]):
            for g in model.hffn_train.gradients(index).values():
                g.fill_(7.0)
    pythia.causal_lm_loss(whole, ids, labels).backward()
    pythia.train_step(frozen, torch.optim.SGD([frozen.embed_out.weight], lr=0.0), ids, labels)
    for a, b in zip(compact(frozen), compact(whole)):
        assert torch.equal(a, b)
    assert torch.equal(frozen.embed_out.weight.grad, whole.embed_out.weight.grad)
    assert all(p.grad is None for name, p in frozen.named_parameters() if name != "embed_out.weight")
