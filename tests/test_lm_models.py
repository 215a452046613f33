"""The language models on the framework's operators (``fused=True``), as a training step uses them together:
embedding, residual norms, backward, exchange, clipped update."""
import copy

import pytest
import torch
import torch.nn.functional as F

import lm_oracle as O
from grace_amd import grace_from_params
from grace_amd.models.bert import BertMLM
from grace_amd.models.lstm import LSTMLM
from grace_amd.parallel import DistributedOptimizer, FusedSGD, clip_grad_norm_
from grace_amd.utils.workloads import WORKLOADS, build_model

BERT = dict(vocab=211, d=72, layers=2, heads=4, ff=96, max_pos=24, p=0.0)
LSTM = dict(vocab=97, emb=50, hidden=50, layers=2, dropout=0.0)


def _models(kind):
    """(unfused, fused) with the same weights, and a batch"""
    made = []
    for fused in (False, True):
        torch.manual_seed(0)
        made.append(BertMLM(**BERT, fused=fused) if kind == "bert" else LSTMLM(**LSTM, fused=fused))
    a, b = made
    assert list(a.state_dict()) == list(b.state_dict())
    for x, y in zip(a.state_dict().values(), b.state_dict().values()):
        assert torch.equal(x, y)
    g = torch.Generator().manual_seed(1)
    vocab = BERT["vocab"] if kind == "bert" else LSTM["vocab"]
    ids = torch.randint(0, vocab, (5, 23), generator=g)
    ids[torch.rand(5, 23, generator=g) < 0.3] = 7  # one token fills a third of the batch
    labels = torch.randint(0, vocab, (5, 23), generator=g)
    return a, b, ids, labels


def _loss(model, ids, labels):
    out = model(ids)
    out = out[0] if isinstance(out, tuple) else out
    return F.cross_entropy(out.reshape(-1, out.shape[-1]), labels.reshape(-1))


def _grads(model, ids, labels):
    model.zero_grad(set_to_none=True)
    loss = _loss(model, ids, labels)
    loss.backward()
    return loss.detach(), {n: p.grad.detach().clone() for n, p in model.named_parameters()}


def _check(fused, plain, exact):
    """No further from fp64 than twice what torch's own operators are (both in fp32), plus 64 roundings."""
    (fl, fg), (pl, pg), (el, eg) = fused, plain, exact
    assert abs(float(fl) - float(el)) <= 2 * abs(float(pl) - float(el)) + 64 * O.U * abs(float(el))
    for n, e in eg.items():
        size = float(e.norm())
        own, ref = (float((g[n].double().cpu() - e).norm()) for g in (fg, pg))
        assert own <= 2 * ref + 64 * O.U * size, (n, own, ref, size)


@pytest.mark.parametrize("kind", ["bert", "lstm"])
def test_fused_model_cpu(kind):
    a, b, ids, labels = _models(kind)
    exact = _grads(copy.deepcopy(a).double(), ids, labels)
    _check(_grads(b, ids, labels), _grads(a, ids, labels), exact)


def test_build_model_lm_ops():
    with pytest.raises(ValueError):
        build_model(WORKLOADS["resnet18_cifar_none"], torch.device("cpu"), "fused")
    with pytest.raises(ValueError):
        build_model(WORKLOADS["lstm_none"], torch.device("cpu"), "fast")
    m = build_model(WORKLOADS["lstm_none"], torch.device("cpu"), "fused")
    assert type(m.encoder).__name__ == "ScaledEmbedding"


def test_clip_with_the_engine_cpu():
    """synchronize, clip, step: the update of the clipped mean gradient, as FusedSGD's own clipping gives it."""
    steps = []
    for inside in (False, True):
        _, model, ids, labels = _models("lstm")
        opt = DistributedOptimizer(FusedSGD(model.parameters(), lr=0.5, max_grad_norm=0.1 if inside else None),
                                   grace_from_params({"compressor": "none", "memory": "none",
                                                      "communicator": "allreduce", "world_size": 1}),
                                   named_parameters=model.named_parameters())
        for _ in range(2):
            opt.zero_grad()
            _loss(model, ids, labels).backward()
            if inside:
                opt.step()
            else:
                opt.synchronize()
                clip_grad_norm_(model.parameters(), 0.1)
                with opt.skip_synchronize():
                    opt.step()
        steps.append([p.detach().clone() for p in model.parameters()])
    for x, y in zip(*steps):
        torch.testing.assert_close(x, y, rtol=1e-6, atol=1e-7)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bert", "lstm"])
def test_fused_model_gpu(kind):
    a, b, ids, labels = _models(kind)
    exact = _grads(copy.deepcopy(a).double(), ids, labels)
    ids, labels = ids.cuda(), labels.cuda()
    _check(_grads(b.cuda(), ids, labels), _grads(a.cuda(), ids, labels), exact)


@pytest.mark.gpu
def test_fused_bert_keeps_the_stream_under_autocast():
    _, b, ids, _ = _models("bert")
    b = b.cuda().train()
    seen = []
    for layer in b.layers:
        layer.ln2.register_forward_hook(lambda m, i, o: seen.append(o.dtype))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        b(ids.cuda())
    assert seen == [torch.float32] * 2


@pytest.mark.gpu
def test_training_steps_gpu():
    """Three steps of the fused encoder through the engine with clipping, against the unfused one with torch's
    clipping and SGD in fp64."""
    a, b, ids, labels = _models("bert")
    a = a.double()
    b = b.cuda()
    oa = torch.optim.SGD(a.parameters(), lr=0.5, momentum=0.9)
    ob = DistributedOptimizer(FusedSGD(b.parameters(), lr=0.5, momentum=0.9, max_grad_norm=0.3),
                              grace_from_params({"compressor": "none", "memory": "none", "communicator": "allreduce",
                                                 "world_size": 1}), named_parameters=b.named_parameters())
    start = [p.detach().clone() for p in a.parameters()]
    for _ in range(3):
        oa.zero_grad()
        _loss(a, ids, labels).backward()
        n = torch.nn.utils.clip_grad_norm_(a.parameters(), 0.3)
        oa.step()
        ob.zero_grad()
        _loss(b, ids.cuda(), labels.cuda()).backward()
        ob.step()
        assert abs(float(ob.grad_norm) - float(n)) <= 1e-4 * float(n)
    # the way that the weights have gone, to a thousandth: far above fp32's rounding of three steps, far below
    # what one gradient left out, doubled or not clipped would make
    for (name, y), x, s in zip(b.named_parameters(), a.parameters(), start):
        assert float((y.detach().cpu().double() - x.detach()).norm()) <= 1e-3 * float((x.detach() - s).norm()), name
