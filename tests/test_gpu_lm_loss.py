"""OrthoSSMLM.loss: the training operators together, as the model uses them."""
import pytest
import torch
import torch.nn.functional as F

from orthossm_b200.lm import OrthoLMConfig, OrthoSSMLM
from tests.test_gpu_lm import ref_forward

pytestmark = pytest.mark.gpu


def model_and_ids(vocab=1000, B=2, S=300, seed=0):
    torch.manual_seed(seed)
    cfg = OrthoLMConfig(vocab_size=vocab, n_layers=2, window=64)
    model = OrthoSSMLM(cfg).to("cuda", torch.bfloat16)
    with torch.no_grad():  # logits with some spread
        model.embedding.weight.mul_(4)
    return model, torch.randint(0, vocab, (B, S), device="cuda")


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def test_loss_against_float64_and_the_logits():
    """Against float64 of the same network, as far as its bf16 logits are (2e-2
    of their norm); and against the cross entropy of the model's own logits."""
    model, ids = model_and_ids()
    st = model.fresh_states(2, "cuda", generator_seed=1)
    ref, finals = ref_forward(model, ids, st)
    t = torch.randint(0, 1000, ids.shape, device="cuda")
    t[0, :50] = -100
    want = F.cross_entropy(ref.reshape(-1, 1000), t.cpu().reshape(-1), reduction="none").view(ids.shape)
    with torch.no_grad():
        each, new = model.loss(ids, t, st, reduction="none", return_state=True)
        plain = F.cross_entropy(model(ids, st).float().view(-1, 1000), t.view(-1), reduction="none").view(ids.shape)
        mean = model.loss(ids, t, st)
    assert each.dtype == torch.float32 and each.shape == ids.shape and (each[0, :50] == 0).all()
    spread = float(ref.std())
    assert float((each.cpu() - want).abs().mean()) < 2e-2 * spread
    assert float((each - plain).abs().mean()) < 2e-2 * spread
    assert abs(float(mean) - float(want.sum() / 550)) < 2e-2 * spread
    for s, f in zip(new, finals):
        assert s.tokens_seen == 300 and rel(s.ema.cpu(), torch.from_numpy(f)) < 5e-3


def test_gradients_against_the_composed_network():
    """Every parameter that forward's cross entropy reaches gets its gradient.
    Both are bf16 networks of some 20 roundings of 2^-9 in a row, forward and
    back: sqrt(40) 2^-9 = 1.2e-2 of the norm each, 3e-2 between them with the
    smaller parameters' sums; 5e-2 is asked."""
    model, ids = model_and_ids()
    st = model.fresh_states(2, "cuda", generator_seed=1)
    got = torch.autograd.grad(model.loss(ids, states=st), list(model.parameters()), allow_unused=True)
    logits = model(ids, st)[:, :-1].reshape(-1, 1000)
    want = torch.autograd.grad(F.cross_entropy(logits.float(), ids[:, 1:].reshape(-1)), list(model.parameters()),
                               allow_unused=True)
    for (name, _), a, b in zip(model.named_parameters(), got, want):
        assert (a is None) == (b is None), name
        if a is not None:
            assert rel(a, b) < 5e-2, (name, rel(a, b))


def test_padding_and_default_targets():
    """Padded ends leave the tokens before them alone: a padded batch's losses are the sequences' own."""
    model, ids = model_and_ids(S=200)
    st = model.fresh_states(2, "cuda", generator_seed=1)
    with torch.no_grad():
        whole = model.loss(ids, states=st, reduction="none")
        assert (whole[:, -1] == 0).all() and (whole[:, :-1] > 0).all()
        padded = ids.clone()
        padded[1, 120:] = -1
        each = model.loss(padded, states=st, reduction="none")
    assert torch.equal(each[0], whole[0])
    assert (each[1, 119:] == 0).all()
    assert float((each[1, :119] - whole[1, :119]).abs().max()) < 1e-3
    with pytest.raises(ValueError):
        OrthoSSMLM(model.cfg).to("cuda").loss(ids)


def test_training_steps_and_capture():
    """A few steps of SGD run; and a step captured into a graph gives what it gives eagerly."""
    model, ids = model_and_ids()
    st = model.fresh_states(2, "cuda", generator_seed=1)
    opt = torch.optim.SGD(model.parameters(), lr=0.1)
    for _ in range(3):
        opt.zero_grad()
        loss = model.loss(ids, states=st, z_loss=1e-4)
        loss.backward()
        opt.step()
        assert loss.isfinite()
    del loss  # torch refuses to capture a backward pass while an eager graph of the same leaves lives
    opt.zero_grad()
    ps = list(model.parameters())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = torch.autograd.grad(model.loss(ids, states=st), ps, allow_unused=True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = torch.autograd.grad(model.loss(ids, states=st), ps, allow_unused=True)
    graph.replay()
    torch.cuda.synchronize()
    for (name, _), a, b in zip(model.named_parameters(), eager, held):
        if a is not None:
            assert rel(b, a) < 1e-2, name
