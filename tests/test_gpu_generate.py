"""Serving the language model: packed prompts, the cache, single tokens and
drawn tokens (orthossm_b200.lm) against the model's own forward."""
import pytest
import torch

from orthossm_b200.lm import OrthoLMConfig, OrthoSSMLM
from orthossm_b200.state import ChebyStreamState
from tests.test_oracle_golden import relerr

pytestmark = pytest.mark.gpu

CFG = OrthoLMConfig(vocab_size=1000, n_layers=2, window=64)


def model_and_coeffs(batch):
    torch.manual_seed(0)
    model = OrthoSSMLM(CFG).to("cuda", torch.bfloat16)
    return model, [st.coeffs for st in model.fresh_states(batch, "cuda", generator_seed=1)]


def whole(model, coeffs, b, ids):
    """Logits of the model's forward over one stream from its first token."""
    states = [ChebyStreamState(coeffs=c[b:b + 1]) for c in coeffs]
    with torch.no_grad():
        return model(ids.view(1, -1), states)[0]


def ids(n):
    return torch.randint(0, CFG.vocab_size, (n,), device="cuda")


# The model's bf16 forward and this path are each within 2e-2 of the exact
# logits (the bound tests/test_gpu_lm.py holds the forward to), so within 4e-2
# of each other.
TOL = 4e-2


@pytest.mark.parametrize("lens", [[1], [200], [5, 130, 1, 77], [96, 96, 96]])
def test_packed_prompts_match_the_forward(lens):
    model, coeffs = model_and_coeffs(len(lens))
    prompts = [ids(n) for n in lens]
    cache = model.new_cache(len(lens), 256, coeffs)
    logits = model.extend(prompts, cache)
    assert logits.shape == (len(lens), CFG.vocab_size) and cache.lengths == lens
    assert cache.lengths_dev.tolist() == lens
    for b, p in enumerate(prompts):
        assert relerr(logits[b].float().cpu().numpy(), whole(model, coeffs, b, p)[-1].float().cpu().numpy()) < TOL


def test_pieces_and_single_tokens_continue_the_stream():
    """A prompt in uneven pieces, then token by token, past the window: the
    logits after each call are those of the forward over the whole stream (the
    local window reaches over the calls' boundaries)."""
    model, coeffs = model_and_coeffs(2)
    streams = [ids(170), ids(150)]
    cache = model.new_cache(2, 170, coeffs)
    at = [0, 0]
    for piece in [(30, 11), (50, 50), (1, 70), (70, 1)] + [(1, 1)] * 18:
        new = [s[a:a + n] for s, a, n in zip(streams, at, piece)]
        logits = model.extend(new, cache)
        at = [a + n for a, n in zip(at, piece)]
        for b in range(2):
            ref = whole(model, coeffs, b, streams[b][:at[b]])[-1]
            assert relerr(logits[b].float().cpu().numpy(), ref.float().cpu().numpy()) < TOL
    assert at == [169, 150]


@pytest.mark.parametrize("where", [1, "head"])
def test_a_call_that_raises_leaves_the_streams(where, monkeypatch):
    model, coeffs = model_and_coeffs(2)
    cache = model.new_cache(2, 128, coeffs)
    first, then = [ids(20), ids(33)], [ids(5), ids(1)]
    model.extend(first, cache)
    ema = [e.clone() for e in cache.ema]

    def fail(*a, **kw):
        raise MemoryError("on purpose")

    with monkeypatch.context() as m:
        m.setattr(model.lm_head if where == "head" else model.layers[where],
                  "forward" if where == "head" else "extend", fail)
        with pytest.raises(MemoryError):
            model.extend([ids(7), ids(9)], cache)
    assert cache.lengths == [20, 33] and cache.lengths_dev.tolist() == [20, 33]
    assert all(torch.equal(a, b) for a, b in zip(cache.ema, ema))
    got = model.extend(then, cache)
    other = model.new_cache(2, 128, coeffs)
    model.extend(first, other)
    assert torch.equal(got, model.extend(then, other))


def test_generate():
    model, coeffs = model_and_coeffs(3)
    prompts = [ids(40), ids(3), ids(90)]
    greedy = model.generate(prompts, 12, temperature=0.0, coeffs=coeffs)
    assert greedy.shape == (3, 12) and int(greedy.min()) >= 0 and int(greedy.max()) < CFG.vocab_size
    # greedy tokens: the largest logit of the same calls made by hand
    cache = model.new_cache(3, 200, coeffs)
    logits = model.extend(prompts, cache)
    for i in range(12):
        best = logits.float().argmax(-1)
        assert greedy[:, i].tolist() == best.tolist()
        logits = model.extend(list(best.split(1)), cache)
    draw = lambda seed: model.generate(  # noqa: E731
        prompts, 8, temperature=0.9, top_k=40, top_p=0.95, generator=torch.Generator("cuda").manual_seed(seed),
        coeffs=coeffs)
    assert torch.equal(draw(1), draw(1)) and not torch.equal(draw(1), draw(2))


@pytest.mark.parametrize("f", [dict(temperature=0.0), dict(temperature=0.9, top_k=40), dict()])
def test_a_stream_without_a_token_ends_alone(f):
    """One stream's logits are NaN: its tokens are -1 and the other streams'
    those that they are without it."""
    model, coeffs = model_and_coeffs(3)
    prompts = [ids(40), ids(3), ids(90)]
    draw = lambda c: model.generate(prompts, 6, coeffs=c, **f,  # noqa: E731
                                    generator=torch.Generator("cuda").manual_seed(5))
    want = draw(coeffs)
    coeffs[0][1] = float("nan")
    got = draw(coeffs)
    assert got[1].tolist() == [-1] * 6 and int(want.min()) >= 0
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])


def test_refusals():
    model, coeffs = model_and_coeffs(2)
    cache = model.new_cache(2, 16, coeffs)
    for bad in [[ids(3)], [ids(3), ids(0)], [ids(17), ids(3)]]:
        with pytest.raises(ValueError):
            model.extend(bad, cache)
    assert cache.lengths == [0, 0]
    with pytest.raises(ValueError, match="bf16"):
        OrthoSSMLM(CFG).cuda().new_cache(1, 8)
