"""Sessions that draw their tokens, without a GPU: ``argmax`` and ``sample`` are stood in for on the host."""
import pytest
import torch

from helpers import pkg
from test_sessions_host_logic import FakeModel


@pytest.fixture
def asked(monkeypatch):
    """The numbers that draws were made by, in order; the token is the one at that share of the vocabulary."""
    calls, mod = [], pkg().sessions

    def sample(logits, uniforms, temperature=None, top_k=None, top_p=None, min_p=None, out=None):
        calls.append(uniforms.item())
        return torch.tensor([int(uniforms.item() * logits.shape[-1])], dtype=torch.int32)

    monkeypatch.setattr(mod, "sample", sample)
    return calls


def generate(*samplings, n=6):
    """The tokens of sessions side by side, each with n of them."""
    mod = pkg().sessions
    engine = mod.SessionEngine(FakeModel(), max_batch=len(samplings), capacity=64)
    live = [engine.prepare_session_with_chunk_size([1, 2], n, sampling=s) for s in samplings]
    while any(not s.finished for s in live):
        for s in live:
            engine.advance(s)
            if not s.finished:
                engine.decode_sessions([s])
    return [s.generated_ids for s in live]


def test_sessions_may_share_their_settings(asked):
    S = pkg().sessions.Sampling
    alone = generate(S(seed=3))[0]
    shared = S(seed=3)
    assert generate(shared, shared, shared) == [alone] * 3
    assert generate(shared)[0] == alone                # and used again they begin anew
    assert generate(S(seed=4), shared) == [generate(S(seed=4))[0], alone]
    assert len(set(alone)) > 1


def test_numbers_of_a_session_are_those_of_its_seed(asked):
    import random
    S = pkg().sessions.Sampling
    generate(S(seed=11))
    want = random.Random(11)
    assert asked == [want.random() for _ in range(6)]


def test_a_draw_by_itself(asked):
    """Without a generator the settings' own goes on, as it does for nobody else."""
    import random
    S = pkg().sessions.Sampling
    s, z, want = S(seed=5), torch.zeros(1, 32), random.Random(5)
    s.draw(z)
    generate(s, s)
    s.draw(z)
    s.draw(z, random.Random(9))
    assert asked[0] == want.random() and asked[-2] == want.random() and asked[-1] == random.Random(9).random()


def last_max(logits):
    v = logits.float()
    return (v.shape[-1] - 1 - torch.flip(v, [-1]).argmax(-1)).to(torch.int32)


class Ties(FakeModel):
    """The likeliest token twice."""

    def _logits(self, tokens):
        out = super()._logits(tokens)
        out[:, 5] = out[:, 20] = 2.0
        return out


@pytest.mark.parametrize("temperature", [0, 0.0, 1e-60])
def test_a_temperature_of_zero_is_greedy_on_ties_too(monkeypatch, temperature):
    """``sample`` takes the first of equal maxima and ``argmax`` the last one."""
    mod = pkg().sessions
    monkeypatch.setattr(mod, "argmax", last_max)
    monkeypatch.setattr(mod, "sample", lambda logits, *rules: logits.float().argmax(-1).to(torch.int32))
    for sampling, token in ((None, 20), (mod.Sampling(temperature=temperature), 20), (mod.Sampling(temperature=temperature, top_k=3, top_p=0.5, min_p=0.1), 20), (mod.Sampling(top_k=1), 5)):
        engine = mod.SessionEngine(Ties(), max_batch=1, capacity=64)
        s = engine.prepare_session_with_chunk_size([1, 2], 4, sampling=sampling)
        assert engine.advance(s) == token, sampling


def test_a_temperature_of_zero_draws_nothing_that_is_not_a_number(monkeypatch):
    mod = pkg().sessions
    monkeypatch.setattr(mod, "argmax", last_max)
    inf, nan = float("inf"), float("nan")
    for z, token in (([1.0, nan, 3.0, 3.0, nan], 3), ([-inf, -inf, -2.0, -inf], 2), ([nan, -inf], -1), ([-inf, -inf, -inf], -1), ([inf, 0.0, inf, nan], 2)):
        for dtype in (torch.float32, torch.bfloat16):
            got = mod.Sampling(temperature=0.0).draw(torch.tensor([z], dtype=dtype))
            assert got.tolist() == [token] and got.dtype == torch.int32
    engine = mod.SessionEngine(FakeModel(), max_batch=1, capacity=64)
    s = engine.prepare_session_with_chunk_size([1, 2], 4, sampling=mod.Sampling(temperature=0.0))
    s.next_logits = torch.full((32,), -inf)
    with pytest.raises(pkg().Ab2Error):
        engine.advance(s)
    assert s.generated_ids == []
