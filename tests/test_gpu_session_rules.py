"""A session's grammar is kept, or the session says that it cannot be."""
import math

import pytest

from helpers import pkg
from model_fixtures import SMALL, build_pair

pytestmark = pytest.mark.gpu


def test_a_token_that_is_not_allowed_is_never_the_choice():
    p = pkg()
    model = build_pair(SMALL, "int8_channel", capacity=64)[0]
    engine = p.sessions.SessionEngine(model, max_batch=1, capacity=64)
    R = p.sessions.LogitRules
    s = engine.prepare_session_with_chunk_size([3, 1, 4], 8, rules=R(allowed=lambda ids: [17, 5], bias={17: -math.inf}))
    assert engine.advance(s) == 5
    s.rules = R(allowed=lambda ids: [17, 5], bias={17: -math.inf, 5: -math.inf})
    with pytest.raises(p.Ab2Error) as e:
        engine.advance(s)
    assert e.value.status == -7 and s.generated_ids == [5] and not s.finished
    s.rules = R(allowed=lambda ids: [17])
    assert engine.advance(s) == 17
