"""Filters of a request on the host: what is refused, and what the scheduler hands to the pick."""
import numpy as np
import pytest

import plain_continuations as plain


@pytest.mark.parametrize("bad", [{"top_k": -1}, {"top_k": 1.5}, {"top_k": True}, {"top_k": 1 << 31}, {"top_p": 0.0}, {"top_p": 1.5},
                                 {"top_p": float("nan")}, {"min_p": -0.1}, {"min_p": 1.1}, {"min_p": float("nan")}])
def test_filters_that_are_refused(bad):
    from imparo_amd import SamplingParams, generate
    with pytest.raises(ValueError, match=next(iter(bad))):
        SamplingParams(**bad)
    with pytest.raises(ValueError, match=next(iter(bad))):
        generate("/nowhere", [[1]], **bad)


def test_the_plain_form_keeps_a_beginning_of_the_order():
    x = np.array([1.0, 3.0, 2.0, 3.0, 0.0], dtype=np.float32)
    assert plain.kept_tokens(x, 1.0, top_k=1)[0].tolist() == [1]
    assert plain.kept_tokens(x, 1.0, top_k=3)[0].tolist() == [1, 2, 3]
    assert plain.kept_tokens(x, 1.0, min_p=0.3)[0].tolist() == [1, 2, 3]
    assert plain.kept_tokens(x, 1.0, top_p=0.5)[0].tolist() == [1, 3]
    assert plain.pick(x, 1.0, 0.0, top_k=1) == 1 and plain.pick(x, 1.0, 1.0, top_p=0.5) == 3


def test_the_scheduler_hands_filters_over_only_where_a_request_has_some():
    from test_scheduler import make
    from imparo_amd.sampling.sampler import SamplingParams
    eng, s = make(n_pages=64)
    seen = []
    plain_pick = s.pick
    s.pick = lambda logits, t, u, *more: seen.append(more) or plain_pick(logits, t, u)
    s.add("a", [1, 2], SamplingParams(max_tokens=2))
    s.run()
    assert seen and all(more == () for more in seen)
    seen.clear()
    s.add("b", [1, 2], SamplingParams(max_tokens=1))
    s.add("c", [1, 2], SamplingParams(max_tokens=1, top_k=4, min_p=0.1))
    s.run()
    assert seen == [([(0, 1.0, 0.0), (4, 1.0, 0.1)],)]


def test_a_vocabulary_that_is_not_filtered_ends_the_request_alone():
    from test_scheduler import make
    from imparo_amd.kernels.ops import PICK_MAX_VOCAB
    from imparo_amd.sampling.sampler import SamplingParams
    eng, s = make(n_pages=64)
    plain_pick = s.pick
    s.pick = lambda logits, t, u, *more: plain_pick(logits, t, u)
    eng.vocab_size = PICK_MAX_VOCAB
    assert s.add("a", [1, 2], SamplingParams(max_tokens=1, top_k=4)).finish_reason == ""
    eng.vocab_size = PICK_MAX_VOCAB + 1
    assert s.add("b", [1, 2], SamplingParams(max_tokens=1, top_k=4)).finish_reason.startswith("error: top_k")
    assert s.add("c", [1, 2], SamplingParams(max_tokens=1)).finish_reason == ""
    s.run()
    assert s.finished["a"].finish_reason == s.finished["c"].finish_reason == "length"
