"""q35_model_sample and q35_model_decode_sampled: the model's logits drawn from by q35_sample.

The drawn ids are those that the definition in float64 gives for the logits of single steps (which a replayed
graph reproduces bit for bit), where u is not within the weights' rounding of a border; temperature 0 gives the greedy
ids."""
import numpy as np
import pytest

import pyq35
from q4_ref import sample64

pytestmark = pytest.mark.gpu


@pytest.fixture
def model(model_dirs):
    m = pyq35.Model(model_dirs["tiny_untied"], 64)
    yield m
    m.close()


def test_temperature_zero_is_greedy(model):
    greedy = model.decode_greedy(5, 11)
    last = model.step(int(greedy[-1]))
    model.reset()
    ids, prob = model.decode_sampled(5, np.full(11, 0.7), temperature=0.0)
    np.testing.assert_array_equal(ids, greedy)
    np.testing.assert_array_equal(prob, np.ones(11, np.float32))
    again = model.step(int(ids[-1]))
    np.testing.assert_array_equal(again[0], last[0])
    assert again[1] == last[1] and model.position == 12


@pytest.mark.parametrize("graph", [True, False])
@pytest.mark.parametrize("how", [dict(temperature=1.0), dict(temperature=3.0, top_k=40), dict(temperature=2.0, top_p=0.9, min_p=0.01)])
def test_steps_draw_from_their_logits(model, how, graph):
    rng = np.random.default_rng(17)
    u = rng.random(13, dtype=np.float32)
    model.set_graph(graph)
    ids, prob = model.decode_sampled(9, u, **how)
    assert model.position == 13
    model.reset()
    token, compared = 9, 0
    setting = (np.float32(how.get("temperature", 1.0)), how.get("top_k", 0), np.float32(how.get("top_p", 1.0)), np.float32(how.get("min_p", 0.0)))
    for i in range(13):
        logits, _ = model.step(token)
        want, p, room = sample64(logits, *setting, u[i])
        drawn, share = model.sample(float(u[i]), **how)  # from the step's logits, by itself
        assert drawn == ids[i] and share == prob[i]
        if room > len(logits) * (2.0 ** -50 + 2.0 ** -52):
            assert ids[i] == want and abs(prob[i] - p) <= p * 2.0 ** -22
            compared += 1
        token = int(ids[i])
    assert compared >= 12


def test_a_prompts_last_logits(model):
    """A prefill's last token is drawn from, and decoding goes on."""
    prompt = np.arange(3, 20, dtype=np.int32)
    lg = model.prefill(prompt)
    token, share = model.sample(0.4, temperature=2.0, top_k=50)
    want, p, room = sample64(lg[-1], np.float32(2.0), 50, np.float32(1.0), np.float32(0.0), np.float32(0.4))
    assert token == want and abs(share - p) <= p * 2.0 ** -22
    ids, _ = model.decode_sampled(token, np.linspace(0.0, 0.99, 6), temperature=2.0, top_k=50)
    assert ids.shape == (6,) and model.position == len(prompt) + 6


def test_one_allocation(model):
    lib = pyq35.lib
    model.step(1)
    before = lib.q35_device_alloc_count()
    model.sample(0.5)
    assert lib.q35_device_alloc_count() == before + 1
    model.decode_sampled(2, np.full(5, 0.5))
    model.sample(0.1, top_k=3)
    assert lib.q35_device_alloc_count() == before + 1
    model.reserve_context(128)
    after = lib.q35_device_alloc_count()
    ids, _ = model.decode_sampled(2, np.full(100, 0.5))
    assert lib.q35_device_alloc_count() == after + 1 and len(ids) == 100


def test_refusals(model):
    lib, u = pyq35.lib, np.full(4, 0.5, np.float32)
    with pytest.raises(pyq35.Q35Error) as e:
        model.sample(0.5)                # no logits yet
    assert e.value.status == -6
    for t in (-1.0, np.nan):
        with pytest.raises(pyq35.Q35Error):
            model.decode_sampled(1, u, temperature=t)
    for token in (-1, model.dims.vocab_size):
        with pytest.raises(pyq35.Q35Error) as e:
            model.decode_sampled(token, u)
        assert e.value.status == -6
    with pytest.raises(pyq35.Q35Error) as e:
        model.decode_sampled(1, np.full(65, 0.5))
    assert e.value.status == -6
    assert lib.q35_model_decode_sampled(model.h, 1, 4, None, pyq35.ptr(u), pyq35.ptr(u), None) < 0
    assert lib.q35_model_sample(None, None, 0.5, None, None) < 0
    assert model.position == 0
    assert len(model.decode_sampled(1, u[:0])[0]) == 0
