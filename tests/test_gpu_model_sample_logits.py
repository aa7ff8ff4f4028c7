"""q35_model_sample draws from logits of the model's own state or not at all: what gives a model another state or position
without a step leaves it without logits until the next step or prompt."""
import numpy as np
import pytest

import pyq35

pytestmark = pytest.mark.gpu
RANGE = -6


@pytest.fixture
def model(model_dirs):
    m = pyq35.Model(model_dirs["tiny_untied"], 64)
    yield m
    m.close()


def refused(m):
    with pytest.raises(pyq35.Q35Error) as e:
        m.sample(0.5)
    return e.value.status == RANGE


def set_position(m, pos):
    pyq35.check(pyq35.lib.q35_model_set_position(m.h, pos))


def test_position_of_a_new_model(model):
    set_position(model, 5)
    assert model.position == 5 and refused(model)
    model.step(3)
    assert model.sample(0.5)[0] >= 0


def test_state_of_another_sequence(model):
    """A state written back: the logits at hand are those of the sequence before."""
    for t in (1, 2, 3):
        model.step(t)
    assert model.sample(0.5)[0] >= 0
    model.reset()
    assert refused(model)
    set_position(model, 2)
    assert refused(model)
    model.prefill(np.arange(4, 9, dtype=np.int32))
    assert model.sample(0.5)[0] >= 0
    set_position(model, model.position)
    assert refused(model)


def test_synthetic_state(model):
    model.step(1)
    pyq35.check(pyq35.lib.q35_model_fill_synthetic(model.h, 9, 1, 0.1))
    assert model.position == 9 and refused(model)
    model.decode_greedy(2, 3)
    assert model.sample(0.25)[0] >= 0


@pytest.mark.parametrize("what", ["gdn", "conv", "kv"])
def test_state_written_in_place(model, what):
    """Another sequence's state of the same length, written without a position."""
    lib, d = pyq35.lib, model.dims
    model.step(1)
    assert model.sample(0.5)[0] >= 0
    if what == "gdn":
        x = np.zeros(d.gdn_v_heads * 128 * 128, np.float32)
        pyq35.check(lib.q35_model_write_gdn_state(model.h, 0, pyq35.ptr(x)))
    elif what == "conv":
        x = np.zeros((2 * d.gdn_k_heads + d.gdn_v_heads) * 128 * 3, np.float32)
        pyq35.check(lib.q35_model_write_conv_state(model.h, 0, pyq35.ptr(x)))
    else:
        x = np.zeros(d.attn_kv_heads * d.attn_head_dim, np.float32)
        pyq35.check(lib.q35_model_write_kv(model.h, 0, 0, 1, pyq35.ptr(x), pyq35.ptr(x)))
    assert refused(model)
    model.step(2)
    assert model.sample(0.5)[0] >= 0


def test_another_context(model):
    model.step(1)
    model.reserve_context(96)
    assert refused(model)
    set_position(model, 1)
    assert refused(model)
    ids, _ = model.decode_sampled(2, np.full(3, 0.5))
    assert len(ids) == 3 and model.sample(0.75)[0] >= 0


def test_a_refused_call_keeps_them(model):
    """What is refused before any work leaves the logits where they were."""
    model.step(7)
    first = model.sample(0.3)
    for ids in ([model.dims.vocab_size], np.zeros(100)):
        with pytest.raises(pyq35.Q35Error):
            model.extend(np.asarray(ids, np.int32))
    assert pyq35.lib.q35_model_set_position(model.h, 65) == RANGE
    assert model.sample(0.3) == first
