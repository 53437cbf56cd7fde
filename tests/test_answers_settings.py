"""What Model.answers refuses before it feeds anything (no GPU needed: nothing is launched)."""
from __future__ import annotations

import numpy as np
import pytest

from flock_amd.decoder import DecoderConfig
from flock_amd.model import Model


class Fed(Exception):
    pass


@pytest.fixture
def model():
    """A model that is never run: what would feed or capture raises."""
    m = Model.__new__(Model)
    m.cfg, m.vocab, m.nKeys = DecoderConfig(maxKeys=64, maxPrefill=8), 500, 0

    def fed(*_):
        raise Fed
    m._feed = m._answers_step = fed
    return m


@pytest.mark.parametrize("settings", [dict(temperature=1e39), dict(temperature=3.5e38),
                                      dict(top_p=1e-50), dict(top_p=7e-46),
                                      dict(temperature=-1e-50), dict(temperature=float("nan"))])
def test_settings_that_f32_does_not_hold(model, settings):
    """They are f32 on the device: infinite or 0 there, which flk_sample refuses."""
    with pytest.raises(ValueError):
        model.answers([1, 2], 2, 2, **settings)


@pytest.mark.parametrize("prompt", [[500], [1, 2, 500], [499, 1 << 31, 3], np.array([-1, 2])])
def test_ids_outside_the_vocabulary(model, prompt):
    """The embedding reads them as zeros."""
    with pytest.raises(ValueError):
        model.answers(prompt, 2, 2)
    assert model.nKeys == 0



@pytest.mark.parametrize("eos,stops", [([-1], 0), ([1 << 32], 0), ([3, 1 << 40, 7, 3], 2),
                                       ([500, 499], 1), (np.array([-5, 4]), 1)])
def test_stops_outside_the_vocabulary(model, eos, stops):
    """As for generate, an id that is never drawn ends nothing."""
    def step(*key):
        assert key == (2, 2, stops)
        raise Fed
    model._answers_step = step
    with pytest.raises(Fed):
        model.answers([1, 2], 2, 2, eos=eos)
