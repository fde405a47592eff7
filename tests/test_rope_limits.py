"""rope_tables refuses what has no tables: numbers that are not finite, and YaRN's ramp
where its dimensions are not in order."""
from __future__ import annotations

import math

import numpy as np
import pytest

from q3ops.rope import rope_tables

YARN = {"scaling": "yarn", "factor": 4.0, "original": 64}


@pytest.mark.parametrize("kw", [
    {"theta": math.nan}, {"theta": math.inf}, {"factor": math.nan, "scaling": "linear"}, {"factor": math.inf, "scaling": "linear"},
    {"factor": math.inf, "scaling": "ntk"}, {**YARN, "factor": math.nan}, {**YARN, "theta": 0.5}, {**YARN, "beta_fast": 0.0},
    {**YARN, "beta_slow": 0.0}, {**YARN, "beta_slow": -1.0}, {**YARN, "beta_fast": 0.5}, {**YARN, "beta_fast": math.nan},
    {**YARN, "attention_factor": math.nan}], ids=str)
def test_refused(kw):
    with pytest.raises(ValueError):
        rope_tables(**{"positions": 8, **kw})


@pytest.mark.parametrize("kw", [{}, {"theta": 0.5}, {"factor": 1e30, "scaling": "linear"}, YARN, {**YARN, "beta_fast": 1.0},
                                {**YARN, "original": 1}, {**YARN, "rot_dim": 2}], ids=str)
def test_finite(kw):
    for t in rope_tables(**{"positions": 8, **kw}):
        assert np.isfinite(t).all()
