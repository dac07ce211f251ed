"""What RotaryTable.for_model refuses, check by check: by its message, as a table on the host is refused whatever its settings."""
import math

import pytest
import torch

from sensenova_u1_amd import RotaryTable, ops

HOST = r"turns must be float64 \[pairs\] on a HIP device"


@pytest.mark.parametrize("message,settings", [
    ("7 elements are no pairs", dict(rotary_dim=7)), ("0 elements are no pairs", dict(rotary_dim=0)), ("-2 elements are no pairs", dict(rotary_dim=-2)),
    ("scaling 'other' by 1.0 on base 10000.0 is not known", dict(rotary_dim=64, scaling="other")), ("by 0.0 on base", dict(rotary_dim=64, factor=0.0)),
    ("by -2.0 on base", dict(rotary_dim=64, scaling="linear", factor=-2.0)), ("by nan on base", dict(rotary_dim=64, scaling="linear", factor=math.nan)),
    ("on base 1.0 is", dict(rotary_dim=64, base=1.0)), ("on base nan is", dict(rotary_dim=64, base=math.nan)),
    ("yarn scaling needs the original context", dict(rotary_dim=64, scaling="yarn", factor=4.0)),
    ("yarn scaling needs the original context", dict(rotary_dim=64, scaling="yarn", factor=4.0, original_context=-1))])
def test_bad_settings(message, settings):
    with pytest.raises(ops.SnGgufError, match=message):
        RotaryTable.for_model(**settings, device="cpu")


@pytest.mark.parametrize("settings", [dict(), dict(scaling="linear", factor=4.0), dict(scaling="yarn", factor=4.0, original_context=4096), dict(factor=0.5),
                                      dict(scaling="yarn", factor=4.0, original_context=1), dict(scaling="yarn", factor=1.0, original_context=4096)])
def test_good_settings_get_as_far_as_the_device(settings):
    with pytest.raises(ops.SnGgufError, match=HOST):
        RotaryTable.for_model(64, **settings, device="cpu")


@pytest.mark.parametrize("turns", [torch.ones(4), torch.ones((2, 2), dtype=torch.float64), torch.ones(0, dtype=torch.float64)])
def test_turns_on_the_host(turns):
    with pytest.raises(ops.SnGgufError, match=HOST):
        RotaryTable(turns)
