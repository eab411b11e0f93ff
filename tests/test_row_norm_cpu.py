"""What the norms of whole rows say of rows without values, before any device is touched."""
from __future__ import annotations

import pytest
import torch


@pytest.mark.parametrize("shape", [(0,), (4, 0), (2, 3, 0), (2, 0, 3, 0)])
def test_rows_without_values_are_refused_in_the_layers_own_words(race, shape):
    x = torch.zeros(shape)
    for call, name in ((race.race_add_norm, "race_add_norm"), (race.race_add_norm_e4m3, "race_add_norm_e4m3")):
        for args in ((x,), (x, x)):
            with pytest.raises(RuntimeError, match=f"{name}: x lives on the CPU"):
                call(*args)
