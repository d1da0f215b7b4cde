"""CPU: the oracle's sampler draws nothing that has no weight."""
import numpy as np
import pytest

import oracle

INF = np.inf


@pytest.mark.parametrize("uniform", [0.0, 2.0**-24, 0.5, 1 - 2.0**-24])
@pytest.mark.parametrize("logits,allowed", [([-INF, -INF, 1, 2, -INF], {2, 3}), ([-INF, 3], {1}), ([3, -INF, -INF], {0}), ([-1e4, 0, 0, -1e4], {1, 2}),
                                            ([1, INF, 2, INF], {1}), ([np.nan, 1, 2, -INF], {1, 2}), ([-INF, np.nan, 4, np.nan], {2})])
def test_plain_temperature_sampling_draws_what_has_a_weight(logits, allowed, uniform):
  assert oracle.sample(np.array(logits, np.float32), 0.8, 1.0, 0, uniform)[0] in allowed


def test_a_variate_of_zero_draws_the_first_token_that_has_a_weight():
  assert oracle.sample(np.array([-INF, -INF, 1, 2], np.float32), 0.8, 1.0, 0, 0.0)[0] == 2
  assert oracle.sample(np.array([0, 5, 1, 2], np.float32), 0.8, 1.0, 0, 0.0)[0] == 0


def test_a_row_without_anything_to_draw():
  row = np.full(7, -INF, np.float32)
  assert [oracle.sample(row, temperature, 1.0, top_k, 0.5)[0] for temperature, top_k in ((0.0, 0), (0.8, 4), (0.8, 0))] == [0, 0, 6]
