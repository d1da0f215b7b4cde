"""GPU: how much of an activation or an inner product enters the adapters' products, beside others of another magnitude."""
import numpy as np
import pytest

from mtlqwen_b200 import device as D
from test_gpu_adapters import TYPES, Adapters, silu

pytestmark = pytest.mark.gpu


def scaled(dev, adapters, factor):
  """The same adapters with other scales."""
  adapters.scale = [scale * factor for scale in adapters.scale]
  adapters.table = dev.records(D.Adapter, [D.Adapter(a.ptr, b.ptr, weights.shape[0], scale) for (a, b), weights, scale in zip(adapters.held, adapters.a, adapters.scale)])
  return adapters


@pytest.mark.parametrize("type_name", sorted(TYPES))
@pytest.mark.parametrize("rows", [1, 8, 40])
@pytest.mark.parametrize("gate_scale,up_scale", [(1e-4, 1e12), (1.0, 1e-12), (1e-6, 1e-20)])
def test_the_matrices_of_a_pair_do_not_share_their_range(dev, type_name, rows, gate_scale, up_scale):
  """An adapter of one of them that is large or small beside the other's."""
  rng, k, n, ranks = np.random.default_rng(rows), 512, 72, [16, 40]
  of_row = (np.arange(rows) % 5 == 4).astype(np.int32)
  gate_set, up_set = (scaled(dev, Adapters(dev, rng, type_name, n, k, ranks), factor) for factor in (gate_scale, up_scale))
  x, zeros, y = rng.standard_normal((rows, k)).astype(np.float32), dev.array(np.zeros((rows, n), np.float32)), dev.empty((rows, n))
  dev.adapters_gate_up(TYPES[type_name][0], gate_set.table, up_set.table, len(ranks), dev.array(of_row), n, k, dev.array(x), rows, zeros, zeros, y)
  (g, eg), (u, eu) = gate_set.product(x, of_row, n), up_set.product(x, of_row, n)
  eg, eu = eg + 2.0**-23 * np.abs(g), eu + 2.0**-23 * np.abs(u)
  want = silu(g) * u
  # silu's slope is below 1.1; the exponential is off by 2^-23 of its argument and two units, what follows by six halves of a unit
  assert (np.abs(y.download() - want) <= 1.1 * eg * (np.abs(u) + eu) + np.abs(silu(g)) * eu + (10 + 2 * np.abs(g)) * 2.0**-24 * np.abs(want) + 1e-37).all()
