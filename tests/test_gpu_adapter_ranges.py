"""GPU: how much of an activation or an inner product enters the adapters' products, beside others of another magnitude."""
import numpy as np
import pytest

from mtlqwen_b200 import device as D
from test_gpu_adapters import TYPES, Adapters, raw, silu

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


def rebuilt(dev, type_name, adapters):
  """The adapters with the weights that they hold now."""
  fresh = Adapters.__new__(Adapters)
  fresh.dtype, fresh.a, fresh.b, fresh.scale = adapters.dtype, adapters.a, adapters.b, adapters.scale
  fresh.held = [(raw(dev, a), raw(dev, b)) for a, b in zip(fresh.a, fresh.b)]
  return scaled(dev, fresh, 1.0)


@pytest.mark.parametrize("type_name", sorted(TYPES))
@pytest.mark.parametrize("rows,ranks", [(3, [24]), (96, [24, 100, 128])])
@pytest.mark.parametrize("larger", [2.0**10, 2.0**17, 2.0**24, 2.0**30])
def test_small_activations_beside_a_large_one(dev, type_name, rows, ranks, larger):
  """Channels that the adapters do not read: what the others keep beside them."""
  rng, k, n = np.random.default_rng(rows), 1024, 40
  adapters, of_row = Adapters(dev, rng, type_name, n, k, ranks), np.arange(rows, dtype=np.int32) * len(ranks) // rows
  x = rng.standard_normal((rows, k)).astype(np.float32)
  x[:, 5::32] *= np.float32(larger)
  for a in adapters.a:
    a[:, 5::32] = 0
  adapters = rebuilt(dev, type_name, adapters)
  zeros, y = dev.array(np.zeros((rows, n), np.float32)), dev.empty((rows, n))
  dev.adapters(TYPES[type_name][0], [adapters.table], len(ranks), dev.array(of_row), [n], k, dev.array(x), rows, [zeros], [y])
  value, error = adapters.product(x, of_row, n)
  if type_name == "f16":  # 2^-39 of the largest of each 32
    largest = np.repeat(np.abs(x.astype(np.float64)).reshape(rows, k // 32, 32).max(-1), 32, axis=1)
    for i, (a, b, scale) in enumerate(zip(adapters.a, adapters.b, adapters.scale)):
      mine = of_row == i
      error[mine] += scale * 2.0**-39 * (largest[mine] @ np.abs(a.double().numpy()).T) @ np.abs(b.double().numpy()).T
  assert (np.abs(y.download() - value) <= error + 2.0**-23 * np.abs(value)).all()


@pytest.mark.parametrize("type_name", sorted(TYPES))
@pytest.mark.parametrize("rows", [3, 96])
@pytest.mark.parametrize("larger", [2.0**10, 2.0**16])
@pytest.mark.parametrize("activation", [1.0, 2.0**14])
def test_small_inner_products_beside_a_large_one(dev, type_name, rows, larger, activation):
  """A rank that no column takes, and activations on it: what the other ranks keep beside it."""
  rng, k, n, rank = np.random.default_rng(rows), 512, 40, 40
  adapters, of_row = Adapters(dev, rng, type_name, n, k, [rank]), np.zeros(rows, np.int32)
  x = rng.standard_normal((rows, k)).astype(np.float32)
  x[:, 0] = activation
  adapters.a[0][:, 0] = 0
  adapters.a[0][7, 0], adapters.b[0][:, 7] = larger / 2, 0  # that rank alone takes the first channel
  adapters = rebuilt(dev, type_name, adapters)
  zeros, y = dev.array(np.zeros((rows, n), np.float32)), dev.empty((rows, n))
  dev.adapters(TYPES[type_name][0], [adapters.table], 1, dev.array(of_row), [n], k, dev.array(x), rows, [zeros], [y])
  value, error = adapters.product(x, of_row, n)
  if type_name == "f16":  # 2^-39 of the largest activation of each 32, and of the row's largest inner product
    a, b, scale = adapters.a[0].double().numpy(), np.abs(adapters.b[0].double().numpy()), adapters.scale[0]
    largest = np.repeat(np.abs(x.astype(np.float64)).reshape(rows, k // 32, 32).max(-1), 32, axis=1)
    error += scale * 2.0**-39 * (largest @ np.abs(a).T) @ b.T
    error += scale * 2.0**-39 * np.abs(x.astype(np.float64) @ a.T).max(-1, keepdims=True) * b.sum(-1)
  assert (np.abs(y.download() - value) <= error + 2.0**-23 * np.abs(value)).all()
