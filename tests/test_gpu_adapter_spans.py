"""GPU: adapters of many rows, whose inner products come from weights and activations that are staged 128 along k at a time."""
import numpy as np
import pytest

from mtlqwen_b200 import device as D
from test_gpu_adapters import TYPES, Adapters, check, run, silu

pytestmark = pytest.mark.gpu
# An eighth of k is staged in several goes, of which the last one may not be whole.
LENGTHS = [1280, 4096, 4352, 12288]
# On 148 SMs: three tiles of 16 ranks an item; eight, four an item; eight an item.
THREE = ([33, 18, 7], [16], [0] * 128)
FOUR = ([33, 18], [64, 64], [0] * 70 + [1] * 58)
EIGHT = ([33, 18], [64, 64], [0] * 300 + [1] * 212)


@pytest.mark.parametrize("type_name", sorted(TYPES))
@pytest.mark.parametrize("k", LENGTHS)
@pytest.mark.parametrize("ns,ranks,of_row", [THREE, FOUR, EIGHT, ([20], [120], [0] * 300), ([20, 9, 40, 11], [3, 50], ([0] * 20 + [1] * 12) * 5 + [-1, 0, 1])])
def test_lengths_of_many_rows(dev, type_name, k, ns, ranks, of_row):
  check(*run(dev, type_name, k, ns, ranks, of_row, seed=k))


@pytest.mark.parametrize("type_name,shift", [("f16", 2), ("f16", 8), ("bf16", 2), ("bf16", 4), ("f32", 4), ("f32", 8)])
@pytest.mark.parametrize("ns,ranks,of_row", [THREE, EIGHT, ([40, 7], [16, 100, 64], [0] * 40 + [1] * 50 + [2] * 40)])
@pytest.mark.parametrize("k", [512, 1280, 4096])
def test_weights_of_many_rows_on_any_boundary(dev, type_name, shift, k, ns, ranks, of_row):
  check(*run(dev, type_name, k, ns, ranks, of_row, shift=shift))


@pytest.mark.parametrize("type_name", sorted(TYPES))
@pytest.mark.parametrize("k", [1280, 4096])
@pytest.mark.parametrize("ranks,of_row", [([64], [0] * 128), ([64, 8], [0] * 300 + [1] * 212), ([130, 16], [0] * 200 + [1, 0] * 90)])
def test_pairs_of_many_rows(dev, type_name, k, ranks, of_row):
  rng, n, m, of_row = np.random.default_rng(k), 50, len(of_row), np.array(of_row, np.int32)
  gate_set, up_set = (Adapters(dev, rng, type_name, n, k, ranks) for _ in range(2))
  x, gate, up = (rng.standard_normal(shape).astype(np.float32) for shape in ((m, k), (m, n), (m, n)))
  y = dev.empty((m, n))
  dev.adapters_gate_up(TYPES[type_name][0], gate_set.table, up_set.table, len(ranks), dev.array(of_row), n, k, dev.array(x), m, dev.array(gate), dev.array(up), y)
  (dg, eg), (du, eu) = gate_set.product(x, of_row, n), up_set.product(x, of_row, n)
  g, u = gate + dg, up + du
  eg, eu = eg + 2.0**-23 * (np.abs(gate) + np.abs(dg)), eu + 2.0**-23 * (np.abs(up) + np.abs(du))
  want = silu(g) * u
  # silu's slope is below 1.1; the exponential is off by 2^-23 of its argument and two units, what follows by six halves of a unit
  assert (np.abs(y.download() - want) <= 1.1 * eg * (np.abs(u) + eu) + np.abs(silu(g)) * eu + (10 + 2 * np.abs(g)) * 2.0**-24 * np.abs(want) + 1e-37).all()


def test_a_call_of_many_rows_gives_the_same_bits_again(dev):
  for type_name in TYPES:
    first, again = (run(dev, type_name, 4352, *EIGHT, seed=1)[-1] for _ in range(2))
    assert all(np.array_equal(a, b) for a, b in zip(first, again))
