"""GPU: operands enter the adapters' products with all of their pieces, the last one too. Activations, inner products and fp32 weights are taken whose last
piece is as large as it gets and has the sign of the others, so that a product without it is off by more than fp32 sums can be."""
import numpy as np
import pytest
import torch

from mtlqwen_b200 import device as D
from test_gpu_adapter_ranges import rebuilt
from test_gpu_adapters import TYPES, Adapters

pytestmark = pytest.mark.gpu


def with_last_piece(rng, shape, half):
  """Positive values of one binade: the last eight of 24 bits set behind eight of which the first is, or the last twelve but one (half a unit of fp16 almost)."""
  return (1 + (2.0**-11 - 2.0**-23 if half else 2.0**-8 + 2.0**-15 - 2.0**-23) + 2.0**-7 * rng.integers(0, 4, shape)).astype(np.float32)


def without_last_piece(values, half):
  if half:
    return values.astype(np.float16).astype(np.float64)
  cut = lambda v: (v.view(np.uint32) & 0xffff0000).view(np.float32)
  first = cut(values)
  return first.astype(np.float64) + cut(values - first)


def call(dev, type_name, adapters, x, of_row, n):
  y = dev.empty((len(x), n))
  dev.adapters(TYPES[type_name][0], [adapters.table], len(adapters.a), dev.array(of_row), [n], x.shape[1], dev.array(x), len(x), [dev.array(np.zeros((len(x), n), np.float32))], [y])
  return y.download()


def compare(got, adapters, x, of_row, lost):
  """`lost`: the products without the last piece."""
  value, error = adapters.product(x, of_row, got.shape[1])
  error = error + 2.0**-23 * np.abs(value)
  assert (np.abs(value - lost) > 2 * error).all()  # the case can tell
  assert (np.abs(got - value) <= error).all()


@pytest.mark.parametrize("type_name", sorted(TYPES))
@pytest.mark.parametrize("k", [256, 1280])
@pytest.mark.parametrize("rows,ranks", [(1, [16]), (8, [16]), (96, [24, 100, 128]), (512, [128, 120])])
def test_activations(dev, type_name, k, rows, ranks):
  rng, n = np.random.default_rng(rows), 24
  adapters, of_row = Adapters(dev, rng, type_name, n, k, ranks), np.arange(rows, dtype=np.int32) * len(ranks) // rows
  for a, b in zip(adapters.a, adapters.b):
    a.copy_(torch.from_numpy(2.0**rng.integers(-3, 3, a.shape)))
    b.zero_()
    b[torch.arange(n), torch.arange(n) % b.shape[1]] = 1  # a column takes a rank
  adapters, x = rebuilt(dev, type_name, adapters), with_last_piece(rng, (rows, k), type_name == "f16")
  short, lost = without_last_piece(x, type_name == "f16"), np.zeros((rows, n))
  for i, (a, scale) in enumerate(zip(adapters.a, adapters.scale)):
    lost[of_row == i] = scale * (short[of_row == i] @ a.double().numpy().T)[:, np.arange(n) % a.shape[0]]
  compare(call(dev, type_name, adapters, x, of_row, n), adapters, x, of_row, lost)


@pytest.mark.parametrize("type_name", sorted(TYPES))
@pytest.mark.parametrize("rows,rank", [(1, 16), (8, 40), (40, 16), (300, 40), (40, 70)])
def test_inner_products(dev, type_name, rows, rank):
  rng, n, k = np.random.default_rng(rows), 24, 256
  adapters, of_row = Adapters(dev, rng, type_name, n, k, [rank]), np.zeros(rows, np.int32)
  adapters.a[0].zero_()
  adapters.a[0][torch.arange(rank), torch.arange(rank) * 3] = 1  # a rank is an activation
  adapters.b[0].copy_(torch.from_numpy(2.0**rng.integers(-3, 3, (n, rank))))
  adapters.scale = [1.0]
  adapters, x = rebuilt(dev, type_name, adapters), np.zeros((rows, k), np.float32)
  x[:, np.arange(rank) * 3] = with_last_piece(rng, (rows, rank), type_name == "f16")
  lost = without_last_piece(x, type_name == "f16")[:, np.arange(rank) * 3] @ adapters.b[0].double().numpy().T
  compare(call(dev, type_name, adapters, x, of_row, n), adapters, x, of_row, lost)


@pytest.mark.parametrize("rows,rank", [(1, 16), (8, 40), (96, 40), (512, 100)])
@pytest.mark.parametrize("which", ["a", "b"])
def test_weights_of_32_bits(dev, rows, rank, which):
  rng, n, k = np.random.default_rng(rows), 24, 256
  adapters, of_row = Adapters(dev, rng, "f32", n, k, [rank]), np.zeros(rows, np.int32)
  x = (2.0**rng.integers(-2, 3, (rows, k))).astype(np.float32)
  a, b = adapters.a[0], adapters.b[0]
  if which == "a":
    a.copy_(torch.from_numpy(with_last_piece(rng, (rank, k), False)))
    b.zero_()
    b[torch.arange(n), torch.arange(n) % rank] = 1
  else:
    a.zero_()
    a[torch.arange(rank), torch.arange(rank)] = 1
    b.copy_(torch.from_numpy(with_last_piece(rng, (n, rank), False)))
  adapters.scale = [1.0]
  short = {"a": a.double().numpy(), "b": b.double().numpy()}
  short[which] = without_last_piece({"a": a, "b": b}[which].numpy(), False)
  lost = x.astype(np.float64) @ short["a"].T @ short["b"].T
  compare(call(dev, "f32", rebuilt(dev, "f32", adapters), x, of_row, n), adapters, x, of_row, lost)
