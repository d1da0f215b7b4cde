"""GPU: plain temperature sampling draws nothing that has no weight, whatever the variate."""
import numpy as np
import pytest

import oracle
from mtlqwen_b200 import device as D

pytestmark = pytest.mark.gpu
ZEROS = [(87, 87586), (93, 84823), (176, 52005)]  # seeds, and indices of a token in its sequence, whose variate is exactly 0


def test_the_variates_are_zero():
  assert all(oracle.uniform(*zero) == 0 for zero in ZEROS)


def sample(dev, logits, draws, temperature=0.9, top_k=0, mode=0):
  """One token a row; a draw is (seed, index of the token in its sequence)."""
  queries = []
  for row, (seed, index) in enumerate(draws):
    q = D.Query()
    q.start, q.count, q.position, q.slot, q.state = row, 1, index - 1, row % 8, D.UNBOUND
    q.logit, q.samples, q.temperature, q.topP, q.topK, q.seed = row, 1, temperature, 1.0, top_k, seed
    queries.append(q)
  tokens = dev.empty(len(draws), np.int32)
  dev.sample(dev.array(logits), logits.shape[1], dev.queries(queries), len(queries), len(draws), mode, tokens)
  return tokens.download().tolist()


@pytest.mark.parametrize("vocab", [2, 33, 130, 4099, 16384, 248320])
def test_a_variate_of_zero_draws_the_first_token_that_has_a_weight(dev, vocab):
  rng = np.random.default_rng(vocab)
  logits = rng.standard_normal((5, vocab)).astype(np.float32)
  first = [0, 1, vocab // 2, vocab - 1, vocab - 2]
  for row, begin in zip(logits, first):
    row[:begin] = -np.inf
  logits[4, :-2] = -1.0e6  # not masked, but without a weight
  draws = [ZEROS[i % 3] for i in range(5)]
  got = sample(dev, logits, draws)
  assert got == first and got == [oracle.sample(row, 0.9, 1.0, 0, 0.0)[0] for row in logits]


@pytest.mark.parametrize("rows,vocab", [(2, 40), (24, 1003), (9, 20000), (200, 4096), (8, 248320)])
@pytest.mark.parametrize("allowed", [1, 2, 17])
def test_rows_of_which_a_mask_leaves_little(dev, rows, vocab, allowed):
  rng = np.random.default_rng(allowed)
  logits = np.full((rows, vocab), -np.inf, np.float32)
  for row in logits:
    where = rng.choice(vocab, allowed, replace=False)
    row[where] = rng.standard_normal(allowed)
  draws = [ZEROS[0]] + [(int(rng.integers(1000)), 1 + r) for r in range(rows - 1)]
  for row, token in zip(logits, sample(dev, logits, draws)):
    assert np.isfinite(row[token])


@pytest.mark.parametrize("vocab", [5, 300, 4099, 248320])
def test_logits_that_are_not_finite(dev, vocab):
  logits = np.random.default_rng(vocab).standard_normal((4, vocab)).astype(np.float32)
  logits[0, [vocab // 2, vocab - 2]] = np.inf
  logits[1, 0] = logits[1, vocab - 1] = np.nan
  logits[2, vocab // 3:], logits[2, vocab - 1] = -np.inf, np.nan
  logits[3] = -np.inf
  draws = [(r, 5) for r in range(3)] + [ZEROS[0]]
  got = sample(dev, logits, draws)
  assert got == [oracle.sample(row, 0.9, 1.0, 0, oracle.uniform(*draw))[0] for row, draw in zip(logits, draws)]
  assert got[0] == vocab // 2 and got[1] not in (0, vocab - 1) and np.isfinite(logits[2, got[2]]) and got[3] == vocab - 1
  assert sample(dev, logits[3:], draws[3:], temperature=0.0) == [0] and sample(dev, logits[3:], draws[3:], top_k=4) == [0]


def test_a_mask_binds_the_sampler(dev):
  """Rules, then plain temperature sampling in the same pass: a token that a mask forbids is not drawn by a variate of 0."""
  vocab, rows = 248320, 3
  rng = np.random.default_rng(0)
  allowed = rng.random((rows, vocab)) < 0.5
  allowed[:, 0] = False
  masks = np.packbits(allowed, axis=1, bitorder="little").view(np.uint32)
  words, rules, queries = dev.array(masks), [], []
  for row, (seed, index) in enumerate(ZEROS):
    rules.append(D.LogitRules(mask=words.ptr + row * masks.shape[1] * 4))
    q = D.Query()
    q.start, q.count, q.position, q.slot, q.state = row, 1, index - 1, row, D.UNBOUND
    q.logit, q.samples, q.temperature, q.topP, q.seed = row, 1, 0.9, 1.0, seed
    queries.append(q)
  logits, records, tokens = dev.array(rng.standard_normal((rows, vocab)).astype(np.float32)), dev.queries(queries), dev.empty(rows, np.int32)
  dev.adjust_logits(logits, vocab, records, rows, rows, dev.records(D.LogitRules, rules), dev.array(np.zeros((rows, 1), np.int32)), 1, None, logits)
  dev.sample(logits, vocab, records, rows, rows, 0, tokens)
  assert tokens.download().tolist() == [int(np.argmax(row)) for row in allowed]
