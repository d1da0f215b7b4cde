"""GPU: what a commit reports where a pass both met a record that is not served and abandoned a bounded wait."""
import numpy as np
import pytest

from mtlqwen_b200 import device as D

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("wait,record,reported", [(True, False, "bounded wait"), (False, True, "record"), ("first", True, "bounded wait"), ("last", True, "bounded wait")])
@pytest.mark.parametrize("rows", [2, 40])
def test_an_abandoned_wait_is_reported_before_a_record(wait, record, reported, rows):
  """The wait spoils the results of all requests, the record those of its own rows."""
  dev = D.Device(0)
  try:
    weights = dev.array(np.zeros(257 * 256, np.uint16))
    table = dev.records(D.Adapter, [D.Adapter(weights.ptr, weights.ptr, 257, 1.0)])
    x, y, index = dev.array(np.zeros((rows, 256), np.float32)), dev.array(np.zeros((rows, 8), np.float32)), dev.array(np.zeros(rows, np.int32))
    abandon = lambda: dev.check(dev.lib.infdev_check_abort_path(dev.ctx, 2000))
    if wait in (True, "first"):
      abandon()
    if record:
      dev.adapters(D.F16, [table], 1, index, [8], 256, x, rows, [y], [y])
    if wait == "last":
      abandon()
    assert dev.lib.infdev_commit(dev.ctx, 10000) == -4 and reported in dev.error()
    assert dev.lib.infdev_commit(dev.ctx, 10000) == 0
  finally:
    dev.close()
