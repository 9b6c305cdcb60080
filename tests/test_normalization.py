"""Host bookkeeping of the normalisers that captured launch sequences share (no GPU needed)."""
import torch

from gnn_amd.normalization import Normalizer


def test_two_captured_users_share_one_device_count():
    """A rollout that starts and ends between the replays of a captured training step leaves the step's count where it is."""
    nr = Normalizer(1, 4, "n", "cpu")
    nr._acc_count = 5
    nr.use_device_count(True)
    count = nr._work()["count_dev"]
    nr._acc_count = 7
    nr.use_device_count(True)
    assert nr._work()["count_dev"] is count and int(count) == 7
    nr._acc_count = 6
    nr.sync_device_count()
    assert nr._work()["count_dev"] is count and int(count) == 6
    nr.use_device_count(False)
    assert nr._work()["count_dev"] is count
    nr.use_device_count(False)
    assert "count_dev" not in nr._work()
    nr.use_device_count(False)                       # one call too many changes nothing
    nr.use_device_count(True)
    assert int(nr._work()["count_dev"]) == 6
    assert any(t is nr._work()["mean_std"] for t in nr.captured_buffers())
