"""What the users of the device status word make of it."""
import pytest

from strata_b200 import _lib, halo, halo_block


def checks():
    for name, owner in (("halo exchange", halo.DistributedTileCopyHaloPadding),
                        ("tiled block run", halo_block.TiledBlockRunner)):
        yield name, lambda owner=owner: owner.check_status(object.__new__(owner))


@pytest.mark.parametrize("status,text", [(101, "kernel wait timed out"), (105, "peer flag wait timed out")])
def test_waits_that_ran_out(monkeypatch, status, text):
    monkeypatch.setattr(_lib, "device_status", lambda reset=True: status)
    for name, check in checks():
        with pytest.raises(RuntimeError, match=rf"{name} failed on the device \(status {status}: {text}\)"):
            check()


def test_a_position_behind_its_table_is_nobody_elses_failure(monkeypatch):
    monkeypatch.setattr(_lib, "device_status", lambda reset=True: 107)
    for _, check in checks():
        with pytest.raises(RuntimeError, match="position given to ops.qk_norm_rope"):
            check()
    monkeypatch.setattr(_lib, "device_status", lambda reset=True: 0)
    for _, check in checks():
        check()
