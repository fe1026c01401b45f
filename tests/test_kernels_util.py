"""The recorder of kernel names, without a device: a recording that misses a kernel is taken again, one of a call that launches none stays."""
import pytest

from tests import kernels_util as U


@pytest.fixture
def recordings(monkeypatch):
    taken = []

    def given(*names):
        def record(fn, lead=0.0):
            taken.append(lead)
            return fn(), set(names[min(len(taken), len(names)) - 1])

        monkeypatch.setattr(U, "record", record)
        return taken

    return given


def test_a_missed_kernel_is_found_in_another_recording(recordings):
    taken = recordings({"copy"}, {"copy"}, {"copy", "lane_bwd_kernel<4, 3>"})
    out, names = U.kernels_of(lambda: 7)
    assert out == 7 and len(taken) == 1
    assert U.launched(names, r"lane_bwd_kernel<4,.* 3>") and len(taken) == 3 and taken[0] == 0.0 < taken[1]
    assert U.launched(names, "copy") and len(taken) == 3


def test_a_kernel_that_is_not_launched_is_not_found(recordings):
    taken = recordings({"copy"})
    _, names = U.kernels_of(lambda: None)
    assert not U.launched(names, "lane_bwd_kernel") and len(taken) == 1 + U.AGAIN


def test_an_empty_recording_is_taken_again(recordings):
    recordings(set(), set(), {"copy"})
    assert U.launched(U.kernels_of(lambda: None)[1], "copy")
    taken = recordings(set())
    taken.clear()
    with pytest.raises(pytest.skip.Exception):
        U.kernels_of(lambda: None)
    assert len(taken) == 1 + U.AGAIN
