"""CPU: the status words' creation and polls from several host threads (the device's side is replaced by plain CPU tensors)."""
import threading

import pytest
import torch

from rise_sdf_amd import _lib


@pytest.fixture
def fake(monkeypatch):
    """A device 0 whose words live in host memory; what was asked of the device is logged."""
    log = []
    zeros = torch.zeros

    def make(*size, **kw):
        kw.pop("device", None)
        log.append("zeros")
        if barrier is not None:
            try:
                barrier.wait(timeout=0.5)
            except threading.BrokenBarrierError:
                pass
        return zeros(*size, **kw)
    barrier = None

    class Stream:
        def synchronize(self):
            log.append("wait")

    class Guard:
        def __init__(self, idx):
            pass

        def __enter__(self):
            return self

        def __exit__(self, *a):
            return False
    state = dict(capturing=False)
    monkeypatch.setattr(_lib, "_STATUS", {})
    monkeypatch.setattr(_lib, "_STATUS_SEEN", {})
    monkeypatch.setattr(_lib, "_BAD_IDS_PTR", {})
    monkeypatch.setattr(_lib, "_STATUS_TOTALS", dict(_lib._STATUS_TOTALS))
    monkeypatch.setattr(torch, "zeros", make)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: Stream())
    monkeypatch.setattr(torch.cuda, "device", Guard)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])

    def both_inside():
        nonlocal barrier
        barrier = threading.Barrier(2)
    return log, state, both_inside


def test_two_threads_that_come_first_share_one_set_of_words(fake):
    """Both are held inside the allocation for as long as the other can get there."""
    log, _, both_inside = fake
    both_inside()
    got = []
    threads = [threading.Thread(target=lambda: got.append(_lib.bad_ids_ptr(0))) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    want = _lib._STATUS[0].data_ptr() + 4 * _lib.ST_BAD_IDS
    assert got == [want, want] and _lib._BAD_IDS_PTR == {0: want}
    assert log.count("zeros") == 1


def test_the_words_are_cleared_before_anyone_gets_them(fake):
    """Whatever stream counts into them first: their creation is waited for."""
    log, _, _ = fake
    _lib.status(torch.device("cuda", 0))
    _lib.status(torch.device("cuda", 0))
    _lib.bad_ids_ptr(0)
    assert log == ["zeros", "wait"]


def test_no_words_are_made_inside_a_capture(fake):
    log, state, _ = fake
    state["capturing"] = True
    assert _lib.bad_ids_ptr(0) == 0 and log == []
    state["capturing"] = False
    p = _lib.bad_ids_ptr(0)
    state["capturing"] = True
    assert p != 0 and _lib.bad_ids_ptr(0) == p


def test_polls_that_overtake_each_other_count_once(fake):
    """A poll that read the words before another one, and is settled after it, adds nothing and takes nothing back."""
    t = torch.zeros(_lib.STATUS_WORDS, dtype=torch.int32)
    early, late = [3, 0, 0, 0, 0, 2, 0, 0], [5, 1, 0, 0, 0, 2, 0, 0]
    assert _lib._status_delta(0, late) == late
    assert _lib._status_delta(0, early) == [0] * 8
    assert _lib._status_delta(0, late) == [0] * 8
    # past the words' 32 bits
    _lib._STATUS_SEEN[0] = [(1 << 31) - 1] * 8
    assert _lib._status_delta(0, [-(1 << 31) + 1] * 8) == [2] * 8
    assert t.numel() == 8


def test_ids_are_reported_beside_a_range_violation(fake, monkeypatch):
    monkeypatch.setenv("RSDF_RANGE_ERROR", "raise")
    _lib._STATUS[0] = torch.tensor([1, 0, 0, 0, 0, 4, 0, 0], dtype=torch.int32)
    with pytest.raises(_lib.RiseSdfHipError, match="non-finite") as e:
        _lib.poll_status(torch.device("cuda", 0))
    assert "4 rows named an id outside the table" in str(e.value)
    _lib.poll_status(torch.device("cuda", 0))                     # reported once
