"""The caller's grow-only scratch: a captured graph keeps the address of a buffer that it was given, so no buffer may go
while the workspace lives, whatever is asked of it afterwards."""

import torch

from dspine_amd.verify import Workspace

CPU = torch.device("cpu")


def test_a_larger_request_keeps_the_buffers_before_it():
    work, kept = Workspace(), set()
    for n in (100, 1000, 50, 5000, 5001):
        buf = work.get(n, CPU)
        assert buf.dtype == torch.uint8 and buf.numel() >= n
        kept.add(buf.data_ptr())
        del buf
    fresh = [torch.empty(n, dtype=torch.uint8) for n in (100, 1000, 5000) * 20]
    assert not kept & {t.data_ptr() for t in fresh}


def test_smaller_requests_get_the_same_buffer():
    work = Workspace()
    at = work.get(1000, CPU).data_ptr()
    assert all(work.get(n, CPU).data_ptr() == at for n in (1, 1000, 0, 999))


def test_buffers_kept_stay_below_twice_the_last():
    work, sizes = Workspace(), []
    for n in range(1, 3000, 7):
        size = work.get(n, CPU).numel()
        if not sizes or size != sizes[-1]:
            sizes.append(size)
    assert sum(sizes) < 2 * sizes[-1]


def test_devices_in_turn_find_their_buffers_again():
    """(A meta tensor stands for another device.)"""
    work, meta = Workspace(), torch.device("meta")
    a, b = work.get(64, CPU), work.get(64, meta)
    for _ in range(5):
        assert work.get(64, CPU) is a and work.get(64, meta) is b
