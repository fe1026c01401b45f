"""Names of the kernels that a call launches, so that a test of a family of kernels can say that it reached it.

A profiler that has been in use for a while may miss what runs in its first milliseconds: a name that is wanted and missing is looked
for again, in new recordings of the same call behind some other work.  A kernel that the call does not launch is in none of them."""
import re
import time

import pytest
import torch
from torch.profiler import ProfilerActivity, profile

AGAIN = 2      # recordings of a call beyond the first
LEAD = 0.02    # seconds of other work in front of the call in these


def record(fn, lead=0.0):
    """-> what fn returns, the names of the kernels recorded"""
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        end = time.perf_counter() + lead
        while time.perf_counter() < end:
            torch.ones(64, device="cuda")
            torch.cuda.synchronize()
        out = fn()
        torch.cuda.synchronize()
    return out, {e.name for e in p.events() if e.device_type == torch.autograd.DeviceType.CUDA}


class Names(set):
    """The names recorded so far of the kernels of the call `fn`"""

    fn = None

    def again(self):
        self.update(record(self.fn, LEAD)[1])


def kernels_of(fn):
    out, first = record(fn)
    names = Names(first)
    names.fn = fn
    for _ in range(AGAIN):
        if names:
            return out, names
        names.again()
    if not names:
        pytest.skip("the profiler records no kernels here")
    return out, names


def launched(names, pattern):
    for left in range(AGAIN, -1, -1):
        if any(re.search(pattern, n) for n in names):
            return True
        if left:
            names.again()
    return False
