"""Which kernels a call launches, for tests that are about one of them: rules on sizes choose a kernel, and a test whose call has left its kernel fails."""
import re

import pytest
import torch


def launched(call):
    """(the call's result, names of the kernels with their template arguments)"""
    call()  # (loads them)
    torch.cuda.synchronize()
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU, torch.profiler.ProfilerActivity.CUDA]) as trace:
        result = call()
        torch.cuda.synchronize()
    names = [e.name for e in trace.events() if "kernel" in e.name]
    if not names:
        pytest.skip("this machine lets no process trace its kernels")
    return result, names


def _argument(a):
    return ("(?:true|1)" if a else "(?:false|0)") if isinstance(a, bool) else str(a)


def through(call, kernel, *arguments):
    """The call's result; `kernel` with these template arguments, behind its element type if it has one, is among what it launches."""
    result, names = launched(call)
    wanted = rf"\b{kernel}<(?:[a-zA-Z_]\w*, )?" + ", ".join(map(_argument, arguments)) + ">"
    assert any(re.search(wanted, re.sub(r"\((?:int|bool)\)", "", name)) for name in names), (wanted, names)
    return result
