"""On a B200: moe_ops_status waits for its stream's work and for nothing else, and counts the products of both kinds once."""
import subprocess
import sys
import time

import pytest

from c0ven_b200 import MoEError, _lib, ops

pytestmark = pytest.mark.gpu
SECOND = 1_900_000_000  # clocks of a spinning kernel, about a second


def hear(stream):
    """A stream that asks for the first time is told of all there ever were, those that other tests counted by hand among them."""
    try:
        ops.status(stream)
    except MoEError as e:
        assert "gave up" in str(e)


@pytest.fixture
def blocking_stream():
    """A stream that waits for the default stream's work queued before its own, and the other way round (torch's do not)."""
    import ctypes

    import torch

    rt = torch.cuda.cudart()
    p = ctypes.c_void_p()
    assert int(rt.cudaStreamCreate(ctypes.addressof(p))) == 0
    yield p.value
    torch.cuda.synchronize()
    assert int(rt.cudaStreamDestroy(p.value)) == 0


def test_nothing_but_the_stream_is_waited_for(blocking_stream):
    """The stream has no work, while the default stream is busy for some 1.5 s: the answer comes at once."""
    import torch

    hear(blocking_stream)
    torch.cuda.synchronize()
    start = time.monotonic()
    torch.cuda._sleep(SECOND * 3 // 2)
    ops.status(blocking_stream, timeout_ms=200)
    asked = time.monotonic() - start
    torch.cuda.synchronize()
    slept = time.monotonic() - start
    assert slept > 1.0 and asked < 0.5, (asked, slept)


def test_the_wait_ends_when_it_says():
    import torch

    s = torch.cuda.Stream()
    hear(s.cuda_stream)
    with torch.cuda.stream(s):
        torch.cuda._sleep(SECOND)
    start = time.monotonic()
    with pytest.raises(MoEError) as e:
        ops.status(s.cuda_stream, timeout_ms=100)
    assert 0.05 < time.monotonic() - start < 0.5
    assert e.value.status == _lib.MOE_TIMEOUT and "did not finish" in str(e.value)
    s.synchronize()
    ops.status(s.cuda_stream)


def in_a_process_of_its_own(code):
    r = subprocess.run([sys.executable, "-c", PRODUCT + code + "\nprint('right')"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "right" in r.stdout, r.stderr[-2000:]


PRODUCT = """
import torch
from c0ven_b200 import MoEError, _lib, ops
w, x = torch.ones((1, 64, 64), dtype=torch.int8, device="cuda"), torch.ones((3, 64), dtype=torch.int8, device="cuda")
scales, y = torch.ones(64, device="cuda"), torch.zeros((3, 64), dtype=torch.float16, device="cuda")
torch.cuda.synchronize()
def product(stream=None):
    ops.i8_product_device(ops.I8Weights(1, 64, 64, w.data_ptr(), scales.data_ptr()), x.data_ptr(), scales.data_ptr(), 3, None, y.data_ptr(), ops.F16, stream=stream)
"""


def test_both_kinds_of_products_share_a_count():
    """A count raised by hand is told once, 8-bit products before and after it (in a process of its own, as streams that ask first hear of all there ever were)."""
    in_a_process_of_its_own("""
product()
ops.status()
assert _lib.lib().moe_ops_note_give_up(None) == _lib.MOE_OK
product()
try:
    ops.status()
    raise SystemExit("not told")
except MoEError as e:
    assert e.status == _lib.MOE_TIMEOUT and "gave up" in str(e)
product()
ops.status()
assert (y == 64).all()
""")


def test_a_first_call_inside_a_capture():
    """A process whose first call of all is captured: nothing had to be set up before, and the graph's result is right."""
    in_a_process_of_its_own("""
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    product(torch.cuda.current_stream().cuda_stream)
torch.cuda.synchronize()
assert (y == 0).all()
graph.replay()
torch.cuda.synchronize()
ops.status()
assert (y == 64).all()
""")
