"""Edges of the serving operators without a GPU: where a handle's runs go, and which
overlaps are refused."""
import os

import pytest

from ktir_cpu_amd import runtime as rt
from tests.test_serving_host import append, attention, rope

pytestmark = pytest.mark.skipif(not os.path.exists(rt.LIB_PATH), reason="libktir_hip.so not built")


# ---- streams -------------------------------------------------------------------------

@pytest.mark.parametrize("make", [rope, append, attention])
def test_a_run_without_a_stream_goes_to_the_library_s(make):
    """Also after one on a stream of the caller's."""
    op, went = make(), []
    op._call = lambda ref: went.append(op.desc.stream) or 0          # nothing launches
    for stream in (None, 7 << 40, None, 0, None):
        op.run(stream)
    assert went == [0, 7 << 40, 0, rt.K["KTIR_STREAM_NULL"], 0]
