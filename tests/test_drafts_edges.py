"""Edges of the operators for drafted tokens without a GPU: what plans ask for."""
import os

import pytest

from ktir_cpu_amd import runtime as rt
from tests.test_drafts_host import attention
from tests.test_serving_host import Fake, cache

pytestmark = pytest.mark.skipif(not os.path.exists(rt.LIB_PATH), reason="libktir_hip.so not built")


@pytest.mark.parametrize("columns,held", [(64, 512), (128, 512), (192, 256), (256, 256)])
def test_one_sequence_is_cut_into_as_many_parts_as_the_chip_holds(columns, held):
    """32 rows of a KV head: sums of 4 wavefronts of 32 rows and up to 256 columns (+ 4) in f32, and b and l, are 36 to 134 KB of a CU's 160, so
    with more than 128 columns each of the 256 CUs holds one workgroup, not two."""
    assert (2 * 4 * 32 * 4 * (columns + 6) <= 160 * 1024) == (held == 512)
    for heads in (1, 2, 4, 8):
        shape = (8, heads * 4, columns)
        op = attention(cache(heads=heads, columns=columns), tokens=8, heads=heads * 4, seqs=1, max_q=8, max_k=1 << 20,
                       out=Fake(shape, "<f2", ptr=1 << 40))
        # (a head's bytes in the workspace are those of 32 rows, so this is the kernel of 32)
        assert op.workspace_bytes == op.desc.attn.splits * heads * 32 * (columns + 4) * 4 + 8
        assert op.desc.attn.splits * heads == held
