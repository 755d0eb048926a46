"""Edges of the operators for drafted tokens without a GPU: what plans ask for, and what the tests' bounds tell apart."""
import math
import os

import pytest
import torch

from ktir_cpu_amd import runtime as rt
from tests import _drafts as P
from tests._serving import close
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


@pytest.mark.parametrize("n,grp,D,k", [(4, 4, 64, 60), (30, 4, 80, 60), (80, 4, 128, 1100)])
@pytest.mark.parametrize("terms,kept", [([torch.float16], False), ([torch.bfloat16], False), ([torch.bfloat16] * 2, True), ([torch.float16] * 2, True)])
def test_the_bound_on_weights_tells_one_term_from_two(n, grp, D, k, terms, kept):
    """Weights rounded to 16 bits once fail the bound that the GPU test puts on the same batch; those of two terms are within it."""
    from tests.test_gpu_drafts_edges import tree_of, two_weights, weights_bound
    b = two_weights(n, grp, D, k, seed=n)
    mask, _ = tree_of(b, 3, 0)
    want, bound = weights_bound(b, mask)
    keys, values = ((c.double() * s.double()[:, None, :, None])[b.table[0].long()].reshape(-1, 2, D)[:k + n] for c, s in ((b.k, b.k_scale), (b.v, b.v_scale)))
    see, out = P.seen_of(mask, n, k + n, 0, None), torch.zeros_like(want)
    for h in range(2 * grp):
        u = (b.q[:n, h].double() @ keys[:, h // grp].T).masked_fill(~see, -math.inf) * math.log2(math.e)
        w = torch.exp2(u - u.amax(1, keepdim=True) + 10.6).float()
        rounded = torch.zeros_like(w)
        for t in terms:
            rounded = rounded + (w - rounded).to(t).float()
        out[:, h] = rounded.double() @ values[:, h // grp] / w.double().sum(1, keepdim=True)
    if kept:
        close(out.half(), want, bound, "f16")
    else:
        with pytest.raises(AssertionError):
            close(out.half(), want, bound, "f16")
