"""Edges of the operators for drafted tokens on the GPU, by each of their kernels: scores of -inf, bounds above
the batch, places that no row sees, uneven batches, how many bits results keep."""
import math

import pytest
import torch

from tests._serving import Batch
from tests.test_gpu_drafts import attend, check, done, tree_of

pytestmark = pytest.mark.gpu

FAR = 1 << 19                  # a bound on the keys with which more than 64 rows of a KV head take the kernels for many rows
# new tokens, query heads of a KV head, columns, bound: tiles of 16 rows and of 32, of 128 rows (64 columns, and 256), of 256
# with half their wavefronts idle, and of 256
KERNELS = [(4, 2, 64, None), (4, 4, 128, None), (20, 2, 64, FAR), (20, 3, 128, FAR), (9, 4, 192, FAR), (30, 4, 64, FAR), (30, 4, 80, FAR),
           (80, 4, 64, FAR), (80, 4, 128, FAR), (40, 4, 256, FAR)]


@pytest.mark.parametrize("n,grp,D,most", KERNELS)
@pytest.mark.parametrize("dt,k", [("f16", 2600), ("bf16", 90)])
def test_attention_of_rows_whose_scores_are_all_minus_infinity(n, grp, D, most, dt, k):
    # such a row is NaN, as softmax has it, and one that sees nothing is 0, whole tiles and cut ones
    b = Batch([(n, n), (n, k + n), (n, n + 70)], hk=2, grp=grp, D=D, page=16, dt=dt, seed=n)
    b.k[..., 0] = b.k[..., 0].abs().clamp(min=1)
    b.q[::3, ::2, 0] = -math.inf
    mask, _ = tree_of(b, 3, 0)
    mask[1:n:2] = 0
    _, out, line = attend(b, mask, **({"max_k": most} if most else {}))
    done()
    none = torch.zeros(b.tokens, dtype=torch.bool)
    none[1:n:2] = True
    some = torch.zeros(b.tokens, 2 * grp, dtype=torch.bool)
    some[::3, ::2] = True
    assert (out.cpu()[none] == 0).all() and torch.isneginf(line.cpu()[none]).all()
    assert out.cpu()[some & ~none[:, None]].isnan().all()
    check(b, out, line, mask)
