"""Edges of the serving operators, on the GPU: how many bits results keep."""
import pytest
import torch

from tests import _serving as S
from tests.test_gpu_serving import attend, serving   # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


# ---- how many bits the weights of prompts keep ---------------------------------------

def sizes(b):
    """The batch with the values' sizes in V's place."""
    v = (b.v.view(torch.uint8) & 0x7f).view(b.v.dtype) if b.code == "e4m3" else b.v.abs()
    return b.k, v, b.k_scale, b.v_scale


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("hk,grp,D,page", [(16, 4, 128, 16), (16, 4, 80, 32), (16, 5, 64, 64), (16, 2, 256, 16)])
def test_weights_of_prompts(serving, hk, grp, D, page, code):  # noqa: F811
    """f16 results of short prompts are the exact ones rounded once, but for f32 sums: no
    weight is rounded to 16 bits on its way."""
    b = S.Batch([(130, 130), (90, 100), (120, 140)], hk=hk, grp=grp, D=D, page=page, code=code, seed=D)
    b.q = b.q * 0.125                                          # (scores near one another: what f32 loses of them is small)
    heads = [0, grp, hk * grp - 1]
    out, _ = attend(serving, b)
    want, _, bound, _ = S.attention(b.q, *b.cache(), *b.where(), scale=D ** -0.5, heads=heads)
    size = S.attention(b.q, *sizes(b), *b.where(), scale=D ** -0.5, heads=heads)[0]
    # `bound` has 2^-11 of every weight; two f16 terms leave 2^-11 of 2^-11
    bound = bound - size * (2.0 ** -11 - 2.0 ** -22)
    S.close(out[:, heads], want[:, heads], bound[:, heads], "f16")
