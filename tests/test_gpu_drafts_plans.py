"""Attention of drafted tokens by each of its plans: the bound on the keys and the batch choose the kernel, its tiles, how
many heads a workgroup has, and whether keys may be cut; small inputs reach all of them by that bound."""
import pytest
import torch

from ktir_cpu_amd import serving as S
from tests._serving import Batch
from tests.test_gpu_drafts import ATTN, attend, cache_of, check, dev, done, tree_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,hk,grp,D,page,code,dt,branch,window,pad,front", [c for c in ATTN if not c[8]])
@pytest.mark.parametrize("most", [6000, 1 << 20])
def test_a_longer_bound(lens, hk, grp, D, page, code, dt, branch, window, pad, front, most):
    b = Batch(lens, hk=hk, grp=grp, D=D, page=page, code=code, dt=dt, pad=pad, front=front, seed=D + branch)
    mask, _ = tree_of(b, branch, 0, seed=2, front=front, pad=pad)
    _, out, line = attend(b, mask, max_k=most)
    done()
    check(b, out, line, mask)


@pytest.mark.parametrize("D", [64, 80, 128, 192, 256])
@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("n,grp", [(5, 8), (20, 3), (33, 4), (61, 4), (80, 4)])
def test_tiles_of_many_rows_and_of_32(D, code, n, grp):
    b = Batch([(n, 700 + n), (1, 90), (n // 2, 300)], hk=2, grp=grp, D=D, page=16, code=code, dt="bf16", seed=D + n)
    mask, _ = tree_of(b, 3, 0)
    _, out, line = attend(b, mask, max_k=1 << 19)
    done()
    check(b, out, line, mask)


@pytest.mark.parametrize("n,grp,D,seqs,window", [(80, 4, 128, 30, 70), (80, 4, 64, 30, 33), (40, 4, 192, 60, 20), (8, 4, 128, 150, 40), (8, 4, 256, 300, 17)])
def test_windows_of_many_tiles(n, grp, D, seqs, window):
    g = torch.Generator().manual_seed(n)
    lens = [(n, n + int(torch.randint(0, 120, (), generator=g))) for _ in range(seqs)]
    b = Batch(lens, hk=1, grp=grp, D=D, page=16, code="i8", dt="f16", seed=n)
    mask, pos = tree_of(b, 4, window)
    _, out, line = attend(b, mask, pos, window=window)
    done()
    check(b, out, line, mask, window, pos)


# many tiles of few keys, of keys that may be many, and of more tiles than are cut; heads in fours, twos and ones
@pytest.mark.parametrize("hk,grp,n,D", [(8, 2, 3, 64), (8, 4, 8, 128), (6, 2, 12, 80), (5, 1, 4, 128), (4, 4, 6, 256), (2, 4, 5, 192), (4, 4, 16, 128)])
@pytest.mark.parametrize("most", [None, 2500, 50000])
def test_heads_together(hk, grp, n, D, most):
    g = torch.Generator().manual_seed(hk + n)
    lens = [(int(torch.randint(0, n + 1, (), generator=g)), 0) for _ in range(140)]
    lens = [(a, a + int(torch.randint(0, 60, (), generator=g))) for a, _ in lens]
    lens[3], lens[100] = (n, 260 + n), (n, 1100 if most else 400)
    b = Batch(lens, hk=hk, grp=grp, D=D, page=16, code="i8", dt="bf16", pad=3, front=2, seed=D)
    mask, _ = tree_of(b, 3, 0, front=2, pad=3)
    _, out, line = attend(b, mask, **({"max_k": most} if most else {}))
    done()
    check(b, out, line, mask)


@pytest.mark.parametrize("n,D", [(6, 128), (16, 64), (12, 256), (40, 128), (50, 256)])
@pytest.mark.parametrize("most", [2600, 1 << 19])
def test_a_nan_page_of_a_cut_tile_is_its_sequences_alone(n, D, most):
    b = Batch([(n, 2600), (n, 900)], hk=2, grp=4, D=D, page=16, code="i8", dt="f16", seed=n)
    mask, _ = tree_of(b, 3, 0)
    _, out, line = attend(b, mask, max_k=most)
    done()
    check(b, out, line, mask)
    page = int(b.table[1, 7])
    b.k_scale[page, 1] = b.v_scale[page, 1] = float("nan")
    _, got, gline = attend(b, mask, max_k=most)
    done()
    assert torch.equal(got[:n], out[:n]) and torch.equal(gline[:n], line[:n])
    assert torch.equal(got[n:, :4], out[n:, :4]) and got[n:, 4:].isnan().all()


@pytest.mark.parametrize("n,D", [(8, 128), (12, 64), (10, 256), (40, 128)])
def test_one_graph_whole_and_cut(n, D):
    # lengths change between the replays of two graphs that share a workspace: tiles are cut, stay whole, and are none
    b = Batch([(n, 4200), (n, 4000), (3, 3900)], hk=2, grp=4, D=D, page=16, code="i8", dt="bf16", seed=n)
    most = dict(max_q=n, max_k=4200)
    cache, _ = cache_of(b)
    q, table, q_start, kv_len = dev(b.q, *b.where())
    mask, _ = tree_of(b, 3, 0)
    at = dev(mask)
    out = [torch.empty_like(q) for _ in range(2)]
    line = [torch.empty(q.shape[:2], device="cuda") for _ in range(2)]
    first = S.KV8TreeAttention(cache, q, out[0], table, q_start, kv_len, at, lse=line[0], **most)
    space = torch.empty(max(16, first.desc.attn.ws_bytes), dtype=torch.uint8, device="cuda")
    ops = [S.KV8TreeAttention(cache, q, o, table, q_start, kv_len, at, lse=x, workspace=space, **most) for o, x in zip(out, line)]
    graphs = []
    for op in ops:
        op.run()
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            op.run()
    for lens in ((4200, 4000, 3900), (n, n, 3), (4200, n, 50), (300, 2000, 3), (n, 4000, 3900), (60, 70, 80), (4200, 4000, 3900)):
        b.kv_len = torch.tensor(lens, dtype=torch.int32)
        b.lens = [(a, k) for (a, _), k in zip(b.lens, lens)]
        kv_len.copy_(b.kv_len)
        for g, o, x in zip(graphs, out, line):
            o.fill_(7.0)
            x.fill_(7.0)
            g.replay()
            done()
            check(b, o, x, mask)
