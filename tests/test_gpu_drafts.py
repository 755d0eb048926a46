"""The operators for drafted tokens on the GPU: against plain implementations in float64
(tests/_drafts.py), and what goes to the cache bit for bit."""
import math

import numpy as np
import pytest
import torch

from ktir_cpu_amd import serving as S
from tests import _drafts as P
from tests._serving import DT, TOP, Batch, append, close, rope

pytestmark = pytest.mark.gpu


def dev(*tensors):
    out = [t.cuda() if isinstance(t, torch.Tensor) else t for t in tensors]
    return out if len(out) > 1 else out[0]


def done():
    """Waits, and raises what the kernels found."""
    from ktir_cpu_amd import runtime as rt
    torch.cuda.synchronize()
    rt.sync()


def same_bits(a, b, what=""):
    a, b = a.cpu().contiguous(), b.cpu().contiguous()
    if a.dtype == torch.float32:
        nan = a.isnan() & b.isnan()
        assert torch.equal(torch.where(nan, 0.0, a), torch.where(nan, 0.0, b)), what
    else:
        x, y = a.view(torch.uint8), b.view(torch.uint8)
        assert torch.equal(x, y), (what, int((x != y).sum()), x.numel())


def cache_of(b):
    arrays = dev(*b.cache())
    return S.KV8Cache(*arrays), arrays


# ---- the tree -----------------------------------------------------------------------

TREES = [([(1, 1)], 1, 1, 0), ([(7, 20), (0, 5), (1, 1), (33, 33)], 3, 2, 0), ([(64, 900)] * 3, 8, 2, 0),
         ([(100, 100), (31, 64), (32, 64), (65, 64 + 65)], 2, 4, 5), ([(1024, 2000), (5, 5), (1000, 1000)], 1, 32, 0),
         ([(1024, 1024)], 1, 32, 700), ([(700, 4000), (1024, 5000)], 300, 32, 1), ([(257, 300)] * 70, 20, 9, 64)]


@pytest.mark.parametrize("lens,branch,words,window", TREES)
def test_tree(lens, branch, words, window):
    b = Batch(lens, front=2, pad=3, hk=1, D=16)
    parents = P.random_parents(lens, branch, seed=len(lens), front=2, pad=3)
    wide = torch.full((b.tokens, words + 1), -3, dtype=torch.int32)
    mask, pos = wide[:, :words], torch.full((b.tokens,), -5, dtype=torch.int32)
    want = P.tree(parents, b.q_start, b.kv_len, words, window, mask, pos)
    wide_d, pos_d = dev(wide, pos)
    S.DraftTree(dev(parents), *dev(b.q_start, b.kv_len), wide_d[:, :words], pos_d, window=window).run()
    done()
    assert torch.equal(wide_d[:, :words].cpu(), want[0]) and torch.equal(pos_d.cpu(), want[1])
    assert (wide_d[:, words:] == -3).all()


def test_tree_refuses_parents_that_are_none():
    lens = [(9, 30), (4, 4)]
    b = Batch(lens, hk=1, D=16)
    parents = P.random_parents(lens, 2)
    parents[5], parents[7], parents[10] = 6, -2, 1         # later, below, the token itself
    mask, pos = torch.zeros((13, 1), dtype=torch.int32), torch.zeros(13, dtype=torch.int32)
    want = P.tree(parents, b.q_start, b.kv_len, 1, 0, mask, pos)
    mask_d, pos_d = dev(mask, pos)
    op = S.DraftTree(dev(parents), *dev(b.q_start, b.kv_len), mask_d, pos_d)
    op.run()
    with pytest.raises(IndexError):
        done()
    assert torch.equal(mask_d.cpu(), want[0]) and torch.equal(pos_d.cpu(), want[1])
    done()


def test_tree_leaves_out_what_is_too_long():
    lens = [(33, 40), (32, 40), (3, 2)]
    b = Batch([(33, 40), (32, 40), (3, 3)], hk=1, D=16)
    parents = P.random_parents(lens, 1)
    mask, pos = torch.full((68, 1), -3, dtype=torch.int32), torch.full((68,), -5, dtype=torch.int32)
    mask_d, pos_d = dev(mask, pos)
    S.DraftTree(dev(parents), *dev(b.q_start, b.kv_len), mask_d, pos_d).run()
    with pytest.raises(IndexError):
        done()
    want = P.tree(parents, b.q_start, b.kv_len, 2, 0, mask.repeat(1, 2), pos)
    assert (mask_d[:33] == -3).all() and (pos_d[:33] == -5).all()
    assert torch.equal(mask_d[33:].cpu(), want[0][33:, :1]) and torch.equal(pos_d[33:].cpu(), want[1][33:])


# ---- rotation and append ----------------------------------------------------------------

def freq_of(rot):
    return torch.as_tensor(S.rope_frequencies(rot, 10000.0)[0])


TURNS = [
    # lens, hk, grp, D, rot, page, code, dt, interleaved, positions, pad, front
    ([(1, 1)], 1, 1, 16, 2, 16, "i8", "f16", False, None, 0, 0),
    ([(1, 1000)], 8, 4, 128, 128, 16, "i8", "bf16", False, None, 0, 0),
    ([(1, 17), (1, 16), (1, 1), (0, 40), (1, 33)], 2, 3, 80, 20, 16, "e4m3", "bf16", True, "i32", 2, 3),
    ([(40, 40), (3, 18), (16, 32), (17, 64)], 3, 2, 80, 20, 16, "i8", "f16", False, "i64", 1, 0),
    ([(100, 300), (5, 70)], 2, 7, 64, 64, 64, "e4m3", "f16", True, "i32", 0, 1),
    ([(70, 71), (300, 300)], 1, 2, 256, 128, 256, "i8", "bf16", False, None, 4, 0),
    ([(33, 50), (2, 500)], 2, 1, 192, 6, 128, "e4m3", "bf16", False, "i32", 0, 0),
    ([(20, 90)], 4, 1, 96, 96, 32, "i8", "f16", True, "i64", 3, 2),
    ([(37, 90)], 1, 5, 112, 70, 32, "i8", "bf16", True, "i64", 0, 0),
    ([(513, 600)], 2, 2, 128, 64, 16, "e4m3", "f16", False, None, 0, 0),
]


@pytest.mark.parametrize("lens,hk,grp,D,rot,page,code,dt,inter,given,pad,front", TURNS)
@pytest.mark.parametrize("place", [False, True])
def test_turn_and_append(lens, hk, grp, D, rot, page, code, dt, inter, given, pad, front, place):
    b = Batch(lens, hk=hk, grp=grp, D=D, page=page, code=code, dt=dt, pad=pad, front=front, seed=D + rot)
    freq, amp = freq_of(rot), 1.25
    where = P.places(b.q_start, b.kv_len, b.tokens)
    live = where >= 0
    pos = where if given is None else torch.randint(0, 1 << 17, (b.tokens,), generator=torch.Generator().manual_seed(1))
    pos = torch.where(live, pos, -9)                      # of tokens outside the sequences: not looked at
    k = P.turned(b.new_k, pos.clamp(min=0), freq, inter, amp)
    want_k = append(k, b.k, b.k_scale, code, page, *b.where())
    want_v = append(b.new_v, b.v, b.v_scale, code, page, *b.where())
    cache, arrays = cache_of(b)
    # queries, keys and values as parts of one projection's rows
    qkv = dev(torch.cat([b.q, b.new_k, b.new_v], 1))
    hq = hk * grp
    q = qkv[:, :hq]
    before = q.clone()
    out = None if place else torch.full(b.q.shape, 3.0, dtype=DT[dt], device="cuda")
    given = None if given is None else dev(pos.to(torch.int32 if given == "i32" else torch.int64))
    op = S.KV8RopeAppend(cache, q, qkv[:, hq:hq + hk], qkv[:, hq + hk:], dev(freq), *dev(*b.where()), out, positions=given,
                         interleaved=inter, amplitude=amp)
    op.run()
    done()
    for got, want, what in zip(arrays, (want_k[0], want_v[0], want_k[1], want_v[1]), ("k", "v", "k_scale", "v_scale")):
        same_bits(got, want, what)
    got = q if place else out
    want, bound = rope(b.q, pos.clamp(min=0), freq, interleaved=inter, amplitude=amp)
    close(got[live], want[live], bound[live], dt)
    untouched = before if place else torch.full_like(out, 3.0)
    same_bits(got[~live], untouched[~live], "rows outside the sequences")
    same_bits(qkv[:, hq:], torch.cat([b.new_k, b.new_v], 1), "keys and values are inputs")
    # and the same bits as the rotation by itself
    alone = torch.empty_like(before)
    S.Rope(before.contiguous(), dev(pos), dev(freq), alone, interleaved=inter, amplitude=amp).run()
    done()
    same_bits(got[live], alone[live], "queries")


def test_turn_odd_strides():
    # rows off 16-byte bounds, heads behind tokens, a cache with keys and values in one allocation
    lens = [(19, 40), (1, 77)]
    b = Batch(lens, hk=2, grp=2, D=48, page=16, code="i8", dt="bf16", seed=3)
    freq = freq_of(48)
    where = P.places(b.q_start, b.kv_len, b.tokens)
    both = torch.zeros((b.pages, b.page, 2, 2, 48), dtype=torch.int8)
    both[:, :, 0], both[:, :, 1] = b.k, b.v
    both = dev(both)
    scales = dev(torch.stack([b.k_scale, b.v_scale], 2))
    cache = S.KV8Cache(both[:, :, 0], both[:, :, 1], scales[:, :, 0], scales[:, :, 1])

    def odd(x):                     # [tokens, heads, columns] with heads outermost, rows of columns + 3
        y = torch.zeros((x.shape[1], x.shape[0], x.shape[2] + 3), dtype=x.dtype, device="cuda")
        y[..., 1:-2] = dev(x.transpose(0, 1).contiguous())
        return y[..., 1:-2].transpose(0, 1)
    q = odd(b.q)
    S.KV8RopeAppend(cache, q, odd(b.new_k), odd(b.new_v), dev(freq), *dev(*b.where())).run()
    done()
    want_k = append(P.turned(b.new_k, where, freq, False, 1.0), b.k, b.k_scale, "i8", 16, *b.where())
    want_v = append(b.new_v, b.v, b.v_scale, "i8", 16, *b.where())
    same_bits(both[:, :, 0], want_k[0])
    same_bits(both[:, :, 1], want_v[0])
    same_bits(scales[:, :, 0], want_k[1])
    same_bits(scales[:, :, 1], want_v[1])
    want, bound = rope(b.q, where, freq)
    close(q, want, bound, "bf16")


@pytest.mark.parametrize("code", ["i8", "e4m3"])
def test_turn_values_that_are_not_finite(code):
    lens = [(20, 40)]
    b = Batch(lens, hk=2, grp=1, D=64, page=16, code=code, dt="f16", seed=4)
    b.new_k[3, 0, 5] = math.inf           # (turned into infinities and NaN)
    b.new_k[19, 1, 63] = math.nan
    b.new_v[0, 1, 0] = -math.inf
    freq = freq_of(32)
    where = P.places(b.q_start, b.kv_len, b.tokens)
    cache, arrays = cache_of(b)
    S.KV8RopeAppend(cache, *dev(b.q, b.new_k, b.new_v, freq, *b.where())).run()
    done()
    want_k = append(P.turned(b.new_k, where, freq, False, 1.0), b.k, b.k_scale, code, 16, *b.where())
    want_v = append(b.new_v, b.v, b.v_scale, code, 16, *b.where())
    assert want_k[1].isnan().sum() == 2 and want_v[1].isnan().sum() == 1
    for got, want in zip(arrays, (want_k[0], want_v[0], want_k[1], want_v[1])):
        same_bits(got, want)


def test_turn_out_of_range():
    """Pages that there are not, a table that ends, and positions below 0: the error word, and nothing else is written."""
    lens = [(20, 40), (10, 100), (5, 30)]
    b = Batch(lens, hk=1, grp=2, D=32, page=16, seed=5)
    freq = freq_of(32)
    where = P.places(b.q_start, b.kv_len, b.tokens)
    pos = where.clone()
    pos[30:] = torch.tensor([3, -1, -4, 7, 8])
    want_pos = pos.clamp(min=0)
    table = b.table.clone()
    table[0, 1] = b.pages                      # its tokens 20 to 31
    short = table[:, :6].contiguous()          # sequence 1 ends at 96 of 100
    kv = torch.tensor([40, 96, 30], dtype=torch.int32)
    cache, arrays = cache_of(b)
    q = dev(b.q)
    op = S.KV8RopeAppend(cache, q, *dev(b.new_k, b.new_v, freq, short, b.q_start, b.kv_len), positions=dev(pos))
    op.run()
    with pytest.raises(IndexError):
        done()
    k = P.turned(b.new_k, want_pos, freq, False, 1.0)
    # what is stored: sequence 0's tokens 32 to 39, sequence 1's 90 to 95, sequence 2's
    part_start, part_kv = torch.tensor([12, 20, 26, 30], dtype=torch.int32), kv
    keep_rows = torch.cat([torch.arange(0, 26), torch.arange(30, 35)])
    rows = torch.cat([torch.arange(12, 26), torch.arange(30, 35)])
    starts = torch.tensor([0, 8, 14, 19], dtype=torch.int32)
    want_k = append(k[rows], b.k, b.k_scale, "i8", 16, b.table, starts, part_kv)
    want_v = append(b.new_v[rows], b.v, b.v_scale, "i8", 16, b.table, starts, part_kv)
    for got, want in zip(arrays, (want_k[0], want_v[0], want_k[1], want_v[1])):
        same_bits(got, want)
    same_bits(q[26:30], b.q[26:30], "queries past the table")
    want, bound = rope(b.q, want_pos, freq)
    close(q[rows], want[rows], bound[rows], "f16")
    assert len(part_start) == 4 and len(keep_rows) == 31
    done()


# ---- attention ------------------------------------------------------------------------------

ATTN = [
    # lens, hk, grp, D, page, code, dt, branch, window, pad, front
    ([(1, 1)], 1, 1, 16, 16, "i8", "f16", 1, 0, 0, 0),
    ([(8, 1000)], 8, 4, 128, 16, "i8", "f16", 3, 0, 0, 0),
    ([(5, 5), (0, 30), (1, 200), (8, 63), (3, 64)], 2, 4, 128, 16, "i8", "bf16", 2, 0, 2, 1),
    ([(16, 300), (7, 31), (2, 18)], 2, 4, 64, 32, "e4m3", "f16", 4, 0, 0, 0),
    ([(64, 2000)], 2, 4, 128, 64, "e4m3", "bf16", 8, 0, 0, 0),
    ([(100, 900), (31, 64), (1, 500), (90, 90)], 3, 7, 80, 32, "i8", "f16", 5, 100, 4, 2),
    ([(33, 500), (20, 40)], 1, 3, 192, 16, "i8", "bf16", 3, 0, 0, 0),
    ([(40, 300), (3, 77)], 2, 2, 256, 16, "e4m3", "f16", 6, 30, 1, 0),
    ([(300, 1200), (129, 129)], 1, 2, 96, 256, "i8", "bf16", 16, 0, 0, 3),
    ([(512, 513), (17, 4000)], 1, 1, 128, 16, "i8", "f16", 30, 0, 0, 0),
    ([(1024, 1100)], 1, 1, 64, 128, "e4m3", "bf16", 200, 0, 0, 0),
    ([(4, 60)] * 40, 2, 8, 128, 16, "i8", "bf16", 2, 0, 0, 0),
    ([(12, 5000), (60, 1500)], 4, 5, 112, 16, "i8", "f16", 4, 0, 3, 0),
]


def attend(b, mask, positions=None, lse=True, out=None, q=None, **kw):
    cache, _ = cache_of(b)
    q = dev(b.q) if q is None else q
    out = torch.full(b.q.shape, 7.0, dtype=DT[b.dt], device="cuda") if out is None else out
    line = torch.full(b.q.shape[:2], 7.0, device="cuda") if lse else None
    op = S.KV8TreeAttention(cache, q, out, *dev(*b.where()), dev(mask), positions=None if positions is None else dev(positions),
                            lse=line, **{**b.most, **kw})
    op.run()
    return op, out, line


def check(b, out, line, mask, window=0, positions=None, scale=None):
    scale = b.D ** -0.5 if scale is None else scale
    want, wline, bound, lbound = P.attention(b.q, *b.cache(), *b.where(), mask, scale=scale, window=window, positions=positions)
    live = P.places(b.q_start, b.kv_len, b.tokens) >= 0
    close(out[live.to(out.device)], want[live], bound[live], b.dt)
    g, w = line.double().cpu()[live], wline[live]
    none = torch.isinf(w)
    assert torch.equal(torch.isinf(g) & (g < 0), none)
    assert ((g - w).abs()[~none] <= lbound[live][~none]).all()
    assert (out.cpu()[~live] == 7.0).all() and (line.cpu()[~live] == 7.0).all()


def tree_of(b, branch, window, seed=0, front=0, pad=0, words=None):
    parents = P.random_parents(b.lens, branch, seed=seed, front=front, pad=pad)
    words = words or max(1, -(-max(n for n, _ in b.lens) // 32))
    return P.tree(parents, b.q_start, b.kv_len, words, window, torch.zeros((b.tokens, words), dtype=torch.int32),
                  torch.zeros(b.tokens, dtype=torch.int32))


@pytest.mark.parametrize("lens,hk,grp,D,page,code,dt,branch,window,pad,front", ATTN)
def test_attention(lens, hk, grp, D, page, code, dt, branch, window, pad, front):
    b = Batch(lens, hk=hk, grp=grp, D=D, page=page, code=code, dt=dt, pad=pad, front=front, seed=D + branch)
    mask, pos = tree_of(b, branch, window, seed=2, front=front, pad=pad)
    _, out, line = attend(b, mask, pos if window else None, window=window)
    done()
    check(b, out, line, mask, window, pos)


@pytest.mark.parametrize("rows", [(3, 2), (30, 4), (90, 4), (200, 1)])
def test_attention_any_mask_and_rows_that_see_nothing(rows):
    # masks that are no tree's, words more than it takes, sequences without tokens before, rows of zeros
    n, grp = rows
    b = Batch([(n, n), (n, n + 70), (1, 1), (n, n)], hk=2, grp=grp, D=64, page=16, seed=n)
    g = torch.Generator().manual_seed(n)
    words = -(-n // 32) + 1
    mask = torch.randint(-(1 << 31), 1 << 31, (b.tokens, words), generator=g, dtype=torch.int64).to(torch.int32)
    mask[::3] = 0
    _, out, line = attend(b, mask)
    done()
    check(b, out, line, mask)
    empty = out[:n][::3]
    assert (empty == 0).all() and torch.isneginf(line[:n][::3]).all()


@pytest.mark.parametrize("n,grp,window", [(6, 2, 1), (40, 4, 33), (80, 4, 100), (8, 4, 7)])
def test_attention_window(n, grp, window):
    # windows within the draft, and pages before the first new token's window that are gone
    b = Batch([(n, 700), (n, n + 5), (1, 400), (n, n)], hk=2, grp=grp, D=128, page=32, seed=window)
    mask, pos = tree_of(b, 2, window, seed=5)
    for s, (new, kv) in enumerate(b.lens):
        gone = max(0, kv - new - window + 1) // b.page
        keep = b.table[s, :gone].clone()
        b.table[s, :gone] = -1
        assert len(keep) == gone
    want = Batch([(n, 700), (n, n + 5), (1, 400), (n, n)], hk=2, grp=grp, D=128, page=32, seed=window)
    _, out, line = attend(b, mask, pos, window=window)
    done()
    check(want, out, line, mask, window, pos)


@pytest.mark.parametrize("n,grp", [(4, 4), (12, 4), (70, 4)])
def test_attention_of_a_line_is_causal_attention(n, grp):
    b = Batch([(n, 500), (1, 77)], hk=2, grp=grp, D=128, page=16, dt="bf16", seed=n)
    mask, _ = tree_of(b, 1, 0)
    _, out, line = attend(b, mask)
    cache, _ = cache_of(b)
    other, oline = torch.empty_like(out), torch.empty_like(line)
    S.KV8Attention(cache, dev(b.q), other, *dev(*b.where()), lse=oline, **b.most).run()
    done()
    want, wline, bound, lbound = P.attention(b.q, *b.cache(), *b.where(), mask, scale=128 ** -0.5)
    # each is within its bound and half a step of the line
    far = (out.double() - other.double()).abs().cpu() - (2 * bound + want.abs() * 2.0 ** -7 * (1 + 2.0 ** -7))
    assert far.max() <= 0
    assert ((line - oline).abs().cpu() <= 2 * lbound).all()


@pytest.mark.parametrize("n,grp", [(5, 2), (20, 2), (90, 4)])
def test_attention_masked_places_are_not_looked_at(n, grp):
    # tokens that no row sees hold NaN and infinite scales and codes: pages of their own, and the last page's rows behind the last token
    b = Batch([(n, 16 * 9 + n)], hk=2, grp=grp, D=64, page=16, code="e4m3", seed=n)
    mask, pos = tree_of(b, 2, 17, seed=1)
    window = 17
    want_cache = [x.clone() for x in b.cache()]
    at = int(b.table[0, 3])                       # whole pages before every window
    b.k_scale[at], b.v_scale[at] = math.nan, math.inf
    b.k.view(torch.uint8)[at] = 0x7f
    b.v.view(torch.uint8)[at] = 0x7f
    last, end = int(b.table[0, (16 * 9 + n - 1) // 16]), (16 * 9 + n - 1) % 16 + 1
    b.k.view(torch.uint8)[last, end:] = 0x7f
    b.v.view(torch.uint8)[last, end:] = 0xff
    _, out, line = attend(b, mask, pos, window=window)
    done()
    b.k, b.v, b.k_scale, b.v_scale = want_cache
    check(b, out, line, mask, window, pos)


@pytest.mark.parametrize("n,grp", [(6, 4), (80, 4)])
def test_attention_in_place_strides_and_scale(n, grp):
    b = Batch([(n, 150), (n - 1, 90)], hk=2, grp=grp, D=80, page=16, dt="f16", seed=9)
    mask, _ = tree_of(b, 3, 0)
    want = P.attention(b.q, *b.cache(), *b.where(), mask, scale=-0.3)
    heads = 2 * grp
    wide = torch.zeros((b.tokens, heads + 1, 83), dtype=torch.float16, device="cuda")
    q = wide[:, :heads, 1:81]
    q.copy_(dev(b.q))
    line = torch.zeros((heads, b.tokens), device="cuda").t()
    wide_mask = torch.full((b.tokens, mask.shape[1] + 2), -1, dtype=torch.int32, device="cuda")
    wide_mask[:, :mask.shape[1]] = dev(mask)
    cache, _ = cache_of(b)
    S.KV8TreeAttention(cache, q, q, *dev(*b.where()), wide_mask[:, :mask.shape[1]], scale=-0.3, lse=line, **b.most).run()
    done()
    close(q, want[0], want[2], "f16")
    assert ((line.cpu() - want[1]).abs() <= want[3]).all()
    assert (wide[:, heads] == 0).all() and (wide[:, :, 0] == 0).all() and (wide[:, :, 81:] == 0).all()


@pytest.mark.parametrize("n,grp,k", [(8, 4, 70000), (64, 4, 40000)])
def test_attention_long(n, grp, k):
    b = Batch([(n, k), (3, 900)], hk=1, grp=grp, D=128, page=64, code="e4m3", dt="bf16", seed=7)
    mask, _ = tree_of(b, 5, 0)
    _, out, line = attend(b, mask)
    done()
    check(b, out, line, mask)


def test_attention_out_of_range():
    # more new tokens than max_q, more cached than max_k, a page that there is not
    for change in ("max_q", "max_k", "page"):
        b = Batch([(10, 200), (4, 100)], hk=1, grp=2, D=64, page=16, seed=6)
        mask, _ = tree_of(b, 2, 0)
        kw = {}
        if change == "page":
            b.table[0, 2] = b.pages + 5
        else:
            kw[change] = 9 if change == "max_q" else 150
        _, out, line = attend(b, mask, **kw)
        with pytest.raises(IndexError):
            done()
        done()
        clean = Batch([(10, 200), (4, 100)], hk=1, grp=2, D=64, page=16, seed=6)
        want, wline, bound, _ = P.attention(clean.q, *clean.cache(), *clean.where(), mask, scale=64 ** -0.5)
        close(out[10:], want[10:], bound[10:], "f16")
        if change == "max_q":
            close(out[:9], want[:9], bound[:9], "f16")
            assert (out[9] == 7).all()


# ---- the kept path ------------------------------------------------------------------------------

def paths(b, branch, seed, most=None):
    """A line of each sequence's tree, cut somewhere."""
    g = torch.Generator().manual_seed(seed)
    parents = P.random_parents(b.lens, branch, seed=seed)
    depth = max(max(n for n, _ in b.lens), 1)
    path, kept = torch.full((len(b.lens), depth), -1, dtype=torch.int32), []
    for s, (n, _) in enumerate(b.lens):
        start = int(b.q_start[s])
        lines = P.family(parents[start:start + n].tolist())
        line = sorted(lines[int(torch.randint(0, n, (), generator=g))]) if n else []
        line = line[:most] if most else line
        path[s, :len(line)] = torch.tensor(line, dtype=torch.int32)
        kept.append(len(line))
    return path, torch.tensor(kept, dtype=torch.int32)


KEEPS = [([(1, 1)], 1, 16, 16, "i8", 1), ([(16, 1016)], 8, 128, 16, "i8", 3), ([(64, 100), (0, 7), (5, 16), (40, 40), (64, 1000)], 2, 80, 16, "i8", 4),
         ([(64, 100), (0, 7), (5, 16), (40, 40), (64, 1000)], 2, 80, 16, "e4m3", 2), ([(200, 300), (300, 300)], 1, 256, 32, "i8", 3),
         ([(500, 900), (100, 120)], 3, 64, 256, "e4m3", 2), ([(9, 40)] * 70, 5, 192, 16, "i8", 3), ([(100, 111)] * 3, 2, 16, 64, "i8", 1)]


@pytest.mark.parametrize("lens,hk,D,page,code,branch", KEEPS)
@pytest.mark.parametrize("spread", [0.0, 1.0])
def test_keep(lens, hk, D, page, code, branch, spread):
    b = Batch(lens, hk=hk, D=D, page=page, code=code, seed=D + page, spread=spread)
    path, kept = paths(b, branch, seed=branch + page)
    cache, arrays = cache_of(b)
    S.KV8Keep(cache, *dev(*b.where(), path, kept)).run()
    done()
    for codes, scale, got, gscale in ((b.k, b.k_scale, arrays[0], arrays[2]), (b.v, b.v_scale, arrays[1], arrays[3])):
        want, wscale, live = P.keep(codes, scale, code, page, *b.where(), path, kept)
        same_bits(got.cpu()[live], want[live])
        same_bits(gscale, wscale)


def test_keep_values():
    """A kept entry's value moves by half a step of its code for each rounding: its own, where its page is another."""
    b = Batch([(60, 300), (33, 48)], hk=2, D=64, page=16, code="i8", seed=1, spread=1.0)
    path, kept = paths(b, 4, seed=3)
    cache, arrays = cache_of(b)
    S.KV8Keep(cache, *dev(*b.where(), path, kept)).run()
    done()
    for s, (n, kv) in enumerate(b.lens):
        for i in range(int(kept[s])):
            to, src = kv - n + i, kv - n + int(path[s, i])
            a, c = int(b.table[s, to // 16]), int(b.table[s, src // 16])
            for codes, scale, got, gscale in ((b.k, b.k_scale, arrays[0], arrays[2]), (b.v, b.v_scale, arrays[1], arrays[3])):
                old = codes[c, src % 16].double() * scale[c].double()[:, None]
                new = got[a, to % 16].double().cpu() * gscale[a].double().cpu()[:, None]
                assert ((new - old).abs() <= gscale[a].double().cpu()[:, None] * (0.5 + 2.0 ** -15)).all()


@pytest.mark.parametrize("code", ["i8", "e4m3"])
def test_keep_scales_and_codes_that_are_not_finite(code):
    b = Batch([(40, 60), (40, 60), (30, 46)], hk=2, D=32, page=16, code=code, seed=2)
    path = torch.full((3, 10), -1, dtype=torch.int32)
    path[0, :6] = torch.tensor([0, 5, 13, 20, 30, 39])
    path[1, :10] = torch.tensor([1, 2, 3, 4, 14, 15, 16, 28, 29, 35])
    path[2, :2] = torch.tensor([17, 29])
    kept = torch.tensor([6, 10, 2], dtype=torch.int32)
    b.k_scale[int(b.table[0, 2]), 0] = math.nan       # comes to the first page
    b.v_scale[int(b.table[0, 1]), 1] = math.nan       # stays in its page
    b.k_scale[int(b.table[1, 3]), 1] = math.inf
    b.v_scale[int(b.table[2, 2])] = 0.0
    if code == "e4m3":
        b.k.view(torch.uint8)[int(b.table[1, 2]), 2:7, 0, 3] = 0x7f
        b.v.view(torch.uint8)[int(b.table[2, 2]), :, 1, 5] = 0xff
    cache, arrays = cache_of(b)
    S.KV8Keep(cache, *dev(*b.where(), path, kept)).run()
    done()
    for codes, scale, got, gscale in ((b.k, b.k_scale, arrays[0], arrays[2]), (b.v, b.v_scale, arrays[1], arrays[3])):
        want, wscale, live = P.keep(codes, scale, code, 16, *b.where(), path, kept)
        same_bits(gscale, wscale)
        nan = want.float().isnan() & got.cpu().float().isnan()
        x, y = (torch.where(nan, 0, t.cpu().contiguous().view(torch.uint8)) for t in (got, want))
        assert torch.equal(x[live], y[live])


def test_keep_out_of_range():
    """Paths that do not rise, leave their sequence, are too long, or reach a page that there is not: cut there."""
    lens = [(20, 52)] * 6
    good = torch.tensor([[0, 3, 9, 17, 19], [0, 3, 9, 17, 19], [0, 3, 9, 17, 19], [0, 3, 9, 17, 19], [0, 3, 9, 17, 19], [1, 2, 3, 4, 5]], dtype=torch.int32)
    b = Batch(lens, hk=1, D=16, page=16, seed=8)
    path, kept = good.clone(), torch.tensor([5, 5, 5, 5, -1, 6], dtype=torch.int32)
    want_kept = torch.tensor([2, 3, 0, 3, 0, 5], dtype=torch.int32)
    path[0, 2] = 3
    path[1, 3] = 20
    path[2, 0] = -1
    table = b.table.clone()
    table[3, 3] = -1                               # places 48 on: new tokens 16 on
    cache, arrays = cache_of(b)
    S.KV8Keep(cache, *dev(table, b.q_start, b.kv_len, path, kept)).run()
    with pytest.raises(IndexError):
        done()
    done()
    for codes, scale, got, gscale in ((b.k, b.k_scale, arrays[0], arrays[2]), (b.v, b.v_scale, arrays[1], arrays[3])):
        want, wscale, live = P.keep(codes, scale, "i8", 16, *b.where(), good, want_kept)
        same_bits(got.cpu()[live], want[live])
        same_bits(gscale, wscale)


def test_keep_nothing_moves():
    b = Batch([(20, 52), (7, 30)], hk=2, D=64, page=16, seed=8)
    path = torch.arange(20, dtype=torch.int32).expand(2, -1).contiguous()
    cache, arrays = cache_of(b)
    S.KV8Keep(cache, *dev(*b.where(), path, torch.tensor([20, 0], dtype=torch.int32))).run()
    done()
    for got, want in zip(arrays, b.cache()):
        same_bits(got, want)
