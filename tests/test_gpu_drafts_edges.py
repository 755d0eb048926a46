"""Edges of the operators for drafted tokens on the GPU, by each of their kernels: scores of -inf, bounds above
the batch, places that no row sees, uneven batches, how many bits results keep."""
import math

import pytest
import torch

from ktir_cpu_amd import serving as S
from tests import _drafts as P
from tests import test_gpu_drafts as G
from tests._serving import Batch, append, close, rope
from tests.test_gpu_drafts import attend, cache_of, check, dev, done, freq_of, same_bits, tree_of

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


@pytest.mark.parametrize("n,grp,D,most", KERNELS)
@pytest.mark.parametrize("k", [90, 2600])
def test_attention_of_rows_whose_scores_are_far_below_zero(n, grp, D, most, k):
    # finite scores of -4e37 and below: the least of them has all the weight, whole tiles and cut ones
    b = Batch([(n, k + n)], hk=2, grp=grp, D=D, page=16, dt="bf16", seed=n)
    b.q.zero_()
    b.q[..., 0] = -1.25 * 2.0 ** 118
    b.k.zero_()
    b.k[..., 0] = 120
    b.k_scale.fill_(1.0)
    page, row = int(b.table[0, 37 // 16]), 37 % 16
    b.k[page, row, :, 0] = 100
    mask, _ = tree_of(b, 3, 0)
    _, out, line = attend(b, mask, scale=1.0, **({"max_k": most} if most else {}))
    done()
    want = (b.v[page, row].double() * b.v_scale[page].double()[:, None]).repeat_interleave(grp, 0).expand(n, -1, -1)
    close(out, want, want.abs() * 2.0 ** -20, "bf16")          # (the weight's sum and quotient in f32)
    assert ((line.double().cpu() / (-125 * 2.0 ** 118) - 1).abs() <= 2.0 ** -20).all()


# ---- rotation with append: a long run of tokens among many sequences of one -------------------

UNEVEN = [
    # lens, hk, grp, D, rot, page, code, dt, interleaved, positions, pad, front
    ([(1, 30 + s) for s in range(70)] + [(40, 300)] + [(1, 77)] * 20, 2, 2, 64, 64, 16, "i8", "bf16", False, None, 0, 0),
    ([(200, 230)] + [(1, 9 + s) for s in range(220)] + [(6, 6), (4, 19), (5, 69)], 1, 3, 128, 128, 256, "e4m3", "f16", False, "i32", 2, 3),
    ([(0, 40)] * 60 + [(90, 90)] + [(0, 5)] * 30, 3, 1, 80, 20, 64, "i8", "f16", True, "i64", 0, 1),
    ([(300, 1000), (2, 40), (3, 3), (0, 9)] + [(0, 1), (1, 1)] * 130 + [(77, 100)], 2, 2, 256, 256, 32, "i8", "bf16", True, None, 3, 0),
    ([(33, 20)] + [(1, 60)] * 40, 1, 1, 32, 16, 16, "e4m3", "bf16", False, None, 0, 0),        # (its first 13 tokens have no place)
]


@pytest.mark.parametrize("lens,hk,grp,D,rot,page,code,dt,inter,given,pad,front", UNEVEN)
def test_turn_of_uneven_batches(lens, hk, grp, D, rot, page, code, dt, inter, given, pad, front):
    # two tokens a sequence at most on average, and more than four of one sequence in a page
    b = Batch(lens, hk=hk, grp=grp, D=D, page=page, code=code, dt=dt, pad=pad, front=front, seed=D + rot)
    assert 8 < b.tokens <= 2 * len(lens)
    freq, where = freq_of(rot), P.places(b.q_start, b.kv_len, b.tokens)
    live = where >= 0
    pos = where if given is None else torch.randint(0, 1 << 17, (b.tokens,), generator=torch.Generator().manual_seed(1))
    want_k = append(P.turned(b.new_k, pos.clamp(min=0), freq, inter, 0.75), b.k, b.k_scale, code, page, *b.where())
    want_v = append(b.new_v, b.v, b.v_scale, code, page, *b.where())
    cache, arrays = cache_of(b)
    q, given = dev(b.q), None if given is None else dev(pos.to(torch.int32 if given == "i32" else torch.int64))
    op = S.KV8RopeAppend(cache, q, *dev(b.new_k, b.new_v, freq, *b.where()), positions=given, interleaved=inter, amplitude=0.75)
    op.run()
    done()
    for got, want, what in zip(arrays, (want_k[0], want_v[0], want_k[1], want_v[1]), ("k", "v", "k_scale", "v_scale")):
        same_bits(got, want, what)
    want, bound = rope(b.q, pos.clamp(min=0), freq, interleaved=inter, amplitude=0.75)
    close(q[live], want[live], bound[live], dt)
    same_bits(q[~live], b.q[~live], "rows that are not stored")


def test_turn_of_uneven_batches_reports_a_page_that_is_not_there():
    b = Batch([(1, 20)] * 60 + [(50, 90), (1, 5)], hk=2, grp=1, D=32, page=16, seed=1)
    freq, where = freq_of(32), P.places(b.q_start, b.kv_len, b.tokens)
    clean = b.table.clone()
    b.table[60, 3] = b.pages                       # its places 48 to 63
    cache, arrays = cache_of(b)
    S.KV8RopeAppend(cache, *dev(b.q, b.new_k, b.new_v, freq, *b.where())).run()
    with pytest.raises(IndexError):
        done()
    done()
    lost = arrays[0][int(clean[60, 3])], arrays[2][int(clean[60, 3])]
    k, ks = append(P.turned(b.new_k, where, freq, False, 1.0), b.k, b.k_scale, "i8", 16, clean, b.q_start, b.kv_len)
    at = int(clean[60, 3])
    k[at], ks[at] = b.k[at], b.k_scale[at]
    same_bits(arrays[0], k)
    same_bits(arrays[2], ks)
    same_bits(lost[0], b.k[at])


def microseconds(op, n=20):
    """The median of seven loops of n launches."""
    a, z = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    times = []
    for _ in range(8):
        a.record()
        for _ in range(n):
            op.run()
        z.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(z) * 1e3 / n)
    return sorted(times[1:])[3]


@pytest.mark.parametrize("ones,run,page", [(256, 200, 16), (0, 100, 64), (0, 100, 256)])
def test_turn_of_a_long_run_among_many_sequences(ones, run, page):
    """The kernel for a token or two a sequence does not hand a long run's rows to one wavefront.  Against the kernel that the same
    batch takes with some tokens of padding: four wavefronts make a page's angles twice where that makes them once, on as many, so
    twice its time and what the launches have in common; a wavefront alone made it eight times (measured: 5 to 7, and 2.6)."""
    lens = [(1, 900)] * ones + [(run, 1100)] + [(0, 900)] * max(0, run - ones)
    took = []
    for pad in (0, 2 * len(lens) + 1 - ones - run):
        pages = sum(-(-k // page) for _, k in lens)
        table = torch.arange(pages, dtype=torch.int32)
        rows = torch.zeros((len(lens), -(-1100 // page)), dtype=torch.int32)
        at = 0
        for s, (_, k) in enumerate(lens):
            n = -(-k // page)
            rows[s, :n], at = table[at:at + n], at + n
        tokens = ones + run + pad
        codes = [torch.zeros((pages, page, 8, 128), dtype=torch.int8, device="cuda") for _ in range(2)]
        scales = [torch.ones((pages, 8), device="cuda") for _ in range(2)]
        q, k, v = (torch.randn((tokens, h, 128), device="cuda").to(torch.bfloat16) for h in (32, 8, 8))
        op = S.KV8RopeAppend(S.KV8Cache(*codes, *scales), q, k, v, *dev(freq_of(128), rows, torch.tensor([0] + [n for n, _ in lens]).cumsum(0).to(torch.int32),
                                                                       torch.tensor([n for _, n in lens], dtype=torch.int32)))
        took.append(microseconds(op))
    done()
    assert took[0] <= 4 * took[1], took


def test_turn_out_of_range_and_its_queries():
    """Queries of tokens whose table entry is no page are turned; those of tokens past the table, or before it, stay."""
    for dt, many in (("f16", False), ("bf16", True)):
        lens = [(20, 40), (10, 100), (5, 30), (9, 4)] + [(600, 600)] * many
        b = Batch(lens, hk=1, grp=2, D=32, page=16, dt=dt, seed=5)
        freq, where = freq_of(32), P.places(b.q_start, b.kv_len, b.tokens)
        table = b.table[:, :6 if not many else 38].contiguous()          # (the first: sequence 1 ends at 96 of 100)
        clean = table.clone()
        table[0, 1] = b.pages                                            # sequence 0's new tokens 0 to 11
        cache, arrays = cache_of(b)
        q = dev(b.q)
        S.KV8RopeAppend(cache, q, *dev(b.new_k, b.new_v, freq, table, b.q_start, b.kv_len)).run()
        with pytest.raises(IndexError):
            done()
        done()
        placed = (where >= 0) & ~((torch.arange(b.tokens) >= 26) & (torch.arange(b.tokens) < 30) & (not many))
        want, bound = rope(b.q, where.clamp(min=0), freq)
        close(q[placed], want[placed], bound[placed], dt)
        same_bits(q[~placed], b.q[~placed], "queries without a place")
        at = int(clean[0, 1])
        same_bits(arrays[0][at], b.k[at], "a page that was not named")


# ---- rotation with append: many tokens -------------------------------------------------------

# several tokens of queries in a workgroup (from 4096 tokens on), and queries read past the caches (more than 64 MB of them in and out)
LARGE = [
    # lens, hk, grp, D, rot, page, code, dt, interleaved, positions, pad, front
    ([(4100, 4200)], 1, 4, 64, 64, 16, "i8", "bf16", False, None, 0, 0),                  # 2 tokens a workgroup, vectors
    ([(3000, 3100), (0, 9), (1500, 1500)], 1, 2, 80, 20, 64, "e4m3", "f16", True, "i32", 7, 5),      # elements
    ([(2000, 2000), (1, 77)] + [(300, 400)] * 21, 1, 3, 64, 16, 32, "i8", "f16", False, "i64", 3, 1),
    ([(16500, 16500)], 1, 2, 32, 32, 256, "i8", "f16", True, None, 2, 3),                  # 8
]
PAST = [
    ([(3000, 3100), (5190, 5200)], 1, 33, 64, 64, 16, "i8", "bf16", False, "i32", 5, 5),
    ([(8200, 8200)], 1, 32, 64, 48, 64, "e4m3", "f16", True, None, 0, 0),
]


@pytest.mark.parametrize("lens,hk,grp,D,rot,page,code,dt,inter,given,pad,front,place", [(*c, x) for c in LARGE for x in (False, True)] + [(*c, False) for c in PAST])
def test_turn_of_many_tokens(lens, hk, grp, D, rot, page, code, dt, inter, given, pad, front, place):
    G.test_turn_and_append(lens, hk, grp, D, rot, page, code, dt, inter, given, pad, front, place)


# ---- attention of many rows ----------------------------------------------------------------------

# tiles of 128 rows (64 columns, and more than 128), of 256 rows with half the wavefronts idle, and of 256
MANY = [(30, 4, 64), (30, 4, 80), (80, 4, 64), (80, 4, 128), (40, 4, 192)]


def plan_of(op, seqs):
    """Which kernels a launch of several parts takes, by what a part of a head has in the workspace: the rows of a tile of 16 or 32, or
    the wavefronts that have 32 rows each."""
    d = op.desc.attn
    J, part = -(-d.cache.columns // 64), (op.workspace_bytes - 8 * seqs) // (4 * d.cache.heads * d.splits)
    wave = 2048 * (4 if J == 3 else J) + 64
    if part % wave == 0:
        return "many", part // wave
    J = 3 if d.cache.columns == 192 else J if J < 3 else 4
    assert part % (64 * J + 4) == 0
    return "few", part // (64 * J + 4)


def parts_of(op, seqs):
    """How many parts each sequence's tiles were cut into, by the note that the last launch left."""
    return op._own[:op.workspace_bytes][-8 * seqs:].view(torch.int32)[1::2].tolist()


def attend_many(b, mask, *args, **kw):
    """attend, by the kernels for many rows."""
    op, out, line = attend(b, mask, *args, **{"max_k": FAR, **kw})
    assert plan_of(op, len(b.lens))[0] == "many"
    return op, out, line


@pytest.mark.parametrize("n,grp,D", MANY)
@pytest.mark.parametrize("k", [70, 3000])
def test_many_rows_any_mask_and_rows_that_see_nothing(n, grp, D, k):
    b = Batch([(n, n), (n, n + k), (1, 1), (n, n)], hk=2, grp=grp, D=D, page=16, seed=n)
    g = torch.Generator().manual_seed(n)
    mask = torch.randint(-(1 << 31), 1 << 31, (b.tokens, -(-n // 32) + 1), generator=g, dtype=torch.int64).to(torch.int32)
    mask[::3] = 0
    op, out, line = attend_many(b, mask)
    done()
    assert (max(parts_of(op, 4)) > 1) == (k == 3000)
    check(b, out, line, mask)
    empty = out[:n][::3]
    assert (empty == 0).all() and torch.isneginf(line[:n][::3]).all()


@pytest.mark.parametrize("n,grp,D", MANY)
@pytest.mark.parametrize("code,k,window", [("e4m3", 16 * 9, 17), ("e4m3", 16 * 190, 16 * 150), ("i8", 16 * 9, 40)])
def test_many_rows_do_not_look_at_masked_places(n, grp, D, code, k, window):
    # what is before every window, and behind the last token, holds NaN and infinite scales and codes.  (The window bounds the keys too:
    # tokens that pad the batch are what brings it to the kernels for many rows)
    b = Batch([(n, k + n)], hk=2, grp=grp, D=D, page=16, code=code, pad=1100, seed=n)
    mask, pos = tree_of(b, 2, window, seed=1, pad=1100)
    clean = [x.clone() for x in b.cache()]
    for p in range((k - window + 1) // 16):
        at = int(b.table[0, p])
        b.k_scale[at], b.v_scale[at] = math.nan, math.inf
        if code == "e4m3":
            b.k.view(torch.uint8)[at] = b.v.view(torch.uint8)[at] = 0x7f
    last, end = int(b.table[0, (k + n - 1) // 16]), (k + n - 1) % 16 + 1
    if code == "e4m3":
        b.k.view(torch.uint8)[last, end:] = 0x7f
        b.v.view(torch.uint8)[last, end:] = 0xff
    op, out, line = attend(b, mask, pos, window=window)
    done()
    assert not op.workspace_bytes or plan_of(op, 1)[0] == "many" and parts_of(op, 1)[0] > 1
    b.k, b.v, b.k_scale, b.v_scale = clean
    check(b, out, line, mask, window, pos)


@pytest.mark.parametrize("n,grp,D", [(30, 4, 48), (30, 4, 112), (80, 4, 80), (80, 4, 64), (40, 4, 208)])
@pytest.mark.parametrize("k", [90, 2500])
def test_many_rows_in_place_strides_and_scale(n, grp, D, k):
    # queries from a 2-byte bound on, heads apart by odd steps, results in their place; a mask's rows apart; a cache in one allocation
    b = Batch([(n, k + n), (n - 1, 90)], hk=2, grp=grp, D=D, page=32, dt="f16", seed=9)
    mask, _ = tree_of(b, 3, 0)
    want = P.attention(b.q, *b.cache(), *b.where(), mask, scale=-0.2)
    heads = 2 * grp
    wide = torch.zeros((b.tokens, heads + 1, D + 3), dtype=torch.float16, device="cuda")
    q = wide[:, :heads, 1:D + 1]
    q.copy_(dev(b.q))
    line = torch.zeros((heads, b.tokens), device="cuda").t()
    wide_mask = torch.full((b.tokens, mask.shape[1] + 2), -1, dtype=torch.int32, device="cuda")
    wide_mask[:, :mask.shape[1]] = dev(mask)
    both = torch.zeros((b.pages, 2, 32, 2, D), dtype=torch.int8, device="cuda")
    both[:, 0], both[:, 1] = dev(b.k, b.v)
    scales = dev(torch.stack([b.k_scale, b.v_scale], 2))
    op = S.KV8TreeAttention(S.KV8Cache(both[:, 0], both[:, 1], scales[:, :, 0], scales[:, :, 1]), q, q, *dev(*b.where()), wide_mask[:, :mask.shape[1]],
                            scale=-0.2, lse=line, max_q=n, max_k=FAR)
    op.run()
    done()
    assert plan_of(op, 2)[0] == "many" and (parts_of(op, 2)[0] > 1) == (k == 2500)
    close(q, want[0], want[2], "f16")
    assert ((line.cpu() - want[1]).abs() <= want[3]).all()
    assert (wide[:, heads] == 0).all() and (wide[:, :, 0] == 0).all() and (wide[:, :, D + 1:] == 0).all()


@pytest.mark.parametrize("n,grp,D", [(10, 2, 64), (10, 4, 128)] + MANY)
@pytest.mark.parametrize("change", ["max_q", "max_k", "page"])
def test_attention_out_of_range_of_each_kernel(n, grp, D, change):
    """More new tokens than max_q, more cached ones than max_k, a page that there is not: the error word, sequences that are in
    range as ever, and of those that are not what is left of them."""
    # (padding brings the launch to the kernels for many rows, whatever bounds the keys)
    b = Batch([(n, 200 + n), (4, 100)], hk=2, grp=grp, D=D, page=16, pad=1100, seed=6)
    mask, _ = tree_of(b, 2, 0, pad=1100)
    clean = [x.clone() for x in (*b.cache(), b.table)]
    most, seq, other = {}, slice(0, n), slice(n, n + 4)
    if change == "page":
        b.table[0, 2] = b.pages + 5
    else:
        most[change] = n - 1 if change == "max_q" else 150
    op, out, line = attend(b, mask, **most)
    with pytest.raises(IndexError):
        done()
    done()
    k, v, ks, vs, table = clean
    where, scale = (table, b.q_start, b.kv_len), D ** -0.5
    want, wline, bound, lbound = P.attention(b.q, k, v, ks, vs, *where, mask, scale=scale)
    close(out[other], want[other], bound[other], "f16")
    assert ((line[other].cpu() - wline[other]).abs() <= lbound[other]).all()
    assert (out[n + 4:] == 7).all() and (line[n + 4:] == 7).all()
    if change == "max_q":                          # the last row is left out
        close(out[:n - 1], want[:n - 1], bound[:n - 1], "f16")
        assert (out[n - 1] == 7).all() and (line[n - 1] == 7).all()
    elif change == "max_k":                        # the first 150 keys, none of them new
        short = torch.tensor([150 + n, 100], dtype=torch.int32)
        none = mask.clone()
        none[seq] = 0
        want, _, bound, _ = P.attention(b.q, k, v, ks, vs, table, b.q_start, short, none, scale=scale)
        close(out[seq], want[seq], bound[seq], "f16")
    else:                                          # (what is read in place of the page is not said, but that it is the cache's)
        assert out[seq].isfinite().all() and not (out[seq] == 7).all(-1).any()


@pytest.mark.parametrize("n,grp", [(40, 4), (20, 4)])
def test_many_rows_of_far_pages(n, grp):
    pages, page, hk, D = 80000, 256, 2, 128                     # 5.2 GB a cache
    lens = [(n, 1700), (9, 500)]
    b = Batch(lens, hk=hk, grp=grp, D=D, page=page, code="i8", dt="bf16", seed=5)
    spots = torch.randperm(200, generator=torch.Generator().manual_seed(2))[:b.pages] + pages - 200
    k, v = (torch.zeros((pages, page, hk, D), dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros((pages, hk), device="cuda") for _ in range(2))
    at = spots.cuda()
    k[at], v[at], ks[at], vs[at] = dev(*b.cache())
    table = torch.where(b.table >= 0, spots[b.table.clamp(min=0).long()].to(torch.int32), b.table)
    mask, _ = tree_of(b, 2, 0)
    out = torch.zeros((b.tokens, 2 * grp, D), dtype=torch.bfloat16, device="cuda")
    op = S.KV8TreeAttention(S.KV8Cache(k, v, ks, vs), dev(b.q), out, *dev(table, b.q_start, b.kv_len), dev(mask), max_q=n, max_k=FAR)
    op.run()
    done()
    assert plan_of(op, 2) == ("many", -(-n * grp // 32))
    want, _, bound, _ = P.attention(b.q, *b.cache(), *b.where(), mask, scale=D ** -0.5)
    close(out, want, bound, "bf16")


@pytest.mark.parametrize("n,grp,D", MANY)
def test_many_rows_of_a_line_are_causal_attention(n, grp, D):
    b = Batch([(n, 1500), (1, 77)], hk=2, grp=grp, D=D, page=16, dt="bf16", seed=n)
    mask, _ = tree_of(b, 1, 0)
    _, out, line = attend_many(b, mask)
    cache, _ = cache_of(b)
    other, oline = torch.empty_like(out), torch.empty_like(line)
    S.KV8Attention(cache, dev(b.q), other, *dev(*b.where()), lse=oline, **b.most).run()
    done()
    want, _, bound, lbound = P.attention(b.q, *b.cache(), *b.where(), mask, scale=D ** -0.5)
    # each is within its bound and half a step of the line
    assert ((out.double() - other.double()).abs().cpu() - (2 * bound + want.abs() * 2.0 ** -7 * (1 + 2.0 ** -7))).max() <= 0
    assert ((line - oline).abs().cpu() <= 2 * lbound).all()


@pytest.mark.parametrize("n,grp,D", MANY)
def test_many_rows_repeat_at_once_and_with_a_shared_workspace(n, grp, D):
    batches = [Batch([(m, k + m), (3, 700)], hk=2, grp=grp, D=D, page=16, dt="f16", seed=m) for m, k in ((n, 5000), (n + 9, 70), (n + 1, 2000))]
    masks = [tree_of(b, 3, 0)[0] for b in batches]
    ops = [attend_many(b, m) for b, m in zip(batches, masks)]
    done()
    assert [parts_of(op, 2)[0] > 1 for op, _, _ in ops] == [True, False, True]
    first = [(out.clone(), line.clone()) for _, out, line in ops]
    for b, m, (_, out, line) in zip(batches, masks, ops):
        check(b, out, line, m)
        out.fill_(7), line.fill_(7)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ops]
    for _ in range(3):
        for (op, _, _), s in zip(ops, streams):
            op.run(s)
    done()
    for (_, out, line), (o, x) in zip(ops, first):
        same_bits(out, o), same_bits(line, x)
    # one workspace for launches that follow one another, of garbage to begin with
    ws = torch.full((max(op.workspace_bytes for op, _, _ in ops),), 0xff, dtype=torch.uint8, device="cuda")
    again = [attend(b, m, max_k=FAR, workspace=ws) for b, m in zip(batches, masks)]
    done()
    for (_, out, line), (o, x) in zip(again, first):
        same_bits(out, o), same_bits(line, x)


@pytest.mark.parametrize("n,grp,D", MANY)
def test_many_rows_in_graphs_whole_and_cut(n, grp, D):
    # lengths change between the replays of two graphs that share a workspace
    b = Batch([(n, 4200), (n, 4000), (3, 3900)], hk=2, grp=grp, D=D, page=16, code="i8", dt="bf16", seed=n)
    cache, _ = cache_of(b)
    q, table, q_start, kv_len = dev(b.q, *b.where())
    mask, _ = tree_of(b, 3, 0)
    at = dev(mask)
    out, line = [torch.empty_like(q) for _ in range(2)], [torch.empty(q.shape[:2], device="cuda") for _ in range(2)]
    first = S.KV8TreeAttention(cache, q, out[0], table, q_start, kv_len, at, lse=line[0], max_q=n, max_k=FAR)
    assert plan_of(first, 3)[0] == "many"
    space = torch.empty(first.workspace_bytes, dtype=torch.uint8, device="cuda")
    ops = [S.KV8TreeAttention(cache, q, o, table, q_start, kv_len, at, lse=x, workspace=space, max_q=n, max_k=FAR) for o, x in zip(out, line)]
    graphs = []
    for op in ops:
        op.run()
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            op.run()
    cut = set()
    for lens in ((4200, 4000, 3900), (n, n, 3), (4200, n, 50), (300, 2000, 3), (4200, 4000, 3900)):
        b.kv_len = torch.tensor(lens, dtype=torch.int32)
        b.lens = [(a, k) for (a, _), k in zip(b.lens, lens)]
        kv_len.copy_(b.kv_len)
        for g, o, x in zip(graphs, out, line):
            o.fill_(7.0)
            x.fill_(7.0)
            g.replay()
            done()
            check(b, o, x, mask)
        cut.add(int(space[-24:].view(torch.int32)[1]) > 1)
    assert cut == {False, True}


# ---- how many bits the weights keep ------------------------------------------------------------------

def two_weights(n, grp, D, k, seed):
    """A batch whose rows see two sizes of weights, e^c and e^-c of their own c, on values that nearly cancel in some column: what a weight is
    rounded by shows, as the result is small against what it is the sum of."""
    b = Batch([(n, k + n)], hk=2, grp=grp, D=D, page=16, dt="f16", seed=seed)
    g = torch.Generator().manual_seed(seed)
    b.q.zero_()
    b.q[..., 0] = (torch.rand(b.q.shape[:2], generator=g) * -2).to(b.q.dtype)
    b.k.zero_()
    b.k[:, ::2, :, 0], b.k[:, 1::2, :, 0] = 64, -64
    b.v[:, ::2] = 100
    b.v[:, 1::2] = -(2 + torch.arange(D) * 125 // D).to(torch.int8)
    b.k_scale.fill_(2.0 ** -6)
    b.v_scale.fill_(2.0 ** -6)
    return b


def weights_bound(b, mask):
    """(out, what it may be off by): a weight to 2^-18 of itself (two bf16 terms, each off by 2^-9 of what it stands for; two f16 terms leave less); its
    exponent, of at most 2^4, in f32 steps (score, scale, sum and difference: 3 roundings of 2^-20 at most), 2^-19 with the exponential's, in
    numerator and denominator; and the f32 sums over the keys, in both."""
    want, _, _, _ = P.attention(b.q, *b.cache(), *b.where(), mask, scale=1.0)
    size, _, _, _ = P.attention(b.q, b.k, b.v.abs(), b.k_scale, b.v_scale, *b.where(), mask, scale=1.0)
    return want, size * (2.0 ** -18 + 2 * 2.0 ** -19 + int(b.kv_len.max()) * 2.0 ** -23)


@pytest.mark.parametrize("n,grp,D,k,kind", [
    (4, 4, 64, 60, "few"), (8, 4, 128, 90, "few"), (9, 3, 192, 60, "few"), (15, 4, 128, 60, "few"), (12, 4, 256, 60, "few"), (8, 4, 128, 1500, "few"),
    (30, 4, 64, 60, "many"), (30, 4, 80, 60, "many"), (80, 4, 64, 60, "many"), (80, 4, 128, 60, "many"), (40, 4, 192, 60, "many"), (30, 4, 80, 1100, "many"),
    (80, 4, 128, 1100, "many")])
def test_weights_keep_their_bits(n, grp, D, k, kind):
    b = two_weights(n, grp, D, k, seed=n)
    mask, _ = tree_of(b, 3, 0)
    op, out, _ = attend(b, mask, scale=1.0, max_k=FAR)
    done()
    assert plan_of(op, 1)[0] == kind and (parts_of(op, 1)[0] > 1) == (k > 1000)
    want, bound = weights_bound(b, mask)
    close(out, want, bound, "f16")
