"""Edges of the operators for drafted tokens on the GPU, by each of their kernels: scores of -inf, bounds above
the batch, places that no row sees, uneven batches, how many bits results keep."""
import math

import pytest
import torch

from ktir_cpu_amd import serving as S
from tests import _drafts as P
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
