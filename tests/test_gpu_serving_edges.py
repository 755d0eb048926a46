"""Edges of the serving operators, on the GPU: both attention kernels (few rows, many
rows) at masks, pages and codes that neither may look at, and how many bits results keep."""
import math

import pytest
import torch

from tests import _serving as S
from tests.test_gpu_serving import attend, check, dev, serving, sync   # noqa: F401 (a fixture)

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


# ---- what lies before a window ---------------------------------------------------------

WINDOWS = [
    # few rows: one sequence, several, in splits, more than one tile a sequence
    ([(1, 333)], 2, 3, 64, 16), ([(1, 333), (2, 90), (5, 700), (1, 16), (3, 3)], 2, 3, 64, 16),
    ([(1, 20000), (2, 9000), (1, 5)], 4, 2, 128, 16), ([(37, 600), (1, 70), (20, 300)], 2, 3, 80, 16),
    # many rows
    ([(130, 700), (90, 300), (64, 1900), (128, 129), (1, 500)], 16, 4, 128, 16),
    ([(130, 700), (90, 300), (64, 1900), (128, 129), (1, 500)], 16, 4, 64, 32),
    ([(70, 700), (90, 300), (64, 1500), (128, 129), (1, 500)], 16, 2, 192, 16),
]


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("window", [1, 37, 100])
@pytest.mark.parametrize("lens,hk,grp,D,page", WINDOWS)
def test_pages_before_the_window_are_not_looked_at(serving, lens, hk, grp, D, page, window, code):  # noqa: F811
    """Their table entries are gone, and what the first page of the window holds before it is
    NaN codes, as the memory of a page that was given away may hold."""
    b = S.Batch(lens, hk=hk, grp=grp, D=D, page=page, code=code, seed=window)
    clean = [x.clone() for x in (*b.cache(), b.table)]
    for s, (n, kv) in enumerate(lens):
        first = max(kv - n - window + 1, 0)                   # what the sequence's first new token sees from on
        gone = first // page
        for p in range(gone):
            at = int(b.table[s, p])
            for x in (b.k, b.v):
                x.view(torch.uint8)[at] = 0x7f
            b.k_scale[at] = b.v_scale[at] = math.nan
        if first % page:
            for x in (b.k, b.v):
                x.view(torch.uint8)[int(b.table[s, gone]), :first % page] = 0x7f
        b.table[s, :gone] = -1
    out, lse = attend(serving, b, window=window)              # (and no IndexError)
    b.k, b.v, b.k_scale, b.v_scale, b.table = clean
    check(b, out, lse, window=window, heads=(0, hk * grp - 1))


# ---- the kernel of many rows, where the one of few rows has been tested ----------------

MANY = dict(hk=16, grp=4)                          # with these, 8 tiles of more than half their rows
COLUMNS = [64, 80, 128, 192]


@pytest.mark.parametrize("D", COLUMNS)
def test_many_rows_not_causal(serving, D):  # noqa: F811
    b = S.Batch([(130, 200), (70, 33), (90, 90), (2, 0)], D=D, page=32, **MANY)
    check(b, *attend(serving, b, causal=False, scale=0.3), causal=False, scale=0.3, heads=(0, 63))


@pytest.mark.parametrize("D", COLUMNS)
@pytest.mark.parametrize("code", ["i8", "e4m3"])
def test_many_rows_do_not_look_behind_the_last_token(serving, code, D):  # noqa: F811
    b = S.Batch([(130, 133), (90, 300), (33, 64), (70, 1100), (1, 129)], D=D, code=code, seed=5, **MANY)
    clean = [x.clone() for x in b.cache()]
    used = set()
    for s, (_, n) in enumerate(b.lens):
        for p in range(-(-n // b.page)):
            at = int(b.table[s, p])
            used.add(at)
            for x in (b.k, b.v):
                x.view(torch.uint8)[at, min(n - p * b.page, b.page):] = 0x7f
    for at in set(range(b.pages)) - used:
        b.k_scale[at] = b.v_scale[at] = math.nan
    out, lse = attend(serving, b)
    b.k, b.v, b.k_scale, b.v_scale = clean
    check(b, out, lse, heads=(0, 63))


@pytest.mark.parametrize("D", COLUMNS)
@pytest.mark.parametrize("first_page", [0, 1, 5])
def test_many_rows_of_a_page_that_is_nan(serving, first_page, D):  # noqa: F811
    """Rows that see a token of the page are NaN, others are as without it."""
    b = S.Batch([(130, 130)] * 4, D=D, **MANY)
    start = 16 * first_page
    for name in ("k_scale", "v_scale"):
        keep = getattr(b, name)
        setattr(b, name, keep.clone())
        getattr(b, name)[int(b.table[1, first_page])] = math.nan
        out, lse = attend(serving, b)
        bad = torch.isnan(out.cpu()).all(-1).all(-1)
        assert bad[130 + start:260].all() and not torch.isnan(out.cpu()[~bad]).any() and int(bad.sum()) == 130 - start, name
        setattr(b, name, keep)
        want, wl, bound, lb = S.attention(b.q, *b.cache(), *b.where(), scale=D ** -0.5, heads=(0, 63))
        for h in (0, 63):
            S.close(out[:, h][~bad.cuda()], want[:, h][~bad], bound[:, h][~bad], b.dt)
            S.close(lse[:, h][~bad.cuda()], wl[:, h][~bad], lb[:, h][~bad], "f32")


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("D", COLUMNS)
def test_many_rows_of_uneven_weights(serving, dt, D):  # noqa: F811
    """One key holds nearly all the weight and has zeros as its value, so the others
    make the result; pages' scales lie far apart, some of values that are all 0."""
    b = S.Batch([(40, 700)] * 8, D=D, dt=dt, seed=9, spread=2.0, **MANY)
    b.q = (torch.ones_like(b.q) + 0.25 * b.q).to(b.q.dtype)
    for s in range(8):
        first = int(b.table[s, 0])
        b.k[first, 0] = 127
        b.k_scale[first] = 12.0 / (D ** 0.5 * 127)        # its score: about 12 above the others
        for p in range(1, b.width):
            b.k_scale[int(b.table[s, p])] = 0.1 / 127
        b.v[first, 0] = 0
        b.v_scale[int(b.table[s, 2])] = 2.0 ** -100
        b.v[int(b.table[s, 2])] = 0
        b.v_scale[int(b.table[s, 3])] = 0.0
        b.v[int(b.table[s, 3])] = 0
    check(b, *attend(serving, b), heads=(0, 63))


def test_many_rows_of_an_empty_v(serving):  # noqa: F811
    for scale in (2.0 ** -100, 0.0):
        b = S.Batch([(40, 200)] * 8, D=64, dt="bf16", **MANY)
        b.v[:] = 0
        b.v_scale[:] = scale
        check(b, *attend(serving, b), heads=(0, 63))


@pytest.mark.parametrize("D", [48, 128, 208])
def test_many_rows_strides_and_odd_bases(serving, D):  # noqa: F811
    """Queries cut from a projection's rows and from a 2-byte bound on, an output with heads
    outside tokens, a cache with both halves in one allocation."""
    b = S.Batch([(40, 90), (130, 177), (90, 90)], D=D, page=32, dt="bf16", **MANY)
    qkv = torch.randn((b.tokens, 70, D)).to(torch.bfloat16)
    qkv[:, 3:67] = b.q
    flat = torch.zeros(qkv.numel() + 9, dtype=torch.bfloat16)
    flat[3:3 + qkv.numel()] = qkv.flatten()
    odd = flat.cuda()[3:3 + qkv.numel()].view(qkv.shape)
    both = torch.stack([b.k.transpose(1, 2), b.v.transpose(1, 2)], 1).contiguous().cuda()
    sc = torch.stack([b.k_scale, b.v_scale], 1).cuda()
    cache = serving.KV8Cache(both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2), sc[:, 0], sc[:, 1])
    want, _, bound, _ = S.attention(b.q, *b.cache(), *b.where(), scale=D ** -0.5, heads=(0, 63))
    for q in (qkv.cuda()[:, 3:67], odd[:, 3:67]):
        out = torch.zeros((64, b.tokens, D), dtype=torch.bfloat16, device="cuda")
        shifted = torch.zeros(out.numel() + 9, dtype=torch.bfloat16, device="cuda")[5:5 + out.numel()].view(b.tokens, 64, D)
        for o in (out.transpose(0, 1), shifted):
            serving.KV8Attention(cache, q, o, *dev(*b.where()), **b.most).run()
            sync()
            for h in (0, 63):
                S.close(o[:, h], want[:, h], bound[:, h], "bf16")


@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 16), (96, 256), (256, 64)])
def test_many_rows_behind_long_contexts(serving, D, page, code):  # noqa: F811
    """Pages and scales are fetched for 16 steps at once: several such fetches, of odd and even numbers."""
    b = S.Batch([(40, 2100), (33, 3333), (40, 4160), (36, 1024), (40, 2048), (40, 1025), (35, 5000), (40, 64)], D=D, page=page, code=code,
                dt="bf16", seed=D, **MANY)
    check(b, *attend(serving, b), heads=(0, 63))


def test_many_rows_out_of_range_is_reported_and_stays_inside(serving):  # noqa: F811
    from ktir_cpu_amd import runtime as rt
    for what in ("page past the cache", "negative page", "length past the table", "tokens past the batch", "max_k", "max_q"):
        b = S.Batch([(130, 140), (90, 1160), (70, 70)], D=64, pad=1, **MANY)
        table, q_start, kv_len = [x.clone() for x in b.where()]
        most = dict(b.most)
        if what == "page past the cache":
            table[1, 3] = b.pages
        elif what == "negative page":
            table[1, 71] = -5
        elif what == "length past the table":
            kv_len[1] = 16 * b.width + 9
            most["max_k"] = 1 << 20
        elif what == "tokens past the batch":
            q_start[3] = 100000
        elif what == "max_k":
            most["max_k"] = 1150
        else:
            most["max_q"] = 100
        print(what, flush=True)
        serving.KV8Attention(serving.KV8Cache(*dev(*b.cache())), b.q.cuda(), torch.zeros_like(b.q).cuda(), *dev(table, q_start, kv_len),
                             **most).run()
        torch.cuda.synchronize()
        with pytest.raises(IndexError, match="outside"):
            rt.sync()
    rt.sync()


# ---- codes that are NaN ------------------------------------------------------------------

@pytest.mark.parametrize("hk,D,page", [(2, 64, 16), (1, 256, 64)])
def test_append_keeps_nan_codes(serving, hk, D, page):  # noqa: F811
    """A page that was filled elsewhere holds NaN codes: they stay NaN when the page's scale grows."""
    b = S.Batch([(3, 13)], hk=hk, D=D, page=page, code="e4m3")
    at = int(b.table[0, 0])
    b.new_k *= 40
    b.new_v *= 40                                              # the scales grow
    for x in (b.k, b.v):
        x.view(torch.uint8)[at, 4, 0, 5], x.view(torch.uint8)[at, 9, hk - 1, D - 1] = 0x7f, 0xff
    d = dev(*b.cache())
    serving.KV8Append(serving.KV8Cache(*d), *dev(b.new_k, b.new_v), *dev(*b.where())).run()
    sync()
    for x, codes, scale, c2, s2 in ((b.new_k, b.k, b.k_scale, d[0], d[2]), (b.new_v, b.v, b.v_scale, d[1], d[3])):
        want, wscale = S.append(x, codes, scale, "e4m3", page, *b.where())
        assert torch.equal(s2.cpu(), wscale) and bool((wscale[at] > scale[at]).all())
        nan = torch.isnan(want.float())
        assert int(nan.sum()) == 2 and torch.equal(torch.isnan(c2.cpu().float()), nan)
        assert torch.equal(c2.cpu().view(torch.uint8)[~nan], want.view(torch.uint8)[~nan])


# ---- the angle's sine and cosine ----------------------------------------------------------

@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("amplitude", [1.0, 1.2079441541679836])
def test_rope_sine_and_cosine_are_rounded_once(serving, amplitude, inter):  # noqa: F811
    g = torch.Generator().manual_seed(7)
    x = torch.randn((700, 2, 128), generator=g)
    pos = torch.randint(0, 1 << 20, (700,), generator=g)
    freq, _ = serving.rope_frequencies(128)
    out = torch.zeros_like(x).cuda()
    serving.Rope(x.cuda(), pos.cuda(), torch.from_numpy(freq).cuda(), out, interleaved=inter, amplitude=amplitude).run()
    sync()
    ang = torch.outer(pos.double(), torch.from_numpy(freq))
    c, s = (ang.cos() * amplitude)[:, None], (ang.sin() * amplitude)[:, None]
    a, b = (x[..., 0::2], x[..., 1::2]) if inter else (x[..., :64], x[..., 64:])
    a, b = a.double(), b.double()
    y, o = (a * c - b * s, b * c + a * s), out.cpu().double()
    o = (o[..., 0::2], o[..., 1::2]) if inter else (o[..., :64], o[..., 64:])
    # c and s rounded once, each product once, their sum once (2^-24 each, the first two on each of the
    # products); the angle in 64 bits: 2^20 radians hold it, in either order of operations, as
    # far as four roundings of 2^-53 and the amplitude go: 2^-30 of the pair's size
    for got, want, size in ((o[0], y[0], (a * c).abs() + (b * s).abs()), (o[1], y[1], (b * c).abs() + (a * s).abs())):
        bound = size * 2 * 2.0 ** -24 * (1 + 2.0 ** -20) + want.abs() * 2.0 ** -24 + (a.abs() + b.abs()) * 2.0 ** -30 + 2.0 ** -126
        assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound).max())


# ---- the own workspace ---------------------------------------------------------------------

def test_own_workspace_after_a_raw_handle(serving):  # noqa: F811
    """A run on a raw handle is the caller's to wait for; the same stream as an object is recorded all the same."""
    b = S.Batch([(1, 5000), (1, 70)], hk=2, grp=4, D=64, dt="bf16")
    q = b.q.cuda()
    op = serving.KV8Attention(serving.KV8Cache(*dev(*b.cache())), q, torch.empty_like(q), *dev(*b.where()), **b.most)
    keep, held = op._own, []

    class Own:
        def record_stream(self, stream):
            held.append(stream.cuda_stream)

    op._own = Own()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    op.run(side.cuda_stream)
    op.run(side)
    torch.cuda.synchronize()
    op.run(side.cuda_stream)
    with torch.cuda.stream(side):
        op.run()
    torch.cuda.synchronize()
    assert held == [side.cuda_stream]
    del keep
