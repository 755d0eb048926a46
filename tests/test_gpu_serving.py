"""The serving operators (rotary positions, the 8-bit cache, attention over it)
against plain float64 implementations, on the GPU."""
import math

import numpy as np
import pytest
import torch

from tests import _serving as S

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def serving():
    from ktir_cpu_amd import serving
    return serving


def dev(*xs):
    out = [x.cuda() if isinstance(x, torch.Tensor) else x for x in xs]
    return out[0] if len(out) == 1 else out


def sync():
    from ktir_cpu_amd import runtime as rt
    torch.cuda.synchronize()
    rt.sync()


# ---- rotary positions ----------------------------------------------------------

@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("tokens,heads,kheads,D,rot,inter", [
    (1, 1, 0, 64, 64, False), (1, 32, 8, 128, 128, False), (7, 5, 2, 80, 20, True), (130, 3, 3, 96, 96, True),
    (67, 4, 1, 128, 64, False), (33, 2, 2, 256, 250, False), (9, 3, 0, 7, 6, True), (300, 8, 8, 64, 64, False),
    (5, 1, 1, 2, 2, False), (64, 40, 40, 128, 128, True)])
def test_rope(serving, tokens, heads, kheads, D, rot, inter, dt):
    g = torch.Generator().manual_seed(tokens + D)
    x = torch.randn((tokens, heads, D), generator=g).to(S.DT[dt])
    k = torch.randn((tokens, max(kheads, 1), D), generator=g).to(S.DT[dt])
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g)
    pos[0] = (1 << 20) - 1
    freq, amp = serving.rope_frequencies(rot, scaling="yarn", factor=8.0)
    out, k_out = torch.zeros_like(x).cuda(), torch.zeros_like(k).cuda()
    f = torch.from_numpy(freq).cuda()
    serving.Rope(x.cuda(), pos.cuda(), f, out, k=k.cuda() if kheads else None, k_out=k_out if kheads else None,
                 interleaved=inter, amplitude=amp).run()
    sync()
    for a, o in ((x, out),) + (((k, k_out),) if kheads else ()):
        want, bound = S.rope(a, pos, freq, interleaved=inter, amplitude=amp)
        S.close(o, want, bound, dt)
        assert torch.equal(o.cpu()[..., rot:], a[..., rot:])


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_rope_in_place_skips_negative_positions_and_turns_back(serving, inter, kind):
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn((50, 12, 64), generator=g)                       # 8 query, 2 key, 2 value heads of a token
    pos = torch.randint(0, 5000, (50,), generator=g)
    pos[[0, 17, 49]] = torch.tensor([-1, -7, -1])
    freq, _ = serving.rope_frequencies(48)
    d, p, f = qkv.cuda(), pos.to(kind).cuda(), torch.from_numpy(freq).cuda()
    q, k = d[:, :8], d[:, 8:10]
    serving.Rope(q, p, f, k=k, interleaved=inter).run()
    sync()
    want, bound = S.rope(qkv[:, :10], pos, freq, interleaved=inter)
    skip = pos < 0
    S.close(d[:, :10][~skip.cuda()], want[~skip], bound[~skip], "f32")
    assert torch.equal(d.cpu()[skip], qkv[skip]) and torch.equal(d.cpu()[:, 10:], qkv[:, 10:])
    serving.Rope(q, p, f, k=k, interleaved=inter, inverse=True).run()
    sync()
    S.close(d[:, :10], qkv[:, :10].double(), 3 * bound.abs() + 1e-30, "f32")


def test_rope_gradient(serving):
    """inverse of the output's gradient is the input's: against differences of the operator in float64."""
    g = torch.Generator().manual_seed(4)
    x, w = torch.randn((3, 2, 12), generator=g), torch.randn((3, 2, 12), generator=g)
    pos = torch.tensor([0, 5, 1000])
    freq, amp = serving.rope_frequencies(8, scaling="yarn", factor=4.0)
    got = torch.zeros_like(x).cuda()
    serving.Rope(w.cuda(), pos.cuda(), torch.from_numpy(freq).cuda(), got, amplitude=amp, inverse=True).run()
    sync()
    want = torch.zeros(x.shape, dtype=torch.float64)
    for i in range(x.numel()):
        step = torch.zeros(x.numel(), dtype=torch.float64)
        step[i] = 0.5                                    # the operator is linear: differences of any step are exact
        up, down = (S.rope(x.double() + sgn * step.reshape(x.shape), pos, freq, amplitude=amp)[0] for sgn in (1, -1))
        want.view(-1)[i] = ((up - down) * w).sum()
    _, bound = S.rope(w, pos, freq, amplitude=amp, inverse=True)
    S.close(got, want, bound + 1e-12, "f32")


@pytest.mark.parametrize("tokens,heads,D,rot,dt,inter", [(9001, 2, 64, 64, "f16", False), (8195, 1, 16, 8, "bf16", True),
                                                         (3, 2, 4096, 4096, "f16", False), (2, 1, 1001, 1000, "f32", True)])
def test_rope_long(serving, tokens, heads, D, rot, dt, inter):
    """Several tokens a workgroup, and rows of more units than it has threads."""
    g = torch.Generator().manual_seed(D)
    x = torch.randn((tokens, heads, D), generator=g).to(S.DT[dt])
    pos = torch.arange(tokens, dtype=torch.int32) * 7
    pos[tokens // 2] = -1
    freq, _ = serving.rope_frequencies(rot)
    out = torch.full_like(x, 5.0).cuda()
    serving.Rope(x.cuda(), pos.cuda(), torch.from_numpy(freq).cuda(), out, interleaved=inter).run()
    sync()
    want, bound = S.rope(x, pos, freq, interleaved=inter)
    want[tokens // 2] = 5.0
    S.close(out, want, bound, dt)


@pytest.mark.parametrize("tokens,heads,kheads,D,rot,dt,inter", [(3501, 32, 8, 128, 96, "bf16", False), (2051, 13, 3, 260, 256, "f32", True)])
def test_rope_larger_than_the_caches(serving, tokens, heads, kheads, D, rot, dt, inter):
    g = torch.Generator().manual_seed(D)
    qkv = torch.randn((tokens, heads + kheads + 1, D), generator=g).to(S.DT[dt])
    assert 2 * tokens * (heads + kheads) * D * qkv.element_size() > 64 << 20
    pos = torch.randint(-3, 1 << 17, (tokens,), generator=g)
    freq, _ = serving.rope_frequencies(rot)
    d = qkv.cuda()
    out, k_out = torch.full((tokens, heads, D), 5.0).to(S.DT[dt]).cuda(), torch.full((tokens, kheads, D), 5.0).to(S.DT[dt]).cuda()
    op = serving.Rope(d[:, :heads], pos.cuda(), torch.from_numpy(freq).cuda(), out, k=d[:, heads:heads + kheads], k_out=k_out,
                      interleaved=inter)
    for _ in range(2):                               # the second on values written by the stream just before
        op.run()
        sync()
        want, bound = S.rope(qkv[:, :heads + kheads], pos, freq, interleaved=inter)
        want[pos < 0] = 5.0
        S.close(out, want[:, :heads], bound[:, :heads], dt)
        S.close(k_out, want[:, heads:], bound[:, heads:], dt)
        qkv = qkv.flip(0).contiguous()
        d.copy_(qkv)


# ---- append ----------------------------------------------------------------------

LENS = {
    "one": [(1, 1)], "decode": [(1, 17), (1, 16), (1, 33), (1, 1), (1, 640)], "prompt": [(100, 100)],
    "chunks": [(37, 50), (5, 300), (64, 64), (1, 129), (0, 40), (200, 333)], "none": [(0, 0), (3, 3), (0, 7)],
    "longer than cached": [(9, 5), (2, 2), (4, 0)],
}


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("hk,D,page", [(1, 64, 16), (3, 80, 32), (8, 128, 16), (2, 256, 64), (2, 16, 256), (1, 208, 128)])
@pytest.mark.parametrize("lens", LENS)
def test_append(serving, lens, hk, D, page, code, dt):
    b = S.Batch(LENS[lens], hk=hk, D=D, page=page, code=code, dt=dt, pad=3, front=2 if lens == "chunks" else 0, seed=len(lens))
    b.new_k[b.tokens // 2] *= 30                     # a page's scale grows by much, another's not
    b.new_v[0] *= 0.0
    d = dev(*b.cache())
    serving.KV8Append(serving.KV8Cache(*d), *dev(b.new_k, b.new_v), *dev(*b.where())).run()
    sync()
    for x, codes, scale, c2, s2 in ((b.new_k, b.k, b.k_scale, d[0], d[2]), (b.new_v, b.v, b.v_scale, d[1], d[3])):
        want, wscale = S.append(x, codes, scale, code, page, *b.where())
        assert torch.equal(s2.cpu(), wscale)
        assert torch.equal(c2.cpu().view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_append_of_values_that_are_not_finite(serving, bad):
    b = S.Batch([(20, 30)], hk=2, D=64)
    b.new_k[3, 1, 5] = bad                           # position 13: the first page, with 10 older tokens, head 1
    d = dev(*b.cache())
    serving.KV8Append(serving.KV8Cache(*d), *dev(b.new_k, b.new_v), *dev(*b.where())).run()
    sync()
    want, wscale = S.append(b.new_k, b.k, b.k_scale, "i8", 16, *b.where())
    assert torch.equal(torch.isnan(d[2].cpu()), torch.isnan(wscale)) and int(torch.isnan(wscale).sum()) == 1
    assert torch.equal(d[0].cpu(), want)
    # the page stays NaN while it fills, and starts over when its first row is written
    one = S.Batch([(1, 31)], hk=2, D=64)
    at = [x.cuda() for x in (b.table, torch.tensor([0, 1], dtype=torch.int32), torch.tensor([14], dtype=torch.int32))]
    serving.KV8Append(serving.KV8Cache(*d), *dev(one.new_k, one.new_v), *at).run()
    sync()
    assert bool(torch.isnan(d[2][int(b.table[0, 0]), 1]))
    at[2].fill_(1)
    serving.KV8Append(serving.KV8Cache(*d), *dev(one.new_k, one.new_v), *at).run()
    sync()
    assert bool(torch.isfinite(d[2]).all())


def test_append_strides(serving):
    """Keys and values cut from one projection's rows, a cache with both in one
    allocation and heads outside tokens, a table of a wider one."""
    b = S.Batch([(40, 90), (1, 5)], hk=3, D=48, page=32, dt="bf16")
    kv = torch.cat([b.new_k, b.new_v], 1).cuda()
    both = torch.zeros((b.pages, 2, b.hk, b.page, b.D), dtype=torch.int8, device="cuda")
    both[:, 0], both[:, 1] = b.k.transpose(1, 2), b.v.transpose(1, 2)
    k, v = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    sc = torch.stack([b.k_scale, b.v_scale], -1).transpose(0, 1).contiguous().cuda().transpose(0, 1)   # heads outside pages
    table = torch.cat([b.table, b.table], 1).cuda()[:, :b.width]
    serving.KV8Append(serving.KV8Cache(k, v, sc[..., 0], sc[..., 1]), kv[:, :3], kv[:, 3:], table, *dev(b.q_start, b.kv_len)).run()
    sync()
    for x, codes, scale, c2, s2 in ((b.new_k, b.k, b.k_scale, k, sc[..., 0]), (b.new_v, b.v, b.v_scale, v, sc[..., 1])):
        want, wscale = S.append(x, codes, scale, "i8", 32, *b.where())
        assert torch.equal(s2.cpu(), wscale) and torch.equal(c2.cpu(), want)


# ---- attention ---------------------------------------------------------------------

def attend(serving, b, **kw):
    out = torch.full_like(b.q, 7.0).cuda()
    lse = torch.full(b.q.shape[:2], 7.0).cuda()
    kw = {**b.most, **kw}
    serving.KV8Attention(serving.KV8Cache(*dev(*b.cache())), b.q.cuda(), out, *dev(*b.where()), lse=lse, **kw).run()
    sync()
    return out, lse


def check(b, out, lse, heads=None, **kw):
    """All query heads, or some of them."""
    want, wl, bound, lb = S.attention(b.q, *b.cache(), *b.where(), scale=kw.pop("scale", b.D ** -0.5), heads=heads, **kw)
    if heads is not None:
        heads = list(heads)
        want, wl, bound, lb, out, lse = want[:, heads], wl[:, heads], bound[:, heads], lb[:, heads], out[:, heads], lse[:, heads]
    inside = torch.zeros(b.tokens, dtype=torch.bool)
    inside[int(b.q_start[0]):int(b.q_start[-1])] = True
    S.close(out[inside.cuda()], want[inside], bound[inside], b.dt, "out")
    S.close(lse[inside.cuda()], wl[inside], lb[inside], "f32", "lse")
    empty = torch.isinf(wl) & (wl < 0)
    assert torch.equal(lse.cpu()[empty], wl[empty].float()) and not out.cpu()[empty].any()
    assert bool((out[~inside.cuda()] == 7).all()) and bool((lse[~inside.cuda()] == 7).all())


ATTN = {
    "one key": [(1, 1)], "decode": [(1, 17), (1, 16), (1, 33), (1, 1), (1, 640)], "prompt": [(70, 70)],
    "chunks": [(37, 50), (5, 300), (33, 64), (1, 129), (0, 40), (90, 333)], "none": [(0, 0), (3, 3), (1, 0), (0, 7)],
    "empty rows": [(9, 5), (2, 2), (4, 0), (20, 19)],
}


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("hk,grp,D,page", [(1, 1, 64, 16), (2, 4, 128, 16), (1, 7, 80, 32), (3, 2, 256, 64), (2, 1, 16, 256),
                                           (1, 16, 192, 16), (1, 3, 144, 128)])
@pytest.mark.parametrize("lens", ATTN)
def test_attention(serving, lens, hk, grp, D, page, code, dt):
    b = S.Batch(ATTN[lens], hk=hk, grp=grp, D=D, page=page, code=code, dt=dt, pad=2, front=1 if lens == "chunks" else 0, seed=len(lens))
    check(b, *attend(serving, b))


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("code", ["i8", "e4m3"])
@pytest.mark.parametrize("hk,grp,D,page,window", [(16, 4, 128, 16, 0), (8, 7, 80, 32, 60), (16, 2, 256, 64, 0), (32, 3, 48, 16, 1),
                                                  (4, 16, 192, 128, 100), (16, 5, 64, 256, 0)])
def test_attention_prompts(serving, hk, grp, D, page, window, code, dt):
    """Enough rows for the kernel of many rows: prompts, chunks behind cached tokens, rows
    that see nothing, sequences of one token or none among them."""
    b = S.Batch([(130, 130), (90, 300), (1, 70), (0, 5), (33, 20), (64, 64), (70, 1100), (128, 129)], hk=hk, grp=grp, D=D, page=page,
                code=code, dt=dt, pad=3, front=1, seed=D)
    check(b, *attend(serving, b, window=window), window=window, heads=(0, grp, hk * grp - 1))


@pytest.mark.parametrize("lens", ["decode", "chunks", "empty rows"])
@pytest.mark.parametrize("window", [1, 2, 15, 16, 40, 1000])
def test_attention_window(serving, lens, window):
    b = S.Batch(ATTN[lens], hk=2, grp=3, D=64, dt="bf16", pad=1, seed=window)
    check(b, *attend(serving, b, window=window), window=window)


@pytest.mark.parametrize("hk,grp,D,dt,lens", [
    (8, 4, 128, "bf16", [(1, 4096 - 61 * i) for i in range(40)] + [(0, 9), (1, 0), (1, 1)]),
    (3, 5, 80, "f16", [(2, 3000), (3, 5000)] + [(1, 7 * i + 1) for i in range(70)]),
    (2, 2, 256, "bf16", [(1, 9000 * i + 5) for i in range(8)]),
    (6, 1, 192, "f16", [(4, 2500 * i + 9) for i in range(9)]), (8, 4, 64, "bf16", [(1, 70001)]), (4, 2, 128, "f16", [(3, 140000)])])
@pytest.mark.parametrize("code", ["i8", "e4m3"])
def test_attention_long(serving, code, hk, grp, D, dt, lens):
    """More keys than one workgroup takes: parts of sequences of all lengths, four, two
    or one head a workgroup, joined."""
    b = S.Batch(lens, hk=hk, grp=grp, D=D, page=32, code=code, dt=dt, pad=1, seed=hk)
    check(b, *attend(serving, b), heads=(0, hk * grp - 1))


def test_attention_long_window(serving):
    b = S.Batch([(1, 60000), (2, 70000), (1, 3), (5, 40000)] * 8, hk=4, grp=2, D=64, page=64, dt="bf16", seed=1)
    check(b, *attend(serving, b, window=30001), window=30001, heads=(3, 7))


def test_attention_of_shared_pages_and_far_ones(serving):
    """Sequences that share a prefix's pages, a page twice in one table, and pages
    whose offset passes 2^32 bytes in a cache of 5 GB."""
    b = S.Batch([(2, 90), (1, 75), (3, 48)], hk=8, grp=2, D=128, dt="bf16")
    pages = (5 << 30) // (16 * 8 * 128)
    big = [torch.empty((pages, 16, 8, 128), dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.full((pages, 8), math.nan, device="cuda") for _ in range(2)]
    at = torch.tensor([pages - 1 - 3 * i for i in range(b.pages)])
    for x, y in zip(big + scales, b.cache()):
        x[at.cuda()] = y.cuda()
    b.table[1, :3] = b.table[0, :3]
    b.table[2, 1] = b.table[2, 0]
    where = [at.to(torch.int32)[b.table.long().clamp(min=0)].cuda(), b.q_start.cuda(), b.kv_len.cuda()]
    out = torch.zeros_like(b.q).cuda()
    cache = serving.KV8Cache(*big, *scales)
    serving.KV8Attention(cache, b.q.cuda(), out, *where, **b.most).run()
    sync()
    want, _, bound, _ = S.attention(b.q, *b.cache(), *b.where(), scale=b.D ** -0.5)
    S.close(out, want, bound, "bf16")
    # appending there, to pages that no other sequence has
    b = S.Batch([(2, 90), (1, 75), (3, 48)], hk=8, grp=2, D=128, dt="bf16")
    where[0] = at.to(torch.int32)[b.table.long().clamp(min=0)].cuda()
    serving.KV8Append(cache, *dev(b.new_k, b.new_v), *where).run()
    sync()
    for x, codes, scale, c2, s2 in ((b.new_k, b.k, b.k_scale, big[0], scales[0]), (b.new_v, b.v, b.v_scale, big[1], scales[1])):
        wc, ws = S.append(x, codes, scale, "i8", 16, *b.where())
        assert torch.equal(c2[at.cuda()].cpu(), wc) and torch.equal(s2[at.cuda()].cpu(), ws)


def test_attention_of_an_empty_v(serving):
    """A cache of zeros at the least scale, and of scale 0: the result is 0, the weights' sum is kept."""
    for scale in (2.0 ** -100, 0.0):
        b = S.Batch([(1, 5000), (40, 200)], hk=1, grp=4, D=64, dt="bf16")
        b.v[:] = 0
        b.v_scale[:] = scale
        check(b, *attend(serving, b))


def test_two_launches_at_once_and_a_shared_workspace(serving):
    """Two launches that split keys, each with its workspace, on two streams; then both one
    after another in one workspace."""
    bs = [S.Batch([(1, 20000), (1, 9000)], hk=2, grp=4, D=128, dt="f16", seed=s) for s in (1, 2)]
    ops, outs = [], []
    for b in bs:
        outs.append(torch.zeros_like(b.q).cuda())
        ops.append(serving.KV8Attention(serving.KV8Cache(*dev(*b.cache())), b.q.cuda(), outs[-1], *dev(*b.where()), **b.most))
        assert ops[-1].workspace_bytes > 0
    want = [S.attention(b.q, *b.cache(), *b.where(), scale=b.D ** -0.5) for b in bs]
    streams = [torch.cuda.Stream() for _ in bs]
    torch.cuda.synchronize()
    for _ in range(20):
        for op, s in zip(ops, streams):
            op.run(s)
    sync()
    for o, w in zip(outs, want):
        S.close(o, w[0], w[2], "f16")
        o.zero_()
    ws = torch.empty(ops[0].workspace_bytes, dtype=torch.uint8, device="cuda")
    shared = [serving.KV8Attention(serving.KV8Cache(*dev(*b.cache())), b.q.cuda(), o, *dev(*b.where()), workspace=ws, **b.most)
              for b, o in zip(bs, outs)]
    for _ in range(5):
        for op in shared:
            op.run()
    sync()
    for o, w in zip(outs, want):
        S.close(o, w[0], w[2], "f16")


def test_results_repeat(serving):
    """The same bits on every run: no order of arrival in any sum."""
    for lens, hk, grp in (([(1, 30000)], 8, 4), ([(1, 3000 + 17 * i) for i in range(30)], 8, 4), ([(700, 900), (300, 2000)], 16, 4)):
        b = S.Batch(lens, hk=hk, grp=grp, D=128, dt="f16", seed=3)
        first = attend(serving, b)
        for _ in range(4):
            again = attend(serving, b)
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("lens,hk,grp", [([(1, 5000), (1, 70)], 2, 4), ([(300, 400), (200, 900)], 16, 4)])
def test_attention_into_the_queries(serving, lens, hk, grp):
    b = S.Batch(lens, hk=hk, grp=grp, D=64, dt="bf16")
    q = b.q.cuda()
    serving.KV8Attention(serving.KV8Cache(*dev(*b.cache())), q, q, *dev(*b.where()), **b.most).run()
    sync()
    heads = [0, hk * grp - 1]
    want, _, bound, _ = S.attention(b.q, *b.cache(), *b.where(), scale=b.D ** -0.5, heads=heads)
    S.close(q[:, heads], want[:, heads], bound[:, heads], "bf16")


def test_own_workspace_is_held_for_every_stream(serving):
    b = S.Batch([(1, 5000), (1, 70)], hk=2, grp=4, D=64, dt="bf16")
    q = b.q.cuda()
    op = serving.KV8Attention(serving.KV8Cache(*dev(*b.cache())), q, torch.empty_like(q), *dev(*b.where()), **b.most)
    assert op.workspace_bytes > 0 and op._own.data_ptr() == op.desc.ws
    keep, held = op._own, []

    class Own:
        def record_stream(self, stream):
            held.append(stream.cuda_stream)

    op._own = Own()
    op.run()
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    op.run(side)
    op.run(side)
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        op.run()
    torch.cuda.synchronize()
    assert held == [side.cuda_stream, other.cuda_stream]
    del keep


def test_attention_not_causal(serving):
    b = S.Batch([(5, 40), (70, 33), (2, 0)], hk=2, grp=3, D=96, page=32)
    check(b, *attend(serving, b, causal=False, scale=0.3), causal=False, scale=0.3)


@pytest.mark.parametrize("lens", ["decode", "chunks"])
@pytest.mark.parametrize("code", ["i8", "e4m3"])
def test_attention_does_not_look_behind_the_last_token(serving, lens, code):
    """Rows of a page behind a sequence's last token, pages that no sequence has,
    and scales of those hold whatever the memory held: NaN codes and scales."""
    b = S.Batch(ATTN[lens], hk=2, grp=2, D=64, code=code, seed=5)
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
    check(b, out, lse)


def test_attention_of_a_page_that_is_nan(serving):
    """Rows that see a token of the page are NaN, others are as without it."""
    b = S.Batch([(40, 40)], hk=1, grp=2, D=64)
    at = int(b.table[0, 1])                          # tokens 16 to 31
    for name in ("k_scale", "v_scale"):
        keep = getattr(b, name)
        setattr(b, name, keep.clone())
        getattr(b, name)[at] = math.nan
        out, lse = attend(serving, b)
        bad = torch.isnan(out.cpu()).all(-1)
        assert not bad[:16].any() and bad[16:].all(), name
        setattr(b, name, keep)
        want, wl, bound, lb = S.attention(b.q, *b.cache(), *b.where(), scale=b.D ** -0.5)
        S.close(out[:16], want[:16], bound[:16], b.dt)
        S.close(lse[:16], wl[:16], lb[:16], "f32")


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("lens", [[(1, 4097)], [(40, 700)]])
def test_attention_of_uneven_weights(serving, dt, lens):
    """One key holds nearly all the weight and has zeros as its value, so the others
    make the result; pages' scales lie far apart, some of values that are all 0."""
    b = S.Batch(lens, hk=1, grp=4, D=64, dt=dt, seed=9, spread=2.0)
    first = int(b.table[0, 0])
    b.q = (torch.ones_like(b.q) + 0.25 * b.q).to(b.q.dtype)
    b.k[first, 0, 0] = 127
    b.k_scale[first] = 12.0 / (64 ** 0.5 * 127)       # its score: about 12 above the others
    for p in range(1, b.width):
        b.k_scale[int(b.table[0, p])] = 0.1 / 127
    b.v[first, 0] = 0
    b.v_scale[int(b.table[0, 2])] = 2.0 ** -100
    b.v[int(b.table[0, 2])] = 0
    b.v_scale[int(b.table[0, 3])] = 0.0
    check(b, *attend(serving, b))


def test_attention_strides(serving):
    """Queries cut from a projection's rows, an output with heads outside tokens, a
    cache with both halves in one allocation."""
    b = S.Batch([(3, 90), (30, 77)], hk=2, grp=2, D=48, page=32, dt="bf16")
    qkv = torch.randn((b.tokens, 12, b.D)).to(torch.bfloat16)
    qkv[:, 3:7] = b.q
    both = torch.stack([b.k.transpose(1, 2), b.v.transpose(1, 2)], 1).contiguous().cuda()
    sc = torch.stack([b.k_scale, b.v_scale], 1).cuda()
    out = torch.zeros((4, b.tokens, b.D), dtype=torch.bfloat16, device="cuda")
    cache = serving.KV8Cache(both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2), sc[:, 0], sc[:, 1])
    serving.KV8Attention(cache, qkv.cuda()[:, 3:7], out.transpose(0, 1), *dev(*b.where()), **b.most).run()
    sync()
    want, _, bound, _ = S.attention(b.q, *b.cache(), *b.where(), scale=b.D ** -0.5)
    S.close(out.transpose(0, 1), want, bound, "bf16")


def test_attention_odd_bases(serving):
    """Queries and output rows that start anywhere (2-byte bounds)."""
    b = S.Batch([(3, 90), (30, 77)], hk=2, grp=2, D=48, page=32)
    n = b.q.numel()
    flat = torch.zeros(n + 9, dtype=torch.float16)
    flat[3:3 + n] = b.q.flatten()
    q = flat.cuda()[3:3 + n].view(b.q.shape)
    out = torch.zeros(n + 9, dtype=torch.float16, device="cuda")[5:5 + n].view(b.q.shape)
    serving.KV8Attention(serving.KV8Cache(*dev(*b.cache())), q, out, *dev(*b.where()), **b.most).run()
    sync()
    want, _, bound, _ = S.attention(b.q, *b.cache(), *b.where(), scale=b.D ** -0.5)
    S.close(out, want, bound, "f16")


# ---- what is out of range, other streams, graphs, the operators together ---------------

def test_out_of_range_is_reported_and_stays_inside(serving):
    from ktir_cpu_amd import runtime as rt
    for what in ("page past the cache", "negative page", "length past the table", "tokens past the batch", "max_k", "max_q"):
        b = S.Batch([(2, 40), (3, 60)], hk=1, grp=2, D=64, pad=1)
        table, q_start, kv_len = [x.clone() for x in b.where()]
        most = dict(b.most)
        if what == "page past the cache":
            table[1, 3] = b.pages
        elif what == "negative page":
            table[1, 3] = -5
        elif what == "length past the table":
            kv_len[1] = 16 * b.width + 9
            most["max_k"] = 1000
        elif what == "tokens past the batch":
            q_start[2] = 1000
        elif what == "max_k":
            most["max_k"] = 50
        else:
            most["max_q"] = 2
        d = dev(*b.cache())
        ops = [serving.KV8Attention(serving.KV8Cache(*d), b.q.cuda(), torch.zeros_like(b.q).cuda(), *dev(table, q_start, kv_len), **most)]
        if not what.startswith("max"):
            ops.append(serving.KV8Append(serving.KV8Cache(*d), *dev(b.new_k, b.new_v), *dev(table, q_start, kv_len)))
        for op in ops:
            print(what, type(op).__name__, flush=True)
            op.run()
            torch.cuda.synchronize()
            with pytest.raises(IndexError, match="outside"):
                rt.sync()
    rt.sync()


def test_device_arrays_on_the_library_stream(serving):
    """The same without torch tensors: host arrays up, the library's stream, results down."""
    from ktir_cpu_amd import runtime as rt
    b = S.Batch([(1, 50), (4, 20)], hk=2, grp=2, D=64, dt="bf16")
    A = serving.DeviceArray
    bits = lambda x: x.view(torch.uint8 if x.dtype == torch.float8_e4m3fn else torch.int16).numpy().view(np.uint16)  # noqa: E731
    cache = serving.KV8Cache(*[A(x.numpy()) for x in b.cache()])
    where = [A(x.numpy()) for x in b.where()]
    q, k, v, out = A(bits(b.q)), A(bits(b.new_k)), A(bits(b.new_v)), A(bits(torch.zeros_like(b.q)))
    freq, _ = serving.rope_frequencies(64)
    pos = torch.tensor([49, 16, 17, 18, 19])
    turn = serving.Rope(q, A(pos.numpy()), A(freq), k=k)
    keep = serving.KV8Append(cache, k, v, *where)
    see = serving.KV8Attention(cache, q, out, *where, **b.most)
    for op in (turn, keep, see):
        op.run()
    rt.sync()
    back = lambda a: torch.from_numpy(a.numpy().view(np.int16)).view(torch.bfloat16)  # noqa: E731
    for a, x in ((q, b.q), (k, b.new_k)):
        want, bound = S.rope(x, pos, freq)
        S.close(back(a), want, bound, "bf16")
    b.q, b.new_k = back(q), back(k)
    for x, name in ((b.new_k, "k"), (b.new_v, "v")):
        c, s = S.append(x, getattr(b, name), getattr(b, name + "_scale"), "i8", 16, *b.where())
        setattr(b, name, c)
        setattr(b, name + "_scale", s)
    assert np.array_equal(cache.arrays[0].numpy(), b.k.numpy()) and np.array_equal(cache.arrays[3].numpy(), b.v_scale.numpy())
    want, _, bound, _ = S.attention(b.q, *b.cache(), *b.where(), scale=b.D ** -0.5)
    S.close(back(out), want, bound, "bf16")


class Decoder:
    """One layer that decodes: rotates, appends and attends, on fixed buffers."""

    def __init__(self, serving, lens, code="i8", hk=2, grp=3, D=64, page=16, steps=40, seed=1):
        self.b = b = S.Batch([(1, n + steps) for n in lens], hk=hk, grp=grp, D=D, page=page, code=code, dt="bf16", seed=seed)
        self.freq, _ = serving.rope_frequencies(D)
        self.d = dev(*b.cache())
        self.where = dev(*b.where())
        self.kv_len = torch.tensor(lens, dtype=torch.int32)
        self.where[2].copy_(self.kv_len)
        rows, heads = len(lens), hk * (grp + 2)
        self.qkv = torch.zeros((rows, heads, D), dtype=torch.bfloat16, device="cuda")
        self.q = torch.zeros((rows, hk * grp, D), dtype=torch.bfloat16, device="cuda")
        self.k = torch.zeros((rows, hk, D), dtype=torch.bfloat16, device="cuda")
        self.out = torch.zeros_like(self.q)
        self.pos = torch.zeros(rows, dtype=torch.int64, device="cuda")
        cache, n = serving.KV8Cache(*self.d), hk * grp
        self.ops = [serving.Rope(self.qkv[:, :n], self.pos, torch.from_numpy(self.freq).cuda(), self.q,
                                 k=self.qkv[:, n:n + hk], k_out=self.k),
                    serving.KV8Append(cache, self.k, self.qkv[:, n + hk:], *self.where),
                    serving.KV8Attention(cache, self.q, self.out, *self.where, max_q=1, max_k=max(lens) + steps)]
        self.n, self.hk = n, hk

    def feed(self, step):
        """A new token of every sequence, its length and position."""
        g = torch.Generator().manual_seed(100 + step)
        self.x = torch.randn(self.qkv.shape, generator=g).to(torch.bfloat16)
        self.kv_len += 1
        self.qkv.copy_(self.x)
        self.where[2].copy_(self.kv_len)
        self.pos.copy_(self.kv_len.long() - 1)

    def run(self):
        for op in self.ops:
            op.run()

    def check(self):
        b, n = self.b, self.n
        b.kv_len = self.kv_len.clone()
        q, k, v = self.x[:, :n], self.x[:, n:n + self.hk], self.x[:, n + self.hk:]
        for a, o in ((q, self.q), (k, self.k)):
            want, bound = S.rope(a, self.kv_len.long() - 1, self.freq)
            S.close(o, want, bound, "bf16")
        for x, name, at in ((self.k.cpu(), "k", 0), (v, "v", 1)):
            c, s = S.append(x, getattr(b, name), getattr(b, name + "_scale"), b.code, b.page, *b.where())
            assert torch.equal(self.d[at].cpu().view(torch.uint8), c.view(torch.uint8)) and torch.equal(self.d[at + 2].cpu(), s)
            setattr(b, name, c)
            setattr(b, name + "_scale", s)
        want, _, bound, _ = S.attention(self.q.cpu(), *b.cache(), *b.where(), scale=b.D ** -0.5)
        S.close(self.out, want, bound, "bf16")


@pytest.mark.parametrize("code", ["i8", "e4m3"])
def test_decoding(serving, code):
    """Forty steps of rotation, append and attention, over page ends, from empty caches on."""
    m = Decoder(serving, [0, 15, 31, 300], code)
    for step in range(40):
        m.feed(step)
        m.run()
        sync()
        m.check()


def test_decoding_on_another_stream_and_in_a_graph(serving):
    """The three launches captured together and replayed on new tokens, with the
    program's own work and waits between the replays, beside a second graph."""
    a, b = Decoder(serving, [5, 40, 200]), Decoder(serving, [64, 1], "e4m3", seed=2)
    side = torch.cuda.Stream()
    graphs = []
    for m in (a, b):
        m.feed(0)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            m.run()
        side.synchronize()
        m.check()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            m.run()
        graphs.append(g)
    for step in range(1, 6):
        for m, g in zip((a, b), graphs):
            m.feed(step)
            g.replay()
        torch.cuda.synchronize()
        for m in (a, b):
            m.check()
        junk = torch.randn(1 << 20, device="cuda").sort()
        torch.cuda.synchronize()
        del junk
    sync()


def test_prompt_in_chunks_is_the_prompt_at_once(serving):
    """Appending and attending 150 tokens in chunks leaves what the cache of the whole holds."""
    b = S.Batch([(150, 150)], hk=2, grp=2, D=64, dt="f16")
    outs = []
    for cuts in ([0, 150], [0, 1, 17, 64, 150]):
        d = [torch.zeros_like(x).cuda() for x in b.cache()]
        cache, out = serving.KV8Cache(*d), torch.zeros_like(b.q).cuda()
        for lo, hi in zip(cuts, cuts[1:]):
            where = dev(b.table, torch.tensor([0, hi - lo], dtype=torch.int32), torch.tensor([hi], dtype=torch.int32))
            serving.KV8Append(cache, *dev(b.new_k[lo:hi], b.new_v[lo:hi]), *where).run()
            serving.KV8Attention(cache, b.q[lo:hi].cuda(), out[lo:hi], *where, max_q=hi - lo, max_k=hi).run()
            sync()
            host = [x.cpu() for x in d]
            want, _, bound, _ = S.attention(b.q[lo:hi], *host, *[x.cpu() for x in where], scale=b.D ** -0.5)
            S.close(out[lo:hi], want, bound, "f16")
        outs.append([x.cpu() for x in d])
    # the scales are the same maxima whichever way the tokens came
    assert torch.equal(outs[0][2], outs[1][2]) and torch.equal(outs[0][3], outs[1][3])
