"""Edges of the serving operators without a GPU: where a handle's runs go, and which
overlaps are refused."""
import os

import numpy as np
import pytest

from ktir_cpu_amd import runtime as rt
from tests.test_serving_host import Fake, append, attention, cache, far, passes, refused, rope

pytestmark = pytest.mark.skipif(not os.path.exists(rt.LIB_PATH), reason="libktir_hip.so not built")


# ---- streams -------------------------------------------------------------------------

@pytest.mark.parametrize("make", [rope, append, attention])
def test_a_run_without_a_stream_goes_to_the_library_s(make):
    """Also after one on a stream of the caller's."""
    op, went = make(), []
    op._call = lambda ref: went.append(op.desc.stream) or 0          # nothing launches
    for stream in (None, 7 << 40, None, 0, None):
        op.run(stream)
    assert went == [0, 7 << 40, 0, rt.K["KTIR_STREAM_NULL"], 0]


# ---- what an output may not overlap ------------------------------------------------------

def at(base, offset, shape, typestr, **kw):
    """An array `offset` bytes behind the start of the made-up array `base`."""
    return Fake(shape, typestr, ptr=base.__cuda_array_interface__["data"][0] + offset, **kw)


def test_rope_over_positions_or_frequencies():
    out, k = far(3, (5, 4, 64), "<f2"), far(5, (5, 2, 64), "<f2")
    refused(rope(out=out, positions=at(out, 5 * 4 * 128 - 8, (5,), "<i8")), match="positions")
    refused(rope(out=out, freq=at(out, -8, (32,), "<f8")), match="frequencies")
    refused(rope(k=k, positions=at(k, 128, (5,), "<i4")), match="positions")
    passes(rope(out=out, positions=at(out, 5 * 4 * 128, (5,), "<i8"), freq=at(out, -256, (32,), "<f8")))
    # in a hole of a strided output
    out = far(3, (5, 4, 64), "<f2", strides=(1024, 128, 2))
    passes(rope(out=out, positions=at(out, 512, (5,), "<i8"), freq=at(out, 1024 + 512, (32,), "<f8")))
    refused(rope(out=out, positions=at(out, 1024 - 8, (5,), "<i8")), match="positions")


def test_append_into_what_it_reads():
    k = far(10, (9, 16, 2, 64), "|i1")                       # codes of 18432 bytes
    ks = far(12, (9, 2), "<f4")
    for what in (dict(k=at(k, 64, (7, 2, 64), "<f2")), dict(v=at(k, 18432 - 2, (7, 2, 64), "<f2")),
                 dict(k=at(ks, 68, (7, 2, 64), "<f2")), dict(v=at(ks, -7 * 256 + 4, (7, 2, 64), "<f2"))):
        refused(append(cache(k=k, k_scale=ks), **what), match="new keys or values")
    for what in (dict(table=at(k, 32, (3, 4), "<i4")), dict(q_start=at(ks, 64, (4,), "<i4")), dict(kv_len=at(k, -8, (3,), "<i4"))):
        refused(append(cache(k=k, k_scale=ks), **what), match="table, offsets or lengths")
    passes(append(cache(k=k, k_scale=ks), k=at(k, 18432, (7, 2, 64), "<f2"), v=at(ks, 72, (7, 2, 64), "<f2"),
                  table=at(k, -48, (3, 4), "<i4"), q_start=at(ks, -16, (4,), "<i4")))
    # (a table of no pages has no place)
    passes(append(table=Fake((3, 0), "<i4", ptr=0)))


def test_append_of_codes_and_scales_in_one_allocation():
    # a page of K's codes, V's codes and the scales of both, heads inside tokens and tokens inside heads
    for strides in ((4160, 128, 64, 1), (4160, 64, 1024, 1)):
        k = far(10, (9, 16, 2, 64), "|i1", strides=strides)
        v = at(k, 2048, (9, 16, 2, 64), "|i1", strides=strides)
        ks, vs = (at(k, 4096 + x, (9, 2), "<f4", strides=(4160, 4)) for x in (0, 8))
        passes(append(cache(k=k, v=v, k_scale=ks, v_scale=vs)))
        for bad in (0, 64, 2048, 4092, 4160):
            refused(append(cache(k=k, v=v, k_scale=at(k, bad, (9, 2), "<f4", strides=(4160, 4)), v_scale=vs)), match="overlap")
    k = far(10, (9, 16, 2, 64), "|i1")
    refused(append(cache(k=k, v_scale=at(k, 18432 - 4, (9, 2), "<f4"))), match="overlap")
    passes(append(cache(k=k, v_scale=at(k, 18432, (9, 2), "<f4"))))


def test_attention_over_what_it_reads():
    k, vs = far(10, (9, 16, 2, 64), "|i1"), far(13, (9, 2), "<f4")
    c = cache(k=k, v_scale=vs)
    table, lengths = far(14, (3, 4), "<i4"), far(16, (3,), "<i4")
    for base, size in ((k, 18432), (vs, 72), (table, 48), (lengths, 12)):
        for offset in (-7 * 512 + 4, size - 4):
            refused(attention(c, table=table, kv_len=lengths, out=at(base, offset, (7, 4, 64), "<f2")), match="overlaps the cache, table")
        for offset in (-7 * 512, size):
            passes(attention(c, table=table, kv_len=lengths, out=at(base, offset, (7, 4, 64), "<f2")))
        refused(attention(c, table=table, kv_len=lengths, lse=at(base, size - 4, (7, 4), "<f4")), match="overlaps the cache, table")


def test_attention_s_workspace_is_its_own():
    more = dict(max_k=1 << 13)
    need = attention(**more).workspace_bytes
    assert need > 0
    ws = far(24, (need,), "|u1")
    q, k = far(22, (7, 4, 64), "<f2"), far(10, (9, 16, 2, 64), "|i1")
    end = -(-need // 4) * 4
    for kw in (dict(q=at(ws, end - 4, (7, 4, 64), "<f2")), dict(out=at(ws, 16, (7, 4, 64), "<f2")), dict(lse=at(ws, end - 4, (7, 4), "<f4")),
               dict(c=cache(k=at(ws, need // 16 * 16 - 16, (9, 16, 2, 64), "|i1"))), dict(kv_len=at(ws, -8, (3,), "<i4"))):
        refused(attention(workspace=ws, **more, **kw), match="workspace")
    passes(attention(workspace=ws, q=q, out=q, c=cache(k=k), **more))
    # not used without splits
    op = attention(q=q)
    assert op.desc.splits == 1
    op.desc.ws, op.desc.ws_bytes = op.desc.q.ptr, 1 << 20
    passes(op)


@pytest.mark.parametrize("seed", range(30))
def test_no_overlap_passes(seed):
    """Random layouts of codes and scales in one allocation, against the set of their bytes: what shares
    a byte is refused, and of what steps alike over pages and lies apart in them, nothing."""
    rng = np.random.default_rng(seed)
    for _ in range(40):
        heads, pages = int(rng.integers(1, 4)), int(rng.integers(1, 4))
        tok, head = [(16 * heads, 16), (16, 256), (16 * heads + 16, 16)][rng.integers(3)]
        inner = max((16 - 1) * tok + (heads - 1) * head + 16, 0)
        page = -(-inner // 16) * 16 + 16 * int(rng.integers(0, 5))
        step = int(rng.choice([4, 8, 4 * heads]))
        offset = 4 * int(rng.integers(-8, (page * pages) // 4 + 8))
        k = far(10, (pages, 16, heads, 16), "|i1", strides=(page, tok, head, 1))
        s_page = int(rng.choice([page, page, 4 * heads if step == 4 else 64]))
        s = at(k, offset, (pages, heads), "<f4", strides=(s_page, step))
        if s_page < (heads - 1) * step + 4:
            continue
        codes = {p * page + t * tok + h * head + x for p in range(pages) for t in range(16) for h in range(heads) for x in range(16)}
        scale = {offset + p * s_page + h * step + x for p in range(pages) for h in range(heads) for x in range(4)}
        op = append(cache(pages=pages, heads=heads, columns=16, k=k, v=far(11, (pages, 16, heads, 16), "|i1"), k_scale=s, v_scale=far(13, (pages, heads), "<f4")))
        if codes & scale:
            refused(op, match="overlap")
        elif s_page == page and offset >= inner and offset + (heads - 1) * step + 4 <= page:
            passes(op)
