"""The serving operators without a GPU: frequencies, and every refusal of the
Python classes and of the C entry points (which check before they touch a device)."""
import ctypes as C
import math
import os
import subprocess

import numpy as np
import pytest

from ktir_cpu_amd import runtime as rt
from ktir_cpu_amd import serving as S

pytestmark = pytest.mark.skipif(not os.path.exists(rt.LIB_PATH), reason="libktir_hip.so not built")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Fake:
    """An array at a made-up address: nothing here launches."""

    def __init__(self, shape, typestr, ptr=1 << 32, strides=None):
        self.__cuda_array_interface__ = dict(shape=tuple(shape), typestr=typestr, version=2, strides=strides, data=(ptr, False))


def far(n, shape, typestr, **kw):
    """the n-th made-up array, a gigabyte from the next"""
    return Fake(shape, typestr, ptr=(n + 4) << 30, **kw)


def launch(op):
    """the status of the C entry point; a good descriptor ends at the missing device"""
    return getattr(rt.opened(), op.entry)(C.byref(op.desc)), rt.opened().ktir_last_error().decode()


def passes(op):
    if rt._lib is not None:
        pytest.skip("a device is in use by this process: a good descriptor would launch on made-up addresses")
    rc, msg = launch(op)
    assert rc == rt.K["KTIR_E_ARG"] and "ktir_init has not run" in msg, msg


def refused(op, code="KTIR_E_ARG", match=""):
    rc, msg = launch(op)
    assert rc == rt.K[code] and match in msg and "ktir_init" not in msg, msg


# ---- frequencies ---------------------------------------------------------------------

def test_frequencies_plain_and_linear():
    f, a = S.rope_frequencies(8, 100.0)
    np.testing.assert_allclose(f, [1.0, 100 ** -0.25, 0.1, 100 ** -0.75], rtol=1e-15)
    assert a == 1.0 and f.dtype == np.float64
    g, _ = S.rope_frequencies(8, 100.0, scaling="linear", factor=4.0)
    np.testing.assert_allclose(g, f / 4, rtol=1e-15)
    g, _ = S.rope_frequencies(8, 100.0, divisors=[1, 2, 4, 8])
    np.testing.assert_allclose(g, f / [1, 2, 4, 8], rtol=1e-15)


def test_frequencies_ntk_keeps_the_fastest_and_slows_the_slowest_by_factor():
    f, _ = S.rope_frequencies(64)
    g, a = S.rope_frequencies(64, scaling="ntk", factor=8.0)
    assert a == 1.0 and g[0] == 1.0
    np.testing.assert_allclose(g[-1], f[-1] / 8, rtol=1e-12)


@pytest.mark.parametrize("scaling", ["yarn", "wavelength"])
def test_frequencies_with_a_ramp(scaling):
    f, _ = S.rope_frequencies(128)
    g, a = S.rope_frequencies(128, scaling=scaling, factor=16.0, trained=4096, fast=32.0, slow=1.0)
    turns = 4096 * f / (2 * np.pi)
    ratio = f / g
    np.testing.assert_allclose(ratio[turns > 40], 1.0, rtol=1e-12)
    np.testing.assert_allclose(ratio[turns < 0.8], 16.0, rtol=1e-12)
    assert (np.diff(ratio) >= -1e-12).all() and ((ratio > 1.01) & (ratio < 15.9)).any()
    assert a == (pytest.approx(0.1 * math.log(16) + 1) if scaling == "yarn" else 1.0)


def test_frequencies_of_one_pair():
    for scaling in (None, "linear", "ntk", "yarn", "wavelength"):
        f, _ = S.rope_frequencies(2, scaling=scaling, factor=2.0)
        assert f.shape == (1,) and np.isfinite(f).all()


@pytest.mark.parametrize("bad", [dict(rot=0), dict(rot=7), dict(rot=8, base=-1.0), dict(rot=8, scaling="cubic"),
                                 dict(rot=8, scaling="yarn", fast=1.0, slow=2.0), dict(rot=8, divisors=[1.0]),
                                 dict(rot=8, scaling="linear", factor=0.0)])
def test_frequencies_refused(bad):
    with pytest.raises(ValueError):
        S.rope_frequencies(**bad)


# ---- rope --------------------------------------------------------------------------------

def rope(shape=(5, 4, 64), rot=64, **kw):
    x = kw.pop("x", far(0, shape, "<f2"))
    return S.Rope(x, kw.pop("positions", far(1, (shape[0],), "<i8")), kw.pop("freq", far(2, (rot // 2,), "<f8")),
                  kw.pop("out", far(3, shape, "<f2")), **kw)


def test_rope_accepted():
    passes(rope())
    passes(rope(out=None))
    passes(rope(k=far(5, (5, 1, 64), "<f2"), positions=far(1, (5,), "<i4"), interleaved=True, inverse=True))
    passes(rope(shape=(1, 1, 2), rot=2))
    x = far(0, (5, 4, 64), "<f2", strides=(12 * 128, 128, 2))
    passes(rope(x=x, out=None, k=Fake((5, 2, 64), "<f2", ptr=(4 << 30) + 512, strides=(12 * 128, 128, 2))))
    assert launch(rope(shape=(0, 4, 64)))[0] == 0       # nothing to do


@pytest.mark.parametrize("seed", range(40))
def test_rope_in_place_side_by_side_or_not(seed):
    # two tensors of equal steps in one allocation, against the set of their elements' addresses
    rng = np.random.default_rng(seed)
    tokens, heads, heads2 = (int(rng.integers(1, 5)) for _ in range(3))
    cols, most = 4, max(heads, heads2)
    head = int(rng.choice([cols, 2 * cols, 3 * cols, 3 * cols + 2]))
    tok = int(rng.choice([most * head, 2 * most * head, most * head + 6]))
    if rng.integers(2):                                # heads apart, their tokens inside
        head, tok = int(rng.choice([1, 2])) * tokens * 3 * cols, int(rng.choice([cols, 2 * cols, 3 * cols]))

    def elements(at, n):
        return {at + i * tok + j * head + c for i in range(tokens) for j in range(n) for c in range(cols)}

    def tensor(at, n):
        return Fake((tokens, n, cols), "<f2", ptr=(8 << 30) + 2 * at, strides=(2 * tok, 2 * head, 2))

    for _ in range(30):
        at = int(rng.integers(-2 * most * head, 2 * most * head + tok))
        op = S.Rope(tensor(0, heads), far(1, (tokens,), "<i8"), far(2, (cols // 2,), "<f8"), k=tensor(at, heads2))
        if elements(0, heads) & elements(at, heads2):
            refused(op, match="overlaps")
        else:
            passes(op)


def test_rope_refused_in_python():
    import torch
    with pytest.raises(ValueError, match="on the GPU"):
        rope(x=torch.zeros((5, 4, 64), dtype=torch.float16))
    with pytest.raises(TypeError, match="no device array"):
        rope(x=np.zeros((5, 4, 64), np.float16))
    for kw in (dict(x=far(0, (5, 64), "<f2")), dict(x=far(0, (5, 4, 64), "<i4")), dict(out=far(3, (5, 4, 32), "<f2")),
               dict(out=far(3, (5, 4, 64), "<f4")), dict(positions=far(1, (4,), "<i8")),
               dict(positions=far(1, (5,), "<f4")), dict(freq=far(2, (32,), "<f4")), dict(rot=128),
               dict(k=far(5, (5, 2, 32), "<f2")), dict(k=far(5, (4, 2, 64), "<f2")), dict(k_out=far(5, (5, 2, 64), "<f2")),
               dict(x=far(0, (5, 4, 64), "<f2", strides=(512, 128, 4))),
               dict(x=far(0, (5, 4, 64), "<f2", strides=(-512, 128, 2))),
               dict(x=far(0, (5, 4, 64), "<f2", strides=(511, 128, 2)))):
        with pytest.raises(ValueError):
            rope(**kw)


def test_rope_refused_in_c():
    refused(rope(out=Fake((5, 4, 64), "<f2", ptr=(4 << 30) + 128)), match="overlaps")
    refused(rope(out=far(3, (5, 4, 64), "<f2", strides=(0, 128, 2))), match="overlap")
    # queries into the keys' place, both outputs in one place, an output over half of the keys
    k = far(5, (5, 4, 64), "<f2")
    refused(rope(out=k, k=k, k_out=far(6, (5, 4, 64), "<f2")), match="overlaps")
    refused(rope(k=k, k_out=far(3, (5, 4, 64), "<f2")), match="overlaps")
    refused(rope(out=None, k=far(0, (5, 2, 64), "<f2")), match="overlaps")
    row = dict(strides=(12 * 128, 128, 2))
    refused(rope(x=far(0, (5, 8, 64), "<f2", **row), shape=(5, 8, 64), out=None, k=Fake((5, 2, 64), "<f2", ptr=(4 << 30) + 7 * 128, **row)),
            match="overlaps")
    refused(rope(out=far(3, (5, 4, 64), "<f2", strides=(512, 64, 2))), match="overlap")
    refused(rope(shape=(5, 0, 64)))
    refused(rope(amplitude=math.inf), match="amplitude")
    refused(rope(shape=(5, 1, 5000)))
    refused(rope(rot=0), match="rotated")
    for name, value, code in (("rot", 7, "KTIR_E_ARG"), ("rot", 66, "KTIR_E_ARG"), ("dtype", rt.K["KTIR_I8"], "KTIR_E_UNSUPPORTED"),
                              ("pos_dtype", rt.K["KTIR_I16"], "KTIR_E_UNSUPPORTED"), ("pos", 0, "KTIR_E_ARG"),
                              ("tokens", -1, "KTIR_E_ARG"), ("heads2", -1, "KTIR_E_ARG")):
        op = rope()
        setattr(op.desc, name, value)
        refused(op, code)
    op = rope()
    op.desc.in_.ptr = 0
    refused(op, match="missing")
    assert rt.opened().ktir_launch_rope(None) == rt.K["KTIR_E_ARG"]


# ---- the cache, append, attention -------------------------------------------------------

def cache(pages=9, page=16, heads=2, columns=64, code="|i1", **kw):
    shape = (pages, page, heads, columns)
    return S.KV8Cache(kw.get("k", far(10, shape, code)), kw.get("v", far(11, shape, code)),
                      kw.get("k_scale", far(12, (pages, heads), "<f4")), kw.get("v_scale", far(13, (pages, heads), "<f4")))


def where(seqs=3, width=4, **kw):
    return (kw.get("table", far(14, (seqs, width), "<i4")), kw.get("q_start", far(15, (seqs + 1,), "<i4")),
            kw.get("kv_len", far(16, (seqs,), "<i4")))


def append(c=None, tokens=7, dt="<f2", **kw):
    c = c or cache()
    shape = (tokens, c.desc.heads, c.desc.columns)
    return S.KV8Append(c, kw.pop("k", far(20, shape, dt)), kw.pop("v", far(21, shape, dt)), *where(**kw))


def attention(c=None, tokens=7, heads=4, dt="<f2", **kw):
    c = c or cache()
    shape = (tokens, heads, c.desc.columns)
    q, out = kw.pop("q", far(22, shape, dt)), kw.pop("out", far(23, shape, dt))
    w = {n: kw.pop(n) for n in ("table", "q_start", "kv_len", "seqs", "width") if n in kw}
    more = {**dict(max_q=3, max_k=64, workspace=far(24, (1 << 28,), "|u1")), **kw}
    return S.KV8Attention(c, q, out, *where(**w), **more)


def test_cache_operators_accepted():
    for page in (16, 32, 64, 128, 256):
        for columns in (16, 80, 128, 256):
            for code in ("|i1", "|u1"):
                c = cache(page=page, columns=columns, code=code)
                passes(append(c))
                passes(append(c, dt="<u2"))
                passes(attention(c))
    passes(attention(heads=14, window=5, scale=0.0, lse=far(25, (7, 14), "<f4")))
    passes(attention(causal=False))
    for op in (append(tokens=0), append(seqs=0), attention(tokens=0), attention(seqs=0)):
        assert launch(op)[0] == 0


def test_cache_refused():
    for kw in (dict(k=far(10, (9, 16, 2, 64), "<f2")), dict(v=far(11, (9, 16, 2, 32), "|i1")),
               dict(v=far(11, (9, 16, 2, 64), "|u1")), dict(k_scale=far(12, (9, 3), "<f4")),
               dict(k_scale=far(12, (9, 2), "<f2")), dict(k=far(10, (9, 16, 128), "|i1")),
               dict(k=far(10, (9, 16, 2, 64), "|i1", strides=(2048 * 2, 256, 128, 2)))):
        with pytest.raises(ValueError):
            cache(**kw)
    for kw in (dict(page=8), dict(page=24), dict(page=512), dict(columns=72), dict(columns=272), dict(columns=8)):
        refused(append(cache(**kw)), "KTIR_E_UNSUPPORTED")
        with pytest.raises(NotImplementedError):
            attention(cache(**kw))
    off = cache(k=Fake((9, 16, 2, 64), "|i1", ptr=(4 << 30) + 8))
    refused(append(off), "KTIR_E_UNSUPPORTED", "16-byte")
    with pytest.raises(NotImplementedError, match="16-byte"):
        attention(off)
    off = cache(v=far(11, (9, 16, 2, 64), "|i1", strides=(2176, 136, 64, 1)))
    refused(append(off), "KTIR_E_UNSUPPORTED", "16-byte")
    # a cache whose pages or heads lie on one another can be read, not written
    same = cache(k=far(10, (9, 16, 2, 64), "|i1", strides=(0, 128, 64, 1)))
    refused(append(same), match="overlap")
    refused(append(cache(v_scale=far(13, (9, 2), "<f4", strides=(0, 4)))), match="share a scale")
    refused(append(cache(v_scale=far(13, (9, 2), "<f4", strides=(8, 0)))), match="share a scale")
    passes(attention(same))
    # keys and values in one allocation: one page behind the other, heads in turn, or on one another
    for strides, v in (((4096, 128, 64, 1), 2048), ((4096, 256, 128, 1), 64), ((4096, 256, 64, 1), 128)):
        one = cache(k=far(10, (9, 16, 2, 64), "|i1", strides=strides),
                    v=Fake((9, 16, 2, 64), "|i1", ptr=(14 << 30) + v, strides=strides))
        passes(append(one))
    k, s = far(10, (9, 16, 2, 64), "|i1"), far(12, (9, 2), "<f4")
    for c in (cache(k=k, v=k), cache(k=k, v=Fake((9, 16, 2, 64), "|i1", ptr=(14 << 30) + 2048)), cache(k_scale=s, v_scale=s)):
        refused(append(c), match="overlap")
        passes(attention(c))


def test_append_refused():
    for kw in (dict(k=far(20, (7, 3, 64), "<f2")), dict(k=far(20, (7, 2, 32), "<f2")), dict(v=far(21, (6, 2, 64), "<f2")),
               dict(v=far(21, (7, 2, 64), "<u2")), dict(k=far(20, (7, 2, 64), "<f4"), v=far(21, (7, 2, 64), "<f4")),
               dict(table=far(14, (2, 4), "<i4")), dict(table=far(14, (3, 4), "<i8")), dict(q_start=far(15, (3,), "<i4")),
               dict(q_start=far(15, (4,), "<i8")), dict(kv_len=far(16, (3,), "<f4")),
               dict(k=far(20, (7, 2, 64), "<f2", strides=(-256, 128, 2)))):
        with pytest.raises(ValueError):
            append(**kw)
    for path, value in (("dtype", rt.K["KTIR_F32"]), ("cache.dtype", rt.K["KTIR_F16"])):
        op = append()
        at, _, name = path.rpartition(".")
        setattr(getattr(op.desc, at) if at else op.desc, name, value)
        refused(op, "KTIR_E_UNSUPPORTED")
    for path, value in (("cache.k", 0), ("cache.v_scale", 0), ("cache.pages", 0), ("cache.heads", 0), ("batch.table", 0),
                        ("batch.q_start", 0), ("batch.kv_len", 2), ("batch.seqs", -1), ("batch.table_row", -4),
                        ("batch.width", -1), ("k.ptr", 0), ("v.tok", -1), ("cache.k_tok", -16), ("cache.ks_page", -1)):
        op = append()
        at, _, name = path.rpartition(".")
        setattr(getattr(op.desc, at), name, value)
        refused(op)
    assert rt.opened().ktir_launch_kv8_append(None) == rt.K["KTIR_E_ARG"]


def test_attention_refused():
    for kw in (dict(q=far(22, (7, 4, 32), "<f2")), dict(out=far(23, (7, 3, 64), "<f2")), dict(out=far(23, (7, 4, 64), "<u2")),
               dict(heads=3), dict(window=-1), dict(window=1 << 31), dict(window=3, causal=False), dict(scale=math.nan), dict(max_q=-1), dict(max_q=1 << 31),
               dict(max_k=-1), dict(lse=far(25, (7, 3), "<f4")), dict(lse=far(25, (7, 4), "<f2")),
               dict(max_k=1 << 31)):
        with pytest.raises(ValueError):
            attention(**kw)
    refused(attention(out=far(23, (7, 4, 64), "<f2", strides=(512, 64, 2))), match="overlap")
    refused(attention(lse=far(25, (7, 4), "<f4", strides=(4, 4))), match="overlap")
    q = far(22, (7, 4, 64), "<f2")
    passes(attention(out=q))
    refused(attention(out=Fake((7, 4, 64), "<f2", ptr=(26 << 30) + 512)), match="overlaps")
    refused(attention(out=far(22, (7, 4, 64), "<f2", strides=(1024, 128, 2))), match="overlaps")
    refused(attention(lse=far(22, (7, 4), "<f4")), match="overlaps")
    refused(attention(lse=far(23, (7, 4), "<f4")), match="overlaps")
    with pytest.raises(ValueError, match="workspace"):
        attention(max_k=1 << 16, workspace=far(24, (8,), "|u1"))
    with pytest.raises(ValueError, match="workspace"):
        attention(max_k=1 << 16, workspace=Fake((1 << 28,), "|u1", ptr=(1 << 34) + 4))
    op = attention(max_k=1 << 13)
    assert op.desc.splits > 1 and op.workspace_bytes > 0
    for name, value in (("ws", 0), ("ws", (1 << 34) + 8), ("ws_bytes", op.workspace_bytes - 4), ("splits", op.desc.splits * 2)):
        op = attention(max_k=1 << 13)
        setattr(op.desc, name, value)
        refused(op, match="workspace")
    for name, value, code in (("dtype", rt.K["KTIR_F32"], "KTIR_E_UNSUPPORTED"), ("q_heads", 0, "KTIR_E_ARG"),
                              ("splits", -1, "KTIR_E_ARG"), ("scale", math.inf, "KTIR_E_ARG"), ("lse", 2, "KTIR_E_ARG")):
        op = attention()
        setattr(op.desc, name, value)
        refused(op, code)
    assert rt.opened().ktir_launch_kv8_attention(None) == rt.K["KTIR_E_ARG"]
    assert rt.opened().ktir_kv8_attention_plan(None) == rt.K["KTIR_E_ARG"]


def test_plans_are_in_bounds():
    """Splits and workspace of every shape of launch: at most 256 splits, none for launches of many rows."""
    for columns in (16, 64, 80, 128, 192, 256):
        for heads, grp in ((1, 1), (2, 7), (8, 4), (4, 16), (3, 40)):
            for tokens, seqs, max_q, max_k in ((1, 1, 1, 1), (1, 1, 1, 1 << 30), (64, 64, 1, 8192), (7, 3, 0, 64), (7, 3, 3, 0),
                                               (8192, 1, 8192, 8192), (500, 12, 400, 4000), (300, 300, 1, 100)):
                for window in (0, 1, 1000):
                    c = cache(heads=heads, columns=columns)
                    op = attention(c, tokens=tokens, heads=heads * grp, seqs=seqs, max_q=max_q, max_k=max_k, window=window,
                                   out=Fake((tokens, heads * grp, columns), "<f2", ptr=1 << 40), workspace=Fake((1 << 36,), "|u1", ptr=1 << 41))
                    assert 1 <= op.desc.splits <= 256
                    assert (op.workspace_bytes > 0) == (op.desc.splits > 1) and op.workspace_bytes < 1 << 30
                    passes(op)


def test_tensors_of_two_devices_are_refused():
    class On:
        """as a tensor of device n looks"""
        def __init__(self, n, shape, dtype):
            self.device = type("device", (), dict(type="cuda", index=n))()
            self.shape, self.dtype = shape, dtype

        def data_ptr(self):
            return 1 << 34

        def stride(self):
            s = [1]
            for n in self.shape[:0:-1]:
                s.insert(0, s[0] * n)
            return s
    args = [On(0, (5, 4, 64), "torch.float16"), On(1, (5,), "torch.int64"), On(0, (32,), "torch.float64")]
    with pytest.raises(ValueError, match="devices"):
        S.Rope(*args)


def test_descriptors_match_c(tmp_path):
    names = ("ktir_rows3_t", "ktir_rope_t", "ktir_kv8_t", "ktir_kv8_batch_t", "ktir_kv8_append_t", "ktir_kv8_attn_t")
    src = '#include <stdio.h>\n#include <stddef.h>\n#include "ktir_hip.h"\nint main(){' + "".join(
        f'printf("%zu ", sizeof({n}));' for n in names) + 'printf("%zu %zu %zu\\n", offsetof(ktir_rope_t, pos_dtype), ' \
        'offsetof(ktir_kv8_append_t, k), offsetof(ktir_kv8_attn_t, splits));}'
    (tmp_path / "s.c").write_text(src)
    exe = str(tmp_path / "s")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "s.c"), "-o", exe], check=True)
    got = [int(x) for x in subprocess.run([exe], capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(x) for x in (rt.Rows3, rt.Rope, rt.KV8, rt.KV8Batch, rt.KV8Append, rt.KV8Attn)] + [
        rt.Rope.pos_dtype.offset, rt.KV8Append.k.offset, rt.KV8Attn.splits.offset]
