"""The operators for drafted tokens without a GPU: every refusal of the Python classes and of the
C entry points, plans, and descriptors."""
import ctypes as C
import math
import os
import subprocess

import pytest
import torch

from ktir_cpu_amd import runtime as rt
from ktir_cpu_amd import serving as S
from tests import _drafts as P
from tests.test_serving_host import Fake, cache, far, launch, passes, refused, where

pytestmark = pytest.mark.skipif(not os.path.exists(rt.LIB_PATH), reason="libktir_hip.so not built")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def tree(seqs=3, tokens=7, words=2, **kw):
    return S.DraftTree(kw.pop("parents", far(30, (tokens,), "<i4")), kw.pop("q_start", far(15, (seqs + 1,), "<i4")),
                       kw.pop("kv_len", far(16, (seqs,), "<i4")), kw.pop("mask", far(31, (tokens, words), "<i4")),
                       kw.pop("positions", far(32, (tokens,), "<i4")), **kw)


def turn(c=None, tokens=7, heads=4, rot=32, dt="<f2", **kw):
    c = c or cache()
    shape, kv = (tokens, heads, c.desc.columns), (tokens, c.desc.heads, c.desc.columns)
    args = [kw.pop(n, far(i, s, t)) for i, (n, s, t) in enumerate((("q", shape, dt), ("k", kv, dt), ("v", kv, dt),
                                                                  ("freq", (rot // 2,), "<f8")), 33)]
    w = {n: kw.pop(n) for n in ("table", "q_start", "kv_len", "seqs", "width") if n in kw}
    return S.KV8RopeAppend(c, *args, *where(**w), kw.pop("q_out", far(37, shape, dt)), **kw)


def attention(c=None, tokens=7, heads=4, words=2, dt="<f2", **kw):
    c = c or cache()
    shape = (tokens, heads, c.desc.columns)
    q, out, mask = kw.pop("q", far(22, shape, dt)), kw.pop("out", far(23, shape, dt)), kw.pop("mask", far(31, (tokens, words), "<i4"))
    w = {n: kw.pop(n) for n in ("table", "q_start", "kv_len", "seqs", "width") if n in kw}
    more = {**dict(max_q=3, max_k=64, workspace=Fake((1 << 36,), "|u1", ptr=1 << 41)), **kw}
    return S.KV8TreeAttention(c, q, out, *where(**w), mask, **more)


def keep(c=None, seqs=3, depth=5, **kw):
    c = c or cache()
    path, kept = kw.pop("path", far(38, (seqs, depth), "<i4")), kw.pop("kept", far(39, (seqs,), "<i4"))
    return S.KV8Keep(c, *where(seqs=seqs, **kw), path, kept)


def set_in(op, path, value):
    at, _, name = path.rpartition(".")
    part = op.desc
    for n in at.split("."):
        part = getattr(part, n) if n else part
    setattr(part, name, value)
    return op


def test_accepted():
    passes(tree())
    passes(tree(words=32, window=5))
    passes(tree(mask=far(31, (7, 2), "<i4", strides=(40, 4))))
    passes(tree(tokens=1, mask=far(31, (1, 3), "<i4", strides=(0, 4))))
    for kw in (dict(), dict(q_out=None), dict(dt="<u2"), dict(interleaved=True, amplitude=2.0), dict(rot=2), dict(rot=64),
               dict(positions=far(40, (7,), "<i4")), dict(positions=far(40, (7,), "<i8")), dict(heads=1), dict(c=cache(code="|u1"))):
        passes(turn(**kw))
    for kw in (dict(), dict(dt="<u2"), dict(window=3, positions=far(40, (7,), "<i4")), dict(lse=far(25, (7, 4), "<f4")), dict(scale=0.0),
               dict(max_q=64), dict(heads=14), dict(c=cache(columns=256, page=256)), dict(words=32, max_q=1024),
               dict(mask=far(31, (7, 2), "<i4", strides=(0, 4))), dict(c=cache(code="|u1"), max_k=1 << 30)):
        passes(attention(**kw))
    passes(keep())
    passes(keep(c=cache(code="|u1", page=256)))
    passes(keep(path=far(38, (3, 5), "<i4", strides=(44, 4))))
    for op in (tree(seqs=0), tree(tokens=0), turn(seqs=0), turn(tokens=0), attention(seqs=0), attention(tokens=0), keep(seqs=0), keep(depth=0)):
        assert launch(op)[0] == 0


def test_tree_refused():
    for kw in (dict(parents=far(30, (7,), "<i8")), dict(parents=far(30, (7, 1), "<i4")), dict(mask=far(31, (6, 2), "<i4")),
               dict(mask=far(31, (7, 2), "<i8")), dict(mask=far(31, (7,), "<i4")), dict(positions=far(32, (6,), "<i4")),
               dict(positions=far(32, (7,), "<i8")), dict(q_start=far(15, (3,), "<i4")), dict(mask=far(31, (7, 2), "<i4", strides=(16, 8)))):
        with pytest.raises(ValueError):
            tree(**kw)
    refused(tree(words=33), "KTIR_E_UNSUPPORTED", "words")
    refused(tree(mask=far(31, (7, 0), "<i4")), "KTIR_E_UNSUPPORTED", "words")
    refused(tree(window=-1), match="window")
    refused(tree(mask=far(31, (7, 2), "<i4", strides=(4, 4))), match="overlap")
    for name in ("parents", "q_start", "kv_len"):
        refused(tree(mask=far(31, (7, 2), "<i4"), **{name: Fake(dict(parents=(7,), q_start=(4,), kv_len=(3,))[name], "<i4", ptr=(35 << 30) + 8)}), match="overlaps")
        x = dict(parents=(7,), q_start=(4,), kv_len=(3,))[name]
        refused(tree(**{name: far(32, x, "<i4")}), match="overlaps")
    refused(tree(positions=Fake((7,), "<i4", ptr=(35 << 30) + 8)), match="overlaps")
    for path, value in (("parents", 0), ("q_start", 0), ("kv_len", 2), ("mask", 0), ("positions", 1), ("seqs", -1), ("tokens", -1),
                        ("mask_row", -1), ("window", 1 << 31)):
        refused(set_in(tree(), path, value))
    assert rt.opened().ktir_launch_draft_tree(None) == rt.K["KTIR_E_ARG"]


def test_turn_refused():
    shape, kv = (7, 4, 64), (7, 2, 64)
    for kw in (dict(q=far(33, (7, 4, 32), "<f2")), dict(q=far(33, shape, "<f4")), dict(k=far(34, (7, 3, 64), "<f2")), dict(k=far(34, kv, "<u2")),
               dict(v=far(35, (6, 2, 64), "<f2")), dict(q_out=far(37, (7, 3, 64), "<f2")), dict(q_out=far(37, shape, "<u2")),
               dict(freq=far(36, (16,), "<f4")), dict(rot=66), dict(positions=far(40, (6,), "<i4")), dict(positions=far(40, (7,), "<f4")),
               dict(table=far(14, (2, 4), "<i4")), dict(q_start=far(15, (3,), "<i4"))):
        with pytest.raises(ValueError):
            turn(**kw)
    # outputs on inputs
    refused(turn(q_out=Fake(shape, "<f2", ptr=(37 << 30) + 128)), match="overlaps")
    refused(turn(q_out=far(34, shape, "<f2")), match="overlaps")
    refused(turn(q_out=far(35, shape, "<f2")), match="overlaps")
    refused(turn(q_out=far(36, shape, "<f2")), match="overlaps")
    refused(turn(q_out=far(40, shape, "<f2"), positions=far(40, (7,), "<i4")), match="overlaps")
    refused(turn(q_out=far(14, shape, "<f2")), match="overlaps")
    refused(turn(q_out=far(37, shape, "<f2", strides=(512, 64, 2))), match="overlap")
    for n, name in ((10, "k"), (11, "v"), (12, "k"), (13, "v"), (10, "q"), (12, "q")):
        refused(turn(**{name: far(n, shape if name == "q" else kv, "<f2")}), match="cache overlaps")
    refused(turn(positions=far(12, (7,), "<i4")), match="cache overlaps")
    refused(turn(freq=far(10, (16,), "<f8")), match="cache overlaps")
    refused(turn(kv_len=far(13, (3,), "<i4")), match="cache overlaps")
    # queries, keys and values of one projection, in place
    row = dict(strides=(8 * 128, 128, 2))
    qkv = [Fake((7, n, 64), "<f2", ptr=(37 << 30) + 128 * at, **row) for n, at in ((4, 0), (2, 4), (2, 6))]
    passes(turn(q=qkv[0], k=qkv[1], v=qkv[2], q_out=None))
    refused(turn(q=Fake((7, 5, 64), "<f2", ptr=37 << 30, **row), heads=5, k=qkv[1], v=qkv[2], q_out=None), match="overlaps")
    refused(turn(c=cache(k=far(10, (9, 16, 2, 64), "|i1", strides=(0, 128, 64, 1)))), match="overlap")
    refused(turn(amplitude=math.nan), match="amplitude")
    for path, value, code in (("rot", 0, "KTIR_E_ARG"), ("rot", 7, "KTIR_E_ARG"), ("rot", 66, "KTIR_E_ARG"), ("q_heads", 0, "KTIR_E_ARG"),
                              ("dtype", rt.K["KTIR_F32"], "KTIR_E_UNSUPPORTED"), ("freq", 0, "KTIR_E_ARG"), ("freq", 4, "KTIR_E_ARG"),
                              ("pos", 4 << 30, "KTIR_E_UNSUPPORTED"), ("q.ptr", 0, "KTIR_E_ARG"), ("q_out.ptr", 0, "KTIR_E_ARG"),
                              ("k.ptr", 0, "KTIR_E_ARG"), ("v.tok", -1, "KTIR_E_ARG"), ("batch.table", 0, "KTIR_E_ARG"),
                              ("cache.columns", 72, "KTIR_E_UNSUPPORTED"), ("q_heads", 65537, "KTIR_E_ARG")):
        refused(set_in(turn(), path, value), code)
    op = turn(positions=far(40, (7,), "<i8"))
    refused(set_in(op, "pos", (1 << 40) + 4), match="bounds")
    assert rt.opened().ktir_launch_kv8_rope_append(None) == rt.K["KTIR_E_ARG"]


def test_attention_refused():
    for kw in (dict(q=far(22, (7, 4, 32), "<f2")), dict(out=far(23, (7, 3, 64), "<f2")), dict(out=far(23, (7, 4, 64), "<u2")), dict(heads=3),
               dict(window=-1), dict(window=1 << 31, positions=far(40, (7,), "<i4")), dict(window=3), dict(scale=math.nan), dict(max_q=-1),
               dict(max_k=-1), dict(max_k=1 << 31), dict(lse=far(25, (7, 3), "<f4")), dict(mask=far(31, (6, 2), "<i4")),
               dict(mask=far(31, (7, 2), "<i8")), dict(mask=far(31, (7, 2), "<i4", strides=(16, 8))), dict(positions=far(40, (7,), "<i8")),
               dict(positions=far(40, (6,), "<i4")), dict(max_q=65), dict(words=1, max_q=33)):
        with pytest.raises(ValueError):
            attention(**kw)
    for kw in (dict(words=33), dict(mask=far(31, (7, 0), "<i4"), max_q=0), dict(c=cache(columns=72))):
        with pytest.raises(NotImplementedError):
            attention(**kw)
    passes(attention(out=far(22, (7, 4, 64), "<f2")))
    refused(attention(out=Fake((7, 4, 64), "<f2", ptr=(26 << 30) + 512)), match="overlaps")
    refused(attention(out=far(23, (7, 4, 64), "<f2", strides=(512, 64, 2))), match="overlap")
    refused(attention(out=far(31, (7, 4, 64), "<f2")), match="overlaps the mask")
    refused(attention(out=far(40, (7, 4, 64), "<f2"), positions=far(40, (7,), "<i4"), window=2), match="overlaps the mask")
    refused(attention(lse=far(31, (7, 4), "<f4")), match="overlaps the mask")
    refused(attention(lse=far(23, (7, 4), "<f4")), match="overlaps")
    refused(attention(out=far(12, (7, 4, 64), "<f2")), match="overlaps the cache")
    for path, value in (("mask", 0), ("mask", (1 << 40) + 2), ("mask_row", -1), ("pos", 2), ("attn.splits", -1), ("attn.max_q", 65), ("attn.batch.kv_len", 0)):
        refused(set_in(attention(), path, value))
    op = attention(window=2, positions=far(40, (7,), "<i4"))
    refused(set_in(op, "pos", 0), match="positions")
    refused(set_in(attention(), "words", 33), "KTIR_E_UNSUPPORTED")
    refused(set_in(attention(), "attn.dtype", rt.K["KTIR_F32"]), "KTIR_E_UNSUPPORTED")
    assert rt.opened().ktir_launch_kv8_tree_attention(None) == rt.K["KTIR_E_ARG"]
    assert rt.opened().ktir_kv8_tree_attention_plan(None) == rt.K["KTIR_E_ARG"]


def test_keep_refused():
    for kw in (dict(path=far(38, (2, 5), "<i4")), dict(path=far(38, (3, 5), "<i8")), dict(kept=far(39, (2,), "<i4")), dict(kept=far(39, (3,), "<i8")),
               dict(path=far(38, (3, 5), "<i4", strides=(40, 8)))):
        with pytest.raises(ValueError):
            keep(**kw)
    for n in (10, 11, 12, 13):
        refused(keep(path=far(n, (3, 5), "<i4")), match="overlaps")
        refused(keep(kept=far(n, (3,), "<i4")), match="overlaps")
        refused(keep(kv_len=far(n, (3,), "<i4")), match="overlaps")
    refused(keep(c=cache(v_scale=far(13, (9, 2), "<f4", strides=(0, 4)))), match="share a scale")
    for path, value in (("path", 0), ("kept", 0), ("kept", 2), ("depth", -1), ("path_row", -1), ("batch.table", 0), ("cache.k", 0)):
        refused(set_in(keep(), path, value))
    assert rt.opened().ktir_launch_kv8_keep(None) == rt.K["KTIR_E_ARG"]


def test_plans_are_in_bounds():
    """Splits and workspace of every shape of launch."""
    for columns in (16, 64, 80, 128, 192, 256):
        for heads, grp in ((1, 1), (2, 7), (8, 4), (4, 16), (3, 40)):
            for tokens, seqs, max_q, max_k in ((1, 1, 1, 1), (8, 1, 8, 1 << 30), (64, 1, 64, 131072), (512, 64, 8, 8192), (7, 3, 0, 64), (7, 3, 3, 0),
                                               (1024, 1, 1024, 8192), (500, 12, 400, 4000), (300, 300, 1, 100), (1000, 40, 64, 20000)):
                for window in (0, 1, 1000):
                    c = cache(heads=heads, columns=columns)
                    op = attention(c, tokens=tokens, heads=heads * grp, seqs=seqs, words=32, max_q=max_q, max_k=max_k, window=window,
                                   positions=far(40, (tokens,), "<i4"), out=Fake((tokens, heads * grp, columns), "<f2", ptr=1 << 40))
                    d = op.desc.attn
                    assert 1 <= d.splits <= 2048
                    assert (op.workspace_bytes > 0) == (d.splits > 1) and op.workspace_bytes <= 1 << 31
                    passes(op)
                    if d.splits > 1:
                        for name, value in (("ws", 0), ("ws", (1 << 41) + 8), ("ws_bytes", op.workspace_bytes - 4), ("splits", 2 * d.splits)):
                            was = getattr(d, name)
                            setattr(d, name, value)
                            refused(op)
                            setattr(d, name, was)


def test_descriptors_match_c(tmp_path):
    names = ("ktir_draft_tree_t", "ktir_kv8_rope_append_t", "ktir_kv8_tree_attn_t", "ktir_kv8_keep_t")
    src = '#include <stdio.h>\n#include <stddef.h>\n#include "ktir_hip.h"\nint main(){' + "".join(
        f'printf("%zu ", sizeof({n}));' for n in names) + 'printf("%zu %zu %zu %zu\\n", offsetof(ktir_draft_tree_t, stream), ' \
        'offsetof(ktir_kv8_rope_append_t, interleaved), offsetof(ktir_kv8_tree_attn_t, words), offsetof(ktir_kv8_keep_t, depth));}'
    (tmp_path / "s.c").write_text(src)
    exe = str(tmp_path / "s")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "s.c"), "-o", exe], check=True)
    got = [int(x) for x in subprocess.run([exe], capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(x) for x in (rt.DraftTree, rt.KV8RopeAppend, rt.KV8TreeAttn, rt.KV8Keep)] + [
        rt.DraftTree.stream.offset, rt.KV8RopeAppend.interleaved.offset, rt.KV8TreeAttn.words.offset, rt.KV8Keep.depth.offset]


# ---- the plain implementations themselves, on examples done by hand ------------------------------

def test_plain_tree():
    #      0        1
    #     / \       |
    #    2   3      4
    #    |
    #    5
    parents = torch.tensor([-1, -1, 0, 0, 1, 2], dtype=torch.int32)
    q_start, kv_len = torch.tensor([0, 6], dtype=torch.int32), torch.tensor([16], dtype=torch.int32)
    blank = torch.zeros((6, 1), dtype=torch.int32), torch.zeros(6, dtype=torch.int32)
    mask, pos = P.tree(parents, q_start, kv_len, 1, 0, *blank)
    assert mask[:, 0].tolist() == [1, 2, 5, 9, 18, 37] and pos.tolist() == [10, 10, 11, 11, 11, 12]
    mask, _ = P.tree(parents, q_start, kv_len, 1, 2, *blank)
    assert mask[:, 0].tolist() == [1, 2, 5, 9, 18, 36]
    see = P.seen_of(mask, 6, 16, 2, pos)
    assert see[5].nonzero().flatten().tolist() == [12, 15] and see[0].nonzero().flatten().tolist() == [9, 10]
    assert see[3].nonzero().flatten().tolist() == [10, 13]


def test_plain_keep():
    # one head of 16 columns, pages of 16: tokens 14 on are new, 16 and 17 of the next page move to 15 and 16
    codes = torch.zeros((2, 16, 1, 16), dtype=torch.int8)
    codes[0, :, 0, 0] = torch.arange(16, dtype=torch.int8) * 4
    codes[1, :, 0, 0] = torch.arange(100, 116, dtype=torch.int8)
    scale = torch.tensor([[1.0], [2.0]])
    table, q_start, kv_len = torch.tensor([[0, 1]], dtype=torch.int32), torch.tensor([0, 6], dtype=torch.int32), torch.tensor([20], dtype=torch.int32)
    got, new, live = P.keep(codes, scale, "i8", 16, table, q_start, kv_len, torch.tensor([[0, 2, 4]], dtype=torch.int32), torch.tensor([3]))
    # 100 * 2 is the first page's largest: its scale is 200 / 127, and 56 becomes 35.56
    assert new.flatten().tolist() == [pytest.approx(200 / 127), 2.0]
    assert got[0, 15, 0, 0] == 127 and got[0, 14, 0, 0] == 36 and got[1, 0, 0, 0] == 102
    assert live[1].tolist() == [True] + [False] * 3 + [True] * 12
