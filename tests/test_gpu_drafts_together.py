"""The operators for drafted tokens where they can go wrong together: steps of a decoding
program, graphs, streams, large batches, far pages, and what a row does not see."""
import math

import numpy as np
import pytest
import torch

from ktir_cpu_amd import serving as S
from tests import _drafts as P
from tests._serving import DT, Batch, append, close, rope
from tests.test_gpu_drafts import attend, cache_of, check, dev, done, freq_of, same_bits, tree_of

pytestmark = pytest.mark.gpu


# ---- large and uneven batches ------------------------------------------------------------

@pytest.mark.parametrize("grp,D,code,most", [(2, 64, "i8", 9), (4, 128, "e4m3", 40), (1, 192, "i8", 50), (8, 128, "i8", 60)])
def test_attention_of_many_uneven_sequences(grp, D, code, most):
    # more sequences than are looked at together, some without new tokens, one much longer than all others
    g = torch.Generator().manual_seed(most)
    lens = []
    for s in range(150):
        n = int(torch.randint(0, most if s % 7 == 0 else 3, (), generator=g))
        lens.append((n, n + int(torch.randint(0, 90, (), generator=g))))
    lens[70] = (most, 3000 + most)
    b = Batch(lens, hk=2, grp=grp, D=D, page=16, code=code, dt="f16", pad=2, front=1, seed=3)
    mask, _ = tree_of(b, 3, 0, front=1, pad=2)
    _, out, line = attend(b, mask)
    done()
    check(b, out, line, mask)


@pytest.mark.parametrize("lens,grp,D", [([(10, 700), (7, 300)], 4, 256), ([(25, 400)], 2, 192), ([(20, 60), (0, 9), (3, 1500), (16, 16)], 3, 160),
                                        ([(32, 5000)], 2, 256)])
def test_attention_of_wide_heads_in_two_tiles(lens, grp, D):
    # 33 to 64 rows of a KV head of more than 128 columns
    b = Batch(lens, hk=2, grp=grp, D=D, page=16, code="i8", dt="bf16", seed=D)
    mask, pos = tree_of(b, 2, 50)
    _, out, line = attend(b, mask, pos, window=50)
    done()
    check(b, out, line, mask, 50, pos)
    mask, _ = tree_of(b, 2, 0)
    _, out, line = attend(b, mask)
    done()
    check(b, out, line, mask)


def test_turn_and_tree_of_many_sequences():
    g = torch.Generator().manual_seed(8)
    lens = [(int(torch.randint(0, 4, (), generator=g)), 0) for _ in range(200)]
    lens = [(n, n + int(torch.randint(0, 40, (), generator=g))) for n, _ in lens]
    b = Batch(lens, hk=2, grp=2, D=64, page=16, code="i8", dt="bf16", seed=1)
    words = 1
    mask, pos = torch.zeros((b.tokens, words), dtype=torch.int32, device="cuda"), torch.zeros(b.tokens, dtype=torch.int32, device="cuda")
    parents = P.random_parents(lens, 2)
    S.DraftTree(dev(parents), *dev(b.q_start, b.kv_len), mask, pos).run()
    cache, arrays = cache_of(b)
    freq = freq_of(64)
    q = dev(b.q)
    S.KV8RopeAppend(cache, q, *dev(b.new_k, b.new_v, freq, *b.where()), positions=pos).run()
    done()
    want_mask, want_pos = P.tree(parents, b.q_start, b.kv_len, words, 0, torch.zeros((b.tokens, 1), dtype=torch.int32), torch.zeros(b.tokens, dtype=torch.int32))
    assert torch.equal(mask.cpu(), want_mask) and torch.equal(pos.cpu(), want_pos)
    k = P.turned(b.new_k, want_pos.long(), freq, False, 1.0)
    want_k, want_v = append(k, b.k, b.k_scale, "i8", 16, *b.where()), append(b.new_v, b.v, b.v_scale, "i8", 16, *b.where())
    for got, want in zip(arrays, (want_k[0], want_v[0], want_k[1], want_v[1])):
        same_bits(got, want)
    want, bound = rope(b.q, want_pos.long(), freq)
    close(q, want, bound, "bf16")


def test_far_pages():
    """Pages more than 4 GiB into the cache: every operator reads and writes the right ones."""
    pages, page, hk, D = 80000, 256, 2, 128                     # 5.2 GB a cache
    lens = [(20, 300), (9, 500)]
    b = Batch(lens, hk=hk, grp=4, D=D, page=page, code="i8", dt="bf16", seed=5)
    spots = torch.randperm(200, generator=torch.Generator().manual_seed(2))[:b.pages] + pages - 200
    k, v = (torch.zeros((pages, page, hk, D), dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros((pages, hk), device="cuda") for _ in range(2))
    at = spots.cuda()
    k[at], v[at], ks[at], vs[at] = dev(*b.cache())
    table = torch.where(b.table >= 0, spots[b.table.clamp(min=0).long()].to(torch.int32), b.table)
    cache = S.KV8Cache(k, v, ks, vs)
    freq, where = freq_of(128), P.places(b.q_start, b.kv_len, b.tokens)
    args = dev(table, b.q_start, b.kv_len)
    q = dev(b.q)
    S.KV8RopeAppend(cache, q, *dev(b.new_k, b.new_v, freq), *args).run()
    done()
    want_k = append(P.turned(b.new_k, where, freq, False, 1.0), b.k, b.k_scale, "i8", page, *b.where())
    want_v = append(b.new_v, b.v, b.v_scale, "i8", page, *b.where())
    for got, want in zip((k, v, ks, vs), (want_k[0], want_v[0], want_k[1], want_v[1])):
        same_bits(got[at], want)
    b.k, b.k_scale, b.v, b.v_scale = *want_k, *want_v
    mask, _ = tree_of(b, 2, 0)
    for rows in (4, 1):                                          # the kernels for many rows, and for few
        hq = 2 * rows
        out = torch.zeros((b.tokens, hq, D), dtype=torch.bfloat16, device="cuda")
        few = Batch(lens, hk=hk, grp=rows, D=D, page=page, code="i8", dt="bf16", seed=5)
        S.KV8TreeAttention(cache, dev(few.q), out, *args, dev(mask), **b.most).run()
        done()
        want, _, bound, _ = P.attention(few.q, *b.cache(), *b.where(), mask, scale=D ** -0.5)
        close(out, want, bound, "bf16")
    path, kept = torch.tensor([[0, 3, 7, 19], [2, 8, -1, -1]], dtype=torch.int32), torch.tensor([4, 2], dtype=torch.int32)
    S.KV8Keep(cache, *args, *dev(path, kept)).run()
    done()
    for codes, scale, got, gscale in ((b.k, b.k_scale, k, ks), (b.v, b.v_scale, v, vs)):
        want, wscale, live = P.keep(codes, scale, "i8", page, *b.where(), path, kept)
        same_bits(got[at].cpu()[live], want[live])
        same_bits(gscale[at], wscale)
    assert not k[:pages - 200].any() and not v[:pages - 200].any()


# ---- what a row does not see ------------------------------------------------------------------

@pytest.mark.parametrize("n,grp", [(40, 1), (40, 2), (40, 4), (80, 4)])
@pytest.mark.parametrize("code", ["i8", "e4m3"])
def test_a_page_that_is_nan_reaches_only_those_who_see_it(n, grp, code):
    b = Batch([(n, 16 * 5 + n), (2, 40)], hk=2, grp=grp, D=128, page=16, code=code, dt="f16", seed=n)
    mask, _ = tree_of(b, 4, 0, seed=4)
    page = int(b.table[0, 6])                                    # new tokens 16 to 31
    half = mask[:, 0].clone()
    mask[:n:2, 0] = half[:n:2] & 0xffff                          # every second row sees none of them
    sees = ((mask[:n, 0] >> 16) & 0xffff) != 0
    clean = [x.clone() for x in b.cache()]
    b.k_scale[page, 0] = math.nan
    b.v_scale[page, 1] = math.nan
    _, out, line = attend(b, mask)
    done()
    want, wline, bound, lbound = P.attention(b.q, *clean, *b.where(), mask, scale=128 ** -0.5)
    for h in range(2 * grp):
        blind = torch.ones(b.tokens, dtype=torch.bool)
        blind[:n] = ~sees
        close(out[blind.cuda(), h], want[blind, h], bound[blind, h], "f16")
        assert ((line.cpu()[blind, h] - wline[blind, h]).abs() <= lbound[blind, h]).all()
        assert out[:n][sees.cuda(), h].isnan().all()


# ---- repeated, at once, other streams, graphs -----------------------------------------------------

def test_results_repeat():
    for lens, grp in (([(8, 3000), (5, 900), (1, 50)], 4), ([(100, 3000), (40, 900)], 4)):
        b = Batch(lens, hk=2, grp=grp, D=128, page=16, dt="bf16", seed=3)
        mask, _ = tree_of(b, 3, 0)
        op, out, line = attend(b, mask)
        done()
        first = out.clone(), line.clone()
        for _ in range(5):
            out.fill_(3), line.fill_(3)
            op.run()
            done()
            same_bits(out, first[0])
            same_bits(line, first[1])


def test_launches_at_once_and_a_shared_workspace():
    batches = [Batch([(n, k), (3, 700)], hk=2, grp=4, D=128, page=16, dt="f16", seed=n) for n, k in ((8, 5000), (60, 4000), (16, 9000), (100, 2500))]
    masks = [tree_of(b, 3, 0)[0] for b in batches]
    streams = [torch.cuda.Stream() for _ in batches]
    ops = [attend(b, m) for b, m in zip(batches, masks)]
    done()
    for _, out, line in ops:
        out.fill_(7), line.fill_(7)
    torch.cuda.synchronize()
    for _ in range(3):
        for (op, _, _), s in zip(ops, streams):
            op.run(s)
    done()
    for b, m, (_, out, line) in zip(batches, masks, ops):
        check(b, out, line, m)
    # one workspace for launches that follow one another, of garbage to begin with
    most = max(op.workspace_bytes for op, _, _ in ops)
    ws = torch.full((most,), 0xff, dtype=torch.uint8, device="cuda")
    again = [attend(b, m, workspace=ws) for b, m in zip(batches, masks)]
    done()
    for b, m, (_, out, line) in zip(batches, masks, again):
        check(b, out, line, m)


def test_device_arrays_on_the_library_stream():
    b = Batch([(9, 120), (4, 33)], hk=2, grp=2, D=64, page=16, dt="f16", seed=6)
    parents, freq = P.random_parents(b.lens, 2), freq_of(64)
    put = lambda t: S.DeviceArray(t.numpy() if isinstance(t, torch.Tensor) else t)  # noqa: E731
    arrays = [put(x) for x in b.cache()]
    cache, where = S.KV8Cache(*arrays), [put(x) for x in b.where()]
    mask, pos = put(np.zeros((b.tokens, 1), np.int32)), put(np.zeros(b.tokens, np.int32))
    q, out = put(b.q), put(np.zeros(b.q.shape, np.float16))
    path, kept = torch.tensor([[0, 4, 8], [1, -1, -1]], dtype=torch.int32), torch.tensor([3, 1], dtype=torch.int32)
    S.DraftTree(put(parents), where[1], where[2], mask, pos).run()
    S.KV8RopeAppend(cache, q, put(b.new_k), put(b.new_v), put(freq.numpy()), *where, positions=pos).run()
    S.KV8TreeAttention(cache, q, out, *where, mask, **b.most).run()
    got_cache = [x.numpy() for x in arrays]
    S.KV8Keep(cache, *where, put(path), put(kept)).run()
    done()
    want_mask, want_pos = P.tree(parents, b.q_start, b.kv_len, 1, 0, torch.zeros((b.tokens, 1), dtype=torch.int32), torch.zeros(b.tokens, dtype=torch.int32))
    assert (mask.numpy() == want_mask.numpy()).all() and (pos.numpy() == want_pos.numpy()).all()
    want_k = append(P.turned(b.new_k, want_pos.long(), freq, False, 1.0), b.k, b.k_scale, "i8", 16, *b.where())
    want_v = append(b.new_v, b.v, b.v_scale, "i8", 16, *b.where())
    for got, want in zip(got_cache, (want_k[0], want_v[0], want_k[1], want_v[1])):
        np.testing.assert_array_equal(got, want.numpy())
    turned = torch.from_numpy(q.numpy())
    want, _, bound, _ = P.attention(turned, want_k[0], want_v[0], want_k[1], want_v[1], *b.where(), want_mask, scale=64 ** -0.5)
    close(torch.from_numpy(out.numpy()), want, bound, "f16")
    for (codes, scale), got, gscale in ((want_k, arrays[0], arrays[2]), (want_v, arrays[1], arrays[3])):
        end, escale, live = P.keep(codes, scale, "i8", 16, *b.where(), path, kept)
        assert (got.numpy()[live.numpy()] == end[live].numpy()).all()
        same_bits(torch.from_numpy(gscale.numpy()), escale)


class Program:
    """Two layers that draft: the launches of a step, on arrays that stay, and the plain
    implementations of the same beside them."""

    def __init__(self, first, *, most=12, code="i8", dt="bf16", grp=4, seed=0):
        self.g = torch.Generator().manual_seed(seed)
        self.seqs, self.most, self.code, self.dt, self.grp, self.hk, self.D, self.page = len(first), most, code, dt, grp, 2, 64, 16
        self.width = 30
        tokens = self.seqs * most
        self.layers = []
        self.freq = freq_of(64)
        pages = self.seqs * self.width
        self.table = torch.randperm(pages, generator=self.g).to(torch.int32).reshape(self.seqs, self.width)
        self.kv = torch.tensor(first, dtype=torch.int32)           # cached tokens, without drafts
        self.d = {n: dev(t) for n, t in dict(
            table=self.table, q_start=torch.zeros(self.seqs + 1, dtype=torch.int32), kv_len=self.kv.clone(), parents=torch.zeros(tokens, dtype=torch.int32),
            mask=torch.zeros((tokens, 1), dtype=torch.int32), pos=torch.zeros(tokens, dtype=torch.int32),
            path=torch.zeros((self.seqs, most), dtype=torch.int32), kept=torch.zeros(self.seqs, dtype=torch.int32), freq=self.freq).items()}
        d = self.d
        where = d["table"], d["q_start"], d["kv_len"]
        self.tree = S.DraftTree(d["parents"], d["q_start"], d["kv_len"], d["mask"], d["pos"])
        for _ in range(2):
            b = Batch([(1, 16 * self.width)] * self.seqs, hk=2, grp=grp, D=64, page=16, code=code, dt=dt, seed=int(torch.randint(0, 999, (), generator=self.g)))
            cpu = [x[:pages].clone() for x in b.cache()]
            gpu = dev(*[x.clone() for x in cpu])
            cache = S.KV8Cache(*gpu)
            qkv = torch.zeros((tokens, 2 * grp + 4, 64), dtype=DT[dt], device="cuda")
            q, k, v = qkv[:, :2 * grp], qkv[:, 2 * grp:2 * grp + 2], qkv[:, 2 * grp + 2:]
            out = torch.zeros((tokens, 2 * grp, 64), dtype=DT[dt], device="cuda")
            turned = torch.zeros_like(out)
            self.layers.append(dict(
                cpu=cpu, gpu=gpu, qkv=qkv, out=out, turned=turned,
                store=S.KV8RopeAppend(cache, q, k, v, d["freq"], *where, turned, positions=d["pos"]),
                attend=S.KV8TreeAttention(cache, turned, out, *where, d["mask"], max_q=most, max_k=16 * self.width),
                keep=S.KV8Keep(cache, *where, d["path"], d["kept"])))

    def draft(self):
        """The next drafts, and every layer's projections."""
        self.n = [int(torch.randint(1, self.most + 1, (), generator=self.g)) for _ in range(self.seqs)]
        self.lens = [(n, n + int(k)) for n, k in zip(self.n, self.kv)]
        self.q_start = torch.tensor([0] + self.n).cumsum(0).to(torch.int32)
        self.kv_len = self.kv + torch.tensor(self.n, dtype=torch.int32)
        self.tokens = sum(self.n)
        self.parents = P.random_parents(self.lens, 3, seed=int(torch.randint(0, 999, (), generator=self.g)))
        self.qkv = [(torch.randn(x["qkv"].shape, generator=self.g) * 1.3).to(DT[self.dt]) for x in self.layers]
        self.d["q_start"].copy_(self.q_start), self.d["kv_len"].copy_(self.kv_len)
        self.d["parents"][:self.tokens].copy_(self.parents)
        for x, y in zip(self.layers, self.qkv):
            x["qkv"].copy_(y)

    def run(self):
        self.tree.run()
        for x in self.layers:
            x["store"].run()
            x["attend"].run()

    def check(self):
        where = self.table, self.q_start, self.kv_len
        n, hq = self.tokens, 2 * self.grp
        mask, pos = P.tree(self.parents, self.q_start, self.kv_len, 1, 0, torch.zeros((n, 1), dtype=torch.int32), torch.zeros(n, dtype=torch.int32))
        assert torch.equal(self.d["mask"][:n].cpu(), mask) and torch.equal(self.d["pos"][:n].cpu(), pos)
        for x, qkv in zip(self.layers, self.qkv):
            k, v, ks, vs = x["cpu"]
            turned = P.turned(qkv[:n, hq:hq + 2], pos.long(), self.freq, False, 1.0)
            k, ks = append(turned, k, ks, self.code, 16, *where)
            v, vs = append(qkv[:n, hq + 2:], v, vs, self.code, 16, *where)
            x["cpu"] = [k, v, ks, vs]
            for got, want in zip(x["gpu"], x["cpu"]):
                same_bits(got, want)
            want, bound = rope(qkv[:n, :hq], pos.long(), self.freq)
            close(x["turned"][:n], want, bound, self.dt)
            want, _, bound, _ = P.attention(x["turned"][:n].cpu(), *x["cpu"], *where, mask, scale=64 ** -0.5)
            close(x["out"][:n], want, bound, self.dt)

    def accept(self):
        """Paths that the drafts' outputs choose, kept by both; the lengths follow."""
        lines = [P.family(self.parents[int(self.q_start[s]):int(self.q_start[s + 1])].tolist()) for s in range(self.seqs)]
        path, kept = torch.full((self.seqs, self.most), -1, dtype=torch.int32), torch.zeros(self.seqs, dtype=torch.int32)
        score = self.layers[1]["out"][:self.tokens].float().sum((1, 2)).cpu()
        for s in range(self.seqs):
            best = int(score[int(self.q_start[s]):int(self.q_start[s + 1])].argmax())
            line = sorted(lines[s][best])
            path[s, :len(line)], kept[s] = torch.tensor(line, dtype=torch.int32), len(line)
        self.d["path"].copy_(path), self.d["kept"].copy_(kept)
        self.path, self.kept = path, kept

    def keep(self):
        for x in self.layers:
            x["keep"].run()

    def kept_too(self):
        where = self.table, self.q_start, self.kv_len
        for x in self.layers:
            k, v, ks, vs = x["cpu"]
            k, ks, live = P.keep(k, ks, self.code, 16, *where, self.path, self.kept)
            v, vs, _ = P.keep(v, vs, self.code, 16, *where, self.path, self.kept)
            for got, want in zip(x["gpu"], (k, v)):
                same_bits(got.cpu()[live], want[live])
            same_bits(x["gpu"][2], ks), same_bits(x["gpu"][3], vs)
            # entries behind the path are undefined: the plain ones go on with the same
            x["cpu"] = [t.cpu() for t in x["gpu"]]
        self.kv = self.kv + self.kept


@pytest.mark.parametrize("code,dt,grp,most", [("i8", "bf16", 4, 12), ("e4m3", "f16", 2, 20), ("i8", "f16", 4, 28)])
def test_steps_of_a_decoding_program(code, dt, grp, most):
    m = Program([0, 40, 200], most=most, code=code, dt=dt, grp=grp, seed=grp + most)
    for _ in range(5):
        m.draft()
        m.run()
        done()
        m.check()
        m.accept()
        m.keep()
        done()
        m.kept_too()


def test_steps_on_another_stream_and_in_graphs():
    """A step's launches captured once, then replayed on new drafts and lengths, with the program's own
    work and waits between the replays, beside a second program's."""
    a, b = Program([5, 90, 333], seed=1), Program([64, 1], most=30, code="e4m3", dt="f16", seed=2)
    side = torch.cuda.Stream()
    graphs = []
    for m in (a, b):
        m.draft()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            m.run()
        side.synchronize()
        m.check()
        m.accept()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            m.keep()
        side.synchronize()
        m.kept_too()
        step, keep = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(step):
            m.run()
        with torch.cuda.graph(keep):
            m.keep()
        graphs.append((step, keep))
    for _ in range(4):
        for m, (step, _) in zip((a, b), graphs):
            m.draft()
            step.replay()
        torch.cuda.synchronize()
        junk = torch.randn(1 << 20, device="cuda").sort()
        for m, (_, keep) in zip((a, b), graphs):
            m.check()
            m.accept()
            keep.replay()
        torch.cuda.synchronize()
        del junk
        for m in (a, b):
            m.kept_too()
    done()


def test_rope_append_is_rope_and_append_but_for_their_rounding():
    """Against the two launches: the same values, and codes of keys that differ by one step at most where 16 bits round."""
    b = Batch([(300, 400), (1, 77)], hk=2, grp=2, D=128, page=16, code="i8", dt="f16", seed=2)
    freq, where = freq_of(128), P.places(b.q_start, b.kv_len, b.tokens)
    one, two = cache_of(b), cache_of(b)
    args, f = dev(*b.where()), dev(freq)
    q, k, v = dev(b.q, b.new_k, b.new_v)
    q1 = torch.zeros_like(q)
    S.KV8RopeAppend(one[0], q, k, v, f, *args, q1).run()
    q2, k2 = torch.zeros_like(q), torch.zeros_like(k)
    S.Rope(q, dev(where), f, q2, k=k, k_out=k2).run()
    S.KV8Append(two[0], k2, v, *args).run()
    done()
    same_bits(q1, q2)
    same_bits(one[1][1], two[1][1])
    same_bits(one[1][3], two[1][3])
    assert (one[1][0].int() - two[1][0].int()).abs().max() <= 1
    # a page's scale follows its largest value, which f16 rounds by 2^-11
    assert ((one[1][2] - two[1][2]).abs() <= two[1][2] * (2.0 ** -11 + 2.0 ** -22)).all()
