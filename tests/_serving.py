"""Plain implementations, in float64 and sequence by sequence, of the serving
operators, and how far an f32 kernel with 16-bit operands may be from them."""
import math

import torch

TOP = {"i8": 127.0, "e4m3": 448.0}
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
CODE = {"i8": torch.int8, "e4m3": torch.float8_e4m3fn}
# half a step of each type, relative to the value, and the least step's half (subnormals)
HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134, "f32": 2.0 ** -150}


def rope(x, pos, freq, *, interleaved=False, amplitude=1.0, inverse=False):
    """(rotated x in float64, its error bound) of x [tokens, heads, columns]."""
    rot = 2 * len(freq)
    y, size = x.double().clone(), x.double().abs()
    ang = torch.outer(pos.double(), torch.as_tensor(freq, dtype=torch.float64)) * (-1.0 if inverse else 1.0)
    c, s = (ang.cos() * amplitude)[:, None], (ang.sin() * amplitude)[:, None]
    ia = torch.arange(0, rot, 2) if interleaved else torch.arange(rot // 2)
    ib = ia + 1 if interleaved else ia + rot // 2
    a, b = y[..., ia].clone(), y[..., ib].clone()
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    both = torch.zeros_like(y)
    both[..., ia] = both[..., ib] = (size[..., ia] + size[..., ib]) * abs(amplitude)
    # cosine and sine: the angle's remainder in f32 (2^-24 of at most pi), a few
    # units of the function, the product with the amplitude: 2^-21 together; the two
    # products and their sum: 3 roundings
    return y, both * (2.0 ** -21 + 3 * 2.0 ** -24)


def lengths(q_start, kv_len, s):
    return int(q_start[s]), int(q_start[s + 1]) - int(q_start[s]), int(kv_len[s])


def codes_of(x, code):
    """f32 values over their scale as codes."""
    if code == "i8":
        return x.round().clamp(-127, 127).to(torch.int8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def append(x, codes, scale, code, page, table, q_start, kv_len):
    """The codes and scales after x [tokens, heads, columns] was appended: the same
    f32 operations in the same order, so they are equal bit for bit."""
    codes, scale = codes.clone(), scale.clone()
    raw = codes.view(torch.uint8)
    for s in range(len(kv_len)):
        start, n, kv = lengths(q_start, kv_len, s)
        pos0 = kv - n
        for p in range(max(pos0, 0) // page, -(-kv // page)):
            lo, hi = max(p * page, pos0, 0), min((p + 1) * page, kv)
            if lo >= hi:
                continue
            at, r0 = int(table[s, p]), lo - p * page
            new = x[start + lo - pos0:start + hi - pos0].float()
            for h in range(x.shape[1]):
                v = new[:, h]
                before = scale[at, h].clone() if r0 else torch.tensor(0.0)
                now = torch.maximum(v.abs().max() * torch.tensor(1.0 / TOP[code]), torch.tensor(2.0 ** -100))
                now = now if now >= before else before
                if not torch.isfinite(v).all():
                    now = torch.tensor(math.nan)
                if r0 and now > before:
                    old = raw[at, :r0, h].view(codes.dtype).float()
                    raw[at, :r0, h] = codes_of(old * (before * (1.0 / now)), code).view(torch.uint8)
                if torch.isfinite(now):
                    raw[at, r0:r0 + hi - lo, h] = codes_of(v * (1.0 / now), code).view(torch.uint8)
                else:
                    raw[at, r0:r0 + hi - lo, h] = 0
                scale[at, h] = now
    return codes, scale


def attention(q, k, v, k_scale, v_scale, table, q_start, kv_len, *, scale, causal=True, window=0, heads=None):
    """(out, lse, bound of out, bound of lse) in float64; rows of no sequence, and heads
    other than `heads`, are NaN."""
    D, grp, page = q.shape[2], q.shape[1] // k.shape[2], k.shape[1]
    heads = range(q.shape[1]) if heads is None else heads
    out = torch.full(q.shape, math.nan, dtype=torch.float64)
    lse = torch.full(q.shape[:2], math.nan, dtype=torch.float64)
    bound, lbound = torch.zeros_like(out), torch.zeros_like(lse)
    for s in range(len(kv_len)):
        start, n, kv = lengths(q_start, kv_len, s)
        held = table[s, :-(-kv // page)].long()
        kk, vv = ((c.view(torch.uint8)[held].view(c.dtype).double() * sc[held].double()[:, None, :, None])
                  .reshape(-1, k.shape[2], D)[:kv] for c, sc in ((k, k_scale), (v, v_scale)))
        vs = v_scale[held].double().repeat_interleave(page, 0)[:kv]
        j = torch.arange(kv)
        for i in range(n):
            pos = kv - n + i
            seen = (j <= pos) if causal else (j >= 0)
            if window:
                seen &= j > pos - window
            for h in heads:
                a, b = kk[seen, h // grp], vv[seen, h // grp]
                row = q[start + i, h].double()
                if not len(a):
                    out[start + i, h], lse[start + i, h] = 0.0, -math.inf
                    continue
                w = (a @ row) * scale
                p = torch.softmax(w, 0)
                out[start + i, h], lse[start + i, h] = p @ b, torch.logsumexp(w, 0)
                # a score is a sum of `columns` products in f32, times two scales, less the maximum:
                # each of columns + 6 roundings is 2^-24 of the sum of sizes
                ds = ((a.abs() @ row.abs()) * abs(scale)).max() * (D + 6) * 2.0 ** -24 + 2.0 ** -21
                # a weight: its exponential twice that far off above and below the line, f16 (2^-11),
                # and the f32 sums over the keys
                rel = 2 * ds + 2.0 ** -11 + len(a) * 2.0 ** -23
                # and a weight (times its page's scale) that is less than 2^-25 of the row's largest is
                # held in steps of 2^-24 where the largest is at least 2^11: half a step is 2^-36 of it
                unit = vs[seen, h // grp]
                small = 2.0 ** -36 * (p * unit).max() * (b.abs() / unit.clamp(min=2.0 ** -100)[:, None]).sum(0)
                bound[start + i, h] = (p @ b.abs()) * rel + small
                lbound[start + i, h] = ds + len(a) * 2.0 ** -24 + abs(lse[start + i, h]) * 2.0 ** -22
    return out, lse, bound, lbound


def close(got, want, bound, dt, what=""):
    """got (of type dt) is want, rounded once, but for `bound`."""
    g, w = got.double().cpu(), want
    fine = torch.isfinite(w)
    assert torch.equal(torch.isnan(g), torch.isnan(w)), what
    far = (g - w).abs()[fine] - (bound[fine] * (1 + HALF[dt]) + w.abs()[fine] * HALF[dt] + TINY[dt])
    assert not len(far) or far.max() <= 0, (what, float(far.max()), int((far > 0).sum()), int(fine.sum()))


class Batch:
    """A random cache, its table and a batch, on the CPU.  lens: (new, cached) tokens."""

    def __init__(self, lens, *, hk=2, grp=2, D=64, page=16, code="i8", dt="f16", pad=0, front=0, seed=0, spread=0.5):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.code, self.dt, self.page, self.hk, self.D = lens, code, dt, page, hk, D
        need = [-(-k // page) for _, k in lens]
        self.pages = sum(need) + 2
        order = torch.randperm(self.pages, generator=g).to(torch.int32)
        self.width = max(max(need, default=0), 1)
        self.table = torch.full((len(lens), self.width), -1, dtype=torch.int32)     # past the end: nothing that may be read
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        starts = [front]
        for n, _ in lens:
            starts.append(starts[-1] + n)
        self.q_start = torch.tensor(starts, dtype=torch.int32)
        self.kv_len = torch.tensor([k for _, k in lens], dtype=torch.int32)
        self.tokens = starts[-1] + pad
        shape = (self.pages, page, hk, D)

        def codes():
            x = torch.randn(shape, generator=g)
            return codes_of(x * (35 if code == "i8" else 120), code)

        def scales():
            return torch.exp(torch.randn((self.pages, hk), generator=g) * spread) * (3.0 / TOP[code])
        self.k, self.v, self.k_scale, self.v_scale = codes(), codes(), scales(), scales()

        def normal(heads, size):
            return (torch.randn((self.tokens, heads, D), generator=g) * size).to(DT[dt])
        self.q, self.new_k, self.new_v = normal(hk * grp, 1.5), normal(hk, 1.2), normal(hk, 1.2)

    def cache(self):
        return self.k, self.v, self.k_scale, self.v_scale

    def where(self):
        return self.table, self.q_start, self.kv_len

    @property
    def most(self):
        return dict(max_q=max([n for n, _ in self.lens], default=0), max_k=max([k for _, k in self.lens], default=0))
