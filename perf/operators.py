"""Cases of the serving operators: what one layer of a served model does with a
paged key/value cache that is held in 8 bits.

* rope: rotary positions of the queries and keys of a batch of tokens;
* append: new keys and values into the cache, quantised with one scale for
  each page of tokens and KV head;
* attention: the batch's queries over the cache.

``run`` computes each in elementary torch operations where ``own`` is false,
and with the launches of ``ktir_cpu_amd.serving`` where it is true.  ``exact``
computes the same in float64, sequence by sequence.

A batch is `seqs` sequences.  Sequence s brings q_start[s + 1] - q_start[s]
new tokens, the last of its kv_len[s] tokens; its keys lie in the pages
table[s, 0], table[s, 1], ... of the cache.  Tokens from q_start[seqs] on pad
the batch.
"""

import math
import random

import torch

own = False

_DEV = "cuda" if torch.cuda.is_available() else "cpu"
_TORCH = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "i8": torch.int8,
          "e4m3": torch.float8_e4m3fn}
_TOP = {"i8": 127.0, "e4m3": 448.0}
_FLOOR = 2.0 ** -100            # the least scale a page gets


def listed():
    return [
        # one decoded token, 32 query and 8 key heads, a context stretched by the ramp of a long-context model
        dict(name="rope_decode_1", op="rope", tokens=1, heads=32, kheads=8, D=128, rot=128, dt="bf16", inter=False,
             inverse=False, far=131072, stretch=8.0, pad=0),
        # a long prompt, queries and keys cut from one projection's rows
        dict(name="rope_prefill_8192", op="rope", tokens=8192, heads=32, kheads=8, D=128, rot=128, dt="f16",
             inter=False, inverse=False, far=8192, stretch=1.0, pad=0),
        # interleaved pairs in the first half of 40 heads (the rotary example's head count), the rest passed on
        dict(name="rope_pairs_part_4096", op="rope", tokens=4096, heads=40, kheads=40, D=128, rot=64, dt="bf16",
             inter=True, inverse=False, far=32768, stretch=4.0, pad=3),
        # the way back (a gradient through the rotation) in f32, odd sizes, queries alone
        dict(name="rope_back_f32_1151", op="rope", tokens=1151, heads=5, kheads=0, D=80, rot=20, dt="f32", inter=True,
             inverse=True, far=1151, stretch=1.0, pad=1),
        # a decode step of 64 sequences: one token each, most in the middle of a page
        dict(name="append_decode_64", op="append", seqs=64, q_lo=1, q_hi=1, k_lo=16, k_hi=8192, salt=1, hk=8, D=128,
             page=16, code="i8", dt="bf16", pad=0),
        # a prompt of 8192 tokens behind 1000 cached ones
        dict(name="append_prefill_8192", op="append", seqs=1, q_lo=8192, q_hi=8192, k_lo=9192, k_hi=9192, salt=2, hk=8,
             D=128, page=16, code="i8", dt="f16", pad=0),
        # prompts' chunks of uneven length, three heads of 80 columns, pages of 64, floating codes
        dict(name="append_chunks_odd", op="append", seqs=9, q_lo=1, q_hi=700, k_lo=1, k_hi=3000, salt=3, hk=3, D=80,
             page=64, code="e4m3", dt="bf16", pad=5),
        # one decoded token after a short prompt: the least work, latency alone
        dict(name="attn_decode_1000", op="attention", seqs=1, q_lo=1, q_hi=1, k_lo=1000, k_hi=1000, salt=4, hq=32,
             hk=8, D=128, page=16, code="i8", dt="f16", window=0, pad=0, lse=False),
        # a decode step of 64 sequences of 64 to 8192 tokens
        dict(name="attn_decode_64", op="attention", seqs=64, q_lo=1, q_hi=1, k_lo=64, k_hi=8192, salt=5, hq=32, hk=8,
             D=128, page=16, code="i8", dt="bf16", window=0, pad=0, lse=False),
        # one decoded token after a very long document, floating codes
        dict(name="attn_decode_131072", op="attention", seqs=1, q_lo=1, q_hi=1, k_lo=131072, k_hi=131072, salt=6,
             hq=32, hk=8, D=128, page=64, code="e4m3", dt="bf16", window=0, pad=0, lse=True),
        # decoding and chunks of prompts in one batch, a window of 1000 tokens, odd heads
        dict(name="attn_mixed_window", op="attention", seqs=12, q_lo=1, q_hi=500, k_lo=1, k_hi=4000, salt=7, hq=21,
             hk=3, D=80, page=32, code="i8", dt="f16", window=1000, pad=4, lse=True),
        # a whole prompt of 8192 tokens
        dict(name="attn_prefill_8192", op="attention", seqs=1, q_lo=8192, q_hi=8192, k_lo=8192, k_hi=8192, salt=8,
             hq=32, hk=8, D=128, page=16, code="i8", dt="bf16", window=0, pad=0, lse=False),
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["rope", "append", "attention", "attention"])
    pad = rng.choice([0, 0, 1, rng.randint(2, 9)])
    if op == "rope":
        D = rng.choice([32, 64, 80, 96, 128, 128, 192, 256])
        rot = rng.choice([D, D, D // 2, 2 * rng.randint(1, D // 2)])
        heads = _log(rng, 1, 40)
        kheads = rng.choice([0, 1, heads, max(1, heads // 4)])
        dt = rng.choice(["f16", "bf16", "bf16", "f32"])
        tokens = _log(rng, 1, max(1, min(8192, 8192 * 40 * 128 * 2 // ((heads + kheads) * D * (4 if dt == "f32" else 2)))))
        return dict(op=op, tokens=tokens, heads=heads, kheads=kheads, D=D, rot=rot, dt=dt, inter=rng.random() < 0.5,
                    inverse=rng.random() < 0.3, far=_log(rng, 64, 1 << 20), stretch=rng.choice([1.0, 1.0, 4.0, 32.0]),
                    pad=pad)
    c = dict(op=op, hk=rng.choice([1, 2, 3, 4, 8, 8]), D=rng.choice([64, 80, 96, 128, 128, 192, 256]),
             page=rng.choice([16, 16, 32, 64]), code=rng.choice(["i8", "i8", "e4m3"]),
             dt=rng.choice(["f16", "bf16"]), salt=rng.randrange(1 << 30), pad=pad)
    kind = rng.choice(["decode", "few", "prompt", "mixed"])
    c["seqs"] = _log(rng, 1, 8 if kind == "prompt" else 64)
    c["q_hi"] = {"decode": 1, "few": rng.randint(2, 16)}.get(kind) or _log(rng, 17, 4096)
    c["q_lo"] = 1 if kind == "mixed" else max(1, c["q_hi"] // 2)
    c["k_hi"] = _log(rng, max(16, c["q_hi"]), 65536 if c["seqs"] < 4 else 8192)
    c["k_lo"] = max(1, c["k_hi"] // rng.choice([1, 2, 50]))
    if op == "attention":
        c["hq"] = c["hk"] * rng.choice([1, 2, 3, 4, 4, 7, 8])
        c["window"] = rng.choice([0, 0, 0, _log(rng, 1, c["k_hi"])])
        c["lse"] = rng.random() < 0.5
    # no more than the largest listed cases cost, the plain form's padded scores among it
    while True:
        q, k = _lengths(c)
        heads, w = c.get("hq", c["hk"]), work(c)
        most = w["bytes"] / 290e6
        if op == "attention":
            most = max(most, w["flops"] / 5.4e11, len(q) * max(q) * max(k) * heads / 2.1e9,
                       2 * len(q) * max(k) * c["hk"] * c["D"] / 1.1e9)
        else:
            most = max(most, sum(q) * c["hk"] * c["D"] / 1.7e7, len(q) * max(k) * c["hk"] * c["D"] / 6e8)
        if most <= 1:
            return c
        for name in ("q_hi", "q_lo", "k_hi", "k_lo"):
            c[name] = max(1, round(c[name] * (0.7 if c["q_hi"] > 1 or name[0] == "k" else 1)))
        c["k_hi"] = max(c["k_hi"], c["q_hi"])


def _lengths(c):
    """New tokens and cached tokens (the new ones among them) of each
    sequence: the first has the most of both, the others are spread."""
    r = random.Random(c["salt"])
    q, k = [c["q_hi"]], [c["k_hi"]]
    while len(q) < c["seqs"]:
        q.append(_log(r, c["q_lo"], c["q_hi"]))
        k.append(max(q[-1], _log(r, c["k_lo"], c["k_hi"])))
    return q, k


def _frequencies(c):
    """Radians per position of each pair (float64), and the factor on cosine
    and sine.  stretch > 1: pairs that turn less than once in the 4096
    positions that were trained are slowed by it, those that turn more than 32
    times are kept, with a ramp over the pair's number in between."""
    rot, base, trained = c["rot"], 10000.0, 4096
    f = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if c["stretch"] == 1.0:
        return f.to(_DEV), 1.0
    at = lambda turns: rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
    ramp = ((torch.arange(rot // 2, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
    return (f * (1 - ramp) + f / c["stretch"] * ramp).to(_DEV), 0.1 * math.log(c["stretch"]) + 1.0


def prepare(case, seed):
    c = case
    g = torch.Generator(device=_DEV)
    g.manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=_DEV) * scale).to(_TORCH[c["dt"]])

    if c["op"] == "rope":
        rows = c["tokens"] + c["pad"]
        # queries, keys and values of a token lie side by side, as one projection leaves them
        qkv = normal(rows, c["heads"] + 2 * c["kheads"], c["D"])
        q, k = qkv[:, :c["heads"]], qkv[:, c["heads"]:c["heads"] + c["kheads"]]
        pos = torch.randint(0, c["far"], (rows,), generator=g, device=_DEV)
        pos = torch.where(torch.arange(rows, device=_DEV) < c["tokens"], pos, -1)     # tokens that pad the batch
        freq, amp = _frequencies(c)
        s = dict(c=c, q=q, k=k if c["kheads"] else None, pos=pos, freq=freq, amp=amp,
                 q_out=torch.zeros(q.shape, dtype=q.dtype, device=_DEV),
                 k_out=torch.zeros(k.shape, dtype=k.dtype, device=_DEV))
        if own:
            from ktir_cpu_amd import serving
            s["launch"] = serving.Rope(q, pos, freq, s["q_out"], k=s["k"], k_out=s["k_out"] if c["kheads"] else None,
                                       interleaved=c["inter"], amplitude=amp, inverse=c["inverse"])
        return s

    q_len, k_len = _lengths(c)
    need = [-(-n // c["page"]) for n in k_len]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=_DEV).to(torch.int32)
    held = torch.tensor(need, device=_DEV)
    width = torch.arange(max(need), device=_DEV)
    # a sequence's pages are anywhere in the cache; entries past its last page hold nothing
    table = torch.where(width < held[:, None], order[((held.cumsum(0) - held)[:, None] + width).clamp(max=pages - 1)],
                        torch.full((), -1, dtype=torch.int32, device=_DEV)).contiguous()
    q_start = torch.tensor([0] + q_len, device=_DEV).cumsum(0).to(torch.int32)
    kv_len = torch.tensor(k_len, device=_DEV, dtype=torch.int32)
    rows = sum(q_len) + c["pad"]

    def codes():
        x = torch.randn((pages, c["page"], c["hk"], c["D"]), generator=g, device=_DEV, dtype=torch.float32)
        if c["code"] == "i8":
            return (x * 35).round_().clamp_(-127, 127).to(torch.int8)
        return (x * 120).clamp_(-448, 448).to(torch.float8_e4m3fn)

    def scales():                # a page's largest value is about 3.6 of a head's standard deviation
        return torch.exp(torch.randn((pages, c["hk"]), generator=g, device=_DEV) * 0.3) * (3.6 / _TOP[c["code"]])

    s = dict(c=c, k_codes=codes(), v_codes=codes(), k_scale=scales(), v_scale=scales(), table=table, q_start=q_start,
             kv_len=kv_len)
    if c["op"] == "append":
        kv = normal(rows, 2 * c["hk"], c["D"], scale=1.2)
        s.update(k=kv[:, :c["hk"]], v=kv[:, c["hk"]:])
    else:
        q = normal(rows, c["hq"], c["D"], scale=2.0)
        s.update(q=q, out=torch.zeros_like(q), scale=c["D"] ** -0.5,
                 lse=torch.zeros((rows, c["hq"]), dtype=torch.float32, device=_DEV) if c["lse"] else None)
    if own:
        from ktir_cpu_amd import serving
        cache = serving.KV8Cache(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"])
        if c["op"] == "append":
            s["launch"] = serving.KV8Append(cache, s["k"], s["v"], table, q_start, kv_len)
        else:
            s["launch"] = serving.KV8Attention(cache, s["q"], s["out"], table, q_start, kv_len, max_q=max(q_len),
                                               max_k=max(k_len), scale=s["scale"], window=c["window"], lse=s["lse"])
    return s


def run(state):
    op = state["c"]["op"]
    if own:
        state["launch"].run()
    else:
        {"rope": _rope, "append": _append, "attention": _attention}[op](state)
    if op == "rope":
        return [state["q_out"]] + ([state["k_out"]] if state["k"] is not None else [])
    if op == "append":
        return [state[x] for x in ("k_codes", "v_codes", "k_scale", "v_scale")]
    return [state["out"]] + ([state["lse"]] if state["lse"] is not None else [])


# ---- the plain forms -------------------------------------------------------------

def _rope(s):
    c, live = s["c"], s["pos"] >= 0
    angle = s["pos"][:, None].double() * s["freq"]                  # 32 bits lose the angle of a far position
    cos, sin = (angle.cos() * s["amp"]).float()[:, None], (angle.sin() * s["amp"]).float()[:, None]
    if c["inverse"]:
        sin = -sin
    _rotate(c, s["q"], cos, sin, live, s["q_out"])
    if s["k"] is not None:
        _rotate(c, s["k"], cos, sin, live, s["k_out"])


def _rotate(c, x, cos, sin, live, out):
    y, rot = x.float(), c["rot"]
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if c["inter"] else (y[..., :rot // 2], y[..., rot // 2:rot])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if c["inter"] else torch.cat([a, b], -1)
    y = torch.cat([turned, y[..., rot:]], -1).to(x.dtype)
    out.copy_(torch.where(live[:, None, None], y, out))


def _coded(x, code):
    """Values over their page's scale as codes."""
    if code == "i8":
        return x.round().clamp(-127, 127).to(torch.int8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def _bytes(x):
    """Codes as bytes: what indexing of floating codes is done on."""
    return x.view(torch.uint8)


def _append(s):
    c, table, page = s["c"], s["table"], s["c"]["page"]
    q_start, kv_len = s["q_start"].long(), s["kv_len"].long()
    # tokens that pad the batch do again what the last one does
    token = torch.minimum(torch.arange(s["k"].shape[0], device=_DEV), q_start[-1] - 1)
    seq = torch.searchsorted(q_start, token, right=True) - 1
    pos = kv_len[seq] - q_start[seq + 1] + token
    at, row = table[seq, pos // page].long(), pos % page
    pages = s["k_scale"].shape[0]
    # the page that a sequence's first new token goes to, and how many older rows it holds
    first = kv_len - (q_start[1:] - q_start[:-1])
    head = table[torch.arange(c["seqs"], device=_DEV), first // page].long()
    older = first % page
    for x, codes, scale in ((s["k"], s["k_codes"], s["k_scale"]), (s["v"], s["v_codes"], s["v_scale"])):
        x = x[token].float()
        top = torch.full((pages, c["hk"]), -1.0, device=_DEV)
        top.scatter_reduce_(0, at[:, None].expand(-1, c["hk"]), x.abs().amax(-1), "amax")
        touched, fresh = top >= 0, (top / _TOP[c["code"]]).clamp(min=_FLOOR)
        before = scale[head]
        fresh[head] = torch.where((older > 0)[:, None], torch.maximum(before, fresh[head]), fresh[head])
        new = torch.where(touched, fresh, scale)
        inv = 1.0 / new
        # older rows of a page whose scale grew are rounded to the new one
        old = _bytes(codes)[head].view(codes.dtype)
        again = _coded(old.float() * (before * inv[head])[:, None, :, None], c["code"])
        keep = (torch.arange(page, device=_DEV) >= older[:, None])[..., None, None] | (new[head] <= before)[:, None, :, None]
        _bytes(codes)[head] = torch.where(keep, _bytes(old), _bytes(again))
        _bytes(codes)[at, row] = _bytes(_coded(x * inv[at][..., None], c["code"]))
        scale.copy_(new)


def _attention(s):
    c, hk, D = s["c"], s["c"]["hk"], s["c"]["D"]
    q_start, kv_len, table = s["q_start"].long(), s["kv_len"].long(), s["table"].long().clamp(min=0)
    B, n, grp = c["seqs"], table.shape[1] * c["page"], c["hq"] // hk
    q_len = q_start[1:] - q_start[:-1]
    most = c["q_hi"]

    def cached(codes, scale):
        x = _bytes(codes)[table].view(codes.dtype).float() * scale[table][:, :, None, :, None]
        return x.reshape(B, n, hk, D).transpose(1, 2)                             # [B, hk, keys, D]

    # rows past a sequence's end do again what its last one does
    i = torch.minimum(torch.arange(most, device=_DEV), q_len[:, None] - 1)       # [B, most]
    token = q_start[:-1, None] + i
    q = s["q"][token].float().reshape(B, most, hk, grp, D).permute(0, 2, 1, 3, 4).reshape(B, hk, most * grp, D)
    score = q @ cached(s["k_codes"], s["k_scale"]).transpose(2, 3).contiguous()
    score *= s["scale"]
    pos = (kv_len - q_len)[:, None] + i
    key = torch.arange(n, device=_DEV)
    seen = key <= pos[..., None]                                                  # [B, most, keys]
    if c["window"]:
        seen &= key > pos[..., None] - c["window"]
    seen = seen.repeat_interleave(grp, 1)[:, None]
    score = score.masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top)
    l = p.sum(-1, keepdim=True)
    o = (p @ cached(s["v_codes"], s["v_scale"]).contiguous()) / l
    lse = (top + torch.log(l)).squeeze(-1)
    back = lambda x: x.reshape(B, hk, most, grp, -1).permute(0, 2, 1, 3, 4).reshape(B, most, c["hq"], -1)  # noqa: E731
    s["out"][token] = back(o).to(s["out"].dtype)
    if s["lse"] is not None:
        s["lse"][token] = back(lse).squeeze(-1)


# ---- work and exact results --------------------------------------------------------

def work(case):
    c = case
    if c["op"] == "rope":
        n, e = c["tokens"] * (c["heads"] + c["kheads"]), 4 if c["dt"] == "f32" else 2
        return dict(bytes=2 * n * c["D"] * e + 8 * (c["tokens"] + c["rot"] // 2), flops=3 * n * c["rot"])
    q, k = _lengths(c)
    if c["op"] == "append":
        n = sum(q) * 2 * c["hk"]
        pages = sum((b - 1) // c["page"] - (b - a) // c["page"] + 1 for a, b in zip(q, k))
        return dict(bytes=n * c["D"] * 3 + pages * (8 * c["hk"] + 4) + 8 * c["seqs"], flops=2 * n * c["D"])
    pairs, keys = 0, 0
    for a, b in zip(q, k):
        w = c["window"] or b
        keys += min(b, w + a - 1)
        full = max(0, min(a, b - w + 1))              # rows that see w keys; the others see all up to their own
        pairs += full * w + sum(range(b - a + 1, b - full + 1))
    return dict(bytes=4 * sum(q) * c["hq"] * c["D"] + 2 * keys * c["hk"] * c["D"]
                + -(-keys // c["page"]) * (8 * c["hk"] + 4) + 8 * c["seqs"], flops=4 * pairs * c["hq"] * c["D"])


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "rope":
        angle = torch.outer(s["pos"].double(), s["freq"]) * (-1.0 if c["inverse"] else 1.0)
        z = torch.polar(torch.full_like(angle, s["amp"]), angle)                   # amp e^(i angle)
        outs = []
        for x in [s["q"]] + ([s["k"]] if s["k"] is not None else []):
            y = x.double().clone()
            r = y[..., :c["rot"]]
            pair = r.reshape(*r.shape[:-1], -1, 2) if c["inter"] else r.reshape(*r.shape[:-1], 2, -1).transpose(-1, -2)
            t = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * z[:, None])
            y[..., :c["rot"]] = (t if c["inter"] else t.transpose(-1, -2)).reshape(r.shape)
            y[c["tokens"]:] = 0.0
            outs.append(y)
        return outs
    q_len, k_len = _lengths(c)
    start = [0]
    for n in q_len:
        start.append(start[-1] + n)
    page = c["page"]
    if c["op"] == "append":                     # codes are whole numbers: the scales alone have a value in 64 bits
        outs = [None, None]
        table = s["table"].tolist()
        for x, scale in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])):
            new, size = scale.double(), x.double().abs().amax(-1)
            for b, (a, n) in enumerate(zip(q_len, k_len)):
                for lo in range((n - a) // page * page, n, page):
                    t0 = max(lo, n - a)
                    top = size[start[b] + t0 - (n - a):start[b] + min(lo + page, n) - (n - a)].amax(0) / _TOP[c["code"]]
                    old = new[table[b][lo // page]] if t0 > lo else torch.zeros_like(top)
                    new[table[b][lo // page]] = torch.maximum(old, top).clamp(min=_FLOOR)
            outs.append(new)
        return outs
    out, lse = s["out"].double(), torch.zeros((s["out"].shape[0], c["hq"]), dtype=torch.float64, device=_DEV)
    grp = c["hq"] // c["hk"]
    for b, (a, n) in enumerate(zip(q_len, k_len)):
        t = s["table"][b, :-(-n // page)].long()
        k, v = ((x.view(torch.uint8)[t].view(x.dtype).double() * y[t].double()[:, None, :, None]).reshape(-1, c["hk"], c["D"])[:n]
                for x, y in ((s["k_codes"], s["k_scale"]), (s["v_codes"], s["v_scale"])))
        key = torch.arange(n, device=_DEV)
        for h in range(c["hk"]):
            kt, vh = k[:, h].t().contiguous(), v[:, h].contiguous()
            for r in range(0, a, 1024):
                rows = slice(start[b] + r, start[b] + min(r + 1024, a))
                x = s["q"][rows, h * grp:(h + 1) * grp].double()
                pos = n - a + r + torch.arange(x.shape[0], device=_DEV)
                hide = key[None] > pos[:, None]
                if c["window"]:
                    hide |= key[None] <= pos[:, None] - c["window"]
                w = (x.reshape(-1, c["D"]) @ kt * s["scale"]).reshape(x.shape[0], grp, n)
                w = w.masked_fill(hide[:, None], -math.inf)
                lse[rows, h * grp:(h + 1) * grp] = torch.logsumexp(w, -1)
                out[rows, h * grp:(h + 1) * grp] = (torch.softmax(w, -1).reshape(-1, n) @ vh).reshape(x.shape)
    return [out] + ([lse] if s["lse"] is not None else [])
