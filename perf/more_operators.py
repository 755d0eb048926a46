"""Cases of the operators for drafted tokens: what a served model's layer does
with a tree of tokens that a draft proposed, over a paged key / value cache in 8 bits.

* tree: positions and ancestor masks of the drafted tokens, from their parents;
* turn: rotary positions of queries and keys, the keys and values appended to
  the cache on the way;
* attention: the drafted tokens over the cache, each seeing its ancestors;
* keep: the accepted path's entries moved to where they belong in the cache.

``run`` computes each in elementary torch operations where ``own`` is false,
and with the launches of ``ktir_cpu_amd.serving`` where it is true.  ``exact``
computes the same in float64, sequence by sequence.

A batch is `seqs` sequences.  Sequence s brings q_start[s + 1] - q_start[s]
new tokens, the last of its kv_len[s] tokens; its keys lie in the pages
table[s, 0], table[s, 1], ... of the cache.  New token i's parent is an earlier
new token of its sequence, or -1: it follows the tokens cached before.  Tokens
from q_start[seqs] on pad the batch.
"""

import math
import random

import torch

own = False

_DEV = "cuda" if torch.cuda.is_available() else "cpu"
_TORCH = {"f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8, "e4m3": torch.float8_e4m3fn}
_TOP = {"i8": 127.0, "e4m3": 448.0}
_FLOOR = 2.0 ** -100            # the least scale a page gets


def listed():
    heads = dict(hq=32, hk=8, D=128)
    return [
        # the drafts of a decode step of 64 sequences, as one layer's or all layers' launches read them
        dict(name="tree_64x64", op="tree", seqs=64, q_lo=4, q_hi=64, k_lo=64, k_hi=8192, salt=1, branch=6, window=0, pad=0),
        # deep, wide drafts and chunks of prompts (chains) of up to 500 tokens, a window, padded
        dict(name="tree_deep_window", op="tree", seqs=24, q_lo=1, q_hi=500, k_lo=500, k_hi=4000, salt=2, branch=2,
             window=100, pad=4),
        # one decoded token: the least work, latency alone
        dict(name="turn_decode_1", op="turn", seqs=1, q_lo=1, q_hi=1, k_lo=1000, k_hi=1000, salt=3, **heads, page=16,
             code="i8", dt="bf16", rot=128, inter=False, stretch=8.0, branch=0, pad=0),
        # a prompt of 8192 tokens behind 1000 cached ones, queries, keys and values cut from one projection's rows
        dict(name="turn_prefill_8192", op="turn", seqs=1, q_lo=8192, q_hi=8192, k_lo=9192, k_hi=9192, salt=4, **heads,
             page=16, code="i8", dt="f16", rot=128, inter=False, stretch=1.0, branch=0, pad=0),
        # drafts and chunks of uneven length, 21 / 3 heads of 80 with 20 interleaved columns turned, pages of 64
        dict(name="turn_drafts_odd", op="turn", seqs=40, q_lo=1, q_hi=100, k_lo=100, k_hi=3000, salt=5, hq=21, hk=3, D=80,
             page=64, code="e4m3", dt="bf16", rot=20, inter=True, stretch=4.0, branch=3, pad=5),
        # eight drafted tokens after a short prompt
        dict(name="attn_8_after_1000", op="attention", seqs=1, q_lo=8, q_hi=8, k_lo=1008, k_hi=1008, salt=6, **heads,
             page=16, code="i8", dt="f16", branch=3, window=0, pad=0, lse=False),
        # a step of 64 sequences, up to eight drafted tokens each after 64 to 8192
        dict(name="attn_64x8", op="attention", seqs=64, q_lo=1, q_hi=8, k_lo=64, k_hi=8192, salt=7, **heads, page=16,
             code="i8", dt="bf16", branch=3, window=0, pad=0, lse=False),
        # 64 drafted tokens after a very long document, floating codes
        dict(name="attn_64_after_131072", op="attention", seqs=1, q_lo=64, q_hi=64, k_lo=131072, k_hi=131072, salt=8,
             **heads, page=64, code="e4m3", dt="bf16", branch=8, window=0, pad=0, lse=True),
        # drafts of uneven size, a window of 1000 tokens, odd heads, padded
        dict(name="attn_odd_window", op="attention", seqs=12, q_lo=1, q_hi=100, k_lo=100, k_hi=4000, salt=9, hq=21, hk=3,
             D=80, page=32, code="i8", dt="f16", branch=5, window=1000, pad=4, lse=True),
        # wide drafts of eight long sequences
        dict(name="attn_8x256", op="attention", seqs=8, q_lo=128, q_hi=256, k_lo=2048, k_hi=16384, salt=10, **heads,
             page=16, code="i8", dt="bf16", branch=16, window=0, pad=0, lse=False),
        # one sequence's accepted tokens, a few of sixteen
        dict(name="keep_1", op="keep", seqs=1, q_lo=16, q_hi=16, k_lo=1016, k_hi=1016, salt=11, hk=8, D=128, page=16,
             code="i8", branch=3),
        # the accepted paths of a large batch, over several pages
        dict(name="keep_256", op="keep", seqs=256, q_lo=8, q_hi=64, k_lo=64, k_hi=4096, salt=12, hk=8, D=128, page=16,
             code="e4m3", branch=4),
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["tree", "turn", "attention", "attention", "keep"])
    pad = rng.choice([0, 0, 1, rng.randint(2, 9)])
    c = dict(op=op, salt=rng.randrange(1 << 30), branch=_log(rng, 1, 16))
    if op == "tree":
        c.update(seqs=_log(rng, 1, 64), q_hi=_log(rng, 1, 500), window=rng.choice([0, 0, _log(rng, 1, 1000)]), pad=pad)
        c["q_lo"] = max(1, c["q_hi"] // rng.choice([1, 2, 16]))
        c["k_hi"] = _log(rng, c["q_hi"], 65536)
        c["k_lo"] = max(1, c["k_hi"] // rng.choice([1, 50]))
        return c
    c.update(hk=rng.choice([1, 2, 3, 4, 8, 8]), D=rng.choice([64, 80, 96, 128, 128, 192, 256]),
             page=rng.choice([16, 16, 32, 64]), code=rng.choice(["i8", "i8", "e4m3"]))
    if op == "keep":
        c.update(seqs=_log(rng, 1, 256), q_hi=_log(rng, 1, 128))
    else:
        c.update(dt=rng.choice(["f16", "bf16"]), hq=c["hk"] * rng.choice([1, 2, 3, 4, 4, 7, 8]), pad=pad)
        kind = rng.choice(["one", "few", "drafts", "mixed"])
        c["seqs"] = _log(rng, 1, 64)
        c["q_hi"] = {"one": 1, "few": rng.randint(2, 16)}.get(kind) or _log(rng, 17, 4096 if op == "turn" else 512)
    c["q_lo"] = max(1, c["q_hi"] // rng.choice([1, 2, 16]))
    c["k_hi"] = _log(rng, max(16, c["q_hi"]), 65536 if c["seqs"] < 4 else 8192)
    c["k_lo"] = max(1, c["k_hi"] // rng.choice([1, 2, 50]))
    if op == "turn":
        c.update(rot=rng.choice([c["D"], c["D"], c["D"] // 2, 2 * rng.randint(1, c["D"] // 2)]), inter=rng.random() < 0.5,
                 stretch=rng.choice([1.0, 1.0, 4.0, 32.0]), branch=rng.choice([0, c["branch"] if c["q_hi"] <= 512 else 0]))
    if op == "attention":
        c.update(window=rng.choice([0, 0, 0, _log(rng, 1, c["k_hi"])]), lse=rng.random() < 0.5)
    # no more than the largest listed cases cost, the plain form's padded scores and gathered codes among it
    while True:
        q, k = _lengths(c)
        w, lot = work(c), len(q) * max(k) * c["hk"] * c["D"]
        most = max(w["bytes"] / 290e6, lot / 6e8)
        if op == "attention":
            most = max(most, w["flops"] / 1.9e11, len(q) * max(q) * max(k) * c["hq"] / 1.07e9, 2 * lot / 1.1e9)
        else:
            most = max(most, sum(q) * (c.get("hq", 0) + 2 * c["hk"]) * c["D"] / 5e7)
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


def _words(c):
    """32-bit words of a token's mask."""
    return -(-c["q_hi"] // 32)


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


def _padded(c, q_start, x, fill):
    """x [tokens, ...] as [seqs, q_hi, ...], `fill` behind a sequence's tokens; and whether a token is there."""
    i = torch.arange(c["q_hi"], device=_DEV)
    q_start = q_start.long()
    there = i < (q_start[1:] - q_start[:-1])[:, None]
    at = torch.where(there, q_start[:-1, None] + i, 0)
    return torch.where(there.reshape(there.shape + (1,) * (x.dim() - 1)), x[at], fill), there


def _family(c, q_start, parents):
    """Whether new token j of a sequence is i or an ancestor of it, [seqs, q_hi, q_hi] (i, j); and which are there."""
    p, there = _padded(c, q_start, parents.long(), -1)
    n = c["q_hi"]
    # one column more stands for the tokens before, which are their own parent
    jump = torch.where(p < 0, n, p)
    jump = torch.cat([jump, torch.full((c["seqs"], 1), n, device=_DEV)], 1)
    up = torch.eye(n + 1, dtype=torch.bool, device=_DEV).expand(c["seqs"], -1, -1)
    for _ in range(max(1, (n - 1).bit_length())):
        up = up | up.gather(1, jump[:, :, None].expand(-1, -1, n + 1))
        jump = jump.gather(1, jump)
    return up[:, :n, :n] & there[:, :, None], there


def _bits(c, family):
    """Truth values [..., q_hi] as 32-bit words [..., words]."""
    w = _words(c)
    x = torch.nn.functional.pad(family, (0, 32 * w - c["q_hi"])).reshape(*family.shape[:-1], w, 32).long()
    x = (x << torch.arange(32, device=_DEV)).sum(-1)
    return torch.where(x >= 1 << 31, x - (1 << 32), x).to(torch.int32)


def prepare(case, seed):
    c = case
    g = torch.Generator(device=_DEV)
    g.manual_seed(seed)
    q_len, k_len = _lengths(c)
    q_start = torch.tensor([0] + q_len, device=_DEV).cumsum(0).to(torch.int32)
    kv_len = torch.tensor(k_len, device=_DEV, dtype=torch.int32)
    tokens, rows = sum(q_len), sum(q_len) + c.get("pad", 0)
    s = dict(c=c, q_start=q_start, kv_len=kv_len)
    # the draft: a token's parent is one of the `branch` tokens before it, or it follows the tokens before the draft
    first = torch.repeat_interleave(q_start[:-1], q_start[1:] - q_start[:-1], output_size=tokens)
    i = torch.arange(tokens, device=_DEV, dtype=torch.int32) - first
    back = torch.rand(tokens, generator=g, device=_DEV) * max(1, c["branch"])
    s["parents"] = torch.nn.functional.pad((i - 1 - back.to(torch.int32)).clamp(min=-1), (0, rows - tokens))
    if c["op"] == "tree":
        s.update(mask=torch.zeros((rows, _words(c)), dtype=torch.int32, device=_DEV),
                 positions=torch.zeros(rows, dtype=torch.int32, device=_DEV))
        if own:
            from ktir_cpu_amd import serving
            s["launch"] = serving.DraftTree(s["parents"], q_start, kv_len, s["mask"], s["positions"], window=c["window"])
        return s

    need = [-(-n // c["page"]) for n in k_len]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=_DEV).to(torch.int32)
    held = torch.tensor(need, device=_DEV)
    width = torch.arange(max(need), device=_DEV)
    # a sequence's pages are anywhere in the cache; entries past its last page hold nothing
    table = torch.where(width < held[:, None], order[((held.cumsum(0) - held)[:, None] + width).clamp(max=pages - 1)],
                        torch.full((), -1, dtype=torch.int32, device=_DEV)).contiguous()

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=_DEV) * scale).to(_TORCH[c["dt"]])

    def codes():
        x = torch.randn((pages, c["page"], c["hk"], c["D"]), generator=g, device=_DEV, dtype=torch.float32)
        if c["code"] == "i8":
            return (x * 35).round_().clamp_(-127, 127).to(torch.int8)
        return (x * 120).clamp_(-448, 448).to(torch.float8_e4m3fn)

    def scales():                # a page's largest value is about 3.6 of a head's standard deviation
        return torch.exp(torch.randn((pages, c["hk"]), generator=g, device=_DEV) * 0.3) * (3.6 / _TOP[c["code"]])

    s.update(k_codes=codes(), v_codes=codes(), k_scale=scales(), v_scale=scales(), table=table)
    if c["op"] != "turn" or c["branch"]:
        # what a program has from the drafts' tree once a step, for all layers
        family, there = _family(c, q_start, s["parents"])
        positions = ((kv_len - (q_start[1:] - q_start[:-1]))[:, None] - 1 + family.sum(-1))[there].to(torch.int32)
        s["positions"] = torch.nn.functional.pad(positions, (0, rows - tokens))
    if c["op"] == "turn":
        qkv = normal(rows, c["hq"] + 2 * c["hk"], c["D"])
        freq, amp = _frequencies(c)
        s.update(q=qkv[:, :c["hq"]], k=qkv[:, c["hq"]:c["hq"] + c["hk"]], v=qkv[:, c["hq"] + c["hk"]:], freq=freq, amp=amp,
                 q_out=torch.zeros((rows, c["hq"], c["D"]), dtype=qkv.dtype, device=_DEV))
        s.setdefault("positions", None)         # (without a tree: their places in the cache)
    elif c["op"] == "attention":
        near = torch.ones_like(family)
        if c["window"]:
            depth = family.sum(-1)
            near = depth[:, :, None] - depth[:, None] < c["window"]
        q = normal(rows, c["hq"], c["D"], scale=2.0)
        s.update(q=q, out=torch.zeros_like(q), scale=c["D"] ** -0.5,
                 mask=torch.nn.functional.pad(_bits(c, family & near)[there], (0, 0, 0, rows - tokens)).contiguous(),
                 lse=torch.zeros((rows, c["hq"]), dtype=torch.float32, device=_DEV) if c["lse"] else None)
    else:
        # the path from the draft's first tokens to one of its tokens, anywhere in it
        at = (torch.rand(c["seqs"], generator=g, device=_DEV) * torch.tensor(q_len, device=_DEV)).long()
        on = family[torch.arange(c["seqs"], device=_DEV), at]
        path = torch.full((c["seqs"], c["q_hi"] + 1), -1, dtype=torch.int32, device=_DEV)
        path.scatter_(1, torch.where(on, on.long().cumsum(1) - 1, c["q_hi"]),
                      torch.arange(c["q_hi"], device=_DEV, dtype=torch.int32).expand(c["seqs"], -1).contiguous())
        s.update(path=path[:, :c["q_hi"]].contiguous(), kept=on.sum(1).to(torch.int32))
    if own:
        from ktir_cpu_amd import serving
        cache = serving.KV8Cache(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"])
        if c["op"] == "turn":
            s["launch"] = serving.KV8RopeAppend(cache, s["q"], s["k"], s["v"], s["freq"], table, q_start, kv_len, s["q_out"],
                                                positions=s["positions"], interleaved=c["inter"], amplitude=s["amp"])
        elif c["op"] == "attention":
            s["launch"] = serving.KV8TreeAttention(cache, s["q"], s["out"], table, q_start, kv_len, s["mask"], max_q=max(q_len),
                                                   max_k=max(k_len), scale=s["scale"], window=c["window"],
                                                   positions=s["positions"], lse=s["lse"])
        else:
            s["launch"] = serving.KV8Keep(cache, table, q_start, kv_len, s["path"], s["kept"])
    return s


def run(state):
    op = state["c"]["op"]
    if own:
        state["launch"].run()
    else:
        {"tree": _tree, "turn": _turn, "attention": _attention, "keep": _keep}[op](state)
    cache = ["k_codes", "v_codes", "k_scale", "v_scale"]
    names = {"tree": ["mask", "positions"], "turn": ["q_out"] + cache, "attention": ["out", "lse"], "keep": cache}[op]
    return [state[x] for x in names if state[x] is not None]


# ---- the plain forms -------------------------------------------------------------

def _tree(s):
    c, q_start = s["c"], s["q_start"].long()
    family, there = _family(c, q_start, s["parents"])
    depth = family.sum(-1)                                                        # and one: of the token itself
    if c["window"]:
        family = family & (depth[:, :, None] - depth[:, None] < c["window"])
    tokens = torch.where(there, q_start[:-1, None] + torch.arange(c["q_hi"], device=_DEV), s["mask"].shape[0])
    pos = (s["kv_len"].long() - (q_start[1:] - q_start[:-1]))[:, None] + depth - 1
    for x, to in ((_bits(c, family), s["mask"]), (pos.to(torch.int32), s["positions"])):
        wide = torch.cat([to, to[:1]])                                            # a row more takes what is behind the sequences
        wide[tokens.reshape(-1)] = x.reshape(-1, *to.shape[1:])
        to.copy_(wide[:-1])


def _coded(x, code):
    """Values over their page's scale as codes."""
    if code == "i8":
        return x.round().clamp(-127, 127).to(torch.int8)
    return x.clamp(-448, 448).to(torch.float8_e4m3fn)


def _bytes(x):
    """Codes as bytes: what indexing of floating codes is done on."""
    return x.view(torch.uint8)


def _turned(c, x, cos, sin):
    y, rot = x.float(), c["rot"]
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if c["inter"] else (y[..., :rot // 2], y[..., rot // 2:rot])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if c["inter"] else torch.cat([a, b], -1)
    return torch.cat([turned, y[..., rot:]], -1)


def _turn(s):
    c, table, page = s["c"], s["table"], s["c"]["page"]
    q_start, kv_len = s["q_start"].long(), s["kv_len"].long()
    # tokens that pad the batch do again what the last one does
    token = torch.minimum(torch.arange(s["k"].shape[0], device=_DEV), q_start[-1] - 1)
    seq = torch.searchsorted(q_start, token, right=True) - 1
    place = kv_len[seq] - q_start[seq + 1] + token
    pos = place if s["positions"] is None else s["positions"].long()[token]
    turns = pos[:, None].double() * s["freq"] * (0.5 / math.pi)     # 32 bits lose the angle of a far position
    angle = (turns - turns.round()) * (2 * math.pi)
    cos, sin = (angle.cos() * s["amp"]).float()[:, None], (angle.sin() * s["amp"]).float()[:, None]
    y = _turned(c, s["q"][token], cos, sin).to(s["q_out"].dtype)
    live = torch.arange(s["k"].shape[0], device=_DEV) < q_start[-1]
    s["q_out"].copy_(torch.where(live[:, None, None], y, s["q_out"]))
    at, row = table[seq, place // page].long(), place % page
    pages = s["k_scale"].shape[0]
    # the page that a sequence's first new token goes to, and how many older rows it holds
    first = kv_len - (q_start[1:] - q_start[:-1])
    head = table[torch.arange(c["seqs"], device=_DEV), first // page].long()
    older = first % page
    for x, codes, scale in ((_turned(c, s["k"][token], cos, sin), s["k_codes"], s["k_scale"]),
                            (s["v"][token].float(), s["v_codes"], s["v_scale"])):
        top = torch.full((pages, c["hk"]), -1.0, device=_DEV)
        top.scatter_reduce_(0, at[:, None].expand(-1, c["hk"]), x.abs().amax(-1), "amax")
        touched, fresh = top >= 0, (top * (1 / _TOP[c["code"]])).clamp(min=_FLOOR)
        before = scale[head]
        fresh[head] = torch.where((older > 0)[:, None], torch.maximum(before, fresh[head]), fresh[head])
        new = torch.where(touched, fresh, scale)
        inv = 1.0 / new
        # older rows of a page whose scale grew are rounded to the new one
        old = _bytes(codes)[head].view(codes.dtype)
        again = _coded(old.float() * (before * inv[head])[:, None, :, None], c["code"])
        same = (torch.arange(page, device=_DEV) >= older[:, None])[..., None, None] | (new[head] <= before)[:, None, :, None]
        _bytes(codes)[head] = torch.where(same, _bytes(old), _bytes(again))
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
    before = (kv_len - q_len)[:, None]
    key = torch.arange(n, device=_DEV)
    seen = (key < before)[:, None].expand(-1, most, -1)                           # [B, most, keys]
    if c["window"]:
        seen = seen & (key > s["positions"].long()[token][..., None] - c["window"])
    bit = key - before                                                            # a key's number in the draft
    word = s["mask"][token].gather(2, (bit // 32).clamp(0, _words(c) - 1)[:, None].expand(-1, most, -1))
    seen = seen | ((bit >= 0) & (bit < q_len[:, None]))[:, None] & ((word >> (bit % 32)[:, None]) & 1).bool()
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


def _keep(s):
    c, page, most = s["c"], s["c"]["page"], s["c"]["q_hi"]
    q_start, kv_len, path = s["q_start"].long(), s["kv_len"].long(), s["path"].long()
    before = (kv_len - (q_start[1:] - q_start[:-1]))[:, None]
    i = torch.arange(most, device=_DEV)
    there = i < s["kept"][:, None]
    to = before + torch.where(there, i, 0)
    src = before + torch.where(there, path, 0)                                     # (places past the last: the first new token's)
    seq = torch.arange(c["seqs"], device=_DEV)[:, None]
    to_page, from_page = s["table"][seq, to // page].long(), s["table"][seq, src // page].long()
    came, stays = there & (to_page != from_page), there & (to_page == from_page)
    pages = s["k_scale"].shape[0]
    # a page keeps its scale if it keeps a token: one of before, or one of the draft's that lay there
    held = torch.zeros(pages + 1, dtype=torch.bool, device=_DEV)
    held[torch.where(stays, to_page, pages)] = True
    held[torch.where(before % page > 0, to_page[:, :1], pages)] = True
    gets = torch.zeros(pages + 1, dtype=torch.bool, device=_DEV)
    gets[torch.where(came, to_page, pages)] = True
    held, gets = held[:pages, None], gets[:pages, None]
    last = torch.zeros((), device=_DEV)
    for codes, scale in ((s["k_codes"], s["k_scale"]), (s["v_codes"], s["v_scale"])):
        x = _bytes(codes)[from_page, src % page].view(codes.dtype).float()        # [seqs, most, heads, columns]
        top = torch.where(came[..., None], x.abs().amax(-1) * scale[from_page], last)
        new = torch.zeros((pages, c["hk"]), device=_DEV)
        new.scatter_reduce_(0, to_page.reshape(-1, 1).expand(-1, c["hk"]), top.reshape(-1, c["hk"]), "amax")
        new = (new * (1 / _TOP[c["code"]])).clamp(min=_FLOOR)
        new = torch.where(gets, torch.where(held, torch.maximum(new, scale), new), scale)
        inv = 1.0 / new
        # older rows of a page whose scale grew are rounded to the new one
        head = to_page[:, 0]
        old = _bytes(codes)[head].view(codes.dtype)
        again = _coded(old.float() * (scale[head] * inv[head])[:, None, :, None], c["code"])
        same = (torch.arange(page, device=_DEV) >= before % page)[..., None, None] | (new[head] <= scale[head])[:, None, :, None]
        _bytes(codes)[head] = torch.where(same, _bytes(old), _bytes(again))
        ratio = torch.where((from_page == to_page)[..., None] & (new[to_page] <= scale[to_page]), torch.ones_like(top),
                            scale[from_page] * inv[to_page])
        y = _bytes(_coded(x * ratio[..., None], c["code"]))
        _bytes(codes)[to_page[there], (to % page)[there]] = y[there]
        scale.copy_(new)


# ---- work and exact results --------------------------------------------------------

def work(case):
    c = case
    q, k = _lengths(c)
    n = sum(q)
    if c["op"] == "tree":
        return dict(bytes=n * (8 + 4 * _words(c)) + 8 * c["seqs"], flops=0)
    row = c["hk"] * c["D"]
    if c["op"] == "turn":
        pages = sum((b - 1) // c["page"] - (b - a) // c["page"] + 1 for a, b in zip(q, k))
        return dict(bytes=n * (4 * c["hq"] * c["D"] + 6 * row) + pages * (8 * c["hk"] + 4) + 4 * c["rot"],
                    flops=3 * n * (c["hq"] + c["hk"]) * c["rot"] + 4 * n * row)
    if c["op"] == "keep":       # the paths follow from the seed: of a draft of n tokens about 2 n / (branch + 1) lie on one, half of them are kept
        kept = sum(max(1, round(a / (c["branch"] + 1))) for a in q)
        return dict(bytes=kept * (4 * row + 4) + 16 * c["seqs"], flops=4 * kept * row)
    # a drafted token's ancestors, two in (branch + 1) of those before it, and the tokens before the draft
    pairs = keys = 0
    for a, b in zip(q, k):
        near = min(b - a, c["window"] or b)
        keys += near + a
        pairs += a * near + round(a + a * (a - 1) / (c["branch"] + 1))
    return dict(bytes=4 * n * c["hq"] * c["D"] + 2 * keys * row + -(-keys // c["page"]) * (8 * c["hk"] + 4) + 4 * n * _words(c),
                flops=4 * pairs * c["hq"] * c["D"])


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "tree":                       # whole numbers
        return None
    q_len, k_len = _lengths(c)
    start = [0]
    for n in q_len:
        start.append(start[-1] + n)
    page, table, tokens = c["page"], s["table"].tolist(), start[-1]
    if c["op"] == "keep":                       # codes are whole numbers, and have no value in 64 bits: the scales alone
        outs, paths, kept = [None, None], s["path"].tolist(), s["kept"].tolist()
        for codes, scale in ((s["k_codes"], s["k_scale"]), (s["v_codes"], s["v_scale"])):
            new, old, size = scale.double().cpu(), scale.double().cpu(), codes.double().abs().amax(-1).cpu()
            for b, (a, n) in enumerate(zip(q_len, k_len)):
                ctx, pages = n - a, {}
                for i, j in enumerate(paths[b][:kept[b]]):
                    pages.setdefault((ctx + i) // page, []).append((ctx + j) // page * page + (ctx + j) % page)
                for p, places in pages.items():
                    came = [x for x in places if x // page != p]
                    if came:
                        stays = len(came) < len(places) or p * page < ctx
                        top = torch.stack([size[table[b][x // page], x % page] * old[table[b][x // page]] for x in came]).amax(0)
                        top = (top / _TOP[c["code"]]).clamp(min=_FLOOR)
                        new[table[b][p]] = torch.maximum(top, old[table[b][p]]) if stays else top
            outs.append(new.to(_DEV))
        return outs
    if c["op"] == "turn":
        place = torch.cat([torch.arange(n - a, n, device=_DEV) for a, n in zip(q_len, k_len)])
        pos = place if s["positions"] is None else s["positions"][:tokens]
        angle = torch.outer(pos.double(), s["freq"])
        z = torch.polar(torch.full_like(angle, s["amp"]), angle)                   # amp e^(i angle)

        def turned(x):
            y = x.double().clone()
            r = y[..., :c["rot"]]
            pair = r.reshape(*r.shape[:-1], -1, 2) if c["inter"] else r.reshape(*r.shape[:-1], 2, -1).transpose(-1, -2)
            t = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * z[:, None])
            y[..., :c["rot"]] = (t if c["inter"] else t.transpose(-1, -2)).reshape(r.shape)
            return y

        outs = [torch.nn.functional.pad(turned(s["q"][:tokens]), (0, 0, 0, 0, 0, s["q"].shape[0] - tokens)), None, None]
        for x, scale in ((turned(s["k"][:tokens]), s["k_scale"]), (s["v"][:tokens].double(), s["v_scale"])):
            new, size = scale.double(), x.abs().amax(-1)
            for b, (a, n) in enumerate(zip(q_len, k_len)):
                for lo in range((n - a) // page * page, n, page):
                    t0 = max(lo, n - a)
                    top = size[start[b] + t0 - (n - a):start[b] + min(lo + page, n) - (n - a)].amax(0) / _TOP[c["code"]]
                    old = new[table[b][lo // page]] if t0 > lo else torch.zeros_like(top)
                    new[table[b][lo // page]] = torch.maximum(old, top).clamp(min=_FLOOR)
            outs.append(new)
        return outs
    out, lse = s["out"].double(), torch.zeros((s["out"].shape[0], c["hq"]), dtype=torch.float64, device=_DEV)
    grp, parents = c["hq"] // c["hk"], s["parents"].tolist()
    for b, (a, n) in enumerate(zip(q_len, k_len)):
        t = s["table"][b, :-(-n // page)].long()
        k, v = ((x.view(torch.uint8)[t].view(x.dtype).double() * y[t].double()[:, None, :, None]).reshape(-1, c["hk"], c["D"])[:n]
                for x, y in ((s["k_codes"], s["k_scale"]), (s["v_codes"], s["v_scale"])))
        hide = torch.zeros((a, n), dtype=torch.bool)
        hide[:, n - a:] = True
        for i in range(a):                       # up from the token to the draft's first, then the tokens before it
            line, j = [], i
            while j >= 0:
                line.append(j)
                j = parents[start[b] + j]
            hide[i, [n - a + j for j in line[:c["window"] or None]]] = False
            if c["window"]:
                hide[i, :max(0, min(n - a, n - a + len(line) - c["window"]))] = True
        hide = hide.to(_DEV)
        for h in range(c["hk"]):
            kt, vh = k[:, h].t().contiguous(), v[:, h].contiguous()
            x = s["q"][start[b]:start[b + 1], h * grp:(h + 1) * grp].double()
            w = (x.reshape(-1, c["D"]) @ kt * s["scale"]).reshape(a, grp, n).masked_fill(hide[:, None], -math.inf)
            lse[start[b]:start[b + 1], h * grp:(h + 1) * grp] = torch.logsumexp(w, -1)
            out[start[b]:start[b + 1], h * grp:(h + 1) * grp] = (torch.softmax(w, -1).reshape(-1, n) @ vh).reshape(x.shape)
    return [out] + ([lse] if s["lse"] is not None else [])
