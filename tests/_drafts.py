"""Plain implementations of the operators for drafted tokens, sequence by sequence, and how far an
f32 kernel with 16-bit operands may be from them."""
import math

import torch

from tests._serving import TOP, codes_of, lengths


def family(parents):
    """The lists of every token's line, from itself up."""
    lines = []
    for i, p in enumerate(parents):
        lines.append([i] + (lines[p] if 0 <= p < i else []))
    return lines


def tree(parents, q_start, kv_len, words, window=0, mask=None, positions=None):
    """(mask, positions) with the rows of the batch's sequences written."""
    mask, positions = mask.clone(), positions.clone()
    for s in range(len(kv_len)):
        start, n, kv = lengths(q_start, kv_len, s)
        for i, line in enumerate(family(parents[start:start + n].tolist())):
            row = [0] * words
            for j in line[:window or None]:
                row[j // 32] |= 1 << (j % 32)
            mask[start + i] = torch.tensor([w - (1 << 32) if w >> 31 else w for w in row], dtype=torch.int32)
            positions[start + i] = kv - n + len(line) - 1
    return mask, positions


def random_parents(lens, branch, seed=0, front=0, pad=0):
    """A random forest for each of the sequences: a parent is one of the `branch` tokens before, or -1."""
    g = torch.Generator().manual_seed(seed)
    out = [-7] * front
    for n, _ in lens:
        for i in range(n):
            out.append(max(-1, i - 1 - int(torch.randint(0, branch, (), generator=g))))
    return torch.tensor(out + [-7] * pad, dtype=torch.int32)


def turned(x, pos, freq, interleaved, amplitude):
    """x [tokens, heads, columns] in f32, turned by the same f32 operations in the same order: equal bit for bit."""
    turns = pos.double()[:, None] * torch.as_tensor(freq, dtype=torch.float64) * (0.5 / math.pi)
    angle = (turns - turns.round()) * (2 * math.pi)
    c, s = ((f * amplitude).float()[:, None] for f in (angle.cos(), angle.sin()))
    rot, y = 2 * len(freq), x.float().clone()
    ia = torch.arange(0, rot, 2) if interleaved else torch.arange(rot // 2)
    ib = ia + 1 if interleaved else ia + rot // 2
    a, b = x.float()[..., ia], x.float()[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    return y


def places(q_start, kv_len, tokens):
    """Every token's place in the cache; -1 outside the sequences."""
    out = torch.full((tokens,), -1, dtype=torch.int64)
    for s in range(len(kv_len)):
        start, n, kv = lengths(q_start, kv_len, s)
        out[start:start + n] = torch.arange(kv - n, kv)
    return out


def seen_of(mask_rows, n, kv, window, pos):
    """Which of kv cached tokens each of the n new ones sees, [n, kv]."""
    ctx = kv - n
    j = torch.arange(kv)
    see = (j < ctx).expand(n, -1).clone()
    if window:
        see &= j[None] > torch.clamp(pos.long(), min=ctx)[:, None] - window
    bits = (j - ctx).clamp(min=0)
    word = (bits // 32).clamp(max=mask_rows.shape[1] - 1)
    named = ((mask_rows[:, word] >> (bits % 32)) & 1).bool() & (bits < 32 * mask_rows.shape[1])
    return torch.where(j >= ctx, named, see)


def attention(q, k, v, k_scale, v_scale, table, q_start, kv_len, mask, *, scale, window=0, positions=None, heads=None):
    """(out, lse, bound of out, bound of lse) in float64; rows of no sequence, and heads other than `heads`, are NaN."""
    D, grp, page = q.shape[2], q.shape[1] // k.shape[2], k.shape[1]
    heads = range(q.shape[1]) if heads is None else heads
    out = torch.full(q.shape, math.nan, dtype=torch.float64)
    lse = torch.full(q.shape[:2], math.nan, dtype=torch.float64)
    bound, lbound = torch.zeros_like(out), torch.zeros_like(lse)
    for s in range(len(kv_len)):
        start, n, kv = lengths(q_start, kv_len, s)
        if not n:
            continue
        rows = slice(start, start + n)
        held = table[s, :-(-kv // page)].long()
        kk, vv = ((c.view(torch.uint8)[held].view(c.dtype).double() * sc[held].double()[:, None, :, None])
                  .reshape(-1, k.shape[2], D)[:kv] for c, sc in ((k, k_scale), (v, v_scale)))
        vs = v_scale[held].double().repeat_interleave(page, 0)[:kv]
        see = seen_of(mask[rows], n, kv, window, None if positions is None else positions[rows])
        some, count = see.any(1), see.sum(1)
        for h in heads:
            a, b, unit, x = kk[:, h // grp], vv[:, h // grp], vs[:, h // grp], q[rows, h].double()
            w = ((x @ a.T) * scale).masked_fill(~see, -math.inf)
            p = torch.where(some[:, None], torch.softmax(w, 1), 0.0)
            line = torch.logsumexp(w, 1)
            out[rows, h], lse[rows, h] = p @ b, line
            # a score is a sum of `columns` products in f32, times two scales, less the maximum:
            # each of columns + 6 roundings is 2^-24 of the sum of sizes
            ds = ((x.abs() @ a.abs().T) * abs(scale)).masked_fill(~see, 0.0).amax(1) * (D + 6) * 2.0 ** -24 + 2.0 ** -21
            # a weight: its exponential twice that far off above and below the line, f16 (2^-11),
            # and the f32 sums over the keys
            rel = 2 * ds + 2.0 ** -11 + count * 2.0 ** -23
            # and a weight (times its page's scale) that is less than 2^-25 of the row's largest is
            # held in steps of 2^-24 where the largest is at least 2^11: half a step is 2^-36 of it
            small = 2.0 ** -36 * (p * unit).amax(1)[:, None] * (see.double() @ (b.abs() / unit.clamp(min=2.0 ** -100)[:, None]))
            bound[rows, h] = (p @ b.abs()) * rel[:, None] + small
            lbound[rows, h] = torch.where(some, ds + count * 2.0 ** -24 + line.abs() * 2.0 ** -22, 0.0)
    return out, lse, bound, lbound


def keep(codes, scale, code, page, table, q_start, kv_len, path, kept):
    """The codes and scales after the paths were kept: the same f32 operations, so they are equal bit for bit.
    (What the entries behind a path hold is undefined: `live` says which rows of the cache count.)"""
    raw, scale = codes.clone().view(torch.uint8), scale.clone()
    old_raw, old_scale = raw.clone(), scale.clone()
    live = torch.ones(codes.shape[:2], dtype=torch.bool)
    per = torch.tensor(1.0 / TOP[code])

    def values(rows):
        return rows.view(codes.dtype).float()

    def rounded(x):
        y = codes_of(x, code)
        return y.view(torch.uint8)
    for s in range(len(kv_len)):
        start, n, kv = lengths(q_start, kv_len, s)
        ctx, entries = kv - n, {}
        for j in range(ctx + int(kept[s]), kv):
            live[int(table[s, j // page]), j % page] = False
        for i in range(int(kept[s])):
            entries.setdefault((ctx + i) // page, []).append((ctx + i, ctx + int(path[s, i])))
        for p, moves in entries.items():
            at = int(table[s, p])
            older = max(0, ctx - p * page)
            came = [m for m in moves if m[1] // page != p]
            stays = older > 0 or len(came) < len(moves)
            for h in range(codes.shape[2]):
                before = now = old_scale[at, h]
                if came:
                    top, finite = torch.tensor(0.0), True
                    for _, src in came:
                        sc = old_scale[int(table[s, src // page]), h]
                        x = values(old_raw[int(table[s, src // page]), src % page, h]).abs()
                        top = torch.maximum(top, torch.where(x.isnan(), 0.0, x).max() * sc)
                        finite = finite and bool(torch.isfinite(sc))
                    now = torch.maximum(top * per, torch.tensor(2.0 ** -100))
                    now = before if stays and not now >= before else now
                    now = now if finite else torch.tensor(math.nan)
                inv = 1.0 / now
                grown = bool(came) and stays and bool(now > before)
                if grown and older:
                    raw[at, :older, h] = rounded(values(old_raw[at, :older, h]) * (before * inv))
                for dst, src in moves:
                    x = old_raw[int(table[s, src // page]), src % page, h]
                    if (dst, src) in came:
                        x = rounded(values(x) * (old_scale[int(table[s, src // page]), h] * inv)) if torch.isfinite(now) else x * 0
                    elif grown:
                        x = rounded(values(x) * (before * inv))
                    raw[at, dst % page, h] = x
                scale[at, h] = now
    return raw.view(codes.dtype), scale, live
