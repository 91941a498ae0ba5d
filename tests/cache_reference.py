"""The state cache's operators restated in float64 (torch, any device): block tables in plain Python, the block write
and the attention from their definitions."""

from __future__ import annotations

import math

import torch

BLOCK = 64
E_MIN, E_MAX = -100, 120


def assign(lens, new, table, free, count, width):
    """(kv_len, seqpos, slots, table, count, outcome) from host lists; nothing changes when blocks are missing."""
    table = [list(row) for row in table]
    need = [-(-(a + b) // BLOCK) - -(-a // BLOCK) for a, b in zip(lens, new)]
    positions = [p for a, b in zip(lens, new) for p in range(a, a + b)]
    if any(-(-(a + b) // BLOCK) > width for a, b in zip(lens, new)):
        return list(lens), positions, [-1] * len(positions), table, count, -1
    if sum(need) > count:
        return list(lens), positions, [-1] * len(positions), table, count, sum(need) - count
    slots = []
    for i, (a, b) in enumerate(zip(lens, new)):
        have = -(-a // BLOCK)
        for k in range(need[i]):
            count -= 1
            table[i][have + k] = free[count]
        slots += [table[i][p // BLOCK] * BLOCK + p % BLOCK for p in range(a, a + b)]
    return [a + b for a, b in zip(lens, new)], positions, slots, table, count, 0


def exponent(amax: float) -> int:
    """The least e with amax * 2^-e <= 448, within the bounds."""
    if amax == 0:
        return E_MIN
    m, x = math.frexp(amax / 448.0)
    return min(max(x - (m == 0.5), E_MIN), E_MAX)


def to_e4m3(x: torch.Tensor) -> torch.Tensor:
    """Float64 values rounded to e4m3 ones, to nearest even, saturating; NaN stays."""
    mag = x.abs()
    _, e = torch.frexp(mag.clamp(2.0 ** -6, 1e300))
    step = torch.ldexp(torch.ones_like(x), e - 4)
    return torch.where(x.isnan(), x, (torch.round(x / step) * step).clamp(-448.0, 448.0))


def store(x, other, cu, slots, codes, scale, is_key):
    """The pool after writing rows ``x`` (T, H, hd) float64 (CPU): codes' values (float64) and scales, new tensors."""
    values, scales = codes.clone(), scale.clone()
    for a, b in zip(cu[:-1], cu[1:]):
        r = a
        while r < b and slots[a] >= 0:
            block, off = divmod(slots[r], BLOCK)
            stop = min(b, r + BLOCK - off)
            for h in range(x.shape[1]):
                part = x[r:stop, h]
                fin = part[part.isfinite()]
                e = exponent(float(fin.abs().max()) if fin.numel() else 0.0)
                if off > 0:
                    old = int(math.frexp(float(scales[block, h]))[1]) - 1
                    if e > old:
                        values[block, h, :off] = to_e4m3(values[block, h, :off] * 2.0 ** (old - e))
                    e = max(e, old)
                scales[block, h] = 2.0 ** e
                got = to_e4m3((part * 2.0 ** -e).clamp(-1e30, 1e30))
                bad = part.isnan().any(1) | other[r:stop, h].isnan().any(1)
                got[bad] = math.nan if is_key else 0.0
                values[block, h, off:off + stop - r] = got
            r = stop
    return values, scales


def attention(q, k, v, ks, vs, table, cu, kv_len, scale, window, gate=None):
    """(out, spread, size): the definition in float64; per output the sum of p |v| / sum of p (times the gate), which
    bounds what relative errors of the probabilities do to it; the largest sum |q k| * scale of a visible pair and the
    largest max |q| * sum |k| * scale. ``k``, ``v``: codes' values; rows outside every request are NaN."""
    tq, hq, hd = q.shape
    hkv = k.shape[1]
    group = hq // hkv
    out = torch.full((tq, hq, hd), math.nan, dtype=torch.float64, device=q.device)
    spread = torch.zeros_like(out)
    size = reach = 0.0
    blocks = k.shape[0]
    for i in range(len(kv_len)):
        a, b, lk = cu[i], cu[i + 1], kv_len[i]
        lq = b - a
        if lq == 0:
            continue
        out[a:b] = 0.0
        lk = min(lk, table.shape[1] * BLOCK)
        pos = torch.arange(lk, device=q.device)
        ids = table[i].long()[pos // BLOCK] if lk else pos
        there = (ids >= 0) & (ids < blocks)
        pos, ids = pos[there], ids[there]
        at = torch.arange(lq, device=q.device)[:, None] + (lk - lq)
        see = torch.ones(lq, pos.numel(), dtype=torch.bool, device=q.device)
        if window[0] >= 0:
            see &= pos[None, :] >= at - window[0]
        if window[1] >= 0:
            see &= pos[None, :] <= at + window[1]
        some = see.any(1)
        if not bool(some.any()):
            continue
        used = see.any(0)  # keys no row sees may hold anything
        pos, ids, see = pos[used], ids[used], see[:, used]
        for h in range(hq):
            g = h // group
            kk = k[ids, g, pos % BLOCK] * ks[ids, g].double()[:, None]
            vv = v[ids, g, pos % BLOCK] * vs[ids, g].double()[:, None]
            size = max(size, float((q[a:b, h].double().abs() @ kk.abs().T * scale)[see].max()))
            top = q[a:b, h].double().abs().amax(1, keepdim=True)
            reach = max(reach, float((top * kk.abs().sum(1) * scale)[see].max()))
            x = torch.where(see, q[a:b, h].double() @ kk.T * scale, -math.inf)
            x = torch.where(some[:, None], x, 0.0)
            p = torch.softmax(x, -1)
            # a hidden key's value harms nobody: 0 times anything is 0 there
            o = torch.where(some[:, None], torch.where(see, p, 0.0) @ vv, 0.0)
            out[a:b, h] = o
            spread[a:b, h] = torch.where(some[:, None], torch.where(see, p, 0.0) @ vv.abs(), 0.0)
    out, spread = out.reshape(tq, hq * hd), spread.reshape(tq, hq * hd)
    if gate is not None:
        s = torch.sigmoid(gate.double())
        live = spread > 0
        out, spread = torch.where(live, out * s, out), spread * s
    return out, spread, (size, reach)
