"""The operators of the state cache, as cases to time and compare: block tables and slot maps from request lengths,
the write of keys and values into blocks of e4m3 codes, and attention over those blocks.

``own`` chooses who computes: false, the plain form below in elementary torch operations; true, the framework's entry
points. A case is a dict of plain values; its request lengths follow from it (``_lengths``), its values from the seed.

The cache (one layer): ``k``, ``v`` e4m3 codes (blocks, Hkv, 64, hd), ``k_scale``, ``v_scale`` float32 (blocks, Hkv),
powers of two; ``table`` int32 (requests, width) holds each request's block ids, -1 where it has none.
"""

import math

import torch

own = False

BLOCK = 64  # tokens of a block
E_MIN, E_MAX = -100, 120  # the scales' exponents
DEV = "cuda"


# ------------------------------------------------------------------------------------------------ cases


def listed():
    return [
        # One question token against one cached state of a page or two of text: the smallest call, all latency
        # (heads of the 0.8B configuration).
        dict(name="ask_one", op="attention", n=1, lo=4096, hi=4096, qlo=1, qhi=1, hq=16, hkv=8, hd=128, left=-1,
             gate=True),
        # A serving step: one new token in each of 48 states of very different lengths (4B configuration).
        dict(name="step_48", op="attention", n=48, lo=700, hi=30011, qlo=1, qhi=1, hq=32, hkv=8, hd=128, left=-1,
             gate=True),
        # One token against one 131,072-token state (31B configuration, a global layer).
        dict(name="ask_131k", op="attention", n=1, lo=131072, hi=131072, qlo=1, qhi=1, hq=32, hkv=16, hd=128, left=-1,
             gate=False),
        # A few tokens each (an option's tokens, scored together) in a sliding layer of the 12B configuration.
        dict(name="options_sliding", op="attention", n=24, lo=300, hi=16001, qlo=2, qhi=9, hq=16, hkv=8, hd=256,
             left=1023, gate=False),
        # Questions of 20 to 200 tokens about 8 cached states (4B configuration): the framework's ordinary request.
        dict(name="questions", op="attention", n=8, lo=1500, hi=24001, qlo=20, qhi=201, hq=32, hkv=8, hd=128, left=-1,
             gate=True),
        # The next 4,096 tokens of one long state (12B configuration, a global layer): the largest work.
        dict(name="chunk_4096", op="attention", n=1, lo=32768, hi=32768, qlo=4096, qhi=4096, hq=16, hkv=8, hd=256,
             left=-1, gate=False),
        # A global layer with heads of 512 and few key/value heads: short questions about 4 states.
        dict(name="global_512", op="attention", n=4, lo=2000, hi=12007, qlo=3, qhi=61, hq=16, hkv=2, hd=512, left=-1,
             gate=False),
        # One new token written per state (4B configuration): every write lands in a half-filled block.
        dict(name="store_step", op="store", n=64, lo=100, hi=9000, qlo=1, qhi=1, hkv=8, hd=128),
        # A pack of whole states written after their prefill (0.8B configuration, 32,000 tokens or so).
        dict(name="store_pack", op="store", n=24, lo=0, hi=0, qlo=300, qhi=4001, hkv=8, hd=128),
        # Blocks and slots of one question on one state.
        dict(name="tables_one", op="tables", n=1, lo=4000, hi=4000, qlo=70, qhi=70),
        # Blocks and slots of a pack of 512 requests of all lengths.
        dict(name="tables_512", op="tables", n=512, lo=1, hi=16001, qlo=1, qhi=500),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "attention", "store", "store", "tables"])
    if op == "tables":
        n = _log(rng, 1, 700)
        hi = _log(rng, 2, 30000)
        qhi = _log(rng, 1, max(1, 120000 // n))
        return dict(op=op, n=n, lo=rng.randint(0, hi), hi=hi, qlo=rng.randint(0, qhi), qhi=qhi)
    hkv, hd = rng.choice([(8, 128), (8, 128), (16, 128), (8, 256), (2, 512), (2, 64), (1, 128), (5, 64)])
    if op == "store":
        n = _log(rng, 1, 200)
        hi = rng.choice([0, _log(rng, 1, 3000)])
        qhi = _log(rng, 1, max(1, 24000 // n))
        return dict(op=op, n=n, lo=rng.randint(0, hi), hi=hi, qlo=rng.randint(0, qhi), qhi=qhi, hkv=hkv, hd=hd)
    group = rng.choice([1, 2, 4, 8, 3])
    kind = rng.choice(["token", "few", "question", "chunk"])
    n = _log(rng, 1, 96) if kind != "chunk" else rng.randint(1, 3)
    qhi = {"token": 1, "few": rng.randint(2, 12), "question": _log(rng, 12, 300), "chunk": _log(rng, 300, 3000)}[kind]
    hi = qhi + _log(rng, 1, max(2, (400000 // n if kind in ("token", "few") else 60000 // n) * 128 // hd))
    lo = rng.randint(max(qhi, hi // 8), hi)
    left = rng.choice([-1, -1, 1023, rng.randint(0, 2000)])
    case = dict(op=op, n=n, lo=lo, hi=hi, qlo=max(1, qhi // rng.choice([1, 2, 9])), qhi=qhi, hq=hkv * group, hkv=hkv,
                hd=hd, left=left, gate=rng.random() < 0.5)
    while work(case)["flops"] > 1.5e12:  # no dearer than the largest case above
        case["hi"] = max(case["qhi"], case["hi"] * 2 // 3)
        case["lo"] = min(case["lo"], case["hi"])
        if case["hi"] == case["qhi"]:
            case["n"] = max(1, case["n"] // 2)
    return case


def _lengths(case):
    """Each request's tokens before (``store``, ``tables``) or in all (``attention``), and its new rows: spread
    log-uniformly over the case's bounds by two irrational rotations, so that they are the case's own."""
    def spread(lo, hi, n, step, start):
        out = []
        for i in range(n):
            u = (start + i * step) % 1.0 if n > 1 else 1.0
            out.append(min(hi, max(lo, int(round((lo + 1) * ((hi + 1) / (lo + 1)) ** u)) - 1)))
        return out

    lens = spread(case["lo"], case["hi"], case["n"], 0.6180339887498949, 0.37)
    new = spread(case["qlo"], case["qhi"], case["n"], 0.4142135623730951, 0.81)
    return lens, new


def _visible(case):
    """Per request (new rows, first key any row sees, keys, visible pairs)."""
    out = []
    for lk, lq in zip(*_lengths(case)):
        left = case["left"]
        first = 0 if left < 0 else max(0, lk - lq - left)
        pairs = 0
        if left < 0:
            pairs = lq * (lk - lq) + lq * (lq + 1) // 2
        else:
            pairs = sum(min(lk - lq + i + 1, left + 1) for i in range(lq))
        out.append((lq, first, lk, pairs))
    return out


def work(case):
    lens, new = _lengths(case)
    if case["op"] == "tables":
        added = sum(-(-(a + b) // BLOCK) - -(-a // BLOCK) for a, b in zip(lens, new))
        # lengths, bounds, the blocks taken and given back; slots and positions of the new rows
        return dict(bytes=4 * (4 * case["n"] + 1) + 16 * sum(new) + 16 * added, flops=0)
    if case["op"] == "store":
        per = case["hkv"] * case["hd"]
        # the rows, their codes, the scales and the slots; a half-filled block's old codes only where its scale grows
        blocks = sum(-(-(a + b) // BLOCK) - a // BLOCK for a, b in zip(lens, new) if b)
        return dict(bytes=2 * per * 3 * sum(new) + 8 * blocks * case["hkv"] + 8 * sum(new), flops=0)
    vis = _visible(case)
    rows = sum(v[0] for v in vis)
    keys = sum(v[2] - v[1] for v in vis)
    wide = 2 * rows * case["hq"] * case["hd"]
    return dict(bytes=2 * keys * case["hkv"] * case["hd"] + wide * (3 if case["gate"] else 2),
                flops=4 * case["hd"] * case["hq"] * sum(v[3] for v in vis))


# ------------------------------------------------------------------------------------------------ inputs


def _bounds(new):
    cu = [0]
    for x in new:
        cu.append(cu[-1] + x)
    return cu


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _exponent(amax):
    """The least e with amax * 2^-e <= 448, inside the exponents' bounds (float32 in, int32 out)."""
    m, x = torch.frexp(amax)  # amax = m 2^x, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(m > 0.875, x - 8, x - 9)
    return torch.where(amax > 0, e, E_MIN).clamp(E_MIN, E_MAX).to(torch.int32)


def _power(e):
    """2^e in float32, exactly (a device's exp2 need not be exact at whole numbers)."""
    return torch.tensor([2.0 ** i for i in range(-126, 128)], device=DEV)[(e + 126).long()]


def _fill(g, blocks, hkv, hd, spread):
    """A pool's codes and scales: normal values whose size differs from head to head and from block to block."""
    codes = torch.empty(blocks, hkv, BLOCK, hd, dtype=torch.float8_e4m3fn, device=DEV)
    scale = torch.empty(blocks, hkv, dtype=torch.float32, device=DEV)
    step = max(1, (1 << 26) // (hkv * BLOCK * hd))
    for a in range(0, blocks, step):
        b = min(blocks, a + step)
        x = torch.randn(b - a, hkv, BLOCK, hd, generator=g, device=DEV)
        x *= torch.exp2(spread * torch.randn(b - a, hkv, 1, 1, generator=g, device=DEV))
        s = _power(_exponent(x.abs().amax((2, 3))))
        codes[a:b] = (x / s[:, :, None, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
        scale[a:b] = s
    return codes, scale


def _table(g, have, spare):
    """(table, free, count): every request's blocks dealt from a shuffled pool, the rest on the free stack."""
    total = sum(have) + spare
    order = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    width = max(1, max(have) + spare)
    table = torch.full((len(have), width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, h in enumerate(have):
        table[i, :h] = order[at:at + h]
        at += h
    free = torch.full((total,), -1, dtype=torch.int32, device=DEV)
    free[:total - at] = order[at:]
    return table, free, _int32([total - at, 0]), total


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    lens, new = _lengths(case)
    n, cu = case["n"], _bounds(new)
    s = dict(case=case, lens=lens, new=new, bounds=cu, cu=_int32(cu), rows=cu[-1])
    if case["op"] == "tables":
        have = [-(-x // BLOCK) for x in lens]
        added = sum(-(-(a + b) // BLOCK) for a, b in zip(lens, new)) - sum(have)
        s["table"], s["free"], s["count"], _ = _table(g, have, added + 7)
        s["lens_dev"], s["added"] = _int32(lens), added
        return s
    hkv, hd = case["hkv"], case["hd"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    if case["op"] == "store":
        have = [-(-(a + b) // BLOCK) for a, b in zip(lens, new)]
        s["table"], _, _, blocks = _table(g, have, 3)
        s["k"], s["ks"] = _fill(g, blocks, hkv, hd, 0.5)
        s["v"], s["vs"] = _fill(g, blocks, hkv, hd, 1.0)
        size = torch.exp2(0.7 * normal(s["rows"], hkv, 1))
        s["k_new"] = normal(s["rows"], hkv, hd).bfloat16()
        s["v_new"] = (normal(s["rows"], hkv, hd) * size).bfloat16()
        req = torch.repeat_interleave(torch.arange(n, device=DEV), torch.tensor(new, device=DEV))
        pos = torch.arange(s["rows"], device=DEV) - s["cu"].long()[req] + torch.tensor(lens, device=DEV)[req]
        s["slots"] = s["table"].long()[req, pos // BLOCK] * BLOCK + pos % BLOCK
    else:
        have = [-(-x // BLOCK) for x in lens]
        s["table"], _, _, blocks = _table(g, have, 3)
        s["k"], s["ks"] = _fill(g, blocks, hkv, hd, 0.25)
        s["v"], s["vs"] = _fill(g, blocks, hkv, hd, 1.0)
        s["q"] = (1.5 * normal(s["rows"], case["hq"], hd)).bfloat16()
        s["gate"] = normal(s["rows"], case["hq"] * hd).bfloat16() if case["gate"] else None
        s["kv_len"] = _int32(lens)
        s["scale"] = hd ** -0.5
    if own:
        from karpo_decision_b200 import ops
        s["blocks"] = ops.KVBlocks(s["k"], s["v"], s["ks"], s["vs"])
    return s


# ------------------------------------------------------------------------------------------------ one pass


def run(s):
    case = s["case"]
    if own:
        from karpo_decision_b200 import ops
        if case["op"] == "tables":
            # a request's blocks taken for its new rows and given back, as a question about a state does
            kv_len, seqpos, slots = ops.kv_assign(s["lens_dev"], s["cu"], s["table"], s["free"], s["count"], s["rows"])
            ops.kv_release(s["table"], kv_len, s["lens_dev"], s["free"], s["count"])
            return kv_len, seqpos, slots, s["table"], s["free"], s["count"]
        if case["op"] == "store":
            ops.kv_store_e4m3(s["k_new"], s["v_new"], s["cu"], s["slots"], s["blocks"])
            return s["k"], s["v"], s["ks"], s["vs"]
        return ops.attention_cache(s["q"], s["blocks"], s["table"], s["cu"], s["kv_len"], max(s["new"]), s["scale"],
                                   (case["left"], 0), gate=s["gate"])
    if case["op"] == "tables":
        return _plain_tables(s)
    if case["op"] == "store":
        _plain_store(s["k_new"], s["slots"], s["k"], s["ks"], s, s["v_new"], True)
        _plain_store(s["v_new"], s["slots"], s["v"], s["vs"], s, s["k_new"], False)
        return s["k"], s["v"], s["ks"], s["vs"]
    return _plain_attention(s)


def _plain_tables(s):
    lens, cu, table, free, count = s["lens_dev"].long(), s["cu"].long(), s["table"], s["free"], s["count"]
    new = cu[1:] - cu[:-1]
    have = (lens + BLOCK - 1) // BLOCK
    add = (lens + new + BLOCK - 1) // BLOCK - have
    base = torch.cumsum(add, 0) - add
    j = torch.arange(s["added"], device=DEV)
    req = torch.repeat_interleave(add, output_size=s["added"])
    at = count[0].long() - 1 - j
    table[req, have[req] + j - base[req]] = free[at]
    t = torch.arange(s["rows"], device=DEV)
    row = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    seqpos = lens[row] + t - cu[row]
    slots = table.long()[row, seqpos // BLOCK] * BLOCK + seqpos % BLOCK
    kv_len = (lens + new).to(torch.int32)
    # and back: the blocks return to their places on the stack
    free[at] = table[req, have[req] + j - base[req]]
    table[req, have[req] + j - base[req]] = -1
    return kv_len, seqpos, slots, table, free, count


def _plain_store(x, slots, codes, scale, s, other, is_key):
    """Rows x into the pool: per (block, head) the power of two that holds its old part and its new rows."""
    rows = x.shape[0]
    blocks, hkv, _, hd = codes.shape
    x = x.float()
    bad = x.isnan().any(2) | other.float().isnan().any(2)
    fin = torch.where(x.isfinite(), x, 0.0)
    blk, off = slots // BLOCK, slots % BLOCK
    amax = torch.zeros(blocks, hkv, device=DEV)
    amax.index_reduce_(0, blk, fin.abs().amax(2), "amax")
    first = torch.full((blocks,), BLOCK, dtype=torch.int64, device=DEV)  # the first new row of each block
    first.index_reduce_(0, blk, off, "amin")
    touched = first < BLOCK
    before = torch.frexp(scale)[1].to(torch.int32) - 1
    e = _exponent(amax)
    e = torch.where((first > 0)[:, None], torch.maximum(e, before), e)
    e = torch.where(touched[:, None], e, before)
    # the old part of the blocks whose scale grew
    ids = blk[torch.cat([torch.ones(1, dtype=torch.bool, device=DEV), blk[1:] != blk[:-1]])] if rows else blk
    part = codes[ids].float() * _power((before - e)[ids].clamp_min(-126))[:, :, None, None]
    keep = (torch.arange(BLOCK, device=DEV)[None, :] < first[ids][:, None])[:, None, :, None]
    codes[ids] = torch.where(keep, part, codes[ids].float()).to(torch.float8_e4m3fn)
    y = (x * _power(-e)[blk][:, :, None]).clamp(-448, 448)
    y = torch.where(bad[:, :, None], float("nan") if is_key else 0.0, y)
    codes[blk, :, off] = y.to(torch.float8_e4m3fn)
    scale.copy_(_power(e))


def _plain_attention(s):
    case = s["case"]
    hq, hkv, hd, left = case["hq"], case["hkv"], case["hd"], case["left"]
    group = hq // hkv
    out = torch.empty(s["rows"], hq * hd, dtype=torch.bfloat16, device=DEV)
    for i, (lk, lq) in enumerate(zip(s["lens"], s["new"])):
        if lq == 0:
            continue
        a = s["bounds"][i]
        first = 0 if left < 0 else max(0, lk - lq - left) // BLOCK
        ids = s["table"][i, first:-(-lk // BLOCK)].long()
        span = lk - first * BLOCK
        step = max(1, (1 << 28) // (span * hq))
        k = (s["k"][ids].float() * s["ks"][ids][:, :, None, None]).permute(1, 0, 2, 3).reshape(hkv, -1, hd)[:, :span]
        v = (s["v"][ids].float() * s["vs"][ids][:, :, None, None]).permute(1, 0, 2, 3).reshape(hkv, -1, hd)[:, :span]
        key = torch.arange(span, device=DEV) + first * BLOCK
        for b in range(0, lq, step):
            e = min(lq, b + step)
            q = s["q"][a + b:a + e].float().reshape(e - b, hkv, group * hd).transpose(0, 1)
            q = q.reshape(hkv, (e - b) * group, hd)
            x = (q @ k.transpose(1, 2)) * s["scale"]
            pos = torch.arange(b, e, device=DEV).repeat_interleave(group) + lk - lq
            see = key[None, :] <= pos[:, None]
            if left >= 0:
                see &= key[None, :] >= pos[:, None] - left
            x = x.masked_fill(~see, -math.inf)
            p = torch.exp(x - x.amax(-1, keepdim=True))
            o = (p @ v) / p.sum(-1, keepdim=True)
            o = o.reshape(hkv, e - b, group * hd).transpose(0, 1).reshape(e - b, hq * hd)
            if s["gate"] is not None:
                o = o / (1 + torch.exp(-s["gate"][a + b:a + e].float()))
            out[a + b:a + e] = o.to(torch.bfloat16)
    return out


# ------------------------------------------------------------------------------------------------ in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    lens, new = s["lens"], s["new"]
    if case["op"] == "tables":
        table, free = s["table"].cpu().tolist(), s["free"].cpu().tolist()
        top = int(s["count"][0])
        seqpos, slots = [], []
        for i, (a, b) in enumerate(zip(lens, new)):
            blocks = table[i][:-(-a // BLOCK)]
            while len(blocks) * BLOCK < a + b:
                top -= 1
                blocks.append(free[top])
            for p in range(a, a + b):
                seqpos.append(p)
                slots.append(blocks[p // BLOCK] * BLOCK + p % BLOCK)
        return (_int32([a + b for a, b in zip(lens, new)]), torch.tensor(seqpos, dtype=torch.int64, device=DEV),
                torch.tensor(slots, dtype=torch.int64, device=DEV), s["table"], s["free"], s["count"])
    if case["op"] == "store":
        return _exact_store(s)
    pairs = sum(v[3] for v in _visible(case))
    if pairs * case["hq"] * case["hd"] * 4 > 3e13:
        return None
    hd, group = case["hd"], case["hq"] // case["hkv"]
    out = torch.zeros(s["rows"], case["hq"], hd, dtype=torch.float64, device=DEV)
    for i, (lk, lq) in enumerate(zip(lens, new)):
        lo = 0 if case["left"] < 0 else max(0, lk - lq - case["left"])
        where = torch.arange(lo, lk, device=DEV)
        ids, off = s["table"][i].long()[where // BLOCK], where % BLOCK
        for h in range(case["hkv"]):
            k = s["k"][ids, h, off].double() * s["ks"][ids, h].double()[:, None]
            v = s["v"][ids, h, off].double() * s["vs"][ids, h].double()[:, None]
            rows = max(1, (1 << 27) // (lk - lo))
            for g in range(group):
                for b in range(0, lq, rows):
                    e = min(lq, b + rows)
                    r = s["bounds"][i]
                    x = s["q"][r + b:r + e, h * group + g].double() @ k.T * s["scale"]
                    dist = torch.arange(b, e, device=DEV)[:, None] + (lk - lq) - where[None, :]
                    hide = dist < 0
                    if case["left"] >= 0:
                        hide |= dist > case["left"]
                    x[hide] = -math.inf
                    out[r + b:r + e, h * group + g] = torch.softmax(x, -1) @ v
    out = out.reshape(s["rows"], -1)
    return out if s["gate"] is None else out * torch.sigmoid(s["gate"].double())


def _exact_store(s):
    """The pool after the write, block by block: the codes' values and the scales."""
    got = []
    # 2^i at index i, negative ones counted from the end
    two = torch.tensor([2.0 ** (i if i < 300 else i - 600) for i in range(600)], dtype=torch.float64, device=DEV)
    runs = {}  # block -> its new rows in order
    slots = s["slots"].cpu().tolist()
    for t, slot in enumerate(slots):
        runs.setdefault(slot // BLOCK, []).append(t)
    ids = torch.tensor(list(runs), dtype=torch.int64, device=DEV)
    for x, codes, scale in ((s["k_new"], s["k"], s["ks"]), (s["v_new"], s["v"], s["vs"])):
        values = codes.double()
        scales = scale.double().clone()
        first = torch.tensor([slots[r[0]] % BLOCK for r in runs.values()], device=DEV)
        full = torch.zeros(len(runs), codes.shape[1], BLOCK, codes.shape[3], dtype=torch.float64, device=DEV)
        at = torch.tensor([i for i, r in enumerate(runs.values()) for _ in r], device=DEV)
        row = torch.tensor([t for r in runs.values() for t in r], device=DEV)
        full[at, :, s["slots"][row] % BLOCK] = x[row].double()
        m, x2 = torch.frexp(full.abs().amax((2, 3)) / 448)
        need = (x2 - (m == 0.5).to(x2.dtype)).clamp(E_MIN, E_MAX)
        need[m == 0] = E_MIN
        old = torch.frexp(scales[ids])[1] - 1
        e = torch.where((first > 0)[:, None], torch.maximum(need, old), need)
        # e4m3 to nearest even: 3 bits after the leading one, steps of 2^-9 below 2^-6
        mine = torch.zeros_like(full, dtype=torch.bool)
        mine[at, :, s["slots"][row] % BLOCK] = True
        y = full * two[-e.long()][:, :, None, None]
        keep = values[ids] * two[(old - e).long()][:, :, None, None]
        for z in (y, keep):
            step = two[(torch.frexp(z.abs().clamp_min(2.0 ** -6))[1] - 4).long()]
            z.copy_((torch.round(z / step) * step).clamp(-448, 448))
        before = (torch.arange(BLOCK, device=DEV)[None, :] < first[:, None])[:, None, :, None].expand_as(full)
        values[ids] = torch.where(mine, y, torch.where(before, keep, values[ids]))
        scales[ids] = two[e.long()]
        got.append((values, scales))
    return got[0][0], got[1][0], got[0][1], got[1][1]
