"""The state cache's operators on the GPU against their float64 restatement (tests/cache_reference.py): block tables and
slot maps, the e4m3 block write, attention over the blocks, and the three of them together."""

import ctypes
import math

import numpy as np
import pytest
import torch

import cache_reference as ref
from karpo_decision_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BLOCK = ops.KV_BLOCK


def ints(x, device=DEV):
    return torch.tensor(x, dtype=torch.int32, device=device)


def bounds(new):
    return [0, *np.cumsum(new).tolist()]


def dealt(lens, new, width, spare, seed=0):
    """(table rows, free list, count): the requests' blocks dealt from a shuffled pool, the rest on the stack."""
    g = np.random.default_rng(seed)
    have = [-(-x // BLOCK) for x in lens]
    total = sum(have) + spare
    order = g.permutation(total).tolist()
    rows, at = [], 0
    for h in have:
        rows.append(order[at:at + h] + [-1] * (width - h))
        at += h
    free = order[at:]
    return rows, free + [-7] * (total - len(free)), len(free)


# ------------------------------------------------------------------------------------------------ block tables


CASES = {
    "one token": ([4000], [1]),
    "one new block": ([64], [1]),
    "empty request": ([0], [0]),
    "from nothing": ([0], [129]),
    "mixed": ([0, 63, 64, 65, 1, 500, 0, 127], [1, 1, 1, 0, 63, 64, 0, 130]),
    "one long": ([10], [70001]),
    "many": ([(7 * i) % 301 for i in range(1500)], [(13 * i) % 40 for i in range(1500)]),
}


@pytest.mark.parametrize("name", CASES)
@pytest.mark.parametrize("pad", [0, 5])
def test_assign_and_its_inverse(name, pad):
    lens, new = CASES[name]
    width = max(-(-(a + b) // BLOCK) for a, b in zip(lens, new)) + 1
    need = sum(-(-(a + b) // BLOCK) - -(-a // BLOCK) for a, b in zip(lens, new))
    rows, free, count = dealt(lens, new, width, need + 3)
    table, stack, height = ints(rows), ints(free), ints([count, 9])
    got = ops.kv_assign(ints(lens), ints(bounds(new)), table, stack, height, sum(new) + pad)
    kv_len, seqpos, slots, want_table, left, outcome = ref.assign(lens, new, rows, free, count, width)
    assert [x.tolist() for x in got] == [kv_len, seqpos + [0] * pad, slots + [-1] * pad]
    assert table.tolist() == want_table and height.tolist() == [left, outcome] and outcome == 0
    ops.kv_release(table, got[0], ints(lens), stack, height)
    assert table.tolist() == rows and height.tolist() == [count, 0] and stack.tolist() == free


def test_tables_of_the_most_requests():
    """Counts around the 48 KB of shared memory that a launch has without asking (with its static arrays: 4,085 to 4,095
    requests for the assignment, 6,127 to 6,143 for the release), up to the most; smaller ones first, so that no larger
    call has asked before."""
    for n in (4084, 4085, 4095, 4096, 6126, 6127, 6128, 6143, 6144):
        lens, new = [0] * n, [0] * n
        new[n // 2], new[n - 1] = 70, 3
        table, stack, height = ints([[-1] * 2] * n), ints(list(range(32))), ints([32, 0])
        got = ops.kv_assign(ints(lens), ints(bounds(new)), table, stack, height, 73)
        want = ref.assign(lens, new, [[-1] * 2] * n, list(range(32)), 32, 2)
        assert [x.tolist() for x in got] == list(want[:3]) and table.tolist() == want[3] and height.tolist() == [29, 0]
        ops.kv_release(table, got[0], ints(lens), stack, height)
        assert (table == -1).all() and stack.tolist() == list(range(32)) and height.tolist() == [32, 0]
    n = 16384
    g = np.random.default_rng(7)
    lens, new = g.integers(0, 130, n).tolist(), g.integers(0, 70, n).tolist()
    need = sum(-(-(a + b) // BLOCK) - -(-a // BLOCK) for a, b in zip(lens, new))
    rows, free, count = dealt(lens, new, 4, need + 3)
    table, stack, height = ints(rows), ints(free), ints([count, 0])
    got = ops.kv_assign(ints(lens), ints(bounds(new)), table, stack, height, sum(new))
    want = ref.assign(lens, new, rows, free, count, 4)
    assert [x.tolist() for x in got] == list(want[:3]) and table.tolist() == want[3] and height.tolist() == [3, 0]
    ops.kv_release(table, got[0], ints(lens), stack, height)
    assert table.tolist() == rows and stack.tolist() == free and height.tolist() == [count, 0]


def test_tables_of_the_most_requests_on_a_large_pool():
    """The largest shared memory a call can ask for, in a cluster of eight: 16,384 requests, ids in two parts."""
    n, capacity = 16384, 2 ** 18 + 70000
    lens, new = [5] * n, [1] * n
    for i in range(0, n, 7):
        new[i] = 64
    need = len(range(0, n, 7))
    ids = np.random.default_rng(8).permutation(capacity).tolist()
    rows, free = [[x, -1] for x in ids[:n]], ids[n:] + [-1] * n
    count = capacity - n
    table, stack, height = ints(rows), ints(free), ints([count, 0])
    got = ops.kv_assign(ints(lens), ints(bounds(new)), table, stack, height, sum(new))
    want = ref.assign(lens, new, rows, free, count, 2)
    assert [x.tolist() for x in got] == list(want[:3]) and table.tolist() == want[3]
    assert height.tolist() == [count - need, 0]
    ops.kv_release(table, got[0], ints(lens), stack, height)
    assert table.tolist() == rows and stack.tolist() == free and height.tolist() == [count, 0]


def test_assign_takes_nothing_when_blocks_are_missing():
    lens, new = [70, 0, 10], [200, 65, 4]
    rows, free, count = dealt(lens, new, 8, 4)  # 3 + 2 + 0 new blocks, 4 free
    table, stack, height = ints(rows), ints(free), ints([count, 0])
    kv_len, seqpos, slots = ops.kv_assign(ints(lens), ints(bounds(new)), table, stack, height, sum(new))
    assert height.tolist() == [4, 1] and table.tolist() == rows and stack.tolist() == free
    assert kv_len.tolist() == lens and set(slots.tolist()) == {-1}
    assert seqpos.tolist() == ref.assign(lens, new, rows, free, count, 8)[1]


@pytest.mark.parametrize("lens,cu,width,outcome", [
    ([600], [0, 10], 9, ops.KV_TABLE_FULL),     # 10 blocks in a table of 9
    ([-1, 5], [0, 4, 8], 9, ops.KV_MALFORMED),  # a negative length
    ([5, 5], [0, 4, 2], 9, ops.KV_MALFORMED),   # bounds that fall
    ([5], [0, 12], 9, ops.KV_MALFORMED),        # bounds past the rows
])
def test_assign_refuses_on_the_device(lens, cu, width, outcome):
    table, stack, height = ints([[0] * width] * len(lens)), ints(list(range(20))), ints([20, 0])
    before = table.clone()
    kv_len, _, slots = ops.kv_assign(ints(lens), ints(cu), table, stack, height, 10)
    assert height.tolist() == [20, outcome] and torch.equal(table, before)
    assert kv_len.tolist() == lens and set(slots.tolist()) == {-1}


@pytest.mark.parametrize("rows,outcome", [(7, 0), (8, ops.KV_MALFORMED)])
def test_assign_to_the_last_length_an_int32_holds(rows, outcome):
    """A table wide enough for 2^31 tokens: up to 2^31 - 1 of them, the next one is refused."""
    n = 2 ** 31 - 8
    table = torch.full((1, 2 ** 25), 3, dtype=torch.int32, device=DEV)
    stack, height = ints([0, 1, 2, -1, -1]), ints([3, 0])
    kv_len, seqpos, slots = ops.kv_assign(ints([n]), ints([0, rows]), table, stack, height, rows)
    assert height.tolist() == [3, outcome]
    if outcome == 0:
        assert kv_len.item() == n + rows and seqpos.tolist() == list(range(n, n + rows))
        assert slots.tolist() == [3 * BLOCK + 56 + i for i in range(rows)]
    else:
        assert kv_len.item() == n and (slots == -1).all()


@pytest.mark.parametrize("bad", [-1, 40, -2 ** 31, 2 ** 31 - 1])
@pytest.mark.parametrize("where", ["half-filled block", "top of the stack", "deep in the stack"])
def test_assign_refuses_ids_outside_the_pool(bad, where):
    """An id the rows would use: all or nothing, as for missing blocks. The same call with the id put right succeeds."""
    # 40 blocks: requests hold 5 (4 full ones, 6 tokens in the last) and 0 tokens; 1,500 more for the deep entry
    deep = 1500 if where == "deep in the stack" else 0
    capacity = 40 + deep
    lens, new = [262, 0], [100, 64 * (deep or 2)]
    width = 2 + new[1] // BLOCK + 5
    rows, free, count = dealt(lens, new, width, capacity - 5)
    need = 1 + new[1] // BLOCK
    table, stack, height = ints(rows), ints(free), ints([count, 0])
    wrong = bad if bad != 40 else capacity
    entry = {"half-filled block": (table, (0, 4)), "top of the stack": (stack, (count - 1,)),
             "deep in the stack": (stack, (count - need,))}[where]
    right = entry[0][entry[1]].item()
    entry[0][entry[1]] = wrong
    before = table.clone(), stack.clone()
    args = ints(lens), ints(bounds(new)), table, stack, height, sum(new)
    kv_len, _, slots = ops.kv_assign(*args)
    assert height.tolist() == [count, ops.KV_MALFORMED] and kv_len.tolist() == lens and (slots == -1).all()
    assert torch.equal(table, before[0]) and torch.equal(stack, before[1])
    entry[0][entry[1]] = right
    got = ops.kv_assign(*args)
    want = ref.assign(lens, new, rows, free, count, width)
    assert [x.tolist() for x in got] == list(want[:3]) and table.tolist() == want[3] and height.tolist() == [want[4], 0]


def test_assign_looks_at_the_ids_it_uses_only():
    """Holes in earlier blocks, a half-filled block without new rows and stack entries below the new blocks' harm nobody."""
    lens, new = [262, 70, 64], [100, 0, 1]
    rows, free, count = dealt(lens, new, 9, 6)
    rows[0][1], rows[0][3], rows[1][1], rows[2][0] = -1, 10 ** 9, -5, 99
    free[:count - 2] = [-3] * (count - 2)
    table, stack, height = ints(rows), ints(free), ints([count, 0])
    got = ops.kv_assign(ints(lens), ints(bounds(new)), table, stack, height, sum(new))
    want = ref.assign(lens, new, rows, free, count, 9)
    assert [x.tolist() for x in got] == list(want[:3]) and table.tolist() == want[3] and height.tolist() == [want[4], 0]


@pytest.mark.parametrize("capacity", [40, 700000])  # ids in one part of the kernel's bitmap, and in three
@pytest.mark.parametrize("twice", ["half-filled blocks", "half-filled block and stack", "stack"])
def test_assign_refuses_a_block_twice(capacity, twice):
    """Two requests' rows for one block: neither gets a slot. The same call with another id succeeds."""
    lens, new, width = [70, 200, 0], [5, 60, 130], 6
    high = capacity - 1
    rows = [[1, high] + [-1] * 4, [2, 3, 4, 5, -1, -1], [-1] * 6]
    free = list(range(6, 30)) + [-1] * (capacity - 24)  # 1 + 3 new blocks: 29, 28, 27, 26
    count = 24
    if twice == "half-filled blocks":
        at, rows[1][3] = (0, (1, 3)), high
    elif twice == "half-filled block and stack":
        at, free[21] = (1, (21,)), high
    else:
        at, free[20], free[22] = (1, (22,)), high - 1, high - 1
    table, stack, height = ints(rows), ints(free), ints([count, 0])
    args = ints(lens), ints(bounds(new)), table, stack, height, sum(new)
    kv_len, _, slots = ops.kv_assign(*args)
    assert height.tolist() == [count, ops.KV_MALFORMED] and kv_len.tolist() == lens and (slots == -1).all()
    assert table.tolist() == rows and stack.tolist() == free
    (table, stack)[at[0]][at[1]] = 33
    rows, free = table.tolist(), stack.tolist()
    got = ops.kv_assign(*args)
    want = ref.assign(lens, new, rows, free, count, width)
    assert [x.tolist() for x in got] == list(want[:3]) and table.tolist() == want[3] and height.tolist() == [want[4], 0]


def test_requests_share_blocks_that_get_no_rows():
    """Two questions on a state that ends with its block, and on a half-filled one that only one of them goes on in;
    release to the state's length gives back their own blocks only."""
    lens, new = [128, 128, 100, 100], [70, 3, 0, 9]
    rows = [[1, 2, -1, -1], [1, 2, -1, -1], [3, 4, -1, -1], [3, 4, -1, -1]]
    free = [9, 8, 7, 6, 5, -1, -1, -1, -1, -1]
    table, stack, height = ints(rows), ints(free), ints([5, 0])
    got = ops.kv_assign(ints(lens), ints(bounds(new)), table, stack, height, sum(new))
    want = ref.assign(lens, new, rows, free, 5, 4)
    assert [x.tolist() for x in got] == list(want[:3]) and table.tolist() == want[3] and height.tolist() == [2, 0]
    ops.kv_release(table, got[0], ints(lens), stack, height)
    assert table.tolist() == rows and stack.tolist() == free and height.tolist() == [5, 0]


@pytest.mark.parametrize("capacity", [40, 700000])
def test_release_of_a_block_twice_gives_nothing_back(capacity):
    high = capacity - 1
    rows, free = [[3, high, 5], [4, high, 6]], [0, 1, 2] + [-1] * (capacity - 3)
    table, stack, height = ints(rows), ints(free), ints([3, 0])
    ops.kv_release(table, ints([150, 150]), ints([0, 0]), stack, height)
    assert height.tolist() == [3, ops.KV_MALFORMED] and table.tolist() == rows and stack.tolist() == free
    table[1, 1] = 7
    ops.kv_release(table, ints([150, 150]), ints([0, 100]), stack, height)
    assert height.tolist()[0] == 7 and table.tolist() == [[-1] * 3, [4, 7, -1]]
    assert stack.tolist()[:7] == [0, 1, 2, 6, 5, high, 3]


def test_assign_in_place_and_release_to_a_length():
    """kv_len may be lens; a release keeps each request's first tokens and the blocks that hold them."""
    lens, new, keep = ints([100, 0, 64]), [300, 70, 1], [130, 0, 500]
    rows, free, count = dealt([100, 0, 64], new, 9, 12)
    table, stack, height = ints(rows), ints(free), ints([count, 0])
    seqpos = torch.empty(371, dtype=torch.int64, device=DEV)
    slots = torch.empty_like(seqpos)
    ops.kv_assign(lens, ints(bounds(new)), table, stack, height, 371, out=(lens, seqpos, slots))
    assert lens.tolist() == [400, 70, 65]
    full = table.tolist()
    taken = count - height[0].item()
    ops.kv_release(table, lens, ints(keep), stack, height)
    kept = [-(-130 // BLOCK), 0, 2]  # a `keep` past the length gives nothing back
    assert table.tolist() == [row[:k] + [-1] * (9 - k) for row, k in zip(full, kept)]
    dropped = [row[j] for row, k, h in zip(full, kept, (7, 2, 2)) for j in range(k, h)]
    assert height.tolist() == [count - taken + len(dropped), 0]
    assert stack.tolist()[count - taken:count - taken + len(dropped)] == dropped[::-1]


@pytest.mark.parametrize("entry", [-1, 20])
def test_release_of_a_block_outside_the_pool_gives_nothing_back(entry):
    table, stack, height = ints([[3, entry, 5]]), ints(list(range(20))), ints([8, 0])
    before, held = table.clone(), stack.clone()
    ops.kv_release(table, ints([150]), ints([0]), stack, height)
    assert height.tolist() == [8, ops.KV_MALFORMED] and torch.equal(table, before) and torch.equal(stack, held)


def test_release_onto_a_full_stack_gives_nothing_back():
    table, stack, height = ints([[3, 4, 5]]), ints(list(range(6))), ints([4, 0])
    ops.kv_release(table, ints([150]), ints([0]), stack, height)
    assert height.tolist() == [4, ops.KV_MALFORMED] and table.tolist() == [[3, 4, 5]]


@pytest.mark.parametrize("free,outcome", [(2, 1), (9, ops.KV_TABLE_FULL)])
def test_a_failed_assignment_shows_after_its_release(free, outcome):
    """A step of assignment and release that takes nothing and gives nothing back; the next assignment clears the word."""
    lens, width = ints([70, 10]), 3 if outcome > 0 else 2
    rows = [[20, 21] + [-1] * (width - 2), [22] + [-1] * (width - 1)]
    table, stack, height = ints(rows), ints(list(range(free)) + [-1] * (30 - free)), ints([free, 0])
    kv_len, _, slots = ops.kv_assign(lens, ints([0, 100, 230]), table, stack, height, 230)
    ops.kv_release(table, kv_len, lens, stack, height)
    assert (slots == -1).all() and height.tolist() == [free, outcome] and table.tolist() == rows
    ops.kv_release(table[:0], kv_len[:0], lens[:0], stack, height)
    assert height.tolist() == [free, outcome]
    kv_len, _, _ = ops.kv_assign(lens, ints([0, 50, 60]), table, stack, height, 60)
    assert height.tolist() == [free, 0]


# ------------------------------------------------------------------------------------------------ the write


def pool(blocks, heads, hd, seed, junk=True):
    """A pool of random codes and scales 2^-6 .. 2^2; with ``junk`` some codes are NaN, as unwritten memory holds."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    k, v = (torch.randint(0, 256, (blocks, heads, BLOCK, hd), generator=g, device=DEV, dtype=torch.uint8)
            for _ in range(2))
    if not junk:
        k, v = (torch.where(x & 0x7f == 0x7f, x & 0x80, x) for x in (k, v))
    ks, vs = (torch.randint(-6, 3, (blocks, heads), generator=g, device=DEV) for _ in range(2))
    ones = torch.ones(blocks, heads, device=DEV)
    return ops.KVBlocks(k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), torch.ldexp(ones, ks),
                        torch.ldexp(ones, vs))


def placed(lens, new, seed=0, spare=3):
    """(blocks in the pool, table, slots) of requests holding ``lens`` tokens that get ``new`` rows."""
    width = max(1, max(-(-(a + b) // BLOCK) for a, b in zip(lens, new)))
    grown = [a + b for a, b in zip(lens, new)]
    rows, free, _ = dealt(grown, new, width, spare, seed)
    slots = [rows[i][p // BLOCK] * BLOCK + p % BLOCK for i, (a, b) in enumerate(zip(lens, new)) for p in range(a, a + b)]
    return len(free), rows, slots


def check_store(k, v, cu, slots, cache, rows):
    before = [x.clone() for x in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    ops.kv_store_e4m3(k, v, ints(cu), torch.tensor(slots, dtype=torch.int64, device=DEV), cache)
    kd, vd = k.double().cpu(), v.double().cpu()
    for got, scale, was, was_scale, x, other, is_key in (
            (cache.k, cache.k_scale, before[0], before[2], kd, vd, True),
            (cache.v, cache.v_scale, before[1], before[3], vd, kd, False)):
        values, scales = ref.store(x, other, cu, slots, was.double().cpu(), was_scale.double().cpu(), is_key)
        assert torch.equal(scale.double().cpu(), scales)
        assert torch.equal(got.double().cpu().nan_to_num(1e9), values.nan_to_num(1e9))


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("heads", [1, 5])
@pytest.mark.parametrize("lens,new", [([0], [1]), ([63], [2]), ([64], [64]), ([10, 0, 70, 5], [200, 0, 1, 64]),
                                      ([1] * 70, [3] * 70)])
def test_store_matches_its_definition(hd, heads, lens, new):
    blocks, _, slots = placed(lens, new, seed=hd)
    g = torch.Generator(device=DEV)
    g.manual_seed(hd + heads)
    rows = sum(new)
    k = (torch.randn(rows, heads, hd, generator=g, device=DEV) *
         torch.exp2(3 * torch.randn(rows, heads, 1, generator=g, device=DEV))).bfloat16()
    v = torch.randn(rows, heads, hd, generator=g, device=DEV).bfloat16()
    check_store(k, v, bounds(new), slots, pool(blocks, heads, hd, 3), rows)


@pytest.mark.parametrize("fill", [0.0, 448.0, 449.0, 447.0, 2.0 ** -110, 3.3e38, 2.0 ** -133, math.inf, math.nan])
def test_store_of_special_values(fill):
    """Zeros, the largest magnitude that still fits a scale, one past it, the ends of bf16's range, infinities, NaN."""
    lens, new = [0, 30], [5, 7]
    blocks, _, slots = placed(lens, new)
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    k = torch.randn(12, 2, 64, generator=g, device=DEV).bfloat16()
    v = torch.randn(12, 2, 64, generator=g, device=DEV).bfloat16()
    k[2, 0, 5] = fill
    v[7, 1, 9] = -fill
    if fill in (0.0, 2.0 ** -133):
        k[:5] = fill
    cache = pool(blocks, 2, 64, 4, junk=False)
    check_store(k, v, bounds(new), slots, cache, 12)


def test_store_grows_a_scale_and_keeps_what_it_can():
    """A half-filled block's old codes move to the larger scale: exact where they stay normal, rounded where not."""
    cache = ops.kv_blocks(2, 1, 64, DEV)
    slots = list(range(64))
    k = torch.randn(64, 1, 64, generator=torch.Generator().manual_seed(0)).to(DEV).bfloat16()
    k[32:] *= 2.0 ** 14
    check_store(k[:32], k[:32], [0, 32], slots[:32], cache, 32)
    check_store(k[32:], k[32:], [0, 32], slots[32:], cache, 32)


def test_store_reads_strided_rows_and_leaves_the_rest():
    """k and v as columns of one projection; rows behind the last request and requests without slots are not written."""
    lens, new = [10, 20, 0], [70, 3, 9]
    blocks, _, slots = placed(lens, new)
    slots[70:73] = [-1] * 3  # the second request got no blocks
    g = torch.Generator(device=DEV)
    g.manual_seed(5)
    qkv = torch.randn(100, 8 * 64, generator=g, device=DEV).bfloat16()
    k, v = (qkv[:, a:a + 128].unflatten(1, (2, 64)) for a in (128, 256))
    check_store(k, v, bounds(new), slots + [0] * 18, pool(blocks, 2, 64, 6), 100)


# ------------------------------------------------------------------------------------------------ attention


def make(lens, new, hq, hkv, hd, seed=0, spread=1.0, pad=0):
    """Requests' cached tokens in a pool whose unwritten places hold anything, NaN codes too."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    blocks, rows, _ = placed(lens, [0] * len(lens), seed)
    cache = pool(blocks, hkv, hd, seed + 1)
    for codes, scale, apart in ((cache.k, cache.k_scale, 1.0), (cache.v, cache.v_scale, spread)):
        for i, n in enumerate(lens):
            for j in range(-(-n // BLOCK)):
                live = min(BLOCK, n - j * BLOCK)
                x = torch.randn(hkv, live, hd, generator=g, device=DEV) * 60.0
                codes[rows[i][j], :, :live] = x.clamp(-448, 448).to(torch.float8_e4m3fn)
                scale[rows[i][j]] = 2.0 ** -6 * torch.exp2(torch.round(
                    apart * torch.randn(hkv, generator=g, device=DEV)))
    q = (1.5 * torch.randn(sum(new) + pad, hq, hd, generator=g, device=DEV)).bfloat16()
    gate = torch.randn(sum(new) + pad, hq * hd, generator=g, device=DEV).bfloat16()
    return cache, ints(rows), q, gate


def tolerance(want, spread, size, hd, keys):
    """What the definition's value may move by (derived, not fitted); spread = sum p |v| / sum p, size = (the largest
    sum |q k| * scale, the largest max |q| * sum |k| * scale):
    - the output's rounding to bf16: 2^-8 |o|;
    - the probabilities' rounding to f16: 2^-11 relative each, so 2^-11 spread; those below f16's normal numbers, 2^-29
      of the row's largest scaled probability, lose at most 2^-40 of it each: keys * 2^-40 of 448 block units, which the
      largest one's own term in spread covers unless its codes are all under 2^-6;
    - a score's error d moves every probability by at most 2 d relative: d <= (hd / 8) 2^-23 size[0] for the products'
      float32 sums (hd / 16 products of 16 terms, each added with an error of one unit), 2^-22 size[0] for its scaling,
      the subtraction of the maximum and the exponential, and 2^-17 size[1] for the queries: as two e4m3 values of a row
      scaled to more than 224, an element is off by half of e4m3's least step, 2^-10 (one f16 value of a row scaled to
      at least 1 is off by 2^-25 at most);
    - the float32 sums over keys: keys / 16 additions of 2^-23 relative at most, in numerator and denominator."""
    d = (hd / 8 * 2.0 ** -23 + 2.0 ** -22) * size[0] + 2.0 ** -17 * size[1]
    return 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -14 + keys / 8 * 2.0 ** -23 + 2 * d) * spread + 1e-30


def check_attention(lens, new, hq, hkv, hd, window=(-1, 0), gated=False, seed=0, table=None, **kw):
    cache, rows, q, gate = make(lens, new, hq, hkv, hd, seed, **kw)
    table = rows if table is None else table(rows)
    scale = hd ** -0.5
    cu = bounds(new)
    got = ops.attention_cache(q, cache, table, ints(cu), ints(lens), max(new), scale, window,
                              gate=gate if gated else None)
    ops.check_status(DEV)
    want, spread, size = ref.attention(q, cache.k.double(), cache.v.double(), cache.k_scale, cache.v_scale, table, cu, lens,
                                 scale, window, gate if gated else None)
    n = cu[-1]
    err = (got[:n].double() - want[:n]).abs()
    tol = tolerance(want[:n], spread[:n], size, hd, max(lens))
    assert torch.isfinite(got[:n]).all()
    worst = (err / tol).max().item() if n else 0.0
    assert worst <= 1.0, f"error {worst:.3f} of the tolerance"
    return got


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 4), (6, 2), (16, 2), (5, 1)])
@pytest.mark.parametrize("gated", [False, True])
def test_attention_of_single_tokens(hd, hq, hkv, gated):
    check_attention([1, 64, 65, 130, 1000, 3, 2049], [1] * 7, hq, hkv, hd, gated=gated)


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("hq,hkv", [(2, 2), (8, 2), (3, 1)])
@pytest.mark.parametrize("window", [(-1, 0), (-1, -1), (20, 0), (0, 0), (63, 5), (200, -1)])
def test_attention_of_questions(hd, hq, hkv, window):
    """Ragged questions about states of all lengths, causal, windowed and whole; a request without new rows."""
    check_attention([40, 129, 700, 64, 1500], [40, 17, 33, 0, 70], hq, hkv, hd, window, gated=hq == 8)


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
def test_attention_of_a_whole_prompt(hd):
    check_attention([391], [391], 4, 2, hd)
    check_attention([1111, 300], [1111, 300], 2, 2, hd, window=(127, 0), gated=True)


def test_attention_of_one_long_state():
    check_attention([70001], [1], 8, 2, 128)
    check_attention([33000], [65], 8, 2, 128, gated=True)


def test_attention_of_many_requests():
    g = np.random.default_rng(3)
    lens = g.integers(1, 400, 300).tolist()
    check_attention(lens, [1] * 300, 8, 4, 64)
    check_attention(lens, [min(n, 3) for n in lens], 8, 4, 128, window=(100, 0))


@pytest.mark.parametrize("hd,hq,hkv", [(64, 8, 8), (128, 8, 4), (256, 8, 4), (512, 8, 2)])
def test_attention_of_long_states_with_few_rows(hd, hq, hkv):
    """Some hundred tiles a block: every slot of its ring is used many times over, by warps that run ahead of one another.
    Two runs are equal bit by bit."""
    lens = [40000, 1, 52345, 30017, 64, 47111, 38000, 20000]
    first = check_attention(lens, [1] * 8, hq, hkv, hd)
    assert torch.equal(first, check_attention(lens, [1] * 8, hq, hkv, hd))


@pytest.mark.parametrize("rows", [1, 20])
def test_attention_of_more_requests_than_threads(rows):
    """900 requests, empty ones and ones without new rows among them, single tokens and rows for the 128-row tiles."""
    g = np.random.default_rng(4)
    lens = g.integers(0, 150, 900).tolist()
    new = [min(n, int(r)) for n, r in zip(lens, g.integers(0, rows + 1, 900))]
    check_attention(lens, new, 4, 2, 64)
    check_attention(lens, new, 4, 4, 128, window=(30, 0), gated=True)


def test_rows_that_see_nothing_are_zero():
    """No cached token, fewer cached tokens than rows (the first rows lie before key 0), a state whose blocks are all
    absent; the gate does not matter there."""
    got = check_attention([0, 3, 70], [5, 9, 2], 4, 2, 128, gated=True,
                          table=lambda t: torch.cat([t[:2], torch.full_like(t[2:], -1)]))
    assert not got[:5].any() and not got[5:11].any() and not got[14:].any() and got[11:14].any()


def test_absent_blocks_are_not_seen():
    """Table entries outside the pool, negative and too large, in the middle of a state."""
    def holes(t):
        t = t.clone()
        t[0, 1], t[0, 4], t[1, 0] = -1, 10 ** 9, -5
        return t

    check_attention([500, 130], [3, 40], 4, 2, 128, table=holes)


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("hq,hkv", [(4, 1), (2, 2), (6, 3)])
@pytest.mark.parametrize("window", [(-1, -1), (20, 0), (0, 0), (0, 3), (63, 5), (200, -1), (5000, 5000)])
def test_few_rows_and_their_windows(hd, hq, hkv, window):
    """The kernel for up to 16 rows a head, under the windows that questions are tested with: whole, to both sides."""
    check_attention([40, 129, 700, 64, 1500, 2], [2, 1, 4, 0, 3, 4], hq, hkv, hd, window, gated=hq == 4)


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("window", [(-1, 0), (7, 0)])
def test_few_rows_that_see_nothing_are_zero(hd, window):
    """As for questions: no cached token, fewer cached tokens than rows, a state whose blocks are all absent."""
    got = check_attention([0, 3, 70, 65], [2, 4, 1, 1], 4, 1, hd, window, gated=True,
                          table=lambda t: torch.cat([t[:2], torch.full_like(t[2:3], -1), t[3:]]))
    assert not got[:3].any() and not got[6].any() and got[3:6].any(1).all() and got[7].any()
    assert not check_attention([0, 0], [1, 3], 4, 1, hd, window).any()


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
def test_few_rows_do_not_see_absent_blocks(hd):
    """Holes in the middle of a state, at its end (where the rows are), and in one that several CTAs share."""
    def holes(t):
        t = t.clone()
        t[0, 1], t[0, 4], t[1, 0], t[2, 0] = -1, 10 ** 9, -5, t.max() + 100
        t[3, ::3], t[3, 1::7] = -1, 2 ** 31 - 1
        return t

    check_attention([500, 130, 65, 30000], [3, 1, 1, 2], 4, 1, hd, table=holes)


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("more", [0, 9000])
def test_a_nan_token_reaches_only_the_few_rows_that_see_it(hd, more):
    """A NaN in a value, seen by the first of two rows through its window; head 0 has none. Also in a longer state, whose
    other tiles are finite."""
    n = 200 + more
    cache = ops.kv_blocks(n // BLOCK + 3, 2, hd, DEV)
    g = torch.Generator(device=DEV)
    g.manual_seed(2)
    k, v = (torch.randn(n, 2, hd, generator=g, device=DEV).bfloat16() for _ in range(2))
    q = torch.randn(2, 2, hd, generator=g, device=DEV).bfloat16()
    v[120, 1, 7] = math.nan
    table = torch.randperm(n // BLOCK + 1, generator=g, device=DEV).int()[None, :]
    t = torch.arange(n, device=DEV)
    ops.kv_store_e4m3(k, v, ints([0, n]), table[0].long()[t // 64] * 64 + t % 64, cache)
    # the rows' positions are n - 2 and n - 1; the window's first key is 120 for the first of them, 121 for the second
    out = ops.attention_cache(q, cache, table, ints([0, 2]), ints([n]), 2, 0.1, (n - 122, 0)).float()
    assert torch.isfinite(out[:, :hd]).all() and out[0, hd:].isnan().all() and torch.isfinite(out[1, hd:]).all()


def test_few_rows_strides_and_rows_behind_the_last_request():
    """q, gate and out as columns of wider buffers, a table with a row stride, rows of padding left as they were."""
    lens, new = [300, 77], [1, 4]
    cache, table, q, gate = make(lens, new, 4, 1, 64, pad=7)
    wide = torch.zeros(2, 40, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    qs = torch.zeros(12, 768, dtype=torch.bfloat16, device=DEV)
    gs, outs = torch.zeros_like(qs), torch.full_like(qs, 5.0)
    qs[:, 256:512], gs[:, 512:] = q.reshape(12, 256), gate
    args = (ints(bounds(new)), ints(lens), 4, 0.125, (-1, 0))
    want = ops.attention_cache(q, cache, table, *args, gate=gate)
    got = ops.attention_cache(qs[:, 256:512].unflatten(1, (4, 64)), cache, wide[:, :table.shape[1]], *args,
                              gate=gs[:, 512:], out=outs[:, 256:512])
    assert torch.equal(got[:5], want[:5])
    assert (outs[5:] == 5).all() and (outs[:, :256] == 5).all() and (outs[:, 512:] == 5).all()


@pytest.mark.parametrize("rows", [1, 30])
def test_a_pool_past_four_gigabytes(rows):
    """Blocks whose codes lie past 2^32 bytes: written and read as in a small pool, bit by bit."""
    blocks, heads, hd, n = 70000, 8, 128, 300
    shape = (blocks, heads, BLOCK, hd)
    k, v = (torch.empty(shape, dtype=torch.float8_e4m3fn, device=DEV) for _ in range(2))
    big = ops.KVBlocks(k, v, *(torch.ones(blocks, heads, device=DEV) for _ in range(2)))
    small = ops.kv_blocks(5, heads, hd, DEV)
    ids = torch.tensor([69999, 3, 66000, 69998, 32768], device=DEV)
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    rows_k, rows_v = (torch.randn(n, heads, hd, generator=g, device=DEV).bfloat16() for _ in range(2))
    q = torch.randn(rows, 2 * heads, hd, generator=g, device=DEV).bfloat16()
    at = torch.arange(n, device=DEV)
    outs = []
    for cache, order in ((big, ids), (small, torch.arange(5, device=DEV))):
        ops.kv_store_e4m3(rows_k, rows_v, ints([0, n]), order[at // BLOCK] * BLOCK + at % BLOCK, cache)
        outs.append(ops.attention_cache(q, cache, order.int()[None, :], ints([0, rows]), ints([n]), rows, 0.1, (-1, 0)))
    held = torch.arange(5 * BLOCK, device=DEV).reshape(5, 1, BLOCK, 1) < n
    for x, y in ((big.k, small.k), (big.v, small.v)):
        assert torch.equal(torch.where(held, x[ids].view(torch.uint8), 0), torch.where(held, y.view(torch.uint8), 0))
    assert torch.equal(big.k_scale[ids], small.k_scale) and torch.equal(big.v_scale[ids], small.v_scale)
    assert torch.equal(*outs) and torch.isfinite(outs[0]).all()


@pytest.mark.parametrize("new", [[1, 1], [30, 41]])
def test_scales_far_apart(new):
    """Blocks whose value scales differ by up to 2^40 or so: the largest values need not have the largest probability."""
    check_attention([640, 333], new, 8, 2, 128, spread=8.0)


@pytest.mark.parametrize("rows", [1, 40])
def test_zero_queries_and_zero_blocks(rows):
    """Every score 0 (a zero query, blocks of zeros with the smallest scale): the mean of the values, not NaN."""
    cache = ops.kv_blocks(4, 1, 128, DEV)
    cache.k_scale.fill_(2.0 ** -100)
    cache.v.fill_(2.0)
    q = torch.zeros(rows, 2, 128, dtype=torch.bfloat16, device=DEV)
    out = ops.attention_cache(q, cache, ints([[2, 0, 1]]), ints([0, rows]), ints([150]), rows, 0.1, (-1, 0))
    assert (out == 2).all()


@pytest.mark.parametrize("new", [[3, 1], [60, 41]])
def test_scales_at_the_ends_of_their_range(new):
    """Value scales 2^-100 beside 2^100: small probabilities of large values, and the reverse."""
    cache, table, q, _ = make([640, 333], new, 4, 2, 64)
    for i, n in enumerate((640, 333)):
        cache.v_scale[table[i, :-(-n // BLOCK)].long()] = 2.0 ** -100
    cache.v_scale[table[0, 3].long()] = 2.0 ** 100
    cache.v_scale[table[1, 0].long()] = 2.0 ** 20
    cu, scale = bounds(new), 0.125
    got = ops.attention_cache(q, cache, table, ints(cu), ints([640, 333]), max(new), scale, (-1, 0))
    want, spread, size = ref.attention(q, cache.k.double(), cache.v.double(), cache.k_scale, cache.v_scale, table, cu,
                                       [640, 333], scale, (-1, 0))
    assert ((got.double() - want).abs() <= tolerance(want, spread, size, 64, 640)).all()


def test_a_nan_token_reaches_only_rows_that_see_it():
    cache = ops.kv_blocks(8, 2, 128, DEV)
    g = torch.Generator(device=DEV)
    g.manual_seed(2)
    k, v, q = (torch.randn(200, 2, 128, generator=g, device=DEV).bfloat16() for _ in range(3))
    v[120, 1, 7] = math.nan
    table = ints([[5, 0, 7, 2]])
    t = torch.arange(200, device=DEV)
    ops.kv_store_e4m3(k, v, ints([0, 200]), table[0].long()[t // 64] * 64 + t % 64, cache)
    out = ops.attention_cache(q, cache, table, ints([0, 200]), ints([200]), 200, 0.1, (40, 0)).float()
    assert torch.isfinite(out[:, :128]).all()
    nan = out[:, 128:].isnan()
    assert nan[120:161].all() and not nan[:120].any() and not nan[161:].any()


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("rows", [1, 3, 40])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_a_query_that_is_not_finite_makes_its_row_nan(hd, rows, value):
    """Also where every score is -inf (the keys are positive at that place); rows that see nothing stay 0, others are not
    touched. The cases span the tiles of 8 and 16 rows and of 128, states of one tile and of several shares."""
    for lens in ([rows, 5, 30], [70, 64, 9001], [1, 1, 300]):
        cache, table, q, _ = make(lens, [rows] * 3, 4, 1, hd)
        for codes in (cache.k[..., 3], cache.k[..., hd - 1]):
            codes.view(torch.uint8)[:] = 0x40  # 2
        q[::2, 1, 3], q[::2, 3, hd - 1] = value, value
        out = ops.attention_cache(q, cache, table, ints(bounds([rows] * 3)), ints(lens), rows, 0.1, (-1, 0))
        ops.check_status(DEV)
        out = out.float().unflatten(1, (4, hd))
        clean = q.clone()
        clean[::2, 1::2] = 0
        want = ops.attention_cache(clean, cache, table, ints(bounds([rows] * 3)), ints(lens), rows, 0.1, (-1, 0))
        want = want.float().unflatten(1, (4, hd))
        for i, n in enumerate(lens):
            for r in range(rows):
                at = i * rows + r
                seen = r + n - rows >= 0
                assert torch.equal(out[at, ::2], want[at, ::2])
                if at % 2 == 0 and seen:
                    assert out[at, 1::2].isnan().all(), (lens, i, r)
                else:
                    assert torch.equal(out[at, 1::2], want[at, 1::2]) and (seen or not out[at].any())


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("new", [[1, 2, 1], [40, 9, 60]])
@pytest.mark.parametrize("spread", [0.0, 8.0])
def test_scores_near_their_limit(hd, new, spread):
    """Every row's query along one key, so that its score is about 2^21.5 in log2 units and the others' far lower: the row
    is that key's value. Off by the output's rounding, 2^-8, and the one probability's to f16, 2^-11 (its exponent may be
    off by a half here, in numerator and sum alike up to a float32 rounding)."""
    lens, hkv, group = [300, 64, 9000], 2, 2
    cache, table, q, _ = make(lens, new, hkv * group, hkv, hd, spread=spread)
    cache.k_scale.fill_(2.0 ** -6)
    scale, cu = hd ** -0.5, bounds(new)
    g = np.random.default_rng(hd)
    want = torch.zeros(sum(new), hkv * group, hd, dtype=torch.float64, device=DEV)
    for i, (n, rows) in enumerate(zip(lens, new)):
        pos = torch.arange(n, device=DEV)
        ids, at = table[i].long()[pos // BLOCK], pos % BLOCK
        for h in range(hkv * group):
            k = cache.k[ids, h // group, at].double() * 2.0 ** -6
            v = cache.v[ids, h // group, at].double() * cache.v_scale[ids, h // group].double()[:, None]
            for r in range(rows):
                key = int(g.integers(0, n - rows + r + 1))
                x = k[key] * 2.0 ** 21.5 / (scale * math.log2(math.e) * (k[key] @ k[key]))
                q[cu[i] + r, h] = x.bfloat16()
                scores = k[:n - rows + r + 1] @ q[cu[i] + r, h].double() * scale * math.log2(math.e)
                assert scores.argmax() == key and scores.abs().max() < 2 ** 22
                assert scores.numel() == 1 or scores.topk(2).values.diff().item() < -2.0 ** 17
                want[cu[i] + r, h] = v[key]
    out = ops.attention_cache(q, cache, table, ints(cu), ints(lens), max(new), scale, (-1, 0)).double()
    ops.check_status(DEV)
    want = want.flatten(1)
    assert ((out - want).abs() <= (2.0 ** -8 + 2.0 ** -11 + 2.0 ** -14) * want.abs()).all()


def test_strides_and_rows_behind_the_last_request():
    """q, gate and out as columns of wider buffers, a table with a row stride, rows of padding left as they were."""
    lens, new = [300, 77], [5, 20]
    cache, table, q, gate = make(lens, new, 4, 2, 64, pad=7)
    wide = torch.zeros(2, 40, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    qs = torch.zeros(32, 768, dtype=torch.bfloat16, device=DEV)
    gs, outs = torch.zeros_like(qs), torch.full_like(qs, 5.0)
    qs[:, 256:512], gs[:, 512:] = q.reshape(32, 256), gate
    args = (ints(bounds(new)), ints(lens), 20, 0.125, (-1, 0))
    want = ops.attention_cache(q, cache, table, *args, gate=gate)
    got = ops.attention_cache(qs[:, 256:512].unflatten(1, (4, 64)), cache, wide[:, :table.shape[1]], *args,
                              gate=gs[:, 512:], out=outs[:, 256:512])
    assert torch.equal(got[:25], want[:25])
    assert (outs[25:] == 5).all() and (outs[:, :256] == 5).all() and (outs[:, 512:] == 5).all()


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 9, 60]])
def test_repeated_calls_are_equal_and_streams_do_not_mix(new):
    """Bit-equal results from launches in flight on two streams at once, again and again."""
    cache, table, q, gate = make([900, 64, 5000], new, 8, 2, 128)
    args = (cache, table, ints(bounds(new)), ints([900, 64, 5000]), max(new), 0.1, (-1, 0))
    want = ops.attention_cache(q, *args, gate=gate)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(ops.attention_cache(q, *args, gate=gate))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("max_q", [1, 2, 10])
@pytest.mark.parametrize("n", [3, 900])
def test_bounds_that_fall_compute_nothing(hd, max_q, n):
    """Bounds that name rows twice (0, 10, 0, 10): nothing is computed, nothing is written behind the workspace, and the
    same buffers serve a good call next. 900 requests are more than a block's threads, the fall is in the last part."""
    hq, rows = 8, 10
    cache, table, q, _ = make([70] * n, [0] * n, hq, 1, hd, pad=rows)
    cu = ints([0, 10] + [10] * (n - 3) + [0, 10])
    lens, out = ints([70] * n), torch.full((rows, hq * hd), 5.0, dtype=torch.bfloat16, device=DEV)
    size = ctypes.c_int64()
    _lib.call("kd_attention_cache_workspace", n, max_q, rows, hq, 1, hd, ctypes.addressof(size))
    scratch = torch.full((size.value + (1 << 24),), 0xab, dtype=torch.uint8, device=DEV)

    def run(bounds_):
        _lib.call("kd_attention_cache", q.data_ptr(), hq * hd, cache.k.data_ptr(), cache.v.data_ptr(),
                  cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), cache.blocks, table.data_ptr(), table.stride(0),
                  table.shape[1], bounds_.data_ptr(), lens.data_ptr(), n, max_q, rows, out.data_ptr(), hq * hd, None, 0,
                  hq, 1, hd, hd ** -0.5, -1, 0, scratch.data_ptr(), size.value, ops.status_word(DEV).data_ptr(),
                  torch.cuda.current_stream().cuda_stream)

    run(cu)
    ops.check_status(DEV)
    assert (out == 5).all() and (scratch[size.value:] == 0xab).all()
    good = ints([0] * (n - 1) + [5, 10])
    run(good)
    assert torch.equal(out, ops.attention_cache(q, cache, table, good, lens, max_q, hd ** -0.5, (-1, 0)))
    assert (scratch[size.value:] == 0xab).all()


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
@pytest.mark.parametrize("new", [[1, 1, 2], [40, 9, 60]])
def test_a_launch_that_gives_up_ends_by_itself(hd, new):
    """With an error already in the status word every wait that is not over at once gives up. The launches end, write
    nothing behind their buffers, and the next ones are right."""
    lens = [900, 64, 30000]
    cache, table, q, gate = make(lens, new, 8, 2, hd, pad=3)
    args = (cache, table, ints(bounds(new)), ints(lens), max(new), 0.1, (-1, 0))
    want = ops.attention_cache(q, *args, gate=gate)
    word = ops.status_word(DEV)
    for _ in range(3):
        out = torch.full_like(want, 5.0)
        word.fill_(_lib.KD_DEVICE_TIMEOUT)
        ops.attention_cache(q, *args, gate=gate, out=out)
        with pytest.raises(_lib.KernelError, match="gave up"):
            ops.check_status(DEV)
        assert (out[sum(new):] == 5).all()
        got = ops.attention_cache(q, *args, gate=gate)
        ops.check_status(DEV)
        assert torch.equal(got[:sum(new)], want[:sum(new)])


# ------------------------------------------------------------------------------------------------ together


@pytest.mark.parametrize("hd", [64, 128])
def test_states_grown_in_pieces(hd):
    """Assign, store and attend over the same tokens in different pieces, as a captured graph would run each step: the
    outputs stay within rounding of the definition on the cache as it stood, and giving blocks back leaves the stack
    full."""
    hq, hkv, total = 4, 2, [150, 70, 333]
    g = torch.Generator(device=DEV)
    g.manual_seed(8)
    q = [torch.randn(n, hq, hd, generator=g, device=DEV).bfloat16() for n in total]
    k = [torch.randn(n, hkv, hd, generator=g, device=DEV).bfloat16() for n in total]
    v = [torch.randn(n, hkv, hd, generator=g, device=DEV).bfloat16() for n in total]
    cache = pool(16, hkv, hd, 9)
    table, stack, height = ints([[-1] * 6] * 3), ints(list(range(16))), ints([16, 0])
    lens, done = ints([0, 0, 0]), [0, 0, 0]
    for step in ([100, 1, 200], [1, 0, 1], [1, 69, 100], [48, 0, 32]):
        new = list(step)
        pick = [slice(d, d + s) for d, s in zip(done, new)]
        rows = [torch.cat([x[i][pick[i]] for i in range(3)]) for x in (q, k, v)]
        cu = ints(bounds(new))
        kv_len, seqpos, slots = ops.kv_assign(lens, cu, table, stack, height, sum(new))
        ops.kv_store_e4m3(rows[1], rows[2], cu, slots, cache)
        out = ops.attention_cache(rows[0], cache, table, cu, kv_len, max(new), hd ** -0.5, (-1, 0))
        done = [d + s for d, s in zip(done, new)]
        assert kv_len.tolist() == done
        want, spread, size = ref.attention(rows[0], cache.k.double(), cache.v.double(), cache.k_scale, cache.v_scale, table,
                                     bounds(new), done, hd ** -0.5, (-1, 0))
        tol = tolerance(want, spread, size, hd, 333)
        assert ((out.double() - want).abs() <= tol).all()
        lens = kv_len
    # what the cache holds is the rows within e4m3's rounding: half a step, 2^-4 relative, and under a block's smallest
    # normal code (2^-6) half of its 2^-9 steps, each a second time where a scale grew
    for i, n in enumerate(total):
        pos = torch.arange(n, device=DEV)
        ids = table[i].long()[pos // BLOCK]
        for codes, scale, x in ((cache.k, cache.k_scale, k[i]), (cache.v, cache.v_scale, v[i])):
            held = codes[ids, :, pos % BLOCK].double() * scale[ids].double()[:, :, None]
            step = 2.0 ** -9 * scale[ids].double()[:, :, None]
            assert ((held - x.double()).abs() <= 2 * (2.0 ** -4 * x.double().abs() + step)).all()
    ops.kv_release(table, lens, ints([0, 0, 0]), stack, height)
    assert height.tolist() == [16, 0] and sorted(stack.tolist()) == list(range(16)) and (table == -1).all()


def test_a_captured_step_follows_the_lengths_on_the_device():
    """One graph of assign, store and attend, replayed as the requests grow by a token each."""
    hq, hkv, hd, n = 4, 2, 64, 3
    cache = ops.kv_blocks(24, hkv, hd, DEV)
    table, stack, height = ints([[-1] * 6] * n), ints(list(range(24))), ints([24, 0])
    lens, cu = ints([0] * n), ints([0, 1, 2, 3])
    q = torch.zeros(n, hq, hd, dtype=torch.bfloat16, device=DEV)
    k, v = (torch.zeros(n, hkv, hd, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    seqpos, slots = (torch.zeros(n, dtype=torch.int64, device=DEV) for _ in range(2))

    def step():
        ops.kv_assign(lens, cu, table, stack, height, n, out=(lens, seqpos, slots))
        ops.kv_store_e4m3(k, v, cu, slots, cache)
        return ops.attention_cache(q, cache, table, cu, lens, 1, hd ** -0.5, (-1, 0))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    ops.kv_release(table, lens, ints([0] * n), stack, height)
    lens.zero_()
    g = torch.Generator(device=DEV)
    g.manual_seed(4)
    for i in range(130):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g, device=DEV))
        graph.replay()
        if i in (0, 1, 62, 63, 64, 65, 129):
            assert lens.tolist() == [i + 1] * n and seqpos.tolist() == [i] * n and height[1].item() == 0
            want, spread, size = ref.attention(q, cache.k.double(), cache.v.double(), cache.k_scale, cache.v_scale, table,
                                         [0, 1, 2, 3], [i + 1] * n, hd ** -0.5, (-1, 0))
            tol = tolerance(want, spread, size, hd, 130)
            assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("hd", [64, 128, 256, 512])
def test_captured_questions_follow_the_bounds_on_the_device(hd):
    """One graph of assign, store, attend and release for up to 64 rows of 3 requests, padding behind them: replayed with
    other questions each time, and with one too many for the pool, whose failure shows at the end."""
    hq, hkv, rows, width = 4, 2, 64, 12
    lens0 = [100, 640, 64]
    cache, table, _, _ = make(lens0, [0, 0, 0], hq, hkv, hd)
    have = [-(-n // BLOCK) for n in lens0]
    blocks = cache.blocks
    rows_ = [table[i, :h].tolist() for i, h in enumerate(have)]
    taken = {x for r in rows_ for x in r}
    free = [i for i in range(blocks) if i not in taken]  # three blocks
    table = ints([r + [-1] * (width - len(r)) for r in rows_])
    stack, height = ints(free + [-1] * (blocks - len(free))), ints([len(free), 0])
    lens, cu, kv_len = ints(lens0), ints([0, 20, 20, 45]), ints(lens0)
    q = torch.zeros(rows, hq, hd, dtype=torch.bfloat16, device=DEV)
    k, v = (torch.zeros(rows, hkv, hd, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    seqpos, slots = (torch.zeros(rows, dtype=torch.int64, device=DEV) for _ in range(2))
    out = torch.zeros(rows, hq * hd, dtype=torch.bfloat16, device=DEV)

    def step():
        ops.kv_assign(lens, cu, table, stack, height, rows, out=(kv_len, seqpos, slots))
        ops.kv_store_e4m3(k, v, cu, slots, cache)
        ops.attention_cache(q, cache, table, cu, kv_len, 40, hd ** -0.5, (-1, 0), out=out)
        during.copy_(table)
        ops.kv_release(table, kv_len, lens, stack, height)

    during = torch.zeros_like(table)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    g = torch.Generator(device=DEV)
    g.manual_seed(5)
    for new, fails in (([20, 0, 25], 0), ([1, 1, 1], 0), ([40, 20, 4], 0), ([0, 40, 1], 0), ([0, 0, 0], 0),
                       ([64, 0, 0], 0), ([30, 33, 1], 0)):
        cu.copy_(ints(bounds(new)))
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g, device=DEV))
        out.fill_(7.0)
        graph.replay()
        n = sum(new)
        grown = [a + b for a, b in zip(lens0, new)]
        assert kv_len.tolist() == grown and height.tolist() == [len(free), fails] and stack.tolist()[:len(free)] == free
        want, spread, size = ref.attention(q, cache.k.double(), cache.v.double(), cache.k_scale, cache.v_scale, during,
                                     bounds(new), grown, hd ** -0.5, (-1, 0))
        err, tol = (out.double() - want).abs(), tolerance(want, spread, size, hd, max(grown))
        assert (err[:n] <= tol[:n]).all() and (out[n:] == 7).all()
    height[0] = 1
    cu.copy_(ints([0, 30, 60, 64]))  # three blocks: 100 + 30, 640 + 30 and 64 + 4 tokens
    graph.replay()
    assert height.tolist() == [1, 2] and kv_len.tolist() == lens0


@pytest.mark.parametrize("hd", [64, 128])
def test_questions_on_one_state(hd):
    """Four questions on one state in one pack. The state ends with its block, so its blocks are shared and stay as they
    are bit by bit; the tokens behind its last whole block go in front of each question. The same questions one to a pack,
    too: each pack's answers against the definition."""
    hq, hkv, whole, tail, asks = 4, 2, 256, 37, [5, 20, 1, 64]
    g = torch.Generator(device=DEV)
    g.manual_seed(6)

    def normal(n, heads):
        return torch.randn(n, heads, hd, generator=g, device=DEV).bfloat16()

    state_k, state_v = normal(whole, hkv), normal(whole, hkv)
    new = [tail + n for n in asks]
    q, k, v = normal(sum(new), hq), normal(sum(new), hkv) * 3, normal(sum(new), hkv) * 100
    cache = pool(40, hkv, hd, 9)
    table, stack, height = ints([[-1] * 6] * 4), ints(list(range(40))), ints([40, 0])
    none = ints([0])
    state, _, slots = ops.kv_assign(none, ints([0, whole]), table[:1], stack, height, whole)
    ops.kv_store_e4m3(state_k, state_v, ints([0, whole]), slots, cache)
    table[1:] = table[0]
    lens, before = ints([whole] * 4), table.clone()
    ids = table[0, :whole // BLOCK].long()
    held = [x[ids].clone().view(torch.uint8) for x in (cache.k, cache.v)] + [cache.k_scale[ids], cache.v_scale[ids]]
    outs = []
    for picks in ([0, 1, 2, 3], [0], [1], [2], [3]):
        sizes = [new[i] for i in picks]
        at = torch.cat([torch.arange(bounds(new)[i], bounds(new)[i + 1], device=DEV) for i in picks])
        cu, t = ints(bounds(sizes)), table[picks[0]:picks[-1] + 1]
        kv_len, _, slots = ops.kv_assign(lens[picks[0]:picks[-1] + 1], cu, t, stack, height, sum(sizes))
        assert height[1].item() == 0
        ops.kv_store_e4m3(k[at], v[at], cu, slots, cache)
        outs.append(ops.attention_cache(q[at], cache, t, cu, kv_len, 101, 0.1, (-1, 0)))
        want, spread, size = ref.attention(q[at], cache.k.double(), cache.v.double(), cache.k_scale, cache.v_scale, t,
                                           bounds(sizes), kv_len.tolist(), 0.1, (-1, 0))
        assert ((outs[-1].double() - want).abs() <= tolerance(want, spread, size, hd, whole + 101)).all()
        ops.kv_release(t, kv_len, lens[picks[0]:picks[-1] + 1], stack, height)
        assert torch.equal(table, before)
        after = [x[ids].view(torch.uint8) for x in (cache.k, cache.v)] + [cache.k_scale[ids], cache.v_scale[ids]]
        assert all(torch.equal(x, y) for x, y in zip(held, after))


def test_a_question_leaves_its_scale_in_a_half_filled_block():
    """What a release does not give back: rows that share a state's last block may have made its scale grow, and the
    state's codes there stay rounded to it, each once (to nearest even), until the block is written anew."""
    cache = ops.kv_blocks(2, 1, 64, DEV)
    table, stack, height = ints([[-1, -1]]), ints([0, 1]), ints([2, 0])
    g = torch.Generator(device=DEV)
    g.manual_seed(7)
    small = torch.randn(40, 1, 64, generator=g, device=DEV).bfloat16()
    lens, _, slots = ops.kv_assign(ints([0]), ints([0, 40]), table, stack, height, 40)
    ops.kv_store_e4m3(small, small, ints([0, 40]), slots, cache)
    block = table[0, 0].item()
    values, scale = cache.k[block, 0, :40].double(), cache.k_scale[block, 0].item()
    kv_len, _, slots = ops.kv_assign(lens, ints([0, 10]), table, stack, height, 10)
    ops.kv_store_e4m3(small[:10] * 64, small[:10] * 64, ints([0, 10]), slots, cache)
    ops.kv_release(table, kv_len, lens, stack, height)
    grown = cache.k_scale[block, 0].item()
    assert grown > scale and height.tolist() == [1, 0]
    assert torch.equal(cache.k[block, 0, :40].double(), ref.to_e4m3(values * scale / grown))
