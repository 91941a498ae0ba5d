"""The state cache's operators refuse malformed calls before any launch (no GPU needed), and the float64 restatement the
GPU tests compare with agrees with torch's own e4m3 rounding."""

import ctypes
import math

import pytest
import torch

import cache_reference as ref
from karpo_decision_b200 import _lib, ops


def refused(name, *args):
    assert getattr(_lib.load(), name)(*args) == -1
    return _lib.last_error()


P = 4096  # an aligned address that is never read: the calls below are refused


def test_assign_refusals():
    ok = [P, P, 4, 100, P, 8, 8, P, 10, P, P, P, P, None]
    for at, bad in ((2, -1), (2, 16385), (3, -1), (3, 2 ** 31), (5, 7), (6, -1), (8, -1), (0, None), (1, None),
                    (4, None), (7, None), (9, None), (10, None), (11, None), (12, None)):
        args = list(ok)
        args[at] = bad
        assert "kv_assign" in refused("kd_kv_assign", *args)


def test_release_refusals():
    ok = [P, 8, 8, P, P, 4, P, 10, P, None]
    for at, bad in ((1, 7), (2, -1), (5, -1), (5, 16385), (7, -1), (0, None), (3, None), (4, None), (6, None), (8, None)):
        args = list(ok)
        args[at] = bad
        assert "kv_release" in refused("kd_kv_release", *args)


def test_store_refusals():
    ok = [P, 256, P, 256, 10, P, 2, P, 2, 128, P, P, P, P, 5, None]
    for at, bad in ((1, 255), (1, 128), (3, 250), (4, -1), (6, -1), (8, 0), (8, 70000), (9, 96), (14, -1), (14, 2 ** 31),
                    (0, None), (0, P + 2), (2, None), (5, None), (7, None), (10, P + 8), (11, None), (12, None), (13, None)):
        args = list(ok)
        args[at] = bad
        assert "kv_store" in refused("kd_kv_store_e4m3", *args)


def test_attention_refusals():
    #     q  ldq  k  v  ks vs blk tab ldt w  cu kv n mq tq  out ldo gate ldg hq hkv hd scale l  r  ws bytes st stream
    ok = [P, 512, P, P, P, P, 5, P, 8, 8, P, P, 2, 1, 10, P, 512, P, 512, 4, 2, 128, 0.1, -1, 0, P, 1 << 40, P, None]
    for at, bad in ((1, 511), (1, 256), (6, 0), (6, -1), (6, 2 ** 31), (8, 7), (9, -1), (9, 2 ** 25), (12, -1), (13, -1), (14, -1),
                    (14, 2 ** 30), (16, 500), (18, 130), (19, 3), (19, 0), (20, 0), (21, 96), (22, 0.0), (22, -1.0),
                    (22, math.nan), (0, None), (0, P + 2), (2, P + 8), (3, None), (4, None), (5, None), (7, None),
                    (10, None), (11, None), (15, None), (17, P + 4), (25, None), (25, P + 8), (26, 16), (27, None)):
        args = list(ok)
        args[at] = bad
        assert "attention_cache" in refused("kd_attention_cache", *args), (at, bad)
    size = ctypes.c_int64()
    for bad in ((-1, 1, 10, 4, 2, 128), (1, -1, 10, 4, 2, 128), (1, 1, -1, 4, 2, 128), (1, 1, 10, 3, 2, 128),
                (1, 1, 10, 4, 0, 128), (1, 1, 10, 4, 2, 96)):
        assert "workspace" in refused("kd_attention_cache_workspace", *bad, ctypes.addressof(size))


def test_the_wrappers_check_types_shapes_and_devices():
    """On CPU tensors: every wrapper refuses them by name before it calls the library."""
    cache = ops.kv_blocks(4, 2, 64, torch.device("cpu"))
    i32 = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="lens"):
        ops.kv_assign(i32, torch.zeros(4, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32), i32, i32[:2], 5)
    with pytest.raises(ValueError, match="lens"):
        ops.kv_release(torch.zeros(3, 2, dtype=torch.int32), i32, i32, i32, i32[:2])
    rows = torch.zeros(5, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv_store_e4m3(rows, rows, i32, torch.zeros(5, dtype=torch.int64), cache)
    with pytest.raises(ValueError, match="CUDA"):
        ops.attention_cache(rows, cache, torch.zeros(2, 2, dtype=torch.int32), i32, i32[:2], 1, 0.1, (-1, 0))
    with pytest.raises(ValueError, match="scales"):
        ops.KVBlocks(cache.k, cache.v, torch.ones(4, 3), cache.v_scale)
    with pytest.raises(ValueError, match="e4m3"):
        ops.KVBlocks(cache.k.float(), cache.v.float(), cache.k_scale, cache.v_scale)
    with pytest.raises(ValueError, match="codes"):
        ops.KVBlocks(cache.k[:, :, :32], cache.v[:, :, :32], cache.k_scale, cache.v_scale)


@pytest.mark.parametrize("current,switched", [(0, []), (1, [0])])
def test_a_call_goes_to_its_tensors_device(monkeypatch, current, switched):
    """With another device current, the wrapper's call runs with the tensors' one current, on that one's stream."""
    device, seen, calls = [current], [], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            seen.append(self.index)
            self.before, device[0] = device[0], self.index

        def __exit__(self, *error):
            device[0] = self.before

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: device[0], raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 1000 + index, raising=False)
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(ops, "call", lambda name, *args: calls.append((name, args, device[0])))
    ops._call_on(0, "kd_kv_release", 7, 8)
    assert calls == [("kd_kv_release", (7, 8, 1000), 0)] and seen == switched and device == [current]


def test_the_restatement_rounds_as_torch_does():
    x = torch.cat([torch.linspace(-460, 460, 4001, dtype=torch.float64), torch.logspace(-4, 2, 3001, dtype=torch.float64)])
    want = x.float().clamp(-448, 448).to(torch.float8_e4m3fn).double()
    assert torch.equal(ref.to_e4m3(x.float().double()), want)


@pytest.mark.parametrize("amax,e", [(448.0, 0), (449.0, 1), (447.0, 0), (224.0, -1), (1.0, -8), (1.75, -8), (1.76, -7),
                                    (0.0, -100), (2.0 ** -130, -100), (3.38e38, 120)])
def test_the_scale_is_the_least_power_of_two_that_fits(amax, e):
    assert ref.exponent(amax) == e
    assert amax * 2.0 ** -e <= 448 or e == 120
