"""Rotary tables and the argument checks of the paged cache that need no GPU."""
from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest


def angles(table):
    R = table.rotary_dim
    c, s = table.cos_sin[:, :R // 2].double(), table.cos_sin[:, R // 2:].double()
    return np.hypot(c.numpy(), s.numpy()), np.arctan2(s.numpy(), c.numpy())


def table(*args, **kw):
    import torch
    from ffn_residual_mesh_b200.kvcache import RotaryTable
    return RotaryTable(*args, device=torch.device("cpu"), **kw)


@pytest.mark.parametrize("kind,factor", [(None, 1.0), ("linear", 4.0), ("ntk", 4.0), ("yarn", 8.0)])
def test_rotary_table(kind, factor):
    R, n, base, orig = 64, 300, 10000.0, 4096
    t = table(R, n, base=base, scaling=kind, factor=factor, original_positions=orig)
    gain, angle = angles(t)
    want_gain = 0.1 * math.log(factor) + 1 if kind == "yarn" else 1.0
    assert np.abs(gain - want_gain).max() < 3e-7
    for i in range(R // 2):
        f = base ** (-2 * i / R)
        if kind == "linear":
            f /= factor
        elif kind == "ntk":
            f = (base * factor ** (R / (R - 2))) ** (-2 * i / R)
        elif kind == "yarn":
            turns = lambda r: R * math.log(orig / (r * 2 * math.pi)) / (2 * math.log(base))
            low, high = math.floor(turns(32)), math.ceil(turns(1))
            ramp = min(max((i - low) / (high - low), 0), 1)
            f = f * (1 - ramp) + f / factor * ramp
        p = np.arange(n) * f
        off = (angle[:, i] - p + math.pi) % (2 * math.pi) - math.pi
        assert np.abs(off).max() < 1e-6
    if kind == "ntk":  # the fastest pair as it was, the slowest slowed by the factor
        assert abs(base ** (-(R - 2) / R) / factor - (base * factor ** (R / (R - 2))) ** (-(R - 2) / R)) < 1e-12


@pytest.mark.parametrize("kw", [dict(rotary_dim=3, max_positions=4), dict(rotary_dim=0, max_positions=4), dict(rotary_dim=4, max_positions=0),
                                dict(rotary_dim=4, max_positions=4, scaling="cubic"), dict(rotary_dim=4, max_positions=4, base=1.0),
                                dict(rotary_dim=4, max_positions=4, scaling="linear", factor=0.5),
                                dict(rotary_dim=4, max_positions=4, scaling="yarn", factor=2.0)])
def test_rotary_table_refuses(kw):
    with pytest.raises(ValueError):
        table(**kw)


def test_rotary_table_from_tensor_refuses():
    import torch
    from ffn_residual_mesh_b200.kvcache import RotaryTable
    for bad in (torch.zeros(4, 6, dtype=torch.float64), torch.zeros(4, 5), torch.zeros(8), torch.zeros(8, 4)[:, :2], torch.zeros(0, 4)):
        with pytest.raises(ValueError):
            RotaryTable.from_tensor(bad)


@pytest.mark.parametrize("cfg", [(0, 4, 1, 64, 16, 1), (1, 0, 1, 64, 16, 1), (1, (1 << 20) + 1, 1, 64, 16, 1), (1, 4, 0, 64, 16, 1),
                                 (1, 4, 1, 96, 16, 1), (1, 4, 1, 64, 24, 1), (1, 4, 1, 64, 256, 1), (1, 4, 1, 64, 16, 0),
                                 (1, 4, 1, 64, 16, 4097), (1, 4, 2000, 64, 16, 1)])
def test_create_refuses_shapes_before_any_device(cfg):
    from ffn_residual_mesh_b200 import _native as N
    from ffn_residual_mesh_b200 import build
    build.build()
    handle = ctypes.c_void_p()
    rc = N.lib().ffnrm_kv_create(ctypes.byref(handle), 0, ctypes.byref(N.KvConfig(*cfg)), 16, 16, 16, 16)
    assert rc == N.ERR_ARG and not handle.value
    with pytest.raises(ValueError):
        N.check(rc)


def test_create_refuses_pools():
    from ffn_residual_mesh_b200 import _native as N
    cfg, handle = N.KvConfig(1, 4, 1, 64, 16, 1), ctypes.c_void_p()
    for pools in ((None, 16, 16, 16), (16, 16, 16, None), (8, 16, 16, 16), (16, 24, 16, 16), (16, 16, 18, 16)):
        assert N.lib().ffnrm_kv_create(ctypes.byref(handle), 0, ctypes.byref(cfg), *pools) == N.ERR_ARG
    assert N.lib().ffnrm_kv_create(None, 0, ctypes.byref(cfg), 16, 16, 16, 16) == N.ERR_ARG


def test_null_cache_and_rotary_arguments_are_refused():
    from ffn_residual_mesh_b200 import _native as N
    lib, null = N.lib(), None
    batch = N.KvBatch(16, 16, None, 1, 1, 1)
    rows = N.Rows(64, 64, 64)
    assert lib.ffnrm_kv_attend(null, 0, ctypes.byref(batch), 0, ctypes.byref(rows), ctypes.byref(rows), None, 1, 1.0, 1, 0, None) == N.ERR_ARG
    assert lib.ffnrm_kv_check(null, None) == N.ERR_ARG and lib.ffnrm_kv_destroy(null) == N.OK
    assert lib.ffnrm_kv_copy_pages(null, 16, 16, 1, None) == N.ERR_ARG

    def rotary(x=rows, y=rows, dtype=0, tokens=2, heads=1, dim=64, pos=16, table=16, rot=64, most=4, flags=0):
        return lib.ffnrm_rotary(ctypes.byref(x), ctypes.byref(y), dtype, tokens, heads, dim, pos, table, rot, most, flags, None)

    for kw in (dict(dtype=3), dict(dtype=-1), dict(tokens=-1), dict(dim=0), dict(rot=66), dict(rot=7), dict(rot=0), dict(most=0),
               dict(flags=4), dict(table=None), dict(pos=None), dict(pos=18), dict(x=N.Rows(None, 64, 64)),
               dict(y=N.Rows(64, 128, 64)), dict(x=N.Rows(65, 64, 64))):
        assert rotary(**kw) == N.ERR_ARG, kw
    assert rotary(tokens=0) == N.OK and rotary(heads=0) == N.OK


@pytest.mark.parametrize("R,base,orig,factor", [(128, 1e4, 131072, 8.0), (128, 1e4, 8192, 4.0), (64, 1e4, 65536, 16.0), (32, 500.0, 1000000, 2.0),
                                                (256, 1e6, 4096, 8.0), (16, 1e4, 300, 32.0)])
def test_yarn_ramp_where_the_last_pair_lies_inside_it(R, base, orig, factor):
    """Pairs of more than 32 turns stay and those below one turn are divided, whichever end of the head the ramp
    reaches; between them the ramp is straight from floor to ceil of its fractional pairs, held to [0, R - 1]."""
    t = table(R, 64, base=base, scaling="yarn", factor=factor, original_positions=orig)
    angle = angles(t)[1]
    low = max(math.floor(R * math.log(orig / (64 * math.pi)) / (2 * math.log(base))), 0)
    high = min(math.ceil(R * math.log(orig / (2 * math.pi)) / (2 * math.log(base))), R - 1)
    for i in range(R // 2):
        f = base ** (-2 * i / R)
        turns = orig * f / (2 * math.pi)
        ramp = min(max((i - low) / (high - low), 0.0), 1.0)
        assert (turns <= 32 or ramp == 0) and (turns >= 1 or ramp == 1)
        p = np.arange(64) * (f * (1 - ramp) + f / factor * ramp)
        off = (angle[:, i] - p + math.pi) % (2 * math.pi) - math.pi
        assert np.abs(off).max() < 1e-5, (i, f, ramp)


def test_yarn_last_pair_of_a_long_trained_context():
    """2.4 turns in 131072 positions: 0.37 of its frequency, not an eighth."""
    t = table(128, 8, base=1e4, scaling="yarn", factor=8.0, original_positions=131072)
    got = angles(t)[1][1, 63] / 1e4 ** (-126 / 128)
    assert abs(got - 0.37) < 0.01


def test_overlapping_rows_are_refused():
    """Written rows lie apart from one another, and on the rows that are read or apart from them: against the sets
    of elements, over random layouts. (Null positions end each call before any launch.)"""
    import random
    from ffn_residual_mesh_b200 import _native as N
    lib, rng, seen = N.lib(), random.Random(1), [0, 0, 0]

    def elements(at, T, H, st, sh, dim):
        return [at + t * st + h * sh + i for t in range(T) for h in range(H) for i in range(dim)]

    for _ in range(6000):
        T, H, dim = rng.randint(1, 4), rng.randint(1, 3), rng.choice([2, 4, 6])
        sx = rng.choice([(H * dim, dim), (dim, T * dim), (2 * H * dim, dim), (3 * dim * H, 3 * dim), (dim + 1, 9), (rng.randint(0, 40), rng.randint(0, 12))])
        sy = sx if rng.random() < 0.6 else (rng.randint(0, 40), rng.choice([dim, dim + 1, 2 * dim]))
        d = rng.choice([0, dim, H * dim, rng.randint(-60, 60)])
        x, y = elements(1000, T, H, *sx, dim), elements(1000 + d, T, H, *sy, dim)
        size = 4
        xr, yr = N.Rows(size * 1000, *sx), N.Rows(size * (1000 + d), *sy)
        assert lib.ffnrm_rotary(ctypes.byref(xr), ctypes.byref(yr), N.F32, T, H, dim, None, 16, 2, 4, 0, None) == N.ERR_ARG
        message = lib.ffnrm_last_error().decode()
        if len(set(y)) < len(y):
            assert "on one another" in message
            seen[0] += 1
        elif x != y and set(x) & set(y):
            assert "itself or lie apart" in message, (T, H, dim, sx, sy, d)
            seen[1] += 1
        elif T == 1 or sx[0] == sy[0] or x == y or max(x) < min(y) or max(y) < min(x):
            assert "positions" in message, (message, T, H, dim, sx, sy, d)
            seen[2] += 1
    assert min(seen) > 300, seen
