"""Refusals of the gated linear recurrence that need no GPU, and the 64-bit restatement's gradients against differences."""
import ctypes as C

import numpy as np
import pytest
import torch

from tacotron2_amd import _lib
from tests import recurrence_ref as ref


def _args(**kw):
    a = _lib.T2ScanArgs()
    a.dtype, a.B, a.T, a.H = 0, 2, 3, 4
    for name in ("z", "f", "y", "dy", "dz", "df"):
        setattr(a, name, (16, 12, 4))
    a.tape = 16
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_library_refuses_bad_arguments_before_any_device_work():
    lib = _lib.load()
    ctx = C.create_string_buffer(64)                 # never looked into: every call below is refused first
    null = (None, 0, 0)
    for fn, bad in ((lib.t2_gated_scan, [{"dtype": 3}, {"dtype": -1}, {"B": 0}, {"B": 65536}, {"T": 0}, {"T": (1 << 30) + 1}, {"H": 0}, {"H": (1 << 24) + 1},
                                         {"z": null}, {"f": null}, {"y": null}]),
                    (lib.t2_gated_scan_backward, [{"dy": null}, {"dz": null}, {"df": null}, {"o": (16, 12, 4)}, {"tape": None}, {"z": null}, {"dtype": 7}])):
        assert fn(None, _args()) == _lib.T2_EINVAL and fn(ctx, None) == _lib.T2_EINVAL
        for kw in bad:
            assert fn(ctx, _args(**kw)) == _lib.T2_EINVAL, kw
    assert fn is lib.t2_gated_scan_backward
    both = {"state": 1 << 20, "final_state": (1 << 20) + 4 * 7}                       # of the 8 floats of each, one is shared
    assert lib.t2_gated_scan(ctx, _args(**both)) == _lib.T2_EINVAL and b"overlap" in lib.t2_last_error()
    assert lib.t2_gated_scan_backward(ctx, _args(dfinal=1 << 20, dstate=1 << 20)) == _lib.T2_EINVAL and b"overlap" in lib.t2_last_error()
    at = 1 << 20
    apart = {"z": (at, 12, 4), "f": (2 * at, 12, 4), "dy": (3 * at, 12, 4), "y": (4 * at, 12, 4), "dz": (5 * at, 12, 4), "df": (6 * at, 12, 4), "ws": None}

    def meets(fn, **kw):
        assert fn(ctx, _args(**{**apart, **kw})) == _lib.T2_EINVAL, kw
        return b"overlap" in lib.t2_last_error()
    # the same place; one channel, one step, one row on; time-major; another layout of the same place
    for y in ((at, 12, 4), (at + 4, 12, 4), (at - 4 * 4, 12, 4), (at + 4 * 12, 12, 4), (at + 4 * 12 - 12, 12, 4), (at, 100, 8)):
        assert meets(lib.t2_gated_scan, y=y), y
    assert meets(lib.t2_gated_scan, z=(at, 4, 8), y=(at + 4 * 8 - 4, 4, 8)) and meets(lib.t2_gated_scan, o=(7 * at, 12, 4), y=(7 * at + 4, 12, 4))
    for kw in ({"dz": (3 * at, 12, 4)}, {"df": (5 * at + 12, 12, 4)}, {"dz": (2 * at, 12, 4)}, {"o": (7 * at, 12, 4), "do_": (at, 12, 4)},
               {"o": (7 * at, 12, 4), "do_": (6 * at, 12, 4)}):
        assert meets(lib.t2_gated_scan_backward, **kw), kw
    # parts of one [2, 3, 8] tensor: apart, so what is refused is the missing workspace (T = 300) and nothing else
    slab = {"T": 300, "z": (at, 2400, 8), "y": (at + 16, 2400, 8), "f": (2 * at, 2400, 8)}
    assert not meets(lib.t2_gated_scan, **slab)
    step = lambda **kw: lib.t2_gated_scan_step(*{**dict(ctx=ctx, dtype=0, B=2, H=4, z=16, zs=4, f=16, fs=4, o=None, os=0, state=16, ss=4, active=None,  # noqa: E731
                                                        y=16, ys=4), **kw}.values())
    for kw in ({"ctx": None}, {"dtype": 5}, {"B": 0}, {"H": 0}, {"z": None}, {"f": None}, {"state": None}, {"y": None}, {"ss": 3}, {"ys": 3}):
        assert step(**kw) == _lib.T2_EINVAL, kw
    ok = {"z": at, "f": 2 * at, "o": 3 * at, "os": 4, "state": 4 * at, "y": 5 * at}
    for kw in ({"y": 4 * at}, {"y": 4 * at + 12}, {"y": at + 4}, {"y": 2 * at + 4 * 4}, {"state": at}, {"state": 3 * at + 4}, {"y": at, "ys": 8},
               {"dtype": 1, "state": at, "ss": 4}):
        assert step(**{**ok, **kw}) == _lib.T2_EINVAL and b"overlap" in lib.t2_last_error(), kw
    assert lib.t2_gated_scan_tape(2, 65, 3) == 2 * 2 * 3 and lib.t2_gated_scan_tape(0, 1, 1) < 0 and lib.t2_gated_scan_ws(1, 0, 1) < 0
    big = lib.t2_gated_scan_tape(64, 1 << 30, 1 << 12)                               # counts beyond 32 bits
    assert big == 64 * (1 << 24) * (1 << 12)


def test_python_layer_refuses_host_tensors():
    from tacotron2_amd import recurrence as R
    z = torch.zeros(1, 2, 3)
    with pytest.raises(ValueError):
        R.gated_scan(None, z, z)
    with pytest.raises(ValueError):
        R.gated_scan_step(None, z[0], z[0], None, z[0])


@pytest.mark.parametrize("reverse", [False, True])
def test_restatement_against_a_loop_and_differences(reverse):
    rng = np.random.default_rng(3)
    z, f, o, dy = (rng.standard_normal((2, 6, 3)) for _ in range(4))
    state, dfinal, lens = rng.standard_normal((2, 3)), rng.standard_normal((2, 3)), np.array([6, 4])

    def loss(z, f, o, state):
        total = 0.0
        for b in range(2):
            h = state[b].copy()
            order = range(lens[b] - 1, -1, -1) if reverse else range(lens[b])
            for t in order:
                a = 1 / (1 + np.exp(-f[b, t]))
                h = a * h + (1 - a) * z[b, t]
                total += (dy[b, t] * h / (1 + np.exp(-o[b, t]))).sum()
            total += (dfinal[b] * h).sum()
        return total
    x = ref.forward(z, f, o, lens, state, reverse)
    assert abs((x["y"] * dy).sum() + (x["final"] * dfinal).sum() - loss(z, f, o, state)) < 1e-12
    g = ref.backward(x, dy, dfinal, lens, reverse)
    for i, k in enumerate(("dz", "df", "do", "dstate")):
        base = [z, f, o, state]
        for at in np.ndindex(base[i].shape):
            up, down = [v.copy() for v in base], [v.copy() for v in base]
            up[i][at] += 1e-5
            down[i][at] -= 1e-5
            assert abs((loss(*up) - loss(*down)) / 2e-5 - g[k][at]) < 1e-8


def test_overlaps_of_every_kind_are_refused_before_any_device_work():
    """What a tile writes, another tile may still have to read: the states, the tape, the lengths and the workspace count like z, f and o."""
    lib = _lib.load()
    ctx = C.create_string_buffer(64)
    at, T, H, B = 1 << 20, 300, 4, 2
    place = lambda k: (k * at, T * H, H)  # noqa: E731
    base = {"B": B, "T": T, "H": H, "z": place(1), "f": place(2), "y": place(3), "dy": place(4), "dz": place(5), "df": place(6), "tape": 7 * at, "state": 8 * at,
            "final_state": 9 * at, "dfinal": 10 * at, "dstate": 11 * at, "lens": 12 * at, "ws": 13 * at, "ws_bytes": 0}

    def refused(fn, **kw):
        assert fn(ctx, _args(**{**base, **kw})) == _lib.T2_EINVAL
        return lib.t2_last_error()
    for fn in (lib.t2_gated_scan, lib.t2_gated_scan_backward):
        assert b"workspace" in refused(fn)                                          # apart: only the workspace is too small
    last = 3 * at + (T * H - H) * 4                                                 # the last row of y's first sequence
    n_tape = lib.t2_gated_scan_tape(B, T, H) * 4
    for kw in ({"state": last}, {"state": last + 12}, {"state": last - B * H * 4 + 4}, {"final_state": last}, {"lens": last - 8}, {"lens": 9 * at + 28},
               {"tape": last}, {"tape": 3 * at - n_tape + 4}, {"tape": 8 * at + 28}, {"tape": 12 * at - n_tape + 4}, {"ws": last - 4}, {"ws": 7 * at},
               {"final_state": 8 * at}, {"y": (3 * at, 0, H)}, {"y": (3 * at, T * H, 0)}, {"y": (3 * at, T * H, H - 1)}, {"y": (3 * at, T * H - 1, H)},
               {"y": (3 * at, H - 1, 2 * H)}):
        assert b"overlap" in refused(lib.t2_gated_scan, **kw), kw
    for kw in ({"dz": (7 * at + n_tape - 4, T * H, H)}, {"df": (10 * at + 28, T * H, H)}, {"dz": (12 * at + 15, T * H, H)}, {"dstate": 7 * at}, {"dstate": 10 * at},
               {"dstate": 6 * at + 4}, {"dstate": 12 * at}, {"ws": 10 * at}, {"ws": 6 * at}, {"dz": (5 * at, T * H, 0)}):
        assert b"overlap" in refused(lib.t2_gated_scan_backward, **kw), kw
    # states that lie in front of the first and behind the last element are apart
    for kw in ({"state": 3 * at - B * H * 4}, {"state": 3 * at + B * T * H * 4}, {"lens": 3 * at - B * 8}, {"tape": 3 * at + B * T * H * 4}):
        assert b"workspace" in refused(lib.t2_gated_scan, **kw), kw
    # strides that no memory holds
    assert b"strides" in refused(lib.t2_gated_scan, z=(at, 1 << 62, H)) and b"strides" in refused(lib.t2_gated_scan, y=(at, H, -(1 << 62)))
    step = lambda **kw: lib.t2_gated_scan_step(*{**dict(ctx=ctx, dtype=0, B=2, H=4, z=at, zs=4, f=2 * at, fs=4, o=None, os=0, state=4 * at, ss=4, active=6 * at,  # noqa: E731
                                                        y=5 * at, ys=4), **kw}.values())
    for kw in ({"active": 4 * at + 31}, {"active": 5 * at}, {"zs": 5, "z": 4 * at + 8}, {"zs": 0, "z": 5 * at + 16}, {"zs": -4, "z": 5 * at + 40}):
        assert step(**kw) == _lib.T2_EINVAL and b"overlap" in lib.t2_last_error(), kw


def test_overlaps_of_different_strides_are_found_exactly():
    """Against the sets of bytes themselves: broadcast, reversed, windowed and interleaved inputs around an output in one buffer."""
    lib = _lib.load()
    ctx = C.create_string_buffer(64)
    rng = np.random.default_rng(12)
    T, far, seen = 257, 1 << 30, [0, 0]
    for _ in range(400):
        B, H = int(rng.integers(1, 4)), int(rng.integers(1, 6))
        if rng.random() < 0.5:
            st = H + int(rng.integers(0, 9))
            sb = (T - 1) * st + H + int(rng.integers(0, 40))
        else:
            sb = H + int(rng.integers(0, 9))
            st = (B - 1) * sb + H + int(rng.integers(0, 20))
        zb, zt = (int(rng.choice([0, sb, -sb, st, 1, H, 3 * H, T * H])), int(rng.choice([0, st, -st, sb, 1, H, 2 * H, B * H])))
        if B == 1:
            zb = int(rng.choice([0, 7, -7]))

        def covered(ptr, b, t, row):
            rows = ptr + 4 * (np.arange(B)[:, None] * b + np.arange(T)[None, :] * t)
            return np.unique(rows[..., None] + np.arange(row))
        span = 4 * ((B - 1) * sb + (T - 1) * st + H)
        y = far
        z = far + 4 * int(rng.integers(-200, span // 4 + 200)) + 4 * (max(0, -zb) * (B - 1) + max(0, -zt) * (T - 1))
        state = far + 4 * int(rng.integers(-40, span // 4 + 40))
        ours = covered(y, sb, st, 4 * H)
        for kw, theirs in (({"z": (z, zb, zt)}, covered(z, zb, zt, 4 * H)), ({"state": state}, np.arange(state, state + 4 * B * H))):
            args = _args(**{"B": B, "T": T, "H": H, "z": (far // 2, T * H, H), "f": (far // 4, T * H, H), "y": (y, sb, st), "tape": None, **kw})
            assert lib.t2_gated_scan(ctx, args) == _lib.T2_EINVAL
            want = bool(np.intersect1d(ours, theirs, assume_unique=True).size)
            got = b"overlap" in lib.t2_last_error()
            assert got == want and (got or b"workspace" in lib.t2_last_error()), (B, T, H, sb, st, kw, lib.t2_last_error())
            seen[want] += 1
    assert min(seen) > 100, seen


def test_context_options():
    lib = _lib.load()
    ctx = C.create_string_buffer(256)                # takes the option's value; no device work
    assert lib.t2_ctx_set_option(ctx, b"scan_wait_us", 0) == _lib.T2_OK and lib.t2_ctx_set_option(ctx, b"scan_wait_us", 2000000) == _lib.T2_OK
    for bad in ((None, b"scan_wait_us", 1), (ctx, None, 1), (ctx, b"scan_wait", 1), (ctx, b"scan_wait_us", -1)):
        assert lib.t2_ctx_set_option(*bad) == _lib.T2_EINVAL, bad


def test_sizes_whose_tape_has_no_count_are_refused():
    lib = _lib.load()
    assert lib.t2_gated_scan_tape(65535, 1 << 30, 1 << 24) < 0 and lib.t2_gated_scan_tape(1 << 14, 1 << 30, 1 << 24) < 0
    assert lib.t2_gated_scan_tape(1 << 12, 1 << 30, 1 << 24) < 0 < lib.t2_gated_scan_tape(1 << 11, 1 << 30, 1 << 24) == 1 << 59 and lib.t2_gated_scan_ws(65535, 1 << 30, 1 << 24) < 0
