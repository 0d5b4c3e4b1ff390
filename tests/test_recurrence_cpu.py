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
