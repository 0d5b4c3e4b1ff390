"""The gated linear recurrence (tacotron2_amd/recurrence.py) on the GPU against 64-bit restatements (recurrence_ref.py), which also
give the bound of every element.  A result in fewer bits may be off by half a step of its type on top, and by half the
smallest subnormal; gates below 2^-126 count as 2^-126, times values under 2^15 here."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from tests import recurrence_ref as ref

torch = pytest.importorskip("torch")
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TINY = {"f32": 2.0 ** -110, "bf16": 2.0 ** -110, "f16": 2.0 ** -25}


def _close(got, want, bound, what, dtype=None):
    got = got.detach().double().cpu().numpy()
    with np.errstate(invalid="ignore"):
        tol = np.abs(bound) + TINY["f32"]                     # results that stay fp32: the gates' own floor alone
        if dtype is not None:
            tol = tol * 1.01 + np.abs(want) * (torch.finfo(DTYPES[dtype]).eps / 2) + TINY[dtype]
        off = np.abs(got - want)
    special = ~np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    assert np.array_equal(got[special & ~np.isnan(want)], want[special & ~np.isnan(want)]), what
    bad = ~special & ~(off <= tol)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:3].tolist(), float(np.nanmax(np.where(bad, off / tol, 0))))


def _inputs(B, T, H, dtype, gate, seed, spread=2.0, shift=1.0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    dt = DTYPES[dtype]
    z, f = r(B, T, H).to(dt).cuda(), (r(B, T, H) * spread + shift).to(dt).cuda()
    o = r(B, T, H).to(dt).cuda() if gate else None
    return z, f, o, r(B, H).cuda(), r(B, T, H).to(dt).cuda(), r(B, H).cuda()


def _np(x):
    return None if x is None else x.detach().double().cpu().numpy()


def _check(z, f, o, lens, state, dy, dfinal, reverse, dtype, out=None, ctx=None):
    from tacotron2_amd import recurrence as R
    B, T, H = z.shape
    n = np.full(B, T) if lens is None else np.asarray(lens.cpu() if isinstance(lens, torch.Tensor) else lens).clip(0, T)
    y, final, tape = R.gated_scan(ctx, z, f, o, lens=lens, state=state, reverse=reverse, tape=True, out=out)
    y2, final2 = R.gated_scan(ctx, z, f, o, lens=lens, state=state, reverse=reverse)
    dz, df, do, dstate = R.gated_scan_backward(ctx, tape, dy, dfinal)
    x = ref.forward(_np(z), _np(f), _np(o), n, np.zeros((B, H)) if state is None else _np(state), reverse)
    g = ref.backward(x, _np(dy), np.zeros((B, H)) if dfinal is None else _np(dfinal), n, reverse)
    _close(y, x["y"], x["ey"], "y", dtype)
    _close(final, x["final"], x["efinal"], "final")
    assert torch.equal(y.nan_to_num(7), y2.nan_to_num(7)) and torch.equal(final.nan_to_num(7), final2.nan_to_num(7))
    _close(dz, g["dz"], g["edz"], "dz", dtype)
    _close(df, g["df"], g["edf"], "df", dtype)
    assert (do is None) == (o is None)
    if o is not None:
        _close(do, g["do"], g["edo"], "do", dtype)
    _close(dstate, g["dstate"], g["edstate"], "dstate")
    return y, final, (dz, df, do, dstate)


SHAPES = [(1, 1, 1), (2, 2, 4), (3, 5, 7), (2, 63, 64), (2, 64, 65), (1, 65, 128), (3, 127, 12), (2, 129, 66), (5, 140, 256), (1, 257, 36), (2, 513, 100)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,T,H", SHAPES)
def test_scan_and_gradients(B, T, H, dtype):
    for k, (gate, reverse, ragged) in enumerate([(True, False, False), (False, True, True), (True, True, True), (False, False, True)]):
        z, f, o, state, dy, dfinal = _inputs(B, T, H, dtype, gate, 100 * T + H + k)
        lens = None
        if ragged:
            lens = torch.from_numpy(np.random.default_rng(T + k).integers(0, T + 1, B)).cuda()
        _check(z, f, o, lens, state if k % 2 == 0 else None, dy, dfinal if k < 2 else None, reverse, dtype)


@pytest.mark.parametrize("dtype,B,T,H", [("f32", 1, 9001, 20), ("bf16", 2, 12345, 68), ("f16", 1, 20000, 64)])
def test_long_sequences(dtype, B, T, H):
    for reverse in (False, True):
        z, f, o, state, dy, dfinal = _inputs(B, T, H, dtype, True, T, spread=1.5, shift=4.0)
        lens = torch.tensor([T - 131 * b for b in range(B)], device="cuda") if reverse else None
        _check(z, f, o, lens, state, dy, dfinal, reverse, dtype)


@pytest.mark.parametrize("dtype,B,T,H,reverse", [("bf16", 8, 12300, 512, True), ("f16", 2, 25000, 1001, False), ("f32", 3, 16500, 517, False)])
def test_large_calls(dtype, B, T, H, reverse):
    """Enough work for the wide tiles; channels are independent, so some of them are held to the restatement."""
    from tacotron2_amd import recurrence as R
    gen = torch.Generator(device="cuda").manual_seed(T)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    dt = DTYPES[dtype]
    z, f, o, dy = r(B, T, H).to(dt), (r(B, T, H) * 1.5 + 3).to(dt), r(B, T, H).to(dt), r(B, T, H).to(dt)
    state, dfinal = r(B, H), r(B, H)
    lens = torch.tensor([T - 700 * b for b in range(B)], device="cuda")
    y, final, tape = R.gated_scan(None, z, f, o, lens=lens, state=state, reverse=reverse, tape=True)
    dz, df, do, dstate = R.gated_scan_backward(None, tape, dy, dfinal)
    rows, cols = [0, B - 1], sorted({0, 1, 63, 64, 127, 128, 255, 256, 400, H - 5, H - 4, H - 2, H - 1})
    pick = lambda t: t[rows][..., cols]  # noqa: E731
    n = lens.cpu().numpy()[rows]
    x = ref.forward(_np(pick(z)), _np(pick(f)), _np(pick(o)), n, _np(pick(state)), reverse)
    g = ref.backward(x, _np(pick(dy)), _np(pick(dfinal)), n, reverse)
    for got, want, bound, what, d in ((y, x["y"], x["ey"], "y", dtype), (final, x["final"], x["efinal"], "final", None), (dz, g["dz"], g["edz"], "dz", dtype),
                                      (df, g["df"], g["edf"], "df", dtype), (do, g["do"], g["edo"], "do", dtype), (dstate, g["dstate"], g["edstate"], "dstate", None)):
        _close(pick(got), want, bound, what, d)
    live = torch.arange(T, device="cuda")[None, :, None] < lens[:, None, None]
    for t in (y, dz, df, do):
        assert torch.isfinite(t).all() and not t.masked_select(~live).any()


@pytest.mark.parametrize("H", [1, 2, 3])
def test_narrow_rows(H):
    for T in (63, 300, 900):
        z, f, o, state, dy, dfinal = _inputs(3, T, H, "bf16", True, T + H)
        _check(z, f, o, torch.tensor([T, T // 3, 0], device="cuda"), state, dy, dfinal, True, "bf16")


def test_distances_beyond_32_bits():
    """Rows 2^31 elements apart, and steps further apart than a tile's offsets reach."""
    from tacotron2_amd import recurrence as R
    for dtype, stride_b, stride_t, T in (("bf16", 2 ** 31 + 24, 24, 300), ("f32", 24, 2 ** 22, 300), ("f16", 2 ** 23, 2 ** 23, 90)):
        z, f, o, state, dy, dfinal = _inputs(1 if stride_b == stride_t else 2, T, 24, dtype, True, 6)

        def far(x):
            size = (x.shape[0] - 1) * stride_b + (T - 1) * stride_t + 24
            v = torch.empty(size, dtype=x.dtype, device="cuda").as_strided(x.shape, (stride_b, stride_t, 1))
            v.copy_(x)
            return v
        a = R.gated_scan(None, z, f, o, state=state, tape=True)
        b = R.gated_scan(None, far(z), f, o, state=state, tape=True, out=far(z))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        for want, got in zip(R.gated_scan_backward(None, a[2], dy, dfinal), R.gated_scan_backward(None, b[2], far(dy), dfinal)):
            assert torch.equal(want, got)


def test_many_rows():
    z, f, o, state, dy, dfinal = _inputs(300, 131, 70, "bf16", True, 5)
    lens = torch.arange(300, device="cuda", dtype=torch.int32) % 132
    _check(z, f, o, lens, state, dy, dfinal, False, "bf16")


@pytest.mark.parametrize("T", [1, 64, 65, 200, 1000])
def test_lengths_of_zero_one_and_outside(T):
    z, f, o, state, dy, dfinal = _inputs(6, T, 33, "f32", True, T)
    lens = torch.tensor([0, 1, T, max(0, T - 1), -5, T + 7], device="cuda")
    y, final, (dz, df, do, dstate) = _check(z, f, o, lens, state, dy, dfinal, True, "f32")
    assert torch.equal(final[0], state[0]) and torch.equal(dstate[0], dfinal[0]) and torch.equal(final[4], state[4])
    assert not y[0].any() and not dz[0].any() and not df[4].any() and not do[4].any()
    with pytest.raises(ValueError):
        _check(z, f, o, [0, 1, T, 0, -1, 0], state, dy, dfinal, False, "f32")
    with pytest.raises(ValueError):
        _check(z, f, o, [0, 1, T, 0, T + 1, 0], state, dy, dfinal, False, "f32")
    _check(z, f, o, [0, 1, T, max(0, T - 1), 0, T], state, dy, dfinal, False, "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("reverse", [False, True])
def test_nothing_behind_a_length_is_read_into_a_result(dtype, reverse):
    z, f, o, state, dy, dfinal = _inputs(4, 150, 40, dtype, True, 8)
    lens = torch.tensor([0, 1, 149, 77], device="cuda")
    a = _check(z, f, o, lens, state, dy, dfinal, reverse, dtype)
    junk = torch.arange(150, device="cuda")[None, :, None] >= lens[:, None, None]
    poison = [x.masked_fill(junk, v) for x, v in ((z, float("nan")), (f, float("inf")), (o, float("nan")), (dy, float("-inf")))]
    from tacotron2_amd import recurrence as R
    y, final, tape = R.gated_scan(None, poison[0], poison[1], poison[2], lens=lens, state=state, reverse=reverse, tape=True)
    grads = R.gated_scan_backward(None, tape, poison[3], dfinal)
    assert torch.equal(y, a[0]) and torch.equal(final, a[1])
    for got, want in zip(grads, a[2]):
        assert torch.equal(got, want)


def test_extreme_gates_and_values():
    """Gates that are shut, open, or infinite; infinities and NaN in z spread only along their own channel, and only forwards."""
    z, f, o, state, dy, dfinal = _inputs(2, 300, 12, "f32", True, 3)
    f[:, :, 0], f[:, :, 1] = -200.0, 200.0
    f[:, :, 2], f[:, :, 3] = float("-inf"), float("inf")
    f[:, :, 4] = 17.0
    y, final, _ = _check(z, f, o, None, state, dy, dfinal, False, "f32")
    assert torch.equal(final[:, 1], state[:, 1]) and torch.equal(final[:, 3], state[:, 3])      # a = 1 exactly
    from tacotron2_amd import recurrence as R
    z2 = z.clone()
    z2[0, 100, 5], z2[1, 200, 6] = float("nan"), float("inf")
    y2, final2 = R.gated_scan(None, z2, f, o, state=state)
    assert torch.equal(y2[0, :100], y[0, :100]) and torch.isnan(y2[0, 100:, 5]).all() and torch.isnan(final2[0, 5])
    assert torch.isposinf(y2[1, 200, 6]) and torch.equal(y2[:, :, 7:], y[:, :, 7:]) and torch.equal(y2[1, :200], y[1, :200])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_strides_orders_and_alignment(dtype):
    from tacotron2_amd import recurrence as R
    B, T, H = 3, 150, 48
    z, f, o, state, dy, dfinal = _inputs(B, T, H, dtype, True, 21)
    want = R.gated_scan(None, z, f, o, state=state, tape=True)
    grads = R.gated_scan_backward(None, want[2], dy, dfinal)

    def same(zz, ff, oo, dd, out=None):
        y, final, tape = R.gated_scan(None, zz, ff, oo, state=state, tape=True, out=out)
        assert torch.equal(y, want[0]) and torch.equal(final, want[1])
        for got, exp in zip(R.gated_scan_backward(None, tape, dd, dfinal), grads):
            assert torch.equal(got, exp)

    packed = torch.cat([z, f, o], 2)                                             # one projection
    same(packed[..., :H], packed[..., H:2 * H], packed[..., 2 * H:], dy)
    flip = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731   time-major memory
    same(flip(z), flip(f), flip(o), flip(dy), out=torch.empty((T, B, H), dtype=z.dtype, device="cuda").transpose(0, 1))

    def odd(x):                                                                  # rows that start at any element
        buf = torch.zeros(B * T * (H + 1) + 1, dtype=x.dtype, device="cuda")
        v = buf[1:].view(B, T, H + 1)[..., :H]
        v.copy_(x)
        return v
    same(odd(z), odd(f), odd(o), odd(dy), out=odd(z))
    both = torch.full((B, T, 2 * H), 3.0, dtype=z.dtype, device="cuda")          # one half of a two-directional layer's output
    same(z, f, o, dy, out=both[..., H:])
    assert (both[..., :H] == 3).all()
    row = z[:1].expand(B, T, H)                                                  # broadcast inputs
    a, b = R.gated_scan(None, row, f, o), R.gated_scan(None, row.contiguous(), f, o)
    assert torch.equal(a[0], b[0])
    narrow = [x[..., :1].contiguous() for x in (z, f, o, dy)]
    _check(narrow[0], narrow[1], narrow[2], None, state[:, :1], narrow[3], dfinal[:, :1], False, dtype)


def test_gradients_against_differences():
    """Central differences of sum(c1 y) + sum(c2 final) in the 64-bit restatement, at a few places."""
    z, f, o, state, dy, dfinal = _inputs(2, 70, 5, "f32", True, 77)
    lens = np.array([70, 31])
    from tacotron2_amd import recurrence as R
    _, _, tape = R.gated_scan(None, z, f, o, lens=lens, state=state, reverse=True, tape=True)
    got = dict(zip(("z", "f", "o", "state"), R.gated_scan_backward(None, tape, dy, dfinal)))
    base = {"z": _np(z), "f": _np(f), "o": _np(o), "state": _np(state)}

    def loss(v):
        x = ref.forward(v["z"], v["f"], v["o"], lens, v["state"], True)
        return (x["y"] * _np(dy)).sum() + (x["final"] * _np(dfinal)).sum()
    rng = np.random.default_rng(0)
    for k in base:
        for _ in range(12):
            at = tuple(rng.integers(0, s) for s in base[k].shape)
            h = 1e-5
            up, down = dict(base), dict(base)
            up[k], down[k] = base[k].copy(), base[k].copy()
            up[k][at] += h
            down[k][at] -= h
            diff = (loss(up) - loss(down)) / (2 * h)
            # differences: h^2 / 6 of a third derivative of order 10, and 1e-15 / h of rounding of a loss of order 100; gradient: fp32
            assert abs(diff - float(got[k][at])) <= 2e-8 + 2e-5 * max(1.0, abs(diff)), (k, at)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("B,H", [(1, 1), (1, 1024), (3, 5), (64, 130), (7, 66)])
def test_step(B, H, dtype):
    from tacotron2_amd import recurrence as R
    for gate, idle in ((True, True), (False, False)):
        z, f, o, state, _, _ = _inputs(B, 1, H, dtype, gate, B * H)
        flat = [None if x is None else x[:, 0] for x in (z, f, o)]
        active = (torch.arange(B, device="cuda") % 3 != 1) if idle else None
        pool = torch.full((B, H + 3), 5.0, device="cuda")
        st = pool[:, 1:H + 1]
        st.copy_(state)
        y = R.gated_scan_step(None, *flat, st, active=active)
        x = ref.forward(_np(z), _np(f), _np(o), np.ones(B, int), _np(state), False)
        on = np.ones(B, bool) if active is None else active.cpu().numpy()
        _close(y, np.where(on[:, None], x["y"][:, 0], 0), x["ey"][:, 0], "y", dtype)
        _close(st, np.where(on[:, None], x["final"], _np(state)), x["efinal"], "state")
        assert (pool[:, 0] == 5).all() and (pool[:, H + 1:] == 5).all()


def test_steps_continue_a_sequence():
    """A prompt of 90 positions as one scan, ten more as steps: the same as one scan over 100 (fp32: reassociation only)."""
    from tacotron2_amd import recurrence as R
    z, f, o, state, _, _ = _inputs(4, 100, 72, "f32", True, 9)
    y, final = R.gated_scan(None, z, f, o, state=state)
    ya, st = R.gated_scan(None, z[:, :90], f[:, :90], o[:, :90], state=state)
    yb = [R.gated_scan_step(None, z[:, t], f[:, t], o[:, t], st) for t in range(90, 100)]
    x = ref.forward(_np(z), _np(f), _np(o), np.full(4, 100), _np(state), False)
    _close(torch.cat([ya, torch.stack(yb, 1)], 1), x["y"], x["ey"], "y", "f32")
    _close(st, x["final"], x["efinal"], "final")


def test_on_another_stream_and_with_a_context_of_its_own():
    from tacotron2_amd import recurrence as R
    from tacotron2_amd.engine import shared_context
    z, f, o, state, dy, dfinal = _inputs(2, 700, 130, "bf16", True, 4)
    _check(z, f, o, None, state, dy, dfinal, False, "bf16", ctx=shared_context(0))
    want = R.gated_scan(None, z, f, o, state=state)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append([R.gated_scan(None, z, f, o, state=state) for _ in range(4)])
    torch.cuda.synchronize()
    for runs in got:
        for y, final in runs:
            assert torch.equal(y, want[0]) and torch.equal(final, want[1])


def test_a_stream_context_is_ordered_against_other_streams():
    from tacotron2_amd import recurrence as R
    from tacotron2_amd.engine import stream_context
    z, f, o, state, _, _ = _inputs(2, 700, 130, "f32", True, 4)
    want = R.gated_scan(None, z, f, o, state=state)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ctx = stream_context()
    assert ctx.stream == side
    for _ in range(8):
        # what the call reads is written on this stream just before, what it wrote is read just behind
        z2 = z * 1.0
        y, final = R.gated_scan(ctx, z2, f, o, state=state)
        del z2
        assert torch.equal(y, want[0]) and torch.equal(final, want[1])
    ctx.close()
    with torch.cuda.stream(side):
        again = R.gated_scan(None, z, f, o, state=state)                   # a closed one is made anew
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again[0], want[0])


def test_in_place_and_in_parts_of_one_tensor():
    from tacotron2_amd import recurrence as R
    from tacotron2_amd._lib import T2Error
    z, f, o, state, _, _ = _inputs(3, 70, 66, "f32", True, 4)
    want, final = R.gated_scan(None, z, f, o, state=state)
    slab = torch.cat([z, f, o, torch.full_like(z, 7.0)], 2)
    parts = slab.split(66, 2)
    got, _ = R.gated_scan(None, *parts[:3], state=state, out=parts[3])
    assert torch.equal(got, want) and torch.equal(slab[:, :, :198], torch.cat([z, f, o], 2))
    for out in (parts[0], slab[:, :, 60:126]):
        with pytest.raises(T2Error):
            R.gated_scan(None, *parts[:3], state=state, out=out)
    s1, s2 = state.clone(), state.clone()
    a, b, c = (t[:, 0].contiguous() for t in (z, f, o))
    y = R.gated_scan_step(None, a, b, c, s1)
    assert R.gated_scan_step(None, a, b, c, s2, out=a) is a and torch.equal(a, y) and torch.equal(s1, s2)
    with pytest.raises(T2Error):
        R.gated_scan_step(None, a, b, c, s1, out=s1)


@pytest.mark.parametrize("T", [50, 1500])
def test_captured_calls_replay(T):
    """Two graphs captured one after the other, replayed in turn and side by side, with eager calls between."""
    from tacotron2_amd import recurrence as R
    made = []
    side = torch.cuda.Stream()
    for seed in (1, 2):
        z, f, o, state, dy, dfinal = _inputs(3, T, 96, "bf16", True, seed)
        lens = torch.tensor([T, T // 2, 0], device="cuda")

        def work(z=z, f=f, o=o, lens=lens, state=state, dy=dy, dfinal=dfinal):
            y, final, tape = R.gated_scan(None, z, f, o, lens=lens, state=state, tape=True)
            return (y, final) + R.gated_scan_backward(None, tape, dy, dfinal)
        with torch.cuda.stream(side):
            work()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = work()
        made.append((graph, outs, work, (z, f, o, lens, state, dy, dfinal)))
    other = torch.cuda.Stream()
    for turn in range(4):
        for graph, outs, work, data in made:
            data[0].add_(0.125)
            for t in outs:
                t.fill_(9)
        torch.cuda.synchronize()
        made[0][0].replay()
        with torch.cuda.stream(other):
            made[1][0].replay()
        torch.cuda.synchronize()
        for graph, outs, work, data in made:
            for got, want in zip(outs, work()):
                assert torch.equal(got, want), turn


def test_refusals():
    from tacotron2_amd import recurrence as R
    from tacotron2_amd.engine import shared_context
    z, f, o, state, dy, dfinal = _inputs(2, 9, 8, "f32", True, 1)
    bad = [
        lambda: R.gated_scan(None, z.cpu(), f), lambda: R.gated_scan(None, z, f.half()), lambda: R.gated_scan(None, z, f[:, :8]),
        lambda: R.gated_scan(None, z.double(), f.double()), lambda: R.gated_scan(None, z[0], f[0]), lambda: R.gated_scan(None, z[:, :0], f[:, :0]),
        lambda: R.gated_scan(None, z.transpose(1, 2).contiguous().transpose(1, 2), f), lambda: R.gated_scan(None, z, f, state=state.half()),
        lambda: R.gated_scan(None, z, f, state=state[:1]), lambda: R.gated_scan(None, z, f, lens=[1, 2, 3]), lambda: R.gated_scan(None, z, f, lens=[1.0, 2.0]),
        lambda: R.gated_scan(None, z, f, lens=torch.ones(2, device="cuda")), lambda: R.gated_scan(None, z, f, out=torch.empty_like(z[:1]).expand(2, 9, 8)),
        lambda: R.gated_scan(None, z, f, out=torch.empty((2, 9, 8), device="cuda", dtype=torch.float16)),
        lambda: R.gated_scan_step(None, z[:, 0], f[:, 0], None, state.half()), lambda: R.gated_scan_step(None, z[:, 0], f[:, 0], None, state[:1]),
        lambda: R.gated_scan_step(None, z[:, 0], f[:, 0], None, state, active=torch.ones(2, device="cuda")),
        lambda: R.gated_scan_step(None, z, f, None, state),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was accepted")
    _, _, tape = R.gated_scan(shared_context(0), z, f, o, tape=True)
    for call in (lambda: R.gated_scan_backward(None, tape, dy[:, :3]), lambda: R.gated_scan_backward(None, tape, dy, dfinal.half())):
        with pytest.raises(ValueError):
            call()
