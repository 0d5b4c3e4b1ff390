"""Calls of the gated linear recurrence at the edge of what its documentation allows."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from tests.test_gpu_recurrence import _check, _inputs

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("T", [200, 1500])
def test_a_state_that_lies_in_the_output(T):
    """Chunks through one buffer: the state in front is the last row of the chunk before, which y replaces."""
    from tacotron2_amd import recurrence as R
    from tacotron2_amd._lib import T2Error
    z, f, _, state, _, _ = _inputs(1, T, 96, "f32", False, 3)
    out = torch.empty_like(z)
    for turn in range(3):
        want, final = R.gated_scan(None, z, f, state=state if turn == 0 else want[:, -1].clone())
        got, last = R.gated_scan(None, z, f, state=state if turn == 0 else out[:, -1], out=out)
        assert got is out and torch.equal(out, want) and torch.equal(last, final)
    lens = out.view(torch.int64).view(-1)[:1]
    with pytest.raises(T2Error):
        R.gated_scan(None, z, f, lens=lens, out=out)


@pytest.mark.parametrize("dtype,B,T,H,gate,reverse", [("f32", 2, 700, 36, True, False), ("bf16", 3, 1500, 130, True, True), ("f16", 1, 2300, 3, False, True),
                                                      ("f32", 1, 5000, 66, False, False), ("bf16", 8, 12300, 512, True, True)])
def test_a_tile_that_does_not_wait_gets_the_same_bits(dtype, B, T, H, gate, reverse):
    """scan_wait_us 0: every tile computes what enters it from the inputs of the tiles before it; 1: some do."""
    from tacotron2_amd import recurrence as R
    from tacotron2_amd.engine import Context
    gen = torch.Generator(device="cuda").manual_seed(T)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    dt = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[dtype]
    z, f, dy = r(B, T, H).to(dt), (r(B, T, H) * 1.5 + 4).to(dt), r(B, T, H).to(dt)
    o = r(B, T, H).to(dt) if gate else None
    state, dfinal = r(B, H), r(B, H)
    ctx = Context(0)
    for lens in (None, torch.tensor([T - 301 * b for b in range(B)], device="cuda").clamp(min=0)):
        got = []
        for us in (2_000_000, 0, 1):
            ctx.set_option("scan_wait_us", us)
            y, final, tape = R.gated_scan(ctx, z, f, o, lens=lens, state=state, reverse=reverse, tape=True)
            dz, df, do, dstate = R.gated_scan_backward(ctx, tape, dy, dfinal)
            got.append([y, final, tape.states if lens is None else final, dz, df, dz if do is None else do, dstate])
        for other in got[1:]:
            for a, b in zip(got[0], other):
                assert torch.isfinite(a).all() and torch.equal(a, b)
    ctx.close()


@pytest.mark.parametrize("dtype,B,T,H", [("f32", 2, 60, 12), ("bf16", 2, 200, 12), ("f32", 2, 1500, 12), ("f16", 3, 700, 3), ("f32", 9, 250, 2048)])
@pytest.mark.parametrize("reverse", [False, True])
def test_an_infinity_stays_one(dtype, B, T, H, reverse):
    """Behind an infinite value or state h is infinite for good, however small the product of the gates since then has become; the
    gradients likewise behind an infinite gradient.  Channels without one are what they were."""
    z, f, o, state, dy, dfinal = _inputs(B, T, H, dtype, True, T)
    f[..., 0] = -20.0                                                     # a product of four of these gates is below 2^-115
    plain = _check(z, f, o, None, state, dy, dfinal, reverse, dtype)
    inf = float("inf")
    z[0, T // 3, 0], z[1, T // 2, 1], state[0, 1], state[1, 2] = inf, -inf, inf, -inf
    _, final, _ = _check(z, f, o, None, state, dy, dfinal, reverse, dtype)
    assert final[0, 0] == inf and final[1, 1] == -inf and final[0, 1] == inf and final[1, 2] == -inf
    from tacotron2_amd.engine import Context
    ctx = Context(0)
    ctx.set_option("scan_wait_us", 0)
    _check(z, f, o, None, state, dy, dfinal, reverse, dtype, ctx=ctx)
    z, f, o, state, dy, dfinal = _inputs(B, T, H, dtype, True, T)
    f[..., 0] = -20.0
    dy[0, T // 3, 0], dy[1, T // 2, 1], dfinal[0, 1], dfinal[1, 2] = inf, -inf, inf, -inf
    y, final, (dz, df, do, dstate) = _check(z, f, o, None, state, dy, dfinal, reverse, dtype)
    assert dstate[0, 0] == inf and dstate[1, 1] == -inf and dstate[0, 1] == inf and dstate[1, 2] == -inf
    _check(z, f, o, None, state, dy, dfinal, reverse, dtype, ctx=ctx)
    ctx.close()
    assert torch.equal(y, plain[0]) and torch.equal(final, plain[1])
    for got, want in zip((dz, df, do), plain[2]):
        assert torch.equal(got[..., 3:], want[..., 3:])


def test_an_infinity_stays_one_in_large_calls():
    """The same across the wide tiles of a large call."""
    from tacotron2_amd import recurrence as R
    B, T, H = 8, 12300, 512
    gen = torch.Generator(device="cuda").manual_seed(5)
    r = lambda *s: torch.randn(s, generator=gen, device="cuda")  # noqa: E731
    z, f, dy, dfinal = r(B, T, H).bfloat16(), (r(B, T, H) - 1).bfloat16(), r(B, T, H).bfloat16(), r(B, H)
    inf = float("inf")
    z[1, 5000, 130], dfinal[2, 300] = inf, -inf
    y, final, tape = R.gated_scan(None, z, f, tape=True)
    dz, _, _, dstate = R.gated_scan_backward(None, tape, dy, dfinal)
    assert (y[1, 5000:, 130] == inf).all() and final[1, 130] == inf and (dz[2, :, 300] == -inf).all() and dstate[2, 300] == -inf
    assert int(torch.isfinite(y).logical_not().sum()) == T - 5000 and int(torch.isfinite(dz).logical_not().sum()) == T


@pytest.mark.parametrize("lens", [None, [2000, 3]])
def test_a_tape_used_on_another_stream_and_dropped_at_once(lens):
    from tacotron2_amd import recurrence as R
    z, f, o, state, dy, dfinal = _inputs(2, 2000, 300, "f32", True, 6)
    _, _, tape = R.gated_scan(None, z, f, o, lens=lens, state=state, tape=True)
    want = R.gated_scan_backward(None, tape, dy, dfinal)
    del tape
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(4):
        _, _, tape = R.gated_scan(None, z, f, o, lens=lens, state=state, tape=True)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
            got = R.gated_scan_backward(None, tape, dy, dfinal)
        made = [tape.states] + ([] if tape.lens is None else [tape.lens])
        at, sizes = [t.data_ptr() for t in made], [t.numel() * t.element_size() for t in made]
        del tape, made
        # the side stream is not done with the states and the lengths: their memory is not anyone else's yet
        new = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for n in sizes]
        assert side.query() or not {t.data_ptr() for t in new} & set(at)
        torch.cuda.current_stream().wait_stream(side)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
            a.record_stream(torch.cuda.current_stream())


def test_lengths_on_the_host_do_not_wait_for_the_stream():
    from tacotron2_amd import recurrence as R
    z, f, o, state, dy, dfinal = _inputs(3, 300, 40, "f32", True, 2)
    want = R.gated_scan(None, z, f, o, lens=torch.tensor([300, 17, 0], device="cuda"), state=state)
    for lens in ([300, 17, 0], np.array([300, 17, 0], np.int32), torch.tensor([300, 17, 0])):
        got = R.gated_scan(None, z, f, o, lens=lens, state=state)             # also: memory and code are there before the wait below
        torch.cuda.synchronize()
        torch.cuda._sleep(400_000_000)
        busy = torch.cuda.Event()
        busy.record()
        got = R.gated_scan(None, z, f, o, lens=lens, state=state)
        assert not busy.query(), "the call waited for what was queued before it"
        if isinstance(lens, np.ndarray):
            lens[:] = 1                                                        # the call has taken its lengths
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_lengths_on_the_host_are_refused_in_a_capture():
    from tacotron2_amd import recurrence as R
    z, f, o, state, _, _ = _inputs(2, 30, 40, "f32", True, 2)
    want = R.gated_scan(None, z, f, o, lens=[30, 17], state=state)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(ValueError):
            R.gated_scan(None, z, f, o, lens=[30, 17], state=state)
        got = R.gated_scan(None, z, f, o, lens=None, state=state)
    graph.replay()                                           # the refusal left the capture whole
    torch.cuda.synchronize()
    assert torch.equal(got[0][0], want[0][0]) and torch.equal(got[1], R.gated_scan(None, z, f, o, state=state)[1])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T", [1, 2, 7, 140, 700])
def test_gradients_that_cancel(dtype, T):
    """dfinal next to -dy of the last step: what is left is as exact as the steps one after the other have it."""
    z, f, _, state, dy, dfinal = _inputs(5, T, 140, dtype, False, T)
    f[:, :-1] += 6.0                                                       # long memories: it reaches the first step
    for reverse in (False, True):
        last = dy[:, 0 if reverse else -1].float()
        dfinal = -last * (1 + 2.0 ** -12 * torch.rand(5, 140, generator=torch.Generator().manual_seed(T)).cuda())
        _check(z, f, None, None, state, dy, dfinal, reverse, dtype)
