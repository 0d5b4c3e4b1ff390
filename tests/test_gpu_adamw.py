"""AdamW over many tensors (training.AdamW) against adamw_ref.py: fp32 results within derived bounds, codes in 8 bits equal."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from tests import adamw_ref as ref

torch = pytest.importorskip("torch")
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HYPER = dict(learning_rate=1e-2, beta1=0.9, beta2=0.99, epsilon=1e-8)


def _np(t):
    return t.detach().double().cpu().numpy().reshape(-1)


def _tensors(sizes, dtypes, seed, scale=1.0, shift=0):
    """Separate tensors; `shift` starts each that many elements into its memory."""
    gen = torch.Generator().manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        dt = DTYPES[dtypes[i % len(dtypes)]]
        buf = torch.zeros(n + shift, dtype=dt, device="cuda")
        buf[shift:] = (torch.randn(n, generator=gen) * scale * 10.0 ** -(i % 4)).to(dt).cuda()
        out.append(buf[shift:])
    return out


def _off(got, want, bound, dt, what):
    tol = bound + (0 if dt is None else np.abs(want) * torch.finfo(dt).eps / 2 * 1.01 + (2.0 ** -25 if dt == torch.float16 else 0))
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:3].tolist(), float((np.abs(got - want) / tol).max()))


class Twin:
    """The restatement of an optimizer, one tensor after the other."""

    def __init__(self, opt, decay, lr, b1, b2, eps):
        self.o, self.decay, self.h, self.t = opt, decay, (lr, b1, b2, eps), 0

    def check(self, params, grads, clip=0.0, grad_scale=1.0, copies=None, **kw):
        """Runs a step of the optimizer on params and holds it to the restatement of the same step."""
        o, (lr, b1, b2, eps) = self.o, self.h
        before = [t.clone() if t is not None else None for t in (o.m, o.v, o.m_scale, o.v_scale)]
        p0 = [_np(p) for p in params]
        g0 = [_np(g) for g in grads]
        o.apply_gradients(grads, params, clip_norm=clip, grad_scale=grad_scale, copies=copies, **kw)
        self.t += 1
        assert o.steps() == self.t
        norm, gs = ref.factor(g0, clip, grad_scale)
        np.testing.assert_allclose(float(o.global_norm(grads, grad_scale)), norm, rtol=2e-7)
        raw = lambda t: t.view(torch.uint8).cpu().numpy()  # noqa: E731
        for i, (n, at) in enumerate(zip(o.sizes, o.offsets)):
            if o.state_bits == 32:
                m, v = _np(before[0][at:at + n]), _np(before[1][at:at + n])
            else:
                k = (n + 127) // 128
                cut = lambda t: raw(t)[at:at + 128 * k]  # noqa: E731
                cuts = lambda t: raw(t)[at // 128:at // 128 + k]  # noqa: E731
                g = np.zeros(128 * k, np.float32)
                g[:n] = g0[i]
                mc, ms, vc, vs, m, r = ref.step8(cut(before[0]), cuts(before[2]), cut(before[1]), cuts(before[3]), g, self.t, gs, b1, b2, o.seed, at)
                assert np.array_equal(cut(o.m), mc) and np.array_equal(cuts(o.m_scale), ms), i
                assert np.array_equal(cut(o.v), vc) and np.array_equal(cuts(o.v_scale), vs), i
                m, v = m[:n].astype(np.float64), r[:n].astype(np.float64) ** 2
            pn, mn, vn, ep, em, ev = ref.step64(p0[i], g0[i], m, v, self.t, gs, lr, b1, b2, eps, self.decay[i])
            _off(_np(params[i]), pn, ep, params[i].dtype, ("p", i))
            if copies is not None and copies[i] is not None:
                _off(_np(copies[i]), pn, ep, copies[i].dtype, ("copy", i))
            if o.state_bits == 32:
                _off(_np(o.m[at:at + n]), mn, em, None, ("m", i))
                _off(_np(o.v[at:at + n]), vn, ev, None, ("v", i))


def _make(sizes, bits, decay=None, seed=0, ctx=None, **kw):
    from tacotron2_amd.training import AdamW
    decay = [0.1 * (i % 3) for i in range(len(sizes))] if decay is None else decay
    h = {**HYPER, **kw}
    opt = AdamW(ctx, sizes, weight_decay=decay, state_bits=bits, seed=seed, **h)
    return opt, Twin(opt, decay, h["learning_rate"], h["beta1"], h["beta2"], h["epsilon"])


SIZES = [1, 7, 127, 128, 129, 2049, 8192, 8193, 20000, 3]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("pt,gt,ct", [(["f32"], ["f32"], None), (["f32"], ["bf16"], ["bf16", "f16"]), (["bf16"], ["bf16"], None), (["f16"], ["f16"], None),
                                      (["f32", "bf16", "f16"], ["f16", "f32"], ["f16"])])
def test_steps_of_mixed_tensors(bits, pt, gt, ct):
    params = _tensors(SIZES, pt, 1)
    copies = None if ct is None else _tensors(SIZES, ct, 9)
    if copies is not None:
        copies[2] = None
    opt, twin = _make(SIZES, bits, seed=77)
    for it in range(4):
        grads = _tensors(SIZES, gt, 100 + it, scale=[0.5, 1e-3, 2.0, 0.1][it])
        grads[8][5000:9000] = 0                                       # whole blocks without a gradient
        twin.check(params, grads, clip=[0.0, 1.0, 1.0, 0.5][it], grad_scale=[1.0, 1.0, 0.25, 2.0][it], copies=copies)
    opt.close()


@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_that_start_anywhere(bits):
    for shift, dt in ((1, "f32"), (1, "bf16"), (3, "f16"), (4, "bf16"), (4, "f32")):
        sizes = [130, 8195]
        params, grads, copies = _tensors(sizes, [dt], 3, shift=shift), _tensors(sizes, ["bf16"], 4, shift=shift), _tensors(sizes, ["f16"], 5, shift=1)
        opt, twin = _make(sizes, bits)
        twin.check(params, grads, clip=1.0, copies=copies)
        assert not params[0]._base[:shift].any() and not copies[1]._base[:1].any()
        opt.close()


@pytest.mark.parametrize("bits", [32, 8])
def test_hundreds_of_tensors(bits):
    sizes = [1 + (37 * i) % 400 for i in range(300)]
    params = _tensors(sizes, ["f32", "bf16"], 6)
    opt, twin = _make(sizes, bits)
    for it in range(2):
        twin.check(params, _tensors(sizes, ["f32"], 50 + it), clip=1.0)
    opt.close()


@pytest.mark.parametrize("bits", [32, 8])
def test_extreme_gradients(bits):
    """Zeros, the smallest and very large values; nothing moves where everything is zero and there is no decay."""
    sizes = [384, 128]
    params = _tensors(sizes, ["f32"], 7)
    opt, twin = _make(sizes, bits, decay=[0.0, 0.5])
    g = torch.zeros(384, device="cuda")
    g[:3] = torch.tensor([1e-30, -1e-20, 1e15])
    g[128:256] = 3e-38
    p0 = params[0].clone()
    for _ in range(3):
        twin.check(params, [g, torch.zeros(128, device="cuda")])
    assert torch.equal(params[0][256:], p0[256:])
    opt.close()


def test_not_finite_gradients():
    from tacotron2_amd.training import AdamW
    for bits in (32, 8):
        for bad in (float("inf"), float("nan")):
            params, grads = _tensors([300, 200], ["f32"], 1), _tensors([300, 200], ["f32"], 2)
            opt = AdamW(None, [300, 200], state_bits=bits, learning_rate=1e-2)
            opt.apply_gradients(grads, params)
            keep = [p.clone() for p in params] + list(opt.state())
            grads[0][150] = bad
            opt.apply_gradients(grads, params, skip_nonfinite=True)
            opt.apply_gradients(grads, params, clip_norm=0.0, skip_nonfinite=True)
            for a, b in zip(params + list(opt.state()), keep):
                assert a is None and b is None or (a == b if isinstance(a, int) else torch.equal(a.view(torch.uint8), b.view(torch.uint8)))
            opt.apply_gradients(grads, params, clip_norm=0.0)                  # without the check: only where it is
            assert opt.steps() == 2
            nan = torch.isnan(params[0])
            assert nan[150] and int(nan.sum()) == 1 and not torch.isnan(params[1]).any()
            grads[0][150] = 0.0
            opt.apply_gradients(grads, params, clip_norm=0.0)
            nan = torch.isnan(params[0])
            assert nan[150] and int(nan.sum()) == (1 if bits == 32 else 128) and not torch.isnan(params[1]).any()
            opt.close()


def test_stochastic_rounding_lets_the_second_moment_decay():
    """400 steps without gradients: every root shrinks by sqrt(0.999), far less than half a code.  A step's rounding has a variance of at
    most 0.0005 / 8 (relative), so a mean over 8192 elements is within 6 sigma = 0.011 of the decay."""
    from tacotron2_amd.training import AdamW
    n = 8192
    opt = AdamW(None, n, weight_decay=0.0, state_bits=8, seed=5)
    g = torch.rand(n, device="cuda") + 0.5
    p, z = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    opt.apply_gradients(g, p)
    root = lambda: opt.v.float().view(-1, 128) * opt.v_scale.float()[:, None]  # noqa: E731
    before = root()
    bound = opt.bind(z, p)
    for _ in range(400):
        opt.apply_gradients(bound)
    ratio = float((root() / before).mean())
    assert abs(ratio - 0.999 ** 200) < 0.011, ratio
    opt.close()


@pytest.mark.parametrize("bits", [32, 8])
def test_state_round_trip_and_other_streams(bits):
    from tacotron2_amd.engine import shared_context
    sizes = [1000, 130]
    params = _tensors(sizes, ["f32"], 1)
    a, twin = _make(sizes, bits, seed=3, ctx=shared_context(0))            # a stream of its own
    for it in range(2):
        twin.check(params, _tensors(sizes, ["f32"], 20 + it), clip=1.0)
    b, _ = _make(sizes, bits, seed=3)
    b.load_state(*a.state())
    pb = [p.clone() for p in params]
    g = _tensors(sizes, ["f32"], 30)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        for _ in range(3):
            b.apply_gradients(g, pb)
    for _ in range(3):
        a.apply_gradients(g, params)
    torch.cuda.synchronize()
    for x, y in zip(params + [a.m, a.v], pb + [b.m, b.v]):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    for o in (a, b):
        o.close()


def test_a_binding_used_on_another_stream_and_dropped_at_once():
    opt, _ = _make([3000, 40], 32, seed=3)
    params = _tensors([3000, 40], ["f32"], 1)
    g = _tensors([3000, 40], ["f32"], 2)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(4):
        b = opt.bind(g, params)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(2000000)
            opt.apply_gradients(b, clip_norm=1.0)
        at = b.table.data_ptr()
        n = b.table.numel()
        del b
        # the side stream is not done with the table: its memory is not anyone else's yet
        new = torch.empty(n, dtype=torch.uint8, device="cuda")
        assert side.query() or new.data_ptr() != at
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
    assert opt.steps() == 4
    opt.close()


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step(bits):
    """Replays count and match an eager twin, with eager steps and a learning rate on the device in between; tensors given to a captured
    call stay those of the capture whatever is bound later."""
    sizes = [3000, 9000, 5]
    lr = torch.tensor([1e-2], device="cuda")
    p1 = _tensors(sizes, ["f32"], 1)
    p2 = [p.clone() for p in p1]
    g = _tensors(sizes, ["bf16"], 2)
    other_g, other_p = _tensors(sizes, ["f32"], 3), _tensors(sizes, ["f32"], 4)
    other_p2 = [p.clone() for p in other_p]
    a, _ = _make(sizes, bits, learning_rate=lr)
    b, _ = _make(sizes, bits, learning_rate=lr)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        a.apply_gradients(g, p1)
    torch.cuda.synchronize()
    b.apply_gradients(g, p2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.apply_gradients(g, p1)
    for turn in range(4):
        for t in g:
            t.mul_(-0.75)
        lr.mul_(0.5)
        graph.replay()
        b.apply_gradients(g, p2)
        a.apply_gradients(other_g, other_p)
        b.apply_gradients(other_g, other_p2)
        torch.cuda.synchronize()
        assert a.steps() == b.steps() == 3 + 2 * turn
        for x, y in zip(p1 + other_p + [a.m, a.v], p2 + other_p2 + [b.m, b.v]):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), turn
    for o in (a, b):
        o.close()


def test_a_tensor_of_more_than_32_bits():
    """4.3 G elements with states in 8 bits: blocks at the start, around 2^31 and 2^32 and at the end are held to the restatement."""
    from tacotron2_amd.training import AdamW
    n = 2 ** 32 + 700
    opt = AdamW(None, n, learning_rate=1e-2, beta2=0.99, weight_decay=0.1, state_bits=8, seed=9)
    p, g = (torch.zeros(n, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    places = [0, 2 ** 31 - 256, 2 ** 32 - 256, 2 ** 32 + 128]
    gen = torch.Generator(device="cuda").manual_seed(1)
    for at in places:
        for t in (p, g):
            t[at:at + 512] = torch.randn(512, generator=gen, device="cuda").to(torch.bfloat16)
    raw = lambda t: t.view(torch.uint8).cpu().numpy()  # noqa: E731
    for step in (1, 2):
        before = [(raw(opt.m[at:at + 512]), raw(opt.m_scale[at // 128:at // 128 + 4]), raw(opt.v[at:at + 512]), raw(opt.v_scale[at // 128:at // 128 + 4]),
                   _np(p[at:at + 512])) for at in places]
        opt.apply_gradients(g, p, clip_norm=0.0)
        for at, (m8, ms, v8, vs, p0) in zip(places, before):
            gn = _np(g[at:at + 512])
            mc, ms, vc, vs, m, r = ref.step8(m8, ms, v8, vs, gn.astype(np.float32), step, 1.0, 0.9, 0.99, 9, at)
            assert np.array_equal(raw(opt.m[at:at + 512]), mc) and np.array_equal(raw(opt.v[at:at + 512]), vc), (step, at)
            assert np.array_equal(raw(opt.m_scale[at // 128:at // 128 + 4]), ms) and np.array_equal(raw(opt.v_scale[at // 128:at // 128 + 4]), vs), (step, at)
            pn, _, _, ep, _, _ = ref.step64(p0, gn, m.astype(np.float64), r.astype(np.float64) ** 2, step, 1.0, 1e-2, 0.9, 0.99, 1e-8, 0.1)
            _off(_np(p[at:at + 512]), pn, ep, torch.bfloat16, (step, at))
    assert not p[n - 60:].any() and not p[1000:100000].any()
    opt.close()


def test_refusals():
    from tacotron2_amd._lib import T2Error
    from tacotron2_amd.training import AdamW
    for kw in ({"sizes": 0}, {"sizes": []}, {"sizes": [4, -1]}, {"beta1": 1.0}, {"epsilon": 0.0}, {"state_bits": 16}, {"weight_decay": -1.0}):
        with pytest.raises(T2Error):
            AdamW(None, **{"sizes": [4], **kw})
    with pytest.raises(ValueError):
        AdamW(None, [4, 4], weight_decay=[0.1])
    opt = AdamW(None, [4, 6])
    t = lambda n, dt=torch.float32: torch.zeros(n, dtype=dt, device="cuda")  # noqa: E731
    good = ([t(4), t(6)], [t(4), t(6)])
    shared = t(8)
    for bad in ((good[0][:1], good[1]), ([t(4), t(5)], good[1]), ([t(4), torch.zeros(6)], good[1]), ([t(4), t(6, torch.float64)], good[1]),
                ([t(4), t(12)[::2]], good[1]), (good[0], [shared[:4], shared[2:8]]), (good[0], [good[0][0], t(6)]), (good[0], None)):
        with pytest.raises(ValueError):
            opt.apply_gradients(*bad)
    with pytest.raises(ValueError):
        opt.apply_gradients(opt.bind(good[0]))                              # no parameters
    with pytest.raises(ValueError):
        opt.apply_gradients(opt.bind(*good), good[1])
    with pytest.raises(ValueError):
        opt.bind(good[0], copies=good[1])
    with pytest.raises(ValueError):
        opt.load_state(opt.m, opt.v[:5], 0)
    with pytest.raises(ValueError):
        opt.load_state(opt.m, opt.v, -1)
    # a table bound for the norm alone cannot reach a parameter even through the C entry
    from tacotron2_amd import _lib
    from tacotron2_amd.engine import stream_context
    b, c = opt.bind(good[0]), stream_context(0)
    _lib.check(c.lib.t2_adamw_step(c.handle, opt._h, b.table.data_ptr(), 1e-3, None, 1.0, 1.0, 0))
    torch.cuda.synchronize()
    opt.close()


def test_trainer_takes_adamw():
    """Trainer.train_step with AdamW in AdamOptimizer's place: kernels are decayed, biases, norms and moving statistics are not."""
    from tacotron2_amd import training as TR
    from tacotron2_amd.engine import Engine
    from tacotron2_amd.hparams import PROFILE_TINY as d
    from tacotron2_amd.weights import init_weights
    w = init_weights(d, 3, perturb=True)
    rng = np.random.default_rng(0)
    B, T, S = 3, 8, 4
    r = d.outputs_per_step
    labels = {"mel": rng.uniform(0, 1, (B, S * r, d.num_mels)).astype(np.float32), "done": np.eye(S, dtype=np.float32)[[S - 1] * B],
              "spec_loss_mask": np.ones((B, S * r), np.float32), "binary_loss_mask": np.ones((B, S), np.float32)}
    feats = {"source": rng.integers(0, d.num_symbols, (B, T)), "source_length": np.array([T, T - 2, T], np.int64)}
    eng = Engine(d, w)
    spec = TR.flatten_spec(w)
    tr = TR.Trainer(eng, B, T, S)
    tr.bind_gradients(spec)
    flat = torch.tensor(TR.flatten(w, spec), device="cuda")
    grads = torch.zeros_like(flat)
    opt = TR.AdamW(eng, spec, learning_rate=1e-2, beta2=0.99, weight_decay=0.5)
    before = TR.unflatten(flat, spec)
    step, losses = tr.train_step(opt, flat, grads, feats, labels, global_step=0, seed=1)
    assert step == 1 and bool(torch.isfinite(losses).all())
    after, g = TR.unflatten(flat, spec), TR.unflatten(grads, spec)
    _, gs = ref.factor(list(g.values()), 1.0, 1.0)
    for name, shape, _, _ in spec:
        if "moving_" in name:
            continue
        z = np.zeros(g[name].size)
        pn, _, _, ep, _, _ = ref.step64(before[name].astype(np.float64).reshape(-1), g[name].astype(np.float64).reshape(-1), z, z, 1, gs, 1e-2, 0.9, 0.99,
                                        1e-8, 0.5 if len(shape) >= 2 else 0.0)
        _off(after[name].astype(np.float64).reshape(-1), pn, ep, torch.float32, name)
    for o in (tr, eng):
        o.close()
    opt.close()
