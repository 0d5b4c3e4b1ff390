"""AdamW with the smallest and largest factors, scales and tables that its documentation allows."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

from tests import adamw_ref as ref
from tests.test_gpu_adamw import _make, _tensors

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("bits", [32, 8])
def test_an_infinite_limit_does_not_clip(bits):
    from tacotron2_amd._lib import T2Error
    sizes = [3000, 40]
    a, twin = _make(sizes, bits, seed=3)
    b, _ = _make(sizes, bits, seed=3)
    params = _tensors(sizes, ["f32"], 1)
    other = [p.clone() for p in params]
    inf, nan = float("inf"), float("nan")
    for it in range(2):
        grads = _tensors(sizes, ["f32"], 10 + it, scale=100.0)
        twin.check(params, grads, clip=0.0, grad_scale=0.5)
        b.apply_gradients(grads, other, clip_norm=inf, grad_scale=0.5)
        for x, y in zip(params + [a.m, a.v], other + [b.m, b.v]):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    # factors that are no numbers are refused, and nothing has moved
    for kw in ({"clip_norm": nan}, {"grad_scale": nan}, {"grad_scale": inf}, {"grad_scale": 1e39}):
        with pytest.raises(T2Error):
            b.apply_gradients(grads, other, **kw)
    for lr in (nan, inf, -1e39):
        b.learning_rate = lr
        with pytest.raises(T2Error):
            b.apply_gradients(grads, other)
    with pytest.raises(T2Error):
        b.global_norm(grads, grad_scale=nan)
    assert b.steps() == 2
    for x, y in zip(params, other):
        assert torch.equal(x, y)
    for o in (a, b):
        o.close()


@pytest.mark.parametrize("bits", [32, 8])
def test_elements_without_a_gradient_stay_with_the_smallest_epsilon(bits):
    eps = float(np.finfo(np.float32).tiny)
    opt, _ = _make([300], bits, decay=[0.0], epsilon=eps)
    p = _tensors([300], ["f32"], 1)
    g = torch.zeros(300, device="cuda")
    g[:128] = torch.randn(128, generator=torch.Generator().manual_seed(2)).cuda()
    before = p[0].clone()
    for _ in range(2):
        opt.apply_gradients([g], p, clip_norm=0.0)
    assert torch.isfinite(p[0]).all() and torch.equal(p[0][128:], before[128:]) and not torch.equal(p[0][:128], before[:128])
    opt.close()


def test_roots_of_subnormal_second_moments():
    """Gradients of 1e-21 to 1e-17: v is subnormal or next to it, and with an epsilon of 1e-30 the root of v alone is the divisor.  The
    state is the formula's in fp32, bit for bit; from there the update passes lr_t, m, two products, a root and a reciprocal of one ulp
    each, a product and a sum: less than 12 roundings."""
    n = 4096
    lr, b1, b2, eps = 1e-2, 0.9, 0.99, 1e-30
    opt, _ = _make([n], 32, decay=[0.0], epsilon=eps)
    rng = np.random.default_rng(4)
    x = (rng.choice([-1.0, 1.0], n) * 10.0 ** rng.uniform(-21, -17, n)).astype(np.float32)
    g, p = torch.from_numpy(x).cuda(), torch.zeros(n, device="cuda")
    opt.apply_gradients([g], [p], clip_norm=0.0)
    with np.errstate(under="ignore"):
        v = (x * x) * np.float32(1 - b2)
    assert np.array_equal(opt.v[:n].cpu().numpy(), v)
    want = -(lr / (1 - b1)) * ((1 - b1) * x.astype(np.float64)) / (np.sqrt(v.astype(np.float64)) / np.sqrt(1 - b2) + eps)
    off = np.abs(p.double().cpu().numpy() - want)
    assert (off <= 12 * 2.0 ** -24 * np.abs(want)).all(), float((off / np.abs(want)).max())
    opt.close()


def test_the_smallest_scale_of_loaded_states():
    """A scale byte of 0 is 2^-127, as every other one is 2^(byte - 127)."""
    opt, _ = _make([512], 8, decay=[0.0], seed=11)
    rng = np.random.default_rng(7)
    codes = rng.integers(0, 0x7F, 512).astype(np.uint8) | (rng.integers(0, 2, 512).astype(np.uint8) << 7)
    roots = rng.integers(0, 0x7F, 512).astype(np.uint8)
    ms, vs = np.array([0, 1, 0, 20], np.uint8), np.array([0, 0, 90, 1], np.uint8)
    dev = lambda a, dt: torch.from_numpy(a).cuda().view(dt)  # noqa: E731
    opt.load_state(dev(codes, torch.float8_e4m3fn), dev(roots, torch.float8_e4m3fn), 4, m_scale=dev(ms, torch.float8_e8m0fnu), v_scale=dev(vs, torch.float8_e8m0fnu))
    p, g = torch.zeros(512, device="cuda"), torch.zeros(512, device="cuda")
    opt.apply_gradients([g], [p], clip_norm=0.0)
    raw = lambda t: t.view(torch.uint8).cpu().numpy()  # noqa: E731
    mc, msn, vc, vsn, _, _ = ref.step8(codes, ms, roots, vs, np.zeros(512, np.float32), 5, 1.0, 0.9, 0.99, opt.seed, 0)
    assert mc[:128].any() and np.array_equal(raw(opt.m), mc) and np.array_equal(raw(opt.m_scale), msn)
    assert np.array_equal(raw(opt.v), vc) and np.array_equal(raw(opt.v_scale), vsn)
    opt.close()
