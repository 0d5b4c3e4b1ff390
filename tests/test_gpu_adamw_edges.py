"""AdamW with the smallest and largest factors, scales and tables that its documentation allows."""
import pytest

pytestmark = pytest.mark.gpu

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
