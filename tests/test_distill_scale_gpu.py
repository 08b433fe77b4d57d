"""Distillation where t / T is large: the probabilities depend on the list's differences alone.

Tolerances as in test_distill_gpu.py, with R the range of the student's row and of the teacher's list alike: an exponent's argument is
(t - max t) / T, off by three roundings of its own size, whatever the logits' common level and T."""
import pytest
import torch

from tests.test_distill_gpu import DEV, _exact, _make, _ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,V,K", [(3, 40, 5), (70, 900, 70), (9, 3000, 9), (5, 20000, 200), (2, 40000, 6)])
@pytest.mark.parametrize("level,T", [(30000.0, 0.7), (-5e6, 3.0), (40.0, 0.003), (0.0, 1e-4)])
def test_lists_far_from_zero_and_small_temperatures(B, V, K, level, T):
    ops = _ops()
    s, _, idx, top = _make(B, V, K, "f32", B + V, ragged=False)
    s, top = s * T, top * T + level   # differences of the size of T
    loss, d = ops.distill_topk(s.to(DEV), idx.to(DEV), top.to(DEV), temperature=T)
    t32 = torch.tensor(T, dtype=torch.float32).double().item()  # (the temperature is a 32-bit number)
    el, eg, mass = _exact(s, idx, top, t32, None, None, 1 / B)
    R = max((s.amax(1) - s.amin(1)).max().item(), (top.amax(1) - top.amin(1)).max().item()) / T
    C = (3 * min(88.0, R) + 70 + V / 64) * 2.0 ** -24
    assert abs(loss.item() - el.sum().item()) <= T * T * (4 * C + 64 * 2.0 ** -24) + el.sum().item() * (B * 2.0 ** -24 + 4 * C)
    p = torch.softmax(top.double() / t32, 1) * (t32 / B)
    part = eg.abs().scatter_add(1, idx, 2 * p)
    assert ((d.cpu().double() - eg).abs() <= part * 4 * C + 1e-37).all()
