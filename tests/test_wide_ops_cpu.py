"""The distillation loss and the embedding ops: what their C entries and wrappers refuse (no kernel runs here)."""
import pytest
import torch

from celligner2_amd import ops
from celligner2_amd._lib import C2Error, lib

P = 4096  # never followed


def test_cpu_tensors_are_refused():
    z, i = torch.zeros(2, 4), torch.zeros(2, 1, dtype=torch.int64)
    for f in (lambda: ops.distill_topk(z, i, z[:, :1]), lambda: ops.embed_fwd(z, i[:, 0]), lambda: ops.embed_grad(z, i[:, 0], 3)):
        with pytest.raises(C2Error, match="MI355X"):
            f()


def test_distill_entry_refuses():
    def call(s=P, dt=0, ldl=50, idx=P, ib=8, ldi=3, top=P, ldt=3, K=3, T=1.0, B=4, V=50, loss=P, d=P + 64, ddt=0, lddl=50, ws=P):
        return lib.c2_distill_topk_fwd_bwd(s, dt, ldl, idx, ib, ldi, top, ldt, K, None, None, T, B, V, 1.0, loss, 1, d, ddt, lddl, ws,
                                           None, None)
    for bad in (dict(dt=3), dict(ddt=4), dict(ib=2), dict(T=0.0), dict(T=-1.0), dict(T=float("inf")), dict(T=float("nan")), dict(T=1e-39), dict(T=2e19),
                dict(K=1025, ldi=1025, ldt=1025), dict(K=-1), dict(B=-1), dict(V=1 << 31), dict(s=None), dict(loss=None),
                dict(ws=None), dict(ldl=49), dict(lddl=49), dict(idx=None), dict(top=None), dict(ldi=2), dict(ldt=2),
                dict(d=P, ddt=1), dict(d=P, lddl=60)):
        assert call(**bad) != 0, bad
        assert lib.c2_last_error()
    assert call(B=0) == 0 and call(V=0) == 0


def test_embed_entries_refuse():
    def fwd(t=P, dt=1, ldt=8, V=5, D=8, ids=P, ib=8, N=3, o=P, odt=1, ldo=8):
        return lib.c2_embed_fwd(t, dt, ldt, V, D, ids, ib, N, 1.0, o, odt, ldo, None, None)
    for bad in (dict(dt=3), dict(odt=4), dict(ib=1), dict(V=-1), dict(N=-1), dict(t=None), dict(ids=None), dict(o=None), dict(ldt=7),
                dict(ldo=7)):
        assert fwd(**bad) != 0, bad
    assert fwd(N=0) == 0 and fwd(D=0) == 0

    def grad(d=P, dt=0, ldd=8, ids=P, ib=4, N=3, V=5, D=8, o=P, ldt=8, ws=P):
        return lib.c2_embed_grad(d, dt, ldd, ids, ib, N, V, D, 1.0, o, ldt, 0, ws, None, None)
    for bad in (dict(dt=3), dict(ib=1), dict(V=-1), dict(N=1 << 31), dict(N=(1 << 26) + 1), dict(V=(1 << 27) + 1),
                dict(D=(1 << 23) + 1, ldd=1 << 24, ldt=1 << 24), dict(N=200, ws=None), dict(N=200, ws=P + 4), dict(d=None), dict(ids=None), dict(o=None), dict(ldd=7), dict(ldt=7)):
        assert grad(**bad) != 0, bad
    assert grad(V=0) == 0 and grad(D=0) == 0


@pytest.mark.parametrize("T", [1e-19, 1e-20, 1e-23, 3e-39, 4e-39])
def test_temperatures_whose_square_is_not_a_normal_number_are_refused(T):
    """T^2 scales the loss: at 1e-20 it keeps a few bits, at 1e-23 it is zero; at 3e-39 log2(e) / T is infinite."""
    rc = lib.c2_distill_topk_fwd_bwd(P, 0, 50, P, 8, 3, P, 3, 3, None, None, T, 4, 50, 1.0, P, 1, P + 64, 0, 50, P, None, None)
    assert rc != 0 and b"temperature" in lib.c2_last_error()


@pytest.mark.parametrize("scale", [float("inf"), float("-inf"), float("nan")])
def test_gradient_scales_that_are_not_finite_are_refused(scale):
    """A row without a token is zero, not 0 * scale."""
    assert lib.c2_embed_grad(P, 0, 8, P, 4, 3, 5, 8, scale, P, 8, 0, P, None, None) != 0 and b"finite" in lib.c2_last_error()
