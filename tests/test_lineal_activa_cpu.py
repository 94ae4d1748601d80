"""What the product with its epilogue refuses: by the wrapper before any device work, and by the C entries."""
import os

import pytest
import torch

import asrn_amd
from asrn_amd import _lib


def t(*forma, dt=torch.float32):
    return torch.zeros(*forma, dtype=dt)


@pytest.mark.parametrize('args,que', [
    ((t(3, 4), t(5, 3)), 'chain'), ((t(3, 4), t(5, 4), t(4)), 'chain'), ((t(3, 4), t(4)), 'chain'), ((t(3, 0), t(5, 0)), 'chain'),
    ((t(3, 4), t(5, 4), t(5), 'relu'), 'activacion'), ((t(3, 4), t(5, 4), t(5), None, t(3, 4)), 'residuo'),
    ((t(3, 4), t(5, 4), t(5), None, t(5)), 'residuo'), ((t(3, 4), t(5, 4), t(5), None, t(3, 5, dt=torch.bfloat16)), 'residuo'),
    ((t(3, 4, dt=torch.float64), t(5, 4, dt=torch.float64)), 'float64'), ((t(3, 4), t(5, 4, dt=torch.bfloat16)), 'bfloat16'),
    ((t(3, 4, dt=torch.bfloat16), t(5, 4, dt=torch.bfloat16), t(5)), 'b of'),
])
def test_refusals(args, que):
    with pytest.raises(ValueError, match=que):
        asrn_amd.lineal_activa(*args)


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match='GPU only'):
        asrn_amd.lineal_activa(t(3, 4), t(5, 4))


def test_entries_refuse():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip('libasrn_hip.so not built (run `python -m asrn_amd.build`)')
    lib = _lib.load()

    def falla(rc, que):
        assert rc != 0 and que in lib.asrn_hip_last_error().decode(), lib.asrn_hip_last_error().decode()

    def fwd(x=64, ldx=8, ldw=8, type=0, M=20, N=8, K=8, act=0, ldy=8, tile=0, ws=None, wsb=0):
        return lib.asrn_linear_act_fwd(x, ldx, 64, ldw, type, None, M, N, K, act, None, 0, 0, None, 0, 64, ldy, 1, tile, ws, wsb, None)
    falla(fwd(type=3), 'type 3')
    falla(fwd(K=0), 'K=0')
    falla(fwd(act=5), 'act=5')
    falla(fwd(x=None), 'null')
    falla(fwd(ldx=7), 'leading')
    falla(fwd(ldy=4), 'leading')
    falla(fwd(ldw=1 << 21), '2^21')
    falla(fwd(tile=7), 'unknown tile 7')
    falla(fwd(M=64, N=64, K=4096, ldx=4096, ldw=4096, ldy=64), 'workspace')
    assert fwd(M=0) == 0 and fwd(N=0) == 0
    assert lib.asrn_linear_act_workspace(64, 64, 4096, 0) > 0 and lib.asrn_linear_act_workspace(64, 64, 4096, 1) == 0
    assert lib.asrn_linear_act_workspace(64, 64, 0, 1) == -1 and lib.asrn_act_grad_workspace(-1, 4) == -1
    falla(lib.asrn_act_grad(64, 8, 1, None, 0, 1, 4, 8, 1, 64, None, None, 0, None), 'null')
    falla(lib.asrn_act_grad(64, 8, 1, 64, 8, 1, 4, 8, 1, 64, 64, None, 0, None), 'workspace')
    falla(lib.asrn_act_grad(64, 4, 1, 64, 8, 1, 4, 8, 1, 64, None, None, 0, None), 'leading')


def test_weight_gradient_refuses():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip('libasrn_hip.so not built (run `python -m asrn_amd.build`)')
    lib = _lib.load()

    def falla(que, g=64, ldg=16, x=64, ldx=16, type=1, M=64, N=16, K=16, out=64, tile=0, slabs=0, ws=None, wsb=0):
        rc = lib.asrn_weight_grad(g, ldg, x, ldx, type, M, N, K, out, 1, tile, slabs, ws, wsb, None)
        assert rc != 0 and que in lib.asrn_hip_last_error().decode(), lib.asrn_hip_last_error().decode()
    falla('type 0', type=0)
    falla('multiples of 8', N=12)
    falla('multiples of 8', K=1 << 21, ldx=1 << 21)
    falla('unknown tile', tile=64)
    falla('unknown tile', slabs=-1)
    falla('null', x=None)
    falla('leading', ldg=8)
    falla('leading', ldx=20)
    falla('misaligned', g=72)
    falla('workspace', M=4096, slabs=4)
    assert lib.asrn_weight_grad(64, 16, 64, 16, 1, 0, 16, 16, 64, 1, 0, 0, None, 0, None) == 0
    assert lib.asrn_weight_grad_workspace(4096, 16, 16, 0, 4) == 4 * 16 * 16 * 4
    assert lib.asrn_weight_grad_workspace(64, 12, 16, 0, 0) == -1 and lib.asrn_weight_grad_workspace(64, 16, 16, 3, 0) == -1
