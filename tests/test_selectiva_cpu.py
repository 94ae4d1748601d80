"""What the per-channel convolution and the selective scan refuse: by the wrappers before any device work, and by the C
entries."""
import os

import pytest
import torch

import asrn_amd
from asrn_amd import _lib

N = None


def t(*forma, dt=torch.float32):
    return torch.zeros(*forma, dtype=dt)


@pytest.mark.parametrize('args,que', [
    ((t(4, 8), t(8, 4)), 'axes'),
    ((t(2, 4, 8, dt=torch.float64), t(8, 4)), 'float64'),
    ((t(2, 4, 8), t(7, 4)), 'peso'),
    ((t(2, 4, 8), t(8, 17)), 'peso'),
    ((t(2, 4, 8), t(8, 0)), 'peso'),
    ((t(2, 4, 8), t(8, 2, 4)), 'peso'),
    ((t(2, 4, 8), t(8, 4), t(7)), 'sesgo'),
    ((t(2, 4, 8), t(8, 4, dt=torch.float64)), 'peso'),
    ((t(2, 4, 8), t(8, 4), t(8), 'relu'), 'activacion'),
    ((t(2, 4, 0), t(0, 4)), 'axes'),
])
def test_conv_canal_refuses(args, que):
    with pytest.raises(ValueError, match=que):
        asrn_amd.conv_canal(*args)


@pytest.mark.parametrize('args,que', [
    ((t(2, 8), t(2, 8, 2), t(8, 4)), 'ventana'),
    ((t(2, 8), t(2, 8, 3, dt=torch.bfloat16), t(8, 4)), 'ventana'),
    ((t(2, 8), t(2, 3, 8).transpose(1, 2), t(8, 4)), 'contiguous'),
    ((t(2, 1, 8), t(2, 8, 3), t(8, 4)), 'axes'),
])
def test_paso_conv_canal_refuses(args, que):
    with pytest.raises(ValueError, match=que):
        asrn_amd.paso_conv_canal(*args)


def base(**kw):
    e = dict(u=t(2, 5, 8), delta=t(2, 5, 8), A=t(8, 3), Bm=t(2, 5, 3), C=t(2, 5, 3))
    e.update(kw)
    return e


@pytest.mark.parametrize('kw,que', [
    (dict(delta=t(2, 5, 7)), 'delta'), (dict(delta=t(2, 5, 8, dt=torch.bfloat16)), 'delta'), (dict(A=t(7, 3)), 'A'),
    (dict(A=t(8, 33), Bm=t(2, 5, 33), C=t(2, 5, 33)), 'A'), (dict(A=t(8, 0)), 'A'), (dict(Bm=t(2, 5, 4)), 'Bm'),
    (dict(C=t(5, 3)), 'C'), (dict(D=t(3)), 'D'), (dict(puerta=t(2, 5, 3)), 'puerta'), (dict(sesgo_delta=t(2, 8)), 'sesgo_delta'),
    (dict(estado=t(2, 3, 8)), 'estado'), (dict(A=t(8, 3, dt=torch.float64)), 'A'), (dict(u=t(5, 8)), 'axes'),
    (dict(u=t(2, 5, 8, dt=torch.int32)), 'axes'),
])
def test_escaneo_selectivo_refuses(kw, que):
    with pytest.raises(ValueError, match=que):
        asrn_amd.escaneo_selectivo(**base(**kw))


@pytest.mark.parametrize('estado,que', [(t(2, 8, 4), 'estado'), (t(2, 8, 3, dt=torch.bfloat16), 'estado'),
                                        (t(2, 3, 8).transpose(1, 2), 'estado')])
def test_paso_selectivo_refuses(estado, que):
    with pytest.raises(ValueError, match=que):
        asrn_amd.paso_selectivo(t(2, 8), t(2, 8), t(8, 3), t(2, 3), t(2, 3), estado)


def test_cpu_tensors_are_refused():
    for f in (lambda: asrn_amd.conv_canal(t(2, 4, 8), t(8, 4)), lambda: asrn_amd.escaneo_selectivo(**base()),
              lambda: asrn_amd.paso_conv_canal(t(2, 8), t(2, 8, 3), t(8, 4)),
              lambda: asrn_amd.paso_selectivo(t(2, 8), t(2, 8), t(8, 3), t(2, 3), t(2, 3), t(2, 8, 3))):
        with pytest.raises(RuntimeError, match='GPU only'):
            f()


@pytest.fixture(scope='module')
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip('libasrn_hip.so not built (run `python -m asrn_amd.build`)')
    return _lib.load()


def test_entries_refuse(lib):
    def falla(rc, que):
        assert rc != 0 and que in lib.asrn_hip_last_error().decode()
    conv = lambda type=0, B=2, L=8, d=8, k=4, act=0: lib.asrn_channel_conv_fwd(N, type, L * d, d, N, N, B, L, d, k, act, N, N)
    falla(conv(type=3), 'type 3')
    falla(conv(k=17), 'k=17')
    falla(conv(act=3), 'act=3')
    falla(conv(d=0), 'd=0')
    falla(conv(), 'null')
    assert conv(B=0) == 0 and conv(L=0) == 0
    falla(lib.asrn_channel_conv_bwd(1, 0, 64, 8, 1, N, 1, 2, 8, 8, 4, 0, 1, 1, 16, 4, N), 'workspace')
    assert lib.asrn_channel_conv_bwd_workspace(2, 8, 8, 17) == -1
    falla(lib.asrn_channel_conv_step(N, 0, 8, N, N, N, N, 2, 8, 4, 0, N, N), 'null')
    sel = lambda type=0, B=2, L=8, d=8, n=4: lib.asrn_selective_fwd(*([N] * 5), type, N, *([N] * 4), B, L, d, n, 1, *([N] * 4), 0, N)
    falla(sel(type=7), 'type 7')
    falla(sel(n=33), 'N=33')
    falla(sel(n=0), 'N=0')
    falla(sel(B=1 << 16), 'too many')
    falla(sel(), 'null')
    assert sel(B=0) == 0 and sel(L=0) == 0
    # 5 waves of 64 channels are 2 workgroups of 3
    assert lib.asrn_selective_checks(2, 17, 300, 9) == 2 * 3 * 6 * 64 * 16 and lib.asrn_selective_checks(2, 0, 8, 4) == 0
    assert lib.asrn_selective_fwd_workspace(0, 5, 8, 4) == 0 and lib.asrn_selective_fwd_workspace(2, 5, 0, 4) == -1
    # 12 waves fill 1/170 of the card: a long text is cut, and its chunks' states need room
    assert lib.asrn_selective_fwd_workspace(1, 1 << 15, 768, 16) > 0


def test_blocks_and_configurations():
    from asrn_amd.modelo import ESTADOS, BloqueLocal
    b = BloqueLocal(40, 4, 80, mezcla='selectiva', memoria_max=64)
    assert b.conv.weight.shape == (40, 1, 4) and b.rango == 3 and b.decaimientos().shape == (40, ESTADOS)
    assert torch.allclose(b.decaimientos()[7], -torch.arange(1.0, ESTADOS + 1))
    pasos = torch.nn.functional.softplus(b.sel_dt.bias)
    assert torch.allclose(pasos[[0, -1]], torch.tensor([1.0, 1 / 64]), rtol=1e-4)
    with pytest.raises(ValueError, match='taps'):
        BloqueLocal(40, 17, 80, mezcla='selectiva')
    with pytest.raises(ValueError, match='k=17'):
        asrn_amd.ConfigASRN(V=10, k=17, mezcla='selectiva')
    c = asrn_amd.ConfigASRN(V=48, d=32, n_capas=10, mezcla='selectiva')
    m = asrn_amd.crear_desde_config(c, semilla=1)
    assert c.contar_parametros() == m.num_parametros() and asrn_amd.ConfigASRN.desde_modelo(m) == c.con(init_profundo=True)
    # the deep start shrinks what writes into the residual stream, and weight decay leaves the decays alone
    recto = asrn_amd.crear_desde_config(c.con(init_profundo=False), semilla=1)
    f = 20 ** -0.5
    for a, r in zip(m.bloques, recto.bloques):
        assert torch.allclose(a.sel_o.weight, f * r.sel_o.weight) and torch.equal(a.conv.weight, r.conv.weight)
    from asrn_amd.entrenamiento import grupos_optimizador
    for nombres, _, decae, _ in grupos_optimizador(m):
        assert not decae or not any(n.endswith(('sel_log_a', 'sel_d')) for n in nombres)
    # the other blocks' weights for a seed are what they were
    assert list(BloqueLocal(8, 4, 16).state_dict()) == ['ln1.weight', 'ln1.bias', 'conv.weight', 'conv.bias', 'ln2.weight', 'ln2.bias',
                                                        'ff.0.weight', 'ff.0.bias', 'ff.2.weight', 'ff.2.bias']


def test_entries_refuse_grids_past_the_launches(lib):
    """A launch has fewer than 2^32 threads."""
    def falla(rc):
        assert rc != 0 and 'too many' in lib.asrn_hip_last_error().decode(), lib.asrn_hip_last_error().decode()
    grande = (1 << 22, 1, 1025)                    # a lane a channel and text
    falla(lib.asrn_channel_conv_fwd(64, 0, 1025, 1025, 64, N, *grande, 4, 0, 64, N))
    wsb = lib.asrn_channel_conv_bwd_workspace(*grande, 4)
    falla(lib.asrn_channel_conv_bwd(64, 0, 1025, 1025, 64, N, 64, *grande, 4, 0, 64, 64, 64, wsb, N))
    falla(lib.asrn_channel_conv_step(64, 0, 1024, 64, 64, 64, N, 1 << 22, 1024, 4, 0, 64, N))
    falla(lib.asrn_linear_act_fwd(64, 1, 64, 1, 0, N, 1, 1 << 26, 1, 0, N, 0, 0, N, 0, 64, 1 << 26, 1, 0, N, 0, N))
    falla(lib.asrn_act_grad(64, (1 << 28) + 1, 1, 64, (1 << 28) + 1, 0, 1, (1 << 28) + 1, 1, 64, N, N, 0, N))     # 16 lanes of one column
