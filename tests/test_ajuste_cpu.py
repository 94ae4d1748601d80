"""The fine-tuning entry points' argument checks, which fail before any device work, and the public names."""
import os
import subprocess
import sys

import pytest
import torch

import asrn_amd
from asrn_amd import _lib
from asrn_amd import ops
from asrn_amd.lineal import lineal8

N = None


@pytest.fixture(scope='module')
def lib():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip('libasrn_hip.so not built (run `python -m asrn_amd.build`)')
    return _lib.load()


def _mal(lib, rc, texto):
    assert rc != 0 and texto in lib.asrn_hip_last_error().decode(), lib.asrn_hip_last_error().decode()


def test_token_logp_checks(lib):
    f = lambda *a: lib.asrn_token_logp_fwd(N, *a, N, -100, 1.0, N, N, N, N)
    _mal(lib, f(3, 4, 2, 10, 20, 10), 'type=3')
    _mal(lib, f(0, 5, 2, 10, 20, 10), 'bad sizes')          # rows that are no multiple of L
    _mal(lib, f(0, 4, 2, 0, 20, 10), 'bad sizes')
    _mal(lib, f(0, 4, 2, 10, -20, 10), 'bad sizes')
    _mal(lib, f(0, 1 << 31, 1, 10, 20, 10), 'bad sizes')
    _mal(lib, f(0, 1 << 26, 1, 10, 20, 10), 'too many rows')
    _mal(lib, f(1, 1 << 24, 1, 5000, 5000, 5000), 'too many rows')
    _mal(lib, f(0, 4, 2, 10, 20, 10), 'null pointer')
    assert f(0, 0, 2, 10, 20, 10) == 0                      # no rows: no launch
    _mal(lib, lib.asrn_token_logp_fwd(N, 0, 4, 2, 10, 20, 10, N, -100, 0.0, N, N, N, N), 'temperature')
    _mal(lib, lib.asrn_token_logp_bwd(N, 1, 4, 2, 10, 20, 10, N, -100, 1.0, N, N, N, 16, N, N), 'entropy')
    _mal(lib, lib.asrn_token_logp_bwd(N, 1, 4, 2, 10, 20, 10, N, -100, 1.0, N, N, 16, N, N, N), 'null pointer')


def test_preference_checks(lib):
    f = lambda P, L, kind, beta, e, margin, ws=0: lib.asrn_preference_fwd(16, 16, N, N, 0, N, N, P, L, kind, beta, e, margin, 0,
                                                                          16, 16, 16, 16, ws, N)
    _mal(lib, f(0, 5, 0, 0.1, 0.0, 0.0), 'bad sizes')
    _mal(lib, f(1 << 30, 5, 0, 0.1, 0.0, 0.0), 'bad sizes')
    _mal(lib, f(1, 5, 3, 0.1, 0.0, 0.0), 'kind=3')
    _mal(lib, f(1, 5, 0, 0.0, 0.0, 0.0), 'beta')
    _mal(lib, f(1, 5, 0, 0.1, 1.5, 0.0), 'smoothing')
    _mal(lib, f(1, 5, 0, 0.1, 0.0, float('nan')), 'margin')
    _mal(lib, f(2, 5000, 0, 0.1, 0.0, 0.0, 4 * 3 * 16 - 1), 'workspace')
    assert lib.asrn_preference_workspace(2, 5000) == 4 * 3 * 16 and lib.asrn_preference_workspace(0, 5) == -1
    _mal(lib, lib.asrn_preference_bwd(N, N, N, N, 1, 5, N, N), 'null pointer')
    assert lib.asrn_preference_bwd(N, N, N, N, 1, 0, N, N) == 0


def test_policy_checks(lib):
    f = lambda B, L, lo, hi, cap, beta, w, ws=0: lib.asrn_policy_fwd(16, 16, N, N, N, N, 16, B, L, lo, hi, cap, beta, w, 0, 16, 16,
                                                                     16, 16, 16, ws, N)
    _mal(lib, f(0, 5, 0.2, 0.2, 0.0, 0.0, 0.0), 'bad sizes')
    _mal(lib, f(1, 5, 1.2, 0.2, 0.0, 0.0, 0.0), 'clip_low')
    _mal(lib, f(1, 5, 0.2, -0.2, 0.0, 0.0, 0.0), 'clip_high')
    _mal(lib, f(1, 5, 0.2, 0.2, 0.5, 0.0, 0.0), 'cap')
    _mal(lib, f(1, 5, 0.2, 0.2, 0.0, -1.0, 0.0), 'beta')
    _mal(lib, f(1, 5, 0.2, 0.2, 0.0, 0.0, float('inf')), 'entropy_weight')
    _mal(lib, f(3, 2049, 0.2, 0.2, 0.0, 0.0, 0.0, 3 * 2 * 48 - 1), 'workspace')
    assert lib.asrn_policy_workspace(3, 2049) == 3 * 2 * 48 and lib.asrn_policy_workspace(1, -1) == -1
    _mal(lib, lib.asrn_policy_bwd(N, N, N, N, N, 1, 5, 0.0, 16, N, N), 'null pointer')
    assert lib.asrn_policy_bwd(N, N, N, N, N, 1, 5, 0.0, N, N, N) == 0


def test_eight_bit_checks(lib):
    _mal(lib, lib.asrn_pack8(16, 0, 4, 0, 16, 16, N), 'bad sizes')
    _mal(lib, lib.asrn_pack8(16, 0, 1 << 30, 1 << 20, 16, 16, N), 'bad sizes')
    _mal(lib, lib.asrn_pack8(16, 0, 4, 32, N, 16, N), 'null pointer')
    _mal(lib, lib.asrn_unpack8(16, 16, -1, 32, 0, 0, 16, N), 'bad sizes')
    _mal(lib, lib.asrn_gelu8_fwd(16, 1, N, 4, 32, N, 16, 16, N), 'null pointer')
    _mal(lib, lib.asrn_gelu8_bwd(16, 16, N, 1, 4, 32, 1, 16, N), 'null pointer')
    _mal(lib, lib.asrn_norm8_fwd(16, 16, 16, 4, 30, 1e-5, 0, 16, 16, 16, 16, N), 'multiple of 4')
    _mal(lib, lib.asrn_norm8_fwd(16, 16, 16, 4, 8196, 1e-5, 0, 16, 16, 16, 16, N), 'multiple of 4')
    _mal(lib, lib.asrn_norm8_fwd(16, 16, 16, 4, 32, 0.0, 0, 16, 16, 16, 16, N), 'eps')
    _mal(lib, lib.asrn_norm8_fwd(24, 16, 16, 4, 32, 1e-5, 0, 16, 16, 16, 16, N), 'aligned')
    need = lib.asrn_norm8_bwd_workspace(100, 64)
    assert need >= 4 * 2 * 64 * 4 and lib.asrn_norm8_bwd_workspace(-1, 64) == -1 and lib.asrn_norm8_bwd_workspace(1, 8196) == -1
    _mal(lib, lib.asrn_norm8_bwd(16, 16, 16, 16, 100, 64, 16, 0, N, 16, 16, 256, need - 1, N), 'workspace')
    _mal(lib, lib.asrn_norm8_read(16, 16, 16, 16, 16, 2, 5, 64, 17, 0, 16, N), 'k=17')
    _mal(lib, lib.asrn_norm8_read(16, 16, 16, 16, 16, 2, 5, 62, 4, 0, 16, N), 'multiple of 4')
    for rc in (lib.asrn_pack8(N, 0, 0, 32, N, N, N), lib.asrn_unpack8(N, N, 0, 32, 0, 0, N, N), lib.asrn_gelu8_fwd(N, 0, N, 0, 32, N, N, N, N),
               lib.asrn_gelu8_bwd(N, N, N, 0, 0, 32, 0, N, N), lib.asrn_norm8_fwd(N, N, N, 0, 32, 1e-5, 0, N, N, N, N, N),
               lib.asrn_norm8_read(N, N, N, N, N, 0, 5, 64, 4, 0, N, N)):
        assert rc == 0                                      # no rows: no launch


def test_public_names_refuse_cpu_tensors():
    lp = torch.zeros(2, 3)
    for f in (lambda: asrn_amd.token_log_probs(torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.long)),
              lambda: asrn_amd.preference_loss(lp), lambda: asrn_amd.policy_loss(lp, lp)):
        with pytest.raises(RuntimeError, match='GPU only'):
            f()


def test_window_reads_only_what_norma8_kept():
    """The columns of a window have rows of another width than the ones kept: reading them as norma8's would leave their
    buffers."""
    leer = lambda ts, dt: pytest.fail('read')
    t = (torch.zeros(1), torch.zeros(4), torch.zeros(4))
    z = torch.zeros(2, 5, 12)
    for guardado in (ops.Guardado8(leer, t, (10, 12)), ops.Guardado8(leer, t[:1], (10, 12)),
                     ops.Guardado8(leer, t, (10, 4), norma=True)):
        with pytest.raises(ValueError, match='did not keep'):
            ops.ventana8(z, 3, torch.float32, guardado)


def test_what_was_kept_on_another_device_is_refused():
    """The weight gradient reads the product's gradient and the kept rows in one kernel: they must be on one device."""
    leer = lambda ts, dt: pytest.fail('read')
    t = tuple(torch.zeros(4, device='meta') for _ in range(3))
    x, w = torch.zeros(2, 5, 4), torch.zeros(3, 4, requires_grad=True)
    with pytest.raises(ValueError, match='kept on meta'):
        lineal8(x, w, None, ops.Guardado8(leer, t, (10, 4)))
    with pytest.raises(ValueError, match='kept on meta'):
        ops.ventana8(x, 3, torch.float32, ops.Guardado8(leer, t, (10, 4), norma=True))


def test_graph_memsets_without_a_graph(lib):
    assert lib.asrn_graph_memsets(N) == -1 and 'no graph' in lib.asrn_hip_last_error().decode()


def test_one_stream_can_be_switched_off():
    m = asrn_amd.crear_modelo(61, 64, 2, semilla=1).train()
    x = torch.zeros(1, 8, dtype=torch.long)
    E = m.emb(x)
    assert m._una_corriente(E, x)
    m.permite_una_corriente = False
    assert not m._una_corriente(E, x)


def test_extras_are_values():
    """An extra that carries a graph: its values are copied, nothing flows back through it and no step keeps its graph."""
    torch.manual_seed(2)
    fuente = torch.nn.Parameter(torch.randn(2, 7))
    m = torch.nn.Sequential(torch.nn.Embedding(11, 8), torch.nn.Linear(8, 11))
    opt = torch.optim.SGD(m.parameters(), lr=0.1)
    perdida = lambda logits, y, ref: ((torch.log_softmax(logits, -1).gather(-1, y[..., None])[..., 0] - ref) ** 2).mean()
    paso = asrn_amd.PasoGrafado(m, opt, 2, 7, precision='fp32', grabar=False, perdida=perdida, extras=(fuente * 2,))
    x = torch.randint(0, 11, (2, 8))
    for i in range(3):
        extra = fuente * (i + 1)
        antes = [p.detach().clone() for p in m.parameters()]
        valor, _, salto = paso(x[:, :-1], x[:, 1:], lr=0.1, extras=(extra,))
        e = paso.extras[0]
        assert not e.requires_grad and e.grad_fn is None and torch.equal(e, extra) and fuente.grad is None
        assert salto == 0 and any(not torch.equal(a, b) for a, b in zip(antes, m.parameters()))


def test_preference_reference_sums_check(lib):
    for filas in (-1, 3):
        _mal(lib, lib.asrn_preference_fwd(16, 16, 16, 16, filas, N, N, 1, 5, 0, 0.1, 0.0, 0.0, 0, 16, 16, 16, 16, 0, N), 'ref_rows')


def test_import_without_a_gpu_build_of_torch():
    """A CPU build of PyTorch has no streams; the package is still imported there (file formats, the model on the CPU)."""
    prog = ("import torch\n"
            "for n in [n for n in dir(torch._C) if 'RawStream' in n]: delattr(torch._C, n)\n"
            "import asrn_amd\n"
            "print(asrn_amd.crear_modelo(11, 64, 2, semilla=1).num_parametros())")
    raiz = os.path.dirname(os.path.dirname(os.path.abspath(asrn_amd.__file__)))
    r = subprocess.run([sys.executable, '-c', prog], cwd=raiz, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and int(r.stdout) > 0, r.stderr


def _compilador(ruta, rc):
    """A stand-in for a compiler: writes the file after -o and ends with rc."""
    ruta.write_text(f'#!{sys.executable}\nimport sys\na = sys.argv\nopen(a[a.index("-o") + 1], "w").write(a[-1])\nsys.exit({rc})\n')
    ruta.chmod(0o755)
    return str(ruta)


@pytest.mark.parametrize('falla', ['no', 'nodos', 'sin_cxx', 'hipcc'])
def test_build_places_the_library_without_the_nodes(tmp_path, monkeypatch, falla):
    """The C ABI needs hipcc alone: nodes that do not compile are reported after the library is in its place."""
    from asrn_amd import build
    cc = _compilador(tmp_path / 'cc', int(falla == 'hipcc'))
    monkeypatch.setattr(build, 'hipcc', lambda: cc)
    monkeypatch.setenv('CXX', str(tmp_path / 'none') if falla == 'sin_cxx' else _compilador(tmp_path / 'cxx', int(falla == 'nodos')))
    monkeypatch.setattr(build, 'LIB', str(tmp_path / 'lib.so'))
    monkeypatch.setattr(build, 'NODOS', str(tmp_path / 'nodos.so'))
    if falla in ('nodos', 'sin_cxx'):
        (tmp_path / 'nodos.so').write_text('of an earlier build')
    if falla == 'no':
        assert build.build() == build.LIB
    else:
        with pytest.raises(RuntimeError, match='hipcc failed' if falla == 'hipcc' else 'autograd nodes are not'):
            build.build()
    assert os.path.exists(build.LIB) == (falla != 'hipcc') and os.path.exists(build.NODOS) == (falla == 'no')
