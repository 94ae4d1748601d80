"""ModeloASRN's 'selectiva' blocks: the block against its formula in 64 bits, the model trained eagerly and from a graph,
written step by step and as a whole text, stored and loaded; and 'memoria' blocks on the per-channel convolution's kernel."""
import copy

import pytest
import torch
import torch.nn.functional as F

import asrn_amd
from asrn_amd import synth
from asrn_amd.modelo import ESTADOS, BloqueLocal, conv_canal_causal

pytestmark = pytest.mark.gpu
DEV = 'cuda'
U = 2.0 ** -24
REDUCIDA = dict(n_tablas=2, tablas_contexto=1, n_bits=6, afin_oculto=16, confirmar=4, vistos=2, nodos_racha=4)


@pytest.fixture(autouse=True)
def semilla():
    torch.manual_seed(0)


def bloque64(b, h):
    """The block's formula in float64."""
    p = {n: t.double() for n, t in b.named_parameters()}
    h = h.double()
    B, L, d = h.shape
    z = F.layer_norm(h, (d,), p['ln1.weight'], p['ln1.bias'], b.ln1.eps)
    c = F.silu(F.conv1d(F.pad(z.transpose(1, 2), (b.k - 1, 0)), p['conv.weight'], p['conv.bias'], groups=d).transpose(1, 2))
    dt, Bm, C = (c @ p['sel_x.weight'].t()).split((b.rango, ESTADOS, ESTADOS), -1)
    dt = F.softplus(dt @ p['sel_dt.weight'].t() + p['sel_dt.bias'], threshold=1e9)
    A = -p['sel_log_a'].exp().view(d, ESTADOS)
    s, ys = h.new_zeros(B, d, ESTADOS), []
    for t in range(L):
        s = s * torch.exp(dt[:, t, :, None] * A) + (dt[:, t] * c[:, t])[..., None] * Bm[:, t, None]
        ys.append((s * C[:, t, None]).sum(-1))
    y = (torch.stack(ys, 1) + p['sel_d'] * c) * F.silu(z @ p['sel_g.weight'].t() + p['sel_g.bias'])
    h = h + y @ p['sel_o.weight'].t()
    y = F.layer_norm(h, (d,), p['ln2.weight'], p['ln2.bias'], b.ln2.eps)
    u = y @ p['ff.0.weight'].t() + p['ff.0.bias']
    return h + (u * 0.5 * torch.erfc(-u / 2 ** 0.5)) @ p['ff.2.weight'].t() + p['ff.2.bias'], s


def bloque(d, k=4, ff=None, **kw):
    b = BloqueLocal(d, k, ff or 2 * d, mezcla='selectiva', memoria_max=64, **kw).to(DEV)
    with torch.no_grad():
        for n, p in b.named_parameters():       # away from the values they start at
            if 'ln' in n or n in ('sel_d',) or n.endswith('bias') and 'sel_dt' not in n:
                p.add_(0.2 * torch.randn_like(p))
    return b


@pytest.mark.parametrize('B,L,d,k', [(2, 33, 32, 4), (1, 1, 64, 2), (3, 150, 48, 1), (2, 70, 50, 4)])
def test_block_is_its_formula(B, L, d, k):
    """Roundings along the block, each of fp32: LayerNorms 40, convolution k + 12, products K + 24 (d, the rank, d, 2 d), the scan
    4 L + 64; every one reaches the output through slopes of a few, taken as 8, and the gradients through as many again."""
    b = bloque(d, k)
    h, gy = torch.randn(B, L, d, device=DEV).requires_grad_(), torch.randn(B, L, d, device=DEV)
    y = b(h)
    n = 2 * 40 + k + 12 + 5 * 24 + 6 * d + 4 * L + 64
    ps = [p for _, p in b.named_parameters()]
    gs = torch.autograd.grad(y, [h, *ps], gy)
    h64 = h.detach().double().requires_grad_()
    b64 = copy.deepcopy(b).double()
    yr, fin = bloque64(b64, h64)
    gr = torch.autograd.grad(yr, [h64, *b64.parameters()], gy.double())
    assert (y.double() - yr).abs().max() <= 8 * n * U * yr.abs().max()
    for (nombre, _), a, v in zip([('h', h), *b.named_parameters()], gs, gr):
        assert (a.double() - v).norm() <= 64 * n * U * v.norm() + 64 * n * U * gy.norm(), nombre
    with torch.no_grad():
        assert torch.equal(b(h), y)
        y2, (z, s) = b.adelante_selectiva(h, devolver_estado=True)
        assert torch.equal(y2, y) and (s.double() - fin).abs().max() <= 8 * n * U * fin.abs().max() and z.shape == h.shape


@pytest.mark.parametrize('dt', [torch.bfloat16, torch.float16])
def test_block_under_autocast(dt):
    """16-bit products: about a dozen roundings of the type on the way, each through slopes of a few."""
    b = bloque(64)
    h = torch.randn(2, 60, 64, device=DEV).requires_grad_()
    gy = torch.randn(2, 60, 64, device=DEV)
    with torch.autocast('cuda', dtype=dt):
        y = b(h)
    assert y.dtype == torch.float32
    gs = torch.autograd.grad(y, [h, *b.parameters()], gy)
    assert all(g.dtype == torch.float32 and torch.isfinite(g).all() for g in gs)
    h64 = h.detach().double().requires_grad_()
    b64 = copy.deepcopy(b).double()
    yr, _ = bloque64(b64, h64)
    gr = torch.autograd.grad(yr, [h64, *b64.parameters()], gy.double())
    e = 12 * 4 * torch.finfo(dt).eps / 2
    assert (y.double() - yr).norm() <= e * yr.norm()
    total = torch.stack([v.norm() for v in gr]).norm()
    for (nombre, _), a, v in zip([('h', h), *b.named_parameters()], gs, gr):
        assert (a.double() - v).norm() <= 2 * e * (v.norm() + 0.05 * total), nombre


def test_dropout_and_replaced_activations():
    b = bloque(32, dropout=0.5)
    h = torch.randn(2, 20, 32, device=DEV)
    entera = b.eval()(h)
    torch.manual_seed(3)
    y1 = b.train()(h)
    torch.manual_seed(3)
    assert torch.equal(y1, b(h)) and not torch.equal(y1, entera)
    b.eval()
    b.ff[1] = torch.nn.GELU()
    assert torch.equal(b(h), entera)
    b.ff[1] = torch.nn.ReLU()
    y = b(h)
    assert not torch.equal(y, entera)
    vistos = []
    b.ff[1].register_forward_hook(lambda m, a, o: vistos.append(o.shape))
    assert torch.equal(b(h), y) and len(vistos) == 1


def _modelo(B, L, **kw):
    m = asrn_amd.crear_modelo(97, 64, n_capas=2, semilla=3, mezcla='selectiva', memoria_max=64, **REDUCIDA, **kw).to(DEV)
    w = synth.tokens(3 * B, L + 1, 97, seed=4).to(DEV)
    return m, [(w[B * i:B * (i + 1), :-1].contiguous(), w[B * i:B * (i + 1), 1:].contiguous()) for i in range(3)]


@pytest.mark.parametrize('precision', ['fp32', 'bf16'])
def test_graphed_training_step_is_an_ordinary_one(precision):
    B, L = 3, 120
    m, lotes = _modelo(B, L)
    m.train()
    m2 = copy.deepcopy(m)
    opt = asrn_amd.crear_optimizador(m, lr=0.0, capturable=True)
    paso = asrn_amd.PasoGrafado(m, opt, B, L, precision=precision, calentar=2)
    for i in range(6):
        x, y = lotes[i % 3]
        perdida, _, salto = paso(x, y, lr=0.0)
        torch.cuda.synchronize()
        got = [p.grad.clone() for p in m.parameters()]
        with torch.autocast('cuda', torch.bfloat16, enabled=precision == 'bf16'):
            logits = m2(x)
        ref_perdida = asrn_amd.ops.cross_entropy(logits, y)
        ref = torch.autograd.grad(ref_perdida, list(m2.parameters()))
        assert salto.item() == 0 and abs(perdida.item() - ref_perdida.item()) <= 1e-5
        norma = torch.stack([g.norm() for g in ref]).norm().item()
        factor = min(1.0, 1.0 / (norma + 1e-6))
        for (n, _), a, b in zip(m.named_parameters(), got, ref):
            assert (a - factor * b).norm().item() <= 1e-5 * (factor * b).norm().item() + 1e-7 * min(norma, 1.0), (i, n)


@pytest.mark.parametrize('checkpoint', ['asrn', 'todo', 'ocho'])
def test_memory_modes_give_the_same_step(checkpoint):
    m, lotes = _modelo(2, 90)
    m.train()
    x, y = lotes[0]
    ref = torch.autograd.grad(m.perdida(x, y), list(m.parameters()))
    m.checkpoint = checkpoint
    got = torch.autograd.grad(m.perdida(x, y), list(m.parameters()))
    for (n, _), a, b in zip(m.named_parameters(), got, ref):
        assert (a - b).norm() <= 1e-5 * b.norm() + 1e-9, n


def test_training_runs_and_its_weights_move(monkeypatch):
    for b in (torch.backends.cuda.matmul, torch.backends.cudnn):      # entrenar allows what other tests' products must not have
        monkeypatch.setattr(b, 'allow_tf32', b.allow_tf32)
    m, lotes = _modelo(2, 64)
    antes = {n: p.detach().clone() for n, p in m.named_parameters()}
    piezas = torch.randint(0, 97, (3000,))
    asrn_amd.entrenar(m, piezas, largo=64, lote=4, pasos=3, precision='bf16')
    for n, p in m.named_parameters():
        assert torch.isfinite(p).all() and ('sel_' not in n or not torch.equal(p, antes[n])), n


@pytest.mark.parametrize('k', [1, 4])
def test_written_step_by_step_is_the_whole_text(k):
    m = asrn_amd.crear_modelo(60, d=32, n_capas=3, largo_cada=1, semilla=1, chunk=8, n_bits=3, mezcla='selectiva', memoria_max=64,
                              k=k).to(DEV).eval()
    x0 = synth.tokens(2, 40, 60, seed=0).to(DEV)
    for grafo in (True, False):
        sec, pasos = asrn_amd.escribir(m, x0, n_nuevos=60, memoria_de_lo_ajeno=False, top_k=0, grafo=grafo)
        with torch.no_grad():
            entero = m(sec[:, :-1].to(DEV))[:, 40 - 1:].cpu()
        assert sec.shape == (2, 100) and (entero - pasos).abs().max().item() < 1e-4


def test_written_from_a_graph_and_eagerly():
    m, lotes = _modelo(2, 50)
    a, la = asrn_amd.escribir(m, lotes[0][0], n_nuevos=30, top_k=5, semilla=3, grafo=True)
    b, lb = asrn_amd.escribir(m, lotes[0][0], n_nuevos=30, top_k=5, semilla=3, grafo=False)
    assert torch.equal(a, b) and torch.equal(la, lb)


def test_stored_and_loaded(tmp_path):
    m, lotes = _modelo(1, 30)
    m.eval()
    asrn_amd.guardar(m, tmp_path / 'm.pt')
    m2 = asrn_amd.cargar(tmp_path / 'm.pt')
    with torch.no_grad():
        assert m2.config == m.config and torch.equal(m(lotes[0][0]), m2(lotes[0][0]))


@pytest.mark.parametrize('k,dt', [(4, torch.float32), (3, torch.bfloat16), (1, torch.float32), (17, torch.float32),
                                  (4, torch.float64)])
def test_per_channel_convolution_of_memoria_blocks(k, dt):
    """conv_canal_causal keeps its result where the kernel takes it and where it does not (17 taps, 64 bits)."""
    z, w, b = torch.randn(2, 50, 24, device=DEV).to(dt), torch.randn(24, 1, k, device=DEV).to(dt), torch.randn(24, device=DEV).to(dt)
    y = conv_canal_causal(z, w, b)
    v = F.pad(z.double(), (0, 0, k - 1, 0)).unfold(1, k, 1)
    ref, m = (v * w.double()[:, 0]).sum(-1) + b.double(), (v * w.double()[:, 0]).abs().sum(-1) + b.double().abs()
    assert y.dtype == dt
    assert ((y.double() - ref).abs() <= (k + 2) * min(U, torch.finfo(dt).eps) * m + torch.finfo(dt).eps / 2 * (ref.abs() + 1e-6)).all()


@pytest.mark.parametrize('como', ['subclase', 'ejemplar'])
def test_block_with_its_own_feed_forward(como):
    """A block whose feed-forward was replaced runs it, over a text and for a token."""
    b, vistas = bloque(32), []

    def propia(y):
        vistas.append(y.shape)
        return torch.tanh(y) / 2
    h = torch.randn(2, 9, 32, device=DEV)
    sin = copy.deepcopy(b)                          # the same block without a feed-forward
    with torch.no_grad():
        sin.ff[2].weight.zero_()
        sin.ff[2].bias.zero_()
        medio = sin(h)
        if como == 'subclase':
            b.__class__ = type('Otro', (BloqueLocal,), {'_ff': lambda s, y: propia(y)})
        else:
            b._ff = propia
        y = b(h)
        assert (y - medio - torch.tanh(b.ln2(medio)) / 2).abs().max() <= 1e-5 and vistas == [h.shape]
        z, s = b.adelante_selectiva(h[:, :-1], devolver_estado=True)[1]
        ventana = F.pad(z, (0, 0, b.k - 1, 0))[:, z.shape[1]:].transpose(1, 2).contiguous()
        paso = b.paso_selectiva(h[:, -1].contiguous(), ventana, s, b.decaimientos())
    assert (paso - y[:, -1]).abs().max() <= 1e-4 and vistas[-1] == (2, 32)


def test_block_with_an_activation_in_place():
    """An activation that changes what it is given, in the GELU's place, trains as the one that does not."""
    b, h, gy = bloque(32), torch.randn(2, 20, 32, device=DEV), torch.randn(2, 20, 32, device=DEV)
    gs = []
    for en_sitio in (False, True):
        b.ff[1] = torch.nn.ReLU(inplace=en_sitio)
        gs.append(torch.autograd.grad(b(h), list(b.parameters()), gy))
    assert all(torch.equal(x, y) for x, y in zip(*gs))


def test_memoria_without_the_nodes(monkeypatch):
    """A library that was built alone runs 'memoria' models on torch's operators: trained and written as with the nodes."""
    from asrn_amd import _lib
    m = asrn_amd.crear_modelo(60, d=32, n_capas=2, semilla=1, mezcla='memoria', memoria_max=64, **REDUCIDA).to(DEV)
    x = synth.tokens(2, 41, 60, seed=0).to(DEV)

    def todo():
        m.train()
        gs = torch.autograd.grad(m.perdida(x[:, :-1], x[:, 1:]), list(m.parameters()))
        m.eval()
        return gs, asrn_amd.escribir(m, x, n_nuevos=20, top_k=1)[1]
    gs, escrito = todo()

    def faltan():
        raise _lib.ASRNHipError('_nodos.so is missing')
    for sitio in ('selectiva', 'ops', 'entrenamiento', '_lib'):
        monkeypatch.setattr(f'asrn_amd.{sitio}.nodos', faltan)
    gs2, escrito2 = todo()
    for a, b in zip(gs, gs2):
        assert (a - b).norm() <= 1e-4 * a.norm() + 1e-7
    assert (escrito - escrito2).abs().max() <= 1e-3
    b = m.bloques[0]
    with pytest.raises(_lib.ASRNHipError, match='missing'):
        asrn_amd.conv_canal(torch.randn(1, 3, 32, device=DEV), b.conv.weight)


@pytest.mark.parametrize('act', [None, 'gelu', 'silu'])
@pytest.mark.parametrize('forma', ['densa', 'traspuesta'])
def test_second_gradient_of_the_convolution_where_it_is_recorded(act, forma):
    """registrable: the gradients that are recorded are the formula's, and so are theirs (fp32 sums of some 20 terms around 1: 64
    roundings of the largest value)."""
    z, w, b = torch.randn(2, 9, 8, device=DEV), torch.randn(8, 1, 4, device=DEV), torch.randn(8, device=DEV)
    if forma == 'traspuesta':
        z = z.transpose(1, 2).contiguous().transpose(1, 2)
    g1, g2 = torch.randn(2, 9, 8, device=DEV), [torch.randn_like(t) for t in (z, w, b)]

    def formula(z, w, b):
        v = F.pad(z, (0, 0, 3, 0)).unfold(1, 4, 1)
        pre = (v * w[:, 0]).sum(-1) + b
        return pre if act is None else F.gelu(pre) if act == 'gelu' else F.silu(pre)

    def dos(f, dt):
        hojas = [t.to(dt).requires_grad_() for t in (z.detach(), w, b)]
        gs = torch.autograd.grad(f(*hojas), hojas, g1.to(dt).requires_grad_(), create_graph=True)
        total = sum((a * c.to(dt)).sum() for a, c in zip(gs, g2))
        return [*gs, *torch.autograd.grad(total, hojas, allow_unused=True, materialize_grads=True)]    # without act b enters none
    propia = dos(lambda *a: asrn_amd.conv_canal(*a, act, registrable=True), torch.float32)
    for a, v in zip(propia, dos(formula, torch.float64)):
        assert (a - v).abs().max() <= 64 * U * 20 * max(1, v.abs().max())
    solo = torch.randn(2, 5, 8, device=DEV).requires_grad_()         # one argument alone asks for a gradient
    g, = torch.autograd.grad(asrn_amd.conv_canal(solo, w, b, act, registrable=True).sum(), solo, create_graph=True)
    ref, = torch.autograd.grad(asrn_amd.conv_canal(solo, w, b, act).sum(), solo)
    assert (g - ref).abs().max() <= 64 * U * 20


def test_memoria_model_with_a_recorded_gradient():
    """Gradients with create_graph=True are those without."""
    m = asrn_amd.crear_modelo(60, d=32, n_capas=2, semilla=1, mezcla='memoria', memoria_max=64, **REDUCIDA).to(DEV)
    x = synth.tokens(2, 41, 60, seed=0).to(DEV)
    ps = list(m.parameters())
    ref, got = (torch.autograd.grad(m.perdida(x[:, :-1], x[:, 1:]), ps, create_graph=c) for c in (False, True))
    for a, b in zip(ref, got):
        assert (a - b).norm() <= 2e-3 * a.norm() + 1e-7
    z, w = torch.randn(2, 9, 8, device=DEV).requires_grad_(), torch.randn(8, 1, 4, device=DEV).requires_grad_()
    g, = torch.autograd.grad(conv_canal_causal(z, w, torch.randn(8, device=DEV)).square().sum(), z, create_graph=True)
    assert torch.autograd.grad(g.square().sum(), w)[0].abs().sum() > 0


def test_hooks_see_a_recorded_gradient_once():
    hojas = [torch.randn(2, 9, 8, device=DEV).requires_grad_(), torch.randn(8, 1, 4, device=DEV).requires_grad_(),
             torch.randn(8, device=DEV).requires_grad_()]
    vistas = []
    for t in hojas:
        t.register_hook(lambda g: vistas.append(g.shape) or 2 * g)
    ref, got = (torch.autograd.grad(asrn_amd.conv_canal(1 * hojas[0], *hojas[1:], 'gelu', registrable=True).sum(), hojas, create_graph=c)
                for c in (False, True))
    assert len(vistas) == 6
    for a, b in zip(ref, got):
        assert (a - b).abs().max() <= 64 * U * 20
