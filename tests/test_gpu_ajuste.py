"""The fine-tuning losses (asrn_amd.log_probabilidades, perdida_preferencia, perdida_politica) against plain
implementations in float64: vocabularies at the lengths where a kernel changes, every type, strides and slices, masks
that hide NaN and whole texts, values at the ends of their types, refusals, graph replays.

Tolerances count roundings. u = 2^-24, half a step of fp32. The sum of a row's exponentials: each exponent z carries
three roundings (difference, product, the constant), so its exponential 3 |z| u, and only terms with |z| < 104 count
(exp(-104) is below fp32's range); the exponential itself and the changes of base at most 40 u more (a few steps each);
n = the additions in a row, at most V / 64 by one thread. So s is within (n + 3 * 104 * 2 + 40) u, the factor 2 for the
changes of base: ERR(V) below."""
import math

import pytest
import torch

import asrn_amd
from asrn_amd import ajuste

pytestmark = pytest.mark.gpu
DEV = 'cuda'
U = 2.0 ** -24
TIPOS = [torch.float32, torch.bfloat16, torch.float16]


def ERR(V):
    return (V / 64 + 6 * 104 + 40) * U


def exacto(x, y, T, g, gh):
    """(lp, H, dx, p, log p, log s) in float64 for rows of x (N, V), y (N), -100 ignored."""
    xd = x.detach().double() / T
    ve = (y != -100)[:, None]
    logp = torch.log_softmax(xd, -1)
    p = logp.exp()
    plogp = torch.where(p > 0, p * logp, 0.0)
    H = -plogp.sum(1, keepdim=True)
    uno = torch.zeros_like(xd).scatter_(1, y.clamp(min=0)[:, None], 1.0)
    lp = torch.where(ve, logp.gather(1, y.clamp(min=0)[:, None]), 0.0)[:, 0]
    dx = (g.double()[:, None] * (uno - p) - gh.double()[:, None] * (plogp + p * H)) / T
    z = xd - xd.amax(1, keepdim=True)
    return lp, torch.where(ve, H, 0.0)[:, 0], torch.where(ve, dx, 0.0), p, logp, z.exp().sum(1).log(), z


def comprobar(x, y, T, entropia, g, gh, lp, H, dx):
    V = x.shape[-1]
    lp0, H0, dx0, p, logp, ls, z = exacto(x, y, T, g, gh if entropia else 0 * gh)
    zf = torch.where(p > 0, z, 0.0)
    ve = y != -100
    zy = torch.where(ve, zf.gather(1, y.clamp(min=0)[:, None])[:, 0].abs(), 0.0)
    assert ((lp.double() - lp0).abs() <= ve * (ERR(V) + U * (4 * zy + 2 * ls + lp0.abs()))).all()
    Ez = (p * zf.abs()).sum(1)
    if entropia:
        assert ((H.double() - H0).abs() <= ve * (ERR(V) * (1 + 2 * Ez) + 4 * U * (ls + Ez))).all()
    ga, ha = g.double().abs()[:, None], gh.double().abs()[:, None] * entropia
    peso = p * (ga + ha * (torch.where(p > 0, logp, 0.0).abs() + H0[:, None].abs() + 2 * ls[:, None] + 1))
    tol = (2 * ERR(V) * peso + 4 * U * ga) / T + torch.finfo(dx.dtype).eps / 2 * dx0.abs()
    tol = tol + torch.finfo(dx.dtype).tiny           # results below the type's range
    assert ((dx.double() - dx0).abs() <= tol * ve[:, None]).all()


@pytest.mark.parametrize('V', [1, 2, 7, 8, 9, 255, 256, 259, 2047, 2048, 4096, 4099, 8192, 16384, 16391, 50304, 70001])
@pytest.mark.parametrize('dtype', TIPOS)
@pytest.mark.parametrize('entropia,T', [(False, 1.0), (True, 0.7)])
def test_logp_lengths(V, dtype, entropia, T):
    g = torch.Generator(device=DEV).manual_seed(V)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    x = (3 * r(7, V)).to(dtype).requires_grad_()
    y = torch.randint(0, V, (7,), generator=g, device=DEV)
    y[3] = -100
    ga, gh = r(7), r(7)
    out = asrn_amd.log_probabilidades(x, y, temperatura=T, entropia=entropia)
    lp, H = out if entropia else (out, None)
    dx, = torch.autograd.grad(out, x, (ga, gh) if entropia else ga)
    assert lp.dtype == torch.float32 and dx.dtype == dtype
    comprobar(x, y, T, entropia, ga, gh, lp, H, dx)


@pytest.mark.parametrize('filas,V', [(1, 131072), (3, 40000), (1025, 16400), (2000, 300), (5, 33)])
def test_logp_rows(filas, V):
    """One row to many: the backward's splits, the forward's workgroup a row and four rows a workgroup."""
    g = torch.Generator(device=DEV).manual_seed(filas)
    x = (2 * torch.randn(filas, V, generator=g, device=DEV)).bfloat16().requires_grad_()
    y = torch.randint(0, V, (filas,), generator=g, device=DEV)
    y[::5] = V - 1
    y[1::7] = -100
    ga, gh = (torch.randn(filas, generator=g, device=DEV) for _ in range(2))
    lp, H = asrn_amd.log_probabilidades(x, y, entropia=True)
    comprobar(x, y, 1.0, True, ga, gh, lp, H, torch.autograd.grad((lp, H), x, (ga, gh))[0])


def _vistas():
    g = torch.Generator(device=DEV).manual_seed(3)
    base = 2 * torch.randn(4, 9, 331, generator=g, device=DEV)
    return {'recorte': base[:, :-1], 'columnas': base[..., 5:322], 'traspuesta': base.transpose(0, 1),
            'salto': base[::2, 1::3], 'cuatro': base[:, :8].reshape(2, 2, 8, 331)[:, :, 1:], 'una': base[0, 0],
            'columna_suelta': base.transpose(1, 2), 'expandida': base[:1].expand(3, 9, 331), 'filas': base[2],
            'sin_filas': base[:0], 'sin_fichas': base[:, :0]}


@pytest.mark.parametrize('cual', ['recorte', 'columnas', 'traspuesta', 'salto', 'cuatro', 'una', 'columna_suelta',
                                  'expandida', 'filas', 'sin_filas', 'sin_fichas'])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_logp_strides(cual, dtype):
    hoja = _vistas()[cual].to(dtype) if dtype == torch.float32 else None
    if hoja is None:                                 # the same view of a 16-bit tensor, an odd number of elements in
        v = _vistas()[cual]
        plano = torch.zeros(v.numel() + 1 if v.is_contiguous() else 1, device=DEV, dtype=dtype)
        hoja = plano[1:].view(v.shape).copy_(v) if v.is_contiguous() and v.numel() else v.to(dtype)
    x = hoja.detach().requires_grad_()
    V = x.shape[-1]
    g = torch.Generator(device=DEV).manual_seed(4)
    y = torch.randint(0, V, x.shape[:-1], generator=g, device=DEV)
    ga, gh = (torch.randn(x.shape[:-1], generator=g, device=DEV) for _ in range(2))
    lp, H = asrn_amd.log_probabilidades(x, y, entropia=True)
    dx, = torch.autograd.grad((lp, H), x, (ga, gh))
    assert lp.shape == y.shape and dx.shape == x.shape
    if y.numel():
        comprobar(x.reshape(-1, V), y.reshape(-1), 1.0, True, ga.reshape(-1), gh.reshape(-1), lp.reshape(-1), H.reshape(-1),
                  dx.reshape(-1, V))


@pytest.mark.parametrize('forma', [(2, 3, 0), (0, 3, 4), (2, 0, 4), (0, 0, 0, 0)])
def test_logp_many_axes_without_tokens(forma):
    x = torch.randn(*forma, 5, device=DEV, requires_grad=True)
    lp, H = asrn_amd.log_probabilidades(x, torch.zeros(forma, dtype=torch.long, device=DEV), entropia=True)
    assert lp.shape == H.shape == forma and torch.autograd.grad(lp.sum() + H.sum(), x)[0].shape == x.shape


@pytest.mark.parametrize('dtype', TIPOS)
def test_logp_extremes(dtype):
    """Infinities, the type's ends, NaN and targets outside the vocabulary, against torch's log_softmax."""
    inf, bajo, alto = math.inf, torch.finfo(dtype).min, torch.finfo(dtype).max
    V = 600
    x = torch.randn(10, V, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(dtype)
    x[0, 100:] = -inf                                # masked words
    x[1, 3:] = bajo
    x[2, 5] = inf
    x[3, 17] = float('nan')
    x[4] = -inf
    x[5] = bajo                                      # a row of the lowest value: uniform
    x[6, 0], x[6, 1:] = alto, bajo
    x[7] = float('nan')                              # ignored: nothing of it may show
    y = torch.tensor([99, 0, 5, 17, 0, 599, 0, -100, 600, -7], device=DEV)
    xr = x.clone().requires_grad_()
    lp, H = asrn_amd.log_probabilidades(xr, y, entropia=True)
    dx, = torch.autograd.grad((lp, H), xr, (torch.ones(10, device=DEV), torch.ones(10, device=DEV)))
    ref = torch.log_softmax(x.double(), -1)
    for i in (0, 1, 5, 6):
        e = ref[i, y[i]]
        assert abs(lp[i].double() - e) <= ERR(V) + 4 * U * e.abs(), i
        p = ref[i].exp()
        assert abs(H[i].double() + torch.where(p > 0, p * ref[i], 0.0).sum()) <= ERR(V) * 8 * math.log(V) and torch.isfinite(dx[i]).all()
    assert torch.isnan(lp[[2, 3, 4, 8, 9]]).all() and torch.isnan(dx[[2, 3, 4, 8, 9]]).any(1).all()
    assert lp[7] == 0 and H[7] == 0 and (dx[7] == 0).all()
    assert (dx[0, 100:] == 0).all()
    xr = x[:1].clone().requires_grad_()              # the log-probability of a word that is masked
    lp = asrn_amd.log_probabilidades(xr, torch.tensor([200], device=DEV))
    assert lp.item() == -inf and torch.isfinite(torch.autograd.grad(lp.sum(), xr)[0]).all()


def test_logp_differences():
    """The gradient along random directions against central differences of the float64 definition."""
    g = torch.Generator(device=DEV).manual_seed(9)
    x = (2 * torch.randn(5, 777, generator=g, device=DEV)).requires_grad_()
    y = torch.randint(0, 777, (5,), generator=g, device=DEV)
    ga, gh = (torch.randn(5, generator=g, device=DEV) for _ in range(2))
    lp, H = asrn_amd.log_probabilidades(x, y, temperatura=1.3, entropia=True)
    dx, = torch.autograd.grad((lp, H), x, (ga, gh))
    f = lambda v: sum((a * b.double()).sum() for a, b in zip(exacto(v, y, 1.3, ga, gh)[:2], (ga, gh)))
    for _ in range(3):
        d = torch.randn(5, 777, generator=g, device=DEV).double()
        num = (f(x.detach().double() + 1e-5 * d) - f(x.detach().double() - 1e-5 * d)) / 2e-5
        assert abs((dx.double() * d).sum() - num) <= 1e-6 * (dx.double() * d).abs().sum() + 1e-8


def test_logp_past_32_bits():
    """More than 2^31 logits: the last rows against the same rows alone, bit for bit, gradient included."""
    filas, V = 43_001, 50_304
    x = torch.empty(filas, V, dtype=torch.bfloat16, device=DEV).fill_(0.5)
    g = torch.Generator(device=DEV).manual_seed(6)
    cola = (2 * torch.randn(5, V, generator=g, device=DEV)).bfloat16()
    x[-5:] = cola
    y = torch.full((filas,), 7, device=DEV)
    y[-5:] = torch.randint(0, V, (5,), generator=g, device=DEV)
    y[:20_000] = -100
    x.requires_grad_()
    lp = asrn_amd.log_probabilidades(x, y)
    dx, = torch.autograd.grad(lp, x, torch.ones_like(lp))
    c = torch.cat([x.detach()[:1200], cola]).requires_grad_()        # past 1,024 rows: the same kernels
    yc = torch.cat([torch.full((1200,), 7, device=DEV), y[-5:]])
    l2 = asrn_amd.log_probabilidades(c, yc)
    d2, = torch.autograd.grad(l2, c, torch.ones_like(l2))
    assert torch.equal(lp[-5:], l2[-5:]) and torch.equal(dx[-5:], d2[-5:]) and torch.equal(lp[20_000:20_010], l2[:10])
    assert (lp[:20_000] == 0).all() and (dx[19_990:20_000] == 0).all()


def test_logp_gradients_of_one_output_and_expanded():
    x = torch.randn(2, 3, 50, device=DEV).requires_grad_()
    y = torch.randint(0, 50, (2, 3), device=DEV)
    lp, H = asrn_amd.log_probabilidades(x, y, entropia=True)
    a, = torch.autograd.grad(lp.sum(), x, retain_graph=True)          # an expanded gradient, none for H
    b, = torch.autograd.grad(H.sum(), x)
    xd = x.detach().double().requires_grad_()
    l = torch.log_softmax(xd, -1)
    ra, = torch.autograd.grad(l.gather(-1, y[..., None]).sum(), xd, retain_graph=True)
    rb, = torch.autograd.grad(-(l.exp() * l).sum(), xd)
    assert (a - ra).abs().max() <= 2 * ERR(50) and (b - rb).abs().max() <= 8 * ERR(50)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(asrn_amd.log_probabilidades(x, y).sum(), x, create_graph=True)[0].sum(), x)


# ---------------------------------------------------------------------------------------------------------------------
# the preference loss
# ---------------------------------------------------------------------------------------------------------------------

def preferencia_exacta(lp, m, ref, beta, tipo, suavizado, margen, por_longitud):
    P = lp.shape[0] // 2
    v = lp.detach().double().requires_grad_()
    on = torch.ones_like(lp, dtype=torch.bool) if m is None else m != 0
    d = torch.where(on, v if ref is None or ref.dim() == 1 else v - torch.where(on, ref.double(), 0.0), 0.0).sum(1)
    if ref is not None and ref.dim() == 1:
        d = d - ref.double()
    R = d / on.sum(1).clamp(min=1) if por_longitud else d
    h = beta * (R[:P] - R[P:]) - margen
    ls = torch.nn.functional.logsigmoid
    por = {'sigmoide': lambda: -(1 - suavizado) * ls(h) - suavizado * ls(-h), 'ipo': lambda: ((h - 0.5) / beta) ** 2,
           'bisagra': lambda: torch.relu(1 - h)}[tipo]()
    loss = por.mean()
    return loss.detach(), (beta * R).detach(), torch.autograd.grad(loss, v)[0]


@pytest.mark.parametrize('P,L', [(1, 1), (1, 60), (3, 257), (8, 512), (8, 513), (9, 100), (2, 4096), (2, 4097), (5, 9001), (300, 33)])
@pytest.mark.parametrize('tipo,suavizado,margen,por_longitud', [
    ('sigmoide', 0.0, 0.0, False), ('sigmoide', 0.1, 0.3, True), ('ipo', 0.0, 0.0, True), ('ipo', 0.0, -0.2, False),
    ('bisagra', 0.0, 0.0, False), ('bisagra', 0.0, 0.5, True)])
@pytest.mark.parametrize('ref', ['no', 'fichas', 'textos'])
def test_preference(P, L, tipo, suavizado, margen, por_longitud, ref):
    g = torch.Generator(device=DEV).manual_seed(P * L)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    lp = (-r(2 * P, L).abs()).requires_grad_()
    m = torch.rand(2 * P, L, generator=g, device=DEV) < 0.6
    m[0] = False                                     # a text without tokens
    rf = {'no': None, 'fichas': lp.detach() + 0.1 * r(2 * P, L), 'textos': -10 * r(2 * P).abs()}[ref]
    with torch.no_grad():                            # what the mask hides is not used
        lp[~m] = float('nan')
        if ref == 'fichas':
            rf[~m] = float('inf')
    kw = dict(beta=0.15, tipo=tipo, suavizado=suavizado, margen=margen, por_longitud=por_longitud)
    perdida, rec = asrn_amd.perdida_preferencia(lp, m, rf, **kw)
    dlp, = torch.autograd.grad(perdida, lp, torch.tensor(1.7, device=DEV))
    e, er, ed = preferencia_exacta(lp, m, rf, **kw)
    # one rounding of a double each (the double's own error, 2^-40 of the sums, beside it); the gradient's coefficient,
    # its product with the loss's gradient
    s = 2.0 ** -40 * (1 + er.abs().max())
    assert abs(perdida.double() - e) <= U * e.abs() + s * (1 + 2 / 0.15 * er.abs().max()) and ((rec.double() - er).abs() <= U * er.abs() + s).all()
    lim = s * 4 if tipo != 'bisagra' else 0.0
    assert ((dlp.double() - 1.7 * ed).abs() <= 3 * U * (1.7 * ed).abs() + lim).all()


def test_preference_long_texts_and_strides():
    """Texts past 2^17 tokens whose sums cancel, rows and tokens read through their strides, masks of other types."""
    P, L = 2, 150_001
    g = torch.Generator(device=DEV).manual_seed(2)
    ancho = -torch.rand(2 * P, 2 * L, generator=g, device=DEV)
    lp = ancho[:, ::2].requires_grad_()
    ref = (ancho.detach()[:, ::2] + 1e-4 * torch.randn(L, 2 * P, generator=g, device=DEV).t())      # a transposed reference
    m = (torch.rand(2 * P, L, generator=g, device=DEV) < 0.5).to(torch.int64) * 3
    for mm in (None, m, m.float(), m.bool()[:, :1].expand(2 * P, L), m.t().contiguous().t()):
        perdida, rec = asrn_amd.perdida_preferencia(lp, mm, ref)
        dlp, = torch.autograd.grad(perdida, lp)
        e, er, ed = preferencia_exacta(lp, mm, ref, 0.1, 'sigmoide', 0.0, 0.0, False)
        assert abs(perdida.double() - e) <= U * e.abs() + 1e-12 * L and ((rec.double() - er).abs() <= U * er.abs() + 1e-12 * L).all()
        assert ((dlp.double() - ed).abs() <= 4 * U * ed.abs() + 1e-13 * L).all()


@pytest.mark.parametrize('P,L', [(1, 3), (9, 600)])
def test_preference_sums_in_float64(P, L):
    """The reference's sums in fp64 (also strided): their digits past fp32's reach the difference of large sums."""
    g = torch.Generator(device=DEV).manual_seed(P)
    lp = (-8e4 / L * (1 + 1e-3 * torch.rand(2 * P, L, generator=g, device=DEV))).requires_grad_()
    ref = lp.detach().double().sum(1) + 3e-3 * torch.randn(2 * P, generator=g, device=DEV).double()
    for r in (ref, torch.stack([ref, ref + 1], 1)[:, 0]):
        perdida, rec = asrn_amd.perdida_preferencia(lp, None, r, beta=50.0)
        d, = torch.autograd.grad(perdida, lp)
        e, er, ed = preferencia_exacta(lp, None, r, 50.0, 'sigmoide', 0.0, 0.0, False)
        # double sums of L values of 8e4 in all: (L + 2) half steps of double, times beta
        s = 50 * 8e4 * (L + 2) * 2.0 ** -53 * 2
        assert abs(perdida.double() - e) <= U * e.abs() + 2 * s and ((rec.double() - er).abs() <= U * er.abs() + s).all()
        assert ((d.double() - ed).abs() <= 4 * U * ed.abs() + 50 * s).all()
    assert abs(perdida.item() - math.log(2)) > 1e-4     # what fp32 sums would leave


def test_losses_of_very_many_texts():
    """Tens of thousands of one-token texts, and gradients against central differences of the float64 definitions."""
    g = torch.Generator(device=DEV).manual_seed(11)
    lp = (-torch.rand(70_000, 1, generator=g, device=DEV)).requires_grad_()
    perdida, rec = asrn_amd.perdida_preferencia(lp)
    e, er, ed = preferencia_exacta(lp, None, None, 0.1, 'sigmoide', 0.0, 0.0, False)
    d, = torch.autograd.grad(perdida, lp)
    assert abs(perdida.double() - e) <= 2 * U and (rec.double() - er).abs().max() <= U and ((d.double() - ed).abs() <= 3 * U * ed.abs()).all()
    A = torch.randn(70_000, generator=g, device=DEV)
    old = lp.detach() + 0.1
    for reduccion in ajuste.REDUCCIONES:
        perdida, est = asrn_amd.perdida_politica(lp, A, old, reduccion=reduccion)
        (e, ee, ed), tam = politica_exacta(lp, A, old, None, 0.2, 0.2, None, None, 0.0, None, 0.0, reduccion)
        d, = torch.autograd.grad(perdida, lp)
        assert abs(perdida.double() - e) <= U * e.abs() + EXP * tam[0].sum() and ((d.double() - ed).abs() <= 6 * U * ed.abs() + EXP * tam[0]).all()


def test_losses_differences():
    """The gradients along random directions against central differences of the float64 definitions, away from the clips'
    and the hinge's corners (the step is far smaller than any token's distance from them)."""
    g = torch.Generator(device=DEV).manual_seed(12)
    lp = (-torch.rand(6, 33, generator=g, device=DEV)).requires_grad_()
    old, A = lp.detach() + 0.3 * torch.randn(6, 33, generator=g, device=DEV), torch.randn(6, 33, generator=g, device=DEV)
    m = torch.rand(6, 33, generator=g, device=DEV) < 0.7
    casos = [(asrn_amd.perdida_preferencia(lp, m, old, beta=0.3, tipo=t)[0],
              lambda v, t=t: preferencia_exacta(v, m, old, 0.3, t, 0.0, 0.0, False)[0]) for t in ajuste.FORMAS]
    casos.append((asrn_amd.perdida_politica(lp, A, old, m, lp_ref=old, beta=0.1)[0],
                  lambda v: politica_exacta(v, A, old, m, 0.2, 0.2, None, old, 0.1, None, 0.0, 'fichas')[0][0]))
    for perdida, f in casos:
        dlp, = torch.autograd.grad(perdida, lp)
        for _ in range(2):
            d = torch.randn(6, 33, generator=g, device=DEV).double()
            v = lp.detach().double()
            num = (f(v + 1e-6 * d) - f(v - 1e-6 * d)) / 2e-6
            assert abs((dlp.double() * d).sum() - num) <= 1e-6 * (dlp.double() * d).abs().sum() + 1e-8


def test_preference_degenerate():
    lp = torch.zeros(2, 0, device=DEV, requires_grad=True)
    perdida, rec = asrn_amd.perdida_preferencia(lp)                  # no tokens at all: h = 0
    assert abs(perdida.item() - math.log(2)) <= 1e-7 and (rec == 0).all()
    assert torch.autograd.grad(perdida, lp)[0].shape == (2, 0)
    lp = torch.full((4, 3), -500.0, device=DEV, requires_grad=True)  # far apart: no overflow
    with torch.no_grad():
        lp[:1] = 0.0
    perdida, _ = asrn_amd.perdida_preferencia(lp, beta=2.0)
    d, = torch.autograd.grad(perdida, lp)
    assert torch.isfinite(d).all() and abs(perdida.item() - math.log(2) / 2) <= 1e-7
    lp = torch.tensor([[-1.0], [float('nan')]], device=DEV, requires_grad=True)
    for tipo in ajuste.FORMAS:
        perdida, _ = asrn_amd.perdida_preferencia(lp, tipo=tipo)
        assert torch.isnan(perdida) and torch.isnan(torch.autograd.grad(perdida, lp)[0]).all(), tipo
    lp = torch.randn(4, 5, device=DEV).bfloat16().requires_grad_()   # 16-bit log-probabilities
    perdida, _ = asrn_amd.perdida_preferencia(lp)
    assert torch.autograd.grad(perdida, lp)[0].dtype == torch.bfloat16


# ---------------------------------------------------------------------------------------------------------------------
# the policy loss
# ---------------------------------------------------------------------------------------------------------------------

def politica_exacta(lp, A, vieja, m, lo, hi, tope, ref, beta, H, peso, reduccion):
    v = lp.detach().double().requires_grad_()
    h = None if H is None else H.detach().double().requires_grad_()
    on = torch.ones_like(lp, dtype=torch.bool) if m is None else m != 0
    limpio = lambda t: torch.where(on, t.double(), 0.0)
    vm = torch.where(on, v, 0.0)
    A = limpio(A if A.dim() == 2 else A[:, None].expand(lp.shape))
    d = vm - (vm.detach() if vieja is None else limpio(vieja))
    r = d.exp()
    rec = r.clamp(1 - lo, 1 + hi)
    pg = -torch.minimum(r * A, rec * A)
    fuera = (r * A > rec * A)
    if tope is not None:
        sobre = (A < 0) & (r > tope)
        pg, fuera = torch.where(sobre, -tope * A, pg), fuera | sobre
    kl = torch.zeros_like(vm) if ref is None else torch.expm1(limpio(ref) - vm) - (limpio(ref) - vm)
    por = pg + beta * kl - (0.0 if h is None else peso * torch.where(on, h, 0.0))
    on = on.double()
    n = on.sum(1)
    if reduccion == 'textos':
        loss = ((por * on).sum(1) / n.clamp(min=1)).sum() / (n > 0).sum()
    else:
        loss = (por * on).sum() / n.sum()
    media = lambda t: ((t * on).sum() / n.sum()).detach()
    est = torch.stack([media(fuera.double()), media(torch.expm1(d) - d), media(kl),
                       media(torch.zeros_like(vm) if h is None else torch.where(on > 0, h, 0.0))])
    peso_de = on / (n[:, None].clamp(min=1) * (n > 0).sum() if reduccion == 'textos' else n.sum())
    q = torch.zeros_like(vm) if ref is None else torch.where(on > 0, ref.double(), 0.0) - vm
    tam = [(t * peso_de).detach() for t in ((r * A).abs(), beta * torch.expm1(q).abs(), beta * kl)]
    return (loss.detach(), est, *torch.autograd.grad(loss, [v] + ([] if h is None else [h]))), tam


# The policy kernel's exponentials are fp32's, all else double. Up to |d| = 1 the series for exp d - 1 - d: its eleven
# steps shrink, so their roundings and the argument's come to 5 U of it, and of exp d - 1 and exp d (1 + d and it, in
# double) to less. Past it expf within one step (2 U) and the factor of its argument's rounding, 3 U of exp d, so 3 U e /
# |e - 1| <= 4.8 U of exp d - 1 and 3 U e / (e - 2) <= 11.4 U of exp d - 1 - d (the worst at d = 1). So a token's loss is
# within 3 U r |A| + 12 U beta kl and its gradient within 3 U r |A| + 7 U beta |expm1 q| (here with the divisor: tam), the
# statistics within 12 U of themselves, before the last roundings.
EXP, EXPM1, KL = 3 * U, 7 * U, 12 * U


@pytest.mark.parametrize('B,L', [(1, 1), (2, 50), (8, 512), (8, 513), (9, 100), (3, 2048), (3, 2049), (2, 7001), (700, 9)])
@pytest.mark.parametrize('ventaja', ['fichas', 'textos'])
@pytest.mark.parametrize('tope,kl,entropia,vieja', [(None, False, False, True), (1.5, True, True, True),
                                                    (None, True, False, False)])
@pytest.mark.parametrize('reduccion', ajuste.REDUCCIONES)
def test_policy(B, L, ventaja, tope, kl, entropia, vieja, reduccion):
    g = torch.Generator(device=DEV).manual_seed(B * L)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    old = -r(B, L).abs()
    lp = (old + 0.4 * r(B, L)).requires_grad_()
    A = r(B, L) if ventaja == 'fichas' else r(B)
    ref = old + 0.01 * r(B, L) if kl else None
    H = r(B, L).abs().requires_grad_() if entropia else None
    m = torch.rand(B, L, generator=g, device=DEV) < 0.6
    m[-1] = B == 1                                   # a text without tokens
    with torch.no_grad():
        for t in (lp, old, ref, H):
            if t is not None:
                t[~m] = float('nan')
    args = dict(lp_ref=ref, beta=0.05 if kl else 0.0, entropia=H, peso_entropia=0.02 if entropia else 0.0)
    perdida, est = asrn_amd.perdida_politica(lp, A, old if vieja else None, m, recorte=(0.2, 0.3), tope=tope,
                                             reduccion=reduccion, **args)
    hojas = [lp] + ([H] if entropia else [])
    ds = torch.autograd.grad(perdida, hojas, torch.tensor(-0.6, device=DEV))
    (e, ee, *ed), tam = politica_exacta(lp, A, old if vieja else None, m, 0.2, 0.3, tope, ref, args['beta'], H, 0.02, reduccion)
    s = 2.0 ** -40
    assert abs(perdida.double() - e) <= U * e.abs() + EXP * tam[0].sum() + KL * tam[2].sum() + s
    assert ((est.double() - ee).abs() <= (U + KL) * ee.abs() + s).all()
    # a token's gradient: rounded once, divided by its divisor (rounded twice more), times the loss's gradient
    for a, b, t in zip(ds, ed, (EXP * tam[0] + EXPM1 * tam[1], 0.0)):
        assert ((a.double() + 0.6 * b).abs() <= 6 * U * b.abs() + t + s / L).all()


def test_policy_borders():
    """Tokens at a clip's border and next to it: the gradient is cut exactly where log r passes log(1 + e), in double."""
    alto = math.log1p(0.28)
    x = torch.tensor(alto, dtype=torch.float32, device=DEV)
    pasos = torch.stack([torch.nextafter(x, torch.tensor(s, device=DEV)) for s in (-9.0, 9.0)] + [x])
    lp = pasos[None].clone().requires_grad_()
    old = torch.zeros_like(lp)
    perdida, est = asrn_amd.perdida_politica(lp, torch.ones(1, device=DEV), old, recorte=(0.2, 0.28))
    d, = torch.autograd.grad(perdida, lp)
    fuera = lp.detach().double() > alto
    assert ((d == 0) == fuera).all() and abs(est[0].item() - fuera.double().mean().item()) <= 1e-7
    # far apart: r past fp32's range under an advantage of 0, ratios at the ends of the type, a wide KL
    lp = torch.tensor([[95.0, -3e38, -30.0, 1.0]], device=DEV, requires_grad=True)
    old = torch.tensor([[0.0, 3e38, 30.0, 1.0]], device=DEV)
    perdida, est = asrn_amd.perdida_politica(lp, torch.tensor([[0.0, 1.0, 1.0, 2.0]], device=DEV), old,
                                             lp_ref=torch.zeros(1, 4, device=DEV))
    d, = torch.autograd.grad(perdida, lp)
    assert abs(perdida.item() + 0.5) <= 1e-7 and torch.allclose(d, torch.tensor([[0.0, 0.0, 0.0, -0.5]], device=DEV), atol=1e-20)
    lp = torch.tensor([[0.0, -math.inf, 200.0, -3.0]], device=DEV, requires_grad=True)
    A = torch.tensor([[0.0, 1.0, 1.0, -1.0]], device=DEV)
    perdida, _ = asrn_amd.perdida_politica(lp, A, torch.zeros(1, 4, device=DEV))
    d, = torch.autograd.grad(perdida, lp)            # r = 0, r = inf clipped, A = 0, r clipped from below
    assert abs(perdida.item() - (0.0 + 0.0 - 1.2 + 0.8) / 4) <= 1e-7 and (d == 0).all()


@pytest.mark.parametrize('B', [1, 9])                   # one launch, and the tokens' own
def test_policy_far_ratios(B):
    """Ratios past fp32's range, against float64: nothing of them under an advantage of 0 (at any finite d, 64 bits' own
    range passed too), finite under one that is small enough, and in a KL term of a small weight."""
    lp = torch.tensor([[177.0, 178.0, 300.0, 709.0, 800.0, 3e38, -3e38, 0.5]] * B, device=DEV, requires_grad=True)
    A = torch.zeros(B, 8, device=DEV)
    A[:, -1] = -1.0
    perdida, est = asrn_amd.perdida_politica(lp, A, torch.zeros_like(lp))
    d, = torch.autograd.grad(perdida, lp)
    e = math.exp(0.5) / 8
    assert abs(perdida.item() - e) <= 2 * EXP * e and (d[:, :-1] == 0).all() and ((d[:, -1] - e / B).abs() <= 6 * U * e).all()
    assert torch.isfinite(est[:1]).all()
    # exp d for d > 160 is the eighth power of expf's, each within a step (2 U): 16 U, and the loss's own rounding
    for v in (161.0, 177.75, 178.0, 185.3):
        lp = torch.full((B, 3), v, device=DEV, requires_grad=True)
        A = torch.full((B,), -1e-43, device=DEV)         # subnormal: r A is finite in fp32
        perdida, _ = asrn_amd.perdida_politica(lp, A, torch.zeros_like(lp))
        d, = torch.autograd.grad(perdida, lp)
        e = math.exp(lp[0, 0].item()) * -A[0].double().item()
        assert abs(perdida.item() - e) <= 18 * U * e and ((d.double() * 3 * B - e).abs() <= 22 * U * e).all(), v
    for q, beta in ((170.0, 1e-60), (178.0, 1e-60), (300.0, 1e-120), (700.0, 1e-290)):
        lp = torch.zeros(B, 2, device=DEV, requires_grad=True)
        perdida, _ = asrn_amd.perdida_politica(lp, torch.zeros(B, device=DEV), lp_ref=torch.full((B, 2), q, device=DEV), beta=beta)
        d, = torch.autograd.grad(perdida, lp)
        e = beta * (math.expm1(q) - q)
        assert abs(perdida.item() - e) <= 18 * U * e and ((d.double() * 2 * B + e).abs() <= 22 * U * e).all(), q


def test_policy_strides_and_masks():
    g = torch.Generator(device=DEV).manual_seed(5)
    B, L = 6, 3001
    ancho = -torch.rand(B, L + 9, 2, generator=g, device=DEV)
    lp = ancho[:, 4:-5, 1].requires_grad_()
    old = torch.randn(L, B, generator=g, device=DEV).t() * 0.1 + lp.detach()
    A = torch.randn(B, generator=g, device=DEV).double()
    for m in (None, (torch.rand(B, L, generator=g, device=DEV) < 0.4).half(), torch.ones(B, 1, device=DEV).expand(B, L)):
        perdida, est = asrn_amd.perdida_politica(lp, A, old, m)
        d, = torch.autograd.grad(perdida, lp)
        (e, ee, ed), tam = politica_exacta(lp, A.float(), old, m, 0.2, 0.2, None, None, 0.0, None, 0.0, 'fichas')
        assert abs(perdida.double() - e) <= U * e.abs() + EXP * tam[0].sum() + 2.0 ** -40
        assert ((est.double() - ee).abs() <= (U + KL) * ee.abs() + 2.0 ** -40).all()
        assert ((d.double() - ed).abs() <= 6 * U * ed.abs() + EXP * tam[0]).all()


def test_policy_without_tokens_and_one_gradient():
    lp = torch.randn(2, 3, device=DEV, requires_grad=True)
    H = torch.rand(2, 3, device=DEV, requires_grad=True)
    A = torch.ones(2, device=DEV)
    nada = torch.zeros(2, 3, dtype=torch.bool, device=DEV)
    for reduccion in ajuste.REDUCCIONES:
        perdida, est = asrn_amd.perdida_politica(lp, A, mascara=nada, reduccion=reduccion)
        assert torch.isnan(perdida) and torch.isnan(est).all()
        assert (torch.autograd.grad(perdida, lp)[0] == 0).all()
    perdida, _ = asrn_amd.perdida_politica(lp.detach(), A, entropia=H, peso_entropia=0.5)
    d, = torch.autograd.grad(perdida, H)
    assert torch.allclose(d, torch.full_like(d, -0.5 / 6), rtol=1e-6)
    perdida, _ = asrn_amd.perdida_politica(lp[:, :0], A)
    assert torch.isnan(perdida)


# ---------------------------------------------------------------------------------------------------------------------
# refusals, graphs, streams
# ---------------------------------------------------------------------------------------------------------------------

def test_refusals():
    x, y = torch.randn(2, 3, 10, device=DEV), torch.zeros(2, 3, dtype=torch.long, device=DEV)
    lp = torch.zeros(2, 3, device=DEV)
    L, P, Q = asrn_amd.log_probabilidades, asrn_amd.perdida_preferencia, asrn_amd.perdida_politica
    malas = [lambda: L(x, y[:1]), lambda: L(x.double(), y), lambda: L(x, y.float()), lambda: L(x[..., :0], y),
             lambda: L(x, y, temperatura=0.0), lambda: L(x, y, temperatura=float('nan')), lambda: L(x, y.cpu()),
             lambda: P(lp[:1]), lambda: P(lp[0]), lambda: P(lp.long()), lambda: P(lp, lp[:, :2]), lambda: P(lp, None, lp[:1]),
             lambda: P(lp, tipo='otra'), lambda: P(lp, beta=0.0), lambda: P(lp, suavizado=2.0), lambda: P(lp, lp.cpu()),
             lambda: P(lp, suavizado=0.1, tipo='ipo'), lambda: P(lp, margen=float('inf')), lambda: P(lp, ref=lp.cpu()),
             lambda: Q(lp, lp[:, :2]), lambda: Q(lp, lp, lp[:1]), lambda: Q(lp, lp, recorte=-0.1), lambda: Q(lp, lp, recorte=(0.1, 0.2, 0.3)),
             lambda: Q(lp, lp, recorte=(1.5, 0.2)), lambda: Q(lp, lp, tope=1.0), lambda: Q(lp, lp, beta=0.1),
             lambda: Q(lp, lp, peso_entropia=0.1), lambda: Q(lp, lp, reduccion='otra'), lambda: Q(lp, lp, mascara=lp[:1]),
             lambda: Q(lp, lp.cpu()), lambda: Q(lp, lp.long())]
    for i, mala in enumerate(malas):
        with pytest.raises(ValueError):
            mala()
            print('taken:', i)
    for mala in (lambda: L(x.cpu(), y.cpu()), lambda: P(lp.cpu()), lambda: Q(lp.cpu(), lp.cpu())):
        with pytest.raises(RuntimeError, match='GPU only'):
            mala()


def test_graph_replays():
    """Scores, both losses and their gradients captured together, replayed with eager work between, on new inputs."""
    g = torch.Generator(device=DEV).manual_seed(8)
    x = torch.randn(4, 40, 1003, generator=g, device=DEV).bfloat16().requires_grad_()
    y = torch.randint(0, 1003, (4, 40), generator=g, device=DEV)
    y[:, :7] = -100
    A = torch.randn(4, generator=g, device=DEV)
    old = torch.empty(4, 40, device=DEV)

    def paso():
        m = y != -100
        lp, H = asrn_amd.log_probabilidades(x, y, entropia=True)
        a, rec = asrn_amd.perdida_preferencia(lp, m, old)
        b, est = asrn_amd.perdida_politica(lp, A, old, m, entropia=H, peso_entropia=0.01, lp_ref=old, beta=0.02,
                                           reduccion='textos')
        return [t.detach() for t in (lp, H, a, rec, b, est, *torch.autograd.grad(a + b, x))]    # no graph outlives the step

    old.copy_(asrn_amd.log_probabilidades(x, y).detach())
    lado = torch.cuda.Stream()
    lado.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(lado):
        paso()
    torch.cuda.current_stream().wait_stream(lado)
    torch.cuda.synchronize()
    grafo = torch.cuda.CUDAGraph()
    with torch.cuda.graph(grafo):
        salida = paso()
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=g, device=DEV))
            old.copy_(-torch.rand(4, 40, generator=g, device=DEV) * 7)
        y[i % 4, 20:] = -100 if i % 2 else 5
        grafo.replay()
        torch.cuda.synchronize()
        for a, b in zip(salida, paso()):
            assert torch.equal(a, b), i


def test_side_stream():
    x = torch.randn(3, 17, 500, device=DEV).requires_grad_()
    y = torch.randint(0, 500, (3, 17), device=DEV)

    def paso():
        lp = asrn_amd.log_probabilidades(x, y)
        return lp.detach(), torch.autograd.grad(lp.sum(), x)[0]

    base = paso()
    lado = torch.cuda.Stream()
    lado.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(lado):
        otra = paso()
    torch.cuda.current_stream().wait_stream(lado)
    assert all(torch.equal(a, b) for a, b in zip(base, otra))


@pytest.mark.parametrize('B,L', [(4, 50), (6, 5001)])
def test_losses_on_a_side_stream(B, L):
    """Both losses and their gradients on another stream, work before them on it: the default stream's bits."""
    g = torch.Generator(device=DEV).manual_seed(B)
    lp0 = -torch.rand(B, L, generator=g, device=DEV)
    old, A = lp0 + 0.1 * torch.randn(B, L, generator=g, device=DEV), torch.randn(B, generator=g, device=DEV)
    m = torch.rand(B, L, generator=g, device=DEV) < 0.6

    def paso():
        lp = (lp0 * 2 - lp0).requires_grad_()        # written on the current stream
        a, rec = asrn_amd.perdida_preferencia(lp, m, old)
        b, est = asrn_amd.perdida_politica(lp, A, old, m, lp_ref=old, beta=0.1)
        return [t.detach() for t in (a, rec, b, est, *torch.autograd.grad(a + b, lp))]

    base = paso()
    torch.cuda.synchronize()
    lado = torch.cuda.Stream()
    with torch.cuda.stream(lado):
        otra = paso()
    lado.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(base, otra))
