"""The per-channel convolution and the selective scan against their formulas in 64 bits, term by term: the tolerances are
those of fp32 sums whose terms' magnitudes the same formulas add up (`magnitud`), and half a step of the output's type."""
import pytest
import torch

import asrn_amd
from asrn_amd import _lib

pytestmark = pytest.mark.gpu
DEV = 'cuda'
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24                     # half a step of fp32


@pytest.fixture(autouse=True)
def semilla():
    torch.manual_seed(0)


def r(*forma, dt=F32):
    return torch.randn(*forma, device=DEV).to(dt)


def cerca(x, ref, termino, n, nombre):
    """|x - ref| within n roundings of fp32 on the sum of the terms' magnitudes and half a step of x's type."""
    assert x.shape == ref.shape, (nombre, x.shape, ref.shape)
    medio = torch.finfo(x.dtype).eps / 2
    # below the type's normal range a step is its smallest subnormal
    cota = n * U * termino + medio * (ref.abs() + n * U * termino) + torch.finfo(x.dtype).smallest_normal * 2 * medio
    mal = (x.double() - ref).abs() > cota
    assert not mal.any(), (nombre, int(mal.sum()), ((x.double() - ref).abs() / cota.clamp(min=1e-300)).max().item())


# ---------------------------------------------------------------------------------------------------------------------
# the convolution
# ---------------------------------------------------------------------------------------------------------------------

def act64(x, act):
    if act == 'gelu':
        fi = 0.5 * torch.erfc(-x / 2 ** 0.5)
        return x * fi, fi + x * torch.exp(-x * x / 2) / (2 * torch.pi) ** 0.5
    if act == 'silu':
        s = torch.sigmoid(x)
        return x * s, s * (1 + x * (1 - s))
    return x, torch.ones_like(x)


def conv64(z, w, b, gy, act):
    """y, dz, dw, db and the sums of their terms' magnitudes."""
    z, gy = z.double(), gy.double()
    d, k = z.shape[2], w.shape[-1]
    w = w.double().reshape(d, k)
    b = torch.zeros(d, device=DEV, dtype=torch.float64) if b is None else b.double()
    v = torch.nn.functional.pad(z, (0, 0, k - 1, 0)).unfold(1, k, 1)
    pre, pre_m = (v * w).sum(-1) + b, (v * w).abs().sum(-1) + b.abs()
    y, der = act64(pre, act)
    # the pre-activation's error reaches y through a slope of at most 1.13 and the derivative through one of at most 0.8
    g = gy * der
    g_m = gy.abs() * (der.abs() + 1 + pre_m)
    y_m = 1.13 * pre_m + y.abs()

    def atras(g, w, v):
        gp = torch.nn.functional.pad(g, (0, 0, 0, k - 1)).unfold(1, k, 1)             # g[t .. t + k - 1]
        return (gp * w.flip(-1)).sum(-1), torch.einsum('bld,bldk->dk', g, v), g.sum((0, 1))
    return (y, *atras(g, w, v)), (y_m, *atras(g_m, w.abs(), v.abs()))


CONVS = [(2, 1, 8, 4, 'silu', F32), (1, 3, 1, 4, None, BF16), (3, 50, 12, 1, 'gelu', F32), (2, 37, 64, 2, 'gelu', BF16),
         (2, 129, 20, 4, 'silu', F16), (1, 300, 36, 3, None, F32), (2, 65, 7, 7, 'gelu', F32), (1, 40, 8, 8, 'silu', BF16),
         (2, 33, 5, 16, 'gelu', F32), (2, 33, 16, 11, 'silu', F16), (1, 2, 260, 9, None, F32), (5, 700, 128, 4, 'silu', BF16)]


@pytest.mark.parametrize('B,L,d,k,act,dt', CONVS)
@pytest.mark.parametrize('con_sesgo', [True, False])
def test_conv_canal(B, L, d, k, act, dt, con_sesgo):
    z, w = r(B, L, d, dt=dt).requires_grad_(), (r(d, 1, k) * k ** -0.5).requires_grad_()
    b, gy = r(d).requires_grad_() if con_sesgo else None, r(B, L, d, dt=dt)
    y = asrn_amd.conv_canal(z, w, b, act)
    assert y.dtype == dt and y.is_contiguous()
    gs = torch.autograd.grad(y, [t for t in (z, w, b) if t is not None], gy)
    (yr, dz, dw, db), (ym, dzm, dwm, dbm) = conv64(z.detach(), w.detach(), None if b is None else b.detach(), gy, act)
    # roundings: k + 1 of the sum, about 8 of the activation or its derivative
    n = k + 12
    cerca(y.detach(), yr, ym, n, 'y')
    cerca(gs[0], dz, dzm, n + k, 'dz')
    cerca(gs[1], dw.view(d, 1, k), dwm.view(d, 1, k), n + B * L, 'dw')
    if con_sesgo:
        cerca(gs[2], db, dbm, n + B * L, 'db')


def test_conv_canal_differences():
    """The gradients against differences of the forward in fp32: a step of 2^-6 leaves 2^-12 / 6 of curvature and 2^-18 of
    rounding a value, both below 1e-3 of gradients around 1."""
    z, w, b = r(2, 9, 5).requires_grad_(), r(5, 4).requires_grad_(), r(5).requires_grad_()
    gy = r(2, 9, 5)
    f = lambda *a: (asrn_amd.conv_canal(*a, 'gelu').double() * gy.double()).sum()
    gs = torch.autograd.grad(f(z, w, b), (z, w, b))
    e = 2.0 ** -6
    for i, t in enumerate((z, w, b)):
        v = r(*t.shape)
        mas, menos = [[s.detach() + (sg * e * v if j == i else 0) for j, s in enumerate((z, w, b))] for sg in (1, -1)]
        dif = (f(*mas) - f(*menos)) / (2 * e)
        assert abs(dif - (gs[i].double() * v.double()).sum()) <= 2e-3 * (1 + (gs[i] * v).abs().sum().item())


@pytest.mark.parametrize('forma', ['columnas', 'traspuesta', 'expandida', 'desplazada'])
def test_conv_canal_strides(forma):
    B, L, d, k = 3, 41, 24, 4
    z = {'columnas': lambda: r(B, L, 3 * d)[..., d:2 * d], 'traspuesta': lambda: r(B, d, L).transpose(1, 2),
         'expandida': lambda: r(1, L, d).expand(B, L, d), 'desplazada': lambda: r(B * L * d + 1)[1:].view(B, L, d)}[forma]()
    w, b = r(d, k), r(d)
    assert torch.equal(asrn_amd.conv_canal(z, w, b, 'gelu'), asrn_amd.conv_canal(z.contiguous().clone(), w, b, 'gelu'))
    zg, zc = z.detach().requires_grad_(), z.detach().contiguous().clone().requires_grad_()
    gy = r(B, L, d)
    g1, g2 = (torch.autograd.grad(asrn_amd.conv_canal(t, w, b, 'silu'), t, gy)[0] for t in (zg, zc))
    assert torch.equal(g1, g2)


@pytest.mark.parametrize('dt', [F32, BF16, F16])
@pytest.mark.parametrize('k', [1, 2, 4, 16])
def test_conv_canal_step_is_the_text(dt, k):
    B, L, d = 3, 20, 37
    z, w, b = r(B, L, d, dt=dt), r(d, k), r(d)
    y = asrn_amd.conv_canal(z, w, b, 'silu')
    v = torch.zeros(B, d, k - 1, device=DEV, dtype=dt)
    for t in range(L):
        antes = v.clone()
        y1, v1 = asrn_amd.paso_conv_canal(z[:, t], v, w, b, 'silu', en_sitio=False)
        assert torch.equal(v, antes)
        yt, v = asrn_amd.paso_conv_canal(z[:, t], v, w, b, 'silu')
        assert torch.equal(y1, yt) and torch.equal(v1, v)
        # the taps are added in another order
        m = (torch.nn.functional.pad(z.double(), (0, 0, k - 1, 0))[:, t:t + k].transpose(1, 2) * w.double()).abs().sum(-1)
        cerca(yt, y[:, t].double(), 1.13 * (m + b.double().abs()) + y[:, t].double().abs() / torch.finfo(F32).eps
              * torch.finfo(dt).eps, 2 * k + 24, t)


def test_conv_canal_empty_and_nonfinite():
    w, b = r(6, 3), r(6)
    for B, L in ((0, 5), (2, 0)):
        z = r(B, L, 6).requires_grad_()
        wg = w.clone().requires_grad_()
        y = asrn_amd.conv_canal(z, wg, b, 'gelu')
        assert y.shape == (B, L, 6)
        gz, gw = torch.autograd.grad(y.sum(), (z, wg))
        assert gz.shape == z.shape and not gw.any()
    # a NaN or an infinity reaches the k outputs whose window holds it, no others
    for malo in (float('nan'), float('inf')):
        z = r(1, 30, 8)
        z[0, 11, 3] = malo
        y = asrn_amd.conv_canal(z, r(8, 3), r(8))
        fin = torch.isfinite(y)
        assert not fin[0, 11:14, 3].any() and fin.sum() == y.numel() - 3


# ---------------------------------------------------------------------------------------------------------------------
# the scan
# ---------------------------------------------------------------------------------------------------------------------

def escaneo64(u, dl, A, Bm, C, D, z, sesgo, h0, gy, gh, sp, magnitud=False):
    """y, the last state and the gradients (u, dl, A, Bm, C, D, z, sesgo, h0), token by token; magnitud: with every term
    replaced by its magnitude."""
    m = (lambda x: None if x is None else x.double().abs()) if magnitud else (lambda x: None if x is None else x.double())
    B, L, d = u.shape
    N = A.shape[1]
    cero = torch.zeros(d, device=u.device, dtype=torch.float64)
    x = dl.double() + (cero if sesgo is None else sesgo.double())
    dt = torch.nn.functional.softplus(x, threshold=1e9) if sp else x
    ddt = torch.sigmoid(x) if sp else torch.ones_like(x)
    a = torch.exp(dt[..., None] * A.double())
    dtm = dt.abs() if magnitud else dt
    if magnitud and sp:
        # the hardware's exponential and reciprocal give 0 for results below 2^-126 (no subnormals): softplus and its
        # derivative are off by up to that besides their roundings, so their magnitudes are at least 2^-126 of roundings, U each
        dtm, ddt = dtm + 2.0 ** -126 / U, ddt + 2.0 ** -126 / U
    uu, Bv, Cv, Dv = m(u), m(Bm), m(C), cero if D is None else m(D)
    s = torch.ones_like(x) if z is None else torch.sigmoid(z.double())
    puerta = torch.ones_like(x) if z is None else z.double() * s
    dpuerta = s * (1 + (0 if z is None else z.double()) * (1 - s))
    if magnitud:
        # silu' = s (1 + z (1 - s)) is a sum of two terms that cancel at z = -1.278, where its own value says nothing of its
        # rounding: their magnitudes add up to s (1 + |z| (1 - s))
        puerta, dpuerta = puerta.abs(), s * (1 + (0 if z is None else z.double().abs()) * (1 - s))
    h = torch.zeros(B, d, N, device=u.device, dtype=torch.float64) if h0 is None else m(h0)
    hs, ys = [h], []
    for t in range(L):
        h = a[:, t] * h + (dtm[:, t] * uu[:, t])[..., None] * Bv[:, t, None]
        hs.append(h)
        ys.append((h * Cv[:, t, None]).sum(-1) + Dv * uu[:, t])
    y0 = torch.stack(ys, 1) if L else torch.zeros(B, 0, d, device=u.device, dtype=torch.float64)
    if gy is None:
        return y0 * puerta, h
    g = m(gy) * puerta
    G = torch.zeros_like(h) if gh is None else m(gh)
    du, ddl, dB, dC = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(Bv), torch.zeros_like(Cv)
    dA = torch.zeros_like(A, dtype=torch.float64)
    Av = m(A)
    for t in reversed(range(L)):
        G = G + g[:, t, :, None] * Cv[:, t, None]
        dC[:, t] = (g[:, t, :, None] * hs[t + 1]).sum(1)
        dB[:, t] = (G * (dtm[:, t] * uu[:, t])[..., None]).sum(1)
        ds = (G * Bv[:, t, None]).sum(-1)
        w = G * a[:, t] * hs[t]
        dA += (w * dtm[:, t, :, None]).sum(0)
        ddl[:, t] = ((w * Av).sum(-1) + ds * uu[:, t]) * ddt[:, t]
        du[:, t] = ds * dtm[:, t] + g[:, t] * Dv
        G = G * a[:, t]
    dz = None if z is None else m(gy) * y0 * dpuerta
    return (y0 * puerta, h, du, ddl, dA, dB, dC, None if D is None else (g * uu).sum((0, 1)), dz,
            None if sesgo is None else ddl.sum((0, 1)), None if h0 is None else G)


NOMBRES = ('y', 'fin', 'u', 'delta', 'A', 'Bm', 'C', 'D', 'puerta', 'sesgo', 'estado')


def entradas(B, L, d, N, dt, D=True, puerta=True, sesgo=True, estado=True, sp=True):
    """u, delta, A, Bm, C, D, puerta, sesgo, estado with decays from one token to hundreds."""
    A = -torch.rand(d, N, device=DEV) * 4 - 0.01
    tau = torch.logspace(0, 2.5, d, device=DEV)
    dl = r(B, L, d, dt=dt) if sp else (r(B, L, d).abs() / 8).to(dt)
    return [r(B, L, d, dt=dt), dl, A, r(B, L, N, dt=dt), r(B, L, N, dt=dt), r(d) if D else None, r(B, L, d, dt=dt) if puerta else None,
            (torch.log(torch.expm1(1 / tau)) if sp else 0.01 + torch.rand(d, device=DEV) / 8) if sesgo else None,
            r(B, d, N) if estado else None]


def llamar(e, **kw):
    u, dl, A, Bm, C, D, z, s, h0 = e
    return asrn_amd.escaneo_selectivo(u, dl, A, Bm, C, D=D, puerta=z, sesgo_delta=s, estado=h0, **kw)


def revisar(e, gy, gh, sp=True, con_fin=True, transformar=lambda t: t):
    hojas = [None if t is None else t.detach().requires_grad_() for t in e]
    y, fin = llamar([None if t is None else transformar(t) for t in hojas], devolver_estado=True, softplus=sp)
    pide = [t for t in hojas if t is not None]
    salidas, gs = ((y, fin), (gy, gh)) if con_fin else ((y,), (gy,))
    gr = iter(torch.autograd.grad(salidas, pide, gs))
    got = [y.detach(), fin.detach()] + [None if t is None else next(gr) for t in hojas]
    ref = escaneo64(*e, gy, gh if con_fin else None, sp)
    mag = escaneo64(*e, gy, gh if con_fin else None, sp, magnitud=True)
    L = e[0].shape[1]
    # a term passes up to L decays, each off by 3 roundings and, times the decay's exponent, 8 more (softplus, the product, the
    # exponential's); a wave's and the workgroups' sums add the channels, the parameters' sums all tokens
    n = 4 * L + 64 + e[0].shape[2] // 4 + e[0].shape[0] * L // 4
    for nombre, x, v, m in zip(NOMBRES, got, ref, mag):
        assert (x is None) == (v is None), nombre
        if x is not None:
            cerca(x, v, m, n, nombre)
    return got


@pytest.mark.parametrize('B,L,d,N,dt', [
    (1, 1, 1, 1, F32), (2, 1, 64, 16, BF16), (3, 7, 5, 3, F32), (2, 8, 65, 16, F32), (1, 9, 130, 8, F16), (2, 63, 20, 11, F32),
    (2, 64, 64, 16, BF16), (1, 65, 300, 17, F32), (3, 200, 70, 16, F32), (2, 333, 33, 32, BF16), (1, 1000, 12, 5, F32),
    (1, 129, 520, 9, F32), (9, 40, 257, 2, BF16), (2, 170, 100, 24, F32), (1, 90, 64, 25, BF16), (2, 77, 130, 20, F16)])
def test_escaneo_selectivo(B, L, d, N, dt):
    e = entradas(B, L, d, N, dt)
    revisar(e, r(B, L, d, dt=dt), r(B, d, N))


@pytest.mark.parametrize('falta', ['D', 'puerta', 'sesgo', 'estado', 'todo'])
@pytest.mark.parametrize('sp', [True, False])
def test_escaneo_selectivo_without(falta, sp):
    B, L, d, N = 2, 150, 40, 6
    kw = {n: falta not in (n, 'todo') for n in ('D', 'puerta', 'sesgo', 'estado')}
    revisar(entradas(B, L, d, N, F32, sp=sp, **kw), r(B, L, d), None, sp=sp, con_fin=False)


def test_escaneo_selectivo_gradient_of_the_state_alone():
    e = entradas(2, 70, 9, 4, F32)
    hojas = [t.detach().requires_grad_() for t in e]
    fin = llamar(hojas, devolver_estado=True)[1]
    gh = r(2, 9, 4)
    gs = torch.autograd.grad(fin, hojas, gh, allow_unused=True)
    ref = escaneo64(*e, torch.zeros(2, 70, 9, device=DEV), gh, True)
    mag = escaneo64(*e, torch.zeros(2, 70, 9, device=DEV), gh, True, magnitud=True)
    for nombre, x, v, m in zip(NOMBRES[2:], gs, ref[2:], mag[2:]):
        cerca(x, v, m, 4 * 70 + 64 + 35, nombre)


def test_escaneo_selectivo_differences():
    e = [t.detach().requires_grad_() for t in entradas(2, 21, 5, 3, F32)]
    gy, gh = r(2, 21, 5), r(2, 5, 3)

    def f(a):
        y, h = llamar(a, devolver_estado=True)
        return (y.double() * gy.double()).sum() + (h.double() * gh.double()).sum()
    gs = torch.autograd.grad(f(e), e)
    paso = 2.0 ** -8               # curvature 2^-16 / 6 and rounding 2^-16, times third derivatives and sums of a few units
    for i, t in enumerate(e):
        v = r(*t.shape)
        mas, menos = [[s.detach() + (sg * paso * v if j == i else 0) for j, s in enumerate(e)] for sg in (1, -1)]
        dif = (f(mas) - f(menos)) / (2 * paso)
        assert abs(dif - (gs[i].double() * v.double()).sum()) <= 5e-3 * (1 + (gs[i] * v).abs().sum().item()), NOMBRES[i + 2]


def test_escaneo_selectivo_strides():
    """Slices of wider projections, an expanded text, a transposed gate."""
    B, L, d, N = 3, 90, 24, 5
    ancho, proy = r(B, L, 2 * d + 1), r(B, L, 3 + 2 * N)
    _, _, A, _, _, D, _, s, h0 = entradas(B, L, d, N, F32)
    e = [ancho[..., 1:d + 1], r(1, L, d).expand(B, L, d), A, proy[..., 3:3 + N], proy[..., 3 + N:], D,
         r(B, d, L).transpose(1, 2), s, h0]
    gy, gh = r(B, L, d), r(B, d, N)
    got = revisar(e, gy, gh)
    denso = revisar([t.contiguous().clone() for t in e], gy, gh)
    for a, b in zip(got, denso):
        assert torch.equal(a, b)


@pytest.mark.parametrize('cortes', [(1,), (64, 65), (100, 200, 299)])
def test_escaneo_selectivo_in_pieces(cortes):
    """A text in pieces, the state handed on, is the text in one."""
    B, L, d, N = 2, 300, 50, 16
    e = entradas(B, L, d, N, F32)
    y, fin = llamar(e, devolver_estado=True)
    ys, h, mag = [], e[-1], escaneo64(*e, None, None, True, magnitud=True)
    for i, j in zip((0, *cortes), (*cortes, L)):
        trozo = [t[:, i:j] if n in (0, 1, 3, 4, 6) else t for n, t in enumerate(e[:-1])] + [h]
        y1, h = llamar(trozo, devolver_estado=True)
        ys.append(y1)
    cerca(torch.cat(ys, 1), y.double(), mag[0], 8 * L + 64, 'y')
    cerca(h, fin.double(), mag[1], 8 * L + 64, 'fin')


@pytest.mark.parametrize('N,dt', [(16, F32), (3, F32), (32, BF16), (1, F16)])
def test_paso_selectivo_is_the_text(N, dt):
    B, L, d = 3, 12, 37
    u, dl, A, Bm, C, D, z, s, h = entradas(B, L, d, N, dt)
    y, fin = llamar([u, dl, A, Bm, C, D, z, s, h], devolver_estado=True)
    ref, href = escaneo64(u, dl, A, Bm, C, D, z, s, h, None, None, True)
    ym, hm = escaneo64(u, dl, A, Bm, C, D, z, s, h, None, None, True, magnitud=True)
    h = h.clone()
    for t in range(L):
        kw = dict(D=D, puerta=z[:, t], sesgo_delta=s)
        antes = h.clone()
        y1, h1 = asrn_amd.paso_selectivo(u[:, t], dl[:, t], A, Bm[:, t], C[:, t], h, **kw, en_sitio=False)
        assert torch.equal(h, antes)
        yt, h2 = asrn_amd.paso_selectivo(u[:, t], dl[:, t], A, Bm[:, t], C[:, t], h, **kw)
        assert h2 is h or h2.data_ptr() == h.data_ptr()
        assert torch.equal(y1, yt) and torch.equal(h1, h)
        cerca(yt, ref[:, t], ym[:, t], 4 * L + 64, t)
    cerca(h, href, hm, 4 * L + 64, 'fin')


def test_escaneo_selectivo_empty():
    for B, L in ((0, 4), (2, 0)):
        e = entradas(B, L, 6, 3, F32)
        hojas = [t.detach().requires_grad_() for t in e]
        y, fin = llamar(hojas, devolver_estado=True)
        assert y.shape == (B, L, 6) and torch.equal(fin, e[-1])
        gs = torch.autograd.grad(y.sum() + (2 * fin).sum(), hojas)
        assert all(g.shape == t.shape for g, t in zip(gs, hojas))
        assert torch.equal(gs[-1], torch.full_like(e[-1], 2.0)) and not any(g.any() for g in gs[:-1])
        y, fin = llamar([*e[:-1], None], devolver_estado=True)
        assert not fin.any()


def test_escaneo_selectivo_extremes():
    """Step sizes from 0 to 1e4 and states that decay at once: no NaN, and the values of the formula."""
    B, L, d, N = 1, 80, 8, 4
    e = entradas(B, L, d, N, F32, sesgo=False)
    e[1] = torch.linspace(-200, 200, L, device=DEV)[None, :, None].expand(B, L, d).contiguous()
    e[1][:, -1] = 1e4
    got = revisar(e, r(B, L, d), r(B, d, N))
    assert all(torch.isfinite(t).all() for t in got if t is not None)
    # a NaN stays in its channel, from its token on; the tokens before it and the other channels are as they were
    e2 = [None if t is None else t.clone() for t in e]
    e2[0][0, 40, 3] = float('nan')
    y, y2 = llamar(e), llamar(e2)
    assert torch.equal(y[:, :40], y2[:, :40]) and torch.isnan(y2[0, 40:, 3]).any()
    resto = [c for c in range(d) if c != 3]
    assert torch.equal(y[..., resto], y2[..., resto])


def test_second_gradient_is_refused():
    z, w = r(2, 5, 4).requires_grad_(), r(4, 2)
    e = [t.detach().requires_grad_() for t in entradas(1, 5, 4, 2, F32)]
    for y, x in ((asrn_amd.conv_canal(z, w), z), (llamar(e), e[0])):
        with pytest.raises((RuntimeError, _lib.ASRNHipError), match='create_graph'):
            torch.autograd.grad(y.sum(), x, create_graph=True)


def test_steps_refuse_gradients():
    with pytest.raises(_lib.ASRNHipError, match='no_grad'):
        asrn_amd.paso_conv_canal(r(2, 4).requires_grad_(), r(2, 4, 2), r(4, 3))
    u, dl, A, Bm, C, D, z, s, h = entradas(2, 1, 4, 3, F32)
    with pytest.raises(_lib.ASRNHipError, match='no_grad'):
        asrn_amd.paso_selectivo(u[:, 0], dl[:, 0], A.requires_grad_(), Bm[:, 0], C[:, 0], h)


def test_steps_refuse_their_parameters_gradients():
    with pytest.raises(_lib.ASRNHipError, match='no_grad'):
        asrn_amd.paso_conv_canal(r(2, 4), r(2, 4, 2), r(4, 3), r(4).requires_grad_())
    u, dl, A, Bm, C, D, z, s, h = entradas(2, 1, 4, 3, F32)
    for de, con in ((D.detach().requires_grad_(), s), (D, s.detach().requires_grad_())):
        with pytest.raises(_lib.ASRNHipError, match='no_grad'):
            asrn_amd.paso_selectivo(u[:, 0], dl[:, 0], A, Bm[:, 0], C[:, 0], h, D=de, sesgo_delta=con)


def test_a_step_in_place_is_seen_by_a_graph_that_kept_its_state():
    p = r(2, 4, 3).requires_grad_()
    u, dl, A, Bm, C, D, z, s, h = entradas(2, 1, 4, 3, F32)
    for estado, paso in ((r(2, 4, 3), lambda v: asrn_amd.paso_conv_canal(u[:, 0], v, r(4, 4))),
                         (h, lambda v: asrn_amd.paso_selectivo(u[:, 0], dl[:, 0], A, Bm[:, 0], C[:, 0], v))):
        q = (p * estado).sum()
        with torch.no_grad():
            paso(estado)
        with pytest.raises(RuntimeError, match='inplace'):
            q.backward()
        with torch.inference_mode():
            paso(estado.clone())


def test_infinite_decay():
    """A state of A = -inf forgets all but the newest token, also where the last tile and chunk are not whole."""
    for L in (5, 16, 37, 300):
        e = [t.detach() for t in entradas(1, L, 70, 3, F32)]
        e[2][:, 1] = -torch.inf
        e[2][3, 0] = -3e38              # beyond fp32 in units of the binary exponent
        hojas = [t.requires_grad_() for t in e]
        y, fin = llamar(hojas, devolver_estado=True)
        ult = [t[:, -1].detach().double() for t in (e[0], e[1], e[3])]
        dt = torch.nn.functional.softplus(ult[1] + e[7].detach().double())
        espera = dt * ult[0] * ult[2][:, 1:2]
        # 20 roundings of softplus from its exponential on, 10 of the exponential's argument (|x| < 10), the two products'
        cerca(fin[..., 1].detach(), espera, espera.abs(), 32, 'fin')
        gs = torch.autograd.grad(y.sum() + fin.sum(), hojas)
        assert y.isfinite().all() and all(g.isfinite().all() for i, g in enumerate(gs) if i != 2)


def test_captured_and_replayed():
    """A training call of both in a graph, replayed on new values with eager work between, on another stream than theirs."""
    B, L, d, N, k = 2, 200, 70, 16, 4
    e = [t.detach().requires_grad_() for t in entradas(B, L, d, N, F32, estado=False) if t is not None]
    w, b, gy = r(d, k).requires_grad_(), r(d).requires_grad_(), r(B, L, d)

    def paso():
        u, dl, A, Bm, C, D, z, s = e
        c = asrn_amd.conv_canal(u, w, b, 'silu')
        y = asrn_amd.escaneo_selectivo(c, dl, A, Bm, C, D=D, puerta=z, sesgo_delta=s)
        return [y.detach(), *torch.autograd.grad(y, [*e, w, b], gy)]
    lado = torch.cuda.Stream()
    lado.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(lado):
        paso()
    torch.cuda.current_stream().wait_stream(lado)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        fijos = paso()
    for i in range(4):
        with torch.no_grad():
            e[0].copy_(r(B, L, d))
            gy.copy_(r(B, L, d))
        eager = [t.clone() for t in paso()]
        g.replay()
        torch.cuda.synchronize()
        for a, v in zip(fijos, eager):
            assert torch.equal(a, v), i


def test_same_bits_again_and_on_another_stream():
    e = entradas(3, 500, 200, 16, BF16)
    gy, gh = r(3, 500, 200, dt=BF16), r(3, 200, 16)

    def todo():
        hojas = [t.detach().requires_grad_() for t in e]
        y, h = llamar(hojas, devolver_estado=True)
        return [y.detach(), h.detach(), *torch.autograd.grad((y, h), hojas, (gy, gh))]
    uno = todo()
    lado = torch.cuda.Stream()
    lado.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(lado):
        dos = todo()
    tres = todo()
    torch.cuda.synchronize()
    for a, b, c in zip(uno, dos, tres):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_offsets_past_32_bits():
    """Texts of more than 2^31 values: the end of the last one against the same tokens alone. Steps of 5 and more forget what lies
    100 tokens back (exp(-500)); both round once to bf16 from fp32 values some 2^-18 apart."""
    B, L, d, N, m = 2, 2 ** 20 + 19, 1024, 4, 128
    u, dl = (torch.empty(B, L, d, device=DEV, dtype=BF16).normal_() for _ in range(2))
    dl += 9
    Bm, C, A = r(B, L, N, dt=BF16), r(B, L, N, dt=BF16), -1 - torch.rand(d, N, device=DEV)
    fin = [t[1:, -m:].clone() for t in (u, dl, Bm, C)]
    with torch.no_grad():
        w, b = r(d, 4), r(d)
        c = asrn_amd.conv_canal(u, w, b, 'silu')
        assert torch.equal(c[1, -m + 3:], asrn_amd.conv_canal(fin[0], w, b, 'silu')[0, 3:])
        del c
        y = asrn_amd.escaneo_selectivo(u, dl, A, Bm, C)[1, -20:].double()
    torch.cuda.empty_cache()
    hojas = [t.requires_grad_() for t in fin]
    ref = asrn_amd.escaneo_selectivo(hojas[0], hojas[1], A, hojas[2], hojas[3])[0, -20:].detach().double()
    assert ((y - ref).abs() <= 2 ** -7 * ref.abs() + 2 ** -14 * ref.abs().max()).all()
    # the gradients of the last tokens from a gradient of theirs alone
    for t in (u, dl, Bm, C):
        t.requires_grad_()
    gy = r(20, d, dt=BF16)
    largo = torch.autograd.grad(asrn_amd.escaneo_selectivo(u, dl, A, Bm, C)[1, -20:], (u, dl, Bm, C), gy)
    corto = torch.autograd.grad(asrn_amd.escaneo_selectivo(hojas[0], hojas[1], A, hojas[2], hojas[3])[0, -20:], hojas, gy)
    for a, b in zip(largo, corto):
        a, b = a[1, -20:].double(), b[0, -20:].double()
        assert ((a - b).abs() <= 2 ** -7 * b.abs() + 2 ** -14 * b.abs().max()).all()
        assert not largo[0][0].any()
    torch.cuda.empty_cache()


@pytest.mark.parametrize('L', [5, 37, 64, 301])
def test_tokens_past_a_texts_end_enter_no_gradient(L):
    """States that forget at once, by a decay of -inf, one beyond fp32 in units of the binary exponent and one of -1e7 (step sizes
    of 2^-16 and more: exp(-150) is 0), and a gradient of the last state in the hundreds: the same bits from each, also where
    the last tile is not whole."""
    e = [t.detach() for t in entradas(1, L, 70, 3, F32)]
    gy, gh = r(1, L, 70), 300 * r(1, 70, 3)

    def todo(uno, otro):
        e[2][:, 1], e[2][3, 0] = uno, otro
        hojas = [t.clone().requires_grad_() for t in e]
        y, fin = llamar(hojas, devolver_estado=True)
        return y.detach(), fin.detach(), *torch.autograd.grad((y, fin), hojas, (gy, gh))
    for nombre, a, b in zip(NOMBRES, todo(-1e7, -1e7), todo(-torch.inf, -3e38)):
        assert b.isfinite().all() and torch.equal(a, b), nombre


def test_forward_tangents_are_refused():
    import torch.autograd.forward_ad as fwd
    z, w, b = r(2, 5, 4), r(4, 3), r(4)
    e = [t.detach() for t in entradas(2, 5, 4, 3, F32)]
    u, dl, A, Bm, C, D, p, s, h = e
    casos = [(lambda *a: asrn_amd.conv_canal(*a, 'silu'), (z, w, b)), (lambda *a: llamar(a), e),
             (lambda *a: asrn_amd.paso_conv_canal(a[0], a[1], a[2], a[3]), (z[:, 0], r(2, 4, 2), w, b)),
             (lambda *a: asrn_amd.paso_selectivo(a[0], a[1], a[2], a[3], a[4], a[5], D=a[6], puerta=a[7], sesgo_delta=a[8]),
              (u[:, 0], dl[:, 0], A, Bm[:, 0], C[:, 0], h, D, p[:, 0], s))]
    for f, args in casos:
        for i in range(len(args)):
            for grad in (True, False):
                with fwd.dual_level(), torch.set_grad_enabled(grad):
                    dual = [fwd.make_dual(t.clone(), torch.ones_like(t)) if j == i else t for j, t in enumerate(args)]
                    with pytest.raises(RuntimeError, match='jvp|forward'):
                        f(*dual)


def lejos(t):
    """t (B, 1, .) as a token-major text of that many values has it: the stride of its one token is 2^24 and more."""
    return torch.as_strided(t.contiguous(), t.shape, (t.stride(0), 2 ** 24 + 8, 1))


@pytest.mark.parametrize('dt', [F32, BF16])
def test_one_token_of_any_stride(dt):
    B, d, N = 3, 24, 5
    e = entradas(B, 1, d, N, dt)
    gy, gh = r(B, 1, d, dt=dt), r(B, d, N)

    def todo(f):
        hojas = [f(t.detach()).requires_grad_() if n in (0, 1, 3, 4, 6) else t.detach().requires_grad_() for n, t in enumerate(e)]
        y, fin = llamar(hojas, devolver_estado=True)
        return y.detach(), fin.detach(), *torch.autograd.grad((y, fin), hojas, (f(gy), gh))
    for nombre, a, b in zip(NOMBRES, todo(lambda t: t.clone()), todo(lejos)):
        assert torch.equal(a, b), nombre
    # no text of such strides
    hojas = [t.detach()[:0].requires_grad_() if n in (8,) else lejos(t.detach())[:0].requires_grad_() if n in (0, 1, 3, 4, 6)
             else t for n, t in enumerate(e)]
    y, fin = llamar(hojas, devolver_estado=True)
    assert y.shape == (0, 1, d) and torch.autograd.grad(y.sum() + fin.sum(), hojas[0])[0].shape == (0, 1, d)
    z, w = e[0], r(d, 4)
    assert torch.equal(asrn_amd.conv_canal(lejos(z), w), asrn_amd.conv_canal(z, w))


@pytest.mark.parametrize('B,L,d,k,act,dt', [(2, 9001, 768, 4, 'silu', BF16), (2, 9001, 768, 3, 'gelu', F32),
                                            (1, 3301, 1021, 7, None, F32), (3, 1501, 801, 4, 'silu', F16)])
def test_conv_canal_in_long_pieces(B, L, d, k, act, dt):
    """So many values that a piece has more than the 16 tokens of the smallest ones (12.6 M of four channels a lane, 3.1 M of one)."""
    test_conv_canal(B, L, d, k, act, dt, True)
