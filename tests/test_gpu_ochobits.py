"""Activations in 8 bits: the format bit for bit against its definition, the LayerNorm, the GELU and the products that
read it back against float64 at the 8-bit values, and local blocks and models that train with it.

Tolerances: u = 2^-24, half a step of fp32; a 16-bit result adds half a step of its own. The GELU's derivative and the
GELU read back come from an approximation of erfc within 1.5e-7 (Abramowitz and Stegun 7.1.26) with a handful of fp32
roundings: 4e-7 of a derivative of order 1 and 4e-7 (1 + |u|) of the GELU."""
import math

import pytest
import torch
import torch.nn.functional as F

import asrn_amd
from asrn_amd import ops
from asrn_amd.lineal import lineal, lineal8

pytestmark = pytest.mark.gpu
DEV = 'cuda'
U = 2.0 ** -24


def ocho(x):
    """(codes, scale bytes, values) of x (..., d) from the definition, in float64 on the CPU."""
    v = x.detach().double().cpu().reshape(-1, x.shape[-1])
    N, d = v.shape
    g = F.pad(v, (0, -d % 32)).view(N, -1, 32)
    top = g.abs().amax(-1, keepdim=True)
    # past 127 2^121 the smallest scale is 2^122 and the integer 64, which stands for 2^128: no fp32 value
    mal = ~(top <= 127 * 2.0 ** 121)
    e = torch.where(mal | (top == 0), torch.full_like(top, -126.0), torch.ceil(torch.log2(torch.where(mal, 1.0, top) / 127)))
    e = torch.where(torch.ldexp(torch.ones_like(e), e.int()) * 127 < torch.where(mal, 0.0, top), e + 1, e)      # log2's rounding
    e = torch.where(torch.ldexp(torch.ones_like(e), e.int() - 1) * 127 >= torch.where(mal, 1e300, top), e - 1, e).clamp(min=-126)
    dos = torch.ldexp(torch.ones_like(e), e.int())
    q = torch.where(mal, 0.0, torch.round(torch.where(mal, 0.0, g) / dos))
    val = torch.where(mal, math.nan, q * dos)
    byte = torch.where(mal, 255.0, e + 127)[..., 0]
    return q.reshape(N, -1)[:, :d].to(torch.int8), byte.to(torch.uint8), val.reshape(N, -1)[:, :d].view(x.shape)


def gelu64(v):
    return v * 0.5 * torch.erfc(-v / math.sqrt(2))


def dgelu64(v):
    return 0.5 * torch.erfc(-v / math.sqrt(2)) + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)


def dentro(a, b, tol):
    """|a - b| <= tol, and NaN in the same places."""
    a, b = a.double().cpu(), b.double().cpu()
    assert torch.equal(a.isnan(), b.isnan())
    d = torch.where(b.isnan() | (a == b), 0.0, (a - b).abs())
    assert (d <= torch.as_tensor(tol).double().cpu()).all(), (d - torch.as_tensor(tol).double().cpu()).max()


@pytest.mark.parametrize('N,d', [(1, 1), (3, 7), (5, 8), (2, 31), (7, 32), (4, 33), (65, 40), (33, 260), (9, 1024), (3, 1537), (700, 96)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_format(N, d, dtype):
    g = torch.Generator(device=DEV).manual_seed(N * d)
    x = torch.randn(N, d, generator=g, device=DEV) * torch.exp(4 * torch.randn(N, 1, generator=g, device=DEV))
    x[0, d // 2] = 0.0
    x = x.to(dtype)
    q, e = ops.guardar8(x)
    q0, e0, v0 = ocho(x)
    assert torch.equal(q.cpu(), q0) and torch.equal(e.cpu(), e0)
    assert torch.equal(ops.leer8(q, e).cpu().double(), v0)
    assert torch.equal(ops.leer8(q, e, torch.bfloat16).cpu().double(), v0)            # exact in bf16
    assert ((v0 - x.cpu().double()).abs() <= 2.0 ** (e0.double() - 128).repeat_interleave(32, 1)[:, :d]).all()


def test_format_extremes():
    """Powers of two at the border of a scale, ties, the ends of fp32, zeros, infinities and NaN, the neighbours kept."""
    x = torch.zeros(14, 64, device=DEV)
    x[0, 0] = 127.0                                  # 127 2^0 exactly
    x[1, 0] = torch.nextafter(torch.tensor(127.0), torch.tensor(200.0)).item()
    x[2, :4] = torch.tensor([127.0, 0.5, 1.5, -2.5])                # ties to even
    x[3, 0], x[3, 32] = torch.finfo(torch.float32).max, torch.finfo(torch.float32).tiny
    x[4, 5] = 1e-45
    x[5, :2] = torch.tensor([2.0 ** -126, -2.0 ** -127])
    x[6, 3] = math.inf
    x[7, 40] = math.nan
    x[8, 1] = -math.inf
    x[8, 33] = 5.0
    x[9] = 128.0
    x[10] = -127.5
    x[11, 0] = 254.0
    x[12, 0] = 254.00002
    x[13] = torch.finfo(torch.float32).min
    for t in (x, x.bfloat16()):
        q, e = ops.guardar8(t)
        q0, e0, v0 = ocho(t)
        assert torch.equal(q.cpu(), q0) and torch.equal(e.cpu(), e0)
        got = ops.leer8(q, e).cpu().double()
        assert torch.equal(got.isnan(), v0.isnan()) and torch.equal(got.nan_to_num(), v0.nan_to_num())
    assert e.cpu()[6].tolist() == [255, 1] and e.cpu()[7].tolist() == [1, 255]


@pytest.mark.parametrize('N,d', [(1, 4), (5, 33), (37, 64), (130, 260), (64, 1536), (3, 7)])
@pytest.mark.parametrize('dtype,gdt', [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)])
def test_gelu(N, d, dtype, gdt):
    g = torch.Generator(device=DEV).manual_seed(N + d)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    u = (2.5 * r(N, d)).to(dtype).requires_grad_()
    y, guardado = ops.gelu8(u)
    gy = r(N, d).to(gdt)
    du, = torch.autograd.grad(y, u, gy.to(y.dtype), retain_graph=True)
    v0 = ocho(u)[2].cpu()
    assert y.dtype == dtype and du.dtype == dtype and torch.equal(y.cpu(), F.gelu(u.detach()).cpu()) or dtype == torch.float32
    dentro(y.detach(), gelu64(u.detach().double()), 4 * U * (1 + u.detach().abs().double()) + torch.finfo(dtype).eps / 2 * y.detach().abs().double())
    ref = dgelu64(v0) * gy.to(y.dtype).double().cpu()
    dentro(du, ref, 4e-7 * gy.abs().double().cpu() + torch.finfo(dtype).eps / 2 * ref.abs())
    for dt in (torch.float32, torch.bfloat16):
        w = guardado.leer(guardado.tensores, dt)
        dentro(w, gelu64(v0).view(N, d), 4e-7 * (1 + v0.abs()).view(N, d) + torch.finfo(dt).eps / 2 * gelu64(v0).abs().view(N, d))
    h = (3 * r(N, d)).requires_grad_()               # the sum: gelu rounds to u's type first
    x = ops.suma_gelu8(h, u)
    gx = r(N, d)
    dh, du = torch.autograd.grad(x, (h, u), gx)
    assert torch.equal(dh, gx) and x.dtype == torch.float32
    dentro(x.detach(), h.detach().double() + gelu64(u.detach().double()),
           4 * U * (1 + u.detach().abs().double()) + U * x.detach().abs().double() + torch.finfo(dtype).eps / 2 * gelu64(u.detach().double()).abs())
    ref = dgelu64(v0) * gx.double().cpu()
    dentro(du, ref, 4e-7 * gx.abs().double().cpu() + torch.finfo(dtype).eps / 2 * ref.abs())


def test_gelu_far_values_and_differences():
    """The tails, where the value or the derivative vanishes; the derivative against central differences of the GELU."""
    u = torch.tensor([[-90.0, -14.0, -9.0, -6.0, -4.0, -1.0, -0.0, 0.0, 1e-30, 1.0, 4.0, 9.0, 60.0, 126.0, 3.0, -3.0] * 2], device=DEV, requires_grad=True)
    y, g8 = ops.gelu8(u)
    du, = torch.autograd.grad(y.sum(), u)
    v = ocho(u)[2]
    h = 1e-5
    dentro(du, (gelu64(v + h) - gelu64(v - h)) / (2 * h), 6e-7)
    dentro(g8.leer(g8.tensores, torch.float32), gelu64(v), 4e-7 * (1 + v.abs()))
    mal = torch.ones(2, 64, device=DEV)
    mal[0, 40], mal[1, 0] = math.inf, math.nan
    u = mal.requires_grad_()
    y, _ = ops.gelu8(u)
    du, = torch.autograd.grad(y.sum(), u)
    assert torch.isnan(du[0, 32:]).all() and torch.isnan(du[1, :32]).all() and torch.isfinite(du[0, :32]).all()


def norma64(x, w, b, eps):
    x = x.detach().double().cpu()
    mu = x.mean(-1, keepdim=True)
    s = ((x - mu) ** 2).mean(-1, keepdim=True).add(eps).rsqrt()
    return (x - mu) * s * w.double().cpu() + b.double().cpu(), mu, s


@pytest.mark.parametrize('forma,d', [((1,), 4), ((3, 11), 64), ((2, 33), 260), ((70,), 768), ((9,), 1024), ((5,), 1028),
                                     ((2, 3), 2048), ((35,), 2052), ((3,), 4096), ((33,), 8192), ((2,), 8200), ((7,), 10), ((33000,), 16)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_norm(forma, d, dtype):
    g = torch.Generator(device=DEV).manual_seed(d)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    ln = torch.nn.LayerNorm(d).to(DEV)
    with torch.no_grad():
        ln.weight.copy_(1 + 0.2 * r(d))
        ln.bias.copy_(0.2 * r(d))
    x = (r(*forma, d) * (1 + 3 * r(d).abs()) + 0.5).requires_grad_()
    y, alias, guardado = ops.norma8(ln, x, dtype)
    y0, mu, s = norma64(x, ln.weight.detach(), ln.bias.detach(), ln.eps)
    half = torch.finfo(dtype).eps / 2
    n = 40 + d / 64                                  # roundings of a row's sums and of the formula's steps
    assert y.dtype == dtype and torch.equal(alias.detach(), x.detach())
    dentro(y.detach(), y0, n * U * (1 + y0.abs() + (mu * s).abs()) + half * y0.abs())
    gy, gx = r(*forma, d).to(dtype), r(*forma, d)
    dx, dw, db = torch.autograd.grad((y, alias), (x, ln.weight, ln.bias), (gy, gx), retain_graph=True)
    xh = (ocho(x)[2] - mu) * s
    f, w = gy.double().cpu(), ln.weight.detach().double().cpu()
    p = f * w
    ref = s * (p - p.mean(-1, keepdim=True) - xh * (p * xh).mean(-1, keepdim=True)) + gx.double().cpu()
    tam = s * (p.abs() + p.abs().mean(-1, keepdim=True) + xh.abs() * (p * xh).abs().mean(-1, keepdim=True)) * (1 + (mu * s).abs())
    dentro(dx, ref, 4 * n * U * (tam + gx.double().cpu().abs()))
    filas = math.prod(forma)
    suma = lambda t: t.reshape(-1, d).sum(0)
    m = (n + filas ** 0.5 + 40) * U                  # sums over the rows in parts: at most 32 + the parts' roundings
    dentro(dw, suma(f * xh), 4 * m * suma((f * xh).abs() + f.abs() * (mu * s).abs()))
    dentro(db, suma(f), 4 * m * suma(f.abs()))
    for dt in (torch.float32, torch.bfloat16):       # formed again, for the next product
        yr = (xh * w + ln.bias.detach().double().cpu()).view(-1, d)
        dentro(guardado.leer(guardado.tensores, dt), yr, n * U * (1 + yr.abs() + (mu * s).abs().view(-1, 1)) + torch.finfo(dt).eps / 2 * yr.abs())


@pytest.mark.parametrize('B,L,d,k', [(2, 9, 64, 4), (3, 5, 20, 3), (1, 1, 8, 4), (2, 3, 36, 16), (2, 40, 12, 5), (1, 6, 10, 4), (2, 4, 1028, 2), (1, 3, 8196, 4), (2, 7, 64, 1)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_window(B, L, d, k, dtype):
    """The columns formed again against the window of the LayerNorm's output formed again."""
    g = torch.Generator(device=DEV).manual_seed(k)
    ln = torch.nn.LayerNorm(d).to(DEV)
    with torch.no_grad():
        ln.weight.copy_(1 + torch.randn(d, generator=g, device=DEV))
        ln.bias.copy_(torch.randn(d, generator=g, device=DEV))
    x = torch.randn(B, L, d, generator=g, device=DEV, requires_grad=True)
    z, _, guardado = ops.norma8(ln, x, torch.float32)
    cols, gc = ops.ventana8(z, k, dtype, guardado)
    y = guardado.leer(guardado.tensores, torch.float32).view(B, L, d)
    ref = F.pad(y, (0, 0, k - 1, 0)).unfold(1, k, 1).reshape(B * L, d * k).to(dtype)
    got = gc.leer(gc.tensores, dtype)
    assert cols.shape == (B, L, d * k) and torch.equal(got, ref)


@pytest.mark.parametrize('bits', [16, 32])
@pytest.mark.parametrize('N,d,m,con_sesgo', [(1, 32, 8, True), (70, 64, 96, True), (513, 260, 40, False), (2048, 128, 256, True)])
def test_products(N, d, m, con_sesgo, bits):
    """lineal8 on what norma8 and gelu8 keep: lineal's output and input gradient bit for bit, the weight gradient that of
    the 8-bit values."""
    dt = torch.bfloat16 if bits == 16 else torch.float32
    g = torch.Generator(device=DEV).manual_seed(N)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    w, b = (r(m, d) * 0.1).requires_grad_(), r(m).requires_grad_() if con_sesgo else None
    ln = torch.nn.LayerNorm(d).to(DEV)
    x, gy = r(N, d).requires_grad_(), r(N, m).to(dt)
    with torch.autocast('cuda', torch.bfloat16, enabled=bits == 16):
        for op in (lambda: ops.norma8(ln, x, dt), lambda: ops.gelu8(x.to(dt))):
            salida = op()
            e, guardado = salida[0], salida[-1]
            e = e.detach().requires_grad_()
            y, y0 = lineal8(e, w, b, guardado), lineal(e, w, b)
            assert torch.equal(y, y0)
            hojas = [e, w] + ([b] if con_sesgo else [])
            got, ref = torch.autograd.grad(y, hojas, gy), torch.autograd.grad(y0, hojas, gy)
            assert torch.equal(got[0], ref[0]) and (not con_sesgo or torch.equal(got[2], ref[2]))
            leido = guardado.leer(guardado.tensores, dt)
            exacto = gy.double().t() @ leido.double()
            # each product's terms summed in fp32: N roundings at most of the sum of the terms' sizes
            lim = (N ** 0.5 + 16) * 2 * U * (gy.double().abs().t() @ leido.double().abs())
            dentro(got[1], exacto, lim + (torch.finfo(dt).eps / 2 * exacto.abs() if bits == 16 else 0))
    with torch.no_grad():                            # nothing kept without gradients
        assert ops.norma8(ln, x, dt)[2] is None and ops.gelu8(x)[1] is None and torch.equal(lineal8(x, w, b, None), lineal(x, w, b))


def _bloque(d, mezcla='conv', dropout=0.0, k=4):
    torch.manual_seed(3)
    return asrn_amd.BloqueLocal(d, k, 2 * d, dropout, mezcla).to(DEV)


@pytest.mark.parametrize('d,mezcla,k', [(64, 'conv', 4), (256, 'conv', 4), (36, 'conv', 3), (64, 'memoria', 4), (1028, 'conv', 2), (10, 'conv', 4)])
@pytest.mark.parametrize('bits', [16, 32])
def test_block(d, mezcla, k, bits):
    """A block's output is the same with 8 bits; its gradients are within what the 8 bits' rounding moves them: an input
    is off by at most max |x| / 127 of its group, 1.5% of a typical value, so a few percent of a gradient's norm."""
    b = _bloque(d, mezcla, k=k)
    g = torch.Generator(device=DEV).manual_seed(1)
    h = torch.randn(3, 50, d, generator=g, device=DEV, requires_grad=True)
    gy = torch.randn(3, 50, d, generator=g, device=DEV)
    out = []
    for ocho in (False, True):
        with torch.autocast('cuda', torch.bfloat16, enabled=bits == 16):
            y = b(h, ocho=ocho)
        out.append((y.detach(), *torch.autograd.grad(y, [h, *b.parameters()], gy)))
    assert torch.allclose(out[0][0], out[1][0], rtol=1e-5, atol=1e-5) if bits == 32 else \
        (out[0][0] - out[1][0]).norm() <= 2e-3 * out[0][0].norm()
    if d % 4 == 0 and d <= 1024:                     # where both modes run the library's LayerNorm: the same bits
        assert torch.equal(out[0][0], out[1][0])
    for a, c in zip(out[0][1:], out[1][1:]):
        assert (a - c).norm() <= 0.04 * a.norm() + 1e-6


def test_block_keeps_less():
    """Bytes kept for the backward of a bf16 block: 28 d a token, and 5 d with the scales in 8 bits."""
    d, N = 256, 4096
    b = _bloque(d)
    h = torch.randn(2, N // 2, d, device=DEV, requires_grad=True)
    medidas = []
    for ocho in (False, True, False, True):
        torch.cuda.synchronize()
        antes = torch.cuda.memory_allocated()
        with torch.autocast('cuda', torch.bfloat16, cache_enabled=False):
            y = b(h, ocho=ocho)
        medidas.append((torch.cuda.memory_allocated() - antes) / (N * d))
        del y
    # beside what is kept: the output (4), the products' 16-bit weights (8 d^2 in all: 1 a value here) and allocator rounding
    assert medidas[2] >= 28 and medidas[3] <= 5.2 + 4 + 2.5, medidas


def test_block_with_hooks_dropout_and_other_activations():
    h = torch.randn(2, 9, 64, device=DEV, requires_grad=True)
    b = _bloque(64, dropout=0.5)
    y = b(h, ocho=True)
    torch.autograd.grad(y.sum(), h)
    b = _bloque(64)
    b.ff[1] = torch.nn.SiLU()
    assert torch.allclose(b(h), b(h, ocho=True), atol=1e-5)
    b = _bloque(64)
    visto = []
    b.ff[1].register_forward_hook(lambda *a: visto.append(1))
    b(h, ocho=True)
    assert visto
    with torch.autocast('cuda', torch.float16):      # products in fp16: the block runs as without
        assert torch.equal(b(h), b(h, ocho=True))


def _modelo(checkpoint, mezcla='conv'):
    m = asrn_amd.crear_modelo(61, 64, 4, semilla=5, checkpoint=checkpoint, mezcla=mezcla).to(DEV)
    return m.train()


@pytest.mark.parametrize('mezcla', ['conv', 'memoria'])
def test_model(mezcla):
    """ModeloASRN(checkpoint='ocho'): the same loss, gradients near those without, and none of it in evaluation."""
    g = torch.Generator().manual_seed(2)
    x, y = (torch.randint(0, 61, (2, 70), generator=g).to(DEV) for _ in range(2))
    res = {}
    for modo in ('no', 'ocho'):
        m = _modelo(modo, mezcla)
        p = m.perdida(x, y)
        p.backward()
        res[modo] = (p.item(), {n: v.grad for n, v in m.named_parameters() if v.grad is not None}, m.eval()(x))
    assert abs(res['no'][0] - res['ocho'][0]) <= 1e-5 and torch.equal(res['no'][2], res['ocho'][2])
    assert res['no'][1].keys() == res['ocho'][1].keys()
    total = sum(v.norm() ** 2 for v in res['no'][1].values()) ** 0.5
    dif = sum((v - res['ocho'][1][n]).norm() ** 2 for n, v in res['no'][1].items()) ** 0.5
    assert dif <= 0.04 * total


def test_wrapped_block_is_called_with_its_own_arguments():
    m = _modelo('ocho')

    class Envuelto(torch.nn.Module):
        def __init__(self, b):
            super().__init__()
            self.b, self.mezcla = b, b.mezcla

        def forward(self, h):
            return self.b(h)

    m.bloques[1] = Envuelto(m.bloques[1])
    m.perdida(torch.zeros(1, 8, dtype=torch.long, device=DEV), torch.zeros(1, 8, dtype=torch.long, device=DEV)).backward()


@pytest.mark.parametrize('precision', ['fp32', 'bf16'])
def test_graphed_step(precision):
    """PasoGrafado over a model in 8 bits: replays equal the eager steps from the same state."""
    g = torch.Generator().manual_seed(3)
    lotes = [torch.randint(0, 61, (2, 48), generator=g).to(DEV) for _ in range(7)]
    perdidas = []
    for grabar in (True, False):
        m = _modelo('ocho')
        opt = asrn_amd.crear_optimizador(m, 1e-3, capturable=grabar)
        paso = asrn_amd.PasoGrafado(m, opt, 2, 47, precision=precision, grabar=grabar)
        fila = []
        for x in lotes:
            p, _, salto = paso(x[:, :-1], x[:, 1:], lr=1e-3)
            fila.append(p.item())
            assert salto.item() == 0
        perdidas.append(fila)
    assert all(abs(a - b) <= (1e-5 if precision == 'fp32' else 2e-3) * abs(b) for a, b in zip(*perdidas)), perdidas


def _pref(logits, y, ref):
    return asrn_amd.perdida_preferencia(asrn_amd.log_probabilidades(logits, y), y != -100, ref, beta=0.3)[0]


def _pol(logits, y, A, vieja):
    lp, H = asrn_amd.log_probabilidades(logits, y, entropia=True)
    return asrn_amd.perdida_politica(lp, A, vieja, y != -100, lp_ref=vieja, beta=0.04, entropia=H, peso_entropia=0.01,
                                     reduccion='textos')[0]


@pytest.mark.parametrize('cual', ['preferencia', 'politica'])
@pytest.mark.parametrize('checkpoint', ['no', 'ocho'])
def test_graphed_fine_tuning(cual, checkpoint):
    """PasoGrafado with the preference or the policy loss and its per-step inputs: replays equal the eager steps."""
    g = torch.Generator().manual_seed(7)
    P, L = 2, 40
    pasos = []
    for _ in range(7):
        x = torch.randint(0, 61, (2 * P, L + 1), generator=g).to(DEV)
        y = x[:, 1:].clone()
        y[:, :9] = -100
        y[1, 20:] = -100
        pasos.append((x[:, :-1], y, torch.randn(2 * P, generator=g).to(DEV), (-3 * torch.rand(2 * P, L, generator=g)).to(DEV)))
    perdidas = []
    for grabar in (True, False):
        m = _modelo(checkpoint)
        opt = asrn_amd.crear_optimizador(m, 1e-3, capturable=grabar)
        de = (lambda p: (p[3],)) if cual == 'preferencia' else (lambda p: p[2:])
        paso = asrn_amd.PasoGrafado(m, opt, 2 * P, L, precision='fp32', grabar=grabar, perdida=_pref if cual == 'preferencia' else _pol,
                                    extras=de(pasos[0]))
        with pytest.raises(ValueError, match='extras'):
            paso(*pasos[0][:2], lr=1e-3)
        fila = []
        for p in pasos:
            perdida, _, salto = paso(*p[:2], lr=1e-3, extras=de(p))
            fila.append(perdida.item())
            assert salto.item() == 0
        perdidas.append(fila)
    assert all(abs(a - b) <= 2e-5 * (1 + abs(b)) for a, b in zip(*perdidas)), perdidas


def test_graphed_step_refuses_a_living_eager_graph():
    """A score kept with its graph holds the parameters' accumulators on the default stream: the capture is refused, and
    runs once the score is dropped."""
    from asrn_amd._lib import nodos
    x = torch.randint(0, 61, (2, 31), generator=torch.Generator().manual_seed(3)).to(DEV)
    m = _modelo('no')
    opt = asrn_amd.crear_optimizador(m, 1e-3, capturable=True)
    paso = asrn_amd.PasoGrafado(m, opt, 2, 30, precision='fp32', calentar=1)
    paso(x[:, :-1], x[:, 1:], lr=1e-3)
    assert not nodos().hojas_en_uso(paso.params)
    lp = m.log_probabilidades(x[:, :-1], x[:, 1:])
    assert nodos().hojas_en_uso(paso.params)
    with pytest.raises(RuntimeError, match='eager graph'):
        paso(x[:, :-1], x[:, 1:], lr=1e-3)
    esperada = -lp.detach().mean()
    del lp
    assert not nodos().hojas_en_uso(paso.params)
    for _ in range(3):
        perdida, _, salto = paso(x[:, :-1], x[:, 1:], lr=0.0)
        assert abs(perdida.item() - esperada.item()) <= 1e-5 * esperada.item() and salto.item() == 0


def test_fine_tuning_step():
    """The operators together, as a fine-tuning step runs them: a reference's scores, then preference and policy steps on
    a model in 8 bits. The losses and gradients are finite, every parameter moves, and the step in 8 bits takes the same
    loss and nearly the gradient of the one without."""
    g = torch.Generator().manual_seed(4)
    P, L = 3, 40
    x = torch.randint(0, 61, (2 * P, L + 1), generator=g).to(DEV)
    entra, y = x[:, :-1], x[:, 1:].clone()
    y[:, :10] = -100
    y[1, 25:] = -100
    m = y != -100
    A = torch.randn(2 * P, generator=g).to(DEV)
    res = {}
    for modo in ('no', 'ocho'):
        mod = _modelo(modo)
        with torch.no_grad():
            ref = mod.log_probabilidades(entra, y)
        lp, H = mod.log_probabilidades(entra, y, entropia=True)
        pref, rec = asrn_amd.perdida_preferencia(lp, m, ref)
        pol, est = asrn_amd.perdida_politica(lp, A, ref, m, lp_ref=ref, beta=0.04, entropia=H, peso_entropia=0.01, reduccion='textos')
        assert abs(pref.item() - math.log(2)) <= 1e-6 and (rec.abs() <= 1e-6).all() and est[0] == 0
        (pref + pol).backward()
        res[modo] = [pref.item(), pol.item(), {n: v.grad.clone() for n, v in mod.named_parameters() if v.grad is not None}]
        antes = {n: v.detach().clone() for n, v in mod.named_parameters()}
        asrn_amd.crear_optimizador(mod, 1e-3).step()
        assert all(torch.isfinite(v).all() for v in mod.parameters())
        assert not torch.equal(mod.bloques[0].ff[0].weight, antes['bloques.0.ff.0.weight'])
    assert abs(res['no'][1] - res['ocho'][1]) <= 1e-5
    total = sum(v.norm() ** 2 for v in res['no'][2].values()) ** 0.5
    assert sum((v - res['ocho'][2][n]).norm() ** 2 for n, v in res['no'][2].items()) ** 0.5 <= 0.04 * total


def test_refusals():
    with pytest.raises(RuntimeError, match='GPU only'):
        ops.guardar8(torch.zeros(2, 32))
    for mal in (torch.zeros(2, 32, device=DEV).half(), torch.zeros((), device=DEV), torch.zeros(2, 0, device=DEV)):
        with pytest.raises(ValueError):
            ops.guardar8(mal)
    q, e = ops.guardar8(torch.zeros(2, 40, device=DEV))
    for a in ((q, e[:1]), (q.int(), e), (q, e.int()), (q[0], e), (q, e, torch.float16)):
        with pytest.raises(ValueError):
            ops.leer8(*a)
    assert ops.guardar8(torch.zeros(0, 40, device=DEV))[0].shape == (0, 40)


def test_past_32_bits():
    """More than 2^31 values: the last rows against the same rows alone."""
    N, d = 70_001, 30_720
    u = torch.zeros(N, d, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(6)
    cola = torch.randn(3, d, generator=g, device=DEV).bfloat16()
    u[-3:] = cola
    q, e = ops.guardar8(u)
    q2, e2 = ops.guardar8(cola)
    assert torch.equal(q[-3:], q2) and torch.equal(e[-3:], e2) and (q[-4] == 0).all()
    assert torch.equal(ops.leer8(q, e, torch.bfloat16)[-3:], ops.leer8(q2, e2, torch.bfloat16))


@pytest.mark.parametrize('d', [64, 2048, 10])
def test_one_output_or_input_alone(d):
    """Gradients of one output only, and of one input only."""
    g = torch.Generator(device=DEV).manual_seed(d)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    ln = torch.nn.LayerNorm(d).to(DEV)
    x, gy = r(9, d).requires_grad_(), r(9, d)
    y, a, _ = ops.norma8(ln, x, torch.float32)
    solo = torch.autograd.grad(y, (x, ln.weight), gy, retain_graph=True)
    cero = torch.autograd.grad((y, a), (x, ln.weight), (gy, torch.zeros_like(gy)), retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(solo, cero))
    dx, dw = torch.autograd.grad(a, (x, ln.weight), gy, allow_unused=True)
    assert torch.equal(dx, gy) and (dw is None or (dw == 0).all())
    y, a, _ = ops.norma8(ln, x.detach(), torch.float32)
    assert torch.allclose(torch.autograd.grad(y, ln.bias, gy)[0], gy.sum(0), atol=1e-4)
    u, h = r(9, d), r(9, d).requires_grad_()
    assert torch.equal(torch.autograd.grad(ops.suma_gelu8(h, u), h, gy)[0], gy)
    s = ops.suma_gelu8(h.detach(), u.requires_grad_())
    assert torch.equal(torch.autograd.grad(s, u, gy)[0], torch.autograd.grad(ops.gelu8(u)[0], u, gy)[0])
    w = r(3, d)
    e, guardado = ops.gelu8(u)
    y, y0 = lineal8(e, w, None, guardado), lineal(e, w)      # a weight without a gradient: nothing is read back
    gy = r(9, 3)
    assert torch.equal(torch.autograd.grad(y, e, gy, retain_graph=True)[0], torch.autograd.grad(y0, e, gy)[0])


def test_second_gradients_are_refused():
    x = torch.randn(4, 64, device=DEV, requires_grad=True)
    for y in (ops.gelu8(x)[0], ops.norma8(torch.nn.LayerNorm(64).to(DEV), x, torch.float32)[0]):
        with pytest.raises(RuntimeError, match='create_graph'):
            torch.autograd.grad((y * y).sum() + (x ** 3).sum(), x, create_graph=True)


def test_strided_inputs_and_offsets():
    """Inputs that are slices, and rows off a 16-byte boundary."""
    base = torch.randn(2, 9, 130, device=DEV)
    u = base[..., 1:65].detach().requires_grad_()
    y, _ = ops.gelu8(u)
    assert torch.allclose(y, F.gelu(u), atol=1e-6) and torch.autograd.grad(y.sum(), u)[0].shape == u.shape
    ln = torch.nn.LayerNorm(64).to(DEV)
    plano = torch.randn(64 * 9 + 1, device=DEV)
    for x in (base[..., 2:66], plano[1:].view(9, 64), base[:, ::2, :64]):
        x = x.detach().requires_grad_()
        y, a, g = ops.norma8(ln, x, torch.float32)
        assert torch.allclose(y, ln(x), atol=1e-5)
        gy = torch.randn(64 * x.numel() // 64 + 1, device=DEV)[1:].view(x.shape)       # off the boundary too
        dx, = torch.autograd.grad((y, a), x, (gy, gy))
        z = ocho(x)[2].to(DEV)
        s = (x.detach().double().var(-1, unbiased=False, keepdim=True) + ln.eps).rsqrt()
        xh = (z - x.detach().double().mean(-1, keepdim=True)) * s
        f = gy.double()
        ref = s * (f - f.mean(-1, keepdim=True) - xh * (f * xh).mean(-1, keepdim=True)) + f
        assert (dx - ref).abs().max() <= 1e-5 * (1 + s.max())


@pytest.mark.parametrize('d', [64, 30])
@pytest.mark.parametrize('dt', [torch.float16, torch.float64])
def test_products_in_other_dtypes(d, dt):
    """Products in fp16 (autocast) and fp64 after ops that kept fp32 inputs: the weight gradient is lineal's on the values
    read back, rounded to the product's dtype."""
    g = torch.Generator(device=DEV).manual_seed(11)
    x = torch.randn(2, 9, d, generator=g, device=DEV)
    w = torch.randn(8, d, generator=g, device=DEV)
    ln = torch.nn.LayerNorm(d).to(DEV)

    def gw(op, y, peso, *resto):
        peso = peso.detach().to(torch.float64 if dt == torch.float64 else torch.float32).requires_grad_()
        with torch.autocast('cuda', dtype=torch.float16, enabled=dt == torch.float16):
            z = op(y.double() if dt == torch.float64 else y, peso, None, *resto)
        assert z.dtype == dt
        return torch.autograd.grad(z, peso, torch.ones_like(z))[0]

    for y, guardado in (ops.gelu8(x.clone().requires_grad_()), ops.norma8(ln, x, torch.float32)[::2]):
        leido = guardado.leer(guardado.tensores, dt)
        assert leido.dtype == dt and torch.equal(leido, guardado.leer(guardado.tensores, torch.float32).to(dt))
        assert torch.equal(gw(lineal8, y, w, guardado), gw(lineal, leido.float().view(x.shape), w))
    z, _, guardado = ops.norma8(ln, x, torch.float32)
    cols, guardado = ops.ventana8(z, 3, torch.float32, guardado)
    w3 = torch.randn(8, 3 * d, generator=g, device=DEV)
    leido = guardado.leer(guardado.tensores, dt)
    assert torch.equal(gw(lineal8, cols, w3, guardado), gw(lineal, leido.float().view(cols.shape), w3))


def test_what_was_kept_belongs_to_its_tensor():
    """ventana8 and lineal8 refuse what an op kept of a tensor of another size, norma8 parameters on another device."""
    x = torch.randn(2, 9, 64, device=DEV)
    w = torch.randn(8, 64, device=DEV, requires_grad=True)
    ln = torch.nn.LayerNorm(64).to(DEV)
    z, _, guardado = ops.norma8(ln, x, torch.float32)
    y, del_gelu = ops.gelu8(x.requires_grad_())
    for otro in (torch.randn(2, 10, 64, device=DEV), torch.randn(1, 9, 64, device=DEV), torch.randn(4, 9, 32, device=DEV)):
        with pytest.raises(ValueError, match='ventana8'):
            ops.ventana8(otro, 3, torch.float32, guardado)
        with pytest.raises(ValueError, match='lineal8'):
            lineal8(otro, w, None, guardado)
    for args in ((z, 3, torch.float32, del_gelu), (z, 3, torch.float16, guardado), (z.bfloat16(), 3, torch.bfloat16, guardado),
                 (z.view(18, 64), 3, torch.float32, guardado), (z, 3, torch.float16, None)):
        with pytest.raises(ValueError, match='ventana8'):
            ops.ventana8(*args)
    with pytest.raises(ValueError, match='norma8'):
        ops.norma8(torch.nn.LayerNorm(64), x, torch.float32)
    assert lineal8(y, w, None, del_gelu).shape == (2, 9, 8)


def test_window_of_a_window_is_refused():
    """What ventana8 itself returns goes to lineal8, not back into ventana8."""
    ln = torch.nn.LayerNorm(64).to(DEV)
    z, _, guardado = ops.norma8(ln, torch.randn(2, 9, 64, device=DEV), torch.float32)
    for k in (1, 3):
        cols, gc = ops.ventana8(z, k, torch.float32, guardado)
        with pytest.raises(ValueError, match='did not keep'):
            ops.ventana8(cols, k, torch.float32, gc)


@pytest.mark.parametrize('N,d', [(40_000, 66), (3, 8198)])
def test_other_widths_in_a_graph(N, d):
    """The widths that torch's LayerNorm runs: a captured backward replays as the eager one, step after step."""
    g = torch.Generator(device=DEV).manual_seed(d)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    ln = torch.nn.LayerNorm(d).to(DEV)
    x, gy = r(N, d).requires_grad_(), r(N, d)

    def paso():
        y, a, _ = ops.norma8(ln, x, torch.float32)
        return [y.detach(), *torch.autograd.grad((y, a), (x, ln.weight, ln.bias), (gy, gy))]

    lado = torch.cuda.Stream()
    lado.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(lado):
        paso()
    torch.cuda.current_stream().wait_stream(lado)
    torch.cuda.synchronize()
    grafo = torch.cuda.CUDAGraph()
    with torch.cuda.graph(grafo):
        salida = paso()
    for _ in range(4):
        with torch.no_grad():
            x.copy_(r(N, d))
            gy.copy_(r(N, d))
        grafo.replay()
        torch.cuda.synchronize()
        for a, b in zip(salida, paso()):
            assert torch.equal(a, b)


def _grande(logits, y):
    """A loss with a torch sum over all logits, which many workgroups share: torch clears their counter with a memset."""
    return asrn_amd.log_probabilidades(logits, y).mean() * -1 + 1e-3 * (logits.float() ** 2).sum() / y.numel()


def _propia(logits, y):
    return -asrn_amd.log_probabilidades(logits, y).mean()


@pytest.mark.parametrize('perdida,una', [(_grande, False), (_propia, True)])
def test_graphed_losses_with_memsets_keep_two_streams(perdida, una):
    """A captured step whose loss records a memset branches, and its replays, with eager work between, equal ordinary
    steps; one without memsets stays on one stream."""
    V, B, L = 997, 4, 250
    g = torch.Generator().manual_seed(9)
    lotes = [torch.randint(0, V, (B, L + 1), generator=g).to(DEV) for _ in range(7)]
    filas = []
    for grabar in (True, False):
        m = asrn_amd.crear_modelo(V, 64, 4, semilla=5).to(DEV).train()
        vistas = []
        m.largos[0].register_forward_pre_hook(lambda c, a, kw: vistas.append(kw.get('una_corriente', False)), with_kwargs=True)
        opt = asrn_amd.crear_optimizador(m, 1e-3, capturable=grabar)
        paso = asrn_amd.PasoGrafado(m, opt, B, L, precision='fp32', calentar=1, grabar=grabar, perdida=perdida)
        fila = []
        for x in lotes:
            p, _, salto = paso(x[:, :-1], x[:, 1:], lr=1e-3)
            fila.append(p.item())
            assert salto.item() == 0 and torch.rand(1 << 16, device=DEV).sum() > 0
        filas.append(fila)
        if grabar:
            assert vistas[-1] == una and m.permite_una_corriente
            assert una or vistas[1] is True           # the capture that was dropped
    assert all(abs(a - b) <= 2e-5 * (1 + abs(b)) for a, b in zip(*filas)), filas


@pytest.mark.parametrize('d', [64, 66, 1028])
def test_norms_with_hooks_or_of_other_kinds(d):
    """norma8 of what norma_residual calls as a module: its hooks and its own forward run, and nothing is kept."""
    x = torch.randn(3, d, device=DEV, requires_grad=True)
    con_gancho, propia, otra = torch.nn.LayerNorm(d).to(DEV), torch.nn.LayerNorm(d).to(DEV), torch.nn.RMSNorm(d).to(DEV)
    con_gancho.register_forward_hook(lambda m, i, o: 2 * o)
    propia.forward = lambda t: t + 1
    # up to 1,024 channels, multiples of 4, norma_residual fuses any affine LayerNorm (and asks for its bias)
    for ln in [con_gancho, propia] + [otra] * (d == 66):
        y, a, guardado = ops.norma8(ln, x, torch.float32)
        y0, a0 = ops.norma_residual(ln, x, torch.float32)
        assert torch.equal(y, y0) and torch.equal(a, a0) and (guardado is None) == (d != 64)
    assert ops.norma8(otra.cpu(), x.cpu(), torch.float32)[2] is None
    assert ops.norma8(torch.nn.LayerNorm(d, bias=False).to(DEV), x, torch.float32)[2] is None
    assert ops.norma8(torch.nn.LayerNorm(d).to(DEV), x, torch.float32)[2] is not None


@pytest.mark.parametrize('d', [66, 1028])
def test_norm_without_eps(d):
    """The library's kernels take a positive eps only; at widths that torch's LayerNorm runs without 8 bits, 0 runs with
    them too."""
    ln = torch.nn.LayerNorm(d, eps=0.0).to(DEV)
    x = torch.randn(3, d, device=DEV, requires_grad=True)
    y, _, guardado = ops.norma8(ln, x, torch.float32)
    assert guardado is None and torch.equal(y, ops.norma_residual(ln, x, torch.float32)[0])


@pytest.mark.parametrize('como', ['subclase', 'instancia'])
def test_block_with_its_own_feed_forward(como):
    """A block whose feed-forward was replaced runs it, with 8 bits asked for or not."""
    b = _bloque(64)
    if como == 'subclase':
        b.__class__ = type('Otro', (asrn_amd.BloqueLocal,), {'_ff': lambda s, y: 3 * asrn_amd.BloqueLocal._ff(s, y)})
    else:
        b._ff = lambda y: torch.zeros_like(y)
    h = torch.randn(2, 9, 64, device=DEV, requires_grad=True)
    assert torch.equal(b(h), b(h, ocho=True))


def test_graphed_step_without_the_nodes(monkeypatch):
    """A library that was built alone: the ordinary captured step runs as before."""
    from asrn_amd import _lib

    def faltan():
        raise _lib.ASRNHipError('_nodos.so is missing')

    monkeypatch.setattr('asrn_amd.entrenamiento.nodos', faltan)
    monkeypatch.setattr('asrn_amd.ops.nodos', faltan)
    x = torch.randint(0, 61, (2, 31), generator=torch.Generator().manual_seed(3)).to(DEV)
    filas = []
    for grabar in (True, False):
        m = _modelo('no')
        opt = asrn_amd.crear_optimizador(m, 1e-3, capturable=grabar)
        paso = asrn_amd.PasoGrafado(m, opt, 2, 30, precision='fp32', calentar=1, grabar=grabar)
        filas.append([paso(x[:, :-1], x[:, 1:], lr=1e-3)[0].item() for _ in range(4)])
    assert all(abs(a - b) <= 1e-5 * abs(b) for a, b in zip(*filas))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_gelu_types_and_values(dtype):
    """The output and the gradient come in the input's type; in bf16 the output is F.gelu's bit for bit, in fp32 both are
    within their roundings of the definition."""
    u = (2.5 * torch.randn(37, 64, generator=torch.Generator(device=DEV).manual_seed(5), device=DEV)).to(dtype).requires_grad_()
    y, _ = ops.gelu8(u)
    du, = torch.autograd.grad(y, u, torch.ones_like(y))
    assert y.dtype == dtype and du.dtype == dtype
    if dtype == torch.bfloat16:
        assert torch.equal(y, F.gelu(u))
    else:
        dentro(y.detach(), F.gelu(u.detach()), 8 * U * (1 + u.detach().abs().double()))


@pytest.mark.parametrize('mezcla', ['conv', 'memoria'])
@pytest.mark.parametrize('bits', [16, 32])
def test_block_with_dropout(mezcla, bits):
    """Active dropout from the same seed: the output of the block without 8 bits, its gradients within the 8 bits' share."""
    b = _bloque(64, mezcla, dropout=0.3)
    g = torch.Generator(device=DEV).manual_seed(1)
    h = torch.randn(3, 50, 64, generator=g, device=DEV, requires_grad=True)
    gy = torch.randn(3, 50, 64, generator=g, device=DEV)
    out = []
    for ocho in (False, True):
        torch.manual_seed(11)
        with torch.autocast('cuda', torch.bfloat16, enabled=bits == 16):
            y = b(h, ocho=ocho)
        out.append((y.detach(), *torch.autograd.grad(y, [h, *b.parameters()], gy)))
    assert torch.allclose(out[0][0], out[1][0], rtol=1e-5, atol=1e-5) if bits == 32 else \
        (out[0][0] - out[1][0]).norm() <= 2e-3 * out[0][0].norm()
    for a, c in zip(out[0][1:], out[1][1:]):
        assert (a - c).norm() <= 0.04 * a.norm() + 1e-6


def test_block_on_a_side_stream():
    """A block in 8 bits on another stream, its input written there: the default stream's output and gradients."""
    b = _bloque(256)
    h0 = torch.randn(3, 50, 256, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)

    def paso():
        h = (h0 * 2 - h0).requires_grad_()
        y = b(h, ocho=True)
        return [y.detach(), *torch.autograd.grad(y, [h, *b.parameters()], h0)]

    base = paso()
    torch.cuda.synchronize()
    lado = torch.cuda.Stream()
    with torch.cuda.stream(lado):
        otra = paso()
    lado.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(base, otra))


def test_graphed_loss_with_memsets_and_dropout():
    """A step captured twice whose model draws: every replay draws anew, and its loss is an eager step's but for the draw."""
    V, B, L = 997, 4, 250
    x = torch.randint(0, V, (B, L + 1), generator=torch.Generator().manual_seed(9)).to(DEV)
    m = asrn_amd.crear_modelo(V, 64, 4, semilla=5, dropout=0.3).to(DEV).train()
    opt = asrn_amd.crear_optimizador(m, 1e-3, capturable=True)
    paso = asrn_amd.PasoGrafado(m, opt, B, L, precision='fp32', calentar=1, perdida=_grande)
    vals = []
    for _ in range(5):
        p, _, salto = paso(x[:, :-1], x[:, 1:], lr=0.0)
        vals.append(p.item())
        assert salto.item() == 0
    eager = _grande(m(x[:, :-1]), x[:, 1:]).item()
    assert len(set(vals)) == 5 and all(abs(v - eager) <= 0.1 * abs(eager) for v in vals), (vals, eager)
