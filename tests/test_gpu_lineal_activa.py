"""The product with its epilogue (asrn_amd.lineal_activa) against the formula in 64 bits. Tolerances: fp32 sums of n terms are
within n + 24 roundings of the terms' magnitudes (24: the three-part fp32 products, bias, activation, residual), through the
activation's slope of at most 1.13; results carry half a step of their type, the 16-bit activations' input and the gradient
before the activation one each of their own."""
import pytest
import torch

import asrn_amd
from asrn_amd import _lib

pytestmark = pytest.mark.gpu
DEV = 'cuda'
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24


@pytest.fixture(autouse=True)
def semilla():
    torch.manual_seed(0)


def r(*forma, dt=F32):
    return torch.randn(*forma, device=DEV).to(dt)


def act64(x, act):
    if act == 'gelu':
        fi = 0.5 * torch.erfc(-x / 2 ** 0.5)
        return x * fi, fi + x * torch.exp(-x * x / 2) / (2 * torch.pi) ** 0.5
    if act == 'silu':
        s = torch.sigmoid(x)
        return x * s, s * (1 + x * (1 - s))
    return x, torch.ones_like(x)


def medio(dt):
    return torch.finfo(dt).eps / 2


def menor(dt):
    """The smallest step, below the type's normal range: half of it is lost there."""
    return torch.finfo(dt).smallest_normal * 2 * medio(dt)


def cerca(x, ref, cota, nombre):
    assert x.shape == ref.shape, nombre
    cota = cota + medio(x.dtype) * (ref.abs() + cota) + menor(x.dtype)
    mal = ~((x.double() - ref).abs() <= cota)
    assert not mal.any(), (nombre, int(mal.sum()), ((x.double() - ref).abs() / cota).max().item())


def revisar(x, w, b, act, res, gy, y, gs):
    """y and the gradients (x, w, b, res as they are given) against 64 bits."""
    dt = x.dtype
    K, N = w.shape[1], w.shape[0]
    x2, w2 = x.double().reshape(-1, K), w.double()
    M = x2.shape[0]
    pre = x2 @ w2.t() + (0 if b is None else b.double())
    pre_m = x2.abs() @ w2.abs().t() + (0 if b is None else b.double().abs())
    yr, der = act64(pre, act)
    # erfc within 1.5e-7 in 16-bit results' GELU: |x| / 2 of it
    e_y = 1.13 * (K + 24) * U * pre_m + 24 * U * yr.abs() + (8e-8 * pre.abs() if dt != F32 else 0)
    if res is not None:
        yr = yr + res.double().reshape(M, N)
        e_y = e_y + U * (res.double().reshape(M, N).abs() + yr.abs())
    cerca(y.reshape(M, N), yr, e_y, 'y')
    if gs is None:
        return
    g2 = gy.double().reshape(M, N)
    gp = g2 * der
    # the derivative at an input that was rounded to dt (slope at most 0.8), its own sums, the rounding of gp to dt
    e_gp = g2.abs() * (0.8 * (medio(dt) * pre.abs() + menor(dt) + (K + 24) * U * pre_m) + 16 * U * (1 + pre.abs()))
    if act is None:
        e_gp = torch.zeros_like(gp)
    e_gp = e_gp + (medio(dt) * (gp.abs() + e_gp) + menor(dt) if dt != F32 or act is not None else 0)
    gp_m = gp.abs() + e_gp
    gs = list(gs)
    cerca(gs.pop(0).reshape(M, K), gp @ w2, e_gp @ w2.abs() + (N + 24) * U * (gp_m @ w2.abs()), 'x')
    # a weight gradient in slabs is rounded to dt slab by slab where the library forms it (16 at most)
    slab = 16 * medio(dt) if dt != F32 else 0
    cerca(gs.pop(0), gp.t() @ x2, e_gp.t() @ x2.abs() + ((M + 24) * U + slab) * (gp_m.t() @ x2.abs()), 'w')
    if b is not None:
        cerca(gs.pop(0), gp.sum(0), e_gp.sum(0) + (M + 24) * U * gp_m.sum(0), 'b')
    if res is not None:
        assert torch.equal(gs.pop(0).reshape(M, N), gy.reshape(M, N))


CASOS = [
    (1, 4, 4, F32), (1, 768, 64, BF16), (3, 17, 5, F32), (16, 389, 130, BF16), (16, 256, 72, F16), (16, 1024, 100, F32),
    (8, 8, 1, F32), (4, 100, 33, F16), (5, 2048, 7, BF16), (13, 64, 300, F32),
    (17, 8, 8, BF16), (17, 5, 3, F32), (64, 64, 64, BF16), (65, 72, 66, F16), (100, 389, 517, F32), (200, 40, 129, BF16),
    (129, 33, 257, BF16), (333, 128, 96, F32), (1000, 776, 64, F16), (2048, 256, 2048, BF16), (2100, 200, 2300, BF16),
    (2049, 100, 2040, F32), (300, 3, 50, F16), (70, 2500, 80, F32), (40, 4096, 36, BF16)]


@pytest.mark.parametrize('M,K,N,dt', CASOS)
@pytest.mark.parametrize('act,con_res', [('gelu', False), ('silu', True), (None, True), (None, False), ('gelu', True)])
def test_lineal_activa(M, K, N, dt, act, con_res):
    x, w = r(M, K, dt=dt).requires_grad_(), (r(N, K) * K ** -0.5).to(dt).requires_grad_()
    b = (r(N) / 2).to(dt).requires_grad_()
    res = r(M, N).requires_grad_() if con_res else None
    gy = r(M, N, dt=F32 if con_res else dt)
    y = asrn_amd.lineal_activa(x, w, b, act, res)
    assert y.dtype == (F32 if con_res else dt) and y.is_contiguous()
    gs = torch.autograd.grad(y, [t for t in (x, w, b, res) if t is not None], gy)
    revisar(x.detach(), w.detach(), b.detach(), act, None if res is None else res.detach(), gy, y.detach(), gs)
    with torch.no_grad():
        assert torch.equal(asrn_amd.lineal_activa(x, w, b, act, res), y)


@pytest.mark.parametrize('M', [7, 200])
@pytest.mark.parametrize('dt', [F32, BF16])
def test_without_bias_and_with_a_residual_of_the_products_type(M, dt):
    x, w, res = r(M, 96, dt=dt).requires_grad_(), (r(40, 96) / 10).to(dt).requires_grad_(), r(M, 40, dt=dt).requires_grad_()
    gy = r(M, 40, dt=dt)
    y = asrn_amd.lineal_activa(x, w, activacion='silu', residuo=res)
    assert y.dtype == dt
    revisar(x.detach(), w.detach(), None, 'silu', res.detach(), gy, y.detach(), torch.autograd.grad(y, (x, w, res), gy))


@pytest.mark.parametrize('M', [3, 150])
@pytest.mark.parametrize('dt', [F32, BF16, F16])
@pytest.mark.parametrize('forma', ['columnas', 'traspuestos', 'desplazados', 'ejes', 'expandidos'])
def test_strides(M, dt, forma):
    K, N = 64, 48
    x, w, res = r(M, K, dt=dt), r(N, K, dt=dt), r(M, N)
    b = r(N, dt=dt)
    if forma == 'expandidos':
        x, res = x[:1].expand(M, K), res[:1].expand(M, N)
    x1, w1, res1 = {
        'expandidos': lambda: (x, w, res),
        'columnas': lambda: (torch.cat([x, x], 1)[:, K:], torch.cat([w, w], 1)[:, :K], torch.cat([res, res], 1)[:, N:]),
        'traspuestos': lambda: (x.t().contiguous().t(), w.t().contiguous().t(), res.t().contiguous().t()),
        'desplazados': lambda: tuple(torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape) for t in (x, w, res)),
        'ejes': lambda: (x.view(1, M, K), w, res.view(1, M, N))}[forma]()
    x, w, res = (t.contiguous().clone() for t in (x, w, res))
    y, y1 = asrn_amd.lineal_activa(x, w, b, 'gelu', res), asrn_amd.lineal_activa(x1, w1, b, 'gelu', res1)
    assert y1.shape == res1.shape
    # one order of sums where the operands may be read as vectors, another where not
    e = 2 * (K + 24) * U * 1.13 * (x.double().abs() @ w.double().abs().t() + b.double().abs()) + 4 * U * y.double().abs()
    assert ((y1.reshape(M, N).double() - y.double()).abs() <= e).all()


def test_under_autocast():
    x, w, b, res = r(70, 40).requires_grad_(), r(24, 40).requires_grad_(), r(24).requires_grad_(), r(70, 24).requires_grad_()
    with torch.autocast('cuda', dtype=BF16):
        y = asrn_amd.lineal_activa(x, w, b, 'gelu', res)
        y2 = asrn_amd.lineal_activa(x, w, b, 'gelu')
    assert y.dtype == F32 and y2.dtype == BF16
    gs = torch.autograd.grad(y, (x, w, b, res), r(70, 24))
    assert all(g.dtype == F32 for g in gs)
    xb, wb, bb = (t.detach().to(BF16) for t in (x, w, b))
    assert torch.equal(y, asrn_amd.lineal_activa(xb, wb, bb, 'gelu', res))
    # a backward inside an autocast region is the one outside: the operands were cast, or not, by the call
    x, w = r(300, 40).requires_grad_(), r(24, 40).requires_grad_()
    y, gy = asrn_amd.lineal_activa(x, w, activacion='silu'), r(300, 24)
    fuera = torch.autograd.grad(y, (x, w), gy, retain_graph=True)
    with torch.autocast('cuda', dtype=BF16):
        dentro = torch.autograd.grad(y, (x, w), gy)
    assert all(torch.equal(a, b) for a, b in zip(fuera, dentro))


def test_empty():
    w, b = r(6, 4).requires_grad_(), r(6).requires_grad_()
    for forma in ((0, 4), (2, 0, 4)):
        x = r(*forma).requires_grad_()
        y = asrn_amd.lineal_activa(x, w, b, 'gelu')
        assert y.shape == (*forma[:-1], 6)
        gx, gw, gb = torch.autograd.grad(y.sum(), (x, w, b))
        assert gx.shape == x.shape and not gw.any() and not gb.any()


@pytest.mark.parametrize('dt', [F32, BF16])
@pytest.mark.parametrize('act', [None, 'gelu'])
def test_no_columns(act, dt):
    for forma in ((3, 8), (2, 3, 8), (2, 0, 8)):
        x, w, b = r(*forma, dt=dt).requires_grad_(), r(0, 8, dt=dt).requires_grad_(), r(0, dt=dt).requires_grad_()
        y = asrn_amd.lineal_activa(x, w, b, act)
        assert y.shape == (*forma[:-1], 0)
        gs = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
        assert [g.shape for g in gs] == [x.shape, w.shape, b.shape] and not gs[0].any()


@pytest.mark.parametrize('dt', [F32, BF16])
@pytest.mark.parametrize('M,N', [(1, 8), (1, 1), (40, 1)])
def test_one_row_of_any_stride(M, N, dt):
    """A matrix of one row is contiguous with whatever stride its row has."""
    def fila(n, K):
        t = r(K, n, dt=dt).t()
        assert n > 1 or (t.is_contiguous() and t.stride(0) == 1)
        return t.requires_grad_()
    x, w, b, res, gy = fila(M, 8), fila(N, 8), r(N, dt=dt).requires_grad_(), r(M, N, dt=dt).requires_grad_(), r(M, N, dt=dt)
    y = asrn_amd.lineal_activa(x, w, b, 'silu', res)
    revisar(x.detach(), w.detach(), b.detach(), 'silu', res.detach(), gy, y.detach(), torch.autograd.grad(y, (x, w, b, res), gy))


@pytest.mark.parametrize('M', [5, 100])
@pytest.mark.parametrize('dt', [F32, BF16])
def test_nonfinite(M, dt):
    """An infinity or a NaN of x stays in its row and comes out as the formula's."""
    x, w, b = r(M, 64, dt=dt), r(32, 64, dt=dt), r(32, dt=dt)
    limpio = asrn_amd.lineal_activa(x, w, b, 'silu')
    for malo in (float('inf'), float('nan')):
        x2 = x.clone()
        x2[3, 7] = malo
        y = asrn_amd.lineal_activa(x2, w, b)
        pre = x2.double() @ w.double().t() + b.double()
        assert torch.equal(torch.isnan(y), torch.isnan(pre)) and torch.equal(torch.isinf(y), torch.isinf(pre))
        for act in ('gelu', 'silu'):
            y = asrn_amd.lineal_activa(x2, w, b, act)
            ref = pre * torch.special.ndtr(pre) if act == 'gelu' else pre * torch.sigmoid(pre)
            assert torch.equal(torch.isfinite(y[3]), torch.isfinite(ref[3])) and torch.isfinite(y).sum() >= y.numel() - 32
        y = asrn_amd.lineal_activa(x2, w, b, 'silu')
        otras = [i for i in range(M) if i != 3]
        if dt != F32:
            assert torch.equal(y[otras], limpio[otras])


def test_gradients_by_differences():
    x, w, b, res = (t.requires_grad_() for t in (r(20, 12), r(9, 12) / 4, r(9), r(20, 9)))
    gy = r(20, 9)
    for act in (None, 'gelu', 'silu'):
        f = lambda *a: (asrn_amd.lineal_activa(*a[:3], act, a[3]).double() * gy.double()).sum()
        gs = torch.autograd.grad(f(x, w, b, res), (x, w, b, res))
        e = 2.0 ** -7              # curvature 2^-14 / 6 of a few units, rounding 2^-17: below 2e-3 of gradients around 1
        for i, t in enumerate((x, w, b, res)):
            v = r(*t.shape)
            mas, menos = [[s.detach() + (sg * e * v if j == i else 0) for j, s in enumerate((x, w, b, res))] for sg in (1, -1)]
            dif = (f(*mas) - f(*menos)) / (2 * e)
            assert abs(dif - (gs[i].double() * v.double()).sum()) <= 2e-3 * (1 + (gs[i] * v).abs().sum().item())


def test_second_gradient_is_refused():
    x, w = r(20, 8).requires_grad_(), r(8, 8)
    with pytest.raises(RuntimeError, match='create_graph'):
        torch.autograd.grad(asrn_amd.lineal_activa(x, w, activacion='gelu').sum(), x, create_graph=True)


def test_captured_and_replayed():
    for dt in (F32, BF16):
        x, w, b = r(300, 64, dt=dt).requires_grad_(), r(80, 64, dt=dt).requires_grad_(), r(80, dt=dt).requires_grad_()
        res, gy = r(300, 80).requires_grad_(), r(300, 80)

        def paso():
            y = asrn_amd.lineal_activa(x, w, b, 'gelu', res)
            return [y.detach(), *torch.autograd.grad(y, (x, w, b, res), gy)]
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
                x.copy_(r(300, 64))
                gy.copy_(r(300, 80))
            eager = [t.clone() for t in paso()]
            g.replay()
            torch.cuda.synchronize()
            for a, v in zip(fijos, eager):
                assert torch.equal(a, v), (dt, i)


def test_same_bits_again():
    x, w, b, res = r(3000, 200, dt=BF16), r(600, 200, dt=BF16), r(600, dt=BF16), r(3000, 600)
    y = asrn_amd.lineal_activa(x, w, b, 'gelu', res)
    lado = torch.cuda.Stream()
    lado.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(lado):
        y2 = asrn_amd.lineal_activa(x, w, b, 'gelu', res)
    torch.cuda.synchronize()
    assert torch.equal(y, y2) and torch.equal(y, asrn_amd.lineal_activa(x, w, b, 'gelu', res))
    # a row's result does not depend on the rows beside it
    assert torch.equal(y[:200], asrn_amd.lineal_activa(x[:200], w, b, 'gelu', res[:200]))


@pytest.mark.parametrize('tile', [256 << 8, 256 << 8 | 192, 128 << 8 | 128, 64 << 8 | 64])
@pytest.mark.parametrize('M,K,N', [(300, 128, 272), (17, 72, 40), (513, 200, 515), (260, 333, 193), (256, 64, 256)])
@pytest.mark.parametrize('dt', [BF16, F16])
def test_every_tile(tile, M, K, N, dt):
    """Each tile at whole, partial and single steps and edges, with everything in the epilogue: the formula, and the same bits
    from every tile (a result's sums have one order)."""
    x, w, b, res = r(M, K, dt=dt), (r(N, K) * K ** -0.5).to(dt), r(N, dt=dt), r(M, N)
    y, pre = torch.empty(M, N, device=DEV), torch.empty(M, N, device=DEV, dtype=dt)
    _lib.call('asrn_linear_act_fwd', x.data_ptr(), K, w.data_ptr(), K, {BF16: 1, F16: 2}[dt], b.data_ptr(), M, N, K, 2, res.data_ptr(),
              N, 1, pre.data_ptr(), N, y.data_ptr(), N, 1, tile, None, 0, torch.cuda.current_stream().cuda_stream)
    revisar(x, w, b, 'silu', res, None, y, None)
    p = x.double() @ w.double().t() + b.double()
    cerca(pre, p, (K + 24) * U * (x.double().abs() @ w.double().abs().t() + b.double().abs()), 'pre')
    assert torch.equal(y, asrn_amd.lineal_activa(x, w, b, 'silu', res))


@pytest.mark.parametrize('tile', [0, 128, 256])
@pytest.mark.parametrize('M,N,K,slabs', [(1, 8, 8, 0), (64, 128, 128, 1), (63, 136, 8, 1), (65, 8, 264, 2), (130, 256, 256, 3),
                                         (1000, 264, 520, 0), (2049, 768, 72, 5), (5000, 40, 1032, 0), (700, 520, 392, 100)])
@pytest.mark.parametrize('dt', [BF16, F16])
def test_weight_gradient(tile, M, N, K, slabs, dt):
    """The entry itself: every tile, slabs that leave steps and rows over, rows with other values between them, both results."""
    g, x = r(M, N + 24, dt=dt)[:, 8:8 + N], r(M, K + 8, dt=dt)[:, :K]
    ref, mag = g.double().t() @ x.double(), g.double().abs().t() @ x.double().abs()
    lib = _lib.load()
    ws = torch.empty(lib.asrn_weight_grad_workspace(M, N, K, tile, slabs), device=DEV, dtype=torch.uint8)
    for tipo in (F32, dt):
        out = torch.full((N + 1, K), 7.0, device=DEV, dtype=tipo)
        _lib.call('asrn_weight_grad', g.data_ptr(), N + 24, x.data_ptr(), K + 8, {BF16: 1, F16: 2}[dt], M, N, K, out.data_ptr(),
                  int(tipo == F32), tile, slabs, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
        cerca(out[:N], ref, M * U * mag, 'dw')
        assert (out[N] == 7).all()


def test_weight_gradient_keeps_infinities_in_their_rows():
    """Rows past the last and columns past the edge enter nothing: an infinite g reaches its own row of dW alone."""
    g, x = r(70, 40, dt=BF16), r(70, 48, dt=BF16)
    g[69, 39], x[3, 47] = torch.inf, torch.nan
    w = r(40, 48, dt=BF16).requires_grad_()
    dw, = torch.autograd.grad(asrn_amd.lineal_activa(x, w), w, g)
    assert dw[:39, :47].isfinite().all() and not dw[39, :47].isfinite().any() and dw[:, 47].isnan().all()


def test_offsets_past_32_bits():
    """More than 2^31 values of x, y and its gradient: the last rows are those of the same rows alone, up to the sums' order."""
    M, K, N = 2 ** 20 + 70, 2056, 2072
    x = torch.empty(M, K, device=DEV, dtype=BF16).normal_().requires_grad_()
    w, b = (r(N, K, dt=BF16) / 64).requires_grad_(), r(N, dt=BF16).requires_grad_()
    y = asrn_amd.lineal_activa(x, w, b, 'gelu')
    fin = x.detach()[-300:].clone().requires_grad_()
    z = asrn_amd.lineal_activa(fin, w, b, 'gelu')
    gz = r(300, N, dt=BF16)
    gy = torch.zeros_like(y)
    gy[-300:] = gz
    cota = 4 * medio(BF16)
    a, c = y.detach()[-300:].double(), z.detach().double()
    assert ((a - c).abs() <= cota * c.abs() + 2 ** -12).all()
    largo, corto = torch.autograd.grad(y, (x, w, b), gy), torch.autograd.grad(z, (fin, w, b), gz)
    for g, h in ((largo[0][-300:], corto[0]), *zip(largo[1:], corto[1:])):
        g, h = g.double(), h.double()
        assert ((g - h).abs() <= cota * h.abs() + 2 ** -7 * h.abs().max()).all()
    assert not largo[0][:-300].any()
    torch.cuda.empty_cache()


def test_forward_tangents_are_refused():
    import torch.autograd.forward_ad as fwd
    args = [r(20, 8), r(6, 8), r(6), r(20, 6)]
    for i in range(4):
        for grad in (True, False):
            with fwd.dual_level(), torch.set_grad_enabled(grad):
                x, w, b, res = [fwd.make_dual(t.clone(), torch.ones_like(t)) if j == i else t for j, t in enumerate(args)]
                with pytest.raises(RuntimeError, match='jvp|forward'):
                    asrn_amd.lineal_activa(x, w, b, 'gelu', res)


@pytest.mark.parametrize('forma', [(5, 8), (100, 8), (2, 60, 8), (8,)])
def test_result_changed_in_place(forma):
    """As F.linear's result, this one may be changed in place, under autograd and when it was made without."""
    x, w, b = r(*forma).requires_grad_(), r(6, 8).requires_grad_(), r(6).requires_grad_()
    y = asrn_amd.lineal_activa(x, w, b, 'silu')
    gy = torch.randn_like(y)
    ref = torch.autograd.grad(torch.relu(2 * y), (x, w, b), gy)
    y = asrn_amd.lineal_activa(x, w, b, 'silu')
    y *= 2
    y.relu_()
    for a, v in zip(torch.autograd.grad(y, (x, w, b), gy), ref):
        assert torch.equal(a, v)
    p = r(6).requires_grad_()
    with torch.no_grad():
        y = asrn_amd.lineal_activa(x, w, b)
    antes = y.clone()
    y *= p
    assert torch.equal(torch.autograd.grad(y, p, gy)[0], (antes * gy).reshape(-1, 6).sum(0))


@pytest.mark.parametrize('dt', [BF16, F16])
def test_weight_gradient_of_odd_widths_keeps_its_sums(dt):
    """16-bit rows that no vector divides: the sums over the rows stay in fp32 to their end, as those of whole units do. Values
    in sixteenths whose sums fp32 holds exactly, in 16 blocks of rows that nearly cancel: only the result is rounded."""
    M, N, K = 16384, 9, 7
    x = 1 + torch.randint(0, 16, (M, K), device=DEV) / 16
    x = x * (1 - 2 * (torch.arange(M, device=DEV) // 1024 % 2))[:, None]
    g = torch.randint(-2, 3, (M, N), device=DEV).float()
    g[:, 0] = 1
    ref = g.double().t() @ x.double()
    w, x, g = r(N, K, dt=dt).requires_grad_(), x.to(dt), g.to(dt)
    dw, = torch.autograd.grad(asrn_amd.lineal_activa(x, w), w, g)
    assert torch.equal(dw, ref.to(dt))
    w = r(N, K).requires_grad_()
    with torch.autocast('cuda', dtype=dt):
        y = asrn_amd.lineal_activa(x, w)
    assert torch.equal(torch.autograd.grad(y, w, g)[0].double(), ref)


@pytest.mark.parametrize('dt', [BF16, F16])
def test_odd_widths_captured_and_replayed(dt):
    """The weight gradient in slabs in a graph, on new values each time, with eager work between."""
    x, w, b, gy = r(4096, 33, dt=dt), r(41, 33, dt=dt).requires_grad_(), r(41, dt=dt).requires_grad_(), r(4096, 41, dt=dt)

    def paso():
        return torch.autograd.grad(asrn_amd.lineal_activa(x, w, b, 'silu'), (w, b), gy)
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
        x.copy_(r(4096, 33))
        gy.copy_(r(4096, 41))
        eager = [t.clone() for t in paso()]
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, v) for a, v in zip(fijos, eager)), i


@pytest.mark.parametrize('dt', [BF16, F16])
def test_gelu_of_16_bit_products(dt):
    """GELU alone (the product with the unit matrix, results in fp32) and its derivative. Phi of erfc's approximation is within
    0.75e-7, and fp32 adds at most: the reciprocal's 2^-23 and its argument's 2^-24 by the slope of t p(t), up to 1.72, 3.1e-7;
    three coefficients and two sums below 1, 2^-25 each, two coefficients below 1/4, two sums and a product below 1/2, 2.1e-7;
    of the exponential, whose square's 5 roundings count x^2 / 2 times, and the last product, Phi (2^-23 + 5 x^2 2^-25) and
    2^-26, 1.0e-7: together below 7e-7 (2.7e-7 found)."""
    x = torch.linspace(-9, 9, 64 * 4000, device=DEV).to(dt).view(-1, 64).requires_grad_()
    uno, cero = torch.eye(64, device=DEV, dtype=dt), torch.zeros(x.shape, device=DEV)
    y = asrn_amd.lineal_activa(x, uno, activacion='gelu', residuo=cero)
    x64 = x.detach().double()
    ref, der = act64(x64, 'gelu')
    assert ((y.double() - ref).abs() <= 7e-7 * x64.abs() + 2 * U * ref.abs()).all()
    # its derivative, rounded to dt: Phi as above and x phi(x), whose roundings are 6 U and the exponential's
    g, = torch.autograd.grad(y, x, torch.ones_like(y))
    cota = 7e-7 + 12 * U * x64.abs()
    assert ((g.double() - der).abs() <= cota + medio(dt) * (der.abs() + cota) + menor(dt)).all()
