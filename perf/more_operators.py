"""Performance cases of a local block's operators with a per-channel state, through the public API.

Kinds of case (the key 'tipo'):
  conv       the causal convolution of each channel with its bias and activation: a text's forward and backward
             (conv_canal), or one token's step on its window (paso_conv_canal)
  selectiva  the selective state space scan: a text's forward and backward, a prompt's forward with its final state
             (escaneo_selectivo), or one token's step on the state (paso_selectivo)
  lineal     the product with bias, activation and residual in its epilogue, forward and backward or forward alone
             (lineal_activa)

own = True runs the framework's kernels; else the same formulas in elementary torch operations. exact() restates them in
float64. dato is the activations' dtype; parameters that a model keeps in fp32 (the convolution's, A, D, the step sizes'
bias) are fp32.
"""
import math

import torch

own = False

DEV = 'cuda'
TIPOS = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
TAU_MAX = 1024                    # the longest time scale of a channel's state at the start, in tokens


def listed():
    return [
        # one token of 16 texts on a d = 768 model: launches count
        dict(name='conv_paso', tipo='conv', modo='paso', B=16, L=1, d=768, k=4, act='silu', dato='fp32'),
        # that model's training batch under autocast
        dict(name='conv_media', tipo='conv', modo='entrenar', B=8, L=2048, d=768, k=4, act='silu', dato='bf16'),
        # a wider window, rows and channels that no vector or tile divides
        dict(name='conv_irregular', tipo='conv', modo='entrenar', B=3, L=1537, d=390, k=7, act='gelu', dato='fp32'),
        # the state's step for the same 16 texts
        dict(name='selectiva_paso', tipo='selectiva', modo='paso', B=16, L=1, d=768, N=16, puerta=True, estado=True,
             dato='fp32'),
        # two long prompts read before writing; few channels, so the text itself is split
        dict(name='selectiva_texto', tipo='selectiva', modo='texto', B=2, L=32768, d=768, N=16, puerta=True, estado=False,
             dato='bf16'),
        # the training batch
        dict(name='selectiva_media', tipo='selectiva', modo='entrenar', B=8, L=2048, d=768, N=16, puerta=True, estado=False,
             dato='bf16'),
        # continued texts of an odd length, a narrow model, a state that fills no register tile, no gate
        dict(name='selectiva_irregular', tipo='selectiva', modo='entrenar', B=3, L=1021, d=200, N=11, puerta=False,
             estado=True, dato='fp32'),
        # a feed-forward's first product for one token of 16 texts: the weights' bytes count
        dict(name='lineal_paso', tipo='lineal', modo='texto', M=16, K=768, N=1536, act='gelu', residuo=False, dato='fp32'),
        # the feed-forward of the training batch: its first product and GELU, then its second onto the fp32 residual
        dict(name='lineal_media', tipo='lineal', modo='entrenar', M=16384, K=768, N=1536, act='gelu', residuo=False,
             dato='bf16'),
        dict(name='lineal_residuo', tipo='lineal', modo='entrenar', M=16384, K=1536, N=768, act='no', residuo=True,
             dato='bf16'),
        # sizes that no tile divides, in fp32
        dict(name='lineal_irregular', tipo='lineal', modo='entrenar', M=1003, K=389, N=517, act='silu', residuo=True,
             dato='fp32'),
        # a d = 2048 model's feed-forward over a prompt
        dict(name='lineal_grande', tipo='lineal', modo='texto', M=8192, K=2048, N=4096, act='gelu', residuo=False,
             dato='bf16'),
    ]


def draw(rng):
    def log(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    tipo = rng.choice(['conv', 'selectiva', 'lineal'])
    dato = rng.choice(['fp32', 'bf16', 'bf16', 'fp16'])
    act = rng.choice(['no', 'gelu', 'silu'])
    if tipo == 'conv':
        modo = rng.choice(['paso', 'entrenar', 'entrenar'])
        B, d, k = rng.randint(1, 16), log(24, 2048), rng.randint(1, 8)
        L = 1 if modo == 'paso' else max(1, min(log(1, 8192), 8 * 2048 * 768 // (B * d)))
        return dict(tipo=tipo, modo=modo, B=B, L=L, d=d, k=k, act=act, dato=dato)
    if tipo == 'selectiva':
        modo = rng.choice(['paso', 'texto', 'entrenar', 'entrenar'])
        B, d, N = rng.randint(1, 16), log(24, 1536), rng.randint(2, 24)
        most = {'paso': 1, 'texto': 2 * 32768 * 768 * 16, 'entrenar': 8 * 2048 * 768 * 16}[modo] // (B * d * N)
        L = 1 if modo == 'paso' else max(1, min(log(1, 32768 if modo == 'texto' else 4096), most))
        return dict(tipo=tipo, modo=modo, B=B, L=L, d=d, N=N, puerta=rng.random() < 0.6,
                    estado=modo == 'paso' or rng.random() < 0.4, dato=dato)
    modo = rng.choice(['texto', 'entrenar'])
    K, N = log(48, 3000), log(48, 4096)
    M = max(1, min(log(1, 16384), 16384 * 768 * 1536 // (K * N)))
    return dict(tipo=tipo, modo=modo, M=M, K=K, N=N, act=act, residuo=rng.random() < 0.5, dato=dato)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = TIPOS[case['dato']]

    def r(*forma):
        return torch.randn(*forma, generator=g, device=DEV)

    st = {'case': dict(case)}
    entrena = case['modo'] == 'entrenar'
    if case['tipo'] == 'conv':
        B, L, d, k = (case[n] for n in 'BLdk')
        cota = k ** -0.5
        st |= {'w': cota * (2 * torch.rand(d, 1, k, generator=g, device=DEV) - 1), 'b': 0.2 * r(d)}
        if case['modo'] == 'paso':
            return st | {'z': r(B, d).to(dt), 'ventana': r(B, d, k - 1).to(dt)}
        st |= {'z': r(B, L, d).to(dt), 'gy': r(B, L, d).to(dt)}
        for n in ('z', 'w', 'b'):
            st[n].requires_grad_(entrena)
        return st
    if case['tipo'] == 'selectiva':
        B, L, d, N = (case[n] for n in 'BLdN')
        forma = (B, d) if case['modo'] == 'paso' else (B, L, d)
        # channels' time scales from 1 to TAU_MAX tokens, the step sizes around them by the text
        tau = torch.logspace(0, math.log10(TAU_MAX), d, device=DEV)
        st |= {'u': r(*forma).to(dt), 'dl': (0.7 * r(*forma)).to(dt), 'sesgo': torch.log(torch.expm1(1 / tau)),
               'A': -torch.arange(1, N + 1, device=DEV, dtype=torch.float32).repeat(d, 1) * torch.exp(0.1 * r(d, N)),
               'Bm': r(*forma[:-1], N).to(dt), 'C': r(*forma[:-1], N).to(dt), 'D': 1 + 0.1 * r(d),
               'z': r(*forma).to(dt) if case['puerta'] else None, 'h': r(B, d, N) if case['estado'] else None}
        if entrena:
            st |= {'gy': r(*forma).to(dt), 'gh': r(B, d, N) if case['estado'] else None}
            for n in HOJAS:
                if st[n] is not None:
                    st[n].requires_grad_()
        return st
    M, K, N = (case[n] for n in 'MKN')
    st |= {'x': r(M, K).to(dt), 'w': (K ** -0.5 * r(N, K)).to(dt), 'b': (0.2 * r(N)).to(dt),
           # the residual stream is fp32 whatever the products' dtype
           'res': r(M, N) if case['residuo'] else None}
    if entrena:
        st |= {'gy': r(M, N).to(torch.float32 if case['residuo'] else dt)}
        for n in ('x', 'w', 'b', 'res'):
            if st[n] is not None:
                st[n].requires_grad_()
    return st


HOJAS = ('u', 'dl', 'A', 'Bm', 'C', 'D', 'z', 'sesgo', 'h')


# ---------------------------------------------------------------------------------------------------------------------
# plain forms: elementary operations in 32 bits, long sums in 64
# ---------------------------------------------------------------------------------------------------------------------

def _sigma(x):
    return 1 / (1 + torch.exp(-x))


def _activar(x, act):
    if act == 'gelu':
        return 0.5 * x * (1 + torch.erf(x * 0.5 ** 0.5))
    return x * _sigma(x) if act == 'silu' else x


def _derivada(x, act):
    if act == 'gelu':
        return 0.5 * (1 + torch.erf(x * 0.5 ** 0.5)) + x * torch.exp(-0.5 * x * x) * (2 * math.pi) ** -0.5
    if act == 'silu':
        s = _sigma(x)
        return s * (1 + x * (1 - s))
    return torch.ones_like(x)


def _conv(st):
    c, w, b = st['case'], st['w'][:, 0].float(), st['b']
    k, act = c['k'], c['act']
    if c['modo'] == 'paso':
        v = torch.cat([st['ventana'], st['z'][..., None]], -1)
        return _activar((v.float() * w).sum(-1) + b, act).to(v.dtype), v[..., 1:].contiguous()
    z = st['z'].detach()
    B, L, d = z.shape
    zf = torch.cat([z.new_zeros(B, k - 1, d), z], 1).float()
    pre = b + sum(zf[:, j:j + L] * w[:, j] for j in range(k))
    gp = st['gy'].float() * _derivada(pre, act)
    gz = torch.zeros_like(zf)
    gw = []
    for j in range(k):
        gz[:, j:j + L] += gp * w[:, j]
        gw.append((gp * zf[:, j:j + L]).double().sum((0, 1)))
    return (_activar(pre, act).to(z.dtype), gz[:, k - 1:].to(z.dtype), torch.stack(gw, -1)[:, None].float(),
            gp.double().sum((0, 1)).float())


def _recorrer(a, b, h):
    """h_t = a_t h_{t-1} + b_t over axis 1 by doubling, from h: every h_t."""
    a, b = a.clone(), b.clone()
    b[:, 0] += a[:, 0] * h
    n = 1
    while n < a.shape[1]:
        b[:, n:] += a[:, n:] * b[:, :-n].clone()
        a[:, n:] = a[:, n:] * a[:, :-n].clone()
        n *= 2
    return b


def _paso_delta(st, i, j):
    x = st['dl'][:, i:j].float() + st['sesgo']
    return x, x.clamp(min=0) + torch.log1p(torch.exp(-x.abs()))


TROZO = 256


def _selectiva(st):
    c, A, D = st['case'], st['A'], st['D']
    if c['modo'] == 'paso':
        st = {n: v[:, None] if n in ('u', 'dl', 'Bm', 'C', 'z') and v is not None else v for n, v in st.items()}
    u, Bm, C, z = st['u'], st['Bm'], st['C'], st['z']
    B, L, d = u.shape
    h = torch.zeros(B, d, c['N'], device=DEV) if st['h'] is None else st['h']
    hs, ys = [h], []
    for i in range(0, L, TROZO):
        j = min(i + TROZO, L)
        delta = _paso_delta(st, i, j)[1]
        todas = _recorrer(torch.exp(delta[..., None] * A), (delta * u[:, i:j].float())[..., None] * Bm[:, i:j, None].float(),
                          hs[-1])
        hs.append(todas[:, -1].clone())
        y = (todas * C[:, i:j, None].float()).sum(-1) + D * u[:, i:j].float()
        if z is not None:
            zf = z[:, i:j].float()
            y = y * zf * _sigma(zf)
        ys.append(y.to(u.dtype))
    y = torch.cat(ys, 1)
    if c['modo'] == 'paso':
        return y[:, 0], hs[-1]
    if c['modo'] == 'texto':
        return y, hs[-1]
    # backward, the pieces from the last to the first: g is the gradient of the state that leaves the piece
    g = torch.zeros_like(h) if st['h'] is None else st['gh']
    gu, gdl, gz = (torch.empty(B, L, d, device=DEV) for _ in range(3))
    gB, gC = (torch.empty(B, L, c['N'], device=DEV) for _ in range(2))
    gA, gD = torch.zeros(d, c['N'], device=DEV, dtype=torch.float64), torch.zeros(d, device=DEV, dtype=torch.float64)
    for n, i in reversed(list(enumerate(range(0, L, TROZO)))):
        j = min(i + TROZO, L)
        x, delta = _paso_delta(st, i, j)
        uf, Bf, Cf, gy = u[:, i:j].float(), Bm[:, i:j, None].float(), C[:, i:j, None].float(), st['gy'][:, i:j].float()
        a = torch.exp(delta[..., None] * A)
        todas = _recorrer(a, (delta * uf)[..., None] * Bf, hs[n])
        antes = torch.cat([hs[n][:, None], todas[:, :-1]], 1)
        if z is not None:
            zf = z[:, i:j].float()
            s = _sigma(zf)
            gz[:, i:j] = gy * ((todas * Cf).sum(-1) + D * uf) * s * (1 + zf * (1 - s))
            gy = gy * zf * s
        # the gradient of h_t: gy_t C_t + a_{t+1} (that of h_{t+1}), the same recurrence from the end
        alreves = torch.flip(torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1), (1,))
        gh = torch.flip(_recorrer(alreves, torch.flip(gy[..., None] * Cf, (1,)), g), (1,))
        gC[:, i:j] = (gy[..., None] * todas).sum(2)
        gB[:, i:j] = (gh * (delta * uf)[..., None]).sum(2)
        gdu = (gh * Bf).sum(-1)
        ga = gh * antes * a
        gA += (ga * delta[..., None]).double().sum((0, 1))
        gdelta = (ga * A).sum(-1) + gdu * uf
        gdl[:, i:j] = gdelta * _sigma(x)
        gu[:, i:j] = gdu * delta + gy * D
        gD += (gy * uf).double().sum((0, 1))
        g = gh[:, 0] * a[:, 0]
    dt = u.dtype
    salida = [y] + ([] if st['h'] is None else [hs[-1]])
    salida += [gu.to(dt), gdl.to(dt), gA.float(), gB.to(dt), gC.to(dt), gD.float()]
    salida += [] if z is None else [gz.to(dt)]
    salida += [gdl.double().sum((0, 1)).float()] + ([] if st['h'] is None else [g])
    return tuple(salida)


def _lineal(st):
    act = st['case']['act']
    x, w = st['x'].detach().float(), st['w'].detach().float()
    pre = x @ w.t() + st['b'].detach().float()
    y = _activar(pre, act)
    y = y.to(st['x'].dtype) if st['res'] is None else st['res'].detach() + y
    if st['case']['modo'] == 'texto':
        return y
    gp = st['gy'].float() * _derivada(pre, act)
    dt = st['x'].dtype
    gs = ((gp @ w).to(dt), (gp.t() @ x).to(dt), gp.double().sum(0).to(dt))
    return (y, *gs) + (() if st['res'] is None else (st['gy'].clone(),))


def run(state):
    c = state['case']
    if not own:
        with torch.no_grad():
            return {'conv': _conv, 'selectiva': _selectiva, 'lineal': _lineal}[c['tipo']](state)
    import asrn_amd
    st, act = state, None if c.get('act') == 'no' else c.get('act')
    if c['tipo'] == 'conv':
        if c['modo'] == 'paso':
            return asrn_amd.paso_conv_canal(st['z'], st['ventana'], st['w'], st['b'], act, en_sitio=False)
        y = asrn_amd.conv_canal(st['z'], st['w'], st['b'], act)
        return y.detach(), *torch.autograd.grad(y, (st['z'], st['w'], st['b']), st['gy'])
    if c['tipo'] == 'selectiva':
        if c['modo'] == 'paso':
            return asrn_amd.paso_selectivo(st['u'], st['dl'], st['A'], st['Bm'], st['C'], st['h'], D=st['D'], puerta=st['z'],
                                           sesgo_delta=st['sesgo'], en_sitio=False)
        con_estado = c['modo'] == 'texto' or c['estado']
        y = asrn_amd.escaneo_selectivo(st['u'], st['dl'], st['A'], st['Bm'], st['C'], D=st['D'], puerta=st['z'],
                                       sesgo_delta=st['sesgo'], estado=st['h'], devolver_estado=con_estado)
        if c['modo'] == 'texto':
            return y
        hojas = [st[n] for n in HOJAS if st[n] is not None]
        if con_estado:
            y, h = y
            return y.detach(), h.detach(), *torch.autograd.grad((y, h), hojas, (st['gy'], st['gh']))
        return y.detach(), *torch.autograd.grad(y, hojas, st['gy'])
    y = asrn_amd.lineal_activa(st['x'], st['w'], st['b'], activacion=act, residuo=st['res'])
    if c['modo'] == 'texto':
        return y
    hojas = [st[n] for n in ('x', 'w', 'b', 'res') if st[n] is not None]
    return y.detach(), *torch.autograd.grad(y, hojas, st['gy'])


def work(case):
    """Bytes: each input read once and each output written once, of the backward too (which reads the inputs again, as a
    training step's backward does); flops as the formulas count them."""
    b = 4 if case['dato'] == 'fp32' else 2
    entrena = case['modo'] == 'entrenar'
    if case['tipo'] == 'conv':
        B, L, d, k = (case[n] for n in 'BLdk')
        n = B * L * d
        if case['modo'] == 'paso':
            return {'bytes': n * b * (2 + 2 * (k - 1)) + 4 * d * (k + 1), 'flops': 2 * n * k}
        return {'bytes': n * b * (5 if entrena else 2) + 8 * d * (k + 1), 'flops': n * k * (8 if entrena else 2)}
    if case['tipo'] == 'selectiva':
        B, L, d, N, p = (case[n] for n in ('B', 'L', 'd', 'N', 'puerta'))
        n, m, e = B * L * d, B * L * N, B * d * N
        bytes_ = b * (n * (3 + p) + 2 * m) + 4 * (d * N + e * (1 + case['estado']))
        if entrena:       # reads u, delta, z, gy, B, C; writes the gradients of the first three and of B and C
            bytes_ += b * (n * (5 + 2 * p) + 4 * m) + 4 * (d * N + 2 * e * case['estado'])
        return {'bytes': bytes_, 'flops': n * N * (22 if entrena else 6)}
    M, K, N = (case[n] for n in 'MKN')
    br = 4 if case['residuo'] else b
    bytes_ = b * (M * K + N * K) + M * N * br * (1 + case['residuo'])
    if entrena:
        bytes_ += b * 2 * (M * K + N * K) + M * N * br * (1 + case['residuo'])
    return {'bytes': bytes_, 'flops': 2 * M * K * N * (3 if entrena else 1)}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------

def _exacta_act(x, act):
    if act == 'gelu':
        return x * 0.5 * torch.erfc(-x / math.sqrt(2))
    return x * torch.sigmoid(x) if act == 'silu' else x


def _exacta_conv(st):
    c = st['case']
    k = c['k']
    if c['modo'] == 'paso':
        v = torch.cat([st['ventana'], st['z'][..., None]], -1)
        y = torch.einsum('bdk,dk->bd', v.double(), st['w'][:, 0].double()) + st['b'].double()
        return [_exacta_act(y, c['act']), v[..., 1:].double()]
    hojas = [st[n].detach().double().requires_grad_() for n in ('z', 'w', 'b')]
    z, w, b = hojas
    ventanas = torch.nn.functional.pad(z, (0, 0, k - 1, 0)).unfold(1, k, 1)          # (B, L, d, k)
    y = _exacta_act((ventanas * w[:, 0]).sum(-1) + b, c['act'])
    return [y.detach(), *torch.autograd.grad(y, hojas, st['gy'].double())]


def _exacta_selectiva(st):
    c = st['case']
    if c['modo'] == 'paso':
        st = {n: v.unsqueeze(1) if n in ('u', 'dl', 'Bm', 'C', 'z') and v is not None else v for n, v in st.items()}
    v = {n: None if st[n] is None else st[n].detach().double() for n in HOJAS}
    entrena = c['modo'] == 'entrenar'
    hojas = [t.requires_grad_(entrena) for t in v.values() if t is not None]
    h = v['u'].new_zeros(c['B'], c['d'], c['N']) if v['h'] is None else v['h']
    delta = torch.nn.functional.softplus(v['dl'] + v['sesgo'], threshold=1e9)
    du, ys = delta * v['u'], []
    for dt, dut, Bt, Ct in zip(*(t.unbind(1) for t in (delta, du, v['Bm'], v['C']))):     # one token after the other
        h = h * torch.exp(dt.unsqueeze(-1) * v['A']) + dut.unsqueeze(-1) * Bt.unsqueeze(1)
        ys.append((h * Ct.unsqueeze(1)).sum(-1))
    y = torch.stack(ys, 1) + v['D'] * v['u']
    if v['z'] is not None:
        y = y * (v['z'] * torch.sigmoid(v['z']))
    if c['modo'] == 'paso':
        return [y[:, 0], h]
    if not entrena:
        return [y, h]
    if st['h'] is None:
        return [y.detach(), *torch.autograd.grad(y, hojas, st['gy'].double())]
    return [y.detach(), h.detach(), *torch.autograd.grad((y, h), hojas, (st['gy'].double(), st['gh'].double()))]


def _exacta_lineal(st):
    hojas = [st[n].detach().double().requires_grad_() for n in ('x', 'w', 'b', 'res') if st[n] is not None]
    x, w, b = hojas[:3]
    y = _exacta_act(torch.mm(x, w.t()) + b, st['case']['act'])
    if st['res'] is not None:
        y = y + hojas[3]
    if st['case']['modo'] == 'texto':
        return [y.detach()]
    return [y.detach(), *torch.autograd.grad(y, hojas, st['gy'].double())]


def exact(case, seed):
    r = {'conv': _exacta_conv, 'selectiva': _exacta_selectiva, 'lineal': _exacta_lineal}[case['tipo']](prepare(case, seed))
    return r[0] if case['tipo'] == 'lineal' and case['modo'] == 'texto' else tuple(r)
