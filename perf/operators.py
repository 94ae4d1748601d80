"""Performance cases of the fine-tuning operators: training on preferences and on rewards, through the public API.

Kinds of case (the key 'tipo'):
  logp         the log-probabilities of given tokens from a vocabulary's logits, forward and backward, with the rows'
               entropy and a temperature where the case has them (log_probabilidades)
  preferencia  the preference loss of pairs of texts from their tokens' log-probabilities (perdida_preferencia)
  politica     the clipped policy loss with its KL and entropy terms (perdida_politica)
  norma8       a local block's LayerNorm that keeps its input in 8 bits for the backward (ops.norma8)
  gelu8        its GELU with the input kept in 8 bits (ops.gelu8)

Tokens outside the answers are ignored or masked, as a prompt's and the padding of a batch are. own = True runs the
framework's kernels; else the same formulas in elementary torch operations. exact() restates them in float64.
"""
import math

import torch

own = False

DEV = 'cuda'
NADA = -100                       # the label of tokens that are not scored
GRUPO = 32                        # neighbouring channels that share a scale in 8 bits


def listed():
    return [
        # a toy model's answers, byte vocabulary, float32: launches count
        dict(name='logp_minima', tipo='logp', B=2, L=100, V=256, bits=32, libres=0.3, entropia=False, T=1.0),
        # texts of a d = 768 model's training batch scored over its vocabulary, half of each a prompt
        dict(name='logp_media', tipo='logp', B=8, L=1024, V=50304, bits=16, libres=0.5, entropia=False, T=1.0),
        # sampled answers scored at the sampling temperature, with the entropy; a vocabulary no vector load divides
        dict(name='logp_irregular', tipo='logp', B=7, L=311, V=32003, bits=32, libres=0.25, entropia=True, T=0.7),
        # one pair of short texts, the reference's sums at hand
        dict(name='preferencia_minima', tipo='preferencia', P=1, L=60, forma='ipo', ref='textos', libres=0.3),
        # long texts, a ragged batch
        dict(name='preferencia_larga', tipo='preferencia', P=24, L=50001, forma='sigmoide', ref='fichas', libres=0.4),
        # a few short answers
        dict(name='politica_minima', tipo='politica', B=4, L=50, ventaja='textos', kl=True, entropia=False,
             reduccion='fichas', tope=None, libres=0.3),
        # a group of answers to each prompt, an advantage per answer, a KL to the reference
        dict(name='politica_media', tipo='politica', B=256, L=1024, ventaja='textos', kl=True, entropia=False,
             reduccion='textos', tope=None, libres=0.5),
        # long answers with an advantage per token, an entropy bonus and the second clip
        dict(name='politica_grande', tipo='politica', B=160, L=20001, ventaja='fichas', kl=True, entropia=True,
             reduccion='fichas', tope=3.0, libres=0.25),
        # the LayerNorms of the d = 768 model's blocks at its training batch, bf16 products
        dict(name='norma8_ancha', tipo='norma8', B=8, L=2048, d=768, bits=16),
        # ragged texts in float32
        dict(name='norma8_irregular', tipo='norma8', B=5, L=301, d=260, bits=32),
        # the feed-forward's hidden activations at the d = 768 model's training batch
        dict(name='gelu8_ancha', tipo='gelu8', B=8, L=2048, d=1536, bits=16),
        # a short ragged batch in float32
        dict(name='gelu8_irregular', tipo='gelu8', B=3, L=407, d=520, bits=32),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _libres(rng):
    return rng.choice([0.0, 0.25, 0.5, 0.75])


def draw(rng):
    tipo = rng.choice(['logp', 'logp', 'preferencia', 'politica', 'norma8', 'gelu8'])
    bits = rng.choice([16, 32])
    if tipo == 'logp':
        V = rng.choice([256, 1000, 8000, 8191, 32000, 32003, 50304])
        fichas = _log(rng, 16, min(16384, 200_000_000 // V))
        B = rng.choice([1, 2, 3, 5, 8])
        return dict(tipo=tipo, B=B, L=max(2, fichas // B), V=V, bits=bits, libres=_libres(rng),
                    entropia=rng.random() < 0.5, T=rng.choice([0.7, 1.0, 1.3]))
    if tipo == 'preferencia':
        fichas = _log(rng, 64, 2_400_000)
        P = min(_log(rng, 1, 128), fichas // 32)
        return dict(tipo=tipo, P=P, L=fichas // (2 * P), forma=rng.choice(['sigmoide', 'ipo', 'bisagra']),
                    ref=rng.choice(['fichas', 'textos', 'no']), libres=_libres(rng))
    if tipo == 'politica':
        fichas = _log(rng, 64, 3_200_000)
        B = min(_log(rng, 1, 512), fichas // 16)
        return dict(tipo=tipo, B=B, L=fichas // B, ventaja=rng.choice(['textos', 'fichas']), kl=rng.random() < 0.7,
                    entropia=rng.random() < 0.4, reduccion=rng.choice(['fichas', 'textos']),
                    tope=rng.choice([None, 3.0]), libres=_libres(rng))
    fichas = _log(rng, 64, 16384)
    B = rng.choice([1, 2, 5, 8])
    d = rng.choice([64, 96, 256, 260, 384, 512, 768])
    return dict(tipo=tipo, B=B, L=max(8, fichas // B), d=d if tipo == 'norma8' else 2 * d, bits=bits)


def _tipo_de(case):
    return torch.bfloat16 if case['bits'] == 16 else torch.float32


def _vistas(case, g, filas, L):
    """(filas, L) bools: the tokens of an answer. Each text opens with a prompt and ends in padding, together `libres`
    of its length on average; every text keeps one token at least."""
    r = torch.rand(filas, 2, generator=g, device=DEV)
    ini = (r[:, :1] * case['libres'] * L).long().clamp(max=L - 1)
    fin = L - (r[:, 1:] * case['libres'] * L).long()
    t = torch.arange(L, device=DEV)
    return (t >= ini) & (t < torch.maximum(fin, ini + 1))


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)
    dt = _tipo_de(case) if 'bits' in case else None
    st = {'case': case}
    if case['tipo'] == 'logp':
        B, L, V = case['B'], case['L'], case['V']
        x = torch.empty(B, L, V, dtype=dt, device=DEV)
        for b in range(B):
            x[b] = 2 * r(L, V)
        y = torch.randint(0, V, (B, L), generator=g, device=DEV)
        x.scatter_add_(2, y[..., None], torch.full((B, L, 1), 6.0, dtype=dt, device=DEV))     # tokens a model expects
        st |= {'x': x.requires_grad_(), 'y': y.masked_fill(~_vistas(case, g, B, L), NADA), 'g': r(B, L) / (B * L),
               'gh': r(B, L) * 1e-2 / (B * L)}
    elif case['tipo'] == 'preferencia':
        P, L = case['P'], case['L']
        lp = -r(2 * P, L).abs() * 2 - 0.01
        m = _vistas(case, g, 2 * P, L)
        ref = lp + 0.02 * r(2 * P, L)
        if case['ref'] == 'textos':
            ref = (ref.double() * m).sum(1).float()
        st |= {'lp': lp.requires_grad_(), 'm': m, 'ref': None if case['ref'] == 'no' else ref}
    elif case['tipo'] == 'politica':
        B, L = case['B'], case['L']
        vieja = -r(B, L).abs() * 2 - 0.01
        lp = (vieja + 0.15 * r(B, L)).clamp(max=0)
        st |= {'lp': lp.requires_grad_(), 'vieja': vieja, 'm': _vistas(case, g, B, L),
               'A': r(B) if case['ventaja'] == 'textos' else r(B, L),
               'ref': (vieja + 0.1 * r(B, L)).clamp(max=0) if case['kl'] else None,
               'H': (3 * torch.rand(B, L, generator=g, device=DEV)).requires_grad_() if case['entropia'] else None}
    elif case['tipo'] == 'norma8':
        B, L, d = case['B'], case['L'], case['d']
        ln = torch.nn.LayerNorm(d, device=DEV)
        with torch.no_grad():
            ln.weight.copy_(1 + 0.2 * r(d))
            ln.bias.copy_(0.2 * r(d))
        # a residual stream: a few channels far larger than the rest
        st |= {'ln': ln, 'x': (r(B, L, d) * (1 + 4 * r(d).abs() * (r(d) > 1.5))).requires_grad_(),
               'gy': r(B, L, d).to(dt), 'gx': r(B, L, d)}
    else:
        B, L, d = case['B'], case['L'], case['d']
        st |= {'u': (1.5 * r(B, L, d)).to(dt).requires_grad_(), 'gy': r(B, L, d).to(dt)}
    return st


# the preference loss's and the policy loss's constants in the cases
BETA, SUAVIZADO, RECORTE, BETA_KL, PESO_H = 0.1, 0.05, (0.2, 0.28), 0.04, 0.01


# ---------------------------------------------------------------------------------------------------------------------
# plain forms: elementary operations, in 32 bits (64 for long sums and for values next to a border)
# ---------------------------------------------------------------------------------------------------------------------

def _logp(st):
    c, y = st['case'], st['y']
    x = st['x'].detach().float() / c['T']
    ve = y != NADA
    t = y.clamp(min=0)[..., None]
    z = x - x.amax(-1, keepdim=True)
    e = z.exp()
    s = e.sum(-1, keepdim=True)
    lp = torch.where(ve, (z.gather(-1, t) - s.log())[..., 0], 0.0)
    p = e / s
    salida = [lp]
    gl = (st['g'] * ve)[..., None]
    dx = -gl * p
    dx.scatter_add_(-1, t, gl)
    if c['entropia']:
        logp = z - s.log()
        H = -(p * logp).sum(-1, keepdim=True)
        salida.append(H[..., 0] * ve)
        dx = dx - (st['gh'] * ve)[..., None] * p * (logp + H)
    return (*salida, (dx / c['T']).to(st['x'].dtype))


def _preferencia(st):
    c, m, ref = st['case'], st['m'], st['ref']
    P, n = c['P'], m.sum(1).double()
    fila = (st['lp'].detach().double() * m).sum(1)
    if ref is not None:
        fila = fila - (ref.double() if ref.dim() == 1 else (ref.double() * m).sum(1))
    div = n.clamp(min=1) if c['forma'] == 'ipo' else torch.ones_like(n)
    r = fila / div
    h = BETA * (r[:P] - r[P:])
    if c['forma'] == 'sigmoide':
        a, b = torch.log1p(torch.exp(-h.abs())) + (-h).clamp(min=0), torch.log1p(torch.exp(-h.abs())) + h.clamp(min=0)
        por, dh = (1 - SUAVIZADO) * a + SUAVIZADO * b, SUAVIZADO - 1 / (1 + torch.exp(h))
    elif c['forma'] == 'ipo':
        por, dh = (h / BETA - 0.5 / BETA) ** 2, 2 * (h / BETA - 0.5 / BETA) / BETA
    else:
        por, dh = (1 - h).clamp(min=0), -(h < 1).double()
    coef = torch.cat([dh, -dh]) * BETA / (P * div)
    return por.mean().float(), (BETA * r).float(), (coef[:, None] * m).float()


def _politica(st):
    c, m = st['case'], st['m']
    lp, A = st['lp'].detach().double(), st['A'].double()
    A = A[:, None].expand(lp.shape) if A.dim() == 1 else A
    d = lp - st['vieja'].double()
    r = d.exp()
    bajo, alto = RECORTE
    fuera = ((A > 0) & (d > math.log1p(alto))) | ((A < 0) & (d < math.log1p(-bajo)))
    pg = -torch.minimum(r * A, r.clamp(1 - bajo, 1 + alto) * A)
    dl = torch.where(fuera, 0.0, -r * A)
    if c['tope'] is not None:
        sobre = (A < 0) & (d > math.log(c['tope']))
        pg, dl = torch.where(sobre, -c['tope'] * A, pg), torch.where(sobre, 0.0, dl)
        fuera = fuera | sobre
    kl = torch.zeros_like(lp)
    if st['ref'] is not None:
        q = st['ref'].double() - lp
        kl = torch.expm1(q) - q
        pg, dl = pg + BETA_KL * kl, dl - BETA_KL * torch.expm1(q)
    H = torch.zeros_like(lp) if st['H'] is None else st['H'].detach().double()
    n = m.sum(1, keepdim=True)
    if c['reduccion'] == 'textos':
        peso = m.double() / (n.clamp(min=1) * (n > 0).sum())
    else:
        peso = m.double() / n.sum()
    todas = m.double() / n.sum()
    out = ((pg - PESO_H * H) * peso).sum().float()
    est = torch.stack([(fuera * todas).sum(), ((torch.expm1(d) - d) * todas).sum(), (kl * todas).sum(), (H * todas).sum()]).float()
    return (out, est, (dl * peso).float()) + (() if st['H'] is None else ((-PESO_H * peso).float(),))


def _ocho(x):
    """x as 8 bits hold it: per GRUPO channels the smallest power of two 2^e with max |x| <= 127 2^e, and integers."""
    d = x.shape[-1]
    v = torch.nn.functional.pad(x.detach().float(), (0, -d % GRUPO)).unflatten(-1, (-1, GRUPO))
    f, k = torch.frexp(v.abs().amax(-1, keepdim=True))
    e = (k - 7 + (f > 127 / 128).int()).clamp(min=-126)
    dos = lambda n: ((n + 127) << 23).view(torch.float32)          # 2^n from its bits (pow may be an ulp off)
    return (torch.round(v * dos(-e)) * dos(e)).flatten(-2)[..., :d]


def _norma8(st):
    ln, x = st['ln'], st['x'].detach()
    w, gy = ln.weight.detach(), st['gy'].float()
    mu = x.mean(-1, keepdim=True)
    rstd = 1 / (((x - mu) ** 2).mean(-1, keepdim=True) + ln.eps).sqrt()
    y = ((x - mu) * rstd * w + ln.bias.detach()).to(st['gy'].dtype)
    xh = (_ocho(x) - mu) * rstd
    q = gy * w
    dx = rstd * (q - q.mean(-1, keepdim=True) - xh * (q * xh).mean(-1, keepdim=True)) + st['gx']
    return y, dx, (gy * xh).sum((0, 1)), gy.sum((0, 1))


def _gelu8(st):
    u, gy = st['u'].detach(), st['gy'].float()
    v = u.float()
    y = 0.5 * v * (1 + torch.erf(v * 0.5 ** 0.5))
    v = _ocho(u)
    du = gy * (0.5 * (1 + torch.erf(v * 0.5 ** 0.5)) + v * torch.exp(-0.5 * v * v) * (2 * math.pi) ** -0.5)
    return y.to(u.dtype), du.to(u.dtype)


def run(state):
    c, tipo = state['case'], state['case']['tipo']
    if not own:
        with torch.no_grad():
            return {'logp': _logp, 'preferencia': _preferencia, 'politica': _politica, 'norma8': _norma8,
                    'gelu8': _gelu8}[tipo](state)
    import asrn_amd
    from asrn_amd import ops
    if tipo == 'logp':
        x = state['x']
        if c['entropia']:
            lp, H = asrn_amd.log_probabilidades(x, state['y'], ignorar=NADA, temperatura=c['T'], entropia=True)
            return lp.detach(), H.detach(), *torch.autograd.grad((lp, H), x, (state['g'], state['gh']))
        lp = asrn_amd.log_probabilidades(x, state['y'], ignorar=NADA, temperatura=c['T'])
        return lp.detach(), *torch.autograd.grad(lp, x, state['g'])
    if tipo == 'preferencia':
        perdida, recompensas = asrn_amd.perdida_preferencia(
            state['lp'], state['m'], state['ref'], beta=BETA, tipo=c['forma'],
            suavizado=SUAVIZADO if c['forma'] == 'sigmoide' else 0.0, por_longitud=c['forma'] == 'ipo')
        return perdida.detach(), recompensas, *torch.autograd.grad(perdida, state['lp'])
    if tipo == 'politica':
        perdida, est = asrn_amd.perdida_politica(
            state['lp'], state['A'], state['vieja'], state['m'], recorte=RECORTE, tope=c['tope'], lp_ref=state['ref'],
            beta=BETA_KL if c['kl'] else 0.0, entropia=state['H'], peso_entropia=PESO_H if c['entropia'] else 0.0,
            reduccion=c['reduccion'])
        hojas = [state['lp']] + ([] if state['H'] is None else [state['H']])
        return perdida.detach(), est, *torch.autograd.grad(perdida, hojas)
    if tipo == 'norma8':
        ln = state['ln']
        y, x, _ = ops.norma8(ln, state['x'], state['gy'].dtype)
        return y.detach(), *torch.autograd.grad((y, x), (state['x'], ln.weight, ln.bias), (state['gy'], state['gx']))
    y, _ = ops.gelu8(state['u'])
    return y.detach(), *torch.autograd.grad(y, state['u'], state['gy'])


def work(case):
    """Bytes: each input read once and each output written once (the logits of rows that are not scored need not be
    read); flops as the formulas count them."""
    tipo = case['tipo']
    if tipo == 'logp':
        n, V, b = case['B'] * case['L'], case['V'], case['bits'] // 8
        vistas = 1 - 0.9 * case['libres']
        return {'bytes': n * V * b * (1 + vistas) + n * (12 + 8 * (1 + case['entropia'])),
                'flops': n * V * vistas * (13 if case['entropia'] else 6)}
    if tipo == 'preferencia':
        n = 2 * case['P'] * case['L']
        return {'bytes': n * (4 + 1 + 4 + 4 * (case['ref'] == 'fichas')), 'flops': 4 * n}
    if tipo == 'politica':
        n = case['B'] * case['L']
        return {'bytes': n * (4 + 4 + 1 + 4 + 4 * (case['ventaja'] == 'fichas') + 4 * case['kl'] + 8 * case['entropia']),
                'flops': 40 * n}
    n, b = case['B'] * case['L'] * case['d'], case['bits'] // 8
    if tipo == 'norma8':
        return {'bytes': n * (4 + b + b + 4 + 4), 'flops': 25 * n}
    return {'bytes': 4 * n * b, 'flops': 30 * n}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------

def _exacta_logp(st):
    c, lps, hs, dxs = st['case'], [], [], []
    x, y = st['x'].detach().flatten(0, 1), st['y'].flatten()
    g, gh = st['g'].double().flatten(), st['gh'].double().flatten()
    paso = max(1, 50_000_000 // c['V'])
    for i in range(0, x.shape[0], paso):
        xi, yi = x[i:i + paso].double() / c['T'], y[i:i + paso]
        ve = (yi != NADA).double()
        logp = torch.log_softmax(xi, -1)
        p, uno = logp.exp(), torch.zeros_like(logp).scatter_(1, yi.clamp(min=0)[:, None], 1.0)
        lps.append((logp * uno).sum(1) * ve)
        dx = (g[i:i + paso] * ve)[:, None] * (uno - p)
        if c['entropia']:
            H = -(p * logp).sum(1)
            hs.append(H * ve)
            dx -= (gh[i:i + paso] * ve)[:, None] * p * (logp + H[:, None])
        dxs.append((dx / c['T']).float() if c['bits'] == 16 else dx / c['T'])
    forma = st['y'].shape
    return [torch.cat(v).view(*forma, *v[0].shape[1:]) for v in (lps, hs, dxs) if v]


def _exacta_preferencia(st):
    c, m = st['case'], st['m'].double()
    P = c['P']
    lp = st['lp'].detach().double().requires_grad_()
    suma = (lp * m).sum(1)
    if st['ref'] is not None:
        suma = suma - (st['ref'].double() if st['ref'].dim() == 1 else (st['ref'].double() * m).sum(1))
    r = suma / m.sum(1) if c['forma'] == 'ipo' else suma
    delta = r[:P] - r[P:]
    ls = torch.nn.functional.logsigmoid
    por = {'sigmoide': lambda: -(1 - SUAVIZADO) * ls(BETA * delta) - SUAVIZADO * ls(-BETA * delta),
           'ipo': lambda: (delta - 0.5 / BETA) ** 2, 'bisagra': lambda: torch.relu(1 - BETA * delta)}[c['forma']]()
    perdida = por.sum() / P
    return [perdida.detach(), (BETA * r).detach(), *torch.autograd.grad(perdida, lp)]


def _exacta_politica(st):
    c, m = st['case'], st['m'].double()
    hojas = [st['lp'].detach().double().requires_grad_()]
    if st['H'] is not None:
        hojas.append(st['H'].detach().double().requires_grad_())
    lp, A = hojas[0], st['A'].double()
    A = A[:, None] if A.dim() == 1 else A
    r = torch.exp(lp - st['vieja'].double())
    dentro = r.clamp(1 - RECORTE[0], 1 + RECORTE[1])
    pg = torch.minimum(r * A, dentro * A)
    fuera = r * A > dentro * A
    if c['tope'] is not None:
        sobre = (A < 0) & (r > c['tope'])
        pg, fuera = torch.where(sobre, c['tope'] * A, pg), fuera | sobre
    por = -pg
    kl = torch.zeros_like(lp)
    if st['ref'] is not None:
        kl = torch.exp(st['ref'].double() - lp) - 1 - (st['ref'].double() - lp)
        por = por + BETA_KL * kl
    if st['H'] is not None:
        por = por - PESO_H * hojas[1]
    media = lambda v: (v * m).sum() / m.sum()
    if c['reduccion'] == 'textos':
        n = m.sum(1)
        perdida = ((por * m).sum(1) / n.clamp(min=1)).sum() / (n > 0).sum()
    else:
        perdida = media(por)
    est = [media(fuera.double()), media(r - 1 - (lp - st['vieja'].double())), media(kl),
           media(hojas[1]) if st['H'] is not None else media(torch.zeros_like(lp))]
    return [perdida.detach(), torch.stack(est).detach(), *torch.autograd.grad(perdida, hojas)]


def _exacto_ocho(x):
    """x as 8 bits hold it, from the definition of the scale: 2^e, e the smallest with max |x| / 127 <= 2^e."""
    d = x.shape[-1]
    v = torch.nn.functional.pad(x.detach().double(), (0, -d % GRUPO)).unflatten(-1, (-1, GRUPO))
    e = torch.ceil(torch.log2(v.abs().amax(-1, keepdim=True) / 127)).clamp(min=-126)
    dos = torch.ldexp(torch.ones((), dtype=torch.float64), e.long().cpu()).to(v.device)
    return (torch.round(v / dos) * dos).flatten(-2)[..., :d]


def _exacta_norma8(st):
    ln, x, gy = st['ln'], st['x'].detach().double(), st['gy'].double()
    w = ln.weight.detach().double()
    var, mu = torch.var_mean(x, -1, unbiased=False, keepdim=True)
    s = (var + ln.eps).sqrt()
    xh = (_exacto_ocho(x) - mu) / s
    q = gy * w
    dx = (q - q.mean(-1, keepdim=True) - xh * (q * xh).mean(-1, keepdim=True)) / s + st['gx'].double()
    return [(x - mu) / s * w + ln.bias.detach().double(), dx, (gy * xh).flatten(0, 1).sum(0), gy.flatten(0, 1).sum(0)]


def _exacta_gelu8(st):
    v, gy = st['u'].detach().double(), st['gy'].double()
    fi = lambda t: 0.5 * torch.erfc(-t / math.sqrt(2))
    q = _exacto_ocho(v)
    return [v * fi(v), gy * (fi(q) + q * torch.exp(-q * q / 2) / math.sqrt(2 * math.pi))]


def exact(case, seed):
    st = prepare(case, seed)
    return tuple({'logp': _exacta_logp, 'preferencia': _exacta_preferencia, 'politica': _exacta_politica,
                  'norma8': _exacta_norma8, 'gelu8': _exacta_gelu8}[case['tipo']](st))
