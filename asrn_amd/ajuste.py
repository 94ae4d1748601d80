"""Losses for fine-tuning a model on answers: the log-probabilities of given tokens, the preference loss of pairs of
texts and the clipped policy loss, each with its gradient, on the library's kernels (include/asrn_hip.h).

    lp = modelo.log_probabilidades(x, y)                      # (B, L): log p of y under the logits of x
    perdida, recompensas = perdida_preferencia(lp, y != -100, ref)         # rows: the chosen texts, then the rejected
    perdida, datos = perdida_politica(lp, ventaja, lp_vieja, y != -100)    # sampled answers and their advantages

The reference package has no counterpart; the functions stand beside the model's loss (ops.cross_entropy). GPU only.
Nothing waits on the host, so a step over them can be captured in a HIP graph.
"""
import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from ._lib import ptr, query
from .ops import _dev, _en

TIPOS = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}     # the kernels' logits
FORMAS = ('sigmoide', 'ipo', 'bisagra')
REDUCCIONES = ('fichas', 'textos')


def _denso(g):
    """An upstream gradient as contiguous fp32."""
    return (g if g.dtype == torch.float32 else g.float()).contiguous()


def _mismo_gpu(quien, dev, **tensores):
    for n, t in tensores.items():
        if t is not None and t.device != dev:
            raise ValueError(f'{quien}: {n} is on {t.device}, the rest on {dev}')


def _pasos(*ts):
    """The row and token strides of (B, L) tensors (0, 0 for None) as the C array the kernels' entry points take."""
    s = [v for t in ts for v in ((0, 0) if t is None else t.stride())]
    return (ctypes.c_int64 * len(s))(*s)


def _mascara(quien, m, forma, dev):
    """A (B, L) mask as bytes (nonzero keeps the token), or None."""
    if m is None:
        return None
    if tuple(m.shape) != tuple(forma):
        raise ValueError(f'{quien}: mascara {tuple(m.shape)} against {tuple(forma)} tokens')
    _mismo_gpu(quien, dev, mascara=m)
    return (m if m.dtype == torch.bool else m != 0).view(torch.uint8)


def _f32(t):
    return t if t is None or t.dtype == torch.float32 else t.float()


def _fijo(t):
    """A constant input: fp32, outside autograd."""
    return t if t is None or (t.dtype == torch.float32 and not t.requires_grad) else t.detach().float()


def _numero(quien, nombre, v, minimo, maximo=math.inf, abierto=False):
    if not isinstance(v, (int, float)) or isinstance(v, bool) or not (minimo < v if abierto else minimo <= v) or not v <= maximo \
            or not math.isfinite(v):
        raise ValueError(f'{quien}: {nombre}={v!r}: a number {"above" if abierto else "from"} {minimo}'
                         + (f' to {maximo}' if maximo < math.inf else ''))
    return float(v)


# ---------------------------------------------------------------------------------------------------------------------
# log-probabilities of given tokens
# ---------------------------------------------------------------------------------------------------------------------

def _filas(x):
    """logits (..., V) as (row count, L, stride over b, stride over t) for rows b L + t read in place, and the tensor
    they are read from: a (B, L, V) slice needs no copy, more leading axes are flattened."""
    V = x.shape[-1]
    if x.stride(-1) != 1 and V > 1:
        x = x.contiguous()
    if x.dim() > 3:
        x = x.reshape(-1, *x.shape[-2:])
    if x.dim() == 1:
        return 1, 1, 0, 0, x
    if x.dim() == 2:
        return x.shape[0], x.shape[0], 0, x.stride(0), x
    return x.shape[0] * x.shape[1], x.shape[1], x.stride(0), x.stride(1), x


class LogProbabilidades(torch.autograd.Function):
    """asrn_token_logp_fwd/bwd: (log-probabilities, entropies or None) of rows of logits, fp32; the gradient comes back
    in the logits' dtype."""

    @staticmethod
    def forward(ctx, logits, y, ignorar, inv_t, entropia):
        dev, V = logits.device, logits.shape[-1]
        filas, L, sb, st, x = _filas(logits)
        t = y.reshape(-1)
        lp = torch.empty(y.shape, dtype=torch.float32, device=dev)
        stats = torch.empty((filas, 2), dtype=torch.float32, device=dev)
        H = torch.empty(y.shape, dtype=torch.float32, device=dev) if entropia else None
        if filas:
            _en(dev, 'asrn_token_logp_fwd', ptr(x), TIPOS[x.dtype], filas, L, V, sb, st, ptr(t), ignorar, inv_t, ptr(lp),
                    ptr(H), ptr(stats))
        ctx.save_for_backward(x, t, stats, H)
        ctx.meta = (filas, L, sb, st, ignorar, inv_t, logits.shape)
        ctx.set_materialize_grads(False)
        return lp, H

    @staticmethod
    @once_differentiable
    def backward(ctx, g, gh):
        x, t, stats, H = ctx.saved_tensors
        filas, L, sb, st, ignorar, inv_t, forma = ctx.meta
        if g is None and gh is None:
            return None, None, None, None, None
        g = None if g is None else _denso(g)
        gh = None if gh is None else _denso(gh)
        dx = torch.empty(forma, dtype=x.dtype, device=x.device)
        if filas:
            _en(x.device, 'asrn_token_logp_bwd', ptr(x), TIPOS[x.dtype], filas, L, forma[-1], sb, st, ptr(t), ignorar, inv_t,
                    ptr(stats), ptr(H), ptr(g), ptr(gh), ptr(dx))
        return dx, None, None, None, None


def log_probabilidades(logits, y, ignorar=-100, temperatura=1.0, entropia=False):
    """log softmax(logits / temperatura) at the tokens y, in fp32: logits (..., V) fp32, bf16 or fp16, read as they are
    through their strides (no fp32 copy), y (...) integers. 0 where y == ignorar, and no gradient there; NaN for a token
    outside [0, V). entropia=True: (log-probabilities, the rows' entropy), both with gradients; an ignored row's entropy
    is 0. The gradient is in the logits' dtype. Sums are held in fp32, as cross_entropy's."""
    quien = 'log_probabilidades'
    dev = _dev(logits)
    if logits.dim() < 1 or tuple(logits.shape[:-1]) != tuple(y.shape):
        raise ValueError(f'{quien}: logits {tuple(logits.shape)} against tokens {tuple(y.shape)}')
    if logits.dtype not in TIPOS:
        raise ValueError(f'{quien}: logits of {logits.dtype} (fp32, bf16 or fp16 are taken)')
    if logits.shape[-1] < 1 or y.is_floating_point() or y.is_complex() or y.dtype == torch.bool:
        raise ValueError(f'{quien}: a vocabulary of {logits.shape[-1]} tokens and token ids of {y.dtype}')
    if y.numel() >= 1 << 31:
        raise ValueError(f'{quien}: {y.numel()} tokens (up to 2**31 - 1)')
    _mismo_gpu(quien, dev, y=y)
    T = _numero(quien, 'temperatura', temperatura, 1e-6, 1e6)
    lp, H = LogProbabilidades.apply(logits, y.to(torch.int64), int(ignorar), 1.0 / T, bool(entropia))
    return (lp, H) if entropia else lp


# ---------------------------------------------------------------------------------------------------------------------
# the preference loss
# ---------------------------------------------------------------------------------------------------------------------

class Preferencia(torch.autograd.Function):
    """asrn_preference_fwd/bwd: (loss, rewards) of lp (2P, L); the gradient of a row is one coefficient, kept from the
    forward."""

    @staticmethod
    def forward(ctx, lp, fijos):
        m, ref, forma, beta, suavizado, margen, por_longitud = fijos      # constants: no autograd around them
        dev = lp.device
        P, L = lp.shape[0] // 2, lp.shape[1]
        perdida = torch.empty((), dtype=torch.float32, device=dev)
        rec = torch.empty((2 * P,), dtype=torch.float32, device=dev)
        wsb = query('asrn_preference_workspace', P, L)
        ws = torch.empty((max(wsb, 0) + 8 * P,), dtype=torch.uint8, device=dev)
        coef = ws.data_ptr() + max(wsb, 0)           # the rows' coefficients, kept for the backward, behind the workspace
        por_fila = ref is not None and ref.dim() == 1
        ref_pasos = None if ref is None else (ctypes.c_int64 * 2)(ref.stride(0), 0) if por_fila else _pasos(ref)
        _en(dev, 'asrn_preference_fwd', ptr(lp), _pasos(lp), ptr(ref), ref_pasos, int(por_fila), ptr(m),
                None if m is None else _pasos(m), P, L, FORMAS.index(forma), beta, suavizado, margen, int(por_longitud),
                ptr(perdida), ptr(rec), coef, ptr(ws), wsb)
        ctx.save_for_backward(ws, m)
        ctx.meta = (P, L, max(wsb, 0))
        ctx.mark_non_differentiable(rec)
        ctx.set_materialize_grads(False)
        return perdida, rec

    @staticmethod
    @once_differentiable
    def backward(ctx, g, _):
        ws, m = ctx.saved_tensors
        P, L, wsb = ctx.meta
        if g is None:
            return None, None
        dlp = torch.empty((2 * P, L), dtype=torch.float32, device=ws.device)
        gc = _denso(g)
        _en(ws.device, 'asrn_preference_bwd', ws.data_ptr() + wsb, ptr(gc), ptr(m), None if m is None else _pasos(m), P, L,
                ptr(dlp))
        return dlp, None


def perdida_preferencia(lp, mascara=None, ref=None, beta=0.1, tipo='sigmoide', suavizado=0.0, margen=0.0,
                        por_longitud=False):
    """The preference loss of P pairs of texts, averaged over the pairs, and the texts' rewards beta R (2P, no gradient):

        R_i = sum over the masked tokens of lp - ref  (por_longitud: over their count),  h = beta (R_chosen - R_rejected) - margen
        'sigmoide'  -(1 - suavizado) log sigma(h) - suavizado log sigma(-h)
        'ipo'       ((h - 1/2) / beta)^2          'bisagra'  max(0, 1 - h)

    lp (2P, L): the tokens' log-probabilities under the model, rows 0 .. P - 1 the chosen texts and P .. 2P - 1 the
    rejected ones (log_probabilidades); mascara (2P, L): nonzero on the answers' tokens (None: all); ref: the reference
    model's, (2P, L) a token or (2P,) summed a text already, or None for none. The gradient goes to lp; mascara and ref
    are constants. What the mask hides is not used, NaN and infinities included; a text without tokens has R = 0 (less
    its ref sum). Sums are held in double."""
    quien = 'perdida_preferencia'
    dev = _dev(lp)
    if lp.dim() != 2 or lp.shape[0] < 2 or lp.shape[0] % 2 or not lp.is_floating_point():
        raise ValueError(f'{quien}: lp {tuple(lp.shape)} of {lp.dtype}: (2P, L) log-probabilities, P >= 1, are needed')
    m = _mascara(quien, mascara, lp.shape, dev)
    if ref is not None:
        if tuple(ref.shape) not in (tuple(lp.shape), (lp.shape[0],)) or not ref.is_floating_point():
            raise ValueError(f'{quien}: ref {tuple(ref.shape)} of {ref.dtype} against lp {tuple(lp.shape)}')
        _mismo_gpu(quien, dev, ref=ref)
        ref = _fijo(ref)
    if tipo not in FORMAS:
        raise ValueError(f'{quien}: tipo={tipo!r}: one of {FORMAS}')
    beta = _numero(quien, 'beta', beta, 0.0, abierto=True)
    suavizado = _numero(quien, 'suavizado', suavizado, 0.0, 1.0)
    if suavizado and tipo != 'sigmoide':
        raise ValueError(f"{quien}: suavizado belongs to tipo='sigmoide'")
    margen = _numero(quien, 'margen', margen, -math.inf)
    return Preferencia.apply(_f32(lp), (m, ref, tipo, beta, suavizado, margen, bool(por_longitud)))


# ---------------------------------------------------------------------------------------------------------------------
# the policy loss
# ---------------------------------------------------------------------------------------------------------------------

class Politica(torch.autograd.Function):
    """asrn_policy_fwd/bwd: (loss, statistics) of lp and the entropies H (B, L); the tokens' gradients before the
    reduction are kept from the forward, in fp32."""

    @staticmethod
    def forward(ctx, lp, H, fijos):
        A, vieja, ref, m, lo, hi, tope, beta, peso, por_texto = fijos     # constants: no autograd around them
        dev = lp.device
        B, L = lp.shape
        perdida = torch.empty((), dtype=torch.float32, device=dev)
        datos = torch.empty((4,), dtype=torch.float32, device=dev)
        # one buffer: the workspace, then what the backward needs: the texts' divisors and the tokens' gradients
        wsb = query('asrn_policy_workspace', B, L)
        fin = max(wsb, 0)
        ws = torch.empty((fin + 4 * B + (4 * B * L if ctx.needs_input_grad[0] else 0),), dtype=torch.uint8, device=dev)
        div = ws.data_ptr() + fin
        crudo = div + 4 * B if ctx.needs_input_grad[0] else None
        _en(dev, 'asrn_policy_fwd', ptr(lp), ptr(A), ptr(vieja), ptr(ref), ptr(H), ptr(m), _pasos(lp, A, vieja, ref, H, m),
                B, L, lo, hi, tope, beta, peso, int(por_texto), crudo, ptr(perdida), ptr(datos), div, ptr(ws), wsb)
        ctx.save_for_backward(ws, m)
        ctx.meta = (B, L, peso, fin)
        ctx.mark_non_differentiable(datos)
        ctx.set_materialize_grads(False)
        return perdida, datos

    @staticmethod
    @once_differentiable
    def backward(ctx, g, _):
        ws, m = ctx.saved_tensors
        B, L, peso, fin = ctx.meta
        if g is None:
            return None, None, None
        dev = ws.device
        dlp = torch.empty((B, L), dtype=torch.float32, device=dev) if ctx.needs_input_grad[0] else None
        dH = torch.empty((B, L), dtype=torch.float32, device=dev) if ctx.needs_input_grad[1] else None
        gc = _denso(g)
        div = ws.data_ptr() + fin
        _en(dev, 'asrn_policy_bwd', div + 4 * B, div, ptr(gc), ptr(m), None if m is None else _pasos(m), B, L, peso, ptr(dlp),
            ptr(dH))
        return dlp, dH, None


def perdida_politica(lp, ventaja, lp_vieja=None, mascara=None, recorte=0.2, tope=None, lp_ref=None, beta=0.0,
                     entropia=None, peso_entropia=0.0, reduccion='fichas'):
    """The clipped policy loss of sampled answers and four statistics (no gradient). Per token, with
    r = exp(lp - lp_vieja) and q = lp_ref - lp:

        -min(r A, clip(r, 1 - recorte, 1 + recorte) A)   (tope c, A < 0 and r > c: -c A instead)
        + beta (exp(q) - 1 - q) - peso_entropia H

    lp (B, L): the sampled tokens' log-probabilities under the model (log_probabilidades); ventaja: A, (B, L) a token or
    (B,) a text; lp_vieja (B, L): those under the model that sampled them (None: lp itself, so r = 1); recorte: one number
    or (below, above); lp_ref (B, L): the reference model's, for the KL term; entropia (B, L): H, the rows' entropies.
    mascara (B, L): nonzero on the answers' tokens (None: all); what it hides is not used, NaN and infinities included.
    reduccion: 'fichas' averages over the masked tokens, 'textos' over the texts' own means (texts without tokens left
    out); NaN when no token is left. The gradient goes to lp and entropia; the rest are constants. Statistics (means over
    the masked tokens): [share of clipped tokens, r - 1 - log r, exp(q) - 1 - q, H]. Everything per token and every sum
    is formed in double."""
    quien = 'perdida_politica'
    dev = _dev(lp)
    if lp.dim() != 2 or lp.shape[0] < 1 or not lp.is_floating_point():
        raise ValueError(f'{quien}: lp {tuple(lp.shape)} of {lp.dtype}: (B, L) log-probabilities, B >= 1, are needed')
    if tuple(ventaja.shape) == (lp.shape[0],):
        ventaja = ventaja[:, None].expand(lp.shape)
    for n, t in (('ventaja', ventaja), ('lp_vieja', lp_vieja), ('lp_ref', lp_ref), ('entropia', entropia)):
        if t is not None and (tuple(t.shape) != tuple(lp.shape) or not t.is_floating_point()):
            raise ValueError(f'{quien}: {n} {tuple(t.shape)} of {t.dtype} against lp {tuple(lp.shape)}')
    _mismo_gpu(quien, dev, ventaja=ventaja, lp_vieja=lp_vieja, lp_ref=lp_ref, entropia=entropia)
    m = _mascara(quien, mascara, lp.shape, dev)
    lo, hi = recorte if isinstance(recorte, (tuple, list)) and len(recorte) == 2 else (recorte, recorte)
    lo, hi = _numero(quien, 'recorte', lo, 0.0, 1.0), _numero(quien, 'recorte', hi, 0.0)
    tope = 0.0 if tope is None else _numero(quien, 'tope', tope, 1.0, abierto=True)
    beta = _numero(quien, 'beta', beta, 0.0)
    peso = _numero(quien, 'peso_entropia', peso_entropia, -math.inf)
    if beta and lp_ref is None:
        raise ValueError(f'{quien}: beta={beta} needs lp_ref')
    if peso and entropia is None:
        raise ValueError(f'{quien}: peso_entropia={peso} needs entropia')
    if reduccion not in REDUCCIONES:
        raise ValueError(f'{quien}: reduccion={reduccion!r}: one of {REDUCCIONES}')
    return Politica.apply(_f32(lp), _f32(entropia), (_fijo(ventaja), _fijo(lp_vieja), _fijo(lp_ref), m, lo, hi, tope, beta,
                                                     peso, reduccion == 'textos'))


token_log_probs, preference_loss, policy_loss = log_probabilidades, perdida_preferencia, perdida_politica
