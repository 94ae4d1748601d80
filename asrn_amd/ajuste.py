"""Losses for fine-tuning a model on answers: the log-probabilities of given tokens, the preference loss of pairs of
texts and the clipped policy loss, each with its gradient, on the library's kernels (include/asrn_hip.h).

    lp = modelo.log_probabilidades(x, y)                      # (B, L): log p of y under the logits of x
    perdida, recompensas = perdida_preferencia(lp, y != -100, ref)         # rows: the chosen texts, then the rejected
    perdida, datos = perdida_politica(lp, ventaja, lp_vieja, y != -100)    # sampled answers and their advantages

The reference package has no counterpart; the functions stand beside the model's loss (ops.cross_entropy). GPU only.
Nothing waits on the host, so a step over them can be captured in a HIP graph.
"""
import math

import torch

from ._lib import nodos
from .ops import _dev

TIPOS = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}     # the kernels' logits
FORMAS = ('sigmoide', 'ipo', 'bisagra')
REDUCCIONES = ('fichas', 'textos')


def _igual(quien, lp, **tensores):
    """Floating tensors of lp's shape on its device, or None."""
    for n, t in tensores.items():
        if t is not None:
            if t.shape != lp.shape or not t.is_floating_point():
                raise ValueError(f'{quien}: {n} {tuple(t.shape)} of {t.dtype} against lp {tuple(lp.shape)}')
            if t.device != lp.device:
                raise ValueError(f'{quien}: {n} is on {t.device}, the rest on {lp.device}')


def _mascara(quien, m, forma, dev):
    """A (B, L) mask as bytes (nonzero keeps the token), or None."""
    if m is None:
        return None
    if m.shape != forma:
        raise ValueError(f'{quien}: mascara {tuple(m.shape)} against {tuple(forma)} tokens')
    if m.device != dev:
        raise ValueError(f'{quien}: mascara is on {m.device}, the rest on {dev}')
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

def log_probabilidades(logits, y, ignorar=-100, temperatura=1.0, entropia=False):
    """log softmax(logits / temperatura) at the tokens y, in fp32: logits (..., V) fp32, bf16 or fp16, read as they are
    through their strides (no fp32 copy), y (...) integers. 0 where y == ignorar, and no gradient there; NaN for a token
    outside [0, V). entropia=True: (log-probabilities, the rows' entropy), both with gradients; an ignored row's entropy
    is 0. The gradient is in the logits' dtype. Sums are held in fp32, as cross_entropy's."""
    quien = 'log_probabilidades'
    dev = _dev(logits)
    if logits.dim() < 1 or logits.shape[:-1] != y.shape:
        raise ValueError(f'{quien}: logits {tuple(logits.shape)} against tokens {tuple(y.shape)}')
    if logits.dtype not in TIPOS:
        raise ValueError(f'{quien}: logits of {logits.dtype} (fp32, bf16 or fp16 are taken)')
    if logits.shape[-1] < 1 or y.is_floating_point() or y.is_complex() or y.dtype == torch.bool:
        raise ValueError(f'{quien}: a vocabulary of {logits.shape[-1]} tokens and token ids of {y.dtype}')
    if y.device != dev:
        raise ValueError(f'{quien}: y is on {y.device}, the logits on {dev}')
    T = _numero(quien, 'temperatura', temperatura, 1e-6, 1e6)
    x, t = logits, y.to(torch.int64).contiguous()
    if x.stride(-1) != 1 and x.shape[-1] > 1:
        x = x.contiguous()
    if x.dim() > 3:                                  # more leading axes are flattened; a (B, L, V) slice needs no copy
        n = math.prod(x.shape[:-2])
        x, t = x.reshape(n, *x.shape[-2:]), t.view(n, t.shape[-1])
    lp, H = nodos().logp(x, t, TIPOS[x.dtype], int(ignorar), 1.0 / T, bool(entropia))
    if logits.dim() > 3:
        lp, H = lp.view(y.shape), H if H is None else H.view(y.shape)
    return (lp, H) if entropia else lp


# ---------------------------------------------------------------------------------------------------------------------
# the preference loss
# ---------------------------------------------------------------------------------------------------------------------

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
    its ref sum). Sums are held in double; lp and a ref a token are taken in fp32 (fp64 ones are rounded to it), the sums
    (2P,) in fp32 or fp64 as they come."""
    quien = 'perdida_preferencia'
    dev = _dev(lp)
    if lp.dim() != 2 or lp.shape[0] < 2 or lp.shape[0] % 2 or not lp.is_floating_point():
        raise ValueError(f'{quien}: lp {tuple(lp.shape)} of {lp.dtype}: (2P, L) log-probabilities, P >= 1, are needed')
    m = _mascara(quien, mascara, lp.shape, dev)
    if ref is not None:
        if ref.dim() != 1:
            _igual(quien, lp, ref=ref)
        elif ref.shape[0] != lp.shape[0] or not ref.is_floating_point() or ref.device != dev:
            raise ValueError(f'{quien}: ref {tuple(ref.shape)} of {ref.dtype} on {ref.device} against lp {tuple(lp.shape)} on {dev}')
        ref = ref.detach() if ref.dim() == 1 and ref.dtype == torch.float64 else _fijo(ref)
    if tipo not in FORMAS:
        raise ValueError(f'{quien}: tipo={tipo!r}: one of {FORMAS}')
    beta = _numero(quien, 'beta', beta, 0.0, abierto=True)
    suavizado = _numero(quien, 'suavizado', suavizado, 0.0, 1.0)
    if suavizado and tipo != 'sigmoide':
        raise ValueError(f"{quien}: suavizado belongs to tipo='sigmoide'")
    margen = _numero(quien, 'margen', margen, -math.inf)
    return nodos().preferencia(_f32(lp), m, ref, FORMAS.index(tipo), beta, suavizado, margen, bool(por_longitud))


# ---------------------------------------------------------------------------------------------------------------------
# the policy loss
# ---------------------------------------------------------------------------------------------------------------------

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
    the masked tokens): [share of clipped tokens, r - 1 - log r, exp(q) - 1 - q, H]. Inputs are taken in fp32 (fp64
    ones are rounded to it); their differences, products and sums are formed in double, exponentials to fp32's accuracy."""
    quien = 'perdida_politica'
    dev = _dev(lp)
    if lp.dim() != 2 or lp.shape[0] < 1 or not lp.is_floating_point():
        raise ValueError(f'{quien}: lp {tuple(lp.shape)} of {lp.dtype}: (B, L) log-probabilities, B >= 1, are needed')
    if ventaja.dim() == 1 and ventaja.shape[0] == lp.shape[0]:
        ventaja = ventaja[:, None].expand(lp.shape)
    _igual(quien, lp, ventaja=ventaja, lp_vieja=lp_vieja, lp_ref=lp_ref, entropia=entropia)
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
    return nodos().politica(_f32(lp), _f32(entropia), _fijo(ventaja), _fijo(lp_vieja), _fijo(lp_ref), m, lo, hi, tope, beta, peso,
                            reduccion == 'textos')


token_log_probs, preference_loss, policy_loss = log_probabilidades, perdida_preferencia, perdida_politica
