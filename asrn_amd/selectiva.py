"""A local block's operators with a state a channel, on the library's kernels (include/asrn_hip.h): the causal convolution
of each channel with its activation and the selective state space scan, for texts (with their gradients) and for single
tokens.

    c = conv_canal(z, peso, sesgo, 'silu')                                  # (B, L, d)
    y = escaneo_selectivo(c, delta, A, Bm, C, D=D, puerta=g, sesgo_delta=b) # (B, L, d)
    c, ventana = paso_conv_canal(z_t, ventana, peso, sesgo, 'silu')         # (B, d): the next token
    y, estado = paso_selectivo(c, delta_t, A, Bm_t, C_t, estado, D=D, puerta=g_t, sesgo_delta=b)

They stand beside escaneo (the affine scan with its coefficients given); ModeloASRN's 'selectiva' blocks are made of them.
GPU only. Nothing waits on the host, so a step over them can be captured in a HIP graph.
"""
import torch

from ._lib import ASRNHipError, nodos
from .ops import _dev

TIPOS = (torch.float32, torch.bfloat16, torch.float16)       # what the kernels read and write
ACTIVACIONES = (None, 'gelu', 'silu')
K_MAX = 16                        # taps of a channel's convolution
ESTADOS_MAX = 32                  # states a channel


def disponible(tipo, k):
    """Whether the convolution of each channel runs here on values of dtype `tipo` with k taps: a library that was built without
    the nodes has none of this module's operators."""
    if tipo not in TIPOS or not 1 <= k <= K_MAX:
        return False
    try:
        nodos()
    except ASRNHipError:
        return False
    return True


def _activacion(quien, a):
    if a not in ACTIVACIONES:
        raise ValueError(f'{quien}: activacion={a!r}: one of {ACTIVACIONES}')
    return ACTIVACIONES.index(a)


def _valores(quien, nombre, t, forma, como):
    """t as a tensor of `forma` in como's dtype on como's device."""
    if tuple(t.shape) != tuple(forma) or t.dtype != como.dtype:
        raise ValueError(f'{quien}: {nombre} {tuple(t.shape)} of {t.dtype}: {tuple(forma)} of {como.dtype} is needed')
    _mismo(quien, nombre, t, como)


def _parametro(quien, nombre, t, forma, como):
    """t, if given, as a floating parameter of `forma` on como's device (the kernels take parameters in fp32)."""
    if t is None:
        return
    if tuple(t.shape) != tuple(forma) or t.dtype not in TIPOS:
        raise ValueError(f'{quien}: {nombre} {tuple(t.shape)} of {t.dtype}: {tuple(forma)} is needed, fp32 at most')
    _mismo(quien, nombre, t, como)


def _mismo(quien, nombre, t, como):
    if t.device != como.device:
        raise ValueError(f'{quien}: {nombre} is on {t.device}, the rest on {como.device}')


def _tipo(quien, nombre, t, ejes):
    if t.dim() != ejes or t.dtype not in TIPOS or t.shape[-1] < 1:
        raise ValueError(f'{quien}: {nombre} {tuple(t.shape)} of {t.dtype}: {ejes} axes of fp32, bf16 or fp16 are needed')


def _conv(quien, z, peso, sesgo, ejes):
    """The checks of a convolution's arguments; its taps."""
    _tipo(quien, 'z', z, ejes)
    d = z.shape[-1]
    if peso.dim() not in (2, 3) or peso.shape[0] != d or peso.numel() != d * peso.shape[-1] or not 1 <= peso.shape[-1] <= K_MAX:
        raise ValueError(f'{quien}: peso {tuple(peso.shape)} for {d} channels: (d, k) or (d, 1, k), k from 1 to {K_MAX}')
    k = peso.shape[-1]
    _parametro(quien, 'peso', peso, peso.shape, z)
    _parametro(quien, 'sesgo', sesgo, (d,), z)
    return k


def conv_canal(z, peso, sesgo=None, activacion=None, registrable=False):
    """act(sesgo + sum_j peso[:, j] z[:, t - (k - 1) + j]) of each channel, zeros before a text's start: z (B, L, d) fp32,
    bf16 or fp16, read through its strides; peso (d, k) or nn.Conv1d's depthwise (d, 1, k), k <= 16; activacion None, 'gelu'
    (erf's) or 'silu'. The result is dense in z's dtype; products, sums and the activation are in fp32, rounded once.
    The backward forms the activation's input again: nothing but z is kept. A backward that is itself recorded
    (create_graph=True) is refused, or with registrable=True runs in torch's operators, which have a second derivative."""
    quien = 'conv_canal'
    _conv(quien, z, peso, sesgo, 3)
    a = _activacion(quien, activacion)
    _dev(z)
    return nodos().conv_canal(z, peso, sesgo, a, bool(registrable))


def paso_conv_canal(z, ventana, peso, sesgo=None, activacion=None, en_sitio=True):
    """conv_canal's next token: z (B, d) and ventana (B, d, k - 1), the values before it, oldest first, dense in z's dtype ->
    (result (B, d), the window after it). en_sitio: the window is updated in place and returned; else it is left as it is.
    No gradient: under grad mode, tensors that ask for one are refused."""
    quien = 'paso_conv_canal'
    k = _conv(quien, z, peso, sesgo, 2)
    _valores(quien, 'ventana', ventana, (*z.shape, k - 1), z)
    if not ventana.is_contiguous():
        raise ValueError(f'{quien}: ventana must be contiguous (strides {ventana.stride()})')
    a = _activacion(quien, activacion)
    _dev(z)
    return nodos().paso_conv_canal(z, ventana, peso, sesgo, a, bool(en_sitio))


def _escaneo(quien, u, delta, A, Bm, C, D, puerta, sesgo_delta, ejes):
    """The checks that the scan and its step share."""
    _tipo(quien, 'u', u, ejes)
    d = u.shape[-1]
    if A.dim() != 2 or A.shape[0] != d or not 1 <= A.shape[1] <= ESTADOS_MAX:
        raise ValueError(f'{quien}: A {tuple(A.shape)} for {d} channels: (d, N), N from 1 to {ESTADOS_MAX}')
    _valores(quien, 'delta', delta, u.shape, u)
    for nombre, t in (('Bm', Bm), ('C', C)):
        _valores(quien, nombre, t, (*u.shape[:-1], A.shape[1]), u)
    if puerta is not None:
        _valores(quien, 'puerta', puerta, u.shape, u)
    _parametro(quien, 'A', A, A.shape, u)
    _parametro(quien, 'D', D, (d,), u)
    _parametro(quien, 'sesgo_delta', sesgo_delta, (d,), u)
    return u.shape[0], d, A.shape[1]


def escaneo_selectivo(u, delta, A, Bm, C, D=None, puerta=None, sesgo_delta=None, estado=None, devolver_estado=False,
                      softplus=True):
    """The selective state space scan over a text: with dt = softplus(delta + sesgo_delta) (softplus=False: delta + sesgo_delta)

        h_t = exp(dt_t A) h_{t-1} + dt_t u_t Bm_t        y_t = (sum_n C_t h_t + D u_t) silu(puerta_t)

    u, delta, puerta (B, L, d) and Bm, C (B, L, N) in one dtype (fp32, bf16, fp16), read through their strides; A (d, N),
    N <= 32, at most 0 for a state that does not grow; D and sesgo_delta (d,). The state h (B, d, N) starts from `estado`
    (None: zeros) and is held in fp32; devolver_estado: (y, the last state), for another piece of the text or for
    paso_selectivo. D, puerta and sesgo_delta may be None. y is dense in u's dtype, rounded once from fp32.
    Gradients go to every tensor argument and come from y and the last state; the parameters' are summed in fp32. A training
    call keeps its inputs and the state of every eighth token."""
    quien = 'escaneo_selectivo'
    B, d, N = _escaneo(quien, u, delta, A, Bm, C, D, puerta, sesgo_delta, 3)
    _parametro(quien, 'estado', estado, (B, d, N), u)
    _dev(u)
    y, fin = nodos().selectivo(u, delta, A, Bm, C, D, puerta, sesgo_delta, estado, bool(softplus), bool(devolver_estado))
    return (y, fin) if devolver_estado else y


def paso_selectivo(u, delta, A, Bm, C, estado, D=None, puerta=None, sesgo_delta=None, softplus=True, en_sitio=True):
    """escaneo_selectivo's next token: u, delta, puerta (B, d), Bm, C (B, N) and the state (B, d, N), fp32 and contiguous ->
    (y (B, d), the state after it). en_sitio: the state is updated in place and returned; else it is left as it is. No
    gradient: under grad mode, tensors that ask for one are refused."""
    quien = 'paso_selectivo'
    B, d, N = _escaneo(quien, u, delta, A, Bm, C, D, puerta, sesgo_delta, 2)
    if tuple(estado.shape) != (B, d, N) or estado.dtype != torch.float32 or not estado.is_contiguous():
        raise ValueError(f'{quien}: estado {tuple(estado.shape)} of {estado.dtype}: {(B, d, N)} fp32, contiguous, is needed')
    _mismo(quien, 'estado', estado, u)
    _dev(u)
    return nodos().paso_selectivo(u, delta, A, Bm, C, estado, D, puerta, sesgo_delta, bool(softplus), bool(en_sitio))


channel_conv, channel_conv_step = conv_canal, paso_conv_canal
selective_scan, selective_step = escaneo_selectivo, paso_selectivo
