"""Dense projections on MI355X: the library's own products (asrn_gemm) where they are the faster ones, and a weight
gradient that fits a long token axis.

For y = x W^T + b over N tokens, the weight gradient dW = dY^T X reduces over all N (32768 at the layer benchmark's
shape) into a small (out, in) matrix. As one GEMM it has only (out / tile) x (in / tile) output tiles to spread over
256 CUs. asrn_gemm cuts the token axis into slabs whose partial products are added in order, and sums the bias
gradient (dY's columns) from the values it loads anyway. fp32 products run there on the bf16 matrix cores, each operand
split into three bf16 parts: fp32's error (for operands from 2^-110 on) at more than fp32's matrix rate. Where hipBLASLt
is faster (below), it is called as before: the weight gradient as one batched product over slabs of tokens.
Under autocast the operands are cast as autocast casts F.linear's, and the products run in that dtype.

On the GPU, the sums (the slab partials, and the bias gradients' column sums) run in the library's asrn_column_sums
(fp32 accumulation in a fixed order, no memset-cleared semaphores, safe to capture in a HIP graph). fp64 operands,
and CPU tensors (the math checked on the CPU), use torch's sums.
"""
import math

import torch
import torch.nn.functional as F

from . import _lib

MIN_SLAB = 1024            # tokens per slab: below this the batched GEMM's own overhead dominates
MAX_SLAB_WEIGHT = 1 << 20  # weights with this many elements or more keep one GEMM: enough output tiles already, and
                           # S partial copies of them would cost more traffic than they save


def slabs_for(n, weight_elems=0):
    """Slab count for a token axis of n: 16 (or fewer) slabs of at least MIN_SLAB tokens that divide n exactly; 1 for
    weights of MAX_SLAB_WEIGHT elements or more."""
    if weight_elems >= MAX_SLAB_WEIGHT:
        return 1
    for s in (16, 8, 4, 2):
        if n % s == 0 and n // s >= MIN_SLAB:
            return s
    return 1


def _rows(t):
    """(N, k) view of a (..., k) tensor whose last axis is contiguous; copies only when the leading axes do not
    flatten to one stride."""
    k = t.shape[-1]
    n = math.prod(t.shape[:-1])                      # stated: -1 has no value for a zero-wide t
    if t.stride(-1) != 1:
        t = t.contiguous()
    try:
        return t.view(n, k)
    except RuntimeError:
        return t.reshape(n, k)


def _slab(t, s):
    """(s, N / s, k) view of an (N, k) matrix with unit last stride (splitting the row axis never needs a copy)."""
    n, k = t.shape
    return t.view(s, n // s, k)


# fp32 products of fewer multiply-adds than this stay on hipBLASLt, measured (us, it / asrn_gemm): 2048 x 64 x 256
# 5.9 / 9.1, 4611 x 384 x 192 10.7 / 11.3, 5005 x 256 x 512 19.1 / 17.8, 4611 x 384 x 384 17.6 / 16.0, 32768 x 256 x 256
# 39.1 / 33.1, 12000 x 768 x 3072 492 / 303: below, a launch's few steps wait for their loads
MIN_PRODUCTO = 400_000_000
# fp32 weight gradients over fewer tokens stay there too: 64 x 64 over 200 tokens 7.7 / 9.9, 64 x 256 over 2048 19.0 / 9.6
MIN_FICHAS = 512
# bf16 weight gradients on asrn_gemm: weights too large for slab copies (768 x 3072 over 16384 tokens 154 / 120,
# 1536 x 768 115 / 72) and small ones (112 x 128 12.4 / 11.4, 64 x 1024 over 65536 34 / 32, 512 x 256 over 5008
# 18.7 / 15.1); between them hipBLASLt's batched slabs win (768 x 768 35 / 51, 512 x 512 over 65536 55 / 69)
MAX_PESO_16 = 1 << 17
# Of the large ones, only over enough tokens for their partial products: tokens times this at least the weight's elements,
# with the bias gradient (13 us or more as a launch of its own) and without. 768 x 3072 with it over 2048 tokens 37 / 48,
# over 5001 68 / 63, 512 x 2048 over 3000 41 / 33, 8000 x 512 over 8192 105 / 111; without it 768 x 3072 over 8192 77 / 81,
# 1536 x 768 over 4097 35 / 39, over 8192 60 / 52, 32768 x 768 over 16384 763 / 1109
FICHAS_PESO = {True: 400, False: 200}


def _apto(t):
    """Whether asrn_gemm can read the 2-D matrix t in place."""
    return (t.dim() == 2 and t.stride(1) == 1 and t.stride(0) % 4 == 0 and t.stride(0) >= t.shape[1]
            and t.data_ptr() % (4 * t.element_size()) == 0)


def gemm(a, ta, b, tb, sesgo=None, columnas=False):
    """op(a) op(b) (+ sesgo) in fp32 on asrn_gemm, op the transpose where ta, tb. columnas (ta): returns (product, the
    sums of a's columns). Shapes that do not chain are refused here: the kernels see leading dimensions only and would
    read whatever lies there."""
    M, K = (a.shape[1], a.shape[0]) if ta else a.shape
    Kb, N = (b.shape[1], b.shape[0]) if tb else b.shape
    if K != Kb or (sesgo is not None and tuple(sesgo.shape) != (N,)):
        raise ValueError(f'gemm: shapes {tuple(a.shape)}{" transposed" if ta else ""}, {tuple(b.shape)}'
                         f'{" transposed" if tb else ""} and bias {None if sesgo is None else tuple(sesgo.shape)} do not chain')
    bf = int(a.dtype == torch.bfloat16)
    out = torch.empty((M, N), dtype=torch.float32, device=a.device)
    cols = torch.empty((M,), dtype=torch.float32, device=a.device) if columnas else None
    wsb = _lib.query('asrn_gemm_workspace', M, N, K, bf, int(columnas), 0, 0)
    ws = torch.empty((wsb,), dtype=torch.uint8, device=a.device) if wsb > 0 else None
    _lib.call('asrn_gemm', _lib.ptr(a), a.stride(0), int(ta), _lib.ptr(b), b.stride(0), int(tb), bf, _lib.ptr(out),
              out.stride(0), M, N, K, _lib.ptr(sesgo), 0, _lib.ptr(cols), 0, 0, _lib.ptr(ws), wsb,
              _lib.stream_of(a.device))
    return (out, cols) if columnas else out


def gemm_ok(a, b, tb, sesgo=None):
    """Whether a @ op(b) (+ sesgo) runs on asrn_gemm: fp32 on the GPU, aligned, MIN_PRODUCTO multiply-adds or more, and
    shapes that chain with one bias value per column (F.linear broadcasts a bias or refuses the rest)."""
    if b.dim() != 2 or a.shape[1] != b.shape[1 if tb else 0]:
        return False
    (M, K), N = a.shape, b.shape[0 if tb else 1]
    return (a.is_cuda and a.dtype == b.dtype == torch.float32 and b.device == a.device and M * N * K >= MIN_PRODUCTO
            and max(M, N, K) < 1 << 30 and N >= 64 and N % 4 == 0 and K % 4 == 0 and _apto(a) and _apto(b)
            and (sesgo is None or (sesgo.dtype == torch.float32 and sesgo.device == a.device and tuple(sesgo.shape) == (N,)
                                   and sesgo.is_contiguous() and sesgo.data_ptr() % 16 == 0)))


def _gradiente_ok(g2, x2, sesgo):
    """Whether dW = g2^T x2 runs on asrn_gemm (see the constants above)."""
    if not (g2.is_cuda and g2.dtype == x2.dtype and g2.dtype in (torch.float32, torch.bfloat16) and _apto(g2)
            and _apto(x2) and g2.shape[1] % 4 == 0 and x2.shape[1] % 4 == 0 and 1 <= g2.shape[0] < 1 << 30):
        return False
    n, peso = g2.shape[0], g2.shape[1] * x2.shape[1]
    if peso == 0:                      # no product to form, but the bias gradient still is (asrn_gemm returns at once)
        return False
    if g2.dtype == torch.float32:
        return sesgo or n >= MIN_FICHAS
    if peso >= MAX_SLAB_WEIGHT:
        return n * FICHAS_PESO[sesgo] >= peso
    return peso <= MAX_PESO_16 or slabs_for(n, peso) == 1


def _acc_dtype(t):
    return torch.float64 if t.dtype == torch.float64 else torch.float32


def _hip_sums(x, rows, cols, ld):
    """fp32 column sums of the (rows, cols) matrix at x (row stride ld) through asrn_column_sums."""
    out = torch.empty((cols,), dtype=torch.float32, device=x.device)
    wsb = _lib.query('asrn_column_sums_workspace', rows, cols)
    ws = torch.empty((wsb,), dtype=torch.uint8, device=x.device) if wsb > 0 else None
    _lib.call('asrn_column_sums', _lib.ptr(x), int(x.dtype == torch.bfloat16), rows, cols, ld, _lib.ptr(out),
              _lib.ptr(ws), wsb, _lib.stream_of(x.device))
    return out


def _on_hip(t):
    return t.is_cuda and t.dtype in (torch.float32, torch.bfloat16)


def sum_rows(t):
    """t (S, ...) summed over its first axis in fp32 (fp64 for fp64), in order."""
    if _on_hip(t):
        t = t.contiguous()
        n = t[0].numel() if t.shape[0] else 0
        return _hip_sums(t, t.shape[0], n, max(n, 1)).view(t.shape[1:])
    return t.sum(0, dtype=_acc_dtype(t))


def weight_grad(g2, x2, sesgo=False):
    """dW = g2^T x2, summed in fp32 (fp64 for fp64 operands): g2 (N, out), x2 (N, in), both with unit last stride.
    sesgo: (dW, the bias gradient column_sums(g2))."""
    if _gradiente_ok(g2, x2, sesgo):
        return gemm(g2, True, x2, False, columnas=sesgo)
    if sesgo:
        return weight_grad(g2, x2), column_sums(g2)
    s = slabs_for(g2.shape[0], g2.shape[1] * x2.shape[1])
    if s == 1:
        return g2.t().mm(x2).to(_acc_dtype(g2))
    # left operand: the transposed slab of g2; right operand: x2's slab as stored (never a transposed view)
    return sum_rows(torch.bmm(_slab(g2, s).transpose(1, 2), _slab(x2, s)))


def column_sums(g2):
    """Sum over the rows of g2 (N, k) with unit last stride, in fp32 (fp64 for fp64)."""
    if _on_hip(g2):
        return _hip_sums(g2, g2.shape[0], g2.shape[1], max(g2.stride(0), g2.shape[1], 1))
    return g2.sum(0, dtype=_acc_dtype(g2))


def _producto(xc, wc, bc, propio):
    """F.linear(xc, wc, bc), on asrn_gemm where that is faster."""
    # rows flattened (which may copy) only for products that asrn_gemm takes by their size
    x2 = None
    if propio and xc.is_cuda and xc.dtype == torch.float32 and xc.numel() * wc.shape[0] >= MIN_PRODUCTO:
        x2 = _rows(xc)
    if x2 is not None and gemm_ok(x2, wc, True, bc):
        return gemm(x2, False, wc, True, sesgo=bc).view(*xc.shape[:-1], wc.shape[0])
    with torch.autocast(device_type=xc.device.type, enabled=False):
        return F.linear(xc, wc, bc)


def _gradientes(g, wc, leer, tipos, quiere):
    """The gradients of a product's x, w and b (None where `quiere` is false) from its output's; leer() gives x's rows."""
    xdt, wdt, bdt = tipos
    gx = gw = gb = None
    with torch.autocast(device_type=g.device.type, enabled=False):
        g = g.to(wc.dtype)
        g2 = _rows(g)
        if quiere[0]:
            if gemm_ok(g2, wc, False):
                gx = gemm(g2, False, wc, False).view(*g.shape[:-1], wc.shape[1]).to(xdt)
            else:
                gx = g.matmul(wc).to(xdt)
        con_sesgo = bdt is not None and quiere[2]
        if quiere[1]:
            gw = weight_grad(g2, leer(), con_sesgo)
            if con_sesgo:
                gw, gb = gw[0], gw[1].to(bdt)
            gw = gw.to(wdt)
        elif con_sesgo:
            gb = column_sums(g2).to(bdt)
    return gx, gw, gb


class _Lineal(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, w, b, dt, propio):
        xc, wc = x.to(dt), w.to(dt)
        y = _producto(xc, wc, b.to(dt) if b is not None else None, propio)
        ctx.save_for_backward(xc, wc)
        ctx.meta = (x.dtype, w.dtype, None if b is None else b.dtype)
        return y

    @staticmethod
    def backward(ctx, g):
        xc, wc = ctx.saved_tensors
        return (*_gradientes(g, wc, lambda: _rows(xc), ctx.meta, ctx.needs_input_grad), None, None)


class _Lineal8(torch.autograd.Function):
    """_Lineal whose weight gradient reads x back from the 8 bits that the op before it keeps (ops.Guardado8)."""

    @staticmethod
    def forward(ctx, x, w, b, dt, leer, *guardados):
        wc = w.to(dt)
        y = _producto(x.to(dt), wc, b.to(dt) if b is not None else None, True)
        ctx.save_for_backward(wc, *guardados)
        ctx.meta = ((x.dtype, w.dtype, None if b is None else b.dtype), leer, dt, len(guardados))
        return y

    @staticmethod
    def backward(ctx, g):
        if torch.is_grad_enabled():
            raise RuntimeError('lineal8: its gradient cannot be recorded (create_graph=True)')
        wc, *guardados = ctx.saved_tensors
        tipos, leer, dt, n = ctx.meta
        return (*_gradientes(g, wc, lambda: leer(guardados, dt), tipos, ctx.needs_input_grad), *(None,) * (2 + n))


def lineal(x, w, b=None, propio=True):
    """F.linear(x, w, b) with its products on asrn_gemm where that is faster; honours autocast like F.linear.
    propio=False: the forward stays F.linear's (outputs whose signs are hashed keep its rounding)."""
    dev = x.device.type
    dt = torch.get_autocast_dtype(dev) if torch.is_autocast_enabled(dev) else x.dtype
    return _Lineal.apply(x, w, b, dt, propio)


def lineal8(x, w, b, guardado):
    """lineal(x, w, b) that does not keep x: the weight gradient reads it back through `guardado`, what ops.norma8,
    ops.ventana8 or ops.gelu8 returned with x (None: lineal itself). The product and x's gradient are lineal's."""
    if guardado is None or not torch.is_grad_enabled():
        return lineal(x, w, b)
    N, d = guardado.forma
    if x.shape[-1] != d or x.numel() != N * d:
        raise ValueError(f'lineal8: x {tuple(x.shape)} and rows ({N}, {d}) kept of another tensor')
    if any(t.device != x.device for t in guardado.tensores):     # the weight gradient's kernels read both
        raise ValueError(f'lineal8: x is on {x.device}, the rows kept on {guardado.tensores[0].device}')
    dev = x.device.type
    dt = torch.get_autocast_dtype(dev) if torch.is_autocast_enabled(dev) else x.dtype
    return _Lineal8.apply(x, w, b, dt, guardado.leer, *guardado.tensores)


# ---------------------------------------------------------------------------------------------------------------------
# the product with its epilogue
# ---------------------------------------------------------------------------------------------------------------------

TIPOS = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVACIONES = {None: 0, 'gelu': 1, 'silu': 2}


def _plan_gradientes(x, w, M, N, K, dt):
    """How the backward of lineal_activa forms x's gradient (on asrn_gemm or not) and w's (on asrn_gemm, or in so many slabs),
    by the rules above for rows of a dense gradient (M, N), x (M, K) and w (N, K) in dt. w's from 16-bit rows of whole 16-byte
    units is asrn_weight_grad's, which is faster at most sizes (its figures: csrc/weight_grad.hip)."""
    f32 = dt == torch.float32
    # _apto for both operands: dense rows of a multiple of 4 (fresh tensors and contiguous inputs are aligned)
    cuatro = N % 4 == 0 and K % 4 == 0 and x.is_contiguous() and x.data_ptr() % 16 == 0
    gx = f32 and cuatro and M * N * K >= MIN_PRODUCTO and K >= 64 and w.is_contiguous() and w.data_ptr() % 16 == 0
    peso = N * K
    if not cuatro or dt == torch.float16 or M == 0:
        gw = False
    elif f32:
        gw = True
    elif peso >= MAX_SLAB_WEIGHT:
        gw = M * FICHAS_PESO[True] >= peso
    else:
        gw = peso <= MAX_PESO_16 or slabs_for(M, peso) == 1
    return int(gx), int(gw), slabs_for(M, peso)


def lineal_activa(x, w, b=None, activacion=None, residuo=None):
    """[residuo +] act(F.linear(x, w, b)) in one pass of the library's kernels: x (..., K), w (N, K), b (N,), residuo (..., N);
    activacion None, 'gelu' (erf's) or 'silu'. fp32, bf16 or fp16; under autocast the product's operands are cast as F.linear's
    are. The result is in the residual's dtype (fp32 or the product's), else in the product's; sums, the activation and the
    residual's addition are in fp32, rounded once. Gradients go to all four tensors; the activation's input is kept in the
    product's dtype. Second gradients and tangents of forward mode are refused, and rows of 2^21 values and more."""
    quien = 'lineal_activa'
    if activacion not in ACTIVACIONES:
        raise ValueError(f'{quien}: activacion={activacion!r}: one of {tuple(ACTIVACIONES)}')
    if x.dim() < 1 or w.dim() != 2 or x.shape[-1] != w.shape[1] or w.shape[1] < 1 or (b is not None and tuple(b.shape) != (w.shape[0],)):
        raise ValueError(f'{quien}: x {tuple(x.shape)}, w {tuple(w.shape)} and b {None if b is None else tuple(b.shape)} do not chain')
    forma = (*x.shape[:-1], w.shape[0])
    dev = x.device.type
    dt = torch.get_autocast_dtype(dev) if torch.is_autocast_enabled(dev) else x.dtype
    if residuo is not None and (tuple(residuo.shape) != forma or residuo.dtype not in (torch.float32, dt)):
        raise ValueError(f'{quien}: residuo {tuple(residuo.shape)} of {residuo.dtype}: {forma} of fp32 or {dt} is needed')
    for nombre, t in (('x', x), ('w', w), ('b', b)):
        if t is not None and (dt not in TIPOS or t.dtype not in TIPOS or (dt == x.dtype and t.dtype != dt and not
                                                                         torch.is_autocast_enabled(dev))):
            raise ValueError(f'{quien}: {nombre} of {t.dtype}: fp32, bf16 or fp16, one for all of them, is needed')
    for nombre, t in (('w', w), ('b', b), ('residuo', residuo)):
        if t is not None and t.device != x.device:
            raise ValueError(f'{quien}: {nombre} is on {t.device}, x on {x.device}')
    if not x.is_cuda:
        raise RuntimeError('asrn_amd runs on the GPU only: got a CPU tensor (move the model and inputs to cuda)')
    N, K = w.shape
    M = x.numel() // K
    plan = _plan_gradientes(x, w, M, N, K, dt) if torch.is_grad_enabled() else (0, 0, 1)
    return _lib.nodos().lineal_activa(x, w, b, residuo, ACTIVACIONES[activacion], dt, *plan)


linear_act = lineal_activa
