"""Matrix products grouped by expert, their gradients, and products of 8-bit integers.

A compiled GEMM KernelOp has fixed shapes and 16-bit or f32 operands.  These calls cover what it
cannot express: products whose row counts are known only on the device (the experts of a routed
layer) and s8 operands with a scale for each row and each channel.  Like the rest of the package
they launch on the caller's buffers and stream and allocate nothing (C ABI: include/emmy_b200.h,
csrc/emmy_products.cu).

* :func:`grouped_matmul`     ``out[r] = x[r] @ w[e].T`` for the rows ``r`` of expert ``e``
* :func:`grouped_matmul_dw`  ``dw[e] = dy_e.T @ x_e`` over expert ``e``'s rows
* :func:`int8_matmul`        ``out[r, n] = (xq[r] . wq[e, n]) * x_scale[r] * w_scale[e, n] + bias[e, n]``
* :func:`quantize_rows`      ``scale[r] = max|x[r]| / 127``, ``q[r] = round(x[r] / scale[r])``

The gradient of a grouped product by its rows is the same product with the weights' two axes
exchanged: ``grouped_matmul(dy, w.transpose(1, 2), offsets, dx)``.

``offsets`` holds ``experts + 1`` int32 values on the device: expert ``e`` owns rows
``offsets[e]`` to ``offsets[e + 1]``.  Rows outside every group are neither used nor written.

Arguments are device tensors (anything with ``data_ptr``, ``shape``, ``stride``, ``dtype`` and
``device``); rows may be padded (any row stride), the innermost axis is contiguous.  Outputs are
the caller's buffers and must not overlap an input.  Launches are asynchronous on ``stream`` (0 =
the legacy default stream) of the tensors' device, whichever device is current.

Every call has a ``bind_`` form that checks the arguments once and returns a callable for loops
that repeat it on the same buffers (as :meth:`.runtime.Module.bind` does for compiled kernels).
"""

from __future__ import annotations

import ctypes as C

from . import runtime

F32, BF16, F16 = 0, 1, 2
MAX_EXPERTS = 1024
MAX_K8 = 131071  # longest 8-bit contraction whose s32 sum cannot overflow

_TYPES = {"float32": F32, "bfloat16": BF16, "float16": F16}


class BoundProduct:
    """A launch with its arguments prepared once (the tensors stay alive and must keep their
    storage): each call is one C-ABI launch."""

    _fns: dict = {}

    def __init__(self, fn: str, args: tuple, keep: tuple):
        f = self._fns.get(fn)
        if f is None:
            f = self._fns[fn] = getattr(runtime.lib(), fn)
        self._fn = f
        self._args = args
        self._keep = keep

    def __call__(self) -> None:
        rc = self._fn(*self._args)
        if rc:
            runtime._check(rc)


_dtype_names: dict = {}


def _dtype(t) -> str:
    name = _dtype_names.get(t.dtype)
    if name is None:
        name = _dtype_names[t.dtype] = str(t.dtype).rpartition(".")[2]
    return name


def _matrix(name: str, t, shape: tuple, dtypes: tuple) -> int:
    """Check a tensor's shape (None: any extent), dtype and contiguous innermost axis; its row stride."""
    have = tuple(t.shape)
    if have != shape:
        fits = len(have) == len(shape)
        for h, w in zip(have, shape):
            if w is not None and h != w:
                fits = False
        if not fits:
            want = ", ".join("any" if w is None else str(w) for w in shape)
            raise ValueError(f"{name} has shape {have}, expected ({want})")
    if _dtype(t) not in dtypes:
        raise ValueError(f"{name} is {_dtype(t)}, expected {' or '.join(dtypes)}")
    stride, cols = t.stride(), have[-1]
    if cols > 1 and stride[-1] != 1:
        raise ValueError(f"{name}'s innermost axis must be contiguous, its stride is {stride[-1]}")
    if len(shape) == 1:
        return 1
    # a single row has no stride to speak of; report one that any check accepts
    return stride[-2] if have[-2] > 1 else max(stride[-2], cols)


def _rows_apart(name: str, t, row_stride: int) -> None:
    if t.shape[-2] > 1 and row_stride < t.shape[-1]:
        raise ValueError(f"{name}'s rows overlap: row stride {row_stride} for {t.shape[-1]} values")


def _device(**tensors) -> int:
    dev = None
    for name, t in tensors.items():
        if t is None:
            continue
        if dev is None:
            dev = t.device
            if dev.type != "cuda":
                raise ValueError(f"{name} is on {dev}, expected a CUDA device")
        elif t.device != dev:
            raise ValueError(f"{name} is on {t.device}, the other tensors on {dev}")
    runtime.init(dev.index)
    return dev.index


def _experts(n: int) -> None:
    if n > MAX_EXPERTS:
        raise ValueError(f"{n} experts, at most {MAX_EXPERTS} are supported")


def bind_grouped_matmul(x, w, offsets, out, stream: int = 0) -> BoundProduct:
    """:func:`grouped_matmul` with its arguments checked and prepared once."""
    if len(w.shape) != 3:
        raise ValueError(f"w has shape {tuple(w.shape)}, expected (experts, n, k)")
    e, n, k = w.shape
    _experts(e)
    ldx = _matrix("x", x, (None, k), ("bfloat16", "float16"))
    rows, dt = x.shape[0], _dtype(x)
    if _dtype(w) != dt:
        raise ValueError(f"w is {_dtype(w)}, x is {dt}")
    se, sn, sk = w.stride()
    if k <= 1:
        sk = 1
    elif n <= 1 and sk != 1:
        sn = 1
    if sn != 1 and sk != 1:
        raise ValueError(f"w's strides are {w.stride()}: one of its last two axes must be contiguous")
    _matrix("offsets", offsets, (e + 1,), ("int32",))
    ldo = _matrix("out", out, (rows, n), (dt, "float32"))
    _rows_apart("out", out, ldo)
    dev = _device(x=x, w=w, offsets=offsets, out=out)
    return BoundProduct("emmy_grouped_matmul",
                        (dev, _TYPES[dt], _TYPES[_dtype(out)], x.data_ptr(), ldx, w.data_ptr(), se, sn, sk,
                         offsets.data_ptr(), out.data_ptr(), ldo, rows, e, n, k, stream), (x, w, offsets, out))


def grouped_matmul(x, w, offsets, out, stream: int = 0) -> None:
    """``out[r] = x[r] @ w[e].T`` for the rows ``r`` of each expert ``e``.

    ``x`` [rows, k], ``w`` [experts, n, k] of the same type (bfloat16 or float16) with either of its
    last two axes contiguous, ``out`` [rows, n] of that type or float32.  Sums are held in f32 and
    rounded once.  Tensor cores truncate where they add: a float32 output is off by up to 1e-6 of its
    size, or 5e-6 and towards zero where all products have one sign, however many terms it has."""
    bind_grouped_matmul(x, w, offsets, out, stream)()


def bind_grouped_matmul_dw(dy, x, offsets, dw, stream: int = 0) -> BoundProduct:
    """:func:`grouped_matmul_dw` with its arguments checked and prepared once."""
    if len(dw.shape) != 3:
        raise ValueError(f"dw has shape {tuple(dw.shape)}, expected (experts, n, k)")
    e, n, k = dw.shape
    _experts(e)
    ldy = _matrix("dy", dy, (None, n), ("bfloat16", "float16"))
    rows, dt = dy.shape[0], _dtype(dy)
    ldx = _matrix("x", x, (rows, k), (dt,))
    _matrix("offsets", offsets, (e + 1,), ("int32",))
    ldw = _matrix("dw", dw, (e, n, k), (dt, "float32"))
    _rows_apart("dw", dw, ldw)
    se = dw.stride()[0]
    if e > 1 and n and k and se < (n - 1) * ldw + k:
        raise ValueError(f"dw's matrices overlap: stride {se} between experts")
    dev = _device(dy=dy, x=x, offsets=offsets, dw=dw)
    return BoundProduct("emmy_grouped_matmul_dw",
                        (dev, _TYPES[dt], _TYPES[_dtype(dw)], dy.data_ptr(), ldy, x.data_ptr(), ldx,
                         offsets.data_ptr(), dw.data_ptr(), se, ldw, rows, e, n, k, stream), (dy, x, offsets, dw))


def grouped_matmul_dw(dy, x, offsets, dw, stream: int = 0) -> None:
    """``dw[e] = dy_e.T @ x_e``: the gradient of :func:`grouped_matmul` by its weights.

    ``dy`` [rows, n] and ``x`` [rows, k] of one type (bfloat16 or float16), ``dw`` [experts, n, k] of
    that type or float32, as precise as :func:`grouped_matmul`'s outputs.  An expert without rows gets
    zeros."""
    bind_grouped_matmul_dw(dy, x, offsets, dw, stream)()


def bind_int8_matmul(xq, x_scale, wq, w_scale, out, offsets=None, bias=None, stream: int = 0) -> BoundProduct:
    """:func:`int8_matmul` with its arguments checked and prepared once."""
    grouped = offsets is not None
    if len(wq.shape) != (3 if grouped else 2):
        raise ValueError(f"wq has shape {tuple(wq.shape)}, expected "
                         + ("(experts, n, k) with offsets" if grouped else "(n, k) without offsets"))
    e = wq.shape[0] if grouped else 1
    n, k = wq.shape[-2:]
    _experts(e)
    if k > MAX_K8:
        raise ValueError(f"k is {k}: an 8-bit product of more than {MAX_K8} terms could pass 32 bits")
    ldx = _matrix("xq", xq, (None, k), ("int8",))
    ldw = _matrix("wq", wq, tuple(wq.shape), ("int8",))
    rows = xq.shape[0]
    _matrix("x_scale", x_scale, (rows,), ("float32",))
    for name, t in (("w_scale", w_scale), ("bias", bias)):
        if t is None:
            continue
        ld = _matrix(name, t, tuple(wq.shape[:-1]), ("float32",))
        if grouped and e > 1 and n and ld != n:
            raise ValueError(f"{name} must be contiguous, its row stride is {ld} for {n} channels")
    if grouped:
        _matrix("offsets", offsets, (e + 1,), ("int32",))
    ldo = _matrix("out", out, (rows, n), ("float32", "bfloat16", "float16"))
    _rows_apart("out", out, ldo)
    dev = _device(xq=xq, x_scale=x_scale, wq=wq, w_scale=w_scale, out=out, offsets=offsets, bias=bias)
    return BoundProduct("emmy_int8_matmul",
                        (dev, _TYPES[_dtype(out)], xq.data_ptr(), ldx, x_scale.data_ptr(), wq.data_ptr(),
                         wq.stride()[0] if grouped else 0, ldw, w_scale.data_ptr(),
                         None if bias is None else bias.data_ptr(), offsets.data_ptr() if grouped else None,
                         out.data_ptr(), ldo, rows, e, n, k, stream),
                        (xq, x_scale, wq, w_scale, out, offsets, bias))


def int8_matmul(xq, x_scale, wq, w_scale, out, offsets=None, bias=None, stream: int = 0) -> None:
    """``out[r, n] = (xq[r] . wq[n]) * x_scale[r] * w_scale[n] (+ bias[n])`` of int8 values.

    ``xq`` [rows, k], ``x_scale`` float32 [rows]; ``wq`` [n, k], ``w_scale`` and ``bias`` float32 [n],
    or, with ``offsets``, one of each for every expert: [experts, n, k] and [experts, n].  ``out``
    [rows, n] is float32, bfloat16 or float16.  The integer sum is exact (``k`` at most 131071); the
    scaling runs in f32 and is rounded once to the output's type."""
    bind_int8_matmul(xq, x_scale, wq, w_scale, out, offsets, bias, stream)()


def bind_quantize_rows(x, q, scale, stream: int = 0) -> BoundProduct:
    """:func:`quantize_rows` with its arguments checked and prepared once."""
    ldx = _matrix("x", x, (None, None), ("float32", "bfloat16", "float16"))
    rows, k = x.shape
    ldq = _matrix("q", q, (rows, k), ("int8",))
    _rows_apart("q", q, ldq)
    _matrix("scale", scale, (rows,), ("float32",))
    dev = _device(x=x, q=q, scale=scale)
    return BoundProduct("emmy_quantize_rows",
                        (dev, _TYPES[_dtype(x)], x.data_ptr(), ldx, q.data_ptr(), ldq, scale.data_ptr(), rows, k,
                         stream), (x, q, scale))


def quantize_rows(x, q, scale, stream: int = 0) -> None:
    """8-bit rows: ``scale[r] = max|x[r]| / 127`` in float32 and ``q[r, c] = x[r, c] / scale[r]`` rounded
    to the nearest integer, exact ties to even.

    ``x`` [rows, k] is float32, bfloat16 or float16, ``q`` int8 [rows, k], ``scale`` float32 [rows].  A row
    of zeros gives scale 0; a row that holds an infinity or NaN gives scale NaN and zeros, so that
    a product with it is NaN.  Weights are quantized the same way, one channel a row."""
    bind_quantize_rows(x, q, scale, stream)()


def variant(rows: int, experts: int, n: int, k: int, dw: bool = False, esize: int = 2,
            aligned: bool = True) -> tuple[bool, int, int]:
    """The kernel that a product of these extents runs on: whether pairs of CTAs, the output rows of a
    tile (0: nothing to launch), and how many CTAs divide a sum.

    ``dw`` asks for :func:`grouped_matmul_dw`, ``esize`` 1 for :func:`int8_matmul`; ``aligned`` says that
    both operands' bases and strides are multiples of 16 bytes.  Needs no GPU."""
    v = (C.c_int32 * 3)()
    runtime._check(runtime.lib().emmy_products_variant(esize, dw, aligned, rows, experts, n, k, v))
    return bool(v[0]), v[1], v[2]


def status(device: int = 0) -> int:
    """Read and clear the EMMY_STATUS_* bits of these kernels on ``device`` (0: every wait ended in
    time); synchronises the device."""
    runtime.init(device)
    st = C.c_uint32(0)
    runtime._check(runtime.lib().emmy_products_status(device, C.byref(st)))
    return st.value
