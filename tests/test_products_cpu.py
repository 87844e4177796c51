"""Refusals of the expert and 8-bit products, before anything reaches a GPU (CPU only)."""

from __future__ import annotations

import ctypes

import pytest
import torch

from emmy_ptx_compiler_b200 import products, runtime

BF16, F16, F32, I8, I32 = torch.bfloat16, torch.float16, torch.float32, torch.int8, torch.int32


def _t(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


def _grouped(**kw):
    a = dict(x=_t(6, 16), w=_t(2, 8, 16), offsets=_t(3, dtype=I32), out=_t(6, 8))
    a.update(kw)
    products.grouped_matmul(**a)


def _dw(**kw):
    a = dict(dy=_t(6, 8), x=_t(6, 16), offsets=_t(3, dtype=I32), dw=_t(2, 8, 16))
    a.update(kw)
    products.grouped_matmul_dw(**a)


def _int8(**kw):
    a = dict(xq=_t(6, 16, dtype=I8), x_scale=_t(6, dtype=F32), wq=_t(2, 8, 16, dtype=I8), w_scale=_t(2, 8, dtype=F32),
             out=_t(6, 8), offsets=_t(3, dtype=I32))
    a.update(kw)
    products.int8_matmul(**a)


def _quantize(**kw):
    a = dict(x=_t(6, 16), q=_t(6, 16, dtype=I8), scale=_t(6, dtype=F32))
    a.update(kw)
    products.quantize_rows(**a)


@pytest.mark.parametrize("call,change,message", [
    (_grouped, dict(x=_t(6, 15)), "x has shape"),
    (_grouped, dict(x=_t(6, 16, dtype=F32)), "x is float32"),
    (_grouped, dict(x=_t(16, 6).t()), "x's innermost axis"),
    (_grouped, dict(w=_t(2, 8, 16, dtype=F16)), "w is float16, x is bfloat16"),
    (_grouped, dict(w=_t(8, 16)), "w has shape"),
    (_grouped, dict(w=_t(8, 16, 2).permute(2, 0, 1)), "one of its last two axes"),
    (_grouped, dict(offsets=_t(2, dtype=I32)), "offsets has shape"),
    (_grouped, dict(offsets=_t(3, dtype=torch.int64)), "offsets is int64"),
    (_grouped, dict(out=_t(6, 8, dtype=F16)), "out is float16"),
    (_grouped, dict(out=_t(5, 8)), "out has shape"),
    (_grouped, dict(out=_t(8).expand(6, 8)), "out's rows overlap"),
    (_grouped, dict(w=_t(1025, 8, 16), offsets=_t(1026, dtype=I32)), "1025 experts"),
    (_grouped, dict(), "x is on cpu"),
    (_dw, dict(x=_t(5, 16)), "x has shape"),
    (_dw, dict(x=_t(6, 16, dtype=F16)), "x is float16"),
    (_dw, dict(dy=_t(6, 9)), "dy has shape"),
    (_dw, dict(dw=_t(2, 8, 16, dtype=F16)), "dw is float16"),
    (_dw, dict(dw=_t(8, 16)), "dw has shape"),
    (_dw, dict(dw=_t(2, 16, 8).transpose(1, 2)), "dw's innermost axis"),
    (_dw, dict(dw=_t(1, 8, 16).expand(2, 8, 16)), "dw's matrices overlap"),
    (_dw, dict(), "dy is on cpu"),
    (_int8, dict(xq=_t(6, 16, dtype=torch.uint8)), "xq is uint8"),
    (_int8, dict(x_scale=_t(5, dtype=F32)), "x_scale has shape"),
    (_int8, dict(x_scale=_t(6, dtype=BF16)), "x_scale is bfloat16"),
    (_int8, dict(x_scale=_t(12, dtype=F32)[::2]), "x_scale's innermost axis"),
    (_int8, dict(w_scale=_t(2, 7, dtype=F32)), "w_scale has shape"),
    (_int8, dict(w_scale=_t(2, 9, dtype=F32)[:, :8]), "w_scale must be contiguous"),
    (_int8, dict(bias=_t(8, dtype=F32)), "bias has shape"),
    (_int8, dict(offsets=None), "without offsets"),
    (_int8, dict(wq=_t(8, 16, dtype=I8)), "with offsets"),
    (_int8, dict(xq=_t(1, 131072, dtype=I8), wq=_t(2, 8, 131072, dtype=I8)), "could pass 32 bits"),
    (_int8, dict(out=_t(6, 8, dtype=torch.float64)), "out is float64"),
    (_int8, dict(), "xq is on cpu"),
    (_quantize, dict(x=_t(6, 16, dtype=torch.float64)), "x is float64"),
    (_quantize, dict(q=_t(6, 15, dtype=I8)), "q has shape"),
    (_quantize, dict(q=_t(16, dtype=I8).expand(6, 16)), "q's rows overlap"),
    (_quantize, dict(scale=_t(6, 1, dtype=F32)), "scale has shape"),
    (_quantize, dict(), "x is on cpu"),
])
def test_refusals(call, change, message):
    with pytest.raises(ValueError, match=message):
        call(**change)


def _error() -> bytes:
    buf = ctypes.create_string_buffer(512)
    runtime.lib().emmy_last_error(buf, 512)
    return buf.value


GROUPED = dict(dev=0, dtype=1, out_dtype=1, x=256, x_stride=16, w=256, w_stride_e=128, w_stride_n=16, w_stride_k=1,
               offsets=256, out=256, out_stride=8, rows=6, experts=2, n=8, k=16, stream=0)
DW = dict(dev=0, dtype=1, out_dtype=0, dy=256, dy_stride=8, x=256, x_stride=16, offsets=256, dw=256, dw_stride_e=128,
          dw_stride_n=16, rows=6, experts=2, n=8, k=16, stream=0)
INT8 = dict(dev=0, out_dtype=0, xq=256, x_stride=16, x_scale=256, wq=256, w_stride_e=128, w_stride_n=16, w_scale=256,
            bias=None, offsets=256, out=256, out_stride=8, rows=6, experts=2, n=8, k=16, stream=0)
QUANTIZE = dict(dev=0, dtype=1, x=256, x_stride=16, q=256, q_stride=16, scale=256, rows=6, k=16, stream=0)


@pytest.mark.parametrize("fn,base,change,message", [
    ("emmy_grouped_matmul", GROUPED, dict(dev=-1), b"bad device"),
    ("emmy_grouped_matmul", GROUPED, dict(dev=64), b"bad device"),
    ("emmy_grouped_matmul", GROUPED, dict(dtype=0, out_dtype=0), b"operands"),
    ("emmy_grouped_matmul", GROUPED, dict(out_dtype=2), b"output"),
    ("emmy_grouped_matmul", GROUPED, dict(rows=-1), b"2^31"),
    ("emmy_grouped_matmul", GROUPED, dict(rows=1 << 31), b"2^31"),
    ("emmy_grouped_matmul", GROUPED, dict(n=1 << 31, out_stride=1 << 31), b"2^31"),
    ("emmy_grouped_matmul", GROUPED, dict(experts=1025), b"experts"),
    ("emmy_grouped_matmul", GROUPED, dict(w_stride_k=2), b"strides"),
    ("emmy_grouped_matmul", GROUPED, dict(out_stride=7), b"overlap"),
    ("emmy_grouped_matmul", GROUPED, dict(x_stride=-1), b"negative"),
    ("emmy_grouped_matmul", GROUPED, dict(offsets=None), b"NULL"),
    ("emmy_grouped_matmul", GROUPED, dict(x=None), b"NULL"),
    ("emmy_grouped_matmul_dw", DW, dict(dtype=3), b"operands"),
    ("emmy_grouped_matmul_dw", DW, dict(k=-2), b"2^31"),
    ("emmy_grouped_matmul_dw", DW, dict(dw_stride_n=15), b"overlap"),
    ("emmy_grouped_matmul_dw", DW, dict(dw_stride_e=127), b"overlap"),
    ("emmy_grouped_matmul_dw", DW, dict(dw=None), b"NULL"),
    ("emmy_int8_matmul", INT8, dict(out_dtype=3), b"output"),
    ("emmy_int8_matmul", INT8, dict(k=131072, x_stride=131072, w_stride_n=131072), b"32 bits"),
    ("emmy_int8_matmul", INT8, dict(offsets=None), b"one expert"),
    ("emmy_int8_matmul", INT8, dict(w_scale=None), b"NULL"),
    ("emmy_quantize_rows", QUANTIZE, dict(dtype=3), b"rows must be"),
    ("emmy_quantize_rows", QUANTIZE, dict(q_stride=15), b"overlap"),
    ("emmy_quantize_rows", QUANTIZE, dict(scale=None), b"NULL"),
])
def test_library_refuses_before_any_launch(fn, base, change, message):
    assert getattr(runtime.lib(), fn)(*{**base, **change}.values()) == -3
    assert message in _error()


def test_calls_without_work_need_no_gpu():
    lib = runtime.lib()
    assert lib.emmy_grouped_matmul(*{**GROUPED, "rows": 0}.values()) == 0
    assert lib.emmy_grouped_matmul(*{**GROUPED, "n": 0}.values()) == 0
    assert lib.emmy_grouped_matmul_dw(*{**DW, "experts": 0}.values()) == 0
    assert lib.emmy_quantize_rows(*{**QUANTIZE, "rows": 0}.values()) == 0
    assert lib.emmy_products_status(0, None) == -3


def test_the_kernel_that_a_product_runs_on():
    assert products.variant(0, 3, 64, 64) == (False, 0, 1)            # nothing to launch
    assert products.variant(0, 3, 64, 64, dw=True) == (False, 128, 1)  # zeros to write
    assert products.variant(5, 1, 64, 0) == products.variant(5, 1, 64, 0, aligned=False)
    for bad in (dict(rows=-1), dict(experts=1025), dict(esize=3), dict(esize=1, dw=True),
                dict(rows=1 << 30, n=1 << 30)):
        with pytest.raises(runtime.EmmyError):
            products.variant(**{**dict(rows=5, experts=2, n=64, k=64), **bad})


def test_the_gpu_tests_reach_every_kernel():
    """A change of the rule that picks kernels must not take one away from the cases that test it."""
    import test_products_gpu as gpu

    forward, rows_gradient, int8, dw = set(), set(), set(), set()

    def aligned(unit, *strides):
        return all(s % unit == 0 for s in strides)

    for counts, n, k, pad in gpu.SHAPES:
        rows, e = sum(counts), len(counts)
        a = aligned(8, k + pad)
        forward.add((a, products.variant(rows + 5, e, n, k, aligned=a)[:2]))
        a = aligned(8, k + pad, n + pad)
        rows_gradient.add((a, products.variant(rows, e, k, n, aligned=a)[:2]))
        dw.add((a, products.variant(rows + 8, e, n, k, dw=True, aligned=a)[:2]))
    for counts, grouped, n, k, pad in gpu.INT8_SHAPES:
        a = aligned(16, k + pad)
        int8.add((a, products.variant(sum(counts) + (4 if grouped else 0), len(counts), n, k, esize=1, aligned=a)[:2]))
    for counts, n, k, esize, kernel in gpu.WIDTHS:
        a = aligned(16 // esize, k)
        for s in (int8,) if esize == 1 else (forward, rows_gradient):
            s.add((a, kernel[:2]))
    rows = sum(gpu.PAIR_COUNTS) + 8
    for n, k, width in gpu.DW_PAIRS:
        dw.add((True, products.variant(rows, len(gpu.PAIR_COUNTS), n, k, dw=True)[:2]))
    every = {(True, (False, w)) for w in (16, 32, 64, 128)} | {(False, (False, w)) for w in (32, 64, 128)}
    every |= {(True, (True, w)) for w in (128, 256)}
    assert forward == every and rows_gradient == every and int8 == every
    assert dw == {(True, (False, 128)), (False, (False, 128)), (True, (True, 128)), (True, (True, 256))}


def test_the_gpu_tests_reach_every_kernel_with_long_sums():
    import test_products_gpu as gpu

    every = {(0, (False, w)) for w in (16, 32, 64, 128)} | {(1, (False, w)) for w in (32, 64, 128)}
    every |= {(0, (True, w)) for w in (128, 256)}
    assert {(odd, kernel[:2]) for _, _, odd, kernel in gpu.LONG_FORWARD} == every
    for rows, n, odd, kernel in gpu.LONG_FORWARD:
        assert products.variant(rows, 1, n, 32768 + odd, aligned=not odd) == kernel
    reached = {(n % 8 == 0 and k % 8 == 0, kernel[:2]) for _, n, k, kernel in gpu.LONG_DW}
    assert reached == {(True, (False, 128)), (False, (False, 128)), (True, (True, 128)), (True, (True, 256))}
