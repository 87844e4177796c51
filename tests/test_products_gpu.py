"""Products grouped by expert, their gradients, 8-bit products and row quantization on the GPU,
against plain 64-bit implementations.

Tolerances.  A sum of ``k`` products held in f32 is off by at most about ``k`` half steps of the sum
of magnitudes; tensor cores may truncate instead of rounding, which is a whole step (2^-23) for
each addition.  Rounding to the output's type adds half a step of it, ``finfo.eps / 2`` relative to
the value (and, for f16, half of its smallest subnormal).  8-bit sums are exact, so only their
scaling in f32 (four roundings, and one of the s32 sum) and the output's rounding count.
"""

from __future__ import annotations

import pytest
import torch

from emmy_ptx_compiler_b200 import products, runtime

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _clean(cuda_device):
    yield
    assert products.status(cuda_device) == 0


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _gen(seed: int):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _offsets(counts, first=0):
    ends = [first]
    for c in counts:
        ends.append(ends[-1] + c)
    return torch.tensor(ends, dtype=torch.int32, device="cuda")


def _padded(rows, cols, dtype, g, pad=0, std=1.0, lead=0):
    """A [rows, cols] view of a wider buffer: row stride cols + pad, starting ``lead`` values in."""
    buf = torch.empty(rows * (cols + pad) + lead, dtype=F32, device="cuda").normal_(0, std, generator=g).to(dtype)
    return buf[lead:].view(rows, cols + pad)[:, :cols]


def _half_step(dtype, want):
    tiny = 2.0 ** -25 if dtype == F16 else 0.0
    return torch.finfo(dtype).eps / 2 * want.abs() + tiny


def _close(got, want, magnitude, terms):
    """``magnitude``: the sum of the magnitudes of each output's ``terms`` products."""
    tol = _half_step(got.dtype, want) * 1.01 + (terms + 2) * 2.0 ** -23 * magnitude
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), (got.double() - want).abs().max().item())


SHAPES = [
    # counts, n, k, row padding
    ([1], 64, 64, 0),
    ([0, 1, 0, 1, 1], 136, 72, 0),
    ([3, 0, 17, 16, 1], 128, 128, 8),
    ([33, 64, 0, 65, 2], 264, 520, 0),
    ([129, 1, 127, 0], 1000, 200, 24),
    ([300, 0, 513], 512, 1096, 0),
    ([257, 600, 255, 1], 776, 64, 8),
    ([2, 5], 100, 33, 0),            # rows of 66 bytes
    ([40, 7, 130], 77, 101, 3),      # odd extents and strides
    ([5, 0, 64], 1, 1, 0),
    ([1100], 640, 320, 0),
    # enough tiles for pairs of CTAs
    ([300, 7, 300, 256, 0, 64, 257, 1000], 1536, 1032, 0),
    ([100, 64, 1, 128, 200, 0, 65, 130], 2604, 1544, 8),
    ([70, 1, 64, 0, 16, 63, 100, 17], 160, 2056, 0),
    # odd rows, in tiles of 64 and of 128
    ([221, 162, 129, 132, 103, 116, 84, 75], 777, 1001, 0),
    ([128, 100, 156, 128, 0, 255, 128, 129], 2301, 135, 0),
    # enough tiles for a single CTA's widest
    ([60] * 8 + [50, 0, 61, 49, 50, 50, 64, 63], 2048, 2056, 0),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("out_f32", [False, True])
@pytest.mark.parametrize("counts,n,k,pad", SHAPES)
def test_grouped_matmul(counts, n, k, pad, dtype, out_f32):
    g = _gen(len(counts) * 1000 + n + k)
    first, spare = 2, 3   # rows before and behind the groups
    rows, e = first + sum(counts) + spare, len(counts)
    x = _padded(rows, k, dtype, g, pad)
    wide = _padded(e * n, k, dtype, g, pad, std=0.1).unflatten(0, (e, n))
    off = _offsets(counts, first)
    out = torch.full((rows, n + pad), 7.0, dtype=F32 if out_f32 else dtype, device="cuda")[:, :n]
    products.grouped_matmul(x, wide, off, out, stream=_stream())
    at = first
    for i, c in enumerate(counts):
        xs, ws = x[at:at + c].double(), wide[i].double()
        _close(out[at:at + c], xs @ ws.t(), xs.abs() @ ws.abs().t(), k)
        at += c
    assert (out[:first] == 7).all() and (out[at:] == 7).all(), "rows outside the groups stay as they were"
    if pad:
        assert (out.as_strided((rows, pad), (n + pad, 1), out.storage_offset() + n) == 7).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("counts,n,k,pad", SHAPES)
def test_grouped_matmul_by_the_other_axis(counts, n, k, pad, dtype):
    """Weights whose n axis is contiguous: the gradient by the rows."""
    g = _gen(len(counts) * 1000 + n + k + 1)
    rows, e = sum(counts), len(counts)
    w = _padded(e * n, k, dtype, g, pad, std=0.1).unflatten(0, (e, n))
    dy = _padded(rows, n, dtype, g, pad)
    off = _offsets(counts)
    dx = torch.empty(rows, k, dtype=dtype, device="cuda")
    products.grouped_matmul(dy, w.transpose(1, 2), off, dx, stream=_stream())
    at = 0
    for i, c in enumerate(counts):
        d, wi = dy[at:at + c].double(), w[i].double()
        _close(dx[at:at + c], d @ wi, d.abs() @ wi.abs(), n)
        at += c


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("out_f32", [False, True])
@pytest.mark.parametrize("counts,n,k,pad", SHAPES)
def test_grouped_matmul_dw(counts, n, k, pad, dtype, out_f32):
    g = _gen(len(counts) * 1000 + n + k + 2)
    first, spare = 3, 5
    rows, e = first + sum(counts) + spare, len(counts)
    dy, x = _padded(rows, n, dtype, g, pad), _padded(rows, k, dtype, g, pad)
    # what stands outside the groups must not reach the sums, not even as 0 * inf
    dy[:first], x[:first], dy[rows - spare:], x[rows - spare:] = float("inf"), float("nan"), float("nan"), float("inf")
    off = _offsets(counts, first)
    dw = torch.full((e, n, k + pad), 7.0, dtype=F32 if out_f32 else dtype, device="cuda")[..., :k]
    products.grouped_matmul_dw(dy, x, off, dw, stream=_stream())
    at = first
    for i, c in enumerate(counts):
        d, xi = dy[at:at + c].double(), x[at:at + c].double()
        _close(dw[i], d.t() @ xi, d.abs().t() @ xi.abs(), c)
        if c == 0:
            assert (dw[i] == 0).all()
        at += c


def test_one_experts_infinity_stays_with_it():
    """Neighbouring groups share tiles' loads: nothing of one may reach the other."""
    g = _gen(5)
    counts, n, k = [5, 11, 40, 3], 256, 192
    rows, e = sum(counts), len(counts)
    x, dy = _padded(rows, k, BF16, g), _padded(rows, n, BF16, g)
    w = _padded(e * n, k, BF16, g).unflatten(0, (e, n))
    off = _offsets(counts)
    x[5:16], dy[5:16], w[1] = float("nan"), float("inf"), float("nan")
    out = torch.empty(rows, n, dtype=BF16, device="cuda")
    dw = torch.empty(e, n, k, dtype=BF16, device="cuda")
    products.grouped_matmul(x, w, off, out, stream=_stream())
    products.grouped_matmul_dw(dy, x, off, dw, stream=_stream())
    assert out[5:16].isnan().all() and dw[1].isnan().all()
    assert out[:5].isfinite().all() and out[16:].isfinite().all() and dw[[0, 2, 3]].isfinite().all()


@pytest.mark.parametrize("offsets,meaning", [
    ([0, -5, 8, 4, 20], [(0, 0), (0, 8), (8, 8), (8, 12)]),
    ([5, 3, 200, 7, 9], [(5, 5), (5, 12), (12, 12), (12, 12)]),
    ([-3, 2, 2, 6, 6], [(0, 2), (2, 2), (2, 6), (6, 6)]),
])
def test_offsets_out_of_order_or_range(offsets, meaning):
    """An offset counts as the largest up to it, within the rows there are."""
    g = _gen(6)
    n, k, rows = 72, 80, 12
    x, w = _padded(rows, k, F16, g), _padded(4 * n, k, F16, g).unflatten(0, (4, n))
    off = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    out = torch.full((rows, n), 7.0, dtype=F32, device="cuda")
    products.grouped_matmul(x, w, off, out, stream=_stream())
    dw = torch.empty(4, n, k, dtype=F32, device="cuda")
    products.grouped_matmul_dw(out.to(F16), x, off, dw, stream=_stream())
    covered = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for i, (a, b) in enumerate(meaning):
        xs, ws = x[a:b].double(), w[i].double()
        _close(out[a:b], xs @ ws.t(), xs.abs() @ ws.abs().t(), k)
        d = out[a:b].to(F16).double()
        _close(dw[i], d.t() @ xs, d.abs().t() @ xs.abs(), b - a)
        covered[a:b] = True
    assert (out[~covered] == 7).all()


def test_empty_extents():
    z = dict(dtype=BF16, device="cuda")
    off0 = torch.zeros(4, dtype=torch.int32, device="cuda")
    products.grouped_matmul(torch.empty(0, 64, **z), torch.empty(3, 32, 64, **z), off0, torch.empty(0, 32, **z))
    products.grouped_matmul(torch.empty(5, 64, **z), torch.empty(0, 32, 64, **z), off0[:1], torch.empty(5, 32, **z))
    products.grouped_matmul(torch.empty(5, 64, **z), torch.empty(3, 0, 64, **z), off0, torch.empty(5, 0, **z))
    out = torch.full((5, 32), 7.0, **z)
    off = torch.tensor([0, 2, 2, 4], dtype=torch.int32, device="cuda")
    products.grouped_matmul(torch.empty(5, 0, **z), torch.empty(3, 32, 0, **z), off, out)
    assert (out[:4] == 0).all() and (out[4] == 7).all()      # a sum of nothing is zero
    dw = torch.full((3, 32, 64), 7.0, **z)
    products.grouped_matmul_dw(torch.empty(0, 32, **z), torch.empty(0, 64, **z), off0, dw)
    assert (dw == 0).all()
    i8 = dict(dtype=torch.int8, device="cuda")
    bias = torch.arange(32, dtype=F32, device="cuda")
    ones = torch.ones(32, dtype=F32, device="cuda")
    products.int8_matmul(torch.empty(5, 0, **i8), ones[:5], torch.empty(32, 0, **i8), ones, out, bias=bias)
    assert (out == bias.to(BF16)).all()
    scale = torch.full((3,), 7.0, device="cuda")
    products.quantize_rows(torch.empty(3, 0, **z), torch.empty(3, 0, **i8), scale)
    assert (scale == 0).all()
    products.quantize_rows(torch.empty(0, 8, **z), torch.empty(0, 8, **i8), scale[:0])


def test_gradients_against_differences():
    """The product is linear in each operand: along a direction, loss(x + h) - loss(x - h) is exact."""
    g = _gen(7)
    counts, n, k = [9, 0, 30, 25], 48, 56
    rows, e = sum(counts), len(counts)
    # small integers: every sum below is exact in f32
    def ints(*shape):
        return torch.randint(-3, 4, shape, device="cuda", generator=g).to(BF16)
    x, w, dy = ints(rows, k), ints(e, n, k), ints(rows, n)
    off = _offsets(counts)

    def loss(x, w):
        out = torch.empty(rows, n, dtype=F32, device="cuda")
        products.grouped_matmul(x, w, off, out, stream=_stream())
        return (out.double() * dy.double()).sum().item()

    dx, dw = torch.empty(rows, k, dtype=F32, device="cuda"), torch.empty(e, n, k, dtype=F32, device="cuda")
    products.grouped_matmul(dy, w.transpose(1, 2), off, dx, stream=_stream())
    products.grouped_matmul_dw(dy, x, off, dw, stream=_stream())
    hx, hw = ints(rows, k), ints(e, n, k)
    assert loss(x + hx, w) - loss(x - hx, w) == 2 * (dx.double() * hx.double()).sum().item()
    assert loss(x, w + hw) - loss(x, w - hw) == 2 * (dw.double() * hw.double()).sum().item()


INT8_SHAPES = [
    # rows of each expert (one entry, grouped False: a plain product), n, k, padding
    ([1], False, 64, 128, 0),
    ([1], False, 4096, 4096, 0),
    ([16], False, 512, 2048, 16),
    ([70], False, 200, 144, 0),
    ([333], False, 1001, 1111, 0),
    ([600], False, 768, 640, 32),
    ([3, 0, 50, 129], True, 272, 160, 0),
    ([300, 1, 0, 280], True, 520, 1024, 16),
    ([5, 9, 0], True, 33, 17, 1),
    ([600], False, 4120, 640, 0),
    ([150], False, 5120, 400, 0),
    ([500, 0, 130, 1, 700], True, 1030, 528, 0),
]


@pytest.mark.parametrize("out_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("counts,grouped,n,k,pad", INT8_SHAPES)
def test_int8_matmul(counts, grouped, n, k, pad, with_bias, out_dtype):
    g = _gen(n + k)
    first = 2 if grouped else 0
    rows, e = first + sum(counts) + first, len(counts)
    xq = torch.randint(-128, 128, (rows, k + pad), dtype=torch.int8, device="cuda", generator=g)[:, :k]
    wq = torch.randint(-128, 128, (e, n, k + pad), dtype=torch.int8, device="cuda", generator=g)[..., :k]
    xs = torch.rand(rows, device="cuda", generator=g) + 0.5
    ws = (torch.rand(e, n, device="cuda", generator=g) + 0.5) * 2.0 ** -14
    bias = torch.empty(e, n, device="cuda").normal_(generator=g) if with_bias else None
    out = torch.full((rows, n + pad), 7.0, dtype=out_dtype, device="cuda")[:, :n]
    if grouped:
        products.int8_matmul(xq, xs, wq, ws, out, offsets=_offsets(counts, first), bias=bias, stream=_stream())
    else:
        products.int8_matmul(xq, xs, wq[0], ws[0], out, bias=None if bias is None else bias[0], stream=_stream())
    at = first
    for i, c in enumerate(counts):
        y = xq[at:at + c].double() @ wq[i].double().t() * xs[at:at + c, None].double() * ws[i].double()
        want = y if bias is None else y + bias[i].double()
        tol = _half_step(out_dtype, want) * 1.01 + 5 * 2.0 ** -24 * (y.abs() + want.abs())
        assert ((out[at:at + c].double() - want).abs() <= tol).all()
        at += c
    assert (out[:first] == 7).all() and (out[at:] == 7).all()


@pytest.mark.parametrize("k", [8192, 131071])
def test_int8_sums_are_exact(k):
    """The largest sums, beyond what f32 holds exactly, come out as the s32 sum rounded once."""
    xq = torch.full((3, k), -128, dtype=torch.int8, device="cuda")
    wq = torch.full((40, k), -128, dtype=torch.int8, device="cuda")
    wq[1], wq[2, 0] = 127, -127
    one = torch.ones(40, device="cuda")
    out = torch.empty(3, 40, device="cuda")
    products.int8_matmul(xq, one[:3], wq, one, out, stream=_stream())
    want = (xq.double() @ wq.double().t()).float()
    assert torch.equal(out, want)


def _quantize_reference(x):
    # the quotient in 64 bits rounds to the f32 quotient: 53 bits are more than twice 24 and two
    scale = (x.abs().amax(1).double() / 127.0).float()
    q = (x.double() / scale.double()[:, None]).round().clamp(-127, 127)
    return torch.where(scale[:, None] > 0, q, torch.zeros_like(q)).to(torch.int8), scale


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows,k,pad,lead", [(1, 1, 0, 0), (1, 4096, 0, 0), (7, 100, 0, 0), (33, 1000, 24, 0),
                                             (5, 1111, 2, 1), (300, 256, 0, 8), (4, 20000, 8, 0), (2, 70001, 0, 0),
                                             (1500, 64, 0, 3), (19, 8192, 0, 0)])
def test_quantize_rows(rows, k, pad, lead, dtype):
    g = _gen(rows + k)
    x = _padded(rows, k, dtype, g, pad, lead=lead)
    x *= torch.rand(rows, 1, device="cuda", generator=g) * 10 + 0.01
    q = torch.full((rows, k + pad), 99, dtype=torch.int8, device="cuda")[:, :k]
    scale = torch.empty(rows, device="cuda")
    products.quantize_rows(x, q, scale, stream=_stream())
    want_q, want_s = _quantize_reference(x)
    assert torch.equal(scale, want_s) and torch.equal(q, want_q)
    if pad:
        assert (q.as_strided((rows, pad), (k + pad, 1), q.storage_offset() + k) == 99).all()


@pytest.mark.parametrize("k", [96, 4097])
def test_quantize_rows_ties_extremes_and_non_finite(k):
    x = torch.zeros(12, k, device="cuda")
    # scale 1: exact halves go to the even integer, and their f32 neighbours to their own side
    halves = torch.arange(-40, 40, device="cuda") + 0.5
    x[0, 0], x[0, 1:81] = 127.0, halves
    up, down = torch.full_like(halves, 1e9), torch.full_like(halves, -1e9)
    x[1, 0], x[1, 1:81] = 127.0, torch.nextafter(halves, up)
    x[2, 0], x[2, 1:81] = -127.0, torch.nextafter(halves, down)
    x[3, 5] = 1e-45                                   # a scale that vanishes
    x[4, 5], x[4, 6] = 1e-43, -6e-44                  # a subnormal scale
    x[5, :] = 3.4e38
    x[6, 3] = float("inf")
    x[7, 3], x[7, 4] = float("nan"), 5.0
    x[8, k - 1] = float("-inf")
    x[10] = torch.linspace(-1, 1, k, device="cuda") * 2.0 ** -126
    x[11] = torch.linspace(-3, 3, k, device="cuda")
    q = torch.full((12, k), 99, dtype=torch.int8, device="cuda")
    scale = torch.empty(12, device="cuda")
    products.quantize_rows(x, q, scale, stream=_stream())
    finite = [0, 1, 2, 3, 4, 5, 9, 10, 11]
    want_q, want_s = _quantize_reference(x[finite])
    assert torch.equal(scale[finite], want_s) and torch.equal(q[finite], want_q)
    assert scale[6:9].isnan().all() and (q[6:9] == 0).all()


def test_halves_of_a_scale_that_is_not_a_power_of_two():
    """Values next to (j + 1/2) * scale, where the quotient in f32 alone can round to the wrong side."""
    g = _gen(9)
    rows, k = 64, 254
    peak = torch.rand(rows, 1, device="cuda", generator=g) * 100 + 1
    scale = (peak / 127.0).double()
    j = torch.arange(-126, 126, device="cuda").double() + 0.5
    x = torch.empty(rows, k, device="cuda")
    x[:, 0], x[:, 1] = peak[:, 0], -peak[:, 0]
    x[:, 2:] = (j * scale).float()
    q, s = torch.empty(rows, k, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    products.quantize_rows(x, q, s, stream=_stream())
    want_q, want_s = _quantize_reference(x)
    assert torch.equal(s, want_s) and torch.equal(q, want_q)


def test_a_quantized_expert_layer_and_its_training_twin():
    """The calls as a program strings them together: experts in 16 bits with their gradients, the same
    weights quantized (a channel a row) and run on rows quantized on the way, on a side stream, then
    recorded into a graph and replayed on new rows and new groups."""
    g = _gen(11)
    e, hidden, inner, rows = 6, 256, 320, 96
    side = torch.cuda.Stream()
    up = _padded(e * inner, hidden, BF16, g, std=hidden ** -0.5).unflatten(0, (e, inner))
    down = _padded(e * hidden, inner, BF16, g, std=inner ** -0.5).unflatten(0, (e, hidden))
    x = _padded(rows, hidden, BF16, g)
    off = _offsets([10, 0, 40, 1, 25, 20])
    z = dict(device="cuda")
    q = {}
    h, y = torch.empty(rows, inner, dtype=BF16, **z), torch.empty(rows, hidden, dtype=BF16, **z)
    h8, y8 = torch.empty_like(h), torch.empty_like(y)
    dh, dx = torch.empty_like(h), torch.empty_like(x)
    dup, ddown = torch.empty_like(up), torch.empty_like(down)
    xq, xs = torch.empty(rows, hidden, dtype=torch.int8, **z), torch.empty(rows, **z)
    hq, hs = torch.empty(rows, inner, dtype=torch.int8, **z), torch.empty(rows, **z)
    torch.cuda.synchronize()
    s = side.cuda_stream
    for name, w in (("up", up), ("down", down)):
        wq = torch.empty(w.shape, dtype=torch.int8, **z)
        ws = torch.empty(w.shape[:2], **z)
        products.quantize_rows(w.view(-1, w.shape[2]), wq.view(-1, w.shape[2]), ws.view(-1), stream=s)
        q[name] = (wq, ws)

    def layer():
        products.grouped_matmul(x, up, off, h, stream=s)
        products.grouped_matmul(h, down, off, y, stream=s)
        # gradients for dy = y
        products.grouped_matmul_dw(y, h, off, ddown, stream=s)
        products.grouped_matmul(y, down.transpose(1, 2), off, dh, stream=s)
        products.grouped_matmul_dw(dh, x, off, dup, stream=s)
        products.grouped_matmul(dh, up.transpose(1, 2), off, dx, stream=s)
        products.quantize_rows(x, xq, xs, stream=s)
        products.int8_matmul(xq, xs, *q["up"], h8, offsets=off, stream=s)
        products.quantize_rows(h8, hq, hs, stream=s)
        products.int8_matmul(hq, hs, *q["down"], y8, offsets=off, stream=s)

    def check():
        torch.cuda.synchronize()
        ends = off.tolist()
        for i in range(e):
            r = slice(ends[i], ends[i + 1])
            X, U, D = x[r].double(), up[i].double(), down[i].double()
            H, Y = h[r].double(), y[r].double()
            _close(h[r], X @ U.t(), X.abs() @ U.abs().t(), hidden)
            _close(y[r], H @ D.t(), H.abs() @ D.abs().t(), inner)
            _close(ddown[i], Y.t() @ H, Y.abs().t() @ H.abs(), H.shape[0])
            _close(dh[r], Y @ D, Y.abs() @ D.abs(), hidden)
            DH = dh[r].double()
            _close(dup[i], DH.t() @ X, DH.abs().t() @ X.abs(), X.shape[0])
            _close(dx[r], DH @ U, DH.abs() @ U.abs(), inner)
            for src, (a, sa), (w, sw), dst in ((x, (xq, xs), q["up"], h8), (h8, (hq, hs), q["down"], y8)):
                wantq, wants = _quantize_reference(src[r])
                assert torch.equal(a[r], wantq) and torch.equal(sa[r], wants)
                want = wantq.double() @ w[i].double().t() * wants[:, None].double() * sw[i].double()
                assert ((dst[r].double() - want).abs() <= _half_step(BF16, want) * 1.01 + 2.0 ** -21 * want.abs()).all()

    layer()
    check()
    with runtime.Graph.record(0, s) as graph:
        layer()
    x.copy_(_padded(rows, hidden, BF16, g))
    off.copy_(_offsets([0, 33, 3, 0, 59, 1]))
    for t in (h, y, h8, y8, dh, dx, dup, ddown):
        t.zero_()
    torch.cuda.synchronize()
    graph.launch(s)
    check()
    graph.close()


def test_calls_that_overlap_on_two_streams():
    """Nothing is shared between calls: the same product on two streams at once gives the same bits."""
    g = _gen(12)
    counts = [20, 3, 0, 60, 45]
    rows, n, k, e = sum(counts), 384, 2048, len(counts)
    x, w = _padded(rows, k, BF16, g), _padded(e * n, k, BF16, g).unflatten(0, (e, n))
    off = _offsets(counts)
    outs = [torch.empty(rows, n, dtype=BF16, device="cuda") for _ in range(3)]
    dws = [torch.empty(e, n, k, dtype=BF16, device="cuda") for _ in range(3)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    products.grouped_matmul(x, w, off, outs[2], stream=_stream())
    products.grouped_matmul_dw(outs[2], x, off, dws[2], stream=_stream())
    torch.cuda.synchronize()
    for _ in range(10):
        for st, o, d in zip(streams, outs, dws):
            products.grouped_matmul(x, w, off, o, stream=st.cuda_stream)
            products.grouped_matmul_dw(outs[2], x, off, d, stream=st.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[2])
    assert torch.equal(dws[0], dws[2]) and torch.equal(dws[1], dws[2])


def test_bound_calls_repeat_on_their_buffers():
    g = _gen(13)
    n, k = 512, 1024
    wq = torch.randint(-127, 128, (n, k), dtype=torch.int8, device="cuda", generator=g)
    ws = torch.rand(n, device="cuda", generator=g)
    x = torch.empty(4, k, dtype=F16, device="cuda")
    xq, xs = torch.empty(4, k, dtype=torch.int8, device="cuda"), torch.empty(4, device="cuda")
    out = torch.empty(4, n, device="cuda")
    calls = [products.bind_quantize_rows(x, xq, xs, stream=_stream()),
             products.bind_int8_matmul(xq, xs, wq, ws, out, stream=_stream())]
    for _ in range(3):
        x.normal_(generator=g)
        for call in calls:
            call()
        q, s = _quantize_reference(x)
        want = q.double() @ wq.double().t() * s[:, None].double() * ws.double()
        assert ((out.double() - want).abs() <= 5 * 2.0 ** -24 * 2 * want.abs()).all()


def test_more_experts_than_any_tile_has_lanes():
    g = _gen(14)
    e, n, k = 1000, 40, 48
    counts = torch.randint(0, 4, (e,), generator=torch.Generator().manual_seed(3)).tolist()
    rows = sum(counts)
    x, w = _padded(rows, k, F16, g), _padded(e * n, k, F16, g).unflatten(0, (e, n))
    off = _offsets(counts)
    out = torch.empty(rows, n, dtype=F32, device="cuda")
    dw = torch.empty(e, n, k, dtype=F32, device="cuda")
    products.grouped_matmul(x, w, off, out, stream=_stream())
    products.grouped_matmul_dw(out.to(F16), x, off, dw, stream=_stream())
    owner = torch.repeat_interleave(torch.arange(e), torch.tensor(counts)).cuda()
    want = torch.einsum("rk,rnk->rn", x.double(), w.double()[owner])
    size = torch.einsum("rk,rnk->rn", x.double().abs(), w.double()[owner].abs())
    _close(out, want, size, k)
    outer = out.to(F16).double()[:, :, None] * x.double()[:, None, :]
    want = torch.zeros(e, n, k, dtype=torch.float64, device="cuda").index_add_(0, owner, outer)
    size = torch.zeros_like(want).index_add_(0, owner, outer.abs())
    _close(dw, want, size, 4)


NAN_PADS = [([3, 20, 0, 9], 200, 72), ([3, 20, 0, 9], 136, 101), ([150, 40, 260], 1000, 100), ([300] * 8, 1544, 1000)]


@pytest.mark.parametrize("counts,n,k", NAN_PADS)
def test_what_lies_between_rows_is_never_used(counts, n, k):
    """Rows padded with NaN, in every operand of all three products and of the 8-bit one."""
    g = _gen(21)
    rows, e, pad = sum(counts), len(counts), 8
    x, dy = _padded(rows, k, BF16, g, pad), _padded(rows, n, BF16, g, pad)
    w = _padded(e * n, k, BF16, g, pad, std=0.1)
    for t, cols in ((x, k), (dy, n), (w, k)):
        t.as_strided((t.shape[0], pad), (cols + pad, 1), t.storage_offset() + cols).fill_(float("nan"))
    w = w.unflatten(0, (e, n))
    off = _offsets(counts)
    out = torch.empty(rows, n, dtype=BF16, device="cuda")
    dx = torch.empty(rows, k, dtype=BF16, device="cuda")
    dw = torch.empty(e, n, k, dtype=F32, device="cuda")
    products.grouped_matmul(x, w, off, out, stream=_stream())
    products.grouped_matmul(dy, w.transpose(1, 2), off, dx, stream=_stream())
    products.grouped_matmul_dw(dy, x, off, dw, stream=_stream())
    assert out.isfinite().all() and dx.isfinite().all() and dw.isfinite().all()
    at = 0
    for i, c in enumerate(counts):
        X, D, W = x[at:at + c].double(), dy[at:at + c].double(), w[i].double()
        _close(out[at:at + c], X @ W.t(), X.abs() @ W.abs().t(), k)
        _close(dx[at:at + c], D @ W, D.abs() @ W.abs(), n)
        _close(dw[i], D.t() @ X, D.abs().t() @ X.abs(), c)
        at += c


def test_broadcast_rows_and_shared_weights():
    """Strides of 0: one row for all rows of x, one matrix for all experts."""
    g = _gen(22)
    counts, n, k = [4, 0, 70, 6], 264, 128
    rows, e = sum(counts), len(counts)
    x = _padded(1, k, F16, g).expand(rows, k)
    w = _padded(n, k, F16, g).unsqueeze(0).expand(e, n, k)
    off = _offsets(counts)
    out = torch.empty(rows, n, dtype=F32, device="cuda")
    products.grouped_matmul(x, w, off, out, stream=_stream())
    _close(out, x.double() @ w[0].double().t(), x.double().abs() @ w[0].double().abs().t(), k)
    dw = torch.empty(e, n, k, dtype=F32, device="cuda")
    dy = _padded(rows, n, F16, g)
    products.grouped_matmul_dw(dy, x, off, dw, stream=_stream())
    for i, (a, b) in enumerate(zip(off.tolist(), off.tolist()[1:])):
        d, X = dy[a:b].double(), x[a:b].double()
        _close(dw[i], d.t() @ X, d.abs().t() @ X.abs(), b - a)


def test_weights_in_the_other_order_and_single_axes():
    """[experts, k, n] weights as a view, and extents of 1, whose strides mean nothing."""
    g = _gen(23)
    for n, k in ((96, 64), (1, 64), (96, 1), (1, 1)):
        w = _padded(3 * k, n, BF16, g).unflatten(0, (3, k)).transpose(1, 2)
        x = _padded(9, k, BF16, g)
        off, out = _offsets([2, 0, 7]), torch.empty(9, n, dtype=F32, device="cuda")
        products.grouped_matmul(x, w, off, out, stream=_stream())
        for i, (a, b) in enumerate(((0, 2), (2, 2), (2, 9))):
            X, W = x[a:b].double(), w[i].double()
            _close(out[a:b], X @ W.t(), X.abs() @ W.abs().t(), k)


@pytest.mark.parametrize("k", [2048, 2041])
def test_positions_beyond_31_bits(k):
    """Operands and outputs of more than 2^31 values: the last rows' addresses need 64 bits."""
    rows, n = 1_100_000, 2048
    x = torch.zeros(rows, k, dtype=torch.int8, device="cuda")
    tail = 300
    g = _gen(24)
    x[-tail:] = torch.randint(-127, 128, (tail, k), dtype=torch.int8, device="cuda", generator=g)
    w = torch.randint(-127, 128, (n, k), dtype=torch.int8, device="cuda", generator=g)
    xs, ws = torch.ones(rows, device="cuda"), torch.ones(n, device="cuda")
    out = torch.empty(rows, n, dtype=F32, device="cuda")
    assert x.numel() > 1 << 31 and out.numel() > 1 << 31
    products.int8_matmul(x, xs, w, ws, out, stream=_stream())
    assert torch.equal(out[-tail:], (x[-tail:].double() @ w.double().t()).float())
    assert (out[:100] == 0).all() and (out[-tail - 100:-tail] == 0).all()


def test_experts_beyond_31_bits():
    """Weights and their gradients of more than 2^31 values."""
    g = _gen(25)
    e, n, k = 600, 2048, 2048
    counts = [0] * (e - 2) + [5, 11]
    w = torch.empty(e, n, k, dtype=BF16, device="cuda")
    assert w.numel() > 1 << 31
    w[-2:].normal_(generator=g)
    x, dy = _padded(16, k, BF16, g), _padded(16, n, BF16, g)
    off = _offsets(counts)
    out = torch.empty(16, n, dtype=F32, device="cuda")
    products.grouped_matmul(x, w, off, out, stream=_stream())
    for i, a, b in ((-2, 0, 5), (-1, 5, 16)):
        X, W = x[a:b].double(), w[i].double()
        _close(out[a:b], X @ W.t(), X.abs() @ W.abs().t(), k)
    products.grouped_matmul_dw(dy, x, off, w, stream=_stream())
    for i, a, b in ((-2, 0, 5), (-1, 5, 16)):
        D, X = dy[a:b].double(), x[a:b].double()
        _close(w[i], D.t() @ X, D.abs().t() @ X.abs(), b - a)
    assert (w[:2] == 0).all() and (w[-4:-2] == 0).all()


def test_long_sums_are_split_and_joined_in_order():
    """Few tiles and long sums: parts of them on several SMs, with the same bits every time."""
    g = _gen(26)
    off = _offsets([20011, 0])
    dy, x = _padded(20011, 264, BF16, g), _padded(20011, 200, BF16, g)
    dws = [torch.empty(2, 264, 200, dtype=F32, device="cuda") for _ in range(3)]
    for dw in dws:
        products.grouped_matmul_dw(dy, x, off, dw, stream=_stream())
    D, X = dy.double(), x.double()
    _close(dws[0][0], D.t() @ X, D.abs().t() @ X.abs(), 20011)
    assert torch.equal(dws[0], dws[1]) and torch.equal(dws[0], dws[2]) and (dws[0][1] == 0).all()
    for rows in (1, 9, 20, 40, 100):
        xq = torch.randint(-127, 128, (rows, 16384), dtype=torch.int8, device="cuda", generator=g)
        wq = torch.randint(-127, 128, (300, 16384), dtype=torch.int8, device="cuda", generator=g)
        ones = torch.ones(300, device="cuda")
        out = torch.empty(rows, 300, device="cuda")
        products.int8_matmul(xq, ones[:rows], wq, ones, out, stream=_stream())
        assert torch.equal(out, (xq.double() @ wq.double().t()).float())
        xb, wb = _padded(rows, 8192, F16, g), _padded(300, 8192, F16, g).unsqueeze(0)
        outs = [torch.empty(rows, 300, dtype=F16, device="cuda") for _ in range(2)]
        for o in outs:
            products.grouped_matmul(xb, wb, _offsets([rows]), o, stream=_stream())
        _close(outs[0], xb.double() @ wb[0].double().t(), xb.double().abs() @ wb[0].double().abs().t(), 8192)
        assert torch.equal(outs[0], outs[1])


FIRST_CALL_RECORDED = """
import torch
from emmy_ptx_compiler_b200 import products, runtime
runtime.init(0)
rows, n, k, e = 40, 256, 512, 2
x = torch.randint(-3, 4, (rows, k), device="cuda").to(torch.bfloat16)
w = torch.randint(-3, 4, (e, n, k), device="cuda").to(torch.bfloat16)
off = torch.tensor([0, 30, 40], dtype=torch.int32, device="cuda")
out = torch.zeros(rows, n, device="cuda")
q, s = torch.zeros(rows, k, dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda")
side = torch.cuda.Stream()
torch.cuda.synchronize()
with runtime.Graph.record(0, side.cuda_stream) as graph:
    runtime._check(runtime.lib().emmy_memset_d8(0, out.data_ptr(), 1, out.numel() * 4, side.cuda_stream))
    products.grouped_matmul(x, w, off, out, stream=side.cuda_stream)
    products.quantize_rows(x, q, s, stream=side.cuda_stream)
graph.launch(side.cuda_stream)
torch.cuda.synchronize()
want = torch.cat([x[:30].double() @ w[0].double().t(), x[30:].double() @ w[1].double().t()])
assert torch.equal(out.double(), want)
assert torch.equal(s, (x.abs().amax(1).double() / 127).float())
assert products.status(0) == 0
graph.close()
print("recorded")
"""

FIRST_CALL_IN_A_TORCH_GRAPH = """
import torch
from emmy_ptx_compiler_b200 import products
x = torch.randint(-3, 4, (600, 512), device="cuda").to(torch.float16)
w = torch.randint(-3, 4, (2, 2560, 512), device="cuda").to(torch.float16)
off = torch.tensor([0, 250, 600], dtype=torch.int32, device="cuda")
out, dw = torch.zeros(600, 2560, device="cuda"), torch.zeros(2, 2560, 512, device="cuda")
dy = torch.randint(-3, 4, (600, 2560), device="cuda").to(torch.float16)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    s = torch.cuda.current_stream().cuda_stream
    products.grouped_matmul(x, w, off, out, stream=s)
    products.grouped_matmul_dw(dy, x, off, dw, stream=s)
    out.mul_(2)
for _ in range(3):
    graph.replay()
torch.cuda.synchronize()
for e, (a, b) in enumerate(((0, 250), (250, 600))):
    assert torch.equal(out[a:b].double(), 2 * (x[a:b].double() @ w[e].double().t()))
    assert torch.equal(dw[e].double(), dy[a:b].double().t() @ x[a:b].double())
assert products.status(0) == 0
print("recorded")
"""


@pytest.mark.parametrize("code", [FIRST_CALL_RECORDED, FIRST_CALL_IN_A_TORCH_GRAPH])
def test_a_first_call_can_be_recorded(code, cuda_device):
    """In a process that has made no call before: loading the kernels does not disturb the recording."""
    import subprocess
    import sys

    from conftest import REPO

    r = subprocess.run([sys.executable, "-c", code], cwd=REPO, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "recorded" in r.stdout, r.stderr[-2000:]


def test_two_host_threads_at_once():
    """Calls from two threads on their own streams: nothing on the host side is shared either."""
    import threading

    g = _gen(27)
    counts, n, k = [33, 0, 80], 256, 264
    rows, e = sum(counts), len(counts)
    x, w = _padded(rows, k, F16, g), _padded(e * n, k, F16, g).unflatten(0, (e, n))
    off = _offsets(counts)
    want = torch.empty(rows, n, dtype=F16, device="cuda")
    products.grouped_matmul(x, w, off, want, stream=_stream())
    torch.cuda.synchronize()
    outs = [torch.empty_like(want) for _ in range(2)]
    errors = []

    def run(o):
        try:
            s = torch.cuda.Stream()
            for _ in range(50):
                products.grouped_matmul(x, w, off, o, stream=s.cuda_stream)
            s.synchronize()
        except Exception as exc:  # reported below, on the test's thread
            errors.append(exc)

    threads = [threading.Thread(target=run, args=(o,)) for o in outs]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors and torch.equal(outs[0], want) and torch.equal(outs[1], want)


def _ints(g, *shape, dtype=BF16, pad=0):
    """Values whose sums of up to 2^24 / 9 products are exact in f32, in rows ``pad`` apart."""
    return torch.randint(-3, 4, (*shape[:-1], shape[-1] + pad), device="cuda", generator=g).to(dtype)[..., :shape[-1]]


# rows of each expert of gradients that run on pairs of CTAs: last blocks of 1, 15, 16, 17, 63, 64 rows, an
# empty group, groups that end on a block between others, a single row
PAIR_COUNTS = [513, 527, 528, 529, 575, 512, 576, 0, 1, 64, 1100, 640]
# n, k, rows of a tile; the first has several tiles for each pair of CTAs
DW_PAIRS = [(1032, 1032, 256), (264, 384, 256), (104, 776, 128), (200, 392, 128)]


@pytest.mark.parametrize("dtype,out_dtype", [(BF16, F32), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("n,k,width", DW_PAIRS)
def test_dw_on_pairs_of_ctas(n, k, width, dtype, out_dtype):
    """Against exact sums, in two orders of the groups, with infinities and NaN in some groups and
    outside all of them."""
    g = _gen(n + k)
    first, spare, pad = 3, 5, 8
    rows, e = first + sum(PAIR_COUNTS) + spare, len(PAIR_COUNTS)
    assert products.variant(rows, e, n, k, dw=True) == (True, width, 1)
    dw = torch.full((e, n, k + pad), 7.0, dtype=out_dtype, device="cuda")[..., :k]
    for counts in (PAIR_COUNTS, PAIR_COUNTS[::-1]):
        dy, x = _ints(g, rows, n, dtype=dtype, pad=pad), _ints(g, rows, k, dtype=dtype)
        off = _offsets(counts, first)
        ends = off.tolist()
        lost = [counts.index(528), counts.index(64)]
        for a, b in [(0, first), (rows - spare, rows)] + [(ends[i], ends[i + 1]) for i in lost]:
            dy[a:b], x[a:b] = float("inf"), float("nan")
        for _ in range(3):
            products.grouped_matmul_dw(dy, x, off, dw, stream=_stream())
        for i in range(e):
            r = slice(ends[i], ends[i + 1])
            if i in lost:
                assert dw[i].isnan().all()
            else:
                want = (dy[r].double().t() @ x[r].double()).float().to(out_dtype)
                assert torch.equal(dw[i], want), (i, counts[i])
        assert (dw.as_strided((e, n, pad), dw.stride(), dw.storage_offset() + k) == 7).all()


def test_dw_on_pairs_of_ctas_recorded():
    """A recorded call follows new offsets, whichever of the groups end inside a block."""
    g = _gen(41)
    n, k, e = 264, 384, len(PAIR_COUNTS)
    rows = sum(PAIR_COUNTS)
    assert products.variant(rows, e, n, k, dw=True)[0]
    dy, x, off = _ints(g, rows, n), _ints(g, rows, k), _offsets(PAIR_COUNTS)
    dw = torch.empty(e, n, k, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with runtime.Graph.record(0, s.cuda_stream) as graph:
        products.grouped_matmul_dw(dy, x, off, dw, stream=s.cuda_stream)
    for counts in (PAIR_COUNTS, sorted(PAIR_COUNTS), [0] * (e - 1) + [rows], [rows - 11] + [1] * (e - 1), [64] * e):
        off.copy_(_offsets(counts))
        dw.fill_(7)
        torch.cuda.synchronize()
        graph.launch(s.cuda_stream)
        torch.cuda.synchronize()
        at = 0
        for i, c in enumerate(counts):
            assert torch.equal(dw[i].double(), dy[at:at + c].double().t() @ x[at:at + c].double()), (counts, i)
            at += c
    graph.close()


# rows of each expert, n, k, operands' size, the kernel: tiles that the shapes above do not reach
WIDTHS = [
    ([20, 14, 24], 136, 136, 2, (False, 32, 1)),
    ([1700], 1100, 65, 2, (False, 128, 1)),
    ([700], 1100, 65, 1, (False, 64, 1)),
    ([1700], 1100, 65, 1, (False, 128, 1)),
    ([60] * 16, 1300, 144, 1, (False, 128, 1)),
]
# sums divided among 2, 4 and 8 CTAs, for each width of a tile
SPLITS = [
    ([40], 2080, 1025, 2, (False, 32, 2)),
    ([9], 136, 1025, 2, (False, 32, 4)),
    ([9], 136, 4097, 2, (False, 32, 8)),
    ([9], 136, 1024, 2, (False, 16, 4)),
    ([9], 136, 4096, 2, (False, 16, 8)),
    ([20], 136, 1024, 2, (False, 32, 4)),
    ([20], 136, 4096, 2, (False, 32, 8)),
    ([100], 2080, 4096, 2, (False, 64, 2)),
    ([40], 2080, 4096, 2, (False, 64, 4)),
    ([40], 136, 4096, 2, (False, 64, 8)),
    ([9], 136, 1024, 1, (False, 16, 2)),
    ([9], 4112, 4096, 1, (False, 16, 4)),
    ([9], 136, 4096, 1, (False, 16, 8)),
    ([20], 136, 1024, 1, (False, 32, 2)),
    ([20], 4112, 4096, 1, (False, 32, 4)),
    ([20], 136, 4096, 1, (False, 32, 8)),
    ([100], 2080, 4096, 1, (False, 64, 2)),
    ([40], 136, 4096, 1, (False, 64, 4)),
    ([40], 136, 8192, 1, (False, 64, 8)),
    ([9], 136, 1025, 1, (False, 32, 2)),
    ([9], 2080, 4097, 1, (False, 32, 4)),
    ([9], 136, 4097, 1, (False, 32, 8)),
]


@pytest.mark.parametrize("counts,n,k,esize,kernel", WIDTHS + SPLITS)
def test_tile_widths_and_split_sums(counts, n, k, esize, kernel):
    g = _gen(n + k + esize)
    rows, e = sum(counts), len(counts)
    assert products.variant(rows, e, n, k, esize=esize, aligned=k % (16 // esize) == 0) == kernel
    off, out = _offsets(counts), torch.empty(rows, n, device="cuda")
    x, w = _ints(g, rows, k), _ints(g, e, n, k)
    if esize == 1:
        one = torch.ones(e, max(n, rows), device="cuda")
        products.int8_matmul(x.to(torch.int8), one[0, :rows], w.to(torch.int8), one[:, :n].contiguous(), out, offsets=off,
                             stream=_stream())
    else:
        products.grouped_matmul(x, w, off, out, stream=_stream())
        # weights whose n axis is contiguous take the same kernels' other layout
        wt = _ints(g, e, k, n).transpose(1, 2)
        out2 = torch.empty_like(out)
        products.grouped_matmul(x, wt, off, out2, stream=_stream())
    at = 0
    for i, c in enumerate(counts):
        X = x[at:at + c].double()
        assert torch.equal(out[at:at + c].double(), X @ w[i].double().t())
        if esize == 2:
            assert torch.equal(out2[at:at + c].double(), X @ wt[i].double().t())
        at += c


@pytest.mark.parametrize("rows,n,k,split", [(2100, 72, 72, 2), (4100, 72, 72, 4), (9000, 72, 72, 8), (2100, 72, 71, 2),
                                            (4100, 71, 72, 4), (9001, 71, 71, 8), (20011, 264, 200, 8)])
def test_split_sums_of_dw_are_exact(rows, n, k, split):
    """Every row counts once: integers whose sums of any order are exact, some rows outside the group."""
    g = _gen(rows + n)
    aligned = n % 8 == 0 and k % 8 == 0
    assert products.variant(rows + 7, 1, n, k, dw=True, aligned=aligned) == (False, 128, split)
    dy, x = _ints(g, rows + 7, n), _ints(g, rows + 7, k)
    dy[:2], x[:2], dy[-5:], x[-5:] = float("nan"), float("inf"), float("inf"), float("nan")
    dw = torch.full((1, n, k), 7.0, device="cuda")
    products.grouped_matmul_dw(dy, x, torch.tensor([2, rows + 2], dtype=torch.int32, device="cuda"), dw, stream=_stream())
    assert torch.equal(dw[0].double(), dy[2:-5].double().t() @ x[2:-5].double())


def test_a_launch_of_more_than_two_seconds():
    """The blocks that end inside come last, in an expert of their own: what waits for them waits for
    the whole launch, 2.8e15 operations (2.9 s), and this is no failure."""
    n, rows, last = 73728, 256_000, 33
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 70 << 30:
        pytest.skip("needs 60 GB of device memory")
    assert rows % 64 == 0 and products.variant(rows + last, 2, n, n, dw=True) == (True, 256, 1)
    x = torch.empty(rows + last, n, dtype=BF16, device="cuda").random_(-3, 4, generator=_gen(51))
    dw = torch.empty(2, n, n, dtype=BF16, device="cuda")
    products.grouped_matmul_dw(x, x, _offsets([rows, last]), dw, stream=_stream())
    torch.cuda.synchronize()
    assert products.status(0) == 0
    for i, r in enumerate((slice(0, rows), slice(rows, rows + last))):
        for a, b in ((0, 0), (n - 64, 256), (4096, n - 64)):
            want = x[r, a:a + 64].double().t() @ x[r, b:b + 64].double()   # exact in f32, rounded once
            assert torch.equal(dw[i, a:a + 64, b:b + 64], want.float().to(BF16)), (i, a, b)
    del x, dw
    torch.cuda.empty_cache()


def _positive(g, *shape, dtype=BF16, scale=1.0):
    return (torch.rand(*shape, device="cuda", generator=g) * scale).to(dtype)


def _product64(a, b):
    """a.T @ b in 64 bits, some rows at a time."""
    out = torch.zeros(a.shape[1], b.shape[1], dtype=torch.float64, device="cuda")
    for i in range(0, a.shape[0], 16384):
        out += a[i:i + 16384].double().t() @ b[i:i + 16384].double()
    return out


def _assert_long_sum(got, want, terms):
    """A sum of ``terms`` products of one sign.  It is joined from parts of 768 terms (f32 outputs) or 8192, which
    lose at most a step (2^-23) of the sum for each term, in additions that lose at most half a step each;
    then it is rounded to the output's type."""
    part = 768 if got.dtype == F32 else 8192
    tol = (part + 2 + terms / part / 2) * 2.0 ** -23 * want + _half_step(got.dtype, want) * 1.01
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), (int(bad.sum()), ((got.double() - want) / want).abs().max().item())


# rows, n, k, kernel; the sums are n * k wide and as long as the rows
LONG_DW = [(262144, 256, 256, (False, 128, 8)), (262144, 256, 255, (False, 128, 8)), (65536, 1024, 1280, (True, 128, 1)),
           (65536, 1032, 2048, (True, 256, 1)), (262144, 1024, 1280, (True, 128, 1)), (65537, 1500, 1001, (False, 128, 1))]


@pytest.mark.parametrize("dtype,out_dtype", [(BF16, F32), (F16, F32), (BF16, BF16), (F16, F16)])
@pytest.mark.parametrize("rows,n,k,kernel", LONG_DW)
def test_long_sums_of_dw_keep_their_precision(rows, n, k, kernel, dtype, out_dtype):
    g = _gen(rows + k)
    assert products.variant(rows, 1, n, k, dw=True, aligned=n % 8 == 0 and k % 8 == 0) == kernel
    dy, x = _positive(g, rows, n, dtype=dtype, scale=0.25), _positive(g, rows, k, dtype=dtype, scale=0.25)
    dw = torch.empty(1, n, k, dtype=out_dtype, device="cuda")
    products.grouped_matmul_dw(dy, x, _offsets([rows]), dw, stream=_stream())
    _assert_long_sum(dw[0], _product64(dy, x), rows)


# rows, n, kernel of sums of 32768 terms, or 32769
LONG_FORWARD = [(300, 2048, 0, (False, 64, 1)), (2048, 2048, 0, (True, 256, 1)),
                (12, 20000, 0, (False, 16, 1)), (24, 20000, 0, (False, 32, 1)), (100, 20000, 0, (True, 128, 1)),
                (60, 20000, 0, (False, 128, 1)), (20, 300, 0, (False, 32, 8)), (100, 300, 0, (False, 64, 8)),
                (30, 5000, 1, (False, 32, 2)), (100, 9000, 1, (False, 64, 1)), (1700, 1100, 1, (False, 128, 1))]


@pytest.mark.parametrize("dtype,out_dtype", [(BF16, F32), (F16, F16)])
@pytest.mark.parametrize("other_axis", [False, True])
@pytest.mark.parametrize("rows,n,odd,kernel", LONG_FORWARD)
def test_long_sums_keep_their_precision(rows, n, odd, kernel, other_axis, dtype, out_dtype):
    g, k = _gen(rows + n), 32768 + odd
    assert products.variant(rows, 1, n, k, aligned=not odd) == kernel
    x = _positive(g, rows, k, dtype=dtype, scale=0.25)
    w = _positive(g, 1, k, n, dtype=dtype, scale=0.25).transpose(1, 2) if other_axis else _positive(g, 1, n, k, dtype=dtype, scale=0.25)
    out = torch.empty(rows, n, dtype=out_dtype, device="cuda")
    products.grouped_matmul(x, w, _offsets([rows]), out, stream=_stream())
    _assert_long_sum(out, _product64(x.t(), w[0].t()), k)


def test_segments_of_many_groups():
    """Sums of one segment, of several and of none follow one another on the same accumulators: exact integers."""
    g = _gen(61)
    counts, n, k = [768, 769, 0, 1023, 1536, 1537, 5, 4096, 4097, 9000, 0, 64], 776, 1032
    rows, e, off = sum(counts), len(counts), _offsets(counts)
    dy, x, w = _ints(g, rows, n), _ints(g, rows, k), _ints(g, e, n, k)
    assert products.variant(rows, e, n, k, dw=True)[0] and products.variant(rows, e, n, k)[0]
    dw, out, dx = torch.empty(e, n, k, device="cuda"), torch.empty(rows, n, device="cuda"), torch.empty(rows, k, device="cuda")
    products.grouped_matmul_dw(dy, x, off, dw, stream=_stream())
    products.grouped_matmul(x, w, off, out, stream=_stream())
    products.grouped_matmul(dy, w.transpose(1, 2), off, dx, stream=_stream())
    at = 0
    for i, c in enumerate(counts):
        D, X, W = dy[at:at + c].double(), x[at:at + c].double(), w[i].double()
        assert torch.equal(dw[i].double(), D.t() @ X), c
        assert torch.equal(out[at:at + c].double(), X @ W.t()) and torch.equal(dx[at:at + c].double(), D @ W), c
        at += c


def test_kernels_of_every_width_at_once():
    """Divided and joined sums of all tile widths on streams of their own: what they hold of an SM leaves
    room for the others, and none waits for good."""
    g = _gen(71)
    calls, checks = [], []
    for rows, n in ((9, 136), (20, 136), (9, 4112), (20, 4112), (40, 136), (100, 2080), (600, 2600), (2048, 2048)):
        k, s = 8192, torch.cuda.Stream()
        x, w, off, out = _ints(g, rows, k), _ints(g, 1, n, k), _offsets([rows]), torch.empty(rows, n, device="cuda")
        calls.append(products.bind_grouped_matmul(x, w, off, out, stream=s.cuda_stream))
        checks.append((out, x.double() @ w[0].double().t()))
    for rows, n, k in ((9000, 72, 72), (5000, 1032, 1032), (3000, 777, 129)):
        s = torch.cuda.Stream()
        dy, x, off, dw = _ints(g, rows, n), _ints(g, rows, k), _offsets([rows]), torch.empty(1, n, k, device="cuda")
        calls.append(products.bind_grouped_matmul_dw(dy, x, off, dw, stream=s.cuda_stream))
        checks.append((dw[0], dy.double().t() @ x.double()))
    torch.cuda.synchronize()
    for _ in range(30):
        for call in calls:
            call()
    torch.cuda.synchronize()
    for out, want in checks:
        assert torch.equal(out.double(), want)
