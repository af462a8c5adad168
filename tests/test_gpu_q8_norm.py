"""rms_norm_q8 / add_rms_norm_q8 against their definition in 64 bits.

Codes are whole numbers decided exactly: they have to be equal.  The stored sum
has to be the same bits.  The scale takes, beside exact steps, a sum of squares
in f32 and five rounded steps: its relative error is at most half the sum's
(the square root) plus 5 u, u = 2^-24.  A thread's chain is at most
max(32, cols / 256) terms and ten shuffles and joins follow."""
import pytest
import torch

import _q8
from oxide_b200 import _lib, ops

pytestmark = pytest.mark.gpu
EPS = 1e-5
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _inputs(dev, rows, cols, dtype, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed * 1000 + rows + cols)
    x, r = (torch.randn(rows, cols, generator=g, device=dev) * 3 for _ in range(2))
    w = torch.rand(cols, generator=g, device=dev) + 0.5
    return x.to(DT[dtype]), r.to(DT[dtype]), w.to(DT[dtype])


def _check(x, r, w, got, eps=EPS):
    h, codes, scale = _q8.norm_q8(x, r, w, eps)
    gh, gc, gs = got if r is not None else (None, *got)
    if r is not None:
        assert torch.equal(gh, h)
    assert gc.dtype == torch.int8 and gc.shape == x.shape and gs.shape == x.shape[:-1]
    bad = (gc != codes).nonzero()
    assert bad.numel() == 0, f"{len(bad)} codes differ, first at {bad[0].tolist()}"
    cols = x.shape[-1]
    tol = ((max(32, cols / 256) + 10) / 2 + 5) * 2.0 ** -24
    assert torch.equal(torch.isnan(gs), torch.isnan(scale))
    ok = ~torch.isnan(scale)
    err = (gs.double() - scale).abs()[ok]
    # below 2^-126 a scale is held with an absolute step of 2^-149
    lim = tol * scale[ok] + 2.0 ** -149
    assert bool((err <= lim).all()), float((err / lim).max())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 8), (9, 37), (1, 256), (17, 1000), (8, 1024), (5, 1032), (64, 4096),
                                       (2, 8200), (7, 16384), (3, 16385), (2, 40000)])
@pytest.mark.parametrize("residual", [False, True])
def test_against_definition(cuda, dtype, rows, cols, residual):
    x, r, w = _inputs(cuda, rows, cols, dtype)
    r = r if residual else None
    got = ops.rms_norm_q8(x, w, EPS) if r is None else ops.add_rms_norm_q8(x, r, w, EPS)
    _check(x, r, w, got)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [64, 2048, 65])
def test_exact_ties(cuda, dtype, cols):
    """Rows whose quotients are half-integers: 127 p / max|p| with max|p| = 127."""
    x = (torch.arange(6 * cols, device=cuda).view(6, cols) % 509 - 254).float() / 2
    x[:, 3] = torch.tensor([127, -127, 63.5, 254, 31.75, 127], device=cuda)
    x = x.clamp(-127, 127).to(DT[dtype])
    w = torch.full((cols,), 0.5, device=cuda).to(DT[dtype])
    _check(x, None, w, ops.rms_norm_q8(x, w, EPS))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [512, 4096, 77])
def test_extreme_rows(cuda, dtype, cols):
    """All zeros; the smallest and largest magnitudes; rows whose products or
    squares leave the range of f32; NaN and infinities, in x and in w."""
    x, _, w = _inputs(cuda, 12, cols, dtype, seed=3)
    x[0] = 0
    x[1] = 0
    x[1, 5] = 1.0
    for i, s in enumerate((1e-38, 1e-30, 1e18, 1e25, 3e37, 1e-41)):
        x[2 + i] = (x[2 + i].double().clamp(-8, 8) * s).to(x.dtype)
    x[9, 1] = float("nan")
    x[10, cols - 1] = float("inf")
    x[11, 0] = float("-inf")
    _check(x, None, w, ops.rms_norm_q8(x, w, EPS))
    big = (w.double() * 1e3).to(w.dtype)
    _check(x, None, big, ops.rms_norm_q8(x, big, EPS))
    w[7] = float("nan")
    _, scale = ops.rms_norm_q8(x, w, EPS)
    assert bool(torch.isnan(scale).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,cols", [(9000, 512), (5000, 515), (4000, 1024), (3000, 4096), (900, 5121), (700, 8191),
                                       (500, 9001), (300, 8192)])
def test_many_rows(cuda, dtype, residual, rows, cols):
    """Several rows in turn to a warp and a CTA, some with codes that the
    definition has to decide (every tenth f32 row at 4096 columns) and some not."""
    x, r, w = _inputs(cuda, rows, cols, dtype, seed=11)
    if residual:
        _check(x, r, w, ops.add_rms_norm_q8(x, r, w, EPS))
    else:
        _check(x, None, w, ops.rms_norm_q8(x, w, EPS))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [1024, 4096, 99])
def test_in_place_sum_and_given_outputs(cuda, dtype, cols):
    x, r, w = _inputs(cuda, 33, cols, dtype, seed=5)
    want = ops.add_rms_norm_q8(x, r, w, EPS)
    codes = torch.empty(33, cols, dtype=torch.int8, device=cuda)
    scale = torch.empty(33, device=cuda)
    for alias in (0, 1):
        a, b = x.clone(), r.clone()
        got = ops.add_rms_norm_q8(a, b, w, EPS, h=(a, b)[alias], out=codes, scale=scale)
        assert got[1] is codes and got[2] is scale
        assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_unaligned_and_large_counts(cuda, dtype):
    """Rows that start off a 16-byte boundary give the aligned call's result, and
    nothing is written behind the last row."""
    x, r, w = _inputs(cuda, 11, 264, dtype, seed=7)
    want = ops.add_rms_norm_q8(x, r, w, EPS)
    off = torch.zeros(11 * 264 + 1, dtype=x.dtype, device=cuda)
    off[1:] = x.reshape(-1)
    out = torch.full((11 * 264 + 9,), 99, dtype=torch.int8, device=cuda)
    sc = torch.full((12,), 7.0, device=cuda)
    h = torch.empty_like(x)
    ops.add_rms_norm_q8(off[1:].view(11, 264), r, w, EPS, h=h, out=out[1:1 + 11 * 264].view(11, 264),
                        scale=sc[:11])
    assert torch.equal(h, want[0]) and torch.equal(out[1:1 + 11 * 264].view(11, 264), want[1])
    # the unaligned call sums in another order
    assert bool(((sc[:11] - want[2]).abs() <= 64 * 2.0 ** -24 * want[2]).all())
    assert int(out[0]) == 99 and bool((out[1 + 11 * 264:] == 99).all()) and float(sc[11]) == 7.0


def test_leading_dims_empty_and_launch_failure(cuda):
    x, _, w = _inputs(cuda, 6, 128, "bf16")
    codes, scale = ops.rms_norm_q8(x.view(2, 3, 128), w, EPS)
    assert codes.shape == (2, 3, 128) and scale.shape == (2, 3)
    c, s = ops.rms_norm_q8(x[:0], w, EPS)
    assert c.shape == (0, 128) and s.shape == (0,)
    _lib.lib().oxide_debug_fail_next(b"oxide_rms_norm_q8_bf16")
    with pytest.raises(_lib.OxideError, match="injected"):
        ops.rms_norm_q8(x, w, EPS)


def test_other_stream_and_graph(cuda):
    x, r, w = _inputs(cuda, 40, 4096, "bf16", seed=9)
    want = ops.add_rms_norm_q8(x, r, w, EPS)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.add_rms_norm_q8(x, r, w, EPS)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    h, codes, scale = (torch.empty_like(t) for t in want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.add_rms_norm_q8(x, r, w, EPS, h=h, out=codes, scale=scale)
    x.copy_(r)
    graph.replay()
    torch.cuda.synchronize()
    _check(x, r, w, (h, codes, scale))


def _integer_codes(h, w):
    """nearest(127 p / max|p|), ties to even, of one row of f32 values, in whole
    numbers: products of two significands have 48 bits and do not fit f64's 127 p."""
    from fractions import Fraction
    p = [Fraction(a) * Fraction(b) for a, b in zip(h.tolist(), w.tolist())]
    top = max(abs(v) for v in p)
    return [round(127 * v / top) for v in p]  # round() of a Fraction takes ties to even


@pytest.mark.parametrize("cols", [64, 1024, 8192, 77, 4097, 17000])
@pytest.mark.parametrize("residual", [False, True])
def test_exact_ties_of_full_products(cuda, cols, residual):
    """f32 rows whose products fill 48 bits and whose quotients are half-integers:
    w the same everywhere, the largest h 254 a units and the others (2 n + 1) a,
    with an a of 16 bits, so 127 p / max|p| is n + 1/2.  Some elements stand a
    unit beside their tie.  Rows above and below the range of f32 products too."""
    g = torch.Generator().manual_seed(cols)
    scales = [1.0, 2.0 ** 60, 2.0 ** -70, 2.0 ** 40] * 3
    x = torch.zeros(len(scales), cols, dtype=torch.float64)
    w = (2 ** 23 + int(torch.randint(0, 2 ** 22, (1,), generator=g)) * 2 + 1) / 2.0 ** 23
    for i, s in enumerate(scales):
        a = int(torch.randint(2 ** 15, 2 ** 16, (1,), generator=g)) | 1
        n = torch.randint(-127, 127, (cols,), generator=g)
        u = (2 * n + 1) * a
        u[::7] += (n[::7] % 3) - 1
        u.clamp_(-254 * a, 254 * a)
        u[int(torch.randint(0, cols, (1,), generator=g))] = 254 * a
        x[i] = u.double() * s / 2.0 ** 22
    x, w = x.float(), torch.full((cols,), w, dtype=torch.float32)
    r = torch.zeros_like(x)
    if residual:
        codes = ops.add_rms_norm_q8(x.to(cuda), r.to(cuda), w.to(cuda), EPS)[1]
    else:
        codes = ops.rms_norm_q8(x.to(cuda), w.to(cuda), EPS)[0]
    for i in range(len(scales)):
        assert codes[i].tolist() == _integer_codes(x[i], w), i
