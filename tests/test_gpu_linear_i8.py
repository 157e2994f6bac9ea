"""The 8-bit linear path (csrc/rows_i8.cu, csrc/linear_i8.cu) against its formulas in 64 bits.

Tolerances follow from the arithmetic. U = 2^-24 is half an ulp of fp32. A statistic of d values is
summed in chains of at most d / 32 + 14 additions (32 threads a row at the least, then the trees), so
its relative error is below E(d) = (d / 32 + 16) U. A code is the rounding of t * (1 / u): t and u carry
at most 2 U and 3 U, so before rounding it is within 127 * 5 U of the exact quotient (plus what the
norm's statistics add).
"""
import math

import pytest
import torch

from streaming_sparse_b200 import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _e(d):
    return (d / 32 + 16) * U


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rows(seed, n, d, dtype, pad=0, spread=1.0):
    g = _gen(seed)
    x = torch.randn(n, d + pad, device=DEV, generator=g) * spread
    x *= 0.25 + 2 * torch.rand(n, 1, device=DEV, generator=g)
    return x.to(dtype)[:, :d]


def _check_codes(q, s, y, slack, s_tol):
    """q, s: the operator's; y: what the codes stand for, float64 [n, d]."""
    top = y.abs().amax(1)
    s64 = (top / 127).clamp_min(1e-30)
    assert q.dtype == torch.int8 and s.dtype == torch.float32
    assert ((s.double() - s64).abs() <= s_tol * s64 + 1e-37).all()
    exact = y / s64[:, None]
    assert ((q.double() - exact).abs() <= 0.5 + slack).all()
    full = top > 1e-20
    assert (q.abs().amax(1)[full] == 127).all()   # the largest value uses the whole range


SIZES = [(1, 1), (1, 1536), (3, 5), (7, 8960), (33, 1537), (129, 256), (65, 2048), (6, 5112), (5, 10240), (4, 16391), (3, 24576), (2, 40003), (1560, 1536)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d", SIZES)
def test_quant_rows(n, d, dtype):
    for pad in (0, 3, 16):
        x = _rows(n + d, n, d, dtype, pad)
        q, s = ops.quant_rows(x)
        assert q.shape == (n, d) and s.shape == (n,)
        _check_codes(q, s, x.double(), 127 * 3 * U, 2 * U)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d", SIZES)
def test_rms_norm_i8(n, d, dtype):
    for pad, residual in ((0, False), (3, True), (8, True)):
        x, w = _rows(n + d, n, d, dtype, pad), _rows(5, 1, d, dtype)[0]
        r = _rows(n + d + 1, n, d, dtype, pad, 0.5) if residual else None
        got = ops.rms_norm_i8(x, w, 1e-6, residual=r)
        assert len(got) == (3 if residual else 2)
        v = x.double()
        if residual:
            assert torch.equal(got[2], (x.float() + r.float()).to(dtype))
            v = v + r.double()
        y = v * w.double() * torch.rsqrt(v.square().mean(1, keepdim=True) + 1e-6)
        _check_codes(got[0], got[1], y, 127 * 5 * U, _e(d) / 2 + 8 * U)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d", SIZES)
def test_adaln_i8(n, d, dtype):
    if d < 5:
        return
    for pad, form, res in ((0, "mod", False), (3, "mod", True), (8, "affine", True), (0, "mod", "gate")):
        x, y = _rows(n + d, n, d, dtype, pad), _rows(n + d + 1, n, d, dtype, pad, 0.5)
        w, b = _rows(5, 1, d, dtype)[0], _rows(6, 1, d, dtype)[0]
        ft = max(1, n // 2)
        em = 0.3 * torch.randn(-(-n // ft), 3, d, device=DEV, generator=_gen(7))
        f = torch.arange(n, device=DEV) // ft
        kw = dict(weight=w, bias=b) if form == "affine" else dict(shift=em[:, 0], scale=em[:, 1], frame_tokens=ft)
        if res:
            kw["y"] = y
        if res == "gate":
            kw["gate"] = em[:, 2]
        got = ops.adaln_i8(x, eps=1e-6, **kw)
        v = x.double()
        if res:
            step = y.float() * em[f, 2] if res == "gate" else y.float()
            assert torch.equal(got[2], (x.float() + step).to(dtype))
            v = v + (y.double() * em[f, 2].double() if res == "gate" else y.double())
        z = v - v.mean(1, keepdim=True)
        z = z * torch.rsqrt(z.square().mean(1, keepdim=True) + 1e-6)
        o = z * w.double() + b.double() if form == "affine" else z * (1 + em[f, 1].double()) + em[f, 0].double()
        # an output's error, in units of the row's largest: the mean's (E times mean |v|, over the
        # deviation), the deviation's and a few roundings, each times |1 + scale| <= 3
        tol = 8 * _e(d) + 16 * U
        _check_codes(got[0], got[1], o, 127 * tol, tol)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [40, 1536, 1537, 2000, 8960, 20000, 30000])
def test_adaln_i8_affine_with_a_gated_addition(d, dtype):
    """The form between a block's self-attention and its cross-attention: LayerNorm(x + y gate[f]) w + b, its sum over x."""
    for n, ft, pad in ((1, 1, 0), (13, 5, 0), (24, 8, 3), (300, 100, 8)):
        x, y = _rows(n + d, n, d, dtype, pad), _rows(n + d + 1, n, d, dtype, pad, 0.5)
        w, b = _rows(5, 1, d, dtype)[0], _rows(6, 1, d, dtype)[0]
        em = 0.3 * torch.randn(-(-n // ft), 6, d, device=DEV, generator=_gen(8))
        f = torch.arange(n, device=DEV) // ft
        kw = dict(eps=1e-6, weight=w, bias=b, y=y, gate=em[:, 2], frame_tokens=ft)
        got = ops.adaln_i8(x, **kw)
        assert torch.equal(got[2], (x.float() + y.float() * em[f, 2]).to(dtype))
        v = x.double() + y.double() * em[f, 2].double()
        z = v - v.mean(1, keepdim=True)
        o = z * torch.rsqrt(z.square().mean(1, keepdim=True) + 1e-6) * w.double() + b.double()
        tol = 8 * _e(d) + 16 * U   # as in test_adaln_i8
        _check_codes(got[0], got[1], o, 127 * tol, tol)
        for over in ("x", "y"):
            to = (x if over == "x" else y).clone()
            again = ops.adaln_i8(to if over == "x" else x, **dict(kw, y=to if over == "y" else y), sum_out=to)
            assert again[2] is to and all(torch.equal(a, c) for a, c in zip(again, got))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [40, 1536, 1537, 2000, 8960, 20000, 30000])
def test_sum_without_an_addition(d, dtype):
    """The C entries store v also where there is nothing to add to x; past the row nothing is written."""
    from streaming_sparse_b200._lib import lib

    n, kind = 9, ops._I8_TYPES[dtype]
    x, w, b = _rows(1, n, d, dtype, 8), _rows(2, 1, d, dtype)[0], _rows(3, 1, d, dtype)[0]
    em = 0.3 * torch.randn(1, 2, d, device=DEV, generator=_gen(7))
    q, s = ops.rows_i8(n, d, DEV), torch.empty(n, device=DEV)
    st = torch.cuda.current_stream().cuda_stream
    to = (q.data_ptr(), q.stride(0), s.data_ptr(), st)
    for call, want in (
            (lambda v: lib().ss_rms_norm_i8(x.data_ptr(), d + 8, None, 0, kind, n, d, w.data_ptr(), 1e-6, v, d + 8, *to),
             ops.rms_norm_i8(x, w, 1e-6)),
            (lambda v: lib().ss_adaln_i8(x.data_ptr(), d + 8, None, 0, None, 0, kind, n, d, 0, None, None, 0, w.data_ptr(),
                                         b.data_ptr(), 1e-6, v, d + 8, *to), ops.adaln_i8(x, eps=1e-6, weight=w, bias=b)),
            (lambda v: lib().ss_adaln_i8(x.data_ptr(), d + 8, None, 0, None, 0, kind, n, d, n, em.data_ptr(),
                                         em[:, 1].data_ptr(), d, None, None, 1e-6, v, d + 8, *to),
             ops.adaln_i8(x, eps=1e-6, shift=em[:, 0], scale=em[:, 1], frame_tokens=n))):
        v = torch.full((n, d + 8), 3.0, dtype=dtype, device=DEV)
        assert call(v.data_ptr()) == 0
        assert torch.equal(v[:, :d], x) and (v[:, d:] == 3).all()
        assert torch.equal(q, want[0]) and torch.equal(s, want[1])


def test_sum_written_over_an_input():
    for which in ("x", "residual"):
        x, r, w = _rows(1, 50, 1536, torch.bfloat16), _rows(2, 50, 1536, torch.bfloat16), _rows(3, 1, 1536, torch.bfloat16)[0]
        q0, s0, v0 = ops.rms_norm_i8(x, w, 1e-6, residual=r)
        to = x if which == "x" else r
        q1, s1, v1 = ops.rms_norm_i8(x, w, 1e-6, residual=r, sum_out=to)
        assert v1 is to and torch.equal(v0, v1) and torch.equal(q0, q1) and torch.equal(s0, s1)
    for d in (1536, 1537):
        x, y = _rows(1, 50, d, torch.bfloat16), _rows(2, 50, d, torch.bfloat16)
        w, b = _rows(3, 1, d, torch.bfloat16)[0], _rows(4, 1, d, torch.bfloat16)[0]
        q0, s0, v0 = ops.adaln_i8(x, eps=1e-6, weight=w, bias=b, y=y)
        q1, s1, v1 = ops.adaln_i8(x, eps=1e-6, weight=w, bias=b, y=y, sum_out=x)
        assert v1 is x and torch.equal(v0, v1) and torch.equal(q0, q1) and torch.equal(s0, s1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [40, 1400, 1700, 2000, 5000, 8968, 20000, 24584])
def test_sum_written_over_an_input_at_widths_that_leave_threads_idle(d, dtype):
    """Threads past the row's end must not see the sum that others store over the inputs: with equal
    signs a value that is added twice would be the row's largest."""
    n = 400
    x, r, w = _rows(1, n, d, dtype).abs(), _rows(2, n, d, dtype).abs(), torch.ones(d, dtype=dtype, device=DEV)
    b = torch.zeros_like(w)
    x[:, -8:] += 30
    em = torch.zeros(1, d, device=DEV)
    for call in (lambda **kw: ops.rms_norm_i8(kw["a"], w, 1e-6, residual=kw["b"], sum_out=kw.get("to")),
                 lambda **kw: ops.adaln_i8(kw["a"], eps=1e-6, weight=w, bias=b, y=kw["b"], sum_out=kw.get("to")),
                 lambda **kw: ops.adaln_i8(kw["a"], eps=1e-6, shift=em, scale=em, frame_tokens=n, y=kw["b"],
                                           gate=em + 1, sum_out=kw.get("to"))):
        ref = call(a=x, b=r)
        for over in ("a", "b"):
            for _ in range(3):
                kw = dict(a=x.clone(), b=r.clone())
                got = call(**kw, to=kw[over])
                assert all(torch.equal(g, t) for g, t in zip(got, ref))


@pytest.mark.parametrize("d", [64, 1536, 1537, 8960, 40000])
def test_rows_of_zeros_tiny_and_not_finite(d):
    x = _rows(9, 8, d, torch.float32)
    x[0] = 0
    x[1, d // 2] = math.inf
    x[2, d - 1] = math.nan
    x[3, 0] = -math.inf
    x[4] = 1e-36
    x[5] *= 1e-20
    q, s = ops.quant_rows(x)
    assert s[0] == torch.tensor(1e-30) and not q[0].any()
    for r in (1, 2, 3):
        assert s[r].isnan() and not q[r].any()
    assert s[4] == torch.tensor(1e-30) and not q[4].any()
    _check_codes(q[5:], s[5:], x[5:].double(), 127 * 3 * U, 2 * U)
    w, b = torch.ones(d, device=DEV), torch.zeros(d, device=DEV)
    for got in (ops.rms_norm_i8(x, w, 1e-6), ops.adaln_i8(x, eps=1e-6, weight=w, bias=b)):
        assert not got[0][:4].any() and got[1][1:4].isnan().all() and got[1][0].isfinite()
        assert got[1][4:].isfinite().all() and (got[0][6:].abs().amax(1) == 127).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [64, 1000, 1536, 1537, 2048, 8960, 20000, 40000])
def test_rows_whose_squares_overflow(d, dtype):
    """Finite rows whose sum of squares is no fp32 number count as not finite; their neighbours are what they were."""
    x, w, b = _rows(9, 6, d, dtype), _rows(2, 1, d, dtype)[0], _rows(3, 1, d, dtype)[0]
    em = 0.3 * torch.randn(1, 2, d, device=DEV, generator=_gen(7))
    big = x.clone()
    big[1] *= 1e20
    big[3, d // 2] = 3e19
    big[4, d - 1] = -1e38
    keep = torch.tensor([0, 2, 5], device=DEV)
    for f in (lambda v, **kw: ops.rms_norm_i8(v, w, 1e-6, **kw),
              lambda v, residual=None: ops.adaln_i8(v, eps=1e-6, weight=w, bias=b, y=residual),
              lambda v, residual=None: ops.adaln_i8(v, eps=1e-6, shift=em[:, 0], scale=em[:, 1], frame_tokens=6, y=residual)):
        for kw in ({}, dict(residual=torch.zeros_like(x))):
            ref, got = f(x, **kw), f(big, **kw)
            assert got[1][[1, 3, 4]].isnan().all() and not got[0][[1, 3, 4]].any()
            assert torch.equal(got[0][keep], ref[0][keep]) and torch.equal(got[1][keep], ref[1][keep])
    # the largest power of two whose d squares sum to less than 2^127 is no overflow
    x[1] = 2.0 ** int((126.99 - math.log2(d)) / 2)
    got = ops.rms_norm_i8(x, torch.ones_like(w), 1e-6)
    assert (got[0][1] == 127).all() and got[1].isfinite().all()


def _linear64(x, xs, w, ws, bias, gelu):
    acc = x.double() @ w.double().t()                      # exact: below 2^53
    scaled = acc * xs.double()[:, None] * ws.double()[None, :]
    v = scaled if bias is None else scaled + bias.double()
    size = scaled.abs() + (0 if bias is None else bias.double().abs())
    tol = 4 * U * size
    if gelu:
        u2 = math.sqrt(8 / math.pi) * (v + 0.044715 * v ** 3)
        v = v / (1 + torch.exp(-u2))
        # 1.13 is GELU's steepest slope; the exponential is a few ulp and carries its argument's error
        tol = 1.13 * tol + v.abs() * (16 * U + 8 * U * u2.abs())
    return v, tol


def _between(got, ref, tol):
    """got is the one rounding to its type of an fp32 value within tol of ref (rounding is monotone)."""
    lo, hi = (ref - tol).to(got.dtype), (ref + tol).to(got.dtype)
    assert ((lo <= got) & (got <= hi)).all(), ((got.double() - ref).abs() / tol).max().item()


def _codes(seed, n, k, top=127):
    g = _gen(seed)
    q = ops.rows_i8(n, k, DEV)
    q.copy_(torch.randint(-top, top + 1, (n, k), device=DEV, generator=g))
    return q, 0.01 + torch.rand(n, device=DEV, generator=g) / 20


def _check_linear(M, N, K, out_dtype, bias_dtype, gelu, seed=0, **kw):
    x, xs = _codes(seed + 1, M, K)
    w, ws = _codes(seed + 2, N, K)
    ws = ws / math.sqrt(K) / 30
    b = None if bias_dtype is None else torch.randn(N, device=DEV, generator=_gen(3)).to(bias_dtype)
    got = ops.linear_i8(x, xs, w, ws, bias=b, gelu=gelu, out_dtype=out_dtype, validate=True, **kw)
    ref, tol = _linear64(x, xs, w, ws, b, gelu)
    assert got.shape == (M, N) and got.dtype == out_dtype
    _between(got, ref, tol)
    return x, xs, w, ws, b, got


@pytest.mark.parametrize("M", [1, 2, 3, 7, 8, 9, 16, 17, 31, 64, 77, 128, 129, 200, 257, 300])
@pytest.mark.parametrize("N,K", [(1, 1), (5, 3), (64, 64), (1531, 1549), (1536, 1536), (130, 8960), (4608, 128),
                                 (257, 129)])
def test_linear_i8_small(M, N, K):
    i = M + N + K
    _check_linear(M, N, K, TYPES[i % 3], [None, *TYPES][i % 4], i % 2 == 1, seed=i)


@pytest.mark.parametrize("M", [3, 4, 5, 6])
@pytest.mark.parametrize("N,K", [(1, 1), (5, 3), (64, 64), (1531, 1549), (1536, 1536), (130, 8960), (333, 65000)])
def test_linear_i8_on_both_sides_of_the_dot_products(M, N, K):
    """Four tokens are the most of the dot-product kernel; five go to the tensor cores."""
    for i, dtype in enumerate(TYPES):
        x, xs, w, ws, b, got = _check_linear(M, N, K, dtype, [None, *TYPES][(i + M) % 4], (i + M) % 2 == 1, seed=M + i)
        xs = xs.clone()
        xs[M - 1] = math.nan
        again = ops.linear_i8(x, xs, w, ws, bias=b, gelu=(i + M) % 2 == 1, out_dtype=dtype)
        assert again[M - 1].isnan().all() and torch.equal(again[:M - 1], got[:M - 1])


@pytest.mark.parametrize("out_dtype", TYPES)
@pytest.mark.parametrize("bias_dtype", [None, *TYPES])
@pytest.mark.parametrize("gelu", [False, True])
@pytest.mark.parametrize("M", [1, 40, 700])
def test_linear_i8_types(M, out_dtype, bias_dtype, gelu):
    _check_linear(M, 333, 272, out_dtype, bias_dtype, gelu)


@pytest.mark.parametrize("M,N,K", [(4680, 1536, 1536), (4680, 4608, 1536), (1560, 8960, 1536), (4680, 1536, 8960),
                                   (4681, 1543, 1000), (2049, 257, 65), (1000, 64, 12345), (20000, 16, 48),
                                   (5, 20000, 33), (70000, 130, 17)])
def test_linear_i8_large(M, N, K):
    _check_linear(M, N, K, torch.bfloat16, torch.bfloat16, K == 1536)
    _check_linear(M, N, K, torch.float32, None, False)


def test_linear_i8_sums_are_exact():
    """All products of one sign at the largest codes: sums near 2^31 stay exact, the whole int8 range counts."""
    for M in (1, 40, 300):
        K = ops.LINEAR_I8_MAX_K
        x, w = ops.rows_i8(M, K, DEV), ops.rows_i8(40, K, DEV)
        x.fill_(-128)
        w.fill_(-128)
        w[1::2] = 127
        one = torch.ones(max(M, 40), device=DEV)
        got = ops.linear_i8(x, one[:M], w, one[:40], out_dtype=torch.float32)
        assert (got[:, 0::2] == torch.tensor(128 * 128 * K).float().item()).all()
        assert (got[:, 1::2] == torch.tensor(-127 * 128 * K).float().item()).all()


def test_linear_i8_strides_and_buffers():
    for M in (3, 50, 1100):
        N, K = 200, 300
        bx = torch.full((M, 352), 77, dtype=torch.int8, device=DEV)
        bw = torch.full((N, 400), -77, dtype=torch.int8, device=DEV)
        x, w = bx[:, 16:16 + K], bw[:, 32:32 + K]
        x.copy_(_codes(1, M, K)[0])
        w.copy_(_codes(2, N, K)[0])
        xs, ws = _codes(3, M, 4)[1], _codes(4, N, 4)[1] / 400
        for dtype in TYPES:
            buf = torch.full((M + 2, N + 7), 5.0, dtype=dtype, device=DEV)
            out = buf[1:M + 1, 3:3 + N]
            assert ops.linear_i8(x, xs, w, ws, out=out) is out
            ref = ops.linear_i8(x.contiguous() if K % 16 == 0 else ops.rows_i8(M, K, DEV).copy_(x), xs, w, ws, out_dtype=dtype)
            assert torch.equal(out, ref)
            buf[1:M + 1, 3:3 + N] = 5.0
            assert (buf == 5.0).all()              # nothing outside the rows was written
            r, tol = _linear64(x, xs, w, ws, None, False)
            _between(ref, r, tol)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [2, 40, 300, 2000])
def test_linear_i8_writes_nothing_past_its_columns(M, dtype):
    """Rows that start at 16 bytes and end inside 16 bytes, at a tile's end and inside one."""
    for N in (128, 130, 133, 250, 257, 1531, 1539):
        x, xs = _codes(1, M, 200)
        w, ws = _codes(2, N, 200)
        ref = ops.linear_i8(x, xs, w, ws / 300, out_dtype=dtype)
        for off in (0, 8, 1):
            buf = torch.full((M + 1, -(-N // 8) * 8 + 16), 7.0, device=DEV, dtype=dtype)
            out = buf[:M, off:off + N]
            assert torch.equal(ops.linear_i8(x, xs, w, ws / 300, out=out), ref)
            out.fill_(7.0)
            assert (buf == 7.0).all(), (N, off)


@pytest.mark.parametrize("M", [1, 6, 20, 130, 2000])
def test_linear_i8_not_finite_rows(M):
    x, xs, w, ws, b, ref = _check_linear(M, 500, 600, torch.bfloat16, torch.bfloat16, False)
    xs = xs.clone()
    xs[M // 2] = math.nan
    ws = ws.clone()
    ws[7] = math.inf
    got = ops.linear_i8(x, xs, w, ws, bias=b)
    assert got[M // 2].isnan().all()
    keep = torch.ones(M, dtype=torch.bool, device=DEV)
    keep[M // 2] = False
    cols = torch.arange(500, device=DEV) != 7
    assert torch.equal(got[keep][:, cols], ref[keep][:, cols])
    assert not got[keep][:, 7].isfinite().any()


def test_no_rows():
    x = torch.empty(0, 64, dtype=torch.bfloat16, device=DEV)
    q, s = ops.quant_rows(x)
    assert q.shape == (0, 64) and s.shape == (0,)
    w, ws = _codes(1, 32, 64)
    assert ops.linear_i8(q, s, w, ws).shape == (0, 32)
    q, s, v = ops.rms_norm_i8(x, torch.ones(64, dtype=torch.bfloat16, device=DEV), 1e-6, residual=x)
    assert q.shape == v.shape == (0, 64)


def test_offsets_past_32_bits():
    n, d, ld = 520, 40, 1 << 22                       # 520 * 2^22 > 2^31 elements
    x = torch.empty(n * ld, dtype=torch.bfloat16, device=DEV).as_strided((n, d), (ld, 1))
    x.copy_(_rows(1, n, d, torch.bfloat16))
    q, s = ops.quant_rows(x)
    q2, s2 = ops.quant_rows(x.contiguous())
    assert torch.equal(q, q2) and torch.equal(s, s2)
    del x
    M, N, K = 270000, 8192, 32                        # 2.2e9 outputs
    x, xs = _codes(1, M, K)
    w, ws = _codes(2, N, K)
    out = ops.linear_i8(x, xs, w, ws)
    for r in (0, 131071, 262144, M - 1):
        assert torch.equal(out[r:r + 1], ops.linear_i8(x[r:r + 1], xs[r:r + 1], w, ws))


def test_a_frame_longer_than_32_bits():
    x = _rows(1, 6, 64, torch.bfloat16)
    em = 0.3 * torch.randn(1, 2, 64, device=DEV, generator=_gen(7))
    kw = dict(eps=1e-6, shift=em[:, 0], scale=em[:, 1])
    for ft in (2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 1):
        assert all(torch.equal(a, b) for a, b in zip(ops.adaln_i8(x, frame_tokens=ft, **kw),
                                                     ops.adaln_i8(x, frame_tokens=6, **kw)))


def test_the_longest_row():
    """2^31 - 1 values: the steps past the row's end pass 2^31."""
    d = 2 ** 31 - 1
    x = torch.zeros(1, d, dtype=torch.bfloat16, device=DEV)
    at = torch.tensor([0, 2 ** 30, d - 511, d - 2, d - 1], device=DEV)
    codes = torch.tensor([1, -2, 50, 3, -127], dtype=torch.int8, device=DEV)
    x[0, at] = codes.bfloat16()
    q, s = ops.quant_rows(x)
    assert s.item() == 1.0 and torch.equal(q[0, at], codes)
    q[0, at] = 0
    assert not any(part.any() for part in q[0].split(1 << 28))


def test_same_bits_every_time_other_streams_and_graphs():
    x, r, w = _rows(1, 300, 1536, torch.bfloat16), _rows(2, 300, 1536, torch.bfloat16), _rows(3, 1, 1536, torch.bfloat16)[0]
    wq, ws = ops.quant_rows(_rows(4, 520, 1536, torch.bfloat16))

    def step(rows):
        q, s, v = ops.rms_norm_i8(x[:rows], w, 1e-6, residual=r[:rows])
        return ops.linear_i8(q, s, wq, ws, gelu=True), v

    for rows in (1, 5, 60, 300):
        ref = step(rows)
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            got = step(rows)
        st.synchronize()
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = step(rows)
        for _ in range(3):
            got[0].zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


def test_refusals():
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device=DEV)
    w = torch.zeros(64, dtype=torch.bfloat16, device=DEV)
    q, s = ops.quant_rows(x)
    bad = [
        lambda: ops.quant_rows(x.int()),
        lambda: ops.quant_rows(x[0]),
        lambda: ops.quant_rows(x.cpu()),
        lambda: ops.quant_rows(x.t()),
        lambda: ops.quant_rows(x[:1].expand(4, 64)),                      # rows that overlap
        lambda: ops.quant_rows(torch.zeros(4, 0, device=DEV)),
        lambda: ops.quant_rows(x, out=torch.zeros(4, 63, dtype=torch.int8, device=DEV)),
        lambda: ops.quant_rows(x, scales=torch.zeros(5, device=DEV)),
        lambda: ops.quant_rows(x.float().requires_grad_()),
        lambda: ops.rms_norm_i8(x, w.float(), 1e-6),
        lambda: ops.rms_norm_i8(x, w[:32], 1e-6),
        lambda: ops.rms_norm_i8(x, w, 1e-6, residual=x[:3]),
        lambda: ops.rms_norm_i8(x, w, 1e-6, residual=x.float()),
        lambda: ops.rms_norm_i8(x, w, 1e-6, sum_out=x),                   # a sum without a residual
        lambda: ops.adaln_i8(x, eps=1e-6),
        lambda: ops.adaln_i8(x, eps=1e-6, weight=w),
        lambda: ops.adaln_i8(x, eps=1e-6, weight=w, bias=w, shift=w[None].float(), scale=w[None].float()),
        lambda: ops.adaln_i8(x, eps=1e-6, shift=w[None].float(), scale=w[None].float(), frame_tokens=3),
        lambda: ops.adaln_i8(x, eps=1e-6, shift=w[None].float(), scale=w[None].float()),
        lambda: ops.adaln_i8(x, eps=1e-6, shift=w[None], scale=w[None], frame_tokens=4),
        lambda: ops.adaln_i8(x, eps=1e-6, weight=w, bias=w, gate=w[None].float(), frame_tokens=4),
        lambda: ops.linear_i8(q, s, q[:, :32], s),
        lambda: ops.linear_i8(q.float(), s, q, s),
        lambda: ops.linear_i8(q, s.double(), q, s),
        lambda: ops.linear_i8(q, s[:3], q, s),
        lambda: ops.linear_i8(q, s, q[:0], s[:0]),
        lambda: ops.linear_i8(q[:, 1:49], s, q[:, :48], s),               # rows off 16 bytes
        lambda: ops.linear_i8(torch.zeros(4, 33, dtype=torch.int8, device=DEV), s,
                              torch.zeros(4, 33, dtype=torch.int8, device=DEV), s),
        lambda: ops.linear_i8(q, s, q, s, bias=torch.zeros(4, dtype=torch.int32, device=DEV)),
        lambda: ops.linear_i8(q, s, q, s, bias=torch.zeros(3, device=DEV)),
        lambda: ops.linear_i8(q, s, q, s, out_dtype=torch.int32),
        lambda: ops.linear_i8(q, s, q, s, out=torch.zeros(4, 5, device=DEV)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was not refused")
