"""The dense operators on the GPU (run with -m gpu on a B200) against plain statements in 64 bits.

Tolerances are sums of the roundings each formula makes, written beside it; U = 2^-24 is half a step of f32, HALF[t] half a
step of the output type.  Integers (int8 values, and so the products' sums) are compared exactly.  __expf is off by at
most 2 + 1.173 |x| steps of f32, __fdividef and rsqrtf by 2."""
import math

import pytest
import torch

import okc_muse_kernels_b200 as okc
from okc_muse_kernels_b200 import synth

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: U}
TINY = 2.0 ** -120


def _gen(seed):
    assert torch.cuda.is_available(), "these tests need a CUDA device"
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(shape, g, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _quant_ref(x):
    """The definition of quantize_rows.  The quotients are made in 64 bits and rounded to f32 (53 bits are more than twice
    24 and two, so this is the f32 quotient), and so is the product (exact in 64 bits)."""
    x = x.double()
    peak = x.abs().amax(dim=1)
    ok = torch.isfinite(peak) & (peak >= TINY)
    steps = torch.full_like(peak, 127)
    inv = torch.where(ok, steps / peak, 0.0).float().double()
    q = torch.where(ok[:, None], torch.round((x * inv[:, None]).float()), 0.0).to(torch.int8)
    scale = torch.where(ok, peak / steps, 0.0).float()
    return q, torch.where(torch.isfinite(peak), scale, float("nan"))


def _int_sum(q, w):
    return q.double() @ w.double().t()             # exact: below 2^53


def _close(got, ref, tol, what):
    got, ref = got.double(), ref.double()
    assert got.shape == ref.shape, what
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{what}: NaN in other places"
    fine = ~torch.isnan(ref)
    off = ((got - ref).abs() - tol)[fine]
    assert off.numel() == 0 or off.max() <= 0, f"{what}: {off.max().item():.3g} beyond the tolerance"


def _weight(rows, cols, g):
    q = torch.randint(-127, 128, (rows, cols), generator=g, device="cuda", dtype=torch.int8)
    return okc.int8_rows(q, torch.rand(rows, generator=g, device="cuda") * 1e-2 + 1e-4)


def _linear_ref(q, scale, w, bias, dtype):
    """(values, tolerance): the sum's conversion, the two products and the bias add round once each, then the type."""
    y0 = _int_sum(q, w.q) * (scale.double()[:, None] * w.scale.double()[None, :])
    y = y0 if bias is None else y0 + bias.double()
    tol = 3.01 * U * y0.abs() + (0 if bias is None else 1.01 * U * y.abs() + 3.01 * U * y0.abs() * U)
    return y, tol + (HALF[dtype] if dtype is torch.bfloat16 else 0) * (y.abs() + tol) + 1e-37


def _gated_ref(q, scale, w, dtype):
    """g and u are off by 3 U relative (see _linear_ref); g / (1 + e^-g) multiplies g's error by 1 + |g| at most; e^-g is off
    by (2 + 1.173 |g|) * 2 U, the sum 1 + e^-g rounds (U), the division is off by 4 U, the product by U.  Below
    e^-g = 2^126 the division gives 0 for less than 2^-119."""
    y = _int_sum(q, w.q) * (scale.double()[:, None] * w.scale.double()[None, :])
    n = w.q.shape[0] // 2
    g, u = y[:, :n], y[:, n:]
    h = torch.special.expit(g) * g * u
    rel = U * (3 * (1 + g.abs()) + 2 * (2 + 1.173 * g.abs()) + 1 + 4 + 1 + 3) * 1.01
    tol = rel * h.abs() + 2.0 ** -119 * (1 + u.abs())
    return h, tol + (HALF[dtype] if dtype is torch.bfloat16 else 0) * (h.abs() + tol) + 1e-37


# ------------------------------------------------------------------------------------------------ quantize_rows
@pytest.mark.parametrize("R,cols", [(1, 1), (3, 7), (2, 16), (5, 1000), (33, 4096), (2, 16385), (400, 2880), (301, 9000), (2, 131071), (7, 131064),
                                    (593, 8), (595, 1016), (600, 2048), (700, 4088), (601, 8192), (599, 8200), (600, 1001), (640, 8185), (640, 8186), (700, 3), (600, 4089), (593, 250), (601, 257)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_rows_is_exact(R, cols, dtype):
    x = _randn((R, cols), _gen(R * cols), dtype)
    got = okc.quantize_rows(x)
    q, scale = _quant_ref(x)
    assert torch.equal(got.q, q) and torch.equal(got.scale, scale)
    assert got.q.stride(0) % 16 == 0 or R == 1


@pytest.mark.parametrize("rows,dtype", [(12, torch.float32), (12, torch.bfloat16), (700, torch.bfloat16)])
def test_quantize_rows_special_rows(rows, dtype):
    x = torch.randn((rows, 40), device="cuda").to(dtype)
    x[1] = 0
    x[2, 5] = float("inf")
    x[3, 39] = float("-inf")
    x[4, 0] = float("nan")
    x[5] *= 2.0 ** -130 / x[5].abs().max()            # below 2^-120: zeros
    x[6] = x[6] / x[6].abs().max() * 2.0 ** -119      # above
    x[7] = x[7] / x[7].abs().max() * 3.3e38           # near the largest values
    x[8, :] = 254.0                                   # multiplier 1/2: halves ...
    x[8, 1:5] = torch.tensor([1.0, 3.0, 5.0, -7.0])   # ... go to the even neighbour
    x[9, 3] = float("nan")
    x[9, 4] = float("inf")
    got = okc.quantize_rows(x)
    q, scale = _quant_ref(x)
    assert torch.equal(got.q, q)
    assert torch.equal(got.scale.isnan(), scale.isnan()) and got.scale.isnan().tolist() == [i in (2, 3, 4, 9) for i in range(rows)]
    assert torch.equal(got.scale.nan_to_num(), scale.nan_to_num())
    assert q[8, 1:5].tolist() == [0, 2, 2, -4] and not q[5].any() and q[6].any()


def test_quantize_rows_strided_and_unaligned_input():
    g = _gen(5)
    many = _randn((700, 301), g, torch.bfloat16)
    wide = _randn((6, 301), g)
    for x in (many, many[:, 3:200], many[1:, 1:], many[::1, 8:136], many[5:, 7:8], many[:, :296], wide[:, 3:200], wide[::2, :100], wide.t(), wide[1:, 1:2], wide.bfloat16()[:, 8:136], wide[0:1, 5:]):
        got = okc.quantize_rows(x)
        q, scale = _quant_ref(x)
        assert torch.equal(got.q, q) and torch.equal(got.scale, scale)
    assert okc.quantize_rows(wide[:0]).q.shape == (0, 301)


# ------------------------------------------------------------------------------------------------ products
SHAPES = [(1, 1, 1), (1, 16384, 40), (1, 16385, 9), (1, 9001, 1200), (1, 520, 3001), (1, 64, 160000), (1, 16384, 1500), (1, 5000, 9000), (1, 2048, 20000), (1, 300, 700), (1, 12000, 2960), (2, 520, 3001), (1, 16, 5), (2, 511, 130), (3, 513, 7), (5, 1000, 301), (8, 4100, 149), (1, 20000, 33), (4, 16400, 64),
          (9, 1, 1), (9, 128, 128), (16, 129, 127), (17, 1000, 301), (40, 4096, 640), (65, 333, 1000), (130, 2048, 257), (256, 520, 384),
          (257, 17, 3), (257, 128, 256), (300, 1000, 301), (513, 2047, 129), (1025, 640, 2050)]


@pytest.mark.parametrize("T,K,N", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_int8_linear(T, K, N, dtype):
    g = _gen(T + K + N)
    x, w = _randn((T, K), g, dtype), _weight(N, K, g)
    bias = _randn(N, g)
    q, scale = _quant_ref(x)
    for b in (None, bias):
        for out_f32 in (False, True):
            y = okc.int8_linear(x, w, bias=b, out_f32=out_f32)
            assert y.dtype == (torch.float32 if out_f32 else torch.bfloat16)
            _close(y, *_linear_ref(q, scale, w, b, y.dtype), f"bias {b is not None} f32 {out_f32}")
            assert torch.equal(y, okc.int8_linear(okc.quantize_rows(x), w, bias=b, out_f32=out_f32)), "int8 tokens"
    assert okc.dense_status() == (0, 0)


@pytest.mark.parametrize("T,K,N", SHAPES)
def test_int8_gated(T, K, N):
    g = _gen(T + K + N + 1)
    x, w = _randn((T, K), g, torch.bfloat16), _weight(2 * N, K, g)
    w = okc.QuantRows(w.q, w.scale * (40.0 / math.sqrt(K)))          # sums of some size: both tails of the sigmoid
    q, scale = _quant_ref(x)
    for out_f32 in (False, True):
        h = okc.int8_gated(x, w, out_f32=out_f32)
        _close(h, *_gated_ref(q, scale, w, h.dtype), f"f32 {out_f32}")
    assert torch.equal(h, okc.int8_gated(okc.quantize_rows(x), w, out_f32=True))
    assert okc.dense_status() == (0, 0)


@pytest.mark.parametrize("T,K,N", [(7, 7168, 2048), (40, 7168, 2040), (31, 4096, 2560), (100, 2304, 2568), (33, 16512, 130), (9, 2944, 4100),
                                   (16, 1408, 520), (200, 512, 1536), (250, 384, 600), (130, 1152, 9601), (2, 131068 // 128 * 128, 24)])
def test_products_of_several_k_blocks_a_copy(T, K, N):
    """K of whole blocks of 128, in stages of different lengths; weight and token rows with other values behind their columns."""
    g = _gen(T + K + N + 2)
    wide = torch.randint(-127, 128, (2 * N, K + 144), generator=g, device="cuda", dtype=torch.int8)
    x = okc.QuantRows(torch.randint(-127, 128, (T, K + 16), generator=g, device="cuda", dtype=torch.int8)[:, :K],
                      torch.rand(T, generator=g, device="cuda") * 1e-2 + 1e-4)
    scale = torch.rand(2 * N, generator=g, device="cuda") * (0.2 / math.sqrt(K))
    w, both = okc.QuantRows(wide[:N, :K], scale[:N]), okc.QuantRows(wide[:, :K], scale)
    for out_f32 in (False, True):
        y, h = okc.int8_linear(x, w, out_f32=out_f32), okc.int8_gated(x, both, out_f32=out_f32)
        _close(y, *_linear_ref(x.q, x.scale, w, None, y.dtype), f"linear f32 {out_f32}")
        _close(h, *_gated_ref(x.q, x.scale, both, h.dtype), f"gated f32 {out_f32}")
    store = torch.full((T + 1, N + 5), 7.0, device="cuda")
    okc.int8_linear(x, w, out_f32=True, out=store[:T, 3:3 + N])
    assert torch.equal(store[:T, 3:3 + N], y) and (store[T] == 7).all() and (store[:, :3] == 7).all() and (store[:, 3 + N:] == 7).all()
    assert okc.dense_status() == (0, 0)


def test_gated_far_tails():
    """Gate values of thousands: silu is g or 0, never NaN."""
    for T in (2, 20, 300):
        x = torch.ones((T, 64), device="cuda")
        x[1::2] = -1
        w = okc.int8_rows(torch.full((32, 64), 127, dtype=torch.int8, device="cuda"), torch.ones(32, device="cuda"))
        h = okc.int8_gated(x, w, out_f32=True)
        q, scale = _quant_ref(x)
        _close(h, *_gated_ref(q, scale, w, torch.float32), f"T {T}")
        assert torch.isfinite(h).all() and (h[1::2] == 0).all() and (h[0::2] > 1e6).all()


@pytest.mark.parametrize("T", [1, 3, 40, 300])
def test_longest_sums_stay_in_32_bits(T):
    """Every product 127 * 127 (and -128 * -128 of rows made elsewhere) over the longest K."""
    K = 131071
    ones = torch.ones((T, K), device="cuda", dtype=torch.bfloat16)
    w = okc.int8_rows(torch.full((2, K), 127, dtype=torch.int8, device="cuda"), torch.ones(2, device="cuda"))
    y = okc.int8_linear(ones, w, out_f32=True)
    q, scale = _quant_ref(ones)
    _close(y, *_linear_ref(q, scale, w, None, torch.float32), "127")
    low = okc.int8_rows(torch.full((T, K), -128, dtype=torch.int8, device="cuda"), torch.ones(T, device="cuda"))
    wl = okc.int8_rows(torch.full((2, K), -128, dtype=torch.int8, device="cuda"), torch.ones(2, device="cuda"))
    y = okc.int8_linear(low, wl, out_f32=True)
    assert (y == float(16384 * K)).all()        # 2^14 * 131071: 17 significant bits


def test_a_tokens_bits_do_not_depend_on_the_batch():
    g = _gen(11)
    x, w = _randn((700, 1500), g), _weight(400, 1500, g)
    full, full_g = okc.int8_linear(x, w, out_f32=True), okc.int8_gated(x, w, out_f32=True)
    for T in (1, 2, 4, 8, 9, 31, 64, 200, 256, 257, 699):
        assert torch.equal(okc.int8_linear(x[:T], w, out_f32=True), full[:T]), T
        assert torch.equal(okc.int8_gated(x[:T], w, out_f32=True), full_g[:T]), T


@pytest.mark.parametrize("T", [4, 70, 333])
def test_rows_that_are_not_finite_or_empty(T):
    g = _gen(T)
    x, w = _randn((T, 200), g), _weight(96, 200, g)
    bias = _randn(96, g)
    x[0] = 0
    x[1, 7] = float("inf")
    x[2, 199] = float("nan")
    y = okc.int8_linear(x, w, bias=bias)
    assert torch.equal(y[0], bias.bfloat16()) and y[1:3].isnan().all() and torch.isfinite(y[3:]).all()
    h = okc.int8_gated(x, w)
    assert not h[0].any() and h[1:3].isnan().all() and torch.isfinite(h[3:]).all()


@pytest.mark.parametrize("T", [1, 2, 6, 50, 400])
def test_strides_padding_and_rows_behind_the_last(T):
    g = _gen(T + 77)
    K, N = 200, 120
    wide = _randn((T + 1, 333), g, torch.bfloat16)
    x = wide[:T, 5:5 + K]                                       # rows off every 16-byte boundary
    qw = torch.randint(-127, 128, (N, 256), generator=g, device="cuda", dtype=torch.int8)
    w = okc.QuantRows(qw[:, :K], torch.rand(N, generator=g, device="cuda"))     # the columns behind K hold other values
    q, scale = _quant_ref(x)
    store = torch.full((T + 2, N + 9), 7.0, device="cuda", dtype=torch.bfloat16)
    y = okc.int8_linear(x, w, out=store[1:T + 1, 3:3 + N])
    _close(y, *_linear_ref(q, scale, w, None, torch.bfloat16), "strided")
    assert y.data_ptr() == store[1:, 3:].data_ptr()
    assert (store[0] == 7).all() and (store[T + 1] == 7).all() and (store[:, :3] == 7).all() and (store[:, 3 + N:] == 7).all()
    # int8 tokens whose row padding holds other values too
    xq = torch.randint(-127, 128, (T + 1, 256), generator=g, device="cuda", dtype=torch.int8)[:T, :K]
    xs = torch.rand(T, generator=g, device="cuda")
    _close(okc.int8_linear((xq, xs), w, out_f32=True), *_linear_ref(xq, xs, w, None, torch.float32), "int8 strided")
    # transposed tokens, strided scales
    _close(okc.int8_linear(x.t().contiguous().t(), w), *_linear_ref(q, scale, w, None, torch.bfloat16), "transposed")
    two = torch.rand((N, 2), generator=g, device="cuda")
    w2 = okc.QuantRows(w.q, two[:, 1])
    _close(okc.int8_linear(x, w2), *_linear_ref(q, scale, w2, None, torch.bfloat16), "strided scales")


@pytest.mark.parametrize("T", [1, 3, 40, 106, 300, 600])
@pytest.mark.parametrize("N", [1, 8, 33, 36, 37, 40, 71, 266])
def test_columns_behind_the_last_are_left_alone(T, N):
    """Rows on 16-byte boundaries with a caller's columns behind them, of every remainder."""
    g = _gen(T + N)
    for K in (128, 1000):
        x, w, both = okc.quantize_rows(_randn((T, K), g)), _weight(N, K, g), _weight(2 * N, K, g)
        for dtype in (torch.bfloat16, torch.float32):
            for fn, weight in ((okc.int8_linear, w), (okc.int8_gated, both)):
                store = torch.full((T + 1, (N + 7) // 8 * 8 + 32), 7.0, device="cuda", dtype=dtype)
                y = fn(x, weight, out_f32=dtype is torch.float32, out=store[:T, :N])
                assert torch.equal(y, fn(x, weight, out_f32=dtype is torch.float32))
                assert (store[:, N:] == 7).all() and (store[T] == 7).all(), (K, dtype, fn.__name__)


@pytest.mark.parametrize("T", [6, 40, 300])
def test_outputs_and_inputs_beyond_32_bit_offsets(T):
    """Row strides that put the last rows more than 2^32 bytes into a buffer."""
    g = _gen(T)
    K, N = 64, 48
    stride = ((1 << 31) // (T - 1) + 64) // 8 * 8
    big = torch.empty((T - 1) * stride + 64, dtype=torch.bfloat16, device="cuda")
    x = big.as_strided((T, K), (stride, 1))
    x.copy_(_randn((T, K), g, torch.bfloat16))
    w = _weight(N, K, g)
    q, scale = _quant_ref(x.clone())
    assert (T - 1) * stride * 2 > 1 << 32
    _close(okc.int8_linear(x, w), *_linear_ref(q, scale, w, None, torch.bfloat16), "input")
    y = okc.int8_linear(x.clone(), w, out=big.as_strided((T, N), (stride, 1)))
    _close(y, *_linear_ref(q, scale, w, None, torch.bfloat16), "output")
    r, n = okc.block_norm(x.clone().contiguous(), pre_gain=torch.ones(K, device="cuda"))
    x.copy_(r)
    assert torch.equal(okc.block_norm(x, pre_gain=torch.ones(K, device="cuda"))[1], n)


def test_empty_batches():
    w = _weight(32, 64, _gen(0))
    x = torch.zeros((0, 64), device="cuda", dtype=torch.bfloat16)
    assert okc.int8_linear(x, w).shape == (0, 32) and okc.int8_gated(x, w).shape == (0, 16) and okc.int8_ffn(x, w, _weight(5, 16, _gen(1))).shape == (0, 5)
    r, n = okc.block_norm(x, x, pre_gain=torch.ones(64, device="cuda"), out="int8")
    assert r.shape == (0, 64) and n.q.shape == (0, 64) and n.scale.shape == (0,)


def test_refusals_on_the_device():
    g = _gen(3)
    x, w = _randn((4, 64), g), _weight(32, 64, g)
    gain = torch.ones(64, device="cuda")
    bad = [
        lambda: okc.int8_linear(x, w, bias=torch.ones(31, device="cuda")),
        lambda: okc.int8_linear(x, w, bias=torch.ones(32, device="cuda", dtype=torch.bfloat16)),
        lambda: okc.int8_linear(x, w, bias=torch.ones(32)),
        lambda: okc.int8_linear(x, (w.q, w.scale.cpu())),
        lambda: okc.int8_linear(x, w, out=torch.empty((4, 31), device="cuda", dtype=torch.bfloat16)),
        lambda: okc.int8_linear(x, w, out=torch.empty((4, 32), device="cuda")),
        lambda: okc.int8_linear(x, w, out=torch.empty((32, 4), device="cuda", dtype=torch.bfloat16).t()),
        lambda: okc.int8_linear(x, w, out=torch.empty((1, 32), device="cuda", dtype=torch.bfloat16).expand(4, 32)),
        lambda: okc.int8_linear(x, w, out_f32=True, out=x[:, :32]),
        lambda: okc.block_norm(x, x[:3]),
        lambda: okc.block_norm(x, x.cpu()),
        lambda: okc.block_norm(x),
        lambda: okc.block_norm(x, pre_gain=gain, gate=gain),
        lambda: okc.block_norm(x, pre_gain=gain, residual_scale=0.5),
        lambda: okc.block_norm(x, pre_gain=gain, residual_out=x),
        lambda: okc.block_norm(x, x, pre_gain=gain[:63]),
        lambda: okc.block_norm(x, x, pre_gain=gain.bfloat16()),
        lambda: okc.block_norm(x, x, gate=torch.ones((4, 2), device="cuda")),
        lambda: okc.block_norm(x, x, gate=gain.double()),
        lambda: okc.block_norm(x, x.clone(), residual_out=x.bfloat16()),
        lambda: okc.block_norm(x[:3], x[:3].clone(), residual_out=x[1:]),
        lambda: okc.block_norm(x[:3], x[1:], residual_out=x[:3]),      # the block's rows are the stream's, one further on
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


# ------------------------------------------------------------------------------------------------ block_norm
def _norm_ref(res, blk, *, post_gain=None, gate=None, gate_sigmoid=False, residual_scale=1.0, block_scale=1.0, pre_gain=None, eps=1e-5):
    """(r', its tolerance, x, its tolerance) before the rounding to a type.  A sum of H squares in chains of at most 32 and
    two trees of 5 is off by 43 U relative, the mean by two more, the root halves that and adds 4 U: 27 U a norm; z takes
    two products on top, the gate and the scales five with a sigmoid's error, r' two products and a sum."""
    res, y = res.double(), None
    r, tol = res, torch.zeros_like(res)
    if blk is not None:
        y = blk.double()
        rel = 0.0
        if post_gain is not None:
            y = y * (y.square().mean(1, keepdim=True) + eps).rsqrt() * post_gain.double()
            rel = 29 * U
        if gate is not None:
            gd = gate.double()
            y = y * (torch.special.expit(gd) if gate_sigmoid else gd)
            rel = rel + (U * (2 * (2 + 1.173 * gd.abs()) + 3) if gate_sigmoid else 0)
        r = residual_scale * res + block_scale * y
        # the scales themselves round to f32 (U each)
        tol = ((rel + 5 * U) * (block_scale * y).abs() + 3 * U * (residual_scale * res).abs()) * 1.01
    if pre_gain is None:
        return r, tol, None, None
    rstd = (r.square().mean(1, keepdim=True) + eps).rsqrt()
    x = r * rstd * pre_gain.double()
    share = tol.norm(dim=1, keepdim=True) / r.norm(dim=1, keepdim=True).clamp_min(1e-300)
    xtol = (tol * rstd * pre_gain.double().abs() + x.abs() * (29 * U + share)) * 1.01
    return r, tol, x, xtol


def _check_norm(res, blk, out, **kw):
    r, x = okc.block_norm(res, blk, out=out, **kw)
    rr, rt, xr, xt = _norm_ref(res, blk, **kw)
    assert r.dtype == res.dtype
    _close(r, rr, rt + HALF[res.dtype] * (rr.abs() + rt) + 1e-37, "residual")
    if xr is None:
        assert x is None
    elif out == "int8":
        # within half a step of the kernel's own x; the scale is its maximum / 127, rounded
        s = x.scale.double()[:, None]
        peak, pt = xr.abs().amax(1), xt.amax(1)
        assert ((x.scale.double() * 127 - peak).abs() <= pt + 2 * U * peak + 2 * TINY).all()
        _close(x.q.double() * s, xr, xt + 0.5 * s * (1 + 2.0 ** -15) + 2 * TINY, "int8 rows")
    else:
        _close(x, xr, xt + HALF[x.dtype] * (xr.abs() + xt) + 1e-37, "normed")
    return r, x


@pytest.mark.parametrize("T,H", [(1, 1), (1, 4096), (2, 63), (7, 1000), (33, 5120), (3, 16384), (2, 16383), (300, 2048), (297, 2056), (310, 6500), (500, 8200), (298, 12289),
                                 (593, 8), (600, 2040), (700, 5120), (597, 8192), (599, 12296),
                                 (593, 1), (600, 2051), (650, 5121), (593, 16383), (700, 1001)])
@pytest.mark.parametrize("res,blk", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)])
def test_block_norm(T, H, res, blk):
    g = _gen(T * H + 1)
    r, y = _randn((T, H), g, res), _randn((T, H), g, blk)
    gains = dict(post_gain=1 + 0.1 * _randn(H, g), pre_gain=1 + 0.1 * _randn(H, g))
    _check_norm(r, y, "bf16", **gains)
    _check_norm(r, y, "f32", residual_scale=0.7, block_scale=-1.3, gate=_randn(H, g), **gains)
    _check_norm(r, y, "int8", gate=_randn((T, 1), g, torch.bfloat16), gate_sigmoid=True, **gains)
    _check_norm(r, y, "f32", gate=_randn((T, H), g, torch.bfloat16), pre_gain=gains["pre_gain"])
    _check_norm(r, y, "bf16", gate=_randn((T, H), g), gate_sigmoid=True, post_gain=gains["post_gain"])
    _check_norm(r, None, "f32", pre_gain=gains["pre_gain"], eps=1e-2)


def test_block_norm_strides_in_place_and_unaligned():
    g = _gen(9)
    T, H = 12, 136
    wide = _randn((T + 2, 3 * H + 1), g)
    gain = 1 + 0.1 * _randn(H + 1, g)
    for lo in (0, 1, 8):
        res, blk = wide[:T, lo:lo + H], wide.bfloat16()[2:, H + lo:2 * H + lo]
        _check_norm(res, blk, "f32", post_gain=gain[:H], pre_gain=gain[1:], gate=wide[:T, -1:])
        _check_norm(res, blk, "int8", post_gain=gain[1:], pre_gain=gain[:H], gate=wide[2:, 5:5 + H])
    _check_norm(wide.t()[:H, :T], wide.t()[:H, 1:T + 1], "bf16", pre_gain=gain[:T].contiguous())
    # many rows of all starts, each copied ahead of its turn
    many = _randn((800, 3 * H + 1), g, torch.bfloat16)
    for lo in (0, 1, 2, 3):
        res, blk = many[:700, lo:lo + H - 1], many[100:, H + lo:2 * H - 1 + lo]
        _check_norm(res, blk, "f32", post_gain=gain[1:H], pre_gain=gain[2:], gate=many[3:703, 2 * H:3 * H - 1])
        _check_norm(res, blk.float(), "int8", post_gain=gain[1:H], pre_gain=gain[:H - 1], gate=many[0, 5:H + 4], gate_sigmoid=True)
        _check_norm(res.float(), blk, "bf16", pre_gain=gain[:H - 1], gate=many[3:703, -1:], gate_sigmoid=True)
        _check_norm(res, blk, "bf16", post_gain=gain[1:H])
    # many rows in place, each copied ahead of its turn: the same bits as out of place, twice over
    for dtype, width in ((torch.float32, H), (torch.bfloat16, H), (torch.float32, H - 3), (torch.bfloat16, H - 3)):
        H = width
        many, blk = _randn((2000, H), g, dtype), _randn((2000, H), g, dtype)
        first, x = okc.block_norm(many, blk, pre_gain=gain[:H], post_gain=gain[:H], gate=many, out="int8")
        second, x2 = okc.block_norm(first, blk, pre_gain=gain[:H], post_gain=gain[:H], gate=first, out="int8")
        store = many.clone()
        for want, wx in ((first, x), (second, x2)):
            _, y = okc.block_norm(store, blk, pre_gain=gain[:H], post_gain=gain[:H], gate=store, out="int8", residual_out=store)
            assert torch.equal(store, want) and torch.equal(y.q, wx.q) and torch.equal(y.scale, wx.scale)
    H = 136
    # in place: the same bits as out of place (from the same addresses: the order of a row's sum goes by its alignment),
    # the columns and rows around them untouched
    store = wide.clone()
    blk = _randn((T, H), g)
    ref, x = okc.block_norm(store[1:T + 1, 7:7 + H], blk, pre_gain=gain[:H], post_gain=gain[:H])
    view = store[1:T + 1, 7:7 + H]
    r, x2 = okc.block_norm(view, blk, pre_gain=gain[:H], post_gain=gain[:H], residual_out=view)
    assert r is view and torch.equal(view, ref) and torch.equal(x, x2)
    around = torch.ones_like(store, dtype=torch.bool)
    around[1:T + 1, 7:7 + H] = False
    assert torch.equal(store[around], wide[around])
    # one memory for all three, element for element
    same = blk.clone()
    assert torch.equal(okc.block_norm(same, same, post_gain=gain[:H], residual_out=same)[0], okc.block_norm(blk, blk.clone(), post_gain=gain[:H])[0])


@pytest.mark.parametrize("T", [9, 640])
def test_block_norm_special_rows(T):
    """Rows of zeros, the largest values, infinities and NaN: what the formula gives, each in its own row only."""
    g = _gen(10)
    H = 520
    r, y = _randn((T, H), g), _randn((T, H), g)
    gain = torch.ones(H, device="cuda")
    r[0] = y[0] = 0
    r[1, 3] = float("nan")
    y[2, 519] = float("inf")
    y[3] = 0
    for out in ("bf16", "f32"):
        r2, x = okc.block_norm(r, y, post_gain=gain, pre_gain=gain, out=out)
        assert not r2[0].any() and not x[0].any()
        assert x[1].isnan().all() and r2[1].isnan().sum() == 1
        assert x[2].isnan().all() and r2[2].isnan().sum() == 1         # inf * rsqrt(inf) in its column, 0 * y beside it
        assert torch.equal(r2[3], r[3]) and torch.isfinite(x[3:]).all()
    _, x = okc.block_norm(r, y, post_gain=gain, pre_gain=gain, out="int8")
    assert x.scale[0] == 0 and x.scale[1:3].isnan().all() and not x.q[:3].any() and torch.isfinite(x.scale[3:]).all()
    # a gate that is not finite, in a width that leaves threads without columns
    gate = torch.ones((T, 1), device="cuda")
    gate[5] = float("inf")
    r2, x = okc.block_norm(r[:, :500].contiguous(), y[:, :500].contiguous(), gate=gate, pre_gain=gain[:500], out="f32")
    assert not torch.isfinite(r2[5]).any() and torch.isfinite(x[6:]).all()


# ------------------------------------------------------------------------------------------------ streams, graphs, together
def _calls(seed):
    g = _gen(seed)
    w13, w2 = _weight(256, 192, g), _weight(192, 128, g)
    gain = 1 + 0.1 * _randn(192, g)
    def run(r, T):
        r2, x = okc.block_norm(r[:T], r[:T].flip(0).contiguous(), post_gain=gain, pre_gain=gain, out="int8")
        return r2, x.q, x.scale, okc.int8_ffn(x, w13, w2), okc.int8_linear(r[:T], w13, out_f32=True)
    return run, _randn((900, 192), g)


@pytest.mark.parametrize("T", [1, 30, 400, 900])
def test_captured_graphs_replay_on_new_inputs_and_side_by_side(T):
    run, r = _calls(T)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    ins = [r.clone(), r.clone()]
    run(r, T)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(x, T))
        graphs.append(g)
    for step in range(4):
        new = [_randn(r.shape, _gen(100 * step + k)) for k in (0, 1)]
        want = [run(n, T) for n in new]
        for x, n in zip(ins, new):
            x.copy_(n)
        torch.cuda.synchronize()
        for g, s in zip(graphs, (s1, s2)):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(o, w))


@pytest.mark.parametrize("T", [5, 100, 400, 900])
def test_two_streams_at_once_and_back_to_back_calls(T):
    run, r = _calls(T + 1)
    others = [_randn(r.shape, _gen(k)) for k in range(8)]
    want = [run(o, T) for o in others]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = [None] * 8
    for k, o in enumerate(others):
        with torch.cuda.stream(streams[k % 4]):
            got[k] = run(o, T)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert okc.dense_status() == (0, 0)


def test_one_token_sequence_after_sequence_reuses_memory_safely():
    """Back to back calls whose temporaries the allocator hands on: scratch of one call is the next one's output."""
    g = _gen(21)
    w = _weight(192, 192, g)
    x = _randn((64, 192), g, torch.bfloat16)
    want, y = [], x
    for _ in range(6):
        y = okc.int8_linear(y, w)
        torch.cuda.synchronize()
        want.append(y.clone())
    for _ in range(20):
        y = x
        for k in range(6):
            y = okc.int8_linear(y, w)
        assert torch.equal(y, want[-1])


@pytest.mark.parametrize("T", [1, 8, 33, 300])
def test_dense_layer_from_norm_to_norm(T):
    """Norm into int8 rows, gated feed-forward, norm with gate and residual: against the same steps in 64 bits."""
    g = _gen(T)
    H, I = 512, 704
    r = _randn((T, H), g)
    def weight(rows, cols):
        return okc.quantize_rows(0.02 * _randn((rows, cols), g))
    w13, w2 = weight(2 * I, H), weight(H, I)
    gain, post, gate = (1 + 0.1 * _randn(H, g) for _ in range(3))
    _, x = okc.block_norm(r, pre_gain=gain, out="int8")
    y = okc.int8_ffn(x, w13, w2, out_f32=True)
    r2, n = okc.block_norm(r, y, post_gain=post, gate=gate, block_scale=0.5, pre_gain=gain)
    deq = lambda q: q.q.double() * q.scale.double()[:, None]  # noqa: E731
    rd = r.double()
    xd = rd * (rd.square().mean(1, keepdim=True) + 1e-5).rsqrt() * gain.double()
    h = xd @ deq(w13).t()
    h = torch.nn.functional.silu(h[:, :I]) * h[:, I:]
    yd = h @ deq(w2).t()
    # The two quantisations of the activations: an error of at most half a step of max / 127 a value, so below
    # max|x| / (254 * rms) relative to a row's norm, about 4 / 254, and as much again for h (whose maximum may be 8 times
    # its rms: 8 / 254); products of independent weights keep the relative size.
    rel = ((y.double() - yd).norm() / yd.norm()).item()
    assert rel < 2 * (4 + 8) / 254, rel
    rr, rt, xr, xt = _norm_ref(r, y, post_gain=post, gate=gate, block_scale=0.5, pre_gain=gain)
    _close(r2, rr, rt + U * (rr.abs() + rt), "residual")
    _close(n, xr, xt + HALF[torch.bfloat16] * (xr.abs() + xt), "next input")


def test_expert_block_on_the_residual_stream():
    """moe_block_step is its parts: norm, router and experts in f32, norm with gate and residual."""
    g = _gen(4)
    plan = okc.MoEPlan(hidden=512, inter=256, n_experts=16, top_k=2, max_tokens=64)
    weights = synth.make_weights(synth.Workload("small", 5, 512, 256, 16, 2), seed=11, device=torch.device("cuda"))
    state, router = okc.prepare(weights, plan), _randn((16, 512), g)
    gain, post = 1 + 0.1 * _randn(512, g), 1 + 0.1 * _randn(512, g)
    lin = okc.quantize_rows(0.02 * _randn((256, 512), g))
    for T in (1, 5, 40):
        r = _randn((T, 512), g)
        gate = _randn((T, 1), g)
        r2, x = okc.moe_block_step(r, router, state, pre_gain=gain, post_gain=post, gate=gate, gate_sigmoid=True, residual_scale=0.9,
                                   next_gain=gain, out="int8")
        hidden = okc.block_norm(r, pre_gain=gain)[1]
        y = okc.moe_layer_step(hidden, router, state, out_f32=True)
        rr, rt, xr, xt = _norm_ref(r, y, post_gain=post, gate=gate, gate_sigmoid=True, residual_scale=0.9, pre_gain=gain)
        _close(r2, rr, rt + U * (rr.abs() + rt), "residual")
        s = x.scale.double()[:, None]
        _close(x.q.double() * s, xr, xt + 0.5 * s * (1 + 2.0 ** -15) + 2 * TINY, "int8 rows")
        _close(okc.int8_linear(x, lin, out_f32=True), *_linear_ref(x.q, x.scale, lin, None, torch.float32), "next projection")
        assert okc.read_status(state)[0] == 0
        again = r.clone()
        r3, none = okc.moe_block_step(again, router, state, pre_gain=gain, post_gain=post, gate=gate, gate_sigmoid=True, residual_scale=0.9,
                                      residual_out=again)
        assert r3 is again and torch.equal(again, r2) and none is None
