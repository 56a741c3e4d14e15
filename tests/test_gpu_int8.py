"""8-bit integer operators on the GPU (rcvpose_amd.int8, rcv_i8_* in include/rcvpose_hip.h) against the definitions in 64 bits."""
import ctypes

import numpy as np
import pytest
import torch

from rcvpose_amd import _hip, int8

pytestmark = pytest.mark.gpu

NP = {torch.float32: np.float32, torch.float16: np.float16}
U32 = 2.0 ** -24                                             # half a step of float32, relative
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step of the output type: finfo.eps / 2
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}       # half a step among the subnormals


def f64(t):
    return t.detach().cpu().double().numpy()


def ref_quantize(x):
    """x float64 [rows, C] (values of the input type) -> codes, scales."""
    with np.errstate(invalid="ignore"):
        s = (np.abs(x).max(axis=1) / 127).astype(np.float32)
    s[s < 2.0 ** -126] = 0
    bad = ~np.isfinite(x).all(axis=1)
    s[bad] = np.nan
    live = (s > 0) & ~bad
    q = np.zeros(x.shape, dtype=np.int8)
    q[live] = np.round(x[live] / s[live, None].astype(np.float64)).astype(np.int8)  # (float64 quotients of float32 numbers never round onto a half)
    return q, s


def ref_product(a, sa, w, sw, bias, residual, relu, image=None):
    """-> (value, magnitude of what was added) in float64.  a [rows, K], w [N, taps, K]."""
    a, w = a.astype(np.float64), w.astype(np.float64)
    rows, n = a.shape[0], w.shape[0]
    v, mag = np.zeros((rows, n)), np.zeros((rows, n))
    if image is None:
        taps = [(0, np.arange(rows), np.arange(rows))]
    else:
        b, h, wd = image
        idx = np.arange(rows).reshape(b, h, wd)
        taps = []
        for t in range(9):
            dy, dx = t // 3 - 1, t % 3 - 1
            dst = idx[:, max(0, -dy):h - max(0, dy), max(0, -dx):wd - max(0, dx)].reshape(-1)
            taps.append((t, dst, dst + dy * wd + dx))
    for t, dst, src in taps:
        part = (a[src] @ w[:, t].T) * sa[src, None].astype(np.float64)
        v[dst] += part
        mag[dst] += np.abs(part)
    v, mag = v * sw.astype(np.float64), mag * sw.astype(np.float64)
    if bias is not None:
        v, mag = v + bias, mag + np.abs(bias)
    if residual is not None:
        v, mag = v + residual, mag + np.abs(residual)
    return (np.where(v < 0, 0, v) if relu else v), mag


def bound(value, mag, dtype, taps):
    """float32: an exact integer sum is rounded once, scaled, and each of the `taps` additions (and up to sixteen more where a long
    sum was split), the weight scale, the bias and the residual round once more, each by at most half a step of a number no larger
    than `mag`.  Then one rounding to the output's type."""
    return (taps + 22) * U32 * mag + HALF[dtype] * (np.abs(value) + (taps + 22) * U32 * mag) + TINY[dtype]


def check_product(got, value, mag, dtype, taps):
    g = f64(got).reshape(value.shape)
    assert np.isfinite(g).all()
    err = np.abs(g - value)
    lim = bound(value, mag, dtype, taps)
    worst = np.unravel_index(np.argmax(err - lim), err.shape)
    assert (err <= lim).all(), (worst, g[worst], value[worst], lim[worst])


def random_codes(rng, rows, k, pitch=None, garbage=True):
    """Codes as a view of a wider buffer whose other bytes hold garbage."""
    pitch = pitch or (k + 15) // 16 * 16
    buf = rng.integers(-128, 128, size=(rows, pitch)).astype(np.int8) if garbage else np.zeros((rows, pitch), np.int8)
    return torch.from_numpy(buf).cuda()[:, :k]


def make(rng, rows, k, n, taps, dtype, residual, pitch=None):
    a = random_codes(rng, rows, k, pitch)
    sa = torch.from_numpy(np.exp(rng.standard_normal(rows)).astype(np.float32) * 0.02).cuda()
    w = torch.from_numpy(rng.integers(-128, 128, size=(n, k) if taps == 1 else (n, 3, 3, k)).astype(np.int8)).cuda()
    sw = torch.from_numpy(np.exp(0.3 * rng.standard_normal(n)).astype(np.float32) / np.float32(74 * np.sqrt(k * taps))).cuda()
    bias = torch.from_numpy(rng.standard_normal(n).astype(np.float32)).cuda()
    res = torch.from_numpy(rng.standard_normal((rows, n)).astype(np.float32)).cuda().to(dtype) if residual else None
    return a, sa, w, sw, bias, res


QUANT = [(1, 1), (1, 4096), (3, 16), (5, 333), (67, 64), (130, 128), (9, 2048), (4, 5000), (2, 40000),
         (70, 30), (71, 100), (40, 1500), (33, 3000), (3, 8192), (4, 10000), (2, 131071)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows, c", QUANT)
def test_quantize(rows, c, dtype):
    rng = np.random.default_rng(rows * 7919 + c)
    x = rng.standard_normal((rows, c)) * np.exp(2 * rng.standard_normal((rows, 1)))
    x[:, 0] *= 3
    x[rows // 2] = 0
    t = torch.from_numpy(x.astype(np.float32)).cuda().to(dtype)
    codes, scales = int8.quantize_tokens(t)
    q, s = ref_quantize(f64(t))
    np.testing.assert_array_equal(scales.cpu().numpy(), s)
    np.testing.assert_array_equal(codes.cpu().numpy(), q)
    assert codes.stride(0) % 16 == 0


def test_quantize_halves_go_to_even():
    """Quotients that are exactly a half, and the nearest float32 numbers beside them: scale 1 (maximum 127) and scale 3."""
    for s in (1.0, 3.0):
        h = (np.arange(-126, 126) + 0.5).astype(np.float32) * np.float32(s)
        x = np.concatenate([h, np.nextafter(h, np.float32(np.inf)), np.nextafter(h, np.float32(-np.inf)), [np.float32(127 * s)]])[None]
        t = torch.from_numpy(x.astype(np.float32)).cuda()
        codes, scales = int8.quantize_tokens(t)
        q, ref = ref_quantize(f64(t))
        np.testing.assert_array_equal(scales.cpu().numpy(), ref)
        np.testing.assert_array_equal(codes.cpu().numpy(), q)


@pytest.mark.parametrize("c0, c1", [(64, 128), (1024, 1024), (33, 16), (16, 7), (5, 3)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_quantize_two_sources_and_strides(c0, c1, dtype):
    rng = np.random.default_rng(c0 + c1)
    wide0 = torch.from_numpy(rng.standard_normal((2, 3, 5, c0 + 24)).astype(np.float32)).cuda().to(dtype)
    x1 = torch.from_numpy(5 * rng.standard_normal((2, 3, 5, c1)).astype(np.float32)).cuda().to(dtype)
    x0 = wide0[..., 8:8 + c0]  # rows at a wider pitch
    codes, scales = int8.quantize_tokens(x0, x1)
    assert tuple(codes.shape) == (2, 3, 5, c0 + c1) and tuple(scales.shape) == (2, 3, 5)
    q, s = ref_quantize(f64(torch.cat([x0, x1], dim=-1)).reshape(30, -1))
    np.testing.assert_array_equal(scales.cpu().numpy().reshape(-1), s)
    np.testing.assert_array_equal(codes.cpu().numpy().reshape(30, -1), q)
    xt = x1.transpose(1, 2)  # rows that walk memory at no single pitch
    np.testing.assert_array_equal(int8.quantize_tokens(xt)[0].cpu().numpy(), int8.quantize_tokens(xt.contiguous())[0].cpu().numpy())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_quantize_extremes(dtype):
    """Rows of zeros, of the type's largest and smallest numbers, and rows that hold a NaN or an infinity."""
    info = torch.finfo(dtype)
    x = torch.zeros(8, 96, dtype=dtype)
    x[1] = info.max
    x[1, ::2] = -info.max
    x[2, 5] = info.tiny  # the smallest normal number alone
    x[3, 7] = float("nan")
    x[4, 95] = float("inf")
    x[5, 0], x[5, 1:] = -float("inf"), 2.0
    x[6] = -0.0
    x[7] = torch.linspace(-1, 1, 96).to(dtype)
    codes, scales = int8.quantize_tokens(x.cuda())
    q, s = ref_quantize(f64(x))
    np.testing.assert_array_equal(scales.cpu().numpy(), s)
    np.testing.assert_array_equal(codes.cpu().numpy(), q)
    assert np.isnan(s[3:6]).all() and np.isfinite(s[[0, 1, 2, 6, 7]]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("c", [24, 100, 700, 1500, 5000])
def test_quantize_at_every_magnitude(c, dtype):
    """Rows from the smallest scale that counts to the largest numbers, with equal values, halves and powers of two of the row's largest among
    them (quotients beside a half): every code and every scale exact."""
    rng = np.random.default_rng(c)
    lo, hi = (-16, 14) if dtype == torch.float16 else (-119, 126)
    e = np.linspace(lo, hi, 200)
    x = rng.standard_normal((200, c)) / 4
    x[:, 0] = 1 + rng.random(200)
    x[:, 1::5] = x[:, :1] * 2.0 ** -rng.integers(0, 9, size=(200, len(range(1, c, 5))))
    x[:, 2::7] = x[:, :1] * (rng.integers(-127, 127, size=(200, len(range(2, c, 7)))) + 0.5) / 127
    t = torch.from_numpy(x * 2.0 ** np.floor(e)[:, None]).to(dtype)
    assert bool(torch.isfinite(t).all())
    codes, scales = int8.quantize_tokens(t.cuda())
    q, s = ref_quantize(f64(t))
    np.testing.assert_array_equal(scales.cpu().numpy(), s)
    np.testing.assert_array_equal(codes.cpu().numpy(), q)


def test_quantize_leaves_the_pitch_alone():
    """Codes written into rows of a wider buffer: the bytes behind the last code and the rows behind the last token stay."""
    L = _hip.lib()
    for c, off in ((50, 0), (64, 16), (37, 5)):
        x = torch.randn(6, c, device="cuda")
        buf = torch.full((9, 112), 77, dtype=torch.int8, device="cuda")
        scales = torch.full((9,), -1.0, device="cuda")
        _hip.check(L.rcv_i8_quantize_tokens(x.data_ptr(), c, c, None, 0, 0, _hip.RCV_F32, 6, buf.data_ptr() + off, 112, scales.data_ptr(),
                                            _hip.current_stream()))
        want = np.full((9, 112), 77, np.int8)
        want[:6, off:off + c], s = ref_quantize(f64(x))
        np.testing.assert_array_equal(buf.cpu().numpy(), want)
        np.testing.assert_array_equal(scales.cpu().numpy(), np.concatenate([s, np.full(3, -1, np.float32)]))


MATMUL = [(1, 1, 1), (1, 16, 5), (1, 4096, 300), (2, 131, 17), (3, 100, 33), (16, 512, 64), (17, 320, 130), (64, 64, 64), (65, 1000, 63),
          (100, 2048, 96), (130, 130, 129), (256, 128, 128), (257, 384, 257), (300, 2048, 512), (515, 96, 40), (2049, 256, 200), (5000, 64, 8),
          (777, 1500, 333),
          # enough output tiles for the large-product kernel: many rows of few channels, few rows of many
          (33000, 70, 40), (33023, 200, 9), (300, 150, 16500),
          (12300, 1030, 1025), (12300, 1900, 1032), (12300, 3600, 1025),
          # a long sum over few tiles, divided over workgroups
          (200, 8200, 900), (70, 20000, 1300),
          # wide layers of few rows
          (20, 200, 8300), (50, 130, 8200), (64, 8200, 4100), (3, 300, 20000)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m, k, n", MATMUL)
def test_matmul(m, k, n, dtype):
    rng = np.random.default_rng(m * 31 + k * 7 + n)
    residual, relu = bool((m + k) % 2), bool((k + n) % 2)
    a, sa, w, sw, bias, res = make(rng, m, k, n, 1, dtype, residual)
    weight = int8.pack_codes(w, sw)
    got = int8.matmul(a, sa, weight, bias=bias, residual=res, relu=relu, dtype=dtype)
    assert got.dtype == dtype and tuple(got.shape) == (m, n)
    v, mag = ref_product(a.cpu().numpy(), sa.cpu().numpy(), w.cpu().numpy().reshape(n, 1, k), sw.cpu().numpy(), f64(bias),
                         None if res is None else f64(res), relu)
    check_product(got, v, mag, dtype, 1)
    again = int8.matmul(a, sa, weight, bias=bias, residual=res, relu=relu, dtype=dtype)
    assert torch.equal(got, again)


CONV = [(1, 1, 1, 16, 1), (1, 1, 9, 64, 32), (2, 9, 1, 48, 24), (2, 5, 7, 33, 19), (1, 15, 20, 256, 96), (3, 37, 53, 96, 80), (1, 2, 2, 1, 1),
        (5, 8, 8, 128, 130), (2, 15, 20, 640, 64), (1, 61, 70, 64, 200),
        # enough output tiles for the large-product kernel
        (9, 61, 70, 33, 24), (7, 47, 101, 130, 120), (7, 47, 101, 40, 136), (33001, 1, 1, 20, 8), (1, 33000, 2, 16, 4),
        # a long sum over few tiles, divided by taps
        (1, 13, 21, 1100, 300), (3, 40, 41, 700, 260), (1, 30, 41, 300, 260), (2, 31, 33, 450, 61)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b, h, wd, c, n", CONV)
def test_conv3x3(b, h, wd, c, n, dtype):
    rng = np.random.default_rng(b * 131 + h * 17 + wd * 7 + c + n)
    residual, relu = bool((h + c) % 2), bool((wd + n) % 2)
    m = b * h * wd
    a, sa, w, sw, bias, res = make(rng, m, c, n, 9, dtype, residual)
    sa[m // 2] = 0
    weight = int8.pack_codes(w, sw)
    call = lambda: int8.conv3x3(a.unflatten(0, (b, h, wd)), sa.view(b, h, wd), weight, bias=bias,
                                residual=None if res is None else res.view(b, h, wd, n), relu=relu, dtype=dtype)
    got = call()
    assert got.dtype == dtype and tuple(got.shape) == (b, h, wd, n)
    v, mag = ref_product(a.cpu().numpy(), sa.cpu().numpy(), w.cpu().numpy().reshape(n, 9, c), sw.cpu().numpy(), f64(bias),
                         None if res is None else f64(res), relu, (b, h, wd))
    check_product(got, v, mag, dtype, 9)
    assert torch.equal(got, call())


def test_largest_sum_does_not_overflow():
    """131071 products of -128 * -128 fill 31 bits; one of the two rows has the opposite sign."""
    k = int8.MAX_CHANNELS
    a = torch.full((2, k + 1), -128, dtype=torch.int8, device="cuda")
    a[1] = 127
    w = torch.full((3, k), -128, dtype=torch.int8, device="cuda")
    got = int8.matmul(a[:, :k], torch.ones(2, device="cuda"), int8.pack_codes(w, torch.ones(3, device="cuda")), dtype=torch.float32)
    want = np.array([[128.0 * 128 * k], [-127.0 * 128 * k]])
    assert (np.abs(f64(got) - want) <= U32 * np.abs(want)).all()


def test_codes_inside_a_wider_matrix():
    """Channels 32 .. 132 of rows of 160 codes; the neighbours' codes have no influence, no bias, residual at a pitch of its own."""
    rng = np.random.default_rng(5)
    wide = torch.from_numpy(rng.integers(-128, 128, size=(70, 160)).astype(np.int8)).cuda()
    _, sa, w, sw, _, _ = make(rng, 70, 100, 48, 1, torch.float32, False)
    res = torch.randn(70, 64, device="cuda")[:, 8:56]
    a = wide[:, 32:132]
    got = int8.matmul(a, sa, int8.pack_codes(w, sw), residual=res, dtype=torch.float32)
    v, mag = ref_product(a.cpu().numpy(), sa.cpu().numpy(), w.cpu().numpy().reshape(48, 1, 100), sw.cpu().numpy(), None, f64(res), False)
    check_product(got, v, mag, torch.float32, 1)


@pytest.mark.parametrize("rows, n, pitch", [(5, 7, 12), (70, 64, 72), (300, 130, 131), (520, 128, 160), (2500, 260, 261), (20000, 1100, 1101), (20000, 1152, 1160)])
def test_output_rows_at_a_pitch(rows, n, pitch):
    """The columns between two rows and the rows behind the last stay as they were, the residual may be the output itself."""
    rng = np.random.default_rng(rows)
    L = _hip.lib()
    k = 1056 if n > 1000 else 96  # (the last case is one of the large-product kernel's widest tiles)
    a, sa, w, sw, bias, _ = make(rng, rows, k, n, 1, torch.bfloat16, False)
    weight = int8.pack_codes(w, sw)
    buf = torch.randn(rows + 2, pitch, device="cuda").bfloat16()
    before = f64(buf)
    args = _hip.I8Args(ctypes.sizeof(_hip.I8Args), _hip.RCV_BF16, a.data_ptr(), sa.data_ptr(), weight.codes.data_ptr(), weight.scales.data_ptr(),
                       bias.data_ptr(), buf.data_ptr(), buf.data_ptr(), rows, a.stride(0), pitch, pitch, k, n, 0, 0, 1, 0)
    need = L.rcv_i8_matmul_workspace_bytes(rows, k, n)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    _hip.check(L.rcv_i8_matmul(ctypes.byref(args), ws.data_ptr(), need, _hip.current_stream()))
    after = f64(buf)
    v, mag = ref_product(a.cpu().numpy(), sa.cpu().numpy(), w.cpu().numpy().reshape(n, 1, k), sw.cpu().numpy(), f64(bias), before[:rows, :n], True)
    check_product(torch.from_numpy(after[:rows, :n]), v, mag, torch.bfloat16, 1)
    after[:rows, :n] = before[:rows, :n]
    np.testing.assert_array_equal(after, before)


@pytest.mark.parametrize("seed", range(8))
def test_sizes_drawn_at_random(seed):
    """Sizes over the ranges in which the choice of kernel changes, every type, with and without bias, residual and ReLU."""
    rng = np.random.default_rng(1000 + seed)
    log = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))
    for _ in range(8):
        dtype = [torch.float32, torch.bfloat16, torch.float16][rng.integers(3)]
        residual, relu, with_bias = rng.random(3) < 0.5
        taps = 1 if rng.random() < 0.5 else 9
        if taps == 1:
            m, k, n = log(1, 3000), log(1, 6000), log(1, 3000)
            while m * k * n > 3e9:
                m, n = max(1, m // 2), max(1, n // 2)
            image = None
        else:
            b, h, wd, k, n = log(1, 4), log(1, 50), log(1, 50), log(1, 900), log(1, 400)
            while b * h * wd * k * n > 3e8:
                k, n = max(1, k // 2), max(1, n // 2)
            m, image = b * h * wd, (b, h, wd)
        a, sa, w, sw, bias, res = make(rng, m, k, n, taps, dtype, residual)
        bias = bias if with_bias else None
        weight = int8.pack_codes(w, sw)
        if taps == 1:
            got = int8.matmul(a, sa, weight, bias=bias, residual=res, relu=bool(relu), dtype=dtype)
        else:
            got = int8.conv3x3(a.unflatten(0, image), sa.view(image), weight, bias=bias, residual=None if res is None else res.view(image + (n,)),
                               relu=bool(relu), dtype=dtype)
        v, mag = ref_product(a.cpu().numpy(), sa.cpu().numpy(), w.cpu().numpy().reshape(n, taps, k), sw.cpu().numpy(),
                             None if bias is None else f64(bias), None if res is None else f64(res), relu, image)
        check_product(got, v, mag, dtype, taps)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_token_has_the_same_product_in_any_batch(dtype):
    """One token, sixteen, a few hundred and many run on different kernels; the integer sums are exact, so a row's bits are the same."""
    rng = np.random.default_rng(17)
    for k, n in ((1100, 520), (8200, 140)):
        a, sa, w, sw, bias, res = make(rng, 9000, k, n, 1, dtype, True)
        weight = int8.pack_codes(w, sw)
        full = int8.matmul(a, sa, weight, bias=bias, residual=res, relu=True, dtype=dtype)
        for start, stop in ((0, 1), (8999, 9000), (100, 116), (200, 264), (300, 500), (1000, 3000)):
            part = slice(start, stop)
            assert torch.equal(int8.matmul(a[part], sa[part], weight, bias=bias, residual=res[part], relu=True, dtype=dtype), full[part])


def test_offsets_past_32_bits():
    """Codes, outputs and tokens of more than 2^31 bytes or elements: the last rows against the definitions."""
    rng = np.random.default_rng(11)
    # codes: 1100000 rows of 2048
    rows, k, n = 1100000, 2048, 20
    a = torch.randint(-128, 128, (rows, k), dtype=torch.int8, device="cuda")
    _, _, w, sw, bias, _ = make(rng, 1, k, n, 1, torch.float32, False)
    sa = torch.rand(rows, device="cuda")
    got = int8.matmul(a, sa, int8.pack_codes(w, sw), bias=bias, dtype=torch.float32)
    v, mag = ref_product(a[-300:].cpu().numpy(), sa[-300:].cpu().numpy(), w.cpu().numpy().reshape(n, 1, k), sw.cpu().numpy(), f64(bias), None, False)
    check_product(got[-300:], v, mag, torch.float32, 1)
    # the same codes as 2200 images of 20 x 25 pixels
    _, _, w, sw, bias, _ = make(rng, 1, k, n, 9, torch.float32, False)
    got = int8.conv3x3(a.view(2200, 20, 25, k), sa.view(2200, 20, 25), int8.pack_codes(w, sw), bias=bias, dtype=torch.float16)
    v, mag = ref_product(a[-500:].cpu().numpy(), sa[-500:].cpu().numpy(), w.cpu().numpy().reshape(n, 9, k), sw.cpu().numpy(), f64(bias), None, False,
                         (1, 20, 25))
    check_product(got[-1], v, mag, torch.float16, 9)
    # tokens: more than 2^31 bfloat16 numbers
    del a, got
    x = torch.randn(1100000, k, dtype=torch.bfloat16, device="cuda")
    codes, scales = int8.quantize_tokens(x)
    q, s = ref_quantize(f64(x[-50:]))
    np.testing.assert_array_equal(codes[-50:].cpu().numpy(), q)
    np.testing.assert_array_equal(scales[-50:].cpu().numpy(), s)
    del x, codes
    # outputs: 70000 x 32768
    a, sa, w, sw, bias, _ = make(rng, 70000, 64, 32768, 1, torch.bfloat16, False)
    got = int8.matmul(a, sa, int8.pack_codes(w, sw), bias=bias)
    v, mag = ref_product(a[-40:].cpu().numpy(), sa[-40:].cpu().numpy(), w.cpu().numpy().reshape(32768, 1, 64), sw.cpu().numpy(), f64(bias), None, False)
    check_product(got[-40:], v, mag, torch.bfloat16, 1)


def test_quantize_more_tokens_than_a_launch_has_threads_for():
    """2^30 + 77 tokens of 17 channels: the first rows, those about 2^30 and the last; zeros between."""
    rows, c = (1 << 30) + 77, 17
    x = torch.zeros(rows, c, dtype=torch.float16, device="cuda")
    parts = [slice(0, 500), slice((1 << 30) - 500, rows)]
    for part in parts:
        x[part].normal_()
    codes, scales = torch.full((rows, c), 5, dtype=torch.int8, device="cuda"), torch.full((rows,), -1.0, device="cuda")
    _hip.check(_hip.lib().rcv_i8_quantize_tokens(x.data_ptr(), c, c, None, 0, 0, _hip.RCV_F16, rows, codes.data_ptr(), c, scales.data_ptr(),
                                                 _hip.current_stream()))
    for part in parts:
        q, s = ref_quantize(f64(x[part]))
        np.testing.assert_array_equal(codes[part].cpu().numpy(), q)
        np.testing.assert_array_equal(scales[part].cpu().numpy(), s)
    for start in range(500, (1 << 30) - 500, 1 << 28):
        part = slice(start, min(start + (1 << 28), (1 << 30) - 500))
        assert int(scales[part].count_nonzero()) == 0 and int(codes[part].count_nonzero()) == 0
    del x, codes, scales
    torch.cuda.empty_cache()


def test_two_streams_and_two_graphs_at_once():
    """Products whose sums are divided (they use a workspace): on two streams at once, and from two graphs replayed in turn and together."""
    rng = np.random.default_rng(3)
    calls, want = [], []
    for rows, k, n in ((200, 8200, 900), (70, 20000, 1300)):
        a, sa, w, sw, bias, _ = make(rng, rows, k, n, 1, torch.float32, False)
        weight = int8.pack_codes(w, sw)
        assert _hip.load_library().rcv_i8_matmul_workspace_bytes(rows, k, n) > 0
        calls.append(lambda a=a, sa=sa, weight=weight, bias=bias: int8.matmul(a, sa, weight, bias=bias, dtype=torch.float32))
        want.append(calls[-1]())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = [[], []]
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i] = [calls[i]() for _ in range(4)]
        torch.cuda.synchronize()
        assert all(torch.equal(y, want[i]) for i in range(2) for y in got[i])
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(calls[i]())
        graphs.append(g)
    for turn in range(4):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for i in (0, 1) if turn % 2 else (1, 0):
            with torch.cuda.stream(streams[i if turn > 1 else 0]):
                graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(outs[i], want[i]) for i in range(2))
        assert torch.equal(calls[0](), want[0])


def test_nan_tokens_poison_their_window_and_nothing_else():
    b, h, wd, c, n = 1, 9, 11, 64, 32
    x = torch.randn(b, h, wd, c, device="cuda")
    x[0, 4, 5, 3] = float("nan")
    x[0, 0, 0, 0] = float("inf")
    codes, scales = int8.quantize_tokens(x)
    w = torch.randn(n, 3, 3, c, device="cuda")
    bad = torch.isnan(int8.conv3x3(codes, scales, int8.quantize_weight(w), relu=True, dtype=torch.float32)).cpu().numpy()
    want = np.zeros((b, h, wd, n), bool)
    want[:, 3:6, 4:7] = True
    want[:, 0:2, 0:2] = True
    np.testing.assert_array_equal(bad, want)
    y = int8.matmul(codes, scales, int8.quantize_weight(w[:, 0, 0]), relu=True, dtype=torch.float16)
    np.testing.assert_array_equal(torch.isnan(y).any(dim=-1).cpu().numpy(), torch.isnan(scales).cpu().numpy())


def test_empty_inputs():
    weight = int8.quantize_weight(torch.ones(8, 32, device="cuda"))
    codes, scales = int8.quantize_tokens(torch.ones(0, 32, device="cuda"))
    assert tuple(int8.matmul(codes, scales, weight).shape) == (0, 8)
    wc = int8.quantize_weight(torch.ones(8, 3, 3, 32, device="cuda"))
    codes, scales = int8.quantize_tokens(torch.ones(2, 0, 5, 32, device="cuda"))
    assert tuple(int8.conv3x3(codes, scales, wc).shape) == (2, 0, 5, 8)


def test_refusals():
    w = int8.quantize_weight(torch.ones(8, 32, device="cuda"))
    codes, scales = int8.quantize_tokens(torch.ones(4, 32, device="cuda"))
    wc = int8.quantize_weight(torch.ones(8, 3, 3, 32, device="cuda"))
    for call in (lambda: int8.matmul(codes, scales, wc), lambda: int8.conv3x3(codes, scales, wc), lambda: int8.conv3x3(codes, scales, w),
                 lambda: int8.matmul(codes[:, :16], scales, w), lambda: int8.matmul(codes, scales[:3], w),
                 lambda: int8.matmul(codes, scales.double(), w), lambda: int8.matmul(codes.float(), scales, w),
                 lambda: int8.matmul(codes, scales, w, dtype=torch.float64), lambda: int8.matmul(codes, scales, w, bias=torch.ones(7, device="cuda")),
                 lambda: int8.matmul(codes, scales, w, residual=torch.ones(4, 8, device="cuda")),
                 lambda: int8.quantize_tokens(torch.ones(4, 32, device="cuda", dtype=torch.int32)),
                 lambda: int8.quantize_tokens(torch.ones(4, 32, device="cuda"), torch.ones(5, 32, device="cuda")),
                 # rows that start 4 bytes apart from a 16-byte border, and a last row that ends with its storage
                 lambda: int8.matmul(torch.ones(4, 40, dtype=torch.int8, device="cuda")[:, :32], scales, w),
                 lambda: int8.matmul(torch.ones(64 + 33, dtype=torch.int8, device="cuda").as_strided((3, 33), (32, 1)), scales[:3],
                                     int8.quantize_weight(torch.ones(8, 33, device="cuda")))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError):
        int8.matmul(codes.cpu(), scales.cpu(), w)


def test_two_layers_as_a_network_runs_them():
    """Concatenated sources -> quantise -> 3x3 -> quantise -> 1x1 with residual: eager on a side stream, and captured, replayed with
    other inputs and other work between the replays; every replay equals the eager result bit for bit."""
    torch.manual_seed(0)
    w1 = int8.quantize_weight(torch.randn(64, 3, 3, 96, device="cuda") * 0.03)
    w2 = int8.quantize_weight(torch.randn(48, 64, device="cuda") * 0.1)
    b1, b2 = torch.randn(64, device="cuda"), torch.randn(48, device="cuda")
    x0, x1 = torch.randn(2, 12, 13, 64, device="cuda").half(), torch.randn(2, 12, 13, 32, device="cuda").half()
    res = torch.randn(2, 12, 13, 48, device="cuda").half()

    def net():
        y = int8.conv3x3(*int8.quantize_tokens(x0, x1), w1, bias=b1, relu=True, dtype=torch.float16)
        return int8.matmul(*int8.quantize_tokens(y), w2, bias=b2, residual=res, relu=True, dtype=torch.float16)

    first = net()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = net()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, second)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = net()
    for i in range(4):
        x0.copy_(torch.randn_like(x0))
        res.mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        want = net()
        assert torch.equal(out, want), i
        torch.randn(1 << 20, device="cuda").sort()
    # the same two layers in float arithmetic on the dequantised operands
    q, s = int8.quantize_tokens(x0, x1)
    xf = (q.double() * s[..., None].double()).cpu().permute(0, 3, 1, 2)
    y = torch.nn.functional.conv2d(xf, w1.dequantize().double().cpu().permute(0, 3, 1, 2), b1.double().cpu(), padding=1).clamp_min(0)
    got = int8.conv3x3(q, s, w1, bias=b1, relu=True, dtype=torch.float32)
    assert float((got.cpu().double() - y.permute(0, 2, 3, 1)).abs().max()) <= 1e-5 * float(y.abs().max())


@pytest.mark.parametrize("h, n", [(6556022, 4), (6556022, 72), (8399926, 4), (65537, 4), (257, 8)])
def test_tall_images(h, n):
    """Images of one column and of more rows than float32 numbers count exactly: the last rows of the first image and the first of the
    second, whose windows end at the border between them (H = 6556022 is the smallest height whose last row a float32 quotient
    misplaces, 8399926 the smallest whose next image's first row it does)."""
    rng = np.random.default_rng(h)
    c, dtype = 16, torch.bfloat16
    images = 2 if h > 1000 else 4001  # (enough rows for the tiles through LDS)
    a = torch.randint(-128, 128, (images * h, c), dtype=torch.int8, device="cuda")
    sa = torch.rand(images * h, device="cuda") + 0.5
    _, _, w, sw, bias, _ = make(rng, 1, c, n, 9, dtype, False)
    got = int8.conv3x3(a.view(images, h, 1, c), sa.view(images, h, 1), int8.pack_codes(w, sw), bias=bias, dtype=dtype).view(images * h, n)
    m = min(h - 1, 300)
    for start, stop, first, last in ((h - m - 1, h, 1, m + 1), (h, h + m + 1, 0, m)):  # rows read, and those of them whose window is among them
        part = slice(start, stop)
        v, mag = ref_product(a[part].cpu().numpy(), sa[part].cpu().numpy(), w.cpu().numpy().reshape(n, 9, c), sw.cpu().numpy(), f64(bias), None, False,
                             (1, m + 1, 1))
        check_product(got[part][first:last], v[first:last], mag[first:last], dtype, 9)


@pytest.mark.parametrize("c", [64, 40, 33, 1])
def test_views_of_quantised_images(c):
    """Crops, every second row, and a transposition of quantise_tokens' codes walk memory at no single pitch: they are copied, whatever the
    number of channels."""
    torch.manual_seed(c)
    codes, scales = int8.quantize_tokens(torch.randn(2, 9, 10, c, device="cuda"))
    wc, wm = int8.quantize_weight(torch.randn(24, 3, 3, c, device="cuda")), int8.quantize_weight(torch.randn(24, c, device="cuda"))
    for view in (lambda t: t[:, 1:-1, 1:-1], lambda t: t[:, ::2], lambda t: t.transpose(1, 2), lambda t: t[:, :, ::3], lambda t: t[:1, 2:3], lambda t: t[:, 3:4, 5:6]):
        q, s = view(codes), view(scales)
        whole = torch.zeros(*q.shape[:-1], (c + 15) // 16 * 16, dtype=torch.int8, device="cuda")
        whole[..., :c] = q
        for call, w in ((int8.conv3x3, wc), (int8.matmul, wm)):
            assert torch.equal(call(q, s, w, dtype=torch.float32), call(whole[..., :c], s.contiguous(), w, dtype=torch.float32))


@pytest.mark.parametrize("c", [64, 40])
def test_rows_farther_apart_than_the_kernels_take(c):
    """A few channels of very wide matrices: x, codes and the residual are copied where their rows lie beyond the kernels' pitches."""
    torch.manual_seed(c)
    weight = int8.quantize_weight(torch.randn(24, c, device="cuda"))
    x = torch.zeros(3, (1 << 24) + 16, dtype=torch.bfloat16, device="cuda")[:, 8:8 + c]
    x.normal_()
    codes, scales = int8.quantize_tokens(x)
    want = int8.quantize_tokens(x.contiguous())
    assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])
    far = torch.full((3, (1 << 22) + 16), 99, dtype=torch.int8, device="cuda")[:, 16:16 + c]
    far.copy_(codes)
    res = torch.zeros(3, (1 << 24) + 16, dtype=torch.float16, device="cuda")[:, 1:25]
    res.normal_()
    y = int8.matmul(codes, scales, weight, residual=res.contiguous(), dtype=torch.float16)
    assert torch.equal(int8.matmul(far, scales, weight, residual=res, dtype=torch.float16), y)
    assert torch.equal(int8.quantize_tokens(x, x)[1], scales)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("k", [2300, 2700, 4400])
def test_matmul_of_many_rows_with_a_residual(k, dtype):
    """Both sides of the sums from which the widest tiles take odd rows and residuals."""
    test_matmul(12301, k, 1025, dtype)


def test_a_float16_token_has_the_same_product_in_any_batch():
    """float16 too: the float32 sum is rounded before it is rounded to half, in every kernel."""
    test_a_token_has_the_same_product_in_any_batch(torch.float16)
