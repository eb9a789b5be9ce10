"""GPU: microscaled 4-bit packing and products against 64-bit references."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ref_pack(x):
    """(values (n, k) float64, scale bytes (n, 4P)) of x, by comparison with the grid's midpoints."""
    x = x.detach().cpu().double().numpy()
    n, k = x.shape
    p = (k + 127) // 128
    b = np.zeros((n, p * 128))
    b[:, :k] = x
    b = b.reshape(n, -1, 32)
    bad = ~np.isfinite(b).all(-1)
    top = np.abs(np.where(bad[..., None], 0, b)).max(-1)
    _, e = np.frexp(top)
    e = np.where(top > 0, np.maximum(e - 3, -127), -127)
    a = np.abs(np.where(bad[..., None], 0, b)) * np.exp2(-e.astype(float))[..., None]
    lo = np.clip(np.searchsorted(GRID, a, side="right") - 1, 0, 7)
    hi = np.minimum(lo + 1, 7)
    up = (a - GRID[lo] > GRID[hi] - a) | ((a - GRID[lo] == GRID[hi] - a) & (hi % 2 == 0))
    v = np.copysign(np.where(up, GRID[hi], GRID[lo]), b) * np.exp2(e.astype(float))[..., None]
    v[bad] = np.nan
    return v.reshape(n, -1)[:, :k], np.where(bad, 255, e + 127)


def same(got, want):
    got = got.cpu().double().numpy()
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want))
    fine = ~np.isnan(want)
    assert np.array_equal(got[fine], want[fine])
    assert np.array_equal(np.signbit(got[fine]), np.signbit(want[fine]))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("n,k", [(1, 1), (1, 31), (3, 32), (5, 33), (17, 127), (16, 128), (1000, 129), (33, 960), (2, 1000)])
def test_pack_values(n, k, dtype):
    from lira_amd import mx4_quantize
    x = (torch.randn(n, k, generator=gen(n * k), device="cuda") * torch.exp(3 * torch.randn(n, 1, generator=gen(1), device="cuda"))).to(DT[dtype])
    t = mx4_quantize(x)
    want, scale = ref_pack(x)
    assert t.shape == (n, k) and t.codes.shape == ((k + 127) // 128, n, 64)
    assert np.array_equal(t.scales.cpu().numpy().transpose(1, 0, 2).reshape(n, -1), scale)
    same(t.dequantize(torch.float32), want)


def test_pack_ties_and_extremes():
    from lira_amd import mx4_quantize
    x = torch.zeros(12, 128)
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.9])
    x[0, :8], x[0, 32:40], x[0, 64:72] = ties, -ties * 2 ** -20, ties * 2 ** 60
    x[1, :8] = torch.nextafter(ties, torch.zeros(8))
    x[2, :8] = torch.nextafter(ties, torch.full((8,), 9.0))
    x[3, 5] = -0.0
    x[4, :4] = torch.tensor([2.0 ** -149, 2.0 ** -148, -2.0 ** -140, 2.0 ** -130])  # below the normal range
    x[5, :4] = torch.tensor([2.0 ** -126, 1.5 * 2.0 ** -126, 2.0 ** -124, -2.0 ** -125])
    x[6, :4] = torch.tensor([3.4028234e38, -3.4028234e38, 2.0 ** 127, 2.0 ** 100])
    x[7, 1], x[7, 33], x[7, 70] = float("nan"), float("inf"), float("-inf")
    x[8] = 7.999
    x[9] = torch.linspace(-6, 6, 128)
    x[10, 64:] = 2.0 ** -127
    x[11, :32] = torch.linspace(2.0 ** -128, 2.0 ** -123, 32)
    t = mx4_quantize(x.cuda())
    want, scale = ref_pack(x)
    assert np.array_equal(t.scales.cpu().numpy()[0], scale)
    same(t.dequantize(torch.float32), want)
    assert not t.codes[0, 7, :48].any()  # (codes of a NaN block are 0)


def test_views_of_a_packed_tensor():
    from lira_amd import MX4Tensor, mx4_linear, mx4_quantize
    x = torch.randn(50, 300, generator=gen(4), device="cuda")
    t = mx4_quantize(x)
    assert t.codes.shape == (3, 50, 64) and t.scales.shape == (3, 50, 4) and t.nbytes() == 3 * 50 * 68 and len(t) == 50
    assert t.codes.data_ptr() == t.codes_ptr and t.scales.data_ptr() == t.scales_ptr and t.device == x.device
    want, _ = ref_pack(x)
    same(MX4Tensor(t.codes, t.scales, 300).dequantize(), want)
    same(t[10:10].dequantize(), want[10:10])
    same(t[49:].dequantize(), want[49:])
    same(t[5:40][3:4].dequantize(), want[8:9])
    # parts whose rows are spaced differently, or that lie apart, are brought together
    wide = torch.zeros(3, 50, 80, dtype=torch.uint8, device="cuda")
    wide[..., 16:] = t.codes
    same(MX4Tensor(wide[..., 16:], t.scales, 300).dequantize(), want)
    q = torch.randn(3, 300, generator=gen(5), device="cuda")
    assert torch.equal(mx4_linear(q, t[7:30]), mx4_linear(q, mx4_quantize(x[7:30])))


def every_code():
    """All 16 codes under all 256 scales: (256, 128) packed rows and their values in 64 bits."""
    codes = torch.zeros(1, 256, 64, dtype=torch.uint8)
    codes[0, :, :8] = torch.arange(8, dtype=torch.uint8) * 2 + (torch.arange(8, dtype=torch.uint8) * 2 + 1) * 16
    scales = torch.arange(256, dtype=torch.uint8)[None, :, None].expand(1, 256, 4).contiguous()
    v = np.zeros((256, 128))
    v[:, :16] = np.concatenate([GRID, -GRID]) * np.exp2(np.arange(256.0) - 127)[:, None]
    v[:, 16:] = 0
    v[255] = np.nan
    return codes.cuda(), scales.cuda(), v


@pytest.mark.parametrize("dtype", list(DT))
def test_unpack_every_code_and_scale(dtype):
    from lira_amd import MX4Tensor
    codes, scales, v = every_code()
    for k in (128, 77):
        want = torch.from_numpy(v[:, :k]).float().to(DT[dtype])  # (one rounding: fp32 holds every value but 6 * 2^127 and its like)
        same(MX4Tensor(codes, scales, k).dequantize(DT[dtype]), want.double().numpy())


@pytest.mark.parametrize("offset,step", [(0, 1), (1, 1), (3, 1), (0, 2), (5, 3)])
@pytest.mark.parametrize("dtype", list(DT))
def test_pack_strided_rows(dtype, offset, step):
    from lira_amd import mx4_quantize
    base = torch.randn(40, 300, generator=gen(offset), device="cuda").to(DT[dtype])
    x = base[::step, offset:offset + 201]
    same(mx4_quantize(x).dequantize(torch.float32), ref_pack(x)[0])
    y = base.t()  # (rows that are not runs of elements are copied first)
    same(mx4_quantize(y).dequantize(torch.float32), ref_pack(y)[0])


def test_unpack_leaves_the_rest_of_out():
    from lira_amd import mx4_quantize
    x = torch.randn(19, 130, generator=gen(2), device="cuda")
    out = torch.full((21, 140), 7.0, device="cuda")
    t = mx4_quantize(x)
    t.dequantize(torch.float32, out=out[1:20, 3:133])
    want, _ = ref_pack(x)
    same(out[1:20, 3:133], want)
    out[1:20, 3:133] = 7.0
    assert bool((out == 7.0).all())
    same(t[5:9].dequantize(torch.float32), want[5:9])


def ref_product(av, bv, alpha, bias, act):
    """The product in 64 bits and the sum of its terms' magnitudes."""
    y = alpha * (av @ bv.T) + (0 if bias is None else bias)
    mag = abs(alpha) * (np.abs(av) @ np.abs(bv).T) + (0 if bias is None else np.abs(bias))
    if act == "relu":
        y = np.maximum(y, 0)
    if act == "sigmoid":
        y = 1 / (1 + np.exp(-y))
    return y, mag


def check_product(got, av, bv, alpha, bias, act, dtype):
    """fp32 sums: every one of the k / 32 block sums and the epilogue's two operations may lose 2^-22 of
    the magnitudes' sum (a matrix instruction's adds need not round to nearest); a sigmoid passes a
    quarter of it on and its own exp and division lose 2^-20; then one rounding to the output's type."""
    want, mag = ref_product(av, bv, alpha, bias, act)
    k = av.shape[1]
    tol = (k / 32 + 4) * 2.0 ** -22 * mag
    if act == "sigmoid":
        tol = tol / 4 + 2.0 ** -20
    tol = tol + torch.finfo(dtype).eps / 2 * (np.abs(want) + tol) + torch.finfo(dtype).tiny
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= tol).all(), (err / tol).max()


SHAPES = [(1, 1, 1), (1, 16, 128), (1, 33, 500), (2, 100, 96), (7, 257, 1000), (15, 64, 129), (16, 31, 256), (17, 130, 384),
          (33, 1000, 960), (64, 64, 64), (65, 65, 4097), (100, 1, 128), (128, 256, 512), (129, 300, 1152), (257, 513, 130),
          (300, 1024, 128), (2100, 2111, 390), (4111, 4113, 260), (1000, 255, 2049), (1, 5000, 128), (3, 4099, 8192), (48, 2000, 3000),
          (1, 65600, 1100), (3, 70001, 1024), (9, 65537, 1030), (2, 30011, 700), (4, 8200, 4100), (1, 20000, 1100), (16, 66000, 100)]  # (columns enough for a loop of groups)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear(m, n, k, dtype):
    from lira_amd import mx4_linear, mx4_matmul, mx4_quantize
    dt = DT[dtype]
    g = gen(m + n + k)
    x = torch.randn(m, k, generator=g, device="cuda").to(dt)
    w = mx4_quantize(torch.randn(n, k, generator=g, device="cuda") * k ** -0.5)
    bias = torch.randn(n, generator=g, device="cuda")
    xv, wv = ref_pack(x)[0], w.dequantize().double().cpu().numpy()
    for b, act, alpha in ((None, None, 1.0), (bias, "relu", -0.5), (bias, "sigmoid", 2.0)):
        bv = None if b is None else b.double().cpu().numpy()
        check_product(mx4_linear(x, w, b, act, alpha), xv, wv, alpha, bv, act, dt)
        check_product(mx4_matmul(mx4_quantize(x), w, b, act, alpha, out_dtype=dt), xv, wv, alpha, bv, act, dt)


# (one of every tile, in the order of the kernels' list; then rows that the product packs by itself, and that it no longer does)
@pytest.mark.parametrize("m,n,k", [(17, 700, 2000), (20, 9000, 4000), (50, 9001, 4000), (20, 20001, 300), (60, 20001, 300),
                                   (130, 20001, 40), (65, 65537, 2000), (700, 20001, 1000), (16, 1000, 2048), (5, 8200, 4096),
                                   (12, 40000, 2000), (13, 70001, 900), (16, 9000, 1700), (9, 300, 3600), (6, 501, 5000)])
@pytest.mark.parametrize("dtype", list(DT))
def test_linear_by_every_tile(m, n, k, dtype):
    from lira_amd import mx4_linear, mx4_matmul, mx4_quantize
    g = gen(m + n + k)
    x = torch.randn(m, k, generator=g, device="cuda").to(DT[dtype])
    w = mx4_quantize(torch.randn(n, k, generator=g, device="cuda") * k ** -0.5)
    bias = torch.randn(n, generator=g, device="cuda")
    xv, wt = mx4_quantize(x).dequantize().double(), w.dequantize().double().t().contiguous()
    want, mag = 0.5 * (xv @ wt) + bias, 0.5 * (xv.abs() @ wt.abs()) + bias.abs()
    tol = (k / 32 + 4) * 2.0 ** -22 * mag  # (as in check_product)
    tol = tol + torch.finfo(DT[dtype]).eps / 2 * (want.abs() + tol) + torch.finfo(DT[dtype]).tiny
    for got in (mx4_linear(x, w, bias, alpha=0.5), mx4_matmul(mx4_quantize(x), w, bias, alpha=0.5, out_dtype=DT[dtype])):
        err = (got.double() - want).abs()
        assert bool((err <= tol).all()), float((err / tol).max())


# (rows packed by the product itself or by a launch of their own: the same numbers in the same order, so the same bits)
@pytest.mark.parametrize("m,n,k", [(17, 64, 8), (17, 1, 8), (17, 130, 16), (64, 257, 128), (65, 129, 96), (1000, 333, 104), (300, 200, 256), (129, 1000, 248),
                                   (40, 9001, 136), (4000, 64, 200), (20, 100001, 64), (64, 64, 8), (16, 70, 2000), (10, 40000, 2000)])
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("dtype", list(DT))
def test_rows_packed_inside(m, n, k, offset, dtype):
    from lira_amd import mx4_linear, mx4_matmul, mx4_quantize
    g = gen(m + n + k)
    room = torch.full((m, k + 11 * offset), float("nan"), device="cuda", dtype=DT[dtype])
    x = room[:, offset:offset + k]
    x.copy_(torch.randn(m, k, generator=g, device="cuda") * torch.exp(4 * torch.randn(m, 1, generator=g, device="cuda")))
    if m > 20:
        x[3, k // 2] = float("inf")
        x[5] = 0
    w = mx4_quantize(torch.randn(n, k, generator=g, device="cuda"))
    out = torch.full((m + 1, n + 3), 7.0, device="cuda", dtype=DT[dtype])
    mx4_linear(x, w, out=out[:m, :n])
    want = mx4_matmul(mx4_quantize(x), w, out_dtype=DT[dtype])
    assert torch.equal(out[:m, :n].nan_to_num(nan=-1.0), want.nan_to_num(nan=-1.0))
    assert bool((out[m] == 7).all()) and bool((out[:, n:] == 7).all())
    if m > 20:
        assert bool(out[3, :n].isnan().all()) and not bool(out[5, :n].any())


@pytest.mark.parametrize("m,n", [(0, 40), (40, 0), (0, 0)])
def test_linear_of_nothing(m, n):
    from lira_amd import mx4_linear, mx4_quantize
    x = torch.randn(m, 70, device="cuda")
    w = mx4_quantize(torch.randn(n, 70, device="cuda"))
    assert w.shape == (n, 70) and w.dequantize().shape == (n, 70)
    assert mx4_linear(x, w, torch.zeros(n, device="cuda")).shape == (m, n)


@pytest.mark.parametrize("m", [1, 5, 40, 200])
def test_linear_strides_and_views(m):
    """Odd row strides of input and output, a row range of the packed operand, what lies round the output."""
    from lira_amd import mx4_linear, mx4_quantize
    g = gen(m)
    x = torch.randn(m, 411, generator=g, device="cuda").bfloat16()[:, 3:404]
    w = mx4_quantize(torch.randn(90, 401, generator=g, device="cuda"))
    out = torch.full((m + 2, 80), 7.0, device="cuda", dtype=torch.bfloat16)
    view = out[1:m + 1, 5:72]
    got = mx4_linear(x, w[11:78], out=view)
    assert got.data_ptr() == view.data_ptr()
    check_product(view, ref_pack(x)[0], w.dequantize()[11:78].double().cpu().numpy(), 1.0, None, None, torch.bfloat16)
    view.fill_(7.0)
    assert bool((out == 7.0).all())


@pytest.mark.parametrize("m", [1, 3, 20, 70, 300])
def test_linear_nan_rows_stay_apart(m):
    """NaN and Inf make their own row (or column) NaN and no other."""
    from lira_amd import mx4_linear, mx4_quantize
    g = gen(m)
    x = torch.randn(m, 300, generator=g, device="cuda")
    w = torch.randn(150, 300, generator=g, device="cuda")
    x[m // 2, 299] = float("inf")
    w[7, 0] = float("nan")
    y = mx4_linear(x, mx4_quantize(w))
    nan = torch.zeros_like(y, dtype=torch.bool)
    nan[m // 2], nan[:, 7] = True, True
    assert torch.equal(torch.isnan(y), nan)


@pytest.mark.parametrize("m", [1, 4, 40, 130])
def test_linear_far_apart_scales(m):
    """Blocks whose scales differ by 2^40 keep the large one's sum exact to fp32."""
    from lira_amd import mx4_linear, mx4_quantize
    g = gen(m)
    x = torch.randn(m, 512, generator=g, device="cuda")
    x[:, 128:160] *= 2.0 ** 20
    w = torch.randn(70, 512, generator=g, device="cuda")
    w[:, 128:160] *= 2.0 ** 20
    w = mx4_quantize(w)
    check_product(mx4_linear(x, w), ref_pack(x)[0], w.dequantize().double().cpu().numpy(), 1.0, None, None, torch.float32)


@pytest.mark.parametrize("m,n,k", [(1, 8192, 8192), (16, 4096, 4096), (300, 700, 1000), (64, 512, 2048)])
def test_linear_repeats_bit_for_bit(m, n, k):
    from lira_amd import mx4_linear, mx4_quantize
    x = torch.randn(m, k, generator=gen(0), device="cuda").bfloat16()
    w = mx4_quantize(torch.randn(n, k, generator=gen(1), device="cuda"))
    first = mx4_linear(x, w)
    for _ in range(5):
        assert torch.equal(mx4_linear(x, w), first)


def test_linear_on_a_stream_and_in_a_graph():
    from lira_amd import mx4_linear, mx4_quantize
    g = gen(3)
    xs = [torch.randn(50, 700, generator=g, device="cuda") for _ in range(4)]
    w = mx4_quantize(torch.randn(333, 700, generator=g, device="cuda"))
    b = torch.randn(333, generator=g, device="cuda")
    want = [mx4_linear(x, w, b, "relu") for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = [mx4_linear(x, w, b, "relu", stream=side) for x in xs]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, c in zip(got, want):
        assert torch.equal(a, c)
    x = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t = mx4_quantize(x)
        y = mx4_linear(x, w, b, "relu")
        v = t.dequantize()
    for i in (1, 2, 3, 0, 2):
        x.copy_(xs[i])
        graph.replay()
        eager = mx4_linear(xs[i], w, b, "relu")  # (the program's own work between replays)
        torch.cuda.synchronize()
        assert torch.equal(y, want[i]) and torch.equal(eager, want[i])
        assert torch.equal(v, mx4_quantize(xs[i]).dequantize())


def test_many_rows():
    """More rows than a grid's second dimension would hold tiles of 16."""
    from lira_amd import mx4_linear, mx4_quantize
    g = gen(6)
    x = torch.randn(1 << 21, 40, generator=g, device="cuda").bfloat16()
    w = mx4_quantize(torch.randn(20, 40, generator=g, device="cuda"))
    y = mx4_linear(x, w)
    at = torch.tensor([0, 1, 77777, (1 << 20) + 5, (1 << 21) - 2, (1 << 21) - 1], device="cuda")
    check_product(y[at], ref_pack(x[at])[0], w.dequantize().double().cpu().numpy(), 1.0, None, None, torch.bfloat16)


def test_more_than_2_31_elements():
    from lira_amd import mx4_linear, mx4_quantize
    g = gen(5)
    n = (1 << 31) // 128 + 100
    x = torch.zeros(n, 128, dtype=torch.bfloat16, device="cuda")
    x[-50:] = torch.randn(50, 128, generator=g, device="cuda").bfloat16()
    t = mx4_quantize(x)
    same(t[n - 50:].dequantize(), ref_pack(x[-50:])[0])
    same(t.dequantize(torch.bfloat16)[-50:], ref_pack(x[-50:])[0])
    del x
    q = torch.randn(3, 128, generator=g, device="cuda")
    y = mx4_linear(q, t)
    assert not y[:, :-50].any()
    check_product(y[:, -50:], ref_pack(q)[0], t[n - 50:].dequantize().double().cpu().numpy(), 1.0, None, None, torch.float32)
    del t, y
    m = (1 << 31) // 65536 + 70  # a result of more than 2^31 elements
    a = torch.randn(m, 64, generator=g, device="cuda").bfloat16()
    w = mx4_quantize(torch.randn(65536, 64, generator=g, device="cuda"))
    y = mx4_linear(a, w)
    check_product(y[-3:], ref_pack(a[-3:])[0], w.dequantize().double().cpu().numpy(), 1.0, None, None, torch.bfloat16)


def test_refusals():
    from lira_amd import MX4Tensor, mx4_linear, mx4_matmul, mx4_quantize
    x = torch.randn(4, 200, device="cuda")
    w = mx4_quantize(torch.randn(9, 200, device="cuda"))
    for call, text in ((lambda: mx4_quantize(x.double()), "float32"), (lambda: mx4_quantize(x[0]), "2 dimensions"),
                       (lambda: mx4_quantize(x[:, :0]), "column"), (lambda: mx4_linear(x[:, :100], w), "columns"),
                       (lambda: mx4_linear(x, w, torch.zeros(8, device="cuda")), "bias"), (lambda: mx4_linear(x, w, torch.zeros(9)), "bias"),
                       (lambda: mx4_linear(x, w, activation="gelu"), "activation"), (lambda: mx4_linear(x, w, out_dtype=torch.int8), "out_dtype"),
                       (lambda: mx4_linear(x, w, out=torch.zeros(4, 8, device="cuda")), "out"),
                       (lambda: mx4_linear(x, w, out=torch.zeros(9, 4, device="cuda").t()), "out"),
                       (lambda: mx4_linear(x, w, out=torch.zeros(1, 9, device="cuda").expand(4, 9)), "out"),
                       (lambda: mx4_matmul(mx4_quantize(x[:, :100]), w), "columns"),
                       (lambda: MX4Tensor(w.codes, w.scales, 257), "planes"), (lambda: MX4Tensor(w.codes, w.scales[:, :8], 200), "same"),
                       (lambda: MX4Tensor(w.codes.int(), w.scales, 200), "uint8"),
                       (lambda: mx4_quantize(x.clone().requires_grad_()), "gradient"),
                       (lambda: mx4_linear(x.clone().requires_grad_(), w), "gradient"),
                       (lambda: w.dequantize(torch.float64), "dtype")):
        with pytest.raises(ValueError, match=text):
            call()
    buf = torch.randn(4, 409, device="cuda")
    with pytest.raises(ValueError, match="share memory"):
        mx4_linear(buf[:, :200], w, out=buf[:, 200:209])  # (between the rows: the spans overlap)
    with pytest.raises(ValueError, match="share memory"):
        mx4_linear(x, w, out=x.view(-1)[:36].view(4, 9))
    with pytest.raises(TypeError):
        w[::2]
    with torch.no_grad():
        assert mx4_linear(x.clone().requires_grad_(), w).shape == (4, 9)
