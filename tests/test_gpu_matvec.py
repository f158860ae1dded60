"""Products of 4-bit matrices (frc_matrix_open, frc_matvec_device) against float64.

Tolerance.  With A = sum_j a_j |x_j| (a_j: the size of weight j's terms, Q4_K: |d sc q| + |dmin mi|), an fp32 sum
of n terms that is formed 16 terms at a time and truncated at each step is off by at most 2 n/16 steps of 2^-23 A,
plus two roundings for every 256 weights' scales and 16 for joining the parts: (n/8 + n/128 + 16) 2^-23 A.  The
vector may be carried with 22 significant bits (2^-23 A, inside the 16), and not below 2^-34 of the largest value in
its span of 256 weights: + 2^-34 sum_j a_j max|x|.  A bf16 result adds half a step, 2^-8 of the value."""
import ctypes

import numpy as np
import pytest

import fronk_b200 as fb
from tests import quant

pytestmark = pytest.mark.gpu


def bound(a, x, n):
    spans = -(-n // 256) * 256
    xp = np.zeros((x.shape[0], spans))
    xp[:, :n] = np.abs(x)
    top = np.repeat(xp.reshape(x.shape[0], -1, 256).max(-1), 256, axis=1)[:, :n]
    return (n / 8 + n / 128 + 16) * 2.0 ** -23 * (np.abs(x) @ a.T) + 2.0 ** -34 * (top @ a.T)


def to_device(x, dtype):
    import torch
    t = torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda()
    return t.to(torch.bfloat16 if dtype == fb.BF16 else torch.float32)


def host(t):
    return t.float().cpu().numpy().astype(np.float64)


def check(y, x, w, a, n, y_type):
    ref = x @ w.T
    tol = bound(a, x, n) + (2.0 ** -8 * np.abs(ref) if y_type == fb.BF16 else 0)
    err = np.abs(y - ref)
    assert np.all(err <= tol), (err / tol).max()


@pytest.fixture(scope="module")
def ctx(gpu):
    with fb.Context(0, 512) as c:
        yield c


def run(ctx, type_, raw, n, xd, x_type, y_type, x_stride=None, y_stride=None):
    import torch
    rows, tokens = raw.shape[0], xd.shape[0]
    y = torch.full((tokens, rows), float("nan"), dtype=torch.bfloat16 if y_type == fb.BF16 else torch.float32,
                   device="cuda")
    with ctx.matrix(type_, rows, n, raw) as m:
        m.matvec_device(tokens, xd.data_ptr(), y.data_ptr(), x_type, y_type, x_stride, y_stride,
                        torch.cuda.current_stream().cuda_stream)
        assert ctx.status(torch.cuda.current_stream().cuda_stream) == fb.OK
    return y


SHAPES = [(fb.Q4_K, 1, 256), (fb.Q4_K, 15, 512), (fb.Q4_K, 17, 2304), (fb.Q4_K, 513, 2048), (fb.Q4_K, 130, 8192),
          (fb.Q4_K, 5000, 256), (fb.MXFP4, 1, 32), (fb.MXFP4, 16, 64), (fb.MXFP4, 33, 288), (fb.MXFP4, 513, 2048),
          (fb.MXFP4, 75, 4192), (fb.MXFP4, 3, 16384), (fb.MXFP4, 2051, 672)]


@pytest.mark.parametrize("type_,rows,n", SHAPES)
@pytest.mark.parametrize("tokens", [1, 2, 3, 4, 5, 8, 9, 16])
def test_shapes(ctx, type_, rows, n, tokens):
    rng = np.random.default_rng(rows * 1000 + n + tokens)
    raw = quant.random_rows(type_, rows, n, rng)
    w, a = quant.weights(type_, raw, n)
    x = rng.standard_normal((tokens, n))
    for x_type, y_type in [(fb.F32, fb.F32), (fb.BF16, fb.BF16), (fb.F32, fb.BF16), (fb.BF16, fb.F32)]:
        xd = to_device(x, x_type)
        y = run(ctx, type_, raw, n, xd, x_type, y_type)
        check(host(y), host(xd), w, a, n, y_type)


@pytest.mark.parametrize("type_,n", [(fb.Q4_K, 256), (fb.Q4_K, 2304), (fb.Q4_K, 5120), (fb.MXFP4, 32), (fb.MXFP4, 672),
                                     (fb.MXFP4, 2560)])
@pytest.mark.parametrize("tokens", [5, 8, 9, 16])
def test_bursts_of_many_rows(ctx, type_, n, tokens):
    """Bursts of five tokens and more over matrices of many rows; rows between the runs of the CTAs, odd strides."""
    import torch
    rows = 19111
    rng = np.random.default_rng(n + tokens)
    base = quant.random_rows(type_, 509, n, rng)
    raw = np.tile(base, (rows // 509 + 1, 1))[:rows]
    w, a = quant.weights(type_, base, n)
    for x_type, y_type in [(fb.F32, fb.F32), (fb.BF16, fb.BF16)]:
        xb = torch.full((tokens, n + 3), float("nan"), dtype=torch.bfloat16 if x_type == fb.BF16 else torch.float32, device="cuda")
        xb[:, :n] = to_device(rng.standard_normal((tokens, n)), x_type)
        yb = torch.full((tokens, rows + 1), -7.0, dtype=torch.bfloat16 if y_type == fb.BF16 else torch.float32, device="cuda")
        s = torch.cuda.current_stream().cuda_stream
        with ctx.matrix(type_, rows, n, raw) as m:
            m.matvec_device(tokens, xb.data_ptr(), yb.data_ptr(), x_type, y_type, n + 3, rows + 1, s)
            assert ctx.status(s) == fb.OK
            first = yb.clone()
            m.matvec_device(tokens, xb.data_ptr(), yb.data_ptr(), x_type, y_type, n + 3, rows + 1, s)
            assert ctx.status(s) == fb.OK and torch.equal(first, yb)
        assert bool((yb[:, rows] == -7).all())
        y, x = host(yb[:, :rows]), host(xb[:, :n])
        for r in range(0, rows, 509):
            k = min(509, rows - r)
            check(y[:, r:r + k], x, w[:k], a[:k], n, y_type)


def test_bursts_with_scales_far_apart(ctx):
    """MXFP4 rows whose exponents differ by more than fp16 holds, in a matrix of many rows."""
    n, rows, tokens = 512, 19000, 7
    rng = np.random.default_rng(77)
    base = quant.random_rows(fb.MXFP4, 100, n, rng, exponents=(90, 127))
    raw = np.tile(base, (rows // 100, 1))
    w, a = quant.weights(fb.MXFP4, base, n)
    x = rng.standard_normal((tokens, n))
    x[3, :480] = 0  # only one block of each row counts
    xd = to_device(x, fb.F32)
    y = host(run(ctx, fb.MXFP4, raw, n, xd, fb.F32, fb.F32))
    for r in range(0, rows, 100):
        check(y[:, r:r + 100], host(xd), w, a, n, fb.F32)


@pytest.mark.parametrize("type_", [fb.Q4_K, fb.MXFP4])
@pytest.mark.parametrize("tokens,x_type", [(1, fb.F32), (4, fb.BF16), (16, fb.F32)])
def test_long_rows(ctx, type_, tokens, x_type):
    """The longest rows: the vectors do not fit a CTA's shared memory as a whole."""
    n, rows = 65536 - (0 if type_ == fb.Q4_K else 96), 300
    rng = np.random.default_rng(tokens)
    raw = quant.random_rows(type_, rows, n, rng)
    w, a = quant.weights(type_, raw, n)
    xd = to_device(rng.standard_normal((tokens, n)), x_type)
    y = run(ctx, type_, raw, n, xd, x_type, fb.F32)
    check(host(y), host(xd), w, a, n, fb.F32)


@pytest.mark.parametrize("type_,rows", [(fb.Q4_K, 70001), (fb.MXFP4, 65537)])
def test_many_rows(ctx, type_, rows):
    """More row tiles than the GPU holds at a time.  Blocks of equal rows: each is held to the bound, which counts an
    fp32 rounding for every addition of a span's or a part's sum whatever the order, so it covers a tile whose spans
    two warps share (the parts are added to one another) and one that a warp sums alone; the two may differ in the last
    bits, the same call twice may not."""
    rng = np.random.default_rng(rows)
    n = 512
    raw = np.tile(quant.random_rows(type_, 257, n, rng), (rows // 257 + 1, 1))[:rows]
    w, a = quant.weights(type_, raw[:257], n)
    for tokens in (1, 7, 16):
        xd = to_device(rng.standard_normal((tokens, n)), fb.F32)
        y = host(run(ctx, type_, raw, n, xd, fb.F32, fb.F32))
        for r in range(0, rows, 257):
            k = min(257, rows - r)
            check(y[:, r:r + k], host(xd), w[:k], a[:k], n, fb.F32)
        again = host(run(ctx, type_, raw, n, xd, fb.F32, fb.F32))
        assert np.array_equal(again, y)


def test_offsets_past_32_bits(ctx):
    """A matrix of more than 4 GiB (rows given on the device): its first and last rows."""
    import torch
    rows, n = 130001, 65536
    rng = np.random.default_rng(8)
    few = quant.random_rows(fb.MXFP4, 64, n, rng)
    w, a = quant.weights(fb.MXFP4, few, n)
    raw = torch.zeros(rows, few.shape[1], dtype=torch.uint8, device="cuda")
    raw[:32] = torch.from_numpy(few[:32]).cuda()
    raw[-32:] = torch.from_numpy(few[32:]).cuda()
    raw[32:-32, ::17] = 120
    assert raw.numel() > 1 << 32
    torch.cuda.synchronize()
    s = torch.cuda.current_stream().cuda_stream
    with ctx.matrix(fb.MXFP4, rows, n, raw.data_ptr(), raw.numel()) as m:
        for tokens in (1, 6):
            xd = to_device(rng.standard_normal((tokens, n)), fb.F32)
            y = torch.full((tokens, rows), float("nan"), device="cuda")
            m.matvec_device(tokens, xd.data_ptr(), y.data_ptr(), stream=s)
            assert ctx.status(s) == fb.OK
            got = host(torch.cat([y[:, :32], y[:, -32:]], 1))
            check(got, host(xd), w, a, n, fb.F32)
            assert not bool(y[:, 32:-32].any())


@pytest.mark.parametrize("type_", [fb.Q4_K, fb.MXFP4])
@pytest.mark.parametrize("x_type,y_type", [(fb.F32, fb.F32), (fb.BF16, fb.BF16)])
def test_strides_and_alignment(ctx, type_, x_type, y_type):
    """Odd row strides, x and y that start on an odd element; what lies between the rows of y stays."""
    import torch
    rng = np.random.default_rng(11)
    rows, n, tokens = 45, 768, 5
    raw = quant.random_rows(type_, rows, n, rng)
    w, a = quant.weights(type_, raw, n)
    dt = torch.bfloat16 if x_type == fb.BF16 else torch.float32
    xb = torch.full((1 + tokens * (n + 3),), float("nan"), dtype=dt, device="cuda")
    xv = xb[1:].view(tokens, n + 3)
    xv[:, :n] = to_device(rng.standard_normal((tokens, n)), x_type)
    yb = torch.full((1 + tokens * (rows + 2),), -7.0, dtype=torch.bfloat16 if y_type == fb.BF16 else torch.float32,
                    device="cuda")
    yv = yb[1:].view(tokens, rows + 2)
    s = torch.cuda.current_stream().cuda_stream
    with ctx.matrix(type_, rows, n, raw) as m:
        m.matvec_device(tokens, xv.data_ptr(), yv.data_ptr(), x_type, y_type, n + 3, rows + 2, s)
        assert ctx.status(s) == fb.OK
    check(host(yv[:, :rows]), host(xv[:, :n]), w, a, n, y_type)
    assert bool((yv[:, rows:] == -7).all()) and float(yb[0]) == -7


@pytest.mark.parametrize("tokens", [1, 3, 16])
def test_range_of_values(ctx, tokens):
    """Spans of very different size in one vector, single large and tiny values, rows of zeros."""
    rng = np.random.default_rng(3)
    for type_, n in [(fb.Q4_K, 1536), (fb.MXFP4, 1440)]:
        raw = quant.random_rows(type_, 40, n, rng)
        w, a = quant.weights(type_, raw, n)
        x = rng.standard_normal((tokens, n)).astype(np.float32)
        x[:, :256] *= 1e-18
        x[:, 256:512] *= 1e12
        x[:, 512:768] = 0
        x[0, 800] = 3e4
        x[0, 900] = 1e-39  # subnormal
        if tokens > 1:
            x[1] = 0
            x[2] *= 1e-30
        xd = to_device(x, fb.F32)
        y = host(run(ctx, type_, raw, n, xd, fb.F32, fb.F32))
        xr = host(xd)
        ref, tol = xr @ w.T, bound(a, xr, n) + 2.0 ** -126  # results below the normal range may be flushed
        assert np.all(np.abs(y - ref) <= tol), (np.abs(y - ref) / tol).max()


def test_scales_at_the_border(ctx):
    """Q4_K super scales that are subnormal, zero or large; MXFP4 exponents far apart in one row, 0 and 200."""
    rng = np.random.default_rng(4)
    n = 768
    raw = quant.random_rows(fb.Q4_K, 48, n, rng)
    b = raw.reshape(48, 3, 144)
    b[:8, :, :4] = np.array([2 ** -24, 2 ** -20], np.float16).view(np.uint8)
    b[8:16, :, :4] = 0
    b[16:24, :, :4] = np.array([60000, -60000], np.float16).view(np.uint8)
    b[24:32, :, 4:16] = 255  # all scales and minima 63
    b[32:40, :, 4:16] = 0
    w, a = quant.weights(fb.Q4_K, raw, n)
    xd = to_device(rng.standard_normal((2, n)), fb.F32)
    check(host(run(ctx, fb.Q4_K, raw, n, xd, fb.F32, fb.F32)), host(xd), w, a, n, fb.F32)

    raw = quant.random_rows(fb.MXFP4, 48, n, rng)
    b = raw.reshape(48, 24, 17)
    b[:8, :, 0] = rng.integers(60, 180, (8, 24))
    b[8:16, :, 0] = 0
    b[16:24, :, 0] = 200
    b[24:32, ::2, 0] = 1
    b[32:40, :, 1:] = 0x88  # minus zero
    w, a = quant.weights(fb.MXFP4, raw, n)
    xd = to_device(rng.standard_normal((2, n)), fb.F32)
    y, x = host(run(ctx, fb.MXFP4, raw, n, xd, fb.F32, fb.F32)), host(xd)
    tol = bound(a, x, n) + 2.0 ** -126
    assert np.all(np.abs(y - x @ w.T) <= tol)


def test_numeric_status(ctx):
    import torch
    rng = np.random.default_rng(5)
    s = torch.cuda.current_stream().cuda_stream
    for type_ in (fb.Q4_K, fb.MXFP4):
        n, rows = 512, 20
        raw = quant.random_rows(type_, rows, n, rng)
        for value in (float("nan"), float("inf"), -float("inf")):
            x = torch.randn(3, n, device="cuda")
            x[1, 77] = value
            y = torch.zeros(3, rows, device="cuda")
            with ctx.matrix(type_, rows, n, raw) as m:
                m.matvec_device(3, x.data_ptr(), y.data_ptr(), stream=s)
                assert ctx.status(s) == fb.NUMERIC
                good = torch.zeros(2, rows, device="cuda")
                m.matvec_device(2, x[::2].contiguous().data_ptr(), good.data_ptr(), stream=s)
                assert ctx.status(s) == fb.OK
            assert bool(torch.isfinite(y[::2]).all()) and not bool(torch.isfinite(y[1]).all())
        big = torch.full((1, n), 3e38, device="cuda")
        y = torch.zeros(1, rows, device="cuda")
        raw = quant.random_rows(fb.MXFP4, rows, n, rng, exponents=(140, 141))
        with ctx.matrix(fb.MXFP4, rows, n, raw) as m:
            m.matvec_device(1, big.data_ptr(), y.data_ptr(), stream=s)
            assert ctx.status(s) == fb.NUMERIC


def test_refusals(ctx):
    import torch
    rng = np.random.default_rng(6)
    raw = quant.random_rows(fb.Q4_K, 4, 256, rng)

    def refused(code, *args):
        with pytest.raises(fb.FrcError) as e:
            ctx.matrix(*args)
        assert e.value.code == code

    refused(fb.INVALID, fb.Q4_K, 5, 256, raw)
    refused(fb.INVALID, fb.Q4_K, 4, 128, raw)
    refused(fb.UNSUPPORTED, fb.Q8_0, 4, 256, raw)
    for at, v in [(1, 0x7c), (3, 0xfc), (1, 0x7e)]:
        broken = raw.copy()
        broken[3, at] = v
        refused(fb.NUMERIC, fb.Q4_K, 4, 256, broken)
    mx = quant.random_rows(fb.MXFP4, 4, 96, rng)
    mx[2, 34] = 255
    refused(fb.NUMERIC, fb.MXFP4, 4, 96, mx)
    x = torch.zeros(17, 256, device="cuda")
    y = torch.zeros(17, 4, device="cuda")
    before = ctx.launches
    with ctx.matrix(fb.Q4_K, 4, 256, raw) as m:
        opened = ctx.launches
        for kw in [dict(tokens=0), dict(tokens=17), dict(x_type=2), dict(y_type=2), dict(tokens=2, x_stride=255),
                   dict(tokens=2, y_stride=3), dict(x_ptr=None), dict(y_ptr=None), dict(x_ptr=x.data_ptr() + 2),
                   dict(y_ptr=y.data_ptr() + 1, y_type=fb.BF16)]:
            a = dict(tokens=1, x_ptr=x.data_ptr(), y_ptr=y.data_ptr())
            a.update(kw)
            with pytest.raises(fb.FrcError) as e:
                m.matvec_device(**a)
            assert e.value.code == fb.INVALID
        assert ctx.launches == opened > before


def test_device_rows_graph_and_streams(ctx):
    """Rows given in device memory; a captured call that is replayed on new values; two streams at once; the same
    call twice gives the same bits."""
    import torch
    rng = np.random.default_rng(7)
    rows, n = 300, 1024
    raw = quant.random_rows(fb.MXFP4, rows, n, rng)
    w, a = quant.weights(fb.MXFP4, raw, n)
    dev = torch.from_numpy(raw).cuda()
    torch.cuda.synchronize()
    m = ctx.matrix(fb.MXFP4, rows, n, dev.data_ptr(), dev.numel())
    del dev
    x = torch.zeros(2, n, device="cuda")
    y = torch.zeros(2, rows, device="cuda")
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        m.matvec_device(2, x.data_ptr(), y.data_ptr(), stream=side.cuda_stream)
    for k in range(3):
        x.copy_(torch.from_numpy(rng.standard_normal((2, n)).astype(np.float32)))
        g.replay()
        torch.cuda.synchronize()
        check(host(y), host(x), w, a, n, fb.F32)
    streams = [torch.cuda.Stream() for _ in range(2)]
    ys = [torch.zeros(2, rows, device="cuda") for _ in range(8)]
    torch.cuda.synchronize()
    for k in range(8):
        m.matvec_device(2, x.data_ptr(), ys[k].data_ptr(), stream=streams[k % 2].cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(v, y) for v in ys)
    assert ctx.status() == fb.OK
    m.close()


def far_apart(n, rng, pairs):
    """Eight MXFP4 rows for each pair (small, large) of exponents: blocks of either kind mixed, and the columns of the
    small ones."""
    small = rng.random(n // 32) < 0.6
    small[0] = True
    raw = np.concatenate([quant.random_rows(fb.MXFP4, 8, n, rng, (lo, lo + 1)) for lo, _ in pairs])
    b = raw.reshape(len(pairs), 8, n // 32, 17)
    for k, (_, hi) in enumerate(pairs):
        b[k, :, ~small, 0] = hi
    return raw, np.repeat(small, 32)


@pytest.mark.parametrize("tokens", [1, 2, 3, 5, 16])
@pytest.mark.parametrize("x_type", [fb.F32, fb.BF16])
def test_block_scales_far_apart(ctx, tokens, x_type):
    """MXFP4 rows whose block scales lie 100 to 229 binades apart, x zero where they are large: what the small ones
    give counts in full.  A zero of x adds nothing and is exact, so the bound's terms are those of the small blocks."""
    rng = np.random.default_rng(31)
    for n in (544, 2560):
        for pairs in ([(20, 120), (20, 146), (20, 147), (20, 148), (20, 220), (20, 229), (21, 248), (25, 254)],
                      [(0, 229), (0, 127), (0, 128), (1, 230), (1, 128), (2, 200)]):
            raw, small = far_apart(n, rng, pairs)
            w, a = quant.weights(fb.MXFP4, raw, n)
            x = np.where(small, rng.standard_normal((tokens, n)), 0) * 2.0 ** 105
            xd = to_device(x, x_type)
            y = host(run(ctx, fb.MXFP4, raw, n, xd, x_type, fb.F32))
            xr = host(xd)
            ref = xr @ w.T
            tol = bound(a * small, xr, n) + 2.0 ** -126
            assert np.all(np.abs(y - ref) <= tol), (np.abs(y - ref) / tol).max()
            assert np.abs(ref).min() > 2.0 ** -60


@pytest.mark.parametrize("tokens", [1, 2, 3, 5, 16])
def test_blocks_without_weights(ctx, tokens):
    """The exponent of a block whose weights are all +-0 means nothing, to 254."""
    rng = np.random.default_rng(32)
    n = 1056
    raw = quant.random_rows(fb.MXFP4, 40, n, rng)
    b = raw.reshape(40, n // 32, 17)
    zero = rng.random((40, n // 32)) < 0.3
    b[zero, 1:] = rng.choice(np.array([0, 0x80, 0x08, 0x88], np.uint8), (int(zero.sum()), 16))
    b[zero, 0] = rng.choice(np.array([0, 1, 200, 254], np.uint8), int(zero.sum()))
    b[5, :, 1:] = 0
    b[5, :, 0] = 254
    w, a = quant.weights(fb.MXFP4, raw, n)
    assert not w.reshape(40, -1, 32)[zero].any()
    xd = to_device(rng.standard_normal((tokens, n)), fb.F32)
    y = host(run(ctx, fb.MXFP4, raw, n, xd, fb.F32, fb.F32))
    check(y, host(xd), w, a, n, fb.F32)
    assert not y[:, 5].any()


@pytest.mark.parametrize("tokens", [1, 2, 3, 5, 16])
@pytest.mark.parametrize("exponents,size", [((60, 90), 2.0 ** 125), ((0, 1), 2.0 ** 125), ((0, 40), 2.0 ** 110), ((224, 255), 2.0 ** -120),
                                            ((254, 255), 2.0 ** -122), ((100, 130), 2.0 ** 100)])
def test_products_of_extremes(ctx, exponents, size, tokens):
    """MXFP4 scales and vectors at opposite ends of their ranges: results that are finite come out finite and right."""
    rng = np.random.default_rng(33)
    for n in (288, 4096):
        raw = quant.random_rows(fb.MXFP4, 33, n, rng, exponents)
        w, a = quant.weights(fb.MXFP4, raw, n)
        x = rng.uniform(0.5, 1.0, (tokens, n)) * rng.choice((-1, 1), (tokens, n)) * size
        xd = to_device(x, fb.F32)
        xr = host(xd)
        assert np.all(np.abs(xr) @ a.T < 2.0 ** 126)
        y = host(run(ctx, fb.MXFP4, raw, n, xd, fb.F32, fb.F32))
        tol = bound(a, xr, n) + 2.0 ** -126
        assert np.all(np.abs(y - xr @ w.T) <= tol)


def test_block_scales_too_far_apart(ctx):
    """Scales of one row more than 229 binades apart are refused, at any place of the matrix; zero weights do not count."""
    rng = np.random.default_rng(34)
    n, rows = 320, 50
    for row, refused, taken in [(0, (0, 230), (1, 230)), (17, (24, 254), (25, 254)), (49, (0, 254), (0, 229))]:
        raw = quant.random_rows(fb.MXFP4, rows, n, rng)
        b = raw.reshape(rows, n // 32, 17)
        b[row, 0, 1] = b[row, 9, 16] = 0x10  # one weight of 0.5
        b[row, 0, 0], b[row, 9, 0] = refused
        with pytest.raises(fb.FrcError) as e:
            ctx.matrix(fb.MXFP4, rows, n, raw)
        assert e.value.code == fb.UNSUPPORTED
        b[row, 0, 0], b[row, 9, 0] = taken
        ctx.matrix(fb.MXFP4, rows, n, raw).close()
        b[row, 0, 0], b[row, 9, 0] = refused
        b[row, 0, 1:] = 0x80
        ctx.matrix(fb.MXFP4, rows, n, raw).close()


@pytest.mark.parametrize("type_", [fb.Q4_K, fb.MXFP4])
@pytest.mark.parametrize("tokens", [1, 3, 4, 5, 16])
@pytest.mark.parametrize("exponent", [-97, -104, -112, -122, -130, -147])
def test_tiny_vectors(ctx, type_, tokens, exponent):
    """Vectors near the bottom of fp32's range, subnormal ones too, times large weights: they are carried as exactly
    as others."""
    rng = np.random.default_rng(35)
    n = 256
    raw = quant.random_rows(type_, 40, n, rng, exponents=(180, 190))
    if type_ == fb.Q4_K:
        raw.reshape(40, 1, 144)[..., :4] = (rng.choice((-1, 1), (40, 1, 2)) * rng.uniform(20000, 60000, (40, 1, 2))).astype(np.float16).view(np.uint8)
    w, a = quant.weights(type_, raw, n)
    xd = to_device(rng.standard_normal((tokens, n)) * 2.0 ** exponent, fb.F32)
    x = host(xd)
    assert x.any(1).all()
    y = host(run(ctx, type_, raw, n, xd, fb.F32, fb.F32))
    tol = bound(a, x, n) + 2.0 ** -126
    assert np.all(np.abs(y - x @ w.T) <= tol), (np.abs(y - x @ w.T) / tol).max()


@pytest.mark.parametrize("type_,rows,n", [(fb.Q4_K, 513, 2048), (fb.Q4_K, 300, 8192), (fb.Q4_K, 200, 65536),
                                          (fb.MXFP4, 513, 2048), (fb.MXFP4, 300, 16384), (fb.MXFP4, 200, 65440)])
def test_size_of_the_error(ctx, type_, rows, n):
    """The error's L2 norm over the rows, which a worst-case bound leaves room for a hundred times over.  With S = the
    root of the sum of (a_j x_j)^2, the size of a sum of n terms of either sign, and roundings that are independent of
    one another: 26 in a span of 256 (8 groups of 2 steps and a scale, 2 for the span's own), each up to 2^-23 of the
    span's S, make sqrt(26) = 5.1; one an added span, up to 2^-24 of all of S, sqrt(spans) / 2; truncation moves a
    group's sum by up to 2 steps the same way, 2; the vector's 22 bits 1; joining 16 parts 4.  Together
    (sqrt(spans) / 2 + 13) 2^-23 S."""
    rng = np.random.default_rng(rows + n)
    raw = quant.random_rows(type_, rows, n, rng)
    w, a = quant.weights(type_, raw, n)
    for tokens in (1, 2, 4, 5, 9, 16):
        for x_type in (fb.F32, fb.BF16):
            xd = to_device(rng.standard_normal((tokens, n)), x_type)
            x = host(xd)
            y = host(run(ctx, type_, raw, n, xd, x_type, fb.F32))
            size = np.sqrt((x ** 2 @ (a ** 2).T).sum(1))
            err = np.sqrt(((y - x @ w.T) ** 2).sum(1))
            limit = (np.sqrt(n / 256) / 2 + 13) * 2.0 ** -23
            assert np.all(err <= limit * size), (tokens, x_type, (err / size).max() / limit)


@pytest.mark.parametrize("type_", [fb.Q4_K, fb.MXFP4])
@pytest.mark.parametrize("n,tokens,x_type", [(65536, 16, fb.F32), (65536, 16, fb.BF16), (65536, 3, fb.F32), (8192, 1, fb.F32),
                                             (8192, 8, fb.BF16)])
def test_one_span_at_a_time(ctx, type_, n, tokens, x_type):
    """Vectors that are zero but for one span of 256 columns, each span in turn: a span that is lost, taken twice or
    taken from another place shows.  The zeros are exact, so the bound is that of a single span."""
    rng = np.random.default_rng(n + tokens)
    n -= 0 if type_ == fb.Q4_K else 96
    spans, rows = -(-n // 256), 70
    raw = quant.random_rows(type_, rows, n, rng)
    w, a = quant.weights(type_, raw, n)
    with ctx.matrix(type_, rows, n, raw) as m:
        for first in range(0, spans, tokens):
            x = np.zeros((tokens, n))
            for t in range(tokens):
                s = (first + t) % spans
                x[t, 256 * s:256 * s + 256] = rng.standard_normal(min(256, n - 256 * s))
            xd = to_device(x, x_type)
            yd = to_device(np.full((tokens, rows), np.nan), fb.F32)
            m.matvec_device(tokens, xd.data_ptr(), yd.data_ptr(), x_type)
            assert ctx.status() == fb.OK
            for t in range(tokens):
                s = (first + t) % spans
                cols = slice(256 * s, 256 * s + 256)
                xs, ys = host(xd[t:t + 1, cols]), host(yd[t:t + 1])
                ref, tol = xs @ w[:, cols].T, bound(a[:, cols], xs, xs.shape[1])
                assert np.all(np.abs(ys - ref) <= tol), (s, (np.abs(ys - ref) / tol).max())


@pytest.mark.parametrize("tokens", [1, 2, 3, 5, 16])
@pytest.mark.parametrize("x_type", [fb.F32, fb.BF16])
@pytest.mark.parametrize("exponent", [0, 228, 229, 230, 254])
def test_largest_sums(ctx, exponent, x_type, tokens):
    """Every weight 6, every x just under a power of two: the largest sum a span can have, at the scales around which
    rows take a common shift."""
    n, rows = 1024, 20
    rng = np.random.default_rng(36)
    raw = quant.random_rows(fb.MXFP4, rows, n, rng, (exponent, exponent + 1))
    raw.reshape(rows, n // 32, 17)[..., 1:] = 0x77
    w, a = quant.weights(fb.MXFP4, raw, n)
    xd = to_device(np.full((tokens, n), (2.0 - 2.0 ** -7) * 2.0 ** (80 if exponent == 0 else -60)), x_type)
    x = host(xd)
    y = host(run(ctx, fb.MXFP4, raw, n, xd, x_type, fb.F32))
    assert np.all(np.abs(y - x @ w.T) <= bound(a, x, n) + 2.0 ** -126)
