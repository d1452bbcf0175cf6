"""The MXFP4 kernels against their definition in 64 bits (MI355X only).

Codes and scales have to be equal. A product's terms are exact (a code has two
significant bits), so that a sum of K of them in float32 is off by at most K
steps of 2^-23 times the sum of the magnitudes, and a result in bfloat16 by
another 2^-8 of itself."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from code2vec_amd.ops import functional as F  # noqa: E402
from code2vec_amd.ops import reference as R  # noqa: E402

BF, F32 = torch.bfloat16, torch.float32


def same(got, want):
    assert got.k == want.k
    assert torch.equal(got.scales.cpu(), want.scales)
    assert torch.equal(got.codes.cpu(), want.codes)


def rows(N, K, seed, dtype=F32):
    g = torch.Generator().manual_seed(seed)
    spread = torch.exp2(torch.rand(N, 1, generator=g) * 12 - 6)
    return (torch.randn(N, K, generator=g) * spread).to(dtype)


@pytest.mark.parametrize('dtype', [F32, BF])
@pytest.mark.parametrize('N,K', [(1, 1), (1, 32), (3, 31), (5, 33), (70, 384), (1000, 128),
                                 (17, 301), (4, 8), (300, 100), (2, 5000)])
def test_quantize(N, K, dtype):
    x = rows(N, K, N + K, dtype)
    want = R.mxfp4_quantize(x)
    got = F.mxfp4_quantize(x.cuda())
    same(got, want)
    for out in (F32, BF):
        back = F.mxfp4_dequantize(got, out)
        assert back.shape == (N, K) and back.dtype == out
        assert torch.equal(back.cpu(), R.mxfp4_dequantize(want, out))


def test_quantize_borders_and_ties():
    """Every middle of the grid, the values next to it, at every binary order."""
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.99, 4.0, 0.5, 0.0])
    v = torch.cat((mids, torch.nextafter(mids, torch.tensor(100.0)),
                   torch.nextafter(mids, torch.tensor(-1.0))))
    v = torch.cat((v, -v))[:77]
    block = torch.zeros(3 * 32)
    block[:77] = v
    block[31], block[63], block[95] = 4.0, 7.5, -6.5   # each block spans 4..8
    x = torch.stack([block * 2.0 ** e for e in (-120, -60, -3, 0, 5, 100, 124)])
    same(F.mxfp4_quantize(x.cuda()), R.mxfp4_quantize(x))
    b = x.to(BF)
    same(F.mxfp4_quantize(b.cuda()), R.mxfp4_quantize(b))


def test_quantize_ends_of_the_range():
    x = torch.zeros(9, 64)
    x[0, 3] = torch.finfo(F32).max
    x[1, 3] = torch.finfo(F32).min
    x[2, 40] = 2.0 ** -126
    x[3, 40], x[3, 41] = 2.0 ** -140, -2.0 ** -149    # below the smallest scale
    x[4, 7], x[4, 8] = 2.0 ** -127, 2.0 ** -128
    x[5, 0] = float('nan')
    x[6, 63] = float('-inf')
    x[7, 1] = -0.0
    want = R.mxfp4_quantize(x)
    got = F.mxfp4_quantize(x.cuda())
    same(got, want)
    back = F.mxfp4_dequantize(got, F32).cpu()
    assert back[5, :32].isnan().all() and back[5, 32:].eq(0).all()
    assert back[6, 32:].isnan().all() and back[6, :32].eq(0).all()
    assert torch.equal(back[8], torch.zeros(64))
    assert torch.equal(torch.nan_to_num(back, 7.0),
                       torch.nan_to_num(R.mxfp4_dequantize(want), 7.0))


def test_quantize_strided_rows():
    for dtype in (F32, BF):
        for K in (96, 50):
            wide = rows(40, K + 20, 5, dtype)
            for at in (4, 8, 3):
                v = wide[:, at:at + K]
                same(F.mxfp4_quantize(wide.cuda()[:, at:at + K]), R.mxfp4_quantize(v))
        t = rows(64, 40, 6, dtype)
        same(F.mxfp4_quantize(t.cuda().t()), R.mxfp4_quantize(t.t()))
        same(F.mxfp4_quantize(t[:1].cuda().expand(9, 40)), R.mxfp4_quantize(t[:1].expand(9, 40)))


def check_product(x, w, y, out):
    """x a tensor or Mxfp4, on the CPU; w Mxfp4 on the CPU."""
    xd = R.mxfp4_dequantize(x, torch.float64) if isinstance(x, F.Mxfp4) else x.double()
    wd = R.mxfp4_dequantize(w, torch.float64)
    ref = xd @ wd.t()
    size = xd.abs() @ wd.abs().t()
    tol = 2.0 ** -23 * (w.k + 4) * size
    if out == BF:
        tol = tol + 2.0 ** -8 * (ref.abs() + tol)
    assert y.dtype == out and y.shape == ref.shape
    bad = (y.cpu().double() - ref).abs() > tol + 2.0 ** -126
    # magnitudes of a sum of 2^128 and more: a partial sum may lie outside of
    # float32 (6 * 2^123 times 4, 96 times, is 2^134), and nothing is said
    bad &= size < 2.0 ** 128
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist())


def on_gpu(q):
    return F.Mxfp4(q.codes.cuda(), q.scales.cuda(), q.k)


@pytest.mark.parametrize('out', [BF, F32])
@pytest.mark.parametrize('N,M,K', [
    (1, 1000, 384), (1, 1, 1), (3, 7, 5), (16, 512, 128), (17, 513, 32), (15, 511, 384),
    (37, 501, 201), (64, 700, 96), (65, 1030, 160), (130, 520, 384), (200, 77, 640),
    (40, 300, 1030), (5, 200, 2500), (129, 1500, 385), (300, 4100, 384), (513, 5003, 33),
    (260, 9001, 100), (700, 3000, 511), (1030, 2050, 384), (2100, 1501, 64),
    (530, 70, 300), (600, 64, 40), (140, 129, 7), (257, 1027, 545), (600, 3002, 768),
    (130, 500, 641), (200, 300, 769)])
def test_products(N, M, K, out):
    x = rows(N, K, N, BF) * 0.5
    w = R.mxfp4_quantize(rows(M, K, M + 1))
    wg = on_gpu(w)
    check_product(x, w, F.mxfp4_matmul(x.cuda(), wg, out), out)
    xq = R.mxfp4_quantize(x)
    got = F.mxfp4_quantize(x.cuda())
    same(got, xq)
    check_product(xq, w, F.mxfp4_matmul(got, wg, out), out)


def test_whole_numbers_are_exact():
    g = torch.Generator().manual_seed(1)
    x = torch.randint(-4, 5, (33, 200), generator=g).float()
    w = torch.randint(-4, 5, (700, 200), generator=g).float()
    wq = F.mxfp4_quantize(w.cuda())
    assert torch.equal(F.mxfp4_dequantize(wq, F32).cpu(), w)
    assert torch.equal(F.mxfp4_matmul(x.to(BF).cuda(), wq, F32).cpu(), x @ w.t())
    assert torch.equal(F.mxfp4_matmul(F.mxfp4_quantize(x.cuda()), wq, F32).cpu(), x @ w.t())


@pytest.mark.parametrize('N,M,K,out', [(2040, 50001, 70, BF), (1020, 50003, 300, F32),
                                       (2048, 50004, 130, BF), (4000, 25002, 40, BF)])
def test_more_than_the_caches_hold(N, M, K, out):
    """Whole numbers again, so that each result is exact up to its own rounding."""
    g = torch.Generator(device='cuda').manual_seed(1)
    x = torch.randint(-4, 5, (N, K), generator=g, device='cuda').float()
    w = torch.randint(-4, 5, (M, K), generator=g, device='cuda').float()
    want = (x @ w.t()).to(out)
    wq = F.mxfp4_quantize(w)
    assert torch.equal(F.mxfp4_matmul(x.to(BF), wq, out), want)
    assert torch.equal(F.mxfp4_matmul(F.mxfp4_quantize(x), wq, out), want)


@pytest.mark.parametrize('N', [5, 100])
def test_product_of_strided_rows(N):
    w = R.mxfp4_quantize(rows(600, 100, 3))
    wide = rows(N, 130, 4, BF)
    for at in (8, 3):
        check_product(wide[:, at:at + 100], w,
                      F.mxfp4_matmul(wide.cuda()[:, at:at + 100], on_gpu(w), F32), F32)
    t = rows(100, N, 4, BF)
    check_product(t.t(), w, F.mxfp4_matmul(t.cuda().t(), on_gpu(w), F32), F32)
    check_product(wide[:1, :100].expand(N, 100), w,
                  F.mxfp4_matmul(wide[:1, :100].cuda().expand(N, 100), on_gpu(w), F32), F32)


def test_scales_at_both_ends_and_nan_blocks():
    w = R.mxfp4_quantize(rows(300, 96, 9))
    w.scales[::3] = 1
    w.scales[1::3] = 250
    x = rows(20, 96, 2, BF).clamp(-4, 4)
    x = torch.where(x.abs() < 0.01, torch.ones_like(x), x)
    for N in (3, 20):
        check_product(x[:N], w, F.mxfp4_matmul(x[:N].cuda(), on_gpu(w), F32), F32)
    w.scales[7, 1] = 255
    # rows 1, 4, 7, .. may leave float32, as above: the claim is on the others
    tame = torch.arange(300) % 3 != 1
    y = F.mxfp4_matmul(x.cuda(), on_gpu(w), F32).cpu()
    y4 = F.mxfp4_matmul(F.mxfp4_quantize(x.cuda()), on_gpu(w), F32).cpu()
    for v in (y, y4):
        assert v[:, 7].isnan().all()
        assert v[:, tame].isfinite().all()
    x[4, 50] = float('nan')
    for v in (F.mxfp4_matmul(x.cuda(), on_gpu(w), F32).cpu(),
              F.mxfp4_matmul(F.mxfp4_quantize(x.cuda()), on_gpu(w), F32).cpu()):
        assert v[4].isnan().all()
        assert v[:4, tame].isfinite().all() and v[5:, tame].isfinite().all()


@pytest.mark.parametrize('K', [20, 32, 50, 96, 128, 160, 270, 385])
@pytest.mark.parametrize('N', [130, 300])
def test_nan_blocks_stay_in_their_columns(N, K):
    """More rows than the kernel for few of them takes. Rows of the table with a NaN
    block and rows whose scales leave bfloat16 (4 * 2^126 and more), the table's
    first, last and those at a tile's border among them: only their own columns
    may see them."""
    M = 333
    bad, nan = [0, 5, 64, 100, 127, 200, M - 1], [5, 64, 200, M - 1]
    w = R.mxfp4_quantize(rows(M, K, 3))
    blocks = w.scales.shape[1]
    w.scales[0, -1], w.scales[100, 0], w.scales[127] = 254, 253, 253
    for k, m in enumerate(nan):
        w.scales[m, k % blocks] = 255
    x = rows(N, K, 4, BF)
    xq = R.mxfp4_quantize(x)
    tame = torch.ones(M, dtype=torch.bool)
    tame[bad] = False
    for out in (F32, BF):
        for a, ag in ((x, x.cuda()), (xq, on_gpu(xq))):
            y = F.mxfp4_matmul(ag, on_gpu(w), out)
            assert y[:, nan].isnan().all()
            assert y.cpu()[:, tame].isfinite().all()
            check_product(a, F.Mxfp4(w.codes[tame], w.scales[tame], K), y[:, tame.cuda()], out)


def test_nan_blocks_of_a_table_beyond_the_caches():
    """The same where rows of y are taken that lie alike on cache lines. Whole
    numbers: each clean column is exact."""
    g = torch.Generator(device='cuda').manual_seed(2)
    N, M, K = 2040, 50001, 70
    x = torch.randint(-4, 5, (N, K), generator=g, device='cuda').float()
    w = torch.randint(-4, 5, (M, K), generator=g, device='cuda').float()
    nan = torch.arange(17, M, 211, device='cuda')
    want = x @ w.t()
    want[:, nan] = float('nan')
    wq = F.mxfp4_quantize(w)
    wq.scales[nan, 0] = 255
    for a in (x.to(BF), F.mxfp4_quantize(x)):
        y = F.mxfp4_matmul(a, wq, BF)
        assert torch.equal(y.isnan(), want.isnan())
        assert torch.equal(y.nan_to_num(7.0), want.to(BF).nan_to_num(7.0))


def test_what_fills_up_a_row_does_not_count():
    """Codes behind K are the table owner's: whatever they are, no result changes."""
    w = F.mxfp4_quantize(rows(200, 40, 1).cuda())
    x = rows(9, 40, 2, BF).cuda()
    want = F.mxfp4_matmul(x, w, F32)
    want4 = F.mxfp4_matmul(F.mxfp4_quantize(x), w, F32)
    w.codes[:, 20:] = 0x77
    assert torch.equal(F.mxfp4_matmul(x, w, F32), want)
    assert torch.equal(F.mxfp4_matmul(F.mxfp4_quantize(x), w, F32), want4)


@pytest.mark.parametrize('K', [20, 96, 130, 700])
@pytest.mark.parametrize('N', [1, 40, 200])
def test_rows_of_a_table(N, K):
    """Some rows of a table, and of quantised rows, are as good as a copy of them: an
    odd number of blocks a row lets their scales start on any byte."""
    w, x = (on_gpu(R.mxfp4_quantize(rows(n, K, n))) for n in (700, N + 3))

    def part(q, at, n):
        return F.Mxfp4(q.codes[at:at + n], q.scales[at:at + n], K)

    def copy(q):
        return F.Mxfp4(q.codes.clone(), q.scales.clone(), K)

    rows_bf = rows(N, K, 9, BF).cuda()
    for at in (1, 2, 3):
        wp, xp = part(w, at, 690), part(x, at, N)
        for out in (F32, BF):
            assert torch.equal(F.mxfp4_dequantize(wp, out), F.mxfp4_dequantize(copy(wp), out))
            assert torch.equal(F.mxfp4_matmul(rows_bf, wp, out),
                               F.mxfp4_matmul(rows_bf, copy(wp), out))
            assert torch.equal(F.mxfp4_matmul(xp, wp, out),
                               F.mxfp4_matmul(copy(xp), copy(wp), out))


def test_nothing_to_do():
    w = F.mxfp4_quantize(rows(10, 40, 1).cuda())
    assert F.mxfp4_matmul(torch.empty(0, 40, dtype=BF, device='cuda'), w).shape == (0, 10)
    none = F.mxfp4_quantize(torch.empty(0, 40, device='cuda'))
    assert none.codes.shape == (0, 32) and F.mxfp4_dequantize(none).shape == (0, 40)
    assert F.mxfp4_matmul(torch.ones(3, 40, dtype=BF, device='cuda'), none).shape == (3, 0)
    flat = F.mxfp4_quantize(torch.empty(4, 0, device='cuda'))
    y = F.mxfp4_matmul(torch.ones(3, 0, dtype=BF, device='cuda'), flat)
    assert y.shape == (3, 4) and (y == 0).all()


def test_another_stream_and_a_captured_graph():
    w = F.mxfp4_quantize(rows(3000, 384, 1).cuda())
    x = rows(50, 384, 2, BF).cuda()

    def both(v):
        q = F.mxfp4_quantize(v)
        return F.mxfp4_matmul(v, w), F.mxfp4_matmul(q, w), F.mxfp4_dequantize(q)

    want = both(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both(x)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both(x)
    for k in range(3):
        x2 = rows(50, 384, 20 + k, BF).cuda()
        eager = both(x2)
        x.copy_(x2)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager, out):
            assert torch.equal(a, b)


def test_offsets_beyond_32_bits():
    """An output of over 2^32 bytes: its last rows are where they belong."""
    w = R.mxfp4_quantize(rows(140000, 32, 1))
    x = rows(16400, 32, 2, BF)
    y = F.mxfp4_matmul(x.cuda(), on_gpu(w))
    assert y.numel() * 2 > 2 ** 32
    for sl in (slice(0, 2), slice(16398, 16400)):
        check_product(x[sl], w, y[sl], BF)


@pytest.mark.parametrize('k', [-1, -5, -62])
def test_rows_of_no_length(k):
    none = torch.empty(3, 0, dtype=torch.uint8, device='cuda')
    bad = F.Mxfp4(none, none, k)
    for call in (lambda: F.mxfp4_dequantize(bad), lambda: F.mxfp4_matmul(bad, bad),
                 lambda: F.mxfp4_matmul(torch.empty(3, 0, dtype=BF, device='cuda'), bad)):
        with pytest.raises(ValueError, match='does not hold rows'):
            call()


def test_refusals():
    w = F.mxfp4_quantize(rows(10, 40, 1).cuda())
    x = rows(3, 40, 2, BF).cuda()
    with pytest.raises(RuntimeError):
        F.mxfp4_matmul(x.float(), w)
    with pytest.raises(ValueError):
        F.mxfp4_matmul(x.cpu(), w)
    with pytest.raises(ValueError):
        F.mxfp4_matmul(x[:, :39], w)
    with pytest.raises(ValueError):
        F.mxfp4_quantize(x.half())
    for bad in (F.Mxfp4(w.codes[:, :16], w.scales, 40), F.Mxfp4(w.codes, w.scales[:9], 40),
                F.Mxfp4(w.codes, w.scales, 70), F.Mxfp4(w.codes.float(), w.scales, 40),
                F.Mxfp4(w.codes, w.scales.cpu(), 40),
                F.Mxfp4(w.codes.t().contiguous().t(), w.scales, 40)):
        with pytest.raises(ValueError):
            F.mxfp4_matmul(x, bad)
        with pytest.raises(ValueError):
            F.mxfp4_dequantize(bad)
        with pytest.raises(ValueError):
            F.mxfp4_matmul(bad, w)
    with pytest.raises(ValueError):
        F.mxfp4_matmul(x, w.codes)
    shifted = torch.empty(w.codes.numel() + 1, dtype=torch.uint8, device='cuda')[1:]
    with pytest.raises(RuntimeError):
        F.mxfp4_matmul(x, F.Mxfp4(shifted.view(w.codes.shape), w.scales, w.k))
