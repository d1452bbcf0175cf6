"""The gated transform's kernels against its formula in 64 bits (MI355X only).

Bounds: a value rounded to bfloat16 is off by at most EB = 2^-8 of itself, one
rounded to float32 by E = 2^-24. A sum of n products in float32 is off by at
most n steps of 2E times the sum of the magnitudes (a matrix instruction may
cut off where an adder rounds, hence 2E); the activation's own evaluation adds
a few more steps, 32 of them in all."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from code2vec_amd.ops import functional as F  # noqa: E402
from code2vec_amd.ops import reference as R  # noqa: E402

EB, E = 2.0 ** -8, 2.0 ** -24
TINY = 2.0 ** -126


def make(N, K, H, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(N, K, generator=g) * scale).to(torch.bfloat16)
    w = (torch.randn(2, K, H, generator=g) * K ** -0.5).to(torch.bfloat16)
    dy = torch.randn(N, H, generator=g).to(torch.bfloat16)
    w_oi = w.transpose(1, 2).contiguous()
    w_io = w.permute(1, 0, 2).reshape(K, 2 * H).contiguous()
    return x, w_oi, w_io, dy


def check_fwd(x, w_oi, act, y, kept):
    xd, wd = x.cpu().double(), w_oi.cpu().double()
    N, K = xd.shape
    H = wd.shape[1]
    g, u = xd @ wd[0].t(), xd @ wd[1].t()
    off = 2 * E * (K + 32)
    sg, su = off * (xd.abs() @ wd[0].abs().t()), off * (xd.abs() @ wd[1].abs().t())
    a, _ = R.gate_activation(act, g)
    ref = a * u
    # |act'| is at most 1.13 for all five; the activation itself is within 32 steps
    tol = EB * ref.abs() + (1 + EB) * (1.13 * sg * (u.abs() + su) + a.abs() * su
                                      + 32 * 2 * E * ref.abs()) + TINY
    assert y.shape == (N, H) and y.dtype == torch.bfloat16
    bad = (y.cpu().double() - ref).abs() > tol
    assert not bad.any(), ('y', int(bad.sum()), bad.nonzero()[:4].tolist())
    assert kept is None or torch.equal(kept.cpu(), w_oi.cpu())


def check_bwd(x, w_io, dy, act, d_ctx, d_w, keep=None):
    xd, wd, dyd = x.cpu().double(), w_io.cpu().double(), dy.cpu().double()
    N, K = xd.shape
    H = dyd.shape[1]
    g, u = xd @ wd[:, :H], xd @ wd[:, H:]
    off = 2 * E * (K + 32)
    sg, su = off * (xd.abs() @ wd[:, :H].abs()), off * (xd.abs() @ wd[:, H:].abs())
    a, da = R.gate_activation(act, g)
    # act' cancels where it is near zero: 64 steps of its largest term
    steps = 64 * 2 * E
    dgu = torch.cat((dyd * u * da, dyd * a), 1)
    d_tol = steps * torch.cat(
        (dyd.abs() * u.abs() * (1 + g.abs()), dyd.abs() * (1 + g.abs())), 1) + TINY
    # what g and u are off by: |act'| is at most 1.13, |act''| at most 1; relu's
    # slope jumps where g may be of either sign
    jump = (g.abs() <= sg).double() if act == 'relu' else 0.0
    d_tol = d_tol + dyd.abs().repeat(1, 2) * torch.cat(
        (su * 1.13 + (u.abs() + su) * (sg + jump), 1.13 * sg), 1)
    d_tol = d_tol + EB * (dgu.abs() + d_tol)
    ref = dgu @ wd.t()
    tol = d_tol @ wd.abs().t() + 2 * E * (2 * H + 32) * (dgu.abs() @ wd.abs().t())
    if keep is not None:
        mask, p = keep
        ref, tol = ref * mask / p, tol * mask / p + 4 * E * (ref * mask / p).abs()
    tol = tol + EB * (ref.abs() + tol) + TINY
    bad = (d_ctx.cpu().double() - ref).abs() > tol
    assert not bad.any(), ('d_ctx', int(bad.sum()), bad.nonzero()[:4].tolist())
    refw = xd.t() @ dgu
    tolw = xd.abs().t() @ d_tol + 2 * E * (N + 64) * (xd.abs().t() @ dgu.abs())
    tolw = tolw + EB * (refw.abs() + tolw) + TINY
    got = d_w.cpu().double().permute(1, 0, 2).reshape(K, 2 * H)
    bad = (got - refw).abs() > tolw
    assert not bad.any(), ('d_w', int(bad.sum()), bad.nonzero()[:4].tolist())


def run(x, w_oi, w_io, dy, act, **kw):
    x, w_oi, w_io, dy = (t.cuda() if not t.is_cuda else t for t in (x, w_oi, w_io, dy))
    y, kept = F.transform_gated_fwd(x, w_oi, act, save=True)
    y2, none = F.transform_gated_fwd(x, w_oi, act)
    # bit by bit: NaN is not equal to itself
    assert none is None and torch.equal(y.view(torch.int16), y2.view(torch.int16))
    d_ctx, d_w = F.transform_gated_bwd(x, w_io, kept, dy, act, **kw)
    return y, kept, d_ctx, d_w


@pytest.mark.parametrize('act', F.GATE_ACTIVATIONS)
@pytest.mark.parametrize('N,K,H', [(150, 96, 72), (150, 1000, 72), (2100, 40, 264)])
def test_each_activation(act, N, K, H):
    x, w_oi, w_io, dy = make(N, K, H, seed=1, scale=2.0)
    y, kept, d_ctx, d_w = run(x, w_oi, w_io, dy, act)
    check_fwd(x, w_oi, act, y, kept)
    check_bwd(x, w_io, dy, act, d_ctx, d_w)


@pytest.mark.parametrize('N,K,H', [
    (1, 384, 384), (2, 8, 8), (3, 1, 1), (200, 384, 384), (256, 64, 128),
    (257, 72, 136), (255, 200, 120), (1000, 24, 24), (64, 768, 40),
    (33, 99, 101), (300, 31, 7), (129, 7, 250), (513, 390, 391), (5000, 192, 192),
    (300, 760, 130), (1000, 1030, 264), (5, 900, 17), (4097, 1440, 72), (4097, 136, 520)])
def test_sizes(N, K, H):
    x, w_oi, w_io, dy = make(N, K, H, seed=N + K + H)
    y, kept, d_ctx, d_w = run(x, w_oi, w_io, dy, 'silu')
    check_fwd(x, w_oi, 'silu', y, kept)
    check_bwd(x, w_io, dy, 'silu', d_ctx, d_w)


@pytest.mark.parametrize('N,K,H', [
    (1, 384, 384), (3, 1, 1), (200, 384, 384), (33, 99, 101), (300, 31, 7), (513, 390, 391),
    (5000, 192, 192), (4097, 136, 520), (20001, 390, 250)])
def test_weight_gradient_in_float32(N, K, H):
    """float32 on request, as it is summed: rounded it is the default's, bit by
    bit. Of small whole numbers and relu each value on the way has a bfloat16
    and each sum is below 2^24, so that the sums are exact."""
    x, w_oi, w_io, dy = make(N, K, H, seed=N + K + H)
    g = torch.Generator().manual_seed(N)
    whole = torch.zeros(N, K)
    for _ in range(2):
        whole[torch.arange(N), torch.randint(0, K, (N,), generator=g)] = 1.0
    w = torch.randint(0, 3, (2, K, H), generator=g).float()
    sums = (whole, w.transpose(1, 2).contiguous(), w.permute(1, 0, 2).reshape(K, 2 * H),
            torch.randint(0, 4, (N, H), generator=g).float())
    want = R.transform_gated_bwd(*(sums[i].double() for i in (0, 2, 1, 3)), 'relu')[1]
    for inputs, act in (((x, w_oi, w_io, dy), 'silu'), (sums, 'relu')):
        inputs = [t.to(torch.bfloat16).cuda() for t in inputs]
        _, kept, d_ctx, d_w = run(*inputs, act)
        again, d_w32 = F.transform_gated_bwd(inputs[0], inputs[2], kept, inputs[3], act,
                                             dw_dtype=torch.float32)
        assert d_w32.dtype == torch.float32 and d_w.dtype == torch.bfloat16
        assert torch.equal(again, d_ctx) and torch.equal(d_w32.to(torch.bfloat16), d_w)
    assert torch.equal(d_w32.cpu().double(), want)


@pytest.mark.parametrize('K', [40, 904])
def test_whole_numbers_are_exact(K):
    """Small whole numbers and relu: every value on the way has a bfloat16."""
    g = torch.Generator().manual_seed(3)
    N, H = 70, 48
    x = torch.zeros(N, K)
    x[torch.arange(N), torch.randint(0, K, (N,), generator=g)] = 1.0
    x[torch.arange(N), torch.randint(0, K, (N,), generator=g)] = 2.0
    w = torch.randint(-2, 3, (2, K, H), generator=g).float()
    dy = torch.zeros(N, H)
    dy[torch.arange(N), torch.randint(0, H, (N,), generator=g)] = 1.0
    w_oi, w_io = w.transpose(1, 2).contiguous(), w.permute(1, 0, 2).reshape(K, 2 * H)
    b = [t.to(torch.bfloat16) for t in (x, w_oi, w_io, dy)]
    y, kept, d_ctx, d_w = run(*b, 'relu')
    yr = R.transform_gated_fwd(x, w_oi, 'relu')
    dxr, dwr = R.transform_gated_bwd(x, w_io, w_oi, dy, 'relu')
    for got, want in ((y, yr), (d_ctx, dxr), (d_w, dwr)):
        assert torch.equal(got.cpu().float(), want)


@pytest.mark.parametrize('K,H', [(96, 96), (99, 61), (800, 48), (901, 21)])
def test_strided_inputs(K, H):
    x, w_oi, w_io, dy = make(130, K, H, seed=7)
    want = run(x, w_oi, w_io, dy, 'tanh')
    wide = torch.full((130, K + 24), float('nan'), dtype=torch.bfloat16)
    for at in (8, 3):                      # rows on 16 bytes and rows that are not
        wide[:, at:at + K] = x
        dwide = torch.full((130, H + 24), float('nan'), dtype=torch.bfloat16)
        dwide[:, at:at + H] = dy
        got = run(wide.cuda()[:, at:at + K], w_oi, w_io, dwide.cuda()[:, at:at + H], 'tanh')
        for a, b in zip((want[0], *want[2:]), (got[0], *got[2:])):
            assert torch.equal(a, b)
    got = run(x.t().contiguous().cuda().t(), w_oi, w_io, dy.t().contiguous().cuda().t(), 'tanh')
    for a, b in zip((want[0], *want[2:]), (got[0], *got[2:])):
        assert torch.equal(a, b)
    # one row for all: a stride of zero
    one = x[:1].cuda().expand(130, K)
    y, kept = F.transform_gated_fwd(one, w_oi.cuda(), 'tanh', save=True)
    check_fwd(one, w_oi, 'tanh', y, kept)
    d_ctx, d_w = F.transform_gated_bwd(one, w_io.cuda(), kept, dy[:1].cuda().expand(130, H), 'tanh')
    check_bwd(one, w_io, dy[:1].expand(130, H), 'tanh', d_ctx, d_w)


def test_no_rows():
    x, w_oi, w_io, dy = make(0, 24, 16, seed=1)
    y, kept, d_ctx, d_w = run(x, w_oi, w_io, dy, 'silu')
    assert y.shape == (0, 16) and d_ctx.shape == (0, 24)
    assert d_w.shape == (2, 24, 16) and (d_w == 0).all()


@pytest.mark.parametrize('act', F.GATE_ACTIVATIONS)
def test_no_columns(act):
    x, w_oi, w_io, dy = make(70, 24, 16, seed=1)
    y, kept, d_ctx, d_w = run(x[:, :0], w_oi[:, :, :0].contiguous(), w_io[:0], dy, act)
    assert y.shape == (70, 16) and (y == 0).all()
    assert d_ctx.shape == (70, 0) and d_w.shape == (2, 0, 16)
    y, kept, d_ctx, d_w = run(x, w_oi[:, :0].contiguous(), w_io[:, :0].contiguous(),
                              dy[:, :0], act)
    assert y.shape == (70, 0) and d_w.shape == (2, 24, 0)
    assert d_ctx.shape == (70, 24) and (d_ctx == 0).all()


@pytest.mark.parametrize('on_device', [False, True])
def test_dropout_mask_of_the_context(on_device):
    N, K, H = 140, 72, 80
    x, w_oi, w_io, dy = make(N, K, H, seed=11)
    seed = 987654321987
    seed_t = torch.tensor([seed], dtype=torch.int64, device='cuda') if on_device else None
    y, kept, d_ctx, d_w = run(x, w_oi, w_io, dy, 'gelu', keep_prob=0.75,
                            seed=0 if on_device else seed, seed_t=seed_t)
    mask = R.dropout_keep_mask(seed, N * K, 0.75, 'cpu').reshape(N, K).double()
    assert ((d_ctx.cpu() == 0) >= (mask == 0)).all()
    check_bwd(x, w_io, dy, 'gelu', d_ctx, d_w, keep=(mask, 0.75))


@pytest.mark.parametrize('act', F.GATE_ACTIVATIONS)
def test_each_activation_in_the_largest_tile(act):
    """256 rows by 128 columns, which a last tile of 33 rows by 122 columns leaves ragged,
    over a reduction that no step divides."""
    x, w_oi, w_io, dy = make(20001, 390, 250, seed=6, scale=2.0)
    y, kept, d_ctx, d_w = run(x, w_oi, w_io, dy, act)
    check_fwd(x, w_oi, act, y, kept)
    check_bwd(x, w_io, dy, act, d_ctx, d_w)


@pytest.mark.parametrize('N,K,H', [(18000, 320, 256), (9003, 520, 500), (33001, 40, 120),
                                   (50001, 64, 128), (14351, 136, 1440)])
def test_sizes_of_the_largest_tile(N, K, H):
    """Whole and ragged tiles, and reductions of one step, of two and of several."""
    x, w_oi, w_io, dy = make(N, K, H, seed=N + K + H)
    y, kept, d_ctx, d_w = run(x, w_oi, w_io, dy, 'silu')
    check_fwd(x, w_oi, 'silu', y, kept)
    check_bwd(x, w_io, dy, 'silu', d_ctx, d_w)


@pytest.mark.parametrize('N,K,H', [(1, 24, 40), (300, 70, 1000), (5003, 192, 190),
                                   (5003, 195, 190), (4099, 136, 520), (20011, 200, 190),
                                   (20011, 198, 190)])
def test_dropout_mask_in_every_tile(N, K, H):
    """d_ctx in tiles of 32 by 32, 64 by 64 and 128 by 128, whole and ragged, with rows
    of whole 16 bytes and others."""
    x, w_oi, w_io, dy = make(N, K, H, seed=N + K + H)
    seed = 2 ** 40 + N
    y, kept, d_ctx, d_w = run(x, w_oi, w_io, dy, 'silu', keep_prob=0.75, seed=seed)
    mask = R.dropout_keep_mask(seed, N * K, 0.75, 'cpu').reshape(N, K).double()
    plain, same = F.transform_gated_bwd(x.cuda(), w_io.cuda(), kept, dy.cuda(), 'silu')
    assert torch.equal(d_w, same)
    assert torch.equal(d_ctx.cpu() == 0, (mask == 0) | (plain.cpu() == 0))
    check_bwd(x, w_io, dy, 'silu', d_ctx, d_w, keep=(mask, 0.75))


def test_nan_and_inf_stay_in_their_rows():
    x, w_oi, w_io, dy = make(100, 64, 64, seed=5)
    clean = run(x, w_oi, w_io, dy, 'silu')
    x2 = x.clone()
    x2[17, 3], x2[60, 5] = float('nan'), float('inf')
    y, kept, d_ctx, _ = run(x2, w_oi, w_io, dy, 'silu')
    other = torch.ones(100, dtype=torch.bool)
    other[[17, 60]] = False
    assert torch.equal(y.cpu()[other], clean[0].cpu()[other])
    assert torch.equal(d_ctx.cpu()[other], clean[2].cpu()[other])
    assert y.cpu()[17].isnan().all()
    assert not y.cpu()[60].isfinite().all()


def test_far_values_saturate_quietly():
    """Gates far out: silu, gelu and sigmoid end in their limits, not in NaN."""
    for act in F.GATE_ACTIVATIONS:
        x = torch.tensor([[200.0], [-200.0]], dtype=torch.bfloat16, device='cuda')
        w = torch.ones(2, 1, 1, dtype=torch.bfloat16, device='cuda')
        y, kept = F.transform_gated_fwd(x, w, act, save=True)
        top = 1.0 if act in ('sigmoid', 'tanh') else 200.0
        bottom = -1.0 if act == 'tanh' else 0.0
        want = torch.tensor([[top * 200.0], [bottom * -200.0]], dtype=torch.bfloat16)
        assert torch.equal(y.cpu(), want)
        dx, dw = F.transform_gated_bwd(x, torch.ones(1, 2, dtype=torch.bfloat16, device='cuda'),
                                       kept, torch.ones_like(y), act)
        assert dx.isfinite().all() and dw.isfinite().all()


def test_results_do_not_depend_on_timing():
    x, w_oi, w_io, dy = (t.cuda() for t in make(20000, 192, 192, seed=2))
    first = run(x, w_oi, w_io, dy, 'silu')
    for _ in range(3):
        for a, b in zip(first, run(x, w_oi, w_io, dy, 'silu')):
            assert torch.equal(a, b)


@pytest.mark.parametrize('K', [192, 800])
def test_another_stream_and_a_captured_graph(K):
    x, w_oi, w_io, dy = (t.cuda() for t in make(600, K, 192, seed=8))
    want = run(x, w_oi, w_io, dy, 'silu')
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(x, w_oi, w_io, dy, 'silu')
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, kept = F.transform_gated_fwd(x, w_oi, 'silu', save=True)
        d_ctx, d_w = F.transform_gated_bwd(x, w_io, kept, dy, 'silu')
    for k in range(3):
        x2 = make(600, K, 192, seed=30 + k)[0].cuda()
        eager = run(x2, w_oi, w_io, dy, 'silu')
        x.copy_(x2)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager, (y, kept, d_ctx, d_w)):
            assert torch.equal(a, b)


def test_offsets_beyond_32_bits():
    """Whole numbers and relu, exact as above: dg and du are 9 GB. dy is not zero in
    the first and last rows alone."""
    g = torch.Generator().manual_seed(4)
    K = H = 384
    N, some = 6000131, 1000
    x = torch.zeros(some, K)
    x[torch.arange(some), torch.randint(0, K, (some,), generator=g)] = 1.0
    x[torch.arange(some), torch.randint(0, K, (some,), generator=g)] = 2.0
    w = torch.randint(-2, 3, (2, K, H), generator=g).float()
    w_oi, w_io = w.transpose(1, 2).contiguous(), w.permute(1, 0, 2).reshape(K, 2 * H)
    b = [t.to(torch.bfloat16).cuda() for t in (x, w_oi, w_io)]
    ctx = b[0].repeat(N // some + 1, 1)[:N]
    dy = torch.zeros(N, H, dtype=torch.bfloat16, device='cuda')
    ends = [0, 1, N - 2, N - 1]
    dy[ends, torch.randint(0, H, (4,), generator=g).cuda()] = 1.0
    y, kept = F.transform_gated_fwd(ctx, b[1], 'relu', save=True)
    yr = R.transform_gated_fwd(x, w_oi, 'relu')
    rows = torch.arange(N - 3000, N)
    assert torch.equal(y[N - 3000:].cpu().float(), yr[rows % some])
    assert torch.equal(y[:some].cpu().float(), yr)
    d_ctx, d_w = F.transform_gated_bwd(ctx, b[2], kept, dy, 'relu')
    xe = x[torch.tensor(ends) % some]
    dxr, dwr = R.transform_gated_bwd(xe, w_io, w_oi, dy[ends].cpu().float(), 'relu')
    assert torch.equal(d_ctx[ends].cpu().float(), dxr)
    assert not d_ctx[2:N - 2].any()
    assert torch.equal(d_w.cpu().float(), dwr)


def test_refusals():
    x, w_oi, w_io, dy = (t.cuda() for t in make(10, 16, 8, seed=1))
    with pytest.raises(ValueError):
        F.transform_gated_bwd(x, w_io, w_oi[:, :5].contiguous(), dy, 'silu')
    with pytest.raises(ValueError):
        F.transform_gated_bwd(x, w_io, w_oi.cpu(), dy, 'silu')
    y, kept = F.transform_gated_fwd(x, w_oi, 'silu', save=True)
    with pytest.raises(RuntimeError):
        F.transform_gated_fwd(x.float(), w_oi.float(), 'silu')
    with pytest.raises(RuntimeError):
        F.transform_gated_fwd(x, w_oi.transpose(1, 2).contiguous().transpose(1, 2), 'silu')
    with pytest.raises(ValueError):
        F.transform_gated_fwd(x, w_oi.cpu(), 'silu')
    with pytest.raises(ValueError):
        F.transform_gated_bwd(x, w_io, None, dy, 'silu')
    with pytest.raises(ValueError):
        F.transform_gated_bwd(x, w_io, kept[:1], dy, 'silu')
    with pytest.raises(RuntimeError):
        F.transform_gated_bwd(x, w_io, kept, dy, 'silu', keep_prob=0.5,
                              seed_t=torch.zeros(1, dtype=torch.int64))
