"""The gated transform and MXFP4 without a GPU: the formulas against
differences and autograd, the format against its definition, and what the
entry points refuse."""

import math

import pytest
import torch

from code2vec_amd.ops import functional as F
from code2vec_amd.ops import reference as R


def gated_inputs(N=5, K=6, H=11, seed=0, dtype=torch.float64):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, K, generator=g, dtype=torch.float64).to(dtype)
    w = torch.randn(2, K, H, generator=g, dtype=torch.float64).to(dtype)
    dy = torch.randn(N, H, generator=g, dtype=torch.float64).to(dtype)
    return x, w.transpose(1, 2).contiguous(), w.permute(1, 0, 2).reshape(K, 2 * H), dy


@pytest.mark.parametrize('act', F.GATE_ACTIVATIONS)
def test_gated_backward_against_differences(act):
    """Central differences in 64 bits with a step of 1e-5: off by about
    step^2 = 1e-10 times a third derivative, and 1e-16 / step = 1e-11."""
    x, w_oi, w_io, dy = gated_inputs()
    _, kept = F.transform_gated_fwd(x, w_oi, act, save=True)
    d_ctx, d_w = F.transform_gated_bwd(x, w_io, kept, dy, act)

    def loss(xv, wv):
        return float((F.transform_gated_fwd(xv, wv, act)[0] * dy).sum())

    step = 1e-5
    for n in range(x.shape[0]):
        for k in range(x.shape[1]):
            a, b = x.clone(), x.clone()
            a[n, k] += step
            b[n, k] -= step
            diff = (loss(a, w_oi) - loss(b, w_oi)) / (2 * step)
            assert abs(diff - float(d_ctx[n, k])) < 1e-7 * (1 + abs(diff))
    for part in range(2):
        for h in range(0, w_oi.shape[1], 3):
            for k in range(x.shape[1]):
                a, b = w_oi.clone(), w_oi.clone()
                a[part, h, k] += step
                b[part, h, k] -= step
                diff = (loss(x, a) - loss(x, b)) / (2 * step)
                assert abs(diff - float(d_w[part, k, h])) < 1e-7 * (1 + abs(diff))


@pytest.mark.parametrize('act', F.GATE_ACTIVATIONS)
def test_gated_backward_against_autograd(act):
    x, w_oi, w_io, dy = gated_inputs(N=9, K=16, H=8, seed=2)
    fn = {'silu': torch.nn.functional.silu, 'gelu': torch.nn.functional.gelu,
          'sigmoid': torch.sigmoid, 'tanh': torch.tanh, 'relu': torch.relu}[act]
    xr, wr = x.clone().requires_grad_(True), w_oi.clone().requires_grad_(True)
    y = fn(xr @ wr[0].t()) * (xr @ wr[1].t())
    y.backward(dy)
    got, kept = F.transform_gated_fwd(x, w_oi, act, save=True)
    d_ctx, d_w = F.transform_gated_bwd(x, w_io, kept, dy, act)
    for a, b in ((got, y.detach()), (d_ctx, xr.grad), (d_w, wr.grad.transpose(1, 2))):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)


def test_gated_dropout_mask_is_the_gathers():
    x, w_oi, w_io, dy = gated_inputs(N=40, K=24, H=16, dtype=torch.float32)
    _, kept = F.transform_gated_fwd(x, w_oi, 'silu', save=True)
    plain, _ = F.transform_gated_bwd(x, w_io, kept, dy, 'silu')
    got, _ = F.transform_gated_bwd(x, w_io, kept, dy, 'silu', keep_prob=0.75, seed=77)
    again, _ = F.transform_gated_bwd(x, w_io, kept, dy, 'silu', keep_prob=0.75,
                                     seed_t=torch.tensor([77]))
    mask = R.dropout_keep_mask(77, x.numel(), 0.75, 'cpu').reshape(x.shape)
    assert torch.equal(got, again)
    assert torch.equal(got == 0, ~mask | (plain == 0))
    assert torch.equal(got, F.gather_concat_bwd(plain, 0.75, 77, True))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32, torch.float64])
def test_gated_weight_gradient_in_float32(dtype):
    """float32 on request, from the same sums: rounded they are the default's."""
    x, w_oi, w_io, dy = gated_inputs(N=9, K=16, H=8, seed=3, dtype=dtype)
    _, kept = F.transform_gated_fwd(x, w_oi, save=True)
    d_ctx, d_w = F.transform_gated_bwd(x, w_io, kept, dy)
    again, d_w32 = F.transform_gated_bwd(x, w_io, kept, dy, dw_dtype=torch.float32)
    same = F.transform_gated_bwd(x, w_io, kept, dy, dw_dtype=dtype)[1]
    assert d_w.dtype == same.dtype == dtype and d_w32.dtype == torch.float32
    assert torch.equal(d_ctx, again) and torch.equal(d_w, same)
    small = dtype if dtype == torch.bfloat16 else torch.float32
    assert torch.equal(d_w32.to(small), d_w.to(small))
    for bad in (torch.float16, torch.int32):
        with pytest.raises(ValueError, match='dw_dtype'):
            F.transform_gated_bwd(x, w_io, kept, dy, dw_dtype=bad)


def test_gated_weights_that_changed_in_between():
    """The forward keeps no copy of the weights: the backward of others would be wrong."""
    x, w_oi, w_io, dy = gated_inputs()
    _, kept = F.transform_gated_fwd(x, w_oi, save=True)
    own = kept.clone()
    want = F.transform_gated_bwd(x, w_io, kept, dy)
    w_oi[1].mul_(2.0)
    with pytest.raises(ValueError, match='changed'):
        F.transform_gated_bwd(x, w_io, kept, dy)
    for a, b in zip(F.transform_gated_bwd(x, w_io, own, dy), want):
        assert torch.equal(a, b)
    # kept anew; two forwards keep apart; a read is no change
    _, kept = F.transform_gated_fwd(x, w_oi, save=True)
    w_oi.sum(), w_oi.cpu()
    F.transform_gated_bwd(x, w_io, kept, dy)
    w_oi.zero_()
    F.transform_gated_bwd(x, w_io, F.transform_gated_fwd(x, w_oi, save=True)[1], dy)
    with pytest.raises(ValueError, match='changed'):
        F.transform_gated_bwd(x, w_io, kept, dy)
    with torch.inference_mode():
        v = w_oi.clone()
        F.transform_gated_bwd(x, w_io, F.transform_gated_fwd(x, v, save=True)[1], dy)
        F.transform_gated_bwd(x, w_io, F.transform_gated_fwd(x, w_oi, save=True)[1], dy)
    F.transform_gated_bwd(x, w_io, F.transform_gated_fwd(x, v, save=True)[1], dy)


def test_gated_refusals():
    x, w_oi, w_io, dy = gated_inputs()
    y, kept = F.transform_gated_fwd(x, w_oi, 'silu', save=True)
    assert y.shape == (5, 11) and torch.equal(kept, w_oi)
    assert F.transform_gated_fwd(x, w_oi)[1] is None
    for bad in (lambda: F.transform_gated_fwd(x, w_oi, 'softplus'),
                lambda: F.transform_gated_fwd(x, w_oi[:1]),
                lambda: F.transform_gated_fwd(x[:, :5], w_oi),
                lambda: F.transform_gated_fwd(x[0], w_oi),
                lambda: F.transform_gated_fwd(x.float(), w_oi),
                lambda: F.transform_gated_bwd(x, w_io, None, dy),
                lambda: F.transform_gated_bwd(x, w_io, kept[:1], dy),
                lambda: F.transform_gated_bwd(x, w_io, kept[..., :5], dy),
                lambda: F.transform_gated_bwd(x, w_io.t(), kept, dy),
                lambda: F.transform_gated_bwd(x, w_io, kept, dy[:4]),
                lambda: F.transform_gated_bwd(x, w_io, kept, dy.float()),
                lambda: F.transform_gated_bwd(x, w_io, kept, dy, 'swish'),
                lambda: F.transform_gated_bwd(x, w_io, kept, dy, keep_prob=0.0),
                lambda: F.transform_gated_bwd(x, w_io, kept, dy, keep_prob=1.5)):
        with pytest.raises(ValueError):
            bad()


# ---------------------------------------------------------------------------

def nearest(v, unit):
    """The definition, value by value: the code with the smallest distance,
    of two with the same the even one."""
    size = abs(v) / unit
    best = min(range(8), key=lambda c: (abs(size - R.MXFP4_VALUES[c]), c % 2))
    return math.copysign(R.MXFP4_VALUES[best] * unit, v)


@pytest.mark.parametrize('N,K', [(1, 1), (3, 32), (4, 45), (2, 96)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_mxfp4_against_its_definition(N, K, dtype):
    g = torch.Generator().manual_seed(N + K)
    x = (torch.randn(N, K, generator=g) * 3).to(dtype)
    x[0, 0] = 5.0                                   # a tie when the unit is one
    q = F.mxfp4_quantize(x)
    blocks = -(-K // 32)
    assert q.codes.shape == (N, 16 * blocks) and q.scales.shape == (N, blocks) and q.k == K
    got = F.mxfp4_dequantize(q, torch.float32)
    for n in range(N):
        for b in range(blocks):
            v = [float(t) for t in x[n, 32 * b:32 * b + 32]]
            unit = 2.0 ** (math.frexp(max(map(abs, v)))[1] - 3)
            assert int(q.scales[n, b]) == round(math.log2(unit)) + 127
            assert got[n, 32 * b:32 * b + 32].tolist() == [nearest(t, unit) for t in v]
    assert torch.equal(F.mxfp4_dequantize(q), got.to(torch.bfloat16))
    assert torch.equal(got.to(torch.bfloat16).float(), got)     # exact in either type


def test_mxfp4_packing_and_special_blocks():
    x = torch.zeros(4, 64)
    x[0, :8] = torch.tensor([0.5, -1.0, 1.5, 2.0, -3.0, 4.0, 6.0, -0.5])
    x[1, 40] = float('nan')
    x[2, 3] = float('-inf')
    q = F.mxfp4_quantize(x)
    assert q.codes[0, :4].tolist() == [0xA1, 0x43, 0x6D, 0x97]
    assert q.scales.tolist() == [[127, 0], [0, 255], [255, 0], [0, 0]]
    v = F.mxfp4_dequantize(q, torch.float32)
    assert v[1, 32:].isnan().all() and v[2, :32].isnan().all()
    assert torch.equal(v[0], x[0]) and (v[3] == 0).all() and (v[1, :32] == 0).all()


def test_mxfp4_product_is_that_of_the_values():
    g = torch.Generator().manual_seed(4)
    x, w = torch.randn(6, 70, generator=g), torch.randn(9, 70, generator=g)
    xb = x.to(torch.bfloat16)
    wq, xq = F.mxfp4_quantize(w), F.mxfp4_quantize(xb)
    wv, xv = F.mxfp4_dequantize(wq, torch.float32), F.mxfp4_dequantize(xq, torch.float32)
    y = F.mxfp4_matmul(xb, wq, torch.float32)
    assert torch.allclose(y, xb.float() @ wv.t(), atol=1e-5)
    assert torch.allclose(F.mxfp4_matmul(xq, wq, torch.float32), xv @ wv.t(), atol=1e-5)
    assert F.mxfp4_matmul(xb, wq).dtype == torch.bfloat16


@pytest.mark.parametrize('k', [-1, -5, -62])
def test_mxfp4_rows_of_no_length(k):
    """Rows of fewer than no values, for which the number of blocks comes out as none."""
    none = torch.empty(3, 0, dtype=torch.uint8)
    bad = F.Mxfp4(none, none, k)
    good = F.Mxfp4(none, none, 0)
    assert F.mxfp4_matmul(good, good).shape == (3, 3)
    for call in (lambda: F.mxfp4_dequantize(bad), lambda: F.mxfp4_matmul(bad, bad),
                 lambda: F.mxfp4_matmul(torch.empty(3, 0, dtype=torch.bfloat16), bad)):
        with pytest.raises(ValueError):
            call()


def test_mxfp4_refusals():
    q = F.mxfp4_quantize(torch.randn(4, 40))
    x = torch.randn(3, 40).to(torch.bfloat16)
    for bad in (lambda: F.mxfp4_quantize(torch.zeros(4)),
                lambda: F.mxfp4_quantize(torch.zeros(4, 4, dtype=torch.float16)),
                lambda: F.mxfp4_quantize(torch.zeros(4, 4, dtype=torch.int32)),
                lambda: F.mxfp4_dequantize(q.codes),
                lambda: F.mxfp4_dequantize(q, torch.float16),
                lambda: F.mxfp4_dequantize(F.Mxfp4(q.codes, q.scales, 65)),
                lambda: F.mxfp4_dequantize(F.Mxfp4(q.codes, q.scales[:3], 40)),
                lambda: F.mxfp4_dequantize(F.Mxfp4(q.codes.int(), q.scales, 40)),
                lambda: F.mxfp4_matmul(x, F.Mxfp4(q.codes[:, ::2], q.scales, 40)),
                lambda: F.mxfp4_matmul(x[:, :39], q),
                lambda: F.mxfp4_matmul(x[0], q),
                lambda: F.mxfp4_matmul(x, x),
                lambda: F.mxfp4_matmul(x, q, torch.float16),
                lambda: F.mxfp4_matmul(F.mxfp4_quantize(torch.randn(3, 41)), q)):
        with pytest.raises(ValueError):
            bad()
