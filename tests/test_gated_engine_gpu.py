"""The gated transform and MXFP4 targets together, as a user runs them on the
GPU: training steps, eager and captured, then answers, eager and captured."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from code2vec_amd.config import GATE_ACTIVATIONS, Config  # noqa: E402
from code2vec_amd.models.network import Code2VecNetwork  # noqa: E402
from code2vec_amd.ops import functional as F  # noqa: E402
from code2vec_amd.ops import reference as R  # noqa: E402

V = (500, 300, 203)


def make_net(device='cuda:0', fmt='full', act='silu', keep=1.0, targets=V[2], C=20):
    cfg = Config(set_defaults=True)
    cfg.TRAIN_DATA_PATH_PREFIX = 'unused'
    cfg.MAX_CONTEXTS = C
    cfg.TOKEN_EMBEDDINGS_SIZE = cfg.PATH_EMBEDDINGS_SIZE = 64
    cfg.CODE_VECTOR_SIZE = cfg.TARGET_EMBEDDINGS_SIZE = 192
    cfg.DROPOUT_KEEP_RATE = keep
    cfg.TRANSFORM, cfg.GATE_ACTIVATION, cfg.TARGET_FORMAT = 'gated', act, fmt
    return Code2VecNetwork(cfg, V[0], V[1], targets, device=device)


def batch(seed, B=16, C=20, device='cuda:0'):
    g = torch.Generator().manual_seed(seed)
    src = torch.randint(0, V[0], (B, C), generator=g, dtype=torch.int32)
    pth = torch.randint(0, V[1], (B, C), generator=g, dtype=torch.int32)
    tgt = torch.randint(0, V[0], (B, C), generator=g, dtype=torch.int32)
    mask = (torch.rand(B, C, generator=g) > 0.3).float()
    mask[:, 0] = 1.0
    mask[B // 2] = 0.0                       # a method without contexts
    labels = torch.randint(1, V[2], (B,), generator=g)
    return [t.to(device) for t in (src, pth, tgt, mask, labels)]


@pytest.mark.parametrize('act', GATE_ACTIVATIONS)
def test_gradients_against_the_cpu_engine(act):
    """The CPU engine in fp32 against the GPU's in bf16. From zero moments a
    step leaves a tenth of the gradient as Adam's first. On the way to one are
    at most twelve tensors rounded to bf16 (context, weights, g, u, y, code,
    targets, logits, their gradient, the code's, y's, the pair's, the weights'),
    each by 2^-8 of its elements at most, which comes through one linear or
    smooth step after another: 12 * 2^-8 = 4.7 % of the gradient's norm, twice
    that where relu's slope jumps for the few g that change their sign."""
    gpu, cpu = make_net(act=act), make_net('cpu', act=act)
    cpu.compute_dtype = torch.float32
    for name in ('w_oi', 'w_io', 'target_shadow'):
        setattr(cpu, name, getattr(cpu, name).float())
    cpu._refresh_shadows()
    for n in gpu.param_names():
        assert torch.equal(gpu.get_param(n).cpu(), cpu.get_param(n))
    b = batch(1)
    loss, want = float(gpu.train_step(*b)), float(cpu.train_step(*[t.cpu() for t in b]))
    assert abs(loss - want) < 0.047 * abs(want)
    part = 0.094 if act == 'relu' else 0.047
    for n in gpu.param_names():
        g, w = gpu._adam_m[n].cpu().double(), cpu._adam_m[n].double()
        assert (g - w).norm() < part * w.norm(), (n, float((g - w).norm() / w.norm()))


def test_captured_steps_are_the_eager_ones():
    """With dropout, over several replays. The attention adds its parts up in
    any order, and so do the tables' gradients, as in the engine with tanh: two
    runs may round a few values to bf16 differently. Their gradients then agree
    like two that were rounded at most twelve times (see above), and the
    parameters to the 1e-3 that is Adam's step, as that engine's test has it."""
    eager, graphed = make_net(keep=0.75), make_net(keep=0.75)
    other = make_net(keep=0.75)              # an eager engine that lives meanwhile
    captured = graphed.make_graph_step(16)
    for i, b in enumerate([batch(s) for s in range(4)]):
        le = float(eager.train_step(*b))
        other.train_step(*b)
        lg = float(captured.step(*b))
        assert abs(le - lg) < 5e-3
        if i == 0:
            for n in eager.param_names():
                g, w = graphed._adam_m[n], eager._adam_m[n]
                assert (g - w).norm() < 0.047 * w.norm(), n
    for n in eager.param_names():
        assert (eager.get_param(n) - graphed.get_param(n)).abs().max() < 1e-3, n
    assert torch.equal(graphed.w_oi, graphed.w.transpose(1, 2).to(torch.bfloat16))
    assert torch.equal(graphed.w_io, torch.cat((graphed.w[0], graphed.w[1]), 1)
                       .to(torch.bfloat16))


def check_answers(net, indices, scores, code):
    """What was answered against the codes of the table as it is now. Code
    vectors may differ in their last place from run to run, and a 4-bit float
    by a whole step then, so that scores are held against their own vectors'."""
    q = R.mxfp4_quantize(net.target_table.cpu())
    for got, want in zip(net.target_codes()[:2], q[:2]):
        assert torch.equal(got.cpu(), want)
    x = code.cpu()
    x = (R.mxfp4_dequantize(R.mxfp4_quantize(x), torch.float32)
         if net.config.TARGET_FORMAT == 'w4a4' else x.to(torch.bfloat16)).double()
    w = R.mxfp4_dequantize(q, torch.float32).double()
    exact, size = x @ w.t(), x.abs() @ w.abs().t()
    tol = 192 * 2.0 ** -23 * size + 2.0 ** -8 * exact.abs()
    got = net.logits(code)
    assert ((got.cpu().double() - exact).abs() <= tol).all()
    # the ten best of what was scored
    best, where = F.topk(got, k=scores.shape[1])
    assert torch.equal(best, scores) and torch.equal(where, indices)
    assert torch.equal(scores.double(), got.double().topk(scores.shape[1])[0])


@pytest.mark.parametrize('fmt', ['w4', 'w4a4'])
@pytest.mark.parametrize('B', [1, 7, 200])
def test_train_then_answer(fmt, B):
    """Captured training, then the answers of an eager and of two captured
    predictors that read the same codes, before and after further steps."""
    from code2vec_amd.serving.graph_infer import GraphCapturedPredictor
    net = make_net(fmt=fmt, act='gelu', targets=3001)
    step = net.make_graph_step(16)
    step.step(*batch(1))
    src, pth, tgt, mask, labels = batch(5, B)
    one = GraphCapturedPredictor(net, B, 10)
    two = GraphCapturedPredictor(net, B + 9, 10)

    def check(first):
        # the first to be asked has to see the table that the last step left
        for p in (first, one, two):
            idx, scores, code = p.predict(src, pth, tgt, mask)
            assert idx.shape == scores.shape == (B, 10) and code.shape == (B, 192)
            assert p.out[2].data_ptr() == code.data_ptr()
            check_answers(net, *p.out)
        eager = net.predict_batch(src, pth, tgt, mask, 10)
        check_answers(net, *eager[:3])
        assert torch.allclose(eager[2], one.out[2], atol=1e-5)
        # (the rows' products may add up in another order in a larger batch)
        assert (eager[2] - two.out[2][:B]).norm() <= 2.0 ** -7 * eager[2].norm()
        return net.target_codes().codes.clone()

    before = check(two)
    for s in range(3):
        step.step(*batch(10 + s))
    after = check(one)
    assert not torch.equal(before, after)
    # a captured predictor goes on when others answer from the full table
    net.config.TARGET_FORMAT = 'full'
    full = GraphCapturedPredictor(net, B, 10)
    step.step(*batch(20))
    idx, scores, code = full.predict(src, pth, tgt, mask)
    assert torch.equal(scores, F.topk(code.to(torch.bfloat16) @ net.target_shadow.t(), k=10)[0])
    one.predict(src, pth, tgt, mask)
    net.config.TARGET_FORMAT = fmt
    check_answers(net, *one.out)
    # the loss of an evaluation
    loss = net.eval_batch(src, pth, tgt, mask, labels, 10)[4]
    st = net.forward(src, pth, tgt, mask, training=False)
    want = torch.nn.functional.cross_entropy(net.logits(st.code).float(), labels,
                                             reduction='sum')
    assert abs(float(loss) - float(want)) < 1e-3 * max(1.0, abs(float(want)))


def test_codes_made_on_another_stream():
    net = make_net(fmt='w4', targets=100003)
    b = batch(3)
    side = torch.cuda.Stream()
    for s in range(3):
        net.train_step(*batch(s))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            first = net.predict_batch(*b[:4], 5)
        second = net.predict_batch(*b[:4], 5)      # no wait in between
        torch.cuda.synchronize()
        for answers in (first, second):
            check_answers(net, *answers[:3])


def test_two_calls_at_once():
    """The same calls on two streams, each with tensors of its own, and two captured
    graphs of them that are replayed at once."""
    def inputs(seed, N):
        g = torch.Generator(device='cuda').manual_seed(seed)
        x = torch.randn(N, 200, generator=g, device='cuda').to(torch.bfloat16)
        w = torch.randn(2, 120, 200, generator=g, device='cuda').to(torch.bfloat16) * 0.1
        dy = torch.randn(N, 120, generator=g, device='cuda').to(torch.bfloat16)
        table = torch.randn(3001, 120, generator=g, device='cuda')
        return x, w, w.permute(2, 0, 1).reshape(200, 240).contiguous(), dy, table

    def run(x, w_oi, w_io, dy, table):
        y, kept = F.transform_gated_fwd(x, w_oi, 'silu', save=True)
        d_ctx, d_w = F.transform_gated_bwd(x, w_io, kept, dy, 'silu')
        q = F.mxfp4_quantize(table)
        return y, d_ctx, d_w, F.mxfp4_matmul(y, q), F.mxfp4_matmul(F.mxfp4_quantize(y), q)

    both = [inputs(1, 3000), inputs(2, 2777)]
    want = [run(*i) for i in both]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        got = []
        for s, i in zip(streams, both):
            with torch.cuda.stream(s):
                got.append(run(*i))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(u, v) for u, v in zip(a, b))
    graphs, outs = [], []
    for i in both:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(run(*i))
    for _ in range(4):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert all(torch.equal(u, v) for u, v in zip(a, b))
