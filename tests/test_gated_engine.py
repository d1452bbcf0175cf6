"""The engine with a gated transform and with MXFP4 targets, on the CPU: its
gradients against autograd's, data parallelism, checkpoints, the command line
and what is refused. In fp32, where a sum of D = 24 terms is off by 24 * 2^-24
of its magnitudes, so that 1e-5 is some ten times what all steps add up to."""

import os
import subprocess
import sys

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from code2vec_amd.config import GATE_ACTIVATIONS, Config
from code2vec_amd.models.network import Code2VecNetwork, NullReducer
from code2vec_amd.ops import functional as F
from code2vec_amd.ops import reference as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
B, C, d = 6, 7, 8
V_TOK, V_PATH, V_TGT = 30, 20, 45


def make_cfg(act='silu', **more):
    cfg = Config(set_defaults=True)
    cfg.TRAIN_DATA_PATH_PREFIX = 'unused'
    cfg.MAX_CONTEXTS = C
    cfg.TOKEN_EMBEDDINGS_SIZE = cfg.PATH_EMBEDDINGS_SIZE = d
    cfg.CODE_VECTOR_SIZE = cfg.TARGET_EMBEDDINGS_SIZE = 3 * d
    cfg.DROPOUT_KEEP_RATE = 1.0
    cfg.COMPUTE_DTYPE = 'fp32'
    cfg.DEVICE = 'cpu'
    cfg.TRANSFORM = 'gated'
    cfg.GATE_ACTIVATION = act
    for name, value in more.items():
        setattr(cfg, name, value)
    return cfg


def make_net(act='silu', **more):
    return Code2VecNetwork(make_cfg(act, **more), V_TOK, V_PATH, V_TGT, device='cpu')


def make_batch(seed=3):
    g = torch.Generator().manual_seed(seed)
    src = torch.randint(0, V_TOK, (B, C), generator=g, dtype=torch.int32)
    pth = torch.randint(0, V_PATH, (B, C), generator=g, dtype=torch.int32)
    tgt = torch.randint(0, V_TOK, (B, C), generator=g, dtype=torch.int32)
    mask = (torch.rand(B, C, generator=g) > 0.3).float()
    mask[:, 0] = 1.0
    labels = torch.randint(1, V_TGT, (B,), generator=g)
    return src, pth, tgt, mask, labels


ACT = {'silu': torch.nn.functional.silu, 'gelu': torch.nn.functional.gelu,
       'sigmoid': torch.sigmoid, 'tanh': torch.tanh, 'relu': torch.relu}


def autograd(net, src, pth, tgt, mask, labels, keep=None):
    p = {n: net.get_param(n).detach().double().requires_grad_(True)
         for n in net.param_names()}
    ctx = torch.cat([p['tok_table'][src.long()], p['path_table'][pth.long()],
                     p['tok_table'][tgt.long()]], dim=-1).reshape(B * C, -1)
    if keep is not None:
        ctx = ctx * keep
    comb = ACT[net.config.GATE_ACTIVATION](ctx @ p['w'][0]) * (ctx @ p['w'][1])
    comb = comb.reshape(B, C, -1)
    alpha = torch.softmax(comb @ p['a'] + torch.log(mask), dim=1)
    code = (comb * alpha[..., None]).sum(dim=1)
    loss = torch.nn.functional.cross_entropy(code @ p['target_table'].t(), labels)
    loss.backward()
    return float(loss.detach()), {n: p[n].grad for n in p}


@pytest.mark.parametrize('act', GATE_ACTIVATIONS)
@pytest.mark.parametrize('keep_rate', [1.0, 0.75])
def test_train_step_against_autograd(act, keep_rate):
    """From zero moments a step leaves a tenth of the gradient as Adam's first."""
    net = make_net(act, DROPOUT_KEEP_RATE=keep_rate)
    batch = make_batch()
    keep = None
    if keep_rate < 1.0:
        seed = (net._seed_counter + 2654435761) & 0x7FFFFFFFFFFFFFFF
        keep = R.dropout_keep_mask(seed, B * C * 3 * d, keep_rate, 'cpu')
        keep = keep.reshape(B * C, -1).double() / keep_rate
    want_loss, grads = autograd(net, *batch, keep=keep)
    loss = float(net.train_step(*batch))
    assert abs(loss - want_loss) < 1e-5
    for n in net.param_names():
        got = net._adam_m[n].double() / 0.1
        assert (got - grads[n]).abs().max() < 1e-5, n
    assert net.w.shape == (2, 3 * d, 3 * d)
    # the shadows follow the weights
    assert torch.equal(net.w_oi, net.w.transpose(1, 2))
    assert torch.equal(net.w_io, torch.cat((net.w[0], net.w[1]), dim=1))


def test_the_tanh_engine_is_what_it_was():
    a = Code2VecNetwork(make_cfg(TRANSFORM='tanh'), V_TOK, V_PATH, V_TGT, device='cpu')
    assert a.w.shape == (3 * d, 3 * d) and not a.gated
    assert 'gate_activation' not in a.state_dict()
    src, pth, tgt, mask, _ = make_batch()
    st = a.forward(src, pth, tgt, mask, training=False)
    ctx = torch.cat([a.tok_table[src.long()], a.path_table[pth.long()],
                     a.tok_table[tgt.long()]], dim=-1).reshape(B * C, -1)
    assert torch.allclose(st.comb, torch.tanh(ctx @ a.w), atol=1e-5)
    assert st.kept is None


def test_weight_gradient_is_not_rounded(monkeypatch):
    """In bf16, too, ranks and Adam get the weights' gradient as it was summed, in
    32 bits: next to all of the sums have more than bf16's 8."""
    net = make_net(COMPUTE_DTYPE='bf16')
    seen = {}

    class Watch:
        def __getattr__(self, name):
            return getattr(NullReducer(), name)

        def allreduce_dense(self, name, grad):
            seen[name] = grad.clone()

    calls = []
    inner = F.transform_gated_bwd
    monkeypatch.setattr(F, 'transform_gated_bwd',
                        lambda *a, **kw: calls.append([t.clone() for t in a[:4]])
                        or inner(*a, **kw))
    net.train_step(*make_batch(), reducer=Watch())
    d_w = seen['w']
    assert d_w.dtype == torch.float32
    ctx, w_io, kept, d_y = calls[0]
    want = R.transform_gated_bwd(ctx.float(), w_io.float(), kept.float(), d_y.float(),
                                 'silu')[1]
    assert torch.equal(d_w, want)
    assert (d_w != d_w.to(torch.bfloat16).float()).float().mean() > 0.9
    assert torch.equal(net._adam_m['w'], d_w.mul(1 - net.config.ADAM_BETA1))


def test_forward_for_answers_keeps_nothing():
    st = make_net().forward(*make_batch()[:4], training=False)
    assert st.kept is None


def test_checkpoints(tmp_path):
    net = make_net('gelu')
    for s in range(2):
        net.train_step(*make_batch(s))
    torch.save(net.state_dict(), tmp_path / 'a.pt')
    again = make_net('gelu')
    again.load_state_dict(torch.load(tmp_path / 'a.pt', weights_only=True))
    for s in range(2, 4):
        assert torch.equal(net.train_step(*make_batch(s)), again.train_step(*make_batch(s)))
    for n in net.param_names():
        assert torch.equal(net.get_param(n), again.get_param(n)), n

    release = net.weights_state_dict()
    make_net('gelu').load_state_dict(release)
    for state in (release, net.state_dict()):
        other = make_net('silu')
        before = other.w.clone()
        with pytest.raises(ValueError, match='gelu gates'):
            other.load_state_dict(state)
        with pytest.raises(ValueError, match='tanh transform'):
            make_net(TRANSFORM='tanh').load_state_dict(state)
        assert torch.equal(other.w, before)
    plain = make_net(TRANSFORM='tanh')
    before = net.w.clone()
    with pytest.raises(ValueError, match='gated transform'):
        net.load_state_dict(plain.state_dict())     # (D,D) would fit by broadcasting
    assert torch.equal(net.w, before)


def test_choices():
    for name in ('TRANSFORM', 'GATE_ACTIVATION', 'TARGET_FORMAT'):
        with pytest.raises(ValueError, match=name):
            make_net(**{name: 'softplus'})
    assert GATE_ACTIVATIONS == F.GATE_ACTIVATIONS


@pytest.mark.parametrize('fmt', ['w4', 'w4a4'])
def test_answers_from_mxfp4_targets(fmt):
    net = make_net(TARGET_FORMAT=fmt)
    src, pth, tgt, mask, labels = make_batch()
    buffers = net.target_codes().codes.data_ptr(), net.target_codes().scales.data_ptr()

    def check():
        st = net.forward(src, pth, tgt, mask, training=False)
        q = R.mxfp4_quantize(net.target_table)
        for got, want in zip(net.target_codes()[:2], q[:2]):
            assert torch.equal(got, want)
        x = st.code
        if fmt == 'w4a4':
            x = R.mxfp4_dequantize(R.mxfp4_quantize(x), torch.float32)
        want = x.double() @ R.mxfp4_dequantize(q, torch.float32).double().t()
        idx, scores, code, _ = net.predict_batch(src, pth, tgt, mask, 10)
        assert torch.equal(code, st.code)
        assert torch.allclose(scores.double(), want.topk(10)[0], atol=1e-5)
        assert torch.allclose(want.gather(1, idx.long()), want.topk(10)[0], atol=1e-5)
        _, s2, _, _, loss = net.eval_batch(src, pth, tgt, mask, labels, 10)
        assert torch.equal(s2, scores)
        ce = torch.nn.functional.cross_entropy(want, labels, reduction='sum')
        assert abs(float(loss) - float(ce)) < 1e-4
        assert buffers == (net.target_codes().codes.data_ptr(),
                           net.target_codes().scales.data_ptr())

    check()
    net.train_step(src, pth, tgt, mask, labels)
    check()
    other = make_net(TARGET_FORMAT='full')
    for s in range(3):
        other.train_step(*make_batch(s))
    net.load_state_dict(other.state_dict())
    check()
    # asked for later
    late = make_net()
    late.config.TARGET_FORMAT = fmt
    assert torch.equal(late.predict_batch(src, pth, tgt, mask, 10)[1],
                       make_net(TARGET_FORMAT=fmt).predict_batch(src, pth, tgt, mask, 10)[1])
    # training does not look at the format
    a, b = make_net(TARGET_FORMAT=fmt), make_net()
    assert torch.equal(a.train_step(*make_batch()), b.train_step(*make_batch()))
    assert torch.equal(a.target_table, b.target_table)


def _worker(rank, world_size, init_file, result):
    dist.init_process_group('gloo', init_method='file://' + init_file, rank=rank,
                            world_size=world_size)
    from code2vec_amd.parallel.ddp import Reducer
    net, batch = make_net(), make_batch()
    part = [t[rank * (B // world_size):(rank + 1) * (B // world_size)] for t in batch]
    reducer = Reducer()
    for _ in range(2):
        net.train_step(*part, reducer=reducer)
    if rank == 0:
        torch.save(net.state_dict(), result)
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.timeout(240)
def test_two_ranks_are_one(tmp_path):
    """The ranks' gradients only add up in another order; Adam's first steps
    divide by the gradient's own size, so that 1e-6 of error may become 1e-3 *
    1e-6 / |g| in a parameter: 2e-5 allows for gradients down to 5e-5."""
    result = str(tmp_path / 'n.pt')
    mp.spawn(_worker, args=(2, str(tmp_path / 'init'), result), nprocs=2, join=True)
    got = torch.load(result, weights_only=True)
    net = make_net()
    for _ in range(2):
        net.train_step(*make_batch())
    for n in net.param_names():
        assert (got['adam_m.' + n] - net._adam_m[n]).abs().max() < 1e-6, n
    big = net._adam_m['w'].abs() > 1e-5
    assert (got['w'] - net.w)[big].abs().max() < 2e-5


@pytest.mark.timeout(400)
def test_command_line(tmp_path):
    from test_cli import write_tiny_dataset
    prefix = write_tiny_dataset(tmp_path)
    save = str(tmp_path / 'm' / 'model')
    env = dict(os.environ, PYTHONPATH=ROOT)

    def run(*args, ok=True):
        r = subprocess.run([sys.executable, os.path.join(ROOT, 'code2vec.py'),
                            '--dtype', 'fp32', '--device', 'cpu', '-v', '0', *args],
                           capture_output=True, text=True, env=env, cwd=str(tmp_path))
        assert (r.returncode == 0) == ok, r.stderr[-2000:]
        return r

    gated = ('--transform', 'gated', '--gate-activation', 'gelu')
    run('--data', prefix, '--test', prefix + '.val.c2v', '--save', save,
        '--target-format', 'w4', *gated)
    saved = [f for f in os.listdir(tmp_path / 'm') if f.endswith('__entire-model')]
    model = str(tmp_path / 'm' / saved[0][:-len('__entire-model')])
    run('--load', model, '--test', prefix + '.val.c2v', '--target-format', 'w4a4', *gated)
    run('--load', model, '--release', *gated)
    made = os.listdir(tmp_path / 'm')
    assert any(f.endswith('.release') for f in made)
    assert not any(f.endswith('.index') for f in made)
    # a gated model does not load as another one
    r = run('--load', model, '--test', prefix + '.val.c2v', ok=False)
    assert 'tanh transform' in r.stderr
    r = run('--load', model, '--test', prefix + '.val.c2v', '--transform', 'gated', ok=False)
    assert 'gelu gates' in r.stderr
