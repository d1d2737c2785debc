"""The Muon optimizer in training: the flat store's update (core/params.py enable_muon), the Trainer, captured
steps and data parallelism.  The update itself is checked in test_muon.py; here it must be applied to the right
matrices, with everything else left to SGD."""
import os
import tempfile

import pytest
import torch
import torch.multiprocessing as mp

from mx_rcnn_amd.core.lr_scheduler import FactorScheduler
from mx_rcnn_amd.core.params import FlatParamStore, MUON_EXCLUDE
from mx_rcnn_amd.core.trainer import GraphedStep, Trainer
from mx_rcnn_amd.models import FasterRCNN
from mx_rcnn_amd.ops import precision
from mx_rcnn_amd.ops.muon import muon_update_
from mx_rcnn_amd.ops.sgd import sgd_momentum_
from tests.test_dist import _batch as _rcnn_batch
from tests.test_dist import _free_port
from tests.test_model import _batch, _cfg

FIXED = ['conv0', 'stage1', 'stage2', 'bn_data', 'bn0']


def _store(dev, x2=0, dtype=torch.float32):
    torch.manual_seed(0)
    m = FasterRCNN('resnet18', 21, cfg=_cfg()).to(dev)
    st = FlatParamStore(m, FIXED, dtype, dev, dev.type == 'cuda', x2=x2)
    gen = torch.Generator().manual_seed(1)
    for g in st.groups:
        g.grad.copy_(torch.randn(g.numel, generator=gen) * 1e-3)
        g.mom.copy_(torch.randn(g.numel, generator=gen) * 1e-3)
    return st


def _expected(st, lr, mlr):
    """Per parameter, from copies: one muon_update_ of a group's matrices, sgd_momentum_ of everything else.  (The
    matrices of a group in one call: the tiles, and with them the order of the sums, are chosen for the call.)"""
    want = {}
    for g in st.groups:
        wd = 0.0005 if g.decay else 0.0
        mats = tuple((off, e[4][0], e[3] // e[4][0]) for e, off in zip(g.entries, g.offsets)
                     if e[0].endswith('_weight') and len(e[4]) >= 2 and e[0][:-7] not in MUON_EXCLUDE)
        mw, mm = g.master.clone(), g.mom.clone()
        muon_update_(mw, mm, g.grad.clone(), mats, mlr, momentum=0.95, wd=wd, clip=1.0)
        sw, sm = g.master.clone(), g.mom.clone()
        sgd_momentum_(sw, sm, g.grad.clone(), lr, 0.9, wd, 1.0, 1.0)
        inside = {o for o, _, _ in mats}
        for e, off in zip(g.entries, g.offsets):
            w, m = (mw, mm) if off in inside else (sw, sm)
            want[e[0]] = (w[off:off + e[3]], m[off:off + e[3]])
    return want


@pytest.mark.parametrize('dev', ['cpu', pytest.param('cuda', marks=pytest.mark.gpu)])
@pytest.mark.parametrize('clear', [False, True])
def test_store_update(request, dev, clear):
    dev = request.getfixturevalue('cuda') if dev == 'cuda' else torch.device('cpu')
    for x2, dtype in (((0, torch.bfloat16), (2, torch.float32), (3, torch.float32)) if dev.type == 'cuda' else
                      ((0, torch.float32),)):
        st = _store(dev, x2, dtype)
        lr, mlr = torch.tensor([0.01], device=dev), torch.tensor([0.05], device=dev)
        names = st.enable_muon(mlr)
        assert 'stage3_unit1_conv1_weight' in names and 'rpn_conv_3x3_weight' in names
        assert not [n for n in names if n.startswith('stage1') or n[:-7] in MUON_EXCLUDE]
        want = _expected(st, lr, mlr)
        st.sgd_step(lr, 0.9, 0.0005, 1.0, 1.0, refresh=False, clear=clear)
        for g in st.groups:
            if clear:
                assert not bool(g.grad.any())
            for (n, _, _, numel, _, _), off in zip(g.entries, g.offsets):
                assert torch.equal(g.master[off:off + numel], want[n][0]), n
                assert torch.equal(g.mom[off:off + numel], want[n][1]), n
            if g.x2:
                parts = precision.split(g.master, g.x2)
                for k in range(g.x2):
                    assert torch.equal(g.shadow[k * g.plane:k * g.plane + g.numel], parts[k * g.numel:(k + 1) * g.numel])
            elif g.shadow is not None:
                assert torch.equal(g.shadow, g.master.to(g.shadow.dtype))


def test_trainer_options_cpu():
    torch.manual_seed(0)
    m = FasterRCNN('resnet18', 21, cfg=_cfg())
    with pytest.raises(ValueError):
        Trainer(m, 'e2e', device='cpu', optimizer='adam')
    sched = FactorScheduler(2, 0.1)
    tr = Trainer(m, 'e2e', fixed_param_prefix=FIXED, lr=0.001, device='cpu', optimizer='muon', muon_lr_mult=5.0,
                 lr_scheduler=sched)
    assert tr.muon_names and float(tr.muon_lr_t) == pytest.approx(0.005)
    assert tr.store._muon_args[1] == 0.95
    for _ in range(4):
        tr.update_lr()
    assert float(tr.lr_t) == pytest.approx(0.0001) and float(tr.muon_lr_t) == pytest.approx(0.0005)
    sgd = Trainer(m, 'e2e', fixed_param_prefix=FIXED, device='cpu')
    assert sgd.muon_lr_t is None and not sgd.store._muon


def test_step_cpu():
    """A step moves every matrix by about lr along an orthogonal direction, and nothing that is frozen."""
    torch.manual_seed(0)
    m = FasterRCNN('resnet18', 21, cfg=_cfg())
    tr = Trainer(m, 'e2e', fixed_param_prefix=FIXED, lr=0.001, wd=0.0, device='cpu', optimizer='muon')
    before = {k: v.clone() for k, v in tr.store.state_arrays().items()}
    out = tr.step(_batch())
    assert torch.isfinite(out['loss'])
    after = tr.store.state_arrays()
    n = 'stage3_unit1_conv1_weight'
    d = (after[n] - before[n]).reshape(after[n].shape[0], -1)
    s = torch.linalg.svdvals(d.double()) / (0.02 * max(1.0, d.shape[0] / d.shape[1]) ** 0.5)
    assert float(s[0]) < 1.21 and float(s.median()) > 0.3
    assert torch.equal(after['stage1_unit1_conv1_weight'], before['stage1_unit1_conv1_weight'])


def test_states_of_the_other_optimizer(tmp_path):
    """A states file restores the momentum of its own optimizer; of the other one's, all but the matrices'."""
    from tests.test_observability import _tiny_module
    opt = {'learning_rate': 1e-3, 'momentum': 0.9, 'wd': 5e-4}
    files = {}
    for name in ('sgd', 'muon'):
        torch.manual_seed(3)
        mod, data = _tiny_module()
        files[name] = str(tmp_path / name) + '-0001.states'
        mod.fit(data, num_epoch=1, states_prefix=str(tmp_path / name), optimizer=name, optimizer_params=opt)
        if name == 'muon':
            names = mod.trainer.muon_names
            assert names
        kept = {k: v.clone() for k, v in mod.trainer.store.optimizer_state().items()}
        for other in ('sgd', 'muon'):
            mod2, _ = _tiny_module()
            mod2.init_optimizer(optimizer=other, optimizer_params=opt)
            if other == name:
                mod2.load_optimizer_states(files[name])
                for k, v in mod2.trainer.store.optimizer_state().items():
                    assert torch.equal(v, kept[k]), k
    for name, other in (('sgd', 'muon'), ('muon', 'sgd')):
        mod2, _ = _tiny_module()
        mod2.init_optimizer(optimizer=other, optimizer_params=opt)
        mod2.load_optimizer_states(files[name])
        for k, v in mod2.trainer.store.optimizer_state().items():
            assert bool(v.any()) != (k in names), (name, k)


def _worker(rank, world, port, out_dir):
    os.environ.update({'MASTER_ADDR': '127.0.0.1', 'MASTER_PORT': str(port), 'RANK': str(rank),
                       'WORLD_SIZE': str(world), 'LOCAL_RANK': str(rank)})
    from mx_rcnn_amd.parallel import dist as pdist
    pdist.init_distributed(backend='gloo')
    tr = _dp_trainer()
    for k in range(2):
        tr.step(_rcnn_batch(rank + k * world))
    torch.save({k: v.clone() for k, v in tr.store.state_arrays().items()}, os.path.join(out_dir, 'r%d.pt' % rank))
    pdist.barrier()
    pdist.destroy()


def _dp_trainer():
    from tests.test_dist import _make_model
    return Trainer(_make_model(), 'rcnn', fixed_param_prefix=['conv0'], lr=0.001, device='cpu', optimizer='muon')


def test_two_ranks_stay_equal_cpu():
    """Data parallel: each rank updates from the summed gradient, bitwise the same weights; the update is that of the
    sum of both ranks' gradients."""
    with tempfile.TemporaryDirectory() as d:
        mp.spawn(_worker, args=(2, _free_port(), d), nprocs=2, join=True)
        r = [torch.load(os.path.join(d, 'r%d.pt' % k), weights_only=True) for k in range(2)]
    for k in r[0]:
        assert torch.equal(r[0][k], r[1][k]), k
    start = _dp_trainer().store.state_arrays()
    moved = [k for k in start if not torch.equal(start[k], r[0][k])]
    assert 'stage4_unit1_conv1_weight' in moved and 'cls_score_weight' in moved


@pytest.mark.gpu
def test_overlapped_sgd_is_refused(cuda, monkeypatch):
    monkeypatch.setenv('MXR_OVERLAP_SGD', '1')
    with pytest.raises(ValueError):
        Trainer(FasterRCNN('resnet18', 21, cfg=_cfg()), 'e2e', fixed_param_prefix=FIXED, device=cuda, optimizer='muon')


@pytest.mark.gpu
@pytest.mark.parametrize('net,prec', [('resnet50', 'bf16'), ('resnet50', 'fp32'), ('vgg16', 'bf16'), ('vgg16', 'bf16x3')])
def test_graphed_steps_equal_eager_steps(cuda, net, prec):
    """Whole training steps, captured and replayed, against eager ones: the same weights, momentum and shadows."""
    gen = torch.Generator().manual_seed(5)
    rois = torch.tensor([[0., 10, 20, 180, 150], [0., 30, 30, 90, 120], [0., 60, 5, 200, 140], [0., 0, 0, 100, 60]])
    batches = []
    for _ in range(3):
        tgt = torch.zeros(4, 84)
        tgt[0, 12:16] = torch.randn(4, generator=gen)
        inside = torch.zeros(4, 84)
        inside[0, 12:16] = 1
        b = {'data': torch.randn(1, 3, 160, 224, generator=gen) * 50, 'rois': rois,
             'label': torch.tensor([3, 0, 0, 0], dtype=torch.int32), 'bbox_target': tgt, 'bbox_inside_weight': inside,
             'bbox_outside_weight': inside.clone()}
        batches.append({k: v.to(cuda) for k, v in b.items()})

    def trainer():
        torch.manual_seed(0)
        m = FasterRCNN(net, 21, cfg=_cfg())
        if net == 'vgg16':
            m.head.dropout = 0.0
        fixed = FIXED if net == 'resnet50' else ['conv1', 'conv2']
        t = Trainer(m, 'rcnn', fixed_param_prefix=fixed, lr=0.001, device=cuda, precision=prec, optimizer='muon')
        assert not t.fused_fc_sgd and t.muon_names
        return t

    eager, graphed = trainer(), trainer()
    step = GraphedStep(graphed, batches[0], warmup=2)
    for b in batches:
        eager.step(b)
        step(b)
    torch.cuda.synchronize()
    for a, g in zip(eager.store.groups, graphed.store.groups):
        assert torch.equal(a.master, g.master) and torch.equal(a.mom, g.mom)
        assert a.shadow is None or torch.equal(a.shadow, g.shadow)
        assert bool(torch.isfinite(a.master).all())
