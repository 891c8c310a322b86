"""The framework's paths through the learning operators: FedOpt with Muon,
row-sparse uploads through FedAvg and FedOpt, the server's select_rows, and a
round of all of them together.

Tolerances: a FedAvg key is exact (the float32 oracle); a row of a sparse
update is a float32 sum of c products, (c + 2) 2^-24 of the absolute terms;
a Muon step is lr' times the orthogonalisation's error (1e-4 is over ten
times the 8e-6 a float32 chain has on such spectra, and a missing limb or
term is 1e-3 and more) and three roundings of the parameter."""
import math
from collections import OrderedDict
from types import SimpleNamespace

import numpy as np
import pytest
import torch

import oracle as O
from test_gpu_learning import _chain, _matrix

pytestmark = pytest.mark.gpu


def _cfg(optimizer=None, **fedopt):
    return SimpleNamespace(
        federate=SimpleNamespace(ignore_weight=False, use_ss=False,
                                 client_num=10),
        aggregator=SimpleNamespace(byzantine_node_num=0),
        fedopt=SimpleNamespace(optimizer=optimizer or {}, annealing=False,
                               **fedopt))


class _Net(torch.nn.Module):
    def __init__(self, bias):
        super().__init__()
        torch.manual_seed(3)
        self.emb = torch.nn.Embedding(40, 24)
        self.a = torch.nn.Linear(24, 70, bias=bias)
        self.b = torch.nn.Linear(70, 10, bias=bias)
        if bias:
            self.conv = torch.nn.Conv2d(2, 3, 3)


def _uploads(model, n, seed, dev, skip=()):
    out = []
    for i in range(n):
        g = torch.Generator().manual_seed(100 * seed + i)
        d = OrderedDict()
        for k, v in model.state_dict().items():
            if k not in skip:
                x = v.detach().cpu() + 0.01 * torch.randn(
                    v.shape, generator=g)
                d[k] = x.to(dev)
        out.append((10 + 3 * i, d))
    return out


def _avg(ups, k):
    w = O.fedavg_weights([s for s, _ in ups])
    return sum(x * d[k].cpu().double() for x, (_, d) in zip(w, ups))


def _muon_ref(p, avg, m, lr, mu=0.95, wd=0.1, nesterov=True, adjust=None):
    g = p - avg
    m = m + (1 - mu) * (g - m)
    y = _chain(g + mu * (m - g) if nesterov else m, torch.float64)
    r, c = p.shape
    k = 0.2 * math.sqrt(max(r, c)) if adjust else math.sqrt(max(1.0, r / c))
    return (1 - lr * wd) * p - lr * k * y, m, 1e-4 * lr * k


@pytest.mark.parametrize('model_dev', ['cpu', 'cuda'])
@pytest.mark.parametrize('kw', [
    dict(), dict(momentum=0.5, nesterov=False, weight_decay=0.0),
    dict(adjust_lr_fn='match_rms_adamw')])
def test_fedopt_muon_chain(kw, model_dev):
    from federatedscope_amd.core.aggregators import FedOptAggregator
    model = _Net(bias=False).to(model_dev)
    agg = FedOptAggregator(
        config=_cfg(dict(type='Muon', lr=0.05, **kw)), model=model)
    ref = {k: v.detach().cpu().double() for k, v in
           model.named_parameters()}
    mom = {k: torch.zeros_like(v) for k, v in ref.items()}
    for r in range(3):
        ups = _uploads(model, 4, r, 'cpu')
        tols = {}
        for k in ref:
            # from the parameters as they are: a chain's later steps do not
            # add the earlier ones' errors
            p = model.state_dict()[k].cpu().double()
            ref[k], mom[k], tols[k] = _muon_ref(
                p, _avg(ups, k), mom[k], 0.05,
                kw.get('momentum', 0.95), kw.get('weight_decay', 0.1),
                kw.get('nesterov', True), kw.get('adjust_lr_fn'))
        got = agg.aggregate({'client_feedback': ups, 'recover_fun': None})
        assert list(got) == list(ref)
        for k in ref:
            off = (got[k].cpu().double() - ref[k]).abs()
            assert float(off.max()) <= tols[k] + 3 * 2.0**-24 * float(
                ref[k].abs().max())
            mom[k] = agg._state[k][0].view(ref[k].shape).cpu().double()


@pytest.mark.parametrize('model_dev', ['cpu', 'cuda'])
def test_fedopt_muon_aux(model_dev):
    """Matrices take Muon, the rest the aux optimizer exactly as alone."""
    from federatedscope_amd.core.aggregators import FedOptAggregator
    aux = dict(type='AdamW', lr=0.01, weight_decay=0.02)
    both, alone = _Net(True).to(model_dev), _Net(True).to(model_dev)
    a1 = FedOptAggregator(config=_cfg(dict(type='Muon', lr=0.05, aux=aux),
                                      annealing_step_size=1,
                                      annealing_gamma=0.5), model=both)
    a2 = FedOptAggregator(config=_cfg(aux), model=alone)
    muon_only = [k for k, v in both.named_parameters() if v.dim() == 2]
    for r in range(2):
        ups = _uploads(both, 3, r, model_dev)
        before = {k: v.detach().cpu().double() for k, v in
                  both.named_parameters()}
        got = a1.aggregate({'client_feedback': ups, 'recover_fun': None})
        want = a2.aggregate({'client_feedback': ups, 'recover_fun': None})
        for k in got:
            if k not in muon_only:
                assert torch.equal(got[k], want[k])
            elif r == 0:
                w, _, tol = _muon_ref(before[k], _avg(ups, k),
                                      torch.zeros_like(before[k]), 0.05)
                assert float((got[k].cpu().double() - w).abs().max()) <= \
                    tol + 3 * 2.0**-24 * float(w.abs().max())


def test_fedopt_muon_annealing_reaches_both():
    from federatedscope_amd.core.aggregators import FedOptAggregator
    cfg = _cfg(dict(type='Muon', lr=0.4, aux=dict(type='SGD', lr=0.2)),
               annealing_step_size=1, annealing_gamma=0.5)
    cfg.fedopt.annealing = True
    model = _Net(True).cuda()
    agg = FedOptAggregator(config=cfg, model=model)
    for _ in range(2):
        agg.aggregate({'client_feedback': _uploads(model, 2, 0, 'cuda'),
                       'recover_fun': None})
    assert agg._lr() == 0.1 and agg._aux._lr() == 0.05


def test_fedopt_muon_refuses_float64():
    from federatedscope_amd.core.aggregators import FedOptAggregator
    model = torch.nn.Linear(5, 4, bias=False).double().cuda()
    before = model.weight.detach().clone()
    agg = FedOptAggregator(config=_cfg(dict(type='Muon', lr=0.1)),
                           model=model)
    with pytest.raises(NotImplementedError, match='Muon'):
        agg.aggregate({'client_feedback': _uploads(model, 2, 0, 'cuda'),
                       'recover_fun': None})
    assert torch.equal(model.weight, before)


# -- row-sparse uploads ------------------------------------------------------------
def _sparse(shape, nnz, seed, dev, dup=True):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, shape[0], (nnz, ), generator=g) if dup else \
        torch.randperm(shape[0], generator=g)[:nnz]
    val = 0.01 * torch.randn((nnz, ) + tuple(shape[1:]), generator=g)
    return torch.sparse_coo_tensor(ids[None], val, shape).to(dev)


def _row_ref(base, ups, key):
    w = O.fedavg_weights([s for s, _ in ups])
    tot, mag = base.cpu().double().clone(), base.cpu().double().abs()
    cnt = 0
    for x, (_, d) in zip(w, ups):
        if key in d:
            u = d[key].cpu()
            tot += x * u.double().to_dense()
            absu = torch.sparse_coo_tensor(u._indices(),
                                           u._values().abs().double(),
                                           u.shape)
            mag = mag + x * absu.to_dense()
            cnt += u._indices().shape[1]
    return tot, (cnt + 2) * 2.0**-24 * mag


@pytest.mark.parametrize('dev', ['cpu', 'cuda'])
@pytest.mark.parametrize('model_dev', ['cpu', 'cuda'])
def test_fedavg_of_row_sparse_uploads(model_dev, dev):
    """Dense keys bit-exact as ever, the sparse key the weighted sum of the
    clients' updates on the server's value; a client without the key; one
    without a row; repeated rows."""
    from federatedscope_amd.core.aggregators import ClientsAvgAggregator
    model = _Net(False).to(model_dev)
    ups = _uploads(model, 5, 1, dev, skip=('emb.weight', ))
    for i, (_, d) in enumerate(ups):
        if i != 2:
            d['emb.weight'] = _sparse((40, 24), (0 if i == 3 else 9 + i), i,
                                      dev)
            d.move_to_end('emb.weight', last=False)
    agg = ClientsAvgAggregator(model=model, device='cuda:0', config=_cfg())
    base = model.state_dict()['emb.weight'].clone()
    got = agg.aggregate({'client_feedback': ups, 'recover_fun': None})
    assert list(got) == ['emb.weight', 'a.weight', 'b.weight']
    assert torch.equal(model.state_dict()['emb.weight'], base)
    want, tol = _row_ref(base, ups, 'emb.weight')
    assert got['emb.weight'].device.type == dev
    assert bool(((got['emb.weight'].cpu().double() - want).abs() <=
                 tol).all())
    dense = [(s, {k: v.cpu().numpy() for k, v in d.items()
                  if not v.is_sparse}) for s, d in ups]
    for k, w in O.para_weighted_avg(dense).items():
        assert got[k].cpu().numpy().tobytes() == w.tobytes()


def test_row_sparse_keys_of_other_shapes():
    """A vector key and a key with two row dimensions; every key sparse."""
    from federatedscope_amd.core.aggregators import ClientsAvgAggregator

    class M(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.v = torch.nn.Parameter(torch.randn(30))
            self.t = torch.nn.Parameter(torch.randn(30, 3, 5))
    model = M()
    ups = [(1 + i, OrderedDict(v=_sparse((30, ), 8, i, 'cuda'),
                               t=_sparse((30, 3, 5), 6, 9 + i, 'cuda')))
           for i in range(3)]
    got = ClientsAvgAggregator(model=model, config=_cfg()).aggregate(
        {'client_feedback': ups, 'recover_fun': None})
    for k in ('v', 't'):
        want, tol = _row_ref(model.state_dict()[k], ups, k)
        assert got[k].shape == want.shape
        assert bool(((got[k].cpu().double() - want).abs() <= tol).all())


def test_row_sparse_refusals():
    from federatedscope_amd.core.aggregators import ClientsAvgAggregator
    model = _Net(False).cuda()
    sp = _sparse((40, 24), 5, 0, 'cuda')
    dense = torch.zeros(40, 24, device='cuda')

    def run(vals, model=model):
        ups = [(1, {'emb.weight': v}) for v in vals]
        return ClientsAvgAggregator(model=model, config=_cfg()).aggregate(
            {'client_feedback': ups, 'recover_fun': None})
    with pytest.raises(ValueError, match='model'):
        run([sp], model=None)
    with pytest.raises(ValueError, match='client 1'):
        run([sp, dense])
    with pytest.raises(ValueError, match='client 1'):
        run([sp, _sparse((41, 24), 5, 0, 'cuda')])
    two = torch.zeros(40, 24)
    two[1, 2] = 1.0
    with pytest.raises(ValueError, match='client 0'):
        run([two.to_sparse().cuda()])
    with pytest.raises(ValueError):
        run([sp, sp.half()])
    with pytest.raises(ValueError):
        run([sp.double()])
    with pytest.raises(Exception):     # dense first: no sparse form
        run([dense, sp])


@pytest.mark.parametrize('dev', ['cpu', 'cuda'])
@pytest.mark.parametrize('name', [
    'KrumAggregator', 'MedianAggregator', 'TrimmedmeanAggregator',
    'NormboundingAggregator', 'AsynClientsAvgAggregator',
    'ServerClientsInterpolateAggregator', 'OnlineClientsAvgAggregator'])
def test_other_rules_refuse_row_sparse_uploads(name, dev):
    """They read dense tensors: an upload of rows is an error, not a value."""
    from federatedscope_amd.core import aggregators
    cfg = _cfg(dict(type='SGD', lr=1.0))
    cfg.federate.restore_from = ''
    cfg.aggregator = SimpleNamespace(
        byzantine_node_num=1, inside_weight=0.5,
        BFT_args=SimpleNamespace(krum_agg_num=2, normbounding_norm_bound=1.0,
                                 trimmedmean_excluded_ratio=0.2))
    cfg.asyn = SimpleNamespace(staleness_discount_factor=1.0)
    model = _Net(False).cuda()
    ups = _uploads(model, 8, 0, dev, skip=('emb.weight', ))
    for i, (_, d) in enumerate(ups):
        d['emb.weight'] = _sparse((40, 24), 5, i, dev)
    agg = getattr(aggregators, name)(model=model, device='cuda:0', config=cfg)
    with pytest.raises(RuntimeError, match='sparse'):
        if name == 'OnlineClientsAvgAggregator':
            agg.reset()
            agg.inc(ups[0])
        else:
            agg.aggregate({'client_feedback': ups, 'recover_fun': None,
                           'staleness': [(0, 0)] * 8})


@pytest.mark.parametrize('model_dev', ['cpu', 'cuda'])
def test_fedopt_takes_row_sparse_uploads(model_dev):
    """The pseudo-gradient of a sparse key is the clients' negated sum."""
    from federatedscope_amd.core.aggregators import FedOptAggregator
    model = _Net(False).to(model_dev)
    agg = FedOptAggregator(config=_cfg(dict(type='SGD', lr=0.5)),
                           model=model)
    for r in range(2):
        ups = _uploads(model, 3, r, 'cuda', skip=('emb.weight', ))
        for i, (_, d) in enumerate(ups):
            d['emb.weight'] = _sparse((40, 24), 7, 10 * r + i, 'cuda')
        base = model.state_dict()['emb.weight'].detach().cpu().clone()
        full, tol = _row_ref(base, ups, 'emb.weight')
        got = agg.aggregate({'client_feedback': ups, 'recover_fun': None})
        want = base.double() - 0.5 * (base.double() - full)
        # p - avg, its product and the sum round once each
        tol = tol + 3 * 2.0**-24 * (want.abs() + (base - full).abs())
        assert bool(((got['emb.weight'].cpu().double() - want).abs() <=
                     tol).all())


@pytest.mark.parametrize('idt', [torch.int64, torch.int32])
def test_select_rows_of_a_host_model(idt):
    """Few tokens (their rows travel) and more than the table has rows (all of
    it does), padding among them: as from a model on the device."""
    from federatedscope_amd.core.workers.server import AggregationServer
    host = _Net(False)
    dev = _Net(False).cuda()
    dev.load_state_dict(host.state_dict())
    a, b = (AggregationServer(m, None, sample_client_num=1, device='cuda:0')
            for m in (host, dev))
    for tok in (torch.tensor([[3, -1, 39], [40, 3, 0]]),
                torch.arange(-5, 95).reshape(2, 50),
                torch.empty(0, 4), torch.tensor([-1, 77])):
        tok = tok.to(idt)
        for where in ('cpu', 'cuda'):
            got = a.select_rows('emb.weight', tok.to(where), scale=1.5)
            want = b.select_rows('emb.weight', tok.to(where), scale=1.5)
            assert got.is_cuda and torch.equal(got, want)
            assert got.shape == tuple(tok.shape) + (24, )


def test_server_round_with_rows_and_muon():
    """A whole round: each client gets the rows of its tokens, answers with a
    row-sparse update of the table and dense matrices; the server steps the
    matrices with Muon.  Two rounds, host and device clients."""
    from federatedscope_amd.core.aggregators import FedOptAggregator
    from federatedscope_amd.core.workers.server import AggregationServer
    model = _Net(False).cuda()
    agg = FedOptAggregator(config=_cfg(dict(type='Muon', lr=0.05)),
                           model=model)
    srv = AggregationServer(model, agg, sample_client_num=3, device='cuda:0')
    for rnd in range(2):
        before = {k: v.detach().cpu().double().clone() for k, v in
                  model.state_dict().items()}
        mom = {k: agg._state[k][0].view(v.shape).cpu().double()
               if k in agg._state else torch.zeros_like(v)
               for k, v in before.items()}
        ups = []
        for c in range(3):
            tok = torch.tensor([[c, 5, 39], [5, -1, 40]])
            rows = srv.select_rows('emb.weight', tok, scale=2.0)
            assert rows.shape == (2, 3, 24)
            table = before['emb.weight'].float()
            for i in range(2):
                for j in range(3):
                    t = int(tok[i, j])
                    want = table[t] * 2 if 0 <= t < 40 else torch.zeros(24)
                    assert torch.equal(rows[i, j].cpu(), want)
            # the client's gradient by token, uncoalesced
            up = torch.sparse_coo_tensor(
                torch.tensor([[c, 5, 39, 5]]),
                0.01 * rows[0, [0, 1, 2, 1]].cpu(), (40, 24))
            dev = 'cpu' if c == 1 else 'cuda'
            d = _uploads(model, 1, 10 * rnd + c, dev,
                         skip=('emb.weight', ))[0][1]
            d['emb.weight'] = up.to(dev)
            ups.append((5 + c, d))
        done = [srv.callback_funcs_model_para(rnd, c, u)
                for c, u in enumerate(ups)]
        assert done == [False, False, True]
        for k, v in model.state_dict().items():
            avg = _row_ref(before[k], ups, k)[0] if k == 'emb.weight' else \
                _avg(ups, k)
            w, _, tol = _muon_ref(before[k], avg, mom[k], 0.05)
            assert float((v.cpu().double() - w).abs().max()) <= \
                tol + 3 * 2.0**-24 * float(w.abs().max())
