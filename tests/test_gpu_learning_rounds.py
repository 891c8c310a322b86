"""Rounds of the framework's paths through the learning operators that come
in another order: a first client without a row-sparse key; and of such that
end early: a refused Muon step; without the host extension; with matrices that
Muon is not to step.

Tolerances are those of test_gpu_learning_paths."""
from collections import OrderedDict

import pytest
import torch

from test_gpu_learning_paths import (_Net, _avg, _cfg, _muon_ref, _row_ref,
                                     _sparse, _uploads)

pytestmark = pytest.mark.gpu


def _round(model, seed, dev, without=(0, ), n=4):
    """Dense matrices and a row-sparse table, which the clients ``without``
    leave out (they touched no row of it)."""
    ups = _uploads(model, n, seed, dev, skip=('emb.weight', ))
    for i, (_, d) in enumerate(ups):
        if i not in without:
            d['emb.weight'] = _sparse((40, 24), 5 + i, 10 * seed + i, dev)
    return ups


@pytest.mark.parametrize('dev', ['cpu', 'cuda'])
@pytest.mark.parametrize('without', [(0, ), (0, 1), (1, 3)])
def test_fedavg_of_row_sparse_uploads_whoever_comes_first(without, dev):
    from federatedscope_amd.core.aggregators import ClientsAvgAggregator
    model = _Net(False).cuda()
    ups = _round(model, 1, dev, without)
    agg = ClientsAvgAggregator(model=model, device='cuda:0', config=_cfg())
    got = agg.aggregate({'client_feedback': ups, 'recover_fun': None})
    assert sorted(got) == ['a.weight', 'b.weight', 'emb.weight']
    if 0 in without:       # not in the first client's order: the model's
        assert list(got) == ['emb.weight', 'a.weight', 'b.weight']
    want, tol = _row_ref(model.state_dict()['emb.weight'], ups, 'emb.weight')
    assert bool(((got['emb.weight'].cpu().double() - want).abs() <=
                 tol).all())
    # and whoever comes first, the matrices as without the table
    plain = ClientsAvgAggregator(model=model, device='cuda:0', config=_cfg())
    dense = [(s, OrderedDict((k, v) for k, v in d.items()
                             if not v.is_sparse)) for s, d in ups]
    alone = plain.aggregate({'client_feedback': dense, 'recover_fun': None})
    for k in alone:
        assert torch.equal(got[k], alone[k])


def test_row_sparse_key_that_another_client_sends_dense():
    from federatedscope_amd.core.aggregators import ClientsAvgAggregator
    model = _Net(False).cuda()
    sp = _sparse((40, 24), 5, 0, 'cuda')
    dense = torch.zeros(40, 24, device='cuda')
    other = torch.zeros(70, 24, device='cuda')
    for vals, who in (((sp, dense), 1), ((None, sp, dense), 2),
                      ((None, dense, sp), 1)):
        ups = [(1, OrderedDict([('a.weight', other)] + (
            [('emb.weight', v)] if v is not None else []))) for v in vals]
        with pytest.raises(ValueError, match='client %d' % who):
            ClientsAvgAggregator(model=model, config=_cfg()).aggregate(
                {'client_feedback': ups, 'recover_fun': None})
    for move in ('cpu', 'cuda'):    # an average of dense tensors by then
        ups = [(1, {'emb.weight': v.to(move)}) for v in (dense, sp)]
        with pytest.raises(RuntimeError, match='parse'):
            ClientsAvgAggregator(model=model, config=_cfg()).aggregate(
                {'client_feedback': ups, 'recover_fun': None})


@pytest.mark.parametrize('dev', ['cpu', 'cuda'])
@pytest.mark.parametrize('rule', ['fedavg', 'SGD', 'Muon'])
def test_server_takes_rows_whoever_comes_first(rule, dev):
    """The first upload to arrive has no rows of the table and is staged; the
    others' rows count all the same."""
    from federatedscope_amd.core import aggregators as A
    from federatedscope_amd.core.workers.server import AggregationServer
    model = _Net(False).cuda()
    if rule == 'fedavg':
        agg = A.ClientsAvgAggregator(model=model, device='cuda:0',
                                     config=_cfg())
    else:
        agg = A.FedOptAggregator(config=_cfg(dict(type=rule, lr=0.5)),
                                 model=model)
    srv = AggregationServer(model, agg, sample_client_num=4, device='cuda:0')
    for rnd in range(2):
        before = {k: v.detach().cpu().double().clone()
                  for k, v in model.state_dict().items()}
        mom = {k: agg._state[k][0].view(v.shape).cpu().double()
               if rule == 'Muon' and k in agg._state else torch.zeros_like(v)
               for k, v in before.items()}
        ups = _round(model, 5 + rnd, dev, without=(0, 2))
        done = [srv.callback_funcs_model_para(rnd, c, u)
                for c, u in enumerate(ups)]
        assert done == [False, False, False, True]
        for k, v in model.state_dict().items():
            avg, tol = _row_ref(before[k], ups, k) if k == 'emb.weight' \
                else (_avg(ups, k), 6 * 2.0**-24 * before[k].abs().max())
            if rule == 'fedavg':
                want = avg
            elif rule == 'SGD':
                want = before[k] - 0.5 * (before[k] - avg)
            else:
                want, _, tol = _muon_ref(before[k], avg, mom[k], 0.5)
            tol = tol + 3 * 2.0**-24 * (want.abs() + (before[k] - avg).abs())
            assert bool(((v.cpu().double() - want).abs() <= tol).all())
            assert not torch.equal(v.cpu().double(), before[k])


@pytest.mark.parametrize('dev', ['cpu', 'cuda'])
def test_staged_uploads_beside_row_sparse_ones_have_landed(dev):
    """Host uploads on their way to their slots (held up on the side stream)
    when a list whose first client sent rows is reduced."""
    from federatedscope_amd.core.aggregators import ClientsAvgAggregator
    from federatedscope_amd.core.workers.ingress import DeviceIngress
    from federatedscope_amd.layout import HostStager
    model = _Net(False).cuda()
    agg = ClientsAvgAggregator(model=model, device='cuda:0', config=_cfg())
    # (two, as many as there are pinned buffers: a third would wait for one)
    ups = _uploads(model, 3, 2, 'cpu', skip=('emb.weight', ))
    rows = _sparse((40, 24), 6, 1, dev)
    first = (ups[0][0], OrderedDict(
        [(k, v.to(dev)) for k, v in ups[0][1].items()] +
        [('emb.weight', rows)]))
    want = agg.aggregate({'client_feedback': [first] + ups[1:],
                          'recover_fun': None})
    ing = DeviceIngress(ups[1][1], 2, device='cuda:0')
    ing._stager = HostStager(ing.device)
    torch.cuda.synchronize()
    with torch.cuda.stream(ing._stager.stream):
        torch.cuda._sleep(100000000)
    staged = [ing.receive(n, d) for n, d in ups[1:]]
    got = agg.aggregate({'client_feedback': [first] + staged,
                         'recover_fun': None})
    assert list(got) == list(want)
    for k in want:
        assert torch.equal(got[k], want[k])


def _all_states(agg):
    return [(k, st[3], [None if t is None else t.clone() for t in st[:3]])
            for a in (agg, agg._aux) for k, st in a._state.items()]


@pytest.mark.parametrize('model_dev', ['cpu', 'cuda'])
@pytest.mark.parametrize('first', [True, False])
def test_a_refused_muon_step_changes_nothing(first, model_dev, monkeypatch):
    """Neither the parameters nor the states nor their counts, Muon's and the
    aux optimizer's; and the step that follows is as if it had not been."""
    from federatedscope_amd import ops
    from federatedscope_amd.core.aggregators import FedOptAggregator
    opt = dict(type='Muon', lr=0.05, aux=dict(type='Adam', lr=0.01))
    models = [_Net(True).to(model_dev) for _ in range(2)]
    aggs = [FedOptAggregator(config=_cfg(opt), model=m) for m in models]
    if not first:
        ups = _uploads(models[0], 3, 8, model_dev)
        for a in aggs:
            a.aggregate({'client_feedback': ups, 'recover_fun': None})
    ups = _uploads(models[0], 3, 9, model_dev)
    info = {'client_feedback': ups, 'recover_fun': None}
    before = {k: v.clone() for k, v in models[0].state_dict().items()}
    states, rounds = _all_states(aggs[0]), aggs[0]._rounds

    def unchanged():
        for k, v in models[0].state_dict().items():
            assert torch.equal(v, before[k])
        now = _all_states(aggs[0])
        had = {k: (n, t) for k, n, t in states}
        for k, n, t in now:
            assert n == (had[k][0] if k in had else 0)
            for x, y in zip(t, had[k][1] if k in had else [None] * 3):
                assert x is None or (torch.equal(x, y) if y is not None else
                                     not x.any())
        assert (aggs[0]._rounds, aggs[0]._aux._rounds) == (rounds, rounds)
    keep = aggs[0].ns_coefficients
    aggs[0].ns_coefficients = (9.0, 9.0, 9.0)
    with pytest.raises(Exception, match='coefficients'):
        aggs[0].aggregate(info)
    unchanged()
    aggs[0].ns_coefficients = keep

    def no_memory(*_, **__):
        raise torch.cuda.OutOfMemoryError('no workspace')
    with monkeypatch.context() as m:
        m.setattr(ops, 'muon_step', no_memory)
        with pytest.raises(torch.cuda.OutOfMemoryError):
            aggs[0].aggregate(info)
    unchanged()
    for a in aggs:
        a.aggregate(info)
    for k, v in models[0].state_dict().items():
        assert torch.equal(v, models[1].state_dict()[k])


def _no_host():
    from federatedscope_amd import _lib
    raise _lib.FsaggError('_fsagg_host.so not found')


def test_paths_without_the_host_extension(monkeypatch):
    """The operators and FedAvg need libfsagg alone: where the host extension
    was not built, the Python ways give the same bits."""
    from federatedscope_amd import _lib, ops
    from federatedscope_amd.core.aggregators import (ClientsAvgAggregator,
                                                     _engine)
    from federatedscope_amd.core.workers.server import AggregationServer
    model = _Net(False).cuda()
    ids = torch.tensor([3, -1, 39, 3], device='cuda')
    table = model.state_dict()['emb.weight']
    ups = _round(model, 3, 'cuda', without=(1, ))

    def run():
        agg = ClientsAvgAggregator(model=model, device='cuda:0',
                                   config=_cfg())
        a = agg.aggregate({'client_feedback': ups, 'recover_fun': None})
        b = agg.aggregate({'client_feedback': [
            (s, {k: v for k, v in d.items() if not v.is_sparse})
            for s, d in ups], 'recover_fun': None})
        other = _Net(False).cuda()
        srv = AggregationServer(other, ClientsAvgAggregator(
            model=other, device='cuda:0', config=_cfg()),
            sample_client_num=4, device='cuda:0')
        for c, u in enumerate(ups):
            srv.callback_funcs_model_para(0, c, u)
        return list(a.values()) + list(b.values()) + list(
            other.state_dict().values()) + [
                ops.embedding_lookup(table, ids, scale=2.0),
                ops.embedding_grad(ids, table[:4], 50)]
    want = run()
    monkeypatch.setattr(_lib, 'host', _no_host)
    monkeypatch.setattr(_engine, '_HOST', [None])
    for x, y in zip(run(), want):
        assert torch.equal(x, y)


@pytest.mark.parametrize('model_dev', ['cpu', 'cuda'])
@pytest.mark.parametrize('rows', [False, True])
def test_fedopt_muon_leaves_the_keys_of_aux_alone(rows, model_dev):
    """A table and a head that aux names take its step exactly as without
    Muon (rows that no client touched stay as they are under SGD), the other
    matrix Muon's."""
    from federatedscope_amd.core.aggregators import FedOptAggregator
    aux = dict(type='SGD', lr=0.5) if rows else dict(type='AdamW', lr=0.01)
    both, alone = _Net(True).to(model_dev), _Net(True).to(model_dev)
    a1 = FedOptAggregator(config=_cfg(dict(type='Muon', lr=0.05, aux=dict(
        aux, keys=['emb.weight', 'b.weight']))), model=both)
    a2 = FedOptAggregator(config=_cfg(aux), model=alone)
    for r in range(2):
        before = {k: v.detach().cpu().double() for k, v in
                  both.named_parameters()}
        mom = a1._state['a.weight'][0].view(70, 24).cpu().double() if r \
            else torch.zeros(70, 24, dtype=torch.float64)
        ups = _uploads(both, 3, r, model_dev)
        if rows:
            for i, (_, d) in enumerate(ups):
                d['emb.weight'] = _sparse((40, 24), 4, 10 * r + i, model_dev)
        info = {'client_feedback': ups, 'recover_fun': None}
        got, want = a1.aggregate(info), a2.aggregate(info)
        for k in got:
            if k != 'a.weight':
                assert torch.equal(got[k], want[k])
        w, _, tol = _muon_ref(before['a.weight'], _avg(ups, 'a.weight'), mom,
                              0.05)
        assert float((got['a.weight'].cpu().double() - w).abs().max()) <= \
            tol + 3 * 2.0**-24 * float(w.abs().max())
        if rows:
            named = set(torch.cat([d['emb.weight']._indices()[0].cpu()
                                   for _, d in ups]).tolist())
            rest = [i for i in range(40) if i not in named]
            assert torch.equal(got['emb.weight'].cpu().double()[rest],
                               before['emb.weight'][rest])
    assert sorted(a1._state) == ['a.weight']


@pytest.mark.parametrize('model_dev', ['cpu', 'cuda'])
def test_select_rows_refuses_other_tokens_wherever_the_model_lies(model_dev):
    from federatedscope_amd.core.workers.server import AggregationServer
    srv = AggregationServer(_Net(False).to(model_dev), None,
                            sample_client_num=1, device='cuda:0')
    for dt in (torch.float32, torch.bool, torch.uint8, torch.int16):
        for n in (3, 60):
            with pytest.raises(ValueError, match='int64 or int32'):
                srv.select_rows('emb.weight', torch.ones(n, dtype=dt))
