"""What the learning operators' checks catch, and the host's refusals at
their edges; without a GPU."""
import ctypes
from types import SimpleNamespace

import pytest
import torch

from federatedscope_amd import _lib as L
from federatedscope_amd import ops
from federatedscope_amd.core.aggregators import FedOptAggregator
from test_gpu_learning import A, B, C, _chain, _check_ns, _matrix


def _without_last_columns(g):
    """The steps with the last 32 columns left out of every Gram product."""
    x = g.double() / float(g.double().norm())
    for _ in range(5):
        gram = x[:, :-32] @ x[:, :-32].T
        x = A * x + (B * gram + C * (gram @ gram)) @ x
    return x


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_damaged_results_are_told_from_right_ones(dtype):
    """The check of a Newton-Schulz result takes the rounded exact one and
    rejects it with a block, a piece of a row, a column or an element wrong,
    or a stage of every product missing."""
    g = _matrix(300, 400, 1)
    right = _chain(g, torch.float64).to(dtype)
    _check_ns(right, g)
    bad = [right.clone() for _ in range(4)]
    bad[0][256:288, 320:352] = 0
    bad[1][40:48, 64:96] *= -1
    bad[2][:, -1] = 0
    bad[3][299, 7] = 0.5
    for x in bad + [_without_last_columns(g).to(dtype)]:
        with pytest.raises(AssertionError):
            _check_ns(x, g)


def test_sparse_keys_of_every_client_are_seen():
    from federatedscope_amd.core.aggregators.clients_avg_aggregator import \
        sparse_keys_of_all
    sp = torch.sparse_coo_tensor(torch.tensor([[1, 3]]), torch.ones(2, 4),
                                 (5, 4))
    plain = torch.zeros(2)
    assert sparse_keys_of_all([(1, {'a': plain}), (2, 'no dict'),
                               (3, {'b': sp, 'a': plain}), (4, {}),
                               (5, {'c': torch.nn.Parameter(plain), 'd': sp,
                                    'b': sp})]) == ['b', 'd']
    assert sparse_keys_of_all([(1, {'a': plain, 'b': 'text'})]) == []


def _fedopt(model, **kw):
    cfg = SimpleNamespace(
        federate=SimpleNamespace(ignore_weight=False, use_ss=False),
        fedopt=SimpleNamespace(optimizer=dict(type='Muon', lr=0.1, **kw),
                               annealing=False))
    return FedOptAggregator(config=cfg, model=model)


def test_fedopt_muon_refuses_at_once_what_its_step_would():
    """Coefficients, eps and matrices that the step does not take are refused
    with the configuration, not in the first round."""
    model = torch.nn.Linear(3, 2, bias=False)
    for kw, word in ((dict(ns_coefficients=(9.0, 9.0, 9.0)), 'coefficients'),
                     (dict(ns_coefficients=(float('nan'), 0.0, 0.0)),
                      'coefficients'), (dict(eps=float('inf')), 'eps')):
        with pytest.raises(ValueError, match=word):
            _fedopt(model, **kw)
    with pytest.raises(ValueError, match='20000 x 30000'):
        _fedopt(torch.nn.Linear(30000, 20000, bias=False, device='meta'))
    with pytest.raises(ValueError, match='1073741824 elements'):
        _fedopt(torch.nn.Linear(256000, 5376, bias=False, device='meta'))
    _fedopt(torch.nn.Linear(128000, 4096, bias=False, device='meta'))
    _fedopt(None)


def test_muon_check():
    ops.muon_check([])
    ops.muon_check([(3, 4), (0, 7), (16384, 65536), (1048576, 1024)])
    for shapes, kw in (([(3, 4), (16385, 16385)], {}),
                       ([(1, 1048577)], {}), ([(2048, 1048576)], {}),
                       ([(-1, 4)], {}), ([], dict(steps=0)),
                       ([(3, 4)], dict(steps=100)), ([], dict(eps=0.0)),
                       ([], dict(coefficients=(9.0, 9.0, 9.0))),
                       ([], dict(coefficients=(1.0, 2.0)))):
        with pytest.raises(ValueError):
            ops.muon_check(shapes, **kw)
    lib = L.load()
    hp = L.MuonParams(0.1, 0.9, 0.1, A, B, C, 1e-7, 5, 1, 0, 0)
    t = (L.MuonMat * 1)(L.MuonMat(None, None, None, 4, 600))
    assert lib.fsagg_muon_check(t, 1, ctypes.byref(hp)) == 0
    assert lib.fsagg_muon_check(t, 1, None) == -1
    assert lib.fsagg_muon_check(None, 1, ctypes.byref(hp)) == -1
    assert lib.fsagg_muon_check(t, -1, ctypes.byref(hp)) == -1
    hp.adjust = 2
    assert lib.fsagg_muon_check(t, 1, ctypes.byref(hp)) == -1


def test_sparse_keys_without_the_host_extension(monkeypatch):
    from federatedscope_amd.core.aggregators import _engine
    from federatedscope_amd.core.aggregators.clients_avg_aggregator import (
        sparse_keys, sparse_keys_of_all)
    monkeypatch.setattr(_engine, '_HOST', [None])
    sp = torch.sparse_coo_tensor(torch.tensor([[1, 3]]), torch.ones(2, 4),
                                 (5, 4))
    models = [(1, {'a': torch.zeros(2)}), (2, 'no dict'), (3, {'b': sp})]
    assert list(sparse_keys(models[0][1])) == []
    assert sparse_keys(models[2][1]) == ['b']
    assert sparse_keys_of_all(models) == ['b']


def test_embed_abi_refuses_strides():
    """Result rows that overlap (two workgroups would write one place), and
    rows that lie backwards."""
    lib = L.load()
    look = lib.fsagg_embed_lookup
    assert look(4096, 4, 8, -8, 0, 4096, 1, 1, 1.0, 4096, None) == -1
    part = (L.EmbedPart * 1)(L.EmbedPart(4096, 8192, 5, 8, 1.0, 1))

    def grad(vocab, stride, acc=0):
        # (a call that is taken this far lacks its workspace)
        return lib.fsagg_embed_grad(part, 1, 0, vocab, 8, 1 << 20, 0, stride,
                                    acc, None, 0, None)
    for vocab, stride in ((10, 7), (10, 0), (10, -8), (2, 7), (1, -1)):
        assert grad(vocab, stride) == grad(vocab, stride, 1) == -1
    for vocab, stride in ((10, 8), (10, 9), (1, 0), (1, 3)):
        assert grad(vocab, stride) == grad(vocab, stride, 1) == -3


def test_fedopt_muon_aux_keys_config():
    """Matrices that aux names are not Muon's: neither stepped by it nor
    measured against its limits."""
    aux = dict(type='Adam', lr=0.2, keys=['weight'])
    agg = _fedopt(torch.nn.Linear(30000, 20000, bias=False, device='meta'),
                  aux=aux)
    assert agg._aux.opt_type == 'Adam' and 'keys' in aux
    assert not agg._takes('weight', (20000, 30000))
    assert agg._takes('other', (3, 4)) and not agg._takes('other', (3, ))
    with pytest.raises(ValueError, match='nothing.weight'):
        _fedopt(torch.nn.Linear(3, 2), aux=dict(type='SGD', lr=0.1, keys=[
            'weight', 'nothing.weight']))
    with pytest.raises(TypeError, match='list'):
        _fedopt(torch.nn.Linear(3, 2), aux=dict(type='SGD', lr=0.1,
                                                keys='weight'))
    _fedopt(None, aux=dict(type='SGD', lr=0.1, keys=['weight']))


def test_sparse_search_passes_on_what_a_value_raises():
    """A value whose class cannot be asked for is an error, not an abort."""
    class Odd:
        @property
        def __class__(self):
            raise ZeroDivisionError
    host = L.host()
    with pytest.raises(ZeroDivisionError):
        host.has_sparse({'a': Odd()})
    with pytest.raises(ZeroDivisionError):
        host.sparse_dicts([{'a': torch.zeros(2)}, {'b': Odd()}])
    assert host.has_sparse('no dict') is False
    with pytest.raises(TypeError):
        host.sparse_dicts(({}, ))
