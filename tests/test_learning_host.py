"""Refusals of the learning operators (Newton-Schulz, Muon, embedding rows):
everything the host rejects before a launch, checked without a GPU."""
import ctypes
from types import SimpleNamespace

import pytest
import torch

from federatedscope_amd import _lib as L
from federatedscope_amd import ops

COEF = (3.4445, -4.7750, 2.0315)


def _err():
    return L.load().fsagg_last_error().decode()


def _ns(mats, steps=5, coef=COEF, eps=1e-7, ws=None, ws_bytes=0):
    t = (L.NsMat * max(1, len(mats)))(*mats)
    return L.load().fsagg_newton_schulz(
        t, len(mats), steps, (ctypes.c_double * 3)(*coef), eps, ws, ws_bytes,
        None)


def _mat(rows=4, cols=6, batch=1, g=4096, out=8192, dtype=0, out_dtype=0):
    return L.NsMat(g, out, rows, cols, batch, rows * cols, cols, 1, dtype,
                   out_dtype)


@pytest.mark.parametrize('kw,word', [
    (dict(steps=0), 'steps'), (dict(steps=100), 'steps'),
    (dict(eps=0.0), 'eps'), (dict(eps=float('nan')), 'eps'),
    (dict(eps=float('inf')), 'eps'),
    (dict(coef=(100.0, 0.0, 0.0)), 'coefficients'),
    (dict(coef=(float('nan'), 0.0, 0.0)), 'coefficients'),
    (dict(coef=(3.0, float('inf'), 0.0)), 'coefficients'),
])
def test_newton_schulz_refuses_settings(kw, word):
    assert _ns([_mat()], **kw) == -1
    assert word in _err()


@pytest.mark.parametrize('kw', [
    dict(rows=-1), dict(cols=-2), dict(batch=-1), dict(rows=20000,
                                                       cols=20000),
    dict(cols=1 << 21), dict(rows=16000, cols=1 << 20), dict(batch=70000),
    dict(g=None), dict(out=None), dict(dtype=3), dict(out_dtype=7)])
def test_newton_schulz_refuses_matrices(kw):
    assert _ns([_mat(), _mat(**kw)], ws=4096, ws_bytes=1 << 40) == -1


def test_newton_schulz_workspace():
    lib = L.load()
    m = _mat(62, 2048, 3)

    def bytes_of(*mats):
        return lib.fsagg_newton_schulz_workspace_bytes(
            (L.NsMat * len(mats))(*mats), len(mats))
    need = bytes_of(m)
    assert need > 0 and need % 16 == 0
    assert _ns([m]) == -3 and 'workspace' in _err()
    assert _ns([m], ws=4096, ws_bytes=need - 1) == -3
    assert _ns([m], ws=4104, ws_bytes=need + 64) == -1
    # nothing to do needs nothing
    assert bytes_of(_mat(0, 5), _mat(5, 0), _mat(batch=0)) == 0
    assert _ns([_mat(0, 5), _mat(5, 0), _mat(batch=0)]) == 0
    assert _ns([]) == 0
    # refused sizes
    assert bytes_of(m, _mat(rows=-1)) == 0


def test_newton_schulz_accepts_tame_coefficients():
    """The bound is on the iterates, not on the coefficients themselves."""
    m = _mat(4, 600)
    for coef in (COEF, (2.0, -1.5, 0.5), (1.5, -0.5, 0.0), (15 / 8, -10 / 8,
                                                            3 / 8)):
        assert _ns([m], coef=coef) == -3      # only the workspace is missing


def test_muon_abi_refusals():
    lib = L.load()
    hp = L.MuonParams(0.1, 0.9, 0.1, *COEF, 1e-7, 5, 1, 0, 0)
    t = (L.MuonMat * 1)(L.MuonMat(4096, 8192, 16384, 4, 600))
    assert lib.fsagg_muon_workspace_bytes(t, 1) > 0
    assert lib.fsagg_muon_workspace_bytes(None, 1) == 0
    assert lib.fsagg_muon_step_f32(t, 1, None, None, 0, None) == -1
    assert lib.fsagg_muon_step_f32(None, 1, ctypes.byref(hp), None, 0,
                                   None) == -1
    assert lib.fsagg_muon_step_f32(t, 1, ctypes.byref(hp), None, 0,
                                   None) == -3
    for k in range(3):
        p = [4096, 8192, 16384]
        p[k] = None
        bad = (L.MuonMat * 1)(L.MuonMat(*p, 4, 6))
        assert lib.fsagg_muon_step_f32(bad, 1, ctypes.byref(hp), 4096,
                                       1 << 30, None) == -1
    hp.adjust = 2
    assert lib.fsagg_muon_step_f32(t, 1, ctypes.byref(hp), 4096, 1 << 30,
                                   None) == -1


def test_embed_abi_refusals():
    lib = L.load()
    look = lib.fsagg_embed_lookup
    assert look(4096, -1, 8, 8, 0, 4096, 1, 1, 1.0, 4096, None) == -1
    assert look(4096, 4, 8, 8, 3, 4096, 1, 1, 1.0, 4096, None) == -1
    assert look(4096, 4, 8, 8, 0, None, 1, 1, 1.0, 4096, None) == -1
    assert look(None, 4, 8, 8, 0, 4096, 1, 1, 1.0, 4096, None) == -1
    for many in (1 << 40, (1 << 62) + 1):
        assert look(4096, 4, 8, 8, 0, 4096, 1, many, 1.0, 4096, None) == -1
    assert look(4096, 4, 1 << 50, 8, 0, 4096, 1, 1, 1.0, 4096, None) == -1
    assert look(None, 4, 8, 8, 0, None, 1, 0, 1.0, None, None) == 0
    part = (L.EmbedPart * 1)(L.EmbedPart(4096, 8192, 5, 8, 1.0, 1))

    def grad(p=part, n=1, dt=0, vocab=10, dim=8, out=1 << 20, odt=0, ld=8,
             acc=0, ws=4096, ws_bytes=1 << 30):
        return lib.fsagg_embed_grad(p, n, dt, vocab, dim, out, odt, ld, acc,
                                    ws, ws_bytes, None)
    assert grad(p=None) == -1
    assert grad(n=-1) == -1
    assert grad(dt=4) == -1
    assert grad(odt=3) == -1
    assert grad(out=None) == -1
    assert grad(vocab=1 << 31) == -1
    for dim in (1 << 31, 1 << 40, (1 << 62) + 8):
        assert grad(dim=dim, ld=dim) == -1
        assert lib.fsagg_embed_grad_workspace_bytes(5, dim, 10) == 0
    assert lib.fsagg_embed_grad_workspace_bytes(1 << 40, 8, 10) == 0
    assert grad(ws=None) == -3
    assert grad(ws_bytes=64) == -3
    assert grad(ws=4100) == -1
    for bad in (L.EmbedPart(None, 8192, 5, 8, 1.0, 1),
                L.EmbedPart(4096, None, 5, 8, 1.0, 1),
                L.EmbedPart(4096, 8192, -5, 8, 1.0, 1),
                L.EmbedPart(4096, 8192, 1 << 29, 8, 1.0, 1)):
        assert grad(p=(L.EmbedPart * 1)(bad)) == -1
    # nothing to do
    assert grad(vocab=0, out=None) == 0
    empty = (L.EmbedPart * 1)(L.EmbedPart(None, None, 0, 8, 1.0, 1))
    assert grad(p=empty, acc=1, ws=None, ws_bytes=0) == 0


def test_operators_have_no_cpu_path():
    x = torch.zeros(4, 6)
    with pytest.raises(ValueError, match='GPU'):
        ops.newton_schulz(x)
    with pytest.raises(ValueError, match='GPU'):
        ops.muon_step([x], [x], [x], lr=0.1)
    with pytest.raises(ValueError, match='GPU'):
        ops.embedding_lookup(x, torch.zeros(3, dtype=torch.long))
    with pytest.raises(ValueError, match='GPU'):
        ops.embedding_grad(torch.zeros(4, dtype=torch.long), x, 5)
    with pytest.raises(TypeError):
        ops.newton_schulz([[1.0]])
    with pytest.raises(ValueError, match='3 values'):
        ops.newton_schulz(x, coefficients=(1.0, 2.0))
    assert ops.newton_schulz([]) == []
    assert ops.muon_step([], [], [], lr=0.1) is None
    with pytest.raises(ValueError, match='not supported'):
        ops.muon_step([x], [x], [x], lr=0.1, adjust_lr='x')
    with pytest.raises(ValueError, match='needs out'):
        ops.embedding_grad(torch.zeros(4, dtype=torch.long), x, 5,
                           accumulate=True)
    with pytest.raises(ValueError, match='negative'):
        ops.embedding_grad(torch.zeros(4, dtype=torch.long), x, -1)
    with pytest.raises(ValueError):
        ops.embedding_grad([], [], 5)


def test_disjoint_check():
    buf = torch.zeros(40)
    a, b, c = buf[:10], buf[10:20], buf[15:25]
    ops._check_disjoint([a, b], [buf[20:30], buf[20:30], buf[25:40]])
    for w, r in (([a, a], []), ([b, c], []), ([a], [a]), ([b], [c]),
                 ([c], [b]), ([a, buf[30:]], [b, c, buf[:1]]),
                 ([buf[3:5]], [buf]), ([buf], [buf[3:5]])):
        with pytest.raises(ValueError, match='overlaps'):
            ops._check_disjoint(w, r)
    ops._check_disjoint([a, buf[5:5]], [buf[7:7]])


def _fedopt(opt, model=None):
    from federatedscope_amd.core.aggregators import FedOptAggregator
    cfg = SimpleNamespace(
        federate=SimpleNamespace(ignore_weight=False, use_ss=False),
        fedopt=SimpleNamespace(optimizer=dict(opt), annealing=False))
    return FedOptAggregator(config=cfg, model=model or torch.nn.Linear(
        3, 2, bias=False))


@pytest.mark.parametrize('kw', [
    dict(lr=-1), dict(lr=0.1, momentum=-1), dict(lr=0.1, weight_decay=-1),
    dict(lr=0.1, adjust_lr_fn='x')])
def test_fedopt_muon_rejects_what_torch_optim_rejects(kw):
    with pytest.raises(ValueError) as want:
        torch.optim.Muon([torch.zeros(2, 3, requires_grad=True)], **kw)
    with pytest.raises(ValueError) as got:
        _fedopt(dict(type='Muon', **kw))
    # torch prints the number as it was given
    assert str(got.value).split(':')[0] == str(want.value).split(':')[0]


def test_fedopt_muon_config():
    agg = _fedopt(dict(type='Muon', lr=0.1))
    assert (agg.momentum, agg.nesterov, agg.weight_decay, agg.ns_steps,
            agg.eps, agg.ns_coefficients) == (0.95, True, 0.1, 5, 1e-7, COEF)
    with pytest.raises(ValueError, match='2D') as got:
        _fedopt(dict(type='Muon', lr=0.1), torch.nn.Linear(3, 2))
    with pytest.raises(ValueError) as want:
        torch.optim.Muon([torch.zeros(2, requires_grad=True)])
    assert str(got.value) == str(want.value)
    for bad in (dict(ns_steps=100), dict(ns_steps=0), dict(eps=0.0),
                dict(ns_coefficients=(1.0, 2.0)),
                dict(aux=dict(type='Muon', lr=0.1))):
        with pytest.raises(ValueError):
            _fedopt(dict(type='Muon', lr=0.1, **bad))
    with pytest.raises(TypeError, match='unexpected'):
        _fedopt(dict(type='Muon', lr=0.1, betas=(0.9, 0.99)))
    with pytest.raises(NotImplementedError):
        _fedopt(dict(type='Muon', lr=0.1, aux=dict(type='LBFGS', lr=1.0)))
    agg = _fedopt(dict(type='Muon', lr=0.1, aux=dict(type='Adam', lr=0.2)),
                  torch.nn.Linear(3, 2))
    assert agg._aux.opt_type == 'Adam' and agg._aux.lr0 == 0.2


def test_sparse_keys_are_seen_and_host_packing_refuses_them():
    from federatedscope_amd.core.aggregators.clients_avg_aggregator import \
        sparse_keys
    sp = torch.sparse_coo_tensor(torch.tensor([[1, 3]]), torch.ones(2, 4),
                                 (5, 4))
    assert sparse_keys({'a': torch.zeros(2), 'b': sp, 'c': 'text',
                        'd': [1.0]}) == ['b']
    dst = torch.zeros(20)
    assert L.host().host_pack_dict(
        {'b': sp}, [('b', 0, 80, 6, 0)], [], dst.data_ptr()) is False
