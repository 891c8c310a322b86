"""What the learning operators' checks catch, and the host's refusals at
their edges; without a GPU."""
import pytest
import torch

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
