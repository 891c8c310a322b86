"""Calls of the learning operators at the edges of what they take: results of
16-bit types, neighbours in a list, lazily negated views, the least divisor.

Tolerances are those of test_gpu_learning, where they are not bits."""
import pytest
import torch

from test_gpu_learning import (A, B, C, LARGE, _chain, _check_ns,
                               _limb_error, _matrix)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('shape', LARGE)
def test_newton_schulz_of_16_bits_is_the_float32_result_rounded(shape, dtype):
    """The same numbers in float32 take the same products and sums: the
    results differ by their one rounding and nothing else."""
    from federatedscope_amd import ops
    batch, rows, cols = shape
    g = torch.stack([_matrix(rows, cols, z) for z in range(min(batch, 2))])
    g = g.repeat((batch + 1) // 2, 1, 1)[:batch].to(dtype).cuda()
    full = ops.newton_schulz(g.float())
    assert torch.equal(ops.newton_schulz(g), full.to(dtype))
    out = torch.empty(shape, dtype=dtype, device='cuda')
    ops.newton_schulz(g.float(), out=out)
    assert torch.equal(out, full.to(dtype))
    _check_ns(full[batch - 1], g[batch - 1].float(), where='cuda')


def test_newton_schulz_is_as_exact_beside_others():
    """A bfloat16 matrix of nearly equal singular values, alone and in a list
    with large ones (whose sums are split elsewhere): as far from 64 bits as
    the exact result's rounding is (the rounding of 1.5 million values near
    them is that to 2 %), and the float32 chain's error."""
    from federatedscope_amd import ops
    g = torch.randn(768, 2048, generator=torch.Generator().manual_seed(1))
    g = g.bfloat16().cuda()
    big = _matrix(4096, 1024, 2).bfloat16().cuda()
    want = _chain(g, torch.float64, where='cuda')
    off = _chain(g, torch.float32, where='cuda') - want
    half = float((want.bfloat16().double() - want).norm())
    tol = 1.02 * half + 4 * float(off.norm()) + _limb_error(
        g, 5, (A, B, C), 1e-7, where='cuda')
    for got in (ops.newton_schulz(g), ops.newton_schulz([g, big, big])[0],
                ops.newton_schulz([big] * 4 + [g])[4]):
        assert float((got.cpu().double() - want).norm()) <= tol
        _check_ns(got, g, where='cuda')


@pytest.mark.parametrize('shape', [(9, 14), (60, 2000), (90, 150),
                                   (1200, 1300)])
def test_newton_schulz_of_zeros_at_any_eps(shape):
    """A zero matrix stays zero however small its divisor."""
    from federatedscope_amd import ops
    z = torch.zeros(*shape, device='cuda')
    for eps in (1e-7, 1e-200, 1e-306, 5e-324):
        assert torch.equal(ops.newton_schulz(z, eps=eps), z)
    g = _matrix(*shape, seed=3).cuda()
    assert torch.equal(ops.newton_schulz(g, eps=5e-324),
                       ops.newton_schulz(g, eps=1e-200))


def _negated(*shape):
    """A view whose memory holds the negative of its values."""
    return torch.randn(*shape, dtype=torch.complex64, device='cuda').conj() \
        .imag


def test_lazily_negated_views_are_refused():
    """Their memory is not what they hold: resolved first, they are taken."""
    from federatedscope_amd import ops
    g = _negated(40, 60)
    assert g.is_neg()
    with pytest.raises(ValueError, match='resolve_neg'):
        ops.newton_schulz(g)
    _check_ns(ops.newton_schulz(g.resolve_neg()), g.resolve_neg())
    x = torch.randn(40, 60, device='cuda')
    with pytest.raises(ValueError, match='resolve_neg'):
        ops.newton_schulz(x, out=torch._neg_view(torch.empty_like(x)))
    for k in range(3):
        t = [x.clone(), x.clone(), x.clone()]
        t[k] = torch._neg_view(t[k])
        with pytest.raises(ValueError, match='resolve_neg'):
            ops.muon_step(t[:1], t[1:2], t[2:], lr=0.1)
    ids = torch.arange(40, device='cuda')
    one = _negated(40, 1)
    for table in (one, torch._neg_view(x)):
        with pytest.raises(ValueError, match='resolve_neg'):
            ops.embedding_lookup(table, ids)
        with pytest.raises(ValueError, match='resolve_neg'):
            ops.embedding_grad(ids, table, 40)
        assert torch.equal(
            ops.embedding_lookup(table.resolve_neg(), ids), table)
        assert torch.equal(
            ops.embedding_grad(ids, table.resolve_neg(), 40), table)
    with pytest.raises(ValueError, match='resolve_neg'):
        ops.embedding_lookup(x, torch._neg_view(ids))
    with pytest.raises(ValueError, match='resolve_neg'):
        ops.embedding_grad(torch._neg_view(ids), x, 40)
    with pytest.raises(ValueError, match='resolve_neg'):
        ops.embedding_lookup(x, ids, out=torch._neg_view(x.clone()))
    for acc in (False, True):
        with pytest.raises(ValueError, match='resolve_neg'):
            ops.embedding_grad(ids, x, 40, out=torch._neg_view(x.clone()),
                               accumulate=acc)


@pytest.mark.parametrize('rows,cols', [(8, 1048576), (130, 1048576),
                                       (1025, 4090 * 256)])
def test_newton_schulz_of_the_longest_is_as_exact(rows, cols):
    """The longest rows that are taken, and planes past 2 GB: within four
    times the float32 chain's error and the limbs' own, over all and for
    every 256 columns of a row (a missing limb is off by a thousandth)."""
    from federatedscope_amd import ops
    t = torch.Generator(device='cuda').manual_seed(rows)
    g = torch.randn(rows, cols, generator=t, device='cuda')

    def chain(x):
        for _ in range(5):
            gram = x @ x.T
            x = A * x + (B * gram + C * (gram @ gram)) @ x
        return x
    x = g.double()
    x /= x.norm()
    y = chain(x.float())
    want = chain(x)
    del x
    got = ops.newton_schulz(g)
    limb = _limb_error(g, 5, (A, B, C), 1e-7, where='cuda')
    del g
    errors = []
    for z in (got, y):
        off = torch.empty(rows, cols // 256, device='cuda',
                          dtype=torch.float64)
        for i in range(0, rows, 64):
            d = z[i:i + 64].double() - want[i:i + 64]
            off[i:i + 64] = d.view(len(d), -1, 256).square().sum(-1).sqrt()
        errors.append(off)
    own, plain = errors
    assert float(own.norm()) <= 4 * float(plain.norm()) + limb
    # a block's share of the limbs' error is at most all of it
    assert bool((own <= 4 * float(plain.max()) + limb).all())


@pytest.mark.parametrize('rows,cols', [(9, 14), (60, 2000), (90, 150)])
def test_newton_schulz_of_negative_strides(rows, cols):
    """A matrix that lies backwards, through the C entry point (torch has no
    such views): the same as its copy the right way round."""
    import ctypes

    from federatedscope_amd import _lib as L
    from federatedscope_amd import ops
    g = _matrix(rows, cols, 4).cuda()
    last = g.data_ptr() + 4 * (rows * cols - 1)
    out = torch.empty_like(g)
    table = (L.NsMat * 1)(L.NsMat(last, out.data_ptr(), rows, cols, 1, 0,
                                  -cols, -1, 0, 0))
    lib = L.load()
    ws = torch.empty(max(16, lib.fsagg_newton_schulz_workspace_bytes(
        table, 1)), dtype=torch.uint8, device='cuda')
    assert lib.fsagg_newton_schulz(
        table, 1, 5, (ctypes.c_double * 3)(A, B, C), 1e-7, ws.data_ptr(),
        ws.numel(), torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(out, ops.newton_schulz(g.flip(0, 1)))
