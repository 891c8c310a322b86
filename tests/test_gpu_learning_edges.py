"""Calls of the learning operators at the edges of what they take: results of
16-bit types, neighbours in a list.

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
