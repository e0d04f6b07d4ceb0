"""What the tensor-level serving calls take, refuse and leave behind: operands changed after they were made, gradients, views that
are not what memory holds, more rows than one launch has."""
import numpy as np
import pytest
import torch

from test_gpu_serving import gen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def S():
    from ecog2txt_amd import serving
    return serving


def test_rows_in_8_bits_are_checked_in_every_call(S):
    """An Int8Rows whose attributes or tensors were changed since it was made: refused where they do not fit (the kernels would read beyond
    them), used as they are where they do."""
    x = torch.randn(7, 100, generator=gen(1), device='cuda')

    def pair():
        return S.quantize_rows(x), S.quantize_rows(torch.randn(50, 100, generator=gen(2), device='cuda'))

    def cols(r): r.cols = 4096
    def none(r): r.cols = 0
    def fewer_scales(r): r.scale = r.scale[:3]
    def more_rows(r): r.q = torch.cat([r.q, r.q])
    def elsewhere(r): r.q = r.q.cpu()
    def scale_elsewhere(r): r.scale = r.scale.cpu()
    def type_(r): r.scale = r.scale.double()
    def not_a_tensor(r): r.q = None
    def unaligned(r): r.q = torch.zeros(r.rows, 144, dtype=torch.int8, device='cuda')[:, 8:136]
    def resized(r): r.q.resize_(r.rows, 64)
    def scale_resized(r): r.scale.resize_(2)
    for change in (cols, none, fewer_scales, more_rows, elsewhere, scale_elsewhere, type_, not_a_tensor, unaligned, resized, scale_resized):
        for which in (0, 1):
            p = pair()
            change(p[which])
            with pytest.raises(ValueError):
                S.matmul_i8(*p)
            if which:
                with pytest.raises(ValueError):
                    S.linear_i8(x, p[1])
    a, w = pair()
    want = S.matmul_i8(a, w)
    a.q, a.scale = a.q[2:5], a.scale[2:5]
    wide = torch.zeros(50, 256, dtype=torch.int8, device='cuda')
    wide[:, :128] = w.q
    w.q = wide                                                         # (another row stride)
    assert torch.equal(S.matmul_i8(a, w), want[2:5])
