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


def test_gradients_are_refused_not_lost(S):
    """Every tensor a call takes, asking for a gradient in either mode; without gradients the same calls pass."""
    import torch.autograd.forward_ad as fw
    x, weight = torch.randn(3, 100, generator=gen(1), device='cuda'), torch.randn(50, 100, generator=gen(2), device='cuda')
    a, w = S.quantize_rows(x), S.quantize_rows(weight)
    ones = lambda *n: torch.ones(*n, device='cuda')
    calls = [lambda g: S.quantize_rows(g(x)), lambda g: S.linear_i8(g(x), w), lambda g: S.linear_i8(x, w, bias=g(ones(50))), lambda g: S.matmul_i8(a, w, bias=g(ones(50))),
             lambda g: S.matmul_i8(a, w, out=g(ones(3, 50))), lambda g: S.linear_i8(x, w, out=g(ones(3, 50))), lambda g: S.Int8Rows(w.q, g(ones(50)), 100),
             lambda g: S.sample_rows(g(x), ones(3) / 2), lambda g: S.sample_rows(x, g(ones(3) / 2)), lambda g: S.sample_rows(x, ones(3) / 2, temperature=g(ones(3))),
             lambda g: S.sample_rows(x, ones(3) / 2, top_p=g(ones(3))), lambda g: S.sample_rows(x, ones(3) / 2, min_p=g(ones(3))),
             lambda g: S.sample_config(3, x.get_device(), temperature=g(ones(3)))]
    for c in calls:
        with pytest.raises(ValueError, match='gradient'):
            c(lambda t: t.clone().requires_grad_())
        with pytest.raises(ValueError, match='gradient'):
            c(lambda t: t.clone().requires_grad_() * 1)
        c(lambda t: t)
        with torch.no_grad():
            c(lambda t: t.clone().requires_grad_())
    for c in calls[:-1]:
        with fw.dual_level():
            with pytest.raises(ValueError, match='tangent'):
                c(lambda t: fw.make_dual(t.clone(), torch.ones_like(t)))
    with torch.no_grad():                                              # scales learned elsewhere, used with gradients on
        r = S.Int8Rows(w.q, ones(50).requires_grad_(), 100)
    with pytest.raises(ValueError, match='gradient'):
        S.linear_i8(x, r)


def test_writing_out_is_noticed_by_graphs_that_saved_it(S):
    x, w = torch.randn(3, 100, generator=gen(1), device='cuda'), S.quantize_rows(torch.randn(50, 100, generator=gen(2), device='cuda'))
    for write in (lambda out: S.linear_i8(x, w, out=out), lambda out: S.matmul_i8(S.quantize_rows(x), w, out=out)):
        out = torch.ones(5, 50, device='cuda')
        v = torch.ones(5, 50, device='cuda', requires_grad=True)
        loss = (v * out).sum()
        write(out[1:4])                                                # (a view: the counter is its base's)
        with pytest.raises(RuntimeError, match='inplace'):
            loss.backward()
        with torch.inference_mode():
            o = torch.ones(3, 50, device='cuda')
            assert write(o) is o
        assert torch.equal(write(o), write(None))


def test_negated_views(S):
    """The imaginary part of a conjugate is a view whose memory holds the opposite sign."""
    z = torch.randn(4, 1, dtype=torch.complex64, generator=gen(1), device='cuda')
    x, one = z.conj().imag, z[:1, 0].conj().imag
    assert x.is_neg() and one.is_neg()
    w = S.quantize_rows(torch.ones(1, 1, device='cuda'))
    for call in (lambda f: S.quantize_rows(f(x)), lambda f: S.linear_i8(f(x), w), lambda f: S.linear_i8(x.resolve_neg(), w, bias=f(one)),
                 lambda f: S.sample_rows(f(x), torch.zeros(4, device='cuda')), lambda f: S.sample_rows(x.resolve_neg()[:1], f(one))):
        with pytest.raises(ValueError, match='resolve_neg'):
            call(lambda t: t)
        call(lambda t: t.resolve_neg())
    r = S.quantize_rows(x.resolve_neg()).float()
    assert torch.equal(r.sign(), -z.imag.sign())


@pytest.mark.parametrize('M,N,K', [(1, 50, 100), (7, 300, 640), (700, 300, 64), (2049, 2310, 200), (1942, 1765, 910), (1624, 4899, 144)])
def test_relu_keeps_nan(S, M, N, K):
    """NaN from a bias or a scale stays NaN behind the ReLU, on few rows, tiles and the fused layer."""
    x = torch.randn(M, K, generator=gen(1), device='cuda')
    a, w = S.quantize_rows(x), S.quantize_rows(torch.randn(N, K, generator=gen(2), device='cuda'))
    bias = torch.randn(N, generator=gen(3), device='cuda')
    bias[3] = float('nan'); w.scale[5] = float('nan'); bias[7] = float('-inf'); bias[8] = float('inf')
    for out in (torch.float32, torch.bfloat16):
        for f in (lambda **kw: S.matmul_i8(a, w, bias=bias, out_dtype=out, **kw), lambda **kw: S.linear_i8(x, w, bias=bias, out_dtype=out, **kw)):
            y, r = f(), f(relu=True)
            assert torch.equal(y.isnan().any(0).nonzero()[:, 0], torch.tensor([3, 5], device='cuda')) and y[:, [3, 5]].isnan().all()
            assert torch.equal(r.isnan(), y.isnan()) and torch.equal(r.nan_to_num(nan=1.0), torch.relu(y).nan_to_num(nan=1.0))


@pytest.mark.parametrize('bits', [-1, 0x7FFFFFFF, 0x7FC00000, 0x7F800001, -0x400000])
@pytest.mark.parametrize('M,N,K', [(1, 50, 100), (16, 50, 640), (700, 300, 64)])
def test_nan_of_any_payload_in_bf16_outputs(S, M, N, K, bits):
    """A NaN whose low bits are ones would round up past the largest exponent as a number would."""
    x = torch.randn(M, K, generator=gen(1), device='cuda')
    a, w = S.quantize_rows(x), S.quantize_rows(torch.randn(N, K, generator=gen(2), device='cuda'))
    bias = torch.zeros(N, device='cuda')
    bias.view(torch.int32)[3] = bits
    for y in (S.matmul_i8(a, w, bias=bias, out_dtype=torch.bfloat16), S.linear_i8(x, w, bias=bias, out_dtype=torch.bfloat16)):
        assert torch.equal(y.isnan().any(0).nonzero()[:, 0], torch.tensor([3], device='cuda')) and y[:, 3].isnan().all()
