"""What the tensor-level serving calls take, refuse and leave behind: operands changed after they were made, gradients, views that
are not what memory holds, more rows than one launch has."""
import pytest
import torch

from test_gpu_serving import check_sample, gen

pytestmark = pytest.mark.gpu


@pytest.fixture
def needs():
    """needs(bytes): skips where the card has not that much; what the test took is given back behind it."""
    def check(n):
        torch.cuda.empty_cache()
        if torch.cuda.mem_get_info()[0] < n:
            pytest.skip('not enough free memory')
    yield check
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


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


def settings(B, seed):
    r = torch.rand(4, B, generator=gen(seed), device='cuda')
    return dict(temperature=0.5 + r[0], top_k=(r[1] * 40).int(), top_p=0.5 + r[2], min_p=0.1 * r[3])


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('B,V', [(65535, 70), (65536, 70), (70001, 1806), ((1 << 22) + 5, 3)])
def test_sample_rows_of_any_number(S, B, V, dtype):
    l = (torch.randn(B, V, generator=gen(B), device='cuda') * 2).to(dtype)
    u, kw = torch.rand(B, generator=gen(2), device='cuda'), settings(B, 3)
    tok, lp = S.sample_rows(l, u, **kw)
    for a in range(0, B, 60000 if B < 1 << 20 else 3 << 20):
        z = min(B, a + (60000 if B < 1 << 20 else 3 << 20))
        t, p = S.sample_rows(l[a:z], u[a:z], **{n: v[a:z] for n, v in kw.items()})
        assert torch.equal(t, tok[a:z]) and torch.equal(p, lp[a:z])
    check_sample(S, l[-40:], u[-40:], **{n: v[-40:] for n, v in kw.items()})


def test_sample_long_rows_of_any_number(S, needs):
    """More long rows than a launch has: copies of a few, each like its original (top-p apart, whose sums depend on the split)."""
    B, V, n = 65535 + 700, 16378, 37
    needs(16 << 30)
    few, u = (torch.randn(n, V, generator=gen(1), device='cuda') * 2).bfloat16(), torch.rand(n, generator=gen(2), device='cuda')
    kw = dict(settings(n, 3), top_p=1.0)
    i = torch.arange(B, device='cuda') % n
    big = {k: v[i] if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    tok, lp = check_sample(S, few, u, **kw)
    t, p = S.sample_rows(few[i], u[i], **big)
    assert torch.equal(t, tok[i]) and torch.equal(p, lp[i])


def test_sample_step_of_many_rows(S, needs):
    """The decoder's bookkeeping behind the first piece of a batch."""
    import ctypes as C
    from ecog2txt_amd import hip_lib as H
    needs(16 << 30)
    V, L, eos, pad = 16378, 3, 1, 0
    n, B = 37, 65535 + 45
    i = torch.arange(B, device='cuda') % n
    few, u = (torch.randn(n, V, generator=gen(1), device='cuda') * 2).bfloat16(), torch.rand(n, generator=gen(2), device='cuda')
    few[5, eos] = 90.0
    got = []
    for l, v in ((few, u), (few[i], u[i])):
        b = len(v)
        temp = (0.5 + torch.arange(n, device='cuda') / n)[torch.arange(b, device='cuda') % n].contiguous()
        done = (torch.arange(b, device='cuda') % n == 9).int()
        out, nxt, score = (torch.full(s, -5, dtype=d, device='cuda') for s, d in (((b, L), torch.int32), ((b,), torch.int32), ((b,), torch.float32)))
        cfg = S.sample_config(b, l.get_device(), temperature=temp, top_k=30)
        need = H.lib.e2t_sample_ws_bytes(b, V)
        ws = torch.empty(need, dtype=torch.uint8, device='cuda')
        H.lib.e2t_sample_step(l.data_ptr(), H.DT_BF16, V, b, V, v.data_ptr(), C.byref(cfg), 1, L, eos, pad, done.data_ptr(), out.data_ptr(), nxt.data_ptr(),
                              score.data_ptr(), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        got.append((done, out, nxt, score))
    for one, many in zip(*got):
        assert torch.equal(one[i], many)
    assert got[0][0][5] == 1 and got[0][1][9, 1] == pad and got[0][3][9] == -5 and (got[0][1][:, [0, 2]] == -5).all()


def test_limits_of_sizes_are_value_errors(S):
    ones = torch.ones(3, device='cuda')
    with pytest.raises(ValueError, match='1048576'):
        S.sample_rows(torch.zeros(3, 1048577, dtype=torch.bfloat16, device='cuda'), ones / 2)
    with pytest.raises(ValueError, match='131071'):
        S.quantize_rows(torch.zeros(1, 131072, device='cuda'))
    store = torch.zeros(2 * 8388624 + 128, dtype=torch.int8, device='cuda')
    with pytest.raises(ValueError, match='8388608'):
        S.Int8Rows(store.as_strided((3, 128), (8388624, 1)), ones, 100)
    # the furthest rows that are served, and one row of any width
    far = store.as_strided((3, 128), (8388608, 1))
    far[:, :100] = torch.randint(-127, 128, (3, 100), generator=gen(1), device='cuda', dtype=torch.int32).to(torch.int8)
    w = S.quantize_rows(torch.randn(20, 100, generator=gen(2), device='cuda'))
    near = far.contiguous()
    assert torch.equal(S.matmul_i8(S.Int8Rows(far, ones, 100), w), S.matmul_i8(S.Int8Rows(near, ones, 100), w))
    assert torch.equal(S.matmul_i8(w, S.Int8Rows(far, ones, 100)), S.matmul_i8(w, S.Int8Rows(near, ones, 100)))
    row = store[None, :store.numel() // 64 * 64]
    assert torch.equal(S.matmul_i8(S.Int8Rows(row, ones[:1], 100), w), S.matmul_i8(S.Int8Rows(near[:1], ones[:1], 100), w))


# ---------------------------------------------------------------------------------------------------- more rows or columns than one launch has
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('M,K', [((1 << 26) + 5, 3), ((1 << 22) + 9, 1030)])
def test_quantize_rows_of_any_number(S, M, K, dtype, needs):
    needs(M * (K + 63) // 64 * 64 + 3 * M * K * 4)
    x = torch.randn(M, K, generator=gen(K), device='cuda').to(dtype)
    r = S.quantize_rows(x)
    step = 1 << 20
    for a in list(range(0, M, step * 8)) + [M - step]:
        part = S.quantize_rows(x[a:a + step])
        assert torch.equal(part.q, r.q[a:a + step]) and torch.equal(part.scale, r.scale[a:a + step])
    if K < 8:                                                          # and as rows of a product
        w = S.quantize_rows(torch.randn(2, K, generator=gen(1), device='cuda'))
        y = S.matmul_i8(r, w)
        for a in (0, 1 << 25, M - 4000):
            assert torch.equal(y[a:a + 4000], S.matmul_i8(S.Int8Rows(r.q[a:a + 4000], r.scale[a:a + 4000], K), w))


def test_product_and_layer_of_any_number_of_columns(S, needs):
    N, K = (1 << 28) + 48, 5
    needs(N * 64 + 12 * N * 4)
    q = torch.zeros(N, 64, dtype=torch.int8, device='cuda')
    q[:, :K] = torch.randint(-127, 128, (N, K), generator=gen(1), device='cuda', dtype=torch.int8)
    w = S.Int8Rows(q, torch.ones(N, device='cuda'), K)
    x = torch.randint(-126, 127, (1, K), generator=gen(2), device='cuda').float()
    x[0, 2] = 127                                                      # (its scale is 1: the quantised row is the row)
    bias = torch.arange(N, device='cuda').remainder(17).float()
    want = (q[:, :K].float() * x).sum(1) + bias                        # (whole numbers below 2^24: exact)
    a = S.quantize_rows(x)
    assert a.scale[0] == 1
    assert torch.equal(S.matmul_i8(a, w, bias=bias)[0], want)
    assert torch.equal(S.linear_i8(x, w, bias=bias)[0], want)
    assert torch.equal(S.linear_i8(x, w, bias=bias, out_dtype=torch.bfloat16)[0], want.bfloat16())


def test_product_of_any_number_of_tiles(S, needs):
    M, N, K = (1 << 18) + 100, 1 << 18, 4
    needs(M * N * 2 + (8 << 30))
    a, w = (S.quantize_rows(torch.randn(n, K, generator=gen(n % 7), device='cuda')) for n in (M, N))
    y = S.matmul_i8(a, w, out_dtype=torch.bfloat16)
    rows = torch.cat([torch.arange(i, i + 64) for i in (0, 65200, 65280, 131000, 262048, 262080, M - 64)] + [torch.randint(M, (300,))]).cuda()
    for i in rows.split(64):
        assert torch.equal(y[i], S.matmul_i8(S.Int8Rows(a.q[i], a.scale[i], K), w, out_dtype=torch.bfloat16))
