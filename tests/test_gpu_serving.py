"""The serving operators on the GPU: 8-bit row quantisation, the int8 product and layer, sampling -- against definitions in 64 bits."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
TOP = float(np.finfo(np.float32).max)


@pytest.fixture(scope='module')
def S():
    from ecog2txt_amd import serving
    return serving


def gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


# ---------------------------------------------------------------------------------------------------- quantisation
def quant_oracle(x):
    """(q, scale) by the definition; x float64 holding fp32 / bf16 values.  127 x is exact in double and the quotient's rounding
    cannot reach a border (24-bit operands: at least 2^-33 away from one it does not meet)."""
    fin = np.where(np.isfinite(x), np.abs(x), 0.0)
    top = fin.max(1, keepdims=True)
    with np.errstate(invalid='ignore', divide='ignore'):
        q = np.rint(x * 127.0 / top)
    q = np.where(np.isnan(x) | (top == 0), 0, np.clip(np.where(np.isnan(q), 0, q), -127, 127))
    q = np.where(np.isinf(x), np.where(x > 0, 127, -127), q)
    return q.astype(np.int8), (top[:, 0].astype(np.float32) / np.float32(127)).astype(np.float32)


def check_quant(S, x):
    r = S.quantize_rows(x)
    q, s = quant_oracle(x.double().cpu().numpy())
    K = x.shape[1]
    np.testing.assert_array_equal(r.q.cpu().numpy()[:, :K], q)
    assert not r.q.cpu().numpy()[:, K:].any()
    np.testing.assert_array_equal(r.scale.cpu().numpy(), s)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('M,K', [(1, 1), (3, 7), (5, 64), (2, 65), (17, 800), (64, 801), (9, 2048), (4, 2049), (33, 4104), (3, 16384), (2, 40001),
                                 (700, 130)])
def test_quantize_rows(S, M, K, dtype):
    x = torch.randn(M, K, generator=gen(M * 31 + K), device='cuda').mul(10.0 ** ((M * K) % 7 - 3)).to(dtype)
    check_quant(S, x)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_quantize_rows_borders_and_odd_values(S, dtype):
    K = 301
    x = torch.randn(12, K, generator=gen(5), device='cuda').to(dtype)
    half = torch.arange(-126, 127, device='cuda') + 0.5                # exact borders of the rounding: ties to even
    x[0, :253] = half.to(dtype); x[0, 253:] = 0; x[0, 300] = 127
    x[1] = 0                                                           # a row of zeros
    x[2] = 0; x[2, 7] = -3e38                                          # one value only
    x[3] = float('nan')
    x[4, 3] = float('inf'); x[4, 5] = float('-inf'); x[4, 9] = float('nan')
    x[5] *= 1e-40                                                      # subnormal rows: 127 / top overflows in fp32
    x[6] = 0; x[6, 0] = 1e-45; x[6, 1] = -1e-45
    x[7] = float('inf')
    x[8] = torch.where(x[8] > 0, 1.0, -1.0).to(dtype)
    x[9] *= 1e36
    check_quant(S, x)


def test_quantize_rows_neighbours_of_borders(S):
    """fp32 values one ulp around every border of rows with awkward maxima: each decision is the exact one."""
    tops = torch.tensor([1.0, 3.0, 0.1, 126.99999, 1.9999999, 7e-5, 1.1e30], device='cuda')
    h = torch.arange(0, 127, device='cuda').double() + 0.5
    rows = []
    for t in tops.double():
        b = (h * t / 127).float()
        rows.append(torch.cat([b, torch.nextafter(b, b * 2), torch.nextafter(b, b * 0), -b, t.float()[None]]))
    check_quant(S, torch.stack(rows))


def test_quantize_rows_strided_input(S):
    """Rows of a wider tensor, starting on odd elements: nothing but the view is read."""
    for dtype in (torch.float32, torch.bfloat16):
        big = torch.full((9, 333), float('nan'), dtype=dtype, device='cuda')
        big[1::2, 3:130] = torch.randn(4, 127, generator=gen(3), device='cuda').to(dtype)
        check_quant(S, big[1::2, 3:130])


# ---------------------------------------------------------------------------------------------------- product
def rows_of(S, q, scale=None):
    """Int8Rows of an int8 [rows, cols] array, zero-padded."""
    r, k = q.shape
    buf = torch.zeros(r, (k + 63) // 64 * 64, dtype=torch.int8, device='cuda')
    buf[:, :k] = q
    return S.Int8Rows(buf, scale if scale is not None else torch.ones(r, device='cuda'), k)


def ints(r, c, seed, lo=-127, hi=128):
    return torch.randint(lo, hi, (r, c), generator=gen(seed), device='cuda', dtype=torch.int32).to(torch.int8)


def product_bound(acc, sa, sb, bias, y, out):
    """|error| of the product by its roundings: the sum to fp32, times sa, times sb (2^-24 each), plus bias (2^-24 of the result), and
    the output type's half step; second-order terms are below the one more 2^-24 counted."""
    e = 2.0 ** -24
    b = 4 * e * np.abs(acc * sa[:, None] * sb[None]) + 2 * e * np.abs(y)
    return b + (np.abs(y) + b) * torch.finfo(out).eps / 2 + 1e-44


SHAPES = [(1, 1, 1), (1, 1806, 800), (2, 17, 63), (3, 4100, 129), (8, 257, 2048), (15, 64, 64), (16, 16, 65), (17, 1806, 801), (31, 50, 4104),
          (33, 33, 33), (64, 65, 127), (65, 300, 256), (127, 129, 128), (128, 128, 192), (129, 1806, 320), (300, 257, 1000), (256, 256, 16),
          (513, 770, 801), (1, 5000, 16384), (16, 300, 20000), (5, 8, 70000)]


@pytest.mark.parametrize('M,N,K', SHAPES)
def test_matmul_i8_sums_are_exact(S, M, N, K):
    """Scales of one: the output is the integer sum, rounded once to fp32 (K <= 1040: exact as it stands)."""
    a, b = ints(M, K, M + K), ints(N, K, N * 3 + K)
    want = a.double() @ b.double().t()
    y = S.matmul_i8(rows_of(S, a), rows_of(S, b))
    assert y.shape == (M, N) and y.dtype == torch.float32
    assert torch.equal(y, want.float())


@pytest.mark.parametrize('out', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('bias,relu', [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize('M,N,K', [(1, 1806, 800), (7, 129, 801), (16, 16, 2048), (24, 1806, 2048), (100, 77, 190), (260, 513, 640), (700, 300, 64)])
def test_matmul_i8_scales_bias_relu(S, M, N, K, bias, relu, out):
    a, b = ints(M, K, 1), ints(N, K, 2)
    sa = torch.rand(M, generator=gen(3), device='cuda') * 0.02 + 1e-4
    sb = torch.rand(N, generator=gen(4), device='cuda') * 0.02 + 1e-4
    bi = torch.randn(N, generator=gen(5), device='cuda') if bias else None
    y = S.matmul_i8(rows_of(S, a, sa), rows_of(S, b, sb), bias=bi, out_dtype=out, relu=relu)
    acc = (a.double() @ b.double().t()).cpu().numpy()
    san, sbn = sa.double().cpu().numpy(), sb.double().cpu().numpy()
    want = acc * san[:, None] * sbn[None] + (0 if bi is None else bi.double().cpu().numpy()[None])
    tol = product_bound(acc, san, sbn, bi, want, out)
    if relu:
        want = np.maximum(want, 0)
    assert y.dtype == out
    assert (np.abs(y.double().cpu().numpy() - want) <= tol).all()


@pytest.mark.parametrize('M,N', [(1, 40), (40, 130), (130, 131)])
def test_matmul_i8_at_the_largest_sums(S, M, N):
    """-128 throughout at the longest allowed rows: 128 * 128 * 131071 = 2^31 - 16384 still fits."""
    K = 131071
    a, b = torch.full((M, K), -128, dtype=torch.int8, device='cuda'), torch.full((N, K), -128, dtype=torch.int8, device='cuda')
    b[1::2] = 127
    y = S.matmul_i8(rows_of(S, a), rows_of(S, b))
    want = torch.tensor([128.0 * 128 * K if n % 2 == 0 else -128.0 * 127 * K for n in range(N)], dtype=torch.float64, device='cuda').float()
    assert torch.equal(y, want.expand(M, N))


@pytest.mark.parametrize('out', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('M,N,K', [(1, 77, 100), (9, 33, 65), (70, 130, 129), (300, 260, 70)])
def test_matmul_i8_strides_and_what_lies_around(S, M, N, K, out):
    """Operands that are views of wider buffers full of other numbers, an output that is a view: only the view is written."""
    K64 = (K + 63) // 64 * 64
    bufs = []
    for rows, seed in ((M, 1), (N, 2)):
        buf = torch.full((rows + 2, K64 + 48), 99, dtype=torch.int8, device='cuda')
        buf[1:rows + 1, 16:16 + K64] = 0
        buf[1:rows + 1, 16:16 + K] = ints(rows, K, seed)
        bufs.append(buf)
    v = [b[1:-1, 16:16 + K64] for b in bufs]
    one = lambda n: torch.ones(n, device='cuda')
    frame = torch.full((M + 2, N + 5), -7.0, dtype=out, device='cuda')
    y = S.matmul_i8(S.Int8Rows(v[0], one(M), K), S.Int8Rows(v[1], one(N), K), out_dtype=out, out=frame[1:-1, 3:3 + N])
    want = v[0][:, :K].double() @ v[1][:, :K].double().t()
    assert torch.equal(y, want.to(torch.float32).to(out))
    frame[1:-1, 3:3 + N] = -7.0
    assert (frame == -7.0).all()


@pytest.mark.parametrize('out', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('M,N,K', [(70, 259, 130), (700, 301, 64), (1100, 1305, 700), (2049, 2310, 200), (4099, 4101, 4104), (1030, 9001, 5000)])
def test_matmul_i8_rows_that_start_anywhere(S, M, N, K, out):
    """Every tile size, rows of the output on every alignment: the same values, nothing beside them touched."""
    a, w = ints(M, K, 1), ints(N, K, 2)
    acc = a.double() @ w.double().t()                                  # (whole numbers below 2^53: exact)
    want = acc.float().to(out)
    A, W = rows_of(S, a), rows_of(S, w)
    step = 1 if out is torch.bfloat16 else 2
    for off in range(0, 9, 1 if M < 2000 else 3):
        for more in (0, 1, 2, 4, 7, 8)[::step]:
            big = torch.full((M, N + 8 + more), -7.0, dtype=out, device='cuda')
            y = big[:, off:off + N]
            assert S.matmul_i8(A, W, out_dtype=out, out=y) is y
            assert torch.equal(y, want)
            y.fill_(-7.0)
            assert (big == -7.0).all()


def test_matmul_i8_only_one_operand_needs_zero_padding(S):
    a, b = ints(20, 64, 1), ints(30, 64, 2)
    b[:, 50:] = 0
    y = S.matmul_i8(S.Int8Rows(a, torch.ones(20, device='cuda'), 50), S.Int8Rows(b, torch.ones(30, device='cuda'), 50))
    assert torch.equal(y, (a[:, :50].double() @ b[:, :50].double().t()).float())


# ---------------------------------------------------------------------------------------------------- linear
@pytest.mark.parametrize('out', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('M,N,K', [(1, 1806, 800), (1, 5, 3), (2, 4096, 4096), (3, 257, 801), (4, 300, 16384), (7, 64, 20000), (8, 1806, 2048),
                                   (16, 100, 640), (24, 1806, 2048), (200, 130, 801)])
def test_linear_i8_is_quantise_then_product(S, M, N, K, dtype, out):
    """The same bits as the two calls, and as the definition within the product's roundings."""
    x = torch.randn(M, K, generator=gen(M + N), device='cuda').to(dtype)
    if M > 2:
        x[1] = 0
        x[2, K // 2] = float('inf')
    w = S.quantize_rows(torch.randn(N, K, generator=gen(K), device='cuda'))
    bias = torch.randn(N, generator=gen(9), device='cuda')
    y = S.linear_i8(x, w, bias=bias, out_dtype=out)
    a = S.quantize_rows(x)
    assert torch.equal(y, S.matmul_i8(a, w, bias=bias, out_dtype=out))
    q, s = quant_oracle(x.double().cpu().numpy())
    acc = q.astype(np.float64) @ w.q[:, :K].double().cpu().numpy().T
    sw = w.scale.double().cpu().numpy()
    want = acc * s.astype(np.float64)[:, None] * sw[None] + bias.double().cpu().numpy()[None]
    assert (np.abs(y.double().cpu().numpy() - want) <= product_bound(acc, s.astype(np.float64), sw, bias, want, out)).all()


# ---------------------------------------------------------------------------------------------------- sampling
def sample_oracle(l, u, t=1.0, k=0, p=1.0, m=0.0):
    """One row by the definition (float64): (token, log-probability)."""
    l = np.minimum(np.where(np.isnan(l), -np.inf, l), TOP)
    rank = np.argsort(-l, kind='stable')
    rank = rank[l[rank] > -np.inf]
    if len(rank) == 0:
        return -1, -np.inf
    if not t > 0:
        return int(rank[0]), 0.0
    w = np.exp((l[rank] - l[rank[0]]) / t)
    n = len(rank) if k <= 0 else min(int(k), len(rank))
    if p < 1:
        mass = np.cumsum(w[:n])
        n = min(n, max(1, int(np.searchsorted(mass, p * mass[-1])) + 1))
    if m > 0:
        n = min(n, max(1, int((w >= min(m, 1.0)).sum())))
    left = np.sort(rank[:n])
    w = np.exp((l[left] - l[rank[0]]) / t)
    mass = np.cumsum(w)
    i = min(int(np.searchsorted(mass, u * mass[-1], side='right')), n - 1)
    return int(left[i]), float((l[left[i]] - l[rank[0]]) / t - np.log(mass[-1]))


def lp_bound(lp, V):
    """|error| of a log-probability: half a step of fp32, and the masses' unit -- each of V is off by half of 2^-F of the largest, their
    sum (>= 1) by V * 2^-(F+1), and what lies 32 below the largest may count as nothing (V e^-32)."""
    c = int(np.ceil(np.log2(V))) if V > 1 else 0
    F = min(50, 62 - c)
    return np.abs(lp) * 2.0 ** -24 + V * 2.0 ** -(F + 1) + V * np.exp(-32.0) + 1e-15


def check_sample(S, logits, u, **kw):
    B, V = logits.shape
    tok, lp = S.sample_rows(logits, u, **kw)
    ln, un = logits.double().cpu().numpy(), u.double().cpu().numpy()
    col = lambda n, d: (kw[n].double().cpu().numpy() if isinstance(kw.get(n), torch.Tensor) else np.full(B, float(np.float32(kw.get(n, d)))))
    t, k, p, m = col('temperature', 1.0), col('top_k', 0), col('top_p', 1.0), col('min_p', 0.0)
    want = [sample_oracle(ln[b], un[b], t[b], k[b], p[b], m[b]) for b in range(B)]
    wt, wl = np.array([x[0] for x in want]), np.array([x[1] for x in want])
    np.testing.assert_array_equal(tok.cpu().numpy(), wt)
    got = lp.double().cpu().numpy()
    fin = np.isfinite(wl)
    np.testing.assert_array_equal(np.isfinite(got), fin)
    assert (np.abs(got[fin] - wl[fin]) <= lp_bound(wl[fin], V)).all()
    return tok, lp


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=5), dict(top_k=50, temperature=1.3), dict(top_p=0.9), dict(top_p=0.3, temperature=2.0),
            dict(top_p=0.0), dict(min_p=0.1), dict(min_p=1.0), dict(top_k=40, top_p=0.95, min_p=0.02, temperature=0.8), dict(temperature=0.0),
            dict(top_k=700, top_p=0.999), dict(top_k=10 ** 9, top_p=1.5, min_p=-1.0), dict(temperature=50.0, top_p=0.6), dict(temperature=0.01, top_p=0.99)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('V', [1, 2, 3, 63, 64, 65, 1000, 1806, 2048, 2049, 5003, 8192, 8193, 16384, 16385, 33333, 131072])
def test_sample_rows_settings(S, V, dtype):
    for i, kw in enumerate(SETTINGS):
        B = 5 if V < 20000 else 2
        l = (torch.randn(B, V, generator=gen(100 * i + V), device='cuda') * (1.0 + i % 4)).to(dtype)
        u = torch.rand(B, generator=gen(i + 7 * V), device='cuda')
        check_sample(S, l, u, **kw)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('B,V', [(300, 1806), (70, 5000), (33, 20011), (16, 70001), (513, 70), (8, 128003)])
def test_sample_rows_mixed_settings_a_row(S, B, V, dtype):
    g = gen(B + V)
    r = torch.rand(5, B, generator=g, device='cuda')
    i = torch.arange(B, device='cuda')
    l = (2.5 * torch.randn(B, V, generator=g, device='cuda')).to(dtype)
    l[i % 4 == 1, : V // 2] = float('-inf')
    kw = dict(temperature=torch.where(i % 5 == 0, torch.zeros(()).cuda(), 0.5 + r[1]), top_k=torch.where(i % 2 == 0, (r[2] * 300).int(), torch.zeros((), dtype=torch.int32).cuda()),
              top_p=torch.where(i % 3 != 0, 0.5 + 0.5 * r[3], torch.ones(()).cuda()), min_p=torch.where(i % 7 == 0, 0.1 * r[4], torch.zeros(()).cuda()))
    check_sample(S, l, r[0].contiguous(), **kw)


@pytest.mark.parametrize('V', [8, 1806, 9000, 40000])
def test_sample_rows_ties(S, V):
    """Equal logits rank by index: flat rows, rows of two or of a few dozen levels, borders of u hit exactly."""
    B = 16
    l = torch.zeros(B, V, device='cuda')
    l[4:8] = torch.randint(0, 2, (4, V), generator=gen(V), device='cuda').float()
    l[8:12] = torch.randint(-20, 20, (4, V), generator=gen(V + 1), device='cuda').float() * 0.25
    l[12:] = 1e-3 * torch.randint(0, 3, (4, V), generator=gen(V + 2), device='cuda').float()
    l[::3] *= -1.0                                                     # (-0 among them: ties with +0)
    u = torch.tensor([0.0, 0.5, 0.25, 1 - 2.0 ** -24], device='cuda').repeat(4)
    for kw in (dict(), dict(top_k=3), dict(top_k=V - 1), dict(top_p=0.5), dict(top_p=0.37), dict(top_k=V // 2, top_p=0.8), dict(min_p=0.9), dict(top_k=V // 3, temperature=0.3)):
        check_sample(S, l, u, **kw)
        check_sample(S, l.bfloat16(), u, **kw)


@pytest.mark.parametrize('V', [5, 1806, 30000])
def test_sample_rows_masks_and_extremes(S, V):
    ninf, inf, nan = float('-inf'), float('inf'), float('nan')
    for dtype in (torch.float32, torch.bfloat16):
        low = torch.finfo(dtype).min
        l = torch.randn(14, V, generator=gen(V), device='cuda').to(dtype)
        l[0] = ninf                                                    # nothing left
        l[1] = nan
        l[2] = ninf; l[2, V - 1] = -3.0                                # one left
        l[3] = low                                                     # masks of the lowest value only: a flat row
        l[4] = low; l[4, V // 2] = 1.0
        l[5, 0] = inf                                                  # +inf: the largest finite number
        l[6, ::2] = inf
        l[7, 1] = nan; l[7, 0] = ninf
        l[8] = low; l[8, ::2] = ninf
        l[9] *= 1e30                                                   # far apart
        l[10] = -l[10].abs() * 1e38
        l[11] = 5e4 + l[11]                                            # far from zero
        l[12] *= 1e-30
        l[13] = torch.finfo(dtype).max
        u = torch.rand(14, generator=gen(V + 1), device='cuda')
        for kw in (dict(), dict(top_k=2), dict(top_p=0.7), dict(min_p=0.5), dict(top_k=3, top_p=0.5, min_p=0.01, temperature=0.5), dict(temperature=0.0),
                   dict(temperature=1e-30), dict(temperature=1e30, top_p=0.5), dict(temperature=float('inf'), top_k=4)):
            tok, lp = check_sample(S, l, u, **kw)
            assert tok[0] == -1 and tok[1] == -1 and lp[0] == ninf


def test_sample_rows_uniforms_out_of_range(S):
    l = torch.zeros(6, 10, device='cuda')
    u = torch.tensor([-1.0, float('nan'), 1.0, 7.0, float('inf'), 0.95], device='cuda')
    tok, _ = S.sample_rows(l, u)
    assert tok.tolist() == [0, 0, 9, 9, 9, 9]


def test_sample_rows_strided_and_unaligned(S):
    for dtype in (torch.float32, torch.bfloat16):
        for V in (77, 1806, 20000):
            big = torch.full((7, V + 9), float('inf'), dtype=dtype, device='cuda')
            big[1::2, 3:3 + V] = torch.randn(3, V, generator=gen(V), device='cuda').to(dtype)
            u = torch.rand(3, generator=gen(1), device='cuda')
            check_sample(S, big[1::2, 3:3 + V], u, top_p=0.9, top_k=30)


@pytest.mark.parametrize('T,unit', [(49.0, 49.0), (3.0, 1.0), (7.0, 7.0), (1.0, 0.25), (0.7, 0.7)])
def test_sample_rows_levels_on_bin_borders(S, T, unit):
    """Long rows whose logits are a few whole multiples of one number: workgroups that have not seen the largest one count from another
    level, and every level may lie on a border of the counting."""
    B, V = 6, 40000
    g = gen(int(T * 10))
    level = torch.randint(1, 12, (B, V), generator=g, device='cuda').float()
    level[:, :V // 2] = level[:, :V // 2].clamp(min=5)
    level[3:, V // 2:] += 3
    l = -level * unit
    l[:, 77] = 0
    for kw in (dict(top_k=300), dict(top_k=9000), dict(top_k=V - 5), dict(top_k=30000, top_p=0.83), dict(top_p=0.77), dict(top_k=20000, top_p=0.9, min_p=1e-3)):
        check_sample(S, l, torch.rand(B, generator=g, device='cuda'), temperature=T, **kw)


@pytest.mark.parametrize('V', [3, 40, 1806, 2041, 2042, 6000, 8185, 8186, 16377, 16378, 20011])
@pytest.mark.parametrize('sd,T', [(0.05, 1.0), (1e-4, 1.0), (30.0, 1.0), (1.0, 40.0), (1.0, 1e-3), (1e-30, 1.0), (1e30, 1.0)])
def test_sample_rows_flat_and_steep(S, V, sd, T):
    """Spreads from nothing to beyond what weighs anything."""
    B = 5
    g = gen(V + int(T))
    l = torch.randn(B, V, generator=g, device='cuda') * sd
    l[1, ::2] = float('-inf')
    l[2] = l[2, 0]
    for kw in (dict(top_k=2), dict(top_k=50), dict(top_k=V - 1), dict(top_k=V // 2 + 1, top_p=0.7), dict(top_k=7, min_p=0.9)):
        check_sample(S, l, torch.rand(B, generator=g, device='cuda'), temperature=T, **kw)


def test_sample_rows_logits_closer_than_their_distances(S):
    """Most logits so near zero that their distances to the largest are all the same number in double precision: they still rank by value."""
    B, V = 4, 30000
    l = torch.randn(B, V, generator=gen(8), device='cuda') * 1e-20
    l[:, 5] = 1.0
    l[1, 5] = 2.0
    for kw in (dict(top_k=50), dict(top_k=20000), dict(top_k=29999), dict(top_k=1)):
        check_sample(S, l, torch.rand(B, generator=gen(9), device='cuda'), **kw)
    short = l[:, :6000].contiguous()
    check_sample(S, short, torch.rand(B, generator=gen(9), device='cuda'), top_k=50)


def test_sample_rows_tails_that_weigh_nothing(S):
    """The longest row: one token and a million whose masses are below half a unit; the nucleus asks for more than the one."""
    V = 1 << 20
    l = torch.full((3, V), -29.85, device='cuda')
    l[:, 31] = 0
    l[1, 32:] = float('-inf')
    for kw in (dict(top_p=1 - 2.0 ** -24), dict(top_p=1 - 2.0 ** -24, top_k=500000), dict()):
        tok, lp = S.sample_rows(l, torch.tensor([0.0, 0.5, 0.9], device='cuda'), **kw)
        assert tok.tolist() == [31] * 3
        assert (lp.abs().double().cpu().numpy() <= V * np.exp(-29.85) + lp_bound(0.0, V)).all()      # (at most the whole tail was kept)


def test_sample_rows_frequencies(S):
    """Evenly spread u: token counts are the kept probabilities to one count (the inverse of the running sum)."""
    V, n = 50, 4096
    l = torch.randn(1, V, generator=gen(1), device='cuda')
    u = (torch.arange(n, device='cuda') + 0.5) / n
    tok, _ = S.sample_rows(l.expand(n, V).contiguous(), u, top_p=0.9)
    x = l[0].double().cpu().numpy()
    p = np.exp(x - x.max()); order = np.argsort(-p); c = np.cumsum(p[order]) / p.sum()
    keep = order[:np.searchsorted(c, np.float32(0.9)) + 1]
    q = np.zeros(V); q[keep] = p[keep] / p[keep].sum()
    assert (np.abs(np.bincount(tok.cpu().numpy(), minlength=V) - n * q) <= 1.0 + 1e-6).all()


def test_sample_rows_does_not_depend_on_the_batch(S):
    """A row gives the same token and the same bits alone, in a batch, and at another place of it."""
    for V in (1806, 50000):
        l = torch.randn(64, V, generator=gen(V), device='cuda') * 3
        u = torch.rand(64, generator=gen(2), device='cuda')
        tok, lp = S.sample_rows(l, u, top_p=0.9, temperature=0.9)
        for b in (0, 17, 63):
            t1, l1 = S.sample_rows(l[b:b + 1], u[b:b + 1], top_p=0.9, temperature=0.9)
            assert t1[0] == tok[b] and l1[0] == lp[b]
        t2, l2 = S.sample_rows(l.flip(0).contiguous(), u.flip(0).contiguous(), top_p=0.9, temperature=0.9)
        assert torch.equal(t2.flip(0), tok) and torch.equal(l2.flip(0), lp)


# ---------------------------------------------------------------------------------------------------- one step of a decoder's head
def test_refused_tensors(S):
    """What the tensor-level calls refuse, with the references they took given back."""
    import sys
    dev = 'cuda'
    x, w = torch.randn(3, 100, device=dev), S.quantize_rows(torch.randn(50, 100, device=dev))
    a, bias, u = S.quantize_rows(x), torch.zeros(50, device=dev), torch.zeros(3, device=dev)
    q = torch.zeros(4, 128, dtype=torch.int8, device=dev)
    ones = torch.ones(4, device=dev)
    out = torch.empty(3, 50, device=dev)
    grad = torch.randn(3, 100, device=dev, requires_grad=True)
    calls = [lambda: S.quantize_rows(x.half()), lambda: S.quantize_rows(x[0]), lambda: S.quantize_rows(x.t()), lambda: S.quantize_rows(x[:, :0]),
             lambda: S.quantize_rows(x[:1].expand(3, 100)), lambda: S.quantize_rows(grad), lambda: S.quantize_rows(None),
             lambda: S.Int8Rows(q, ones, 129), lambda: S.Int8Rows(q, ones, 0), lambda: S.Int8Rows(q, ones[:3], 100), lambda: S.Int8Rows(q, ones.double(), 100),
             lambda: S.Int8Rows(q[:, 1:], ones, 64), lambda: S.Int8Rows(q[:, :100], ones, 100), lambda: S.Int8Rows(q.int(), ones, 100),
             lambda: S.matmul_i8(x, w), lambda: S.matmul_i8(a, x), lambda: S.matmul_i8(a, S.quantize_rows(x[:, :64])), lambda: S.matmul_i8(a, w, bias[:49]),
             lambda: S.matmul_i8(a, w, bias.bfloat16()), lambda: S.matmul_i8(a, w, bias.cpu()), lambda: S.matmul_i8(a, w, out_dtype=torch.float16),
             lambda: S.matmul_i8(a, w, out_dtype=None), lambda: S.matmul_i8(a, w, out=out[:2]), lambda: S.matmul_i8(a, w, out=out, out_dtype=torch.bfloat16),
             lambda: S.matmul_i8(a, w, out=out.t()), lambda: S.linear_i8(x[:, :99], w), lambda: S.linear_i8(grad, w), lambda: S.linear_i8(x, w, bias[None]),
             lambda: S.linear_i8(x, w, out=x), lambda: S.sample_rows(x.int(), u), lambda: S.sample_rows(x, u[:2]), lambda: S.sample_rows(x, u.double()),
             lambda: S.sample_rows(x, u.cpu()), lambda: S.sample_rows(x, u, temperature=u.double()), lambda: S.sample_rows(x, u, top_k=u),
             lambda: S.sample_rows(x, u, top_p=u[:2]), lambda: S.sample_rows(x, u, min_p=u[:, None])]
    held = [x, w.q, w.scale, a.q, a.scale, bias, u, q, ones, out]
    before = [sys.getrefcount(t) for t in held]
    for c in calls:
        for _ in range(3):
            with pytest.raises(ValueError):
                c()
    for bad in (dict(top_k='a'), dict(temperature=None), dict(min_p=[1])):
        with pytest.raises((TypeError, ValueError)):
            S.sample_rows(x, u, **bad)
    for _ in range(3):
        S.linear_i8(x, w, bias), S.matmul_i8(a, w, bias, out=out), S.sample_rows(x, u, top_k=10 ** 30, top_p=0.5), S.sample_rows(x, u, top_k=-10 ** 30)
    assert [sys.getrefcount(t) for t in held] == before
    with torch.no_grad():
        S.linear_i8(grad, w)
    assert S.matmul_i8(S.quantize_rows(x[:0]), w).shape == (0, 50) and S.linear_i8(x[:0], w, bias).shape == (0, 50)
    assert [t.shape for t in S.sample_rows(x[:0], u[:0])] == [(0,), (0,)]


def test_head_of_a_decoder_step_in_a_graph_and_on_two_streams(S):
    """quantise + product + draw as a decoding service runs them: eager, captured and replayed with new inputs, two streams at once."""
    M, V, K = 48, 1806, 800
    w = S.quantize_rows(torch.randn(V, K, generator=gen(1), device='cuda') * 0.2)
    bias = torch.randn(V, generator=gen(2), device='cuda')

    def head(h, u):
        return S.sample_rows(S.linear_i8(h, w, bias=bias), u, temperature=0.9, top_k=100, top_p=0.95)
    ins = [(torch.randn(M, K, generator=gen(10 + i), device='cuda').bfloat16(), torch.rand(M, generator=gen(20 + i), device='cuda')) for i in range(4)]
    eager = [[t.clone() for t in head(*x)] for x in ins]
    for (h, u), (tok, lp) in zip(ins, eager):
        y = S.linear_i8(h, w, bias=bias).double().cpu().numpy()
        want = [sample_oracle(y[b], float(u[b]), float(np.float32(0.9)), 100, float(np.float32(0.95)), 0.0) for b in range(M)]
        np.testing.assert_array_equal(tok.cpu().numpy(), [x[0] for x in want])
    h, u = ins[0][0].clone(), ins[0][1].clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        tok, lp = head(h, u)
    for i in (0, 1, 2, 3, 1, 0):
        h.copy_(ins[i][0]); u.copy_(ins[i][1])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(tok, eager[i][0]) and torch.equal(lp, eager[i][1])
        head(*ins[(i + 1) % 4])
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(5):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((j, head(*ins[j])))
    torch.cuda.synchronize()
    for j, (t, l) in got:
        assert torch.equal(t, eager[j][0]) and torch.equal(l, eager[j][1])


def test_sample_step_bookkeeping():
    """e2t_sample_step: e2t_sample_rows' draw with e2t_greedy_step's bookkeeping; finished rows emit padding and keep their score."""
    import ctypes as C
    from ecog2txt_amd import hip_lib as H, serving as S
    B, V, L, eos, pad = 9, 1806, 4, 1, 0
    l = torch.randn(B, V, generator=gen(1), device='cuda')
    l[2] = float('-inf')
    l[3] = float('-inf'); l[3, eos] = 0.0
    u = torch.rand(B, generator=gen(2), device='cuda')
    tok, lp = S.sample_rows(l, u, top_k=20)
    done = torch.zeros(B, dtype=torch.int32, device='cuda'); done[4] = 1
    out = torch.full((B, L), -5, dtype=torch.int32, device='cuda')
    nxt = torch.full((B,), -5, dtype=torch.int32, device='cuda')
    score = torch.full((B,), 0.5, device='cuda')
    cfg = S.sample_config(B, l.get_device(), top_k=20)
    n = H.lib.e2t_sample_ws_bytes(B, V)
    ws = torch.empty(max(n, 16), dtype=torch.uint8, device='cuda')
    H.lib.e2t_sample_step(l.data_ptr(), H.DT_F32, V, B, V, u.data_ptr(), C.byref(cfg), 2, L, eos, pad, done.data_ptr(), out.data_ptr(), nxt.data_ptr(),
                          score.data_ptr(), ws.data_ptr(), n, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    t = tok.tolist(); t[2] = eos
    assert nxt.tolist() == t
    want = list(t); want[4] = pad
    assert out[:, 2].tolist() == want and (out[:, [0, 1, 3]] == -5).all()
    assert done.tolist() == [int(t[b] == eos or b == 4) for b in range(B)]
    ws_ = (score - 0.5).cpu().numpy()
    assert ws_[4] == 0 and ws_[2] == -np.inf
    ok = [b for b in range(B) if b not in (2, 4)]
    np.testing.assert_allclose(ws_[ok], lp.cpu().numpy()[ok], rtol=0, atol=2.0 ** -21)   # (0.5 + lp: sums below 16 round by at most 2^-21)
