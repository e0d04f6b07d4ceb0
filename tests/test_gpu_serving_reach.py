"""The serving operators where the choice of kernel changes: every instance of the int8 product, batches of long rows at every split, rows of the
largest vocabulary, zones around a cut that no list holds, and the 8-bit projection of a decoder at the sizes it is used at."""
import numpy as np
import pytest
import torch

from test_gpu_parity import SPECS, build
from test_gpu_serving import check_sample, gen, ints, product_bound, quant_oracle, rows_of

gpu = pytest.mark.gpu

# sizes by the instance they run on: odd rows and columns, few and many k-blocks, an odd number of them, one more than a multiple
INSTANCES = {
    0: [(1, 16, 1), (16, 1806, 800), (3, 357, 399), (78, 18, 3), (348, 220, 16)],
    1: [(3, 144, 1374), (45, 18, 2110), (2, 252, 7359), (24, 584, 7311), (186, 91, 2682)],
    2: [(427, 3613, 68), (76, 3530, 715), (63, 1017, 3874), (355, 345, 3186), (104, 644, 11446)],
    3: [(256, 1806, 800), (17, 4533, 797), (29, 2889, 1801), (180, 3425, 386), (25, 5632, 3079), (415, 420, 1127)],
    4: [(50, 3345, 1830), (502, 295, 3288), (91, 4494, 1456), (28, 5185, 7241), (54, 1398, 16076)],
    5: [(34, 5455, 4756), (289, 1115, 4680), (271, 944, 6878), (101, 3455, 8188), (130, 1461, 17211)],
    6: [(537, 19, 1), (578, 331, 6), (573, 251, 118), (357, 2209, 630), (763, 2651, 2939)],
    7: [(539, 18, 764), (1361, 23, 2373), (1033, 303, 2336), (126, 4716, 781), (666, 181, 9235)],
    8: [(8704, 3200, 801), (1624, 4899, 144), (1394, 5413, 232), (864, 5828, 425), (1360, 3038, 1340), (1848, 2363, 552)],
    9: [(1624, 2065, 708), (1942, 1765, 910), (600, 4008, 1726), (873, 2486, 1680), (1631, 1426, 2491)],
    10: [(4099, 4101, 4104), (4400, 4300, 1500), (4000, 4096, 1500), (8704, 2300, 1500), (1030, 9001, 5000)],
}
ALL = [(i, *s) for i, shapes in INSTANCES.items() for s in shapes]


def test_every_instance_has_its_sizes():
    from ecog2txt_amd import hip_lib
    f = hip_lib.lib.e2t_gemm_i8_instance
    assert [f(M, N, K) for _, M, N, K in ALL] == [i for i, *_ in ALL]
    assert set(INSTANCES) == set(range(11))
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1, 131072), (-1, 4, 4)):
        assert f(*bad) == -1


@pytest.fixture(scope='module')
def S():
    from ecog2txt_amd import serving
    return serving


# ---------------------------------------------------------------------------------------------------- product
@gpu
@pytest.mark.parametrize('i,M,N,K', ALL)
def test_product_of_every_instance(S, i, M, N, K):
    """Sums with scales of one are exact; with scales, bias and ReLU within the roundings; in a view, nothing beside it is written."""
    a, b = ints(M, K, M + K), ints(N, K, 3 * N + K)
    acc = a.double() @ b.double().t()                                  # (whole numbers below 2^53: exact)
    A, W = rows_of(S, a), rows_of(S, b)
    assert torch.equal(S.matmul_i8(A, W), acc.float())
    sa = torch.rand(M, generator=gen(3), device='cuda') * 0.02 + 1e-4
    sb = torch.rand(N, generator=gen(4), device='cuda') * 0.02 + 1e-4
    bias = torch.randn(N, generator=gen(5), device='cuda')
    A, W = S.Int8Rows(A.q, sa, K), S.Int8Rows(W.q, sb, K)
    e = 2.0 ** -24
    scaled = acc * sa.double()[:, None] * sb.double()[None]
    want = scaled + bias.double()[None]
    for out in (torch.float32, torch.bfloat16):
        tol = 4 * e * scaled.abs() + 2 * e * want.abs()                # (product_bound, on the device)
        tol = tol + (want.abs() + tol) * torch.finfo(out).eps / 2 + 1e-44
        assert ((S.matmul_i8(A, W, bias=bias, out_dtype=out).double() - want).abs() <= tol).all()
        for off, more in ((0, 0), (1, 0), (3, 2), (8, 8)):
            big = torch.full((M + 2, N + 8 + more), -7.0, dtype=out, device='cuda')
            y = S.matmul_i8(A, W, bias=bias, out_dtype=out, relu=True, out=big[1:-1, off:off + N])
            assert ((y.double() - want.clamp(min=0)).abs() <= tol).all()
            y.fill_(-7.0)
            assert (big == -7.0).all()


# ---------------------------------------------------------------------------------------------------- sampling
def mixed(B, seed):
    """Settings a row, every combination of cuts among them."""
    r = torch.rand(4, B, generator=gen(seed), device='cuda')
    i = torch.arange(B, device='cuda')
    zero = torch.zeros((), device='cuda')
    return dict(temperature=torch.where(i % 11 == 3, zero, 0.5 + r[0]), top_k=torch.where(i % 2 == 0, (1 + r[1] * 4000).int(), zero.int()),
                top_p=torch.where(i % 3 != 0, 0.3 + 0.7 * r[2], zero + 1), min_p=torch.where(i % 5 == 0, 0.1 * r[3], zero))


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('B,V', [(129, 50000), (256, 50003), (600, 20011), (129, 128003), (65, 262144)])
def test_sample_long_rows_in_large_batches(S, B, V, dtype):
    """Fewer, longer chunks a row: the counting window of a chunk moves up again and again where the logits rise along the row."""
    g = gen(B + V)
    l = 2.0 * torch.randn(B, V, generator=g, device='cuda')
    i = torch.arange(B, device='cuda')
    rise = torch.linspace(0, 30, V, device='cuda')
    l[i % 4 == 1] += rise
    l[i % 4 == 2] -= rise
    l[i % 8 == 3, V // 3:] = float('-inf')
    check_sample(S, l.to(dtype), torch.rand(B, generator=g, device='cuda'), **mixed(B, V))


@gpu
@pytest.mark.parametrize('V', [786432, 1 << 20])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_sample_largest_vocabularies(S, V, dtype):
    B = 3
    g = gen(V)
    l = (2.0 * torch.randn(B, V, generator=g, device='cuda')).to(dtype)
    l[1, ::3] = float('-inf')
    for kw in (dict(), dict(top_k=50), dict(top_k=200000), dict(top_p=0.9, temperature=1.4), dict(top_p=0.95), dict(top_k=100000, top_p=0.5, min_p=1e-3)):
        check_sample(S, l, torch.rand(B, generator=g, device='cuda'), **kw)


@gpu
@pytest.mark.parametrize('V', [16378, 131072])
def test_sample_zones_wider_than_the_list(S, V):
    """Top-k far behind top-p: the tokens between the two cuts are more than the list holds."""
    B = 4
    g = gen(V)
    l = 2.0 * torch.randn(B, V, generator=g, device='cuda')
    for kw in (dict(top_k=V // 6, top_p=0.5), dict(top_k=V // 2, top_p=0.3), dict(top_k=V - 1, top_p=0.2), dict(top_k=V * 3 // 4, top_p=0.99, min_p=1e-4), dict(top_k=V // 2)):
        check_sample(S, l, torch.rand(B, generator=g, device='cuda'), **kw)
        check_sample(S, l * 0.02, torch.rand(B, generator=g, device='cuda'), **kw)


@gpu
@pytest.mark.parametrize('V', [20011, 50000, 300000])
def test_sample_long_rows_do_not_depend_on_the_split(S, V):
    """1, 70 and 256 rows are cut into different numbers of chunks.  Without top-p the same bits; with it the sum that p is a share of may
    differ by 1e-11, which moves a token only where a border lies that close."""
    n = 256
    l = torch.randn(n, V, generator=gen(V), device='cuda') * 3
    u = torch.rand(n, generator=gen(2), device='cuda')
    for kw in (dict(temperature=0.9), dict(top_k=300), dict(top_k=9000, min_p=1e-3), dict(min_p=0.01), dict(top_p=0.9), dict(top_k=5000, top_p=0.8)):
        tok, lp = S.sample_rows(l, u, **kw)
        for rows in ([0], [17], [255], range(70), range(100, 230)):
            rows = torch.tensor(list(rows), device='cuda')
            t, p = S.sample_rows(l[rows], u[rows], **kw)
            assert torch.equal(t, tok[rows]) and torch.equal(p, lp[rows])


# ---------------------------------------------------------------------------------------------------- the projection in 8 bits
WIDE = dict(SPECS['cfg2_widths'], vocab=1806)


def check_projection(eng, h, out, qw, sw, bias):
    """The logits `out` of the state rows h are the product of the quantised operands with the bias added in fp32."""
    q, s = quant_oracle(h.double().cpu().numpy())
    acc = (torch.from_numpy(q.astype(np.float64)) @ torch.from_numpy(qw.astype(np.float64)).t()).numpy()     # (exact: sums below 2^53)
    b = bias.double().cpu().numpy().reshape(-1)
    want = acc * s.astype(np.float64)[:, None] * sw.astype(np.float64)[None] + b[None]
    assert (np.abs(out.double().cpu().numpy() - want) <= product_bound(acc, s.astype(np.float64), sw.astype(np.float64), bias, want, torch.float32)).all()


def projection_operands(eng):
    pr = eng.proj
    fin = pr.sizes[-2]
    return (fin, *quant_oracle(pr.WT[-1][:, :fin].double().cpu().numpy()), eng.store.view('proj%d.b' % (pr.nl - 1)))


@gpu
@pytest.mark.parametrize('B', [1, 24, 256, 700])
def test_projection_of_a_decode_batch(B):
    eng, ws, *_ = build(WIDE, B, 26, 3, seed=5)
    L, V = ws['L'], eng.spec.vocab
    u = torch.rand(L, B, generator=gen(1), device='cuda')
    eng.sample_decode(ws, u, which='p', int8_projection=True)
    fin, qw, sw, bias = projection_operands(eng)
    for l in range(L):
        h = ws['dec']['Yext'].view(-1, eng.dec.ldy)[(l + 1) * B:(l + 2) * B, :fin]
        check_projection(eng, h, ws['proj']['out'].view(L, B, V)[l], qw, sw, bias)


@gpu
@pytest.mark.parametrize('name,B,W', [('tiny_odd', 19, 4), ('cat_aux_hidden_proj', 7, 3), ('wide', 6, 4), ('wide', 64, 16)])
def test_beams_with_the_projection_in_8_bits(name, B, W, monkeypatch):
    """Every step's logits are the quantised product, and the surviving hypotheses the W best continuations by these logits."""
    eng, ws, *_ = build(dict(SPECS, wide=WIDE)[name], B, 26, 4, seed=7)
    L, V, pr = ws['L'], eng.spec.vocab, eng.proj
    steps, inner = [], eng._proj_rows

    def proj_rows(wb, src, l, q8=None):
        if steps:
            steps[-1].update(rowmap=wb['beam']['rowmap'].clone(), tok=wb['U'].view(L, -1)[l].clone())
        inner(wb, src, l, q8)
        n = wb['B']
        h = wb['dec']['Yext'].view(-1, eng.dec.ldy)[(l + 1) * n:(l + 2) * n] if pr.nl == 1 else wb['proj']['act'][-1][l * n:(l + 1) * n]
        steps.append(dict(h=h.clone(), out=wb['proj']['out'].view(L, n, V)[l].clone(), wb=wb))
    monkeypatch.setattr(eng, '_proj_rows', proj_rows)
    hyp, score = eng.beam_decode(ws, W, which='p', int8_projection=True)
    assert len(steps) == L
    fin, qw, sw, bias = projection_operands(eng)
    steps[-1].update(rowmap=steps[-1]['wb']['beam']['rowmap'].clone())
    have = torch.full((B, W), -float('inf'), dtype=torch.float64)
    have[:, 0] = 0
    done = torch.zeros(B, W, dtype=torch.bool)
    # (a log-probability in fp32: a sum of V terms, its logarithm, a difference, and the running score, all of magnitude below 64 here)
    tol = (V + 64 * 8) * 2.0 ** -24
    for l, s in enumerate(steps):
        check_projection(eng, s['h'][:, :fin], s['out'], qw, sw, bias)
        logp = torch.log_softmax(s['out'].double().cpu(), -1).view(B, W, V)
        cand = torch.where(done[:, :, None], -float('inf'), have[:, :, None] + logp).reshape(B, W * V)
        best = torch.cat([cand, torch.where(done, have, -float('inf'))], 1).topk(W, 1).values
        parent = s['rowmap'].cpu().long().view(B, W) - W * torch.arange(B)[:, None]
        assert ((parent >= 0) & (parent < W)).all()
        was = done.gather(1, parent)
        if l + 1 < L:
            tok = s['tok'].cpu().long().view(B, W)
            cont = cand.view(B, W, V)[torch.arange(B)[:, None], parent, tok]
            have = torch.where(was, have.gather(1, parent), cont)
            done = was | (tok == 1)
            fin_ = torch.isfinite(best)
            assert ((have - best).abs()[fin_] <= (l + 1) * tol).all()
        else:
            fin_ = torch.isfinite(best)
            assert ((score.double().cpu() - best).abs()[fin_] <= L * tol).all()
