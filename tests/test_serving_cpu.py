"""What the serving operators refuse (no GPU needed: every check is made before anything is launched)."""
import ctypes as C

import pytest
import torch


@pytest.fixture(scope='module')
def H():
    from ecog2txt_amd import hip_lib
    hip_lib.load()
    return hip_lib


def refused(fn, *a):
    with pytest.raises(RuntimeError, match='bad argument'):
        fn(*a)


def test_struct_layout(H):
    assert H.lib.e2t_sizeof(7) == C.sizeof(H.SampleCfg)


def test_quant_refusals(H):
    f = H.lib.e2t_quant_rows_i8
    x, q, s = 0x10000, 0x20000, 0x30000
    good = [x, 0, 100, 3, 100, q, 128, s, None]
    for i, v in ((0, None), (0, x + 2), (1, 2), (2, 99), (3, 0), (3, -1), (3, (1 << 30) + 1), (4, 0), (5, None), (5, q + 8), (6, 127), (6, 120), (6, 112), (7, None)):
        a = list(good); a[i] = v
        refused(f, *a)


def test_gemm_refusals(H):
    f = H.lib.e2t_gemm_nt_i8
    good = [0x10000, 128, 0x20000, 0x30000, 128, 0x40000, None, 0x50000, 50, 7, 50, 100, 0, None]
    for i, v in ((0, None), (0, 0x10008), (1, 112), (1, 130), (2, None), (3, None), (3, 0x30004), (4, 64), (4, 136), (5, None), (7, None), (7, 0x50002),
                 (8, 49), (9, 0), (9, (1 << 30) + 1), (10, 0), (10, -4), (11, 0), (11, 131072), (12, 4), (12, 8), (12, 16), (12, 64)):
        a = list(good); a[i] = v
        refused(f, *a)


def test_linear_refusals(H):
    f, n = H.lib.e2t_linear_i8, H.lib.e2t_linear_i8_ws_bytes(200, 50, 100)
    assert n >= 200 * 128 + 800 and H.lib.e2t_linear_i8_ws_bytes(0, 7, 5) == 0
    good = [0x10000, 1, 100, 0x30000, 128, 0x40000, None, 0x50000, 50, 200, 50, 100, 0, 0x60000, n, None]
    for i, v in ((0, None), (0, 0x10001), (1, 5), (2, 99), (3, None), (3, 0x30008), (4, 120), (5, None), (7, None), (8, 49), (9, 0), (10, 0), (11, 0), (11, 131072),
                 (12, 32), (13, None), (13, 0x60004), (14, n - 1)):
        a = list(good); a[i] = v
        refused(f, *a)


def test_sample_refusals(H):
    cfg = H.SampleCfg(1.0, 1.0, 0.0, 0)
    B, V = 3, 40000
    n = H.lib.e2t_sample_ws_bytes(B, V)
    good = [0x10000, 0, V, B, V, 0x20000, C.byref(cfg), 0x30000, 0x40000, 0x50000, n, None]
    bad = [(0, None), (0, 0x10002), (1, 2), (1, -1), (2, V - 1), (3, 0), (4, 0), (4, 1048577), (5, None), (6, None), (7, None)]
    if n:
        bad += [(9, None), (9, 0x50004), (10, n - 1)]
    for i, v in bad:
        a = list(good); a[i] = v
        refused(H.lib.e2t_sample_rows, *a)
    good = [0x10000, 0, V, B, V, 0x20000, C.byref(cfg), 1, 4, 1, 0, 0x30000, 0x40000, None, None, 0x50000, n, None]
    for i, v in ((0, None), (5, None), (6, None), (7, 4), (7, -1), (11, None), (12, None)):
        a = list(good); a[i] = v
        refused(H.lib.e2t_sample_step, *a)


def test_tensor_level_refusals(H):
    from ecog2txt_amd import serving as S
    x = torch.zeros(3, 64)
    with pytest.raises(ValueError, match='device tensor'):
        S.quantize_rows(x)
    with pytest.raises(ValueError, match='device tensor'):
        S.sample_rows(x, torch.zeros(3))
    with pytest.raises(ValueError, match='device tensor'):
        S.linear_i8(x, None)
    with pytest.raises(ValueError, match='Int8Rows'):
        S.matmul_i8(x, None)
    with pytest.raises(ValueError, match='device tensor'):
        S.Int8Rows(torch.zeros(3, 64, dtype=torch.int8), torch.zeros(3), 50)
