"""What the tensor-level serving calls refuse whatever device a tensor lies on (no GPU needed)."""
import pytest
import torch


def test_gradients():
    import torch.autograd.forward_ad as fw
    from ecog2txt_amd import serving as S
    x = torch.zeros(3, 64)
    with pytest.raises(ValueError, match='gradient'):
        S.quantize_rows(x.clone().requires_grad_())
    with pytest.raises(ValueError, match='gradient'):
        S.sample_config(3, -1, top_p=torch.ones(3).requires_grad_())
    with fw.dual_level(), pytest.raises(ValueError, match='tangent'):
        S.linear_i8(fw.make_dual(x, x + 1), None)
    with torch.no_grad(), pytest.raises(ValueError, match='device tensor'):
        S.quantize_rows(x.clone().requires_grad_())


def test_negated_views():
    from ecog2txt_amd import serving as S
    x = torch.zeros(3, 1, dtype=torch.complex64).conj().imag
    assert x.is_neg()
    with pytest.raises(ValueError, match='resolve_neg'):
        S.quantize_rows(x)


def test_workspace_of_a_batch_in_pieces():
    from ecog2txt_amd.hip_lib import lib
    n = lib.e2t_sample_ws_bytes(65535, 20000)
    assert n and lib.e2t_sample_ws_bytes(65536, 20000) == n == lib.e2t_sample_ws_bytes(2 ** 31 - 1, 20000)
    assert lib.e2t_sample_ws_bytes(65534, 20000) < n
    assert lib.e2t_sample_ws_bytes(2 ** 31 - 1, 16377) == 0 == lib.e2t_sample_ws_bytes(3, 1048577)
