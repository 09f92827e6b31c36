"""Host-side argument checks of the recurrent block's C entry points (no GPU, nothing launched)
and of the Python functions on CPU tensors."""
import pytest
import torch

from theorem_b200 import _lib, ops

FAKE = 1 << 20  # never dereferenced: every case returns before touching memory


def test_gated_scan_rejects_arguments_without_gpu():
    lib = _lib.load()
    f, g = lib.thm_gated_scan_fwd, lib.thm_gated_scan_bwd
    q6, q8 = [8] * 6, [8] * 8
    p9, p14 = [FAKE] * 9, [FAKE] * 14
    no_cu = [FAKE] * 5 + [None] + [FAKE] * 3
    no_cu14 = [FAKE] * 7 + [None] + [FAKE] * 6
    # B, T, D, nseq, zero_rest, dtype
    assert f(*no_cu, *q6, 1, 8, 8, 1, 0, 9, None) == _lib.THM_ERR_INVALID    # unknown dtype
    assert f(*no_cu, *q6, -1, 8, 8, -1, 0, 0, None) == _lib.THM_ERR_INVALID  # negative size
    assert f(*no_cu, *q6, 2, 8, 8, 3, 0, 0, None) == _lib.THM_ERR_INVALID    # nseq != B without cu_seqlens
    assert f(*p9, *q6, 2, 8, 8, 2, 0, 0, None) == _lib.THM_ERR_INVALID       # packed with B = 2
    assert f(*no_cu, *q6, 1 << 27, 1, 8, 1 << 27, 0, 0, None) == _lib.THM_ERR_UNSUPPORTED
    assert f(*no_cu, *q6, 1, (1 << 30) + 1, 8, 1, 0, 0, None) == _lib.THM_ERR_UNSUPPORTED
    assert f(*([None] * 9), *q6, 1, 8, 8, 1, 0, 0, None) == _lib.THM_ERR_INVALID  # null pointers
    assert f(*([None] * 9), *q6, 1, 8, 0, 1, 0, 0, None) == _lib.THM_OK      # no channels
    assert f(*([None] * 9), *q6, 0, 8, 8, 0, 0, 0, None) == _lib.THM_OK      # no sequences
    assert g(*no_cu14, *q8, 2, 8, 8, 3, 0, 0, None) == _lib.THM_ERR_INVALID
    assert g(*p14, *q8, 2, 8, 8, 2, 0, 0, None) == _lib.THM_ERR_INVALID
    assert g(*([None] * 14), *q8, 1, 8, 8, 1, 0, 0, None) == _lib.THM_ERR_INVALID
    assert g(*([None] * 14), *q8, 1, 8, 0, 1, 0, 0, None) == _lib.THM_OK
    no_ws = [FAKE] * 7 + [None] + [FAKE] * 5 + [None]
    assert g(*no_ws, *q8, 1, 8, 8, 1, 0, 0, None) == _lib.THM_ERR_INVALID    # no workspace


def test_group_norm_rejects_arguments_without_gpu():
    lib = _lib.load()
    f, g = lib.thm_group_norm_fwd, lib.thm_group_norm_bwd
    p5, p10 = [FAKE] * 5, [FAKE] * 10
    # row strides..., R, C, G, center, activation, eps, dtype
    assert f(*p5, 8, 8, 1, 8, 3, 1, 0, 1e-5, 0, None) == _lib.THM_ERR_INVALID        # 8 % 3
    assert f(*p5, 8, 8, 1, 8, 0, 1, 0, 1e-5, 0, None) == _lib.THM_ERR_INVALID        # empty group
    assert f(*p5, 8, 8, 1, 8, 4, 1, 5, 1e-5, 0, None) == _lib.THM_ERR_INVALID        # unknown activation
    assert f(*p5, 8, 8, 1, 8, 4, 1, 0, 1e-5, 4, None) == _lib.THM_ERR_INVALID        # unknown dtype
    assert f(*p5, 8192, 8192, 1, 8192, 8192, 1, 0, 1e-5, 0, None) == _lib.THM_ERR_UNSUPPORTED
    assert f(*([None] * 5), 8, 8, 1, 8, 4, 1, 0, 1e-5, 0, None) == _lib.THM_ERR_INVALID
    assert f(*([None] * 5), 8, 8, 0, 8, 4, 1, 0, 1e-5, 0, None) == _lib.THM_OK       # no rows
    assert g(*p10, 8, 8, 8, 1, 8, 3, 1, 0, 1e-5, 0, None) == _lib.THM_ERR_INVALID
    assert g(*p10[:9], None, 8, 8, 8, 1, 8, 4, 1, 0, 1e-5, 0, None) == _lib.THM_ERR_INVALID  # no workspace
    no_dgate = [FAKE] * 6 + [None] + [FAKE] * 3
    assert g(*no_dgate, 8, 8, 8, 1, 8, 4, 1, 0, 1e-5, 0, None) == _lib.THM_ERR_INVALID       # gate without dgate


def test_conv_step_and_bwd_reject_arguments_without_gpu():
    lib = _lib.load()
    f, g = lib.thm_causal_conv1d_step, lib.thm_causal_conv1d_bwd
    p6, p8 = [FAKE] * 6, [FAKE] * 8
    # strides, B, S, D, W, dtype, activation
    assert f(*p6, 8, 8, 1, 1, 8, 0, 0, 0, None) == _lib.THM_ERR_INVALID      # W = 0
    assert f(*p6, 8, 8, 1, 1, 8, 9, 0, 0, None) == _lib.THM_ERR_UNSUPPORTED  # W > 8
    assert f(*p6, 8, 8, 1, 1, 8, 4, 7, 0, None) == _lib.THM_ERR_INVALID      # unknown dtype
    assert f(*p6, 8, 8, 1, 1, 8, 4, 0, 7, None) == _lib.THM_ERR_INVALID      # unknown activation
    assert f(*([None] * 6), 8, 8, 1, 1, 8, 4, 0, 0, None) == _lib.THM_ERR_INVALID
    assert f(*([None] * 6), 8, 8, 0, 1, 8, 4, 0, 0, None) == _lib.THM_OK
    assert g(*p8, 8, 8, 8, 8, 1, 1, 8, 9, 0, 0, None) == _lib.THM_ERR_UNSUPPORTED
    assert g(*p8, 8, 8, 8, 8, 1, -1, 8, 4, 0, 0, None) == _lib.THM_ERR_INVALID
    assert g(*p8, 8, 8, 8, 8, 1, (1 << 30) + 1, 8, 4, 0, 0, None) == _lib.THM_ERR_UNSUPPORTED
    assert g(*p8, 8, 8, 8, 8, 65536, 1, 8, 4, 0, 0, None) == _lib.THM_ERR_UNSUPPORTED
    assert g(*([None] * 8), 8, 8, 8, 8, 1, 1, 8, 4, 0, 0, None) == _lib.THM_ERR_INVALID
    assert lib.thm_causal_conv1d_bwd_parts(0, 8, 8) == 0
    assert lib.thm_causal_conv1d_bwd_parts(2, 1, 8) == 2


@pytest.mark.parametrize("call", [
    lambda t, w: ops.gated_scan(t, t, t, w[0]),
    lambda t, w: ops.gated_scan_bwd(t, t, t, w[0], w, t),
    lambda t, w: ops.group_norm(t, 4),
    lambda t, w: ops.group_norm_bwd(t, t, 4),
    lambda t, w: ops.causal_conv1d_step(t, t, w, w[0]),
    lambda t, w: ops.causal_conv1d_bwd(t, w, w[0], t),
])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(AssertionError, match="CUDA"):
        call(torch.zeros(1, 2, 8), torch.zeros(8, 8))
