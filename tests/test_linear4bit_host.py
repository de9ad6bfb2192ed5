"""Host side of the 4-bit linear layer (no GPU): size queries and refusals."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
from next_step_ai_b200 import _lib, linear4bit  # noqa: E402


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        from next_step_ai_b200.build import build

        build()
    return _lib.load()


@pytest.mark.parametrize("N,K,gs", [(1, 2, 32), (16, 128, 64), (17, 130, 64), (1001, 2086, 128), (257, 1026, 96),
                                    (512, 4096, 4096)])
def test_packed_sizes(lib, N, K, gs):
    tiles = -(-N // 128) * -(-K // 128)                    # 128 x 128 weights, 8 KB each
    assert lib.nsm_linear4bit_packed_bytes(N, K) == 8192 * tiles
    per_tile = 1 if gs % 128 == 0 else 2 if gs % 64 == 0 else 4
    steps = -(-K // 128)
    entries = -(-steps // (gs // 128)) if per_tile == 1 else steps
    assert lib.nsm_linear4bit_scale_count(N, K, gs) == -(-N // 128) * 128 * entries * per_tile


def test_sizes_that_are_refused(lib):
    for n, k in ((0, 128), (16, 0), (16, 127), (-1, 128), ((1 << 24) + 1, 128), (16, (1 << 20) + 2)):
        assert lib.nsm_linear4bit_packed_bytes(n, k) == 0
        assert lib.nsm_linear4bit_scale_count(n, k, 64) == 0
    for gs in (0, 16, 48, -32):
        assert lib.nsm_linear4bit_scale_count(16, 128, gs) == 0
    assert lib.nsm_linear4bit_max_rows(_lib.NSM_BF16) == 32 and lib.nsm_linear4bit_max_rows(_lib.NSM_F32) == 16


def test_bad_arguments_are_errors_before_any_device_call(lib):
    one = 256                                              # an address that is never read
    assert lib.nsm_linear4bit_pack(None, 64, one, 0, None, 16, 128, 64, 0, one, one, None, None) == _lib.NSM_ERR_INVALID_ARG
    assert lib.nsm_linear4bit_pack(one, 63, one, 0, None, 16, 128, 64, 0, one, one, None, None) == _lib.NSM_ERR_INVALID_ARG
    assert lib.nsm_linear4bit_pack(one, 64, one, 0, one, 16, 128, 64, 1, one, one, one, None) == _lib.NSM_ERR_INVALID_ARG
    assert lib.nsm_linear4bit_pack(one, 64, one, 7, None, 16, 128, 64, 0, one, one, None, None) == _lib.NSM_ERR_INVALID_ARG
    assert lib.nsm_linear4bit_pack(one, 64, one, 0, None, 16, 128, 64, 0, one + 8, one, None, None) == _lib.NSM_ERR_INVALID_ARG
    assert lib.nsm_linear4bit_pack(one, 64, one, 0, None, 16, 128, 40, 0, one, one, None, None) == _lib.NSM_ERR_UNSUPPORTED
    import ctypes

    w = _lib.Linear4bitWeightsC(one, one, None, None, None, 0, 16, 128, 64)
    ref = ctypes.byref(w)
    call = lib.nsm_linear4bit
    assert call(one, 0, 1, 128, None, one, 0, 16, one, 1 << 20, None) == _lib.NSM_ERR_INVALID_ARG
    assert call(one, 5, 1, 128, ref, one, 0, 16, one, 1 << 20, None) == _lib.NSM_ERR_INVALID_ARG
    assert call(None, 0, 1, 128, ref, one, 0, 16, one, 1 << 20, None) == _lib.NSM_ERR_INVALID_ARG
    assert call(one, 0, 17, 128, ref, one, 0, 16, one, 1 << 20, None) == _lib.NSM_ERR_UNSUPPORTED
    assert call(one + 2, 0, 1, 128, ref, one, 0, 16, one, 1 << 20, None) == _lib.NSM_ERR_INVALID_ARG
    w.group_size = 33
    assert call(one, 0, 1, 128, ref, one, 0, 16, one, 1 << 20, None) == _lib.NSM_ERR_UNSUPPORTED


def test_host_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        linear4bit.Linear4bit(torch.zeros((16, 64), dtype=torch.uint8), torch.zeros((16, 2)), out_features=16,
                              in_features=128)
    with pytest.raises(RuntimeError, match="rank-2"):
        linear4bit.Linear4bit.from_dense(torch.zeros(16))
    with pytest.raises(RuntimeError, match="must divide"):
        linear4bit.Linear4bit.from_dense(torch.zeros((4, 100)), device="cpu")


def test_quant_blocks_across_rows_are_refused():
    from next_step_ai_b200.checkpoint import Nf4Param

    p = Nf4Param("w", torch.zeros(96, dtype=torch.uint8), torch.zeros(3), torch.zeros(16), 2, 96, 64, "nf4", "float16")
    with pytest.raises(RuntimeError, match="do not divide"):
        linear4bit.Linear4bit.from_param(p, "cpu")


def test_wait_limit_is_validated(lib):
    assert lib.nsm_linear4bit_set_wait_limit(-2) == _lib.NSM_ERR_INVALID_ARG
    assert lib.nsm_linear4bit_set_wait_limit(1000) == _lib.NSM_OK
    assert lib.nsm_linear4bit_set_wait_limit(0) == _lib.NSM_OK


def test_error_word_needs_somewhere_to_go(lib):
    assert lib.nsm_linear4bit_error(None, None) == _lib.NSM_ERR_INVALID_ARG
