"""CPU: the 8-bit operators refuse what they cannot take before anything touches a device."""
import pytest
import torch


def test_library_refuses_bad_shapes():
    import ctypes
    from pointcloudsegmentation_amd import _lib
    lib = _lib.lib()
    assert lib.p2n_int8_weight_bytes(0, 4) == -1 and lib.p2n_int8_weight_bytes(4, 65537) == -1
    # 2 k-tiles of 32 (rounded up to even) x 1 channel tile of 1 KiB, 32 scales, 32 biases
    assert lib.p2n_int8_weight_bytes(6, 7) == 2 * 1024 + 8 * 32
    assert lib.p2n_int8_pack_weight(None, None, 0, 4, None, None) == 1
    assert lib.p2n_int8_pack_weight(None, None, 4, 4, None, None) == 1
    assert lib.p2n_quantize_tokens(None, 0, 4, 8, 7, None, None, None) == 1          # rows that overlap
    assert lib.p2n_quantize_tokens(None, 0, 0, 8, 8, None, None, None) == 0
    assert lib.p2n_int8_linear(None, 0, 4, 8, 8, None, 4, 0, None, None, 0, None) == 1
    assert lib.p2n_int8_linear(None, 0, 0, 8, 8, None, 4, 0, None, None, 0, None) == 0
    assert lib.p2n_int8_linear(16, 0, 4, 8, 8, 16, 4, 0, 16, 16, 1, None) == 2       # workspace too small
    assert b"workspace" in lib.p2n_last_error()
    dims = (ctypes.c_int * 3)(6, 32, 300)
    images = (ctypes.c_void_p * 2)(16, 16)
    assert lib.p2n_int8_mlp(16, 1, 8, 2, dims, images, 1, 0, 16, None) == 1
    assert b"output channels" in lib.p2n_last_error()
    dims = (ctypes.c_int * 3)(6, 32, 64)
    assert lib.p2n_int8_mlp(16, 1, 40, 2, dims, images, 1, 32, 16, None) == 1        # 40 columns in groups of 32
    assert lib.p2n_int8_mlp(16, 1, 48, 2, dims, images, 1, 24, 16, None) == 1
    assert lib.p2n_int8_mlp(16, 1, (1 << 24) + 1, 2, dims, images, 1, 0, 16, None) == 1
    assert lib.p2n_int8_mlp(16, 1, 8, 9, dims, images, 1, 0, 16, None) == 1
    assert lib.p2n_int8_mlp(None, 0, 8, 2, dims, images, 1, 0, None, None) == 0
    assert lib.p2n_max_of_columns(None, 4, 0, None, None) == 1


def test_cpu_tensors_are_refused():
    from pointcloudsegmentation_amd import quant
    x = torch.randn(4, 8)
    with pytest.raises(ValueError):
        quant.quantize_tokens(x)
    with pytest.raises(ValueError):
        quant.Int8Weight(x)
    with pytest.raises(ValueError):
        quant.int8_mlp(x.view(1, 4, 8), [])
