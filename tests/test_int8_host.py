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
    assert lib.p2n_int8_pack_weight(None, None, 0, 4, None, None, None, None, 0.0, None, None) == 1
    assert lib.p2n_int8_pack_weight(None, None, 4, 4, None, None, None, None, 0.0, None, None) == 1
    assert lib.p2n_int8_pack_weight(16, None, 4, 4, 16, None, 16, 16, 1e-5, 16, None) == 1       # gamma without beta
    assert lib.p2n_quantize_tokens(None, 0, 4, 8, 7, None, None, None) == 1          # rows that overlap
    assert lib.p2n_quantize_tokens(None, 0, 0, 8, 8, None, None, None) == 0
    assert lib.p2n_int8_linear(None, 0, 4, 8, 8, None, 4, 0, None, None, 0, None) == 1
    assert lib.p2n_int8_linear(None, 0, 0, 8, 8, None, 4, 0, None, None, 0, None) == 0
    assert lib.p2n_int8_linear_workspace_bytes(4, 8, 4) == 0 and lib.p2n_int8_linear_workspace_bytes(100, 8, 4) == 4 * 2048 + 4 * 128
    assert lib.p2n_int8_linear(16, 0, 100, 8, 8, 16, 4, 0, 16, 16, 1, None) == 2     # workspace too small
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
    # more than a launch's 2^32 threads
    assert lib.p2n_int8_linear(16, 0, (1 << 30) + 1, 1, 1, 16, 1, 0, 16, 16, 1 << 62, None) == 1
    for B, wide in ((128, 32), (32, 100), (16, 200)):
        assert lib.p2n_int8_mlp(16, B, 1 << 24, 1, (ctypes.c_int * 2)(6, wide), images, 1, 0, 16, None) == 1
        assert b"too many columns" in lib.p2n_last_error()
    assert lib.p2n_max_of_columns(16, 1 << 32, 1, 16, None) == 1


def test_cpu_tensors_are_refused():
    from pointcloudsegmentation_amd import quant
    x = torch.randn(4, 8)
    with pytest.raises(ValueError):
        quant.quantize_tokens(x)
    with pytest.raises(ValueError):
        quant.Int8Weight(x)
    with pytest.raises(ValueError):
        quant.int8_mlp(x.view(1, 4, 8), [])


def test_checkpoint_layers_refuse_bad_shapes():
    from pointcloudsegmentation_amd import _lib
    lib = _lib.lib()
    # codes, scales, bits, mean and 1/deviation, each part rounded up to 256 bytes
    assert lib.p2n_act8_kept_bytes(2, 64, 300, 1) == 2 * 3 * 64 * 128 + 2 * 3 * 64 * 4 + 2 * 3 * 64 * 16 + 64 * 8
    assert lib.p2n_act8_kept_bytes(2, 6, 300, 0) == 2 * 3 * 6 * 128 + 256                # 6 scales as 8: 192 bytes
    for bad in ((0, 64, 300, 1), (2, 0, 300, 1), (2, 1025, 300, 1), (2, 64, 0, 1), (2, 64, (1 << 24) + 1, 1), (1 << 20, 1024, 3000, 1), (1 << 24, 1, 1, 0)):
        assert lib.p2n_act8_kept_bytes(*bad) == 0
        assert lib.p2n_act8_workspace_bytes(*bad[:3], 8) == 0
    a = 1 << 16     # an address that is never read: every call below is refused first

    def fwd(x=a, K=8, N=8, gamma=None, beta=None, rm=None, rv=None, mom=0.1, h=a, kept=a, nk=1 << 20, ws=a, nw=1 << 24, B=1, L=50):
        return lib.p2n_act8_forward(x, B, K, L, a, a, N, gamma, beta, rm, rv, None, mom, 1e-5, h, kept, nk, ws, nw, None)

    assert fwd(x=None) == 1 and fwd(h=None) == 1 and fwd(N=0) == 1 and fwd(N=1025) == 1 and fwd(K=2000) == 1
    assert fwd(gamma=a) == 1                                  # gamma without beta
    assert fwd(gamma=a, beta=a, rm=a) == 1                    # one running statistic
    assert fwd(gamma=a, beta=a, mom=-1.0) == 1                # frozen statistics that are not there
    assert fwd(gamma=a, beta=a, mom=1.5) == 1
    assert fwd(gamma=a, beta=a, L=1) == 1                     # batch statistics of one value
    assert fwd(kept=a + 16) == 1 and fwd(ws=a + 16) == 1      # alignment
    assert fwd(nk=100) == 2 and fwd(nw=100) == 2 and fwd(kept=None) == 2
    assert lib.p2n_act8_backward(a, 1, 8, 50, a, 8, a, a, 0, a, 1 << 20, None, a, a, a, None, a, 1 << 24, None) == 1   # dgamma without dx
    assert lib.p2n_act8_backward(None, 1, 8, 50, a, 8, None, None, 0, a, 1 << 20, a, a, a, None, None, a, 1 << 24, None) == 1
    assert lib.p2n_act8_norm_relu_forward(a, 1, 8, 50, None, None, None, None, None, 0.1, 1e-5, a, a, 1 << 20, a, 1 << 20, None) == 1
    assert lib.p2n_act8_norm_relu_backward(a, 1, 8, 50, a, 0, a, 10, a, None, None, a, 1 << 20, None) == 2
