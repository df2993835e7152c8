"""What the operators refuse, on the CPU: the Python checks and those of the C entries, which come before any use of the GPU."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def dp(built_library):
    import deepity_b200
    return deepity_b200


def test_only_cuda_tensors_of_two_types(dp):
    h, w, t = torch.zeros(2, 8), torch.zeros(5, 8), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(ValueError, match="no CPU path"):
        dp.vocab_cross_entropy(h, w, t)
    with pytest.raises(TypeError, match="float32 and bfloat16"):
        dp.vocab_cross_entropy(h.half(), w, t)
    with pytest.raises(TypeError, match="torch tensor"):
        dp.residual_norm([1.0])
    with pytest.raises(ValueError, match="no CPU path"):
        dp.residual_norm(h, h)
    with pytest.raises(ValueError, match="no CPU path"):
        dp.activate_and_pack(h, "gelu")
    with pytest.raises(ValueError, match="no CPU path"):
        dp.packed_activation_backward(h, None, "gelu")


def test_packed_containers_are_checked(dp):
    codes, scales = torch.zeros(3, 200, dtype=torch.int8), torch.zeros(3, 2)
    assert dp.PackedActivations(codes, scales).shape == (3, 200)
    for bad in ((codes.float(), scales), (codes, scales.double()), (codes, torch.zeros(3, 1)), (codes[:, ::2], scales),
                (codes[0], scales), (codes, torch.zeros(2, 3).T)):
        with pytest.raises(ValueError):
            dp.PackedActivations(*bad)


def vocab(**more):
    from deepity_b200 import _lib
    base = dict(rows=4, width=8, vocab=16, hidden_stride=8, weight_stride=8, type=1, scale=1.0, ignore_index=-100,
                d_hidden_stride=8, d_weight_stride=8)
    return _lib.VocabCe(**{**base, **more})


@pytest.mark.parametrize("more,status,said", [
    (dict(type=2), -1, b"type"), (dict(type=-1), -1, b"type"), (dict(rows=-1), -1, b"rows"), (dict(width=0), -1, b"width"),
    (dict(vocab=0), -1, b"vocab"), (dict(rows=1 << 29), -6, b"2^28"), (dict(vocab=1 << 29), -6, b"2^28"),
    (dict(hidden_stride=7), -1, b"stride"), (dict(weight_stride=7), -1, b"stride"),
    (dict(weight_stride=1 << 40), -1, b"stride"), (dict(scale=0.0), -1, b"scale"), (dict(scale=-1.0), -1, b"scale"),
    (dict(scale=float("nan")), -1, b"scale"), (dict(scale=float("inf")), -1, b"scale")])
def test_vocab_entries_refuse(built_library, more, status, said):
    from deepity_b200 import _lib
    lib, size = _lib.load(), ctypes.c_size_t()
    c = vocab(**more)
    for rc in (lib.dpc_vocab_ce_forward(None, ctypes.byref(c)), lib.dpc_vocab_ce_backward(None, ctypes.byref(c)),
               lib.dpc_vocab_ce_workspace(ctypes.byref(c), 0, ctypes.byref(size))):
        assert rc == status and said in lib.dpc_last_error()


def test_vocab_entries_refuse_missing_tensors(built_library):
    from deepity_b200 import _lib
    lib, size = _lib.load(), ctypes.c_size_t()
    assert lib.dpc_vocab_ce_forward(None, None) == -1
    assert lib.dpc_vocab_ce_workspace(ctypes.byref(vocab()), 0, None) == -1
    assert lib.dpc_vocab_ce_forward(None, ctypes.byref(vocab())) == -1 and b"null" in lib.dpc_last_error()
    assert lib.dpc_vocab_ce_backward(None, ctypes.byref(vocab())) == -1
    assert lib.dpc_vocab_ce_backward(None, ctypes.byref(vocab(grad_stride=2))) == -1
    assert lib.dpc_vocab_ce_backward(None, ctypes.byref(vocab(d_weight_stride=7))) == -1
    assert lib.dpc_vocab_ce_backward(None, ctypes.byref(vocab(d_weight=256, d_bias=256))) == -1  # a bias gradient without a bias
    assert lib.dpc_vocab_ce_forward(None, ctypes.byref(vocab(rows=0))) == 0  # nothing to do


def norm(**more):
    from deepity_b200 import _lib
    base = dict(rows=4, width=8, groups=1, type=0, norm=0, post_norm=0, stream_scale=1.0, branch_scale=1.0, eps=1e-6,
                stream_stride=8, branch_stride=8, gate_stride=8, new_stream_stride=8, normed_stride=8)
    return _lib.ResidualNorm(**{**base, **more})


@pytest.mark.parametrize("more,status,said", [
    (dict(type=2), -1, b"type"), (dict(norm=2), -1, b"norm"), (dict(rows=-1), -1, b"rows"), (dict(width=0), -1, b"width"),
    (dict(width=16385), -6, b"16384"), (dict(rows=1 << 32), -6, b"2^31"), (dict(eps=-1.0), -1, b"eps"),
    (dict(eps=float("nan")), -1, b"eps"), (dict(branch=256, gate=256, groups=3), -1, b"gate"),
    (dict(branch=256, gate=256, groups=0), -1, b"gate"), (dict(branch=256, gate=256, gate_stride=7), -1, b"gate"),
    (dict(gate=256), -1, b"without a branch"), (dict(post_norm=1), -1, b"without a branch"),
    (dict(stream_scale=0.5), -1, b"without a branch"), (dict(branch=256, post_weight=256), -1, b"post_norm"),
    (dict(), -1, b"null pointer"), (dict(stream=256, normed=256, stats=264), -1, b"16-byte"),
    (dict(stream=256, normed=256, stats=256, stream_stride=7), -1, b"stride")])
def test_norm_forward_refuses(built_library, more, status, said):
    from deepity_b200 import _lib
    lib = _lib.load()
    assert lib.dpc_residual_norm_forward(None, ctypes.byref(norm(**more))) == status
    assert said in lib.dpc_last_error()


@pytest.mark.parametrize("more,said", [
    (dict(), b"null pointer"), (dict(d_gate=256), b"not there"), (dict(d_branch=256), b"not there"),
    (dict(d_post_weight=256), b"not there"), (dict(d_post_bias=256), b"not there"),
    (dict(new_stream=256, stats=256, d_normed=256, d_normed_stride=7), b"stride")])
def test_norm_backward_refuses(built_library, more, said):
    from deepity_b200 import _lib
    lib = _lib.load()
    assert lib.dpc_residual_norm_backward(None, ctypes.byref(norm(**more))) == -1
    assert said in lib.dpc_last_error()


@pytest.mark.parametrize("args,status", [
    ((2, 0, 1, 8, 256, 8, 256, 8, 256, 256), -1), ((0, 1, 1, 8, 256, 8, 256, 8, 256, 256), -1),
    ((0, 14, 1, 8, 256, 8, 256, 8, 256, 256), -1), ((0, -2, 1, 8, 256, 8, 256, 8, 256, 256), -1),
    ((0, 0, -1, 8, 256, 8, 256, 8, 256, 256), -1), ((0, 0, 1, 0, 256, 8, 256, 8, 256, 256), -1),
    ((0, 0, 1 << 32, 8, 256, 8, 256, 8, 256, 256), -6), ((0, 0, 1, 8, None, 8, 256, 8, 256, 256), -1),
    ((0, 0, 1, 8, 256, 7, 256, 8, 256, 256), -1), ((0, 0, 1, 8, 256, 8, 256, 7, 256, 256), -1),
    ((0, 0, 0, 8, None, 8, None, 8, None, None), 0)])
def test_pack_refuses(built_library, args, status):
    from deepity_b200 import _lib
    assert _lib.load().dpc_activate_and_pack(None, *args) == status


@pytest.mark.parametrize("tensors", [
    (None, 256, 256, 8, 256, 8, 256, 8), (256, None, 256, 8, 256, 8, 256, 8), (256, 256, None, 8, 256, 8, 256, 8),
    (256, 256, 256, 8, None, 8, 256, 8), (256, 256, None, 8, None, 8, None, 8), (256, 256, 256, 7, 256, 8, None, 0),
    (256, 256, 256, 8, 256, 7, None, 0), (256, 256, 256, 8, 256, 8, 256, 7)])
def test_packed_backward_refuses(built_library, tensors):
    from deepity_b200 import _lib
    assert _lib.load().dpc_packed_activation_backward(None, 0, 0, 1, 8, *tensors) == -1
