"""What the operators on class scores and leaf products refuse; no device is needed: every check comes before the first device call."""
import ctypes

import pytest
import torch

from falcata_b200 import ops

S = torch.zeros(4, 6)
Y = torch.zeros(4, dtype=torch.int32)
B = torch.tensor([0, 2, 4], dtype=torch.int32)
X, W = torch.zeros(4, 3), torch.zeros(2, 5, 3)
Z = torch.zeros(4)


@pytest.mark.parametrize("error,args,kw", [
    (TypeError, ([[0.0]],), {}),
    (TypeError, (S.double(),), {}),
    (TypeError, (S.int(),), {}),
    (ValueError, (S[0],), {}),
    (ValueError, (torch.zeros(4, 0),), {}),
    (TypeError, (S, [0, 0, 0, 0]), {}),
    (TypeError, (S, Y.float()), {}),
    (ValueError, (S, Y[:3]), {}),
    (ValueError, (S, Y[:, None]), {}),
    (ValueError, (S,), {"top_k": 7}),
    (ValueError, (S,), {"top_k": -1}),
    (ValueError, (torch.zeros(4, 64),), {"top_k": 33}),
    (ValueError, (S, Y), {}),                      # not on a CUDA device
])
def test_class_log_probs_refuses(error, args, kw):
    with pytest.raises(error):
        ops.class_log_probs(*args, **kw)


@pytest.mark.parametrize("error,kw", [
    (ValueError, dict(log_norm=None)),
    (ValueError, dict(entropy=torch.zeros(3))),
    (ValueError, dict(grad_log_prob=Z)),           # no labels
    (ValueError, dict(labels=Y, grad_log_prob=torch.zeros(4, 1))),
    (ValueError, dict(grad_top_log_prob=torch.zeros(4, 2))),
    (ValueError, dict(grad_top_log_prob=torch.zeros(4, 2), top_class=torch.zeros(4, 2))),
    (ValueError, dict(grad_top_log_prob=torch.zeros(4, 2), top_class=torch.zeros(4, 3, dtype=torch.int32))),
    (ValueError, dict(grad_top_log_prob=torch.zeros(4, 7), top_class=torch.zeros(4, 7, dtype=torch.int32))),
    (ValueError, dict()),                          # not on a CUDA device
])
def test_class_log_probs_grad_refuses(error, kw):
    with pytest.raises(error):
        ops.class_log_probs_grad(S, **{"log_norm": Z, "entropy": Z, **kw})


@pytest.mark.parametrize("error,args", [
    (TypeError, (X.double(), W.double(), B)),
    (TypeError, (X, W.half(), B)),
    (ValueError, (X[0], W, B)),
    (ValueError, (torch.zeros(4, 0), torch.zeros(2, 5, 0), B)),
    (ValueError, (X, W[0], B)),
    (ValueError, (X, W[:, :0], B)),
    (ValueError, (X, W[:, :, :2], B)),
    (ValueError, (X, W[:1], B)),
    (ValueError, (X, W, B.float())),
    (ValueError, (X, W, B[:1])),
    (TypeError, (X, W, [0, 2, 4])),
    (ValueError, (X, W, B)),                       # not on a CUDA device
])
def test_leaf_products_refuses(error, args):
    with pytest.raises(error):
        ops.leaf_products(*args)


@pytest.mark.parametrize("error,args,kw", [
    (TypeError, (X, X.half(), B), {}),
    (ValueError, (X, X[:3], B), {}),
    (TypeError, (X, X, B), {"dtype": torch.float16}),
    (TypeError, (X.half(), X.half(), B), {"dtype": torch.bfloat16}),
    (ValueError, (X, X, B[:1]), {}),
    (ValueError, (X, X, B), {}),                   # not on a CUDA device
])
def test_leaf_gram_refuses(error, args, kw):
    with pytest.raises(error):
        ops.leaf_gram(*args, **kw)


def test_native_entry_points_return_errors():
    """The C entry points check their sizes themselves, before any device call, and report instead of throwing."""
    from falcata_b200.basic import _lib

    lib, L, I, P = _lib(), ctypes.c_longlong, ctypes.c_int, ctypes.c_void_p
    lib.FB_OpsLastError.restype = ctypes.c_char_p

    def scores(rows=4, classes=6, label_bits=0, top_k=0):
        return lib.FB_OpClassLogProbs(P(), I(0), L(rows), L(classes), L(classes), L(1), P(), I(label_bits), I(top_k), P(), P(), P(), P(), P(), I(0), P())

    for bad, word in ((dict(rows=-1), b"rows"), (dict(rows=1 << 31), b"rows"), (dict(classes=0), b"classes"), (dict(classes=1 << 31), b"classes"),
                      (dict(label_bits=16), b"labels"), (dict(top_k=33, classes=100), b"alternatives"), (dict(top_k=7), b"alternatives"), (dict(top_k=-1), b"alternatives")):
        assert scores(**bad) == -1 and word in lib.FB_OpsLastError()
    assert lib.FB_OpLeafProducts(P(), L(3), P(), L(15), L(3), L(1), P(), I(32), I(0), L(4), I(3), I(5), I(0), P(), P(), P(), I(0), P()) == -1 and b"leaves" in lib.FB_OpsLastError()
    assert lib.FB_OpLeafProducts(P(), L(3), P(), L(15), L(3), L(1), P(), I(16), I(2), L(4), I(3), I(5), I(0), P(), P(), P(), I(0), P()) == -1 and b"boundaries" in lib.FB_OpsLastError()
    assert lib.FB_OpLeafProducts(P(), L(3), P(), L(15), L(3), L(1), P(), I(32), I(2), L(4), I(0), I(5), I(0), P(), P(), P(), I(0), P()) == -1 and b"feature" in lib.FB_OpsLastError()
    assert lib.FB_OpLeafGram(P(), L(3), P(), L(3), P(), I(32), I(2), L(4), I(0), I(3), I(0), I(0), P(), P(), P(), I(0), P()) == -1 and b"column" in lib.FB_OpsLastError()


def test_forward_mode_derivatives_are_refused():
    """A tangent would be lost without a word; outside forward mode, and for tensors without a tangent, nothing changes."""
    from torch.autograd import forward_ad

    half = torch.zeros(4)
    with forward_ad.dual_level():
        s, x, w = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (S, X, W))
        z = forward_ad.make_dual(Z, torch.ones_like(Z))
        for call in (lambda: ops.class_log_probs(s, Y), lambda: ops.class_log_probs_grad(s, Z, Z), lambda: ops.class_log_probs_grad(S, z, Z), lambda: ops.class_log_probs_grad(S, Z, Z, grad_entropy=z),
                     lambda: ops.leaf_products(x, W, B), lambda: ops.leaf_products(X, w, B), lambda: ops.leaf_gram(x, X, B), lambda: ops.leaf_gram(X, x, B)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with pytest.raises(ValueError, match="CUDA"):
            ops.class_log_probs_grad(S, half, half)


def test_sizes_beyond_the_native_call_are_refused():
    """The native call takes leaves and columns as 32-bit numbers: 2^32 + 3 of them must not pass as 3."""
    from falcata_b200.basic import _lib

    many = (1 << 32) + 3
    one = torch.zeros(1, 1)
    wide, begin = one.expand(1, many), torch.zeros(1, dtype=torch.int32)
    for call, word in ((lambda: ops.leaf_products(wide, one[None].expand(2, 5, many), B), "columns"), (lambda: ops.leaf_products(X, one[None].expand(2, many, 3), B), "outputs"),
                       (lambda: ops.leaf_gram(wide, one, B), "columns"), (lambda: ops.leaf_gram(one, wide, B), "columns"), (lambda: ops.leaf_gram(X, X, begin.expand(many + 1)), "leaves"),
                       (lambda: ops.leaf_products(X, one[None].expand(many, 5, 3), begin.expand(many + 1)), "leaves")):
        with pytest.raises(ValueError, match=f"{word} are covered"):
            call()
    lib, L, I, P = _lib(), ctypes.c_longlong, ctypes.c_int, ctypes.c_void_p
    lib.FB_OpsLastError.restype = ctypes.c_char_p
    over = (1 << 28) + 1
    for leaves, f, k in ((over, 3, 5), (2, over, 5), (2, 3, over)):
        assert lib.FB_OpLeafProducts(P(), L(3), P(), L(15), L(3), L(1), P(), I(32), I(leaves), L(4), I(f), I(k), I(0), P(), P(), P(), I(0), P()) == -1 and (b"leaves" if leaves == over else b"2^28") in lib.FB_OpsLastError()
        assert lib.FB_OpLeafGram(P(), L(3), P(), L(3), P(), I(32), I(leaves), L(4), I(f), I(k), I(0), I(0), P(), P(), P(), I(0), P()) == -1
