"""Without a GPU: the float64 gradients of the training norms and head losses against central differences, and what the
operators refuse before any launch."""
import ctypes

import pytest
import torch


def _directional(f, tensors, grads, seed):
    """|sum <grad, d> - (f(t + h d) - f(t - h d)) / 2h| is O(h^2 |f'''|) + rounding / h: 1e-6 at h = 1e-4 for these sizes."""
    gen = torch.Generator().manual_seed(seed)
    h = 1e-4
    for k, (t, g) in enumerate(zip(tensors, grads)):
        d = torch.randn(t.shape, generator=gen, dtype=torch.float64)
        up = [u + h * d if j == k else u for j, u in enumerate(tensors)]
        down = [u - h * d if j == k else u for j, u in enumerate(tensors)]
        slope = float(f(*up) - f(*down)) / (2 * h)
        assert abs(slope - float((g * d).sum())) <= 1e-6 * max(1.0, float(g.norm()) * float(d.norm())), k


def test_layer_norm_gradients_against_differences():
    from oracle import head_norm_oracle as O

    gen = torch.Generator().manual_seed(1)
    s, w, b, g = (torch.randn(*n, generator=gen, dtype=torch.float64) for n in ((2, 5, 24), (24,), (24,), (2, 5, 24)))
    _directional(lambda *t: (O.layer_norm(*t, 1e-5) * g).sum(), (s, w, b), O.layer_norm_backward(g, s, w, 1e-5), 2)


def _norm_args(C=64):
    t = torch.zeros(2, 3, C, dtype=torch.bfloat16)
    return t, torch.ones(C, dtype=torch.bfloat16), torch.zeros(C, dtype=torch.bfloat16)


def test_norm_refusals_before_any_launch():
    import flashrwkv_b200 as F

    x, w, b = _norm_args()
    with pytest.raises(TypeError, match="x must be a torch.Tensor"):
        F.pretrain_tmix_layer_norm_bf16(None, w, b)
    with pytest.raises(TypeError, match="weight must be a torch.Tensor"):
        F.pretrain_tmix_layer_norm_bf16(x, 1.0, b)
    with pytest.raises(TypeError, match="residual must be a torch.Tensor"):
        F.pretrain_tmix_add_layer_norm_bf16(x, None, w, b)
    with pytest.raises(ValueError, match="contiguous CUDA bfloat16"):
        F.pretrain_tmix_layer_norm_bf16(x, w, b)
    with pytest.raises(ValueError, match="contiguous CUDA bfloat16"):
        F.pretrain_tmix_add_layer_norm_bf16(x.half(), x, w, b)


def test_norm_entries_refuse_bad_arguments_without_a_device():
    from flashrwkv_b200 import _ext

    lib = _ext.capi()
    lib.frwkv_pretrain_layer_norm_workspace_floats.restype = ctypes.c_longlong
    ok, odd, eps = ctypes.c_void_p(4096), ctypes.c_void_p(4096 + 8), ctypes.c_float(1e-5)
    rows = ctypes.c_longlong(4)

    def forward(x=ok, residual=None, sum_out=None, rows=rows, C=64, eps=eps, out=ok):
        return lib.frwkv_pretrain_layer_norm_forward(x, residual, ok, ok, sum_out, out, ok, ok, rows, C, eps, None)

    def backward(grad=ok, gw=ok, gb=ok, ws=ok, floats=1 << 40, rows=rows, C=64):
        return lib.frwkv_pretrain_layer_norm_backward(grad, None, ok, ok, ok, ok, ok, gw, gb, ws, ctypes.c_longlong(floats), rows,
                                                      C, None)

    for call, message in ((lambda: forward(x=None), b"null pointer"), (lambda: forward(x=odd), b"16-byte aligned"),
                          (lambda: forward(residual=ok), b"go together"), (lambda: forward(rows=ctypes.c_longlong(0)), b"positive"),
                          (lambda: forward(C=12), b"multiple of 8"), (lambda: forward(C=16392), b"up to 16384"),
                          (lambda: forward(eps=ctypes.c_float(0.0)), b"eps"),
                          (lambda: forward(eps=ctypes.c_float(float("nan"))), b"eps"),
                          (lambda: forward(eps=ctypes.c_float(float("inf"))), b"eps"),
                          (lambda: backward(grad=None), b"null pointer"), (lambda: backward(grad=odd), b"16-byte aligned"),
                          (lambda: backward(gb=None), b"go together"), (lambda: backward(ws=None), b"null workspace"),
                          (lambda: backward(floats=10, rows=ctypes.c_longlong(4000)), b"workspace is smaller"),
                          (lambda: backward(C=20), b"multiple of 8")):
        assert call() == -1
        assert message in lib.frwkv_last_error(), lib.frwkv_last_error()
    assert lib.frwkv_pretrain_layer_norm_workspace_floats(ctypes.c_longlong(0), 64) == 0
