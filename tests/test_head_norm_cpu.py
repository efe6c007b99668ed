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


def _head_case(T, K):
    gen = torch.Generator().manual_seed(3)
    x, w = torch.randn(6, 9, generator=gen, dtype=torch.float64), torch.randn(13, 9, generator=gen, dtype=torch.float64)
    labels = torch.randint(13, (6, K), generator=gen)
    return x, w, labels, torch.randn(6, generator=gen, dtype=torch.float64), gen


def test_cross_entropy_gradients_against_differences():
    from oracle import head_norm_oracle as O

    x, w, labels, up, _ = _head_case(1.0, 1)
    shares = torch.ones(6, 1, dtype=torch.float64)
    shares[2] = 0
    _directional(lambda x, w: (O.head_losses(x, w, labels, shares) * up).sum(), (x, w), O.head_backward(up, x, w, labels, shares), 5)


@pytest.mark.parametrize("T", [1.0, 2.5])
def test_distillation_gradients_against_differences(T):
    from oracle import head_norm_oracle as O

    x, w, labels, up, gen = _head_case(T, 5)
    logits = torch.randn(6, 5, generator=gen)
    logits[1, 2:] = float("-inf")
    logits[4] = float("-inf")
    shares, used = O.teacher_shares(logits, T)
    assert used.tolist() == [True, True, True, True, False, True]
    _directional(lambda x, w: (O.head_losses(x, w, labels, shares, T) * up).sum(), (x, w),
                 O.head_backward(up, x, w, labels, shares, T), 6)
    assert float(O.head_losses(x, w, labels, shares, T)[4]) == 0


def test_head_refusals_before_any_launch():
    import flashrwkv_b200 as F

    x, w, t = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(5, 8, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(TypeError, match="targets must be a torch.Tensor"):
        F.pretrain_head_cross_entropy_bf16(x, w, [0, 1, 2, 3])
    with pytest.raises(ValueError, match="contiguous CUDA bfloat16"):
        F.pretrain_head_cross_entropy_bf16(x, w, t)
    with pytest.raises(ValueError, match="reduction"):
        F.pretrain_head_cross_entropy_bf16(x, w, t, reduction=None)
    for index in (1.0, None, True, 2 ** 63):
        with pytest.raises(ValueError, match="ignore_index"):
            F.pretrain_head_cross_entropy_bf16(x, w, t, ignore_index=index)
    with pytest.raises(TypeError, match="teacher_indices must be a torch.Tensor"):
        F.pretrain_head_distill_bf16(x, w, t, None)
    with pytest.raises(ValueError, match="contiguous CUDA bfloat16"):
        F.pretrain_head_distill_bf16(x, w, torch.zeros(4, 1), t[:, None])


class _HeadArgs(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_void_p) for n in ("x", "weight", "labels", "teacher_logits", "row_grads", "grad_scale", "row_losses",
                                                "loss", "grad_x", "grad_weight", "workspace")]
                + [("workspace_bytes", ctypes.c_size_t), ("error_flag", ctypes.c_void_p), ("rows", ctypes.c_longlong),
                   ("ignore_index", ctypes.c_longlong)]
                + [(n, ctypes.c_int) for n in ("channels", "vocab", "top", "label_bytes", "mean")] + [("temperature", ctypes.c_float)])


def test_head_entry_refuses_bad_arguments_without_a_device():
    from flashrwkv_b200 import _ext

    lib = _ext.capi()
    lib.frwkv_pretrain_head_loss_workspace_bytes.restype = ctypes.c_size_t

    def call(**changes):
        a = _HeadArgs(x=4096, weight=4096, labels=4096, row_losses=4096, workspace=4096, workspace_bytes=1 << 40, error_flag=4096,
                      rows=4, ignore_index=-100, channels=64, vocab=100, top=1, label_bytes=8, mean=1, temperature=1.0)
        for name, value in changes.items():
            setattr(a, name, value)
        return lib.frwkv_pretrain_head_loss(ctypes.byref(a), None)

    assert lib.frwkv_pretrain_head_loss(None, None) == -1
    for changes, message in (({"x": 0}, b"null pointer"), ({"workspace": 0}, b"null pointer"), ({"error_flag": 0}, b"null pointer"),
                             ({"rows": 0}, b"positive"), ({"rows": (1 << 24) + 1}, b"16777216 rows"), ({"channels": 12}, b"multiple of 8"),
                             ({"channels": 65544}, b"up to 65536"), ({"vocab": (1 << 20) + 1}, b"1048576"), ({"vocab": -3}, b"positive"),
                             ({"label_bytes": 2}, b"int32 or int64"), ({"top": 2}, b"one label"), ({"top": 0}, b"1 to 512"),
                             ({"top": 513, "teacher_logits": 4096}, b"1 to 512"), ({"temperature": 0.0}, b"temperature"),
                             ({"temperature": 2.0}, b"temperature 1"), ({"temperature": float("nan")}, b"temperature"),
                             ({"x": 4104}, b"aligned"), ({"grad_weight": 4104}, b"aligned"), ({"workspace": 4096 + 64}, b"aligned"),
                             ({"labels": 4100}, b"aligned"), ({"workspace_bytes": 16}, b"workspace is smaller")):
        assert call(**changes) == -1, changes
        assert message in lib.frwkv_last_error(), (changes, lib.frwkv_last_error())
    assert lib.frwkv_pretrain_head_loss_workspace_bytes(ctypes.c_longlong(0), 64, 100, 1, 1) == 0
    ok, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4104)
    n, none = ctypes.c_longlong(8), ctypes.c_longlong(0)
    assert lib.frwkv_scale_bf16(None, none, None, none, ok, None) == -1 and b"null pointer" in lib.frwkv_last_error()
    assert lib.frwkv_scale_bf16(None, n, ok, n, ok, None) == -1 and lib.frwkv_scale_bf16(ok, n, None, none, None, None) == -1
    assert lib.frwkv_scale_bf16(ok, ctypes.c_longlong(12), None, none, ok, None) == -1
    assert b"multiples of 8" in lib.frwkv_last_error()
    assert lib.frwkv_scale_bf16(ok, n, odd, n, ok, None) == -1 and b"aligned" in lib.frwkv_last_error()


def test_head_workspace_stays_bounded():
    """The exponentials of a piece take at most 1 GiB (or 256 rows), so a long batch costs the workspace of a piece, its
    compacted rows and the partial sums, not rows x vocabulary."""
    from flashrwkv_b200 import _ext

    lib = _ext.capi()
    lib.frwkv_pretrain_head_loss_workspace_bytes.restype = ctypes.c_size_t

    def size(rows, channels, vocab, grads):
        return lib.frwkv_pretrain_head_loss_workspace_bytes(ctypes.c_longlong(rows), channels, vocab, grads, grads)

    assert size(1 << 17, 2048, 65536, 1) < (5 << 30) and size(1 << 17, 2048, 65536, 0) < (1 << 30)
    assert size(8192, 2048, 65536, 1) < (1400 << 20)
