"""Training LayerNorm and add + LayerNorm (forward and backward) against the float64 oracle, element by element.

Tolerances: every output is computed in fp32 and rounded once to bf16, i.e. off by at most eps(bf16) / 2 = 2^-8 of its
value, plus the fp32 error in front of the rounding.  u = 2^-24.  The row statistics are sums of C terms in a tree of
depth <= 32 per thread + 9 levels, so mean and variance are good to 64 u; the subtraction s - mean carries 64 u max|s|,
i.e. 64 u max|s| rstd in units of xhat.  With A = 1 + max|s| rstd, xhat is therefore within 128 u A, the output within
128 u A max|w| plus its own rounding of the sum (u |b|), and dx within 512 u A^2 rstd max|h| (three products with xhat).  A
column sum over R rows adds R u sum|terms| for any order of addition.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF = torch.finfo(torch.bfloat16).eps / 2
EPS = 1e-5
SHAPES = [(1, 1, 8), (2, 3, 16), (1, 1, 2048), (3, 37, 256), (2, 19, 264), (1, 70, 512), (1, 70, 520), (5, 7, 1024), (1, 1237, 1000),
          (3, 131, 2048), (1, 66, 2056), (1, 9, 4096), (1, 9, 4104), (2, 17, 8192), (1, 5, 8200), (1, 3, 16384), (3000, 1, 64)]


def _inputs(B, T, C, seed, mean=0.3, scale=1.0):
    gen = torch.Generator().manual_seed(seed)

    def rn(*shape, s=1.0, m=0.0):
        return (torch.randn(*shape, generator=gen) * s + m).to(torch.bfloat16).cuda()

    return dict(x=rn(B, T, C, s=scale, m=mean), residual=rn(B, T, C, s=2 * scale), weight=rn(C, s=0.3, m=1.0), bias=rn(C, s=0.2),
                g=rn(B, T, C), gs=rn(B, T, C))


def _amplification(s):
    s = s.double()
    rstd = (s.var(-1, unbiased=False, keepdim=True) + EPS).rsqrt()
    return 1 + s.abs().amax(-1, keepdim=True) * rstd, rstd


def _close(got, want, slack, name):
    got = got.double()
    assert torch.isfinite(got).all(), name
    over = (got - want).abs() - (HALF * want.abs() * (1 + 2 * HALF) + slack)
    assert float(over.max()) <= 0, f"{name}: {float(over.max())} beyond the bound"


def _check_all(i, s, out, ds, dw, db, gs=None):
    from oracle import head_norm_oracle as O

    A, rstd = _amplification(s)
    w = i["weight"].double()
    rows = s.numel() // s.shape[-1]
    _close(out, O.layer_norm(s, w, i["bias"], EPS), 128 * U * A * w.abs().max() + 2 * U * i["bias"].double().abs(), "out")
    want, want_w, want_b = O.layer_norm_backward(i["g"], s, w, EPS)
    slack = 512 * U * A ** 2 * rstd * (i["g"].double() * w).abs().amax(-1, keepdim=True)
    if gs is not None:
        want = want + gs.double()
        slack = slack + 2 * U * gs.double().abs()
    _close(ds, want, slack, "d x")
    g = i["g"].double().abs()
    unit = (s.double() - s.double().mean(-1, keepdim=True)).abs() * rstd
    _close(dw, want_w, (rows + 4) * U * (g * unit).sum((0, 1)) + (128 * U * A * g).sum((0, 1)), "d weight")
    _close(db, want_b, rows * U * g.sum((0, 1)), "d bias")


@pytest.mark.parametrize("B,T,C", SHAPES)
def test_layer_norm(B, T, C):
    import flashrwkv_b200 as F

    i = _inputs(B, T, C, B * 100 + T + C)
    leaves = [i[n].requires_grad_() for n in ("x", "weight", "bias")]
    out = F.pretrain_tmix_layer_norm_bf16(*leaves, eps=EPS)
    grads = torch.autograd.grad(out, leaves, i["g"])
    i = {k: v.detach() for k, v in i.items()}
    _check_all(i, i["x"], out.detach(), *grads)
    # the inference operator normalises the same rows
    infer = F.infer_tmix_layer_norm_forward_varlen(i["x"].view(-1, C), i["weight"], i["bias"], eps=EPS)
    A, _ = _amplification(i["x"])
    gap = (infer.view_as(out).double() - out.detach().double()).abs()
    assert bool((gap <= 2 * HALF * out.detach().double().abs() * (1 + 2 * HALF) + 512 * U * A * 2.5).all())


@pytest.mark.parametrize("B,T,C", SHAPES)
def test_add_layer_norm(B, T, C):
    import flashrwkv_b200 as F

    i = _inputs(B, T, C, B * 100 + T + C + 1)
    leaves = [i[n].requires_grad_() for n in ("x", "residual", "weight", "bias")]
    total, out = F.pretrain_tmix_add_layer_norm_bf16(*leaves, eps=EPS)
    gx, gr, gw, gb = torch.autograd.grad((total, out), leaves, (i["gs"], i["g"]))
    i = {k: v.detach() for k, v in i.items()}
    assert torch.equal(total.detach(), (i["x"].float() + i["residual"].float()).to(torch.bfloat16))
    assert torch.equal(gx, gr)
    _check_all(i, total.detach(), out.detach(), gx, gw, gb, i["gs"])


@pytest.mark.parametrize("mean,scale", [(0.0, 1e-4), (100.0, 1.0), (-30.0, 8.0), (0.0, 1e4)])
def test_layer_norm_of_shifted_and_scaled_rows(mean, scale):
    import flashrwkv_b200 as F

    i = _inputs(2, 40, 776, 5, mean=mean, scale=scale)
    leaves = [i[n].requires_grad_() for n in ("x", "weight", "bias")]
    out = F.pretrain_tmix_layer_norm_bf16(*leaves, eps=EPS)
    grads = torch.autograd.grad(out, leaves, i["g"])
    i = {k: v.detach() for k, v in i.items()}
    _check_all(i, i["x"], out.detach(), *grads)


def test_constant_rows_and_rows_that_are_not_finite():
    """A constant row normalises to the bias; a NaN or infinite value spoils its own row and the parameter gradients only."""
    import flashrwkv_b200 as F

    i = _inputs(1, 50, 328, 9)
    x = i["x"].clone()
    x[0, 3] = 2.5
    x[0, 7, 11] = float("nan")
    x[0, 20, 0] = float("inf")
    good = [r for r in range(50) if r not in (7, 20)]
    leaves = [t.requires_grad_() for t in (x, i["weight"], i["bias"])]
    out = F.pretrain_tmix_layer_norm_bf16(*leaves, eps=EPS)
    dx, dw, db = torch.autograd.grad(out, leaves, i["g"])
    assert torch.equal(out[0, 3], i["bias"])
    assert torch.isnan(out[0, 7]).all() and torch.isnan(dx[0, 7]).all() and torch.isnan(out[0, 20]).all()
    assert torch.isnan(dw).all() and torch.isfinite(db).all()
    alone = F.pretrain_tmix_layer_norm_bf16(x.detach()[:, good].contiguous(), i["weight"], i["bias"], eps=EPS)
    assert torch.equal(out[:, good], alone)


def test_gradients_that_are_missing_expanded_or_not_asked_for():
    import flashrwkv_b200 as F

    i = _inputs(2, 33, 520, 11)
    x, r, w, b = (i[n].requires_grad_() for n in ("x", "residual", "weight", "bias"))
    # the sum alone: its gradient passes through; the norm's parameters take no part
    total, out = F.pretrain_tmix_add_layer_norm_bf16(x, r, w, b, eps=EPS)
    gx, gr, gw = torch.autograd.grad(total, (x, r, w), i["gs"], allow_unused=True)
    assert torch.equal(gx, i["gs"]) and torch.equal(gr, i["gs"]) and gw is None
    # the norm alone equals a zero gradient of the sum
    total, out = F.pretrain_tmix_add_layer_norm_bf16(x, r, w, b, eps=EPS)
    only = torch.autograd.grad(out, (x, r, w, b), i["g"], retain_graph=True)
    both = torch.autograd.grad((total, out), (x, r, w, b), (torch.zeros_like(total), i["g"]))
    for a, c in zip(only, both):
        assert torch.equal(a, c)
    # an expanded gradient, and one that starts in the middle of a 16-byte piece
    out = F.pretrain_tmix_layer_norm_bf16(x, w, b, eps=EPS)
    one = torch.ones((), dtype=torch.bfloat16, device="cuda").expand_as(out)
    got = torch.autograd.grad(out, (x, w, b), one, retain_graph=True)
    store = torch.ones(out.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view_as(out)
    assert store.data_ptr() % 16 != 0
    for a, c in zip(got, torch.autograd.grad(out, (x, w, b), store)):
        assert torch.equal(a, c)
    # frozen parameters, frozen rows
    w0, b0, x0 = w.detach(), b.detach(), x.detach()
    out = F.pretrain_tmix_layer_norm_bf16(x, w0, b0, eps=EPS)
    dx = torch.autograd.grad(out, x, i["g"])[0]
    out = F.pretrain_tmix_layer_norm_bf16(x0, w, b0, eps=EPS)
    dw = torch.autograd.grad(out, w, i["g"])[0]
    out = F.pretrain_tmix_layer_norm_bf16(x, w, b, eps=EPS)
    full = torch.autograd.grad(out, (x, w), i["g"])
    assert torch.equal(dx, full[0]) and torch.equal(dw, full[1])


def test_same_bits_every_time_on_any_stream_and_in_a_graph():
    import flashrwkv_b200 as F

    i = _inputs(4, 300, 1544, 13)
    leaves = [i[n].requires_grad_() for n in ("x", "residual", "weight", "bias")]

    def step():
        outs = F.pretrain_tmix_add_layer_norm_bf16(*leaves, eps=EPS)
        return (*(o.detach() for o in outs), *torch.autograd.grad(outs, leaves, (i["gs"], i["g"])))

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [t.clone() for t in step()]
    side.synchronize()
    for a, c in zip(want, again):
        assert torch.equal(a, c)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(2):
        for t in held:
            t.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(want, held):
            assert torch.equal(a, c)
    # new values in the same leaves
    with torch.no_grad():
        leaves[0].mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    kept = [t.clone() for t in held]
    for a, c in zip(step(), kept):
        assert torch.equal(a, c)


def test_many_rows_fall_into_many_slabs():
    """More rows than one wave of CTAs holds: each column sum of ones is the row count, exactly."""
    import flashrwkv_b200 as F

    x = torch.randn(9000, 136, device="cuda").to(torch.bfloat16)
    w = torch.ones(136, device="cuda", dtype=torch.bfloat16).requires_grad_()
    b = torch.zeros_like(w).requires_grad_()
    out = F.pretrain_tmix_layer_norm_bf16(x, w, b)
    _, db = torch.autograd.grad(out, (w, b), torch.ones_like(out))
    assert torch.equal(db, torch.full_like(db, 9000.0))


def test_second_order_is_refused():
    import flashrwkv_b200 as F

    i = _inputs(1, 4, 64, 3)
    x = i["x"].requires_grad_()
    out = F.pretrain_tmix_layer_norm_bf16(x, i["weight"], i["bias"])
    with pytest.raises(RuntimeError, match="not itself differentiable"):
        torch.autograd.grad(out, x, i["g"], create_graph=True)


def test_refusals_on_the_device():
    import flashrwkv_b200 as F

    i = _inputs(2, 4, 64, 3)
    x, w, b = i["x"], i["weight"], i["bias"]
    shifted = torch.zeros(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view_as(x)
    wide = torch.zeros(1, 16392, dtype=x.dtype, device="cuda")
    for args, message in (((shifted, w, b), "16-byte aligned"), ((x[:, ::2], w, b), "contiguous"),
                          ((x.float(), w, b), "bfloat16"), ((x, w[:8], b), "weight must have shape"),
                          ((x, w, b[:8].contiguous()), "bias must have shape"), ((x[0, 0], w, b), "non-empty shape"),
                          ((x[:0], w, b), "non-empty shape"), ((x.view(-1, 4), w[:4], b[:4]), "multiple of 8"),
                          ((wide, wide[0], wide[0]), "up to 16384"), ((x, w.cpu(), b), "CUDA")):
        with pytest.raises(ValueError, match=message):
            F.pretrain_tmix_layer_norm_bf16(*args)
    with pytest.raises(ValueError, match="same shape as x"):
        F.pretrain_tmix_add_layer_norm_bf16(x, x[:1], w, b)
    for eps in (0.0, -1.0, float("nan"), float("inf"), 1e-60):
        with pytest.raises(ValueError, match="eps must be positive"):
            F.pretrain_tmix_layer_norm_bf16(x, w, b, eps=eps)


def test_offsets_beyond_32_bits():
    import flashrwkv_b200 as F

    rows, C = 270_000, 8192  # 2.2e9 values
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(rows, C, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    w = torch.ones(C, dtype=torch.bfloat16, device="cuda").requires_grad_()
    b = torch.zeros(C, dtype=torch.bfloat16, device="cuda").requires_grad_()
    x.requires_grad_()
    out = F.pretrain_tmix_layer_norm_bf16(x, w, b)
    g = torch.zeros_like(out)
    g[-3:] = torch.empty_like(g[-3:]).normal_(generator=gen)
    dx, dw, db = torch.autograd.grad(out, (x, w, b), g)
    few = x.detach()[-3:].contiguous().requires_grad_()
    want = F.pretrain_tmix_layer_norm_bf16(few, w, b)
    assert torch.equal(out[-3:], want)
    ex, ew, eb = torch.autograd.grad(want, (few, w, b), g[-3:].contiguous())
    assert torch.equal(dx[-3:], ex) and bool((dx[:-3] == 0).all())
    # three terms per column, added in another order among zeros: 3 u of their sum of magnitudes, then the rounding to bf16
    slack = 3 * U * (g[-3:].double().abs() * (1 + want.double().abs())).sum(0)
    assert bool(((dw.double() - ew.double()).abs() <= 2 * HALF * ew.double().abs() + slack).all())
    assert bool(((db.double() - eb.double()).abs() <= 2 * HALF * eb.double().abs() + slack).all())


def test_a_captured_backward_pass_beside_an_eager_graph_of_the_same_leaves():
    """Refused where that graph was made on the default stream and the leaf's gradient is asked for."""
    import flashrwkv_b200 as F

    x, r = (torch.randn(6, 5, 64, device="cuda").bfloat16().requires_grad_() for _ in range(2))
    w, b = (torch.randn(64, device="cuda").bfloat16().requires_grad_() for _ in range(2))
    go = torch.randn_like(x)
    for call in (lambda: F.pretrain_tmix_layer_norm_bf16(x, w, b), lambda: F.pretrain_tmix_add_layer_norm_bf16(x, r, w, b)[1]):
        alive = call()
        with pytest.raises(RuntimeError, match="default stream"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                torch.autograd.grad(call(), (w, b), go)
        torch.cuda.synchronize()
        want = torch.autograd.grad(alive, (w, b), go)
        del alive
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held = torch.autograd.grad(call(), (w, b), go)
        g.replay()
        torch.cuda.synchronize()
        for got, value in zip(held, want):
            assert torch.equal(got, value)


def test_an_eager_backward_pass_behind_a_captured_forward_pass_beside_an_eager_graph():
    """Only a captured backward pass cannot reach leaves of the default stream."""
    import flashrwkv_b200 as F

    x, r = (torch.randn(6, 5, 64, device="cuda").bfloat16().requires_grad_() for _ in range(2))
    w, b = (torch.randn(64, device="cuda").bfloat16().requires_grad_() for _ in range(2))
    go = torch.randn_like(x)
    for call in (lambda: F.pretrain_tmix_layer_norm_bf16(x, w, b), lambda: F.pretrain_tmix_add_layer_norm_bf16(x, r, w, b)[1]):
        alive = call()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        g.replay()
        torch.cuda.synchronize()
        got = torch.autograd.grad(out, (x, w, b), go)
        for a, c in zip((out, *got), (alive, *torch.autograd.grad(alive, (x, w, b), go))):
            assert torch.equal(a, c)


def test_a_backward_pass_captured_apart_from_its_forward_pass():
    """Refused while the leaves belong to a graph of the default stream; without one it is captured and replayed."""
    import flashrwkv_b200 as F

    x, r = (torch.randn(6, 5, 64, device="cuda").bfloat16().requires_grad_() for _ in range(2))
    w, b = (torch.randn(64, device="cuda").bfloat16().requires_grad_() for _ in range(2))
    go = torch.randn_like(x)
    side = torch.cuda.Stream()
    for call in (lambda: F.pretrain_tmix_layer_norm_bf16(x, w, b), lambda: F.pretrain_tmix_add_layer_norm_bf16(x, r, w, b)[1]):
        alive = call()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            out = call()
        side.synchronize()
        for leaves in ((x, w, b), (x,), (b,)):
            with pytest.raises(RuntimeError, match="default stream"):
                with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                    torch.autograd.grad(out, leaves, go, retain_graph=True)
            torch.cuda.synchronize()
        want = torch.autograd.grad(alive, (x, w, b), go)
        del alive, out
        with torch.cuda.stream(side):
            out = call()
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            held = torch.autograd.grad(out, (x, w, b), go)
        g.replay()
        torch.cuda.synchronize()
        for a, c in zip(held, want):
            assert torch.equal(a, c)
        del out


@pytest.mark.parametrize("rows,C", [(9000, 136), (9000, 520), (9000, 1032), (9000, 2056), (4500, 8200), (593, 264), (149, 64)])
def test_every_row_counts_once_in_the_parameter_gradients(rows, C):
    """A row's upstream gradient is 1 in the column of its number, 0 elsewhere: the gradient of the bias is the number of rows
    that share a column, a whole number below 256, exactly, and a row that is lost at a slab's edge, or counted twice, shows as
    one.  The gradient of the weight is the sum of as many units of xhat, within the bounds above."""
    import flashrwkv_b200 as F
    from oracle import head_norm_oracle as O

    i = _inputs(1, rows, C, rows + C)
    w, b = i["weight"].requires_grad_(), i["bias"].requires_grad_()
    g = torch.zeros(1, rows, C, dtype=torch.bfloat16, device="cuda")
    at = torch.arange(rows, device="cuda")
    g[0, at, at % C] = 1.0
    dw, db = torch.autograd.grad(F.pretrain_tmix_layer_norm_bf16(i["x"], w, b, eps=EPS), (w, b), g)
    count = torch.bincount(at % C, minlength=C)
    assert int(count.max()) < 256 and torch.equal(db, count.to(torch.bfloat16))
    _, want, _ = O.layer_norm_backward(g, i["x"], w.detach(), EPS)
    A, rstd = _amplification(i["x"])
    unit = (i["x"].double() - i["x"].double().mean(-1, keepdim=True)).abs() * rstd
    _close(dw, want, (rows + 4) * U * (g.double() * unit).sum((0, 1)) + (128 * U * A * g.double()).sum((0, 1)), "d weight")
