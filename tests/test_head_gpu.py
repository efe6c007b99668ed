"""The head's losses (cross entropy, distillation) and their gradients against the float64 oracle.

Bounds, with u = 2^-24 and rho = eps(bf16) / 2 = 2^-8.  A logit is an fp32 sum of C exact products; for any order of
addition, and one unit per addition rather than half (tensor cores may truncate), it is within delta_n = 2 C u B_n / T of its
value, B_n = max_v sum_c |x_nc w_vc|.  The normaliser sums 256 positive terms per tile, then the tiles: relative error
<= (256 + tiles + 16) u, each exponential 2^-21.  So with zmax_n = max |z_n|:
    |loss error| <= T^2 (2 delta_n + (300 + tiles) u + 2^-20 + 32 u (zmax_n + |loss|))  =: T^2 e_n
A logit gradient g = scale T (q - p) has q's relative error e_n plus that of the fp16 exponential (2^-11, or 2^-24 of the
tile's maximum where it is subnormal), and its own rounding rho |g|:
    gerr = rho |g| + scale T (q (2 e_n + 2^-10) + 2^-23 q_tilemax + 4 u)
dx = g W is then within gerr |W| + V 2 u (|g| |W|) + rho |dx| and dW within gerr^T |x| + N 2 u (|g|^T |x|) + rho |dW|.  These
hold for every element.  Roundings are independent, so in the Frobenius norm the two of them (g, result) stay below
sqrt(2) rho / sqrt(3) = 3.2e-3 of sqrt(|result|^2 + sum g^2 w^2); 4e-3 is asked for.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
RHO = torch.finfo(torch.bfloat16).eps / 2


def _rows(N, C, V, seed, sure=True):
    gen = torch.Generator().manual_seed(seed)
    w = (torch.randn(V, C, generator=gen) * 2 / C ** 0.5).to(torch.bfloat16)
    t = torch.randint(V, (N,), generator=gen)
    x = torch.randn(N, C, generator=gen)
    if sure:
        x = x + 2 * torch.rand(N, 1, generator=gen) * w[t].float()
    return x.to(torch.bfloat16).cuda(), w.cuda(), t.cuda(), gen


def _reference(x, w, labels, shares, T, row_grads):
    """Losses, gradients and the bounds above, in pieces of the rows."""
    N, C = x.shape
    V = w.shape[0]
    xd, wd = x.double(), w.double()
    aw = wd.abs()
    out = {k: [] for k in ("loss", "eloss", "dx", "edx", "fx")}
    dw, edw = torch.zeros_like(wd), torch.zeros_like(wd)
    fw = 0.0
    tiles = -(-V // 256)
    step = max(1, 2 ** 26 // V)
    for lo in range(0, N, step):
        s = slice(lo, min(N, lo + step))
        used = (shares[s].sum(1) > 0).double()[:, None]
        z = xd[s] @ wd.T / T
        B = (xd[s].abs() @ aw.T).amax(1)
        lq = torch.log_softmax(z, 1)
        lab = torch.where(shares[s] > 0, labels[s].long(), 0)
        loss = T * T * (torch.special.xlogy(shares[s], shares[s]) - shares[s] * lq.gather(1, lab)).sum(1)
        e = 2 * (2 * C * U * B / T) + (300 + tiles) * U + 2 ** -20 + 32 * U * (z.abs().amax(1) + loss.abs() / T / T)
        out["loss"].append(loss)
        out["eloss"].append(T * T * e * used[:, 0])
        q = lq.exp()
        g = q.clone().scatter_add_(1, lab, -shares[s])
        sc = (T * row_grads[s].double().abs())[:, None] * used
        g = g * T * row_grads[s].double()[:, None] * used
        pad = torch.zeros(q.shape[0], tiles * 256 - V, dtype=q.dtype, device=q.device)
        top = torch.cat((q, pad), 1).view(-1, tiles, 256).amax(2).repeat_interleave(256, 1)[:, :V]
        gerr = RHO * g.abs() + sc * (q * (2 * e[:, None] + 2 ** -10) + 2 ** -23 * top + 4 * U)
        dx = g @ wd
        out["dx"].append(dx)
        out["edx"].append(gerr @ aw + 2 * V * U * (g.abs() @ aw) + RHO * dx.abs() * 1.01)
        out["fx"].append((dx ** 2).sum() + ((g ** 2) @ (wd ** 2)).sum())
        dw += g.T @ xd[s]
        edw += gerr.T @ xd[s].abs() + 2 * N * U * (g.abs().T @ xd[s].abs())
        fw = fw + ((g ** 2).T @ (xd[s] ** 2)).sum()
    res = {k: torch.cat(v) for k, v in out.items() if k != "fx"}
    res.update(dw=dw, edw=edw + RHO * dw.abs() * 1.01, fx=sum(out["fx"]), fw=fw + (dw ** 2).sum())
    return res


def _near(got, want, bound, name):
    got = got.double()
    assert torch.isfinite(got).all(), name
    over = (got - want).abs() - bound
    assert float(over.max()) <= 1e-30, f"{name}: {float(over.max())} beyond the bound"


def _check_grads(dx, dw, r):
    for got, want, bound, norm, name in ((dx, r["dx"], r["edx"], r["fx"], "d x"), (dw, r["dw"], r["edw"], r["fw"], "d weight")):
        if got is not None:
            _near(got, want, bound, name)
            assert float((got.double() - want).norm()) <= 4e-3 * float(norm) ** 0.5 + 1e-30, name


# rows, channels, vocabulary: one of each; tiles of 256 with their edges; several row and vocabulary tiles; odd vocabularies
SHAPES = [(1, 8, 1), (1, 8, 5), (3, 64, 257), (16, 40, 255), (64, 512, 8191), (130, 72, 1000), (256, 64, 256), (257, 264, 511),
          (300, 1032, 3001), (513, 128, 769), (1000, 2048, 777), (33, 2048, 20011), (2000, 64, 300)]


@pytest.mark.parametrize("N,C,V", SHAPES)
def test_cross_entropy(N, C, V):
    import flashrwkv_b200 as F

    x, w, t, gen = _rows(N, C, V, N + C + V)
    if N > 4:
        t[::5] = -100
    used = t != -100
    shares = used.double()[:, None]
    x.requires_grad_(), w.requires_grad_()
    rows = F.pretrain_head_cross_entropy_bf16(x, w, t, reduction="none")
    count = int(used.sum())
    r = _reference(x.detach(), w.detach(), t[:, None], shares, 1.0, torch.full((N,), 1.0 / max(count, 1), device="cuda"))
    _near(rows.detach(), r["loss"], r["eloss"], "row losses")
    assert bool((rows[~used] == 0).all())
    loss = F.pretrain_head_cross_entropy_bf16(x, w, t)
    assert abs(float(loss.detach()) - float(r["loss"].sum() / count)) <= float(r["eloss"].sum() / count) + (N + 4) * U * float(
        r["loss"].sum() / count)
    dx, dw = torch.autograd.grad(loss, (x, w))
    _check_grads(dx, dw, r)
    assert bool((dx[~used] == 0).all())
    # row losses with an upstream gradient per row
    up = torch.randn(N, generator=gen).cuda()
    dx, dw = torch.autograd.grad(rows, (x, w), up)
    _check_grads(dx, dw, _reference(x.detach(), w.detach(), t[:, None], shares, 1.0, up))


def _teacher(N, K, V, gen, missing=True):
    idx = torch.stack([torch.randperm(max(V, K), generator=gen)[:K] % V for _ in range(N)]).cuda()
    logits = (torch.randn(N, K, generator=gen) * 3).cuda()
    if missing and N > 2:
        logits[torch.rand(N, K, generator=gen).cuda() < 0.3] = float("-inf")
        logits[1] = float("-inf")
    return logits, idx


@pytest.mark.parametrize("N,C,V,K,T", [(1, 8, 3, 1, 1.0), (5, 64, 257, 7, 2.0), (33, 512, 8191, 8, 1.0), (130, 72, 1000, 64, 4.0),
                                       (300, 264, 3001, 300, 1.5), (40, 1032, 600, 512, 0.5), (64, 64, 20, 40, 1.0)])
@pytest.mark.parametrize("wide", [False, True])
def test_distill(N, C, V, K, T, wide):
    """K = 40 of 20 names every token twice; K beyond 256 is more than a CTA's threads."""
    import flashrwkv_b200 as F
    from oracle import head_norm_oracle as O

    x, w, _, gen = _rows(N, C, V, N + C + V + K, sure=False)
    logits, idx = _teacher(N, K, V, gen)
    shares, used = O.teacher_shares(logits, T)
    idx = torch.where(logits == float("-inf"), torch.full_like(idx, -7), idx)  # the index of an absent entry is not looked at
    idx = idx if wide else idx.to(torch.int32)
    x.requires_grad_(), w.requires_grad_()
    count = int(used.sum())
    loss = F.pretrain_head_distill_bf16(x, w, logits, idx, temperature=T)
    r = _reference(x.detach(), w.detach(), idx, shares, T, torch.full((N,), 1.0 / count, device="cuda"))
    want = float(r["loss"].sum() / count)
    # the shares' own fp32 error: (K + 8) u of each, times log p - log q, of which a few tens at most
    share_error = T * T * (K + 8) * U * 64
    assert abs(float(loss.detach()) - want) <= float(r["eloss"].sum() / count) + share_error + N * U * abs(want)
    dx, dw = torch.autograd.grad(loss, (x, w))
    _check_grads(dx, dw, r)
    rows = F.pretrain_head_distill_bf16(x, w, logits, idx, temperature=T, reduction="none")
    _near(rows.detach(), r["loss"], r["eloss"] + share_error, "row losses")
    assert bool((rows[~used] == 0).all()) and bool((dx[~used] == 0).all())
    total = F.pretrain_head_distill_bf16(x, w, logits, idx, temperature=T, reduction="sum")
    assert abs(float(total) - float(rows.double().sum())) <= (N + 4) * U * float(rows.double().abs().sum())


def test_distill_from_one_certain_entry_is_cross_entropy():
    import flashrwkv_b200 as F

    x, w, t, _ = _rows(70, 128, 900, 4)
    x.requires_grad_(), w.requires_grad_()
    a = F.pretrain_head_cross_entropy_bf16(x, w, t)
    b = F.pretrain_head_distill_bf16(x, w, torch.zeros(70, 1, device="cuda"), t[:, None])
    for g, h in zip((a, *torch.autograd.grad(a, (x, w))), (b, *torch.autograd.grad(b, (x, w)))):
        assert torch.equal(g, h)


def test_more_rows_than_one_piece_holds():
    """2^20 vocabulary entries leave 512 rows to a piece of the exponentials."""
    import flashrwkv_b200 as F

    N, C, V = 700, 32, 1 << 20
    x, w, t, _ = _rows(N, C, V, 8)
    t[3:60] = -100
    used = t != -100
    x.requires_grad_(), w.requires_grad_()
    loss = F.pretrain_head_cross_entropy_bf16(x, w, t, reduction="sum")
    dx, dw = torch.autograd.grad(loss, (x, w))
    r = _reference(x.detach(), w.detach(), t[:, None], used.double()[:, None], 1.0, torch.ones(N, device="cuda"))
    assert abs(float(loss) - float(r["loss"].sum())) <= float(r["eloss"].sum()) + N * U * float(r["loss"].sum())
    _check_grads(dx, dw, r)


def test_rows_that_take_no_part_reach_nothing():
    """NaN and infinities where no label is; and a batch without any label."""
    import flashrwkv_b200 as F

    x, w, t, _ = _rows(200, 136, 1500, 5)
    t[10:90] = -100
    clean = x.clone()
    x[10:50] = float("nan")
    x[50:90, ::3] = float("inf")
    w.requires_grad_()
    outs = []
    for rows in (x, clean):
        rows = rows.requires_grad_()
        loss = F.pretrain_head_cross_entropy_bf16(rows, w, t)
        outs.append((loss.detach(), *torch.autograd.grad(loss, (rows, w))))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    kept = [r for r in range(200) if not 10 <= r < 90]
    few = clean.detach()[kept].contiguous().requires_grad_()
    loss = F.pretrain_head_cross_entropy_bf16(few, w, t[kept].contiguous())
    dx, dw = torch.autograd.grad(loss, (few, w))
    # the same row losses and products, added in the order of another batch size: N u of the loss, one rounding of a gradient
    assert abs(float(outs[0][0]) - float(loss.detach())) <= 200 * U * float(loss.detach())
    for a, b in ((outs[0][1][kept], dx), (outs[0][2], dw)):
        assert float((a.double() - b.double()).norm()) <= RHO * float(b.double().norm())
    none = torch.full_like(t, -100)
    for reduction in ("mean", "sum"):
        loss = F.pretrain_head_cross_entropy_bf16(x, w, none, reduction=reduction)
        dx, dw = torch.autograd.grad(loss, (x, w))
        assert float(loss) == 0 and bool((dx == 0).all()) and bool((dw == 0).all())
    gone = torch.full((200, 3), float("-inf"), device="cuda")
    loss = F.pretrain_head_distill_bf16(x, w, gone, torch.zeros(200, 3, dtype=torch.int32, device="cuda"))
    dx, dw = torch.autograd.grad(loss, (x, w))
    assert float(loss) == 0 and bool((dx == 0).all()) and bool((dw == 0).all())


def test_labels_outside_the_vocabulary_are_nan_and_stay_in_bounds():
    import flashrwkv_b200 as F

    x, w, t, _ = _rows(40, 64, 300, 6)
    want = F.pretrain_head_cross_entropy_bf16(x, w, t, reduction="none")
    bad = t.clone()
    bad[3], bad[17], bad[30] = 300, -1, 2 ** 40
    x.requires_grad_(), w.requires_grad_()
    rows = F.pretrain_head_cross_entropy_bf16(x, w, bad, reduction="none")
    hit = torch.zeros(40, dtype=torch.bool, device="cuda")
    hit[[3, 17, 30]] = True
    assert torch.isnan(rows[hit]).all() and torch.equal(rows[~hit].detach(), want[~hit])
    loss = F.pretrain_head_cross_entropy_bf16(x, w, bad)
    dx, dw = torch.autograd.grad(loss, (x, w))
    assert torch.isnan(loss) and torch.isnan(dx[hit]).all() and torch.isfinite(dx[~hit]).all() and torch.isnan(dw).all()
    # another ignore_index, negative or a token
    assert float(F.pretrain_head_cross_entropy_bf16(x, w, torch.full_like(t, 7), ignore_index=7)) == 0
    assert torch.isnan(F.pretrain_head_cross_entropy_bf16(x, w, torch.full_like(t, -100), ignore_index=-1))
    # values that are not finite in a row that takes part
    y = x.detach().clone()
    y[5, 2] = float("nan")
    rows = F.pretrain_head_cross_entropy_bf16(y, w, t, reduction="none")
    assert torch.isnan(rows[5]) and torch.equal(torch.cat((rows[:5], rows[6:])), torch.cat((want[:5], want[6:])))


def test_teacher_values_that_are_not_numbers():
    import flashrwkv_b200 as F

    x, w, _, gen = _rows(12, 64, 300, 7)
    logits, idx = _teacher(12, 5, 300, gen, missing=False)
    want = F.pretrain_head_distill_bf16(x, w, logits, idx, reduction="none")
    logits[2, 1] = float("nan")
    logits[4, 0] = float("inf")
    idx[6, 3] = 300
    rows = F.pretrain_head_distill_bf16(x, w, logits, idx, reduction="none")
    hit = torch.zeros(12, dtype=torch.bool, device="cuda")
    hit[[2, 4, 6]] = True
    assert torch.isnan(rows[hit]).all() and torch.equal(rows[~hit], want[~hit])


def test_upstream_gradients_and_repeated_backward_passes():
    """A scalar upstream gradient scales (one more bf16 rounding unless it is a power of two); a second pass over a retained
    graph makes the same gradients again; only what is asked for is made."""
    import flashrwkv_b200 as F

    x, w, t, _ = _rows(90, 136, 700, 9)
    x.requires_grad_(), w.requires_grad_()
    loss = F.pretrain_head_cross_entropy_bf16(x, w, t)
    one = torch.autograd.grad(loss, (x, w), retain_graph=True)
    kept = [g.clone() for g in one]
    again = torch.autograd.grad(loss, (x, w), retain_graph=True)
    quarter = torch.autograd.grad(loss, (x, w), torch.tensor(0.25, device="cuda"))
    for a, b, c, k in zip(one, again, quarter, kept):
        assert torch.equal(a, k) and torch.equal(b, k) and torch.equal(c, 0.25 * k)
    loss = F.pretrain_head_cross_entropy_bf16(x, w, t)
    scaled = torch.autograd.grad(3.0 * loss, (x, w))
    for a, k in zip(scaled, kept):
        assert bool(((a.double() - 3.0 * k.double()).abs() <= RHO * 3.0 * k.double().abs()).all())
    for leaf, want in ((x, kept[0]), (w, kept[1])):
        loss = F.pretrain_head_cross_entropy_bf16(x, w, t)
        assert torch.equal(torch.autograd.grad(loss, leaf)[0], want)
    assert torch.equal(torch.autograd.grad(F.pretrain_head_cross_entropy_bf16(x, w.detach(), t), x)[0], kept[0])
    assert torch.equal(torch.autograd.grad(F.pretrain_head_cross_entropy_bf16(x.detach(), w, t), w)[0], kept[1])
    with torch.no_grad():
        assert not F.pretrain_head_cross_entropy_bf16(x, w, t).requires_grad
    with pytest.raises(RuntimeError, match="not itself differentiable"):
        torch.autograd.grad(F.pretrain_head_cross_entropy_bf16(x, w, t), x, create_graph=True)


def test_same_bits_every_time_on_any_stream_and_in_graphs():
    """Two captured graphs at once, and eager calls between their replays."""
    import flashrwkv_b200 as F

    x, w, t, _ = _rows(300, 264, 2100, 10)
    t[::7] = -100
    x.requires_grad_(), w.requires_grad_()
    up = torch.tensor(2.0, device="cuda")

    def step():
        loss = F.pretrain_head_cross_entropy_bf16(x, w, t)
        return (loss.detach(), *torch.autograd.grad(loss, (x, w), up))

    want = [v.clone() for v in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [v.clone() for v in step()]
    side.synchronize()
    for a, b in zip(want, again):
        assert torch.equal(a, b)
    graphs, held = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(step())
        graphs.append(g)
    for k in (0, 1, 0):
        for v in held[k]:
            v.fill_(5.0)
        graphs[k].replay()
        step()
        torch.cuda.synchronize()
        for a, b in zip(want, held[k]):
            assert torch.equal(a, b)
    with torch.no_grad():  # other labels, other rows that take part
        t.copy_(t.roll(3))
        t[:40] = -100
    graphs[1].replay()
    torch.cuda.synchronize()
    for a, b in zip(step(), held[1]):
        assert torch.equal(a, b)


def test_leading_shape_label_types_and_refusals():
    import flashrwkv_b200 as F

    x, w, t, _ = _rows(60, 64, 300, 11)
    want = F.pretrain_head_cross_entropy_bf16(x, w, t, reduction="none")
    got = F.pretrain_head_cross_entropy_bf16(x.view(3, 20, 64), w, t.view(3, 20).to(torch.int32), reduction="none")
    assert got.shape == (3, 20) and torch.equal(got.flatten(), want)
    half = torch.randn(60, 4, device="cuda").half()
    idx = torch.randint(300, (60, 4), device="cuda")
    assert torch.equal(F.pretrain_head_distill_bf16(x, w, half, idx), F.pretrain_head_distill_bf16(x, w, half.float(), idx))
    shifted = torch.zeros(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view_as(x)
    for args, message in (((shifted, w, t), "16-byte aligned"), ((x.float(), w, t), "bfloat16"), ((x, w.half(), t), "bfloat16"),
                          ((x, w[:, :32].contiguous(), t), "weight must have shape"), ((x[:, ::2], w, t), "contiguous"),
                          ((x, w, t[:5]), "leading shape"), ((x, w, t.float()), "int32 or int64"), ((x, w, t.cpu()), "CUDA"),
                          ((x, w, t.repeat_interleave(2)[::2]), "contiguous"), ((x[:0], w, t[:0]), "non-empty"),
                          ((x, w[:0], t), "weight must have shape"), ((x[:, :4].contiguous(), w[:, :4].contiguous(), t), "multiple of 8")):
        with pytest.raises(ValueError, match=message):
            F.pretrain_head_cross_entropy_bf16(*args)
    logits = torch.randn(60, 4, device="cuda")
    for args, message in (((logits[:5], idx), "leading shape"), ((logits, idx[:, :3].contiguous()), "teacher_logits' shape"),
                          ((logits.double(), idx), "float32, float16 or bfloat16"), ((logits, idx.float()), "int32 or int64"),
                          ((torch.zeros(60, 513, device="cuda"), torch.zeros(60, 513, dtype=torch.int32, device="cuda")), "K from 1 to 512"),
                          ((logits.clone().requires_grad_(), idx), "must not require"), ((logits.t().contiguous().t(), idx), "contiguous")):
        with pytest.raises(ValueError, match=message):
            F.pretrain_head_distill_bf16(x, w, *args)
    for temperature in (0.0, -1.0, float("nan"), float("inf"), 1e-60, True):
        with pytest.raises(ValueError, match="temperature must be positive"):
            F.pretrain_head_distill_bf16(x, w, logits, idx, temperature=temperature)
    with pytest.raises(ValueError, match="reduction"):
        F.pretrain_head_cross_entropy_bf16(x, w, t, reduction="batchmean")


@pytest.mark.parametrize("C", [256, 1024, 2048, 4096])
def test_logits_carry_no_mean_error(C):
    """With one vocabulary entry a row's loss is its logit's error (the normaliser is the tensor core's logit, the label's an
    fp32 dot product).  An accumulator that truncates each of its C / 16 additions loses up to one unit, 2^-23 of a sum that
    is half of the result on average: C / 16 * 2^-24 of the logit at most.  A tenth of that is allowed to the mean over 40000
    logits, which the random part (3e-7 of each) moves by 1.5e-9; the scale itself is an fp32 number, 2^-24."""
    import flashrwkv_b200 as F

    gen = torch.Generator().manual_seed(C)
    w = (torch.randn(1, C, generator=gen) * 2 / C ** 0.5).to(torch.bfloat16).cuda()
    x = torch.randn(40000, C, generator=gen).cuda() + (2 + 6 * torch.rand(40000, 1, generator=gen)).cuda() * w.float()
    x = x.to(torch.bfloat16)
    z = (x.double() @ w.double().T)[:, 0]
    loss = F.pretrain_head_cross_entropy_bf16(x, w, torch.zeros(40000, dtype=torch.int64, device="cuda"), reduction="none")
    big = z.abs() > 6
    assert int(big.sum()) > 20000
    assert abs(float((loss.double() / z)[big].mean())) <= 0.1 * C / 16 * 2.0 ** -24 + 2.0 ** -24


def test_the_end_of_a_training_step():
    """Residual stream -> add + norm -> head loss, as a training step runs them; the gradients reach the residual stream, the
    norm's parameters and the head.  Three bf16 tensors lie between the loss and the residual stream (normalised rows, their
    gradient, the result): each adds at most rho of its value, so 3 rho in the Frobenius norm (and the oracle takes the
    normalised rows as the operator returned them)."""
    import flashrwkv_b200 as F
    from oracle import head_norm_oracle as O

    gen = torch.Generator().manual_seed(12)
    N, C, V = 150, 264, 1300

    def rn(*shape, s=1.0, m=0.0):
        return (torch.randn(*shape, generator=gen) * s + m).to(torch.bfloat16).cuda().requires_grad_()

    x, r, nw, nb, w = rn(2, 75, C), rn(2, 75, C), rn(C, s=0.2, m=1.0), rn(C, s=0.1), rn(V, C, s=2 / C ** 0.5)
    t = torch.randint(V, (2, 75), generator=gen).cuda()
    t[0, :20] = -100
    total, rows = F.pretrain_tmix_add_layer_norm_bf16(x, r, nw, nb)
    ce = F.pretrain_head_cross_entropy_bf16(rows, w, t)
    logits, idx = _teacher(N, 16, V, gen)
    kd = F.pretrain_head_distill_bf16(rows, w, logits.view(2, 75, 16), idx.view(2, 75, 16), temperature=2.0)
    got = torch.autograd.grad(ce + 0.5 * kd, (x, r, nw, nb, w))
    flat, used = rows.detach().view(N, C), (t.flatten() != -100)
    d1, w1 = O.head_backward(used / used.sum(), flat, w.detach(), t.view(N, 1), used.double()[:, None])
    shares, there = O.teacher_shares(logits, 2.0)
    d2, w2 = O.head_backward(0.5 * there / there.sum(), flat, w.detach(), idx, shares, 2.0)
    ds, dnw, dnb = O.layer_norm_backward((d1 + d2).view(2, 75, C), total.detach(), nw.detach(), 1e-5)
    for g, want, name in zip(got, (ds, ds, dnw, dnb, w1 + w2), ("x", "residual", "norm weight", "norm bias", "head")):
        assert float((g.double() - want).norm()) <= 3 * RHO * float(want.norm()), name


def _plain_rows(x, w, t):
    z = x.double() @ w.double().T
    return torch.logsumexp(z, 1) - z.gather(1, t[:, None])[:, 0], torch.softmax(z, 1)


def test_offsets_beyond_32_bits_in_the_weight():
    """2^20 x 2056 weights are 2.16e9 values; the last vocabulary rows are labels.  The row sum of exponentials takes 8192
    entries.  Bounds as above, with B_n from the rows themselves."""
    import flashrwkv_b200 as F

    N, C, V = 12, 2056, 1 << 20
    gen = torch.Generator(device="cuda").manual_seed(1)
    w = torch.empty(V, C, dtype=torch.bfloat16, device="cuda").normal_(0, 2 / C ** 0.5, generator=gen)
    x = torch.randn(N, C, generator=gen, device="cuda").to(torch.bfloat16)
    t = torch.arange(V - N, V, device="cuda")
    x.requires_grad_(), w.requires_grad_()
    rows = F.pretrain_head_cross_entropy_bf16(x, w, t, reduction="none")
    loss = F.pretrain_head_cross_entropy_bf16(x, w, t, reduction="sum")
    dx, dw = torch.autograd.grad(loss, (x, w))
    z = torch.cat([x.detach().double() @ part.double().T for part in w.detach().split(1 << 16)], 1)
    want = torch.logsumexp(z, 1) - z.gather(1, t[:, None])[:, 0]
    B = torch.stack([(x.detach().double().abs() @ part.double().abs().T).amax(1) for part in w.detach().split(1 << 16)]).amax(0)
    bound = 2 * (2 * C * U * B) + 9000 * U + 2 ** -20 + 32 * U * (z.abs().amax(1) + want)
    _near(rows.detach(), want, bound, "row losses")
    g = torch.softmax(z, 1)
    g[torch.arange(N), t] -= 1
    want_dx = sum(p @ q.double() for p, q in zip(g.split(1 << 16, 1), w.detach().split(1 << 16)))
    assert float((dx.double() - want_dx).norm()) <= 4e-3 * 2 ** 0.5 * float(want_dx.norm())
    for s in (slice(0, 300), slice(V - 300, V)):
        want_dw = g[:, s].T @ x.detach().double()
        assert float((dw[s].double() - want_dw).norm()) <= 4e-3 * 2 ** 0.5 * float(want_dw.norm())


def test_offsets_beyond_32_bits_in_the_rows():
    import flashrwkv_b200 as F

    N, C, V = (1 << 20) + 1003, 2056, 300
    gen = torch.Generator(device="cuda").manual_seed(2)
    w = torch.empty(V, C, dtype=torch.bfloat16, device="cuda").normal_(0, 2 / C ** 0.5, generator=gen)
    x = torch.empty(N, C, dtype=torch.bfloat16, device="cuda").normal_(generator=gen)
    t = torch.randint(V, (N,), generator=gen, device="cuda")
    t[5:900] = -100  # the rows that take part move, the last too
    x.requires_grad_()
    rows = F.pretrain_head_cross_entropy_bf16(x, w, t, reduction="none")
    up = torch.zeros_like(rows)
    up[-700:] = 1
    dx = torch.autograd.grad(rows, x, up)[0]
    last = slice(N - 700, N)
    want, q = _plain_rows(x.detach()[last], w, t[last])
    assert float((rows.detach()[last].double() - want).abs().max()) <= 2 * 2 * C * U * float(
        (x.detach()[last].double().abs() @ w.double().abs().T).max()) + 2 ** -19
    q[torch.arange(700), t[last]] -= 1
    want_dx = q @ w.double()
    assert float((dx[last].double() - want_dx).norm()) <= 4e-3 * 2 ** 0.5 * float(want_dx.norm())
    assert bool((dx[:-700] == 0).all()) and bool((rows[5:900] == 0).all())


def test_inference_mode_and_another_current_stream():
    """Called from a stream of its own right behind the kernels that make its inputs there; and without autograd."""
    import flashrwkv_b200 as F

    x, w, t, _ = _rows(300, 264, 2100, 13)
    want = F.pretrain_head_cross_entropy_bf16(x, w, t)
    with torch.inference_mode():
        assert torch.equal(F.pretrain_head_cross_entropy_bf16(x, w, t), want)
        total, out = F.pretrain_tmix_add_layer_norm_bf16(x, x, w[0], w[1])
        assert out.shape == x.shape
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        y = (x.float() * 2).to(torch.bfloat16).requires_grad_()
        loss = F.pretrain_head_cross_entropy_bf16(y, w, t)
        grad = torch.autograd.grad(loss, y)[0]
    side.synchronize()
    z = (x.float() * 2).to(torch.bfloat16).requires_grad_()
    again = F.pretrain_head_cross_entropy_bf16(z, w, t)
    assert torch.equal(again, loss) and torch.equal(torch.autograd.grad(again, z)[0], grad)


def test_two_calls_at_once_on_two_streams():
    import flashrwkv_b200 as F

    cases = []
    for k, shape in enumerate(((700, 264, 9000), (40, 512, 30000))):
        x, w, t, _ = _rows(*shape, 20 + k)
        x.requires_grad_(), w.requires_grad_()
        loss = F.pretrain_head_cross_entropy_bf16(x, w, t)
        cases.append((x, w, t, [loss.detach(), *torch.autograd.grad(loss, (x, w))], torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for x, w, t, _, stream in cases:
            with torch.cuda.stream(stream):
                loss = F.pretrain_head_cross_entropy_bf16(x, w, t)
                got.append([loss.detach(), *torch.autograd.grad(loss, (x, w))])
        torch.cuda.synchronize()
        for (_, _, _, want, _), have in zip(cases, got):
            for a, b in zip(want, have):
                assert torch.equal(a, b)


def test_losses_accumulate_over_micro_batches_into_one_weight():
    """Two losses alive at once over the same weight, run backward together: the leaves receive the sum of their gradients."""
    import flashrwkv_b200 as F

    x1, w, t1, _ = _rows(70, 72, 600, 30)
    x2, _, t2, _ = _rows(90, 72, 600, 31)
    for v in (x1, x2, w):
        v.requires_grad_()
    a, b = F.pretrain_head_cross_entropy_bf16(x1, w, t1), F.pretrain_head_cross_entropy_bf16(x2, w, t2)
    ((a + b) * 0.5).backward()
    g1 = torch.autograd.grad(F.pretrain_head_cross_entropy_bf16(x1, w, t1), (x1, w), torch.tensor(0.5, device="cuda"))
    g2 = torch.autograd.grad(F.pretrain_head_cross_entropy_bf16(x2, w, t2), (x2, w), torch.tensor(0.5, device="cuda"))
    assert torch.equal(x1.grad, g1[0]) and torch.equal(x2.grad, g2[0]) and torch.equal(w.grad, g1[1] + g2[1])
    # the same row taken from a leaf that is used in place afterwards is refused, as by any operator that needs it again
    loss = F.pretrain_head_cross_entropy_bf16(x1, w, t1)
    with torch.no_grad():
        x1.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("N,C,V", [(40, 64, 300), (25, 1032, 5000), (1, 256, 129), (6, 2048, 900)])
@pytest.mark.parametrize("teacher", [False, True])
def test_rows_that_are_nearly_certain(N, C, V, teacher):
    """Losses from ordinary to 1e-20 keep their relative precision, and so do the gradients of each row by itself: with d the
    distance of the others' log sum from the label's logit the loss is log(1 + e^d), whose relative error is at most d's
    error, e_n above; g then has that relative error and its one rounding.  A teacher that is nearly certain as well (its
    second entry between 1e-9 and 1e-1 of the first) has a loss that is a difference of two such terms, each with a relative
    error of e_n + 16 u."""
    import flashrwkv_b200 as F
    from oracle import head_norm_oracle as O

    gen = torch.Generator().manual_seed(N + C)
    w = (torch.randn(V, C, generator=gen) * 2 / C ** 0.5).to(torch.bfloat16).cuda()
    t = torch.randint(V, (N,), generator=gen).cuda()
    sure = torch.linspace(0, 14, N)[:, None].cuda() if N > 1 else torch.tensor([[7.0]], device="cuda")
    x = (torch.randn(N, C, generator=gen).cuda() * 0.5 + sure * w[t].float()).to(torch.bfloat16)
    x.requires_grad_(), w.requires_grad_()
    if teacher:
        idx = torch.stack((t, (t + 1) % V), 1)
        gap = torch.logspace(-9, -1, N).log().cuda() if N > 1 else torch.tensor([-8.0], device="cuda")
        logits = torch.stack((torch.zeros(N, device="cuda"), gap), 1)
        shares, _ = O.teacher_shares(logits, 1.0)
        rows = F.pretrain_head_distill_bf16(x, w, logits, idx, reduction="none")
    else:
        idx, shares = t[:, None], torch.ones(N, 1, dtype=torch.float64, device="cuda")
        rows = F.pretrain_head_cross_entropy_bf16(x, w, t, reduction="none")
    z = x.detach().double() @ w.detach().double().T
    B = (x.detach().double().abs() @ w.detach().double().abs().T).amax(1)
    e = 2 * (2 * C * U * B) + (300 + V // 128 + 1) * U + 2 ** -20 + 32 * U * z.abs().amax(1)
    others = z.clone()
    others[torch.arange(N), t] = float("-inf")
    d = torch.logsumexp(others, 1) - z[torch.arange(N), t]
    excess = torch.nn.functional.softplus(d)
    if teacher:
        p2 = shares[:, 1]
        second = z[torch.arange(N), idx[:, 1]] - z[torch.arange(N), t]
        want = excess - torch.log1p(torch.exp(gap.double())) + p2 * (gap.double() - second)
        bound = (e + 16 * U) * (excess + torch.exp(gap.double())) + p2 * (e + 16 * U) * (1 + gap.double().abs() + second.abs())
    else:
        want, bound = excess, e * excess
    assert teacher or N == 1 or (float(want.min()) < 1e-6 and float(want.max()) > 1)
    _near(rows.detach(), want, bound + 2.0 ** -140, "row losses")
    # each row's gradient by itself
    g = torch.exp(z - z[torch.arange(N), t][:, None] - excess[:, None])
    missing = torch.sigmoid(d)
    if teacher:
        g[torch.arange(N), idx[:, 1]] -= p2
        g[torch.arange(N), t] = p2 - missing
    else:
        g[torch.arange(N), t] = -missing
    dx = torch.autograd.grad(rows.sum(), x)[0].double()
    want_dx = g @ w.detach().double()
    scale = ((g ** 2) @ (w.detach().double() ** 2)).sum(1) + (want_dx ** 2).sum(1)
    if teacher:  # q - p of an entry is a difference too
        slack = 2 * (e + 16 * U) * (missing + p2) * w.detach().double().norm(dim=1).amax() * 2
    else:
        slack = 2 * e * scale.sqrt()
    assert bool(((dx - want_dx).norm(dim=1) <= 4e-3 * scale.sqrt() + slack).all())


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_a_captured_backward_pass_of_a_call_made_before_may_be_replayed(reduction):
    """The gradients that the loss left behind are used up by one pass; every replay has to make them again."""
    import flashrwkv_b200 as F

    x, w, t, _ = _rows(300, 264, 2100, 21)
    t[::7] = -100
    x.requires_grad_(), w.requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        up = torch.full((300,) if reduction == "none" else (), 2.0, device="cuda")
        loss = F.pretrain_head_cross_entropy_bf16(x, w, t, reduction=reduction)
        again = F.pretrain_head_cross_entropy_bf16(x, w, t, reduction=reduction)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        held = torch.autograd.grad(loss, (x, w), up, retain_graph=True)
    for scale in (2.0, 2.0, 0.5):
        with torch.cuda.stream(side):
            up.fill_(scale)
            g.replay()
            want = torch.autograd.grad(again, (x, w), up, retain_graph=True)
        side.synchronize()
        for a, b in zip(held, want):
            assert torch.allclose(a.float(), b.float(), rtol=2**-6, atol=2**-7 * float(b.abs().max()))


def test_a_captured_backward_pass_beside_an_eager_graph_of_the_same_leaves():
    """Refused where that graph was made on the default stream; made on another stream it is no hindrance."""
    import flashrwkv_b200 as F

    def leaves():
        x, w, t, _ = _rows(40, 128, 500, 22)
        return x.requires_grad_(), w.requires_grad_(), t

    x, w, t = leaves()
    alive = F.pretrain_head_cross_entropy_bf16(x, w, t)
    with pytest.raises(RuntimeError, match="default stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            F.pretrain_head_cross_entropy_bf16(x, w, t).backward()
    torch.cuda.synchronize()
    alive.backward()
    want = [x.grad, w.grad]

    x, w, t = leaves()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = F.pretrain_head_cross_entropy_bf16(x, w, t)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        F.pretrain_head_cross_entropy_bf16(x, w, t).backward()
    g.replay()
    torch.cuda.synchronize()
    for a, b in zip((x.grad, w.grad), want):
        assert torch.equal(a, b)
    del alive


def test_an_eager_backward_pass_behind_a_captured_forward_pass_beside_an_eager_graph():
    """Only a captured backward pass cannot reach leaves of the default stream; this one makes the gradients anew."""
    import flashrwkv_b200 as F

    x, w, t, _ = _rows(40, 128, 500, 23)
    x.requires_grad_(), w.requires_grad_()
    alive = F.pretrain_head_cross_entropy_bf16(x, w, t)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        loss = F.pretrain_head_cross_entropy_bf16(x, w, t)
    g.replay()
    torch.cuda.synchronize()
    got = torch.autograd.grad(loss, (x, w))
    for a, b in zip((loss, *got), (alive, *torch.autograd.grad(alive, (x, w)))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_a_backward_pass_captured_apart_beside_an_eager_graph_of_the_same_leaves(reduction):
    """The forward pass ran eagerly, on a stream that may be captured; the leaves belong to the default stream all the same."""
    import flashrwkv_b200 as F

    x, w, t, _ = _rows(40, 128, 500, 24)
    x.requires_grad_(), w.requires_grad_()
    alive = F.pretrain_head_cross_entropy_bf16(x, w, t, reduction=reduction)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        up = torch.full_like(alive.detach(), 0.5)
        loss = F.pretrain_head_cross_entropy_bf16(x, w, t, reduction=reduction)
    side.synchronize()
    for leaves in ((x, w), (x,), (w,)):
        with pytest.raises(RuntimeError, match="default stream"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                torch.autograd.grad(loss, leaves, up, retain_graph=True)
        torch.cuda.synchronize()
    want = torch.autograd.grad(alive, (x, w), up)
    with torch.cuda.stream(side):
        got = torch.autograd.grad(loss, (x, w), up)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("teacher", [False, True])
@pytest.mark.parametrize("N", [1, 9000, (1 << 20) + 77])
def test_the_scalar_loss_of_many_like_rows(N, teacher):
    """Row losses that are all the same round the same way in every addition of a binade.  Their sum and their mean are each
    rounded once, to half a step (2^-24); the sum of doubles that they are compared with is off by N 2^-53 at most."""
    import flashrwkv_b200 as F

    gen = torch.Generator().manual_seed(N)
    w = torch.randn(3, 8, generator=gen).to(torch.bfloat16).cuda()
    x = torch.randn(1, 8, generator=gen).to(torch.bfloat16).cuda().expand(N, 8).contiguous()
    t = torch.full((N, 1), 2, device="cuda")
    t[N // 2] = 0  # and one that differs

    def call(reduction):
        if teacher:
            return F.pretrain_head_distill_bf16(x, w, torch.zeros(N, 1, device="cuda"), t, reduction=reduction)
        return F.pretrain_head_cross_entropy_bf16(x, w, t[:, 0], reduction=reduction)

    total = float(call("none").double().sum())
    bound = (U + N * 2.0 ** -52) * total
    assert abs(float(call("sum")) - total) <= bound
    assert abs(float(call("mean")) - total / N) <= bound / N


def _growing_row(kind, N, C, gen):
    """Rows x [N,C] and a vector w [C] whose dot products lie between 12 and 31 and gather their magnitude in one way each."""
    def uniform(*shape, low=0.1, high=1.1):
        return low + (high - low) * torch.rand(*shape, generator=gen)

    w = uniform(C, low=0.5, high=1.5)
    if kind == "exact":  # whole numbers times one power of two: every sum of fewer than 2^24 units is exact
        x = torch.randint(1, 128, (N, C), generator=gen).float()
        return (x * 2.0 ** -int(torch.log2(x.sum(1).max() / 30).ceil())).to(torch.bfloat16), torch.ones(C, dtype=torch.bfloat16)
    if kind == "even":
        x = uniform(N, C)
    elif kind == "sparse":
        x = torch.zeros(N, C)
        x.scatter_(1, torch.stack([torch.randperm(C, generator=gen)[:5] for _ in range(N)]), uniform(N, 5))
    elif kind == "random":
        w = torch.randn(C, generator=gen) * 2 / C ** 0.5
        x = torch.randn(N, C, generator=gen) + 6 * w
    else:
        x = 1e-4 * uniform(N, C)
        x[:, slice(0, 16) if kind == "first" else slice(C - 16, C)] = uniform(N, 16)
    x = x * (22 / (x @ w)[:, None])
    return x.to(torch.bfloat16), w.to(torch.bfloat16)


@pytest.mark.parametrize("N", [100, 300])
@pytest.mark.parametrize("kind", ["exact", "even", "first", "last", "sparse", "random"])
@pytest.mark.parametrize("C", [128, 1024, 1032, 2056, 4096, 16384, 65536])
def test_a_logit_however_its_sum_grows(C, kind, N):
    """The label's logit is 0 and the only other one z, so a row's loss is log(1 + e^z).  An accumulator takes 1024 channels at
    most; it loses up to one unit (2 u of the sum of magnitudes so far, B at the end) per product, and its parts are added with
    a rounding of u B each.  Scaling to powers of two, back to natural units and the last addition are six roundings, of the
    numbers that they are done with included: 6 u z.  The scale gives back what random rows lose, 1.03e-9 per channel of an
    accumulator, to rows that lost nothing too: with the roundings that is all that an exact sum may be off by."""
    import flashrwkv_b200 as F

    x, w = _growing_row(kind, N, C, torch.Generator().manual_seed(C))
    x, w = x.cuda(), torch.stack((torch.zeros_like(w), w)).cuda()
    z, B = x.double() @ w[1].double(), x.double().abs() @ w[1].double().abs()
    assert 12 < float(z.min()) and float(z.max()) < 31
    loss = F.pretrain_head_cross_entropy_bf16(x, w, torch.zeros(N, dtype=torch.int64, device="cuda"), reduction="none")
    parts = -(-C // 1024)
    sums = 0 if kind == "exact" else (2 * min(C, 1024 + 64) + parts) * U * B
    _near(loss, torch.nn.functional.softplus(z, threshold=100), sums + (6 * U + 1.03e-9 * C / parts) * z, "row losses")


@pytest.mark.parametrize("C", [256, 1024, 2048, 4096, 8200])
def test_logits_of_random_rows_carry_no_mean_error(C):
    """As above, the label's logit 0 and the other's z, so that a row's loss is z + log(1 + e^-z).  An accumulator of P channels
    that truncates each of its P / 16 additions loses up to one unit, 2^-23 of a sum that is half of the result on average: P /
    16 * 2^-24 of the logit.  A tenth of that is allowed to the mean over 30000 logits; the scale itself is an fp32 number,
    2^-24."""
    import flashrwkv_b200 as F

    gen = torch.Generator().manual_seed(C)
    w = torch.randn(C, generator=gen) * 2 / C ** 0.5
    x = (torch.randn(30000, C, generator=gen) + (4 + 4 * torch.rand(30000, 1, generator=gen)) * w).to(torch.bfloat16).cuda()
    w = torch.stack((torch.zeros(C), w)).to(torch.bfloat16).cuda()
    z = x.double() @ w[1].double()
    loss = F.pretrain_head_cross_entropy_bf16(x, w, torch.zeros(30000, dtype=torch.int64, device="cuda"), reduction="none")
    big = z > 8
    assert int(big.sum()) > 25000
    off = (loss.double() - torch.nn.functional.softplus(z, threshold=100)) / z
    P = C / -(-C // 1024)
    assert abs(float(off[big].mean())) <= 0.1 * P / 16 * 2.0 ** -24 + 2.0 ** -24


@pytest.mark.parametrize("N,C,V", [(300, 2056, 2100), (140, 4104, 700), (20, 4104, 3001), (128, 8200, 300)])
def test_logits_of_several_parts(N, C, V):
    """Odd and even numbers of accumulators to a logit, tiles that follow one another in each, with the gradients behind them."""
    import flashrwkv_b200 as F

    x, w, t, _ = _rows(N, C, V, N + C + V)
    t[::5] = -100
    used = t != -100
    x.requires_grad_(), w.requires_grad_()
    loss = F.pretrain_head_cross_entropy_bf16(x, w, t, reduction="sum")
    r = _reference(x.detach(), w.detach(), t[:, None], used.double()[:, None], 1.0, torch.ones(N, device="cuda"))
    assert abs(float(loss.detach()) - float(r["loss"].sum())) <= float(r["eloss"].sum()) + U * float(r["loss"].sum())
    _check_grads(*torch.autograd.grad(loss, (x, w)), r)


@pytest.mark.parametrize("N,C,V", [(9472, 512, 20011), (100, 37888, 8200)])
def test_gradients_of_several_parts(N, C, V):
    """As many tiles of dx as run at once, so that a tile's contraction over the vocabulary is not cut between pairs (or single
    CTAs) and takes several accumulators; 9472 rows are several of dW's as well."""
    import flashrwkv_b200 as F

    x, w, t, _ = _rows(N, C, V, N + C + V)
    t[::5] = -100
    t[5 * N // 6:] = t.clamp_min(0)[5 * N // 6:]
    used = t != -100
    x.requires_grad_(), w.requires_grad_()
    loss = F.pretrain_head_cross_entropy_bf16(x, w, t, reduction="sum")
    got = torch.autograd.grad(loss, (x, w))
    r = _reference(x.detach(), w.detach(), t[:, None], used.double()[:, None], 1.0, torch.ones(N, device="cuda"))
    assert abs(float(loss.detach()) - float(r["loss"].sum())) <= float(r["eloss"].sum()) + U * float(r["loss"].sum())
    _check_grads(*got, r)


def test_a_weight_gradient_of_many_rows_whose_large_terms_come_first():
    """A label whose logit lies 40 below the others has the logit gradient -up exactly, here a power of two: dW[label] is a sum
    of exact products, of one sign.  An accumulator takes 4096 of them at most and loses up to one unit (2 u of the sum) per
    product, the 32 parts are added with u each.  The roundings of the results to bf16 are independent: in the mean over 9472
    columns they stay below five deviations, 5 rho / sqrt(3 * 9472)."""
    import flashrwkv_b200 as F

    N, C, V = 131072, 9472, 512  # 2 x 37 tiles: none of them is cut between pairs
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = (0.5 + torch.rand(N, C, generator=gen, device="cuda", dtype=torch.float32)).to(torch.bfloat16)
    w = torch.zeros(V, C, device="cuda", dtype=torch.bfloat16)
    w[0] = -(2.0 ** -8)
    w.requires_grad_()
    up = torch.full((N,), 2.0 ** -14, device="cuda")
    up[:64] = 1.0
    rows = F.pretrain_head_cross_entropy_bf16(x, w, torch.zeros(N, dtype=torch.int32, device="cuda"), reduction="none")
    got = torch.autograd.grad(rows, w, up)[0][0].double()
    want = -sum(u.double() @ p.double() for u, p in zip(up.split(8192), x.split(8192)))
    off = float(((got - want) / want).mean())
    assert abs(off) <= 2 * 4096 * U + 32 * U + 5 * RHO / (3 * C) ** 0.5, off


@pytest.mark.parametrize("T", [0.25, 0.7, 3.0])
def test_teacher_logits_far_from_zero(T):
    """A softmax knows no offset: with logits that are multiples of 2^-6 below 16 an offset of 2^14 is exact in fp32, so that
    every result keeps its bits.  Entries of the type's lowest value are entries: beside others they have no share, and among
    themselves equal ones."""
    import flashrwkv_b200 as F
    from oracle import head_norm_oracle as O

    x, w, _, gen = _rows(40, 64, 300, 41)
    logits, idx = _teacher(40, 9, 300, gen, missing=False)
    logits = (logits.clamp(-15, 15) * 64).round() / 64
    logits[3, 2:] = float("-inf")
    x.requires_grad_(), w.requires_grad_()

    def call(logits):
        loss = F.pretrain_head_distill_bf16(x, w, logits, idx, temperature=T)
        return (loss.detach(), *torch.autograd.grad(loss, (x, w)))

    want = call(logits)
    for offset in (2.0 ** 14, -(2.0 ** 14)):
        for a, b in zip(call(logits + offset), want):
            assert torch.equal(a, b)
    # An entry without a share has its logit gradient from fp32, where the column of an absent one has it from an fp16
    # exponential: 2^-11 between them may round to the other bf16 neighbour, so the gradients go by the oracle's bounds.
    count = torch.full((40,), 1 / 40, device="cuda")
    for lowest in (torch.finfo(torch.float32).min, torch.finfo(torch.bfloat16).min):
        low, gone = logits.clone(), logits.clone()
        low[5, 1:], gone[5, 1:] = lowest, float("-inf")
        low[7], gone[7] = lowest, 0.0
        loss, dx, dw = call(low)
        assert torch.equal(loss, call(gone)[0])
        _check_grads(dx, dw, _reference(x.detach(), w.detach(), idx, O.teacher_shares(low, T)[0], T, count))


@pytest.mark.parametrize("N,C,V", [(2047, 64, 6000), (2048, 64, 6000), (65, 40, 4096), (65, 40, 4097), (64, 40, 4096)])
def test_rows_finished_by_warps_and_by_ctas(N, C, V):
    """Both sides of each edge of the rule that gives a row to a warp or to a CTA."""
    import flashrwkv_b200 as F

    x, w, t, _ = _rows(N, C, V, N + C + V)
    t[::6] = -100
    used = t != -100
    x.requires_grad_(), w.requires_grad_()
    loss = F.pretrain_head_cross_entropy_bf16(x, w, t, reduction="sum")
    got = torch.autograd.grad(loss, (x, w))
    r = _reference(x.detach(), w.detach(), t[:, None], used.double()[:, None], 1.0, torch.ones(N, device="cuda"))
    assert abs(float(loss.detach()) - float(r["loss"].sum())) <= float(r["eloss"].sum()) + U * float(r["loss"].sum())
    _check_grads(*got, r)


@pytest.mark.parametrize("teacher", [False, True])
@pytest.mark.parametrize("N", [100, 255])
def test_the_rounding_of_a_mean_is_no_error_that_rows_share(N, teacher):
    """1 / 255 lies in the middle between two bf16 values: as a factor of the logit gradients it would put all of them off by
    2^-8 with one sign.  Labels 40 below the other logits have the gradient -1 / N exactly; dW[label] sums N products, 2 N u
    for any order, and its roundings to bf16 are independent: in the mean over 2048 columns five deviations, 5 rho /
    sqrt(3 * 2048).  Factors and T are a few roundings of u."""
    import flashrwkv_b200 as F

    C, V, T = 2048, 300, 1.0 if not teacher else 1.7
    gen = torch.Generator(device="cuda").manual_seed(N)
    x = (0.5 + torch.rand(N, C, generator=gen, device="cuda")).to(torch.bfloat16)
    w = torch.zeros(V, C, device="cuda", dtype=torch.bfloat16)
    w[7] = -(2.0 ** -5)
    w.requires_grad_()
    label = torch.full((N, 1), 7, device="cuda")
    if teacher:
        loss = F.pretrain_head_distill_bf16(x, w, torch.zeros(N, 1, device="cuda"), label, temperature=T)
    else:
        loss = F.pretrain_head_cross_entropy_bf16(x, w, label[:, 0])
    for up in (1.0, 0.3):
        again = torch.autograd.grad(loss, w, torch.tensor(up, device="cuda"), retain_graph=True)[0][7].double()
        want = -x.double().sum(0) * T * float(torch.tensor(up)) / N
        off = float(((again - want) / want).mean())
        # the first pass scales gradients that are rounded already: a second rounding unless the scale is 1
        assert abs(off) <= (2 * N + 8) * U + 5 * RHO / (3 * C) ** 0.5 * (1 if up == 1.0 else 2 ** 0.5), (up, off)


@pytest.mark.parametrize("N", [64, 255, 9001])
def test_upstream_gradients_that_all_rows_share_are_no_shared_error(N):
    """The mean of row losses taken outside: 1 / rows arrives as every row's upstream gradient.  Labels 40 below the other
    logits, bounds as above; rows without a label do not count, whatever arrives there."""
    import flashrwkv_b200 as F

    C, V = 2048, 300
    gen = torch.Generator(device="cuda").manual_seed(N)
    x = (0.5 + torch.rand(N, C, generator=gen, device="cuda")).to(torch.bfloat16)
    w = torch.zeros(V, C, device="cuda", dtype=torch.bfloat16)
    w[7] = -(2.0 ** -5)
    w.requires_grad_()
    t = torch.full((N,), 7, device="cuda")
    t[3::9] = -100
    used = t != -100
    rows = F.pretrain_head_cross_entropy_bf16(x, w, t, reduction="none")
    for up in (1 / 255, -3e-30, 1.7e30):
        ups = torch.where(used, torch.full((N,), up, device="cuda"), torch.full((N,), float("inf"), device="cuda"))
        got = torch.autograd.grad(rows, w, ups, retain_graph=True)[0][7].double()
        want = -x[used].double().sum(0) * float(ups[0])
        off = float(((got - want) / want).mean())
        assert abs(off) <= (2 * N + 8) * U + 5 * RHO / (3 * C) ** 0.5, (up, off)


def test_upstream_gradients_that_are_not_finite_or_zero():
    """They spoil their own rows and the weight's gradient; no other row's."""
    import flashrwkv_b200 as F

    x, w, t, gen = _rows(50, 64, 300, 50)
    x.requires_grad_(), w.requires_grad_()
    rows = F.pretrain_head_cross_entropy_bf16(x, w, t, reduction="none")
    up = torch.rand(50, generator=gen).cuda()
    want = torch.autograd.grad(rows, (x, w), up, retain_graph=True)
    bad = up.clone()
    bad[4], bad[9] = float("nan"), float("inf")
    dx, dw = torch.autograd.grad(rows, (x, w), bad, retain_graph=True)
    hit = torch.zeros(50, dtype=torch.bool, device="cuda")
    hit[[4, 9]] = True
    if float(up[hit].max()) < float(up[~hit].max()):  # the scale is another row's
        assert torch.equal(dx[~hit], want[0][~hit])
    assert torch.isfinite(dx[~hit]).all() and not torch.isfinite(dx[hit]).all() and not torch.isfinite(dw).any()
    for zero in (torch.zeros(50, device="cuda"), -torch.zeros(50, device="cuda")):
        for g in torch.autograd.grad(rows, (x, w), zero, retain_graph=True):
            assert bool((g == 0).all())
    one = torch.zeros(50, device="cuda")
    one[11] = 2.0
    dx, dw = torch.autograd.grad(rows, (x, w), one, retain_graph=True)
    few = x.detach()[11:12].clone().requires_grad_()
    fx, fw = torch.autograd.grad(F.pretrain_head_cross_entropy_bf16(few, w, t[11:12], reduction="none"), (few, w),
                                 torch.tensor([2.0], device="cuda"))
    assert float((dx[11].double() - fx[0].double()).norm()) <= RHO * float(fx.double().norm()) and bool((dx[:11] == 0).all())
    assert float((dw.double() - fw.double()).norm()) <= RHO * float(fw.double().norm())
