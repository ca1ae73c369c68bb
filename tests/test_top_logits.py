"""ops.top_logits and ops.soft_cross_entropy_top against their definitions in 64 bits.

Selection is compared exactly.  Tolerances of the rest count f32 roundings (F = 2^-24; exp and log are good to a few of them, an
exponent's own rounding enters as its size times F), e being the size of the numbers whose difference is formed:
  lse        16 F (1 + |lse| + max |logits / T|)
  log p, log q, their difference   8 F e, e = |z| + |norm| + |y| + |lse| + 1
  p_rest = 1 - exp(lz - norm)      d = 8 F (|lz| + |norm| + 1), where lz is the log-sum-exp of the kept z
  L          sum_j p_j 16 F e_j (1 + |log p_j - log q_j|) + d (2 + |log p_rest - log q_rest|) + 16 F p_rest e_rest
  gradient   u |g| (storage) + factor * (16 F e q (M + p_rest / q_rest) + 16 F e p + d exp(y - lse_rest)) per class
"""
import math

import pytest
import torch

from efficientvlm_amd import ops

BF16, F32 = torch.bfloat16, torch.float32
F = 2.0 ** -24


def rows(R, C, dtype, seed=0, spread=3.0, layout="padded"):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(R, C, generator=g) * spread).to(dtype)
    width = {"padded": (C + 7) // 8 * 8, "plain": C, "shifted": C + 3}[layout]
    buf = torch.zeros(R, width, dtype=dtype, device="cuda")
    view = buf[:, 3:] if layout == "shifted" else buf[:, :C]
    view.copy_(x)
    return view


def want_top(x, k, T):
    x = x.double().cpu()
    nan_high = torch.where(x.isnan(), torch.full_like(x, math.inf), x)
    # NaN above +inf: sort the pairs (is NaN, value), both stable
    order = torch.sort(nan_high, dim=1, descending=True, stable=True).indices
    isnan = x.gather(1, order).isnan()
    order = order.gather(1, torch.sort(isnan.int(), dim=1, descending=True, stable=True).indices)[:, :k]
    return x.gather(1, order), order, torch.logsumexp(x / T, 1)


def check_top(x, k, T=1.0):
    values, classes, lse = ops.top_logits(x, k, temperature=T)
    v, c, l = want_top(x, k, T)
    assert values.dtype == F32 and classes.dtype == torch.int32 and lse.dtype == F32
    assert torch.equal(classes.long().cpu(), c)
    a, b = values.double().cpu(), v
    assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(0.5), b.nan_to_num(0.5))
    got = lse.double().cpu()
    for g, w, r in zip(got, l, x.double().cpu()):
        if math.isfinite(w):
            assert abs(g - w) <= 16 * F * (1 + abs(w) + r[r.isfinite()].abs().max() / T)
        else:
            assert (math.isnan(g) and math.isnan(w)) or g == w


# ---- refusals (no GPU) ------------------------------------------------------------------------------
def test_refusals():
    x = torch.zeros(3, 10)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.top_logits(x, 2)
    for k in (0, 11, 257, -1):
        with pytest.raises(RuntimeError, match="k ="):
            ops.top_logits(x, k)
    with pytest.raises(RuntimeError, match="k ="):
        ops.top_logits(torch.zeros(3, 300), 257)
    for T in (0.0, -1.0, math.nan, math.inf):
        with pytest.raises(RuntimeError, match="temperature"):
            ops.top_logits(x, 2, temperature=T)
    with pytest.raises(TypeError):
        ops.top_logits(x.half(), 2)
    v, c = torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int32)
    call = ops.soft_cross_entropy_top
    with pytest.raises(RuntimeError, match="GPU only"):
        call(x, v, c)
    for bad, err, match in ((dict(values=torch.zeros(3, 3)), RuntimeError, "must be"), (dict(values=torch.zeros(2, 2), classes=c[:2]), RuntimeError, "must be"),
                            (dict(classes=c.float()), TypeError, "int32"), (dict(classes=c[:2]), RuntimeError, "must be"),
                            (dict(lse=torch.zeros(2)), RuntimeError, "lse"), (dict(row_weight=torch.zeros(3, 1)), RuntimeError, "row_weight"),
                            (dict(row_weight=torch.zeros(3, dtype=torch.int32)), TypeError, "row_weight"), (dict(temperature=0), RuntimeError, "temperature"),
                            (dict(predicts=torch.zeros(0, 10), values=v[:0], classes=c[:0]), RuntimeError, "no rows"),
                            (dict(predicts=x.half()), TypeError, "float16"),
                            (dict(values=torch.zeros(3, 300), classes=torch.zeros(3, 300, dtype=torch.int32)), RuntimeError, "256")):
        with pytest.raises(err, match=match):
            call(**{**dict(predicts=x, values=v, classes=c), **bad})


def test_c_entries_refuse_before_any_launch():
    from efficientvlm_amd import _lib
    lib = _lib.load()
    p = 4096
    assert lib.evlm_top_logits(_lib.BF16, p, 1, 10, 10, 11, 1.0, p, p, p, None) != 0
    assert lib.evlm_top_logits(_lib.BF16, p, 1, 10, 9, 2, 1.0, p, p, p, None) != 0
    assert lib.evlm_top_logits(9, p, 1, 10, 10, 2, 1.0, p, p, p, None) != 0
    assert lib.evlm_top_logits(_lib.F32, None, 1, 10, 10, 2, 1.0, p, p, p, None) != 0
    assert lib.evlm_kl_top_fwd(_lib.F32, p, 1, 10, 10, p, p, None, 257, 1.0, 1.0, None, p, p, p, None) != 0
    assert lib.evlm_kl_top_fwd(_lib.F32, p, 1, 10, 10, p, p, None, 2, -1.0, 1.0, None, p, p, p, None) != 0
    assert lib.evlm_kl_top_bwd(_lib.F32, p, 1, 10, 10, p, p, 0, 2, 1.0, 1.0, None, p, p, p, 12, 0, None) != 0
    assert lib.evlm_kl_top_bwd(_lib.F32, p, 1, 10, 10, p, p, 0, 2, 1.0, 1.0, None, p, p, p + 4, 16, 0, None) != 0
    assert b"16-byte" in lib.evlm_last_error()


# ---- selection --------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("C,k", [(1, 1), (7, 7), (8, 3), (255, 255), (256, 256), (1001, 256), (4099, 64), (30522, 1), (30522, 16),
                                 (32768, 256), (32769, 33), (70001, 100)])
def test_top_sizes(dtype, C, k):
    for layout in ("padded", "plain", "shifted"):
        check_top(rows(3, C, dtype, seed=C, layout=layout), k, 1.5)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("C", [50, 9001, 40000])
def test_top_ties(dtype, C):
    """all equal, two values, few values, descending and ascending runs: the lower class first, always"""
    k = min(C, 200)
    g = torch.Generator().manual_seed(C)
    x = torch.stack([torch.full((C,), -2.5), torch.randint(0, 2, (C,), generator=g).float(), torch.randint(0, 9, (C,), generator=g).float(),
                     -torch.arange(C).float() // 7, torch.arange(C).float() // 3, torch.zeros(C) * torch.randn(C, generator=g)])
    x[5, ::3] = -0.0
    check_top(x.to(dtype).cuda(), k)
    check_top(x.to(dtype).cuda(), 1, 4.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("C", [40, 5000, 33000])
def test_top_values_out_of_the_ordinary(dtype, C):
    x = rows(7, C, dtype, seed=1, layout="plain").clone()
    low = torch.finfo(dtype).min
    x[0, 5:] = -math.inf
    x[1] = -math.inf
    x[2, 3] = math.inf
    x[3, [1, 8, 30]] = math.nan
    x[4, 7], x[4, 2] = math.nan, math.inf
    x[5, 6:] = low                                            # masked by the type's lowest value
    x[6] = low
    check_top(x, 20)
    x[:, :] = math.nan
    check_top(x[:1], 30)


@pytest.mark.gpu
def test_top_shapes():
    x = rows(12, 900, BF16)
    v, c, l = ops.top_logits(x, 9)
    for shaped in (x.view(3, 4, 900), x.unflatten(0, (2, 3, 2))):
        a = ops.top_logits(shaped, 9)
        assert a[0].shape == (*shaped.shape[:-1], 9) and a[2].shape == shaped.shape[:-1]
        assert torch.equal(a[0].view(12, 9), v) and torch.equal(a[1].view(12, 9), c) and torch.equal(a[2].view(12), l)
    a = ops.top_logits(x[5], 9)
    assert torch.equal(a[1], c[5]) and a[2].shape == ()
    t = x.t().contiguous().t()                                # classes not contiguous
    assert torch.equal(ops.top_logits(t, 9)[1], c)
    assert torch.equal(ops.top_logits(x[:1].expand(4, -1), 9)[1], c[:1].expand(4, -1))
    e = ops.top_logits(x[:0], 9)
    assert e[0].shape == (0, 9) and e[1].shape == (0, 9) and e[2].shape == (0,)
    y = x.float().requires_grad_()
    assert not any(t.requires_grad for t in ops.top_logits(y, 3))


# ---- the loss ---------------------------------------------------------------------------------------
def want_loss(x, values, classes, lse, T, weight, gout=1.0, u=0.0):
    """loss, gradient and the bounds of their errors, in 64 bits"""
    T = float(torch.tensor(1.0 / T, dtype=F32).double().reciprocal())         # (the kernels multiply by the f32 1 / T)
    x, z = x.detach().double().cpu(), values.double().cpu() / T
    at = classes.long().cpu()
    R, C = x.shape
    total, bound = 0.0, 0.0
    grad, gtol = torch.zeros_like(x), torch.zeros_like(x)
    for r in range(R):
        w = 1.0 if weight is None else float(weight[r])
        if w == 0:
            continue
        ok = (at[r] >= 0) & (at[r] < C) & (z[r] > -math.inf)
        if lse is None and not ok.any():
            continue
        y = x[r] / T
        lq = torch.logsumexp(y, 0)
        q = torch.exp(y - lq)
        zi, ci = z[r][ok], at[r][ok]
        lz = torch.logsumexp(zi, 0) if len(zi) else torch.tensor(-math.inf, dtype=torch.float64)
        norm = lz if lse is None else lse[r].double().cpu()
        logp, logq = zi - norm, y[ci] - lq
        p = logp.exp()
        e = zi.abs() + norm.abs() + y[ci].abs() + lq.abs() + 1
        L = (p * (logp - logq)).masked_fill(p == 0, 0).sum()
        tol = (p * 16 * F * e * (1 + (logp - logq).abs())).masked_fill(p == 0, 0).sum()
        p_sum = torch.zeros(C, dtype=torch.float64).index_add_(0, ci, p)
        size = y.abs().nan_to_num(posinf=0, neginf=0) + lq.abs() + 1
        mass, p_rest, d = p.sum(), 0.0, 0.0
        g = torch.zeros(C, dtype=torch.float64)
        gt = torch.zeros(C, dtype=torch.float64)
        kept = torch.zeros(C, dtype=torch.bool)
        kept[at[r][(at[r] >= 0) & (at[r] < C)]] = True
        if lse is not None and not kept.all() and torch.logsumexp(y[~kept], 0) > -math.inf:
            p_rest = float((-torch.expm1(lz - norm)).clamp_min(0)) if len(zi) else 1.0
            d = 8 * F * ((abs(lz) if len(zi) else 0) + abs(norm) + 1)
            lr = torch.logsumexp(y[~kept], 0)
            if p_rest > 0:
                L = L + p_rest * (math.log(p_rest) - (lr - lq))
                tol = tol + d * (2 + abs(math.log(p_rest) - (lr - lq))) + 16 * F * p_rest * (lr.abs() + lq.abs() + 1)
            else:
                tol = tol + d * (2 + abs(math.log(d) - (lr - lq)))
        mass = mass + p_rest
        g = mass * q - p_sum
        gt = 16 * F * size * (q * (mass + d) + p_sum * (1 + norm.abs() + (zi.abs().max() if len(zi) else 0))) + d * q
        if lse is not None and (~kept).any() and torch.logsumexp(y[~kept], 0) > -math.inf:
            share = torch.exp(y - lr).masked_fill(kept, 0.0)
            g = torch.where(kept, g, share * (mass * torch.exp(lr - lq) - p_rest))
            gt = gt + share * (2 * d + 16 * F * (size + lr.abs()) * (mass * torch.exp(lr - lq) + p_rest))
        factor = w / T / R * gout
        total, bound = total + w * L / R, bound + w * tol / R
        grad[r], gtol[r] = factor * g, abs(factor) * gt + (u + 4 * F) * (factor * g).abs() + 1e-38
    return total, bound + (R + 4) * F * abs(total), grad, gtol


def check_loss(x, values, classes, lse=None, T=1.0, weight=None, gout=1.0):
    s = x.detach().requires_grad_()
    loss = ops.soft_cross_entropy_top(s, values, classes, lse=lse, temperature=T, row_weight=weight)
    (g,) = torch.autograd.grad(loss, s, torch.tensor(gout, device="cuda"))
    assert loss.dtype == F32 and loss.shape == () and g.shape == x.shape and g.dtype == x.dtype
    L, lt, G, gt = want_loss(x, values, classes, lse, T, weight, gout, 2.0 ** -8 if x.dtype == BF16 else F)
    assert abs(float(loss) - float(L)) <= float(lt) + 1e-30, (float(loss), float(L), float(lt))
    over = ((g.double().cpu() - G).abs() - gt).nan_to_num(math.inf)
    assert over.max() <= 0, f"{int((over > 0).sum())} of {over.numel()} elements off, worst by {over.max():.3e} over its bound"
    return loss, g


def pair(R, C, k, dtype, seed=0, layout="padded", T=1.0, rest=True):
    teacher = rows(R, C, dtype, seed=seed + 100)
    s = rows(R, C, dtype, seed=seed, layout=layout)
    s.copy_((0.7 * teacher.float() + 0.5 * s.float()).to(dtype))
    v, c, l = ops.top_logits(teacher, k, temperature=T)
    return s, v, c, (l if rest else None)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("R,C,k", [(1, 1, 1), (2, 9, 4), (5, 9, 9), (3, 300, 256), (4, 1001, 31), (33, 30522, 16), (2, 33001, 128)])
def test_loss_sizes(dtype, rest, R, C, k):
    for layout, T in (("padded", 1.0), ("plain", 2.0), ("shifted", 0.7)):
        s, v, c, l = pair(R, C, k, dtype, seed=C, layout=layout, T=T, rest=rest)
        check_loss(s, v, c, l, T, torch.rand(R, generator=torch.Generator().manual_seed(R)).cuda() if R > 1 else None, gout=1.7)


@pytest.mark.gpu
@pytest.mark.parametrize("R", [1023, 8192, 9001])
def test_loss_of_many_rows(R):
    check_loss(*pair(R, 9, 4, F32, seed=R, rest=True))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_all_classes_kept_is_the_whole_rows_loss(dtype):
    """k = C: soft_cross_entropy of the same logits"""
    R, C = 6, 40
    t, s = rows(R, C, dtype, 1), rows(R, C, dtype, 2)
    v, c, l = ops.top_logits(t, C, temperature=2.0)
    for lse in (None, l):
        loss, g = check_loss(s, v, c, lse, 2.0)
        a = s.detach().requires_grad_()
        other = ops.soft_cross_entropy(a, t, temperature=2.0)
        assert abs(float(loss) - float(other)) <= 2.0 ** -17 * (1 + abs(float(other)))         # 64 F times logs of size up to 8, both sides
        og, = torch.autograd.grad(other, a)
        assert (g.float() - og.float()).abs().max() <= (2.0 ** -7 if dtype == BF16 else 2.0 ** -16) * og.float().abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rest", [False, True])
def test_entries_left_out_twice_and_masked(dtype, rest):
    R, C, k = 8, 500, 6
    s, v, c, l = pair(R, C, k, dtype, seed=4, rest=rest)
    v, c, s = v.clone(), c.clone(), s.clone()
    c[0, 2:] = -1                                  # padding
    c[1, 3], c[1, 4] = C, 2 ** 31 - 1              # outside
    c[2] = -1                                      # a row without entries
    c[3, 1] = c[3, 0]                              # the same class twice
    c[4] = c[4, 0]                                 # ... always
    v[5, 3:] = -math.inf                           # no mass
    s[6, c[6, 5].long()] = -math.inf if not rest else s[6, 0]
    v[6, 5] = -math.inf                            # ... where the student has none
    w = torch.rand(R, generator=torch.Generator().manual_seed(0)).cuda()
    w[7] = 0.0
    s[7] = math.nan                                # a row of weight 0 holds anything
    loss, g = check_loss(s, v, c, l, 1.0, w)
    assert (g[7] == 0).all()
    if not rest:
        assert (g[2] == 0).all()
    big = check_loss(s, v, c.long(), l, 1.0, w)    # int64 classes
    assert torch.equal(big[0], loss) and torch.equal(big[1], g)
    far = c.long().clone()
    far[1, 4] = 2 ** 40 + 3                        # (a class that 32 bits would fold back into the row)
    assert torch.equal(check_loss(s, v, far, l, 1.0, w)[1], g)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_masked_students_and_extreme_rows(dtype):
    """classes at -inf and at the type's lowest value, rows of one overwhelming class, mass all kept and none kept"""
    R, C, k = 6, 700, 8
    s, v, c, l = pair(R, C, k, dtype, seed=9)
    s, c = s.clone(), c.clone()
    free = [i for i in range(C) if i not in set(c.flatten().tolist())]
    s[0, free[:300]] = -math.inf
    s[1, free] = torch.finfo(dtype).min            # the student has no mass outside the kept classes
    s[2, c[2, 0].long()] = 60.0
    v[3, 0], l[3] = v[3, 0] + 50, v[3, 0] + 50     # the teacher has none
    s[4, free[0]] = 80.0                           # nearly all of the student's mass is not kept
    keep = torch.tensor([0, 2, 3, 4, 5], device="cuda")
    check_loss(s[keep], v[keep], c[keep], l[keep])
    check_loss(s, v, c, None)
    check_loss(s[1:2], v[1:2], c[1:2], l[1:2])     # (the classes that the other rows kept hold its rest)
    s[5, 3] = math.nan                             # a broken row shows
    a = s.detach().requires_grad_()
    loss = ops.soft_cross_entropy_top(a, v, c, lse=l)
    g, = torch.autograd.grad(loss, a)
    assert math.isnan(float(loss)) and g[5].isnan().all() and g[4].isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rest_at_the_lowest_value(dtype):
    """a student whose every class outside the kept ones holds the type's lowest value: the rest lies 3e38 away, and its
    gradient is spread evenly over it (a log-sum-exp in one number would have lost the log of the count)"""
    s, v, c, l = pair(3, 900, 5, dtype, seed=11)
    low = torch.full_like(s, torch.finfo(dtype).min).scatter_(1, c.long(), s.gather(1, c.long()))
    a = low.detach().requires_grad_()
    loss = ops.soft_cross_entropy_top(a, v, c, lse=l)
    assert float(loss) > 1e37
    g = torch.autograd.grad(loss, a)[0].double().cpu()
    kept = torch.zeros(3, 900, dtype=torch.bool).scatter_(1, c.long().cpu(), True)
    p_rest = (1 - torch.exp(v.double() - l.double()[:, None]).sum(1)).cpu()
    want = (-p_rest / 895 / 3)[:, None].expand(3, 900)[~kept]
    assert ((g[~kept] - want).abs() <= (2.0 ** -8 + 2.0 ** -17) * want.abs()).all()


@pytest.mark.gpu
def test_gradient_against_differences():
    """directional differences of the definition in 64 bits against the f32 kernel's gradient"""
    for rest in (False, True):
        s, v, c, l = pair(5, 300, 12, F32, seed=2, T=1.5, rest=rest)
        w = torch.rand(5, generator=torch.Generator().manual_seed(0)).cuda()
        _, g = check_loss(s, v, c, l, 1.5, w)
        _, _, G, gt = want_loss(s, v, c, l, 1.5, w)
        d = torch.randn(5, 300, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
        f = lambda h: want_loss(s.double().cpu() + h * d, v, c, l, 1.5, w)[0]
        diff = (f(1e-5) - f(-1e-5)) / 2e-5
        assert abs((g.double().cpu() * d).sum() - diff) <= (gt * d.abs()).sum() + 1e-8


@pytest.mark.gpu
def test_no_second_derivative():
    s, v, c, l = pair(3, 50, 4, F32)
    a = s.detach().requires_grad_()
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(ops.soft_cross_entropy_top(a, v, c, lse=l), a, create_graph=True)


@pytest.mark.gpu
def test_join_with_the_hard_label_loss():
    """logits that feed the hard-label and the distillation loss: one gradient buffer (join_grads), the sum of both"""
    R, C = 20, 1001
    s, v, c, l = pair(R, C, 16, BF16, seed=6)
    labels = torch.randint(0, C, (R,), generator=torch.Generator().manual_seed(0)).cuda()
    a = s.detach().requires_grad_()
    j = ops.join_grads(a)
    (ops.cross_entropy(j, labels) + 0.5 * ops.soft_cross_entropy_top(j, v, c, lse=l)).backward()
    b = s.detach().requires_grad_()
    ce = torch.autograd.grad(ops.cross_entropy(b, labels), b)[0].double().cpu()
    _, _, G, gt = want_loss(s, v, c, l, 1.0, None, 0.5, 2.0 ** -8)
    both = ce + G
    # the hard-label gradient is rounded once into the buffer on either side, the sum once more
    assert ((a.grad.double().cpu() - both).abs() <= gt + 2 * 2.0 ** -8 * (both.abs() + ce.abs()) + 1e-30).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rest", [False, True])
def test_a_gradient_larger_than_the_cache(dtype, rest):
    """a thousand rows, and the same rows several times over with the loss's gradient as many times larger (powers of two: every
    factor of a row is the same number): the same bits in each copy"""
    C, k, n = 30001, 24, 8 if dtype == BF16 else 4
    x = rows(1024, C, dtype, seed=9)
    values, classes, lse = ops.top_logits(rows(1024, C, dtype, seed=10), k, temperature=2.0)
    weight = torch.rand(1024, device="cuda")
    weight[5] = 0.0

    def grad(copies):
        s = x.repeat(copies, 1).requires_grad_()
        loss = ops.soft_cross_entropy_top(s, values.repeat(copies, 1), classes.repeat(copies, 1), lse=lse.repeat(copies) if rest else None,
                                          temperature=2.0, row_weight=weight.repeat(copies))
        return torch.autograd.grad(loss, s, torch.tensor(float(copies), device="cuda"))[0]

    small, large = grad(1), grad(n)
    assert (small.abs().sum(1) > 0).sum() == 1023
    for i in range(n):
        assert torch.equal(small, large[1024 * i:1024 * (i + 1)])


@pytest.mark.gpu
def test_same_bits_shapes_and_streams():
    s, v, c, l = pair(40, 3001, 32, BF16, seed=7)
    first = check_loss(s, v, c, l)
    a = s.unflatten(0, (8, 5)).detach().requires_grad_()
    loss = ops.soft_cross_entropy_top(a, v.view(8, 5, 32), c.view(8, 5, 32), lse=l.view(8, 5))
    loss.backward()
    assert torch.equal(loss, first[0]) and torch.equal(a.grad.view(40, 3001), first[1])
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    out = []
    for i in range(6):
        with torch.cuda.stream(side[i % 2]):
            b = s.detach().requires_grad_()
            loss = ops.soft_cross_entropy_top(b, v, c, lse=l)
            out.append((loss, *torch.autograd.grad(loss, b), *ops.top_logits(s, 32)))
    torch.cuda.synchronize()
    for o in out:
        assert torch.equal(o[0], first[0]) and torch.equal(o[1], first[1])
        assert all(torch.equal(x, y) for x, y in zip(o[2:], out[0][2:]))


@pytest.mark.gpu
def test_capture():
    """teacher's selection, loss and gradient captured together; replayed on other logits with eager work in between"""
    R, C, k = 30, 5003, 24
    t, s = rows(R, C, BF16, 1), rows(R, C, BF16, 2).detach().requires_grad_()

    def step(t, s):
        v, c, l = ops.top_logits(t, k, temperature=2.0)
        loss = ops.soft_cross_entropy_top(s, v, c, lse=l, temperature=2.0)
        return loss, torch.autograd.grad(loss, s)[0], c
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(t, s)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step(t, s)
    for turn in range(4):
        t.copy_(rows(R, C, BF16, 10 + turn))
        with torch.no_grad():
            s.copy_(rows(R, C, BF16, 20 + turn))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in static]
        for a, b in zip(got, step(t, s.detach().requires_grad_())):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_together():
    """as they are used: a teacher keeps its top logits; the student's packed answers go through attention and the vocabulary
    projection, the distillation loss comes back through all of it (f32, against the same chain in 64 bits)"""
    g = torch.Generator().manual_seed(0)
    H, dh, C, k, T = 4, 32, 1201, 20, 2.0
    lens = [3, 9, 1, 14, 40, 6]
    n, d = sum(lens), H * dh
    cu = torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device="cuda")
    r = lambda *s: torch.randn(*s, generator=g)
    x, W, E, teacher = r(n, d), r(3 * d, d) * d ** -0.5, r(C, d) * 0.3, r(n, C) * 3
    weight = torch.rand(n, generator=g)
    v, c, l = ops.top_logits(teacher.cuda(), k, temperature=T)
    px, pW, pE = (torch.nn.Parameter(t.cuda()) for t in (x, W, E))
    qkv = ops.linear(px, pW, None).view(n, 3, H, dh)
    ctx = ops.packed_attention(qkv[:, 0], qkv[:, 1], qkv[:, 2], cu)
    logits = ops.linear(ctx.reshape(n, d), pE, None)
    loss = ops.soft_cross_entropy_top(logits, v, c, lse=l, temperature=T, row_weight=weight.cuda())
    got = torch.autograd.grad(loss, (px, pW, pE))

    dx, dW, dE = (t.double().requires_grad_() for t in (x, W, E))
    q64, k64, v64 = (dx @ dW.T).view(n, 3, H, dh).unbind(1)
    out, a = [], 0
    for m in lens:
        S = (q64[a:a + m].transpose(0, 1) @ k64[a:a + m].permute(1, 2, 0)) * dh ** -0.5
        S = S.masked_fill(torch.ones(m, m, dtype=torch.bool).triu(1), -math.inf)
        out.append((torch.softmax(S, 2) @ v64[a:a + m].transpose(0, 1)).transpose(0, 1))
        a += m
    lq = torch.log_softmax(torch.cat(out).reshape(n, d) @ dE.T / T, 1)
    lp = torch.log_softmax(teacher.double() / T, 1)
    at = c.long().cpu()
    pk, lk = lp.gather(1, at).exp(), lp.gather(1, at)
    rest = torch.ones(n, C, dtype=torch.bool).scatter_(1, at, False)
    pr = (lp.exp() * rest).sum(1)
    L = (pk * (lk - lq.gather(1, at))).sum(1) + pr * (pr.log() - torch.logsumexp(lq.masked_fill(~rest, -math.inf), 1))
    ref = (L * weight.double()).mean()
    assert abs(float(loss) - float(ref)) <= 1e-5 * (1 + abs(float(ref)))     # f32 products of 128 terms: 128 F = 8e-6 of logits of size 1
    for a, b in zip(got, torch.autograd.grad(ref, (dx, dW, dE))):
        # four products of up to 1201 terms in a row, each good to (terms) F of its largest sums
        assert (a.double().cpu() - b).norm() <= 4 * 1201 * F * b.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("C", [700, 40000])
def test_gradient_of_a_rest_close_to_the_teachers(dtype, C):
    """student and teacher agree on the mass outside the kept classes to a few parts in 10^5: the rest's gradient is that difference,
    formed from terms that carry it (64 bits), not from two f32 numbers next to each other.  The other classes hold 0: their sum is a
    whole number, exact, and every exponent among them 0, so what remains are a dozen f32 roundings of the result itself"""
    R, k = 4, 3
    s = torch.zeros(R, C, dtype=dtype, device="cuda")
    c = torch.randint(0, C // 2, (R, k), generator=torch.Generator().manual_seed(1)).cuda().int() * 2 + torch.tensor([0, 1, 0], device="cuda").int()
    c[:, 2] = C - 1
    v = torch.tensor([[5.0, 3.5, 1.25]], device="cuda").repeat(R, 1)
    s.scatter_(1, c.long(), v.to(dtype))
    lse = torch.logsumexp(s.double(), 1)
    for off in (3e-5, -1e-4, 4e-6):
        l = (lse + off).float()
        a = s.detach().requires_grad_()
        g = torch.autograd.grad(ops.soft_cross_entropy_top(a, v, c, lse=l), a)[0].double().cpu()
        p = torch.exp(v.double() - l.double()[:, None]).sum(1)
        q_rest = torch.exp(-torch.logsumexp(s.double(), 1)) * (C - k)
        want = ((q_rest - (1 - p)) / (C - k) / R).cpu()
        kept = torch.zeros(R, C, dtype=torch.bool).scatter_(1, c.long().cpu(), True)
        want = want[:, None].expand(R, C)[~kept]
        assert ((g[~kept] - want).abs() <= ((2.0 ** -8 if dtype == BF16 else 0) + 16 * F) * want.abs()).all(), off


# ---- large constants (masked classes that are finite) ---------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("C", [900, 40000])
@pytest.mark.parametrize("value", [-1e9, -1e10, -1e12, -1e20, -1e29, 1e10, 1e25])
def test_top_of_rows_at_a_masking_constant(dtype, C, value):
    """the log-sum-exp of rows whose every class holds a large constant is constant / T + log C: finite, and not the constant itself"""
    x = rows(4, C, dtype, seed=2, layout="plain").clone()
    x[0] = value
    x[1, 7:] = value
    x[2, ::2] = value
    for T in (1.0, 1.5, 0.7, 4.0):
        check_top(x, 20, T)
    check_top(rows(3, C, dtype, seed=3), 20, 1e-9)            # ordinary logits, exponents of the same size


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("C", [900, 40000])
@pytest.mark.parametrize("value", [-3e8, -1e10, -1e12, -1e20, -1e29, 1e10, 1e25])
def test_rest_at_a_masking_constant(dtype, C, value):
    """a student whose every class outside the kept ones holds one large constant: the loss is finite, the rest's gradient spread evenly
    over those classes, the kept classes' as in the definition.  Every exponent that enters is a difference of equal numbers, of
    numbers 1e8 apart, or of kept logits (all their size: e), so the errors are those of e"""
    R, k = 3, 5
    for T in (1.0, 1.5, 0.7):
        s, v, c, l = pair(R, C, k, dtype, seed=11, T=T)
        full = torch.full_like(s, value).scatter_(1, c.long(), s.gather(1, c.long()))
        a = full.detach().requires_grad_()
        loss = ops.soft_cross_entropy_top(a, v, c, lse=l, temperature=T)
        g = torch.autograd.grad(loss, a)[0].double().cpu()
        L, _, G, _ = want_loss(full, v, c, l, T, None)
        u = 2.0 ** -8 if dtype == BF16 else F
        assert abs(float(loss) - float(L)) <= 2.0 ** -17 * abs(float(L))
        e = float(s.gather(1, c.long()).abs().max() + v.abs().max()) / T + float(l.abs().max()) + 8
        y, z = s.gather(1, c.long()).double().cpu() / T, v.double().cpu() / T
        p = torch.exp(z - l.double().cpu()[:, None])
        q = torch.softmax(full.double().cpu() / T, 1).gather(1, c.long().cpu())
        got, want = g.gather(1, c.long().cpu()), G.gather(1, c.long().cpu())
        assert ((got - want).abs() <= u * want.abs() + 16 * F * e * (p + q) / T / R + 1e-30).all()
        p_rest = 1 - p.sum(1)
        share = ((1 - p_rest) if value > 0 else -p_rest) / (C - k) / T / R                 # mass q_rest - p_rest; value > 0: q_rest = 1
        kept = torch.zeros(R, C, dtype=torch.bool).scatter_(1, c.long().cpu(), True)
        share = share[:, None].expand(R, C)[~kept]
        # (p_rest of f32 terms: 8 F e of their size 1; C / 512 + 16 terms of the sum in a row)
        slack = 8 * F * e / (C - k) / T / R
        assert ((g[~kept] - share).abs() <= (u + (C / 512 + 32) * F) * share.abs() + slack).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("C", [300, 33000])
@pytest.mark.parametrize("rest", [False, True])
def test_a_row_without_entries_holds_anything(dtype, C, rest):
    """with and without the rest: such a row adds nothing and has a zero gradient, the other rows' are those without it"""
    s, v, c, l = pair(4, C, 6, dtype, seed=3, rest=rest)
    s, v, c = s.clone(), v.clone(), c.clone()
    c[1], c[2] = -1, C
    want, wg = check_loss(s, v, c, l)
    for broken in (math.nan, math.inf, -math.inf):
        s[1], s[2, 5:] = broken, broken
        v[1], v[2] = broken, broken
        if rest:
            l[1] = broken
        a = s.detach().requires_grad_()
        loss = ops.soft_cross_entropy_top(a, v, c, lse=l)
        g, = torch.autograd.grad(loss, a)
        assert torch.equal(loss, want) and torch.equal(g, wg) and not g[1:3].any()


@pytest.mark.gpu
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("size", [3e3, 1e5, 1e6])
def test_gradient_of_logits_far_from_zero(rest, size):
    """logits around +-size, a few units apart: every probability is an exponent of differences (exact in f32), so the gradient is as good as
    around zero.  (logits times the f32 1 / T, rounded before the difference, would be off by size 2^-24: 6 % of a probability at 1e6)"""
    R, C, k, T = 6, 200, 9, 0.7
    g = torch.Generator().manual_seed(4)
    # whole multiples of 2^-4: f32 holds them up to 2^20
    t = (torch.randn(R, C, generator=g) * 32).round() / 16
    s = (t * 16 + (torch.randn(R, C, generator=g) * 8).round()).round() / 16
    inv = float(torch.tensor(1.0 / T, dtype=F32))
    for shift in (size, -size):
        shift = float(round(shift))
        x, y = (s + shift).cuda(), (t + shift).cuda()
        v, c, _ = ops.top_logits(y, k)
        # a log-sum-exp of the teacher as f32 holds it; rows in which it leaves the kept classes more than all mass have no rest
        l = torch.logsumexp(y.double() * inv, 1).float() if rest else None
        a = x.detach().requires_grad_()
        got = torch.autograd.grad(ops.soft_cross_entropy_top(a, v, c, lse=l, temperature=T), a)[0].double().cpu()
        xs, at = s.double() * inv, c.long().cpu()
        q = torch.softmax(xs, 1)
        z = v.double().cpu() * inv
        p = torch.softmax(z, 1) if l is None else torch.exp(z - l.double().cpu()[:, None])
        P = torch.zeros_like(q).scatter_(1, at, p)
        if rest:
            kept = torch.zeros_like(q, dtype=torch.bool).scatter_(1, at, True)
            p_rest = (1 - p.sum(1, keepdim=True)).clamp_min(0)
            mass = p.sum(1, keepdim=True) + p_rest
            q_rest = q.masked_fill(kept, 0).sum(1, keepdim=True)
            want = torch.where(kept, mass * q - P, q / q_rest * (mass * q_rest - p_rest))
        else:
            want = q - P
        # exponents up to e = (spread of the logits) / T: 4 F e each; sums of C terms; p_rest of 64-bit terms
        e = 2 * float((s.max() - s.min()).clamp_min(float(t.max() - t.min()))) * inv + 16
        assert ((got - want / T / R).abs() <= 8 * F * e * (q + P) * (1.5 if not rest else 3) / T / R + 4 * F * want.abs() + 1e-12).all()
