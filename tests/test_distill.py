"""Distillation from a teacher's top logits: the k largest logits, the loss on them and its
gradient, against the definitions in 64 bits, with tolerances from the kernels' roundings.

The rounding unit is u = 2^-24. An exponential's argument is a difference, a product and a constant
(3 roundings, |argument| <= S), the power of two itself is good to 2^-22 = 4 u, and a positive sum
of n terms over 32 or more lanes adds n / 32 + 16 roundings at most, so every probability has a
relative error below e = (4 S + n / 32 + 64) u, with S the largest |logit| / temperature of the row
or its teacher (the entries' arguments include one subtraction of the log-sum-exp).
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import splax_b200 as sx
from splax_b200 import _lib

U = 2.0**-24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF = math.inf


# ------------------------------------------------------------------ oracle (64 bits, host)
def oracle(z, v, ids, lse_t=None, temperature=1.0, weights=None, denom=None):
    """(loss, gradient, loss tolerance, gradient tolerance before the output's rounding)."""
    z, v, ids = z.double().cpu(), v.double().cpu(), ids.long().cpu()
    R, C = z.shape
    tau = float(temperature)
    w = torch.ones(R, dtype=torch.float64) if weights is None else weights.double().cpu()
    denom = float(R if denom is None else denom)
    loss, loss_tol = 0.0, 0.0
    grad, tol = torch.zeros_like(z), torch.zeros_like(z)
    for r in range(R):
        if w[r] == 0:
            continue
        valid = (ids[r] >= 0) & (ids[r] < C)
        a, at = v[r][valid] / tau, ids[r][valid]
        if lse_t is None:
            if a.numel() == 0 or bool((a == -INF).all()):
                continue
            norm = torch.logsumexp(a, 0)
        else:
            norm = lse_t[r].double().cpu()
            if norm == -INF:
                continue
        s = z[r] / tau
        if bool((s == -INF).all()):
            continue
        log_q = torch.log_softmax(s, 0)  # the maximum first: -3e38 + ln C is -3e38 in 64 bits too
        q = log_q.exp()
        log_p = a - norm
        p = log_p.exp()
        named = torch.zeros(C, dtype=torch.bool)
        named[at] = True
        log_qo = torch.logsumexp(log_q[~named], 0) if bool((~named).any()) else torch.tensor(-INF)
        P = float(p.sum())
        rho = max(0.0, 1.0 - P) if lse_t is not None and log_qo > -INF else 0.0
        finite = torch.cat([s, a, norm[None]])
        finite = finite[finite.isfinite()]
        S = float(finite.abs().max()) if finite.numel() else 0.0
        if S > 1e30:  # rows with the type's lowest value: those classes have no probability
            S = float(finite[finite.abs() < 1e30].abs().max()) if bool(
                (finite.abs() < 1e30).any()) else 0.0
        e = (4 * S + C / 32 + 64) * U
        live = p > 0
        terms = p[live] * (log_p[live] - log_q[at[live]])
        row = float(terms.sum())
        bound = e * float((terms.abs() + p[live]).sum())
        if lse_t is not None and log_qo > -INF:
            if rho > 0:
                row += rho * (math.log(rho) - float(log_qo))
            # rho has an absolute error of e P, and may have it where it is zero
            bound += e * max(P, rho) * (2 + abs(math.log(max(rho, e))) + abs(float(log_qo)))
        g = (P + rho) * q
        g_tol = e * (P + rho) * q
        if log_qo > -INF:
            share = (log_q - log_qo).exp()
            out = ~named
            g[out] = ((P + rho) * math.exp(float(log_qo)) - rho) * share[out]
            g_tol[out] = e * ((P + rho) * q[out] + (rho + (P if lse_t is not None else 0))
                              * share[out])
        else:
            g[~named] = 0.0
        for c, x in zip(at.tolist(), p.tolist()):
            g[c] -= x
            g_tol[c] += e * x
        k = float(w[r]) * tau / denom
        grad[r], tol[r] = g * k, (g_tol * abs(k)) + 4 * U * g.abs() * abs(k)
        loss += float(w[r]) * tau * tau / denom * row
        loss_tol += abs(float(w[r])) * tau * tau / denom * bound
    return loss, grad, loss_tol + 2 * U * abs(loss), tol


def rounded(tol, ref, dtype):
    """The tolerance with the output's one rounding: half a step, or half the smallest number."""
    return tol * (1 + torch.finfo(dtype).eps) + ref.abs() * (torch.finfo(dtype).eps / 2) + \
        torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def make(R, C, K, dtype, seed=0, *, pad=0, offset=0, spread=2.5, temperature=1.0):
    g = torch.Generator().manual_seed(seed)
    teacher = torch.randn(R, C, generator=g) * spread
    z = torch.randn(R, C, generator=g) * spread * 0.5 + 0.6 * teacher
    teacher, z = teacher.to(dtype), z.to(dtype)
    v, i = teacher.double().topk(K, dim=1)
    lse = torch.logsumexp(teacher.double() / temperature, 1).float()
    store = torch.zeros(offset + R * (C + pad), dtype=dtype, device="cuda")
    rows = store[offset:].view(R, C + pad)[:, :C]
    rows.copy_(z)
    return rows, v.to(dtype).cuda(), i.to(torch.int32).cuda(), lse.cuda()


def check(z, v, i, lse=None, cot=1.0, **kw):
    """The loss alone, the loss and gradient together, and the gradient computed again."""
    ref, ref_grad, tol, grad_tol = oracle(z, v, i, lse, **kw)
    with torch.no_grad():
        alone = sx.distill_loss(z, v, i, lse, **kw)
    assert alone.dtype == F32 and alone.shape == ()
    assert abs(alone.item() - ref) <= tol, (alone.item(), ref, tol)
    # a non-overlapping leaf with the same strides
    leaf = z.detach().requires_grad_()
    loss = sx.distill_loss(leaf, v, i, lse, **kw)
    assert abs(loss.item() - ref) <= tol
    first, = torch.autograd.grad(loss, leaf, torch.tensor(cot, device="cuda"), retain_graph=True)
    again, = torch.autograd.grad(loss, leaf, torch.tensor(cot, device="cuda"))
    bar = rounded(grad_tol * abs(cot), ref_grad * cot, z.dtype)
    if cot != 1.0:  # scaled in place after the first rounding: one more
        bar = bar + (ref_grad * cot).abs() * torch.finfo(z.dtype).eps / 2 + \
            abs(cot) * torch.finfo(z.dtype).smallest_normal * torch.finfo(z.dtype).eps / 2
    for got in (first, again):
        assert got.shape == z.shape and got.dtype == z.dtype
        err = (got.double().cpu() - ref_grad * cot).abs()
        bad = ~(err <= bar)
        assert not bool(bad.any()), (int(bad.sum()), float((err / bar).max()))
    return ref


# ------------------------------------------------------------------ host
def test_the_oracles_gradient_is_the_losss_difference_quotient():
    g = torch.Generator().manual_seed(1)
    z = torch.randn(4, 9, generator=g, dtype=torch.float64) * 2
    t = torch.randn(4, 9, generator=g, dtype=torch.float64) * 2
    v, i = t.topk(3, 1)
    i[2] = -1
    i[1, 2] = i[1, 0]
    w = torch.tensor([0.5, 1.0, 2.0, 1.5])
    for lse in (None, torch.logsumexp(t / 2.0, 1)):
        kw = dict(temperature=2.0, weights=w, denom=3.0)
        _, grad, _, _ = oracle(z, v, i, lse, **kw)
        h = 1e-5
        for r in range(4):
            for c in range(9):
                d = torch.zeros_like(z)
                d[r, c] = h
                up, down = oracle(z + d, v, i, lse, **kw)[0], oracle(z - d, v, i, lse, **kw)[0]
                # truncation h^2 / 6 times a third derivative below 4, cancellation 1e-15 / h
                assert abs((up - down) / (2 * h) - float(grad[r, c])) <= 1e-9


def test_refusals_without_a_device():
    z, v, i = torch.zeros(4, 9), torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        sx.top_logits(z, 3)
    with pytest.raises(ValueError, match="CUDA"):
        sx.distill_loss(z, v, i)
    for bad in (0, 10, -1):
        with pytest.raises(ValueError, match="k="):
            sx.top_logits(z, bad)
    with pytest.raises(ValueError, match="k="):
        sx.top_logits(torch.zeros(2, 300), 129)
    with pytest.raises(TypeError):
        sx.top_logits(z, 2.5)
    for x in (z.double(), z.long(), torch.zeros(3, 0), torch.zeros(()), torch.zeros(1, 262145)):
        with pytest.raises(ValueError, match="logits"):
            sx.top_logits(x, 1)
        with pytest.raises(ValueError, match="logits"):
            sx.distill_loss(x, v, i)
    for t in (0.0, -1.0, INF, math.nan):
        with pytest.raises(ValueError, match="temperature"):
            sx.top_logits(z, 3, temperature=t)
        with pytest.raises(ValueError, match="temperature"):
            sx.distill_loss(z, v, i, temperature=t)
    for args in ((v[:3], i[:3]), (v, i[:, :2]), (v[:, :0], i[:, :0]), (v[0], i[0]),
                 (torch.zeros(4, 129), torch.zeros(4, 129, dtype=torch.int32))):
        with pytest.raises(ValueError, match="top_values"):
            sx.distill_loss(z, *args)
    with pytest.raises(ValueError, match="top_ids"):
        sx.distill_loss(z, v, i.short())
    with pytest.raises(ValueError, match="top_values"):
        sx.distill_loss(z, v.double(), i)
    with pytest.raises(ValueError, match="top_lse"):
        sx.distill_loss(z, v, i, torch.zeros(3))
    with pytest.raises(ValueError, match="weights"):
        sx.distill_loss(z, v, i, weights=torch.ones(4, dtype=torch.int32))
    for d in (0.0, -2.0, INF, math.nan):
        with pytest.raises(ValueError, match="denom"):
            sx.distill_loss(z, v, i, denom=d)
    with pytest.raises(ValueError, match="denom"):
        sx.distill_loss(z[:0], v[:0], i[:0])


def test_c_entry_refusals():
    """Every call is refused on the host, before any launch: the pointers are never used."""
    lib = _lib.load()
    P = ctypes.c_void_p
    good = P(1 << 20)
    top = dict(z=good, dtype=0, rows=2, classes=9, stride=9, k=3, tau=1.0, values=good, ids=good,
               lse=good)
    for bad in (dict(z=None), dict(z=P((1 << 20) + 2)), dict(dtype=3), dict(dtype=-1),
                dict(rows=-1), dict(classes=0), dict(classes=262145, stride=262145), dict(stride=8),
                dict(k=0), dict(k=10), dict(classes=300, stride=300, k=129), dict(tau=0.0),
                dict(tau=math.nan), dict(tau=INF), dict(values=None), dict(ids=P(1 << 20 | 1)),
                dict(lse=None), dict(rows=1 << 40, stride=1 << 40)):
        a = {**top, **bad}
        rc = lib.splax_top_logits(a["z"], a["dtype"], a["rows"], a["classes"], a["stride"], a["k"],
                                  a["tau"], a["values"], a["ids"], a["lse"], None)
        assert rc == _lib.SPLAX_ERR_INVALID_ARGUMENT, bad
        assert lib.splax_last_error().decode().startswith("top_logits")
    ok = dict(z=good, dtype=1, rows=2, classes=9, stride=9, v=good, vd=0, i=good, bits=32,
              lse=None, k=3, w=None, tau=1.0, denom=2.0, work=good, loss=good, grad=good,
              cot=good)
    for bad in (dict(z=None), dict(dtype=5), dict(v=None), dict(vd=7), dict(i=None), dict(bits=16),
                dict(i=P((1 << 20) + 4), bits=64), dict(lse=P(3)), dict(w=P(6)), dict(denom=0.0),
                dict(denom=math.nan), dict(denom=INF), dict(work=None), dict(work=P(4)),
                dict(loss=None), dict(grad=None), dict(grad=P(1)), dict(cot=None), dict(k=129),
                dict(stride=8), dict(tau=-1.0)):
        a = {**ok, **bad}
        head = (a["z"], a["dtype"], a["rows"], a["classes"], a["stride"], a["v"], a["vd"], a["i"],
                a["bits"], a["lse"], a["k"], a["w"], a["tau"], a["denom"])
        refused = []
        if not {"grad", "cot"} & set(bad):
            refused.append(lib.splax_distill_loss(*head, a["work"], a["loss"], None))
        if not {"cot"} & set(bad):
            refused.append(lib.splax_distill_loss_and_grad(*head, a["work"], a["loss"], a["grad"],
                                                           None))
        if not {"work", "loss"} & set(bad):
            refused.append(lib.splax_distill_loss_bwd(*head, a["cot"], a["grad"], None))
        assert set(refused) == {_lib.SPLAX_ERR_INVALID_ARGUMENT}, bad
    for a in ((None, 0, 4, good), (good, 3, 4, good), (good, 0, -1, good), (good, 0, 4, None),
              (P(2), 0, 4, good)):
        assert lib.splax_distill_scale_grad(*a, None) == _lib.SPLAX_ERR_INVALID_ARGUMENT
    assert lib.splax_capture_id(None, None) == _lib.SPLAX_ERR_INVALID_ARGUMENT


def test_python_limits_are_the_headers():
    from pathlib import Path

    from splax_b200 import _distill

    text = (Path(__file__).resolve().parents[1] / "include" / "splax_b200.h").read_text()
    for name, value in (("MAX_CLASSES", _distill.MAX_CLASSES), ("MAX_K", _distill.MAX_K),
                        ("WORKSPACE", _distill.WORKSPACE)):
        assert f"#define SPLAX_DISTILL_{name} {value}\n" in text


# ------------------------------------------------------------------ top logits
def check_top(z, k, temperature=1.0):
    values, ids, lse = sx.top_logits(z, k, temperature=temperature)
    host = z.cpu()
    key = torch.where(host == 0, torch.zeros_like(host), host).double()  # the zeros are equal
    key = torch.where(key.isnan(), torch.full_like(key, math.nan), key)
    order = torch.sort(torch.where(key.isnan(), torch.full_like(key, 1e300), key).masked_fill(
        key == INF, 1e299), dim=1, descending=True, stable=True).indices[:, :k]
    assert ids.dtype == torch.int32 and torch.equal(ids.cpu().long(), order)
    want = host.gather(1, order)
    assert values.dtype == z.dtype
    assert torch.equal(values.cpu().nan_to_num(7.0), want.nan_to_num(7.0))
    assert torch.equal(values.cpu().isnan(), want.isnan())
    ref = torch.logsumexp(host.double() / temperature, 1)
    got = lse.double().cpu()
    assert lse.dtype == F32 and torch.equal(got.isnan(), ref.isnan() | host.isnan().any(1) |
                                            (host == INF).any(1))
    fine = got.isfinite()
    assert torch.equal(ref[~fine & ~got.isnan()], got[~fine & ~got.isnan()])
    C = z.shape[1]
    S = ref[fine].abs().max() if bool(fine.any()) else torch.tensor(0.0)
    # the probabilities' relative error, and three roundings of the result's size
    assert bool(((got - ref)[fine].abs() <= (C / 32 + 64 + 4 * 40) * U + 3 * U * S).all())


SHAPES = [(1, 1, 1), (2, 2, 2), (3, 5, 3), (300, 7, 1), (7, 31, 8), (5, 32, 32), (64, 33, 5),
          (1000, 21, 8), (129, 150, 8), (70, 255, 3), (17, 257, 16), (9, 513, 16), (4, 1023, 33),
          (40, 1024, 1), (6, 2047, 64), (3, 4097, 64), (150, 5000, 7), (2, 20_001, 128),
          (5, 33_000, 50), (2, 70_001, 20), (1, 131_072, 128), (1, 262_144, 5)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("R,C,k", SHAPES)
def test_top_logits(R, C, k, dtype):
    for pad, offset, temperature in ((0, 0, 1.0), (3, 1, 0.5), (8, 8, 3.0)):
        z, _, _, _ = make(R, C, 1, dtype, seed=R + C, pad=pad, offset=offset)
        check_top(z, k, temperature)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("C,k", [(9, 9), (40, 6), (150, 8), (700, 40), (3000, 128), (40_000, 100)])
def test_top_logits_of_ties_masks_and_extremes(C, k, dtype):
    g = torch.Generator().manual_seed(C)
    low = torch.finfo(dtype).min
    rows = [torch.zeros(C), torch.full((C,), -INF), torch.full((C,), low),
            torch.randint(-2, 3, (C,), generator=g).float(),
            torch.where(torch.rand(C, generator=g) < 0.95, -INF, torch.randn(C, generator=g)),
            torch.where(torch.rand(C, generator=g) < 0.95, low, torch.randn(C, generator=g)),
            torch.arange(C).float() / C, -torch.arange(C).float() / C,
            torch.where(torch.arange(C) % 2 == 0, 0.0, -0.0),
            torch.cat([torch.full((C - k // 2,), -3.0), torch.full((k // 2,), 3.0)])]
    nan = torch.randn(C, generator=g)
    nan[C // 2] = math.nan
    inf = torch.randn(C, generator=g)
    inf[C - 1] = INF
    rows += [nan, torch.full((C,), math.nan), inf]
    check_top(torch.stack(rows).to(dtype).cuda(), k)


@pytest.mark.gpu
def test_top_logits_shapes_and_strides():
    z = torch.randn(2, 3, 4, 50, device="cuda")
    v, i, lse = sx.top_logits(z, 5)
    assert v.shape == i.shape == (2, 3, 4, 5) and lse.shape == (2, 3, 4)
    flat = sx.top_logits(z.view(-1, 50), 5)
    assert torch.equal(v.view(-1, 5), flat[0]) and torch.equal(lse.view(-1), flat[2])
    for view in (z.transpose(0, 3), z[..., ::2], z.permute(1, 0, 2, 3), z[:, :, :1].expand(2, 3, 6, 50)):
        a, b = sx.top_logits(view, 2), sx.top_logits(view.contiguous(), 2)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    v, i, lse = sx.top_logits(z[0, 0, 0], 1)
    assert v.shape == (1,) and lse.shape == ()
    v, i, lse = sx.top_logits(z[:0], 3)
    assert v.shape == (0, 3, 4, 3) and lse.shape == (0, 3, 4)


# ------------------------------------------------------------------ the loss and its gradient
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("R,C,K", SHAPES)
def test_loss_and_gradient(R, C, K, dtype):
    for n, (pad, offset, temperature, rest, cot) in enumerate(
            ((0, 0, 1.0, False, 1.0), (3, 1, 0.5, True, 1.0), (8, 8, 3.0, True, -0.75))):
        if C > 60_000 and n == 1:
            continue
        z, v, i, lse = make(R, C, K, dtype, seed=R + C + n, pad=pad, offset=offset,
                            temperature=temperature)
        w = torch.rand(R, generator=torch.Generator().manual_seed(n)).cuda() if n else None
        check(z, v, i if n else i.long(), lse if rest else None, cot, temperature=temperature,
              weights=w, denom=None if n < 2 else 2.5 * R)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("R,C,K", [(150, 2049, 40), (149, 9001, 8), (150, 20_001, 40),
                                   (149, 70_003, 8), (148, 70_000, 65), (148, 140_001, 33),
                                   (148, 150_000, 3)])
def test_many_long_rows(R, C, K, dtype):
    for n, (pad, rest) in enumerate(((0, True), (5, False))):
        z, v, i, lse = make(R, C, K, dtype, seed=C + n, pad=pad, temperature=2.0)
        i[::7, : K // 2] = -1
        i[3::7, -1] = i[3::7, 0]
        check(z, v, i, lse if rest else None, temperature=2.0)
        check_top(z, min(K, C), 2.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("C", [2049, 9001, 40_000, 140_000])
def test_top_logits_of_long_rows_in_any_order(C, dtype):
    """Rising, falling, constant and masked rows, and rows with few different values: the list of
    candidates overflows or holds nothing but equal logits."""
    g = torch.Generator().manual_seed(C)
    low = torch.finfo(dtype).min
    up = torch.arange(C).float() / 64
    rows = [up, up.flip(0), torch.zeros(C), torch.full((C,), -INF), torch.full((C,), low),
            torch.randint(0, 3, (C,), generator=g).float(),
            torch.where(torch.rand(C, generator=g) < 0.999, -INF, torch.randn(C, generator=g)),
            torch.where(torch.arange(C) > C - 100, 5.0, torch.randn(C, generator=g))]
    nan = torch.randn(C, generator=g)
    nan[C // 3::C // 5] = math.nan
    rows += [nan, torch.full((C,), math.nan)]
    few = torch.stack(rows).to(dtype).cuda()
    for k in (1, 20, 128):
        check_top(few, k)
        check_top(few.repeat(16, 1), k)  # enough rows for a CTA each


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16])
def test_many_short_rows_agree_with_few(dtype):
    """How rows are dealt out depends on their number: any number gives the same answers."""
    g = torch.Generator(device="cuda").manual_seed(11)
    for C in (1, 2, 7, 8, 31, 39, 40, 41, 64, 79, 80, 81, 97, 128, 159, 160, 161, 200, 256, 319,
              320, 321, 511, 512, 639, 640, 700, 1024, 1279, 1280, 1500, 2000, 2047, 2048):
        R = 12_000 + C
        z = torch.randn(R, C, device="cuda", generator=g).mul_(3).to(dtype)
        for K in {min(C, n) for n in (1, 5, 17, 40, 128)}:
            v, i, lse = sx.top_logits(z, K)
            part = slice(R - 150, R - 30)
            few = sx.top_logits(z[part].clone(), K)
            assert torch.equal(v[part], few[0]) and torch.equal(i[part], few[1])
            assert float((lse[part] - few[2]).abs().max()) <= 64 * U * 16
            t = torch.randn(R, K, device="cuda", generator=g)
            full = z.clone().requires_grad_()
            sub = z[part].clone().requires_grad_()
            d = 1.0 / 64
            a, = torch.autograd.grad(sx.distill_loss(full, t, i, denom=d), full)
            b, = torch.autograd.grad(sx.distill_loss(sub, t[part], i[part], denom=d), sub)
            # each within (4 S + C / 32 + 64) u of the probability, which is at most 64 here
            bar = 2 * 64 * (4 * 20 + C / 32 + 64) * U + 64 * torch.finfo(dtype).eps
            assert float((a[part].float() - b.float()).abs().max()) <= bar, (C, K)


@pytest.mark.gpu
@pytest.mark.parametrize("R,C", [(16_500, 131_072), (71_000_000, 31)])
def test_offsets_past_32_bits(R, C):
    z = torch.empty(R, C, device="cuda", dtype=BF16)
    z.normal_(generator=torch.Generator(device="cuda").manual_seed(12))
    v, i, lse = sx.top_logits(z, 3)
    last = slice(R - 5, R)
    few = sx.top_logits(z[last].clone(), 3)
    assert torch.equal(v[last], few[0]) and torch.equal(i[last], few[1])
    z.requires_grad_()
    g, = torch.autograd.grad(sx.distill_loss(z, v, i, lse + 0.5, denom=5.0), z)
    ref, tol = oracle(z.detach()[last], v[last], i[last], lse[last] + 0.5, denom=5.0)[1::2]
    err = (g[last].double().cpu() - ref).abs()
    assert bool((err <= rounded(tol, ref, BF16)).all())


@pytest.mark.gpu
def test_saved_tensors_may_move():
    """The backward takes what autograd saved, wherever it has put it meanwhile."""
    z, v, i, lse = make(40, 300, 5, F32, seed=41, pad=4)
    leaf = z.detach().requires_grad_()
    with torch.autograd.graph.save_on_cpu():
        loss = sx.distill_loss(leaf, v, i, lse)
    del v, i, lse
    first, = torch.autograd.grad(loss, leaf, retain_graph=True)
    torch.empty(1 << 20, device="cuda").fill_(math.nan)
    again, = torch.autograd.grad(loss, leaf)
    assert float((first - again).abs().max()) <= 8 * U


@pytest.mark.gpu
def test_first_call_of_a_process_may_be_captured():
    import subprocess
    import sys
    from pathlib import Path

    code = """
import torch, splax_b200 as sx
z = torch.randn(300, 5000, device='cuda', requires_grad=True)
s = torch.randn(300, 50, device='cuda', requires_grad=True)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = []
    for x in (z, s, z[:9]):
        v, i, lse = sx.top_logits(x, 4)
        loss = sx.distill_loss(x, v, i, lse, temperature=1.0)
        out += [v, i, lse, loss] + list(torch.autograd.grad(loss, x))
g.replay()
torch.cuda.synchronize()
for n, x in enumerate((z, s, z[:9])):
    v, i, lse = sx.top_logits(x, 4)
    loss = sx.distill_loss(x, v, i, lse, temperature=1.0)
    want = [v, i, lse, loss] + list(torch.autograd.grad(loss, x))
    assert all(torch.equal(a, b) for a, b in zip(out[5 * n:], want)), n
print('ok')
"""
    res = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                         cwd=Path(__file__).resolve().parents[1])
    assert res.returncode == 0 and res.stdout.strip().endswith("ok"), res.stderr[-2000:]


@pytest.mark.gpu
def test_without_grad_mode_no_gradient_is_made():
    z, v, i, lse = make(2000, 512, 4, F32, seed=51)
    leaf = z.clone().requires_grad_()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.max_memory_allocated()
    with torch.no_grad():
        loss = sx.distill_loss(leaf, v, i, lse)
    assert not loss.requires_grad
    assert torch.cuda.max_memory_allocated() - before < leaf.numel() * 4


@pytest.mark.gpu
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("C", [11, 150, 1500, 9000, 70_000])
def test_masked_rows_entries_and_classes(C, dtype, rest):
    K = 6
    z, v, i, lse = make(14, C, K, dtype, seed=C)
    i[0, :] = -1  # no entry at all
    i[1, 2:] = -1
    i[2, 0] = C  # outside the classes
    i[2, 1] = 2**31 - 1
    i[2, 2] = -(2**31)
    i[3, 1] = i[3, 0]  # the same class twice, and three times
    i[4, 3] = i[4, 5] = i[4, 0]
    v[5, :] = -INF
    v[6, 1:3] = -INF
    z[7, i[7, 0].item()] = z[7].float().max().to(dtype)
    others = torch.ones(C, dtype=torch.bool, device="cuda")
    others[i[8].long()] = False
    z[8, others] = -INF  # the student gives nothing outside the entries
    z[9, :] = -INF
    z[10, others] = torch.finfo(dtype).min
    z[11, :] = torch.finfo(dtype).min
    w = torch.ones(14, device="cuda")
    w[12] = 0.0
    z[12, C // 2] = math.nan  # masked by its weight
    v[12, 0] = math.nan
    lse[13] = -INF if rest else lse[13]
    check(z, v, i, lse if rest else None, weights=w)


@pytest.mark.gpu
@pytest.mark.parametrize("R,C", [(40, 9), (3, 5000), (200, 5000)])
def test_rows_without_entries_get_exactly_nothing(R, C):
    z, v, i, lse = make(R, C, 4, F32, seed=17)
    i[:] = -1
    i[1, 2] = C
    leaf = z.detach().requires_grad_()
    for t in (None, lse):
        loss = sx.distill_loss(leaf, v, i, t)
        assert loss.item() == 0.0
        assert not bool(torch.autograd.grad(loss, leaf)[0].any())


@pytest.mark.gpu
@pytest.mark.parametrize("C", [5, 300, 9000])
def test_nan_and_infinite_losses_stay_visible(C):
    z, v, i, lse = make(4, C, 2, F32, seed=3)
    for change in (lambda x: x[1].fill_(math.nan), lambda x: x[1, C - 1:].fill_(math.nan),
                   lambda x: x[1, :1].fill_(INF)):
        bad = z.clone()
        change(bad)
        bad.requires_grad_()
        loss = sx.distill_loss(bad, v, i, lse)
        assert math.isnan(loss.item())
        g, = torch.autograd.grad(loss, bad)
        assert bool(g[1].isnan().all()) and bool(g[[0, 2, 3]].isfinite().all())
    # a class that the teacher has and the student masks: an infinite divergence
    bad = z.clone()
    bad[2, i[2, 0].item()] = -INF
    bad.requires_grad_()
    loss = sx.distill_loss(bad, v, i)
    assert loss.item() == INF
    g, = torch.autograd.grad(loss, bad)
    ref = oracle(bad.detach(), v, i)[1]
    assert bool(g.isfinite().all()) and float((g.cpu() - ref).abs().max()) <= 1e-5


@pytest.mark.gpu
def test_all_classes_named_drops_the_rest():
    z, v, i, lse = make(50, 8, 8, F32, seed=5)
    check(z, v, i, lse)
    check(z, v, i, lse - 0.25)  # an inconsistent log-sum-exp: a mass above one
    check(z, v, i, lse + 0.5)


@pytest.mark.gpu
def test_sharp_and_agreeing_distributions():
    """A student that gives the others 1e-30 still has an accurate rest term and gradient."""
    z, v, i, lse = make(20, 400, 4, F32, seed=6, spread=1.0)
    sharp = z.clone()
    sharp.scatter_add_(1, i.long(), torch.full((20, 4), 70.0, device="cuda"))
    check(sharp, v, i, lse)
    check(sharp, v, i)
    same = torch.zeros(20, 400, device="cuda").copy_(z)
    vv, ii, ll = sx.top_logits(same, 4)
    check(same, vv, ii, ll)


@pytest.mark.gpu
@pytest.mark.parametrize("R,C", [(40, 77), (20, 5000), (160, 5000)])
@pytest.mark.parametrize("low", [-1.1e9, -1e10, -1e30, 1e10])
def test_rows_masked_by_large_finite_numbers(R, C, low):
    """A whole row, or most of it, of one number whose product with log2(e) has no exact fp32
    neighbourhood: the row is uniform over those, and what lies far above takes everything."""
    g = torch.Generator().manual_seed(C)
    z = torch.randn(R, C, generator=g)
    z[::2] = low
    z[1::4, 5:] = low
    z[1, :] = torch.where(torch.arange(C) % 3 == 0, low, -math.inf)
    z = z.cuda()
    i = torch.randint(0, C, (R, 3), generator=g).int().cuda()
    v = torch.randn(R, 3, generator=g).cuda()
    check_top(z, 4)
    leaf = z.clone().requires_grad_()
    weights = torch.zeros(R, device="cuda")
    weights[::2] = 1.0
    loss = sx.distill_loss(leaf, v, i, weights=weights, denom=1.0)
    grad, = torch.autograd.grad(loss, leaf)
    # the uniform rows against rows of zeros, which have the same softmax: q = 1 / C either way. The
    # loss adds and subtracts p |low| in 64 bits, some four times an entry and half the rows: below
    # |low| 2^-50 R in all. Beyond 1e12 that is all it promises.
    ref, ref_grad, tol, grad_tol = oracle(torch.zeros_like(z), v, i, weights=weights, denom=1.0)
    assert abs(loss.item() - ref) <= tol + abs(low) * 2.0**-50 * R, (loss.item(), ref, tol)
    err = (grad.double().cpu() - ref_grad).abs()
    assert bool((err <= rounded(grad_tol, ref_grad, F32)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("R,C", [(40, 77), (20, 5000), (160, 5000)])
@pytest.mark.parametrize("middle", [2907271.0, -2907271.0, 2907000.0, 2908000.0])
def test_a_common_offset_changes_nothing(R, C, middle):
    """Steps of 1/4 around numbers of about 2^22 / log2(e), exact in fp32: the softmax is that of the
    steps alone, on either side of the place where references change their form and across it."""
    g = torch.Generator().manual_seed(R + C)
    steps = torch.randint(-20, 21, (R, C), generator=g).float() / 4
    steps[0] = steps[0].sort().values  # a rising row: the running maximum crosses
    z = (steps + middle).cuda()
    assert bool((z.cpu().double() == steps.double() + middle).all())
    i = torch.randint(0, C, (R, 6), generator=g).int().cuda()
    v = torch.randn(R, 6, generator=g).cuda()
    # twice the tolerance: a difference of logits is multiplied by the first part of log2(e) / tau
    # alone, which is up to 2 u off, 2 u |x - m| <= 4 S u more in the exponent
    ref, ref_grad, tol, grad_tol = oracle(steps, v, i)
    leaf = z.clone().requires_grad_()
    loss = sx.distill_loss(leaf, v, i)
    grad, = torch.autograd.grad(loss, leaf)
    # the loss's own 64-bit differences of numbers of 3e6: 2^-30 each
    assert abs(loss.item() - ref) <= 2 * tol + 2.0**-28, (loss.item(), ref, tol)
    err = (grad.double().cpu() - ref_grad).abs()
    bar = rounded(2 * grad_tol, ref_grad, F32)
    assert bool((err <= bar).all()), float((err / bar).max())
    check_top(z, 5)


@pytest.mark.gpu
def test_types_and_shapes_of_the_teacher():
    z, v, i, lse = make(12, 77, 5, F32, seed=7)
    ref = sx.distill_loss(z, v.half(), i, lse)
    assert torch.equal(ref, sx.distill_loss(z, v.half().float(), i.long(), lse))
    assert torch.equal(ref, sx.distill_loss(z.view(3, 4, 77), v.half().view(3, 4, 5),
                                            i.view(3, 4, 5), lse.view(3, 4)))
    t = torch.stack([v, v], -1)[..., 0]  # a strided teacher
    assert torch.equal(sx.distill_loss(z, t, i), sx.distill_loss(z, v, i))
    one = sx.distill_loss(z[3], v[3], i[3], lse[3], weights=torch.tensor(2.0, device="cuda"))
    ref1, _, tol, _ = oracle(z[3:4], v[3:4], i[3:4], lse[3:4], weights=torch.tensor([2.0]))
    assert abs(one.item() - ref1) <= tol
    wide = i.long() + 2**32  # outside the classes, although their low halves are inside
    assert sx.distill_loss(z, v, wide).item() == 0.0
    empty = sx.distill_loss(z[:0].requires_grad_(), v[:0], i[:0], denom=3.0)
    assert empty.item() == 0.0
    # a student shared by several rows: its gradient is their sum
    row = z[:1].clone().requires_grad_()
    g, = torch.autograd.grad(sx.distill_loss(row.expand(12, 77), v, i, lse), row)
    full = z[:1].expand(12, 77).contiguous().requires_grad_()
    h, = torch.autograd.grad(sx.distill_loss(full, v, i, lse), full)
    assert float((g - h.sum(0, keepdim=True)).abs().max()) <= 12 * U


@pytest.mark.gpu
def test_backward_runs_again_and_refuses_a_second_order():
    z, v, i, lse = make(30, 200, 6, F32, seed=8)
    leaf = z.clone().requires_grad_()
    (0.5 * sx.distill_loss(leaf, v, i, lse)).backward()
    first = leaf.grad.clone()
    loss = sx.distill_loss(leaf, v, i, lse)
    (0.25 * loss).backward(retain_graph=True)
    (0.25 * loss).backward()
    assert float((leaf.grad - 2 * first).abs().max()) <= 8 * U * float(first.abs().max())
    loss = sx.distill_loss(leaf, v, i, lse)
    g, = torch.autograd.grad(loss, leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    loss = sx.distill_loss(leaf, v, i, lse)
    with torch.no_grad():
        leaf.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.gpu
@pytest.mark.parametrize("R,C", [(5000, 33), (700, 3001), (600, 40_000)])
def test_results_do_not_depend_on_the_order(R, C):
    z, v, i, lse = make(R, C, 5, BF16, seed=9)
    leaf = z.clone().requires_grad_()

    def once():
        loss = sx.distill_loss(leaf, v, i, lse)
        return [loss.detach(), torch.autograd.grad(loss, leaf)[0], *sx.top_logits(z, 5)]

    first = once()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))


@pytest.mark.gpu
@pytest.mark.parametrize("C", [150, 40_000])
def test_two_captured_graphs_and_side_streams(C):
    """Two captured steps replayed at once on two streams, each on its own new inputs."""
    sets = []
    for n in range(2):
        z, v, i, lse = make(64, C, 5, BF16, seed=20 + n)
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        leaf = z.clone().requires_grad_()
        with torch.cuda.graph(graph, stream=stream):
            loss = sx.distill_loss(leaf, v, i, lse)
            g, = torch.autograd.grad(3.0 * loss, leaf)
            top = sx.top_logits(leaf, 4)
        sets.append((leaf, v, i, lse, stream, graph, loss, g, top))
    for step in range(3):
        for leaf, *_ in sets:
            with torch.no_grad():
                leaf.copy_(torch.randn(64, C, device="cuda") * 2)
        torch.cuda.synchronize()
        for *_, stream, graph, _, _, _ in sets:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for leaf, v, i, lse, _, _, loss, g, top in sets:
            fresh = leaf.detach().clone().requires_grad_()
            want = sx.distill_loss(fresh, v, i, lse)
            assert torch.equal(loss, want)
            assert torch.equal(g, torch.autograd.grad(3.0 * want, fresh)[0])
            assert all(torch.equal(a, b) for a, b in zip(top, sx.top_logits(fresh, 4)))


@pytest.mark.gpu
def test_a_backward_replayed_apart_from_its_forward():
    """The forward is eager, the backward captured and replayed: each replay gives the gradient."""
    z, v, i, lse = make(40, 90, 5, F32, seed=31)
    leaf = z.clone().requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    cot = torch.tensor(0.5, device="cuda")
    with torch.cuda.stream(side):
        loss = sx.distill_loss(leaf, v, i, lse)
    side.synchronize()
    with torch.cuda.graph(graph, stream=side):
        g, = torch.autograd.grad(loss, leaf, cot, retain_graph=True)
    want = oracle(z, v, i, lse)[1] * 0.5
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert float((g.cpu() - want).abs().max()) <= 1e-6 * float(want.abs().max()) + 40 * U / 40


@pytest.mark.gpu
def test_semantic_scene_trains_against_a_teachers_top_logits():
    """The set as it is used: class scores of gaussians rendered three channels at a time, a
    teacher's top logits per pixel, the loss, its gradient through the blend, Adam."""
    from conftest import cam, random_scene, viewmat

    H, W, C, K = 48, 64, 9, 4
    m, s, q, c, op, bg = random_scene(400, 2)
    t = lambda x: torch.tensor(x, device="cuda")  # noqa: E731
    geo = sx.project(t(m), t(s), t(q), t(viewmat()), opacities=t(op), **cam(H, W))
    xys, depths, radii, conics, num, cum = geo

    def scores(features):
        black = torch.zeros(3, device="cuda")
        views = [sx.rasterize(features[:, a:a + 3].contiguous(), t(op), black, xys, depths, radii,
                              conics, cum, img_shape=(H, W)) for a in range(0, C, 3)]
        return torch.cat(views, -1)

    g = torch.Generator(device="cuda").manual_seed(4)
    with torch.no_grad():
        teacher = scores(torch.randn(400, C, device="cuda", generator=g) * 4).view(H, W, C)
    values, ids, lse = sx.top_logits(teacher, K)
    mask = (torch.rand(H, W, device="cuda", generator=g) < 0.8).float()
    feat = (torch.randn(400, C, device="cuda", generator=g) * 0.1).requires_grad_()
    opt = sx.Adam([feat], 0.1)
    img = scores(feat).view(H, W, C)
    loss = sx.distill_loss(img, values, ids, lse, weights=mask)
    ref, ref_grad, tol, grad_tol = oracle(img.detach().view(-1, C), values.view(-1, K),
                                          ids.view(-1, K), lse.view(-1), weights=mask.view(-1))
    assert abs(loss.item() - ref) <= tol
    got, = torch.autograd.grad(loss, feat, retain_graph=True)
    want, = torch.autograd.grad(img, feat, ref_grad.float().cuda().view(H, W, C))
    # both go through the same blend, whose atomics add in any order: 1e-4 of the largest gradient
    assert float((got - want).abs().max()) <= 1e-4 * float(want.abs().max())
    loss = sx.distill_loss(scores(feat).view(H, W, C), values, ids, lse, weights=mask)
    loss.backward()
    before = feat.detach().clone()
    opt.step()
    assert bool(feat.isfinite().all()) and not torch.equal(feat.detach(), before)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("C,K", [(3, 2), (3, 16), (19, 30), (40, 128), (150, 8), (513, 64),
                                 (1500, 128)])
def test_classes_that_many_entries_name(C, K, dtype):
    """All lanes of a row read the logits of the same two classes, and each marks their places."""
    z, v, _, _ = make(90, C, 1, dtype, seed=C + K)
    g = torch.Generator().manual_seed(K)
    v = torch.randn(90, K, generator=g).to(dtype).cuda()
    ids = torch.randint(0, 2, (90, K), generator=g).mul(C - 1).int().cuda()
    ids[::9, K // 2:] = -1
    lse = (torch.logsumexp(v.double(), 1) + 0.5).float()
    check(z, v, ids)
    check(z, v, ids, lse)


def test_rescaling_is_refused_as_the_gradient_is():
    lib = _lib.load()
    P = ctypes.c_void_p
    good = P(1 << 20)
    for bad in (dict(z=None), dict(dtype=3), dict(stride=8), dict(k=0), dict(bits=8),
                dict(denom=0.0), dict(cot=None), dict(cot=P(2)), dict(grad=None), dict(grad=P(1))):
        a = {**dict(z=good, dtype=1, stride=9, bits=32, k=3, denom=1.0, cot=good, grad=good), **bad}
        rc = lib.splax_distill_rescale_grad(a["z"], a["dtype"], 2, 9, a["stride"], good, 0, good,
                                            a["bits"], None, a["k"], None, 1.0, a["denom"],
                                            a["cot"], a["grad"], None)
        assert rc == _lib.SPLAX_ERR_INVALID_ARGUMENT, bad
        assert lib.splax_last_error().decode().startswith("distill_rescale_grad")


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [65536.0, 0.7])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("R,C", [(120, 101), (70, 513), (9, 5000), (160, 5000), (160, 20_001)])
def test_a_loss_scale_reaches_the_gradient_before_its_rounding(R, C, dtype, scale):
    """Rows of a large view under a loss scale: without it most of the fp16 gradient vanishes, with it
    nothing may be missing, and every backward of a graph gives the same."""
    denom, cot = 2_000_000.0, torch.tensor(scale, device="cuda")
    scale = cot.item()
    z, v, i, lse = make(R, C, 6, dtype, seed=R + C, pad=3)
    leaf = z.detach().requires_grad_()
    for t in (None, lse):
        _, ref, _, tol = oracle(z, v, i, t, denom=denom)
        ref, tol = ref * scale, tol * scale
        loss = sx.distill_loss(leaf, v, i, t, denom=denom)
        first, = torch.autograd.grad(loss, leaf, cot, retain_graph=True)
        again, = torch.autograd.grad(loss, leaf, cot)
        if dtype == F32:  # scaled after its rounding: one more
            tol = tol + ref.abs() * U
        for got in (first, again):
            err, bar = (got.double().cpu() - ref).abs(), rounded(tol, ref, dtype)
            assert not bool((err > bar).any()), float((err / bar).max())
        if dtype != F32:
            assert torch.equal(first, again)
        # a cotangent of one leaves what the forward made
        loss = sx.distill_loss(leaf, v, i, t, denom=float(R))
        first, = torch.autograd.grad(loss, leaf, retain_graph=True)
        assert torch.equal(first, torch.autograd.grad(loss, leaf)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("R,C", [(64, 101), (12, 9000), (160, 9000)])
def test_a_captured_backward_follows_its_cotangent(R, C, dtype):
    z, v, i, lse = make(R, C, 5, dtype, seed=C)
    leaf = z.clone().requires_grad_()
    cot = torch.ones((), device="cuda")
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        g, = torch.autograd.grad(sx.distill_loss(leaf, v, i, lse, denom=1e6), leaf, cot)
    for value in (1.0, 4096.0, 1.0, 65536.0, 0.0):
        cot.fill_(value)
        graph.replay()
        torch.cuda.synchronize()
        fresh = leaf.detach().clone().requires_grad_()
        want, = torch.autograd.grad(sx.distill_loss(fresh, v, i, lse, denom=1e6), fresh, cot)
        assert torch.equal(g, want)


def careful(z, v, ids, lse_t=None, temperature=1.0, denom=None):
    """As ``oracle``, for rows of numbers beside which 64 bits have no room for a logarithm: logits
    are subtracted from one another before anything else, and the error of a probability goes by the
    differences that leave one (of what is 200 below the maximum, e^-66 at most is left). Rows that
    count nothing have no place here."""
    z, v, ids = z.double().cpu(), v.double().cpu(), ids.long().cpu()
    R, C = z.shape
    tau, denom = float(temperature), float(R if denom is None else denom)
    loss, loss_tol, grad, tol = 0.0, 0.0, torch.zeros_like(z), torch.zeros_like(z)
    for r in range(R):
        valid = (ids[r] >= 0) & (ids[r] < C)
        at = ids[r][valid]
        a = (v[r][valid] - v[r][valid].max()) / tau
        log_p = a - torch.logsumexp(a, 0) if lse_t is None else \
            v[r][valid] / tau - lse_t[r].double().cpu()
        d = (z[r] - z[r].max()) / tau
        log_q = d - torch.logsumexp(d, 0)
        p, q = log_p.exp(), log_q.exp()
        named = torch.zeros(C, dtype=torch.bool)
        named[at] = True
        o = z[r][~named]
        log_share = torch.full((C,), -INF, dtype=torch.float64)
        log_qo = -INF
        if o.numel() and float(o.max()) > -INF:
            do = (o - o.max()) / tau
            log_share[~named] = do - torch.logsumexp(do, 0)
            log_qo = float((o.max() - z[r].max()) / tau + torch.logsumexp(do, 0) -
                           torch.logsumexp(d, 0))
        P = float(p.sum())
        rho = max(0.0, 1.0 - P) if lse_t is not None and log_qo > -INF else 0.0
        size = torch.cat([d, a, log_share * 1.0,
                          torch.zeros(1) if lse_t is None else v[r][valid] / tau])
        size = size[size.abs() <= min(200.0, 200.0 / tau)]
        e = (4 * float(size.abs().max()) + C / 32 + 64) * U
        live = p > 0
        terms = p[live] * (log_p[live] - log_q[at[live]])
        row, bound = float(terms.sum()), e * float((terms.abs() + p[live]).sum())
        if lse_t is not None and log_qo > -INF:
            if rho > 0:
                row += rho * (math.log(rho) - log_qo)
            bound += e * max(P, rho) * (2 + abs(math.log(max(rho, e))) + abs(log_qo))
        g = (P + rho) * q
        g_tol = e * (P + rho) * q
        share = log_share[~named].exp()
        g[~named] = ((P + rho) * math.exp(log_qo) - rho) * share
        g_tol[~named] = e * ((P + rho) * q[~named] + (rho + (P if lse_t is not None else 0)) * share)
        for c, x in zip(at.tolist(), p.tolist()):
            g[c] -= x
            g_tol[c] += e * x
        k = tau / denom
        grad[r], tol[r] = g * k, g_tol * k + 4 * U * g.abs() * k
        loss += tau * k * row
        loss_tol += tau * k * bound
    return loss, grad, loss_tol + 2 * U * abs(loss), tol


def check_carefully(z, v, i, lse=None, **kw):
    ref, ref_grad, tol, grad_tol = careful(z, v, i, lse, **kw)
    leaf = z.detach().requires_grad_()
    loss = sx.distill_loss(leaf, v, i, lse, **kw)
    with torch.no_grad():
        assert torch.equal(loss, sx.distill_loss(z, v, i, lse, **kw))
    assert abs(loss.item() - ref) <= tol, (loss.item(), ref, tol)
    grad, = torch.autograd.grad(loss, leaf)
    err = (grad.double().cpu() - ref_grad).abs()
    bar = rounded(grad_tol, ref_grad, z.dtype)
    assert not bool((err > bar).any()), float((err / bar).max())


def test_the_careful_oracle_is_the_oracle_where_that_holds():
    g = torch.Generator().manual_seed(2)
    z, t = torch.randn(6, 11, generator=g), torch.randn(6, 11, generator=g)
    v, i = t.topk(4, 1)
    i[1, 1], i[2, 2] = i[1, 0], -1
    for lse in (None, torch.logsumexp(t.double() / 1.5, 1)):
        a, b = oracle(z, v, i, lse, 1.5), careful(z, v, i, lse, 1.5)
        assert abs(a[0] - b[0]) <= 1e-14 and float((a[1] - b[1]).abs().max()) <= 1e-14


def masked_rows(kind, R, C, low, dtype, g):
    """(logits, classes of three entries) of rows of which `low` takes all or a part."""
    z = torch.randn(R, C, generator=g)
    i = torch.stack([torch.randperm(C, generator=g)[:3] for _ in range(R)])
    if kind == "all":
        z[:] = low
    elif kind == "all but the entries":
        z = torch.full_like(z, low).scatter_(1, i, z)
    elif kind == "the entries":
        z = z.scatter_(1, i, low)
    elif kind == "all, others gone":
        z[:] = low
        z[torch.rand(R, C, generator=g) < 0.7] = -INF
        z.scatter_(1, i, low)
    return z.to(dtype).cuda(), i.int().cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("R,C", [(40, 11), (60, 150), (8, 1500), (20, 5000), (160, 5000)])
@pytest.mark.parametrize("kind", ["all", "all but the entries", "the entries", "all, others gone"])
@pytest.mark.parametrize("dtype,low", [(F32, torch.finfo(F32).min), (BF16, torch.finfo(BF16).min),
                                       (F16, torch.finfo(F16).min), (F32, -1e12), (F32, 1e10),
                                       (F32, 3e30), (BF16, -1e30)])
def test_loss_of_rows_masked_by_large_finite_numbers(dtype, low, kind, R, C):
    """A uniform row, one where few classes stand above the mask, and one where entries that the
    teacher gives a probability are masked: there the loss itself is as large as the mask."""
    g = torch.Generator().manual_seed(R + C)
    z, i = masked_rows(kind, R, C, low, dtype, g)
    v = torch.randn(R, 3, generator=g).cuda()
    denom = 1000.0 * R  # a loss of the lowest value's size, times a temperature, in fp32
    for tau in (1.0, 1.5, 3.0):
        lse = (torch.logsumexp(v.double() / tau, 1) + 0.25).float()
        check_carefully(z, v, i, temperature=tau, denom=denom)
        check_carefully(z, v, i, lse, temperature=tau, denom=denom)


@pytest.mark.gpu
@pytest.mark.parametrize("R,C", [(40, 11), (60, 150), (20, 5000), (160, 5000)])
@pytest.mark.parametrize("dtype,low", [(F32, torch.finfo(F32).min), (BF16, torch.finfo(BF16).min),
                                       (F32, -1e12), (F32, 1e30)])
def test_a_teachers_entries_masked_by_large_finite_numbers(dtype, low, R, C):
    """Renormalised entries that are all of the mask: uniform probabilities, whose logarithms count."""
    z, v, i, _ = make(R, C, 5, F32, seed=R + C)
    v = v.to(dtype)
    v[:] = low
    v[::3, 2] = -INF
    for tau in (1.0, 1.5, 3.0):
        check_carefully(z, v, i, temperature=tau)
    if low < 0:
        v[1::3, 0] = 1.0  # one entry above the mask
        check_carefully(z, v, i, temperature=1.5)


@pytest.mark.gpu
@pytest.mark.parametrize("C", [9, 150, 5000])
def test_one_row_of_any_stride(C):
    """The stride between the rows of a single row is never used, however large it is."""
    z, v, i, _ = make(1, C, 4, F32, seed=C)
    lib, s = _lib.load(), torch.cuda.current_stream().cuda_stream
    work = torch.empty(workspace_bytes(), dtype=torch.uint8, device="cuda")
    outs = []
    for stride in (C, C + 1, 1 << 40, (1 << 62) + 4, (1 << 63) - 1):
        values, ids, lse = torch.empty_like(v), torch.empty_like(i), torch.empty(1, device="cuda")
        loss, grad = torch.empty((), device="cuda"), torch.empty_like(z)
        _lib.check(lib.splax_top_logits(z.data_ptr(), 0, 1, C, stride, 4, 1.0, values.data_ptr(),
                                        ids.data_ptr(), lse.data_ptr(), s))
        _lib.check(lib.splax_distill_loss_and_grad(
            z.data_ptr(), 0, 1, C, stride, v.data_ptr(), 0, i.data_ptr(), 32, None, 4, None, 1.0,
            1.0, work.data_ptr(), loss.data_ptr(), grad.data_ptr(), s))
        outs.append((values, ids, lse, loss, grad))
    for other in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], other))


def workspace_bytes():
    from splax_b200 import _distill

    return _distill.WORKSPACE


@pytest.mark.gpu
@pytest.mark.parametrize("R,C", [(40, 150), (20, 5000), (160, 5000)])
def test_temperatures_near_their_limits(R, C):
    """Entries of the lowest value whose quotient by the temperature overflows; and a temperature whose scale leaves almost nothing beyond its first 24 bits."""
    g = torch.Generator().manual_seed(C)
    for tau in (3e-9, 7e-9, 1.1e-8, 1.3e-8, 1.7e-8, 1.9e-8):
        z = (torch.randn(R, C, generator=g) * tau).cuda()
        v = (torch.randn(R, 3, generator=g) * tau).cuda()
        v[:, 1] = torch.finfo(F32).min
        i = torch.stack([torch.randperm(C, generator=g)[:3] for _ in range(R)]).int().cuda()
        lse = (torch.logsumexp(v[:, ::2].double() / tau, 1) + 0.25).float()
        check_carefully(z, v, i, lse, temperature=tau, denom=tau * tau)
        check_carefully(z, v, i, temperature=tau, denom=tau * tau)
    taus = [math.log2(math.e) / torch.tensor(1.5e-30).item()]  # of a float, and a hair beside it
    for _ in range(16):
        taus.append(math.nextafter(taus[-1], 0.0))
    z = torch.randn(R, C, generator=g)
    z[:, ::3] = -INF
    z = z.cuda()
    for tau in taus:
        values, ids, lse = sx.top_logits(z, 4, temperature=tau)
        want = math.log(C - (C + 2) // 3)  # at such a temperature all classes are alike
        assert float((lse - want).abs().max()) <= (C / 32 + 64) * U + 3 * U * want
        loss = sx.distill_loss(z, values, ids, temperature=tau, denom=1e30)
        assert math.isfinite(loss.item())


@pytest.mark.gpu
def test_the_profile_counts_the_kernels_that_were_launched():
    def kernels(call):
        _lib.profile_reset()
        _lib.profile_enable(True)
        try:
            call()
        finally:
            _lib.profile_enable(False)
        torch.cuda.synchronize()
        return _lib.profile_report()["kernels"]["loss"]["kernels"]

    for R, C, loss_kernels in ((1, 9, 1), (3000, 9, 2), (1, 5000, 1), (9, 5000, 2), (200, 5000, 2),
                               (0, 9, 1)):
        z, v, i, _ = make(R, C, 3, F16, seed=R)
        leaf = z.clone().requires_grad_()
        with torch.no_grad():
            assert kernels(lambda: sx.top_logits(z, 3)) == (1 if R else 0)
            assert kernels(lambda: sx.distill_loss(z, v, i, denom=2.0)) == loss_kernels
        loss = sx.distill_loss(leaf, v, i, denom=2.0)
        for _ in range(2):
            assert kernels(lambda: torch.autograd.grad(loss, leaf, retain_graph=True)) == min(R, 1)
