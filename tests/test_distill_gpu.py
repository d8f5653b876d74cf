"""Distillation from a teacher's largest logits against plain 64-bit math, at the sizes where its kernels change shape and at its edges.

Tolerances: an fp32 probability carries the rounding of z - max, of its product with log2 e / T (relative 2^-24 each, so 2^-23 |z - max| / T absolute
in the exponent) and a few units of 2^-24 for exp2, the sum and the product; a bf16 gradient half a step, 2^-8, more."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -8
U32 = 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available()
    from savit_amd import ops as o

    return o


def ref_distill(z, top, at, T, soft, lse, labels, hard, smooth, weight, grad_scale):
    """64-bit loss and gradient, and bounds on the fp32 roundings of both."""
    R, C = z.shape
    zd = z.double().detach().requires_grad_()
    P = torch.zeros(R, C, dtype=torch.float64, device=z.device)
    ok = (at >= 0) & (at < C)
    t = torch.where(ok, top.double() / T, -math.inf)
    j = torch.where(ok, at, 0).long()
    named = torch.zeros(R, C, dtype=torch.float64, device=z.device).scatter_add_(1, j, ok.double()) > 0
    if lse is None:
        m = t.amax(1, keepdim=True) if t.shape[1] else torch.full((R, 1), -math.inf, device=z.device, dtype=torch.float64)
        e = torch.where(ok, (t - torch.where(m == -math.inf, 0.0, m)).exp(), 0.0)
        s = e.sum(1, keepdim=True)
        p = e / torch.where(s == 0, 1.0, s)
        P.scatter_add_(1, j, p)
    else:
        p = torch.where(ok, (t - lse.double()[:, None]).exp(), 0.0)
        P.scatter_add_(1, j, p)
        others = (~named).sum(1, keepdim=True)
        left = torch.where(others > 0, (1 - p.sum(1, keepdim=True)).clamp(min=0), 0.0)
        P = torch.where(named, P, left / others.clamp(min=1))
    lq = torch.log_softmax(zd / T, 1)
    terms = torch.where(P > 0, torch.xlogy(P, P) - P * lq, 0.0)
    loss = soft * T * T * terms.sum(1)
    lz = torch.log_softmax(zd, 1)
    y = torch.zeros_like(P)
    if labels is not None and hard:
        good = (labels >= 0) & (labels < C)
        y = smooth / C + (1 - smooth) * torch.zeros_like(P).scatter_(1, torch.where(good, labels, 0).long()[:, None], 1.0)
        y = torch.where(good[:, None], y, 0.0)
        loss = loss - hard * torch.where(y > 0, y * lz, 0.0).sum(1)
    w = torch.ones(R, device=z.device) if weight is None else weight
    loss = torch.where(w == 0, 0.0, loss * w.double())
    with torch.no_grad():
        gs = grad_scale * w.double()[:, None]
        S = P.sum(1, keepdim=True)
        q, sz = lq.exp(), lz.exp()
        on = y.sum(1, keepdim=True)  # 1, or 0 where the row has no hard term
        dz = gs * (soft * T * (S * q - P) + hard * (on * sz - y))
        dist = (zd - zd.amax(1, keepdim=True)).abs()
        dist = torch.where(dist == math.inf, 0.0, dist)
        er = U32 * (24 + 4 * dist / T + 4 * (q * dist / T).sum(1, keepdim=True))
        eh = U32 * (24 + 4 * dist + 4 * (sz * dist).sum(1, keepdim=True))
        tol = gs.abs() * (soft * T * (S * q * er + 4 * U32 * P) + hard * (on * sz * eh + 4 * U32 * y))
        # the loss is joined in 64 bits; what fp32 leaves in it is the normaliser's relative error (its sum's terms, each er) and, with mass left
        # over or smoothing, a chain of fp32 additions of the logits (a thread's share, then a tree)
        ls = soft * T * T * S[:, 0] * (q * er).sum(1) + hard * on[:, 0] * (sz * eh).sum(1)
        finite = torch.where(zd.isfinite(), zd.abs(), 0.0)
        if lse is not None or smooth:
            ls = ls + (soft * T * (P.sum(1) if lse is not None else 0.0) + hard * smooth) * finite.mean(1) * U32 * 512
        ltol = w.double().abs() * (ls + 2 * U32 * loss.abs() + 1e-12)
    dz = torch.where(w[:, None] == 0, 0.0, dz)
    return loss.detach(), dz, ltol, torch.where(w[:, None] == 0, 0.0, tol)


def make(R, C, K, seed, dtype, spread=2.0, lse=False, T=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = (torch.randn(R, C, generator=g, device="cuda") * spread).to(dtype)
    t = z.float() + torch.randn(R, C, generator=g, device="cuda")
    top, at = t.topk(K, dim=1) if K else (t[:, :0], t[:, :0].long())
    total = torch.logsumexp(t / T, 1) if lse else None
    labels = torch.randint(0, C, (R,), generator=g, device="cuda", dtype=torch.int32)
    return z, top.contiguous(), at.int().contiguous(), total, labels


def run_and_check(ops, z, top, at, T, soft, lse, labels, hard, smooth, weight, gdtype, grad_scale=None):
    R, C = z.shape
    gs = 1.0 / R if grad_scale is None else grad_scale
    buf = torch.full((R, C + 3), 5.0, dtype=gdtype, device="cuda")
    dz = buf[:, :C]
    loss = ops.distill_xent(z, top, at, temperature=T, distill_weight=soft, teacher_lse=lse, labels=labels, hard_weight=hard, label_smoothing=smooth,
                            row_weight=weight, grad_scale=grad_scale, dlogits=dz)
    want, wz, ltol, tol = ref_distill(z, top, at, T, soft, lse, labels, hard, smooth, weight, gs)
    assert bool(((loss.double() - want).abs() <= ltol).all()), float(((loss.double() - want).abs() / ltol).max())
    u = U if gdtype == torch.bfloat16 else U32
    err = (dz.double() - wz).abs()
    lim = tol * (1 + u) + u * wz.abs() + 1e-40
    assert bool((err <= lim).all()), float((err / lim).max())
    assert bool((buf[:, C:] == 5.0).all()), "columns beyond the classes"
    only = ops.distill_xent(z, top, at, temperature=T, distill_weight=soft, teacher_lse=lse, labels=labels, hard_weight=hard, label_smoothing=smooth,
                            row_weight=weight)
    assert torch.equal(only, loss)
    return loss, dz


# the kernels' shapes change at 128, 512, 1024, 2048, 6144 and beyond 16384 pieces of 16 bytes (8 bf16 or 4 fp32 logits)
CLASSES = [1, 2, 3, 7, 100, 511, 513, 1000, 1025, 4097, 8191, 8200, 16385, 21843, 32769, 70001, 140003]


@pytest.mark.parametrize("C", CLASSES)
@pytest.mark.parametrize("dtype,gdtype", [(torch.float32, torch.bfloat16), (torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                          (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("mode", ["pairs", "rest", "hard"])
def test_distill(ops, C, dtype, gdtype, mode):
    R = 5 if C < 5000 else 3
    K = min(C, 1 if mode == "hard" else 67)
    T = {"pairs": 2.0, "rest": 1.0, "hard": 4.0}[mode]
    z, top, at, lse, labels = make(R, C, K, C, dtype, lse=mode == "rest", T=T)
    if mode == "hard":
        labels[0] = at[0, 0]  # the label's class is a pair's class too
        run_and_check(ops, z, top, at, T, 0.7, None, labels, 0.3, 0.1, None, gdtype)
    else:
        run_and_check(ops, z, top, at, T, 1.0, lse, None, 0.0, 0.0, None, gdtype)


@pytest.mark.parametrize("K", [0, 1, 5, 64, 65, 512])
def test_distill_pair_counts(ops, K):
    z, top, at, lse, labels = make(6, 600, K, K, torch.float32, lse=True)
    run_and_check(ops, z, top, at, 1.0, 0.5, lse if K else None, labels, 0.5, 0.0, None, torch.float32)
    run_and_check(ops, z, top, at, 1.0, 1.0, lse, None, 0.0, 0.0, None, torch.float32)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("C", [9, 3000])
def test_distill_edges(ops, C, rest):
    """Absent and repeated pairs, masked teacher logits, rows without any pair, rows of weight 0 full of NaN, labels outside the classes."""
    K = 6
    z, top, at, lse, labels = make(8, C, K, 17, torch.float32, lse=True)
    at[0, 2], at[0, 5] = -1, C  # no pairs
    at[1, :] = at[1, 0]  # one class six times
    at[2, 3] = at[2, 1]
    top[3, 1:] = -math.inf
    at[4, :] = -1  # no pair at all
    top[5, :] = -math.inf
    labels[2], labels[3], labels[4] = -1, C, 2 ** 31 - 1
    labels[1] = at[1, 0]
    weight = torch.tensor([1.0, 0.5, 2.0, 1.0, 1.0, 1.0, 0.0, 3.0], device="cuda")
    z[6], top[6] = math.nan, math.nan
    zc = z.clone()
    zc[6], tc = 0.0, top.clone()
    tc[6] = 0.0
    gs = 0.25
    kw = dict(temperature=1.5, distill_weight=0.6, teacher_lse=lse if rest else None, labels=labels, hard_weight=0.4, label_smoothing=0.1, row_weight=weight, grad_scale=gs)
    dz = torch.empty_like(z)
    loss = ops.distill_xent(z, top, at, dlogits=dz, **kw)
    want, wz, ltol, tol = ref_distill(zc, tc, at, 1.5, 0.6, lse if rest else None, labels, 0.4, 0.1, weight, gs)
    assert bool(((loss.double() - want).abs() <= ltol).all()) and bool(((dz.double() - wz).abs() <= tol + U32 * wz.abs()).all())
    assert float(loss[6]) == 0.0 and bool((dz[6] == 0).all())
    if not rest:  # nothing to distil from: the hard term alone, and that dropped too where the label is none
        assert float(loss[4]) == 0.0 and bool((dz[4] == 0).all())


def test_distill_masked_and_extreme_logits(ops):
    C = 300
    z, top, at, _, _ = make(7, C, 8, 3, torch.float32)
    z[0, 200:] = -math.inf
    at[0] = torch.arange(8, device="cuda", dtype=torch.int32) * 20
    z[1, 100:] = torch.finfo(torch.float32).min
    at[1] = at[0]
    z[2] = torch.finfo(torch.float32).min  # every class masked alike: uniform
    z[3], z[3, 7] = -3e38, 3e38
    at[3, 0] = 7
    top[3, 1:] = -math.inf
    z[4] = -math.inf
    z[5, 0] = math.inf
    z[6, 3] = math.nan
    dz = torch.empty_like(z)
    loss = ops.distill_xent(z, top, at, dlogits=dz, grad_scale=1.0)
    want, wz, ltol, tol = ref_distill(z[:4].clone(), top[:4], at[:4], 1.0, 1.0, None, None, 0.0, 0.0, None, 1.0)
    assert bool(((loss[:4].double() - want).abs() <= ltol).all()) and bool(((dz[:4].double() - wz).abs() <= tol + U32 * wz.abs()).all())
    assert bool((dz[0, 200:] == 0).all()) and bool(loss[4:].isnan().all())


def test_distill_small_divergence(ops):
    """Teacher and student agree but for 1e-3: the loss is 1e-6 of the terms it is joined from, and still right to 2 digits or better."""
    g = torch.Generator(device="cuda").manual_seed(2)
    z = torch.randn(4, 50, generator=g, device="cuda") * 2
    t = z + 1e-2 * torch.randn(4, 50, generator=g, device="cuda")
    top, at = t.topk(50, dim=1)
    loss = ops.distill_xent(z, top.contiguous(), at.int().contiguous(), temperature=4.0)
    p = torch.softmax(t.double() / 4, 1)
    want = 16 * (p * (torch.log_softmax(t.double() / 4, 1) - torch.log_softmax(z.double() / 4, 1))).sum(1)
    # the normaliser's error, 50 terms of 2^-22 each at random signs, times T^2 = 16: 2e-6 at the very most against 1e-5
    assert bool(((loss.double() - want).abs() < 16 * 8 * U32).all()), (loss, want)


def test_distill_in_place_unaligned_and_bias(ops):
    for dtype in (torch.float32, torch.bfloat16):
        z, top, at, _, labels = make(9, 1003, 10, 5, dtype)
        kw = dict(temperature=2.0, labels=labels, hard_weight=0.5, distill_weight=0.5, label_smoothing=0.1)
        dz = torch.empty_like(z)
        db = torch.full((1003,), 0.5, device="cuda")
        loss = ops.distill_xent(z, top, at, dlogits=dz, dbias=db, **kw)
        assert float((db.double() - 0.5 - dz.double().sum(0)).abs().max()) <= 16 * U32
        big = torch.zeros(9, 1010, dtype=dtype, device="cuda")
        view = big[:, 3:1006]  # rows that start at any element
        view.copy_(z)
        assert torch.equal(ops.distill_xent(view, top, at, dlogits=view, **kw), loss) and torch.equal(view, dz)
        assert bool((big[:, :3] == 0).all()) and bool((big[:, 1006:] == 0).all())
    assert ops.distill_xent(z[:0], top[:0], at[:0]).numel() == 0


def test_distill_hard_term_alone_is_softmax_xent(ops):
    z, top, at, _, labels = make(32, 1000, 4, 9, torch.float32)
    a, b = torch.empty(32, 1000, dtype=torch.bfloat16, device="cuda"), torch.empty(32, 1000, dtype=torch.bfloat16, device="cuda")
    rows = torch.empty(32, device="cuda")
    ops.softmax_xent(z, labels, 0.1, loss_rows=rows, dlogits=a)
    loss = ops.distill_xent(z, top, at, distill_weight=0.0, labels=labels, hard_weight=1.0, label_smoothing=0.1, dlogits=b)
    assert float((loss - rows).abs().max()) < 1e-5 and float((a.double() - b.double()).norm() / a.double().norm()) < 2 * U


def test_distill_gradient_by_differences(ops):
    g = torch.Generator(device="cuda").manual_seed(4)
    z, top, at, lse, labels = make(4, 300, 20, 6, torch.float32, lse=True, T=2.0)
    d = torch.randn(4, 300, generator=g, device="cuda")
    for extra in (dict(), dict(teacher_lse=lse)):
        kw = dict(temperature=2.0, distill_weight=0.6, labels=labels, hard_weight=0.4, label_smoothing=0.1, **extra)
        dz = torch.empty_like(z)
        ops.distill_xent(z, top, at, dlogits=dz, grad_scale=1.0, **kw)
        e = 2.0 ** -6
        diff = (ops.distill_xent(z + e * d, top, at, **kw).double() - ops.distill_xent(z - e * d, top, at, **kw).double()) / (2 * e)
        want = (dz.double() * d.double()).sum(1)
        # truncation: e^2 / 6 of a third moment of the direction (below 10); rounding: 2^-20 of a loss below 10, over e
        assert float((diff - want).abs().max()) < 10 * e * e / 6 + 10 * 2.0 ** -20 / e


def test_distill_captured(ops):
    z, top, at, _, labels = make(64, 1000, 10, 12, torch.float32)
    z2 = torch.randn_like(z)
    live, db = z.clone(), torch.zeros(1000, device="cuda")
    dz = torch.empty(64, 1000, dtype=torch.bfloat16, device="cuda")
    kw = dict(temperature=2.0, labels=labels, hard_weight=0.5)

    def eager(v):
        out, b = torch.empty_like(dz), torch.zeros_like(db)
        return ops.distill_xent(v, top, at, dlogits=out, dbias=b, **kw), out, b

    want = [eager(z), eager(z2)]
    gph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gph):
        db.zero_()
        loss = ops.distill_xent(live, top, at, dlogits=dz, dbias=db, **kw)
    for k in (0, 1, 0, 1):
        live.copy_((z, z2)[k])
        gph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((loss, dz, db), want[k]))
        eager(z)


def test_distill_through_a_model(ops):
    """The loss on an engine's logits, its gradient through the engine's custom-loss entry: the hard term alone gives loss_backward's gradients; with a
    teacher the head's gradients are those of the 64-bit loss gradient.  200 classes: the engine's gradient rows are padded."""
    from oracle import vit_ref
    from savit_amd.config import ModelConfig
    from savit_amd.engine import ViTEngine

    kw = dict(kind="vit", num_layers=2, num_heads=3, embed_dim=192, patch=16, num_classes=200, img_size=64)
    B, C, K = 6, 200, 9
    eng = ViTEngine(ModelConfig(**kw), B)
    eng.load_params(vit_ref.init_params(vit_ref.Cfg(**kw), seed=1, randomize=True))
    g = torch.Generator(device="cuda").manual_seed(8)
    images = torch.randn(B, 64, 64, 3, generator=g, device="cuda")
    _, top, at, lse, labels = make(B, C, K, 11, torch.float32, lse=True, T=2.0)
    eng.forward(images)
    eng.loss_backward(labels, 0.1)
    want = eng.grads.double()

    def backward(**loss):
        db = torch.zeros(C, device="cuda")
        rows = ops.distill_xent(eng.logits, top, at, labels=labels, label_smoothing=0.1, dlogits=eng.dlogits[:, :C], dbias=db, **loss)
        eng.backward_from_dlogits()
        off = eng.layout.off["bh"][0]
        eng.grads[off : off + C] += db
        return rows, db

    backward(distill_weight=0.0, hard_weight=1.0)
    # the two kernels' logit gradients may round to neighbours, and so may what follows: a few steps of 2^-8 at random signs
    assert float((eng.grads.double() - want).norm() / want.norm()) < 2 * U
    rows, db = backward(temperature=2.0, distill_weight=0.7, teacher_lse=lse, hard_weight=0.3)
    loss, grad, tol_loss, tol_grad = ref_distill(eng.logits, top, at, 2.0, 0.7, lse, labels, 0.3, 0.1, None, 1.0 / B)
    assert bool(((rows.double() - loss).abs() <= tol_loss).all())
    tol = tol_grad + U * grad.abs()
    off, d = eng.layout.off["Wh"][0], kw["embed_dim"]
    z = eng.zcls.double()
    dwh = eng.grads[off : off + d * C].view(d, C).double()
    assert bool(((dwh - z.T @ grad).abs() <= z.abs().T @ tol * 1.01 + 1e-30).all())  # (a sum of six products in fp32: 2^-21 of them, inside the hundredth)
    assert bool(((db.double() - grad.sum(0)).abs() <= tol.sum(0) * 1.01 + 1e-30).all())


def test_distill_offsets_beyond_32_bits(ops):
    """The last rows of logits of more than 4 GiB come out as they do alone."""
    C, K = 131072, 8
    z, top, at, _, labels = make(16, C, K, 5, torch.bfloat16)
    kw = dict(temperature=2.0, hard_weight=0.5, label_smoothing=0.1, grad_scale=1.0)
    n = 1040  # times 16 rows of 256 KiB
    big = z.repeat(n, 1)
    assert big.numel() * 2 > 1 << 32
    want = torch.empty_like(z)
    rows = ops.distill_xent(z, top, at, labels=labels, dlogits=want, **kw)
    got = ops.distill_xent(big, top.repeat(n, 1), at.repeat(n, 1), labels=labels.repeat(n), dlogits=big, **kw)
    assert torch.equal(got[-16:], rows) and torch.equal(big[-16:], want) and torch.equal(big[:16], want)


# --------------------------------------------------------------------------------------------- logits far from zero
def check_shifted(ops, z, top, at, T, soft, lse, labels, hard, smooth, gdtype=torch.float32):
    """Loss and gradient against 64 bits.  The reference sees the logits less their row's maximum (exact in 64 bits, and neither output changes by it), so
    that its bounds know nothing of a common offset: the exponents are rounded as numbers of the size of z - max, and so is the sum of the logits."""
    R, C = z.shape
    dz = torch.empty(R, C, dtype=gdtype, device="cuda")
    loss = ops.distill_xent(z, top, at, temperature=T, distill_weight=soft, teacher_lse=lse, labels=labels, hard_weight=hard, label_smoothing=smooth, dlogits=dz)
    zd = z.double()
    want, wz, ltol, tol = ref_distill(zd - zd.amax(1, keepdim=True), top, at, T, soft, lse, labels, hard, smooth, None, 1.0 / R)
    assert bool(((loss.double() - want).abs() <= ltol).all()), float(((loss.double() - want).abs() / ltol).max())
    u = U if gdtype == torch.bfloat16 else U32
    err, lim = (dz.double() - wz).abs(), tol * (1 + u) + u * wz.abs() + 1e-40
    assert bool((err <= lim).all()), float((err / lim).max())


OFFSETS = [300.0, -300.0, 5000.0, 40000.0, -40000.0]


@pytest.mark.parametrize("offset", OFFSETS)
@pytest.mark.parametrize("T", [0.5, 1.0, 4.0])
@pytest.mark.parametrize("C", [100, 1000, 21843])
def test_distill_gradient_with_a_common_offset(ops, offset, T, C):
    z, top, at, _, labels = make(4, C, 20, C, torch.float32)
    z = z + offset
    check_shifted(ops, z, top, at, T, 1.0, None, None, 0.0, 0.0)
    check_shifted(ops, z, top, at, T, 0.6, None, labels, 0.4, 0.0)
    check_shifted(ops, z.bfloat16(), top, at, T, 0.6, None, labels, 0.4, 0.0)


@pytest.mark.parametrize("offset", [8e4, -8e4, 2e5, -2e5])
def test_distill_gradient_with_an_offset_that_one_temperature_stretches(ops, offset):
    """At temperature 4 the distillation's exponents are those of ordinary logits and the label term's are not."""
    z, top, at, _, labels = make(4, 1000, 20, 3, torch.float32)
    check_shifted(ops, z + offset, top, at, 4.0, 0.6, None, labels, 0.4, 0.0)


@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("C", [21843, 140003])
def test_distill_maximum_across_the_border_of_the_short_form(ops, C, sign):
    """Exponents beyond 1e5 are taken in another form: a row whose running maximum crosses that (z log2 e = 1e5) between one piece and the next."""
    z, top, at, _, labels = make(4, C, 20, C, torch.float32, spread=0.5)
    z = z + sign * 1e5 * math.log(2.0)
    z[:, : C // 3] -= 1.5
    check_shifted(ops, z, top, at, 1.0, 0.6, None, labels, 0.4, 0.0)


@pytest.mark.parametrize("offset", [0.0] + OFFSETS)
@pytest.mark.parametrize("C,dtype", [(100, torch.float32), (1000, torch.float32), (21843, torch.float32), (70001, torch.float32), (3000, torch.bfloat16)])
def test_distill_sums_of_logits_with_a_common_offset(ops, offset, C, dtype):
    """The rest of the teacher's mass and the smoothing need the sum of all logits: it is no worse for an offset that all of them share."""
    z, top, at, lse, labels = make(4, C, 20, C, dtype, lse=True, T=2.0)
    z = (z.float() + offset).to(dtype)
    check_shifted(ops, z, top, at, 2.0, 1.0, lse, None, 0.0, 0.0)
    check_shifted(ops, z, top, at, 2.0, 0.6, None, labels, 0.4, 0.1)
    check_shifted(ops, z, top, at, 2.0, 0.6, lse, labels, 0.4, 0.1)


def test_distill_small_divergence_with_the_rest_and_an_offset(ops):
    g = torch.Generator(device="cuda").manual_seed(2)
    z = torch.randn(4, 50, generator=g, device="cuda") * 2
    t = z + 1e-2 * torch.randn(4, 50, generator=g, device="cuda")
    top, at = t.topk(30, dim=1)
    lse = torch.logsumexp(t.double() / 4, 1).float()
    for offset in (0.0, 4096.0):  # (a power of two: the differences of the logits stay what they were to 2^-11)
        zo = z + offset
        loss = ops.distill_xent(zo, top.contiguous(), at.int().contiguous(), temperature=4.0, teacher_lse=lse)
        want, _, _, _ = ref_distill(zo.double() - offset, top, at.int(), 4.0, 1.0, lse, None, 0.0, 0.0, None, 1.0)
        # as above: the normaliser's error times T^2, and the sum of 50 logits below 8: 50 roundings of 2^-24 of each, over the classes, times T
        assert bool(((loss.double() - want).abs() < 16 * 8 * U32 + 4 * 50 * 8 * U32).all()), (loss, want)


@pytest.mark.parametrize("C", [300, 140003])
def test_distill_smoothing_over_the_lowest_logits(ops, C):
    """Several classes at the type's lowest value: their sum passes what fp32 holds, their mean does not."""
    z, top, at, _, labels = make(4, C, 8, C, torch.float32)
    z[:, 50:60] = torch.finfo(torch.float32).min
    labels[:] = 7
    loss = ops.distill_xent(z, top, at, distill_weight=0.0, labels=labels, hard_weight=1.0, label_smoothing=0.1)
    want = -0.1 * z.double().mean(1)
    assert bool(((loss.double() / want - 1).abs() < 1e-5).all()), (loss, want)
    z[:] = torch.finfo(torch.float32).min  # every class alike: uniform
    loss = ops.distill_xent(z, top, at, distill_weight=0.0, labels=labels, hard_weight=1.0, label_smoothing=0.1)
    assert bool(((loss.double() - math.log(C)).abs() < 64 * U32 * math.log(C)).all()), loss


@pytest.mark.parametrize("masked", [-math.inf, torch.finfo(torch.float32).min, -1e30])
@pytest.mark.parametrize("C", [300, 5000, 140003])
def test_distill_masked_classes_with_the_rest(ops, C, masked):
    """Classes that teacher and student both exclude, named by pairs of probability 0: they take no part, and the loss is that of the others."""
    g = torch.Generator(device="cuda").manual_seed(C)
    z, _, _, _, labels = make(4, C, 8, C, torch.float32)
    out = torch.tensor([1, 2, 150, C - 1], device="cuda")
    t = torch.randn(4, C, generator=g, device="cuda") * 3
    t[:, out] = -math.inf
    z[:, out] = masked
    at = torch.cat([out.expand(4, 4), torch.arange(20, 40, device="cuda").expand(4, 20)], 1)
    at = torch.cat([at, at[:, :2]], 1)  # one of them twice
    top = t.gather(1, at)
    top[:, -2:] = -math.inf
    lse = torch.logsumexp(t.double(), 1).float()
    dz = torch.empty_like(z)
    loss = ops.distill_xent(z, top.contiguous(), at.int().contiguous(), teacher_lse=lse, dlogits=dz, grad_scale=1.0)
    keep = torch.ones(C, dtype=torch.bool, device="cuda")
    keep[out] = False
    new = (keep.cumsum(0) - 1)[at[:, 4:24]].int()
    want, wz, ltol, tol = ref_distill(z[:, keep], top[:, 4:24], new, 1.0, 1.0, lse, None, 0.0, 0.0, None, 1.0)
    assert bool(((loss.double() - want).abs() <= ltol).all()), (loss, want)
    assert bool((dz[:, ~keep] == 0).all()) and bool(((dz[:, keep].double() - wz).abs() <= tol + U32 * wz.abs()).all())
    # excluded by the student alone: the divergence is infinite (or as large as the mask makes it)
    z[:, 60] = masked
    loss = ops.distill_xent(z, top.contiguous(), at.int().contiguous(), teacher_lse=lse)
    if masked == -math.inf:
        assert bool((loss == math.inf).all())
    else:
        share = ((1 - (top[:, 4:24].double() - lse.double()[:, None]).exp().sum(1)) / (C - 24))
        assert bool(((loss.double() / (share * -masked) - 1).abs() < 1e-4).all()), (loss, share)  # (lse's own rounding, 2^-22 of exp, is in share too)


@pytest.mark.parametrize("C,dtype", [(1003, torch.float32), (30011, torch.float32), (140003, torch.bfloat16)])
def test_distill_masked_classes_in_place(ops, C, dtype):
    """Rows with masked classes are summed a second time: before any of their logits is replaced by its gradient."""
    z, top, at, lse, labels = make(32, C, 8, C, dtype, lse=True)
    z[:, 3::7] = torch.finfo(torch.float32).min if dtype == torch.float32 else -1e30
    kw = dict(teacher_lse=lse, labels=labels, hard_weight=0.5, distill_weight=0.5, label_smoothing=0.1)
    dz = torch.empty_like(z)
    loss = ops.distill_xent(z, top, at, dlogits=dz, **kw)
    for _ in range(5):
        place = z.clone()
        assert torch.equal(ops.distill_xent(place, top, at, dlogits=place, **kw), loss) and torch.equal(place, dz)
