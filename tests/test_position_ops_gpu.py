"""Per-head query / key norm with the rotation, learned relative position biases and attention with a bias, against plain 64-bit math.

Tolerances count roundings: u = 2^-8 is bf16's unit roundoff, 2^-24 fp32's.  A bf16 output is off by u |value|; an MFMA operand rounded to bf16 by
u times its magnitude, carried through the product's absolute values; fp32 terms by a small multiple of 2^-24 of what they are summed from."""
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


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


# --------------------------------------------------------------------------------------------- query / key norm + rotation
def qkn_ref(x, wq, wk, table, pos, H, Hk, hd, eps, q_scale, center, inter, cols=None):
    """64-bit forward on leaf tensors (autograd gives the gradients)."""
    rows = x.shape[0]
    t = None if table is None else table.double()[pos]

    def one(v, w, s):
        v = v.reshape(rows, -1, hd)
        if center:
            v = v - v.mean(-1, keepdim=True)
        v = v / (v.square().mean(-1, keepdim=True) + eps).sqrt() * w * s
        if t is not None:
            c, sn = t[:, None, : hd // 2], t[:, None, hd // 2:]
            a, b = (v[..., 0::2], v[..., 1::2]) if inter else (v[..., : hd // 2], v[..., hd // 2:])
            a, b = a * c - b * sn, a * sn + b * c
            v = torch.stack([a, b], -1).reshape(rows, -1, hd) if inter else torch.cat([a, b], -1)
        return v.reshape(rows, -1)

    nq, nk = H * hd, Hk * hd
    return torch.cat([one(x[:, :nq], wq, q_scale), one(x[:, nq:nq + nk], wk, 1.0), x[:, nq + nk:nq + 2 * nk]], 1)


QKN = [  # B, N, H, Hk, hd
    (1, 1, 1, 1, 16), (3, 1, 32, 8, 128), (2, 5, 3, 3, 64), (1, 197, 12, 12, 64), (4, 33, 6, 2, 48), (2, 7, 4, 1, 256), (5, 50, 5, 5, 32), (1, 19, 2, 2, 80),
    (16, 197, 12, 12, 64), (9, 257, 7, 7, 96),
]


@pytest.mark.parametrize("B,N,H,Hk,hd", QKN)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("center,inter,table,positions", [(False, False, True, False), (True, True, True, True), (False, True, True, False), (True, False, False, False)])
def test_qk_norm_rope(ops, B, N, H, Hk, hd, dtype, center, inter, table, positions):
    g = gen(B * 1000 + N * 10 + hd)
    rows, width, pad = B * N, (H + 2 * Hk) * hd, 16
    full = randn(g, rows, width + pad, dtype=dtype)
    x = full[:, :width]  # a row pitch wider than the row
    x[0, :hd] = 0  # a head of zeros: n = 0
    wq, wk = 1 + randn(g, hd, scale=0.3), randn(g, hd)
    wk[0] = 0.0  # a weight of zero still has a gradient
    T = N + 37
    tab = ops.rope_table(ops.rope_angles_1d(T, hd)) if table else None
    pos = torch.randint(0, T, (rows,), generator=g, device="cuda", dtype=torch.int32) if positions else None
    at = pos.long() if positions else torch.arange(rows, device="cuda") % N
    dy = randn(g, rows, width, dtype=dtype)
    kw = dict(N=N, H=H, Hk=Hk, head_dim=hd, positions=pos, q_scale=hd ** -0.5, center=center, interleaved=inter)
    y = ops.qk_norm_rope_fwd(x, wq, wk, tab, **kw)

    xd, wqd, wkd = x.double().requires_grad_(), wq.double().requires_grad_(), wk.double().requires_grad_()
    ref = qkn_ref(xd, wqd, wkd, tab, at, H, Hk, hd, 1e-6, hd ** -0.5, center, inter)
    ux = U if dtype == torch.bfloat16 else U32
    # fp32 arithmetic: mean, mean square and rsqrt carry (hd + 8) roundings, the products and the two-term rotation about 8 more, of numbers up to |w n| <= sqrt(hd) |w|
    slack = (hd + 16) * U32 * math.sqrt(hd) * max(float(wq.abs().max()) * hd ** -0.5, float(wk.abs().max())) * math.sqrt(2)
    nqk = (H + Hk) * hd
    err = (y.double() - ref).abs()
    assert bool((err[:, :nqk] <= ux * ref[:, :nqk].abs() + slack).all()), float(err.max())
    assert torch.equal(y[:, nqk:], x[:, nqk:])

    dwq, dwk = torch.full((hd,), 2.0, device="cuda"), torch.full((hd,), -1.0, device="cuda")
    out = torch.full((rows, width + 8), 7.0, dtype=dtype, device="cuda")
    dx = ops.qk_norm_rope_bwd(dy, x, wq, wk, tab, dwq, dwk, out=out, **kw)
    gx, gq, gk = torch.autograd.grad(ref, (xd, wqd, wkd), dy.double())
    assert bool((out[:, width:] == 7.0).all()) and torch.equal(out[:, nqk:width], dy[:, nqk:])
    # dx = r (h - mean h - n mean(h n)): its terms are of size r |g| |w| (1 + |n|^2 / hd ..) <= r * 3 sqrt(hd) max|g w|
    xh = xd.detach()[:, :nqk].reshape(rows, -1, hd)
    if center:
        xh = xh - xh.mean(-1, keepdim=True)
    r = 1 / (xh.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    wmax = torch.cat([(wqd.detach().abs().max() * hd ** -0.5).expand(H), wkd.detach().abs().max().expand(Hk)])[None, :, None]
    gmax = dy[:, :nqk].double().reshape(rows, -1, hd).abs().amax(-1, keepdim=True) * math.sqrt(2)
    size = (3 * math.sqrt(hd) * r * gmax * wmax).expand(-1, -1, hd).reshape(rows, nqk)
    err = (dx[:, :nqk].double() - gx[:, :nqk]).abs()
    assert bool((err <= ux * gx[:, :nqk].abs() + (hd + 32) * U32 * size).all()), float((err / (ux * gx[:, :nqk].abs() + (hd + 32) * U32 * size)).max())
    # weight gradients: fp32 sums of rows * heads terms |g n| <= gmax sqrt(hd), each off by (hd + 16) roundings; a sum of n terms in a tree of
    # chains (rows per group, groups of a block, blocks) adds less than 64 + n / 64 roundings of the sum of magnitudes
    n = rows * max(H, Hk)
    bound = (hd + 16 + 64 + n / 64) * U32 * n * float(gmax.max()) * math.sqrt(hd)
    got = torch.stack([dwq - 2.0, dwk + 1.0]).double()
    want = torch.stack([gq, gk])
    assert float((got - want).abs().max()) <= bound + 4 * U32
    assert float((got - want).norm() / want.norm()) < 1e-5

    # in place, and bit by bit the same a second time
    z = x.clone()
    assert ops.qk_norm_rope_fwd(z, wq, wk, tab, out=z, **kw) is z and torch.equal(z, y)
    d2, e2, f2 = dy.clone(), torch.full((hd,), 2.0, device="cuda"), torch.full((hd,), -1.0, device="cuda")
    ops.qk_norm_rope_bwd(d2, x, wq, wk, tab, e2, f2, **kw)
    assert torch.equal(d2, dx[:, :width]), "in place"


def test_qk_norm_rope_repeats_and_far_positions(ops):
    g = gen(5)
    B, N, H, hd = 8, 197, 12, 64
    x, dy = randn(g, B * N, 3 * H * hd, dtype=torch.bfloat16), randn(g, B * N, 3 * H * hd, dtype=torch.bfloat16)
    w = 1 + randn(g, 2, hd, scale=0.1)
    tab = ops.rope_table(ops.rope_angles_2d(14, 14, hd))
    res = []
    for _ in range(3):
        dw = torch.zeros(2, hd, device="cuda")
        dx = ops.qk_norm_rope_bwd(dy, x, w[0], w[1], tab, dw[0], dw[1], N=N, H=H, out=torch.empty_like(dy))
        res.append((dx, dw))
    assert all(torch.equal(a, b) for r in res[1:] for a, b in zip(res[0], r))
    # the class token's angles are zero: only the norm remains
    y = ops.qk_norm_rope_fwd(x, w[0], w[1], tab, N=N, H=H)
    y0 = ops.qk_norm_rope_fwd(x, w[0], w[1], None, N=N, H=H)
    assert torch.equal(y.view(B, N, -1)[:, 0], y0.view(B, N, -1)[:, 0]) and not torch.equal(y, y0)
    # a position outside the table poisons its row and no other
    pos = torch.arange(B * N, device="cuda", dtype=torch.int32) % N
    pos[3], pos[7], pos[9] = N, -1, 2 ** 31 - 1
    y = ops.qk_norm_rope_fwd(x, w[0], w[1], tab, N=N, H=H, positions=pos)
    bad = torch.zeros(B * N, dtype=torch.bool, device="cuda")
    bad[[3, 7, 9]] = True
    assert bool(y[bad][:, : 2 * H * hd].isnan().all()) and not bool(y[~bad].isnan().any()) and torch.equal(y[:, 2 * H * hd:], x[:, 2 * H * hd:])
    assert ops.qk_norm_rope_fwd(x[:0], w[0], w[1], tab, N=N, H=H).shape == (0, 3 * H * hd)


def test_qk_norm_rope_gradient_by_differences(ops):
    """fp32: the directional derivative of sum(y dy) along a random direction, by central differences of the kernel's own forward."""
    g = gen(11)
    B, N, H, hd = 2, 9, 3, 48
    x, dy, d = (randn(g, B * N, 3 * H * hd) for _ in range(3))
    w, dwd = 1 + randn(g, 2, hd, scale=0.2), randn(g, 2, hd)
    tab = ops.rope_table(ops.rope_angles_1d(N, hd))
    kw = dict(N=N, H=H, head_dim=hd, center=True, interleaved=True)
    dw = torch.zeros(2, hd, device="cuda")
    dx = ops.qk_norm_rope_bwd(dy, x, w[0], w[1], tab, dw[0], dw[1], out=torch.empty_like(x), **kw)
    e = 2.0 ** -7

    def f(s):
        return float((ops.qk_norm_rope_fwd(x + s * e * d, w[0] + s * e * dwd[0], w[1] + s * e * dwd[1], tab, **kw).double() * dy.double()).sum())

    diff = (f(1) - f(-1)) / (2 * e)
    want = float((dx.double() * d.double()).sum() + (dw.double() * dwd.double()).sum())
    # truncation e^2 / 6 of a third derivative of order the function's own size (~ sqrt(count) = 51), and 2^-24 sqrt(count) / e of rounding
    assert abs(diff - want) < 50 * e * e * math.sqrt(x.numel()), (diff, want)


# --------------------------------------------------------------------------------------------- relative position bias
@pytest.mark.parametrize("kind,H", [((1, 1, False), 1), ((1, 1, True), 3), ((3, 5, True), 4), ((14, 14, True), 12), ((7, 7, False), 5), ((24, 24, True), 16), (1, 2), (5, 3), (300, 6),
                                    (1024, 2)])
def test_relpos_bias_and_its_gradient(ops, kind, H):
    index, nb = ops.relpos_index_1d(kind) if isinstance(kind, int) else ops.relpos_index_2d(*kind)
    N = index.shape[0]
    g = gen(N + H)
    table = randn(g, nb, H)
    bias = ops.relpos_bias_fwd(table, index)
    assert torch.equal(bias, table[index.long()].permute(2, 0, 1))
    order, start = ops.relpos_order(index, nb)
    buf = ops.relpos_bias_empty(H, N)
    base = buf.as_strided((H, N, buf.stride(1)), (N * buf.stride(1), buf.stride(1), 1))
    base.fill_(float("nan"))  # the padding is never read
    db = randn(g, H, N, N)
    buf.copy_(db)
    before = randn(g, nb, H)
    got = [ops.relpos_bias_bwd(buf, order, start, before.clone()) for _ in range(2)]
    assert torch.equal(got[0], got[1])
    want, size = (torch.zeros(nb, H, dtype=torch.float64, device="cuda").index_add_(0, index.reshape(-1).long(), v.reshape(H, -1).t().double()) for v in (db, db.abs()))
    # a list of n terms: chains of at most n / (64 parts) + parts + 8 additions
    n = int((start[1:] - start[:-1]).max())
    assert bool(((got[0].double() - before.double() - want).abs() <= U32 * ((n / 64 + 140) * size + 2 * before.double().abs() + want.abs())).all())


def test_relpos_bad_lists_stay_inside(ops):
    index, nb = ops.relpos_index_2d(3, 3, cls=False)
    N = 9
    bad = index.clone()
    bad[0, 0], bad[1, 2] = nb, -5
    bias = ops.relpos_bias_fwd(torch.ones(nb, 2, device="cuda"), bad)
    assert bool(bias[:, 0, 0].isnan().all()) and bool(bias[:, 1, 2].isnan().all()) and int(bias.isnan().sum()) == 4
    order, start = ops.relpos_order(index, nb)
    order[0], order[5], start[nb] = -1, N * N, 10 ** 9
    out = ops.relpos_bias_bwd(ops.relpos_bias_fwd(torch.ones(nb, 2, device="cuda"), index), order, start, torch.zeros(nb, 2, device="cuda"))
    assert float(out.sum()) == 2.0 * (N * N - 2)


# --------------------------------------------------------------------------------------------- attention with a bias
def attn_ref(qkv, bias, lens, B, N, H, hd, d_o=None, dq_scale=1.0):
    """64-bit values and elementwise bounds on what the roundings of the kernels may change."""
    q, k, v = qkv[:, : 3 * H * hd].double().reshape(B, N, 3, H, hd).permute(2, 0, 3, 1, 4).contiguous()
    n = torch.full((B,), N, device="cuda") if lens is None else lens.clamp(0, N)
    inside = torch.arange(N, device="cuda")[None, :] < n[:, None]
    rowin = inside[:, None, :, None]
    q, k, v = (torch.where(rowin, t, 0.0) for t in (q, k, v))
    bd = torch.where(bias < -2e38, -math.inf, bias.double())
    s = q @ k.transpose(2, 3) + bd
    s = s.masked_fill(~(rowin & inside[:, None, None, :]), -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where((lse == -math.inf)[..., None], 0.0, (s - torch.where(lse == -math.inf, 0.0, lse)[..., None]).exp())
    o = p @ v
    rows = lambda t: t.permute(0, 2, 1, 3).reshape(B * N, H * hd)  # noqa: E731
    # relative error of a probability: S is an fp32 sum of hd products and the bias, its scaling and the log-sum-exp round once more each
    fin = torch.where(s == -math.inf, 0.0, s.abs())
    ep = 2 * U32 * ((hd + 4) * (q.abs() @ k.abs().transpose(2, 3)) + 4 * fin + 4 * torch.where(lse == -math.inf, 0.0, lse.abs())[..., None] + 8)
    pe = p * ep
    res = {"o": rows(o), "lse": lse, "lse_tol": U32 * (8 * torch.where(lse == -math.inf, 0.0, lse.abs()) + 16) + (pe.sum(-1))}
    res["o_tol"] = rows((U + 0.0) * (p @ v.abs()) + U * o.abs() + (pe + (N + 16) * U32 * p) @ v.abs()) * 1.001 + 1e-30
    if d_o is None:
        return res
    do = torch.where(rowin, d_o.double().reshape(B, N, H, hd).permute(0, 2, 1, 3), 0.0)
    dp = do @ v.transpose(2, 3)
    dpa = do.abs() @ v.abs().transpose(2, 3)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    # dS in fp32: its own factor, dP's sum of hd products, and delta's sum over the keys
    dse = pe * (dp - delta).abs() + p * (hd + 2) * U32 * dpa + p * ((pe * dp.abs() + p * ((hd + N + 4) * U32) * dpa).sum(-1, keepdim=True)) + 4 * U32 * p * (dp.abs() + delta.abs())
    acc = (N + 16) * U32
    dq, dk, dv = ds @ k * dq_scale, ds.transpose(2, 3) @ q, p.transpose(2, 3) @ do
    tq = (dse + (U + acc) * ds.abs()) @ k.abs() * dq_scale + U * dq.abs()
    tk = (dse + (U + acc) * ds.abs()).transpose(2, 3) @ q.abs() + U * dk.abs()
    tv = (pe + (U + acc) * p).transpose(2, 3) @ do.abs() + U * dv.abs()
    res["dqkv"] = torch.cat([rows(t) for t in (dq, dk, dv)], 1)
    res["dqkv_tol"] = torch.cat([rows(t) for t in (tq, tk, tv)], 1) * 1.001 + 1e-30
    res["dbias"], res["dbias_tol"] = ds.sum(0), (dse + (B + 8) * U32 * ds.abs()).sum(0) + 1e-30
    res["inside"] = inside.reshape(-1)
    return res


def check_attention(ops, qkv, bias, lens, B, N, H, hd, d_o, scale):
    o, lse = ops.bias_attention_fwd(qkv, bias, B, N, H, head_dim=hd, lens=lens)
    dqkv, dbias = ops.bias_attention_bwd(qkv, bias, d_o, lse, B, N, H, dq_scale=scale, head_dim=hd, lens=lens)
    ref = attn_ref(qkv, bias, lens, B, N, H, hd, d_o, scale)
    w = 3 * H * hd
    for name, got in (("o", o), ("lse", lse), ("dqkv", dqkv[:, :w]), ("dbias", dbias)):
        want, tol = ref[name], ref[name + "_tol"]
        empty = want == -math.inf
        assert torch.equal(got.double() == -math.inf, empty), name
        err = torch.where(empty, 0.0, (got.double() - want).abs())
        assert bool((err <= tol).all()), (name, float(torch.nan_to_num(err / tol, nan=1e9).max()))
    out = ~ref["inside"]
    assert bool((o[out] == 0).all()) and bool((dqkv[:, :w][out] == 0).all())
    return o, lse, dqkv, dbias


SIZES = [(1, 1, 1), (3, 2, 2), (2, 17, 3), (2, 31, 1), (2, 32, 2), (3, 33, 2), (5, 49, 4), (2, 63, 1), (1, 64, 3), (2, 65, 2), (1, 96, 1), (2, 127, 2), (1, 128, 1), (3, 129, 1),
         (3, 197, 3), (1, 257, 2), (1, 577, 2)]


@pytest.mark.parametrize("hd", [16, 32, 48, 64])
@pytest.mark.parametrize("B,N,H", SIZES)
def test_bias_attention(ops, B, N, H, hd):
    g = gen(B * 100 + N + hd)
    d = H * hd
    qkv = randn(g, B * N, 3 * d + 8 * (N % 3), dtype=torch.bfloat16)  # some with a wider row pitch
    qkv[:, :d] *= hd ** -0.5
    bias = ops.relpos_bias_empty(H, N)
    bias.copy_(randn(g, H, N, N))
    d_o = randn(g, B * N, d, dtype=torch.bfloat16)
    check_attention(ops, qkv, bias, None, B, N, H, hd, d_o, hd ** -0.5)


@pytest.mark.parametrize("N,lens", [(1, [0, 1]), (5, [5, 0, 3, 1]), (50, [50, 33, 1, 0, 32, 31]), (64, [63, 64, 2]), (130, [129, 128, 1, 97, 0, 64]), (200, [-3, 500, 199, 65])])
def test_bias_attention_padded_batch(ops, N, lens):
    """Padding holds NaN everywhere it can: nothing of it reaches a valid row; its own rows come back zero, its log-sum-exp -inf."""
    B, H, hd = len(lens), 2, 64
    g = gen(N)
    lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    qkv = randn(g, B * N, 3 * H * hd, dtype=torch.bfloat16, scale=0.6)
    d_o = randn(g, B * N, H * hd, dtype=torch.bfloat16)
    inside = (torch.arange(N, device="cuda")[None, :] < lens.clamp(0, N)[:, None]).reshape(-1)
    qkv[~inside] = float("nan")
    d_o[~inside] = float("nan")
    bias = ops.relpos_bias_empty(H, N)
    bias.copy_(randn(g, H, N, N))
    o, lse, dqkv, dbias = check_attention(ops, qkv, bias, lens, B, N, H, hd, torch.where(inside[:, None], d_o, 0.0), 1.0)
    again = ops.bias_attention_bwd(qkv, bias, d_o, lse, B, N, H, dq_scale=1.0, head_dim=hd, lens=lens)
    assert torch.equal(again[0], dqkv) and torch.equal(again[1], dbias)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("N,lens,hd", [(20, [3, 0, 9], 32), (64, [47, 33], 16), (130, [100, 128], 48), (224, [197, 1], 64), (300, [7, 290, 257], 64), (330, [129, 0], 32)])
def test_bias_attention_rows_behind_every_sequence(ops, N, lens, hd, bad):
    """Bias rows and columns that no sequence reaches hold anything: no gradient reads them, theirs is zero."""
    B, H, top = len(lens), 2, max(lens)
    g = gen(N + hd)
    lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    qkv = randn(g, B * N, 3 * H * hd, dtype=torch.bfloat16, scale=0.6)
    d_o = randn(g, B * N, H * hd, dtype=torch.bfloat16)
    clean = ops.relpos_bias_empty(H, N)
    clean.copy_(randn(g, H, N, N))
    o, lse = ops.bias_attention_fwd(qkv, clean, B, N, H, head_dim=hd, lens=lens)
    want = ops.bias_attention_bwd(qkv, clean, d_o, lse, B, N, H, dq_scale=1.0, head_dim=hd, lens=lens)
    dirty = ops.relpos_bias_empty(H, N)
    dirty.copy_(clean)
    dirty[:, top:], dirty[:, :, top:] = bad, bad
    o2, lse2 = ops.bias_attention_fwd(qkv, dirty, B, N, H, head_dim=hd, lens=lens)
    got = ops.bias_attention_bwd(qkv, dirty, d_o, lse2, B, N, H, dq_scale=1.0, head_dim=hd, lens=lens)
    assert torch.equal(o2, o) and torch.equal(lse2, lse)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert bool((got[1][:, top:] == 0).all()) and bool((got[1][:, :, top:] == 0).all())


@pytest.mark.parametrize("N", [3, 40, 64, 197])
@pytest.mark.parametrize("masked", [-math.inf, torch.finfo(torch.float32).min, torch.finfo(torch.bfloat16).min])
def test_bias_attention_masks_in_the_bias(ops, N, masked):
    """-inf (and the lowest values) mask keys; a query that keeps none is empty: zero output, -inf, no gradient."""
    B, H, hd = 2, 2, 32
    g = gen(N)
    qkv = randn(g, B * N, 3 * H * hd, dtype=torch.bfloat16)
    qkv[:, : H * hd] *= hd ** -0.5
    bias = ops.relpos_bias_empty(H, N)
    b = randn(g, H, N, N)
    b = torch.where(torch.rand(H, N, N, generator=g, device="cuda") < 0.5, masked, b)
    b[0, 0], b[1, N - 1], b[0, :, : max(1, N - 2)] = masked, masked, masked  # empty rows, and a head that sees the last keys alone
    bias.copy_(b)
    d_o = randn(g, B * N, H * hd, dtype=torch.bfloat16)
    o, lse, dqkv, dbias = check_attention(ops, qkv, bias, None, B, N, H, hd, d_o, hd ** -0.5)
    assert bool((lse[:, 0, 0] == -math.inf).all()) and bool((o.view(B, N, H, hd)[:, 0, 0] == 0).all()) and bool((dbias[0, 0] == 0).all())


def test_bias_attention_large_scores(ops):
    """Scores far apart, growing along the keys (the running reference moves at every tile) and shrinking: no overflow, the same bounds."""
    B, N, H, hd = 1, 300, 2, 64
    g = gen(3)
    qkv = randn(g, B * N, 3 * H * hd, dtype=torch.bfloat16)
    ramp = torch.linspace(-400, 400, N, device="cuda")
    bias = ops.relpos_bias_empty(H, N)
    bias[0], bias[1] = ramp[None, :], -ramp[None, :]
    check_attention(ops, qkv, bias, None, B, N, H, hd, randn(g, B * N, H * hd, dtype=torch.bfloat16), 1.0)


def test_bias_attention_without_bias_is_attention(ops):
    """A bias of zero: the framework's own attention, to its roundings."""
    B, N, H, hd = 4, 197, 6, 64
    g = gen(4)
    qkv = randn(g, B * N, 3 * H * hd, dtype=torch.bfloat16)
    qkv[:, : H * hd] *= hd ** -0.5
    o0, lse0 = ops.attention_fwd(qkv, B, N, H)
    o, lse = ops.bias_attention_fwd(qkv, ops.relpos_bias_empty(H, N).zero_(), B, N, H)
    ref = attn_ref(qkv, torch.zeros(H, N, N, device="cuda"), None, B, N, H, hd)
    assert bool(((o.double() - o0.double()).abs() <= 2 * ref["o_tol"]).all()) and bool(((lse - lse0).abs() <= 2 * ref["lse_tol"]).all())


def test_bias_attention_repeats_bit_by_bit(ops):
    B, N, H, hd = 37, 49, 4, 32
    g = gen(8)
    qkv, d_o = randn(g, B * N, 3 * H * hd, dtype=torch.bfloat16), randn(g, B * N, H * hd, dtype=torch.bfloat16)
    index, nb = ops.relpos_index_2d(7, 7, cls=False)
    order, start = ops.relpos_order(index, nb)
    bias = ops.relpos_bias_fwd(randn(g, nb, H), index)
    res = []
    for _ in range(3):
        o, lse = ops.bias_attention_fwd(qkv, bias, B, N, H, head_dim=hd)
        dqkv, dbias = ops.bias_attention_bwd(qkv, bias, d_o, lse, B, N, H, dq_scale=0.5, head_dim=hd)
        res.append((o, lse, dqkv, dbias.clone(), ops.relpos_bias_bwd(dbias, order, start, torch.zeros(nb, H, device="cuda"))))
    assert all(torch.equal(a, b) for r in res[1:] for a, b in zip(res[0], r))
    only, none = ops.bias_attention_bwd(qkv, bias, d_o, lse, B, N, H, dq_scale=0.5, head_dim=hd, want_dbias=False)
    assert none is None and torch.equal(only, res[0][2])


def test_bias_attention_no_images(ops):
    bias = ops.relpos_bias_empty(2, 5).zero_()
    e = torch.empty(0, 96, dtype=torch.bfloat16, device="cuda")
    o, lse = ops.bias_attention_fwd(e, bias, 0, 5, 2, head_dim=16)
    dqkv, db = ops.bias_attention_bwd(e, bias, o, lse, 0, 5, 2, dq_scale=1.0, head_dim=16)
    assert o.shape == (0, 32) and dqkv.shape == (0, 96) and float(db.abs().sum()) == 0.0


# --------------------------------------------------------------------------------------------- as they are used together
def step(ops, x, w, tab, table_nb, index, order, start, B, N, H, hd, d_o):
    """Norm + rotation, attention with the learned bias, and back: everything a training step of one layer's attention calls."""
    y = ops.qk_norm_rope_fwd(x, w[0], w[1], tab, N=N, H=H, head_dim=hd, q_scale=hd ** -0.5)
    bias = ops.relpos_bias_fwd(table_nb, index)
    o, lse = ops.bias_attention_fwd(y, bias, B, N, H, head_dim=hd)
    dqkv, dbias = ops.bias_attention_bwd(y, bias, d_o, lse, B, N, H, dq_scale=1.0, head_dim=hd)  # q_scale is undone by the norm's backward
    dt, dw = torch.zeros_like(table_nb), torch.zeros_like(w)
    ops.relpos_bias_bwd(dbias, order, start, dt)
    ops.qk_norm_rope_bwd(dqkv, x, w[0], w[1], tab, dw[0], dw[1], N=N, H=H, head_dim=hd, q_scale=hd ** -0.5)
    return o, dqkv, dt, dw


def make_step(ops, seed=21, B=3, gh=6, H=3, hd=64):
    g = gen(seed)
    N = gh * gh + 1
    index, nb = ops.relpos_index_2d(gh, gh)
    order, start = ops.relpos_order(index, nb)
    return dict(x=randn(g, B * N, 3 * H * hd, dtype=torch.bfloat16), w=1 + randn(g, 2, hd, scale=0.2), tab=ops.rope_table(ops.rope_angles_2d(gh, gh, hd)),
                table_nb=randn(g, nb, H), index=index, order=order, start=start, B=B, N=N, H=H, hd=hd, d_o=randn(g, B * N, H * hd, dtype=torch.bfloat16))


def test_attention_step_together(ops):
    a = make_step(ops)
    o, dx, dt, dw = step(ops, **a)
    B, N, H, hd = a["B"], a["N"], a["H"], a["hd"]
    x, w, t = a["x"].double().requires_grad_(), a["w"].double().requires_grad_(), a["table_nb"].double().requires_grad_()
    y = qkn_ref(x, w[0], w[1], a["tab"], torch.arange(B * N, device="cuda") % N, H, H, hd, 1e-6, hd ** -0.5, False, False)
    q, k, v = y.reshape(B, N, 3, H, hd).permute(2, 0, 3, 1, 4)
    p = torch.softmax(q @ k.transpose(2, 3) + t[a["index"].long()].permute(2, 0, 1), -1)
    ro = (p @ v).permute(0, 2, 1, 3).reshape(B * N, H * hd)
    want = torch.autograd.grad(ro, (x, t, w), a["d_o"].double())
    # two chained bf16 roundings of the operands at random signs: a few times 2^-8 / sqrt(3) of the norm
    for name, got, ref in (("o", o, ro.detach()), ("dx", dx, want[0]), ("dtable", dt, want[1]), ("dw", dw, want[2])):
        assert float((got.double() - ref).norm() / ref.norm()) < 3 * U, name


def test_attention_step_captured_and_on_another_stream(ops):
    a, b = make_step(ops, 31), make_step(ops, 32)
    eager = [[t.clone() for t in step(ops, **v)] for v in (a, b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        res = step(ops, **a)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(res, eager[0]))
    live = {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in a.items()}
    graphs = []
    for _ in range(2):  # two graphs of the same step: their workspaces are their own
        gph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gph):
            out = step(ops, **live)
        graphs.append((gph, out))
    for k, src in enumerate((a, b, a, b)):
        for name in ("x", "w", "table_nb", "d_o"):
            live[name].copy_(src[name])
        for gph, _ in graphs:
            gph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for _, out in graphs for x, y in zip(out, eager[k % 2])), k
        step(ops, **src)  # eager work between the replays


def test_offsets_beyond_32_bits(ops):
    """The last head (image, rows) of tensors of more than 4 GiB comes out as it does alone, bit by bit."""
    g = gen(77)
    H, N, hd = 17, 8192, 16  # a bias of 4.25 GiB
    index = ((torch.arange(N, device="cuda")[:, None] * 31 + torch.arange(N, device="cuda")[None, :] * 7) % 97).int()
    table = randn(g, 97, H)
    bias = ops.relpos_bias_fwd(table, index)
    assert bias.numel() * 4 > 1 << 32
    last = ops.relpos_bias_fwd(table[:, -1:].contiguous(), index)
    assert torch.equal(bias[-1], last[0])
    qkv = randn(g, N, 3 * H * hd, dtype=torch.bfloat16)
    d_o = randn(g, N, H * hd, dtype=torch.bfloat16)
    o, lse = ops.bias_attention_fwd(qkv, bias, 1, N, H, head_dim=hd)
    dqkv, dbias = ops.bias_attention_bwd(qkv, bias, d_o, lse, 1, N, H, dq_scale=1.0, head_dim=hd)
    one = qkv.view(N, 3, H, hd)[:, :, -1].reshape(N, 3 * hd).contiguous()
    d_one = d_o[:, -hd:].contiguous()
    o1, lse1 = ops.bias_attention_fwd(one, last, 1, N, 1, head_dim=hd)
    g1, b1 = ops.bias_attention_bwd(one, last, d_one, lse1, 1, N, 1, dq_scale=1.0, head_dim=hd)
    assert torch.equal(o[:, -hd:], o1) and torch.equal(lse[:, -1:], lse1)
    assert torch.equal(dqkv.view(N, 3, H, hd)[:, :, -1].reshape(N, -1), g1) and torch.equal(dbias[-1], b1[0])
    del bias, dbias, last, b1
    B, N, H, hd = 4800, 197, 12, 64  # packed rows of 4.06 GiB
    small = randn(g, 8 * N, 3 * H * hd, dtype=torch.bfloat16, scale=0.5)
    qkv = small.repeat(B // 8, 1)
    assert qkv.numel() * 2 > 1 << 32
    w = 1 + randn(g, 2, hd, scale=0.1)
    tab = ops.rope_table(ops.rope_angles_1d(N, hd))
    y = ops.qk_norm_rope_fwd(qkv, w[0], w[1], tab, N, H)
    assert torch.equal(y[-8 * N :], ops.qk_norm_rope_fwd(small, w[0], w[1], tab, N, H))
    dw = torch.zeros(2, 2, hd, device="cuda")
    dx = ops.qk_norm_rope_bwd(qkv, qkv, w[0], w[1], tab, dw[0, 0], dw[0, 1], N, H, out=y)
    assert torch.equal(dx[-8 * N :], ops.qk_norm_rope_bwd(small, small, w[0], w[1], tab, dw[1, 0], dw[1, 1], N, H, out=torch.empty_like(small)))
    bias = ops.relpos_bias_empty(H, N)
    bias.copy_(randn(g, H, N, N))
    d_small = randn(g, 8 * N, H * hd, dtype=torch.bfloat16)
    o, lse = ops.bias_attention_fwd(qkv, bias, B, N, H)
    o1, lse1 = ops.bias_attention_fwd(small[-N:], bias, 1, N, H)
    assert float((o[-N:].double() - o1.double()).norm() / o1.double().norm()) < 2 * U  # (another tile shape for one image)
    dqkv, _ = ops.bias_attention_bwd(qkv, bias, d_small.repeat(B // 8, 1), lse, B, N, H, dq_scale=1.0, want_dbias=False, dqkv=y)
    g1, _ = ops.bias_attention_bwd(small[-N:], bias, d_small[-N:], lse[-1:].contiguous(), 1, N, H, dq_scale=1.0, want_dbias=False)
    assert torch.equal(dqkv[-N:], g1)
