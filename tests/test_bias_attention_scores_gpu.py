"""Attention with a bias where the scores are far from zero or masked by large finite numbers, against plain 64-bit math.

Softmax does not change by what a row's scores have in common.  The bounds here therefore know nothing of the scores' size: inputs are whole multiples of a
power of two, so that every score is exact in 32 bits and in 64, or a masked score is so large that 32 bits hold nothing of the product beside it (and the
reference takes it so).  What remains are the roundings of exponents of the size of (score - maximum), and bf16's: u = 2^-8, 2^-24 in fp32."""
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


def steps(g, *shape):
    """-1, 0 or 1."""
    return torch.randint(-1, 2, shape, generator=g, device="cuda").float()


def heads(t, B, N, H, hd):
    return t.double().reshape(B, N, H, hd).permute(0, 2, 1, 3).contiguous()


def rows(t):
    B, H, N, hd = t.shape
    return t.permute(0, 2, 1, 3).reshape(B * N, H * hd)


def check(ops, qkv, bias, B, N, H, hd, d_o=None, scale=1.0, lens=None, mask=None, masked=None):
    """mask [H, N, N]: where the score is `masked` itself.  With a cotangent d_o the gradients too."""
    d = H * hd
    o, lse = ops.bias_attention_fwd(qkv, bias, B, N, H, head_dim=hd, lens=lens)
    q, k, v = (heads(qkv[:, i * d:(i + 1) * d], B, N, H, hd) for i in range(3))
    s = q @ k.transpose(2, 3) + bias.double()
    if mask is not None:
        s = torch.where(mask, float(masked), s)
    n = torch.full((B,), N, device="cuda") if lens is None else lens.clamp(0, N).long()
    inside = torch.arange(N, device="cuda")[None, :] < n[:, None]
    keep = inside[:, None, :, None] & inside[:, None, None, :]
    s = torch.where(keep, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    x = s - torch.where(top == -math.inf, 0.0, top)
    e = x.exp()
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    want_lse = (top + total.log())[..., 0]
    assert torch.equal(lse == -math.inf, want_lse == -math.inf)
    live = want_lse != -math.inf
    assert bool(((lse.double() - want_lse).abs()[live] <= U32 * (4 * want_lse.abs() + 32)[live]).all()), "lse"
    # a probability: its exponent rounds a few times as a number of the size of x, the exponential, the sum and the quotient a few times more
    ep = U32 * (4 * torch.where(x == -math.inf, 0.0, x.abs()) + 24)
    pe = p * (ep + (p * ep).sum(-1, keepdim=True))
    want, tol = p @ v, (U * p + pe + (N + 16) * U32 * p) @ v.abs()
    tol = (tol + U * want.abs()) * 1.001 + 1e-30
    err = (heads(o, B, N, H, hd) - want).abs()
    assert bool((err <= tol).all()), ("o", float(torch.nan_to_num(err / tol, nan=1e9).max()))
    if d_o is None:
        return
    dqkv, dbias = ops.bias_attention_bwd(qkv, bias, d_o, lse, B, N, H, dq_scale=scale, head_dim=hd, lens=lens)
    do = torch.where(inside[:, None, :, None], heads(d_o, B, N, H, hd), 0.0)
    dp, dpa = do @ v.transpose(2, 3), do.abs() @ v.abs().transpose(2, 3)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    dse = pe * (dp - delta).abs() + p * (hd + 2) * U32 * dpa + p * (pe * dp.abs() + p * ((hd + N + 4) * U32) * dpa).sum(-1, keepdim=True) + 4 * U32 * p * (dp.abs() + delta.abs())
    acc = (N + 16) * U32
    got = [heads(dqkv[:, i * d:(i + 1) * d], B, N, H, hd) for i in range(3)]
    for name, g, w, t in (("dq", got[0], ds @ k * scale, (dse + (U + acc) * ds.abs()) @ k.abs() * scale),
                          ("dk", got[1], ds.transpose(2, 3) @ q, (dse + (U + acc) * ds.abs()).transpose(2, 3) @ q.abs()),
                          ("dv", got[2], p.transpose(2, 3) @ do, (pe + (U + acc) * p).transpose(2, 3) @ do.abs())):
        err, tol = (g - w).abs(), (t + U * w.abs()) * 1.001 + 1e-30
        assert bool((err <= tol).all()), (name, float(torch.nan_to_num(err / tol, nan=1e9).max()))
    err, tol = (dbias.double() - ds.sum(0)).abs(), (dse + (B + 8) * U32 * ds.abs()).sum(0) + 1e-30
    assert bool((err <= tol).all()), ("dbias", float(torch.nan_to_num(err / tol, nan=1e9).max()))


def inputs(ops, B, N, H, hd, seed):
    """Rows whose scores are multiples of 1/32 below 2; v and the cotangent are anything."""
    g = gen(seed)
    d = H * hd
    qkv = torch.randn(B * N, 3 * d, generator=g, device="cuda").bfloat16()
    qkv[:, :d] = steps(g, B * N, d).bfloat16()
    qkv[:, d:2 * d] = (steps(g, B * N, d) / 32).bfloat16()
    bias = ops.relpos_bias_empty(H, N)
    bias.copy_(torch.randint(-64, 65, (H, N, N), generator=g, device="cuda") / 32)
    return g, qkv, bias, torch.randn(B * N, d, generator=g, device="cuda").bfloat16()


# one and two waves, one segment, several; gradients with resident keys (an even and an odd number of tiles) and streaming ones
SIZES = [(2, 1, 2, 16), (3, 17, 2, 64), (2, 32, 3, 32), (3, 49, 2, 32), (2, 64, 2, 64), (2, 100, 2, 48), (2, 130, 2, 64), (2, 197, 2, 64), (2, 224, 1, 32), (2, 300, 2, 64), (1, 500, 2, 32)]
# the forward with 32 queries a wave takes wide heads and 512 workgroups
WIDE = [(128, 70, 4, 64), (64, 130, 4, 48), (86, 300, 2, 64)]


OFFSETS = [100.0, -1e4, 2.0 ** 17, -2.0 ** 17]


def with_offset(ops, B, N, H, hd, offset):
    g, qkv, bias, d_o = inputs(ops, B, N, H, hd, N)
    bias += offset
    bias[:, N // 2] -= 2 * offset  # (and rows of another)
    return qkv, bias, d_o


@pytest.mark.parametrize("offset", OFFSETS)
@pytest.mark.parametrize("B,N,H,hd", SIZES + WIDE)
def test_scores_with_a_common_offset(ops, B, N, H, hd, offset):
    qkv, bias, _ = with_offset(ops, B, N, H, hd, offset)
    check(ops, qkv, bias, B, N, H, hd)


MASKS = [-1e8, -1e9, -1e10, -1e20, -1e30, torch.finfo(torch.float32).min / 2]


def with_mask(ops, B, N, H, hd, masked):
    """Rows that a mask leaves the last keys of, the first ones, some, or none: a row that is masked all over is uniform, as in a plain softmax."""
    g, qkv, bias, d_o = inputs(ops, B, N, H, hd, N + 1)
    mask = torch.rand(H, N, N, generator=g, device="cuda") < 0.3
    i, j = torch.arange(N, device="cuda")[:, None], torch.arange(N, device="cuda")[None, :]
    mask[0] |= j < i - N // 8  # a window: the first tiles of late queries are masked all over
    mask[-1] |= j > i + 1
    mask[:, N // 3], mask[0, N - 1], mask[-1, 0] = True, True, True
    bias.copy_(torch.where(mask, masked, bias))
    return qkv, bias, d_o, dict(mask=mask, masked=torch.tensor(masked, dtype=torch.float32).double())


@pytest.mark.parametrize("masked", MASKS)
@pytest.mark.parametrize("B,N,H,hd", SIZES + WIDE)
def test_large_finite_masks(ops, B, N, H, hd, masked):
    qkv, bias, _, kw = with_mask(ops, B, N, H, hd, masked)
    check(ops, qkv, bias, B, N, H, hd, **kw)


MANY = [(3, 49, 2, 32), (2, 197, 2, 64), (2, 300, 2, 64), (128, 70, 4, 64)]


def with_masks(ops, B, N, H, hd):
    """One mask on top of another: among masked keys alone, those masked least are what is left.  Row 7 is empty: the lowest value masks."""
    g, qkv, bias, d_o = inputs(ops, B, N, H, hd, N + 2)
    kind = torch.randint(0, 4, (H, N, N), generator=g, device="cuda")
    lowest = torch.finfo(torch.float32).min
    masked = torch.tensor([-1e9, -1e10, -1e30, lowest], device="cuda")[kind]
    masked[:, 5, : N // 2], masked[:, 5, N // 2:], masked[:, 7] = -1e30, -2e30, lowest
    hide = torch.rand(H, N, 1, generator=g, device="cuda") < 0.5
    hide[:, 5], hide[:, 7] = True, True
    bias.copy_(torch.where(hide, masked, bias))
    d = H * hd
    q, k, v = (heads(qkv[:, c * d:(c + 1) * d], B, N, H, hd) for c in range(3))
    s = torch.where(hide.expand(H, N, N), torch.where(masked < -1e38, -math.inf, masked.double()), q @ k.transpose(2, 3) + bias.double())
    return qkv, bias, d_o, torch.softmax(s, -1).nan_to_num(0.0), v


@pytest.mark.parametrize("B,N,H,hd", MANY)
def test_masks_of_several_sizes(ops, B, N, H, hd):
    qkv, bias, _, p, v = with_masks(ops, B, N, H, hd)
    o, lse = ops.bias_attention_fwd(qkv, bias, B, N, H, head_dim=hd)
    # u for P and for the output; the exponents of scores below 4 and what follows them, under 200 roundings, and the sum's N
    assert bool(((heads(o, B, N, H, hd) - p @ v).abs() <= (2 * U + (N + 200) * U32) * (p @ v.abs()) + 1e-30).all())
    assert bool((lse[:, :, 7] == -math.inf).all()) and bool(lse[:, :, 8:].isfinite().all())


# --------------------------------------------------------------------------------------------- gradients
@pytest.mark.parametrize("offset", OFFSETS)
@pytest.mark.parametrize("B,N,H,hd", SIZES + WIDE)
def test_gradients_of_scores_with_a_common_offset(ops, B, N, H, hd, offset):
    qkv, bias, d_o = with_offset(ops, B, N, H, hd, offset)
    check(ops, qkv, bias, B, N, H, hd, d_o, 0.5)


@pytest.mark.parametrize("masked", MASKS)
@pytest.mark.parametrize("B,N,H,hd", SIZES + WIDE)
def test_gradients_with_large_finite_masks(ops, B, N, H, hd, masked):
    """Among them rows that are masked all over: their probabilities are uniform in the gradients too."""
    qkv, bias, d_o, kw = with_mask(ops, B, N, H, hd, masked)
    check(ops, qkv, bias, B, N, H, hd, d_o, 0.5, **kw)


@pytest.mark.parametrize("B,N,H,hd", MANY)
def test_gradients_with_masks_of_several_sizes(ops, B, N, H, hd):
    qkv, bias, d_o, p, v = with_masks(ops, B, N, H, hd)
    d = H * hd
    _, lse = ops.bias_attention_fwd(qkv, bias, B, N, H, head_dim=hd)
    dqkv, dbias = ops.bias_attention_bwd(qkv, bias, d_o, lse, B, N, H, dq_scale=1.0, head_dim=hd)
    do = heads(d_o, B, N, H, hd)
    dv, dva = p.transpose(2, 3) @ do, p.transpose(2, 3) @ do.abs()
    assert bool(((heads(dqkv[:, 2 * d:3 * d], B, N, H, hd) - dv).abs() <= (2 * U + (N + 200) * U32) * dva + 1e-30).all())
    assert bool((dbias[:, 7] == 0).all()) and bool(dqkv[:, : 3 * d].isfinite().all()) and bool(dbias.isfinite().all())


@pytest.mark.parametrize("B,N,H,hd", [(300, 49, 4, 32), (45, 197, 6, 64), (20, 257, 8, 64)])
def test_gradients_with_masks_over_many_images(ops, B, N, H, hd):
    """Several images a workgroup, of different lengths."""
    qkv, bias, d_o, kw = with_mask(ops, B, N, H, hd, -1e9)
    lens = torch.randint(0, N + 1, (B,), generator=gen(1), device="cuda", dtype=torch.int32)
    check(ops, qkv, bias, B, N, H, hd, d_o, 0.5, lens=lens, **kw)
