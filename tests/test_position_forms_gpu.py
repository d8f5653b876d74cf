"""The forms that the position operators' kernels take at larger sizes, against plain 64-bit math: several images a workgroup, 32 queries a wave, several heads a
group of lanes.  Tolerances as in test_position_ops_gpu.py, whose references these use."""
import math

import pytest
import torch

from tests.test_position_ops_gpu import U, U32, check_attention, gen, ops, qkn_ref, randn  # noqa: F401

pytestmark = pytest.mark.gpu


def attention_inputs(ops, B, N, H, hd, seed):  # noqa: F811
    g = gen(seed)
    d = H * hd
    qkv = randn(g, B * N, 3 * d, dtype=torch.bfloat16)
    qkv[:, :d] *= hd ** -0.5
    bias = ops.relpos_bias_empty(H, N)
    bias.copy_(randn(g, H, N, N))
    return g, qkv, bias, randn(g, B * N, d, dtype=torch.bfloat16)


def lengths(g, B, N):
    lens = torch.randint(0, N + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    lens[0], lens[B // 2], lens[B - 1] = 0, N, 1
    return lens


# A workgroup of the gradients of short sequences goes through several images (the batch is cut into 256 parts or fewer times the workgroups a CU, over the
# heads): every number of 16-row tiles up to 14, heads of an image in a row and images of a head in a row; then the streaming form
IMAGES = [(400, 5, 12, 16), (300, 17, 16, 64), (300, 49, 4, 32), (100, 70, 6, 64), (90, 100, 6, 48), (70, 128, 8, 64), (45, 144, 6, 64), (45, 145, 6, 32), (45, 170, 6, 64), (45, 190, 6, 48),
          (45, 197, 6, 64), (25, 197, 12, 64), (45, 209, 6, 16), (45, 224, 6, 64), (25, 224, 12, 32), (20, 257, 8, 64), (25, 300, 6, 48), (20, 385, 6, 32)]


@pytest.mark.parametrize("B,N,H,hd", IMAGES)
@pytest.mark.parametrize("padded", [False, True])
def test_bias_attention_many_images(ops, B, N, H, hd, padded):  # noqa: F811
    g, qkv, bias, d_o = attention_inputs(ops, B, N, H, hd, B + N)
    lens = lengths(g, B, N) if padded else None
    if padded:
        outside = (torch.arange(N, device="cuda")[None, :] >= lens[:, None]).reshape(-1)
        qkv[outside] = math.nan  # nothing of a row behind one sequence may reach the next one's
    _, lse, dqkv, dbias = check_attention(ops, qkv, bias, lens, B, N, H, hd, d_o, hd ** -0.5)
    again = ops.bias_attention_bwd(qkv, bias, d_o, lse, B, N, H, dq_scale=hd ** -0.5, head_dim=hd, lens=lens)
    assert torch.equal(again[0], dqkv) and torch.equal(again[1], dbias)
    only, _ = ops.bias_attention_bwd(qkv, bias, d_o, lse, B, N, H, dq_scale=hd ** -0.5, head_dim=hd, lens=lens, want_dbias=False)
    assert torch.equal(only, dqkv)


# 65 tokens and more, heads of 48 and 64, 512 workgroups of 128 queries and more: the forward with 32 queries a wave
WIDE = [(128, 70, 4, 64), (64, 129, 4, 48), (43, 300, 4, 64), (52, 197, 5, 64), (128, 128, 4, 48)]


@pytest.mark.parametrize("B,N,H,hd", WIDE)
@pytest.mark.parametrize("form", ["plain", "padded", "masked", "ramp"])
def test_bias_attention_wide_forward(ops, B, N, H, hd, form):  # noqa: F811
    g, qkv, bias, d_o = attention_inputs(ops, B, N, H, hd, N)
    lens = lengths(g, B, N) if form == "padded" else None
    if form == "masked":
        b = torch.where(torch.rand(H, N, N, generator=g, device="cuda") < 0.5, -math.inf, bias)
        b[0, 3], b[1, :, : N // 2 + 3], b[2, :, N // 3:] = -math.inf, -math.inf, torch.finfo(torch.float32).min
        bias.copy_(b)
    if form == "ramp":  # the running maximum moves at every tile, or never
        ramp = torch.linspace(-400, 400, N, device="cuda")
        bias[0], bias[1], bias[2:] = ramp[None, :], -ramp[None, :], (ramp * (torch.arange(N, device="cuda") % 3 - 1))[None, :]
    check_attention(ops, qkv, bias, lens, B, N, H, hd, d_o, 1.0)


@pytest.mark.parametrize("B,N,H,hd", [(1, 17, 2, 32), (300, 49, 4, 32), (2, 197, 3, 64), (45, 197, 6, 64), (3, 300, 2, 64), (25, 300, 6, 48), (1, 1, 1, 16)])
def test_bias_gradient_leaves_what_lies_behind_its_columns(ops, B, N, H, hd):  # noqa: F811
    """A gradient that is a part of a wider buffer: the columns beside it keep what they hold."""
    g, qkv, narrow, d_o = attention_inputs(ops, B, N, H, hd, N)
    ld = (N + 3) // 4 * 4 + 12
    bias = torch.full((H, N, ld), math.nan, device="cuda")[:, :, :N]
    bias.copy_(narrow)
    _, lse = ops.bias_attention_fwd(qkv, bias, B, N, H, head_dim=hd)
    buf = torch.full((H, N, ld), 7.0, device="cuda")
    _, db = ops.bias_attention_bwd(qkv, bias, d_o, lse, B, N, H, dq_scale=1.0, head_dim=hd, dbias=buf[:, :, :N])
    _, want = ops.bias_attention_bwd(qkv, narrow, d_o, lse, B, N, H, dq_scale=1.0, head_dim=hd)
    assert torch.equal(db, want) and bool((buf[:, :, N:] == 7.0).all())


@pytest.mark.parametrize("N", [20, 300])
def test_bias_attention_gradient_of_wide_rows(ops, N):  # noqa: F811
    """Rows with columns beside the packed ones: the gradient has those of the packed ones, at the same pitch."""
    B, H, hd = 2, 2, 32
    g, qkv, bias, d_o = attention_inputs(ops, B, N, H, hd, N)
    wide = torch.full((B * N, 3 * H * hd + 24), math.nan, dtype=torch.bfloat16, device="cuda")
    wide[:, : 3 * H * hd] = qkv
    _, lse = ops.bias_attention_fwd(wide, bias, B, N, H, head_dim=hd)
    dqkv, db = ops.bias_attention_bwd(wide, bias, d_o, lse, B, N, H, dq_scale=1.0, head_dim=hd)
    assert dqkv.shape == qkv.shape and dqkv.stride(0) == wide.stride(0)
    want, wb = ops.bias_attention_bwd(qkv, bias, d_o, lse, B, N, H, dq_scale=1.0, head_dim=hd)
    assert torch.equal(dqkv, want) and torch.equal(db, wb)


def test_outputs_beside_their_inputs(ops):  # noqa: F811
    """Column ranges of one buffer share its rows and no memory: inputs and outputs next to each other."""
    B, N, H, hd = 2, 50, 2, 32
    g, qkv, bias, d_o = attention_inputs(ops, B, N, H, hd, 3)
    w = 3 * H * hd
    both = torch.zeros(B * N, 2 * w + 16, dtype=torch.bfloat16, device="cuda")
    both[:, :w] = qkv
    both_bias = torch.zeros(H * N * 120 + 64, device="cuda")[: H * N * 120].view(H, N, 120)  # (rows of 120, the last one's from column 60 on too)
    both_bias[:, :, :N] = bias
    o, lse = ops.bias_attention_fwd(both[:, :w], both_bias[:, :, :N], B, N, H, head_dim=hd)
    dqkv, db = ops.bias_attention_bwd(both[:, :w], both_bias[:, :, :N], d_o, lse, B, N, H, dq_scale=1.0, head_dim=hd, dqkv=both[:, w + 8:2 * w + 8], dbias=both_bias[:, :, 60:60 + N])
    want, wb = ops.bias_attention_bwd(qkv, bias, d_o, lse, B, N, H, dq_scale=1.0, head_dim=hd)
    assert torch.equal(dqkv, want) and torch.equal(db, wb) and torch.equal(both[:, :w], qkv) and bool((both[:, 2 * w + 8:] == 0).all())
    wq = 1 + randn(g, hd, scale=0.1)
    y = ops.qk_norm_rope_fwd(both[:, :w], wq, wq, None, N, H, head_dim=hd, out=both[:, w:2 * w])
    assert torch.equal(y, ops.qk_norm_rope_fwd(qkv, wq, wq, None, N, H, head_dim=hd))
    dw = torch.zeros(4, hd, device="cuda")
    dx = ops.qk_norm_rope_bwd(want, both[:, :w], wq, wq, None, dw[0], dw[1], N, H, head_dim=hd, out=both[:, w + 8:2 * w + 8])
    assert torch.equal(dx, ops.qk_norm_rope_bwd(want, qkv, wq, wq, None, dw[2], dw[3], N, H, head_dim=hd, out=torch.empty_like(want))) and torch.equal(dw[:2], dw[2:])
    z = torch.zeros(9, 210, device="cuda")
    z[:, :100] = randn(g, 9, 100)
    top, at = z[:, :100].topk(5, dim=1)
    dz = torch.empty(9, 100, device="cuda")
    loss = ops.distill_xent(z[:, :100].contiguous(), top, at.int(), dlogits=dz)
    assert torch.equal(ops.distill_xent(z[:, :100], top, at.int(), dlogits=z[:, 101:201]), loss) and torch.equal(z[:, 101:201], dz)


# --------------------------------------------------------------------------------------------- query / key norm
# enough rows that a group of lanes takes four heads in bf16 and two in fp32; numbers of heads that leave a last group fewer
MANY = [(24001, 5, 3, 64), (11000, 7, 1, 256), (33000, 6, 2, 48), (66001, 9, 9, 16)]


@pytest.mark.parametrize("rows,H,Hk,hd", MANY)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("center,inter,positions", [(False, False, False), (True, True, True)])
def test_qk_norm_rope_many_rows(ops, rows, H, Hk, hd, dtype, center, inter, positions):  # noqa: F811
    g = gen(rows + hd)
    width, N, T = (H + 2 * Hk) * hd, 1009, 1100
    x, dy = randn(g, rows, width, dtype=dtype), randn(g, rows, width, dtype=dtype)
    wq, wk = 1 + randn(g, hd, scale=0.3), randn(g, hd)
    tab = ops.rope_table(ops.rope_angles_1d(T, hd))
    pos = torch.randint(0, T, (rows,), generator=g, device="cuda", dtype=torch.int32) if positions else None
    at = pos.long() if positions else torch.arange(rows, device="cuda") % N
    kw = dict(N=N, H=H, Hk=Hk, head_dim=hd, positions=pos, q_scale=hd ** -0.5, center=center, interleaved=inter)
    y = ops.qk_norm_rope_fwd(x, wq, wk, tab, **kw)
    xd, wqd, wkd = x.double().requires_grad_(), wq.double().requires_grad_(), wk.double().requires_grad_()
    ref = qkn_ref(xd, wqd, wkd, tab, at, H, Hk, hd, 1e-6, hd ** -0.5, center, inter)
    ux = U if dtype == torch.bfloat16 else U32
    slack = (hd + 16) * U32 * math.sqrt(hd) * max(float(wq.abs().max()) * hd ** -0.5, float(wk.abs().max())) * math.sqrt(2)
    nqk = (H + Hk) * hd
    err = (y.double() - ref).abs()
    assert bool((err[:, :nqk] <= ux * ref[:, :nqk].abs() + slack).all()), float(err.max())
    assert torch.equal(y[:, nqk:], x[:, nqk:])
    z = x.clone()
    assert ops.qk_norm_rope_fwd(z, wq, wk, tab, out=z, **kw) is z and torch.equal(z, y)
    gq, gk = torch.autograd.grad(ref, (wqd, wkd), dy.double())
    dwq, dwk = torch.zeros(hd, device="cuda"), torch.zeros(hd, device="cuda")
    ops.qk_norm_rope_bwd(dy, x, wq, wk, tab, dwq, dwk, out=torch.empty_like(dy), **kw)
    got, want = torch.stack([dwq, dwk]).double(), torch.stack([gq, gk])
    assert float((got - want).norm() / want.norm()) < 1e-5


@pytest.mark.parametrize("B,N,H,Hk,hd", [(1, 1, 1, 1, 16), (3, 1, 32, 8, 128), (1, 197, 12, 12, 64), (4, 33, 6, 2, 48), (2, 7, 4, 1, 256), (1, 19, 2, 2, 80), (16, 197, 12, 12, 64), (9, 257, 7, 7, 96)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_qk_norm_rope_weight_gradients_in_place(ops, B, N, H, Hk, hd, dtype):  # noqa: F811
    """In place the values are left alone, so that the groups of lanes are other ones: the weights' gradients are those of the formula, twice the same."""
    g = gen(B * 1000 + N * 10 + hd)
    rows, width = B * N, (H + 2 * Hk) * hd
    x, dy = randn(g, rows, width, dtype=dtype), randn(g, rows, width, dtype=dtype)
    wq, wk = 1 + randn(g, hd, scale=0.3), randn(g, hd)
    tab = ops.rope_table(ops.rope_angles_1d(N, hd))
    kw = dict(N=N, H=H, Hk=Hk, head_dim=hd, q_scale=hd ** -0.5)
    res = []
    for _ in range(2):
        d, dw = dy.clone(), torch.stack([torch.full((hd,), 2.0, device="cuda"), torch.full((hd,), -1.0, device="cuda")])
        assert ops.qk_norm_rope_bwd(d, x, wq, wk, tab, dw[0], dw[1], **kw) is d
        res.append((d, dw))
    assert all(torch.equal(a, b) for a, b in zip(*res))
    assert torch.equal(res[0][0][:, (H + Hk) * hd:], dy[:, (H + Hk) * hd:])
    xd, wqd, wkd = x.double(), wq.double().requires_grad_(), wk.double().requires_grad_()
    ref = qkn_ref(xd, wqd, wkd, tab, torch.arange(rows, device="cuda") % N, H, Hk, hd, 1e-6, hd ** -0.5, False, False)
    want = torch.stack(torch.autograd.grad(ref, (wqd, wkd), dy.double()))
    got = res[0][1].double() - torch.tensor([[2.0], [-1.0]], device="cuda")
    gmax = float(dy[:, : (H + Hk) * hd].double().abs().max()) * math.sqrt(2)
    n = rows * max(H, Hk)
    bound = (hd + 16 + 64 + n / 64) * U32 * n * gmax * math.sqrt(hd)
    assert float((got - want).abs().max()) <= bound + 4 * U32
    assert float((got - want).norm() / want.norm()) < 1e-5 + 4 * U32 * math.sqrt(2 * hd) / float(want.norm())
