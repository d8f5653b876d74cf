"""Attention with a bias: outputs and gradients are rounded to bfloat16 once, when they are stored.

Probabilities and score gradients enter the matrix instructions as two bfloat16 numbers, the second what the first one's rounding took off: 2^-16 of each is
lost, beside the 2^-8 of the result's own rounding and fp32's terms.  A single bfloat16 operand loses 2^-8 of the products' absolute values, many times the
bounds here where they cancel."""
import pytest
import torch

from tests.test_position_ops_gpu import U, U32, gen, ops, randn  # noqa: F401

pytestmark = pytest.mark.gpu

# one and two waves, one segment, resident and streaming gradients, the forward with 32 queries a wave (the last three)
SIZES = [(2, 9, 2, 16), (3, 17, 2, 64), (2, 32, 3, 32), (3, 49, 2, 32), (2, 64, 2, 64), (2, 100, 2, 48), (2, 197, 2, 64), (2, 224, 1, 32), (2, 300, 2, 64), (1, 577, 2, 32),
         (128, 70, 4, 64), (64, 130, 4, 48), (86, 300, 2, 64)]


@pytest.mark.parametrize("B,N,H,hd", SIZES)
@pytest.mark.parametrize("padded", [False, True])
def test_one_rounding(ops, B, N, H, hd, padded):  # noqa: F811
    g = gen(B + N)
    d = H * hd
    qkv = randn(g, B * N, 3 * d, dtype=torch.bfloat16)
    qkv[:, :d] *= hd ** -0.5
    bias = ops.relpos_bias_empty(H, N)
    bias.copy_(randn(g, H, N, N))
    d_o = randn(g, B * N, d, dtype=torch.bfloat16)
    lens = torch.randint(1, N + 1, (B,), generator=g, device="cuda", dtype=torch.int32) if padded else torch.full((B,), N, dtype=torch.int32, device="cuda")
    o, lse = ops.bias_attention_fwd(qkv, bias, B, N, H, head_dim=hd, lens=lens)
    dqkv, _ = ops.bias_attention_bwd(qkv, bias, d_o, lse, B, N, H, dq_scale=0.5, head_dim=hd, lens=lens)

    def heads(t):
        return t.double().reshape(B, N, H, hd).permute(0, 2, 1, 3).contiguous()

    there = torch.arange(N, device="cuda")[None, :] < lens[:, None]
    q, k, v = (heads(qkv[:, i * d:(i + 1) * d]) for i in range(3))
    do = heads(d_o) * there[:, None, :, None]
    keep = there[:, None, :, None] & there[:, None, None, :]
    s = (q @ k.transpose(2, 3) + bias.double()).masked_fill(~keep, -1e30)
    p = torch.softmax(s, -1) * keep
    dp, dpa = do @ v.transpose(2, 3), do.abs() @ v.abs().transpose(2, 3)
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    # scores: fp32 sums of hd products and a bias; exponents and what follows them: numbers below 32, a few roundings each
    es = U32 * ((hd + 4) * (q.abs() @ k.abs().transpose(2, 3)) + 4 * torch.where(keep, s.abs(), 0.0) + 4 * 32 + 24)
    pe = p * (es + (p * es).sum(-1, keepdim=True))
    dse = pe * (dp - delta).abs() + p * (pe * dp.abs()).sum(-1, keepdim=True) + (hd + N + 8) * U32 * p * (dpa + (p * dpa).sum(-1, keepdim=True))
    lost = U * U + (N + 16) * U32  # of an operand: its low part's rounding, and the accumulation's
    pt, dst = p.transpose(2, 3), ds.transpose(2, 3)
    for name, got, want, tol in (("o", o, p @ v, (pe + lost * p) @ v.abs()),
                                 ("dq", dqkv[:, :d], ds @ k * 0.5, (dse + lost * ds.abs()) @ k.abs() * 0.5),
                                 ("dk", dqkv[:, d:2 * d], dst @ q, (dse + lost * ds.abs()).transpose(2, 3) @ q.abs()),
                                 ("dv", dqkv[:, 2 * d:3 * d], pt @ do, (pe + lost * p).transpose(2, 3) @ do.abs())):
        err, lim = (heads(got) - want).abs(), (tol + U * (want.abs() + tol)) * 1.001 + 1e-30
        assert bool((err <= lim).all()), (name, float((err / lim).max()))
