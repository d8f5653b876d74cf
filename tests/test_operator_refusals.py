"""What the position, bias-attention and distillation operators refuse, checked on the host: nothing here reaches a GPU."""
import pytest
import torch

P, EINVAL = 0x10000, 1001  # an aligned address that is never followed


@pytest.fixture(scope="module")
def L():
    import os

    from savit_amd import lib

    if not os.path.exists(lib.LIB_PATH):
        import __graft_entry__ as g

        g.build()
    return lib.load()


def qkn(L, bwd=False, **kw):
    a = dict(x=P, ld=192, wq=P, wk=P, table=P, T=50, pos=None, out=2 * P, ldo=192, rows=50, N=50, H=1, Hk=1, hd=64, bf16=1, eps=1e-6, dq=3 * P, ldd=192,
             dwq=P, dwk=P + 256, ws=P, bytes=1 << 30)
    a.update(kw)
    if bwd:
        return L.savit_qk_norm_rope_bwd(a["dq"], a["ldd"], a["x"], a["ld"], a["wq"], a["wk"], a["table"], a["T"], a["pos"], a["out"], a["ldo"], a["dwq"], a["dwk"], a["rows"],
                                        a["N"], a["H"], a["Hk"], a["hd"], a["bf16"], a["eps"], 1.0, 0, 0, a["ws"], a["bytes"], None)
    return L.savit_qk_norm_rope_fwd(a["x"], a["ld"], a["wq"], a["wk"], a["table"], a["T"], a["pos"], a["out"], a["ldo"], a["rows"], a["N"], a["H"], a["Hk"], a["hd"], a["bf16"],
                                    a["eps"], 1.0, 0, 0, None)


@pytest.mark.parametrize("bad", [dict(x=None), dict(out=None), dict(wq=None), dict(wk=None), dict(ld=191), dict(ld=196), dict(ldo=184), dict(hd=24, ld=72), dict(hd=8), dict(hd=272, ld=816),
                                 dict(H=0), dict(Hk=0), dict(N=0), dict(rows=-1), dict(T=49), dict(T=0, pos=P), dict(x=P + 8), dict(out=2 * P + 2), dict(table=P + 4), dict(eps=-1.0),
                                 dict(out=P, ldo=200), dict(rows=(1 << 30) + 1)])
def test_qk_norm_rope(L, bad):
    assert qkn(L, **bad) == EINVAL
    assert qkn(L, bwd=True, **bad) == EINVAL


@pytest.mark.parametrize("bad", [dict(dq=None), dict(ldd=100), dict(ldd=196), dict(dwq=None), dict(dwk=None), dict(dq=3 * P + 2), dict(ws=P + 1), dict(out=P, dq=3 * P), dict(dwk=P), dict(dwk=P + 252),
                                 dict(ws=None, rows=1 << 20, N=1 << 20, T=1 << 20)])
def test_qk_norm_rope_bwd(L, bad):
    assert qkn(L, bwd=True, **bad) == EINVAL


def test_qk_norm_rope_nothing_to_do(L):
    assert qkn(L, rows=0) == 0 and qkn(L, bwd=True, rows=0) == 0
    need = L.savit_qk_norm_rope_bwd_workspace_bytes(1, 1, 64)
    assert need >= 2 * 64 * 4 and L.savit_qk_norm_rope_bwd_workspace_bytes(12, 12, 24) == 0
    assert qkn(L, bwd=True, rows=1 << 20, N=1 << 20, T=1 << 20, bytes=need - 1) == EINVAL


def test_relpos(L):
    ok = dict(t=P, i=P, b=P, N=9, H=2, nb=25, ld=12)

    def fwd(**kw):
        a = {**ok, **kw}
        return L.savit_relpos_bias_fwd(a["t"], a["i"], a["b"], a["N"], a["H"], a["nb"], a["ld"], None)

    def bwd(ws=None, n=0, **kw):
        a = {**ok, **kw}
        return L.savit_relpos_bias_bwd(a["b"], a["i"], a["i"], a["t"], a["N"], a["H"], a["nb"], a["ld"], ws, n, None)

    for bad in (dict(t=None), dict(i=None), dict(b=None), dict(N=0), dict(N=32769, ld=32772), dict(H=0), dict(nb=0), dict(ld=8), dict(ld=9), dict(nb=1 << 28, H=16)):
        assert fwd(**bad) == EINVAL and bwd(**bad) == EINVAL, bad
    assert fwd(b=P + 4) == EINVAL
    need = L.savit_relpos_bias_bwd_workspace_bytes(1000, 2, 32)
    assert need > 0 and L.savit_relpos_bias_bwd_workspace_bytes(9, 2, 25) == 0
    assert bwd(N=1000, nb=32, ld=1000) == EINVAL and bwd(N=1000, nb=32, ld=1000, ws=P, n=need - 1) == EINVAL


def attn(L, bwd=False, **kw):
    a = dict(qkv=P, bias=P, lens=None, o=3 * P, lse=P, do=P, dqkv=2 * P, dbias=3 * P, B=2, N=50, H=3, hd=64, ld=576, ldb=52, ws=P, n=1 << 30)
    a.update(kw)
    if bwd:
        return L.savit_bias_attention_bwd(a["qkv"], a["bias"], a["lens"], a["do"], a["lse"], a["dqkv"], a["dbias"], a["B"], a["N"], a["H"], a["hd"], a["ld"], a["ldb"], 1.0, a["ws"],
                                          a["n"], None)
    return L.savit_bias_attention_fwd(a["qkv"], a["bias"], a["lens"], a["o"], a["lse"], a["B"], a["N"], a["H"], a["hd"], a["ld"], a["ldb"], None)


@pytest.mark.parametrize("bad", [dict(qkv=None), dict(bias=None), dict(lse=None), dict(B=-1), dict(N=0), dict(N=32769, ldb=32772), dict(H=0), dict(hd=40), dict(hd=128, ld=1152),
                                 dict(ld=568), dict(ld=578), dict(ldb=49), dict(ldb=51), dict(qkv=P + 8), dict(bias=P + 4), dict(N=32768, ldb=32768), dict(B=1 << 30)])
def test_bias_attention(L, bad):
    assert attn(L, **bad) == EINVAL
    assert attn(L, bwd=True, **bad) == EINVAL


@pytest.mark.parametrize("bad", [dict(do=None), dict(dqkv=None), dict(dqkv=P), dict(ws=None), dict(ws=P + 4), dict(do=P + 2), dict(dqkv=2 * P + 8), dict(dbias=3 * P + 8), dict(dbias=P), dict(do=2 * P), dict(B=0)])
def test_bias_attention_bwd(L, bad):
    assert attn(L, bwd=True, **bad) == EINVAL


def test_bias_attention_workspace(L):
    assert attn(L, o=None) == EINVAL and attn(L, o=P + 2) == EINVAL and attn(L, o=P) == EINVAL and attn(L, B=0) == 0
    for want in (0, 1):
        need = L.savit_bias_attention_bwd_workspace_bytes(128, 197, 12, 200, want)
        assert need >= 128 * 12 * 2 * 256 * 4
        assert attn(L, bwd=True, B=128, N=197, H=12, ld=2304, ldb=200, n=need - 1, dbias=3 * P if want else None) == EINVAL


def distill(L, **kw):
    a = dict(z=P, ld=100, b=0, top=P, at=P, K=5, lse=None, labels=P, w=None, T=1.0, soft=0.5, hard=0.5, smooth=0.1, loss=P, dz=2 * P, ldz=100, db=0, dbias=None, R=4, C=100)
    a.update(kw)
    return L.savit_distill_xent(a["z"], a["ld"], a["b"], a["top"], a["at"], a["K"], a["lse"], a["labels"], a["w"], a["T"], a["soft"], a["hard"], a["smooth"], 1.0, a["loss"], a["dz"],
                                a["ldz"], a["db"], a["dbias"], a["R"], a["C"], None)


@pytest.mark.parametrize("bad", [dict(z=None), dict(R=-1), dict(C=0), dict(ld=99), dict(K=-1), dict(K=513), dict(top=None), dict(at=None), dict(T=0.0), dict(T=-1.0), dict(T=float("inf")),
                                 dict(T=float("nan")), dict(labels=None), dict(smooth=-0.1), dict(smooth=1.5), dict(loss=None, dz=None), dict(ldz=99), dict(dz=None, dbias=P), dict(z=P + 2),
                                 dict(dz=2 * P + 2), dict(dz=P, db=1), dict(dz=P, ldz=104)])
def test_distill(L, bad):
    assert distill(L, **bad) == EINVAL


@pytest.mark.parametrize("T", [1e-39, 1e-31, 1e31, float("nan")])
def test_distill_temperatures_without_a_scale(L, T):
    """log2 e / T has to be an ordinary number."""
    assert distill(L, T=T) == EINVAL


def test_distill_nothing_to_do(L):
    assert distill(L, R=0) == 0


def test_outputs_over_inputs(L):
    """An output that shares memory with what is still to be read, but for the places that a call names: one row further, one column over, another pitch."""
    assert qkn(L, out=P + 384) == EINVAL and qkn(L, out=P + 16) == EINVAL and qkn(L, out=P + 384, ldo=200) == EINVAL and qkn(L, ld=384, ldo=384, out=P + 368) == EINVAL
    assert qkn(L, bwd=True, out=3 * P + 384) == EINVAL and qkn(L, bwd=True, out=P + 384) == EINVAL and qkn(L, bwd=True, out=P - 384) == EINVAL
    assert qkn(L, bf16=0, out=P + 768) == EINVAL and qkn(L, bf16=0, out=P + 384 * 50) == EINVAL  # (fp32 rows are twice as long)
    assert attn(L, o=P + 1152 * 99) == EINVAL and attn(L, qkv=3 * P, o=3 * P - 16) == EINVAL
    assert attn(L, bwd=True, dqkv=P + 1152) == EINVAL and attn(L, bwd=True, do=2 * P + 1152) == EINVAL and attn(L, bwd=True, dbias=P + 208) == EINVAL
    assert attn(L, bwd=True, dbias=P + 16, ldb=100) == EINVAL
    assert distill(L, dz=P + 4) == EINVAL and distill(L, dz=P + 400) == EINVAL and distill(L, dz=P + 2, db=1) == EINVAL and distill(L, dz=P + 396, ld=100, ldz=200) == EINVAL


def test_wrappers_refuse_cpu_tensors():
    from savit_amd import ops

    z = torch.zeros(4, 192)
    with pytest.raises(ValueError, match="no CPU path"):
        ops.qk_norm_rope_fwd(z, torch.ones(64), torch.ones(64), None, N=4, H=1)
    with pytest.raises(ValueError, match="no CPU path"):
        ops.distill_xent(z, z, z.int())
    with pytest.raises(ValueError, match="no CPU path"):
        ops.relpos_bias_fwd(torch.zeros(3, 2), torch.zeros(2, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="no CPU path"):
        ops.bias_attention_fwd(z.bfloat16(), torch.zeros(1, 4, 4), 1, 4, 1)
    with pytest.raises(ValueError, match="outside"):
        ops.relpos_order(torch.tensor([[0, 3], [1, 0]]), 3)
    with pytest.raises(ValueError):
        ops.relpos_index_1d(10, buckets=6, device="cpu")
    with pytest.raises(ValueError):
        ops.rope_angles_2d(2, 2, 18)


def test_position_tables():
    """The host side: buckets, their lists and the rotation's angles, by their definitions."""
    from savit_amd import ops

    index, n = ops.relpos_index_2d(2, 3, device="cpu")
    assert tuple(index.shape) == (7, 7) and n == 3 * 5 + 3 and int(index.max()) == n - 1
    assert int(index[0, 0]) == n - 1 and bool((index[0, 1:] == n - 3).all()) and bool((index[1:, 0] == n - 2).all())
    assert int(index[1, 1]) == int(index[4, 4]) and int(index[1, 2]) == int(index[5, 6]) and int(index[1, 2]) != int(index[2, 1])
    order, start = ops.relpos_order(index, n)
    flat = index.reshape(-1)
    assert all(bool((flat[order[start[b]:start[b + 1]].long()] == b).all()) for b in range(n)) and int(start[-1]) == 49
    idx, n = ops.relpos_index_1d(300, 32, 128, device="cpu")
    assert n == 32 and int(idx[5, 5]) == 0 and int(idx[5, 6]) == 17 and int(idx[6, 5]) == 1 and int(idx[0, 299]) == 31 and int(idx[299, 0]) == 15
    a = ops.rope_angles_2d(2, 3, 8)
    assert tuple(a.shape) == (7, 4) and float(a[0].abs().sum()) == 0.0 and float(a[1].abs().sum()) == 0.0
    assert a[6, 0] == 1.0 and a[6, 2] == 2.0 and a[3, 0] == 0.0  # row and column of the last patch
    t = ops.rope_table(a, device="cpu")
    assert tuple(t.shape) == (7, 8) and bool((t[0, :4] == 1).all()) and bool((t[0, 4:] == 0).all())
