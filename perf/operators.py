"""Measured cases of the position, attention and distillation operators of the encoder's training step.

Three families, named by a case's "op":

  qk_norm_rope  per-head normalisation of queries and keys with the position rotation in the same pass (packed q|k|v rows)
  relpos        attention whose scores get a learned bias, looked up by relative-position bucket, and the gradient of its table
  distill       distillation from the largest logits of a teacher, with the gradient of the student's logits

`run` computes a case in elementary torch operations where `own` is false, and by this repository's operators where it is true."""
import math

import torch

own = False

CLS_BUCKETS = 3  # class token to patch, patch to class token, class token to itself


# --------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one training step's layer of a base-size encoder at 224 px, batch 128: 196 patches and a class token, 12 heads
        {"name": "qkn_train_128x197x12", "op": "qk_norm_rope", "B": 128, "N": 197, "H": 12, "Hk": 12, "hd": 64, "dtype": "bf16", "train": True,
         "center": False, "interleaved": False, "positions": False},
        # the tiny encoder in its default arithmetic, batch 8, statistics with the mean taken out, neighbours rotated together
        {"name": "qkn_train_fp32_8x197x3", "op": "qk_norm_rope", "B": 8, "N": 197, "H": 3, "Hk": 3, "hd": 64, "dtype": "fp32", "train": True,
         "center": True, "interleaved": True, "positions": False},
        # single tokens of four sequences at far positions, eight shared key heads: only latency counts
        {"name": "qkn_token_4x32", "op": "qk_norm_rope", "B": 4, "N": 1, "H": 32, "Hk": 8, "hd": 128, "dtype": "bf16", "train": False,
         "center": False, "interleaved": False, "positions": True},
        # a long prompt of one sequence, 48-wide heads
        {"name": "qkn_prompt_16384x8x48", "op": "qk_norm_rope", "B": 1, "N": 16384, "H": 8, "Hk": 8, "hd": 48, "dtype": "bf16", "train": False,
         "center": False, "interleaved": False, "positions": False},
        # forward and backward of one encoder layer's attention at 224 px, batch 128, with the table's gradient
        {"name": "relpos_train_128x197x12", "op": "relpos", "B": 128, "gh": 14, "gw": 14, "cls": True, "N": 197, "H": 12, "hd": 64, "train": True,
         "ragged": False},
        # inference at 384 px: 577 tokens, 16 heads
        {"name": "relpos_infer_16x577x16", "op": "relpos", "B": 16, "gh": 24, "gw": 24, "cls": True, "N": 577, "H": 16, "hd": 64, "train": False,
         "ragged": False},
        # attention inside 7 x 7 windows, all windows of a batch at once, narrow heads
        {"name": "relpos_window_2048x49x4", "op": "relpos", "B": 2048, "gh": 7, "gw": 7, "cls": False, "N": 49, "H": 4, "hd": 32, "train": True,
         "ragged": False},
        # long sequences of different lengths in one padded batch, buckets by distance
        {"name": "relpos_long_2x1500x8", "op": "relpos", "B": 2, "gh": 0, "gw": 0, "cls": False, "N": 1500, "H": 8, "hd": 64, "train": True, "ragged": True},
        # one small sequence: launches and latency
        {"name": "relpos_small_1x17x3", "op": "relpos", "B": 1, "gh": 4, "gw": 4, "cls": True, "N": 17, "H": 3, "hd": 64, "train": True, "ragged": False},
        # a classifier's batch with hard labels beside the teacher's ten largest logits
        {"name": "distill_128x1000", "op": "distill", "R": 128, "V": 1000, "K": 10, "T": 2.0, "rest": False, "labels": True, "smoothing": 0.1,
         "dtype": "fp32", "grad": "bf16"},
        # a wide label set of odd size, stored teacher logits whose remaining mass is spread evenly
        {"name": "distill_1024x21843", "op": "distill", "R": 1024, "V": 21843, "K": 100, "T": 1.0, "rest": True, "labels": False, "smoothing": 0.0,
         "dtype": "fp32", "grad": "bf16"},
        # a language model's vocabulary, bf16 in and out
        {"name": "distill_2048x131072", "op": "distill", "R": 2048, "V": 131072, "K": 64, "T": 1.5, "rest": False, "labels": False, "smoothing": 0.0,
         "dtype": "bf16", "grad": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 5e12, w["flops"] / 5e13)


def draw(rng):
    op = rng.choice(("qk_norm_rope", "relpos", "distill"))
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        if op == "qk_norm_rope":
            H = rng.choice((1, 2, 3, 4, 6, 8, 12, 16, 32))
            case = {"op": op, "B": _log_int(rng, 1, 256), "N": _log_int(rng, 1, 16384), "H": H, "Hk": rng.choice([k for k in (1, 2, 3, 4, 6, 8, 12, 16, 32) if H % k == 0]),
                    "hd": rng.choice((16, 32, 48, 64, 80, 96, 128, 256)), "dtype": rng.choice(("bf16", "bf16", "fp32")), "train": rng.random() < 0.6,
                    "center": rng.random() < 0.3, "interleaved": rng.random() < 0.4, "positions": rng.random() < 0.4}
        elif op == "relpos":
            flat = rng.random() < 0.35
            gh, gw, cls = (0, 0, False) if flat else (_log_int(rng, 1, 32), _log_int(rng, 1, 32), rng.random() < 0.6)
            case = {"op": op, "B": _log_int(rng, 1, 2048), "gh": gh, "gw": gw, "cls": cls, "N": _log_int(rng, 1, 2048) if flat else gh * gw + int(cls),
                    "H": rng.choice((1, 2, 3, 4, 6, 8, 12, 16)), "hd": rng.choice((16, 32, 48, 64, 64)), "train": rng.random() < 0.6, "ragged": rng.random() < 0.4}
        else:
            V = _log_int(rng, 2, 160000)
            case = {"op": op, "R": _log_int(rng, 1, 8192), "V": V, "K": min(V, _log_int(rng, 1, 256)), "T": rng.choice((0.5, 1.0, 1.0, 2.0, 4.0)),
                    "rest": rng.random() < 0.4, "labels": rng.random() < 0.5, "smoothing": rng.choice((0.0, 0.1)), "dtype": rng.choice(("bf16", "fp32")),
                    "grad": rng.choice(("bf16", "fp32"))}
        if _cost(case) <= most:
            return case


def work(case):
    if case["op"] == "qk_norm_rope":
        rows, size = case["B"] * case["N"], 2 if case["dtype"] == "bf16" else 4
        row = (case["H"] + 2 * case["Hk"]) * case["hd"] * size
        qk = (case["H"] + case["Hk"]) * case["hd"]
        # forward reads and writes a row; backward reads the cotangent row and the saved queries and keys and writes a row
        return {"bytes": rows * (2 * row + (2 * row + qk * size if case["train"] else 0)), "flops": rows * qk * (12 + (24 if case["train"] else 0))}
    if case["op"] == "relpos":
        B, N, H, hd = case["B"], case["N"], case["H"], case["hd"]
        row = B * N * H * hd * 2
        # q, k, v in, o out; backward: q, k, v, the cotangent in, three gradients out.  Products: 2 forward, 5 backward
        return {"bytes": row * (4 + (7 if case["train"] else 0)) + N * N * 4, "flops": 2.0 * B * H * N * N * hd * (2 + (5 if case["train"] else 0))}
    size, gsize = (2 if case["dtype"] == "bf16" else 4), (2 if case["grad"] == "bf16" else 4)
    return {"bytes": case["R"] * (case["V"] * (size + gsize) + case["K"] * 8.0), "flops": case["R"] * case["V"] * 8.0}


# --------------------------------------------------------------------------------------------- inputs
def _dtype(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


def _relpos_index(case):
    """int32 [N, N] bucket of (query, key), and the number of buckets."""
    N = case["N"]
    if not case["gh"]:  # by distance: half the buckets for either sign, exact up to 8, then by the logarithm up to 128
        d = torch.arange(N)[None, :] - torch.arange(N)[:, None]
        a = d.abs()
        far = 8 + (torch.log(a.clamp(min=1).double() / 8) / math.log(16.0) * 8).long()
        return (torch.where(a < 8, a, far.clamp(max=15)) + 16 * (d > 0).long()).int(), 32
    gh, gw = case["gh"], case["gw"]
    y, x = torch.arange(gh * gw) // gw, torch.arange(gh * gw) % gw
    patch = (y[:, None] - y[None, :] + gh - 1) * (2 * gw - 1) + (x[:, None] - x[None, :] + gw - 1)
    n = (2 * gh - 1) * (2 * gw - 1)
    if not case["cls"]:
        return patch.int(), n
    index = torch.empty((N, N), dtype=torch.long)
    index[1:, 1:] = patch
    index[0, :], index[:, 0], index[0, 0] = n, n + 1, n + 2
    return index.int(), n + CLS_BUCKETS


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, dtype=torch.float32, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int32)

    s = dict(case)
    if case["op"] == "qk_norm_rope":
        rows, hd, dt = case["B"] * case["N"], case["hd"], _dtype(case["dtype"])
        cols = (case["H"] + 2 * case["Hk"]) * hd
        length = max(case["N"], 4096) if case["positions"] else case["N"]
        freq = 10000.0 ** (-torch.arange(hd // 2, device="cuda", dtype=torch.float64) / (hd // 2))
        angle = torch.arange(length, device="cuda", dtype=torch.float64)[:, None] * freq
        s["table"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        s["qkv"] = normal(rows, cols, dtype=dt)
        s["wq"], s["wk"] = 1 + normal(hd, scale=0.2), 1 + normal(hd, scale=0.2)
        s["pos"] = whole(0, length, rows) if case["positions"] else None
        s["dout"] = normal(rows, cols, dtype=dt, scale=1e-2) if case["train"] else None
    elif case["op"] == "relpos":
        B, N, H, hd = case["B"], case["N"], case["H"], case["hd"]
        index, nb = _relpos_index(case)
        s["index"], s["nb"] = index.cuda(), nb
        flat = s["index"].reshape(-1).long()
        s["order"] = torch.sort(flat, stable=True).indices.int()
        s["start"] = torch.cat([torch.zeros(1, dtype=torch.long, device="cuda"), torch.bincount(flat, minlength=nb).cumsum(0)]).int()
        s["table_nb"] = normal(nb, H, scale=0.5)
        s["qkv"] = normal(B * N, 3 * H * hd, dtype=torch.bfloat16)
        s["qkv"][:, : H * hd] *= hd ** -0.5
        s["lens"] = whole(0, N + 1, B) if case["ragged"] else None
        s["dout"] = normal(B * N, H * hd, dtype=torch.bfloat16, scale=1e-2) if case["train"] else None
    else:
        R, V, K = case["R"], case["V"], case["K"]
        s["z"] = normal(R, V, dtype=_dtype(case["dtype"]), scale=2.0)
        apart = max(1, V // 4096)  # a teacher that the student follows roughly, sure of classes spread over the whole set
        teacher = s["z"][:, ::apart][:, :4096].float()
        top, at = (teacher + normal(*teacher.shape)).topk(K, dim=1)
        s["top"], s["at"] = top.contiguous(), (at * apart).int().contiguous()
        tail = math.log(V - K) if V > K else -math.inf
        s["lse"] = torch.logaddexp(torch.logsumexp(top / case["T"], 1), torch.full((R,), tail, device="cuda")) if case["rest"] else None
        s["labels"] = whole(0, V, R) if case["labels"] else None
    return s


# --------------------------------------------------------------------------------------------- one pass
def run(s):
    if own:
        return {"qk_norm_rope": _own_qk, "relpos": _own_relpos, "distill": _own_distill}[s["op"]](s)
    return {"qk_norm_rope": _plain_qk, "relpos": _plain_relpos, "distill": _plain_distill}[s["op"]](s)


def _own_qk(s):
    from savit_amd import ops

    kw = dict(N=s["N"], H=s["H"], Hk=s["Hk"], head_dim=s["hd"], positions=s["pos"], q_scale=s["hd"] ** -0.5, center=s["center"], interleaved=s["interleaved"])
    out = ops.qk_norm_rope_fwd(s["qkv"], s["wq"], s["wk"], s["table"], **kw)
    if not s["train"]:
        return out
    dw = torch.zeros(2, s["hd"], device="cuda")
    dqkv = ops.qk_norm_rope_bwd(s["dout"], s["qkv"], s["wq"], s["wk"], s["table"], dw[0], dw[1], out=torch.empty_like(s["dout"]), **kw)
    return out, dqkv, dw


def _own_relpos(s):
    from savit_amd import ops

    B, N, H, hd = s["B"], s["N"], s["H"], s["hd"]
    bias = ops.relpos_bias_fwd(s["table_nb"], s["index"])
    o, lse = ops.bias_attention_fwd(s["qkv"], bias, B, N, H, head_dim=hd, lens=s["lens"])
    if not s["train"]:
        return o, lse
    dqkv, dbias = ops.bias_attention_bwd(s["qkv"], bias, s["dout"], lse, B, N, H, dq_scale=hd ** -0.5, head_dim=hd, lens=s["lens"])
    dtable = torch.zeros_like(s["table_nb"])
    ops.relpos_bias_bwd(dbias, s["order"], s["start"], dtable)
    return o, lse, dqkv, dtable


def _own_distill(s):
    from savit_amd import ops

    dz = torch.empty(s["z"].shape, dtype=_dtype(s["grad"]), device="cuda")
    loss = torch.empty(s["R"], device="cuda")
    hard = 0.5 if s["labels"] is not None else 0.0
    ops.distill_xent(s["z"], s["top"], s["at"], temperature=s["T"], distill_weight=1.0 - hard, teacher_lse=s["lse"], labels=s["labels"], hard_weight=hard,
                     label_smoothing=s["smoothing"], loss_rows=loss, dlogits=dz)
    return loss, dz


def _rotate(x, c, sn, inter):
    """The pairs of the last axis turned by the angle whose cosine and sine are c, sn."""
    if inter:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * c - b * sn, a * sn + b * c], -1).reshape(x.shape)
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return torch.cat([a * c - b * sn, a * sn + b * c], -1)


def _plain_qk(s):
    H, Hk, hd, N = s["H"], s["Hk"], s["hd"], s["N"]
    rows = s["qkv"].shape[0]
    at = s["pos"].long() if s["pos"] is not None else torch.arange(rows, device="cuda") % N
    t = s["table"][at]
    c, sn = t[:, None, : hd // 2], t[:, None, hd // 2 :]
    x = s["qkv"][:, : (H + Hk) * hd].float().view(rows, H + Hk, hd)
    if s["center"]:
        x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    xn = x * r
    w = torch.cat([s["wq"].expand(H, hd) * hd ** -0.5, s["wk"].expand(Hk, hd)])
    y = _rotate(xn * w, c, sn, s["interleaved"])
    out = torch.cat([y.reshape(rows, -1).to(s["qkv"].dtype), s["qkv"][:, (H + Hk) * hd :]], 1)
    if not s["train"]:
        return out
    dy = s["dout"][:, : (H + Hk) * hd].float().view(rows, H + Hk, hd)
    gw = _rotate(dy, c, -sn, s["interleaved"])
    d = gw * xn
    dw = torch.stack([d[:, :H].sum((0, 1)) * hd ** -0.5, d[:, H:].sum((0, 1))])
    gx = gw * w
    dx = gx - xn * (gx * xn).mean(-1, keepdim=True)
    if s["center"]:
        dx = dx - gx.mean(-1, keepdim=True)
    dqkv = torch.cat([(dx * r).reshape(rows, -1).to(s["dout"].dtype), s["dout"][:, (H + Hk) * hd :]], 1)
    return out, dqkv, dw


def _plain_relpos(s):
    B, N, H, hd = s["B"], s["N"], s["H"], s["hd"]
    q, k, v = s["qkv"].float().view(B, N, 3, H, hd).permute(2, 0, 3, 1, 4).contiguous()
    score = q @ k.transpose(2, 3).contiguous()
    score += s["table_nb"][s["index"].long()].permute(2, 0, 1)
    if s["lens"] is not None:
        inside = torch.arange(N, device="cuda")[None, :] < s["lens"][:, None]
        score.masked_fill_(~(inside[:, None, :, None] & inside[:, None, None, :]), -math.inf)
    top = score.amax(-1, keepdim=True)
    p = (score - torch.where(top == -math.inf, 0.0, top)).exp()
    total = p.sum(-1, keepdim=True)
    lse = (top + total.log()).squeeze(-1)
    p = p / torch.where(total == 0, 1.0, total)
    o = (p @ v).permute(0, 2, 1, 3).reshape(B * N, H * hd).to(torch.bfloat16)
    if not s["train"]:
        return o, lse
    do = s["dout"].float().view(B, N, H, hd).permute(0, 2, 1, 3).contiguous()
    dv = p.transpose(2, 3).contiguous() @ do
    dp = do @ v.transpose(2, 3).contiguous()
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    dq = (ds @ k) * hd ** -0.5
    dk = ds.transpose(2, 3).contiguous() @ q
    dqkv = torch.stack([dq, dk, dv]).permute(1, 3, 0, 2, 4).reshape(B * N, 3 * H * hd).to(torch.bfloat16)
    db = ds.double().sum(0).reshape(H, N * N)[:, s["order"].long()].cumsum(1)
    db = torch.cat([db.new_zeros(H, 1), db], 1)[:, s["start"].long()]
    return o, lse, dqkv, (db[:, 1:] - db[:, :-1]).t().contiguous().float()


def _plain_distill(s):
    R, V, T = s["R"], s["V"], s["T"]
    z, at = s["z"].float(), s["at"].long()
    hard = 0.5 if s["labels"] is not None else 0.0
    soft = 1.0 - hard
    lq = z / T
    top = lq.amax(1, keepdim=True)
    lq = lq - (top + (lq - top).exp().sum(1, keepdim=True).log())
    t = s["top"] / T
    if s["rest"]:
        p = (t - s["lse"][:, None]).exp()
        left = (1 - p.sum(1)).clamp(min=0) if V > p.shape[1] else torch.zeros(R, device="cuda")
        share = left / max(V - p.shape[1], 1)
    else:
        m = t.amax(1, keepdim=True)
        p = (t - m).exp()
        p = p / p.sum(1, keepdim=True)
        left = share = torch.zeros(R, device="cuda")
    at_top = lq.gather(1, at)
    loss = (p * (p.log() - at_top)).sum(1)
    if s["rest"]:
        others = lq.double().sum(1) - at_top.double().sum(1)
        loss = loss + torch.where(left > 0, left * share.log(), 0.0) - (share.double() * others).float()
    target = share[:, None].expand(R, V).scatter(1, at, p)
    dz = (soft * T) * (lq.exp() * (p.sum(1) + left)[:, None] - target)
    loss = (soft * T * T) * loss
    if s["labels"] is not None:
        m = z.amax(1, keepdim=True)
        lz = z - (m + (z - m).exp().sum(1, keepdim=True).log())
        lab, a = s["labels"].long()[:, None], s["smoothing"]
        loss = loss - hard * ((1 - a) * lz.gather(1, lab).squeeze(1) + a * lz.mean(1))
        dz = dz + hard * (lz.exp() - a / V)
        dz.scatter_add_(1, lab, torch.full((R, 1), -hard * (1 - a), device="cuda"))
    return loss, (dz / R).to(_dtype(s["grad"]))


# --------------------------------------------------------------------------------------------- the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"qk_norm_rope": _exact_qk, "relpos": _exact_relpos, "distill": _exact_distill}[case["op"]](s)


def _exact_qk(s):
    H, Hk, hd = s["H"], s["Hk"], s["hd"]
    rows = s["qkv"].shape[0]
    full = s["qkv"].double().requires_grad_()
    wq, wk = s["wq"].double().requires_grad_(), s["wk"].double().requires_grad_()
    at = torch.remainder(torch.arange(rows, device="cuda"), s["N"]) if s["pos"] is None else s["pos"].long()
    turn = torch.complex(s["table"][:, : hd // 2].double(), s["table"][:, hd // 2 :].double())[at][:, None]

    def one(x, w, scale):
        if s["center"]:
            x = x - x.mean(-1, keepdim=True)
        x = w * scale * x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt()
        pair = x.unflatten(-1, (hd // 2, 2)) if s["interleaved"] else x.unflatten(-1, (2, hd // 2)).transpose(-1, -2)
        turned = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        return (turned if s["interleaved"] else turned.transpose(-1, -2)).reshape(rows, -1)

    q, k, v = full.split([H * hd, Hk * hd, Hk * hd], 1)
    out = torch.cat([one(q.reshape(rows, H, hd), wq, hd ** -0.5), one(k.reshape(rows, Hk, hd), wk, 1.0), v], 1)
    if not s["train"]:
        return out.detach()
    dx, dwq, dwk = torch.autograd.grad(out, (full, wq, wk), s["dout"].double())
    return out.detach(), dx, torch.stack([dwq, dwk])


def _exact_relpos(s):
    B, N, H, hd = s["B"], s["N"], s["H"], s["hd"]
    full, table = s["qkv"].double().requires_grad_(), s["table_nb"].double().requires_grad_()
    q, k, v = full.view(B, N, 3, H, hd).unbind(2)
    with torch.set_grad_enabled(s["train"]):
        score = torch.einsum("bihe,bjhe->bhij", q, k) + table.index_select(0, s["index"].reshape(-1).long()).view(N, N, H).permute(2, 0, 1)
        if s["lens"] is not None:
            there = torch.arange(N, device="cuda") < s["lens"].view(B, 1)
            keep = there.view(B, 1, 1, N) & there.view(B, 1, N, 1)
            lse = torch.logsumexp(score.detach().masked_fill(~keep, -math.inf), -1)
            score = torch.where(keep, score, -1e300)
            weight = torch.softmax(score, -1) * keep
        else:
            lse = torch.logsumexp(score.detach(), -1)
            weight = torch.softmax(score, -1)
        del score
        o = torch.einsum("bhij,bjhe->bihe", weight, v).reshape(B * N, H * hd)
        # queries enter already scaled: their gradient is that of the unscaled ones
    if not s["train"]:
        return o.detach(), lse
    dqkv, dtable = torch.autograd.grad(o, (full, table), s["dout"].double())
    dqkv[:, : H * hd] *= hd ** -0.5
    return o.detach(), lse, dqkv, dtable


def _exact_distill(s):
    R, V, T = s["R"], s["V"], s["T"]
    if R * V > 1 << 28:
        return None
    z = s["z"].double().requires_grad_()
    hard = 0.5 if s["labels"] is not None else 0.0
    t = s["top"].double() / T
    target = torch.zeros(R, V, dtype=torch.float64, device="cuda")
    if s["rest"]:
        p = (t - s["lse"].double().view(R, 1)).exp()
        target += (1 - p.sum(1, keepdim=True)).clamp(min=0) / max(V - p.shape[1], 1)
    else:
        p = torch.softmax(t, 1)
    target.scatter_(1, s["at"].long(), p)
    loss = (1 - hard) * T * T * (torch.xlogy(target, target) - target * torch.log_softmax(z / T, 1)).sum(1)
    if s["labels"] is not None:
        loss = loss + hard * torch.nn.functional.cross_entropy(z, s["labels"].long(), reduction="none", label_smoothing=s["smoothing"])
    (dz,) = torch.autograd.grad(loss.sum() / R, z)
    return loss.detach(), dz
