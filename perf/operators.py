"""Work of the packed-prompt operators: token embedding, causal attention over packed sequences, and the 8-bit integer Linear.

Each case is one pass through one operator.  `run` computes it in elementary torch operations (`own` false) or through the package's
entry points (`own` true): `ops.embedding`, `ops.attention_packed` and `kernels.linear_int8`.

  embedding          out[t] = scale * table[ids[t]] + pos[place[t]]; an id outside the table reads a zero row and receives no gradient
                     dtable[v] = scale * sum_{t: ids[t] = v} dout[t],   dpos[p] = sum_{t: place[t] = p} dout[t]
  attention_packed   rows cu[b] .. cu[b+1]-1 of a packed [q | k | v] projection are one sequence; query i of it sees its keys 0 .. i;
                     `heads` query heads share `kv_heads` key / value heads in consecutive groups; rows past cu[-1] give zeros
  linear_int8        xs[m] = max_k |x[m,k]| / 127 (fp32), xq = round_half_even(x / xs); the same for every row of the weight;
                     y = act(xs[m] * ws[n] * sum_k xq[m,k] wq[n,k] + bias[n]) + residual
"""
import math
import random

import numpy as np
import torch

own = False

_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}
_VOCAB = 49408                 # the text tower's vocabulary; its last two ids open and close every prompt


def listed():
    return [
        # one prompt typed by a user: the text tower's attention and embedding at their smallest, where only latency counts
        dict(name="attn one prompt", op="attn", train=False, dtype="f16", heads=8, kv_heads=8, dim=64, seqs=1, lo=11, hi=11, empty=0, spare=0, draw=1),
        # a batch of 256 prompts of 6 .. 32 tokens (the batch of the `encode_text` command), ViT-B/32 text heads
        dict(name="attn 256 prompts", op="attn", train=False, dtype="f16", heads=8, kv_heads=8, dim=64, seqs=256, lo=6, hi=32, empty=0, spare=0, draw=2),
        # training over ragged sequences with grouped heads, a few empty slots and spare rows at the end of a fixed-size buffer
        dict(name="attn train ragged grouped", op="attn", train=True, dtype="bf16", heads=16, kv_heads=4, dim=64, seqs=24, lo=60, hi=2100, empty=2, spare=37, draw=3),
        # long training sequences, one key / value head per query head, 128 features
        dict(name="attn train long", op="attn", train=True, dtype="bf16", heads=16, kv_heads=16, dim=128, seqs=1, lo=8192, hi=8192, empty=0, spare=0, draw=4),
        # whole long prompts, eight query heads per four key / value heads: the largest forward
        dict(name="attn long grouped", op="attn", train=False, dtype="bf16", heads=32, kv_heads=8, dim=128, seqs=2, lo=15000, hi=16384, empty=0, spare=0, draw=5),
        # the embedding of one prompt
        dict(name="embed one prompt", op="embed", train=False, table="f32", out="f32", vocab=_VOCAB, width=512, seqs=1, lo=11, hi=11, empty=0, spare=0, draw=6),
        # prompt tuning on a batch of prompts: table and position gradients, opening / closing tokens in every prompt
        dict(name="embed train prompts", op="embed", train=True, table="f32", out="f16", vocab=_VOCAB, width=512, seqs=509, lo=6, hi=77, empty=0, spare=3, draw=7),
        # an embedding trained from scratch on long documents
        dict(name="embed train long", op="embed", train=True, table="bf16", out="bf16", vocab=_VOCAB, width=1024, seqs=64, lo=1500, hi=2048, empty=0, spare=0, draw=8),
        # one row through one projection
        dict(name="int8 one row", op="int8", dtype="f16", rows=1, n=2048, k=512, act="none", res=False),
        # the packed rows of 256 prompts through the text tower's first MLP product
        dict(name="int8 prompts", op="int8", dtype="f16", rows=4617, n=2048, k=512, act="quickgelu", res=False),
        # 64 images of 257 tokens through ViT-L/14's first MLP product
        dict(name="int8 vit-l", op="int8", dtype="bf16", rows=16448, n=4096, k=1024, act="quickgelu", res=False),
        # ... and its second one, back into the fp32 residual stream
        dict(name="int8 vit-l residual", op="int8", dtype="bf16", rows=16448, n=1024, k=4096, act="none", res=True),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "embed", "int8", "int8"])
    if op == "attn":
        train = rng.random() < 0.5
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 4])
        total = _logint(rng, 4, 24000)
        hi = min(total, _logint(rng, 1, 8192))
        seqs = max(1, min(1024, total // max(1, (hi + 1) // 2)))
        return dict(op="attn", train=train, dtype=rng.choice(["bf16", "f16"]), heads=heads, kv_heads=kv, dim=rng.choice([64, 64, 128, 128, 80, 40]),
                    seqs=seqs, lo=max(1, hi // _logint(rng, 1, 16)), hi=hi, empty=rng.choice([0, 0, 1, 5]), spare=rng.choice([0, 0, 1, 70]), draw=rng.randrange(1 << 30))
    if op == "embed":
        hi = _logint(rng, 1, 2048)
        seqs = max(1, min(2048, _logint(rng, 1, 100000) // hi))
        kind = rng.choice(["f32", "bf16", "f16"])
        return dict(op="embed", train=rng.random() < 0.6, table=kind, out=rng.choice([kind, "f32"]) if kind != "f32" else rng.choice(["f32", "bf16", "f16"]),
                    vocab=_logint(rng, 50, 60000), width=rng.choice([64, 100, 512, 768, 1000, 1024]), seqs=seqs, lo=max(1, hi // 3), hi=hi,
                    empty=0, spare=rng.choice([0, 0, 9]), draw=rng.randrange(1 << 30))
    while True:
        rows, n, k = _logint(rng, 1, 20000), _logint(rng, 33, 4100), 16 * _logint(rng, 2, 256)
        if rows * n * k <= 16448 * 4096 * 1024:
            break
    return dict(op="int8", dtype=rng.choice(["bf16", "f16"]), rows=rows, n=rng.choice([n, 8 * ((n + 7) // 8)]), k=k, act=rng.choice(["none", "gelu", "quickgelu"]),
                res=rng.random() < 0.3)


def _lens(case):
    """The sequences' lengths: the case's own, the same for every seed."""
    rng = random.Random(case["draw"])
    n = [_logint(rng, case["lo"], case["hi"]) for _ in range(case["seqs"])]
    for _ in range(case["empty"]):
        n.insert(rng.randrange(len(n) + 1), 0)
    return n


def _gen(seed, k):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * seed + k)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def prepare(case, seed):
    s = dict(case=case)
    g = _gen(seed, 1)
    if case["op"] == "attn":
        lens = _lens(case)
        rows, cols = sum(lens) + case["spare"], (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        # projections of normalised activations: unit variance, channels of unequal size
        s["qkv"] = (_randn(g, rows, cols) * torch.exp(0.3 * _randn(g, cols))).to(_DT[case["dtype"]])
        s["lens"] = lens
        s["cu"] = torch.tensor(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32), device="cuda")
        s["scale"] = case["dim"] ** -0.5
        if case["train"]:
            s["dout"] = (_randn(g, rows, case["heads"] * case["dim"]) * 0.1).to(_DT[case["dtype"]])
            if own:
                s["qkv"].requires_grad_()
    elif case["op"] == "embed":
        lens, V, W = _lens(case), case["vocab"], case["width"]
        n = sum(lens)
        # Zipf's law over the vocabulary, with the opening and the closing token around every prompt
        ids = torch.exp(torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * math.log(V)).long().clamp_(1, V) - 1
        ends = torch.from_numpy(np.cumsum(lens)).cuda()
        ids[ends - torch.tensor(lens, device="cuda")] = V - 2
        ids[ends - 1] = V - 1
        place = torch.cat([torch.arange(m) for m in lens])
        if case["spare"]:      # unused rows of the buffer
            ids = torch.cat([ids, torch.full((case["spare"],), -1, device="cuda")])
            place = torch.cat([place, torch.full((case["spare"],), -1)])
        s["ids"], s["place"] = ids, place.cuda()
        s["table"] = (_randn(g, V, W) * 0.02).to(_DT[case["table"]])
        s["pos"] = (_randn(g, max(lens), W) * 0.01).to(_DT[case["table"]])
        s["scale"] = math.sqrt(W) if case["table"] == "bf16" else 1.0
        if case["train"]:
            s["dout"] = (_randn(g, len(ids), W) * 0.1).to(_DT[case["out"]])
            if own:
                s["table"].requires_grad_()
                s["pos"].requires_grad_()
    else:
        R, N, K = case["rows"], case["n"], case["k"]
        # normalised activations with a few large channels; a weight of the usual initial size
        s["x"] = (_randn(g, R, K) * torch.exp(0.5 * _randn(g, K))).to(_DT[case["dtype"]])
        w = _randn(g, N, K) * K ** -0.5
        s["bias"] = _randn(g, N) * 0.1
        s["res"] = _randn(g, R, N) if case["res"] else None
        if own:
            from feed_forward_vqgan_clip_amd import kernels as kern
            s["wq"], s["ws"] = kern.int8_quant(w)
        else:
            s["wq"], s["ws"] = _quant(w)
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------------------
def _quant(x):
    """Rows to 8-bit integers (as fp32 values) and their scales; the quotients in 64 bits, so that values next to a border round right."""
    s = (x.float().abs().amax(1).double() / 127.0).float()
    q = (x.double() / s.double()[:, None]).nan_to_num_(0.0).round_()
    return q.float(), s


def _attn_tiles(case, lens):
    """(first row, length, first query, past the last query) pieces whose score matrices stay moderate."""
    for b, n in enumerate(lens):
        r0, step = sum(lens[:b]), max(64, min(n, (1 << 27) // max(1, n * case["heads"])))
        for q0 in range(0, n, step):
            yield r0, n, q0, min(n, q0 + step)


def _plain_attn(s):
    case, lens = s["case"], s["lens"]
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    x = s["qkv"].float()
    rows = x.shape[0]
    if max(lens) <= 128:
        return _plain_attn_short(s, x)
    q = x[:, :H * D].view(rows, G, H // G, D).permute(1, 2, 0, 3)              # [G, H/G, rows, D]
    k = x[:, H * D:(H + G) * D].view(rows, G, D).permute(1, 0, 2).contiguous()
    v = x[:, (H + G) * D:].view(rows, G, D).permute(1, 0, 2).contiguous()
    out = torch.zeros(G, H // G, rows, D, device=x.device)
    if case["train"]:
        do = s["dout"].float().view(rows, G, H // G, D).permute(1, 2, 0, 3)
        dq, dk, dv = torch.zeros_like(out), torch.zeros_like(k), torch.zeros_like(v)
    for r0, n, q0, q1 in _attn_tiles(case, lens):
        m = q1 - q0
        sl, kl = slice(r0 + q0, r0 + q1), slice(r0, r0 + q1)                  # the keys these queries can see
        kt, vt = k[:, kl], v[:, kl]
        qt = q[:, :, sl].reshape(G, -1, D)
        p = torch.bmm(qt, kt.transpose(1, 2).contiguous()).mul_(s["scale"]).view(G, H // G, m, q1)
        p.masked_fill_(torch.ones(m, q1, dtype=torch.bool, device=x.device).triu_(q0 + 1), float("-inf"))
        p = (p - p.amax(-1, keepdim=True)).exp_()
        p = (p / p.sum(-1, keepdim=True)).view(G, -1, q1)
        o = torch.bmm(p, vt)
        out[:, :, sl] = o.view(G, H // G, m, D)
        if case["train"]:
            dot = do[:, :, sl].reshape(G, -1, D)
            dv[:, kl] += torch.bmm(p.transpose(1, 2).contiguous(), dot)
            dp = torch.bmm(dot, vt.transpose(1, 2).contiguous())
            ds = p * (dp - (dot * o).sum(-1, keepdim=True)) * s["scale"]
            dq[:, :, sl] = torch.bmm(ds, kt).view(G, H // G, m, D)
            dk[:, kl] += torch.bmm(ds.transpose(1, 2).contiguous(), qt)
    dt = s["qkv"].dtype
    out = out.permute(2, 0, 1, 3).reshape(rows, H * D).to(dt)
    if not case["train"]:
        return out
    parts = [dq.permute(2, 0, 1, 3).reshape(rows, H * D), dk.permute(1, 0, 2).reshape(rows, G * D), dv.permute(1, 0, 2).reshape(rows, G * D)]
    return out, torch.cat(parts, 1).to(dt)


def _plain_attn_short(s, x):
    """Short sequences, padded to the longest one: one batched product instead of a loop over the batch."""
    case = s["case"]
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    n, m = len(s["lens"]), max(s["lens"])
    cu = s["cu"].long()
    t = torch.arange(m, device=x.device)
    live = t[None] < (cu[1:] - cu[:-1])[:, None]
    at = (cu[:-1, None] + t[None]).clamp_(max=x.shape[0] - 1)
    y = x[at]                                                                 # [n, m, columns]
    q = y[..., :H * D].view(n, m, H, D).permute(0, 2, 1, 3).reshape(n * H, m, D)
    k = y[..., H * D:(H + G) * D].view(n, m, G, 1, D).expand(n, m, G, H // G, D).permute(0, 2, 3, 4, 1).reshape(n * H, D, m)
    v = y[..., (H + G) * D:].view(n, m, G, 1, D).expand(n, m, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(n * H, m, D)
    p = torch.bmm(q, k).mul_(s["scale"]).masked_fill_(t[None, :] > t[:, None], float("-inf"))
    p = (p - p.amax(-1, keepdim=True)).exp_()
    p = p / p.sum(-1, keepdim=True)
    rows = lambda a: a.reshape(n, -1, m, D).permute(0, 2, 1, 3).reshape(n, m, -1)  # noqa: E731 (heads back into the columns)
    pv = torch.bmm(p, v)
    out = torch.zeros(x.shape[0], H * D, dtype=s["qkv"].dtype, device=x.device)
    out[at[live]] = rows(pv)[live].to(out.dtype)
    if not case["train"]:
        return out
    do = s["dout"].float()[at].masked_fill_(~live[..., None], 0.0).view(n, m, H, D).permute(0, 2, 1, 3).reshape(n * H, m, D)
    ds = p * (torch.bmm(do, v.transpose(1, 2).contiguous()) - (do * pv).sum(-1, keepdim=True)) * s["scale"]
    dq = torch.bmm(ds, k.transpose(1, 2).contiguous())
    dk = torch.bmm(ds.transpose(1, 2).contiguous(), q).view(n * G, H // G, m, D).sum(1)
    dv = torch.bmm(p.transpose(1, 2).contiguous(), do).view(n * G, H // G, m, D).sum(1)
    dqkv = torch.zeros(x.shape, dtype=s["qkv"].dtype, device=x.device)
    dqkv[at[live]] = torch.cat([rows(dq), rows(dk), rows(dv)], -1)[live].to(out.dtype)
    return out, dqkv


def _plain_embed(s):
    case, ids, place = s["case"], s["ids"], s["place"]
    ok = (ids >= 0) & (ids < case["vocab"])
    okp = place >= 0
    out = s["scale"] * s["table"][ids.clamp(0, case["vocab"] - 1)].float() * ok[:, None] + s["pos"][place.clamp(min=0)].float() * okp[:, None]
    out = out.to(_DT[case["out"]])
    if not case["train"]:
        return out
    g = s["dout"].float()
    dt = torch.zeros(s["table"].shape, device=g.device).index_add_(0, ids.clamp(0, case["vocab"] - 1), g * ok[:, None]).mul_(s["scale"])
    dp = torch.zeros(s["pos"].shape, device=g.device).index_add_(0, place.clamp(min=0), g * okp[:, None])
    return out, dt.to(s["table"].dtype), dp.to(s["pos"].dtype)


def _act(kind, v):
    if kind == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * 0.7071067811865476))
    if kind == "quickgelu":
        return v / (1.0 + torch.exp(-1.702 * v))
    return v


def _plain_int8(s):
    case = s["case"]
    q, xs = _quant(s["x"])
    v = _act(case["act"], (q @ s["wq"].t()) * (xs[:, None] * s["ws"][None]) + s["bias"])
    return v + s["res"] if case["res"] else v.to(s["x"].dtype)


# ---- one pass ------------------------------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    if not own:
        return {"attn": _plain_attn, "embed": _plain_embed, "int8": _plain_int8}[case["op"]](s)
    from feed_forward_vqgan_clip_amd import kernels as kern
    from feed_forward_vqgan_clip_amd import ops
    if case["op"] == "attn":
        if not case["train"]:
            return ops.attention_packed(s["qkv"], s["cu"], case["heads"], case["kv_heads"], s["scale"])
        o = ops.attention_packed(s["qkv"], s["cu"], case["heads"], case["kv_heads"], s["scale"])
        return (o.detach(),) + torch.autograd.grad(o, s["qkv"], s["dout"])
    if case["op"] == "embed":
        o = ops.embedding(s["ids"], s["table"], s["scale"], pos=s["pos"], pos_ids=s["place"], out_dtype=_DT[case["out"]])
        return (o.detach(),) + torch.autograd.grad(o, (s["table"], s["pos"]), s["dout"]) if case["train"] else o
    act = {"none": kern.ACT_NONE, "gelu": kern.ACT_GELU, "quickgelu": kern.ACT_QUICKGELU}[case["act"]]
    return kern.linear_int8(s["x"], s["wq"], s["ws"], bias=s["bias"], act=act, residual=s["res"], out_dtype=torch.float32 if case["res"] else None)


def work(case):
    if case["op"] == "attn":
        lens = _lens(case)
        rows, H, G, D = sum(lens) + case["spare"], case["heads"], case["kv_heads"], case["dim"]
        pairs = sum(n * (n + 1) // 2 for n in lens)
        qkv, o = rows * (H + 2 * G) * D * 2, rows * H * D * 2
        # scores and the weighted sum; backward: the scores again, dP, dV, dQ, dK
        return dict(bytes=(2 * qkv + 2 * o) if case["train"] else qkv + o, flops=2 * pairs * H * D * (7 if case["train"] else 2))
    if case["op"] == "embed":
        n, W, V = sum(_lens(case)) + case["spare"], case["width"], case["vocab"]
        v = np.arange(1, V + 1, dtype=np.float64)
        distinct = float(np.sum(1.0 - np.exp(n * np.log1p(-np.log1p(1.0 / v) / math.log(V + 1)))))
        b = 16 * n + (distinct + case["hi"]) * W * _SIZE[case["table"]] + n * W * _SIZE[case["out"]]
        if case["train"]:
            b += n * W * _SIZE[case["out"]] + (V + case["hi"]) * W * _SIZE[case["table"]]
        return dict(bytes=int(b), flops=n * W * (4 if case["train"] else 2))
    R, N, K = case["rows"], case["n"], case["k"]
    return dict(bytes=R * K * 2 + N * K + N * 8 + R * N * (8 if case["res"] else 2), flops=2 * R * N * K)


# ---- the same from the definitions, in 64 bits ---------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "attn":
            return _exact_attn(case, s)
        if case["op"] == "embed":
            V, W = case["vocab"], case["width"]
            ext = lambda t: torch.cat([t.detach().double(), torch.zeros(1, W, device="cuda", dtype=torch.float64)])  # noqa: E731 (a zero row for absent ids)
            ids = torch.where((s["ids"] < 0) | (s["ids"] >= V), V, s["ids"])
            P = s["pos"].shape[0]
            place = torch.where(s["place"] < 0, P, s["place"])
            out = s["scale"] * ext(s["table"]).index_select(0, ids) + ext(s["pos"]).index_select(0, place)
            if not case["train"]:
                return out
            res = [out]
            for rows, idx, mul in ((V, ids, s["scale"]), (P, place, 1.0)):
                order = torch.argsort(idx, stable=True)
                sums = torch.cumsum(s["dout"].double()[order], 0)                  # differences of running sums: ~2^-45 of the largest
                sums = torch.cat([torch.zeros(1, W, device="cuda", dtype=torch.float64), sums])
                edge = torch.searchsorted(idx[order].contiguous(), torch.arange(rows + 1, device="cuda"))
                res.append(mul * (sums[edge[1:]] - sums[edge[:-1]]))
            return tuple(res)
        x, K = s["x"].double(), case["k"]
        top = x.abs().max(dim=1).values
        xs = (top / 127.0).float().double()
        unit = torch.where(xs > 0, xs, torch.ones_like(xs))
        xq = torch.round(x / unit[:, None])
        wq, ws = s["wq"].double(), s["ws"].double()
        y = torch.zeros(case["rows"], case["n"], device="cuda", dtype=torch.float64)
        for k0 in range(0, K, 1024):
            y += xq[:, k0:k0 + 1024] @ wq[:, k0:k0 + 1024].T
        y = y * xs[:, None] * ws + s["bias"].double()
        if case["act"] == "gelu":
            y = y * torch.special.ndtr(y)
        elif case["act"] == "quickgelu":
            y = y * torch.sigmoid(1.702 * y)
        return y + s["res"].double() if case["res"] else y


def _exact_attn(case, s):
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    z = s["qkv"].detach()
    out = torch.zeros(z.shape[0], H * D, device="cuda", dtype=torch.float64)
    grad = torch.zeros(z.shape, device="cuda", dtype=torch.float64) if case["train"] else None
    at = 0
    for n in s["lens"]:
        rows = slice(at, at + n)
        at += n
        if n == 0:
            continue
        late = torch.arange(n, device="cuda")[None] > torch.arange(n, device="cuda")[:, None]
        for h in range(H):
            g = h // (H // G)
            cq, ck, cv = slice(h * D, h * D + D), slice((H + g) * D, (H + g + 1) * D), slice((H + G + g) * D, (H + G + g + 1) * D)
            q, k, v = z[rows, cq].double(), z[rows, ck].double(), z[rows, cv].double()
            a = torch.softmax((q @ k.T * s["scale"]).masked_fill_(late, -math.inf), dim=1)
            out[rows, cq] = a @ v
            if grad is not None:
                do = s["dout"][rows, cq].double()
                grad[rows, cv] += a.T @ do
                da = do @ v.T
                dl = a * (da - (a * da).sum(1, keepdim=True)) * s["scale"]
                grad[rows, cq] = dl @ k
                grad[rows, ck] += dl.T @ q
    return out if grad is None else (out, grad)
