"""Packed-prompt operators on the GPU against plain 64-bit forms: ops.embedding, ops.attention_packed, kernels.linear_int8.

Every bound is computed from the inputs: half a step of the 16-bit type per rounding that the kernels make (u), 2^-24 per fp32 operation."""
import math

import pytest
import torch

from feed_forward_vqgan_clip_amd import kernels as K
from feed_forward_vqgan_clip_amd import ops

pytestmark = pytest.mark.gpu
BF, HF, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
E = 2.0 ** -24


def half(dt):
    return torch.finfo(dt).eps / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32, mul=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * mul).to(dtype)


def within(got, want, bound, what):
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} out of bound, worst excess {float((err - bound).max()):.3e} (error {float(err.max()):.3e})"


def offsets(lens):
    return torch.tensor([0] + list(torch.tensor(lens, dtype=torch.long).cumsum(0)), dtype=torch.int32, device="cuda")


# ---- attention -----------------------------------------------------------------------------------------------------------------
def attn_reference(q, k, v, lens, scale, do=None):
    """Outputs, gradients and the bounds of their errors, in 64 bits.  q (T, H, D), k / v (T, G, D)."""
    T, H, D = q.shape
    G = k.shape[1]
    u = half(q.dtype)
    out = torch.zeros(T, H, D, dtype=F64, device=q.device)
    bo = torch.zeros_like(out)
    if do is not None:
        dq, bq = torch.zeros_like(out), torch.zeros_like(out)
        dk, dv, bk, bv = (torch.zeros(T, G, D, dtype=F64, device=q.device) for _ in range(4))
    at = 0
    for n in lens:
        r = slice(at, at + n)
        at += n
        if n == 0:
            continue
        late = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1)
        for h in range(H):
            g = h // (H // G)
            Q, Kk, V = q[r, h].double(), k[r, g].double(), v[r, g].double()
            s = (Q @ Kk.T * scale).masked_fill(late, -math.inf)
            p = torch.softmax(s, 1)
            # a score: D products and sums in fp32, the exponent's own rounding (arguments up to its magnitude)
            es = E * ((D + 4) * float((Q.abs() @ Kk.abs().T).max()) * scale + 16)
            ep = 2 * es + 4 * E                                    # numerator and denominator
            o, a = p @ V, p @ V.abs()
            out[r, h] = o
            # weights rounded to the 16-bit type, fp32 sums over up to n keys, the output's own rounding
            bo[r, h] = u * (a + o.abs()) * (1 + u) + (ep + n * E) * a * 2
            if do is None:
                continue
            dO = do[r, h].double()
            dP = dO @ V.T
            dl = (dO * o).sum(1, keepdim=True)
            ds = p * (dP - dl) * scale
            dq[r, h] = ds @ Kk
            dk[r, g] += ds.T @ Q
            dv[r, g] += p.T @ dO
            # delta is taken from the rounded output; dP and delta are fp32 sums over D
            edl = (dO.abs() * (bo[r, h])).sum(1, keepdim=True) + E * (D + 2) * (dO * o).abs().sum(1, keepdim=True)
            edp = E * (D + 2) * (dO.abs() @ V.abs().T)
            eds = u * ds.abs() + scale * p * (edl + edp) * (1 + u) + (ep + 4 * E) * p * scale * (dP.abs() + dl.abs()) * 2
            m = H // G * n
            bq[r, h] = eds @ Kk.abs() + u * dq[r, h].abs() + n * E * (ds.abs() @ Kk.abs()) * 2
            bk[r, g] += eds.T @ Q.abs() + m * E * (ds.abs().T @ Q.abs()) * 2
            bv[r, g] += (u + 2 * ep + m * E * 2) * (p.T @ dO.abs())
    if do is None:
        return out, bo
    tiny = torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps      # half a step of the subnormal range of the stored result
    bk += u * dk.abs()
    bv += u * dv.abs()
    return (out, dq, dk, dv), (bo + tiny, bq * (1 + u) + tiny, bk * (1 + u) + tiny, bv * (1 + u) + tiny)


ATTN = [  # lens, heads, kv_heads, head_dim
    ([1], 1, 1, 64),
    ([1, 2, 3, 31, 32, 33], 8, 8, 64),
    ([63, 64, 65], 2, 1, 64),
    ([127, 128, 129, 5], 4, 2, 128),
    ([0, 7, 0, 0, 200, 0], 3, 1, 64),
    ([300], 8, 2, 128),
    ([77, 12, 40], 5, 5, 80),
    ([130, 9], 2, 2, 8),
    ([513, 64, 190], 16, 4, 40),
    ([1030], 2, 2, 120),
    ([11] * 70, 2, 2, 64),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("case", range(len(ATTN)))
def test_attention_packed_forward_and_gradients(cuda, case, dtype):
    lens, H, G, D = ATTN[case]
    g = gen(case)
    spare = case % 3
    T = sum(lens) + spare
    qkv = randn(g, T, (H + 2 * G) * D, dtype=dtype)
    do = randn(g, T, H * D, dtype=dtype)
    cu = offsets(lens)
    q, k, v = ops._split_heads(qkv, H, G)
    (o, dq, dk, dv), (bo, bq, bk, bv) = attn_reference(q, k, v, lens, D ** -0.5, do.view(T, H, D))
    leaf = qkv.clone().requires_grad_()
    got = ops.attention_packed(leaf, cu, H, G)
    within(got.view(T, H, D), o, bo, "out")
    (dqkv,) = torch.autograd.grad(got, leaf, do)
    gq, gk, gv = ops._split_heads(dqkv, H, G)
    within(gq, dq, bq, "dq")
    within(gk, dk, bk, "dk")
    within(gv, dv, bv, "dv")
    if spare:
        assert float(got[T - spare:].abs().max()) == 0 and float(dqkv[T - spare:].abs().max()) == 0
    # the same bits again, and without the statistics
    with torch.no_grad():
        assert torch.equal(ops.attention_packed(qkv, cu, H, G), got)
    leaf2 = qkv.clone().requires_grad_()
    (again,) = torch.autograd.grad(ops.attention_packed(leaf2, cu, H, G), leaf2, do)
    assert torch.equal(again, dqkv)


# the backward splits a key tile's walk in four, in two or not at all, by the number of tiles times key heads; among 2 .. 63 sequences it takes
# the tiles by the length of their walks, otherwise in order
MIXED = [300, 200, 129, 0, 511, 33, 256]
SPLITS = [  # lens, rows behind them, heads, kv_heads, head_dim
    (MIXED, 37, 4, 2, 64),
    (MIXED, 300, 4, 2, 128),
    (MIXED, 37, 48, 48, 64),
    (MIXED, 37, 96, 48, 128),
    (MIXED, 37, 64, 64, 72),
    ([1500], 0, 96, 96, 64),
    ([68, 72] * 35, 3, 8, 4, 64),
    ([68, 72] * 35, 3, 8, 8, 128),
    ([68, 72] * 35, 3, 16, 16, 64),
    ([0, 900] + [64] * 61, 130, 4, 4, 64),
]


@pytest.mark.parametrize("case", range(len(SPLITS)))
def test_attention_packed_gradients_at_every_split(cuda, case):
    lens, spare, H, G, D = SPLITS[case]
    g = gen(900 + case)
    T = sum(lens) + spare
    qkv = randn(g, T, (H + 2 * G) * D, dtype=BF).requires_grad_()
    do = randn(g, T, H * D, dtype=BF)
    q, k, v = ops._split_heads(qkv.detach(), H, G)
    (o, dq, dk, dv), (bo, bq, bk, bv) = attn_reference(q, k, v, lens, D ** -0.5, do.view(T, H, D))
    got = ops.attention_packed(qkv, offsets(lens), H, G)
    within(got.view(T, H, D), o, bo, "out")
    (dqkv,) = torch.autograd.grad(got, qkv, do)
    for name, a, b, c in zip(("dq", "dk", "dv"), ops._split_heads(dqkv, H, G), (dq, dk, dv), (bq, bk, bv)):
        within(a, b, c, name)
    if spare:
        assert float(got[T - spare:].abs().max()) == 0 and float(dqkv[T - spare:].abs().max()) == 0


def test_attention_packed_gradient_by_differences(cuda):
    """The change of sum(out * w) along the gradient's own signs, through the forward kernel alone.  What the difference may be off by: the
    truncation (the 64-bit forward's own difference against its gradient), every output's bound on both sides, every gradient's bound."""
    g = gen(5)
    lens, H, G, D = [40, 70], 4, 2, 64
    T = sum(lens)
    qkv = randn(g, T, (H + 2 * G) * D, dtype=HF)
    w = randn(g, T, H * D, dtype=HF)
    cu = offsets(lens)
    leaf = qkv.clone().requires_grad_()
    (d,) = torch.autograd.grad(ops.attention_packed(leaf, cu, H, G), leaf, w)
    h = 2.0 ** -6
    lo, hi = (qkv.float() - h * d.sign()).half(), (qkv.float() + h * d.sign()).half()
    wd = w.double().view(T, H, D)
    ref = lambda x: attn_reference(*ops._split_heads(x, H, G), lens, D ** -0.5)  # noqa: E731
    (o_hi, b_hi), (o_lo, b_lo) = ref(hi), ref(lo)
    (_, *grads), (_, *bounds) = attn_reference(*ops._split_heads(qkv, H, G), lens, D ** -0.5, w.view(T, H, D))
    move = ops._split_heads(hi.double() - lo.double(), H, G)
    exact = sum(float((a * b).sum()) for a, b in zip(grads, move))
    trunc = abs(float(((o_hi - o_lo) * wd).sum()) - exact)
    slack = float(((b_hi + b_lo) * wd.abs()).sum()) + sum(float((a * b.abs()).sum()) for a, b in zip(bounds, move))
    with torch.no_grad():
        fd = float(((ops.attention_packed(hi, cu, H, G).double() - ops.attention_packed(lo, cu, H, G).double()) * w.double()).sum())
    got = float((d.double() * (hi.double() - lo.double())).sum())
    assert abs(fd - got) <= trunc + slack, (fd, got, trunc, slack)
    assert trunc + slack < 0.2 * abs(exact)                        # the comparison says something


def test_attention_packed_strided_views_and_given_output(cuda):
    g = gen(7)
    lens, H, G, D = [50, 90, 3], 4, 2, 64
    T = sum(lens) + 6
    wide = randn(g, T, (H + 2 * G) * D + 64, dtype=BF)
    qkv = wide[:, 32:32 + (H + 2 * G) * D]
    cu = offsets(lens)
    want = ops.attention_packed(qkv.contiguous(), cu, H, G)
    assert torch.equal(ops.attention_packed(qkv, cu, H, G), want)
    # heads outermost (T-strided), an output with rows of its own that keeps its tail
    q, k, v = (t.permute(1, 0, 2).contiguous().permute(1, 0, 2) for t in ops._split_heads(qkv, H, G))
    buf = torch.full((T, H, 2 * D), 3.0, dtype=BF, device="cuda")
    out, _ = K.attn_packed_fwd(q, k, v, cu, D ** -0.5, out=buf[:, :, :D])
    assert torch.equal(out[:T - 6].reshape(T - 6, -1), want[:T - 6])
    assert bool((buf[T - 6:] == 3.0).all()) and bool((buf[:, :, D:] == 3.0).all())
    leaf = wide.clone().requires_grad_()
    do = randn(g, T, H * D, dtype=BF)
    (dw,) = torch.autograd.grad(ops.attention_packed(leaf[:, 32:32 + (H + 2 * G) * D], cu, H, G), leaf, do)
    leaf2 = qkv.contiguous().requires_grad_()
    (d2,) = torch.autograd.grad(ops.attention_packed(leaf2, cu, H, G), leaf2, do)
    assert torch.equal(dw[:, 32:32 + (H + 2 * G) * D], d2)
    # a broadcast output gradient (sum().backward() hands over an expanded scalar)
    leaf3 = qkv.contiguous().requires_grad_()
    ops.attention_packed(leaf3, cu, H, G).sum().backward()
    leaf4 = qkv.contiguous().requires_grad_()
    (d4,) = torch.autograd.grad(ops.attention_packed(leaf4, cu, H, G), leaf4, torch.ones(T, H * D, dtype=BF, device="cuda"))
    assert torch.equal(leaf3.grad, d4)


@pytest.mark.parametrize("D", [64, 128])
def test_attention_packed_matches_single_sequences(cuda, D):
    """Sequences do not see each other: every one alone gives the same bits, whatever its neighbours hold (NaN included)."""
    g = gen(9)
    lens, H, G = [33, 100, 64, 1, 190], 4, 4
    qkv = randn(g, sum(lens), 3 * H * D, dtype=HF)
    want = ops.attention_packed(qkv, offsets(lens), H)
    at = 0
    for i, n in enumerate(lens):
        alone = ops.attention_packed(qkv[at:at + n].contiguous(), offsets([n]), H)
        assert torch.equal(alone, want[at:at + n])
        dirty = torch.full_like(qkv, float("nan"))
        dirty[at:at + n] = qkv[at:at + n]
        assert torch.equal(ops.attention_packed(dirty, offsets(lens), H)[at:at + n], want[at:at + n])
        at += n


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("lens,H,G,D", [([70], 2, 1, 64), ([200, 45], 4, 2, 128), ([20, 9, 31], 2, 2, 64), ([150], 2, 2, 40)])
def test_attention_packed_nonfinite_values_stay_behind_the_mask(cuda, lens, H, G, D, value):
    """An inf / NaN in a token's v or k reaches no earlier query, one in its q or output gradient reaches no later key."""
    T, scale = sum(lens), D ** -0.5
    g = gen(17)
    clean, do = randn(g, T, (H + 2 * G) * D, dtype=BF), randn(g, T, H * D, dtype=BF)
    cu = offsets(lens)

    def run(x, d):
        leaf = x.clone().requires_grad_()
        o = ops.attention_packed(leaf, cu, H, G)
        return (o.detach().view(T, H, D),) + ops._split_heads(torch.autograd.grad(o, leaf, d)[0], H, G)

    start = 0
    for n in lens:
        for t in {start, start + n // 3, start + n - 1}:
            for what in ("v", "k", "q", "do"):
                x, d = clean.clone(), do.clone()
                parts = dict(zip("qkv", ops._split_heads(x, H, G)), do=d.view(T, H, D))
                parts[what][t, :, 3 % D] = value
                parts[what][t, -1] = value
                got = run(x, d)
                # what must not notice the token: as if it held zeros (64 bits), to the usual bounds
                parts[what][t] = 0
                ref, bound = attn_reference(*ops._split_heads(x, H, G), lens, scale, d.view(T, H, D))
                other = [r for r in range(T) if r < start or r >= start + n]
                before, after = list(range(start, t)), list(range(t + 1, start + n))
                rows = {"v": (before, before, [], []), "k": (before, before, [], []), "q": (before + after, before + after, after, after),
                        "do": (list(range(start, start + n)), before + after, after, after)}[what]
                for name, a, b, e, keep in zip(("out", "dq", "dk", "dv"), got, ref, bound, rows):
                    within(a[keep + other], b[keep + other], e[keep + other], f"{name} with {what}[{t}] = {value}")
                if what == "v":
                    assert not bool(torch.isfinite(got[0][t:start + n, -1]).any())
        start += n


def test_attention_packed_bad_offsets_stay_inside(cuda):
    """Offsets that descend or leave the tensor are clamped: other rows' values may come out, nothing outside is touched."""
    g = gen(11)
    H, D, T = 2, 64, 100
    qkv = randn(g, T, 3 * H * D, dtype=BF)
    for cu in ([0, 500], [-7, 30, 90], [0, 80, 20, 100], [100, 0]):
        got = ops.attention_packed(qkv, torch.tensor(cu, dtype=torch.int32, device="cuda"), H)
        torch.cuda.synchronize()
        assert got.shape == (T, H * D)


def test_attention_packed_large_scores(cuda):
    """Scores of hundreds: the running maximum carries the exponent; a row dominated by one key returns that key's value."""
    T, D = 200, 64
    q = torch.zeros(T, 1, D, dtype=BF, device="cuda")
    k = torch.zeros(T, 1, D, dtype=BF, device="cuda")
    q[:, 0, 0] = 64.0
    k[:, 0, 0] = torch.arange(T, device="cuda").to(BF)              # rounds: equal neighbours share the weight
    v = randn(gen(13), T, 1, D, dtype=BF)
    o, lse = K.attn_packed_fwd(q, k, v, offsets([T]), 1.0, want_lse=True)
    ref, bound = attn_reference(q, k, v, [T], 1.0)
    within(o, ref, bound, "out")
    assert bool(torch.isfinite(lse).all())


def test_attention_packed_gradient_that_starts_anywhere(cuda):
    """An incoming gradient that is a piece of a larger buffer, at an odd offset."""
    g = gen(77)
    lens, H, D = [5, 40, 3], 2, 24
    qkv = randn(g, 48, 3 * H * D, dtype=HF).requires_grad_()
    buf = randn(g, 48 * H * D + 3, dtype=HF)
    o = ops.attention_packed(qkv, offsets(lens), H)
    (want,) = torch.autograd.grad(o, qkv, buf[3:].view(48, H * D).clone(), retain_graph=True)
    (got,) = torch.autograd.grad(o, qkv, buf[3:].view(48, H * D), retain_graph=True)
    assert torch.equal(got, want)
    (ones,) = torch.autograd.grad(o.sum(), qkv, retain_graph=True)
    assert torch.equal(ones, torch.autograd.grad(o, qkv, torch.ones_like(o))[0])


def test_attention_packed_other_stream_and_graph(cuda):
    g = gen(15)
    lens, H, G, D = [60, 5, 130], 4, 2, 64
    T = sum(lens) + 5
    qkv, do, cu = randn(g, T, (H + 2 * G) * D, dtype=BF), randn(g, T, H * D, dtype=BF), offsets(lens)

    def step(x):
        leaf = x.detach().requires_grad_()
        o = ops.attention_packed(leaf, cu, H, G)
        return o.detach(), torch.autograd.grad(o, leaf, do)[0]

    want = step(qkv)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step(qkv)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    static = qkv.clone()
    graph = torch.cuda.CUDAGraph()
    q, k, v = ops._split_heads(static, H, G)
    dqkv = torch.empty_like(static)
    with torch.cuda.graph(graph):
        o, lse = K.attn_packed_fwd(q, k, v, cu, D ** -0.5, want_lse=True)
        K.attn_packed_bwd(q, k, v, o, do.view(T, H, D), lse, cu, D ** -0.5, *ops._split_heads(dqkv, H, G))
    for i in range(4):
        x = randn(gen(100 + i), *qkv.shape, dtype=BF)
        static.copy_(x)
        if i == 2:                                                    # other lengths in the same buffers
            cu.copy_(offsets([5, 100, 80]))
        graph.replay()
        want = step(x)
        torch.cuda.synchronize()
        assert torch.equal(o.view(T, -1), want[0]) and torch.equal(dqkv, want[1])


# ---- embedding -----------------------------------------------------------------------------------------------------------------
def embed_check(V, W, ids, place, P, table_dt, out_dt, scale, seed, noncontig=False):
    g = gen(seed)
    table = randn(g, V, W, dtype=table_dt)
    pos = randn(g, P, W, dtype=table_dt) if P else None
    if noncontig:
        table = torch.cat([table, table], 1)[:, :W]
    n = ids.numel()
    dout = randn(g, *ids.shape, W, dtype=out_dt)
    t, p = table.detach().requires_grad_(), (pos.requires_grad_() if P else None)
    out = ops.embedding(ids, t, scale, pos=p, pos_ids=place, out_dtype=out_dt)
    assert out.dtype == out_dt
    pl = place if place is not None else torch.arange(n, device="cuda").view(ids.shape)
    flat, fp = ids.reshape(-1), pl.reshape(-1)
    ok = (flat >= 0) & (flat < V)
    a = torch.where(ok[:, None], table.detach().double()[flat.clamp(0, V - 1)] * scale, 0.0)
    b = torch.zeros_like(a)
    if P:
        okp = (fp >= 0) & (fp < P)
        b = torch.where(okp[:, None], pos.detach().double()[fp.clamp(0, P - 1)], 0.0)
    uo = half(out_dt) if out_dt != F32 else 0.0
    within(out.reshape(n, W), a + b, 2 * E * (a.abs() + b.abs()) + uo * (a + b).abs() * (1 + E) + 1e-30 + (6e-8 if out_dt == HF else 0), "out")
    grads = torch.autograd.grad(out, [t] + ([p] if P else []), dout)
    ut = half(table_dt) if table_dt != F32 else 0.0
    d2 = dout.reshape(n, W).double()
    for got, idx, rows, mul, m in [(grads[0], flat, V, scale, ok)] + ([(grads[1], fp, P, 1.0, (fp >= 0) & (fp < P))] if P else []):
        at = idx.clamp(0, rows - 1)
        want = torch.zeros(rows, W, dtype=F64, device="cuda").index_add_(0, at, d2 * m[:, None]) * mul
        mag = torch.zeros(rows, W, dtype=F64, device="cuda").index_add_(0, at, d2.abs() * m[:, None]) * abs(mul)
        cnt = torch.zeros(rows, dtype=F64, device="cuda").index_add_(0, at, m.double())
        within(got, want, E * (cnt[:, None] + 2) * mag + ut * want.abs() * (1 + E) + (6e-8 if table_dt == HF else 1e-38), "gradient")
        assert got.dtype == table_dt
    out2 = ops.embedding(ids, t, scale, pos=p, pos_ids=place, out_dtype=out_dt)
    for x, y in zip(grads, torch.autograd.grad(out2, [t] + ([p] if P else []), dout)):
        assert torch.equal(x, y)


EMBED = [  # tokens, vocab, width, places, table, out, scale
    (1, 10, 64, 0, F32, F32, 1.0),
    (5, 3, 100, 7, F32, F32, 2.0),
    (31, 1000, 64, 8, BF, BF, 8.0),
    (33, 1, 7, 1, HF, HF, 1.0),
    (700, 50, 512, 77, F32, HF, 1.0),
    (3000, 49408, 128, 77, F32, F32, 1.0),
    (8192, 300, 24, 40, BF, F32, 0.5),
    (8193, 300, 24, 40, F32, BF, 0.5),
    (20000, 70000, 16, 2000, F32, F32, 1.0),
    (50001, 257, 33, 0, HF, F32, 1.0),
]


@pytest.mark.parametrize("case", range(len(EMBED)))
def test_embedding_and_gradients(cuda, case):
    n, V, W, P, td, od, scale = EMBED[case]
    g = gen(40 + case)
    ids = torch.randint(-1, V + 1, (n,), generator=g, device="cuda")           # both ends fall outside the table
    ids[torch.rand(n, generator=g, device="cuda") < 0.3] = V // 2              # one hot token
    place = torch.randint(-1, P + 1, (n,), generator=g, device="cuda") if P else None
    embed_check(V, W, ids, place, P, td, od, scale, case)


@pytest.mark.parametrize("n, V, P, dim", [(1, 1, 1, 8), (700, 300, 77, 24), (5000, 90, 200, 8), (9000, 70000, 3, 16), (9000, 20, 9000, 40), (40000, 300, 66000, 8)])
@pytest.mark.parametrize("places", [False, True])
def test_embedding_both_gradients_at_once(cuda, n, V, P, dim, places):
    """Both tables' gradients in the same launches: the bits of each on its own (the tables sort in one to three passes, or by ranks)."""
    g = gen(n + dim)
    ids = torch.randint(-1, V + 1, (n,), generator=g, device="cuda")
    at = torch.randint(-2, P + 2, (n,), generator=g, device="cuda") if places else torch.arange(n, device="cuda")
    d = randn(g, n, dim, dtype=BF)
    dtable, dpos = K.embed_bwd(d, ids, V, 0.5, F32, P, at if places else None)
    assert torch.equal(dtable, K.embed_bwd(d, ids, V, 0.5, F32))
    ok = (at >= 0) & (at < P)
    want = torch.zeros(P, dim, dtype=F64, device="cuda").index_add_(0, at[ok], d[ok].double())
    size = torch.zeros(P, dim, dtype=F64, device="cuda").index_add_(0, at[ok], d[ok].double().abs())
    within(dpos, want, n * E * size, "dpos")
    assert torch.equal(dpos, K.embed_bwd(d, at, P, 1.0, F32))


def test_embedding_shapes_strides_and_default_places(cuda):
    g = gen(60)
    embed_check(40, 64, torch.randint(0, 40, (6, 9), generator=g, device="cuda"), None, 54, F32, F32, 1.0, 61)
    embed_check(40, 64, torch.randint(0, 40, (9,), generator=g, device="cuda"), None, 0, BF, F32, 1.0, 62, noncontig=True)
    embed_check(9, 64, torch.full((40000,), 4, device="cuda"), None, 0, F32, F32, 1.0, 63)          # every token the same
    embed_check(9, 64, torch.full((50,), -1, device="cuda"), None, 0, F32, F32, 1.0, 64)           # no token at all
    big = torch.full((3,), 2 ** 40, device="cuda")
    assert float(ops.embedding(big, torch.ones(4, 8, device="cuda")).abs().max()) == 0
    assert tuple(ops.embedding(torch.zeros(0, dtype=torch.long, device="cuda"), torch.ones(4, 8, device="cuda")).shape) == (0, 8)
    assert K.embed_bwd(torch.zeros(0, 8, device="cuda"), torch.zeros(0, dtype=torch.long, device="cuda"), 4).abs().sum() == 0


def test_embedding_gradient_of_nonfinite_rows_stays_in_its_row(cuda):
    ids = torch.tensor([0, 1, 2, 1], device="cuda")
    t = torch.zeros(4, 16, device="cuda", requires_grad=True)
    d = torch.ones(4, 16, device="cuda")
    d[1, 3], d[3, 4] = float("inf"), float("nan")
    (gt,) = torch.autograd.grad(ops.embedding(ids, t), t, d)
    assert bool((gt[[0, 2]] == 1).all()) and bool((gt[3] == 0).all())
    assert float(gt[1, 3]) == math.inf and math.isnan(float(gt[1, 4])) and float(gt[1, 0]) == 2


def test_embedding_graph_replays(cuda):
    for n in (300, 9000):
        ids = torch.zeros(n, dtype=torch.long, device="cuda")
        d = randn(gen(70), n, 64)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = K.embed_bwd(d, ids, 100)
        for i in range(4):
            x = torch.randint(0, 100, (n,), generator=gen(71 + i), device="cuda")
            ids.copy_(x)
            graph.replay()
            want = K.embed_bwd(d, x, 100)
            torch.cuda.synchronize()
            assert torch.equal(got, want)


# ---- 8-bit integer Linear ----------------------------------------------------------------------------------------------------------
def quant_reference(x):
    top = x.double().abs().amax(-1)
    s = (top / 127.0).float()
    q = torch.where(s[..., None] > 0, x.double() / s.double()[..., None], 0.0).round()       # (half to even)
    return q, s


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("K_", [16, 48, 512, 1008, 1024, 4096, 8208])
def test_int8_quant_is_exact(cuda, K_, dtype):
    g = gen(K_)
    x = randn(g, 37, K_, dtype=dtype)
    x[3] = 0
    x[5] *= 1e-4 if dtype == HF else 1e-30
    x[7] = x[7].sign() * (torch.arange(K_, device="cuda") % 128 + 0.5).to(dtype)             # every quotient next to a border
    x[7, 0] = 127.0
    q, s = K.int8_quant(x)
    qr, sr = quant_reference(x)
    assert torch.equal(s, sr)
    assert torch.equal(q.double(), qr)
    y = x.clone()
    y[2, 5], y[9, 1] = float("nan"), float("-inf")
    q, s = K.int8_quant(y)
    assert bool(torch.isnan(s[[2, 9]]).all()) and int(torch.isnan(s).sum()) == 2
    keep = [i for i in range(37) if i not in (2, 9)]
    assert torch.equal(q[keep].double(), qr[keep])


def linear_reference(x, wq, ws, bias, act, res, out_dt):
    q, s = quant_reference(x)
    z1 = (q @ wq.double().T) * (s.double()[..., None] * ws.double())
    z = z1 + (bias.double() if bias is not None else 0.0)
    ez = 4 * E * z1.abs() + E * z.abs()
    fast = out_dt != F32
    if act == K.ACT_GELU:
        y = z * torch.special.ndtr(z)
        cdf, pdf = torch.special.ndtr(z), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        dy = cdf + z * pdf
    elif act == K.ACT_QUICKGELU:
        sg = torch.sigmoid(1.702 * z)
        y, dy = z * sg, sg * (1 + 1.702 * z * (1 - sg))
    else:
        y, dy = z, torch.ones_like(z)
    # |act'| <= 1.13; the approximations: |erf error| <= 1.5e-7, exp / rcp a few units of fp32 with arguments up to |1.702 z| or z^2 / 2
    ea = 0.0 if act == K.ACT_NONE else (2e-7 * (1 + z.abs()) + (8 + 4 * z.abs()) * 2 * E * z.abs() if fast else (16 + 4 * z.abs()) * E * z.abs() + 4 * E)
    u = half(out_dt) if out_dt != F32 else E
    yr = y + (res.double() if res is not None else 0.0)
    b = (1.13 * ez + ea + E * yr.abs()) * (1 + u) + u * yr.abs() + (6e-8 if out_dt == HF else 1e-37)
    return yr, b, dy, ez


INT8 = [  # rows, N, K, act, residual dtype, output
    (1, 16, 16, 0, None, None), (1, 2048, 512, 2, None, None), (3, 17, 48, 1, F32, F32), (16, 100, 1024, 0, BF, None), (16, 4096, 4080, 2, F32, F32),
    (17, 128, 128, 0, None, None), (17, 33, 144, 1, None, F32), (130, 129, 272, 2, F32, F32), (257, 512, 512, 1, BF, None), (1000, 1000, 1008, 2, None, None),
    (5000, 2055, 400, 0, None, F32), (6200, 2304, 256, 1, None, None), (8000, 1600, 768, 2, F32, F32), (70, 72, 8208, 0, None, None),
    (8193, 2048, 80, 1, BF, None), (8256, 1930, 192, 0, F32, F32), (8257, 1928, 64, 2, None, None),
    (8392, 2600, 96, 2, None, F32), (600, 2055, 400, 1, F32, None), (300, 1000, 2064, 2, BF, None), (4000, 16, 208, 0, None, None),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("case", range(len(INT8)))
def test_linear_int8(cuda, case, dtype):
    M, N, Kd, act, rd, od = INT8[case]
    act = (K.ACT_NONE, K.ACT_GELU, K.ACT_QUICKGELU)[act]
    rd = dtype if rd == BF else rd
    g = gen(200 + case)
    x = randn(g, M, Kd, dtype=dtype)
    wq, ws = K.int8_quant(randn(g, N, Kd, mul=Kd ** -0.5))
    bias = randn(g, N) if case % 3 else None
    res = randn(g, M, N, dtype=rd) if rd is not None else None
    y, ag = K.linear_int8(x, wq, ws, bias, act, res, od, want_actgrad=True)
    want, bound, dy, ez = linear_reference(x, wq, ws, bias, act, res, od or dtype)
    assert y.dtype == (od or dtype) and ag.dtype == dtype
    within(y, want, bound, "y")
    within(ag, dy, half(dtype) * dy.abs() + ez + 1e-6 + 4e-6 * dy.abs(), "act'")
    assert torch.equal(K.linear_int8(x, wq, ws, bias, act, res, od), y)


def test_linear_int8_rows_are_independent(cuda):
    """One row at a time (the one-launch form) gives the same bits as the tiled product; strided and shifted inputs too."""
    g = gen(300)
    Kd, N = 512, 264
    x = randn(g, 40, Kd, dtype=HF)
    wq, ws = K.int8_quant(randn(g, N, Kd))
    y = K.linear_int8(x, wq, ws)
    for i in (0, 17, 39):
        assert torch.equal(K.linear_int8(x[i:i + 1], wq, ws), y[i:i + 1])
    wide = torch.zeros(40, Kd + 8, dtype=HF, device="cuda")
    wide[:, :Kd] = x
    assert torch.equal(K.linear_int8(wide[:, :Kd], wq, ws), y)
    odd = torch.zeros(40 * Kd + 3, dtype=HF, device="cuda")
    odd[3:] = x.reshape(-1)
    assert torch.equal(K.linear_int8(odd[3:].view(40, Kd), wq, ws), y)
    assert torch.equal(K.linear_int8(x[:1].expand(40, Kd), wq, ws), y[:1].expand(40, N))
    for t in (odd[3:].view(40, Kd), x[:1].expand(40, Kd), wide[:, :Kd], wide.view(-1)[5:5 + 39 * Kd].view(39, Kd)):
        for a, b in zip(K.int8_quant(t), K.int8_quant(t.clone(memory_format=torch.contiguous_format))):
            assert torch.equal(a, b)
    assert torch.equal(K.linear_int8(x.view(4, 10, Kd), wq, ws), y.view(4, 10, N))
    assert tuple(K.linear_int8(x[:0], wq, ws).shape) == (0, N)
    bad = x.clone()
    bad[5, 7] = float("nan")
    z = K.linear_int8(bad, wq, ws)
    assert bool(torch.isnan(z[5]).all()) and torch.equal(z[:5], y[:5]) and torch.equal(z[6:], y[6:])
    bad[3, 1] = float("inf")
    assert bool(torch.isnan(K.linear_int8(bad[3:4], wq, ws)).all())


def test_linear_int8_graph_replays(cuda):
    g = gen(310)
    wq, ws = K.int8_quant(randn(g, 96, 256))
    for M in (2, 60):
        x = randn(g, M, 256, dtype=BF)
        graph = torch.cuda.CUDAGraph()
        K.linear_int8(x, wq, ws)
        with torch.cuda.graph(graph):
            y = K.linear_int8(x, wq, ws, act=K.ACT_GELU)
        for i in range(3):
            x.copy_(randn(gen(311 + i), M, 256, dtype=BF))
            graph.replay()
            want = K.linear_int8(x, wq, ws, act=K.ACT_GELU)
            torch.cuda.synchronize()
            assert torch.equal(y, want)


# ---- together --------------------------------------------------------------------------------------------------------------------
def test_packed_operators_two_graphs_and_two_streams(cuda):
    """Embedding, 8-bit projection and attention with their gradients: two captured graphs replayed in turn, two streams at once; the workspaces
    belong to a call, so each gives its eager results."""
    g = gen(400)
    V, W, H = 600, 128, 2
    lens = [30, 1, 0, 200, 64]
    T, cu = sum(lens), offsets(lens)
    table, pos = randn(g, V, W), randn(g, T, W)
    wq, ws = K.int8_quant(randn(g, 3 * W, W, mul=W ** -0.5))
    scale = (W // H) ** -0.5

    def step(ids, do):
        x = K.embed_fwd(ids, table, 1.0, pos, None, BF)
        qkv = K.linear_int8(x, wq, ws)
        o, lse = K.attn_packed_qkv_fwd(qkv, cu, H, H, scale, want_lse=True)
        dqkv = K.attn_packed_qkv_bwd(qkv, o, do, lse, cu, H, H, scale)
        return (x, qkv, o, dqkv, *K.embed_bwd(dqkv[:, :W].contiguous(), ids, V, 1.0, F32, T))

    def inputs(seed):
        r = gen(seed)
        return torch.randint(0, V, (T,), generator=r, device="cuda"), randn(r, T, W, dtype=BF)

    ins = [inputs(401), inputs(402)]
    step(*ins[0])
    graphs, outs = [], []
    for a in ins:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(*a))
        graphs.append(graph)
    for i in range(3):
        for a, new in zip(ins, (inputs(410 + i), inputs(420 + i))):
            for t, n in zip(a, new):
                t.copy_(n)
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        want = [step(*a) for a in ins]
        torch.cuda.synchronize()
        for got, w in zip(outs, want):
            assert all(torch.equal(p, q) for p, q in zip(got, w))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    res = []
    for st, a in zip(streams, ins):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            res.append([step(*a) for _ in range(3)][-1])
    torch.cuda.synchronize()
    for got, w in zip(res, want):
        assert all(torch.equal(p, q) for p, q in zip(got, w))


def test_packed_operators_past_32_bit_offsets(cuda):
    """More than 2^31 elements per tensor: the last rows equal a call on them alone (zeros before them)."""
    g = gen(500)
    # attention: 1.1 million rows of 2048 columns, sequences of 64
    H, G, D, n, last = 16, 8, 64, 64, 640
    T = 1100032
    qkv = torch.zeros(T, (H + 2 * G) * D, dtype=BF, device="cuda")
    qkv[-last:] = randn(g, last, qkv.shape[1], dtype=BF)
    assert qkv.numel() > 1 << 31
    cu = torch.arange(0, T + 1, n, dtype=torch.int32, device="cuda")
    part = qkv[-last:].clone()
    o, lse = K.attn_packed_qkv_fwd(qkv, cu, H, G, 0.125, want_lse=True)
    o2, lse2 = K.attn_packed_qkv_fwd(part, cu[:last // n + 1].clone(), H, G, 0.125, want_lse=True)
    assert torch.equal(o[-last:], o2) and torch.equal(lse[:, -last:], lse2) and float(o[:T - last].abs().max()) == 0
    do = torch.zeros_like(o)
    do[-last:] = randn(g, last, H * D, dtype=BF)
    dqkv = K.attn_packed_qkv_bwd(qkv, o, do, lse, cu, H, G, 0.125)
    want = K.attn_packed_qkv_bwd(part, o2, do[-last:].clone(), lse2, cu[:last // n + 1].clone(), H, G, 0.125)
    assert torch.equal(dqkv[-last:], want) and float(dqkv[:T - last].abs().max()) == 0
    del o, do, dqkv
    # 8-bit Linear on the same rows: x, its panels and y
    wq, ws = K.int8_quant(randn(g, 2048, 2048, mul=0.02))
    y = K.linear_int8(qkv, wq, ws)
    assert torch.equal(y[-last:], K.linear_int8(part, wq, ws)) and float(y[:T - last].abs().max()) == 0
    del y
    # embedding: a table and a token buffer of that size
    ids = torch.full((T,), -1, device="cuda")
    ids[-last:] = torch.randint(T - last, T, (last,), generator=g, device="cuda")
    out = K.embed_fwd(ids, qkv)
    assert torch.equal(out[-last:], qkv[ids[-last:]]) and float(out[:T - last].abs().max()) == 0
    grad = K.embed_bwd(out, ids, T)
    small = K.embed_bwd(out[-last:].clone(), ids[-last:] - (T - last), last)
    assert torch.allclose(grad[-last:].double(), small.double(), rtol=2.0 ** -7, atol=last * E * float(out.abs().max()))
    assert float(grad[:T - last].abs().max()) == 0
