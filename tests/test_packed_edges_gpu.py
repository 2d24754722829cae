"""Packed-prompt operators at their edges: values, offsets, widths and gradients that the ordinary cases do not reach."""
import math

import pytest
import torch

from feed_forward_vqgan_clip_amd import clip as fclip
from feed_forward_vqgan_clip_amd import kernels as K
from feed_forward_vqgan_clip_amd import ops
from test_packed_gpu import attn_reference, half, within

pytestmark = pytest.mark.gpu
BF, HF, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32, mul=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * mul).to(dtype)


def offsets(lens, first=0):
    return torch.tensor([first] + list(torch.tensor(lens, dtype=torch.long).cumsum(0) + first), dtype=torch.int32, device="cuda")


def attend(qkv, cu, H, G, do):
    """out, dq, dk, dv of the public operator, by heads."""
    leaf = qkv.detach().clone().requires_grad_()
    o = ops.attention_packed(leaf, cu, H, G)
    (d,) = torch.autograd.grad(o, leaf, do)
    return (o.detach().unflatten(1, (H, -1)),) + ops._split_heads(d, H, G)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("lens,H,G,D", [([64], 2, 1, 64), ([128], 2, 2, 128), ([70], 2, 1, 64), ([33], 1, 1, 40), ([200, 45], 4, 2, 128), ([20, 9, 31], 2, 2, 64),
                                        ([700], 2, 2, 64), ([1500], 96, 96, 64)])
def test_a_key_that_every_query_rejects(cuda, lens, H, G, D, dtype):
    """A key of -inf against queries that are positive there has weight 0: its gradients are zeros and nothing else notices it.  The same bits as
    with the lowest finite score in its place (whose weight 2^-1000 is 0 as well), whatever the length is a multiple of."""
    g = gen(len(lens) * 1000 + lens[0] + D)
    T = sum(lens)
    qkv, do, cu = randn(g, T, (H + 2 * G) * D, dtype=dtype), randn(g, T, H * D, dtype=dtype), offsets(lens)
    q, k, _ = ops._split_heads(qkv, H, G)
    q[:, :, 3] = q[:, :, 3].abs() + 0.5
    start = 0
    for n in lens:
        for t in {start + 1, start + n // 2, start + n - 1}:
            res = []
            for value in (-float("inf"), -3e4 if dtype == HF else -1e30):
                keep = k[t].clone()
                k[t, :, 3] = value
                res.append(attend(qkv, cu, H, G, do))
                k[t] = keep
            (o, dq, dk, dv), (o2, dq2, dk2, dv2) = res
            assert torch.equal(o, o2), (n, t)
            assert float(dk[t].abs().max()) == 0 and float(dv[t].abs().max()) == 0, (n, t)
            assert torch.equal(dk, dk2) and torch.equal(dv, dv2), (n, t)
            # dq of the sequence itself: 0 * -inf for the queries that see the key, and those beside it are summed again, in another order
            rest = [r for r in range(T) if r < start or r >= start + n]
            assert torch.equal(dq[rest], dq2[rest]), (n, t)
        start += n


def refill(like, value):
    """Leave `value` in memory of this size, so that whatever a call does not write is likely to show it."""
    t = torch.full_like(like, value)
    torch.cuda.synchronize()
    del t


@pytest.mark.parametrize("first", [1, 5, 31, 32, 200, 700])
@pytest.mark.parametrize("lens,H,G,D", [([5, 9, 30], 2, 2, 64), ([0, 7, 0], 2, 1, 64), ([300], 8, 2, 128), ([130, 90], 4, 4, 64), ([20] * 70, 2, 2, 64), ([900, 400], 48, 48, 64)])
def test_offsets_that_begin_behind_row_0(cuda, lens, H, G, D, first):
    """A slice of a batch's offsets: the sequences' rows as if they stood alone, zeros before the first and behind the last."""
    n, spare = sum(lens), first % 3
    T = first + n + spare
    g = gen(first * 100 + n)
    qkv, do = randn(g, T, (H + 2 * G) * D, dtype=BF), randn(g, T, H * D, dtype=BF)
    alone = attend(qkv[first:first + n].contiguous(), offsets(lens), H, G, do[first:first + n].contiguous())
    refill(qkv, 3.0)
    refill(do, 3.0)
    got = attend(qkv, offsets(lens, first), H, G, do)
    for name, a, b in zip(("out", "dq", "dk", "dv"), got, alone):
        assert not bool(a[:first].any()) and not bool(a[first + n:].any()), name
        # (more rows may choose another split of the backward's sums: equal up to their rounding)
        assert torch.equal(a[first:first + n], b) if name == "out" else torch.allclose(a[first:first + n].double(), b.double(), rtol=2.0 ** -7, atol=1e-2), name
    # buffers that are given: forward leaves those rows alone, backward zeroes them; nothing beside the views is written
    q, k, v = ops._split_heads(qkv, H, G)
    buf = torch.full((T + 2, H * D + 8), 5.0, dtype=BF, device="cuda")
    out, lse = K.attn_packed_fwd(q, k, v, offsets(lens, first), D ** -0.5, out=buf[1:-1, :H * D].unflatten(1, (H, D)), want_lse=True)
    assert torch.equal(out[first:first + n], got[0][first:first + n])
    keep = buf.clone()
    keep[1 + first:1 + first + n, :H * D] = 5.0
    assert bool((keep == 5.0).all())
    grad = torch.full((T + 2, (H + 2 * G) * D + 8), 5.0, dtype=BF, device="cuda")
    views = ops._split_heads(grad[1:-1, :-8], H, G)
    K.attn_packed_bwd(q, k, v, got[0].contiguous(), do.unflatten(1, (H, D)), lse, offsets(lens, first), D ** -0.5, *views)
    assert all(torch.equal(a, b) for a, b in zip(views, got[1:]))
    grad[1:-1, :-8] = 5.0
    assert bool((grad == 5.0).all())


TOWER = dict(embed_dim=64, image_resolution=32, vision_layers=1, vision_width=128, vision_patch_size=8, context_length=77, vocab_size=500,
             transformer_width=128, transformer_heads=2, transformer_layers=2)


def test_packed_text_tower_on_a_slice_of_the_offsets(cuda):
    """Prompts 2 .. of a batch through the whole batch's rows: their features, and no gradient for the tokens of the prompts before them."""
    model = fclip.CLIP(fclip.random_state_dict(TOWER, 3), HF, text_packed=True)
    g = torch.Generator().manual_seed(2)
    text = torch.zeros(6, 77, dtype=torch.long)
    for i in range(6):
        text[i, :9 + i] = torch.arange(60 * i, 60 * i + 9 + i) + 1
        text[i, 9 + i] = 499
    w = torch.randn(6, 64, generator=g).cuda()
    ids, cu = fclip.pack_tokens(text)
    ids, cu = ids.cuda(), cu.cuda()
    table = model.tok_emb.clone().requires_grad_()
    full = model.encode_text_packed(ids, cu, table)
    (gf,) = torch.autograd.grad((full[2:] * w[2:]).sum(), table)
    part = model.encode_text_packed(ids, cu[2:].clone(), table)
    (gp,) = torch.autograd.grad((part * w[2:]).sum(), table)
    # the same rows through the same products (the forward does not depend on company); sums of the backward may be cut differently
    assert torch.allclose(part, full[2:], rtol=1e-5, atol=1e-6)
    before = ids[:int(cu[2])].unique()
    before = before[before != 499]
    assert not bool(gp[before].any()) and bool(torch.isfinite(gp).all())
    assert float((gp - gf).norm() / gf.norm()) < 20 * torch.finfo(HF).eps / 2


# every form of the backward: one-wave tiles; dq in halves and dk / dv in four parts; dq whole and dk / dv in two; both whole
FORMS = [([64], 2, 2), ([30, 9, 64, 17], 4, 2), ([70, 200], 4, 2), ([900], 96, 96), ([1500], 96, 96)]


def hold_gradients(lens, H, G, D, scale, do_size, seed, size=1.0):
    """f16 gradients of a call with output gradients of this size, against the 64-bit formulas and their bounds (which know one rounding of dS to 11
    bits and one of the result, and nothing of overflow or lost bits below it)."""
    g = gen(seed)
    T = sum(lens)
    qkv, do = randn(g, T, (H + 2 * G) * D, dtype=HF, mul=size), randn(g, T, H * D, dtype=HF, mul=do_size).clamp(-6e4, 6e4)
    q, k, v = ops._split_heads(qkv, H, G)
    (o, dq, dk, dv), (bo, bq, bk, bv) = attn_reference(q, k, v, lens, scale, do.view(T, H, D))
    leaf = qkv.clone().requires_grad_()
    got = ops.attention_packed(leaf, offsets(lens), H, G, scale=scale)
    within(got.view(T, H, D), o, bo, "out")
    (d,) = torch.autograd.grad(got, leaf, do)
    for name, a, b, c in zip(("dq", "dk", "dv"), ops._split_heads(d, H, G), (dq, dk, dv), (bq, bk, bv)):
        fits = b.abs() < 65000                                       # (the few others, sums over a group's heads, round to an infinity)
        within(a[fits], b[fits], c[fits], name)
        assert float(fits.double().mean()) > 0.999


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_f16_gradients_of_a_scaled_loss(cuda, form, D):
    """p (dP - delta) passes 65504 although ds = scale p (dP - delta) and all three gradients fit."""
    lens, H, G = FORMS[form]
    hold_gradients(lens, H, G, D, 1.0 / 128, 12000.0, 70 + form)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_f16_gradients_that_grow_along_the_walk(cuda, form, D):
    """Output gradients of 1e-3 for most queries and of thousands for a few: the factor is lowered in the middle of a walk, for some rows and not for others."""
    lens, H, G = FORMS[form]
    g = gen(170 + form)
    T, scale = sum(lens), D ** -0.5
    qkv, do = randn(g, T, (H + 2 * G) * D, dtype=HF), randn(g, T, H * D, dtype=HF, mul=1e-3)
    do[T // 2::7] *= 4e6
    v = ops._split_heads(qkv, H, G)[2]
    v[T // 3::5] *= 8
    q, k, v = ops._split_heads(qkv, H, G)
    (o, dq, dk, dv), (bo, bq, bk, bv) = attn_reference(q, k, v, lens, scale, do.view(T, H, D))
    leaf = qkv.clone().requires_grad_()
    (d,) = torch.autograd.grad(ops.attention_packed(leaf, offsets(lens), H, G), leaf, do)
    for name, a, b, c in zip(("dq", "dk", "dv"), ops._split_heads(d, H, G), (dq, dk, dv), (bq, bk, bv)):
        fits = b.abs() < 65000                                       # (the others round to an infinity)
        within(a[fits], b[fits], c[fits], name)
        assert float(fits.double().mean()) > 0.9


@pytest.mark.parametrize("D", [64, 128])
def test_f16_gradients_of_a_mean_over_many_keys(cuda, D):
    """Output gradients of 1e-4 over 2000 keys: dS of a few 1e-8, sums of a few 1e-6 that f16 holds to its subnormal step."""
    hold_gradients([2000, 40], 2, 2, D, D ** -0.5, 1e-4, 270, size=0.3)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens", [[3000], [3000] + [2] * 60])
def test_many_small_weights_beside_a_large_one(cuda, lens, D, dtype):
    """3000 keys of weight 2^-26 behind one of weight 1: their sum is the output wherever the large key's value is 0."""
    g = gen(370 + D)
    T, scale = sum(lens), D ** -0.5
    q, k = torch.zeros(T, 2, D, dtype=dtype, device="cuda"), torch.zeros(T, 2, D, dtype=dtype, device="cuda")
    q[:, :, 5] = 8.0
    k[0, :, 5] = 18.0 / (8.0 * scale)
    v = randn(g, T, 2, D).abs().add(0.5).to(dtype)
    v[0] = 0
    o, lse = K.attn_packed_fwd(q, k, v, offsets(lens), scale, want_lse=True)
    ref, bound = attn_reference(q, k, v, lens, scale)
    assert float(ref[2000:3000].min()) > 1e-5
    within(o, ref, bound + (2.0 ** -25 if dtype == HF else 0.0), "out")          # (half a step of a subnormal output)
    s = (q[2999].double() * k[:3000].double()).sum(-1) * scale
    assert float((lse[:, 2999].double() - torch.logsumexp(s, 0) / math.log(2)).abs().max()) < 2e-5   # (26 in fp32, l to n 2^-24)


@pytest.mark.parametrize("int8", [False, True])
def test_frozen_mlp_with_a_residual_that_alone_wants_a_gradient(cuda, int8):
    g = gen(470)
    W1, W2 = (ops.Weights.frozen(randn(g, n, k, mul=k ** -0.5), randn(g, n), HF, int8=int8) for n, k in ((256, 64), (64, 256)))
    x, res, dy = randn(g, 40, 64, dtype=HF), randn(g, 40, 64).requires_grad_(), randn(g, 40, 64)
    y = ops.mlp(x, W1, W2, K.ACT_GELU, residual=res, out_dtype=F32)
    (gr,) = torch.autograd.grad(y, res, dy)
    assert torch.equal(gr, dy)
    x2 = x.clone().requires_grad_()
    y2 = ops.mlp(x2, W1, W2, K.ACT_GELU, residual=res, out_dtype=F32)
    gx, gr = torch.autograd.grad(y2, (x2, res), dy)
    assert torch.equal(y2, y) and torch.equal(gr, dy) and bool(gx.any()) and bool(torch.isfinite(gx).all())


def test_a_single_row_of_a_wider_buffer(cuda):
    """One token: the row stride of its tensors is never taken, so an odd one is no reason to refuse the call."""
    g = gen(570)
    H, D = 2, 64
    wide = randn(g, 1, 3 * H * D + 5, dtype=HF)
    qkv, cu = wide[:, :3 * H * D], offsets([1])
    assert qkv.stride(0) % 8
    do = randn(g, 1, H * D, dtype=HF)
    want = attend(qkv.contiguous(), cu, H, H, do)
    leaf = wide.clone().requires_grad_()
    o = ops.attention_packed(leaf[:, :3 * H * D], cu, H)
    (d,) = torch.autograd.grad(o, leaf, do)
    for a, b in zip((o.unflatten(1, (H, D)),) + ops._split_heads(d[:, :3 * H * D], H, H), want):
        assert torch.equal(a, b)
    assert torch.equal(K.attn_packed_qkv_fwd(qkv, cu, H, H, D ** -0.5)[0], o.detach())
    q, k, v = ops._split_heads(qkv, H, H)
    out = torch.zeros(1, H * D + 3, dtype=HF, device="cuda")[:, :H * D].unflatten(1, (H, D))
    K.attn_packed_fwd(q, k, v, cu, D ** -0.5, out=out)
    assert torch.equal(out, want[0])
    # heads apart by more than their width as well: the single row's heads need no room of a row
    buf = randn(g, 1, 3 * H, 2 * D, dtype=HF)
    qq, kk, vv = (buf[:, i * H:(i + 1) * H, :D] for i in range(3))
    o2, _ = K.attn_packed_fwd(qq, kk, vv, cu, D ** -0.5)
    assert torch.equal(o2, K.attn_packed_fwd(qq.contiguous(), kk.contiguous(), vv.contiguous(), cu, D ** -0.5)[0])
    # the other operators take such rows as well
    x = randn(g, 1, 67, dtype=HF)[:, :64]
    wq, ws = K.int8_quant(randn(g, 24, 64))
    assert torch.equal(K.linear_int8(x, wq, ws), K.linear_int8(x.contiguous(), wq, ws))
    assert torch.equal(K.int8_quant(x)[0], K.int8_quant(x.contiguous())[0])
    table = randn(g, 1, 67)[:, :64]
    ids = torch.tensor([0, 0, 1], device="cuda")
    assert torch.equal(K.embed_fwd(ids, table), K.embed_fwd(ids, table.contiguous()))
    assert torch.equal(K.embed_bwd(x, ids[:1], 3), K.embed_bwd(x.contiguous(), ids[:1], 3))


def test_outputs_on_top_of_inputs_are_refused(cuda):
    g = gen(670)
    T, H, D, cu = 40, 2, 64, offsets([40])
    q, k, v, do = (randn(g, T, H, D, dtype=HF) for _ in range(4))
    for t in (q, k, v):
        with pytest.raises(ValueError):
            K.attn_packed_fwd(q, k, v, cu, 0.125, out=t)
    o, lse = K.attn_packed_fwd(q, k, v, cu, 0.125, want_lse=True)
    new = lambda: torch.empty_like(q)  # noqa: E731
    one = new()
    for dq, dk, dv in ((q, new(), new()), (new(), k, new()), (new(), new(), v), (do, new(), new()), (new(), o, new()), (one, one, new()), (one, new(), one), (new(), one, one)):
        with pytest.raises(ValueError):
            K.attn_packed_bwd(q, k, v, o, do, lse, cu, 0.125, dq, dk, dv)
    grads = [new() for _ in range(3)]
    K.attn_packed_bwd(q, k, v, o, do, lse, cu, 0.125, *grads)
    assert all(bool(t.any()) for t in grads)
    both = torch.empty(T, 2 * H, D, dtype=HF, device="cuda")             # interleaved rows of one buffer are no overlap
    K.attn_packed_bwd(q, k, v, o, do, lse, cu, 0.125, new(), both[:, :H], both[:, H:])
    assert torch.equal(both[:, :H], grads[1]) and torch.equal(both[:, H:], grads[2])


@pytest.mark.parametrize("int8", [False, True])
def test_packed_text_tower_without_a_token(cuda, int8):
    """Prompts that are all empty: each the features of an empty prompt beside others, and a gradient of zeros."""
    model = fclip.CLIP(fclip.random_state_dict(TOWER, 3), HF, int8=int8, text_packed=True)
    ids = torch.tensor([498, 5, 6, 499], device="cuda")
    mixed = model.encode_text_packed(ids, torch.tensor([0, 4, 4], dtype=torch.int32, device="cuda"))
    table = model.tok_emb.clone().requires_grad_()
    got = model.encode_text_packed(ids[:0], torch.zeros(4, dtype=torch.int32, device="cuda"), table)
    assert got.shape == (3, 64) and torch.allclose(got, mixed[1].expand(3, 64), rtol=1e-5, atol=1e-6)
    (gt,) = torch.autograd.grad(got.sum(), table)
    assert gt.shape == table.shape and not bool(gt.any())


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("H,G,D", [(2, 2, 64), (4, 2, 128), (96, 96, 64)])
def test_offsets_of_any_kind_write_nothing_outside(cuda, H, G, D, many):
    """Offsets that descend or leave the tensor, forward and backward, into views between guard rows and guard columns."""
    g = gen(770 + D)
    T = 700
    qkv, do = randn(g, T, (H + 2 * G) * D, dtype=BF), randn(g, T, H, D, dtype=BF)
    q, k, v = ops._split_heads(qkv, H, G)
    cases = [[0, 5000], [-7, 30, 690], [0, 650, 20, 700], [700, 0], [-2 ** 31, 2 ** 31 - 1], [100, 100, 100], [900, 800, -1, 350], [0, 700, 0, 700, 0, 700]]
    for cu in cases:
        if many:                                               # more sequences than lanes: the search in place of the order by length
            cu = cu + [cu[-1]] * 70
        cu = torch.tensor(cu, dtype=torch.int32, device="cuda")
        out = torch.full((T + 128, H * D + 64), 7.0, dtype=BF, device="cuda")
        grad = torch.full((T + 128, (H + 2 * G) * D + 64), 7.0, dtype=BF, device="cuda")
        o, lse = K.attn_packed_fwd(q, k, v, cu, D ** -0.5, out=out[64:64 + T, :H * D].unflatten(1, (H, D)), want_lse=True)
        K.attn_packed_bwd(q, k, v, o, do, lse, cu, D ** -0.5, *ops._split_heads(grad[64:64 + T, :-64], H, G))
        torch.cuda.synchronize()
        for buf in (out, grad):
            buf[64:64 + T, :-64] = 7.0
            assert bool((buf == 7.0).all()), cu[:6]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens", [[300], [300] + [2] * 20])
def test_scores_far_beyond_the_exponents(cuda, lens, D, dtype):
    """Scores of 10^6 to 4 10^9 (exponents whose last place is up to 512), every key far above those before it: a query's output is its own value
    row, to the rounding of its one weight and of the result."""
    T = sum(lens)
    for top in (64.0, 1024.0, 49152.0):
        q, k = torch.zeros(T, 2, D, dtype=dtype, device="cuda"), torch.zeros(T, 2, D, dtype=dtype, device="cuda")
        q[:, :, 5] = 49152.0
        k[:, :, 5] = (torch.arange(T, device="cuda", dtype=F32)[:, None] + 1) * (top / 512)
        k[:, 0, 5] = k[:, 0, 5].flip(0).neg()                          # negative scores in one head: the order stays
        v = randn(gen(870), T, 2, D, dtype=dtype)
        o, lse = K.attn_packed_fwd(q, k, v, offsets(lens), 1.0, want_lse=True)
        assert bool(torch.isfinite(o).all()) and bool(torch.isfinite(lse).all())
        if dtype == HF or T <= 256:                                      # (bf16 does not hold so many different keys: equal ones share the weight)
            assert float(k[:, :, 5].double().diff(dim=0).min()) > 0
            want = v.double()
            within(o, want, (2 * half(dtype) + 4 * 2.0 ** -24) * want.abs() * (1 + half(dtype)) + 2.0 ** -25, "out")
        dq, dk, dv = (torch.empty_like(q) for _ in range(3))
        K.attn_packed_bwd(q, k, v, o, randn(gen(871), T, 2, D, dtype=dtype), lse, offsets(lens), 1.0, dq, dk, dv)
        if top == 64.0:                                                  # exponents of 8 10^6: their rounding is below one
            assert all(bool(torch.isfinite(t).all()) for t in (dq, dk, dv))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
def test_scores_far_beyond_the_exponents_beside_a_nan(cuda, D, dtype):
    """The rows that are summed again without a later NaN keep their one weight as well."""
    T = 200
    q, k = torch.zeros(T, 1, D, dtype=dtype, device="cuda"), torch.zeros(T, 1, D, dtype=dtype, device="cuda")
    q[:] = 49152.0                                                       # every feature: scores of 4 10^10
    k[:] = (torch.arange(T, device="cuda", dtype=F32)[:, None, None] + 1) * 64
    v = randn(gen(970), T, 1, D, dtype=dtype)
    for t in (150, T - 1):
        x = v.clone()
        x[t] = float("nan")
        o, _ = K.attn_packed_fwd(q, k, x, offsets([T]), 1.0)
        want = v[:t].double()
        within(o[:t], want, (2 * half(dtype) + 4 * 2.0 ** -24) * want.abs() * (1 + half(dtype)) + 2.0 ** -25, "out")
        assert bool(torch.isnan(o[t]).all())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("scale", [1e-44, 1e-38, 3e-30, 1e-6, 40.0])
@pytest.mark.parametrize("lens,H,G,D", [([70, 3], 2, 1, 64), ([20, 9], 2, 2, 128), ([300], 2, 2, 64)])
def test_scales_of_any_size(cuda, lens, H, G, D, scale, dtype):
    """From scales at which every weight is the same (their smallest is subnormal) to one at which a few keys take all of it."""
    g = gen(1070 + D)
    T = sum(lens)
    qkv, do = randn(g, T, (H + 2 * G) * D, dtype=dtype), randn(g, T, H * D, dtype=dtype)
    q, k, v = ops._split_heads(qkv, H, G)
    (o, dq, dk, dv), bounds = attn_reference(q, k, v, lens, scale, do.view(T, H, D))
    leaf = qkv.clone().requires_grad_()
    got = ops.attention_packed(leaf, offsets(lens), H, G, scale=scale)
    (d,) = torch.autograd.grad(got, leaf, do)
    # fp32 weights end at 2^-126 = 1.2e-38: up to 300 of them, times scale |dp - delta| |q| < 40 * 200 * 6, are less than 1e-30
    small = 2.0 ** -25 if dtype == HF else 1e-30
    for name, a, b, c in zip(("out", "dq", "dk", "dv"), (got.view(T, H, D),) + ops._split_heads(d, H, G), (o, dq, dk, dv), bounds):
        within(a, b, c + small, name)
