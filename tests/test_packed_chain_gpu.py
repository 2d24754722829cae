"""The whole packed text tower, step by step: every Linear, attention, LayerNorm and hand-over of the twelve blocks against 64 bits on its own inputs.

End to end an 8-bit tower is off by what 48 quantised products add up to (3 % of the features and more), and a bound of that size lets a wrong layer
pass.  Here each step is held to its own rounding, and what one hands to the next is compared as it is."""
import math

import pytest
import torch

from feed_forward_vqgan_clip_amd import clip as fclip
from feed_forward_vqgan_clip_amd import kernels as K
from feed_forward_vqgan_clip_amd import ops
from test_packed_gpu import E, attn_reference, half, linear_reference, quant_reference, within

pytestmark = pytest.mark.gpu
BF, HF, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64


def state_dict(seed):
    """ViT-B/32 with biases and norms that are not 0 and 1."""
    sd = fclip.random_state_dict(fclip.VIT_B32, seed)
    g = torch.Generator().manual_seed(seed + 1)
    for k in sd:
        if k.startswith(("transformer.", "ln_final")) and sd[k].dim() == 1:
            sd[k] = torch.randn(sd[k].shape, generator=g) * 0.1 + (1.0 if k.endswith("weight") else 0.0)
    return sd


def prompts(n, seed):
    g = torch.Generator().manual_seed(seed)
    t = torch.zeros(n, 77, dtype=torch.long)
    for i in range(n):
        m = int(torch.randint(1, 30, (1,), generator=g)) if i else 75
        t[i, 0] = 49406
        t[i, 1:1 + m] = torch.randint(1, 49405, (m,), generator=g)
        t[i, 1 + m] = 49407
    return t


def layer_norm(x, gamma, beta):
    """64 bits, and the bound of an fp32 evaluation: two sums over the row, then a handful of operations."""
    x = x.double()
    d = x - x.mean(-1, keepdim=True)
    h = d * (d.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    y = h * gamma.double() + beta.double()
    return y, E * ((2 * x.shape[-1] + 8) * (h.abs() + 1) * gamma.double().abs() + 2 * beta.double().abs())


def check_tower(sd, steps, ids, lens, feats, heads=8):
    """steps: the launches of one encode_text_packed in their order, inputs and outputs."""
    dev = {k: v.cuda() for k, v in sd.items() if not k.startswith("visual")}
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    place = torch.cat([torch.arange(n) for n in lens]).cuda()
    emb = dev["token_embedding.weight"].double()[ids] + dev["positional_embedding"].double()[place]
    it = iter(steps)

    def linear(p, x, act, residual, out_dt, bias):
        kind, rec = next(it, (None, None))
        assert kind == "linear", p
        wq, ws = quant_reference(dev[p])
        assert torch.equal(rec["wq"].double(), wq) and torch.equal(rec["ws"], ws), p
        assert rec["act"] == act and (rec["residual"] is None) == (residual is None), p
        if residual is not None:
            assert torch.equal(rec["residual"], residual), p
        if x is not None:
            assert torch.equal(rec["x"], x), p
        assert torch.equal(rec["bias"], dev[bias]), p
        want, bound, _, _ = linear_reference(rec["x"], wq, ws, dev[bias], act, residual, out_dt)
        within(rec["y"], want, bound, p)
        return rec["x"], rec["y"]

    def normed(got, stream, p):
        want, bound = layer_norm(stream, dev[p + ".weight"], dev[p + ".bias"])
        within(got, want, bound + half(HF) * (want.abs() + bound) + 2.0 ** -25, p)

    stream = None
    blocks = len({k.split(".")[2] for k in sd if k.startswith("transformer.resblocks.")})
    for b in range(blocks):
        p = f"transformer.resblocks.{b}."
        xn, qkv = linear(p + "attn.in_proj_weight", None, K.ACT_NONE, None, HF, p + "attn.in_proj_bias")
        kind, rec = next(it, (None, None))
        assert kind == "attn" and torch.equal(rec["qkv"], qkv) and rec["heads"] == (heads, heads), p
        q, k, v = ops._split_heads(qkv, heads, heads)
        o, bo = attn_reference(q, k, v, lens, (qkv.shape[1] // 3 // heads) ** -0.5)
        within(rec["out"].view_as(o), o, bo + 2.0 ** -25, p + "attention")
        if b == 0:                                          # the stream before the first block is seen as the residual of its first sum
            kind, first = steps[2]
            stream = first["residual"]
            within(stream, emb, 2 * E * (emb.abs() + 0.1), "embedding")
        normed(xn, stream, p + "ln_1")
        _, stream = linear(p + "attn.out_proj.weight", rec["out"], K.ACT_NONE, stream, F32, p + "attn.out_proj.bias")
        xn, h = linear(p + "mlp.c_fc.weight", None, K.ACT_QUICKGELU, None, HF, p + "mlp.c_fc.bias")
        normed(xn, stream, p + "ln_2")
        _, stream = linear(p + "mlp.c_proj.weight", h, K.ACT_NONE, stream, F32, p + "mlp.c_proj.bias")
    assert next(it, None) is None
    eot = stream[torch.tensor(cu[1:], device="cuda") - 1]
    xn, bx = layer_norm(eot, dev["ln_final.weight"], dev["ln_final.bias"])
    P = dev["text_projection"].double()
    within(feats, xn @ P, (bx + (P.shape[0] + 2) * E * xn.abs()) @ P.abs() * 2, "features")


def test_int8_text_tower_step_by_step(cuda, monkeypatch):
    sd = state_dict(11)
    model = fclip.CLIP(sd, HF, int8=True, text_packed=True)
    text = prompts(12, 12)
    ids, cu = fclip.pack_tokens(text)
    ids, cu = ids.cuda(), cu.cuda()
    lens = cu.diff().tolist()
    steps = []
    linear, attn = K.linear_int8, K.attn_packed_qkv_fwd

    def spy_linear(x, wq, ws, bias=None, act=K.ACT_NONE, residual=None, out_dtype=None, want_actgrad=False):
        assert not want_actgrad
        y = linear(x, wq, ws, bias, act, residual, out_dtype)
        steps.append(("linear", dict(x=x.clone(), wq=wq, ws=ws, bias=bias, act=act, residual=None if residual is None else residual.clone(), y=y.clone())))
        return y

    def spy_attn(qkv, cu_, heads, kv_heads, scale, want_lse=False):
        o, lse = attn(qkv, cu_, heads, kv_heads, scale, want_lse)
        steps.append(("attn", dict(qkv=qkv.clone(), heads=(heads, kv_heads), out=o.clone())))
        return o, lse

    monkeypatch.setattr(K, "linear_int8", spy_linear)
    monkeypatch.setattr(K, "attn_packed_qkv_fwd", spy_attn)
    with torch.no_grad():
        feats = model.encode_text_packed(ids, cu)
    check_tower(sd, steps, ids, lens, feats)

    # the check notices a tower that differs from the checkpoint: mistakes planted in what it compares with
    def wrong(**changes):
        with pytest.raises(AssertionError):
            check_tower({**sd, **changes}, steps, ids, lens, feats)

    last, name = "transformer.resblocks.11.", "transformer.resblocks.4.attn.out_proj.weight"
    wrong(positional_embedding=torch.zeros_like(sd["positional_embedding"]))
    wrong(**{last + "attn.out_proj.weight": torch.zeros(512, 512), last + "mlp.c_proj.weight": torch.zeros(512, 2048)})
    wrong(**{name: sd["transformer.resblocks.5.attn.out_proj.weight"]})
    wrong(**{last + "ln_2.bias": torch.zeros(512)})
    wrong(**{"ln_final.bias": torch.zeros(512)})
    with pytest.raises(AssertionError):
        check_tower(sd, steps[:-5], ids, lens, feats)
    # and the padded tower, for the size of the whole: 48 quantised products whose errors of about 1.2 % each are independent
    want = model._encode_text_padded(text)
    err = float((feats - want).norm() / want.norm())
    assert err < 0.012 * math.sqrt(48), err


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("act", [K.ACT_GELU, K.ACT_QUICKGELU])
def test_8_bit_layers_pass_gradients_straight_through(cuda, dtype, act):
    """dx = dy W of the 16-bit weight for ops.linear; with act'(pre) of the 8-bit forward between two of them for ops.mlp."""
    g = torch.Generator(device="cuda").manual_seed(21)
    rn = lambda *s, dt=F32, mul=1.0: (torch.randn(*s, generator=g, device="cuda") * mul).to(dt)  # noqa: E731
    M, D, Hd = 77, 128, 512
    w1, w2, b1, b2 = rn(Hd, D, mul=D ** -0.5), rn(D, Hd, mul=Hd ** -0.5), rn(Hd), rn(D)
    W1, W2 = ops.Weights.frozen(w1, b1, dtype, int8=True), ops.Weights.frozen(w2, b2, dtype, int8=True)
    x, dy = rn(M, D, dt=dtype), rn(M, D, dt=dtype)
    u = half(dtype)
    a1, a2 = w1.to(dtype).double(), w2.to(dtype).double()
    dh = rn(M, Hd, dt=dtype)
    leaf = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(ops.linear(leaf, W1), leaf, dh)
    want = dh.double() @ a1
    within(dx, want, u * want.abs() * (1 + u) + 2 * Hd * E * (dh.double().abs() @ a1.abs()), "linear dx")
    leaf, res = x.clone().requires_grad_(), rn(M, D).requires_grad_()
    y = ops.mlp(leaf, W1, W2, act, residual=res, out_dtype=F32)
    dx, dr = torch.autograd.grad(y, (leaf, res), dy.float())
    assert torch.equal(dr, dy.float())
    _, ag = K.linear_int8(x, *W1.int8, bias=b1, act=act, want_actgrad=True)
    t = dy.double() @ a2
    hid = t * ag.double()
    eh = ag.double().abs() * (2 * D * E) * (dy.double().abs() @ a2.abs()) + u * hid.abs() * (1 + u)        # the hidden gradient is stored in 16 bits
    want = hid @ a1
    within(dx, want, (eh @ a1.abs()) * (1 + u) + u * want.abs() * (1 + u) + 2 * Hd * E * (hid.abs() @ a1.abs()), "mlp dx")


@pytest.mark.parametrize("int8", [False, True])
def test_packed_tower_captured_and_replayed(cuda, int8):
    """A fixed buffer of ids and offsets: one capture serves batches of other lengths, also with empty prompts and rows before the first one."""
    cfg = dict(embed_dim=64, image_resolution=32, vision_layers=1, vision_width=128, vision_patch_size=8, context_length=77, vocab_size=500,
               transformer_width=128, transformer_heads=2, transformer_layers=2)
    model = fclip.CLIP(fclip.random_state_dict(cfg, 3), HF, int8=int8, text_packed=True)
    rows, B = 200, 6
    g = torch.Generator(device="cuda").manual_seed(31)
    ids, cu = torch.zeros(rows, dtype=torch.long, device="cuda"), torch.zeros(B + 1, dtype=torch.int32, device="cuda")
    batches = [[0, 10, 30, 31, 90, 150, 200], [0, 0, 77, 77, 100, 101, 140], [17, 40, 50, 90, 91, 92, 199], [0, 33, 66, 99, 132, 165, 198]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad(), torch.cuda.stream(side):
        for _ in range(2):
            model.encode_text_packed(ids, cu)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        got = model.encode_text_packed(ids, cu)
    for r in range(2):
        for c in batches:
            new = torch.randint(0, 500, (rows,), generator=g, device="cuda")
            off = torch.tensor(c, dtype=torch.int32, device="cuda")
            ids.copy_(new)
            cu.copy_(off)
            graph.replay()
            with torch.no_grad():
                want = model.encode_text_packed(new, off)
            torch.cuda.synchronize()
            assert torch.allclose(got, want, rtol=1e-5, atol=1e-6), (r, c)
            assert bool(torch.isfinite(got).all())
