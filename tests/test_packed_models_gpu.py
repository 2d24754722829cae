"""The packed text tower (CLIP.encode_text_packed: embedding, packed attention, 16-bit or 8-bit Linear layers) against the padded CPU oracle."""
import pytest
import torch

from feed_forward_vqgan_clip_amd import clip as fclip
from feed_forward_vqgan_clip_amd import main as fmain
from oracle import clip as oclip

pytestmark = pytest.mark.gpu
CFG = dict(embed_dim=64, image_resolution=32, vision_layers=2, vision_width=128, vision_patch_size=8, context_length=77, vocab_size=500,
           transformer_width=128, transformer_heads=2, transformer_layers=2)
# Each block rounds about ten tensors to the compute dtype (LayerNorm outputs, qkv, probabilities, attention output, hidden activation, weights of four
# products), the residual stream stays fp32.  The roundings are independent; 20 of them of at most u = eps / 2 each, taken at their worst and
# all in one direction, are 20 u of a tensor of the size of the stream, and LayerNorm at the end divides by a stream of that size.
BLOCKS = 2


def tol16(dt):
    return 10 * BLOCKS * torch.finfo(dt).eps / 2


# 8-bit rows: a step is amax / 127, its rounding error amax / 254 at most and amax / 440 rms; amax is about 3.5 times the rms of a row of 128 normal
# values, so a rounded row is off by 0.8 % rms, a product of two such rows by 1.2 %, and there are four products per block.
TOL8 = 4 * BLOCKS * 0.012


def prompts(n, seed):
    g = torch.Generator().manual_seed(seed)
    t = torch.zeros(n, 77, dtype=torch.long)
    for i in range(n):
        m = int(torch.randint(1, 75, (1,), generator=g)) if i else 75
        t[i, 0] = 498
        t[i, 1:1 + m] = torch.randint(1, 498, (m,), generator=g)
        t[i, 1 + m] = 499
    return t


def rel(a, b):
    return float((a.detach().double().cpu() - b.detach().double()).norm() / b.detach().double().norm())


@pytest.mark.parametrize("cdt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("int8", [False, True])
def test_packed_text_tower_features_and_table_gradient(cuda, cdt, int8):
    sd = fclip.random_state_dict(CFG, 3)
    text = prompts(9, 4)
    model = fclip.CLIP(sd, cdt, int8=int8, text_packed=True)
    want_table = sd["token_embedding.weight"].clone().requires_grad_()
    want = oclip.encode_text({**sd, "token_embedding.weight": want_table}, text)
    w = torch.randn(want.shape, generator=torch.Generator().manual_seed(5))
    (gt,) = torch.autograd.grad((want * w).sum(), want_table)
    tol = TOL8 if int8 else tol16(cdt)
    assert rel(model.encode_text(text), want) < tol                            # packs on the host
    ids, cu = fclip.pack_tokens(text)
    assert int(cu[-1]) == ids.numel() == int((text.argmax(1) + 1).sum())
    table = model.tok_emb.clone().requires_grad_()
    spare = torch.full((3,), 7)                                                # rows behind the last prompt do not matter
    feats = model.encode_text_packed(torch.cat([ids, spare]).cuda(), cu.cuda(), table)
    assert rel(feats, want) < tol
    (g,) = torch.autograd.grad((feats * w.cuda()).sum(), table)
    # the backward pass runs the same products once more each way
    assert rel(g, gt) < 3 * tol
    unused = torch.ones(500, dtype=torch.bool)
    unused[ids] = False
    assert bool(unused.any()) and float(g[unused.cuda()].abs().max()) == 0


def test_packed_prompts_do_not_see_each_other(cuda):
    """With 8-bit Linear layers every step up to the projection is the same for any batch: alone, reordered, next to a NaN prompt."""
    sd = fclip.random_state_dict(CFG, 6)
    model = fclip.CLIP(sd, torch.float16, int8=True, text_packed=True)
    text = prompts(6, 7)
    full = model.encode_text(text)
    flip = model.encode_text(text.flip(0)).flip(0)
    assert torch.allclose(full, flip, rtol=1e-5, atol=1e-6)                     # (the fp32 projection may cut its sum differently)
    for i in range(6):
        assert torch.allclose(model.encode_text(text[i:i + 1]), full[i:i + 1], rtol=1e-5, atol=1e-6)
    ids, cu = fclip.pack_tokens(text)
    empty = torch.cat([cu[:3], cu[2:]])                                        # an empty prompt in the middle
    got = model.encode_text_packed(ids.cuda(), empty.cuda())
    assert torch.allclose(got[[0, 1, 3, 4, 5, 6]], full, rtol=1e-5, atol=1e-6) and bool(torch.isfinite(got[2]).all())


def test_int8_image_tower(cuda):
    sd = fclip.random_state_dict(CFG, 8)
    x = torch.randn(3, 3, 32, 32, generator=torch.Generator().manual_seed(9))
    xr = x.clone().requires_grad_()
    want = oclip.encode_image(sd, xr)
    w = torch.randn(want.shape, generator=torch.Generator().manual_seed(10))
    (gw,) = torch.autograd.grad((want * w).sum(), xr)
    xg = x.cuda().requires_grad_()
    model = fclip.CLIP(sd, torch.float16, int8=True)
    got = model.encode_image(xg)
    assert rel(got, want) < TOL8
    (g,) = torch.autograd.grad((got * w.cuda()).sum(), xg)
    assert rel(g, gw) < 3 * TOL8


def test_constructor_and_argument_refusals(cuda):
    sd = fclip.random_state_dict(CFG, 1)
    with pytest.raises(ValueError):
        fclip.CLIP(sd, torch.float16, int8=True, fp8=True)
    with pytest.raises(ValueError):
        fclip.CLIP(sd, torch.float32, int8=True)
    with pytest.raises(ValueError):
        fclip.CLIP(sd, torch.float32, text_packed=True)
    plain = fclip.CLIP(sd, torch.float16)
    with pytest.raises(RuntimeError):
        plain.encode_text_packed(torch.zeros(4, dtype=torch.long, device="cuda"), torch.tensor([0, 4], dtype=torch.int32, device="cuda"))
    packed = fclip.CLIP(sd, torch.float16, text_packed=True)
    with pytest.raises(TypeError):
        packed.encode_text_packed(torch.zeros(4, dtype=torch.int32, device="cuda"), torch.tensor([0, 4], dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        packed.encode_text(torch.zeros(2, packed.context_length + 1, dtype=torch.long))
    with pytest.raises(ValueError):
        fmain.encode_text("synthetic:2", int8=True)


def test_encode_text_command_packed(cuda, tmp_path):
    """The cache command over ViT-B/32's text tower: packed features next to the padded fp32-grade ones (12 blocks)."""
    a = fmain.encode_text("synthetic:20:3", out=str(tmp_path / "a.pkl"), batch_size=8)
    assert fmain._cli(["encode_text", "synthetic:20:3", str(tmp_path / "b.pkl"), "--packed"]) == 0
    assert fmain._cli(["encode_text", "synthetic:20:3", str(tmp_path / "c.pkl"), "--packed", "--int8"]) == 0
    assert fmain._cli(["encode_text", "synthetic:20:3", "--nonsense"]) == 2
    b, c = torch.load(tmp_path / "b.pkl", weights_only=True), torch.load(tmp_path / "c.pkl", weights_only=True)
    assert a.shape == b.shape == c.shape == (20, 512)
    assert rel(b, a) < 10 * 12 * torch.finfo(torch.float16).eps / 2
    assert rel(c, a) < 4 * 12 * 0.012
