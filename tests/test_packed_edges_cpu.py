"""Packed-prompt operators without a GPU: what the public entry points do around the launches, with the launchers stubbed, and more refusals."""
import ctypes
import os

import pytest
import torch
from torch.autograd import forward_ad

from feed_forward_vqgan_clip_amd import _lib
from feed_forward_vqgan_clip_amd import kernels as K
from feed_forward_vqgan_clip_amd import ops

built = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="libffvc_hip.so not built (run __graft_entry__.build())")
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


class Pack:
    """The part of ops.Weights that the autograd nodes read, on the CPU (Weights.frozen uploads)."""

    def __new__(cls, N, Kd, cdt, int8):
        w = torch.randn(N, Kd)
        W = ops.Weights(None, torch.zeros(N), w.to(cdt), w.t().contiguous().to(cdt))
        if int8:
            W.int8 = (torch.zeros(N, Kd, dtype=torch.int8), torch.ones(N))
        return W


@pytest.fixture
def linear_stubs(monkeypatch):
    """Products that return zeros of the right shape (and the residual they are given); the outputs that were allocated for them."""
    made = []

    def linear_int8(x, wq, ws, bias=None, act=0, residual=None, out_dtype=None, want_actgrad=False):
        y = torch.zeros(*x.shape[:-1], wq.shape[0], dtype=out_dtype or x.dtype)
        if residual is not None:
            y += residual
        made.append(y)
        return (y, torch.ones_like(y)) if want_actgrad else y

    def gemm(x, w, y, *a, residual=None, aux=None, **kw):
        y.zero_()
        if residual is not None:
            y += residual
        made.append(y)

    monkeypatch.setattr(K, "linear_int8", linear_int8)
    monkeypatch.setattr(K, "gemm", gemm)
    monkeypatch.setattr(K, "cast", lambda t, dt: t.to(dt))
    return made


@pytest.mark.parametrize("int8", [False, True])
def test_mlp_gradient_of_the_residual_alone(linear_stubs, int8):
    """A frozen or detached x beside a trainable residual stream: the residual's gradient is the output's, with no product in the backward."""
    W1, W2 = Pack(64, 32, HF, int8), Pack(32, 64, HF, int8)
    x, res = torch.randn(5, 32).half(), torch.randn(5, 32, requires_grad=True)
    y = ops.mlp(x, W1, W2, K.ACT_QUICKGELU, residual=res, out_dtype=F32)
    before = len(linear_stubs)
    dy = torch.randn(5, 32)
    (g,) = torch.autograd.grad(y, res, dy)
    assert torch.equal(g, dy) and len(linear_stubs) == before
    # both, and x alone, still run their products
    x.requires_grad_()
    y = ops.mlp(x, W1, W2, K.ACT_QUICKGELU, residual=res, out_dtype=F32)
    gx, g = torch.autograd.grad(y, (x, res), dy)
    assert torch.equal(g, dy) and gx.shape == x.shape and len(linear_stubs) == before + 4


def test_linear_with_8_bit_weights_allocates_its_output_once(linear_stubs, monkeypatch):
    W = Pack(64, 32, HF, True)
    sizes = []
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **kw: sizes.append(a) or empty(*a, **kw))
    y = ops.linear(torch.randn(5, 32).half(), W, residual=torch.randn(5, 64), out_dtype=F32)
    assert y.shape == (5, 64) and y.dtype == F32 and not sizes and len(linear_stubs) == 1


@pytest.fixture
def stubs(monkeypatch):
    """Launchers that return tensors of the right shape and count their calls."""
    calls = []

    def fwd(qkv, cu, heads, kv_heads, scale, want_lse=False):
        calls.append("attn")
        T, W = qkv.shape
        return qkv.new_zeros(T, heads * (W // (heads + 2 * kv_heads))), torch.zeros(heads, T)

    def embed(ids, table, scale=1.0, pos=None, pos_ids=None, out_dtype=None):
        calls.append("embed")
        return torch.zeros(*ids.shape, table.shape[1], dtype=out_dtype or table.dtype)

    monkeypatch.setattr(K, "attn_packed_qkv_fwd", fwd)
    monkeypatch.setattr(K, "embed_fwd", embed)
    return calls


def test_forward_mode_tangents_are_refused_and_not_dropped(stubs):
    """As by every other operator of the package: none has a forward-mode derivative."""
    qkv, cu = torch.randn(4, 3 * 2 * 64, dtype=HF), torch.tensor([0, 4], dtype=torch.int32)
    ids, table, pos = torch.tensor([0, 2, 1]), torch.randn(5, 8), torch.randn(3, 8)
    for grad in (False, True):
        with torch.set_grad_enabled(grad), forward_ad.dual_level():
            dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
            for call in (lambda: ops.attention_packed(dual(qkv), cu, 2), lambda: ops.embedding(ids, dual(table)), lambda: ops.embedding(ids, table, pos=dual(pos))):
                with pytest.raises(RuntimeError):
                    call()
            # a tangent elsewhere does not matter
            assert ops.attention_packed(qkv, cu, 2).shape == (4, 128) and ops.embedding(ids, table, pos=pos).shape == (3, 8)


def test_calls_without_a_gradient_make_no_node(stubs):
    qkv, cu = torch.randn(4, 3 * 2 * 64, dtype=HF), torch.tensor([0, 4], dtype=torch.int32)
    ids, table = torch.tensor([0, 2, 1]), torch.randn(5, 8)
    assert ops.attention_packed(qkv, cu, 2).grad_fn is None and ops.embedding(ids, table, pos=table).grad_fn is None
    assert ops.attention_packed(qkv.clone().requires_grad_(), cu, 2).grad_fn is not None
    assert ops.embedding(ids, table, pos=table.clone().requires_grad_()).grad_fn is not None
    with torch.no_grad():
        assert ops.attention_packed(qkv.clone().requires_grad_(), cu, 2).grad_fn is None
    assert stubs == ["attn", "embed", "attn", "embed", "attn"]


A = 1 << 12                                                           # an aligned non-null address that nothing may touch


def attn_desc(rows=4, seqs=1, heads=2, kv_heads=2, dim=64):
    d = _lib.AttnPackedDesc()
    for i, n in enumerate(("q", "k", "v", "out", "lse", "cu", "dout", "dq", "dk", "dv", "delta")):
        setattr(d, n, A + (i << 40))
    d.rows, d.seqs, d.heads, d.kv_heads, d.head_dim, d.dtype, d.scale = rows, seqs, heads, kv_heads, dim, _lib.BF16, 1.0
    for n in ("q", "k", "v", "o", "do", "dq", "dk", "dv"):
        setattr(d, n + "_rs", dim * heads)
        setattr(d, n + "_hs", dim)
    return d


def refused(rc, word):
    return rc != 0 and word in _lib.load().ffvc_last_error().decode()


@built
def test_launches_of_2_to_the_32_threads_are_refused():
    """Before anything runs, and by name."""
    lib = _lib.load()
    n = (1 << 26) - 3
    assert refused(lib.ffvc_embed_fwd(A, 1, 8, 5, A, 1.0, 0, 0, 0, 0, A, 1, 8, n, 8, None), "too many")
    ws = lib.ffvc_embed_bwd_ws_bytes(100, n, 8)
    assert refused(lib.ffvc_embed_bwd(A, 1, 8, A, 100, n, 8, 1.0, A, 1, A, ws, None), "too many")
    half = 1 << 25
    ws = lib.ffvc_embed_bwd_pair_ws_bytes(100, half, half, 8)
    assert refused(lib.ffvc_embed_bwd_pair(A, 1, 8, A, 100, half, 8, 1.0, A, A, half, A, 1, A, ws, None), "too many")
    assert refused(lib.ffvc_int8_quant(A, 0, 32, A, 32, A, n, 32, None), "too many")
    assert refused(lib.ffvc_gemm_int8(A, A, A, 16, A, 0, 0, 0, 1, 1 << 14, A, 0, 1 << 14, 0, 0, 1 << 27, 1 << 14, 16, None), "too many")
    for d in (attn_desc(rows=1 << 30, heads=8, kv_heads=8, dim=8), attn_desc(rows=1 << 30, seqs=1 << 29, heads=1, kv_heads=1, dim=8)):
        assert refused(lib.ffvc_attn_packed_fwd(ctypes.byref(d), None), "too many")
        assert refused(lib.ffvc_attn_packed_bwd(ctypes.byref(d), None), "too many")


def test_projections_that_do_not_divide_into_heads_are_refused():
    """By the launchers too, which would otherwise leave the last columns' gradient unwritten."""
    cu = torch.tensor([0, 4], dtype=torch.int32)
    for W, H, G in ((3 * 2 * 64 + 8, 2, 2), (200, 8, 8), (3 * 64, 0, 1), (3 * 64, 1, 0), (3 * 64, -1, 2)):
        qkv = torch.zeros(4, W, dtype=HF)
        with pytest.raises(ValueError):
            K.attn_packed_qkv_fwd(qkv, cu, H, G, 1.0)
        D = max(W // max(H + 2 * G, 1), 1)
        o, lse = torch.zeros(4, H * D if H > 0 else 0, dtype=HF), torch.zeros(max(H, 0), 4)
        with pytest.raises((ValueError, _lib.FFVCError)) as e:
            K.attn_packed_qkv_bwd(qkv, o, o, lse, cu, H, G, 1.0)
        assert isinstance(e.value, ValueError)
