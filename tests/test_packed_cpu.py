"""Packed-prompt operators without a GPU: argument refusals (launchers and C entry points), descriptor layout, the formulas themselves."""
import ctypes
import math
import os
import re

import pytest
import torch

from feed_forward_vqgan_clip_amd import _lib
from feed_forward_vqgan_clip_amd import kernels as K
from feed_forward_vqgan_clip_amd import ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
built = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="libffvc_hip.so not built (run __graft_entry__.build())")
BF, F32 = torch.bfloat16, torch.float32


def test_attn_packed_desc_layout_matches_header():
    text = open(os.path.join(ROOT, "include", "ffvc.h")).read()
    body = text[text.index("typedef struct ffvc_attn_packed_desc {"):text.index("} ffvc_attn_packed_desc;")]
    names, types = [], []
    for line in body.splitlines()[1:]:
        m = re.match(r"\s*(?:const\s+)?(void|float|int32_t|int64_t)\s*(\*?)\s*(.+);", line)
        if m:
            for n in m.group(3).split(","):
                names.append(n.strip())
                types.append(ctypes.c_void_p if m.group(2) else {"float": ctypes.c_float, "int32_t": ctypes.c_int32, "int64_t": ctypes.c_int64}[m.group(1)])
    assert [(n, t) for n, t in zip(names, types)] == _lib.AttnPackedDesc._fields_


def test_attention_packed_refusals():
    cu = torch.tensor([0, 4], dtype=torch.int32)
    x = torch.zeros(4, 3 * 2 * 64, dtype=BF)
    for bad in (dict(heads=0), dict(heads=3), dict(heads=2, kv_heads=3), dict(heads=4, kv_heads=0), dict(heads=2, kv_heads=-1)):
        with pytest.raises(ValueError):
            ops.attention_packed(x, cu, **bad)
    with pytest.raises(ValueError):
        ops.attention_packed(x.view(2, 2, -1), cu, 2)
    for dh in (4, 12, 136):
        with pytest.raises(ValueError):
            ops.attention_packed(torch.zeros(4, 3 * 2 * dh, dtype=BF), cu, 2)
    with pytest.raises(TypeError):
        ops.attention_packed(x.float(), cu, 2)
    for c in (cu.long(), cu[:1], cu.view(1, 2), torch.zeros(4, dtype=torch.int32)[::2]):
        with pytest.raises(TypeError):
            ops.attention_packed(x, c, 2)
    with pytest.raises(_lib.FFVCError):                               # no CPU fallback
        ops.attention_packed(x, cu, 2)
    q = torch.zeros(4, 2, 64, dtype=BF)
    with pytest.raises(ValueError):
        K.attn_packed_fwd(q, q[:3], q, cu, 1.0)
    with pytest.raises(ValueError):
        K.attn_packed_fwd(q, q, q[:, :1], cu, 1.0)
    with pytest.raises(ValueError):
        K.attn_packed_fwd(q.transpose(1, 2), q, q, cu, 1.0)
    with pytest.raises(TypeError):
        K.attn_packed_fwd(q, q.half(), q, cu, 1.0)


def test_embedding_refusals():
    t = torch.zeros(5, 8)
    ids = torch.zeros(3, dtype=torch.long)
    with pytest.raises(TypeError):
        ops.embedding(ids.int(), t)
    with pytest.raises(TypeError):
        ops.embedding(torch.zeros(6, dtype=torch.long)[::2], t)
    with pytest.raises(ValueError):
        ops.embedding(ids, t.view(5, 2, 4))
    with pytest.raises(ValueError):
        ops.embedding(ids, torch.zeros(8, 5).t())
    with pytest.raises(ValueError):
        ops.embedding(ids, t, pos=torch.zeros(5, 9))
    with pytest.raises(ValueError):
        ops.embedding(ids, t, pos=t.half())
    with pytest.raises(ValueError):
        ops.embedding(ids, t, pos=t, pos_ids=torch.zeros(2, dtype=torch.long))
    with pytest.raises(TypeError):
        ops.embedding(ids, t.double())
    with pytest.raises(_lib.FFVCError):
        ops.embedding(ids, t)
    with pytest.raises(ValueError):
        K.embed_bwd(torch.zeros(4, 8), ids, 5)
    with pytest.raises(ValueError):
        K.embed_bwd(torch.zeros(3, 8), ids, 5, pos_ids=ids)
    with pytest.raises(ValueError):
        K.embed_bwd(torch.zeros(3, 8), ids, 5, pos_rows=4, pos_ids=torch.zeros(2, dtype=torch.long))


def test_int8_refusals():
    x = torch.zeros(4, 32, dtype=BF)
    wq, ws = torch.zeros(8, 32, dtype=torch.int8), torch.zeros(8)
    with pytest.raises(ValueError):
        K.int8_quant(torch.zeros(4, 24))
    with pytest.raises(TypeError):
        K.int8_quant(torch.zeros(4, 32, dtype=torch.float64))
    with pytest.raises(_lib.FFVCError):
        K.int8_quant(x)
    with pytest.raises(TypeError):
        K.linear_int8(x.float(), wq, ws)
    with pytest.raises(_lib.FFVCError):
        K.linear_int8(x, wq, ws)


@built
def test_c_entry_points_refuse_bad_arguments():
    """Every call here is turned away by the host checks: no launch, an error code and a message."""
    lib = _lib.load()
    A = 1 << 12                                                       # an aligned non-null address that nothing may touch
    d = _lib.AttnPackedDesc()
    for n in ("q", "k", "v", "out", "lse", "cu", "dout", "dq", "dk", "dv", "delta"):
        setattr(d, n, A)
    d.rows, d.seqs, d.heads, d.kv_heads, d.head_dim, d.dtype, d.scale = 4, 1, 2, 2, 64, _lib.BF16, 1.0
    for n in ("q", "k", "v", "o", "do", "dq", "dk", "dv"):
        setattr(d, n + "_rs", 128)
        setattr(d, n + "_hs", 64)
    for field, value in (("dtype", _lib.F32), ("rows", 0), ("rows", 1 << 31), ("seqs", 0), ("heads", 3), ("kv_heads", 0), ("head_dim", 12),
                         ("head_dim", 136), ("scale", float("nan")), ("scale", 0.0), ("scale", -1.0), ("scale", math.inf), ("q", 0), ("k", A + 2),
                         ("v_rs", 63), ("v_rs", 8), ("o_hs", 4), ("q_rs", 1 << 23), ("cu", 0)):
        e = _lib.AttnPackedDesc.from_buffer_copy(d)
        setattr(e, field, value)
        assert lib.ffvc_attn_packed_fwd(ctypes.byref(e), None) != 0, (field, value)
        assert lib.ffvc_attn_packed_bwd(ctypes.byref(e), None) != 0, (field, value)
        assert lib.ffvc_last_error()
    for field, value in (("dout", 0), ("dq", A + 8), ("dk_rs", 4), ("dv_hs", 1), ("lse", 0), ("delta", 0), ("dq_hs", 0), ("dk_rs", 64), ("dv_hs", 128)):
        e = _lib.AttnPackedDesc.from_buffer_copy(d)
        setattr(e, field, value)
        assert lib.ffvc_attn_packed_bwd(ctypes.byref(e), None) != 0, (field, value)
    for field, value in (("o_hs", 0), ("o_hs", 128), ("o_rs", 64)):                                # written rows and heads that overlap
        e = _lib.AttnPackedDesc.from_buffer_copy(d)
        setattr(e, field, value)
        assert lib.ffvc_attn_packed_fwd(ctypes.byref(e), None) != 0, (field, value)
    assert lib.ffvc_attn_packed_fwd(None, None) != 0 and lib.ffvc_attn_packed_bwd(None, None) != 0

    def embed_fwd(table=A, dt=1, ld=8, V=5, ids=A, pos=0, pld=0, npos=0, out=A, odt=1, ldo=8, n=3, dim=8):
        return lib.ffvc_embed_fwd(table, dt, ld, V, ids, 1.0, pos, pld, npos, 0, out, odt, ldo, n, dim, None)
    for kw in (dict(table=0), dict(dt=7), dict(ld=7), dict(V=0), dict(ids=0), dict(pos=A), dict(out=0), dict(odt=-1), dict(ldo=4), dict(n=0), dict(dim=0)):
        assert embed_fwd(**kw) != 0, kw
    need = lib.ffvc_embed_bwd_ws_bytes(100, 5, 8)
    assert need > 0 and lib.ffvc_embed_bwd_ws_bytes(0, 5, 8) == 0

    def embed_bwd(dout=A, dt=1, ld=8, ids=A, n=100, V=5, dim=8, grad=A, gdt=1, ws=A, nb=need):
        return lib.ffvc_embed_bwd(dout, dt, ld, ids, n, V, dim, 1.0, grad, gdt, ws, nb, None)
    for kw in (dict(dout=0), dict(dt=9), dict(ld=7), dict(ids=0), dict(n=0), dict(n=1 << 31), dict(V=0), dict(V=1 << 31), dict(grad=0), dict(ws=0),
               dict(ws=A + 4), dict(nb=need - 1)):
        assert embed_bwd(**kw) != 0, kw
    both = lib.ffvc_embed_bwd_pair_ws_bytes(100, 5, 7, 8)
    assert both > need and lib.ffvc_embed_bwd_pair_ws_bytes(100, 5, 0, 8) == 0

    def pair(dout=A, dt=1, ld=8, ids=A, n=100, V=5, dim=8, grad=A, place=A, P=7, dpos=A, gdt=1, ws=A, nb=both):
        return lib.ffvc_embed_bwd_pair(dout, dt, ld, ids, n, V, dim, 1.0, grad, place, P, dpos, gdt, ws, nb, None)
    for kw in (dict(dout=0), dict(ids=0), dict(n=0), dict(V=0), dict(P=0), dict(P=1 << 31), dict(grad=0), dict(dpos=0), dict(gdt=8), dict(ws=A + 8), dict(nb=both - 1)):
        assert pair(**kw) != 0, kw

    def quant(x=A, dt=0, ldx=32, q=A, ldq=32, s=A, rows=4, k=32):
        return lib.ffvc_int8_quant(x, dt, ldx, q, ldq, s, rows, k, None)
    for kw in (dict(x=0), dict(x=A + 2), dict(dt=5), dict(ldx=16), dict(ldx=33), dict(q=A + 8), dict(ldq=40), dict(s=0), dict(rows=0), dict(k=24)):
        assert quant(**kw) != 0, kw

    def gemm(x=A, xs=A, w=A, ldw=32, ws=A, act=0, res=0, rdt=1, ldr=8, y=A, ydt=0, ldy=8, lo=0, M=4, N=8, k=32):
        return lib.ffvc_gemm_int8(x, xs, w, ldw, ws, 0, act, res, rdt, ldr, y, ydt, ldy, 0, lo, M, N, k, None)
    for kw in (dict(x=0), dict(x=A + 1), dict(xs=0), dict(w=0), dict(ldw=16), dict(ws=0), dict(act=3), dict(res=A, rdt=2), dict(res=A, ldr=7),
               dict(y=0), dict(ydt=2), dict(ldy=7), dict(lo=1), dict(M=0), dict(N=0), dict(k=0), dict(k=40), dict(k=131088, ldw=131088)):
        assert gemm(**kw) != 0, kw
    assert lib.ffvc_linear_int8_few_ok(16, 512) == 1 and lib.ffvc_linear_int8_few_ok(17, 512) == 0 and lib.ffvc_linear_int8_few_ok(16, 8192) == 0
    assert lib.ffvc_linear_int8_few(A, 0, 512, A, 512, A, 0, 0, 0, 1, 8, A, 0, 8, 0, 17, 8, 512, None) != 0
    assert lib.ffvc_linear_int8_few(A + 2, 0, 512, A, 512, A, 0, 0, 0, 1, 8, A, 0, 8, 0, 1, 8, 512, None) != 0


def test_gradient_formulas_against_autograd():
    """The closed forms the kernels compute (64 bits) are the derivatives of the forward: attention with shared heads, embedding."""
    g = torch.Generator().manual_seed(1)
    H, G, n, D, scale = 4, 2, 9, 8, 0.3
    q, k, v, do = (torch.randn(n, h, D, generator=g, dtype=torch.float64) for h in (H, G, G, H))
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    late = torch.ones(n, n, dtype=torch.bool).triu(1)
    p = torch.softmax((torch.einsum("ihd,jhd->hij", leaves[0], leaves[1].repeat_interleave(H // G, 1)) * scale).masked_fill(late, -math.inf), -1)
    o = torch.einsum("hij,jhd->ihd", p, leaves[2].repeat_interleave(H // G, 1))
    want = torch.autograd.grad(o, leaves, do)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for h in range(H):
        s = h // (H // G)
        P = p[h].detach()
        dP = do[:, h] @ v[:, s].T
        ds = scale * P * (dP - (do[:, h] * o[:, h].detach()).sum(1, keepdim=True))
        dq[:, h] = ds @ k[:, s]
        dk[:, s] += ds.T @ q[:, h]
        dv[:, s] += P.T @ do[:, h]
    for a, b in zip((dq, dk, dv), want):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-13)
