"""Packed-prompt operators without a GPU: what the public entry points do around the launches, with the launchers stubbed, and more refusals."""
import pytest
import torch
from torch.autograd import forward_ad

from feed_forward_vqgan_clip_amd import kernels as K
from feed_forward_vqgan_clip_amd import ops

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


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
