"""Packed-prompt operators at their edges: values, offsets, widths and gradients that the ordinary cases do not reach."""
import pytest
import torch

from feed_forward_vqgan_clip_amd import ops

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
