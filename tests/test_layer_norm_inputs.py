"""`nn.layer_norm` of views: broadcast rows, overlapping rows, transposed and sliced inputs."""

import pytest
import torch

from rig_b200 import nn

VIEWS = {
    "row over rows": lambda t: t[0].expand(7, 40),
    "row over a batch": lambda t: t[:1].expand(3, 7, 40),
    "batch of rows": lambda t: t.unsqueeze(1).expand(9, 5, 40),
    "one number": lambda t: t[:1, :1].expand(6, 40),
    "overlapping rows": lambda t: t.flatten().as_strided((8, 40), (16, 1)),
    "transposed": lambda t: t.flatten()[:320].view(40, 8).t(),
    "every other row": lambda t: t[::2],
    "one row": lambda t: t[3:4],
    "columns": lambda t: t[:, 3:20],
    "a vector": lambda t: t[2],
}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("view", VIEWS)
def test_views_equal_their_copies(cuda, view, dtype):
    g = torch.Generator().manual_seed(3)
    base = torch.randn(9, 40, generator=g).to(dtype).to(cuda)
    one = base.clone().requires_grad_(True)
    x = VIEWS[view](one)
    d = x.shape[-1]
    w, b = (torch.randn(d, generator=g).to(cuda).requires_grad_(True) for _ in range(2))
    dy = torch.randn(x.shape, generator=g).to(dtype).to(cuda)
    y = nn.layer_norm(x, w, b)
    got = torch.autograd.grad(y, (x, w, b), dy)
    copy = VIEWS[view](base).contiguous().requires_grad_(True)
    want_y = nn.layer_norm(copy, w, b)
    want = torch.autograd.grad(want_y, (copy, w, b), dy)
    assert torch.equal(y, want_y) and all(torch.equal(p, q) for p, q in zip(got, want))
    nn.layer_norm(x, w, b).backward(dy)  # the view's own gradient, down to its base
    assert one.grad.shape == one.shape and torch.isfinite(one.grad).all()
