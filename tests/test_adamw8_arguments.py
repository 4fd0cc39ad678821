"""Arguments of the 8-bit AdamW step that the kernels would read or write past the end."""

import ctypes

import pytest
import torch

from rig_b200 import _lib, ops


@pytest.mark.gpu
def test_refused_before_anything_runs(cuda):
    n = 256
    cfg = _lib.AdamWConfig(learning_rate=1e-2, horizon_lr_scale=1.0, min_lr_ratio=0.1, warmup_steps=0,
                           total_steps=4, beta1=0.9, beta2=0.95, eps=1e-8, eps_horizon_scale=1.0,
                           weight_decay=0.1, wd_horizon_scale=1.0, grad_clip=0.0, grad_scale=1.0)
    p, g = torch.zeros(n, device=cuda), torch.ones(n, device=cuda)
    raw = bytes((_lib.TensorGroup * 2)(*(_lib.TensorGroup(offset=o, size=128, lr_mult=1.0, eps_mult=1.0,
                                                          wd_mult=1.0, decay=1) for o in (0, 128))))
    good = dict(groups=torch.frombuffer(bytearray(raw), dtype=torch.uint8).to(cuda),
                step=torch.zeros(1, dtype=torch.int32, device=cuda), loss=torch.ones(1, device=cuda),
                history=torch.zeros(4, 3, device=cuda), ws=ops.adamw_workspace(n, cuda))
    state = ops.adamw8_state(n, cuda)

    def step(**bad):
        a = {**good, **bad}
        ops.adamw8_step(p, state, g, a["groups"], 2, cfg, a["step"], a["loss"], a["history"], None, 0, a["ws"])

    def bucket(**bad):
        a = {**good, **bad}
        ops.adamw8_update_range(p, state, g, 0, n, a["groups"], 2, cfg, 0, None, 0, a["ws"])

    shared = [dict(ws=good["ws"][:-8]), dict(ws=good["ws"][::2]), dict(ws=good["ws"].cpu()),
              dict(groups=good["groups"][:ctypes.sizeof(_lib.TensorGroup)]), dict(groups=good["groups"].cpu())]
    own = [dict(step=good["step"].float()), dict(step=good["step"].cpu()), dict(loss=good["loss"].double()),
           dict(loss=torch.ones(0, device=cuda)), dict(history=torch.zeros(4, 2, device=cuda)),
           dict(history=torch.zeros(4, 6, device=cuda)[:, ::2]), dict(history=good["history"].half()),
           dict(history=torch.zeros(12, device=cuda))]
    before = ops.launch_count()
    for call, cases in ((step, shared + own), (bucket, shared)):
        for bad in cases:
            with pytest.raises(ValueError):
                call(**bad)
    assert ops.launch_count() == before
    step()
    torch.cuda.synchronize()
    assert int(good["step"]) == 1 and (p != 0).all() and good["history"][0, 0] == 1
