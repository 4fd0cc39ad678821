"""The variant's training step repeats bit for bit at sequences of two key tiles: a sum of
two numbers has no order, and every other sum of the step has a fixed one."""

import numpy as np
import pytest
import torch

from rig_b200 import ops
from rig_b200.model import GPTTrainer, init_params
from test_variant_step import _batch, _config


@pytest.mark.gpu
def test_eager_captured_and_overlapped_steps_are_the_same(cuda):
    cfg = _config(steps=6, warmup_steps=1)
    assert cfg.seq_len == 256
    runs = {}
    for how in ("eager", "again", "graph", "overlap"):
        tr = GPTTrainer(cfg, cfg.batch_size, cuda, overlap_optimizer=how == "overlap")
        tr.load_params(init_params(cfg, 0))
        for i in range(4):
            x, y = _batch(cfg, i)
            tr.train_step(x.to(cuda), y.to(cuda))
            if how == "graph" and i == 0:
                tr.capture()
        torch.cuda.synchronize()
        assert ops.device_error() == 0 and int(tr.step_dev) == 4
        runs[how] = [t.cpu().numpy() for t in (tr.params, *tr.state8, tr.history[:4, :2])]
        norms = tr.history[:4, 2].cpu().numpy()
        # (in buckets the squares of the gradients are added up in another order)
        first = norms if how == "eager" else first
        np.testing.assert_allclose(norms, first, rtol=1e-6 if how == "overlap" else 0)
    for how in ("again", "graph", "overlap"):
        for a, b in zip(runs["eager"], runs[how]):
            np.testing.assert_array_equal(a, b)
