"""CPU: what the entries of cross attention, RMS norm and gradient clipping, and the trainer around them, decide on the host."""
import math
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_nothing_turns_graph_packet_capture_on():
    """with it replayed graphs end in a GPU memory fault: no tool, benchmark or module sets the variable to anything but 0"""
    for folder in ("", "tools", "ogmm_amd", "perf", "oracle"):
        for name in sorted(os.listdir(os.path.join(ROOT, folder))):
            if name.endswith((".py", ".sh")):
                text = open(os.path.join(ROOT, folder, name), encoding="utf-8").read()
                assert not re.search(r"PACKET_CAPTURE\W{0,8}=\W{0,3}[1-9]", text), os.path.join(folder, name)


@pytest.mark.parametrize("hits", [(True, False), (False, True), (True, True), (False, False)])
@pytest.mark.parametrize("limit", [None, 0.5])
def test_trainer_returns_a_norm_for_every_step(hits, limit):
    """with a limit "grad_norm" is there for a skipped step too, as a NaN, and for one that left no gradient, as zero"""
    from ogmm_amd.trainer import Trainer

    class Steps(Trainer):
        def _traced(self, src, *_):
            R, t = torch.eye(3).repeat(src.shape[0], 1, 1), torch.zeros(src.shape[0], 3)
            return (R, t), torch.ones(()), {}, None, None

        def _overflow_hits(self, fwd, bwd):
            return hits

    trainer = Steps(torch.nn.Linear(2, 2), max_grad_norm=limit, loss_scale=1.0)
    for p in trainer.model.parameters():
        p.requires_grad_(False)
    info = trainer.step(torch.zeros(2, 3, 4), torch.zeros(2, 3, 4), torch.eye(4).repeat(2, 1, 1), None, None)
    assert info["skipped"] == any(hits) and ("grad_norm" in info) == (limit is not None)
    if limit is not None:
        assert info["grad_norm"].shape == () and (math.isnan(float(info["grad_norm"])) if any(hits) else float(info["grad_norm"]) == 0.0)


def test_heads_that_the_kernels_cannot_reach_are_copied():
    """the attention entries take 64 rows and the heads that share a key head within 4 GB; rows, heads or addresses beyond what they take become a copy"""
    from ogmm_amd import ops
    far = torch.empty((1 << 31) + (1 << 23), dtype=torch.bfloat16)          # (never touched but where the heads lie)
    for heads, step, group, kept in ((256, 1 << 23, 256, False), (256, 1 << 23, 8, True), (250, 1 << 23, 250, True), (2, 1 << 24, 1, False), (4, 64, 4, True), (4, 60, 4, False)):
        t = far.as_strided((1, 3, heads, 8), (8, 8, step, 1))
        if kept:
            assert ops._heads(t, "q", t.dtype, group)[0] is t
        else:
            for i in range(heads):
                t[:, :, i].fill_(i)
            x, _, n, h = ops._heads(t, "q", t.dtype, group)
            assert x.is_contiguous() and (n, h) == (heads * 8, 8) and torch.equal(x, t)
