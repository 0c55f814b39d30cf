"""Paged cache at the edges of what it takes, on the device."""
import pytest
import torch

from elfa_b200 import native, ops

from paged_cases import attend64, close, make

pytestmark = pytest.mark.gpu


def _run(c, **kw):
    return ops.paged_attention(c["q"], c["pages"], c["table"], c["q_start"], c["kv_len"], **kw)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("step", [0.0, 0.05])
def test_blocks_that_follow_each_other(cuda_device, hd, step):
    """Items of 24 blocks: the probabilities of one are written where the product of the block before has just read its own, and, with keys that grow, again when a row's
    maximum has moved. The same bits every time."""
    c = make([(128, 3000), (140, 140)], 4, 2, hd, 64, seed=hd)
    for b, kv in enumerate(c["kv_len"].tolist()):
        pos = torch.arange(kv, device=cuda_device)
        at = (c["table"][b, pos // 64].long(), 0, slice(None), pos % 64)
        c["pages"][at] = (c["pages"][at].float() * (0.5 + step * (pos // 128))[:, None, None]).bfloat16()
    ref, mag = attend64(c)
    outs = [_run(c, max_new=140) for _ in range(8)]
    assert close(outs[0], ref, mag) and all(torch.equal(o, outs[0]) for o in outs)
    assert native.status() == 0
