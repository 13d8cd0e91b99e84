"""Rotary positions of as many rows as the entry point takes: more workgroups of one token each than a grid's first
dimension holds threads for (2^24 of 256)."""
import pytest
import torch

import train_oracle as orc
import tsa
from test_gpu_rope import check

pytestmark = pytest.mark.gpu


def test_more_rows_than_one_grid_dimension(dev):
    B, H, D, rot = 1 << 24, 9, 64, 2  # 288 units a token: a workgroup takes one
    x = torch.randn(1, H, 1, D, device=dev).half()
    out = torch.empty(B, H, 1, D, dtype=torch.float16, device=dev)
    at = [0, 1, (1 << 23) - 1, 1 << 23, (1 << 23) + 1, B - 2, B - 1]
    n, lens = torch.zeros(B, dtype=torch.int32, device=dev), torch.zeros(B, dtype=torch.int32, device=dev)
    for i, b in enumerate(at[::2]):
        n[b], lens[b] = 1, 1000 * i + 7
    out[at] = 5.0
    rope = tsa.Rope(D, rot=rot)
    tsa.rope_fwd(rope, x.expand(B, H, 1, D), len=lens, n_new=n, q_out=out)
    f, amp = orc.freqs(rot)
    for i, b in enumerate(at):
        if i % 2:
            assert (out[b] == 5).all(), b  # padding
        else:
            check(rope, f, amp, x, out[b:b + 1], lens[b].view(1, 1) - 1)
    del out
    torch.cuda.empty_cache()
