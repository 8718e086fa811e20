"""The paged operators at the edges of their arguments: lengths that no sum can
hold, scales of any sign, long spans, workspaces after a wait that ran out."""
from __future__ import annotations

import os
import subprocess
import sys

import numpy as np
import pytest

import paged_helpers as P

pytestmark = pytest.mark.gpu

SUM_END = (1 << 30) - 1  # where the tables' running sums stop


def dev(torch, x, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(x), dtype=dtype, device="cuda")


class Step:
    """One paged_step call over `past`, `new`, `held`; its tables as numpy arrays."""

    def __init__(self, torch, N, past, new, held, queue, ring, table, page, max_blocks, max_tok):
        i32, n = torch.int32, len(past)
        z = lambda k: torch.full((k,), -99, dtype=i32, device="cuda")  # noqa: E731
        self.out = dict(held_out=z(n), queue_out=z(4), seq_len=z(n), q_start=z(n + 1), positions=z(max_tok),
                        slots=z(max_tok), token_req=z(max_tok))
        self.ring = dev(torch, ring, i32)
        N.paged_step_dev(N.paged_step(n_req=n, page_size=page, n_pages=len(ring), max_blocks=max_blocks,
                                      max_tok=max_tok, past=dev(torch, past, i32), n_new=dev(torch, new, i32),
                                      held=dev(torch, held, i32), queue=dev(torch, queue, i32), ring=self.ring,
                                      block_table=table, **self.out))
        torch.cuda.synchronize()

    def check(self, want):
        for name, key in (("held_out", "held"), ("queue_out", "queue"), ("seq_len",) * 2, ("q_start",) * 2,
                          ("positions",) * 2, ("slots",) * 2, ("token_req",) * 2):
            np.testing.assert_array_equal(self.out[name].cpu().numpy(),
                                          np.minimum(np.asarray(want[key], np.int64), SUM_END), err_msg=name)
        np.testing.assert_array_equal(self.ring.cpu().numpy(), np.asarray(want["ring"]))


@pytest.mark.parametrize("new", [[1 << 30, 1 << 30, 3, 2], [3, (1 << 31) - 1, (1 << 31) - 1, 5], [1 << 30] * 40 + [4]])
def test_step_of_lengths_past_any_sum(nncu, torch_cuda, new):
    """New tokens whose sum passes 2^31: nobody behind them is served, and the sums stay at their end."""
    n, page, n_pages, max_blocks, max_tok = len(new), 16, 12, 6, 40
    past, held = [5] * n, [1] * n
    table = np.arange(n * max_blocks).reshape(n, max_blocks) % n_pages
    ring = np.arange(n_pages)
    want = P.step(past, new, held, [3, 9], ring, table, page, n_pages, max_blocks, max_tok)
    Step(torch_cuda, nncu, past, new, held, [3, 9], ring, dev(torch_cuda, table, torch_cuda.int32), page, max_blocks,
         max_tok).check(want)
