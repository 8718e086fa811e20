"""Every array of the 8-bit operators and the log probabilities lies in the
current GPU's memory: the host's is refused before anything is launched."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

N_ROWS, COLS = 4, 64
FLOATS = ("x", "gamma", "scales", "out", "x_scales", "w_scales", "bias", "add", "y", "logits", "logprob", "entropy",
          "top_logprobs")
WHOLE = ("ids", "tokens", "rank", "top_ids")
CALLS = {
    "i8_rows": ("i8_quantise_dev", dict(n=N_ROWS, cols=COLS, norm=1), ("x", "gamma", "codes", "scales")),
    "i8_lookup": ("i8_lookup_dev", dict(n=N_ROWS, cols=COLS, n_rows=N_ROWS), ("ids", "codes", "scales", "out")),
    "i8_linear": ("i8_linear_dev", dict(n_tok=N_ROWS, rows=COLS, cols=COLS),
                  ("x", "x_scales", "w", "w_scales", "bias", "add", "y")),
    "logprobs": ("logprobs_dev", dict(n=N_ROWS, n_vocab=COLS, top=3),
                 ("logits", "tokens", "logprob", "rank", "entropy", "top_ids", "top_logprobs")),
}


def memory(torch, call, name, host=False):
    kind = torch.float32 if name in FLOATS and not (call == "i8_linear" and name == "x") else \
        torch.int32 if name in WHOLE else torch.int8
    x = torch.zeros(COLS * COLS, dtype=kind)
    return x.pin_memory() if host else x.cuda()


@pytest.mark.parametrize("call,name", [(c, n) for c, (_, _, names) in CALLS.items() for n in names])
def test_host_memory_is_refused(nncu, torch_cuda, call, name):
    torch, N = torch_cuda, nncu
    run, sizes, names = CALLS[call]
    arrays = {n: memory(torch, call, n) for n in names}
    given = lambda a: getattr(N, call)(**sizes, **{n: x.data_ptr() for n, x in a.items()})  # noqa: E731
    getattr(N, run)(given(arrays))  # as it should be
    before = N.launch_count()
    arrays[name] = memory(torch, call, name, host=True)
    with pytest.raises(N.NnncError, match="device memory"):
        getattr(N, run)(given(arrays))
    assert N.launch_count() == before
    torch.cuda.synchronize()


def test_alternatives_that_are_not_asked_for_are_not_looked_at(nncu, torch_cuda):
    torch, N = torch_cuda, nncu
    ent = torch.zeros(N_ROWS, device="cuda")
    pinned = torch.zeros(16, dtype=torch.int32).pin_memory()
    N.logprobs_dev(N.logprobs(n=N_ROWS, n_vocab=COLS, logits=torch.zeros(N_ROWS, COLS, device="cuda"), entropy=ent,
                              top=0, top_ids=pinned.data_ptr()))
    torch.cuda.synchronize()
    assert bool((ent > 4.15).all())  # log 64
