"""Each way that adapters' sizes are dispatched, against 64-bit products (MI355X).

The bars are those of the general cases without what a second product of two parts lost:
t and s keep float32's bits.  float16's up is taken in two parts, beside t in three, so
twice the additions.
"""

from __future__ import annotations

import pytest
import torch

from rosellm_amd.rosetrainer import adapter_linear

from _philox import keep
from test_gpu_adapters import DTYPES, _close, _make, _reference

pytestmark = pytest.mark.gpu

CASES = [
    # N, A, H, O, r, runs
    # few rows and more columns than one launch takes: whole and partial slabs and stages
    *[(N, 3, 96, O, r, 1) for N, O in ((16, 16385), (40, 20000), (33, 20480)) for r in (8, 32, 64, 128)],
    # the same of the gradient of x
    *[(N, 3, H, 80, r, 1) for N, H in ((16, 16385), (40, 20480)) for r in (8, 32, 64, 128)],
    # many rows of whole sizes, and of whole sizes in one dimension
    *[(N, A, H, O, r, runs) for r in (16, 32, 64, 128) for N, A, H, O, runs in
      ((1500, 3, 256, 512, 100), (3000, 1, 512, 256, 3000), (2100, 20, 768, 264, 1), (1300, 2, 200, 1024, 700))],
    # many rows of ranks and sizes that are not whole
    *[(N, A, H, O, r, runs) for r in (20, 40, 64, 90) for N, A, H, O, runs in
      ((600, 3, 130, 77, 1), (1100, 2, 71, 515, 300), (2000, 5, 333, 258, 60))],
    # the borders of few rows
    *[(N, 2, 72, 300, r, 9) for r in (16, 32, 64, 128) for N in (512, 513, 1024, 1025)],
]


@pytest.mark.parametrize("dtype", DTYPES, ids=lambda d: str(d)[6:])
@pytest.mark.parametrize("N,A,H,O,r,runs", CASES)
def test_product_and_gradients(device, N, A, H, O, r, runs, dtype):
    print(f"[adapters] N={N} A={A} H={H} O={O} r={r} runs={runs} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(N + H + O + r)
    x, base, down, up, ids, g = (v.to(device) for v in _make(N, A, H, O, r, dtype, gen, runs))
    scales = (torch.rand(A, generator=gen) + 0.1).to(device)
    more = 2 if dtype == torch.float16 else 1
    for b, p in ((base, 0.0), (None, 0.25)):
        kw = dict(dropout_p=p, seed=11, offset=5) if p else {}
        mask, factor = keep(N, H, p, 11, 5) if p else (None, 1.0)
        leaves = [v.clone().requires_grad_() for v in (x, down, up)]
        y = adapter_linear(*leaves, ids, base=b, scales=scales, **kw)
        out = (y, *torch.autograd.grad(y, leaves, g))
        # (the operands as float32: without the part that is for two parts of t)
        want = _reference(x.float(), b, down.float(), up.float(), ids, g, scales,
                          None if mask is None else mask.to(device), factor)
        for got, (w, e), what in zip(out, want, ("y", "dx", "ddown", "dup")):
            assert got.dtype == dtype and got.shape == w.shape
            _close(got, w.cpu(), more * e.cpu(), what)
        none = ids < 0
        assert torch.equal(out[0][none], torch.zeros_like(base)[none] if b is None else base[none])
        assert not out[1][none].any()
