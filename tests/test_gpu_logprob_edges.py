"""GPU tests of log probabilities (b2_logprob_forward) of long rows with a NaN: whatever comes behind it, the row's results are NaN."""
import math

import numpy as np
import pytest

from test_gpu_token_operators import _host, _rand, tm  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab,t", [(5001, "bf16"), (9001, "f32"), (25001, "f16"), (70000, "bf16")])
@pytest.mark.parametrize("rows", [60, 700, 2500])
@pytest.mark.parametrize("behind", ["nothing", "masked", "more", "much more"])
@pytest.mark.parametrize("top", [0, 4])
def test_nan_anywhere_in_a_row(tm, vocab, t, rows, behind, top):  # noqa: F811
    torch, b2 = tm
    x = _rand(torch, (rows, vocab), t, 3, 2.0)
    at = np.linspace(3, vocab - 1, 30).astype(int)             # rows 0, 2, 4, ... 58
    mask = torch.ones(rows, vocab, dtype=torch.uint8, device="cuda") if behind == "masked" else None
    for i, p in enumerate(at):
        for r in (2 * i, 2 * i + 1):
            if behind == "nothing":
                x[r, p + 1:] = -math.inf
            elif behind == "masked":
                mask[r, p + 1:] = 0
            elif behind == "much more":
                x[r, p + 1:] += 100.0
                x[r, p + 1 + (vocab - p) // 2:] += 100.0
        x[2 * i, p] = math.nan
    logprob, lse, entropy = (torch.full((rows,), 7.0, device="cuda") for _ in range(3))
    more = dict(top_tokens=torch.empty(rows, top, dtype=torch.int32, device="cuda"), top_logprobs=torch.empty(rows, top, device="cuda")) if top else {}
    b2.logprob_forward(x, torch.zeros(rows, dtype=torch.int32, device="cuda"), logprob, lse, entropy=entropy, mask=mask, **more)
    bad = np.arange(0, 60, 2)
    good = np.setdiff1d(np.arange(rows), bad)
    for v in (logprob, lse, entropy):
        assert np.isnan(_host(v)[bad]).all() and np.isfinite(_host(v)[good]).all()
    if top:
        assert (more["top_tokens"][torch.from_numpy(bad).cuda(), 0] == torch.from_numpy(at).cuda()).all()       # NaN ranks first
