"""Verification of drafted tokens at the sizes of a serving batch: chunks of more than one round of loads, rows that several ways of ending them divide, long vocabularies."""
import pytest
import torch

import capi_serving as cs
import serving_ref as ref
from test_gpu_verify import LEFT, Case

pytestmark = pytest.mark.gpu


def chunks(n, V):
    """Of a row: the workspace holds a 64-bit sum for each, and a number for every sequence."""
    return (cs.lib().minfer_verify_drafts_workspace_bytes(n, V) - (n * 4 + 255) // 256 * 256) // (8 * n)


@pytest.mark.parametrize("n,most,V,dtype,drafter,parts", [
    (64, 2, 128256, torch.float32, True, 32),        # chunks of 4096, 2048 workgroups
    (64, 1, 128256, torch.bfloat16, True, 32),
    (150, 1, 50257, torch.bfloat16, False, 13),      # 1950 workgroups of 8 KiB
    (300, 1, 50257, torch.bfloat16, True, 7),        # chunks of 8192 16-bit elements: the unrolled rounds
    (300, 1, 50257, torch.float16, False, 7),
    (100, 1, 50257, torch.float32, False, 13),       # 1300 workgroups of 16 KiB: one launch
    (1, 3, 600000, torch.float32, True, 147),        # as many chunks as threads put together, longer ones for that
    (2, 2, 1100000, torch.float16, False, 180),
    (1700, 1, 9001, torch.float32, True, 2),         # more sequences than there are counters, with several chunks
])
def test_large(kerns, n, most, V, dtype, drafter, parts):
    assert chunks(n, V) == parts
    Case(n, most, V, dtype, drafter, seed=V + n).check(kerns)


@pytest.mark.parametrize("n,V,dtype", [(64, 128256, torch.float32), (300, 50257, torch.bfloat16), (1, 600000, torch.float32)])
def test_large_rows_without_weight(kerns, n, V, dtype):
    """Refused drafts where the target has nothing more than the drafter anywhere, rows of zeros, and rows whose only weight lies at an end."""
    c = Case(n, 0, V, dtype, lens=[2] * n, seed=n)
    c.accept_u.fill_(1.0 - 2.0 ** -24)
    c.target = c.draft.clone()
    x = c.tokens[1::2]
    c.draft[torch.arange(0, 2 * n, 2), x] *= 1.5
    if n > 1:
        for s, keep in ((3, None), (4, 0), (5, V - 1), (6, 70 % V)):
            c.target[2 * s] = 0
            if keep is not None:
                c.target[2 * s, keep] = 0.25
        c.draft[8:14] *= 0.5
    want, kept = ref.verify(c.tokens, c.cu, c.target, c.draft, c.accept_u, c.sample_u)
    got = c.call(kerns)
    assert got[1] == kept and got[0] == [LEFT if t is None else t for t in want]
    if n > 1:
        assert got[0][6] == -1 and kept[4] == kept[5] == 0 and got[0][8] == 0 and got[0][10] == V - 1


@pytest.mark.parametrize("n,V,dtype", [(64, 128256, torch.float32), (300, 50257, torch.bfloat16)])
def test_large_rows_off_the_null_stream(kerns, n, V, dtype):
    c = Case(n, 1, V, dtype, seed=5)
    want = c.call(kerns)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        assert c.call(kerns) == want
