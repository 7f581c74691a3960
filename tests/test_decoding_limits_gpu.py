"""The decoding operators at the limits of what their documentation allows, on the GPU against oracle/decoding.py.

Tolerances are those of test_decoding_gpu: pages, whole numbers and held values exactly, attention within half a step of the
bfloat16 result plus 2**-10 of sum p |v| / sum p.  Values far apart cost nothing on top: their products are exact, and a column's
sum is one of float32.  Selection: the large bfloat16 chunk adds up 64 exponentials per lane, 64 * 2**-24 relative, which with the
17 * 1.44 * 2**-24 of their arguments and the 2**-19 of the result is still below 1e-5.
"""
import math

import numpy as np
import pytest
import torch

from oracle import decoding as od
from tests.test_decoding_gpu import _gen, both, same_attention, same_pages, same_tokens

pytestmark = pytest.mark.gpu


# ---- pages


def test_compact_results_stay():
    """The number of pages that a compaction returned is not changed by the next one."""
    c, o = both(4, 256, 1, 64)
    used = []
    for par in ([[0, 1], [0, 1]], [[0, -1], [0, 1]], [[-1, 1], [0, -1]]):
        c.extend(70)
        o.extend(70)
        c.reorder(torch.tensor(par, device="cuda"))
        o.reorder(par)
        used.append((c.compact(), o.compact()))
        same_pages(c, o)
    assert len({want for _, want in used}) == 3
    assert [int(got) for got, _ in used] == [want for _, want in used]
    assert all(got.dtype == torch.int32 and got.dim() == 0 for got, _ in used)
