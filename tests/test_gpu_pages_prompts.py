"""The kernel of paged FP8 attention for many rows, by calls whose bounds are past what the one for few rows takes."""
import numpy as np
import pytest

import w4amd
from test_gpu_pages import Attn

pytestmark = pytest.mark.gpu

FEW_WORK = 7e8  # rows of a call times positions times D, up to which the other kernel takes everything


def prompts(seed, lens, adds, H, group, D, page, **more):
    """Places behind the last sequence until the call is one of the kernel for many rows."""
    longest = min(more.get("max_len") or max(lens), (max(-(-max(lens) // page), 1) + 1) * page)
    pad = max(0, int(FEW_WORK / (H * group * longest * D)) + 1 - sum(adds))
    a = Attn(seed, lens, adds, H, group, D, page, pad=pad, **more)
    a.plan = w4amd.capi().attention_f8_pages_plan_for(a.view, a.batch, group)
    assert a.plan[0] >= 2 and any(n * group > a.plan[1] for n in adds), a.plan
    return a


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("page", [1, 7, 24])
def test_pages_that_are_no_multiple_of_16(D, page):
    """Tiles whose scales are laid out by the four waves; with pages of one position a table holds 448 of them, and what
    is left over is a single tile."""
    prompts(D + page, [449, 512, 64, 40, 960], [120, 64, 64, 33, 50], 1, 4, D, page).check()
    prompts(D + page + 1, [64], [64], 2, 4, D, page).check()
    prompts(D + page + 2, [500], [90], 1, 4, D, page).check()
