"""The 8-bit cache's operators on the GPU at their limits."""
from __future__ import annotations

import pytest
import torch

from test_gpu_q8 import DEV, al, check_attend, make_q, random_cache, status

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("h, T", [(2, 3), (4, 16), (1, 40), (4, 100), (3, 333)])      # single tokens, prompts
def test_a_window_past_the_capacity_hides_nothing(dtype, h, T):
    """Requests padded on the left: positions reach down to -T, and a window that is as large as an int must not wrap
    around below them. Sinks that cover the cache hide nothing either, whatever the window."""
    C, lengths = 350, [350, 5, 1, 0, 100]
    cache = random_cache(h + T, len(lengths), 2, C, spread=1)
    q = make_q(T, len(lengths), 2, h, T, dtype)
    on_gpu = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    want = al().attend_q8(q, cache, on_gpu)
    check_attend(cache, q, lengths, 0, 0, want)
    for window in (C, C + 1, 2 ** 30, 2 ** 31 - 2, 2 ** 31 - 1):
        for sinks in (0, 4, 2 ** 31 - 1):
            assert torch.equal(al().attend_q8(q, cache, on_gpu, window=window, sinks=sinks), want), (window, sinks)
    check_attend(cache, q, lengths, 7, 2 ** 31 - 1, al().attend_q8(q, cache, on_gpu, window=7, sinks=2 ** 31 - 1))
    check_attend(cache, q, lengths, C - 1, 3, al().attend_q8(q, cache, on_gpu, window=C - 1, sinks=3))
    assert status() == 0
