"""GPU checks of speculative decoding's operators at the ends of their ranges; forms and bounds are those of
tests/test_gpu_drafts.py."""

import math

import numpy as np
import pytest
import torch

from tests.test_gpu_attention import say
from tests.test_gpu_drafts import attention, check_probs, sampling  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(7, 1000), (7, 40003), (200, 40003)])
def test_probs_of_far_logits(sampling, rows, vocab, dtype):  # noqa: F811
    """Logits further apart than the largest number, at temperatures that bring them together again."""
    say("far logits", rows, vocab, dtype)
    rng = np.random.default_rng(rows + vocab)
    x = rng.uniform(-3.3e38, 3.3e38, (rows, vocab))
    x[:, 7], x[:, vocab - 3] = 3.3e38, -3.3e38
    x[0, :vocab // 2] = -math.inf
    t = np.float32([1.5e38, 3e38, 4e37, math.inf, 1.0, 0.5, 1e37] + [2e38] * (rows - 7))
    x = torch.from_numpy(x.astype(np.float32)).to(dtype).cuda()
    check_probs(sampling, x, t, torch.empty(rows, vocab, device="cuda"))
