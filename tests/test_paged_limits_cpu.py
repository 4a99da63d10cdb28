"""The paged cache's and the log probabilities' oracle and entry points at their limits, on the CPU."""
import math

import torch

from hrm_text_b200.models.paged import token_logprobs_reference


def test_likeliest_order_is_nan_then_infinity_then_the_lowest_id():
    nan, inf = math.nan, math.inf
    rows = torch.tensor([[inf, 1.0, nan, inf, nan], [-nan, nan, 0.0, -inf, inf], [-0.0, 0.0, -inf, 0.0, -1.0]])
    for dtype in (torch.float32, torch.float64):
        ids = token_logprobs_reference(rows.to(dtype), torch.zeros(3, dtype=torch.long), 5)[2]
        assert ids.tolist() == [[2, 4, 0, 3, 1], [0, 1, 4, 2, 3], [0, 1, 3, 4, 2]]
