"""CPU: the 4-bit layer names the argument that is not a tensor."""

from __future__ import annotations

import pytest
import torch


def test_arguments_that_are_no_tensors(pkg):
    def weights(n, d):
        w = object.__new__(pkg.W4Weights)            # no GPU to lay weights out: only their sizes are looked at
        w.num_experts, w.n, w.d, w.dtype = 4, n, d, torch.bfloat16
        return w
    hidden, ids, w = torch.zeros(3, 64, dtype=torch.bfloat16), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2)
    for args, name in ((([1.0], ids, w), "hidden_states"), ((hidden, ids, 0.5), "topk_weights"), ((hidden, [0], w), "topk_ids"),
                       ((None, ids, w), "hidden_states")):
        with pytest.raises(TypeError, match=name):
            pkg.moe_w4(*args, weights(64, 64), weights(64, 32))
    with pytest.raises(ValueError, match="CUDA"):
        pkg.moe_w4(hidden, ids, w, weights(64, 64), weights(64, 32))
    with pytest.raises(TypeError, match="w13"):
        pkg.moe_w4(hidden, ids, w, hidden, weights(64, 32))
