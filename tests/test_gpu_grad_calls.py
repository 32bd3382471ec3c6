"""Calls of the gradient operators that their documentation allows, beside those of test_gpu_grad.py."""
import numpy as np
import pytest
import torch

from test_gpu_grad import f64, make, message

pytestmark = pytest.mark.gpu


def test_several_messages_for_one_momentum(pkg):
    # three messages for one tensor, and one for a tensor that shares its last elements
    n = 5000
    whole = torch.randn(n + 200, device="cuda")
    u, shared = whole[:n], whole[n - 100:]
    index = [[0, 7, 4999], [7, 8], list(range(4096, 4900)), [0, 99, 100, 299]]
    msgs = [message(i) for i in index]
    want = f64(whole)
    counts = torch.zeros(4, dtype=torch.int32, device="cuda")
    pkg.hp_cuda_gd_mask(msgs, [m.numel() for m in msgs], [u, u, u, shared], [n, n, n, 300], counts)
    for i in index[:3]:
        want[i] = 0
    want[n - 100 + np.array(index[3])] = 0
    assert np.array_equal(f64(whole), want) and counts.tolist() == [len(i) for i in index]
