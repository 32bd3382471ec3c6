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


def test_orders_that_an_int_does_not_hold(pkg):
    x, r = torch.ones(64, device="cuda"), pkg.hp_cuda_grad_result()
    for order in ((1 << 32) + 2, 1 << 32, (1 << 64) + 2):
        with pytest.raises(ValueError, match="order"):
            pkg.hp_cuda_grad_norm([x], [64], r, order)
        with pytest.raises(ValueError, match="order"):
            pkg.hp_cuda_grad_clip([x], [64], None, 1.0, r, order=order)
        with pytest.raises(ValueError, match="order"):
            pkg.hp_cuda_gd_momentum([x], [64], [torch.ones(64, device="cuda")], None, 0.9, 1.0, r, order)
    assert bool((x == 1).all()) and bool((r == 0).all())
    # numbers of other kinds than int are taken as before
    pkg.hp_cuda_grad_norm([x], [np.int64(64)], r, np.int32(2))
    assert r[0].item() == 64.0
