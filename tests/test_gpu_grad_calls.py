"""Calls of the gradient operators that their documentation allows, beside those of test_gpu_grad.py; the tolerances are
those derived there."""
import math

import numpy as np
import pytest
import torch

from gpu_util import stream_ptr
from test_gpu_grad import SIZES, coefficient, f64, intact, make, message, near, near_momentum, squares, types_of

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


def told(result, s, norm, c, scale=1.0):
    assert abs(result[0].item() - s) <= 1e-9 * s
    assert abs(result[1].item() / (abs(scale) * norm) - 1) <= 1e-9
    assert abs(result[2].item() - c) <= abs(c) * 2.0 ** -24 * (1 + 1e-6)


@pytest.mark.parametrize("measured", [0, 1])
@pytest.mark.parametrize("lead", [0, 1, 3])
@pytest.mark.parametrize("which", list(SIZES))
def test_fp32_outputs_in_the_place_of_the_gradients(pkg, which, lead, measured):
    sizes = SIZES[which]
    for share, scale in ((0.3, 1.0), (0.3, -0.5), (2.0, 0.125)):  # of the norm
        g, b = make(sizes, ["fp32"] * len(sizes), 90, lead)
        before = [f64(t) for t in g]
        total = squares(g)
        norm = math.sqrt(total)
        result = pkg.hp_cuda_grad_result()
        if measured:
            result[0] = total
        pkg.hp_cuda_grad_clip(g, sizes, g, share * abs(scale) * norm, result, measured, scale=scale)
        c = coefficient(norm, share * abs(scale) * norm, scale)
        assert c != 0 and c != 1
        told(result, total, norm, c, scale)
        for x, y in zip(before, g):
            near(y, c * x, "fp32", np.abs(c * x) * 2.0 ** -24 * (1 + 1e-6), which)
        intact(b, g)


@pytest.mark.parametrize("which", ["tiny", "ragged", "many", "large"])
def test_some_outputs_in_the_place_of_their_gradients(pkg, which):
    sizes = SIZES[which]
    types = types_of("mixed", sizes)
    g, b = make(sizes, types, 91, 1)
    other, ob = make(sizes, ["fp32"] * len(sizes), 92, 2)
    own = [t == "fp32" and i % 2 == 0 for i, t in enumerate(types)]
    out = [x if mine else o for x, o, mine in zip(g, other, own)]
    before = [f64(t) for t in g]
    norm = math.sqrt(squares(g))
    result = pkg.hp_cuda_grad_result()
    pkg.hp_cuda_grad_clip(g, sizes, out, 0.3 * norm, result)
    c = coefficient(norm, 0.3 * norm)
    for x, o, y, mine in zip(before, out, g, own):
        near(o, c * x, "fp32", np.abs(c * x) * 2.0 ** -24 * (1 + 1e-6), which)
        assert mine or np.array_equal(f64(y), x)
    # Nesterov's direction likewise
    u, ub = make(sizes, ["fp32"] * len(sizes), 93, 3)
    u0, before = [f64(t) for t in u], [f64(t) for t in g]
    pkg.hp_cuda_gd_momentum(g, sizes, u, out, 0.9, 1.0, None, scale=-0.25)
    for x, v, y, d in zip(before, u0, u, out):
        near_momentum(y, d, x, v, 0.9, -0.25)
    for bs, ts in ((b, g), (ob, other), (ub, u)):
        intact(bs, ts)


@pytest.mark.parametrize("measured", [0, 1])
@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16", "mixed"])
@pytest.mark.parametrize("which", list(SIZES))
def test_unscaling_in_place(pkg, which, kind, measured):
    sizes = SIZES[which]
    types = types_of(kind, sizes)
    for share, scale, lead in ((2.0, 2.0 ** -10, 0), (0.3, -0.375, 1), (2.0, 3.0, 5)):
        g, b = make(sizes, types, 94, lead)
        before = [f64(t) for t in g]
        total = squares(g)
        norm = math.sqrt(total)
        result = pkg.hp_cuda_grad_result()
        if measured:
            result[0] = total
        pkg.hp_cuda_grad_clip(g, sizes, None, share * abs(scale) * norm, result, measured, scale=scale)
        c = coefficient(norm, share * abs(scale) * norm, scale)
        told(result, total, norm, c, scale)
        for x, t, y in zip(before, types, g):
            near(y, c * x, t, np.abs(c * x) * 2.0 ** -23, (which, kind))
        intact(b, g)


def test_masks_by_messages_of_the_sparsifier_without_residual(pkg, capi, oracle_cpu):
    # hpx_dgc_encode clears what it sends in the tensor that it is given: here a copy of the momentum
    sizes, seeds = [1000, 65_536, 100_003, 33], [3, 1 << 22, 12_345 << 20, 5]
    rates, shares = [0.05, 0.5, 0.01, 1.0], [0.01, 0.5, 0.001, 0.1]
    u, b = make(sizes, ["fp32"] * len(sizes), 95, 1)
    before = [t.clone() for t in u]
    sent = [t.clone() for t in u]
    rooms = [4 + 8 * math.ceil(n * s) for n, s in zip(sizes, shares)]
    msgs = [torch.full((r,), 0xEE, dtype=torch.uint8, device="cuda") for r in rooms]
    counts = torch.zeros(len(sizes), dtype=torch.int32, device="cuda")
    rc = capi.load().hpx_dgc_encode(len(sizes), capi.ptr_array([t.data_ptr() for t in sent]), capi.i32_array(sizes),
                                    capi.ptr_array([m.data_ptr() for m in msgs]), capi.f64_array(rates), capi.f64_array(shares),
                                    capi.u64_array(seeds), stream_ptr())
    assert rc == 0, capi.last_error()
    pkg.hp_cuda_gd_mask(msgs, rooms, u, sizes, counts)
    for i, n in enumerate(sizes):
        ref, _ = oracle_cpu.dgc_encode(before[i].cpu().numpy(), rates[i], shares[i], seeds[i])
        k = (ref.size - 4) // 8
        assert counts[i].item() == k and (k > 0) == (i > 0)  # the first tensor's samples hold its largest value: nothing lies beyond them
        want = f64(before[i])
        want[ref[4:4 + 4 * k].view(np.int32)] = 0
        assert np.array_equal(f64(u[i]), want)
    intact(b, u)


@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16", "mixed"])
@pytest.mark.parametrize("sizes", [[1], [2048], [1, 3, 7, 0, 9, 1023, 1024, 1025], [33, 16_385, 5000], [49_152], [49_153], [1000] * 48, [1000] * 49])
def test_sum_of_a_clip_that_measures(pkg, sizes, kind):
    # the lists of up to 48 tiles and the shortest beyond: the same bits at every address, in place and not, and but for the order
    # of additions hp_cuda_grad_norm's
    types, n = types_of(kind, sizes), sum(sizes)
    seen, most = set(), set()
    for lead in (0, 1, 3, 64):
        g, _ = make(sizes, types, 96, lead)
        out, _ = make(sizes, ["fp32"] * len(sizes), 97, lead + 1)
        norm, result = pkg.hp_cuda_grad_result(), pkg.hp_cuda_grad_result()
        pkg.hp_cuda_grad_norm(g, sizes, norm)
        pkg.hp_cuda_grad_clip(g, sizes, out, 0.01, result)
        seen.add((norm[0].item(), *result[:3].tolist()))
        pkg.hp_cuda_grad_clip(g, sizes, out, 0.01, result, order=0)
        pkg.hp_cuda_grad_norm(g, sizes, norm, 0)
        most.add((norm[0].item(), *result[:2].tolist()))
        pkg.hp_cuda_grad_clip(g, sizes, None, 0.01, result)
        seen.add((seen.copy().pop()[0], *result[:3].tolist()))
    assert len(seen) == 1 and len(most) == 1
    (of_norm, of_clip, length, c), = seen
    assert abs(of_clip - of_norm) <= 2 * n * 2.0 ** -53 * of_norm
    # the root, the divisor, the quotient and the rounding to fp32
    assert abs(c - coefficient(math.sqrt(of_clip), 0.01)) <= abs(c) * 2.0 ** -24 * (1 + 1e-6)
    (a, b, length), = most
    assert a == b == length


@pytest.mark.parametrize("which", ["tiny", "many", "large"])
def test_every_call_captured(pkg, which):
    # short lists, several tables, long lists; replayed four times with other gradients each, eager work between
    sizes = SIZES[which]
    types = types_of("mixed", sizes)
    side = torch.cuda.Stream()

    def fresh(seed):
        return make(sizes, types, seed)[0], [make(sizes, ["fp32"] * len(sizes), seed + k)[0] for k in (1, 2, 3)]

    index = [list(range(0, n, 3))[:50] for n in sizes]
    msgs = [message(i) for i in index]
    rooms = [m.numel() for m in msgs]
    counts = torch.zeros(len(sizes), dtype=torch.int32, device="cuda")

    def calls(g, out, u, d, results):
        pkg.hp_cuda_grad_clip(g, sizes, out, 0.02, results[0], scale=0.5)
        pkg.hp_cuda_grad_norm(g, sizes, results[1])
        pkg.hp_cuda_grad_norm(out, sizes, results[1], is_add_to=1)
        pkg.hp_cuda_gd_momentum(g, sizes, u, d, 0.9, 0.02, results[1])
        pkg.hp_cuda_gd_mask(msgs, rooms, u, sizes, counts)
        pkg.hp_cuda_grad_clip(g, sizes, None, 0.01, results[1], is_measured=1)
        pkg.hp_cuda_grad_clip(g, sizes, None, math.inf, results[2], scale=-0.5)

    g, (out, u, d) = fresh(200)
    results = [pkg.hp_cuda_grad_result() for _ in range(3)]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            calls(g, out, u, d, results)
    held = [*g, *out, *u, *d]
    for rep in range(4):
        g2, (out2, u2, d2) = fresh(210 + 10 * rep)
        eager = [pkg.hp_cuda_grad_result() for _ in range(3)]
        for a, b in zip(held, [*g2, *out2, *u2, *d2]):
            a.copy_(b)
        calls(g2, out2, u2, d2, eager)
        counts.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, [*g2, *out2, *u2, *d2])), rep
        assert all(torch.equal(a[:3], b[:3]) for a, b in zip(results, eager)) and results[2][2].item() == -0.5
        assert counts.tolist() == [len(i) for i in index]
        assert math.isfinite(float(torch.randn(1 << 20, device="cuda").sum()))
