"""The gradient operators around the codecs against their definitions in 64 bits.

Tolerances.  A square of an fp32 value is exact in fp64, and n of them added in any order are off by at most (n - 1) 2^-53 of the
sum.  The coefficient is rounded to fp32 once (2^-24 of it), the product with it once more, a result in 16 bits a third time
(2^-8 in bf16, 2^-11 in fp16); results below the type's normal range are off by half of its smallest value instead.  In the
momentum the product c g is off by two roundings and the sum by one."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
HALF = {"fp32": 2.0 ** -24, "bf16": 2.0 ** -8, "fp16": 2.0 ** -11}        # a rounding, relative
LEAST = {"fp32": 2.0 ** -149, "bf16": 2.0 ** -133, "fp16": 2.0 ** -24}    # the smallest value
GUARD = 64


def make(sizes, types, seed=0, lead=0, sigma=1e-2):
    """Gradients of the sizes and types, `lead` elements behind a 256-byte boundary, each within a buffer of its own that has
    GUARD elements of a known value on both sides; (views, buffers)."""
    gen = torch.Generator().manual_seed(seed)
    views, buffers = [], []
    for n, t in zip(sizes, types):
        x = torch.full((2 * GUARD + lead + n,), 77.0, dtype=TYPES[t])
        x[GUARD + lead:GUARD + lead + n] = (torch.randn(n, generator=gen) * sigma).to(TYPES[t])
        x = x.cuda()
        buffers.append(x)
        views.append(x[GUARD + lead:GUARD + lead + n])
    return views, buffers


def intact(buffers, views):
    for b, v in zip(buffers, views):
        at = v.storage_offset()
        assert bool((b[:at] == 77).all()) and bool((b[at + v.numel():] == 77).all())


def f64(t):
    return t.detach().cpu().to(torch.float64).numpy()


def squares(ts):
    return math.fsum(float(x) for t in ts for x in np.square(f64(t)))


def coefficient(norm, max_norm, scale=1.0):
    return scale * min(1.0, max_norm / (abs(scale) * norm + 1e-6))


def near(got, want, type_, extra=0.0, what=""):
    """got (a tensor of type_) against want in fp64; extra: an absolute bound beside the rounding to the type."""
    tol = np.abs(want) * (HALF[type_] * (1 + 2.0 ** -20)) + LEAST[type_] / 2 + extra
    off = np.abs(f64(got) - want)
    assert bool((off <= tol).all()), (what, float((off / tol).max()), int(np.argmax(off / tol)))


SIZES = {
    "one": [1],
    "tiny": [1, 3, 7, 8, 9, 0, 15, 16, 17],
    "edges": [2047, 4095, 4096, 4097, 8191, 8192, 8193, 0],
    "ragged": [100_003, 5, 16_385, 65_537],
    "many": [1 + (i * 37) % 900 for i in range(1000)],   # several tables
    "large": [3_000_017, 1_000_001],
}


def types_of(kind, sizes):
    return [("fp32", "bf16", "fp16")[i % 3] if kind == "mixed" else kind for i in range(len(sizes))]


@pytest.mark.parametrize("lead", [0, 1, 5])
@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16", "mixed"])
@pytest.mark.parametrize("which", list(SIZES))
def test_norm(pkg, which, kind, lead):
    sizes = SIZES[which]
    g, _ = make(sizes, types_of(kind, sizes), 1, lead)
    result = pkg.hp_cuda_grad_result()
    want, n = squares(g), sum(sizes)
    pkg.hp_cuda_grad_norm(g, sizes, result)
    s, norm = result[:2].tolist()
    assert abs(s - want) <= n * 2.0 ** -53 * want
    assert abs(norm - math.sqrt(want)) <= (n + 2) * 2.0 ** -53 * math.sqrt(want)
    again = pkg.hp_cuda_grad_result()
    pkg.hp_cuda_grad_norm(g, sizes, again)
    assert again[0].item() == s  # the same bits every time
    pkg.hp_cuda_grad_norm(g, sizes, result, 0)
    most = max(float(np.abs(f64(t)).max()) for t in g if t.numel())
    assert result[:2].tolist() == [most, most]
    assert result[3:16].tolist() == [0.0] * 13  # the count of arrivals is back at zero


@pytest.mark.parametrize("full", [8, 48, 256, 320, 448])
@pytest.mark.parametrize("n", [3, 2000])
def test_empty_tensors_behind_a_full_table(pkg, full, n):
    sizes = [n] * full + [0, 0]
    g, b = make(sizes, types_of("mixed", sizes), 80, 1)
    before = [f64(t) for t in g]
    want = squares(g)
    norm = math.sqrt(want)
    c = coefficient(norm, 0.5 * norm)
    result = pkg.hp_cuda_grad_result()
    pkg.hp_cuda_grad_norm(g, sizes, result)
    assert abs(result[0].item() - want) <= sum(sizes) * 2.0 ** -53 * want
    out, _ = make(sizes, ["fp32"] * len(sizes), 81)
    u, _ = make(sizes, ["fp32"] * len(sizes), 82)
    u0 = [f64(t) for t in u]
    pkg.hp_cuda_grad_clip(g, sizes, out, 0.5 * norm, result)
    pkg.hp_cuda_gd_momentum(g, sizes, u, None, 0.9, 0.5 * norm, result)
    for x, o, v, y in zip(before, out, u0, u):
        near(o, c * x, "fp32", np.abs(c * x) * 2.0 ** -24 * (1 + 1e-6))
        near_momentum(y, None, x, v, 0.9, c)
    pkg.hp_cuda_grad_clip(g, sizes, None, 0.5 * norm, result)
    assert abs(result[0].item() - want) <= sum(sizes) * 2.0 ** -53 * want
    assert abs(result[1].item() / norm - 1) <= 1e-9 and abs(result[2].item() - c) <= c * 2.0 ** -24 * (1 + 1e-6)
    intact(b, g)


def test_norm_of_several_lists(pkg):
    sizes = [70_001, 33, 4096]
    lists = [make(sizes, [t] * 3, seed)[0] for seed, t in enumerate(("fp32", "bf16", "fp16"))]
    result = pkg.hp_cuda_grad_result()
    for i, g in enumerate(lists):
        pkg.hp_cuda_grad_norm(g, sizes, result, is_add_to=int(i > 0))
    want = squares([t for g in lists for t in g])
    assert abs(result[0].item() - want) <= 3 * sum(sizes) * 2.0 ** -53 * want
    for i, g in enumerate(lists):
        pkg.hp_cuda_grad_norm(g, sizes, result, 0, int(i > 0))
    assert result[0].item() == max(float(np.abs(f64(t)).max()) for g in lists for t in g)


def test_norm_of_two_tables_the_second_with_more_tiles(pkg):
    # 448 small tensors fill the first table; the second has more workgroups than the first
    sizes = [1 + i % 7 for i in range(448)] + [9_000_001, 8_000_003]
    g, _ = make(sizes, types_of("fp32", sizes), 50, 1)
    g[449] = g[449].bfloat16()
    want = float(sum(np.square(f64(t)).sum() for t in g))
    for _ in range(2):
        result = pkg.hp_cuda_grad_result()
        result[16:528] = float("nan")  # slots that no call has written yet may hold anything
        pkg.hp_cuda_grad_norm(g, sizes, result)
        assert abs(result[0].item() - want) <= sum(sizes) * 2.0 ** -53 * want
        pkg.hp_cuda_grad_norm(g, sizes, result, 0)
        assert result[0].item() == max(float(np.abs(f64(t)).max()) for t in g)


@pytest.mark.parametrize("kind", ["fp32", "bf16", "mixed"])
@pytest.mark.parametrize("which", ["tiny", "edges", "ragged", "many", "large"])
def test_norm_has_the_same_bits_at_other_addresses(pkg, which, kind):
    sizes = SIZES[which]
    seen = set()
    for lead in (0, 1, 3, 64):
        g, _ = make(sizes, types_of(kind, sizes), 51, lead)
        result = pkg.hp_cuda_grad_result()
        pkg.hp_cuda_grad_norm(g, sizes, result)
        seen.add((result[0].item(), result[1].item()))
    assert len(seen) == 1


def test_norm_of_nothing(pkg):
    result = pkg.hp_cuda_grad_result().fill_(0)
    for g, sizes in (([], []), ([torch.zeros(0, device="cuda")], [0])):
        result[:3] = 5.0
        pkg.hp_cuda_grad_norm(g, sizes, result)
        assert result[:2].tolist() == [0.0, 0.0]
        result[0] = 9.0
        pkg.hp_cuda_grad_norm(g, sizes, result, is_add_to=1)
        assert result[:2].tolist() == [9.0, 3.0]
        pkg.hp_cuda_grad_clip(g, sizes, None, 1.0, result)
        assert result[:3].tolist() == [0.0, 0.0, 1.0]


@pytest.mark.parametrize("value", [1e30, 3e38, 1e-30, 1e-44])
def test_norm_of_extreme_values(pkg, value):
    # their squares are outside fp32's range
    x = torch.full((10_007,), value, device="cuda")
    result = pkg.hp_cuda_grad_result()
    pkg.hp_cuda_grad_norm([x], [x.numel()], result)
    v = float(np.float32(value))
    assert abs(result[0].item() / (x.numel() * v * v) - 1) <= x.numel() * 2.0 ** -53


@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_values_that_are_not_finite(pkg, kind, bad):
    sizes = [4097, 20_000]
    g, b = make(sizes, [kind] * 2, 4, 1)
    g[1][12_345] = bad
    result = pkg.hp_cuda_grad_result()
    for order in (2, 0):
        pkg.hp_cuda_grad_norm(g, sizes, result, order)
        got = result[1].item()
        assert math.isnan(got) if math.isnan(bad) else got == math.inf
        outs = [torch.full((n,), 5.0, device="cuda") for n in sizes]
        pkg.hp_cuda_grad_clip(g, sizes, outs, math.inf, result, 0, order)
        assert result[2].item() == 0.0
        for o in outs:
            assert bool((o == 0).all())
        u = [torch.ones(n, device="cuda") for n in sizes]
        pkg.hp_cuda_gd_momentum(g, sizes, u, outs, 0.5, 1.0, result, order)
        assert all(bool((x == 0.5).all()) for x in u) and all(bool((x == 0.25).all()) for x in outs)
    pkg.hp_cuda_grad_clip(g, sizes, None, 1.0, result)
    assert all(bool((x == 0).all()) for x in g)
    intact(b, g)


@pytest.mark.parametrize("lead, out_lead", [(0, 0), (1, 0), (3, 1), (0, 2)])
@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16", "mixed"])
@pytest.mark.parametrize("which", list(SIZES))
def test_clip(pkg, which, kind, lead, out_lead):
    sizes = SIZES[which]
    types = types_of(kind, sizes)
    g, b = make(sizes, types, 2, lead)
    before = [f64(t) for t in g]
    norm = math.sqrt(squares(g))
    for max_norm, scale in ((0.25 * norm, 1.0), (1e9, 1.0), (0.1 * norm, -0.5), (math.inf, 3.0)):
        out, ob = make(sizes, ["fp32"] * len(sizes), 3, out_lead)
        result = pkg.hp_cuda_grad_result()
        pkg.hp_cuda_grad_clip(g, sizes, out, max_norm, result, scale=scale)
        c = coefficient(norm, max_norm, scale)
        assert abs(result[1].item() / (abs(scale) * norm) - 1) <= 1e-9
        assert abs(result[2].item() - c) <= abs(c) * 2.0 ** -24 * (1 + 1e-6)
        for x, o in zip(before, out):
            near(o, c * x, "fp32", np.abs(c * x) * 2.0 ** -24 * (1 + 1e-6), (which, kind))
        intact(ob, out)
        intact(b, g)
    assert all(np.array_equal(x, f64(t)) for x, t in zip(before, g))  # gradients are only read
    # in place, each in its own type
    result = pkg.hp_cuda_grad_result()
    pkg.hp_cuda_grad_clip(g, sizes, None, 0.25 * norm, result)
    c = coefficient(norm, 0.25 * norm)
    for x, t, y in zip(before, types, g):
        near(y, c * x, t, np.abs(c * x) * 2.0 ** -23, (which, kind))
    intact(b, g)
    # fp32 outputs that are the gradients themselves
    if kind == "fp32":
        now = [f64(t) for t in g]
        pkg.hp_cuda_grad_clip(g, sizes, g, 0.0, result)
        assert all(bool((t == 0).all()) for t in g) and result[2].item() == 0.0
        del now


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_lists_of_many_tiles(pkg, kind):
    # more tiles than workgroups in every pass; beyond 96 MiB for fp32, where loads stream
    sizes = [20_000_003, 70_001, 5, 6_000_000]
    types = [kind, "fp32", kind, kind]
    g, b = make(sizes, types, 40, 1)
    before = [f64(t) for t in g]
    want = float(sum(np.square(x).sum() for x in before))
    norm, n = math.sqrt(want), sum(sizes)
    result = pkg.hp_cuda_grad_result()
    pkg.hp_cuda_grad_norm(g, sizes, result)
    assert abs(result[0].item() - want) <= n * 2.0 ** -53 * want
    measured = result[0].item()
    out, ob = make(sizes, ["fp32"] * 4, 41, 3)
    pkg.hp_cuda_grad_clip(g, sizes, out, 0.3 * norm, result)
    assert result[0].item() == measured  # the same order of additions, whoever joins the partial sums
    c = coefficient(norm, 0.3 * norm)
    for x, o in zip(before, out):
        near(o, c * x, "fp32", np.abs(c * x) * 2.0 ** -24 * (1 + 1e-6))
    intact(ob, out)
    for nesterov in (False, True):
        u, ub = make(sizes, ["fp32"] * 4, 42, 2)
        u0 = [f64(t) for t in u]
        pkg.hp_cuda_gd_momentum(g, sizes, u, out if nesterov else None, 0.9, 0.3 * norm, result)
        for x, v, y, z in zip(before, u0, u, out):
            near_momentum(y, z if nesterov else None, x, v, 0.9, c)
        intact(ub, u)
        intact(ob, out)
    pkg.hp_cuda_grad_clip(g, sizes, None, 2 * norm, result)
    assert result[2].item() == 1.0 and all(np.array_equal(x, f64(t)) for x, t in zip(before, g))
    pkg.hp_cuda_grad_clip(g, sizes, None, 0.3 * norm, result)
    for x, t, y in zip(before, types, g):
        near(y, c * x, t, np.abs(c * x) * 2.0 ** -23)
    intact(b, g)


def test_clip_leaves_what_is_short_enough(pkg):
    g, b = make([5000, 17], ["bf16", "fp32"], 5)
    bits = [t.clone() for t in b]
    result = pkg.hp_cuda_grad_result()
    pkg.hp_cuda_grad_clip(g, [5000, 17], None, 1e6, result)
    assert result[2].item() == 1.0
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(bits, b))


@pytest.mark.parametrize("kind", ["fp32", "bf16", "mixed"])
@pytest.mark.parametrize("which", ["tiny", "ragged", "many", "large"])
def test_clip_by_the_largest_magnitude(pkg, which, kind):
    sizes = SIZES[which]
    types = types_of(kind, sizes)
    g, b = make(sizes, types, 70, 1)
    before = [f64(t) for t in g]
    most = max(float(np.abs(x).max()) for x in before if x.size)
    result = pkg.hp_cuda_grad_result()
    out, ob = make(sizes, ["fp32"] * len(sizes), 71, 2)
    c = coefficient(most, 0.5 * most)
    pkg.hp_cuda_grad_clip(g, sizes, out, 0.5 * most, result, order=0)
    assert result[:2].tolist() == [most, most] and abs(result[2].item() - c) <= c * 2.0 ** -24 * (1 + 1e-6)
    u, _ = make(sizes, ["fp32"] * len(sizes), 72)
    u0 = [f64(t) for t in u]
    pkg.hp_cuda_gd_momentum(g, sizes, u, None, 0.9, 0.5 * most, result, 0)
    for x, v, o, y in zip(before, u0, out, u):
        near(o, c * x, "fp32", np.abs(c * x) * 2.0 ** -24 * (1 + 1e-6))
        near_momentum(y, None, x, v, 0.9, c)
    pkg.hp_cuda_grad_clip(g, sizes, None, 0.5 * most, result, order=0)
    for x, t, y in zip(before, types, g):
        near(y, c * x, t, np.abs(c * x) * 2.0 ** -23)
    intact(b, g)
    intact(ob, out)


@pytest.mark.parametrize("order", [2, 0])
def test_clip_by_a_norm_over_ranks(pkg, order):
    # what an all-reduce leaves in result[0]
    sizes = [9001, 300]
    g, _ = make(sizes, ["bf16", "fp32"], 6)
    before = [f64(t) for t in g]
    result = pkg.hp_cuda_grad_result()
    pkg.hp_cuda_grad_norm(g, sizes, result, order)
    result[0] *= 16
    s = result[0].item()
    norm = math.sqrt(s) if order == 2 else s
    out = [torch.zeros(n, device="cuda") for n in sizes]
    pkg.hp_cuda_grad_clip(g, sizes, out, 0.5 * norm, result, 1, order)
    c = coefficient(norm, 0.5 * norm)
    assert result[0].item() == s and abs(result[1].item() / norm - 1) < 1e-14
    for x, o in zip(before, out):
        near(o, c * x, "fp32", np.abs(c * x) * 2.0 ** -24 * (1 + 1e-6))


def near_momentum(got_u, got_d, g, u, m, c):
    m = float(np.float32(m))
    cg = np.abs(c * g) * (2.0 ** -23 * (1 + 1e-6)) + 2.0 ** -149
    want = m * u + c * g
    near(got_u, want, "fp32", cg)
    if got_d is not None:
        near(got_d, m * want + c * g, "fp32", cg + abs(m) * (cg + np.abs(want) * 2.0 ** -24 + 2.0 ** -149))


@pytest.mark.parametrize("lead, u_lead, d_lead", [(0, 0, 0), (1, 2, 3), (0, 1, 0)])
@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16", "mixed"])
@pytest.mark.parametrize("which", list(SIZES))
def test_momentum(pkg, which, kind, lead, u_lead, d_lead):
    sizes = SIZES[which]
    g, _ = make(sizes, types_of(kind, sizes), 7, lead)
    before = [f64(t) for t in g]
    norm = math.sqrt(squares(g))
    for nesterov in (False, True):
        u, ub = make(sizes, ["fp32"] * len(sizes), 8, u_lead)
        d, db = make(sizes, ["fp32"] * len(sizes), 9, d_lead)
        u0 = [f64(t) for t in u]
        result = pkg.hp_cuda_grad_result()
        pkg.hp_cuda_grad_norm(g, sizes, result)
        pkg.hp_cuda_gd_momentum(g, sizes, u, d if nesterov else None, 0.9, 0.25 * norm, result)
        c = coefficient(norm, 0.25 * norm)
        assert abs(result[2].item() - c) <= c * 2.0 ** -24 * (1 + 1e-6)
        for x, v, y, z in zip(before, u0, u, d):
            near_momentum(y, z if nesterov else None, x, v, 0.9, c)
        intact(ub, u)
        intact(db, d)
    assert all(np.array_equal(x, f64(t)) for x, t in zip(before, g))
    # without a norm, the direction in the place of fp32 gradients
    if kind == "fp32":
        u, _ = make(sizes, ["fp32"] * len(sizes), 10, u_lead)
        u0 = [f64(t) for t in u]
        pkg.hp_cuda_gd_momentum(g, sizes, u, g, 0.5, 1.0, None, scale=0.125)
        for x, v, y, z in zip(before, u0, u, g):
            near_momentum(y, z, x, v, 0.5, 0.125)


def message(indices, room=None, header=None):
    k = len(indices)
    words = np.zeros((1 + 2 * k) if room is None else room, np.int32)
    words[0] = 4 + 8 * k if header is None else header
    words[1:1 + k] = indices
    words[1 + k:1 + 2 * k] = 1 << 20  # the values: no index of a small tensor
    return torch.from_numpy(words).cuda().view(torch.uint8)


@pytest.mark.parametrize("ks, ns", [([1], [1]), ([0, 1, 255, 256, 257], [10, 10, 300, 5000, 4096]), ([7] * 700, [50] * 700), ([20_000], [1_000_003])])
def test_mask(pkg, ks, ns):
    rng = np.random.default_rng(11)
    index = [rng.permutation(n)[:k].astype(np.int32) for k, n in zip(ks, ns)]
    msgs = [message(i) for i in index]
    u, b = make(ns, ["fp32"] * len(ns), 12, 1)
    want = [f64(t) for t in u]
    counts = torch.full((len(ks),), 99, dtype=torch.int32, device="cuda")
    pkg.hp_cuda_gd_mask(msgs, [m.numel() for m in msgs], u, ns, counts)
    assert counts.tolist() == ks
    for w, i, t in zip(want, index, u):
        w[i] = 0
        assert np.array_equal(w, f64(t))
    intact(b, u)


def test_mask_of_bad_messages(pkg):
    n = 100
    cases = [  # message, its room in bytes, entries told, indices cleared
        (message([3, 5], room=9), 36, 2, [3, 5]),             # a message shorter than its room
        (message([3, 5, 7], header=4 + 8 * 4), 28, -1, []),   # longer than its room
        (message([3, 5], header=-12), 20, -1, []),
        (message([3, 5], header=0), 20, -1, []),
        (message([3, 5], header=19), 20, -1, []),
        (message([3, 5], header=12), 20, 1, [3]),
        (message([-1, 100, 99, 1 << 30]), 36, 4, [99]),       # indices outside the tensor
        (message([4, 4, 4]), 28, 3, [4]),                     # the same index more than once
        (message([3]), 11, -1, []),                           # no room for one entry
        (message([3]), 3, -1, []),
        (message([3]), 0, -1, []),
    ]
    u = [torch.ones(n, device="cuda") for _ in cases]
    counts = torch.zeros(len(cases), dtype=torch.int32, device="cuda")
    pkg.hp_cuda_gd_mask([c[0] for c in cases], [c[1] for c in cases], u, [n] * len(cases), counts)
    assert counts.tolist() == [c[2] for c in cases]
    for (_, _, _, gone), t in zip(cases, u):
        want = np.ones(n)
        want[gone] = 0
        assert np.array_equal(want, f64(t))
    pkg.hp_cuda_gd_mask([cases[0][0]], [36], [torch.zeros(0, device="cuda")], [0])  # an empty tensor


@pytest.mark.parametrize("nesterov", [False, True])
def test_a_worker_step_of_the_sparsifier(pkg, oracle_cpu, nesterov):
    # norm of two lists, the ranks' sums, momentum correction, sparsifier with its residual, masks: four steps of two ranks
    sizes, types = [200_003, 5000, 65_536], ["bf16", "fp32", "fp16"]
    rate, drop, m = 0.05, 0.99, 0.9
    rooms = [4 + 8 * math.ceil(n * (1 - drop)) for n in sizes]
    ranks = [{"u": [torch.zeros(n, device="cuda") for n in sizes], "d": [torch.zeros(n, device="cuda") for n in sizes],
              "r": [torch.zeros(n, device="cuda") for n in sizes], "result": pkg.hp_cuda_grad_result()} for _ in range(2)]
    for step in range(4):
        sums = []
        for k, rank in enumerate(ranks):
            rank["g"], _ = make(sizes, types, 100 + 10 * step + k)
            pkg.hp_cuda_grad_norm(rank["g"][:2], sizes[:2], rank["result"])
            pkg.hp_cuda_grad_norm(rank["g"][2:], sizes[2:], rank["result"], is_add_to=1)
            sums.append(rank["result"][0].clone())
        total = sums[0] + sums[1]
        norm = math.sqrt(squares([t for rank in ranks for t in rank["g"]]))
        assert abs(total.sqrt().item() / norm - 1) < 1e-9
        for rank in ranks:
            rank["result"][0] = total
            u0, r0 = [f64(t) for t in rank["u"]], [t.cpu().numpy() for t in rank["r"]]
            pkg.hp_cuda_gd_momentum(rank["g"], sizes, rank["u"], rank["d"] if nesterov else None, m, 0.5 * norm, rank["result"])
            c = coefficient(norm, 0.5 * norm)
            for g, u, v, d in zip(rank["g"], u0, rank["u"], rank["d"]):
                near_momentum(v, d if nesterov else None, f64(g), u, m, c)
            sent = rank["d"] if nesterov else rank["u"]
            msgs = [torch.zeros(b, dtype=torch.uint8, device="cuda") for b in rooms]
            seeds = [7 + step, 8, 9]
            fed = [t.cpu().numpy() for t in sent]
            assert pkg.hp_cuda_gd(sent, sizes, rank["r"], sizes, msgs, [rate] * 3, [drop] * 3, seeds=seeds) == 0
            counts = torch.zeros(3, dtype=torch.int32, device="cuda")
            u1 = [f64(t) for t in rank["u"]]
            pkg.hp_cuda_gd_mask(msgs, rooms, rank["u"], sizes, counts)
            for i in range(3):
                ref, _ = oracle_cpu.gd_encode(fed[i], r0[i], rate, drop, seeds[i])
                assert np.array_equal(msgs[i].cpu().numpy()[:ref.size], ref)
                assert np.array_equal(rank["r"][i].cpu().numpy().view(np.uint32), r0[i].view(np.uint32))
                k = (ref.size - 4) // 8
                index = ref[4:4 + 4 * k].view(np.int32)
                assert counts[i].item() == k > 0
                u1[i][index] = 0
                assert np.array_equal(u1[i], f64(rank["u"][i]))


def test_clipped_gradients_through_a_codec(pkg, oracle_cpu):
    # bf16 gradients, clipped into what the threshold codec encodes
    sizes = [70_001, 300]
    g, _ = make(sizes, ["bf16", "bf16"], 20)
    out = [torch.zeros(n, device="cuda") for n in sizes]
    r = [torch.zeros(n, device="cuda") for n in sizes]
    packed = [torch.zeros((n + 3) // 4, dtype=torch.uint8, device="cuda") for n in sizes]
    result = pkg.hp_cuda_grad_result()
    pkg.hp_cuda_grad_clip(g, sizes, out, 1.0, result)
    assert pkg.hp_cuda_tbq(out, sizes, r, sizes, packed, None, [1e-3] * 2) == 0
    for o, p, n in zip(out, packed, sizes):
        assert np.array_equal(p.cpu().numpy(), oracle_cpu.tbq_encode(o.cpu().numpy(), np.zeros(n, np.float32), 1e-3))


def test_raw_addresses_and_streams(pkg):
    sizes, types = [4099, 1000], ["bf16", "fp32"]
    g, _ = make(sizes, types, 21, 1)
    want = squares(g)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for stream in (side, side.cuda_stream, None):
        result = pkg.hp_cuda_grad_result()
        torch.cuda.synchronize()
        pkg.hp_cuda_grad_norm([t.data_ptr() for t in g], np.array(sizes), result.data_ptr(), types=[TYPES[t] for t in types], stream=stream)
        torch.cuda.synchronize()
        assert abs(result[0].item() - want) <= sum(sizes) * 2.0 ** -53 * want


def test_refused_tensors(pkg):
    x, r = torch.zeros(64, device="cuda"), pkg.hp_cuda_grad_result()
    b = torch.zeros(20, dtype=torch.uint8, device="cuda")
    with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
        pkg.hp_cuda_grad_norm([x.cpu()], [64], r)
    with pytest.raises(RuntimeError, match="contiguous"):
        pkg.hp_cuda_grad_norm([x[::2]], [32], r)
    with pytest.raises(ValueError, match="64 elements, 65"):
        pkg.hp_cuda_grad_norm([x], [65], r)
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        pkg.hp_cuda_grad_norm([x.double()], [64], r)
    with pytest.raises(TypeError, match="not of the type"):
        pkg.hp_cuda_grad_norm([x], [64], r, types=[torch.bfloat16])
    with pytest.raises(TypeError, match="Double"):
        pkg.hp_cuda_grad_norm([x], [64], r.float())
    with pytest.raises(ValueError, match="2064"):
        pkg.hp_cuda_grad_norm([x], [64], r[:16])
    with pytest.raises(ValueError, match="order 1"):
        pkg.hp_cuda_grad_norm([x], [64], r, 1)
    with pytest.raises(TypeError, match="Float"):
        pkg.hp_cuda_grad_clip([x], [64], [x.bfloat16()], 1.0, r)
    with pytest.raises(ValueError, match="an output"):
        pkg.hp_cuda_grad_clip([x], [64], [torch.zeros(63, device="cuda")], 1.0, r)
    with pytest.raises(ValueError, match="an output"):
        pkg.hp_cuda_grad_clip([x, x], [64, 64], [torch.zeros(64, device="cuda")], 1.0, r)
    with pytest.raises(ValueError, match="overlap"):
        pkg.hp_cuda_grad_clip([x, x], [64, 64], None, 1.0, r)
    with pytest.raises(ValueError, match="max_norm"):
        pkg.hp_cuda_grad_clip([x], [64], None, -1.0, r)
    with pytest.raises(ValueError, match="a momentum"):
        pkg.hp_cuda_gd_momentum([x], [64], [torch.zeros(8, device="cuda")], None, 0.9, 1.0, r)
    with pytest.raises(ValueError, match="overlap"):
        pkg.hp_cuda_gd_momentum([x], [64], [x], None, 0.9, 1.0, r)
    with pytest.raises(TypeError, match="Byte"):
        pkg.hp_cuda_gd_mask([x], [20], [x], [64])
    with pytest.raises(ValueError, match="a message"):
        pkg.hp_cuda_gd_mask([b], [21], [x], [64])
    with pytest.raises(ValueError, match="the counts"):
        pkg.hp_cuda_gd_mask([b, b], [20, 20], [x, x], [64, 64], torch.zeros(1, dtype=torch.int32, device="cuda"))


def test_two_graphs_of_one_stream(pkg):
    # both captured on the same stream, replayed at the same time on two others, with eager calls of the same operators between
    sizes, types = [300_001, 17, 4096], ["bf16", "fp32", "fp16"]
    side, others = torch.cuda.Stream(), [torch.cuda.Stream(), torch.cuda.Stream()]
    sets = []
    for k in range(2):
        g, _ = make(sizes, types, 30 + k)
        s = {"g": g, "u": [torch.zeros(n, device="cuda") for n in sizes], "out": [torch.zeros(n, device="cuda") for n in sizes],
             "result": pkg.hp_cuda_grad_result(), "msg": message([1, 5, 16]), "graph": torch.cuda.CUDAGraph()}
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            with torch.cuda.graph(s["graph"], stream=side):
                pkg.hp_cuda_grad_clip(s["g"], sizes, s["out"], 0.5, s["result"])
                pkg.hp_cuda_gd_momentum(s["g"], sizes, s["u"], None, 0.5, 0.5, s["result"])
                pkg.hp_cuda_gd_mask([s["msg"]], [28], s["u"][1:2], [17])
        sets.append(s)
    for rep in range(4):
        wants = []
        for k, s in enumerate(sets):
            fresh, _ = make(sizes, types, 1000 + 10 * rep + k, sigma=10.0 ** -rep)
            for a, b in zip(s["g"], fresh):
                a.copy_(b)
            u = [t.clone() for t in s["u"]]
            out, result = [torch.zeros(n, device="cuda") for n in sizes], pkg.hp_cuda_grad_result()
            pkg.hp_cuda_grad_clip(fresh, sizes, out, 0.5, result)
            pkg.hp_cuda_gd_momentum(fresh, sizes, u, None, 0.5, 0.5, result)
            pkg.hp_cuda_gd_mask([s["msg"]], [28], u[1:2], [17])
            wants.append((out, u, result))
        torch.cuda.synchronize()
        for s, stream in zip(sets, others):
            with torch.cuda.stream(stream):
                s["graph"].replay()
        torch.cuda.synchronize()
        for s, (out, u, result) in zip(sets, wants):
            assert torch.equal(s["result"][:3], result[:3])
            assert all(torch.equal(x, y) for x, y in zip(s["out"], out)) and all(torch.equal(x, y) for x, y in zip(s["u"], u))
        assert math.isfinite(float(torch.randn(1 << 20, device="cuda").sum()))


def test_calls_from_several_threads(pkg):
    # each thread with a stream, a result block and tensors of its own
    import threading
    sizes, types = [200_001, 33, 5000], ["bf16", "fp32", "fp16"]
    jobs = []
    for k in range(4):
        g, _ = make(sizes, types, 60 + k)
        norm = math.sqrt(squares(g))
        jobs.append((g, norm, [torch.zeros(n, device="cuda") for n in sizes], [torch.zeros(n, device="cuda") for n in sizes],
                     pkg.hp_cuda_grad_result(), torch.cuda.Stream()))
    torch.cuda.synchronize()
    failed = []

    def work(g, norm, out, u, result, stream):
        try:
            with torch.cuda.stream(stream):
                for _ in range(50):
                    pkg.hp_cuda_grad_clip(g, sizes, out, 0.5 * norm, result)
                    pkg.hp_cuda_grad_norm(g, sizes, result)
                    pkg.hp_cuda_gd_momentum(g, sizes, u, None, 0.0, 0.5 * norm, result)
                stream.synchronize()
        except Exception as e:
            failed.append(e)

    threads = [threading.Thread(target=work, args=j) for j in jobs]
    for t in threads: t.start()
    for t in threads: t.join()
    assert not failed
    for g, norm, out, u, result, _ in jobs:
        c = coefficient(norm, 0.5 * norm)
        for x, o, v in zip(g, out, u):
            near(o, c * f64(x), "fp32", np.abs(c * f64(x)) * 2.0 ** -24 * (1 + 1e-6))
            assert torch.equal(o, v)


def test_more_elements_than_32_bits_count(pkg):
    n = (1 << 31) + 4099
    if torch.cuda.mem_get_info()[0] < 8 * n:
        pytest.skip("not enough device memory")
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    places = [0, 1, (1 << 31) - 1, 1 << 31, n - 4099, n - 1]
    held = {at: float(k + 1) for k, at in enumerate(places)}  # n - 4099 is 2^31 again: five places
    for at, v in held.items():
        g[at] = v
    result = pkg.hp_cuda_grad_result()
    pkg.hp_cuda_grad_norm([g], [n], result)
    assert result[0].item() == 1 + 4 + 9 + 25 + 36
    pkg.hp_cuda_grad_norm([g], [n], result, 0)
    assert result[0].item() == 6
    pkg.hp_cuda_grad_clip([g], [n], None, 3.0, result, 1, 0)   # c = 3 / (6 + 1e-6): the halves are exact in bf16
    assert {at: g[at].item() for at in places} == {at: 0.5 * v for at, v in held.items()}
    assert int((g != 0).sum()) == 5
    # the gradient in halves, a momentum for each: offsets beyond 2^32 bytes
    h = n // 2
    u = torch.ones(h, device="cuda")
    pkg.hp_cuda_gd_momentum([g[:h]], [h], [u], None, 0.5, 1.0, None)
    assert u[0].item() == 1.0 and u[1].item() == 1.5 and u[h - 1].item() == 0.5 and int((u != 0.5).sum()) == 2
