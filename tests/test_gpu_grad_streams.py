"""The gradient operators on lists that the caches do not hold: dense data over every tile of the streaming loops, in each type,
with tensors that begin at odd elements.

The norm's data are whole numbers, so the sum of their squares is exact in fp64 whatever the order: a tile that is left out or
taken twice, or one element of it, changes it.  Clipped elements are compared with the product in 64 bits: the coefficient and
the product are rounded to fp32 (2^-24 each), a result in 16 bits once more (2^-8 in bf16, 2^-11 in fp16; below fp16's
normal range by half of its smallest value, 2^-25).  Sums that torch and we take in fp64 are off by n 2^-53 of the sum each, their
roots and the coefficients by half as much."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
HALF = {"fp32": 2.0 ** -24, "bf16": 2.0 ** -8, "fp16": 2.0 ** -11}
GUARD = 64
CHUNK = 1 << 24


def types_of(kind, sizes):
    return [("bf16", "fp32", "fp16")[i % 3] if kind == "mixed" else kind for i in range(len(sizes))]


def make(sizes, types, lead, value=None):
    """(views, buffers): GUARD elements of 77 on both sides, `lead` more before."""
    views, buffers = [], []
    for n, t in zip(sizes, types):
        b = torch.full((2 * GUARD + lead + n,), 77.0, dtype=TYPES[t], device="cuda")
        views.append(b[GUARD + lead:GUARD + lead + n])
        if value is not None:
            views[-1].fill_(value)
        buffers.append(b)
    return views, buffers


def intact(buffers, views):
    for b, v in zip(buffers, views):
        at = v.storage_offset()
        assert bool((b[:at] == 77).all()) and bool((b[at + v.numel():] == 77).all())


def chunks(*ts):
    for at in range(0, ts[0].numel(), CHUNK):
        yield [t[at:at + CHUNK].double() for t in ts]


@pytest.mark.parametrize("lead", [0, 1])
@pytest.mark.parametrize("kind", ["fp32", "bf16", "fp16", "mixed"])
def test_norm_of_lists_beyond_the_cache(pkg, kind, lead):
    # 380 MB: the last 192 MiB (6144 tiles of 32 KiB) are loaded one way and what lies before another; the border lies within the
    # second tensor, or for the mixed list the third
    sizes = [30_000_001, 25_000_003, 777, 40_000_005, 5]
    if kind != "fp32":
        sizes = [2 * n + 1 for n in sizes]
    if kind == "mixed":
        sizes = [30_000_001, 25_000_003, 60_000_001, 40_000_005, 5_000_001]
    types = types_of(kind, sizes)
    gen = torch.Generator(device="cuda").manual_seed(5)
    g, b = make(sizes, types, lead)
    for t in g:
        for at in range(0, t.numel(), CHUNK):
            part = t[at:at + CHUNK]
            part.copy_(torch.randint(-3, 4, (part.numel(),), generator=gen, device="cuda", dtype=torch.int32))
    want = sum(int(x.square().sum().item()) for t in g for (x,) in chunks(t))
    result = pkg.hp_cuda_grad_result()
    pkg.hp_cuda_grad_norm(g, sizes, result)
    assert result[0].item() == want and abs(result[1].item() / math.sqrt(want) - 1) <= 2.0 ** -52
    assert result[3:16].tolist() == [0.0] * 13
    # the largest magnitude, wherever it lies
    for k, t in enumerate(g):
        for at in {0, t.numel() // 3, t.numel() // 2, t.numel() - 1}:
            held = t[at].item()
            t[at] = -9.0
            pkg.hp_cuda_grad_norm(g, sizes, result, 0)
            assert result[:2].tolist() == [9.0, 9.0], (k, at)
            t[at] = held
    intact(b, g)


# 60 M elements: the clipping pass joins the partial sums itself; 150 M are more than 65536 tiles, and the norm joins them.  All of
# them are more than 96 MiB, and loads stream.
@pytest.mark.parametrize("lead, out_lead", [(0, 0), (1, 3)])
@pytest.mark.parametrize("kind, sizes", [
    ("bf16", [40_000_001, 70_001, 5, 20_000_003]),
    ("fp16", [40_000_001, 70_001, 5, 20_000_003]),
    ("mixed", [40_000_001, 70_001, 5, 20_000_003]),
    ("fp32", [90_000_001, 70_001, 5, 60_000_003]),
    ("bf16", [90_000_001, 70_001, 5, 60_000_003]),
    ("fp16", [90_000_001, 70_001, 5, 60_000_003]),
    ("mixed", [70_000_001, 60_000_003, 20_000_001, 5]),
])
def test_clip_of_lists_that_stream(pkg, kind, sizes, lead, out_lead):
    types = types_of(kind, sizes)
    gen = torch.Generator(device="cuda").manual_seed(6)
    g, b = make(sizes, types, lead)
    for t in g:
        t.normal_(0, 1e-2, generator=gen)
    total, n = math.fsum(x.square().sum().item() for t in g for (x,) in chunks(t)), sum(sizes)
    norm = math.sqrt(total)
    before = [t.clone() for t in g]
    out, ob = make(sizes, ["fp32"] * len(sizes), out_lead, 5.0)
    result = pkg.hp_cuda_grad_result()

    def told(c, scale):
        s, length, factor = result[:3].tolist()
        assert abs(s - total) <= 2 * n * 2.0 ** -53 * total
        assert abs(length / (abs(scale) * norm) - 1) <= (n + 4) * 2.0 ** -53
        assert abs(factor - c) <= abs(c) * (2.0 ** -24 + 2 * n * 2.0 ** -53)

    def compare(got, ts, c):
        for x, y, t in zip(before, got, ts):
            for wide, seen in chunks(x, y):
                wide = c * wide
                tol = wide.abs() * (2.0 ** -23 + n * 2.0 ** -53 + (HALF[t] if t != "fp32" else 0.0)) * (1 + 2.0 ** -7) + 2.0 ** -25 * (t == "fp16")
                assert bool(((seen - wide).abs() <= tol).all())

    c = 0.3 * norm / (norm + 1e-6)
    pkg.hp_cuda_grad_clip(g, sizes, out, 0.3 * norm, result)
    told(c, 1.0)
    compare(out, ["fp32"] * len(sizes), c)
    intact(ob, out)
    intact(b, g)
    assert all(torch.equal(x, y) for x, y in zip(before, g))
    pkg.hp_cuda_grad_clip(g, sizes, None, math.inf, result, scale=-0.375)
    told(-0.375, -0.375)
    compare(g, types, -0.375)
    for x, y in zip(before, g):
        y.copy_(x)
    pkg.hp_cuda_grad_clip(g, sizes, None, 0.3 * norm, result)
    told(c, 1.0)
    compare(g, types, c)
    intact(b, g)
