"""The gradient operators on tensors of more elements than a launch or a part of a table takes.  Coefficients are 0.5 and values
small multiples of powers of two, so every result is exact."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

CHUNK = 1 << 30


def room_for(nbytes):
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < nbytes + (8 << 30):
        pytest.skip("not enough device memory")


def is_all(t, value, places):
    """Whether t holds `value` everywhere but at `places` (a dict), which it holds the values of."""
    for at, v in places.items():
        assert t[at].item() == v, (at, t[at].item(), v)
        t[at] = value
    for at in range(0, t.numel(), CHUNK):
        lo, hi = (x.item() for x in torch.aminmax(t[at:at + CHUNK]))
        assert lo == hi == value, (at, lo, hi)


def test_clip_of_more_tiles_than_a_launch_has_workgroups(pkg):
    # 2^35 elements are 2^24 tiles of 2048; with 256 lanes each that would be a launch of 2^32 lanes, which are counted in 32 bits
    n = (1 << 35) + 4099
    room_for(4 * n)
    g = torch.full((n,), 1.0, device="cuda")
    places = {0: 4.0, (1 << 32) - 1: 8.0, 1 << 32: 16.0, (1 << 35) - 1: 32.0, 1 << 35: 64.0, n - 1: 128.0}
    for at, v in places.items():
        g[at] = v
    result = pkg.hp_cuda_grad_result()
    pkg.hp_cuda_grad_clip([g], [n], [g], math.inf, result, is_measured=1, scale=0.5)
    is_all(g, 0.5, {at: 0.5 * v for at, v in places.items()})
    assert result[:3].tolist() == [0.0, 0.0, 0.5]


@pytest.mark.parametrize("lead", [0, 3])
def test_tensors_of_more_than_a_part(pkg, lead):
    n, guard = (1 << 32) + 4099, 64
    room_for(2 * n + 8 * n)
    room = 2 * guard + lead + n
    inside = slice(guard + lead, guard + lead + n)
    places = {0: 4.0, (1 << 32) - 2: 8.0, (1 << 32) - 1: 16.0, 1 << 32: 32.0, (1 << 32) + 1: 64.0, n - 1: 128.0}
    halves = {at: 0.5 * v for at, v in places.items()}

    def filled(dtype, value, at=None):
        b = torch.full((room,), 77.0, dtype=dtype, device="cuda")
        b[inside] = value
        for k, v in (at or {}).items():
            b[guard + lead + k] = v
        return b, b[inside]

    def intact(*buffers):
        for b in buffers:
            assert bool((b[:guard + lead] == 77).all()) and bool((b[guard + lead + n:] == 77).all())

    result = pkg.hp_cuda_grad_result()
    gb, g = filled(torch.bfloat16, 1.0, places)
    ob, out = filled(torch.float32, 5.0)
    small = torch.full((5,), 2.0, device="cuda"), torch.zeros(5, device="cuda")
    pkg.hp_cuda_grad_clip([g, small[0]], [n, 5], [out, small[1]], math.inf, result, is_measured=1, scale=0.5)
    is_all(out, 0.5, halves)
    assert small[1].tolist() == [1.0] * 5
    ub, u = ob, out  # u = 0.5 u + 0.5 g, with u all 0.5 again
    db, d = filled(torch.float32, 5.0)
    pkg.hp_cuda_gd_momentum([small[0], g], [5, n], [small[1], u], [torch.zeros(5, device="cuda"), d], 0.5, 1.0, None, scale=0.5)
    is_all(u, 0.75, {at: 0.25 + h for at, h in halves.items()})
    is_all(d, 0.875, {at: 0.5 * (0.25 + h) + h for at, h in halves.items()})
    pkg.hp_cuda_gd_momentum([g], [n], [d], None, 0.0, 1.0, None, scale=0.5)
    is_all(d, 0.5, halves)
    pkg.hp_cuda_grad_clip([g], [n], None, math.inf, result, is_measured=1, scale=0.5)
    is_all(g, 0.5, halves)
    intact(gb, ob, db)
