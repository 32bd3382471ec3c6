"""What the gradient operators (global norm, clipping, momentum correction, momentum masking) refuse, before anything is launched:
no GPU is needed."""
import math

import pytest

A = 1 << 20  # an address that nothing is read from


def _norm(c, ptrs=(A,), sizes=(8,), types=None, order=2, result=A):
    return c.load().hpx_grad_norm(len(ptrs), c.ptr_array(ptrs), c.i64_array(sizes), None if types is None else c.i32_array(types), order, 0, result, None)


def _clip(c, ptrs=(A,), sizes=(8,), types=None, outs=None, order=2, max_norm=1.0, scale=1.0, result=A):
    return c.load().hpx_grad_clip(len(ptrs), c.ptr_array(ptrs), c.i64_array(sizes), None if types is None else c.i32_array(types),
                                  None if outs is None else c.ptr_array(outs), 0, order, max_norm, scale, result, None)


def _momentum(c, ptrs=(A,), sizes=(8,), types=None, us=(2 * A,), outs=None, m=0.9, order=2, max_norm=1.0, scale=1.0, result=A):
    return c.load().hpx_gd_momentum(len(ptrs), c.ptr_array(ptrs), c.i64_array(sizes), None if types is None else c.i32_array(types),
                                    c.ptr_array(us), None if outs is None else c.ptr_array(outs), m, order, max_norm, scale, result, None)


def _mask(c, ins=(A,), in_sizes=(20,), us=(2 * A,), sizes=(8,), counts=None):
    return c.load().hpx_gd_mask(len(ins), c.ptr_array(ins), c.i32_array(in_sizes), c.ptr_array(us), c.i32_array(sizes), counts, None)


@pytest.mark.parametrize("call", [_norm, _clip, _momentum])
@pytest.mark.parametrize("change, text", [
    (dict(sizes=(-1,)), "size -1"),
    (dict(sizes=(1 << 48,)), "size"),
    (dict(types=(3,)), "type 3"),
    (dict(types=(-1,)), "type -1"),
    (dict(ptrs=(0,)), "null pointer"),
    (dict(ptrs=(A + 2,)), "multiple of its element size"),
    (dict(ptrs=(A + 1,), types=(1,)), "multiple of its element size"),
    (dict(order=1), "order 1"),
    (dict(result=A + 4), "result block"),
])
def test_lists(capi, call, change, text):
    assert call(capi, **change) == -3
    assert text in capi.last_error()


def test_null_arguments(capi):
    L = capi.load()
    assert L.hpx_grad_norm(-1, None, None, None, 2, 0, A, None) == -3 and "negative count" in capi.last_error()
    assert L.hpx_grad_norm(1, None, None, None, 2, 0, A, None) == -3 and "null argument" in capi.last_error()
    assert L.hpx_grad_clip(1, None, None, None, None, 0, 2, 1.0, 1.0, A, None) == -3
    assert L.hpx_gd_momentum(1, None, None, None, None, None, 0.9, 2, 1.0, 1.0, A, None) == -3
    assert L.hpx_gd_mask(1, None, None, None, None, None, None) == -3
    assert L.hpx_gd_mask(0, None, None, None, None, None, None) == 0
    assert _norm(capi, result=None) == -3 and "result block" in capi.last_error()
    assert _clip(capi, result=None) == -3 and "result block" in capi.last_error()


@pytest.mark.parametrize("call", [_clip, _momentum])
@pytest.mark.parametrize("change, text", [
    (dict(max_norm=-1.0), "max_norm"),
    (dict(max_norm=math.nan), "max_norm"),
    (dict(scale=math.nan), "scale"),
    (dict(scale=math.inf), "scale"),
    (dict(scale=1e300), "scale"),
    (dict(outs=(0,)), "output 0"),
    (dict(outs=(4 * A + 2,)), "output 0"),
    (dict(types=(1,), outs=(A,)), "cannot take the place"),
])
def test_parameters(capi, call, change, text):
    assert call(capi, **change) == -3
    assert text in capi.last_error()


def test_momentum_parameters(capi):
    for m in (math.nan, math.inf):
        assert _momentum(capi, m=m) == -3 and "momentum" in capi.last_error()
    assert _momentum(capi, us=(0,)) == -3 and "momentum 0" in capi.last_error()
    assert _momentum(capi, us=(2 * A + 2,)) == -3 and "momentum 0" in capi.last_error()


def test_overlapping_tensors(capi):
    # in place: the same tensor twice, in either order of addresses, and a partial overlap
    for ptrs in ((A, A), (A + 16, A), (A, 2 * A, A + 28)):
        assert _clip(capi, ptrs=ptrs, sizes=(8,) * len(ptrs)) == -3 and "overlap" in capi.last_error()
    # bf16: eight elements are sixteen bytes
    assert _clip(capi, ptrs=(A, A + 14), sizes=(8, 8), types=(1, 1)) == -3
    # outputs that overlap each other, or a gradient that is not their own
    assert _clip(capi, ptrs=(A, 2 * A), sizes=(8, 8), outs=(4 * A, 4 * A + 28)) == -3
    assert _clip(capi, ptrs=(A, 2 * A), sizes=(8, 8), outs=(2 * A, 4 * A)) == -3 and "gradient 1" in capi.last_error()
    assert _clip(capi, ptrs=(A, 2 * A), sizes=(8, 8), outs=(A + 4, 4 * A)) == -3 and "gradient 0" in capi.last_error()
    assert _clip(capi, ptrs=(A, A), sizes=(8, 8), outs=(A, 4 * A)) == -3 and "gradient 1" in capi.last_error()
    assert _momentum(capi, us=(A,)) == -3
    assert _momentum(capi, us=(2 * A,), outs=(2 * A,)) == -3
    assert _momentum(capi, us=(2 * A,), outs=(2 * A + 28,)) == -3
    assert _momentum(capi, us=(A + 28,), outs=(4 * A,)) == -3


@pytest.mark.parametrize("at", [0, 8, 24, 2063 * 8])
def test_tensors_apart_from_the_result_block(capi, at):
    R = 16 * A
    for call, kinds in ((_norm, ("ptrs",)), (_clip, ("ptrs", "outs")), (_momentum, ("ptrs", "us", "outs"))):
        for kind in kinds:
            name = {"ptrs": "gradient", "us": "momentum", "outs": "output"}[kind]
            assert call(capi, result=R, **{kind: (R + at,)}) == -3 and f"{name} 0 overlaps the result block" in capi.last_error()
            # from below: eight elements whose last is the block's first
            assert call(capi, result=R, **{kind: (R - 28,)}) == -3 and f"{name} 0 overlaps the result block" in capi.last_error()
    assert _clip(capi, ptrs=(A, R + at), sizes=(8, 2), types=(0, 1), result=R) == -3 and "gradient 1 overlaps" in capi.last_error()


@pytest.mark.parametrize("change, text", [
    (dict(in_sizes=(-1,)), "negative size"),
    (dict(sizes=(-1,)), "negative size"),
    (dict(ins=(0,)), "message 0"),
    (dict(ins=(A + 2,)), "message 0"),
    (dict(us=(0,)), "momentum 0"),
    (dict(us=(2 * A + 1,)), "momentum 0"),
    (dict(counts=A + 2), "counts"),
])
def test_messages(capi, change, text):
    assert _mask(capi, **change) == -3
    assert text in capi.last_error()


def test_messages_and_counts_apart_from_what_is_written(capi):
    # a message of 20 bytes against momenta of 8 elements, whole and by its last or first word
    for ins, us in (((A,), (A,)), ((A,), (A + 16,)), ((A + 28,), (A,)), ((2 * A, 4 * A + 28), (8 * A, 4 * A))):
        n = len(ins)
        assert _mask(capi, ins=ins, in_sizes=(20,) * n, us=us, sizes=(8,) * n) == -3
        assert f"message {n - 1} overlaps a momentum" in capi.last_error()
    # momenta that overlap each other hide none of the first
    assert _mask(capi, ins=(A + 40, 4 * A), in_sizes=(20, 20), us=(A, A + 16), sizes=(64, 2)) == -3 and "message 0" in capi.last_error()
    assert _mask(capi, us=(2 * A,), counts=2 * A + 28) == -3 and "the counts overlap a momentum" in capi.last_error()
    assert _mask(capi, ins=(A, A + 64), in_sizes=(20, 20), us=(2 * A, 3 * A), sizes=(8, 8), counts=A - 4) == -3
    assert "the counts overlap message 0" in capi.last_error()
    assert _mask(capi, ins=(A, A + 64), in_sizes=(20, 20), us=(2 * A, 3 * A), sizes=(8, 8), counts=A + 80) == -3
    assert "the counts overlap message 1" in capi.last_error()


def test_sizes_that_their_type_does_not_hold(pkg):
    # none of them is its lower bits
    for size in ((1 << 64) + 8, 1 << 63, -(1 << 63) - 1):
        with pytest.raises(ValueError, match="sizes"):
            pkg.hp_cuda_grad_norm([A], [size], 2 * A, stream=0)
        with pytest.raises(ValueError, match="sizes"):
            pkg.hp_cuda_grad_clip([A], [size], None, 1.0, 2 * A, stream=0)
        with pytest.raises(ValueError, match="sizes"):
            pkg.hp_cuda_gd_momentum([A], [size], [4 * A], None, 0.9, 1.0, 2 * A, stream=0)
    for size in ((1 << 32) + 8, 1 << 31, -(1 << 31) - 1, (1 << 64) + 8):
        with pytest.raises(ValueError, match="sizes"):
            pkg.hp_cuda_gd_mask([A], [20], [2 * A], [size], stream=0)
        with pytest.raises(ValueError, match="in sizes"):
            pkg.hp_cuda_gd_mask([A], [size], [2 * A], [8], stream=0)
    for code in ((1 << 32) + 1, (1 << 64) + 1):
        with pytest.raises(ValueError, match="types"):
            pkg.hp_cuda_grad_norm([A], [8], 2 * A, types=[code], stream=0)


def test_result_block_is_on_the_device_that_is_named(pkg, monkeypatch):
    import torch
    asked = []
    monkeypatch.setattr(torch, "zeros", lambda *shape, dtype, device: asked.append((shape, dtype, device)))
    for device in (None, 0, 1, "cuda:1"):
        pkg.hp_cuda_grad_result(device)
    assert asked == [((2064,), torch.float64, d) for d in ("cuda", 0, 1, "cuda:1")]


def test_streams_of_another_device(pkg, monkeypatch):
    import torch

    class Stream:
        device_index, cuda_stream = 1, 0

    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    for call in (lambda s: pkg.hp_cuda_grad_norm([], [], A, stream=s), lambda s: pkg.hp_cuda_grad_clip([], [], None, 1.0, A, stream=s),
                 lambda s: pkg.hp_cuda_gd_momentum([], [], [], None, 0.9, 1.0, None, stream=s), lambda s: pkg.hp_cuda_gd_mask([], [], [], [], stream=s)):
        with pytest.raises(RuntimeError, match="one of device 1, the current device is 0"):
            call(Stream())


def test_python_functions_are_there(pkg):
    for name in ("hp_cuda_grad_result", "hp_cuda_grad_norm", "hp_cuda_grad_clip", "hp_cuda_gd_momentum", "hp_cuda_gd_mask"):
        assert callable(getattr(pkg, name)) and name in pkg.__all__
    assert pkg._capi.GRAD_RESULT == 2064
