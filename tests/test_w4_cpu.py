"""CPU: the 4-bit matrix-vector product's argument checks (C ABI and Python),
which return before any device work, and its layer method's loading rules."""
import ctypes as C
import importlib

import pytest
import torch

INVALID = 1  # cudaErrorInvalidValue


def _pointers(count, base=1 << 30):
    return [C.c_void_p(base + (i << 26)) for i in range(count)]


@pytest.mark.parametrize('n,k,group,ok', [
    (1, 32, 32, True), (2048, 512, 128, True), (17, 96, 32, True), (1 << 22, 256, 256, True), (16, 16384, 64, True),
    (0, 128, 128, False), ((1 << 22) + 1, 128, 128, False), (16, 0, 32, False), (16, 16416, 32, False),
    (16, 160, 64, False), (16, 128, 16, False), (16, 128, 48, False), (-16, 128, 128, False)])
def test_shapes(native, n, k, group, ok):
    lib = native.lib()
    x, tiles, scales, out, flags = _pointers(5)
    # M == 0 returns success after the shape test alone
    want = 0 if ok else INVALID
    assert lib.ornith_moe_b200_w4_launch(None, 0, 0, None, None, 0, None, None, 0, None, 0, n, k, group, None) == want
    if ok:
        tile_shape, scale_shape, zero_shape = native.w4_pack_shapes(n, k, group)
        assert tile_shape[0] * 16 >= n and tile_shape[1] * 64 >= k and scale_shape[1] * group == k
        assert zero_shape[2] == scale_shape[2] == 16
    else:
        with pytest.raises(ValueError):
            native.w4_pack_shapes(n, k, group)


def test_launch_refusals(native):
    fn = native.lib().ornith_moe_b200_w4_launch
    x, tiles, scales, zeros, out, flags = _pointers(6)

    def call(x=x, stride=256, x_type=0, tiles=tiles, scales=scales, scale_type=0, zeros=zeros, out=out, out_type=0,
             flags=flags, m=2, n=64, k=256, group=64):
        return fn(x, stride, x_type, tiles, scales, scale_type, zeros, out, out_type, flags, m, n, k, group, None)

    assert call(m=17) == INVALID and call(m=-1) == INVALID
    assert call(x_type=2) == INVALID and call(x_type=-1) == INVALID       # fp32 activations
    assert call(x_type=0, out_type=1) == INVALID                          # bf16 in, fp16 out
    assert call(out_type=3) == INVALID and call(scale_type=2) == INVALID
    assert call(stride=248) == INVALID and call(stride=260) == INVALID    # overlapping rows, rows off 16 bytes
    for missing in ('x', 'tiles', 'scales', 'out', 'flags'):
        assert call(**{missing: None}) == INVALID, missing
    assert call(x=C.c_void_p(x.value + 8)) == INVALID
    assert call(tiles=C.c_void_p(tiles.value + 8)) == INVALID
    assert call(out=C.c_void_p(out.value + 2), out_type=2) == INVALID
    assert call(out=x) == INVALID and call(flags=out) == INVALID and call(out=zeros) == INVALID


def test_pack_refusals(native):
    fn = native.lib().ornith_moe_b200_w4_pack
    codes, scales, zeros, tiles, ts, tz = _pointers(6)
    assert fn(codes, scales, zeros, tiles, ts, None, 64, 256, 64, None) == INVALID   # zeros without a place
    assert fn(codes, scales, None, tiles, ts, tz, 64, 256, 64, None) == INVALID
    assert fn(codes, scales, None, codes, ts, None, 64, 256, 64, None) == INVALID    # in place
    assert fn(codes, scales, zeros, tiles, ts, ts, 64, 256, 64, None) == INVALID
    assert fn(codes, scales, zeros, tiles, ts, tz, 64, 256, 100, None) == INVALID
    assert fn(None, scales, zeros, tiles, ts, tz, 64, 256, 64, None) == INVALID


def test_python_refuses_cpu_tensors(native):
    codes = torch.zeros((16, 16), dtype=torch.int32).view(torch.uint32)
    scales = torch.ones((16, 1), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        native.w4_pack(codes, scales)
    with pytest.raises(ValueError):
        native.w4_launch(torch.zeros((1, 128), dtype=torch.bfloat16), codes, scales, None,
                         torch.zeros((1, 16), dtype=torch.bfloat16), torch.zeros(1, dtype=torch.int32), 16, 128)


def test_method_geometry_and_loading():
    method = importlib.import_module('ornith_b200.method')
    for bad in (dict(dtype=torch.float32), dict(k=200), dict(group=100), dict(has_bias=True), dict(split=2)):
        layer = torch.nn.Module()
        layer.has_bias = bad.get('has_bias', False)
        k, n = bad.get('k', 256), 48
        m = method.W4LinearMethod('layer', group=bad.get('group', 64))
        with pytest.raises(ValueError):
            m.create_weights(layer, k // bad.get('split', 1), [n], k, n, bad.get('dtype', torch.bfloat16))
    for zero_points in (False, True):
        layer = torch.nn.Module()
        m = method.W4LinearMethod('layer', group=64, zero_points=zero_points)
        m.create_weights(layer, 256, [16, 32], 256, 48, torch.bfloat16)
        assert layer.w4_codes.shape == (48, 32) and layer.w4_scales.shape == (48, 4)
        assert hasattr(layer, 'w4_zeros') == zero_points
        with pytest.raises(ValueError):
            m.process_weights_after_loading(layer)          # nothing loaded
        with pytest.raises(ValueError):
            layer.w4_scales.weight_loader(layer.w4_scales, torch.ones((48, 4)))   # another dtype
        with pytest.raises(RuntimeError):
            m.apply(layer, torch.zeros((1, 256), dtype=torch.bfloat16))


def test_sealing_twice_and_after_a_refusal(monkeypatch):
    """A second call of process_weights_after_loading leaves a sealed layer as it is (as for the G256 methods); a
    weight that the layout refuses leaves the layer unsealed and its parameters in place."""
    method = importlib.import_module('ornith_b200.method')
    layer = torch.nn.Module()
    m = method.W4LinearMethod('layer', group=64)
    m.create_weights(layer, 256, [48], 256, 48, torch.bfloat16)
    layer.w4_codes.weight_loader(layer.w4_codes, torch.zeros((48, 32), dtype=torch.uint32))
    layer.w4_scales.weight_loader(layer.w4_scales, torch.ones((48, 4), dtype=torch.bfloat16))

    def refuse(*checkpoint):
        raise ValueError('scales must be finite')

    monkeypatch.setattr(method.native, 'w4_pack', refuse)
    with pytest.raises(ValueError):
        m.process_weights_after_loading(layer)
    assert not layer._g256_ready and hasattr(layer, 'w4_codes')
    packed = []
    monkeypatch.setattr(method.native, 'w4_pack', lambda *checkpoint: packed.append(checkpoint) or ('tiles', 'scales', None))
    m.process_weights_after_loading(layer)
    assert layer._g256_ready and not hasattr(layer, 'w4_codes')
    m.process_weights_after_loading(layer)
    assert layer._g256_ready and layer.w4_bank == ('tiles', 'scales', None) and len(packed) == 1
