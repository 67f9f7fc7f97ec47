"""GPU: the 4-bit matrix-vector product against its definition in 64 bits.

Tolerance.  Products x * (c - z) are exact in fp32, so the error of a result is
that of its sums: at most K/16 accumulations of the tensor core, K/32 scaled
joins, 8 joins of split sums, and 16 additions inside a tensor core step, each
taken as off by 2^-22 (two steps of fp32: the tensor core may truncate) of the
sum of magnitudes A = sum |x| |s (c - z)|, which bounds every partial sum.  The
store adds half a step of the output's type."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device('cuda:0')
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def make(n, k, group, zeros, dtype=BF16, scale_dtype=None, seed=0):
    gen = torch.Generator().manual_seed(seed + n * 7 + k)
    c = torch.randint(0, 16, (n, k), generator=gen)
    z = torch.randint(0, 16, (n, k // group), generator=gen) if zeros else None
    s = (0.02 * torch.randn((n, k // group), generator=gen)).to(scale_dtype or dtype)  # either sign
    words = sum(c[:, d::8] << (4 * d) for d in range(8))
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
    weight = (c.view(n, k // group, group) - (8 if z is None else z[:, :, None])).double() * s.double()[:, :, None]
    return (words.to(DEV).view(torch.uint32), s.to(DEV), None if z is None else z.to(torch.uint8).to(DEV),
            weight.view(n, k))


def rows(m, k, dtype, seed=1, pad=0):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn((m, k + pad), generator=gen).to(dtype).to(DEV)[:, :k]


def check(out, x, weight):
    k = x.shape[1]
    x64 = x.double().cpu()
    want, size = x64 @ weight.t(), x64.abs() @ weight.abs().t()
    steps = k // 16 + k // 32 + 8 + 16
    tol = steps * 2.0 ** -22 * size + torch.finfo(out.dtype).eps / 2 * want.abs() + torch.finfo(out.dtype).tiny
    err = (out.double().cpu() - want).abs()
    assert bool((err <= tol).all()), f'off by {(err / tol).max():.3g} of the bound'


def run(native, x, bank, n, out_dtype=None, flags=None):
    out = torch.full((x.shape[0], n), float('nan'), dtype=out_dtype or x.dtype, device=DEV)
    flags = torch.zeros(1, dtype=torch.int32, device=DEV) if flags is None else flags
    native.w4_launch(x, *bank, out, flags, n, x.shape[1])
    return out, flags


@pytest.mark.parametrize('k,group', [(32, 32), (64, 32), (96, 32), (64, 64), (192, 64), (128, 128), (640, 128),
                                     (256, 256), (2048, 128), (1056, 32), (4352, 256), (16384, 64)])
@pytest.mark.parametrize('n', [1, 15, 16, 17, 250])
def test_sizes(native, n, k, group):
    for zeros, m, dtype in ((False, 1, BF16), (True, 5, FP16), (True, 16, BF16)):
        codes, scales, z, weight = make(n, k, group, zeros, dtype)
        x = rows(m, k, dtype)
        out, flags = run(native, x, native.w4_pack(codes, scales, z), n)
        check(out, x, weight)
        assert int(flags) == 0


@pytest.mark.parametrize('m', range(1, 17))
def test_row_counts(native, m):
    n, k, group = 83, 512, 64
    codes, scales, z, weight = make(n, k, group, True, FP16)
    bank = native.w4_pack(codes, scales, z)
    x = rows(m, k, FP16)
    out, _ = run(native, x, bank, n)
    check(out, x, weight)
    # a row's result does not depend on the rows beside it (one and two tiles of eight rows apart)
    alone, _ = run(native, x[m - 1:], bank, n)
    assert torch.equal(alone[0], out[m - 1])


@pytest.mark.parametrize('n,k', [(2048, 512), (5003, 2048), (40000, 256)])
@pytest.mark.parametrize('out_dtype', [BF16, FP32])
def test_many_rows_of_n(native, n, k, out_dtype):
    """Sizes at which one, two, four and eight warps share a row tile."""
    codes, scales, z, weight = make(n, k, 128, True)
    x = rows(3, k, BF16)
    out, _ = run(native, x, native.w4_pack(codes, scales, z), n, out_dtype)
    check(out, x, weight)


@pytest.mark.parametrize('dtype,scale_dtype,out_dtype', [(BF16, FP16, BF16), (FP16, BF16, FP32), (FP16, FP16, FP16)])
def test_types(native, dtype, scale_dtype, out_dtype):
    codes, scales, z, weight = make(100, 256, 64, True, dtype, scale_dtype)
    x = rows(9, 256, dtype)
    out, _ = run(native, x, native.w4_pack(codes, scales, z), 100, out_dtype)
    check(out, x, weight)


def test_strided_rows_and_untouched_memory(native):
    n, k = 37, 96
    codes, scales, z, weight = make(n, k, 32, True)
    bank = native.w4_pack(codes, scales, z)
    x = rows(4, k, BF16, pad=40)
    assert x.stride(0) == k + 40
    around = torch.full((6, n), 7.0, dtype=BF16, device=DEV)
    flags = torch.zeros(1, dtype=torch.int32, device=DEV)
    native.w4_launch(x, *bank, around[1:5], flags, n, k)
    check(around[1:5], x, weight)
    assert bool((around[0] == 7).all()) and bool((around[5] == 7).all())
    nothing = around[:0]
    native.w4_launch(x[:0], *bank, nothing, flags, n, k)   # no rows: nothing happens
    assert int(flags) == 0


def test_offsets_past_32_bits(native):
    """A weight of 8 GiB, and rows of x further apart than 2^32 bytes."""
    n, k, group, gen = 1 << 20, 16384, 256, torch.Generator(device=DEV).manual_seed(5)
    codes = torch.randint(-2 ** 31, 2 ** 31, (n, k // 8), dtype=torch.int32, device=DEV, generator=gen)
    scales = (0.02 * torch.randn((n, k // group), device=DEV, generator=gen)).to(BF16)
    bank = native.w4_pack(codes.view(torch.uint32), scales)
    at = torch.tensor([0, 17, 2 ** 19 - 1, 2 ** 19, 2 ** 19 + 33, n - 300, n - 16, n - 1], device=DEV)
    c = torch.stack([(codes[at].long() >> (4 * d)) & 15 for d in range(8)], dim=2).view(len(at), k)
    weight = ((c.view(len(at), -1, group) - 8).double() * scales[at].double()[:, :, None]).view(len(at), k).cpu()
    del codes
    stride = 2 ** 31 + 8
    x = torch.empty(2 * stride + k, dtype=BF16, device=DEV).as_strided((3, k), (stride, 1))
    x.copy_(rows(3, k, BF16))
    out, flags = run(native, x, bank, n, FP32)
    check(out[:, at], x, weight)
    assert int(flags) == 0


def test_extreme_codes_and_scales(native):
    """Codes 0 and 15 against zero points 15 and 0, scales at both ends."""
    n, k = 32, 64
    words = torch.full((n, k // 8), -1, dtype=torch.int32, device=DEV)
    words[::2] = 0
    z = torch.zeros((n, 1), dtype=torch.uint8, device=DEV)
    z[::2] = 15
    s = torch.full((n, 1), 2.0 ** -14, dtype=FP16, device=DEV)
    s[:, 0] = torch.where(torch.arange(n, device=DEV) % 4 < 2, 2.0 ** -14, 100.0)
    x = rows(2, k, FP16)
    c = torch.where(torch.arange(n)[:, None] % 2 == 1, 15.0, 0.0).double().expand(n, k)
    weight = (c - z.cpu().double()) * s.cpu().double()
    out, flags = run(native, x, native.w4_pack(words.view(torch.uint32), s, z), n, FP32)
    check(out, x, weight)
    assert int(flags) == 0


def test_nonfinite_values_stay_in_their_row(native):
    n, k = 20, 128
    codes, scales, z, weight = make(n, k, 64, False, FP16)
    bank = native.w4_pack(codes, scales, z)
    x = rows(3, k, FP16)
    x[1, 5] = float('inf')
    out, flags = run(native, x, bank, n)
    assert int(flags) == 4 | 8 and not bool(torch.isfinite(out[1]).any())
    check(out[::2], x[::2], weight)
    x[1, 5] = 0
    x[2] *= 60000.0 / x[2].abs().max()
    big = native.w4_pack(codes, torch.full_like(scales, 100.0), z)
    out, flags = run(native, x, big, n)
    assert int(flags) == 8 and bool(torch.isinf(out[2]).any())     # overflow of fp16 alone
    out, flags = run(native, x, big, n, FP32)
    assert int(flags) == 0 and bool(torch.isfinite(out).all())


def test_capture_replay_and_streams(native):
    n, k = 333, 1024
    codes, scales, z, weight = make(n, k, 128, True)
    bank = native.w4_pack(codes, scales, z)
    x = rows(2, k, BF16)
    out = torch.zeros((2, n), dtype=BF16, device=DEV)
    flags = torch.zeros(1, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        native.w4_launch(x, *bank, out, flags, n, k)
    torch.cuda.current_stream().wait_stream(side)
    check(out, x, weight)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        native.w4_out(x, *bank, out, flags, n, k)
    x.copy_(rows(2, k, BF16, seed=9))
    out.zero_()
    graph.replay()
    check(out, x, weight)


def test_refusals(native):
    n, k = 48, 128
    codes, scales, z, _ = make(n, k, 64, True)
    bank = native.w4_pack(codes, scales, z)
    x = rows(2, k, BF16)
    out = torch.zeros((2, n), dtype=BF16, device=DEV)
    flags = torch.zeros(1, dtype=torch.int32, device=DEV)
    good = dict(x=x, tiles=bank[0], scales=bank[1], zeros=bank[2], out=out, flags=flags, n=n, k=k)
    native.w4_launch(**good)
    bad = [dict(x=rows(17, k, BF16)), dict(x=x.float()), dict(x=rows(2, k, BF16, pad=4)), dict(x=x[:, :64]),
           dict(x=x.t()), dict(x=x.cpu()), dict(x=rows(3, k, BF16)), dict(x=x.to(FP16)),
           dict(x=x[:1].expand(2, k)), dict(x=rows(1, k + 8, BF16)[:, 1:k + 1]),
           dict(out=out.to(FP16)), dict(out=torch.zeros((n, 2), dtype=BF16, device=DEV).t()), dict(out=out[:, :40]),
           dict(tiles=bank[0][:1]), dict(tiles=bank[0].view(torch.int32)), dict(scales=bank[1].float()),
           dict(scales=bank[1][:, :1]), dict(zeros=bank[2][:1]), dict(zeros=bank[2].cpu()), dict(n=n + 16),
           dict(k=64), dict(flags=flags.long()), dict(flags=torch.zeros(2, dtype=torch.int32, device=DEV))]
    for change in bad:
        with pytest.raises(ValueError):
            native.w4_launch(**{**good, **change})
    for change in (dict(codes=codes.view(torch.int32)), dict(codes=codes[:, ::2]), dict(scales=scales.float()),
                   dict(scales=scales[:40]), dict(zeros=z[:, :1]), dict(zeros=z.int()), dict(zeros=z + 16),
                   dict(scales=scales * float('inf')), dict(scales=scales.cpu())):
        with pytest.raises(ValueError):
            native.w4_pack(**{**dict(codes=codes, scales=scales, zeros=z), **change})


def test_layer_method(native):
    method = importlib.import_module('ornith_b200.method')
    runtime = importlib.import_module('ornith_b200.runtime')
    n, k = 200, 256
    codes, scales, z, weight = make(n, k, 64, True)
    rt = runtime.Runtime(['head'], 8, DEV)
    for fp32 in (False, True):
        layer = torch.nn.Module()
        m = method.W4LinearMethod('head', group=64, zero_points=True, logits_fp32=fp32)
        m.create_weights(layer, k, [n], k, n, BF16, device=DEV)
        for name, value in (('w4_codes', codes), ('w4_scales', scales), ('w4_zeros', z)):
            getattr(layer, name).weight_loader(getattr(layer, name), value)
        m.process_weights_after_loading(layer)
        assert not hasattr(layer, 'w4_codes')
        m.bind(rt, 0)
        x = rows(35, k, BF16)                                      # three slices of rows
        out = m.apply(layer, x.view(5, 7, k))
        assert out.shape == (5, 7, n) and out.dtype == (FP32 if fp32 else BF16)
        check(out.view(35, n), x, weight)
    assert rt.check_error_flags() == [0]


@pytest.mark.parametrize('group,k', [(32, 96), (64, 192), (128, 256), (256, 512)])
@pytest.mark.parametrize('zeros,dtype,scale_dtype', [(False, BF16, BF16), (True, FP16, FP16), (True, BF16, FP16),
                                                     (False, FP16, BF16)])
def test_two_row_tiles_a_warp(native, group, k, zeros, dtype, scale_dtype):
    """Weights wide enough for a warp to take two row tiles, the last set with one of its own, ragged."""
    n = 4736 * 16 + 9
    codes, scales, z, weight = make(n, k, group, zeros, dtype, scale_dtype)
    bank = native.w4_pack(codes, scales, z)
    for m, out_dtype in ((1, FP32), (8, dtype), (9, FP32), (16, dtype)):
        x = rows(m, k, dtype, seed=m)
        around = torch.full((m + 2, n), 7.0, dtype=out_dtype, device=DEV)
        flags = torch.zeros(1, dtype=torch.int32, device=DEV)
        native.w4_launch(x, *bank, around[1:-1], flags, n, k)
        check(around[1:-1], x, weight)
        assert bool((around[0] == 7).all()) and bool((around[-1] == 7).all()) and int(flags) == 0


@pytest.mark.parametrize('group', [32, 64, 128])
def test_two_warps_share_a_row_tile(native, group):
    n, k = 20000, 256
    codes, scales, z, weight = make(n, k, group, True)
    bank = native.w4_pack(codes, scales, z)
    for m in (1, 9):
        x = rows(m, k, BF16, seed=m)
        out, flags = run(native, x, bank, n)
        check(out, x, weight)
        assert int(flags) == 0


def test_layer_method_on_other_views(native):
    """No rows, one row of a wider tensor, and a batch whose rows lie apart."""
    method = importlib.import_module('ornith_b200.method')
    runtime = importlib.import_module('ornith_b200.runtime')
    n, k = 96, 128
    codes, scales, _, weight = make(n, k, 32, False)
    layer = torch.nn.Module()
    m = method.W4LinearMethod('layer', group=32)
    m.create_weights(layer, k, [n], k, n, BF16, device=DEV)
    layer.w4_codes.weight_loader(layer.w4_codes, codes)
    layer.w4_scales.weight_loader(layer.w4_scales, scales)
    m.process_weights_after_loading(layer)
    rt = runtime.Runtime(['layer'], 8, DEV)
    m.bind(rt, 0)
    assert m.apply(layer, torch.empty((0, k), dtype=BF16, device=DEV)).shape == (0, n)
    assert m.apply(layer, torch.empty((3, 0, k), dtype=BF16, device=DEV)).shape == (3, 0, n)
    wide = rows(24, 2 * k, BF16)
    check(m.apply(layer, wide[5, k:])[None], wide[5:6, k:], weight)
    check(m.apply(layer, wide[:, :k]), wide[:, :k], weight)
    check(m.apply(layer, wide.view(4, 6, 2 * k).transpose(0, 1)[:, 1:3, k:]).reshape(12, n),
          wide.view(4, 6, 2 * k).transpose(0, 1)[:, 1:3, k:].reshape(12, k), weight)
    with pytest.raises(ValueError):
        m.apply(layer, wide[:, :k].float())
    with pytest.raises(RuntimeError):
        m.apply(layer, wide[:, :k], bias=torch.zeros(n, device=DEV))
    assert rt.check_error_flags() == [0]
